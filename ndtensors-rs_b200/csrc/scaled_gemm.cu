// Products of block-scaled 8-bit matrices on the fifth-generation tensor cores.
//
//   C[i, j] = sum over kb of sa(i, kb) * sb(j, kb) * P_kb[i, j] (+ C[i, j])
//   P_kb[i, j] = sum over the 128 k of block kb of a[i, k] * b[j, k]
//
// The scales change every 128 k, so the tensor core sums one block at a time
// (four k = 32 steps of tcgen05.mma kind::f8f6f4, 32-bit accumulators in
// TMEM) and the epilogue warps multiply each P_kb by its scales and add it to
// accumulators in registers, in 32 bits.  Two TMEM buffers let the tensor
// core work on block kb + 1 meanwhile.
//
// Roles: warp 0 loads the operand tiles by TMA into a ring of 128-byte
// swizzled stages, 1 issues the MMAs, 2 loads the scales into a ring of its
// own (cp.async), 4 - 11 scale and sum (a thread holds one row and half the
// tile's columns).
//
// Two forms.  CTAS = 1: one CTA computes a 128 x BN tile; where there are few
// tiles a cluster of CTAs splits k and adds its parts through distributed
// shared memory, in rank order (no workspace, no atomics).  With few rows of A
// (a decoding batch) the operands trade places, so that B's rows fill the 128
// lanes and A's few the columns.  CTAS = 2: a CTA pair computes 256 x 256 with
// cta_group::2 MMAs, each CTA staging its half of both operands; persistent.
//
// Measured on one B200 (1 x 128 by 128 x 128 scales, bf16 result, L2 flushed):
// 4096^3 90 us = 1530 TFLOP/s, 8192^3 522 us = 2110; with a scale for each row of
// both 135 and 809 us.  Copies of the kernel, 4096^3 / 8192^3 in us: loads alone
// (a quarter of the MMAs, no TMEM reads) 61 / 318, loads and all MMAs 76 / 424,
// all 90 / 522, all but the loads (stages filled once) 90 / 502.  So the bound is
// not L2 but the way of a block's sums: MMAs, reads from TMEM, scales, the buffer
// given back, with two buffers to overlap them; a scale for each column as well
// is one more multiplication there for two values.  The tensor pipe is busy 45 %
// of the time.  One row against 10240 x 8192 weights: 19 us, 4.5 TB/s.
//
// sa * sb is formed in 32 bits: it stays finite while the product of two
// blocks' largest values is below 2^127, and has all its bits while that product
// is above 2^-108.
#include <algorithm>

#include "mbarrier.h"

namespace ndt {
namespace {

constexpr int kBK = 128;     // one scale block, one swizzled row
constexpr int kEpiWarp0 = 4;  // the epilogue is whole warpgroups (setmaxnreg)
constexpr int kSlots = 8;    // scale ring

struct GemmArgs {
  const float* sa;
  const float* sb;
  int64_t sa_rs, sa_cs, sb_rs, sb_cs;
  void* c;
  int64_t crs, ccs;  // strides of C's rows and columns (one of them is 1)
  int m, n, kblocks;
  int tiles_m, tiles_n;
  int ksplit;
  uint32_t idesc;
  int a_row, b_row;  // a scale for each row of A / B (else for each 128)
  int ctype;       // MType of C
  int accumulate;
  int vec;         // rows of C are contiguous and their 16-byte stores aligned
  int early_a;     // A was there before the kernel ahead in the stream: its first tiles need not wait for it
  int* flag;       // set when a bounded wait ran out
};

// ------------------------------------------------------------- PTX pieces
// In another CTA of the cluster.  (What it reports, that TMEM has been read, is
// ordered by the tcgen05 fences; a release at cluster scope would add a memory
// barrier to every k block.)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
template <int CTAS>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if constexpr (CTAS == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
  else  // bar is the leader's
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
        "[%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}

// K-major operand tile of 128-byte rows, 128-byte swizzle: 8-row groups are
// 1024 bytes apart.  (Start address, offsets in units of 16 bytes; bit 46 is
// the descriptor version of sm_100, 2 at bit 61 the 128-byte swizzle.)
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
template <int CTAS>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  if constexpr (CTAS == 1)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
// The barrier (of both CTAs of a pair) is arrived at when the MMAs issued so
// far are done.
template <int CTAS>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  if constexpr (CTAS == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}
// N columns of the warp's 32 lanes.
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t* r) {
  static_assert(N == 8 || N == 16 || N == 32, "columns of one load");
  if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
  if constexpr (N == 16)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
  if constexpr (N == 32)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Two 32-bit operations in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair(uint32_t a, uint32_t b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
// One 4-byte element into shared memory; zero where !valid.
__device__ __forceinline__ void cp4(uint32_t dst, const float* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}

__device__ __forceinline__ float load_c(const void* c, int64_t i, int type) {
  if (type == (int)MType::F32) return ((const float*)c)[i];
  if (type == (int)MType::BF16) return __bfloat162float(((const __nv_bfloat16*)c)[i]);
  return __half2float(((const __half*)c)[i]);
}
__device__ __forceinline__ void store_c(void* c, int64_t i, int type, float v) {
  if (type == (int)MType::F32)
    ((float*)c)[i] = v;
  else if (type == (int)MType::BF16)
    ((__nv_bfloat16*)c)[i] = __float2bfloat16_rn(v);
  else
    ((__half*)c)[i] = __float2half_rn(v);
}

// tile index -> (row tile, column tile): bands of 8 row tiles are walked
// column by column, so the tiles in flight share operand tiles in L2.
__device__ __forceinline__ void tile_at(int t, int tiles_m, int tiles_n, int& tm, int& tn) {
  constexpr int kBand = 8;
  const int band = t / (kBand * tiles_n), first = band * kBand;
  const int rows = min(kBand, tiles_m - first);
  const int in = t - band * kBand * tiles_n;
  tm = first + in % rows;
  tn = in / rows;
}

template <int CTAS, int BN>
struct Shape {
  static constexpr int kEpiWarps = 8;  // (16, with half the registers each, wait in each other's way: 86 -> 107 us for 4096^3)
  static constexpr int kBM = 128;                    // rows of one CTA
  static constexpr int kBRows = BN / CTAS;           // rows of B that one CTA stages
  static constexpr int kABytes = kBM * kBK, kBBytes = kBRows * kBK;
  static constexpr int kStage = kABytes + kBBytes;
  // narrow tiles leave room for two CTAs on an SM: twice the loads in flight
  static constexpr int kResident = BN <= 64 ? 2 : 1;
  static constexpr int kStages = (kResident == 2 ? 100 : 192) * 1024 / kStage;
  static constexpr int kScaleFloats = kBM + (BN + 31) / 32 * 32;  // a slot of the scale ring
  static constexpr int kTmemCols = 2 * BN;
  static constexpr int kCols = BN / (kEpiWarps / 4);  // columns of one epilogue thread
  static constexpr int kThreads = 32 * (kEpiWarp0 + kEpiWarps);
  // rows of C that vectors do not fit go through 32 x 16 values a warp, so that
  // its stores are runs of a row (wide tiles; narrow ones lie along C's columns).
  // 7080 x 2703 x 512, bf16 result, x quantised in the call: 211 -> 60 us.
  static constexpr int kTurn = BN >= 128 ? 32 * 17 : 0;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStage + ((size_t)kSlots * kScaleFloats + kEpiWarps * kTurn) * 4;
  static_assert(kTmemCols >= 32 && kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM columns");
  static_assert((size_t)BN * 129 * 4 <= (size_t)kStages * kStage || CTAS == 2, "the split's buffer reuses the stages");
  static_assert(kStage % 1024 == 0, "swizzled tiles start on 1024 bytes");
};

template <int CTAS, int BN, bool BROW>
__global__ void __launch_bounds__(Shape<CTAS, BN>::kThreads, Shape<CTAS, BN>::kResident)
    scaled_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                       const GemmArgs g) {
  using S = Shape<CTAS, BN>;
  constexpr int kCols = S::kCols, kThreads = S::kThreads, kEpiWarps = S::kEpiWarps;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t bars[2 * S::kStages + 2 * kSlots + 4];
  __shared__ uint32_t tmem_base_s;
  __shared__ int gave_up_s;
  const uint32_t stage0 = (smem_u32(raw) + 1023) & ~1023u;
  float* scale_ring = reinterpret_cast<float*>(raw + (stage0 - smem_u32(raw)) + (size_t)S::kStages * S::kStage);
  const uint32_t full = smem_u32(bars), empty = full + 8 * S::kStages, sfull = empty + 8 * S::kStages,
                 sempty = sfull + 8 * kSlots, tfull = sempty + 8 * kSlots, tempty = tfull + 16;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 2 ? cluster_rank() : 0;
  const bool clustered = CTAS == 2 || g.ksplit > 1;
  volatile int* gave_up = &gave_up_s;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kStages; i++) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < kSlots; i++) mbar_init(sfull + 8 * i, 32), mbar_init(sempty + 8 * i, kEpiWarps);
    for (int i = 0; i < 2; i++) mbar_init(tfull + 8 * i, 1), mbar_init(tempty + 8 * i, CTAS * kEpiWarps);
    gave_up_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    const uint32_t where = smem_u32(&tmem_base_s);
    if constexpr (CTAS == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "n"(S::kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(where), "n"(S::kTmemCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
  }
  fence_before();
  __syncthreads();
  if (clustered) cluster_sync();
  fence_after();
  const uint32_t tmem = tmem_base_s;
  pdl_release();
  if (CTAS == 2 || !g.early_a || warp != 0) pdl_wait();

  const int split = CTAS == 1 && g.ksplit > 1 ? (int)cluster_rank() : 0;
  const int unit = CTAS == 1 ? blockIdx.x / g.ksplit : blockIdx.x / 2;
  const int units = CTAS == 1 ? gridDim.x / g.ksplit : gridDim.x / 2;
  const int ntiles = g.tiles_m * g.tiles_n;
  const int kb0 = CTAS == 1 ? (int)((int64_t)g.kblocks * split / g.ksplit) : 0;
  const int kb1 = CTAS == 1 ? (int)((int64_t)g.kblocks * (split + 1) / g.ksplit) : g.kblocks;

  // wide tiles: the block's 384 x 168 registers, 40 a thread for the loading
  // warpgroup and 232 for the two that sum (40 x 128 + 232 x 256 is their sum)
  auto fewer = [] { if (BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;"); };
  auto more = [] { if (BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;"); };
  if (warp == 0) {
    fewer();
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      int ahead = 0;  // stages whose A is on its way already
      if (CTAS == 1 && g.early_a) {
        int tm, tn;
        tile_at(unit, g.tiles_m, g.tiles_n, tm, tn);
        for (; ahead < S::kStages && kb0 + ahead < kb1; ahead++) {
          mbar_expect_tx(full + 8 * ahead, S::kStage);
          tma_load<CTAS>(stage0 + ahead * S::kStage, &map_a, full + 8 * ahead, (kb0 + ahead) * kBK, tm * 128);
        }
        pdl_wait();
      }
      for (int t = unit; t < ntiles && ok; t += units) {
        int tm, tn;
        tile_at(t, g.tiles_m, g.tiles_n, tm, tn);
        const int row_a = tm * 128 * CTAS + rank * 128, row_b = tn * BN + rank * S::kBRows;
        for (int kb = kb0; kb < kb1; kb++) {
          if (ahead > 0) {
            ahead--;
            tma_load<CTAS>(stage0 + stage * S::kStage + S::kABytes, &map_b, full + 8 * stage, kb * kBK, row_b);
            if (++stage == S::kStages) stage = 0, phase ^= 1;
            continue;
          }
          if (!(ok = mbar_wait(empty + 8 * stage, phase ^ 1, gave_up, g.flag))) break;
          const uint32_t dst = stage0 + stage * S::kStage;
          uint32_t bar = full + 8 * stage;
          if (rank == 0) mbar_expect_tx(bar, CTAS * S::kStage);
          if (CTAS == 2) bar = mapa(bar, 0);
          tma_load<CTAS>(dst, &map_a, bar, kb * kBK, row_a);
          tma_load<CTAS>(dst + S::kABytes, &map_b, bar, kb * kBK, row_b);
          if (++stage == S::kStages) stage = 0, phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    fewer();
    if (rank == 0 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      uint32_t it = 0;  // k blocks so far: TMEM buffer it & 1
      bool ok = true;
      for (int t = unit; t < ntiles && ok; t += units) {
        for (int kb = kb0; kb < kb1; kb++, it++) {
          const uint32_t buf = it & 1;
          if (!(ok = mbar_wait(tempty + 8 * buf, ((it >> 1) & 1) ^ 1, gave_up, g.flag))) break;
          if (!(ok = mbar_wait(full + 8 * stage, phase, gave_up, g.flag))) break;
          fence_after();
          const uint64_t da = tile_desc(stage0 + stage * S::kStage), db = tile_desc(stage0 + stage * S::kStage + S::kABytes);
#pragma unroll
          for (int s = 0; s < 4; s++)  // k = 32 a step: 32 bytes along the swizzled row
            mma_f8<CTAS>(tmem + buf * BN, da + 2 * s, db + 2 * s, g.idesc, s > 0);
          mma_commit<CTAS>(empty + 8 * stage);
          mma_commit<CTAS>(tfull + 8 * buf);
          if (++stage == S::kStages) stage = 0, phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    fewer();
    uint32_t it = 0;
    bool ok = true;
    for (int t = unit; t < ntiles && ok; t += units) {
      int tm, tn;
      tile_at(t, g.tiles_m, g.tiles_n, tm, tn);
      const int row_a = tm * 128 * CTAS + rank * 128, row_b = tn * BN;
      // this lane's rows; those past the matrix read its last and are stored as zeros
      auto scale_a = [&](int j) { return min(row_a + lane + 32 * j, g.m - 1) >> (g.a_row ? 0 : 7); };
      constexpr int kNB = BROW ? (BN + 31) / 32 : 1;
      auto row_of_b = [&](int j) { return BROW ? row_b + lane + 32 * j : row_b + lane * 128; };
      auto scale_b = [&](int j) { return min(row_of_b(j), g.n - 1) >> (BROW && g.b_row ? 0 : 7); };
      for (int kb = kb0; kb < kb1; kb++, it++) {
        const uint32_t slot = it % kSlots, ph = (it / kSlots) & 1;
        if (!(ok = warp_wait(sempty + 8 * slot, ph ^ 1, gave_up, g.flag))) break;
        const uint32_t dst = smem_u32(scale_ring + slot * S::kScaleFloats) + 4 * lane;
#pragma unroll
        for (int j = 0; j < 4; j++)
          cp4(dst + 128 * j, g.sa + scale_a(j) * g.sa_rs + kb * g.sa_cs, row_a + lane + 32 * j < g.m);
#pragma unroll
        for (int j = 0; j < kNB; j++)
          if (BROW ? lane + 32 * j < BN : lane < (BN + 127) / 128)
            cp4(dst + 512 + 128 * j, g.sb + scale_b(j) * g.sb_rs + kb * g.sb_cs, row_of_b(j) < g.n);
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sfull + 8 * slot) : "memory");
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
  } else if (warp == 3) {
    fewer();
  } else {
    more();
    const int quad = warp & 3, band = (warp - kEpiWarp0) >> 2;
    const int row = quad * 32 + lane;
    const uint32_t tmem_row = tmem + ((uint32_t)(quad * 32) << 16) + band * kCols;
    const uint32_t tempty_leader = CTAS == 2 ? mapa(tempty, 0) : tempty;
    constexpr int kLd = kCols < 16 ? kCols : 16, kLoads = kCols / kLd, kFly = kLoads < 4 ? kLoads : 4;
    uint32_t it = 0;
    bool ok = true;
    for (int t = unit; t < ntiles && ok; t += units) {
      int tm, tn;
      tile_at(t, g.tiles_m, g.tiles_n, tm, tn);
      uint64_t acc[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; j++) acc[j] = 0;
      for (int kb = kb0; kb < kb1; kb++, it++) {
        const uint32_t slot = it % kSlots, sph = (it / kSlots) & 1, buf = it & 1, ph = (it >> 1) & 1;
        if (!(ok = warp_wait(sfull + 8 * slot, sph, gave_up, g.flag))) break;
        const float* sc = scale_ring + slot * S::kScaleFloats;
        const float sa = sc[row];
        const float sab = BROW ? sa : sa * sc[128 + (BN == 256 ? band : 0)];
        const uint64_t s2 = pair(sab, sab);
        if (!(ok = warp_wait(tfull + 8 * buf, ph, gave_up, g.flag))) break;
        fence_after();
        // kFly loads at a time, so that their latency is paid once
        uint32_t d[kFly][kLd];
#pragma unroll
        for (int q = 0; q < kFly; q++) tmem_ld<kLd>(tmem_row + buf * BN + q * kLd, d[q]);
#pragma unroll
        for (int q = 0; q < kLoads; q++) {
          float4 b[kLd / 4];  // the columns' scales, on their way before the wait
          if (BROW)
#pragma unroll
            for (int j = 0; j < kLd / 4; j++) b[j] = *reinterpret_cast<const float4*>(sc + 128 + band * kCols + q * kLd + 4 * j);
          if (q % kFly == 0) {
            tmem_ld_wait();
            if (q + kFly >= kLoads) {  // the last column is in registers: the tensor core may have the buffer
              fence_before();
              __syncwarp();
              if (lane == 0) {
                if (CTAS == 2)
                  mbar_arrive_cluster(tempty_leader + 8 * buf);
                else
                  mbar_arrive(tempty + 8 * buf);
              }
            }
          }
          uint32_t* w = d[q % kFly];
#pragma unroll
          for (int j = 0; j < kLd; j += 4) {
            uint64_t f0 = s2, f1 = s2;
            if (BROW) {
              f0 = mul2(s2, pair(b[j / 4].x, b[j / 4].y)), f1 = mul2(s2, pair(b[j / 4].z, b[j / 4].w));
            }
            uint64_t& a0 = acc[(q * kLd + j) / 2];
            uint64_t& a1 = acc[(q * kLd + j) / 2 + 1];
            a0 = fma2(pair(w[j], w[j + 1]), f0, a0);
            a1 = fma2(pair(w[j + 2], w[j + 3]), f1, a1);
          }
          if (q + kFly < kLoads) tmem_ld<kLd>(tmem_row + buf * BN + (q + kFly) * kLd, w);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(sempty + 8 * slot);
      }
      if (!ok) break;
      auto at = [&](int j) { return __uint_as_float((uint32_t)(acc[j / 2] >> (j & 1) * 32)); };
      const int row_c = tm * 128 * CTAS + rank * 128 + row, col_c = tn * BN + band * kCols;
      if (CTAS == 1 && g.ksplit > 1) {
        // this CTA's part, column-major with an odd pitch, over the stages (all consumed)
        float* part = reinterpret_cast<float*>(raw + (stage0 - smem_u32(raw)));
#pragma unroll
        for (int j = 0; j < kCols; j++) part[(band * kCols + j) * 129 + row] = at(j);
      } else if (S::kTurn && (!g.vec || g.accumulate || col_c + kCols > g.n) && g.ccs == 1) {
        float* turn = scale_ring + kSlots * S::kScaleFloats + (warp - kEpiWarp0) * S::kTurn;
        const int first = tm * 128 * CTAS + rank * 128 + quad * 32;
#pragma unroll
        for (int q = 0; q < kCols / 16; q++) {
#pragma unroll
          for (int j = 0; j < 16; j++) turn[lane * 17 + j] = at(q * 16 + j);
          __syncwarp();
          const int col = col_c + q * 16 + (lane & 15);
#pragma unroll 4
          for (int r = lane >> 4; r < 32; r += 2) {
            if (first + r >= g.m || col >= g.n) continue;
            const int64_t i = (int64_t)(first + r) * g.crs + col;
            float v = turn[r * 17 + (lane & 15)];
            if (g.accumulate) v += load_c(g.c, i, g.ctype);
            store_c(g.c, i, g.ctype, v);
          }
          __syncwarp();
        }
      } else if (row_c < g.m) {
        const int64_t base = row_c * g.crs + col_c * g.ccs;
        const int cols = min(kCols, g.n - col_c);
        if (g.vec && cols == kCols && !g.accumulate) {
          if (g.ctype == (int)MType::F32) {
            float4* p = reinterpret_cast<float4*>((float*)g.c + base);
#pragma unroll
            for (int j = 0; j < kCols / 4; j++) p[j] = make_float4(at(4 * j), at(4 * j + 1), at(4 * j + 2), at(4 * j + 3));
          } else {
            uint4* p = reinterpret_cast<uint4*>((uint16_t*)g.c + base);
#pragma unroll
            for (int j = 0; j < kCols / 8; j++) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; i++) {
                if (g.ctype == (int)MType::BF16) {
                  const __nv_bfloat162 h = __floats2bfloat162_rn(at(8 * j + 2 * i), at(8 * j + 2 * i + 1));
                  w[i] = *reinterpret_cast<const uint32_t*>(&h);
                } else {
                  const __half2 h = __floats2half2_rn(at(8 * j + 2 * i), at(8 * j + 2 * i + 1));
                  w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
              }
              p[j] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < kCols; j++)
            if (j < cols) {
              float v = at(j);
              if (g.accumulate) v += load_c(g.c, base + j * g.ccs, g.ctype);
              store_c(g.c, base + j * g.ccs, g.ctype, v);
            }
        }
      }
    }
  }

  // every role is done with this CTA's barriers, TMEM and (pair) the peer's
  fence_before();
  __syncthreads();
  if (*gave_up) settle_in_flight();
  if (CTAS == 1 && g.ksplit > 1) {
    cluster_sync();
    // each CTA adds its share of the tile over all parts, in rank order; neighbouring threads take neighbours in C
    int tm, tn;
    tile_at(unit, g.tiles_m, g.tiles_n, tm, tn);
    const int rows = min(128, g.m - tm * 128), cols = min(BN, g.n - tn * BN);
    const bool by_row = g.crs == 1;
    const int fast = by_row ? rows : cols, total = rows * cols;
    const int end = total * (split + 1) / g.ksplit;
    constexpr int kFly = 8;  // elements a thread fetches at a time: a peer's memory is far
    for (int e0 = total * split / g.ksplit + threadIdx.x; e0 < end; e0 += kThreads * kFly) {
      float v[kFly] = {};
      uint32_t at[kFly];
      int64_t to[kFly];
#pragma unroll
      for (int i = 0; i < kFly; i++) {
        const int e = min(e0 + i * kThreads, end - 1);
        const int lo = e % fast, hi = e / fast;
        const int r = by_row ? lo : hi, j = by_row ? hi : lo;
        at[i] = stage0 + (uint32_t)(j * 129 + r) * 4;
        to[i] = (tm * 128 + r) * g.crs + (tn * BN + j) * g.ccs;
      }
      for (int p = 0; p < g.ksplit; p++) {
        float w[kFly];
#pragma unroll
        for (int i = 0; i < kFly; i++) w[i] = ld_cluster(mapa(at[i], p));
#pragma unroll
        for (int i = 0; i < kFly; i++) v[i] += w[i];
      }
      if (*gave_up) continue;
#pragma unroll
      for (int i = 0; i < kFly; i++) {
        if (e0 + i * kThreads >= end) break;
        if (g.accumulate) v[i] += load_c(g.c, to[i], g.ctype);
        store_c(g.c, to[i], g.ctype, v[i]);
      }
    }
    cluster_sync();
  } else if (CTAS == 2) {
    cluster_sync();
  }
  fence_after();
  if (warp == 1) {
    if constexpr (CTAS == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTmemCols));
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTmemCols));
  }
}

// ------------------------------------------------------------------- host
// Boxes of box_rows x 128 bytes; bytes outside the matrix read as zeros (0.0 in both 8-bit types).
CUtensorMap operand_map(const ScaledOperand& o, int64_t k, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)o.rows}, strides[1] = {(cuuint64_t)o.ld};
  const cuuint32_t box[2] = {kBK, (cuuint32_t)box_rows};
  return byte_map(o.p, 2, dims, strides, box);
}

template <int CTAS, int BN, bool BROW>
void launch(const ScaledOperand& a, const ScaledOperand& b, int64_t k, GemmArgs g, int grid, int cluster, cudaStream_t s) {
  using S = Shape<CTAS, BN>;
  const CUtensorMap ma = operand_map(a, k, 128), mb = operand_map(b, k, S::kBRows);
  auto kern = scaled_gemm_kernel<CTAS, BN, BROW>;
  ensure_dynamic_smem((const void*)kern, S::kSmem);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  NDT_CUDA(cudaLaunchKernelEx(&cfg, kern, ma, mb, g));
  count_launch();
}

}  // namespace

void scaled_gemm(const ScaledOperand& a_, const ScaledOperand& b_, int64_t k, MType ct, void* c, int64_t ldc,
                 bool accumulate, cudaStream_t s, bool b_early) {
  // Up to 64 rows of A: B's rows on the 128 lanes, A's as 16 to 64 columns
  // (8192 x 8192 weights, 17 / 33 / 64 rows: 19.1 / 23.9 / 25.5 us, against
  // 24.9 / 26.3 / 30.1 as they are).
  const bool swap = a_.rows <= 64;
  const ScaledOperand &a = swap ? b_ : a_, &b = swap ? a_ : b_;
  GemmArgs g{};
  g.sa = a.s, g.sa_rs = a.srs, g.sa_cs = a.scs;
  g.sb = b.s, g.sb_rs = b.srs, g.sb_cs = b.scs;
  g.c = c, g.crs = swap ? 1 : ldc, g.ccs = swap ? ldc : 1;
  g.m = (int)a.rows, g.n = (int)b.rows;
  g.kblocks = (int)((k + kBK - 1) / kBK);
  g.a_row = a.per_row, g.b_row = b.per_row, g.ctype = (int)ct, g.accumulate = accumulate;
  g.vec = !swap && (uintptr_t)c % 16 == 0 && ldc * msize(ct) % 16 == 0;
  g.flag = wait_flag_device();
  g.ksplit = 1;
  g.early_a = swap && b_early;
  const int sms = ctx().sm_count;
  auto cdiv = [](int64_t x, int64_t y) { return (int)((x + y - 1) / y); };
  // bits of the instruction descriptor: 32-bit accumulators, the operands'
  // types (0 e4m3, 1 e5m2), both K-major, N / 8 and M / 16
  auto idesc = [&](int m, int n) {
    return 1u << 4 | (a.type == MType::E5M2 ? 1u : 0u) << 7 | (b.type == MType::E5M2 ? 1u : 0u) << 10 |
           (uint32_t)(n / 8) << 17 | (uint32_t)(m / 16) << 24;
  };
  // Waves of 128 x 128 tiles against waves of 256 x 256 pairs, which take 5 / 4
  // of the time.  us of tiles and of pairs, k 512 / 2048 / 8192: 1024 x 2048 12.3,
  // 14.3 / 18.4, 20.5 / 38.9, 45.1 (one wave of each); 1024 x 2560 18.4, 16.4 /
  // 28.7, 22.5 / 69.6, 47.1 (two of tiles, one of pairs); 2048 x 3000 26.6, 24.6 /
  // 41.0, 36.9 / 102.4, 86.0; 4096 x 4096 49.2, 30.7 / 86.0, 57.3 / 229.4, 153.6.
  const int64_t pair_tiles = (int64_t)cdiv(g.m, 256) * cdiv(g.n, 256);
  const int64_t waves = ((int64_t)cdiv(g.m, 128) * cdiv(g.n, 128) + sms - 1) / sms, pair_waves = (pair_tiles + sms / 2 - 1) / (sms / 2);
  if (!swap && 5 * pair_waves < 4 * waves) {
    g.tiles_m = cdiv(g.m, 256), g.tiles_n = cdiv(g.n, 256);
    g.idesc = idesc(256, 256);
    const int grid = 2 * (int)std::min<int64_t>(pair_tiles, sms / 2);
    if (b.per_row)
      launch<2, 256, true>(a, b, k, g, grid, 2, s);
    else
      launch<2, 256, false>(a, b, k, g, grid, 2, s);
    return;
  }
  const int bn = !swap ? 128 : g.n <= 16 ? 16 : g.n <= 32 ? 32 : 64;
  g.tiles_m = cdiv(g.m, 128), g.tiles_n = cdiv(g.n, bn);
  g.idesc = idesc(128, bn);
  // k is split while the CTAs fit the GPU at once and keep enough blocks each.
  // 128 x 128 tiles are costly to add: 128 x 2048 with k 8192 / 16384 / 32768
  // takes 36.9 / 61.4 / 114.6 us unsplit, 36.9 / 51.2 / 69.6 with 64 blocks or
  // more a CTA, 49.2 / 127 / 148 with 16.  Of few rows it costs little (k 8192, one
  // row against 1024 / 10240: 32.8 / 34.8 us unsplit, 16.4 / 28.7 with 4 or more;
  // 16 rows, 8192 x 1024: 12.4 and 14.3).
  const int room = sms * (swap ? 2 : 1), tiles = g.tiles_m * g.tiles_n;
  g.ksplit = std::max(1, std::min({8, room / tiles, g.kblocks / (swap ? 4 : 64)}));
  const int grid = tiles * g.ksplit;
  if (!swap)
    b.per_row ? launch<1, 128, true>(a, b, k, g, grid, g.ksplit, s) : launch<1, 128, false>(a, b, k, g, grid, g.ksplit, s);
  else if (bn == 16)
    launch<1, 16, true>(a, b, k, g, grid, g.ksplit, s);
  else if (bn == 32)
    launch<1, 32, true>(a, b, k, g, grid, g.ksplit, s);
  else
    launch<1, 64, true>(a, b, k, g, grid, g.ksplit, s);
}

}  // namespace ndt
