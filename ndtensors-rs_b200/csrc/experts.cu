// A mixture-of-experts layer for a few tokens, one kernel.
//
//   l[t, e] = sum over h of x[t, h] * router[e, h]
//   the `top` largest l of a token choose its experts (ties to the lowest e);
//   g = exp(l) / sum exp(l) over all experts, or over the chosen (renormalize)
//   a = W_in[e] x_t;  b = silu(a[:i]) * a[i:];  y_t = sum over chosen of g * W_out[e] b
//
// With few tokens the layer is bound by reading each chosen expert's weights
// once.  Which experts those are is known only after the router, so the steps
// are phases of one cooperative kernel (a grid barrier costs about as much as
// a launch's latency overlap saves) and every phase spreads its rows over all
// SMs.
//
// Products run on the warp-level tensor cores (mma.sync) with the weights as
// the 16-row operand and up to 8 tokens a column tile: with so few columns the
// tensor core is never what is waited for.  In the first product a tile is 8
// gate rows and the 8 up rows of the same outputs, so silu(gate) * up needs no
// exchange.
//
// The weights stream through a ring of stages in shared memory, 16 rows x 1 or
// 2 KB each.  Four teams of 4 warps take the tiles in turn; a team splits a
// stage's k and adds its parts through shared memory at a tile's end, while the
// others multiply (one team of 16 lost a quarter of its time there).  The
// ring runs across tiles, and from the first product into the second before
// the grid barrier between them.  One warp fills it.  Rows that are multiples
// of 128 bytes come as two tensor copies a stage (8 rows x 8 pieces of 128
// bytes, swizzled so that ldmatrix meets no bank conflict; 90 KB in flight on
// each SM are needed for HBM's rate, so stages are small); others of whole
// 16-byte vectors as 16 bulk copies of 2 KB, rows 2064 bytes apart, which the
// copy engine takes at 70 - 85 ns each, below the rate of HBM.  Rows of any
// other length come by bulk copies of the 16-byte granules that they touch, and
// seven warps shift them into place: 0.5 - 1.5 TB/s.  Lanes that copied their
// own fragments (cp.async) spent 110 instructions on each KB: 3.2 TB/s.
//
// Measured on one B200: 1 token, 8 of 64 experts, h 2048, i 1024, bf16 39 us
// (router 1.4, choice 5, products 10 and 6, barriers 6, the rest the launch); 8
// tokens of it 114 - 118 us, 4.6 TB/s; 64 tokens, 4 of 64, h 4096, i 1280, 8-bit
// 319 - 324 us, 3.1 TB/s, where the short rows of w_out make each tile mostly
// barriers.
//
// All sums are in 32 bits.  The activations b enter the second product as the
// sum of two 16-bit numbers, which keeps 16 bits of mantissa in bfloat16 (2^-17
// of each b at most) and 22 in float16 (2^-23, and 2^-39 of the row's largest),
// where a 32-bit b has 24: below the rounding of y, 2^-9 and 2^-12, by as much.
// For float16 each row of b is scaled by a power of two first, since b may be
// out of that type's range.  8-bit weights multiply in float16, x scaled
// likewise: exact down to 2^-28 of the token's largest, 2^-40 of it at most below.
#include <cooperative_groups.h>

#include <algorithm>

#include "mbarrier.h"

namespace ndt {
namespace {

namespace cg = cooperative_groups;

constexpr int kConsumers = 16;       // warps that multiply
// (kShift) Warps that shift rows into place; one more issues their copies.  The
// shifts bound such layers: 64 tokens, 4 of 64, h 2049, i 641, bf16 takes 405 us
// with 7 and 496 with 4, which leave no more registers to a thread (80).
constexpr int kShifters = 7;
constexpr int kMaxWarps = kConsumers + kShifters + 1;
enum Copy { kShift, kBulk, kTensor };  // how rows come: at any byte, in 16-byte vectors, in 128-byte pieces
__host__ __device__ constexpr int most_bytes(int copy) { return copy == kTensor ? 1024 : 2048; }  // of a row in one stage
__host__ __device__ constexpr int stage_bytes(int copy) { return copy == kTensor ? 16 * 1024 : 16 * (2048 + 16); }
__host__ __device__ constexpr int warps_of(int copy) { return kConsumers + (copy == kShift ? kShifters + 1 : 1); }
constexpr int kMaxSlots = 2048;      // (token, chosen expert) pairs of one launch
constexpr int kMaxTokens = 256;
constexpr int kMaxExperts = 1024;
constexpr int kGroup = 8;            // tokens of one router product
constexpr int kTeam = 4;             // multiplying warps that take a tile together
constexpr int kMaxStages = 12;
constexpr int kRawPitch = 2048 + 32, kRawBytes = 16 * kRawPitch, kMaxRaw = 4;  // (kShift)

struct LayerArgs {
  ExpertArgs e;
  int tokens, experts, top, h, i;
  int ip;           // i rounded up to 8: the pitch of b's rows
  int unit;         // tokens of an expert that a CTA takes at a time (each unit reads the weights anew)
  int stages;
  int raw;             // slots for rows at any byte (kShift)
  int row_bytes[2];    // of a row in one stage of each product: even parts of the row
  int xpitch, bpitch;  // bytes of a token's row of x / of b's parts in shared memory
  int op_bytes;     // shared memory for either, and for an expert's scales behind it
  int scale_at;     // where those start; -1: they stay in global memory
  float* logits;    // [tokens, experts]
  float* b;         // [slots, ip]
  float* o;         // [slots, h]
  unsigned* bmax;   // [slots] magnitude of the largest b
  unsigned* xmax;   // [tokens] ... of the largest x (8-bit layers)
  unsigned* arrived;  // CTAs whose part of b is written
  int* flag;        // set when a bounded wait ran out
};

struct Maps {
  CUtensorMap m[2];  // w_in and w_out
};

template <typename M>
__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<M, __half>)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename M>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<M, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename M>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same_v<M, __half>)
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
// Two 8-bit weights (the low 16 bits of w) as a pair of float16: exact.
__device__ __forceinline__ uint32_t widen(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The bits of |x|, which order as it does; infinities and NaN do not count.
__device__ __forceinline__ unsigned magnitude(float x) {
  const unsigned u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0;
}

// 16 bytes of a row of n elements from element k; zeros outside it.
template <typename T, bool VEC>
__device__ __forceinline__ uint4 row16(const T* row, int k, int n, bool on) {
  constexpr int kN = 16 / sizeof(T);
  if (!on || k >= n) return make_uint4(0, 0, 0, 0);
  if constexpr (VEC) {
    return __ldg(reinterpret_cast<const uint4*>(row + k));
  } else {
    uint4 v = make_uint4(0, 0, 0, 0);
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int j = 0; j < kN; j++)
      if (k + j < n) e[j] = row[k + j];
    return v;
  }
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, int bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes),
               "r"(bar)
               : "memory");
}
// 8 rows of a box of pieces of 128 bytes, piece by piece, 128-byte swizzle.
__device__ __forceinline__ void tensor_copy(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row, int piece) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(0), "r"(row), "r"(piece)
      : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

struct Lists {
  uint16_t chosen[kMaxSlots];     // the expert of each slot (token * top + place)
  uint16_t slots[kMaxSlots];      // slots expert by expert, in order
  int first[kMaxExperts + 1];     // where an expert's slots start (with few slots only [e + 1] of its experts)
  uint16_t unit_expert[kMaxSlots];  // an expert with up to `unit` of its slots
  uint16_t unit_first[kMaxSlots];   // ... from this place of `slots` on
  int units;
};

// The sortable form of a product: NaN above all, as in a sort; -0 and 0 equal.
__device__ __forceinline__ uint32_t sortable(float f) {
  f += 0.f;
  const uint32_t u = __float_as_uint(f);
  return f != f ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// One token's choice, by a warp that holds PER of its products a lane.
template <int PER>
__device__ __forceinline__ void choose(const LayerArgs& a, const float* l, int t, Lists& L) {
  const int lane = threadIdx.x & 31;
  float v[PER];
  uint32_t key[PER];
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const bool on = j * 32 + lane < a.experts;
    v[j] = on ? l[j * 32 + lane] : -INFINITY;
    key[j] = on ? sortable(v[j]) : 0;  // below every product's
    top = fmaxf(top, v[j]);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
#pragma unroll
  for (int j = 0; j < PER; j++) {
    v[j] = expf(v[j] - top);
    if (j * 32 + lane < a.experts) sum += v[j];
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  float total = 0.f;
  const bool tell = blockIdx.x == 0;
  for (int r = 0; r < a.top; r++) {
    uint32_t best = 0, at = 0;
#pragma unroll
    for (int j = PER - 1; j >= 0; j--)
      if (key[j] >= best) best = key[j], at = j;
    const uint32_t most = __reduce_max_sync(~0u, best);
    const uint32_t e = __reduce_min_sync(~0u, best == most ? at * 32 + lane : ~0u);
    float p = 0.f;
#pragma unroll
    for (int j = 0; j < PER; j++)
      if (j * 32 + lane == e) p = v[j], key[j] = 0;
    p = __shfl_sync(~0u, p, e & 31) / sum;
    total += p;
    if (lane == 0) {
      L.chosen[t * a.top + r] = (uint16_t)e;
      if (tell) a.e.ids[t * a.top + r] = (int)e, a.e.weights[t * a.top + r] = p;
    }
  }
  if (tell && a.e.renormalize) {
    __syncwarp();
    for (int r = lane; r < a.top; r += 32) a.e.weights[t * a.top + r] /= total;
  }
}

// Choose the experts of every token (every CTA does all of them: a barrier
// would cost more) and list the slots of every expert.
template <int kWarps>
__device__ __forceinline__ void route(const LayerArgs& a, Lists& L, int* scratch, float* space, int space_bytes) {
  constexpr int kThreads = kWarps * 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // all products at once where they fit: a load for each token in turn waits for L2 each time
  const int all = a.tokens * a.experts;
  const float* l = a.logits;
  if (all * 4 <= space_bytes) {
#pragma unroll 4
    for (int c = threadIdx.x; c < all; c += kThreads) space[c] = __ldcg(a.logits + c);
    __syncthreads();
    l = space;
  }
  for (int t = warp; t < a.tokens; t += kWarps) {
    const float* lt = l + t * a.experts;
    if (a.experts <= 64)
      choose<2>(a, lt, t, L);
    else if (a.experts <= 256)
      choose<8>(a, lt, t, L);
    else
      choose<32>(a, lt, t, L);
  }
  __syncthreads();
  const int slots = a.tokens * a.top;
  if (slots <= 32) {  // one warp: a slot's place is the number of slots before it by (expert, slot)
    if (warp == 0) {
      const int e = lane < slots ? L.chosen[lane] : 0xffff;
      const unsigned same = __match_any_sync(~0u, e);
      const int rank = __popc(same & ((1u << lane) - 1));
      int before = 0, units = 0;  // slots, and units, of lower experts
      for (int s = 0; s < slots; s++) {
        const int f = __shfl_sync(~0u, e, s), r = __shfl_sync(~0u, rank, s);
        if (f < e) before++, units += r % a.unit == 0;
      }
      const int place = before + rank;
      if (lane < slots) {
        L.slots[place] = (uint16_t)lane;
        if (rank % a.unit == 0) {
          L.unit_expert[units + rank / a.unit] = (uint16_t)e, L.unit_first[units + rank / a.unit] = (uint16_t)place;
          if (rank == 0) L.first[e + 1] = before + __popc(same);
        }
      }
      const int all = __popc(__ballot_sync(~0u, lane < slots && rank % a.unit == 0));
      if (lane == 0) L.units = all;
    }
    __syncthreads();
    return;
  }
  for (int e = warp; e < a.experts; e += kWarps) {
    int n = 0;
    for (int s = 0; s < slots; s += 32) n += __popc(__ballot_sync(~0u, s + lane < slots && L.chosen[s + lane] == e));
    if (lane == 0) scratch[e] = n;
  }
  __syncthreads();
  if (warp == 0) {
    int at = 0, units = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane, n = e < a.experts ? scratch[e] : 0, u = (n + a.unit - 1) / a.unit;
      int x = n, y = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int p = __shfl_up_sync(~0u, x, o), q = __shfl_up_sync(~0u, y, o);
        if (lane >= o) x += p, y += q;
      }
      if (e < a.experts) L.first[e] = at + x - n;
      for (int k = 0; k < u; k++) {
        L.unit_expert[units + y - u + k] = (uint16_t)e;
        L.unit_first[units + y - u + k] = (uint16_t)(at + x - n + k * a.unit);
      }
      at += __shfl_sync(~0u, x, 31), units += __shfl_sync(~0u, y, 31);
    }
    if (lane == 0) L.first[a.experts] = at, L.units = units;
  }
  __syncthreads();
  for (int e = warp; e < a.experts; e += kWarps) {
    int at = L.first[e];
    if (L.first[e + 1] == at) continue;
    for (int s = 0; s < slots; s += 32) {
      const bool on = s + lane < slots && L.chosen[s + lane] == e;
      const unsigned m = __ballot_sync(~0u, on);
      if (on) L.slots[at + __popc(m & ((1u << lane) - 1))] = (uint16_t)(s + lane);
      at += __popc(m);
    }
  }
  __syncthreads();
}

// Sums over the warp of 32 values a lane: lane l ends with the sum of value l.
__device__ __forceinline__ float transpose_sum(float* v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int j = 0; j < o; j++) {
      const bool up = lane & o;
      const float give = up ? v[j] : v[j + o], keep = up ? v[j + o] : v[j];
      v[j] = keep + __shfl_xor_sync(~0u, give, o);
    }
  return v[0];
}

// Router products: a CTA takes RE experts and up to 8 tokens (MAX: and their
// largest magnitudes).
template <typename X, int COPY, bool MAX, int RE>
__device__ __forceinline__ void router(const LayerArgs& a, float* red) {
  static_assert(RE * kGroup <= 32, "");
  constexpr int kWarps = warps_of(COPY), kThreads = kWarps * 32;
  constexpr bool VEC = COPY != kShift;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = (a.tokens + kGroup - 1) / kGroup, es = (a.experts + RE - 1) / RE;
  for (int u = blockIdx.x; u < es * groups; u += gridDim.x) {
    const int e0 = u % es * RE, t0 = u / es * kGroup, nt = min(kGroup, a.tokens - t0), ne = min(RE, a.experts - e0);
    float acc[32] = {};
    unsigned top[kGroup] = {};
    const X* r = (const X*)a.e.router + (int64_t)e0 * a.h;
    const X* x = (const X*)a.e.x + (int64_t)t0 * a.e.ldx;
    for (int k = threadIdx.x * 8; k < a.h; k += kThreads * 8) {
      uint4 rv[RE], xv[kGroup];
#pragma unroll
      for (int j = 0; j < RE; j++) rv[j] = row16<X, VEC>(r + (int64_t)j * a.h, k, a.h, j < ne);
#pragma unroll
      for (int t = 0; t < kGroup; t++) xv[t] = row16<X, VEC>(x + t * a.e.ldx, k, a.h, t < nt);
#pragma unroll
      for (int t = 0; t < kGroup; t++) {
        if (t >= nt) break;
        const X* xe = reinterpret_cast<const X*>(&xv[t]);
        if (MAX)
#pragma unroll
          for (int c = 0; c < 8; c++) top[t] = max(top[t], magnitude(to_f32<X>(xe[c])));
#pragma unroll
        for (int j = 0; j < RE; j++) {
          const X* re = reinterpret_cast<const X*>(&rv[j]);
#pragma unroll
          for (int c = 0; c < 8; c++) acc[j * kGroup + t] = fmaf(to_f32<X>(re[c]), to_f32<X>(xe[c]), acc[j * kGroup + t]);
        }
      }
    }
    red[warp * 32 + lane] = transpose_sum(acc);
    if (MAX && e0 == 0) {
#pragma unroll
      for (int t = 0; t < kGroup; t++) {
        const unsigned m = __reduce_max_sync(~0u, top[t]);
        if (lane == 0) red[(kMaxWarps + t) * 32 + warp] = __uint_as_float(m);
      }
    }
    __syncthreads();
    if (warp == 0) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) s += red[w * 32 + lane];
      const int j = lane / kGroup, t = lane % kGroup;
      if (j < ne && t < nt) a.logits[(int64_t)(t0 + t) * a.experts + e0 + j] = s;
    }
    if (MAX && e0 == 0 && threadIdx.x < nt) {
      unsigned m = 0;
      for (int w = 0; w < kWarps; w++) m = max(m, __float_as_uint(red[(kMaxWarps + threadIdx.x) * 32 + w]));
      a.xmax[t0 + threadIdx.x] = m;
    }
    __syncthreads();
  }
}

// W: the weights' type, X: x's and y's, M: the products', COPY: how rows come,
// NT: column tiles of 8 tokens that a product takes at a time.
template <typename W, typename X, typename M, int COPY, int NT>
struct Layer {
  static constexpr bool VEC = COPY != kShift;
  static constexpr int kWarps = warps_of(COPY), kThreads = kWarps * 32;
  static constexpr bool kScaled = sizeof(W) == 1;
  static constexpr bool kHalf = std::is_same_v<M, __half>;
  static constexpr int kStageBytes = stage_bytes(COPY);
  static constexpr int kRowPitch = most_bytes(COPY) + 16;     // (not kTensor)
  static constexpr int kStepK = kScaled ? 128 : 32;           // k of a warp's step: one scale, or two MMAs
  static constexpr int kStepBytes = kStepK * (int)sizeof(W);
  static constexpr int kRed = kTeam * NT * 128;               // floats of a tile's parts

  // The power of two that brings a row whose largest finite value is at `most`
  // to float16's upper end, from 2^top up (sign 1), or what takes it back.  There
  // the row has its type's bits down to 2^-28 of the largest: a channel that
  // dominates it, and may meet zero weights, costs the others none.  (The sums
  // are in 32 bits; float16 is 2^16 at most.)
  static constexpr int kTopX = 15, kTopB = 14;  // x has no more bits than float16; b may round up
  __device__ static __forceinline__ float power(const unsigned* most, int top, int sign) {
    const int ex = (int)(__ldcg(most) >> 23) - 127;
    const int c = min(top - ex, 126);  // (a smaller row than 2^-111: as far as 32 bits go)
    return __uint_as_float((uint32_t)(127 + sign * c) << 23);
  }

  __device__ static void run(const LayerArgs& a, const CUtensorMap* maps, Lists& L, int* scratch, uint64_t* bars, volatile int* gave_up,
                             unsigned char* dyn) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2;
    unsigned char* op = dyn;                                        // x, then b, of the unit's tokens
    float* red = reinterpret_cast<float*>(dyn + a.op_bytes);        // two buffers of parts a team
    unsigned char* ring = dyn + a.op_bytes + 2 * kConsumers / kTeam * kRed * 4;
    ring += (1024 - (smem_u32(ring) & 1023)) & 1023;
    const uint32_t full = smem_u32(bars), empty = full + 8 * kMaxStages;
    __shared__ float back[NT * 8];  // what takes a token's results back from float16's range
    cg::grid_group grid = cg::this_grid();

    if (threadIdx.x == 0) {
      *gave_up = 0;
      for (int st = 0; st < a.stages; st++) {
        mbar_init(full + 8 * st, VEC ? 1 : kShifters);
        mbar_init(empty + 8 * st, kConsumers);
      }
      for (int st = 0; st < kMaxRaw; st++) {
        mbar_init(empty + 8 * (kMaxStages + st), 1);
        mbar_init(empty + 8 * (kMaxStages + kMaxRaw + st), kShifters);
      }
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (a.tokens <= 8)
      router<X, COPY, kScaled, 1>(a, red);
    else
      router<X, COPY, kScaled, 4>(a, red);
    const int tiles0 = (a.i + 7) / 8, tiles1 = (a.h + 15) / 16;
    if (kHalf)
      for (int s = blockIdx.x * kThreads + threadIdx.x; s < a.tokens * a.top; s += gridDim.x * kThreads) a.bmax[s] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.arrived = 0;
    grid.sync();
    route<kWarps>(a, L, scratch, reinterpret_cast<float*>(ring), a.stages * kStageBytes);
    // (plain writes to the ring before its first copies)
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();

    // the tiles are dealt to the CTAs in even runs
    auto share = [&](int tasks, int cta) { return (int)((int64_t)tasks * cta / gridDim.x); };
    const int first0 = share(L.units * tiles0, blockIdx.x), end0 = share(L.units * tiles0, blockIdx.x + 1);
    const int first1 = share(L.units * tiles1, blockIdx.x), end1 = share(L.units * tiles1, blockIdx.x + 1);

    if (warp >= kConsumers) {
      if (COPY == kShift) {
        shift_tiles(a, L, first0, end0, tiles0, first1, end1, tiles1, ring, full, empty, gave_up);
      } else {
        int stage = 0;
        uint32_t phase = 0;
        if (copy_tiles<0>(a, maps, L, first0, end0, tiles0, ring, full, empty, stage, phase, gave_up))
          copy_tiles<1>(a, maps + 1, L, first1, end1, tiles1, ring, full, empty, stage, phase, gave_up);
      }
      __syncwarp();
    } else {
      const int team = warp / kTeam, part = warp % kTeam;
      int stage = 0, parity = 0;
      uint32_t phase = 0;
      // Over another team's stages.  Every team gives every stage back, so that
      // none is ever a whole round of the ring from another and a barrier's
      // parity stays unambiguous.
      auto pass = [&](int k, int row_bytes) {
        for (int b = 0; b < k * (int)sizeof(W); b += row_bytes) {
          mbar_wait(full + 8 * stage, phase, gave_up, a.flag);
          __syncwarp();
          if (lane == 0) mbar_arrive(empty + 8 * stage);
          if (++stage == a.stages) stage = 0, phase ^= 1;
        }
      };
      auto park = [&](float (*acc)[4]) {  // this warp's part of the tile, for the warps that finish it
        float* at = red + (team * 2 + parity) * kRed;
#pragma unroll
        for (int j = 0; j < NT; j++)
          *reinterpret_cast<float4*>(at + ((part * NT + j) * 32 + lane) * 4) = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
        asm volatile("bar.sync %0, %1;" ::"r"(2 + team), "n"(kTeam * 32) : "memory");  // one a tile: two buffers alternate
        parity ^= 1;
        return (const float*)at;
      };

      // ---- first product: tiles of 8 outputs of one expert
      int unit = -1;
      for (int task = first0; task < end0; task++) {
        const int u = task / tiles0, i0 = (task - u * tiles0) * 8;
        const int e = L.unit_expert[u], n0 = L.unit_first[u], n = min(a.unit, L.first[e + 1] - n0);
        if (u != unit) {
          if (unit < 0 || a.tokens > 1 || kScaled) stage_x(a, L, e, n0, n, op, back);
          unit = u;
        }
        if ((task - first0) % (kConsumers / kTeam) != team) {
          pass(a.h, a.row_bytes[0]);
          continue;
        }
        float acc[NT][4] = {};
        const int row_a = min(i0 + g, a.i - 1);
        multiply<0>(a, acc, e, row_a, a.i + row_a, n, op, ring, full, empty, stage, phase, gave_up);
        const float* parts = park(acc);
        // accumulator (row g: gate; row g + 8: up; columns 2 q, 2 q + 1) of column tile j; which warps finish goes round
        for (int o = ((part + (task / kTeam & 1) * 2) % kTeam) * 32 + lane; o < NT * 64; o += kTeam * 32) {
          const int j = o >> 6, ln = o >> 1 & 31, half = o & 1;
          const int col = j * 8 + (ln & 3) * 2 + half, row = i0 + (ln >> 2);
          if (col >= n || row >= a.i) continue;
          float ga = 0.f, up = 0.f;
#pragma unroll
          for (int w = 0; w < kTeam; w++) {
            const float* p = parts + ((w * NT + j) * 32 + ln) * 4 + half;
            ga += p[0], up += p[2];
          }
          const int64_t slot = L.slots[n0 + col];
          if (kScaled) ga *= back[col], up *= back[col];
          const float v = ga / (1.f + expf(-ga)) * up;
          a.b[slot * a.ip + row] = v;
          if (kHalf) atomicMax(a.bmax + slot, magnitude(v));
        }
      }
      all_consumers_sync(a, gave_up);

      // ---- second product: tiles of 16 rows of one expert
      unit = -1;
      for (int task = first1; task < end1; task++) {
        const int u = task / tiles1, tile = task - u * tiles1, r0 = tile * 16;
        const int e = L.unit_expert[u], n0 = L.unit_first[u], n = min(a.unit, L.first[e + 1] - n0);
        if (u != unit) {
          stage_b(a, L, e, n0, n, op, back);
          unit = u;
        }
        if ((task - first1) % (kConsumers / kTeam) != team) {
          pass(a.i, a.row_bytes[1]);
          continue;
        }
        float acc[NT][4] = {};
        multiply<1>(a, acc, e, min(r0 + g, a.h - 1), min(r0 + g + 8, a.h - 1), n, op, ring, full, empty, stage, phase, gave_up);
        const float* parts = park(acc);
        // warp `part` finishes accumulator `part` of every lane
        static_assert(kTeam == 4, "");
#pragma unroll
        for (int j = 0; j < NT; j++) {
          const int col = j * 8 + (lane & 3) * 2 + (part & 1), row = r0 + (lane >> 2) + (part & 2) * 4;
          if (col >= n || row >= a.h) continue;
          float s = 0.f;
#pragma unroll
          for (int w = 0; w < kTeam; w++) s += parts[((w * NT + j) * 32 + lane) * 4 + part];
          const int slot = L.slots[n0 + col];
          a.o[(int64_t)slot * a.h + row] = kHalf ? s * back[col] : s;
        }
      }
    }
    // ---- the tokens' sums over their experts, in the order of choice
    // (A counter a tile, whose last part sums it, saves this barrier; its
    // fence in every tile cost four times as much.)
    grid.sync();
    const bool four = a.h % 4 == 0 && a.e.ldy % 4 == 0 && (uintptr_t)a.e.y % (4 * sizeof(X)) == 0;
    const int step = four ? 4 : 1, columns = a.h / step;
    for (int c = blockIdx.x * kThreads + threadIdx.x; c < a.tokens * columns; c += gridDim.x * kThreads) {
      const int t = c / columns, row = (c - t * columns) * step;
      float s[4] = {};
#pragma unroll 4
      for (int r = 0; r < a.top; r++) {
        const float w = __ldcg(a.e.weights + t * a.top + r);
        const float* o = a.o + ((int64_t)t * a.top + r) * a.h + row;
        if (four) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(o));
          s[0] = fmaf(w, v.x, s[0]), s[1] = fmaf(w, v.y, s[1]), s[2] = fmaf(w, v.z, s[2]), s[3] = fmaf(w, v.w, s[3]);
        } else {
          s[0] = fmaf(w, __ldcg(o), s[0]);
        }
      }
      X* y = (X*)a.e.y + (int64_t)t * a.e.ldy + row;
      if (four)
        *reinterpret_cast<uint2*>(y) = make_uint2(pack2<X>(s[0], s[1]), pack2<X>(s[2], s[3]));
      else
        *y = from_f32<X>(s[0]);
    }
    if (*gave_up) settle_in_flight();
  }

  __device__ static __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }

  // A barrier of the multiplying warps of all CTAs (the grid is resident as a
  // whole).  The copying warps stay out of it: they may be waiting for room in
  // the ring, which only the second product makes.
  __device__ static __forceinline__ void all_consumers_sync(const LayerArgs& a, volatile int* gave_up) {
    consumers_sync();
    if (threadIdx.x == 0) {
      // (release and acquire at the GPU's scope: the CTA's barriers carry the other warps' writes)
      asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(a.arrived) : "memory");
      const long long t0 = clock64();
      unsigned n;
      do {
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(a.arrived) : "memory");
        if (clock64() - t0 > kWaitLimit) {
          *gave_up = 1;
          atomicExch_system(a.flag, 1);
          break;
        }
      } while (n < gridDim.x);
    }
    consumers_sync();
  }

  // Fill the ring with the tiles' rows.  PRODUCT 0: outputs 8 tile + r, their
  // gate rows of w_in in stage rows 0 - 7, their up rows in 8 - 15; 1: rows
  // 16 tile + r of w_out.  Rows past the end are others or zeros (not used).
  // False after a wait that gave up: a stage still in use takes no copy.
  template <int PRODUCT>
  __device__ static __forceinline__ bool copy_tiles(const LayerArgs& a, const CUtensorMap* map, const Lists& L, int first, int end, int tiles,
                                                    unsigned char* ring, uint32_t full, uint32_t empty, int& stage,
                                                    uint32_t& phase, volatile int* gave_up) {
    const int lane = threadIdx.x & 31;
    const int k = PRODUCT == 0 ? a.h : a.i;
    const int64_t rows = PRODUCT == 0 ? 2 * (int64_t)a.i : a.h;
    const W* w = (const W*)(PRODUCT == 0 ? a.e.w_in : a.e.w_out);
    auto row_of = [&](int tile, int r) {
      return PRODUCT == 0 ? min(tile * 8 + (r & 7), a.i - 1) + (r >= 8 ? a.i : 0) : min(tile * 16 + r, a.h - 1);
    };
    for (int task = first; task < end; task++) {
      const int u = task / tiles, tile = task - u * tiles;
      const int64_t expert = L.unit_expert[u];
      const int row_bytes = a.row_bytes[PRODUCT], row_k = row_bytes / (int)sizeof(W);
      for (int k0 = 0; k0 < k; k0 += row_k) {
        if (!warp_wait(empty + 8 * stage, phase ^ 1, gave_up, a.flag)) return false;
        unsigned char* dst = ring + stage * kStageBytes;
        if constexpr (COPY == kTensor) {
          if (lane == 0) {
            const int bar = full + 8 * stage, piece = k0 * (int)sizeof(W) / 128;
            mbar_expect_tx(bar, 16 * row_bytes);  // whole boxes: what is outside the tensor comes as zeros
            tensor_copy(smem_u32(dst), map, bar, (int)(expert * rows) + (PRODUCT == 0 ? tile * 8 : tile * 16), piece);
            tensor_copy(smem_u32(dst) + 8 * 1024, map, bar, (int)(expert * rows) + (PRODUCT == 0 ? a.i + tile * 8 : tile * 16 + 8), piece);
          }
          __syncwarp();
        } else {
          const int bytes = min(row_bytes, (k - k0) * (int)sizeof(W));
          if (lane == 0) mbar_expect_tx(full + 8 * stage, 16 * bytes);
          __syncwarp();
          if (lane < 16) bulk_copy(smem_u32(dst + lane * kRowPitch), w + (expert * rows + row_of(tile, lane)) * k + k0, bytes, full + 8 * stage);
        }
        if (++stage == a.stages) stage = 0, phase ^= 1;
      }
    }
    return true;
  }

  // The same for rows that start at any byte: the 16-byte granules that a row
  // touches come by a bulk copy into a slot, and the copying warps shift the
  // bytes into a stage.  (Granules that reach past the weights' first or last
  // byte are not copied; what they hold of a row is read byte by byte.)  Rows
  // that one stage holds whole lie one behind the other: one copy brings a tile's
  // 16 of w_out, two its 8 and 8 of w_in (a copy costs 70 - 85 ns of its SM at
  // any size; h 4096, i 181 400 -> 390 us when it came).
  __device__ static __forceinline__ void shift_tiles(const LayerArgs& a, const Lists& L, int first0, int end0, int tiles0, int first1,
                                                     int end1, int tiles1, unsigned char* ring, uint32_t full, uint32_t empty,
                                                     volatile int* gave_up) {
    const int lane = threadIdx.x & 31, copier = (threadIdx.x >> 5) - kConsumers;
    unsigned char* raw = ring + a.stages * kStageBytes;
    const uint32_t arrived = empty + 8 * kMaxStages, read = arrived + 8 * kMaxRaw;  // a slot's copies; its rows' shifts
    struct At {
      int product, task, byte;
    };
    auto settle = [&](At& p) {
      if (p.product == 0 && p.task >= end0) p.product = 1, p.task = first1;
      if (p.product == 1 && p.task >= end1) p.product = 2;
    };
    auto next = [&](At& p) {
      p.byte += a.row_bytes[p.product];
      if (p.byte < (p.product == 0 ? a.h : a.i) * (int)sizeof(W)) return;
      p.byte = 0, p.task++;
      settle(p);
    };
    struct Row {
      uintptr_t at, base, lo, hi;  // the row's first byte; its copy's first granule; the granules that are copied
      int bytes, from;             // where the copy's first granule goes in the slot
    };
    auto whole = [&](int product) { return a.row_bytes[product] >= (product == 0 ? a.h : a.i) * (int)sizeof(W); };
    auto row_of = [&](const At& p, int r) {
      const bool p0 = p.product == 0;
      const int tiles = p0 ? tiles0 : tiles1, u = p.task / tiles, tile = p.task - u * tiles;
      const int row = p0 ? min(tile * 8 + (r & 7), a.i - 1) + (r >= 8 ? a.i : 0) : min(tile * 16 + r, a.h - 1);
      const int64_t rows = p0 ? 2 * (int64_t)a.i : a.h, length = (int64_t)(p0 ? a.h : a.i) * sizeof(W);
      const uintptr_t w = (uintptr_t)(p0 ? a.e.w_in : a.e.w_out), end = w + a.experts * rows * length;
      Row x;
      x.at = w + (L.unit_expert[u] * rows + row) * length + p.byte;
      x.bytes = (int)min((int64_t)a.row_bytes[p.product], length - p.byte);
      uintptr_t first = x.at, last = x.at + x.bytes;  // what the row's copy brings
      x.from = r * kRawPitch;
      if (whole(p.product)) {
        const int run = p0 ? 8 : 16, first_row = tile * run, last_row = min(first_row + run, p0 ? a.i : a.h);
        const uintptr_t block = w + (L.unit_expert[u] * rows + (p0 && r >= 8 ? a.i : 0)) * length;
        first = block + first_row * length, last = block + last_row * length;
        x.from = (p0 ? r & 8 : 0) * kRawPitch;
      }
      x.base = first & ~(uintptr_t)15;
      x.lo = max(x.base, (w + 15) & ~(uintptr_t)15);
      x.hi = max(x.lo, min((last + 15) & ~(uintptr_t)15, end & ~(uintptr_t)15));
      return x;
    };
    auto issue = [&](const At& p, int slot) {  // one warp
      const Row x = row_of(p, lane & 15);
      const bool copies = lane < 16 && (!whole(p.product) || lane == 0 || (lane == 8 && p.product == 0));
      const int bytes = copies ? (int)(x.hi - x.lo) : 0;
      const int all = __reduce_add_sync(~0u, bytes);
      if (lane == 0) mbar_expect_tx(arrived + 8 * slot, all);
      __syncwarp();
      if (bytes)
        bulk_copy(smem_u32(raw + slot * kRawBytes + x.from) + (uint32_t)(x.lo - x.base), (const void*)x.lo, bytes, arrived + 8 * slot);
    };
    At p{0, first0, 0};
    settle(p);
    int stage = 0, slot = 0;
    uint32_t phase = 0, turn = 0;
    // (16 copies take a warp as long as its share of the shifts: a warp of their own)
    if (copier == kShifters) {
      for (; p.product < 2; next(p)) {
        if (!warp_wait(read + 8 * slot, turn ^ 1, gave_up, a.flag)) break;
        issue(p, slot);
        if (++slot == a.raw) slot = 0, turn ^= 1;
      }
      return;
    }
    for (; p.product < 2; next(p)) {
      mbar_wait(arrived + 8 * slot, turn, gave_up, a.flag);
      mbar_wait(empty + 8 * stage, phase ^ 1, gave_up, a.flag);
      __syncwarp();
      for (int r = copier; r < 16; r += kShifters) {
        const Row x = row_of(p, r);
        const unsigned char* from = raw + slot * kRawBytes + x.from;
        const int skew = (int)(x.at - x.base), lo = (int)(x.lo - x.base), hi = (int)(x.hi - x.base);
        unsigned char* to = ring + stage * kStageBytes + r * kRowPitch;
        constexpr int kFly = most_bytes(COPY) / 512;  // a lane's 16-byte pieces of the row: all at once
        uint32_t q[kFly][5];
        const uint32_t shift = (skew & 3) * 8;
#pragma unroll
        for (int f = 0; f < kFly; f++) {  // five words of the slot hold 16 bytes (the slot has room behind the row)
          const uint32_t* words = reinterpret_cast<const uint32_t*>(from) + (skew >> 2) + lane * 4 + f * 128;
          if (lane * 16 + f * 512 < x.bytes)
#pragma unroll
            for (int j = 0; j < 5; j++) q[f][j] = words[j];
        }
#pragma unroll
        for (int f = 0; f < kFly; f++) {
          const int c = lane * 16 + f * 512, n = min(16, x.bytes - c), at = skew + c;
          if (n <= 0) break;
          uint32_t v[4];
          if (at >= lo && at + n <= hi) {
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = __funnelshift_r(q[f][j], q[f][j + 1], shift);
            if (n < 16) {
#pragma unroll
              for (int j = 0; j < 4; j++) {
                const int keep = n - 4 * j;  // zeros past the row's end
                v[j] = keep >= 4 ? v[j] : keep <= 0 ? 0 : v[j] & ((1u << 8 * keep) - 1);
              }
            }
          } else {
            const unsigned char* g = reinterpret_cast<const unsigned char*>(x.at) + c;
#pragma unroll
            for (int j = 0; j < 4; j++) {
              v[j] = 0;
              for (int b = 0; b < 4; b++)
                if (4 * j + b < n) v[j] |= (uint32_t)g[4 * j + b] << 8 * b;
            }
          }
          *reinterpret_cast<uint4*>(to + c) = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(full + 8 * stage);
        mbar_arrive(read + 8 * slot);
      }
      if (++stage == a.stages) stage = 0, phase ^= 1;
      if (++slot == a.raw) slot = 0, turn ^= 1;
    }
  }

  // The scales of one expert's [rows, k] weights behind the tokens, where they
  // fit: a tile's would wait for L2 in every stage.
  __device__ static __forceinline__ void stage_scales(const LayerArgs& a, const float* scales, int expert, int rows, int k,
                                                      unsigned char* op) {
    if (!kScaled || a.scale_at < 0) return;
    const int n = (rows + 127) / 128 * ((k + 127) / 128);
    float* to = reinterpret_cast<float*>(op + a.scale_at);
    for (int c = threadIdx.x; c < n; c += kConsumers * 32) to[c] = __ldg(scales + (int64_t)expert * n + c);
  }

  // The unit's tokens of x as rows of `op`, zeros up to a multiple of 128.  8-bit
  // weights are exact in float16 (one instruction for two), so x goes there too.
  __device__ static __forceinline__ void stage_x(const LayerArgs& a, const Lists& L, int expert, int n0, int n, unsigned char* op, float* back) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    consumers_sync();
    if (kScaled && threadIdx.x < n) back[threadIdx.x] = power(a.xmax + L.slots[n0 + threadIdx.x] / a.top, kTopX, -1);
    stage_scales(a, a.e.in_scales, expert, 2 * a.i, a.h, op);
    const int padded = (a.h + 127) / 128 * 128;
    for (int c = warp * 32 + lane; c < n * (padded / 8); c += kConsumers * 32) {
      const int t = c / (padded / 8), k = (c - t * (padded / 8)) * 8;
      const int token = L.slots[n0 + t] / a.top;
      uint4 v = row16<X, VEC>((const X*)a.e.x + (int64_t)token * a.e.ldx, k, a.h, true);
      if (kScaled) {
        const float f = power(a.xmax + token, kTopX, 1);
        uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const float2 x = unpack2<X>(w[j]);
          w[j] = pack2<M>(x.x * f, x.y * f);
        }
      }
      *reinterpret_cast<uint4*>(op + t * a.xpitch + k * 2) = v;
    }
    consumers_sync();
  }
  // The unit's rows of b as high parts, then low parts.
  __device__ static __forceinline__ void stage_b(const LayerArgs& a, const Lists& L, int expert, int n0, int n, unsigned char* op, float* back) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    consumers_sync();
    if (kHalf && threadIdx.x < n) back[threadIdx.x] = power(a.bmax + L.slots[n0 + threadIdx.x], kTopB, -1);
    stage_scales(a, a.e.out_scales, expert, a.h, a.i, op);
    const int padded = (a.i + 127) / 128 * 128;
    for (int c = warp * 32 + lane; c < n * (padded / 4); c += kConsumers * 32) {
      const int t = c / (padded / 4), k = (c - t * (padded / 4)) * 4;
      const int slot = L.slots[n0 + t];
      const float scale = kHalf ? power(a.bmax + slot, kTopB, 1) : 1.f;
      float4 f = make_float4(0, 0, 0, 0);
      if (k < a.i) f = __ldcg(reinterpret_cast<const float4*>(a.b + (int64_t)slot * a.ip + k));
      float v[4] = {f.x, f.y, f.z, f.w};
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int j = 0; j < 4; j++) v[j] = k + j < a.i ? v[j] * scale : 0.f;
#pragma unroll
      for (int j = 0; j < 2; j++) {
        hi[j] = pack2<M>(v[2 * j], v[2 * j + 1]);
        const float2 h = unpack2<M>(hi[j]);
        // (an infinite high part stands alone: no inf - inf)
        lo[j] = pack2<M>(isinf(h.x) ? 0.f : v[2 * j] - h.x, isinf(h.y) ? 0.f : v[2 * j + 1] - h.y);
      }
      *reinterpret_cast<uint2*>(op + t * a.bpitch + k * 2) = make_uint2(hi[0], hi[1]);
      *reinterpret_cast<uint2*>(op + (a.unit + t) * a.bpitch + k * 2) = make_uint2(lo[0], lo[1]);
    }
    consumers_sync();
  }

  // This warp's part of one tile: its steps of every stage of the tile.
  template <int PRODUCT>
  __device__ static __forceinline__ void multiply(const LayerArgs& a, float (*acc)[4], int expert, int row_a, int row_b, int n,
                                                  const unsigned char* op, const unsigned char* ring, uint32_t full,
                                                  uint32_t empty, int& stage, uint32_t& phase, volatile int* gave_up) {
    constexpr int kParts = PRODUCT == 0 ? 1 : 2;  // b comes in two parts
    const int part = (threadIdx.x >> 5) % kTeam, lane = threadIdx.x & 31;
    const int g = lane >> 2, q = lane & 3;
    const int k = PRODUCT == 0 ? a.h : a.i;
    const int pitch = PRODUCT == 0 ? a.xpitch : a.bpitch;
    const float *sa = nullptr, *sb = nullptr;
    if (kScaled) {
      const int64_t kb = (k + 127) / 128, rb = ((PRODUCT == 0 ? 2 * a.i : a.h) + 127) / 128;
      const float* s = a.scale_at < 0 ? (PRODUCT == 0 ? a.e.in_scales : a.e.out_scales) + expert * rb * kb
                                      : reinterpret_cast<const float*>(op + a.scale_at);
      sa = s + (row_a >> 7) * kb, sb = s + (row_b >> 7) * kb;
    }
    // the lane's row of the weights' 8 x 16 byte pieces: rows 0 - 7, 8 - 15, the same of the next 16 bytes
    const uint32_t wrow = smem_u32(ring) + (COPY == kTensor ? (lane >> 3 & 1) * 8 * 1024 + (lane & 7) * 128
                                                            : (lane & 15) * kRowPitch + (lane >> 4) * 16);
    auto piece = [&](int byte) {  // of the stage's row, a multiple of 32
      return COPY == kTensor ? (byte >> 7) * 1024 + ((((byte >> 4 & 7) + (lane >> 4)) ^ (lane & 7)) << 4) : byte;
    };
    // 16-bit weights: the lane's token and piece of k of the tokens' four 8 x 16 byte pieces
    const uint32_t ops = smem_u32(op);
    float odd[NT][4] = {};  // every second MMA's sums: a chain of dependent ones is half as long
    const int row_bytes = a.row_bytes[PRODUCT], row_k = row_bytes / (int)sizeof(W);
    int turn = part;  // the team's warps take the tile's steps in turn: this stage's first of this warp
    for (int k0 = 0; k0 < k; k0 += row_k) {
      // bytes of a row in this stage, whole 16-byte pieces (zeros past the row's end)
      const int bytes = min(row_bytes, ((k - k0) * (int)sizeof(W) + 15) / 16 * 16);
      mbar_wait(full + 8 * stage, phase, gave_up, a.flag);
      __syncwarp();
      const uint32_t at = wrow + stage * kStageBytes;
      int byte = turn * kStepBytes;  // of the stage's row
#pragma unroll 2
      for (; byte < bytes; byte += kTeam * kStepBytes) {
        const int kk = k0 + byte / (int)sizeof(W);
        if constexpr (!kScaled) {
          uint32_t w[8];
          ldmatrix4(at + piece(byte), w);
          if (byte + 16 >= bytes) w[2] = w[3] = 0;
          if (byte + 32 < bytes) ldmatrix4(at + piece(byte + 32), w + 4);
          else w[4] = w[5] = w[6] = w[7] = 0;
          if (byte + 48 >= bytes) w[6] = w[7] = 0;
#pragma unroll
          for (int j = 0; j < NT; j++) {
            if (j * 8 >= n) break;
#pragma unroll
            for (int p = 0; p < kParts; p++) {
              uint32_t b[4];
              ldmatrix4(ops + (min(j * 8 + (lane & 7), n - 1) + p * a.unit) * pitch + kk * 2 + (lane >> 3) * 16, b);
              mma<M>(acc[j], w[0], w[1], w[2], w[3], b[0], b[1]);
              mma<M>(odd[j], w[4], w[5], w[6], w[7], b[2], b[3]);
            }
          }
        } else {
          const float fa = sa[kk >> 7], fb = sb[kk >> 7];
          float sum[NT][2][4] = {};
          uint32_t w[4][4];  // 32 bytes of k each: two pieces of 16
#pragma unroll
          for (int c = 0; c < 4; c++) {
            if (byte + c * 32 < bytes) ldmatrix4(at + piece(byte + c * 32), w[c]);
            else w[c][0] = w[c][1] = w[c][2] = w[c][3] = 0;
            if (byte + c * 32 + 16 >= bytes) w[c][2] = w[c][3] = 0;
          }
#pragma unroll
          for (int c = 0; c < 4; c++) {
            uint32_t m[8];  // lane q has k 4 q .. 4 q + 3 of a piece: its MMA takes them as 2 q, 2 q + 1 and + 8
#pragma unroll
            for (int r = 0; r < 4; r++) m[2 * r] = widen(w[c][r] & 0xffff), m[2 * r + 1] = widen(w[c][r] >> 16);
#pragma unroll
            for (int j = 0; j < NT; j++) {
              if (j * 8 >= n) break;
#pragma unroll
              for (int p = 0; p < kParts; p++) {
                const unsigned char* b = op + (min(j * 8 + g, n - 1) + p * a.unit) * pitch + (kk + c * 32) * 2 + q * 8;
                const uint2 b0 = *reinterpret_cast<const uint2*>(b), b1 = *reinterpret_cast<const uint2*>(b + 32);
                mma<M>(sum[j][0], m[0], m[2], m[1], m[3], b0.x, b0.y);
                mma<M>(sum[j][1], m[4], m[6], m[5], m[7], b1.x, b1.y);
              }
            }
          }
#pragma unroll
          for (int j = 0; j < NT; j++) {
#pragma unroll
            for (int c = 0; c < 4; c++) acc[j][c] = fmaf(sum[j][0][c] + sum[j][1][c], c < 2 ? fa : fb, acc[j][c]);
          }
        }
      }
      turn = (byte - row_bytes) / kStepBytes;
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * stage);
      if (++stage == a.stages) stage = 0, phase ^= 1;
    }
    if (!kScaled)
#pragma unroll
      for (int j = 0; j < NT; j++)
#pragma unroll
        for (int c = 0; c < 4; c++) acc[j][c] += odd[j][c];
  }
};

template <typename W, typename X, typename M, int COPY, int NT>
__global__ void __launch_bounds__(warps_of(COPY) * 32, 1)
    layer_kernel(const __grid_constant__ LayerArgs a, const __grid_constant__ Maps maps) {
  __shared__ Lists lists;
  __shared__ int scratch[kMaxExperts];
  __shared__ __align__(8) uint64_t bars[2 * (kMaxStages + kMaxRaw)];
  __shared__ int gave_up;
  extern __shared__ __align__(16) unsigned char dyn[];
  Layer<W, X, M, COPY, NT>::run(a, maps.m, lists, scratch, bars, &gave_up, dyn);
}

constexpr int red_bytes(int nt) { return 2 * kConsumers * nt * 128 * 4; }
// Shared memory for the tokens of a unit and the ring.
int room(int nt) { return (int)ctx().smem_optin - (int)sizeof(Lists) - kMaxExperts * 4 - 2048 - red_bytes(nt); }

// Rows of `bytes` as [piece of 128 bytes][row][byte].
CUtensorMap weight_map(const void* w, int64_t rows, int64_t bytes, int stage_row) {
  const cuuint64_t dims[3] = {128, (cuuint64_t)rows, (cuuint64_t)(bytes / 128)}, strides[2] = {(cuuint64_t)bytes, 128};
  const cuuint32_t box[3] = {128, 8, (cuuint32_t)stage_row / 128};
  return byte_map(w, 3, dims, strides, box);
}

template <typename W, typename X, typename M, int COPY, int NT>
void launch(LayerArgs& a, int64_t row, cudaStream_t s) {
  auto kern = layer_kernel<W, X, M, COPY, NT>;
  // as many tokens as fit beside kKeep of stages (at least one, beside two stages), and stages for the rest.
  // 16-bit weights: 8 up to i 3712 and h 7424, 4 for i 6400, 2 for i 14336.  us with 100 KB kept / 66 (two
  // stages of row copies, four of tensor copies): 64 tokens, 2 of 16, 7168 / 2048 519 / 440, 2880 / 2880 282 /
  // 264; 2 of 8, 4096 / 6400 1398 / 1154, 4096 / 14336 7990 / 4790; 8 tokens, 8 of 64, 2048 / 1024 128 / 130.
  // Rows at any byte want two slots beside two stages (132 KB; 100 / 132 / 166: 64 tokens, 2 of 16, 4095 / 2047
  // 939 / 730 / 1664; 4 of 64, 2049 / 641 411 / 411 / 546).
  const int space = room(NT), kStageBytes = stage_bytes(COPY), kKeep = (COPY == kShift ? 132 : 66) * 1024;
  if (row > space - 8192 - 2 * kStageBytes - (COPY == kShift ? kRawBytes : 0)) throw Error(ErrKind::InvalidArgument, "h or i is too large for a token's row to fit shared memory");
  a.unit = (int)std::max<int64_t>(1, std::min<int64_t>({NT * 8, a.tokens, (space - kKeep - (sizeof(W) == 1 ? 8192 : 0)) / row}));
  a.op_bytes = (int)(a.unit * row);
  for (int p = 0; p < 2; p++) {
    const int64_t bytes = (int64_t)(p == 0 ? a.h : a.i) * sizeof(W), n = (bytes + most_bytes(COPY) - 1) / most_bytes(COPY);
    a.row_bytes[p] = (int)((bytes + n * 128 - 1) / (n * 128) * 128);
  }
  a.scale_at = -1;
  if (sizeof(W) == 1) {
    const int64_t hb = (a.h + 127) / 128, ib = (a.i + 127) / 128, jb = (2 * (int64_t)a.i + 127) / 128;
    const int64_t bytes = std::max(hb * jb, hb * ib) * 4;
    if (bytes <= 8192) a.scale_at = a.op_bytes, a.op_bytes += (int)((bytes + 15) / 16 * 16);
  }
  a.stages = COPY == kShift ? 2 : std::min(kMaxStages, (space - a.op_bytes) / kStageBytes);
  a.raw = COPY == kShift ? std::min(kMaxRaw, (space - a.op_bytes - 2 * kStageBytes) / kRawBytes) : 0;
  const size_t smem = (size_t)a.op_bytes + red_bytes(NT) + 1024 + (size_t)a.stages * kStageBytes + (size_t)a.raw * kRawBytes;
  ensure_dynamic_smem((const void*)kern, smem);
  Maps maps{};
  if (COPY == kTensor) {
    maps.m[0] = weight_map(a.e.w_in, 2 * a.e.experts * a.e.i, a.e.h * sizeof(W), a.row_bytes[0]);
    maps.m[1] = weight_map(a.e.w_out, a.e.experts * a.e.h, a.e.i * sizeof(W), a.row_bytes[1]);
  }
  void* args[] = {&a, &maps};
  NDT_CUDA(cudaLaunchCooperativeKernel((const void*)kern, dim3((unsigned)ctx().sm_count), dim3(warps_of(COPY) * 32), args, smem, s));
  count_launch();
}

}  // namespace

void expert_layer(const ExpertArgs& e, cudaStream_t s) {
  if (e.tokens == 0 || e.h == 0) return;
  if (e.experts > kMaxExperts) throw Error(ErrKind::InvalidArgument, "more than 1024 experts");
  // a launch takes as many tokens as its lists hold; more tokens, more launches
  const int64_t step = std::max<int64_t>(1, std::min<int64_t>(kMaxTokens, kMaxSlots / e.top));
  const int64_t most = std::min(step, e.tokens);
  const int64_t ip = (e.i + 7) / 8 * 8;
  const int64_t xs = msize(e.xt), ws_ = msize(e.wt);
  // b first: its rows are read in 16-byte vectors
  Workspace ws((size_t)4 * (most * (e.top * (ip + e.h + 1) + e.experts) + most + 1), s);
  for (int64_t t0 = 0; t0 < e.tokens; t0 += step) {
    LayerArgs a{};
    a.e = e;
    a.tokens = (int)std::min(step, e.tokens - t0);
    a.experts = (int)e.experts, a.top = (int)e.top, a.h = (int)e.h, a.i = (int)e.i, a.ip = (int)ip;
    a.e.x = (const char*)e.x + t0 * e.ldx * xs;
    a.e.y = (char*)e.y + t0 * e.ldy * xs;
    a.e.ids = e.ids + t0 * e.top, a.e.weights = e.weights + t0 * e.top;
    a.b = (float*)ws.p;
    a.o = a.b + most * e.top * ip;
    a.logits = a.o + most * e.top * e.h;
    a.bmax = (unsigned*)(a.logits + most * e.experts);
    a.xmax = a.bmax + most * e.top;
    a.arrived = a.xmax + most;
    a.flag = wait_flag_device();
    const bool vec = e.h * ws_ % 16 == 0 && e.i * ws_ % 16 == 0 && e.h % 8 == 0 && e.ldx % 8 == 0 &&
                     (((uintptr_t)a.e.x | (uintptr_t)e.router | (uintptr_t)e.w_in | (uintptr_t)e.w_out) % 16) == 0;
    const bool pieces = vec && e.h * ws_ % 128 == 0 && e.i * ws_ % 128 == 0 && 2 * e.experts * std::max(e.h, e.i) <= INT32_MAX;
    // tokens' rows start on different banks
    const int pad = e.wt == MType::E4M3 ? 32 : 16;
    a.xpitch = (a.h + 127) / 128 * 256 + pad, a.bpitch = (a.i + 127) / 128 * 256 + pad;
    const int64_t row = std::max((int64_t)a.xpitch, 2 * (int64_t)a.bpitch);
    // An expert's second unit of tokens reads its weights again (from L2): more
    // columns where an expert gets more than 6 tokens on average and 16 fit.  us of
    // 8 / 16 columns, 512 / 256 with 8 experts: 6 tokens each 23.8 / 23.8, 16 each
    // 30.0 / 30.6, 32 each 38.1 / 36.1; 768 / 384 with 64 each 110 / 89.
    const bool many = a.tokens * e.top > 6 * e.experts && a.tokens > 8 && 16 * row <= room(2) - 140 * 1024;
    auto go = [&](auto w, auto x, auto m) {
      using W = decltype(w);
      using X = decltype(x);
      using M = decltype(m);
      if (!vec)
        many ? launch<W, X, M, kShift, 2>(a, row, s) : launch<W, X, M, kShift, 1>(a, row, s);
      else if (!pieces)
        many ? launch<W, X, M, kBulk, 2>(a, row, s) : launch<W, X, M, kBulk, 1>(a, row, s);
      else
        many ? launch<W, X, M, kTensor, 2>(a, row, s) : launch<W, X, M, kTensor, 1>(a, row, s);
    };
    const __nv_bfloat16 bf{};
    const __half hf{};
    if (e.wt == MType::E4M3)
      e.xt == MType::BF16 ? go(__nv_fp8_e4m3{}, bf, hf) : go(__nv_fp8_e4m3{}, hf, hf);
    else if (e.xt == MType::BF16)
      go(bf, bf, bf);
    else
      go(hf, hf, hf);
  }
}

}  // namespace ndt
