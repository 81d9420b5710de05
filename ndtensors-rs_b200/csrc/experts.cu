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
// Products run on the warp-level tensor cores with the weights as the 16-row
// operand and up to 8 tokens a column tile: a lane copies 16 contiguous bytes
// of two weight rows, and since the order of k within a product is free, those
// bytes are its operand fragments as they are (the tokens' fragments are
// loaded with the same order).  In the first product the two rows are the gate
// and the up row of the same output, so silu(gate) * up needs no exchange.
// Four warps share a tile of 16 rows, split its k and add their parts through
// shared memory (with all 16 warps on a tile the barrier and the sums cost as
// much as the product).
//
// The weights stream through a ring of cp.async copies in shared memory, each
// lane reading back only what it copied itself, so no barrier stands between a
// copy and its use.  The ring runs across tasks, and from the first product
// into the second before the grid barrier between them.
//
// All sums are in 32 bits.  The activations b enter the second product as the
// sum of two 16-bit numbers (16 or 22 bits of mantissa), so it loses nothing
// against a 32-bit b; for float16 each row of b is scaled by a power of two
// first, since b may be out of that type's range.
#include <cooperative_groups.h>

#include <algorithm>

#include "model_ops.h"

namespace ndt {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kTeam = 4;             // warps that share a tile
constexpr int kTeams = kWarps / kTeam;
constexpr int kMaxSlots = 4096;    // (token, chosen expert) pairs of one launch
constexpr int kMaxTokens = 256;
constexpr int kMaxExperts = 1024;
constexpr int kGroup = 8;          // tokens of one router product
constexpr int kMaxUnits = kMaxExperts + kMaxSlots / 32;

struct LayerArgs {
  ExpertArgs e;
  int tokens, experts, top, h, i;
  int ip;           // i rounded up to 8: the pitch of b's rows
  float* logits;    // [tokens, experts]
  void* b;          // [slots, 2, ip] bf16 high and low parts, or [slots, ip] floats (float16 layers)
  float* o;         // [slots, h]
  unsigned* bmax;   // [slots] bits of max |b|
  unsigned* done;   // [row tiles of w_out] parts of a tile that are finished
};

template <typename M>
__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<M, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
// Two 8-bit weights (the low 16 bits of w) as a pair of M: exact in both types.
template <typename M>
__device__ __forceinline__ uint32_t widen(uint32_t w) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3);
  if constexpr (std::is_same_v<M, __half>) return *reinterpret_cast<const uint32_t*>(&h);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return pack2<__nv_bfloat16>(f.x, f.y);
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
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes from p, of which n elements are the row's, into shared memory: an
// asynchronous copy where rows are whole vectors.
template <typename T, bool VEC>
__device__ __forceinline__ void copy16(void* dst, const T* p, int n, bool on) {
  if constexpr (VEC) {
    const bool in = on && n > 0;
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(p), "r"(in ? 16 : 0) : "memory");
  } else {
    *reinterpret_cast<uint4*>(dst) = row16<T, false>(p, 0, n, on);
  }
}

// The weights' side of one step of k: a lane's 16 bytes of a row as pairs of M.
template <typename W, typename M>
struct Step {
  static constexpr int kPerLane = 16 / sizeof(W);  // k of a lane
  static constexpr int kK = 4 * kPerLane;          // k of the warp
  static constexpr int kPairs = kPerLane / 2;
  __device__ static __forceinline__ void pairs(const uint4& v, uint32_t* p) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (sizeof(W) == 2) {
#pragma unroll
      for (int j = 0; j < 4; j++) p[j] = w[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) p[2 * j] = widen<M>(w[j] & 0xffff), p[2 * j + 1] = widen<M>(w[j] >> 16);
    }
  }
};

struct Lists {
  uint16_t chosen[kMaxSlots];     // the expert of each slot (token * top + place)
  uint16_t slots[kMaxSlots];      // slots expert by expert, in order
  int first[kMaxExperts + 1];     // where an expert's slots start
  uint16_t unit_expert[kMaxUnits];  // an expert with up to 8 NT of its slots
  uint16_t unit_first[kMaxUnits];   // ... from this place of `slots` on
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
__device__ __forceinline__ void choose(const LayerArgs& a, int t, Lists& L) {
  const int lane = threadIdx.x & 31;
  const float* l = a.logits + (int64_t)t * a.experts;
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
template <int NT>
__device__ __forceinline__ void route(const LayerArgs& a, Lists& L, int* scratch) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int t = warp; t < a.tokens; t += kWarps) {
    if (a.experts <= 64)
      choose<2>(a, t, L);
    else if (a.experts <= 256)
      choose<8>(a, t, L);
    else
      choose<32>(a, t, L);
  }
  __syncthreads();
  const int slots = a.tokens * a.top;
  for (int e = warp; e < a.experts; e += kWarps) {
    int n = 0;
    for (int s = 0; s < slots; s += 32) n += __popc(__ballot_sync(~0u, s + lane < slots && L.chosen[s + lane] == e));
    if (lane == 0) scratch[e] = n;
  }
  __syncthreads();
  if (warp == 0) {
    int at = 0, units = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane, n = e < a.experts ? scratch[e] : 0, u = (n + 8 * NT - 1) / (8 * NT);
      int x = n, y = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int p = __shfl_up_sync(~0u, x, o), q = __shfl_up_sync(~0u, y, o);
        if (lane >= o) x += p, y += q;
      }
      if (e < a.experts) L.first[e] = at + x - n;
      for (int k = 0; k < u; k++) {
        L.unit_expert[units + y - u + k] = (uint16_t)e;
        L.unit_first[units + y - u + k] = (uint16_t)(at + x - n + k * 8 * NT);
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

// Router products: a CTA takes RE experts and up to 8 tokens.
template <typename X, bool VEC, int RE>
__device__ __forceinline__ void router(const LayerArgs& a, float* red) {
  static_assert(RE * kGroup <= 32, "");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int groups = (a.tokens + kGroup - 1) / kGroup, es = (a.experts + RE - 1) / RE;
  for (int u = blockIdx.x; u < es * groups; u += gridDim.x) {
    const int e0 = u % es * RE, t0 = u / es * kGroup, nt = min(kGroup, a.tokens - t0), ne = min(RE, a.experts - e0);
    float acc[32] = {};
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
#pragma unroll
        for (int j = 0; j < RE; j++) {
          const X* re = reinterpret_cast<const X*>(&rv[j]);
#pragma unroll
          for (int c = 0; c < 8; c++) acc[j * kGroup + t] = fmaf(to_f32<X>(re[c]), to_f32<X>(xe[c]), acc[j * kGroup + t]);
        }
      }
    }
    red[warp * 32 + lane] = transpose_sum(acc);
    __syncthreads();
    if (warp == 0) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; w++) s += red[w * 32 + lane];
      const int j = lane / kGroup, t = lane % kGroup;
      if (j < ne && t < nt) a.logits[(int64_t)(t0 + t) * a.experts + e0 + j] = s;
    }
    __syncthreads();
  }
}

// W: the weights' type, M: x's and the products' type, VEC: rows are whole
// 16-byte vectors, NT: column tiles of 8 tokens that a product takes at a time.
template <typename W, typename M, bool VEC, int NT>
struct Layer {
  using S = Step<W, M>;
  static constexpr bool kScaled = sizeof(W) == 1;
  static constexpr bool kHalf = std::is_same_v<M, __half>;
  static constexpr int kRing = NT == 1 ? 8 : 6;          // steps in flight
  static constexpr int kSlot = 2 * 512 + (kScaled ? 64 : 0);  // bytes of a warp's step: two rows a lane, two scales a row
  static constexpr int kRed = kWarps * NT * 128;         // floats of the teams' parts
  static constexpr size_t kSmem = (size_t)kWarps * kRing * kSlot + 2 * kRed * 4;

  // The stream of steps that a warp copies ahead of their use.  product 0:
  // outputs 8 tile + g, their gate and up rows of w_in; product 1: rows
  // 16 tile + g and + 8 of w_out.
  struct Feed {
    int product, task, step, slot;
    const W *a, *b;  // the lane's two rows
    const float *sa, *sb;
    bool ona, onb;
  };

  __device__ static void run(const LayerArgs& a, Lists& L, int* scratch, unsigned char* dyn) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int team = warp / kTeam, part = warp % kTeam;
    const int g = lane >> 2, q = lane & 3;  // row (and token) of the lane, quarter of k
    unsigned char* ring = dyn + (size_t)warp * kRing * kSlot;
    float* red = reinterpret_cast<float*>(dyn + (size_t)kWarps * kRing * kSlot);
    cg::grid_group grid = cg::this_grid();

    if (a.tokens <= 8)
      router<M, VEC, 1>(a, red);
    else
      router<M, VEC, 4>(a, red);
    const int tiles0 = (a.i + 7) / 8, tiles1 = (a.h + 15) / 16;
    for (int s = blockIdx.x * kThreads + threadIdx.x; s < max(a.tokens * a.top, tiles1); s += gridDim.x * kThreads) {
      if (s < a.tokens * a.top) a.bmax[s] = 0;
      if (s < tiles1) a.done[s] = 0;
    }
    grid.sync();
    route<NT>(a, L, scratch);

    // this warp's steps of k in each product; the tiles are dealt to the CTAs in even runs, to their teams in turn
    const int steps0 = (a.h + S::kK - 1) / S::kK, steps1 = (a.i + S::kK - 1) / S::kK;
    const int lo0 = steps0 * part / kTeam, hi0 = steps0 * (part + 1) / kTeam;
    const int lo1 = steps1 * part / kTeam, hi1 = steps1 * (part + 1) / kTeam;
    auto share = [&](int tasks, int cta) { return (int)((int64_t)tasks * cta / gridDim.x); };
    const int tasks0 = L.units * tiles0, tasks1 = L.units * tiles1;
    const int first0 = share(tasks0, blockIdx.x) + team, end0 = share(tasks0, blockIdx.x + 1);
    const int first1 = share(tasks1, blockIdx.x) + team, end1 = share(tasks1, blockIdx.x + 1);

    Feed f;
    f.product = 0, f.task = first0, f.slot = 0;
    auto settle = [&] {  // onto the next task that has steps for this warp
      if (f.product == 0 && (f.task >= end0 || lo0 == hi0)) f.product = 1, f.task = first1;
      if (f.product == 1 && (f.task >= end1 || lo1 == hi1)) f.product = 2;
      if (f.product == 2) return;
      const bool p0 = f.product == 0;
      f.step = p0 ? lo0 : lo1;
      const int tiles = p0 ? tiles0 : tiles1, u = f.task / tiles, tile = f.task - u * tiles;
      const int64_t expert = L.unit_expert[u];
      const int ra = p0 ? tile * 8 + g : tile * 16 + g, n = p0 ? 2 * a.i : a.h, k = p0 ? a.h : a.i;
      f.ona = ra < (p0 ? a.i : a.h);
      f.onb = p0 ? f.ona : ra + 8 < a.h;
      const int qa = f.ona ? ra : 0, qb = !f.onb ? 0 : p0 ? a.i + ra : ra + 8;
      const W* w = (const W*)(p0 ? a.e.w_in : a.e.w_out) + expert * n * k + f.step * S::kK + q * S::kPerLane;
      f.a = w + (int64_t)qa * k, f.b = w + (int64_t)qb * k;
      if (kScaled) {
        const int kb = (k + 127) / 128;
        const float* sc = (p0 ? a.e.in_scales : a.e.out_scales) + expert * ((n + 127) / 128) * kb;
        f.sa = sc + (qa >> 7) * kb, f.sb = sc + (qb >> 7) * kb;
      }
    };
    auto feed = [&] {  // copy the next step; an empty group at the end of the stream
      if (f.product < 2) {
        unsigned char* at = ring + f.slot * kSlot + lane * 16;
        const int n = (f.product == 0 ? a.h : a.i) - (f.step * S::kK + q * S::kPerLane);  // elements from here to the row's end
        copy16<W, VEC>(at, f.a, n, f.ona);
        copy16<W, VEC>(at + 512, f.b, n, f.onb);
        f.a += S::kK, f.b += S::kK;
        if (kScaled && q == 0) {
          const int kb = f.step * S::kK / 128;
          const uint32_t sc = smem_u32(ring + f.slot * kSlot + 1024 + g * 8);
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sc), "l"(f.sa + kb) : "memory");
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sc + 4), "l"(f.sb + kb) : "memory");
        }
        if (++f.slot == kRing) f.slot = 0;
        if (++f.step == (f.product == 0 ? hi0 : hi1)) {
          f.task += kTeams;
          settle();
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    settle();
    for (int p = 0; p < kRing - 1; p++) feed();
    int slot = 0, parity = 0;
    // take the oldest step: its two rows' pairs and scales
    auto take = [&](uint32_t* pa, uint32_t* pb, float& fa, float& fb) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kRing - 2) : "memory");
      if (kScaled) __syncwarp();  // the scales were copied by the row's first lane (and the last ones have been read)
      const unsigned char* at = ring + slot * kSlot;
      S::pairs(*reinterpret_cast<const uint4*>(at + lane * 16), pa);
      S::pairs(*reinterpret_cast<const uint4*>(at + 512 + lane * 16), pb);
      if (kScaled) {
        const float2 sc = *reinterpret_cast<const float2*>(at + 1024 + g * 8);
        fa = sc.x, fb = sc.y;
      }
      if (++slot == kRing) slot = 0;
      feed();
    };
    auto add_scaled = [&](float* acc, const float* part, float fa, float fb) {
      acc[0] = fmaf(part[0], fa, acc[0]), acc[1] = fmaf(part[1], fa, acc[1]);
      acc[2] = fmaf(part[2], fb, acc[2]), acc[3] = fmaf(part[3], fb, acc[3]);
    };
    auto park = [&](float (*acc)[4]) {  // this warp's part of the tile, for its team
      float* at = red + parity * kRed + team * kTeam * NT * 128;
#pragma unroll
      for (int j = 0; j < NT; j++)
        *reinterpret_cast<float4*>(at + ((part * NT + j) * 32 + lane) * 4) = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(kTeam * 32) : "memory");  // one a tile: two buffers alternate
      parity ^= 1;
      return (const float*)at;
    };

    // ---- first product: tiles of 8 outputs of one expert
    for (int task = first0; task < end0; task += kTeams) {
      const int u = task / tiles0, i0 = (task - u * tiles0) * 8;
      const int e = L.unit_expert[u], n0 = L.unit_first[u], n = min(NT * 8, L.first[e + 1] - n0);
      const M* xr[NT];
#pragma unroll
      for (int j = 0; j < NT; j++) xr[j] = (const M*)a.e.x + (int64_t)(j * 8 + g < n ? L.slots[n0 + j * 8 + g] / a.top : 0) * a.e.ldx;
      float acc[NT][4] = {};
      for (int s = lo0; s < hi0; s++) {
        const int k = s * S::kK + q * S::kPerLane;
        uint32_t pa[S::kPairs], pb[S::kPairs];
        float fa, fb;
        take(pa, pb, fa, fb);
#pragma unroll
        for (int j = 0; j < NT; j++) {
          if (j * 8 >= n) break;
          alignas(16) uint32_t px[S::kPairs];
#pragma unroll
          for (int v = 0; v < S::kPairs / 4; v++)
            *reinterpret_cast<uint4*>(px + 4 * v) = row16<M, VEC>(xr[j], k + 8 * v, a.h, j * 8 + g < n);
          float sum[4] = {};
          float* to = kScaled ? sum : acc[j];
#pragma unroll
          for (int v = 0; v < S::kPairs; v += 2) mma<M>(to, pa[v], pb[v], pa[v + 1], pb[v + 1], px[v], px[v + 1]);
          if (kScaled) add_scaled(acc[j], sum, fa, fb);
        }
      }
      const float* parts = park(acc);
      // accumulator (row g: gate; row g + 8: up; columns 2 q, 2 q + 1) of column tile j
      for (int o = part * 32 + lane; o < NT * 64; o += kTeam * 32) {
        const int j = o >> 6, ln = o >> 1 & 31, half = o & 1;
        const int col = j * 8 + (ln & 3) * 2 + half, row = i0 + (ln >> 2);
        if (col >= n) continue;
        float ga = 0.f, up = 0.f;
#pragma unroll
        for (int w = 0; w < kTeam; w++) {
          const float* p = parts + ((w * NT + j) * 32 + ln) * 4 + half;
          ga += p[0], up += p[2];
        }
        const int64_t slot_row = L.slots[n0 + col];
        const float v = ga / (1.f + expf(-ga)) * up;  // rows past i: 0, the padding of b
        if constexpr (kHalf) {
          ((float*)a.b)[slot_row * a.ip + row] = v;
          atomicMax(a.bmax + slot_row, __float_as_uint(fabsf(v)));
        } else {
          const __nv_bfloat16 hi = __float2bfloat16_rn(v);
          const float hf = __bfloat162float(hi);
          __nv_bfloat16* p = (__nv_bfloat16*)a.b + slot_row * 2 * a.ip + row;
          p[0] = hi;
          p[a.ip] = __float2bfloat16_rn(isinf(hf) ? 0.f : v - hf);  // an infinite high part stands alone
        }
      }
    }
    grid.sync();

    // ---- second product: tiles of 16 rows of one expert
    for (int task = first1; task < end1; task += kTeams) {
      const int u = task / tiles1, tile = task - u * tiles1, r0 = tile * 16;
      const int e = L.unit_expert[u], n0 = L.unit_first[u], n = min(NT * 8, L.first[e + 1] - n0);
      const char* br[NT];
      float down[NT][2], up[NT];
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const int sl = L.slots[n0 + min(j * 8 + g, n - 1)];
        br[j] = (const char*)a.b + (int64_t)sl * a.ip * 4;
        if constexpr (kHalf) {
          // 2^-x of the slot's largest value, and back for the lane's two result columns
          auto power = [&](int at, int sign) {
            const int ex = (int)(a.bmax[at] >> 23) - 127;
            const int c = ex < -100 || ex > 127 ? 0 : min(ex, 126);  // tiny, infinite or NaN: as it is
            return __uint_as_float((uint32_t)(127 + sign * c) << 23);
          };
          up[j] = power(sl, -1);
          for (int c = 0; c < 2; c++) down[j][c] = power(L.slots[n0 + min(j * 8 + 2 * q + c, n - 1)], 1);
        }
      }
      float acc[NT][4] = {};
      for (int s = lo1; s < hi1; s++) {
        const int k = s * S::kK + q * S::kPerLane;
        uint32_t pa[S::kPairs], pb[S::kPairs];
        float fa, fb;
        take(pa, pb, fa, fb);
#pragma unroll
        for (int j = 0; j < NT; j++) {
          if (j * 8 >= n) break;
          float sum[4] = {};
          float* to = kScaled ? sum : acc[j];
#pragma unroll
          for (int v = 0; v < S::kPairs / 4; v++) {
            const int kk = k + 8 * v;
            const bool on = j * 8 + g < n && kk < a.ip;
            alignas(16) uint32_t hi[4] = {}, lo[4] = {};
            if constexpr (kHalf) {
              const float4* p = reinterpret_cast<const float4*>((const float*)br[j] + kk);
              const float4 f0 = on ? p[0] : make_float4(0, 0, 0, 0), f1 = on ? p[1] : make_float4(0, 0, 0, 0);
              const float x[8] = {f0.x, f0.y, f0.z, f0.w, f1.x, f1.y, f1.z, f1.w};
#pragma unroll
              for (int c = 0; c < 4; c++) {
                const float y0 = x[2 * c] * up[j], y1 = x[2 * c + 1] * up[j];
                hi[c] = pack2<M>(y0, y1);
                const float2 hf = unpack2<M>(hi[c]);
                // (an infinite high part stands alone: no inf - inf)
                lo[c] = pack2<M>(isinf(hf.x) ? 0.f : y0 - hf.x, isinf(hf.y) ? 0.f : y1 - hf.y);
              }
            } else if (on) {
              const __nv_bfloat16* p = (const __nv_bfloat16*)br[j] + kk;
              *reinterpret_cast<uint4*>(hi) = *reinterpret_cast<const uint4*>(p);
              *reinterpret_cast<uint4*>(lo) = *reinterpret_cast<const uint4*>(p + a.ip);
            }
#pragma unroll
            for (int c = 0; c < 4; c += 2) {
              const int m = 4 * v + c;
              mma<M>(to, pa[m], pb[m], pa[m + 1], pb[m + 1], hi[c], hi[c + 1]);
              mma<M>(to, pa[m], pb[m], pa[m + 1], pb[m + 1], lo[c], lo[c + 1]);
            }
          }
          if (kScaled) add_scaled(acc[j], sum, fa, fb);
        }
      }
      if constexpr (kHalf) {
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
          for (int c = 0; c < 4; c++) acc[j][c] *= down[j][c & 1];
      }
      const float* parts = park(acc);
      // warp `part` finishes accumulator `part` of every lane
#pragma unroll
      for (int j = 0; j < NT; j++) {
        const int col = j * 8 + (lane & 3) * 2 + (part & 1), row = r0 + (lane >> 2) + (part & 2) * 4;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kTeam; w++) s += parts[((w * NT + j) * 32 + lane) * 4 + part];
        if (col < n && row < a.h) a.o[(int64_t)L.slots[n0 + col] * a.h + row] = s;
      }
      if (NT == 1) {
        // the warp that finishes a row tile's last part (of kTeam a unit) sums the tokens' experts there
        __threadfence();
        __syncwarp();
        unsigned before = 0;
        if (lane == 0) before = atomicAdd(a.done + tile, 1u);
        before = __shfl_sync(~0u, before, 0);
        if (before == (unsigned)(kTeam * L.units - 1)) {
          __threadfence();
          for (int c = lane; c < a.tokens * 16; c += 32) combine(a, c >> 4, r0 + (c & 15));
        }
      }
    }
    if (NT > 1) {
      grid.sync();
      const int64_t all = (int64_t)a.tokens * a.h;
      for (int64_t c = blockIdx.x * (int64_t)kThreads + threadIdx.x; c < all; c += (int64_t)gridDim.x * kThreads) {
        const int t = (int)(c / a.h);
        combine(a, t, (int)(c - (int64_t)t * a.h));
      }
    }
  }

  // A token's sum over its experts, in the order of choice.
  __device__ static __forceinline__ void combine(const LayerArgs& a, int t, int row) {
    if (row >= a.h) return;
    float s = 0.f;
#pragma unroll 4
    for (int r = 0; r < a.top; r++) s += __ldcg(a.e.weights + t * a.top + r) * __ldcg(a.o + ((int64_t)t * a.top + r) * a.h + row);
    ((M*)a.e.y)[(int64_t)t * a.e.ldy + row] = from_f32<M>(s);
  }
};

template <typename W, typename M, bool VEC, int NT>
__global__ void __launch_bounds__(kThreads, 1) layer_kernel(const LayerArgs a) {
  __shared__ Lists lists;
  __shared__ int scratch[kMaxExperts];
  extern __shared__ __align__(16) unsigned char dyn[];
  Layer<W, M, VEC, NT>::run(a, lists, scratch, dyn);
}

template <typename W, typename M, bool VEC, int NT>
void launch(LayerArgs& a, cudaStream_t s) {
  auto kern = layer_kernel<W, M, VEC, NT>;
  constexpr size_t smem = Layer<W, M, VEC, NT>::kSmem;
  ensure_dynamic_smem((const void*)kern, smem);
  void* args[] = {&a};
  NDT_CUDA(cudaLaunchCooperativeKernel((const void*)kern, dim3((unsigned)ctx().sm_count), dim3(kThreads), args, smem, s));
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
  Workspace ws((size_t)4 * (most * (e.top * (ip + e.h + 1) + e.experts) + (e.h + 15) / 16), s);
  for (int64_t t0 = 0; t0 < e.tokens; t0 += step) {
    LayerArgs a{};
    a.e = e;
    a.tokens = (int)std::min(step, e.tokens - t0);
    a.experts = (int)e.experts, a.top = (int)e.top, a.h = (int)e.h, a.i = (int)e.i, a.ip = (int)ip;
    a.e.x = (const char*)e.x + t0 * e.ldx * xs;
    a.e.y = (char*)e.y + t0 * e.ldy * xs;
    a.e.ids = e.ids + t0 * e.top, a.e.weights = e.weights + t0 * e.top;
    a.b = ws.p;
    a.o = (float*)ws.p + most * e.top * ip;
    a.logits = a.o + most * e.top * e.h;
    a.bmax = (unsigned*)(a.logits + most * e.experts);
    a.done = a.bmax + most * e.top;
    const bool vec = e.h * ws_ % 16 == 0 && e.i * ws_ % 16 == 0 && e.h % 8 == 0 && e.ldx % 8 == 0 &&
                     (((uintptr_t)a.e.x | (uintptr_t)e.router | (uintptr_t)e.w_in | (uintptr_t)e.w_out) % 16) == 0;
    auto go = [&](auto w, auto x) {
      using W = decltype(w);
      using M = decltype(x);
      if (a.tokens <= 8)
        vec ? launch<W, M, true, 1>(a, s) : launch<W, M, false, 1>(a, s);
      else
        vec ? launch<W, M, true, 4>(a, s) : launch<W, M, false, 4>(a, s);
    };
    if (e.wt == MType::E4M3)
      e.xt == MType::BF16 ? go(__nv_fp8_e4m3{}, __nv_bfloat16{}) : go(__nv_fp8_e4m3{}, __half{});
    else if (e.xt == MType::BF16)
      go(__nv_bfloat16{}, __nv_bfloat16{});
    else
      go(__half{}, __half{});
  }
}

}  // namespace ndt
