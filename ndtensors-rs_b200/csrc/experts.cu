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
// operand and up to 8 tokens a column tile: a lane loads 16 contiguous bytes
// of two weight rows, and since the order of k within a product is free, those
// bytes are its operand fragments as they are (the tokens' fragments are
// loaded with the same order).  In the first product the two rows are the gate
// and the up row of the same output, so silu(gate) * up needs no exchange.
// The warps of a CTA split k and add their parts through shared memory.
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
constexpr int kMaxSlots = 4096;    // (token, chosen expert) pairs of one launch
constexpr int kMaxTokens = 256;
constexpr int kMaxExperts = 1024;
constexpr int kGroup = 8;          // tokens of one router product

struct LayerArgs {
  ExpertArgs e;
  int tokens, experts, top, h, i;
  float* logits;    // [tokens, experts]
  float* b;         // [slots, i]
  float* o;         // [slots, h]
  unsigned* bmax;   // [slots] bits of max |b|
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

// The weights' side of one step of k: a lane's two rows as pairs of M.
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
  int* slots;    // [tokens * top] slots (token * top + place) expert by expert, in order
  int* first;    // [experts + 1]
  int* active;   // experts with tokens
  int n_active;
};

// Choose the experts of every token (every CTA does all of them: a barrier
// would cost more) and list the slots of every expert.
__device__ void route(const LayerArgs& a, int* chosen /* [slots] */, Lists& L, int* scratch) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = (a.experts + 31) / 32;
  for (int t = warp; t < a.tokens; t += kWarps) {
    const float* l = a.logits + (int64_t)t * a.experts;
    float top = -INFINITY, sum = 0.f;
    for (int j = 0; j < per; j++)
      if (j * 32 + lane < a.experts) top = fmaxf(top, __ldcg(l + j * 32 + lane));
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    for (int j = 0; j < per; j++)
      if (j * 32 + lane < a.experts) sum += expf(__ldcg(l + j * 32 + lane) - top);
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    uint32_t taken = 0;  // bit j: expert j * 32 + lane (at most 1024 experts)
    float total = 0.f;
    for (int r = 0; r < a.top; r++) {
      unsigned long long best = 0;
      for (int j = 0; j < per; j++) {
        const int e = j * 32 + lane;
        if (e >= a.experts || (taken >> j & 1)) continue;
        const float f = __ldcg(l + e) + 0.f;  // -0 and 0 are equal
        uint32_t u = __float_as_uint(f);
        u = f != f ? 0xffffffffu : (u & 0x80000000u) ? ~u : u | 0x80000000u;  // NaN above all, as in a sort
        best = max(best, (unsigned long long)u << 32 | (0xffffffffu - e));
      }
      for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
      const int e = (int)(0xffffffffu - (uint32_t)best);
      if ((e & 31) == lane) taken |= 1u << (e >> 5);
      const float p = expf(__ldcg(l + e) - top) / sum;
      total += p;
      if (lane == 0) {
        chosen[t * a.top + r] = e;
        if (blockIdx.x == 0) a.e.ids[t * a.top + r] = e, a.e.weights[t * a.top + r] = p;
      }
    }
    if (a.e.renormalize && blockIdx.x == 0) {
      __syncwarp();
      for (int r = lane; r < a.top; r += 32) a.e.weights[t * a.top + r] /= total;
    }
  }
  __syncthreads();
  // slots of each expert in order: count, scan, place
  const int slots = a.tokens * a.top;
  for (int e = warp; e < a.experts; e += kWarps) {
    int n = 0;
    for (int s = 0; s < slots; s += 32) n += __popc(__ballot_sync(~0u, s + lane < slots && chosen[s + lane] == e));
    if (lane == 0) scratch[e] = n;
  }
  __syncthreads();
  if (warp == 0) {
    int at = 0, act = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane, n = e < a.experts ? scratch[e] : 0;
      int x = n;
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
      }
      if (e < a.experts) L.first[e] = at + x - n;
      const unsigned on = __ballot_sync(~0u, n > 0);
      if (n > 0) L.active[act + __popc(on & ((1u << lane) - 1))] = e;
      act += __popc(on);
      at += __shfl_sync(~0u, x, 31);
    }
    if (lane == 0) L.first[a.experts] = at, scratch[0] = act;
  }
  __syncthreads();
  L.n_active = scratch[0];
  for (int e = warp; e < a.experts; e += kWarps) {
    int at = L.first[e];
    if (L.first[e + 1] == at) continue;
    for (int s = 0; s < slots; s += 32) {
      const bool on = s + lane < slots && chosen[s + lane] == e;
      const unsigned m = __ballot_sync(~0u, on);
      if (on) L.slots[at + __popc(m & ((1u << lane) - 1))] = s + lane;
      at += __popc(m);
    }
  }
  __syncthreads();
}

// W: the weights' type, M: the products' type, VEC: rows are whole 16-byte
// vectors, NT: column tiles of 8 tokens that a product takes at a time.
template <typename W, typename X, typename M, bool VEC, int NT>
__global__ void __launch_bounds__(kThreads, 1) layer_kernel(const LayerArgs a) {
  using S = Step<W, M>;
  constexpr bool kScaled = sizeof(W) == 1;
  constexpr int kBlock = kScaled ? 128 : S::kK;  // k that share a scale
  __shared__ int chosen[kMaxSlots];
  __shared__ int slot_list[kMaxSlots];
  __shared__ int first[kMaxExperts + 1], active[kMaxExperts], scratch[kMaxExperts];
  extern __shared__ __align__(16) float red[];  // [kWarps][NT][32][4]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;  // row (and token) of the lane, quarter of k
  cg::grid_group grid = cg::this_grid();

  // ---- router: a CTA takes one expert and up to 8 tokens
  {
    const int groups = (a.tokens + kGroup - 1) / kGroup;
    for (int u = blockIdx.x; u < a.experts * groups; u += gridDim.x) {
      const int e = u % a.experts, t0 = u / a.experts * kGroup, nt = min(kGroup, a.tokens - t0);
      float acc[kGroup] = {};
      const X* r = (const X*)a.e.router + (int64_t)e * a.h;
      const X* x = (const X*)a.e.x + (int64_t)t0 * a.e.ldx;
      for (int k = threadIdx.x * 8; k < a.h; k += kThreads * 8) {
        const uint4 rv = row16<X, VEC>(r, k, a.h, true);
        const X* re = reinterpret_cast<const X*>(&rv);
#pragma unroll
        for (int t = 0; t < kGroup; t++) {
          const uint4 xv = row16<X, VEC>(x + t * a.e.ldx, k, a.h, t < nt);
          const X* xe = reinterpret_cast<const X*>(&xv);
#pragma unroll
          for (int j = 0; j < 8; j++) acc[t] = fmaf(to_f32<X>(re[j]), to_f32<X>(xe[j]), acc[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < kGroup; t++)
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[t] += __shfl_xor_sync(~0u, acc[t], o);
      if (lane == 0)
#pragma unroll
        for (int t = 0; t < kGroup; t++) red[warp * kGroup + t] = acc[t];
      __syncthreads();
      if (threadIdx.x < nt) {
        float s = 0.f;
        for (int w = 0; w < kWarps; w++) s += red[w * kGroup + threadIdx.x];
        a.logits[(int64_t)(t0 + threadIdx.x) * a.experts + e] = s;
      }
      __syncthreads();
    }
    for (int s = blockIdx.x * kThreads + threadIdx.x; s < a.tokens * a.top; s += gridDim.x * kThreads) a.bmax[s] = 0;
  }
  grid.sync();
  Lists L{slot_list, first, active, 0};
  route(a, chosen, L, scratch);

  // ---- first product: tasks of 8 outputs (their gate and up rows) of one expert
  {
    const int tiles = (a.i + 7) / 8, blocks = (a.h + kBlock - 1) / kBlock;
    const int kb0 = blocks * warp / kWarps, kb1 = blocks * (warp + 1) / kWarps;
    for (int task = blockIdx.x; task < L.n_active * tiles; task += gridDim.x) {
      const int e = L.active[task / tiles], i0 = task % tiles * 8;
      const bool on = i0 + g < a.i;
      const int ra = i0 + g, rb = a.i + i0 + g;
      const W* wa = (const W*)a.e.w_in + ((int64_t)e * 2 * a.i + (on ? ra : 0)) * a.h;
      const W* wb = (const W*)a.e.w_in + ((int64_t)e * 2 * a.i + (on ? rb : 0)) * a.h;
      const int hb = (a.h + 127) / 128, rbs = (2 * a.i + 127) / 128;
      const float* sa = kScaled ? a.e.in_scales + ((int64_t)e * rbs + (on ? ra : 0) / 128) * hb : nullptr;
      const float* sb = kScaled ? a.e.in_scales + ((int64_t)e * rbs + (on ? rb : 0) / 128) * hb : nullptr;
      for (int n0 = L.first[e]; n0 < L.first[e + 1]; n0 += NT * 8) {
        const int n = min(NT * 8, L.first[e + 1] - n0);
        const X* xr[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) xr[j] = (const X*)a.e.x + (int64_t)(j * 8 + g < n ? L.slots[n0 + j * 8 + g] / a.top : 0) * a.e.ldx;
        float acc[NT][4] = {};
        for (int kb = kb0; kb < kb1; kb++) {
          float part[NT][4] = {};
#pragma unroll
          for (int st = 0; st < kBlock / S::kK; st++) {
            const int k = kb * kBlock + st * S::kK + q * S::kPerLane;
            uint32_t pa[S::kPairs], pb[S::kPairs];
            S::pairs(row16<W, VEC>(wa, k, a.h, on), pa);
            S::pairs(row16<W, VEC>(wb, k, a.h, on), pb);
#pragma unroll
            for (int j = 0; j < NT; j++) {
              if (j * 8 >= n) break;
              alignas(16) uint32_t px[S::kPairs];
#pragma unroll
              for (int v = 0; v < S::kPairs / 4; v++)
                *reinterpret_cast<uint4*>(px + 4 * v) = row16<X, VEC>(xr[j], k + 8 * v, a.h, j * 8 + g < n);
#pragma unroll
              for (int v = 0; v < S::kPairs; v += 2) mma<M>(kScaled ? part[j] : acc[j], pa[v], pb[v], pa[v + 1], pb[v + 1], px[v], px[v + 1]);
            }
          }
          if (kScaled) {
            const float fa = sa[kb], fb = sb[kb];
#pragma unroll
            for (int j = 0; j < NT; j++) {
              acc[j][0] = fmaf(part[j][0], fa, acc[j][0]), acc[j][1] = fmaf(part[j][1], fa, acc[j][1]);
              acc[j][2] = fmaf(part[j][2], fb, acc[j][2]), acc[j][3] = fmaf(part[j][3], fb, acc[j][3]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NT; j++)
          *reinterpret_cast<float4*>(red + ((warp * NT + j) * 32 + lane) * 4) = make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
        __syncthreads();
        // accumulator (row g: gate; row g + 8: up; columns 2 q, 2 q + 1) of column tile j
        for (int o = threadIdx.x; o < NT * 64; o += kThreads) {
          const int j = o >> 6, ln = o >> 1 & 31, half = o & 1;
          const int col = j * 8 + (ln & 3) * 2 + half, row = i0 + (ln >> 2);
          float ga = 0.f, up = 0.f;
          for (int w = 0; w < kWarps; w++) {
            const float* p = red + ((w * NT + j) * 32 + ln) * 4 + half;
            ga += p[0], up += p[2];
          }
          if (col < n && row < a.i) {
            const int slot = L.slots[n0 + col];
            const float v = ga / (1.f + expf(-ga)) * up;
            a.b[(int64_t)slot * a.i + row] = v;
            if (std::is_same_v<M, __half>) atomicMax(a.bmax + slot, __float_as_uint(fabsf(v)));
          }
        }
        __syncthreads();
      }
    }
  }
  grid.sync();

  // ---- second product: tasks of 16 rows of one expert
  {
    const int tiles = (a.h + 15) / 16, blocks = (a.i + kBlock - 1) / kBlock;
    const int kb0 = blocks * warp / kWarps, kb1 = blocks * (warp + 1) / kWarps;
    for (int task = blockIdx.x; task < L.n_active * tiles; task += gridDim.x) {
      const int e = L.active[task / tiles], r0 = task % tiles * 16;
      const bool ona = r0 + g < a.h, onb = r0 + g + 8 < a.h;
      const int ra = ona ? r0 + g : 0, rb = onb ? r0 + g + 8 : 0;
      const W* wa = (const W*)a.e.w_out + ((int64_t)e * a.h + ra) * a.i;
      const W* wb = (const W*)a.e.w_out + ((int64_t)e * a.h + rb) * a.i;
      const int ib = (a.i + 127) / 128, rbs = (a.h + 127) / 128;
      const float* sa = kScaled ? a.e.out_scales + ((int64_t)e * rbs + ra / 128) * ib : nullptr;
      const float* sb = kScaled ? a.e.out_scales + ((int64_t)e * rbs + rb / 128) * ib : nullptr;
      for (int n0 = L.first[e]; n0 < L.first[e + 1]; n0 += NT * 8) {
        const int n = min(NT * 8, L.first[e + 1] - n0);
        const float* br[NT];
        float up[NT], down[NT][2];
#pragma unroll
        for (int j = 0; j < NT; j++) {
          const int slot = L.slots[n0 + min(j * 8 + g, n - 1)];
          br[j] = a.b + (int64_t)slot * a.i;
          up[j] = 1.f, down[j][0] = down[j][1] = 1.f;
          if constexpr (std::is_same_v<M, __half>) {
            // 2^-x of the slot's largest value, and back for the lane's two result columns
            auto power = [&](int s, bool inverse) {
              const int ex = (int)(__ldcg(a.bmax + s) >> 23) - 127;
              const int c = ex < -100 || ex > 127 ? 0 : min(ex, 126);  // tiny, infinite or NaN: as it is
              return __uint_as_float((uint32_t)(127 + (inverse ? c : -c)) << 23);
            };
            up[j] = power(slot, false);
            for (int c = 0; c < 2; c++) down[j][c] = power(L.slots[n0 + min(j * 8 + 2 * q + c, n - 1)], true);
          }
        }
        float acc[NT][4] = {};
        for (int kb = kb0; kb < kb1; kb++) {
          float part[NT][4] = {};
#pragma unroll
          for (int st = 0; st < kBlock / S::kK; st++) {
            const int k = kb * kBlock + st * S::kK + q * S::kPerLane;
            uint32_t pa[S::kPairs], pb[S::kPairs];
            S::pairs(row16<W, VEC>(wa, k, a.i, ona), pa);
            S::pairs(row16<W, VEC>(wb, k, a.i, onb), pb);
#pragma unroll
            for (int j = 0; j < NT; j++) {
              if (j * 8 >= n) break;
#pragma unroll
              for (int v = 0; v < S::kPairs; v += 2) {
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int p = 0; p < 2; p++) {
                  const int kk = k + 2 * (v + p);
                  float f0 = 0.f, f1 = 0.f;
                  if (j * 8 + g < n) {
                    if (kk < a.i) f0 = __ldcg(br[j] + kk) * up[j];
                    if (kk + 1 < a.i) f1 = __ldcg(br[j] + kk + 1) * up[j];
                  }
                  hi[p] = pack2<M>(f0, f1);
                  const float2 h = unpack2<M>(hi[p]);
                  // (an infinite high part stands alone: no inf - inf)
                  lo[p] = pack2<M>(isinf(h.x) ? 0.f : f0 - h.x, isinf(h.y) ? 0.f : f1 - h.y);
                }
                mma<M>(kScaled ? part[j] : acc[j], pa[v], pb[v], pa[v + 1], pb[v + 1], hi[0], hi[1]);
                mma<M>(kScaled ? part[j] : acc[j], pa[v], pb[v], pa[v + 1], pb[v + 1], lo[0], lo[1]);
              }
            }
          }
          if (kScaled) {
            const float fa = sa[kb], fb = sb[kb];
#pragma unroll
            for (int j = 0; j < NT; j++) {
              acc[j][0] = fmaf(part[j][0], fa, acc[j][0]), acc[j][1] = fmaf(part[j][1], fa, acc[j][1]);
              acc[j][2] = fmaf(part[j][2], fb, acc[j][2]), acc[j][3] = fmaf(part[j][3], fb, acc[j][3]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NT; j++)
          *reinterpret_cast<float4*>(red + ((warp * NT + j) * 32 + lane) * 4) =
              make_float4(acc[j][0] * down[j][0], acc[j][1] * down[j][1], acc[j][2] * down[j][0], acc[j][3] * down[j][1]);
        __syncthreads();
        for (int o = threadIdx.x; o < NT * 128; o += kThreads) {
          const int j = o >> 7, c = o >> 5 & 3, ln = o & 31;
          const int col = j * 8 + (ln & 3) * 2 + (c & 1), row = r0 + (ln >> 2) + (c & 2) * 4;
          float s = 0.f;
          for (int w = 0; w < kWarps; w++) s += red[((w * NT + j) * 32 + ln) * 4 + c];
          if (col < n && row < a.h) a.o[(int64_t)L.slots[n0 + col] * a.h + row] = s;
        }
        __syncthreads();
      }
    }
  }
  grid.sync();

  // ---- the tokens' sums over their experts, in the order of choice
  for (int64_t u = blockIdx.x * (int64_t)kThreads + threadIdx.x; u < (int64_t)a.tokens * a.h; u += (int64_t)gridDim.x * kThreads) {
    const int t = (int)(u / a.h), c = (int)(u - (int64_t)t * a.h);
    float s = 0.f;
    for (int r = 0; r < a.top; r++) s += __ldcg(a.e.weights + t * a.top + r) * __ldcg(a.o + ((int64_t)t * a.top + r) * a.h + c);
    ((X*)a.e.y)[(int64_t)t * a.e.ldy + c] = from_f32<X>(s);
  }
}

template <typename W, typename X, typename M, bool VEC, int NT>
void launch(LayerArgs& a, cudaStream_t s) {
  auto kern = layer_kernel<W, X, M, VEC, NT>;
  const size_t smem = (size_t)kWarps * NT * 32 * 16;
  ensure_dynamic_smem((const void*)kern, smem);
  void* args[] = {&a};
  NDT_CUDA(cudaLaunchCooperativeKernel((const void*)kern, dim3((unsigned)ctx().sm_count), dim3(kThreads), args, smem, s));
  count_launch();
}

}  // namespace

void expert_layer(const ExpertArgs& e, cudaStream_t s) {
  if (e.tokens == 0 || e.h == 0) return;
  if (e.experts > kMaxExperts) throw Error(ErrKind::InvalidArgument, "expert_layer: more than 1024 experts");
  // a launch takes as many tokens as its lists hold; more tokens, more launches
  const int64_t step = std::max<int64_t>(1, std::min<int64_t>(kMaxTokens, kMaxSlots / e.top));
  const int64_t most = std::min(step, e.tokens);
  const size_t xs = msize(e.xt);
  Workspace ws((size_t)most * 4 * (e.experts + e.top * (e.i + e.h + 1)), s);
  for (int64_t t0 = 0; t0 < e.tokens; t0 += step) {
    LayerArgs a{};
    a.e = e;
    a.tokens = (int)std::min(step, e.tokens - t0);
    a.experts = (int)e.experts, a.top = (int)e.top, a.h = (int)e.h, a.i = (int)e.i;
    a.e.x = (const char*)e.x + t0 * e.ldx * xs;
    a.e.y = (char*)e.y + t0 * e.ldy * xs;
    a.e.ids = e.ids + t0 * e.top, a.e.weights = e.weights + t0 * e.top;
    a.logits = (float*)ws.p;
    a.b = a.logits + most * e.experts;
    a.o = a.b + most * e.top * e.i;
    a.bmax = (unsigned*)(a.o + most * e.top * e.h);
    const int ws_ = msize(e.wt);
    const bool vec = e.h * ws_ % 16 == 0 && e.i * ws_ % 16 == 0 && e.h % 8 == 0 && e.ldx % 8 == 0 &&
                     (((uintptr_t)a.e.x | (uintptr_t)e.router | (uintptr_t)e.w_in | (uintptr_t)e.w_out) % 16) == 0;
    auto go = [&](auto w, auto x) {
      using W = decltype(w);
      using X = decltype(x);
      if (a.tokens <= 8)
        vec ? launch<W, X, X, true, 1>(a, s) : launch<W, X, X, false, 1>(a, s);
      else
        vec ? launch<W, X, X, true, 4>(a, s) : launch<W, X, X, false, 4>(a, s);
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
