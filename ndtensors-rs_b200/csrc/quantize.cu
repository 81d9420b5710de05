// 8-bit block quantisation, and the packing of 8-bit operands.
//
// For a block b of x (block_rows x 128 elements, cut at the matrix edge):
//   amax = max(2^-100, max |x| over the finite x of b)
//   s_b  = amax / F, rounded to 32 bits           (F = 448 e4m3, 57344 e5m2)
//   q    = x / s_b, rounded to 32 bits, then to 8 bits (nearest, ties to even)
// The quotient of a finite x never exceeds F by more than its rounding, and
// saturates there.  NaN becomes NaN; an infinity becomes the type's (e5m2) or
// NaN (e4m3 has none), so an overflow upstream stays visible.  The lower
// bound on amax makes the scale of a zero block a normal number and q zero.
// IEEE divisions, not products with a reciprocal: q is then a function of the
// block alone that any caller can restate.
#include <algorithm>

#include "model_ops.h"

namespace ndt {
namespace {

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100
constexpr int kTile = 128;
constexpr int kThreads = 256;

template <typename Q>
__device__ __forceinline__ float fmax8();
template <>
__device__ __forceinline__ float fmax8<__nv_fp8_e4m3>() { return 448.f; }
template <>
__device__ __forceinline__ float fmax8<__nv_fp8_e5m2>() { return 57344.f; }

// Four elements as 8-bit codes, the first in the lowest byte.
template <typename Q>
__device__ __forceinline__ uint32_t round8(float x0, float x1, float x2, float x3, float s) {
  constexpr bool kE4 = std::is_same_v<Q, __nv_fp8_e4m3>;
  constexpr __nv_fp8_interpretation_t kind = kE4 ? __NV_E4M3 : __NV_E5M2;
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x0 / s, x1 / s), __NV_SATFINITE, kind);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x2 / s, x3 / s), __NV_SATFINITE, kind);
  uint32_t w = lo | hi << 16;
  const float sum = fabsf(x0) + fabsf(x1) + fabsf(x2) + fabsf(x3);
  if (!(sum <= 3.402823466e38f)) {  // rare: an element is not finite (or their sum is not)
    const float x[4] = {x0, x1, x2, x3};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (fabsf(x[j]) <= 3.402823466e38f) continue;
      const uint32_t code = kE4 || x[j] != x[j] ? 0x7fu : x[j] > 0 ? 0x7cu : 0xfcu;
      w = (w & ~(0xffu << (8 * j))) | code << (8 * j);
    }
  }
  return w;
}
__device__ __forceinline__ float mag(float x) {
  x = fabsf(x);
  return x <= 3.402823466e38f ? x : 0.f;  // infinities and NaN do not count
}

struct QArgs {
  const void* x;
  int64_t rows, cols, rs, cs;
  QuantOut q, t;
};

// One 128 x 128 tile a CTA.  A warp takes 16 rows, a lane 4 columns: a row's
// maximum is a warp reduction of values that stay in registers.  The
// transposed output goes through a copy of the tile in shared memory, so x is
// read once for both.  Bound by HBM: 16-bit in, 8-bit out.
template <typename T, typename Q, bool BLOCK, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const QArgs a) {
  __shared__ float red[kThreads / 32];
  __shared__ float half_max[2][kTile];
  extern __shared__ __align__(16) unsigned char dyn[];
  T* tile = reinterpret_cast<T*>(dyn);  // [128][132] when the transpose is wanted
  constexpr int kPitch = kTile + 4;
  pdl_release();
  pdl_wait();
  const int64_t r0 = (int64_t)blockIdx.y * kTile, c0 = (int64_t)blockIdx.x * kTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int nr = (int)min((int64_t)kTile, a.rows - r0);
  const T* x = (const T*)a.x;
  const int64_t c = c0 + lane * 4;
  float v[16][4];
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int r = warp * 16 + i;
    const bool row = r < nr;
    if (VEC) {
      if (row && c < a.cols) {  // cols is a multiple of 4 here
        const T* p = x + (r0 + r) * a.rs + c;
        if constexpr (sizeof(T) == 4) {
          const float4 w = *reinterpret_cast<const float4*>(p);
          v[i][0] = w.x, v[i][1] = w.y, v[i][2] = w.z, v[i][3] = w.w;
        } else {
          const uint2 w = *reinterpret_cast<const uint2*>(p);
          const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
          for (int j = 0; j < 4; j++) v[i][j] = to_f32<T>(e[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; j++) v[i][j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++) v[i][j] = row && c + j < a.cols ? to_f32<T>(x[(r0 + r) * a.rs + (c + j) * a.cs]) : 0.f;
    }
  }
  if (a.t.q) {
#pragma unroll
    for (int i = 0; i < 16; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) tile[(warp * 16 + i) * kPitch + lane * 4 + j] = from_f32<T>(v[i][j]);
  }
  float block_scale = 0.f;
  if (BLOCK) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) m = fmaxf(m, mag(v[i][j]));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (lane == 0) red[warp] = m;
    __syncthreads();
    m = kTiny;
#pragma unroll
    for (int i = 0; i < kThreads / 32; i++) m = fmaxf(m, red[i]);
    block_scale = m / fmax8<Q>();
    if (threadIdx.x == 0) {
      if (a.q.q) a.q.s[blockIdx.y * a.q.srs + blockIdx.x * a.q.scs] = block_scale;
      if (a.t.q) a.t.s[blockIdx.x * a.t.srs + blockIdx.y * a.t.scs] = block_scale;
    }
  }
  if (a.q.q) {
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = warp * 16 + i;
      if (r >= nr) break;
      float s = block_scale;
      if (!BLOCK) {
        float m = fmaxf(fmaxf(mag(v[i][0]), mag(v[i][1])), fmaxf(mag(v[i][2]), mag(v[i][3])));
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        s = fmaxf(m, kTiny) / fmax8<Q>();
        if (lane == 0) a.q.s[(r0 + r) * a.q.srs + blockIdx.x * a.q.scs] = s;
      }
      const uint32_t w = round8<Q>(v[i][0], v[i][1], v[i][2], v[i][3], s);
      // ldq is a multiple of 16: whole words, zeros past the last column
      if (c < a.cols) *reinterpret_cast<uint32_t*>((uint8_t*)a.q.q + (r0 + r) * a.q.ldq + c) = w;
    }
  }
  if (a.t.q) {
    __syncthreads();
    // a thread takes 64 rows of one column; lanes hold neighbouring columns
    const int col = threadIdx.x & 127, part = threadIdx.x >> 7;
    float s = block_scale;
    if (!BLOCK) {
      float m = 0.f;
#pragma unroll 8
      for (int i = 0; i < 64; i++) m = fmaxf(m, mag(to_f32<T>(tile[(part * 64 + i) * kPitch + col])));
      half_max[part][col] = m;
      __syncthreads();
      s = fmaxf(fmaxf(half_max[0][col], half_max[1][col]), kTiny) / fmax8<Q>();
      if (part == 0 && c0 + col < a.cols) a.t.s[(c0 + col) * a.t.srs + blockIdx.y * a.t.scs] = s;
    }
    if (c0 + col < a.cols) {
      uint8_t* out = (uint8_t*)a.t.q + (c0 + col) * a.t.ldq + r0 + part * 64;
#pragma unroll
      for (int g = 0; g < 4; g++) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const T* e = tile + (part * 64 + g * 16 + k * 4) * kPitch + col;
          w[k] = round8<Q>(to_f32<T>(e[0]), to_f32<T>(e[kPitch]), to_f32<T>(e[2 * kPitch]), to_f32<T>(e[3 * kPitch]), s);
        }
        // the leading dimension is a multiple of 16 and covers the rows: whole vectors
        if (part * 64 + g * 16 < nr) *reinterpret_cast<uint4*>(out + g * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

template <typename T, typename Q>
void launch(const QArgs& a, bool block, cudaStream_t s) {
  const dim3 grid((unsigned)((a.cols + kTile - 1) / kTile), (unsigned)((a.rows + kTile - 1) / kTile));
  const size_t smem = a.t.q ? (size_t)kTile * (kTile + 4) * sizeof(T) : 0;
  const bool vec = a.cs == 1 && a.cols % 4 == 0 && a.rs % 4 == 0 && (uintptr_t)a.x % (4 * sizeof(T)) == 0;
  auto go = [&](auto kern) {
    if (smem > 48 * 1024) ensure_dynamic_smem((const void*)kern, smem);
    launch_pdl(kern, grid, dim3(kThreads), smem, s, a);
  };
  if (block)
    vec ? go(quantize_kernel<T, Q, true, true>) : go(quantize_kernel<T, Q, true, false>);
  else
    vec ? go(quantize_kernel<T, Q, false, true>) : go(quantize_kernel<T, Q, false, false>);
  count_launch();
}

__global__ void pack8_kernel(const uint8_t* __restrict__ x, int64_t rows, int64_t cols, int64_t rs, int64_t cs,
                             uint8_t* __restrict__ dst, int64_t ld) {
  pdl_release();
  pdl_wait();
  // four output bytes a thread; the columns past the matrix are zeros
  const int64_t words = rows * (ld / 4);
  for (int64_t e = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; e < words; e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = e / (ld / 4), c = (e - r * (ld / 4)) * 4;
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++)
      if (c + j < cols) w |= (uint32_t)x[r * rs + (c + j) * cs] << (8 * j);
    *reinterpret_cast<uint32_t*>(dst + r * ld + c) = w;
  }
}

}  // namespace

void quantize(MType xt, const MatView& x, int block_rows, MType q8, const QuantOut& q, const QuantOut& t,
              cudaStream_t s) {
  if (x.rows == 0 || x.cols == 0 || (!q.q && !t.q)) return;
  if ((x.rows + kTile - 1) / kTile > 65535)
    throw Error(ErrKind::InvalidArgument, "quantize: more than 65535 * 128 rows");
  QArgs a{x.p, x.rows, x.cols, x.rs, x.cs, q, t};
  const bool block = block_rows != 1;
  auto pick = [&](auto qv) {
    using Q = decltype(qv);
    if (xt == MType::F32)
      launch<float, Q>(a, block, s);
    else if (xt == MType::BF16)
      launch<__nv_bfloat16, Q>(a, block, s);
    else
      launch<__half, Q>(a, block, s);
  };
  if (q8 == MType::E4M3)
    pick(__nv_fp8_e4m3{});
  else
    pick(__nv_fp8_e5m2{});
}

void pack8(const MatView& x, void* dst, int64_t ld, cudaStream_t s) {
  if (x.rows == 0 || x.cols == 0) return;
  const int64_t words = x.rows * (ld / 4);
  const int64_t grid = std::min<int64_t>((words + kThreads - 1) / kThreads, (int64_t)ctx().sm_count * 16);
  launch_pdl(pack8_kernel, dim3((unsigned)grid), dim3(kThreads), 0, s, (const uint8_t*)x.p, x.rows, x.cols, x.rs, x.cs,
             (uint8_t*)dst, ld);
  count_launch();
}

}  // namespace ndt
