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
// The quotient is the correctly rounded one, not a product with a reciprocal,
// so q is a function of the block alone that any caller can restate.  It takes
// three operations by Markstein's method (IBM J. Res. Dev. 34, 1990): with r
// the rounded 1 / s and y = x r, y + r (x - s y) rounds to x / s as long as the
// remainder does not underflow, which a power of two keeps it from.  (CUDA's
// division, a branch for each element, made the kernel six times as long:
// 46 us for 4096 x 4096 bfloat16.)  Measured on one B200: 8192 x 8192 bfloat16
// 56 us by rows (3.6 TB/s; HBM alone would take 31), 122 with the transpose (2.2
// TB/s); in 128 x 128 blocks 68 and 98.  Instructions bound them, not HBM.
#include <algorithm>

#include "model_ops.h"

namespace ndt {
namespace {

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100
constexpr float kMaxFloat = 3.402823466e38f;
constexpr int kTile = 128;
constexpr int kThreads = 256;

template <typename Q>
__device__ __forceinline__ float fmax8();
template <>
__device__ __forceinline__ float fmax8<__nv_fp8_e4m3>() { return 448.f; }
template <>
__device__ __forceinline__ float fmax8<__nv_fp8_e5m2>() { return 57344.f; }

// A scale and what dividing by it takes.
struct Divisor {
  float s, up, r;  // up: a power of two for both sides
};
template <typename Q>
__device__ __forceinline__ Divisor divisor(float amax) {
  Divisor d;
  d.s = fmaxf(amax, kTiny) / fmax8<Q>();
  d.up = d.s < 8.673617379884035e-19f ? 18446744073709551616.f : 1.f;  // 2^64 below 2^-60
  d.r = 1.f / (d.s * d.up);
  return d;
}
__device__ __forceinline__ float quotient(float x, float s, float r) {
  const float y = x * r;
  return fmaf(fmaf(-y, s, x), r, y);
}
// Four elements as 8-bit codes, the first in the lowest byte.
template <typename Q>
__device__ __forceinline__ uint32_t round8(float x0, float x1, float x2, float x3, const Divisor& d) {
  constexpr bool kE4 = std::is_same_v<Q, __nv_fp8_e4m3>;
  constexpr __nv_fp8_interpretation_t kind = kE4 ? __NV_E4M3 : __NV_E5M2;
  const float s = d.s * d.up;
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(quotient(x0 * d.up, s, d.r), quotient(x1 * d.up, s, d.r)), __NV_SATFINITE, kind);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(quotient(x2 * d.up, s, d.r), quotient(x3 * d.up, s, d.r)), __NV_SATFINITE, kind);
  uint32_t w = lo | hi << 16;
  const float sum = fabsf(x0) + fabsf(x1) + fabsf(x2) + fabsf(x3);
  if (!(sum <= kMaxFloat)) {  // rare: an element is not finite (or their sum is not)
    const float x[4] = {x0, x1, x2, x3};
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (fabsf(x[j]) <= kMaxFloat) continue;
      const uint32_t code = kE4 || x[j] != x[j] ? 0x7fu : x[j] > 0 ? 0x7cu : 0xfcu;
      w = (w & ~(0xffu << (8 * j))) | code << (8 * j);
    }
  }
  return w;
}
__device__ __forceinline__ float mag(float x) {
  x = fabsf(x);
  return x <= kMaxFloat ? x : 0.f;  // infinities and NaN do not count
}

struct QArgs {
  const void* x;
  int64_t rows, cols, rs, cs;
  QuantOut q, t;
  uint32_t across;  // CTAs along a row; the grid is one line of them, row after row
};

// How x lies: columns apart; columns together, rows starting anywhere (read in
// aligned words); whole aligned vectors of 8 columns.
enum Lie { kApart, kTogether, kVectors };

// Eight elements of a row from column c (zeros outside the matrix).
template <typename T, int LIE>
__device__ __forceinline__ void load8(const QArgs& a, int64_t r, int64_t c, float* v) {
  const T* p = (const T*)a.x + r * a.rs;
  if (LIE != kApart && r < a.rows && c + 8 <= a.cols) {
    p += c;
    if constexpr (sizeof(T) == 4) {
      if (LIE == kVectors || ((uintptr_t)p & 15) == 0) {
        const float4 w0 = *reinterpret_cast<const float4*>(p), w1 = *reinterpret_cast<const float4*>(p + 4);
        v[0] = w0.x, v[1] = w0.y, v[2] = w0.z, v[3] = w0.w, v[4] = w1.x, v[5] = w1.y, v[6] = w1.z, v[7] = w1.w;
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = p[j];
      }
    } else {
      uint32_t w[4];
      if (LIE == kVectors) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
      } else {  // four aligned words hold the elements, or five where the row starts in the middle of one
        const uint32_t* q = reinterpret_cast<const uint32_t*>((uintptr_t)p & ~(uintptr_t)3);
        const bool odd = (uintptr_t)p & 2;
        uint32_t x[5];
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = q[j];
        x[4] = odd ? q[4] : 0;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = odd ? __funnelshift_r(x[j], x[j + 1], 16) : x[j];
      }
      const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = to_f32<T>(e[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j++)
      v[j] = LIE != kVectors && r < a.rows && c + j < a.cols ? to_f32<T>(p[(c + j) * (LIE == kApart ? a.cs : 1)]) : 0.f;
  }
}
__device__ __forceinline__ float max8(const float* v) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) m = fmaxf(m, mag(v[j]));
  return m;
}
// ld is a multiple of 16 that covers the row: whole words, zeros past the last column
template <typename Q>
__device__ __forceinline__ void store8(const QArgs& a, int64_t r, int64_t c, const float* v, const Divisor& d) {
  const uint2 w = make_uint2(round8<Q>(v[0], v[1], v[2], v[3], d), round8<Q>(v[4], v[5], v[6], v[7], d));
  if (r < a.rows && c < a.cols) *reinterpret_cast<uint2*>((uint8_t*)a.q.q + r * a.q.ldq + c) = w;
}

// Blocks of 1 x 128, x as it lies: half a warp takes a block, a thread 8
// columns of kRows rows.  Bound by instructions, 25 an element: 85 % of the issue
// slots are busy at 8192 x 8192, DRAM 36 % of its peak.
constexpr int kRows = 4;
template <typename T, typename Q, int LIE>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const QArgs a) {
  pdl_wait();
  pdl_release();  // (in this order: the next kernel may read what was ready before this one)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t by = blockIdx.x / a.across, bx = blockIdx.x - by * a.across;
  const int64_t r0 = ((int64_t)by * (kThreads / 32) + warp) * kRows, c = bx * 256ll + lane * 8;
  if (r0 >= a.rows) return;
  float v[kRows][8], m[kRows];
#pragma unroll
  for (int i = 0; i < kRows; i++) load8<T, LIE>(a, r0 + i, c, v[i]);
#pragma unroll
  for (int i = 0; i < kRows; i++) m[i] = max8(v[i]);
#pragma unroll
  for (int o = 8; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < kRows; i++) m[i] = fmaxf(m[i], __shfl_xor_sync(~0u, m[i], o));
#pragma unroll
  for (int i = 0; i < kRows; i++) {
    const Divisor d = divisor<Q>(m[i]);
    store8<Q>(a, r0 + i, c, v[i], d);
    if ((lane & 15) == 0 && r0 + i < a.rows && c < a.cols) a.q.s[(r0 + i) * a.q.srs + c / 128 * a.q.scs] = d.s;
  }
}

// One 128 x 128 tile a CTA: blocks of 128 x 128, or the transpose too.  The
// tile lies in shared memory, so x is read once for both outputs; there a
// thread takes two columns of a quarter of the rows.  Bound by instructions and
// their latency: 17 an element in blocks, 27 with the transpose too, 39 with rows
// of both, at 52 - 61 % of the issue slots with 16 warps an SM (the registers of
// 64 elements a thread).
template <typename T, typename Q, bool BLOCK, int LIE>
__global__ void __launch_bounds__(kThreads) quantize_tile_kernel(const QArgs a) {
  extern __shared__ __align__(16) unsigned char dyn[];
  constexpr int kPitch = kTile + 16 / (int)sizeof(T);
  T* tile = reinterpret_cast<T*>(dyn);  // [128][kPitch]
  __shared__ float red[kThreads / 32];
  __shared__ float quarter[4][kTile];
  pdl_release();
  pdl_wait();
  const uint32_t by = blockIdx.x / a.across, bx = blockIdx.x - by * a.across;
  const int64_t r0 = (int64_t)by * kTile, c0 = (int64_t)bx * kTile;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane >> 4, col8 = (lane & 15) * 8;
  float v[8][8], m[8];
#pragma unroll
  for (int i = 0; i < 8; i++) load8<T, LIE>(a, r0 + warp * 16 + i * 2 + sub, c0 + col8, v[i]);
#pragma unroll
  for (int i = 0; i < 8; i++) m[i] = max8(v[i]);
  if (a.t.q) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      T* to = tile + (warp * 16 + i * 2 + sub) * kPitch + col8;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(to) = make_float4(v[i][0], v[i][1], v[i][2], v[i][3]);
        *reinterpret_cast<float4*>(to + 4) = make_float4(v[i][4], v[i][5], v[i][6], v[i][7]);
      } else {
        alignas(16) T e[8];
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = from_f32<T>(v[i][j]);
        *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(e);
      }
    }
  }
  Divisor block{};
  if (BLOCK) {
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) most = fmaxf(most, m[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
    if (lane == 0) red[warp] = most;
    __syncthreads();
    most = 0.f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; i++) most = fmaxf(most, red[i]);
    block = divisor<Q>(most);
    if (threadIdx.x == 0) {
      if (a.q.q) a.q.s[by * a.q.srs + bx * a.q.scs] = block.s;
      if (a.t.q) a.t.s[bx * a.t.srs + by * a.t.scs] = block.s;
    }
  }
  if (a.q.q) {
    if (!BLOCK)
#pragma unroll
      for (int o = 8; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < 8; i++) m[i] = fmaxf(m[i], __shfl_xor_sync(~0u, m[i], o));
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int64_t r = r0 + warp * 16 + i * 2 + sub;
      const Divisor d = BLOCK ? block : divisor<Q>(m[i]);
      store8<Q>(a, r, c0 + col8, v[i], d);
      if (!BLOCK && (lane & 15) == 0 && r < a.rows) a.q.s[r * a.q.srs + bx * a.q.scs] = d.s;
    }
  }
  if (!a.t.q) return;
  __syncthreads();
  const int col = (threadIdx.x & 63) * 2, part = threadIdx.x >> 6;
  const T* from = tile + part * 32 * kPitch + col;
  auto two = [&](int r, float& x, float& y) {
    if constexpr (sizeof(T) == 4) {
      const float2 w = *reinterpret_cast<const float2*>(from + r * kPitch);
      x = w.x, y = w.y;
    } else {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(from + r * kPitch);
      const T* e = reinterpret_cast<const T*>(&w);
      x = to_f32<T>(e[0]), y = to_f32<T>(e[1]);
    }
  };
  Divisor d[2] = {block, block};
  if (!BLOCK) {
    float mx = 0.f, my = 0.f;
#pragma unroll 8
    for (int i = 0; i < 32; i++) {
      float x, y;
      two(i, x, y);
      mx = fmaxf(mx, mag(x)), my = fmaxf(my, mag(y));
    }
    *reinterpret_cast<float2*>(&quarter[part][col]) = make_float2(mx, my);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; k++) {
      d[k] = divisor<Q>(fmaxf(fmaxf(quarter[0][col + k], quarter[1][col + k]), fmaxf(quarter[2][col + k], quarter[3][col + k])));
      if (part == 0 && c0 + col + k < a.cols) a.t.s[(c0 + col + k) * a.t.srs + by * a.t.scs] = d[k].s;
    }
  }
  const int nr = (int)min((int64_t)kTile, a.rows - r0);
#pragma unroll
  for (int g = 0; g < 2; g++) {  // 16 rows: a vector of each column
    uint32_t w[2][4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      float x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; j++) two(g * 16 + k * 4 + j, x[j], y[j]);
      w[0][k] = round8<Q>(x[0], x[1], x[2], x[3], d[0]);
      w[1][k] = round8<Q>(y[0], y[1], y[2], y[3], d[1]);
    }
    // the leading dimension is a multiple of 16 and covers the rows: whole vectors
    const int row = part * 32 + g * 16;
#pragma unroll
    for (int k = 0; k < 2; k++)
      if (row < nr && c0 + col + k < a.cols)
        *reinterpret_cast<uint4*>((uint8_t*)a.t.q + (c0 + col + k) * a.t.ldq + r0 + row) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
  }
}

template <typename T, typename Q>
void launch(QArgs a, bool block, cudaStream_t s) {
  const Lie lie = a.cs != 1 ? kApart
                  : a.cols % 8 == 0 && a.rs % (16 / sizeof(T)) == 0 && (uintptr_t)a.x % 16 == 0 ? kVectors : kTogether;
  auto grid_of = [&](int64_t rows, int64_t cols) {
    const int64_t across = (a.cols + cols - 1) / cols, all = across * ((a.rows + rows - 1) / rows);
    if (all > INT32_MAX) throw Error(ErrKind::InvalidArgument, "the matrix has too many blocks for one launch");
    a.across = (uint32_t)across;
    return dim3((unsigned)all);
  };
  if (!block && !a.t.q) {
    const dim3 grid = grid_of(kThreads / 32 * kRows, 256);
    auto go = [&](auto kern) { launch_pdl(kern, grid, dim3(kThreads), 0, s, a); };
    lie == kVectors ? go(quantize_rows_kernel<T, Q, kVectors>)
    : lie == kTogether ? go(quantize_rows_kernel<T, Q, kTogether>) : go(quantize_rows_kernel<T, Q, kApart>);
  } else {
    const dim3 grid = grid_of(kTile, kTile);
    const size_t smem = a.t.q ? (size_t)kTile * (kTile + 16 / sizeof(T)) * sizeof(T) : 0;
    auto go = [&](auto kern) {
      if (smem > 48 * 1024) ensure_dynamic_smem((const void*)kern, smem);
      launch_pdl(kern, grid, dim3(kThreads), smem, s, a);
    };
    if (block)
      lie == kVectors ? go(quantize_tile_kernel<T, Q, true, kVectors>)
      : lie == kTogether ? go(quantize_tile_kernel<T, Q, true, kTogether>) : go(quantize_tile_kernel<T, Q, true, kApart>);
    else
      lie == kVectors ? go(quantize_tile_kernel<T, Q, false, kVectors>)
      : lie == kTogether ? go(quantize_tile_kernel<T, Q, false, kTogether>) : go(quantize_tile_kernel<T, Q, false, kApart>);
  }
  count_launch();
}

// Rows of 8-bit elements to rows that start on 16 bytes, zeros past the last:
// a warp takes a row, a lane 16 output bytes at a time.
__global__ void __launch_bounds__(kThreads) pack8_kernel(const uint8_t* __restrict__ x, int64_t rows, int64_t cols, int64_t rs,
                                                         int64_t cs, uint8_t* __restrict__ dst, int64_t ld) {
  pdl_release();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t r = blockIdx.x * (int64_t)(kThreads / 32) + (threadIdx.x >> 5); r < rows; r += warps) {
#pragma unroll 4
    for (int64_t c = lane * 16; c < ld; c += 512) {
      const uint8_t* p = x + r * rs + c * cs;
      uint32_t v[4] = {};
      if (cs == 1 && c + 16 <= cols) {  // five aligned words hold the 16 bytes (four where p is aligned)
        const uint32_t shift = (uint32_t)((uintptr_t)p & 3) * 8;
        const uint32_t* q = reinterpret_cast<const uint32_t*>((uintptr_t)p & ~(uintptr_t)3);
        uint32_t w[5];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = q[j];
        w[4] = shift ? q[4] : 0;
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = __funnelshift_r(w[j], w[j + 1], shift);
      } else {
#pragma unroll
        for (int j = 0; j < 16; j++)
          if (c + j < cols) v[j / 4] |= (uint32_t)p[j * cs] << (8 * (j % 4));
      }
      *reinterpret_cast<uint4*>(dst + r * ld + c) = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

}  // namespace

void quantize(MType xt, const MatView& x, int block_rows, MType q8, const QuantOut& q, const QuantOut& t,
              cudaStream_t s) {
  if (x.rows == 0 || x.cols == 0 || (!q.q && !t.q)) return;
  QArgs a{x.p, x.rows, x.cols, x.rs, x.cs, q, t, 0};
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
  const int64_t grid = std::min<int64_t>((x.rows + kThreads / 32 - 1) / (kThreads / 32), (int64_t)ctx().sm_count * 64);
  launch_pdl(pack8_kernel, dim3((unsigned)grid), dim3(kThreads), 0, s, (const uint8_t*)x.p, x.rows, x.cols, x.rs, x.cs,
             (uint8_t*)dst, ld);
  count_launch();
}

}  // namespace ndt
