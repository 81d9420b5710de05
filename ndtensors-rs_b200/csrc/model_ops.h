// Operators of language models on caller-owned device memory (row-major
// matrices, as torch holds them): block-scaled 8-bit products, embeddings,
// expert layers.
//
//   quantize.cu     8-bit block quantisation and operand packing
//   scaled_gemm.cu  products of block-scaled 8-bit matrices (tcgen05)
//   embedding.cu    embedding lookup and its gradient by sorted ids
//   experts.cu      a mixture-of-experts layer for a few tokens
//   model_ops.cpp   argument checks and the C entry points
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "ndt_internal.h"

namespace ndt {

// Element types of these operators; the numbers are the C ABI's (0 and 1 are
// float64 and complex128, which they do not take).
enum class MType : int { F32 = 2, BF16 = 3, F16 = 4, E4M3 = 5, E5M2 = 6 };
inline int msize(MType t) { return t == MType::F32 ? 4 : (t == MType::BF16 || t == MType::F16) ? 2 : 1; }

// A matrix [rows, cols] in device memory; element (r, c) at r * rs + c * cs.
struct MatView {
  const void* p;
  int64_t rows, cols, rs, cs;
};

// 8-bit block quantisation of x (quantize.cu).  q [rows, cols] with leading
// dimension ldq, scales at (block row, block column) through the strides; qt
// is the same of x's transpose.  q or qt may be null.
struct QuantOut {
  void* q;
  int64_t ldq;
  float* s;
  int64_t srs, scs;
};
void quantize(MType xt, const MatView& x, int block_rows, MType qt_type, const QuantOut& q, const QuantOut& qt,
              cudaStream_t s);
// dst[r * ld + c] = x(r, c) for 8-bit elements (ld a multiple of 16).
void pack8(const MatView& x, void* dst, int64_t ld, cudaStream_t s);

// C[i, j] = sum over blocks of 128 along k of sa * sb * (a . b): scaled_gemm.cu.
struct ScaledOperand {
  const void* p;  // [rows, k], unit stride along k; base and ld multiples of 16 bytes
  int64_t rows, ld;
  MType type;
  const float* s;  // scale of (row block, k block) at rb * srs + kb * scs
  int64_t srs, scs;
  bool per_row;  // a scale for each row; else for each 128 rows
};
// b_early: b was complete before the kernel that the stream ran last began (a
// quantize(), which waits for what is ahead of it before it lets the next
// kernel start), so its loads need not wait for that kernel.
void scaled_gemm(const ScaledOperand& a, const ScaledOperand& b, int64_t k, MType ct, void* c, int64_t ldc,
                 bool accumulate, cudaStream_t s, bool b_early = false);

// Embedding (embedding.cu).
void embedding(MType t, const void* table, int64_t v, int64_t d, int64_t ldt, const void* ids, bool ids64, int64_t n,
               int64_t first, float scale, void* out, int64_t ldo, cudaStream_t s);
void embedding_grad(MType gt, const void* grad, int64_t ldg, const void* ids, bool ids64, int64_t n, int64_t v,
                    int64_t d, int64_t first, float scale, MType ot, void* out, int64_t ldo, bool accumulate,
                    cudaStream_t s);

// A mixture-of-experts layer (experts.cu).
struct ExpertArgs {
  MType xt, wt;        // of x, the router and y; of the experts' weights
  const void* x;       // [tokens, h]
  const void* router;  // [experts, h]
  const void* w_in;    // [experts, 2 i, h]
  const void* w_out;   // [experts, h, i]
  const float* in_scales;   // [experts, ceil(2 i / 128), ceil(h / 128)] with 8-bit weights
  const float* out_scales;  // [experts, ceil(h / 128), ceil(i / 128)]
  int64_t tokens, experts, top, h, i, ldx, ldy;
  bool renormalize;
  void* y;         // [tokens, h], x's type
  int* ids;        // [tokens, top]
  float* weights;  // [tokens, top]
};
void expert_layer(const ExpertArgs& a, cudaStream_t s);

// A word in host memory that a kernel sets when a bounded wait ran out; the
// entry points report it at the next call.
int* wait_flag_device();
bool wait_flag_raised();

// Stream-ordered workspace, returned to the pool when the object goes.
struct Workspace {
  void* p = nullptr;
  cudaStream_t s;
  Workspace(size_t bytes, cudaStream_t st) : s(st) {
    if (bytes) p = pool_alloc(bytes, st);
  }
  ~Workspace() {
    if (p) cudaFreeAsync(p, s);
  }
  Workspace(const Workspace&) = delete;
  Workspace& operator=(const Workspace&) = delete;
};

// ------------------------------------------------------- device helpers
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

}  // namespace ndt
