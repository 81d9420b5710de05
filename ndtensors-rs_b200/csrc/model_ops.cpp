// C entry points of the language-model operators: argument checks, operand
// layout, status codes.  They take a cudaStream_t and device pointers of the
// current device, like ndt_b200_gemm_dev.
#include <climits>
#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/ndtensors_capi.h"
#include "mbarrier.h"

namespace ndt {

namespace {
std::mutex g_flag_mu;
int* g_flag = nullptr;  // host memory, mapped for every device

// One thread waits on a barrier that nothing arrives at.
__global__ void give_up_kernel(long long limit, int* flag) {
  __shared__ __align__(8) uint64_t bar;
  __shared__ int gave_up;
  gave_up = 0;
  mbar_init(smem_u32(&bar), 1);
  mbar_wait_slow(smem_u32(&bar), 0, &gave_up, flag, limit);
}
}  // namespace

int* wait_flag_device() {
  std::lock_guard<std::mutex> lk(g_flag_mu);
  if (!g_flag) {
    void* p = nullptr;
    NDT_CUDA(cudaHostAlloc(&p, sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable));
    g_flag = (int*)p;
    *(volatile int*)g_flag = 0;
  }
  return g_flag;  // unified addressing: the device's pointer is the host's
}
bool wait_flag_raised() {
  std::lock_guard<std::mutex> lk(g_flag_mu);
  if (!g_flag || !*(volatile int*)g_flag) return false;
  *(volatile int*)g_flag = 0;
  return true;
}
static void give_up_wait(long long clocks, cudaStream_t s) {
  give_up_kernel<<<1, 1, 0, s>>>(clocks, wait_flag_device());
  NDT_CUDA(cudaGetLastError());
}

CUtensorMap byte_map(const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    NDT_CUDA(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r));
    if (!p || r != cudaDriverEntryPointSuccess) throw Error(ErrKind::Cuda, "cuTensorMapEncodeTiled is not in this driver");
    return (Encode)p;
  }();
  CUtensorMap m;
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = encode(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, one,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(ErrKind::Cuda, "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
  return m;
}

}  // namespace ndt

using namespace ndt;

namespace {

[[noreturn]] void bad(const std::string& m) { throw Error(ErrKind::InvalidArgument, m); }
[[noreturn]] void bad_shape(const std::string& m) { throw Error(ErrKind::ShapeMismatch, m); }

// Runs the body; maps what it throws to a status code and ndt_b200_last_error.
template <typename F>
int entry(const char* name, F&& body) {
  try {
    ctx();
    if (wait_flag_raised())
      throw Error(ErrKind::Cuda, "an earlier scaled product or expert layer gave up waiting inside its kernel: its result is not valid");
    body();
    return NDT_SUCCESS;
  } catch (const Error& e) {
    set_last_error(std::string(name) + ": " + e.what());
    if (e.kind == ErrKind::Cuda) cudaGetLastError();  // the runtime keeps it for the next kernel launch of the library to find
    switch (e.kind) {
      case ErrKind::Panic:
      case ErrKind::Cuda:
        return NDT_INTERNAL_ERROR;
      case ErrKind::ShapeMismatch:
        return NDT_SHAPE_MISMATCH;
      default:
        return NDT_INVALID_ARGUMENT;
    }
  } catch (const std::exception& e) {
    set_last_error(std::string(name) + ": " + e.what());
    return NDT_INTERNAL_ERROR;
  } catch (...) {
    set_last_error(std::string(name) + ": unknown failure");
    return NDT_INTERNAL_ERROR;
  }
}

MType real_type(int t, const char* what) {
  if (t != NDT_F32 && t != NDT_BF16 && t != NDT_F16) bad(std::string(what) + " must be float32, bfloat16 or float16");
  return (MType)t;
}
MType type8(int t, const char* what) {
  if (t != NDT_E4M3 && t != NDT_E5M2) bad(std::string(what) + " must be float8 e4m3 or e5m2");
  return (MType)t;
}
void size_ok(long n, const char* what) {
  if (n < 0 || n > INT_MAX - 256) bad(std::string(what) + " must be from 0 to 2^31 - 257");
}
int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// A tensor-map operand: as it is, or copied to rows that start on 16 bytes.
struct Laid {
  Workspace copy;
  ScaledOperand o;
  Laid(MType t, const void* p, int64_t rows, int64_t k, int64_t rs, int64_t cs, cudaStream_t s)
      : copy(fits(p, rows, k, rs, cs) ? 0 : (size_t)(rows * up(k, 16)), s) {
    o.p = p, o.rows = rows, o.ld = rs, o.type = t;
    if (rows == 1) o.ld = up(k, 16);  // any stride will do
    if (copy.p) {
      pack8(MatView{p, rows, k, rs, cs}, copy.p, up(k, 16), s);
      o.p = copy.p, o.ld = up(k, 16);
    }
  }
  static bool fits(const void* p, int64_t rows, int64_t k, int64_t rs, int64_t cs) {
    return (uintptr_t)p % 16 == 0 && (k == 1 || cs == 1) && (rows == 1 || (rs % 16 == 0 && rs >= k && rs < ((int64_t)1 << 39)));
  }
};
void set_scales(ScaledOperand& o, const float* s, int block_rows, long rs, long cs, const char* what) {
  if (block_rows != 1 && block_rows != 128) bad(std::string(what) + ": a scale is for 1 or for 128 rows");
  o.s = s, o.srs = rs, o.scs = cs, o.per_row = block_rows == 1;
}

// An 8-bit matrix in a workspace: values with rows on 16 bytes, then scales, a
// column of them for each block of 128 along the rows (as the product reads them).
struct Quantised {
  MatView x;
  int block_rows;
  MType type;
  int64_t ld, sld;
  char* p = nullptr;
  Quantised(const MatView& x_, int br, MType t)
      : x(x_), block_rows(br), type(t), ld(up(x_.cols, 16)), sld(br == 1 ? up(x_.rows, 4) : (x_.rows + 127) / 128) {}
  size_t bytes() const { return (size_t)(up(x.rows * ld, 256) + up((x.cols + 127) / 128 * sld * 4, 256)); }
  void* place(void* at) {
    p = (char*)at;
    return p + bytes();
  }
  float* scales() const { return (float*)(p + up(x.rows * ld, 256)); }
  QuantOut out() const { return QuantOut{p, ld, scales(), 1, sld}; }
  ScaledOperand operand() const { return ScaledOperand{p, x.rows, ld, type, scales(), 1, sld, block_rows == 1}; }
};

void zero_rows(void* c, int64_t m, int64_t n, int64_t ldc, MType t, cudaStream_t s) {
  NDT_CUDA(cudaMemset2DAsync(c, ldc * msize(t), 0, n * msize(t), m, s));
}

}  // namespace

extern "C" {

int ndt_b200_quantize_dev(int x_type, const void* x, long rows, long cols, long row_stride, long col_stride,
                          int block_rows, int q_type, void* q, long ldq, float* scales, long scale_row_stride,
                          long scale_col_stride, void* qt, long ldqt, float* scales_t, long scale_t_row_stride,
                          long scale_t_col_stride, void* stream) {
  return entry("quantize", [&] {
    const MType xt = real_type(x_type, "x"), t8 = type8(q_type, "the result");
    size_ok(rows, "rows"), size_ok(cols, "columns");
    if (block_rows != 1 && block_rows != 128) bad("a block has 1 or 128 rows");
    if (rows == 0 || cols == 0) return;
    if (!x || (!q && !qt) || (q && !scales) || (qt && !scales_t)) bad("NULL pointer");
    auto out = [&](void* p, long ld, long width) {
      if (p && (ld < up(width, 16) || ld % 16 || (uintptr_t)p % 16))
        bad("8-bit results need a 16-byte aligned base and a leading dimension that is a multiple of 16 and covers a row");
    };
    out(q, ldq, cols), out(qt, ldqt, rows);
    quantize(xt, MatView{x, rows, cols, row_stride, col_stride}, block_rows, t8,
             QuantOut{q, ldq, scales, scale_row_stride, scale_col_stride},
             QuantOut{qt, ldqt, scales_t, scale_t_row_stride, scale_t_col_stride}, (cudaStream_t)stream);
  });
}

int ndt_b200_scaled_gemm_dev(long m, long n, long k, int a_type, const void* a, long a_row_stride, long a_col_stride,
                             int a_block_rows, const float* a_scales, long a_scale_row_stride, long a_scale_col_stride,
                             int b_type, const void* b, long b_row_stride, long b_col_stride, int b_block_rows,
                             const float* b_scales, long b_scale_row_stride, long b_scale_col_stride, int c_type,
                             void* c, long ldc, int accumulate, void* stream) {
  return entry("scaled_gemm", [&] {
    const MType at = type8(a_type, "a"), bt = type8(b_type, "b"), ct = real_type(c_type, "c");
    size_ok(m, "m"), size_ok(n, "n"), size_ok(k, "k");
    if (m == 0 || n == 0) return;
    if (!c) bad("NULL pointer");
    if (ldc < n) bad("ldc is smaller than a row of c");
    cudaStream_t s = (cudaStream_t)stream;
    if (k == 0) {
      if (!accumulate) zero_rows(c, m, n, ldc, ct, s);
      return;
    }
    if (!a || !b || !a_scales || !b_scales) bad("NULL pointer");
    Laid la(at, a, m, k, a_row_stride, a_col_stride, s), lb(bt, b, n, k, b_row_stride, b_col_stride, s);
    set_scales(la.o, a_scales, a_block_rows, a_scale_row_stride, a_scale_col_stride, "a");
    set_scales(lb.o, b_scales, b_block_rows, b_scale_row_stride, b_scale_col_stride, "b");
    scaled_gemm(la.o, lb.o, k, ct, c, ldc, accumulate != 0, s);
  });
}

int ndt_b200_scaled_linear_dev(int x_type, const void* x, long tokens, long k, long x_row_stride, long x_col_stride,
                               int w_type, const void* w, long n, long w_row_stride, long w_col_stride,
                               const float* w_scales, long w_scale_row_stride, long w_scale_col_stride, int y_type,
                               void* y, long ldy, void* stream) {
  return entry("scaled_linear", [&] {
    const MType xt = real_type(x_type, "x"), wt = type8(w_type, "w"), yt = real_type(y_type, "y");
    size_ok(tokens, "tokens"), size_ok(n, "outputs"), size_ok(k, "inputs");
    if (tokens == 0 || n == 0) return;
    if (!y) bad("NULL pointer");
    if (ldy < n) bad("ldy is smaller than a row of y");
    cudaStream_t s = (cudaStream_t)stream;
    if (k == 0) {
      zero_rows(y, tokens, n, ldy, yt, s);
      return;
    }
    if (!x || !w || !w_scales) bad("NULL pointer");
    Laid lw(wt, w, n, k, w_row_stride, w_col_stride, s);
    set_scales(lw.o, w_scales, 128, w_scale_row_stride, w_scale_col_stride, "w");
    Quantised qx(MatView{x, tokens, k, x_row_stride, x_col_stride}, 1, MType::E4M3);
    Workspace ws(qx.bytes(), s);
    qx.place(ws.p);
    quantize(xt, qx.x, 1, MType::E4M3, qx.out(), QuantOut{}, s);
    scaled_gemm(qx.operand(), lw.o, k, yt, y, ldy, false, s, !lw.copy.p);
  });
}

int ndt_b200_scaled_linear_fwd_dev(int x_type, const void* x, long tokens, long k, long x_row_stride, long x_col_stride,
                                   int w_type, const void* w, long n, long w_row_stride, long w_col_stride, void* y,
                                   long ldy, void* wt, long ldwt, float* wt_scales, void* stream) {
  return entry("scaled_linear_fwd", [&] {
    const MType xt = real_type(x_type, "x"), wtp = real_type(w_type, "w");
    size_ok(tokens, "tokens"), size_ok(n, "outputs"), size_ok(k, "inputs");
    cudaStream_t s = (cudaStream_t)stream;
    if (ldy < n) bad("ldy is smaller than a row of y");
    if ((tokens && n && !y) || (k && ((tokens && !x) || (n && !w))) || (wt && !wt_scales)) bad("NULL pointer");
    if (wt && (ldwt < up(n, 16) || ldwt % 16 || (uintptr_t)wt % 16)) bad("wt needs a 16-byte aligned base and a leading dimension to match");
    if (n == 0) return;
    if (k == 0) {
      if (tokens) zero_rows(y, tokens, n, ldy, xt, s);
      return;
    }
    Quantised qw(MatView{w, n, k, w_row_stride, w_col_stride}, 128, MType::E4M3),
        qx(MatView{x, tokens, k, x_row_stride, x_col_stride}, 1, MType::E4M3);
    Workspace ws(qw.bytes() + qx.bytes(), s);
    qx.place(qw.place(ws.p));
    const QuantOut t{wt, ldwt, wt_scales, 1, (k + 127) / 128};
    quantize(wtp, qw.x, 128, MType::E4M3, qw.out(), wt ? t : QuantOut{}, s);
    if (tokens == 0) return;
    quantize(xt, qx.x, 1, MType::E4M3, qx.out(), QuantOut{}, s);
    scaled_gemm(qx.operand(), qw.operand(), k, xt, y, ldy, false, s);
  });
}

int ndt_b200_scaled_linear_vjp_dev(int x_type, const void* dy, long tokens, long n, long dy_row_stride, long dy_col_stride,
                                   const void* x, long k, long x_row_stride, long x_col_stride, const void* wt, long ldwt,
                                   const float* wt_scales, int grad8_type, void* dx, long lddx, int dw_type, void* dw,
                                   long lddw, void* stream) {
  return entry("scaled_linear_vjp", [&] {
    const MType xt = real_type(x_type, "x"), g8 = type8(grad8_type, "the gradient's 8-bit type");
    const MType dwt = dw ? real_type(dw_type, "dw") : MType::F32;
    size_ok(tokens, "tokens"), size_ok(n, "outputs"), size_ok(k, "inputs");
    cudaStream_t s = (cudaStream_t)stream;
    if ((dx && lddx < k) || (dw && lddw < k)) bad("a leading dimension is smaller than a row");
    if (k == 0 || (!dx && !dw)) return;
    if (dx && n == 0 && tokens) zero_rows(dx, tokens, k, lddx, xt, s);
    if (dw && tokens == 0 && n) zero_rows(dw, n, k, lddw, dwt, s);
    if (n == 0 || tokens == 0) return;
    if (!dy || (dx && (!wt || !wt_scales)) || (dw && !x)) bad("NULL pointer");
    const MatView g{dy, tokens, n, dy_row_stride, dy_col_stride}, gt{dy, n, tokens, dy_col_stride, dy_row_stride},
        xtr{x, k, tokens, x_col_stride, x_row_stride};
    Quantised qg(g, 1, g8), qgt(gt, 1, g8), qxt(xtr, 1, MType::E4M3);
    Workspace ws((dx ? qg.bytes() : 0) + (dw ? qgt.bytes() + qxt.bytes() : 0), s);
    void* p = ws.p;
    if (dx) p = qg.place(p);
    if (dw) qxt.place(qgt.place(p));
    quantize(xt, g, 1, g8, dx ? qg.out() : QuantOut{}, dw ? qgt.out() : QuantOut{}, s);
    if (dw) quantize(xt, MatView{x, tokens, k, x_row_stride, x_col_stride}, 1, MType::E4M3, QuantOut{}, qxt.out(), s);
    if (dx) {
      ScaledOperand ow{wt, k, ldwt, MType::E4M3, wt_scales, 1, (k + 127) / 128, false};
      scaled_gemm(qg.operand(), ow, n, xt, dx, lddx, false, s);
    }
    if (dw) scaled_gemm(qgt.operand(), qxt.operand(), tokens, dwt, dw, lddw, false, s);
  });
}

int ndt_b200_embedding_dev(int type, const void* table, long rows, long dim, long ld, const void* ids, int ids64, long n,
                           long first, float scale, void* out, long ldo, void* stream) {
  return entry("embedding", [&] {
    const MType t = real_type(type, "the table");
    size_ok(rows, "rows"), size_ok(dim, "columns"), size_ok(n, "ids");
    if (n == 0 || dim == 0) return;
    if ((rows && !table) || !ids || !out) bad("NULL pointer");
    if (ld < dim || ldo < dim) bad("a leading dimension is smaller than a row");
    embedding(t, table, rows, dim, ld, ids, ids64 != 0, n, first, scale, out, ldo, (cudaStream_t)stream);
  });
}

int ndt_b200_embedding_grad_dev(int grad_type, const void* grad, long ldg, const void* ids, int ids64, long n, long rows,
                                long dim, long first, float scale, int out_type, void* out, long ldo, int accumulate,
                                void* stream) {
  return entry("embedding_grad", [&] {
    const MType gt = real_type(grad_type, "grad"), ot = real_type(out_type, "the result");
    size_ok(rows, "rows"), size_ok(dim, "columns"), size_ok(n, "ids");
    if (rows == 0 || dim == 0) return;
    if (!out || (n && (!grad || !ids))) bad("NULL pointer");
    if (ldg < dim || ldo < dim) bad("a leading dimension is smaller than a row");
    embedding_grad(gt, grad, ldg, ids, ids64 != 0, n, rows, dim, first, scale, ot, out, ldo, accumulate != 0, (cudaStream_t)stream);
  });
}

int ndt_b200_expert_layer_dev(int x_type, const void* x, long tokens, long h, long ldx, const void* router, long experts,
                              int w_type, const void* w_in, const float* in_scales, const void* w_out,
                              const float* out_scales, long i, long top, int renormalize, void* y, long ldy, int* ids,
                              float* weights, void* stream) {
  return entry("expert_layer", [&] {
    const MType xt = real_type(x_type, "x");
    if (xt == MType::F32) bad("x must be bfloat16 or float16");
    const bool w8 = w_type == NDT_E4M3;
    if (!w8 && w_type != x_type) bad("the experts' weights must have x's type or be float8 e4m3");
    size_ok(tokens, "tokens"), size_ok(h, "h"), size_ok(experts, "experts"), size_ok(i, "i");
    if (h < 1 || experts < 1 || i < 1) bad_shape("h, i and the number of experts must be positive");
    if (i > INT_MAX / 4 || h > INT_MAX / 4) bad("h and i must be below 2^29");
    if (top < 1 || top > experts) bad("top must be from 1 to the number of experts");
    if (tokens == 0) return;
    if (!x || !router || !w_in || !w_out || !y || !ids || !weights || (w8 && (!in_scales || !out_scales))) bad("NULL pointer");
    if (ldx < h || ldy < h) bad("a leading dimension is smaller than a row");
    ExpertArgs a{};
    a.xt = xt, a.wt = (MType)w_type;
    a.x = x, a.router = router, a.w_in = w_in, a.w_out = w_out, a.in_scales = in_scales, a.out_scales = out_scales;
    a.tokens = tokens, a.experts = experts, a.top = top, a.h = h, a.i = i, a.ldx = ldx, a.ldy = ldy;
    a.renormalize = renormalize != 0;
    a.y = y, a.ids = ids, a.weights = weights;
    expert_layer(a, (cudaStream_t)stream);
  });
}

int ndt_b200_give_up_wait(long clocks, void* stream) {
  return entry("give_up_wait", [&] {
    if (clocks < 1 || clocks > INT_MAX) bad("clocks must be from 1 to 2^31 - 1");
    give_up_wait(clocks, (cudaStream_t)stream);
  });
}

}  // extern "C"
