// Embedding lookup with scaling, and the gradient of the table.
//
//   out[i, :]    = scale * table[ids[i] - first, :]      (zero outside the table)
//   dtable[v, :] = scale * sum over i with ids[i] - first == v of grad[i, :]
//
// Both are bound by memory.  The sum has to have one order, so that a step
// gives the same gradient twice: the ids are sorted by (row, position), then
// tiles of kEntries sorted entries are summed in 32 bits in that order.  A
// row whose entries cross tiles leaves a part in each, and a last kernel adds
// the parts in tile order.  Tiles of entries, not of rows, keep the work even
// when a few ids make up most of a batch.
//
// The sort is one kernel without communication: every CTA owns a range of
// rows, counts over all ids how many lie below its range (its offset in the
// sorted list) and places its own, stably.  It writes the zeros of its rows
// that no id names as well, so the dense result is written once.
//
// Measured on one B200 (16384 ids by frequency, 65536 x 2048 bf16, us under the
// profiler): lookup 15, sort with 180 MB of zeros to DRAM 45, sum 17 for 67 MB,
// join 13; the step 94, 5.0 TB/s of what it has to move.  Eight rows of grad in
// flight a thread made the sum 50 -> 26, and chains added by groups of threads
// the join 193 -> 29.
#include <algorithm>

#include "model_ops.h"

namespace ndt {
namespace {

constexpr int kSortThreads = 1024;
constexpr int kPlacers = 512;                      // threads that place ids while the others write zeros
constexpr int kPerThread = 8;                      // ids a placer takes in turn
constexpr int kList = kPlacers * kPerThread + kPlacers;  // compacted ids of a range
constexpr int kEntries = 32;                       // sorted entries a tile
constexpr int kSumThreads = 128;                   // (256 leave a last wave of half the SMs)

// The table's row of id i; for an id below the table's first the largest number
// (the difference alone comes round to a row where first is near 2^63).
template <bool IDS64>
__device__ __forceinline__ uint64_t row_at(const void* ids, int64_t i, int64_t first) {
  const int64_t id = IDS64 ? ((const int64_t*)ids)[i] : (int64_t)((const int*)ids)[i];
  return id < first ? ~0ull : (uint64_t)id - (uint64_t)first;
}

// ---------------------------------------------------------------- lookup
// A warp takes one row (or one of `parts` pieces of it), four 16-byte vectors
// a lane at a time.
template <typename T, bool IDS64, bool VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const T* __restrict__ table, int64_t v, int64_t d, int64_t ldt,
                                                     const void* __restrict__ ids, int64_t n, int64_t first, float scale,
                                                     T* __restrict__ out, int64_t ldo, int parts) {
  pdl_release();
  pdl_wait();
  constexpr int kN = VEC ? 16 / sizeof(T) : 1;
  const int lane = threadIdx.x & 31;
  const int64_t w = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
  const int64_t i = w / parts;
  if (i >= n) return;
  const int64_t vecs = d / kN, per = (vecs + parts - 1) / parts;
  const int64_t c0 = (w - i * parts) * per, c1 = min(vecs, c0 + per);
  const uint64_t row = row_at<IDS64>(ids, i, first);
  const bool in = row < (uint64_t)v;
  const T* src = table + (in ? row : 0) * ldt;
  T* dst = out + i * ldo;
  if constexpr (VEC) {
    for (int64_t c = c0 + lane; c < c1; c += 128) {
      uint4 x[4];
#pragma unroll
      for (int j = 0; j < 4; j++)
        x[j] = in && c + 32 * j < c1 ? __ldg(reinterpret_cast<const uint4*>(src) + c + 32 * j) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; j++) {
        if (c + 32 * j >= c1) break;
        T* e = reinterpret_cast<T*>(&x[j]);
#pragma unroll
        for (int q = 0; q < kN; q++) e[q] = from_f32<T>(in ? to_f32<T>(e[q]) * scale : 0.f);
        reinterpret_cast<uint4*>(dst)[c + 32 * j] = x[j];
      }
    }
  } else {
    for (int64_t c = c0 + lane; c < c1; c += 32) dst[c] = from_f32<T>(in ? to_f32<T>(src[c]) * scale : 0.f);
  }
}

// ------------------------------------------------------------------ sort
// Exclusive sum over the first N threads of the CTA, which all call it; the
// total too.
template <int N>
__device__ __forceinline__ void group_sync() {
  asm volatile("bar.sync %0, %1;" ::"n"(N == kSortThreads ? 0 : 1), "n"(N) : "memory");
}
template <int N>
__device__ __forceinline__ int exclusive_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto inclusive = [&](int x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, x, o);
      if (lane >= o) x += y;
    }
    return x;
  };
  const int x = inclusive(v);
  if (lane == 31) warp_sums[warp] = x;
  group_sync<N>();
  const int sums = inclusive(lane < N / 32 ? warp_sums[lane] : 0);
  total = __shfl_sync(~0u, sums, 31);
  const int before = __shfl_sync(~0u, sums, (warp + 31) & 31);
  group_sync<N>();
  return (warp ? before : 0) + x - v;
}

struct SortArgs {
  const void* ids;
  int64_t n, first, v, range;  // range: rows of one CTA
  int* order;                  // sorted positions
  int* rows;                   // their rows
  int* count;                  // how many ids are in the table
  void* out;                   // zeros go to the rows without an id; null: nowhere
  int64_t d_bytes, ld_bytes;
};

template <bool IDS64>
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const SortArgs a) {
  extern __shared__ int sm[];
  int* start = sm;                  // [range] counts, then where the next id of a row goes
  int* list_key = sm + a.range;     // [kList]
  int* list_pos = list_key + kList;
  __shared__ int warp_sums[32];
  __shared__ int list_n, below_s, next_row;
  __shared__ unsigned present[1024];  // a bit a row of the range: it has an id
  pdl_release();
  pdl_wait();
  const uint64_t v0 = blockIdx.x * (uint64_t)a.range, v1 = min((uint64_t)a.v, v0 + a.range);
  const int rows = (int)(v1 - v0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < a.range; i += kSortThreads) start[i] = 0;
  if (threadIdx.x == 0) below_s = 0, list_n = 0, next_row = 0;
  __syncthreads();
  int below = 0;
  for (int64_t i0 = threadIdx.x; i0 < a.n; i0 += kSortThreads * 8) {
    uint64_t r[8];
#pragma unroll
    for (int j = 0; j < 8; j++) r[j] = i0 + j * kSortThreads < a.n ? row_at<IDS64>(a.ids, i0 + j * kSortThreads, a.first) : ~0ull;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      if (r[j] < v0) below++;
      if (r[j] >= v0 && r[j] < v1) atomicAdd(&start[r[j] - v0], 1);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) below += __shfl_xor_sync(~0u, below, o);
  if (lane == 0 && below) atomicAdd(&below_s, below);
  __syncthreads();
  // counts -> first places
  const int base0 = below_s;
  int base = base0;
  for (int i0 = 0; i0 < a.range; i0 += kSortThreads) {
    const int i = i0 + threadIdx.x;
    const int c = i < a.range ? start[i] : 0;
    const unsigned on = __ballot_sync(~0u, c > 0);
    if (lane == 0) present[i >> 5] = on;
    int total;
    const int before = exclusive_scan<kSortThreads>(c, warp_sums, total);
    if (i < a.range) start[i] = base + before;
    base += total;
  }
  __syncthreads();
  if (threadIdx.x == 0 && v1 == (uint64_t)a.v) *a.count = base;
  const bool none = base == base0;  // no id in this range
  // the zeros of rows without an id: a warp takes the next four rows
  auto zeros = [&] {
    if (!a.out) return;
    const bool vec = a.d_bytes % 16 == 0 && a.ld_bytes % 16 == 0 && (uintptr_t)a.out % 16 == 0;
    while (true) {
      int r0 = 0;
      if (lane == 0) r0 = atomicAdd(&next_row, 4);
      r0 = __shfl_sync(~0u, r0, 0);
      if (r0 >= rows) return;
      for (int r = r0; r < min(r0 + 4, rows); r++) {
        if (present[r >> 5] >> (r & 31) & 1) continue;
        unsigned char* p = (unsigned char*)a.out + (v0 + r) * a.ld_bytes;
        if (vec)
          for (int64_t c = lane * 16; c < a.d_bytes; c += 512) *reinterpret_cast<uint4*>(p + c) = make_uint4(0, 0, 0, 0);
        else
          for (int64_t c = lane * 2; c < a.d_bytes; c += 64) *reinterpret_cast<uint16_t*>(p + c) = 0;
      }
    }
  };
  if (threadIdx.x >= kPlacers || none) {
    zeros();
    return;
  }
  // ids of the range, compacted in order of position, then placed
  auto place = [&](int upto) {  // the whole list: batches of one entry a thread
    for (int b = 0; b < upto; b += kPlacers) {
      const int m = min(kPlacers, upto - b);
      const bool on = (int)threadIdx.x < m;
      const int key = on ? list_key[b + threadIdx.x] : -1;
      const unsigned same = __match_any_sync(~0u, key);
      const int rank = __popc(same & ((1u << lane) - 1)), leader = __ffs(same) - 1;
      for (int w = 0; w * 32 < m; w++) {
        if (warp == w) {
          int at = 0;
          if (on && lane == leader) {
            at = start[key];
            start[key] = at + __popc(same);
          }
          at = __shfl_sync(~0u, at, leader) + rank;
          if (on) {
            a.order[at] = list_pos[b + threadIdx.x];
            a.rows[at] = (int)(v0 + key);
          }
        }
        group_sync<kPlacers>();
      }
    }
  };
  for (int64_t i0 = 0; i0 < a.n; i0 += kPlacers * kPerThread) {
    uint64_t r[kPerThread];
    int mine = 0;
    const int64_t at0 = i0 + threadIdx.x * kPerThread;
#pragma unroll
    for (int j = 0; j < kPerThread; j++) r[j] = at0 + j < a.n ? row_at<IDS64>(a.ids, at0 + j, a.first) : ~0ull;
#pragma unroll
    for (int j = 0; j < kPerThread; j++) mine += r[j] >= v0 && r[j] < v1;
    int total;
    int at = list_n + exclusive_scan<kPlacers>(mine, warp_sums, total);
#pragma unroll
    for (int j = 0; j < kPerThread; j++)
      if (r[j] >= v0 && r[j] < v1) {
        list_key[at] = (int)(r[j] - v0);
        list_pos[at++] = (int)(at0 + j);
      }
    const int have = list_n + total;
    group_sync<kPlacers>();
    if (have > kPlacers || i0 + kPlacers * kPerThread >= a.n) {
      place(have);
      if (threadIdx.x == 0) list_n = 0;
    } else if (threadIdx.x == 0) {
      list_n = have;
    }
    group_sync<kPlacers>();
  }
  zeros();
}

// ------------------------------------------------------------------- sum
__device__ __forceinline__ void put(void* out, int64_t i, MType t, float v, bool add) {
  if (t == MType::F32) {
    float* p = (float*)out + i;
    *p = add ? *p + v : v;
  } else if (t == MType::BF16) {
    __nv_bfloat16* p = (__nv_bfloat16*)out + i;
    *p = __float2bfloat16_rn(add ? __bfloat162float(*p) + v : v);
  } else {
    __half* p = (__half*)out + i;
    *p = __float2half_rn(add ? __half2float(*p) + v : v);
  }
}

struct SumArgs {
  const void* grad;
  int64_t ldg, d;
  const int* order;
  const int* rows;
  const int* count;
  float scale;
  void* out;
  int64_t ldo;
  MType ot;
  bool accumulate, vec, out_vec;  // out_vec: out has grad's type and 16-byte rows
  float* head;  // [tiles, d] a tile's part of the row it shares with the tile before
  float* tail;  // [tiles, d] ... of the row it shares with the tile after (and not before)
};

template <typename T>
__global__ void __launch_bounds__(kSumThreads) sum_kernel(const SumArgs a) {
  constexpr int kN = 16 / sizeof(T);
  __shared__ int order[kEntries], rows[kEntries + 2];
  pdl_release();
  pdl_wait();
  const int n = *a.count;
  const int64_t e0 = blockIdx.x * (int64_t)kEntries;
  if (e0 >= n) return;
  const int m = (int)min((int64_t)kEntries, n - e0);
  if (threadIdx.x < kEntries + 2) {  // rows[0] and rows[m + 1]: the neighbours' (or -1)
    const int64_t e = e0 + (int)threadIdx.x - 1;
    rows[threadIdx.x] = e >= 0 && e < n ? a.rows[e] : -1;
  }
  if (threadIdx.x < m) order[threadIdx.x] = a.order[e0 + threadIdx.x];
  __syncthreads();
  const int64_t c = (blockIdx.y * (int64_t)kSumThreads + threadIdx.x) * kN;
  if (c >= a.d) return;
  const int nc = (int)min((int64_t)kN, a.d - c);
  float acc[kN] = {};
  bool started_before = rows[0] == rows[1];
  constexpr int kFly = 8;  // rows of grad in flight a thread
  for (int e0 = 0; e0 < m; e0 += kFly) {
    uint4 x[kFly];
#pragma unroll
    for (int j = 0; j < kFly; j++) {
      x[j] = make_uint4(0, 0, 0, 0);
      if (e0 + j >= m) continue;
      const T* p = (const T*)a.grad + (int64_t)order[e0 + j] * a.ldg + c;
      if (a.vec) {
        x[j] = __ldg(reinterpret_cast<const uint4*>(p));
      } else {
        T* v = reinterpret_cast<T*>(&x[j]);
#pragma unroll
        for (int q = 0; q < kN; q++)
          if (q < nc) v[q] = p[q];
      }
    }
#pragma unroll
    for (int j = 0; j < kFly; j++) {
      const int e = e0 + j;
      if (e >= m) break;
      const T* v = reinterpret_cast<const T*>(&x[j]);
#pragma unroll
      for (int q = 0; q < kN; q++) acc[q] += to_f32<T>(v[q]);
      const int row = rows[e + 1];
      if (rows[e + 2] == row && e + 1 < m) continue;
      const bool goes_on = rows[e + 2] == row;  // into the next tile
      if (started_before || goes_on) {
        float* p = (started_before ? a.head : a.tail) + blockIdx.x * a.d + c;
#pragma unroll
        for (int q = 0; q < kN; q++)
          if (q < nc) p[q] = acc[q];
      } else if (nc == kN && a.out_vec && !a.accumulate) {
        if constexpr (sizeof(T) == 4) {  // (out has grad's type here)
          *reinterpret_cast<float4*>((float*)a.out + row * a.ldo + c) = make_float4(acc[0] * a.scale, acc[1] * a.scale, acc[2] * a.scale, acc[3] * a.scale);
        } else {
          alignas(16) T w[kN];
#pragma unroll
          for (int q = 0; q < kN; q++) w[q] = from_f32<T>(acc[q] * a.scale);
          *reinterpret_cast<uint4*>((T*)a.out + row * a.ldo + c) = *reinterpret_cast<const uint4*>(w);
        }
      } else {
#pragma unroll
        for (int q = 0; q < kN; q++)
          if (q < nc) put(a.out, row * a.ldo + c + q, a.ot, acc[q] * a.scale, a.accumulate);
      }
#pragma unroll
      for (int q = 0; q < kN; q++) acc[q] = 0.f;
      started_before = false;
    }
  }
}

// Rows that cross tiles: the CTAs of the tile where the row starts add its
// tail and the heads of the tiles after it, in order.  Four groups of 64
// threads take neighbouring stretches of the tiles and are added in their
// order; a CTA has 256 columns (a few ids make up much of a batch, so one
// row's chain can be most of the work).  Most CTAs find nothing to join:
// they are small, so that the GPU is through with them at once.
constexpr int kJoinThreads = 64, kJoinColumns = 4 * kJoinThreads, kStretches = 4;
__global__ void __launch_bounds__(kJoinThreads* kStretches) join_kernel(const SumArgs a) {
  __shared__ float4 part[kStretches][kJoinThreads];
  pdl_release();
  pdl_wait();
  const int n = *a.count;
  const int64_t t = blockIdx.x, e0 = t * kEntries, e1 = e0 + kEntries;
  if (e1 >= n) return;
  const int row = a.rows[e1 - 1], next = a.rows[e1], first = a.rows[e0], before = e0 > 0 ? a.rows[e0 - 1] : -1;
  if (next != row || (first == row && before == row)) return;  // does not cross, or starts earlier
  // the tiles after t that begin with the row
  int64_t heads = 0;
  for (int more = blockDim.x; more == (int)blockDim.x; heads += more) {
    const int64_t e = e1 + (heads + threadIdx.x) * kEntries;
    more = __syncthreads_count(e < n && a.rows[e] == row);
  }
  const int group = threadIdx.x / kJoinThreads, lane = threadIdx.x % kJoinThreads;
  const int64_t per = (heads + kStretches - 1) / kStretches, h0 = t + 1 + group * per, h1 = min(t + 1 + heads, h0 + per);
  const bool vec = a.d % 4 == 0;  // (head and tail start on 16 bytes)
  auto load = [&](const float* p, int64_t left) {
    if (vec) return *reinterpret_cast<const float4*>(p);
    return make_float4(p[0], left > 1 ? p[1] : 0.f, left > 2 ? p[2] : 0.f, left > 3 ? p[3] : 0.f);
  };
  for (int64_t c0 = blockIdx.y * (int64_t)kJoinColumns; c0 < a.d; c0 += gridDim.y * (int64_t)kJoinColumns) {
    const int64_t c = c0 + lane * 4;
    float4 v = make_float4(0, 0, 0, 0);
    if (c < a.d) {
#pragma unroll 8
      for (int64_t h = h0; h < h1; h++) {
        const float4 x = load(a.head + h * a.d + c, a.d - c);
        v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      }
    }
    part[group][lane] = v;
    __syncthreads();
    if (group == 0 && c < a.d) {
      float4 s = load(a.tail + t * a.d + c, a.d - c);
#pragma unroll
      for (int w = 0; w < kStretches; w++) {
        const float4 x = part[w][lane];
        s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
      }
      const float e[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int q = 0; q < 4; q++)
        if (c + q < a.d) put(a.out, row * a.ldo + c + q, a.ot, e[q] * a.scale, a.accumulate);
    }
    __syncthreads();
  }
}

}  // namespace

void embedding(MType t, const void* table, int64_t v, int64_t d, int64_t ldt, const void* ids, bool ids64, int64_t n,
               int64_t first, float scale, void* out, int64_t ldo, cudaStream_t s) {
  if (n == 0 || d == 0) return;
  auto go = [&](auto tv) {
    using T = decltype(tv);
    const int kn = 16 / (int)sizeof(T);
    const bool vec = d % kn == 0 && ldt % kn == 0 && ldo % kn == 0 && (uintptr_t)table % 16 == 0 && (uintptr_t)out % 16 == 0;
    // few rows: several warps a row, down to 512 bytes each
    const int64_t want = (int64_t)ctx().sm_count * 16;
    const int64_t most = std::max<int64_t>(1, d * (int64_t)sizeof(T) / 512);
    const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(most, want / n));
    const int64_t blocks = (n * parts + 7) / 8;
    if (blocks > 0x7fffffff) throw Error(ErrKind::InvalidArgument, "embedding: too many ids");
    auto launch = [&](auto kern) {
      launch_pdl(kern, dim3((unsigned)blocks), dim3(256), 0, s, (const T*)table, v, d, ldt, ids, n, first, scale, (T*)out, ldo, parts);
    };
    if (ids64)
      vec ? launch(lookup_kernel<T, true, true>) : launch(lookup_kernel<T, true, false>);
    else
      vec ? launch(lookup_kernel<T, false, true>) : launch(lookup_kernel<T, false, false>);
    count_launch();
  };
  if (t == MType::F32)
    go(float{});
  else if (t == MType::BF16)
    go(__nv_bfloat16{});
  else
    go(__half{});
}

void embedding_grad(MType gt, const void* grad, int64_t ldg, const void* ids, bool ids64, int64_t n, int64_t v,
                    int64_t d, int64_t first, float scale, MType ot, void* out, int64_t ldo, bool accumulate,
                    cudaStream_t s) {
  if (v == 0 || d == 0) return;
  if (n >= (int64_t)1 << 31 || v >= (int64_t)1 << 31) throw Error(ErrKind::InvalidArgument, "embedding_grad: 2^31 ids or rows");
  const int sms = ctx().sm_count;
  const int64_t range = std::min<int64_t>((v + sms - 1) / sms, 32768);  // its counters fit shared memory
  const int ctas = (int)((v + range - 1) / range);
  const size_t smem = (size_t)(range + 2 * kList) * 4;
  const int64_t tiles = (n + kEntries - 1) / kEntries;
  Workspace ws((size_t)(2 * n + 4) * 4 + (size_t)(2 * tiles * d) * 4, s);
  SortArgs a{};
  a.ids = ids, a.n = n, a.first = first, a.v = v, a.range = range;
  float* parts = (float*)ws.p;
  a.order = (int*)(parts + 2 * tiles * d), a.rows = a.order + n, a.count = a.rows + n;
  a.out = accumulate ? nullptr : out;
  a.d_bytes = d * msize(ot), a.ld_bytes = ldo * msize(ot);
  auto sort = [&](auto kern) {
    ensure_dynamic_smem((const void*)kern, smem);
    launch_pdl(kern, dim3((unsigned)ctas), dim3(kSortThreads), smem, s, a);
    count_launch();
  };
  ids64 ? sort(sort_kernel<true>) : sort(sort_kernel<false>);
  if (n == 0) return;
  SumArgs b{};
  b.grad = grad, b.ldg = ldg, b.d = d, b.order = a.order, b.rows = a.rows, b.count = a.count;
  b.scale = scale, b.out = out, b.ldo = ldo, b.ot = ot, b.accumulate = accumulate;
  b.head = parts, b.tail = parts + tiles * d;
  const int kn = 16 / msize(gt);
  b.vec = d % kn == 0 && ldg % kn == 0 && (uintptr_t)grad % 16 == 0;
  b.out_vec = ot == gt && ldo % kn == 0 && (uintptr_t)out % 16 == 0;
  const dim3 grid((unsigned)tiles, (unsigned)((d + kSumThreads * kn - 1) / (kSumThreads * kn)));
  if (gt == MType::F32)
    launch_pdl(sum_kernel<float>, grid, dim3(kSumThreads), 0, s, b);
  else if (gt == MType::BF16)
    launch_pdl(sum_kernel<__nv_bfloat16>, grid, dim3(kSumThreads), 0, s, b);
  else
    launch_pdl(sum_kernel<__half>, grid, dim3(kSumThreads), 0, s, b);
  count_launch();
  if (tiles > 1) {
    const unsigned chunks = (unsigned)std::min<int64_t>(8, (d + kJoinColumns - 1) / kJoinColumns);
    launch_pdl(join_kernel, dim3((unsigned)(tiles - 1), chunks), dim3(kJoinThreads * kStretches), 0, s, b);
    count_launch();
  }
}

}  // namespace ndt
