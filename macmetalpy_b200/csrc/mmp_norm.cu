// mmp_global_norm: the Euclidean norm over a list of arrays,
//   norm = sqrt(sum over the arrays of sum x^2),
// and, with outputs, every array times coef = 1 if norm <= max_norm else
// max_norm / norm (clipping by the global norm).  The reference has only
// reductions of one array (reductions.py:74-163).
//
// Squares and their sums are in float64: a float32 square overflows from
// 1.8e19 on, and the sum runs over billions of elements.  The list travels
// as kernel parameters, kTable arrays a launch, so a call needs no copy of
// it to the device.  Every block walks chunks of the concatenated list and
// leaves one partial; the blocks of the second kernel each add all partials
// in the same order, so the result does not depend on timing.
// 290 arrays of 354 M elements, mostly float16: 366 us a call, of which the
// first pass (708 MB) takes 124 us and the second (1416 MB, backwards, as what
// was read last lies in L2) 222: 5.7 and 6.4 TB/s.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "mmp_chain.cuh"
#include "mmp_device.cuh"
#include "mmp_internal.h"

namespace mmpd {

constexpr int kNormTable = 512, kNormFew = 32;  // arrays a launch; a short list travels in 1 KB, not 16
constexpr int kNormThreads = 256;
constexpr long long kNormChunk = 16384;  // elements

struct NormEntry {
  const void *x;
  void *y;
  long long n;
  int first;  // chunks of the entries before this one
  int dtype;
};
template <int N> struct NormTable {
  int count;
  int chunks;
  NormEntry e[N];
};

template <int N> __device__ __forceinline__ const NormEntry &norm_find(const NormTable<N> &t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return t.e[lo];
}

// Sum over the block of one double per thread, in a fixed order; thread 0's
// return value is the sum.
__device__ __forceinline__ double norm_block_sum(double v) {
  __shared__ double s[kNormThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) {
    v = threadIdx.x < kNormThreads / 32 ? s[threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_down_sync(0xffffffffu, v, o);
  }
  return v;
}

template <class T> struct alignas(16) NormVec { T v[16 / sizeof(T)]; };

// The sum of a chunk's squares.  16-byte loads, four ahead, where the chunk is
// aligned to them (chunks start a multiple of 16 bytes into their array).
template <class T>
__device__ __forceinline__ double norm_chunk(const T *x, int n) {
  constexpr int PE = 16 / (int)sizeof(T);
  double acc = 0.0;
  int done = 0;
  if (((uintptr_t)x & 15) == 0) {
    const NormVec<T> *p = reinterpret_cast<const NormVec<T> *>(x);
    const int pieces = n / PE;
    for (int i = threadIdx.x; i < pieces; i += 4 * kNormThreads) {
      NormVec<T> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u * kNormThreads < pieces) v[u] = p[i + u * kNormThreads];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (i + u * kNormThreads < pieces) {
#pragma unroll
          for (int e = 0; e < PE; ++e) {
            const double f = Cvt<double, T>::f(v[u].v[e]);
            acc = fma(f, f, acc);
          }
        }
      }
    }
    done = pieces * PE;
  }
  for (int i = done + threadIdx.x; i < n; i += kNormThreads) {
    const double f = Cvt<double, T>::f(x[i]);
    acc = fma(f, f, acc);
  }
  return acc;
}

template <int N>
__global__ void __launch_bounds__(kNormThreads, 4) norm_sum_kernel(const __grid_constant__ NormTable<N> t,
                                                                   double *partial) {
  double acc = 0.0;
  chain_wait();
  chain_next();
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const NormEntry &e = norm_find(t, c);
    const long long at = (long long)(c - e.first) * kNormChunk;
    const int n = (int)(e.n - at < kNormChunk ? e.n - at : kNormChunk);
    if (e.dtype == MMP_DT_FLOAT16) acc += norm_chunk((const __half *)e.x + at, n);
    else if (e.dtype == MMP_DT_FLOAT32) acc += norm_chunk((const float *)e.x + at, n);
    else acc += norm_chunk((const double *)e.x + at, n);
  }
  acc = norm_block_sum(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// The norm from the partials, the same in every thread of the block.
__device__ __forceinline__ double norm_total(const double *partial, int n) {
  __shared__ double total;
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += kNormThreads) acc += partial[i];
  acc = norm_block_sum(acc);
  if (threadIdx.x == 0) total = sqrt(acc);
  __syncthreads();
  return total;
}

template <class T, class S>
__device__ __forceinline__ void norm_scale(const T *x, T *y, int n, S coef) {
  constexpr int PE = 16 / (int)sizeof(T);
  int done = 0;
  if ((((uintptr_t)x | (uintptr_t)y) & 15) == 0) {
    const NormVec<T> *p = reinterpret_cast<const NormVec<T> *>(x);
    NormVec<T> *q = reinterpret_cast<NormVec<T> *>(y);
    const int pieces = n / PE;
    for (int i = threadIdx.x; i < pieces; i += 4 * kNormThreads) {
      NormVec<T> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u * kNormThreads < pieces) v[u] = p[i + u * kNormThreads];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (i + u * kNormThreads < pieces) {
#pragma unroll
          for (int e = 0; e < PE; ++e) v[u].v[e] = Cvt<T, S>::f(Cvt<S, T>::f(v[u].v[e]) * coef);
          q[i + u * kNormThreads] = v[u];
        }
      }
    }
    done = pieces * PE;
  }
  for (int i = done + threadIdx.x; i < n; i += kNormThreads) y[i] = Cvt<T, S>::f(Cvt<S, T>::f(x[i]) * coef);
}

// The same where float32 holds fewer bits of the coefficient, or none of it
// (below 2^-126: huge arrays and a small limit).  A call of its own, so that
// the usual one keeps its registers.
__device__ __noinline__ void norm_scale_small(const float *x, float *y, int n, double coef) {
  for (int i = threadIdx.x; i < n; i += kNormThreads) y[i] = (float)(x[i] * coef);
}

template <int N>
__global__ void __launch_bounds__(kNormThreads, 4) norm_scale_kernel(const __grid_constant__ NormTable<N> t,
                                                                  const double *partial, int npartial, double max_norm,
                                                                  int norm_f64, void *norm_out) {
  chain_wait();
  chain_next();
  const double norm = norm_total(partial, npartial);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) {
    if (norm_f64) *(double *)norm_out = norm;
    else *(float *)norm_out = (float)norm;
  }
  const double coef = norm <= max_norm ? 1.0 : max_norm / norm;
  const bool small = coef < 0x1p-126 && coef > 0.0;
  for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {  // what was read last lies in L2
    const NormEntry &e = norm_find(t, c);
    if (coef == 1.0 && e.x == e.y) continue;  // in place, nothing to scale
    const long long at = (long long)(c - e.first) * kNormChunk;
    const int n = (int)(e.n - at < kNormChunk ? e.n - at : kNormChunk);
    if (e.dtype == MMP_DT_FLOAT16) norm_scale((const __half *)e.x + at, (__half *)e.y + at, n, (float)coef);
    else if (e.dtype == MMP_DT_FLOAT32 && small) norm_scale_small((const float *)e.x + at, (float *)e.y + at, n, coef);
    else if (e.dtype == MMP_DT_FLOAT32) norm_scale((const float *)e.x + at, (float *)e.y + at, n, (float)coef);
    else norm_scale((const double *)e.x + at, (double *)e.y + at, n, coef);
  }
}

}  // namespace mmpd

namespace {

using mmpd::NormTable;
using mmpd::kNormFew;
using mmpd::kNormTable;

// The first entries of a table, for the kernels of short lists.
NormTable<kNormFew> norm_few(const NormTable<kNormTable> &t) {
  NormTable<kNormFew> f;
  f.count = t.count;
  f.chunks = t.chunks;
  for (int i = 0; i < t.count; ++i) f.e[i] = t.e[i];
  return f;
}

// The next part of the list, from array *at on: at most kNormTable arrays
// with elements.
int norm_fill(NormTable<kNormTable> &t, int64_t *at, int64_t count, const int *dtypes, const void *const *x, void *const *y,
              const int64_t *sizes) {
  t.count = 0;
  long long chunks = 0;
  int64_t i = *at;
  for (; i < count && t.count < mmpd::kNormTable; ++i) {
    if (sizes[i] == 0) continue;
    const long long mine = (sizes[i] + mmpd::kNormChunk - 1) / mmpd::kNormChunk;
    if (chunks + mine > INT32_MAX) return mmp::set_error(MMP_E_ARG, "global_norm: the arrays are too long");
    mmpd::NormEntry &e = t.e[t.count++];
    e.x = x[i];
    e.y = y ? y[i] : nullptr;
    e.n = sizes[i];
    e.first = (int)chunks;
    e.dtype = dtypes[i];
    chunks += mine;
  }
  t.chunks = (int)chunks;
  *at = i;
  return MMP_OK;
}

}  // namespace

extern "C" int mmp_global_norm(int64_t count, const int *dtypes, const void *const *x, void *const *y,
                               const int64_t *sizes, double max_norm, int norm_dtype, void *norm) {
  if (count < 0) return mmp::set_error(MMP_E_ARG, "global_norm: negative count");
  if (!norm || (count && (!dtypes || !x || !sizes))) return mmp::set_error(MMP_E_ARG, "global_norm: null pointer");
  if (norm_dtype != MMP_FLOAT32 && norm_dtype != MMP_FLOAT64)
    return mmp::set_error(MMP_E_ARG, "global_norm: the norm is float32 or float64");
  for (int64_t i = 0; i < count; ++i) {
    if (dtypes[i] != MMP_FLOAT16 && dtypes[i] != MMP_FLOAT32 && dtypes[i] != MMP_FLOAT64)
      return mmp::set_error(MMP_E_ARG, "global_norm: needs floating dtypes");
    if (sizes[i] < 0) return mmp::set_error(MMP_E_ARG, "global_norm: negative size");
    if (sizes[i] && (!x[i] || (y && !y[i]))) return mmp::set_error(MMP_E_ARG, "global_norm: null pointer");
  }
  if (!mmp::device_error_word()) return mmp::set_error(MMP_E_CUDA, "no CUDA device available");
  cudaStream_t st = mmp::stream();
  const int64_t most = (int64_t)mmp::sm_count() * 8;
  const int64_t launches = count ? (count + mmpd::kNormTable - 1) / mmpd::kNormTable : 1;
  double *partial = nullptr;
  MMP_CUDA_TRY(cudaMallocAsync((void **)&partial, (size_t)(launches * most) * sizeof(double), st));
  static thread_local NormTable<kNormTable> t;
  int rc = MMP_OK, npartial = 0;
  for (int64_t at = 0; at < count && !rc;) {
    rc = norm_fill(t, &at, count, dtypes, x, y, sizes);
    if (rc || !t.chunks) continue;
    const int grid = (int)(t.chunks < most ? t.chunks : most);
    rc = t.count <= kNormFew ? mmp::launch_after(mmpd::norm_sum_kernel<kNormFew>, grid, mmpd::kNormThreads, 0, 1,
                                                 norm_few(t), partial + npartial)
                             : mmp::launch_after(mmpd::norm_sum_kernel<kNormTable>, grid, mmpd::kNormThreads, 0, 1, t,
                                                 partial + npartial);
    npartial += grid;
  }
  // with one table the one just filled serves both kernels
  int64_t at = 0;
  bool first = true;
  while (!rc && (first || (y && at < count))) {
    if (y) rc = norm_fill(t, &at, count, dtypes, x, y, sizes);
    else t.count = t.chunks = 0;
    if (rc) break;
    const int grid = (int)(t.chunks < 1 ? 1 : t.chunks < most ? t.chunks : most);
    void *const to = first ? norm : nullptr;
    const int f64 = norm_dtype == MMP_FLOAT64;
    rc = t.count <= kNormFew ? mmp::launch_after(mmpd::norm_scale_kernel<kNormFew>, grid, mmpd::kNormThreads, 0, 1,
                                                 norm_few(t), partial, npartial, max_norm, f64, to)
                             : mmp::launch_after(mmpd::norm_scale_kernel<kNormTable>, grid, mmpd::kNormThreads, 0, 1, t,
                                                 partial, npartial, max_norm, f64, to);
    first = false;
  }
  cudaFreeAsync(partial, st);
  return rc;
}
