// mmp_embedding / mmp_embedding_grad: rows of a table by token id, times a
// scale, and the gradient of the table,
//   out[n, :] = scale * weight[ids[n], :]
//   grad_weight[v, :] = scale * sum over n with ids[n] = v, in order of n, of grad[n, :].
// The reference has take (indexing.py:24-60; numpy on the host) without a
// scale or a gradient.  Products and sums are in float32 (float64 for
// float64 tables) and each output is rounded once.
//
// An id outside [0, rows) gives a row of zeros in the lookup, adds nothing in
// the gradient, and sets device error 5, as mmp_gather does for an offset.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "mmp_device.cuh"
#include "mmp_internal.h"

namespace mmpd {

template <class T> struct EmbAcc { typedef float type; };
template <> struct EmbAcc<double> { typedef double type; };

template <class T, class I>
__global__ void __launch_bounds__(256) emb_kernel(const T *__restrict__ w, long long rows, long long width,
                                                  long long w_stride, const I *__restrict__ ids, long long n,
                                                  typename EmbAcc<T>::type scale, T *__restrict__ out, int *err) {
  typedef typename EmbAcc<T>::type S;
  for (long long r = blockIdx.x; r < n; r += gridDim.x) {
    const long long id = (long long)ids[r];
    const bool ok = id >= 0 && id < rows;
    if (!ok && threadIdx.x == 0) atomicExch(err, 5);
    for (long long j = threadIdx.x; j < width; j += blockDim.x)
      out[r * width + j] = ok ? Cvt<T, S>::f((S)Cvt<S, T>::f(w[id * w_stride + j]) * scale) : Cvt<T, S>::f(S(0));
  }
}

// One warp per row of the table walks the ids and adds the rows of the
// gradient that are its own, 32 columns at a time.
template <class T, class I>
__global__ void __launch_bounds__(256) emb_grad_kernel(const I *__restrict__ ids, long long n, const T *__restrict__ grad,
                                                       long long g_stride, long long rows, long long width,
                                                       typename EmbAcc<T>::type scale, long long padding,
                                                       T *__restrict__ out, int *err) {
  typedef typename EmbAcc<T>::type S;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (blockIdx.x == 0)
    for (long long i = threadIdx.x; i < n; i += blockDim.x) {
      const long long id = (long long)ids[i];
      if (id < 0 || id >= rows) atomicExch(err, 5);
    }
  for (long long v = (long long)blockIdx.x * nw + w; v < rows; v += (long long)gridDim.x * nw) {
    for (long long j0 = 0; j0 < width; j0 += 32) {
      const long long j = j0 + lane;
      S acc = S(0);
      if (v != padding)
        for (long long i0 = 0; i0 < n; i0 += 32) {
          unsigned m = __ballot_sync(0xffffffffu, i0 + lane < n && (long long)ids[i0 + lane] == v);
          for (; m; m &= m - 1)
            if (j < width) acc += Cvt<S, T>::f(grad[(i0 + __ffs(m) - 1) * g_stride + j]);
        }
      if (j < width) out[v * width + j] = Cvt<T, S>::f(acc * scale);
    }
  }
}

}  // namespace mmpd

namespace {

int emb_check(const char *what, int dtype, int ids_dtype, int64_t rows, int64_t width, int64_t n) {
  if (rows < 0 || width < 0 || n < 0) return mmp::set_error(MMP_E_ARG, std::string(what) + ": negative size");
  if (dtype != MMP_FLOAT16 && dtype != MMP_FLOAT32 && dtype != MMP_FLOAT64)
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": needs a floating dtype");
  if (ids_dtype != MMP_INT32 && ids_dtype != MMP_INT64)
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": ids must be int32 or int64");
  if (rows > INT32_MAX || n > INT32_MAX || width > INT32_MAX)
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": a size passes 2^31 - 1");
  return MMP_OK;
}

unsigned emb_grid(long long want) {
  const long long cap = (long long)mmp::sm_count() * 16;
  return (unsigned)(want < cap ? want : cap);
}

template <class T, class I>
int run_emb(const void *w, int64_t rows, int64_t width, int64_t w_stride, const void *ids, int64_t n, double scale,
            void *out) {
  mmpd::emb_kernel<T, I><<<emb_grid(n), 256, 0, mmp::stream()>>>((const T *)w, rows, width, w_stride, (const I *)ids,
                                                               n, (typename mmpd::EmbAcc<T>::type)scale, (T *)out,
                                                               mmp::device_error_word());
  MMP_LAUNCH_CHECK("embedding");
  return MMP_OK;
}

template <class T, class I>
int run_emb_grad(const void *ids, int64_t n, const void *grad, int64_t g_stride, int64_t rows, int64_t width,
                 double scale, int64_t padding, void *out) {
  mmpd::emb_grad_kernel<T, I><<<emb_grid((rows + 7) / 8), 256, 0, mmp::stream()>>>(
      (const I *)ids, n, (const T *)grad, g_stride, rows, width, (typename mmpd::EmbAcc<T>::type)scale, padding,
      (T *)out, mmp::device_error_word());
  MMP_LAUNCH_CHECK("embedding_grad");
  return MMP_OK;
}

}  // namespace

#define MMP_EMB_DISPATCH(F, ...)                                                                           \
  if (dtype == MMP_FLOAT16)                                                                                \
    return ids_dtype == MMP_INT32 ? F<__half, int>(__VA_ARGS__) : F<__half, long long>(__VA_ARGS__);       \
  if (dtype == MMP_FLOAT32)                                                                                \
    return ids_dtype == MMP_INT32 ? F<float, int>(__VA_ARGS__) : F<float, long long>(__VA_ARGS__);         \
  return ids_dtype == MMP_INT32 ? F<double, int>(__VA_ARGS__) : F<double, long long>(__VA_ARGS__)

extern "C" {

int mmp_embedding(int dtype, const void *weight, int64_t rows, int64_t width, int64_t w_stride, int ids_dtype,
                  const void *ids, int64_t n, double scale, void *out) {
  int rc = emb_check("embedding", dtype, ids_dtype, rows, width, n);
  if (rc) return rc;
  if (n == 0 || width == 0) return MMP_OK;
  if (!ids || !out || (rows && !weight)) return mmp::set_error(MMP_E_ARG, "embedding: null pointer");
  if (!mmp::stream()) return mmp::set_error(MMP_E_CUDA, "no CUDA device available");
  MMP_EMB_DISPATCH(run_emb, weight, rows, width, w_stride, ids, n, scale, out);
}

int mmp_embedding_grad(int dtype, int ids_dtype, const void *ids, int64_t n, const void *grad, int64_t g_stride,
                       int64_t rows, int64_t width, double scale, int64_t padding_idx, void *grad_weight) {
  int rc = emb_check("embedding_grad", dtype, ids_dtype, rows, width, n);
  if (rc) return rc;
  if (rows == 0 || width == 0) return MMP_OK;
  if ((n && (!ids || !grad)) || !grad_weight) return mmp::set_error(MMP_E_ARG, "embedding_grad: null pointer");
  if (!mmp::stream()) return mmp::set_error(MMP_E_CUDA, "no CUDA device available");
  MMP_EMB_DISPATCH(run_emb_grad, ids, n, grad, g_stride, rows, width, scale, padding_idx, grad_weight);
}

}  // extern "C"
