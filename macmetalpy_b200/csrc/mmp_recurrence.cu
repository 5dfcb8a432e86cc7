// mmp_recurrence / mmp_recurrence_grad: the first-order linear recurrence
//   h_t = f_t h_{t-1} + u_t          along the middle axis of (outer, steps, inner)
// with f = a, u = x (plain) or f = sigmoid(a), u = (1 - f) x (gated), and its
// gradient
//   g_t = grad_t + c_{t+1},  c_t = f_t g_t,  c_{steps+1} = grad_state
//   plain: grad_a = g_t h_{t-1},                    grad_x = g_t
//   gated: grad_a = g_t (h_{t-1} - x_t) f (1 - f),  grad_x = g_t (1 - f)
//   grad_h0 = c_1.
// The reference has cumsum / cumprod (reductions.py:661-705) and no decayed
// form.  The running state is held in float32 (float64 for float64 arrays)
// and each output is rounded to the array's type once.
//
// A chain is one (outer, inner) pair; its steps depend on one another, the
// chains do not.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "mmp_device.cuh"
#include "mmp_internal.h"

namespace mmpd {

// Element strides of a 3-D operand over (outer, step); inner has stride 1.
struct RecView {
  const void *p;
  long long so, st;
};

template <class T> struct RecState { typedef float type; };
template <> struct RecState<double> { typedef double type; };

__device__ __forceinline__ float rec_load(const __half *p) { return __half2float(*p); }
__device__ __forceinline__ float rec_load(const float *p) { return *p; }
__device__ __forceinline__ double rec_load(const double *p) { return *p; }
__device__ __forceinline__ void rec_store(__half *p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void rec_store(float *p, float v) { *p = v; }
__device__ __forceinline__ void rec_store(double *p, double v) { *p = v; }

// f = sigmoid(z) and 1 - f from e = exp(-|z|) in (0, 1], so that neither
// cancels and z = +-inf gives exactly 1 and 0 (e = 0): a gate of +inf keeps
// the state as it is, one of -inf replaces it.
template <class S>
__device__ __forceinline__ void rec_gate(S z, S &f, S &rest) {
  const S e = exp(-fabs(z));
  const S r = S(1) / (S(1) + e);
  const S q = e * r;
  f = z >= S(0) ? r : q;
  rest = z >= S(0) ? q : r;
  if (z != z) f = rest = z;
}

template <class T, bool GATED>
__global__ void __launch_bounds__(128) rec_kernel(RecView a, RecView x, const typename RecState<T>::type *h0, RecView h,
                                                  typename RecState<T>::type *state, long long chains, long long steps,
                                                  long long inner) {
  typedef typename RecState<T>::type S;
  const long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= chains) return;
  const long long o = c / inner, i = c - o * inner;
  const T *pa = (const T *)a.p + o * a.so + i;
  const T *px = (const T *)x.p + o * x.so + i;
  T *ph = (T *)h.p + o * h.so + i;
  S s = h0 ? h0[c] : S(0);
  for (long long t = 0; t < steps; ++t) {
    S f = rec_load(pa + t * a.st), u = rec_load(px + t * x.st);
    if (GATED) {
      S rest;
      rec_gate(f, f, rest);
      u *= rest;
    }
    s = f * s + u;
    rec_store(ph + t * h.st, s);
  }
  if (state) state[c] = s;
}

template <class T, bool GATED>
__global__ void __launch_bounds__(128) rec_grad_kernel(RecView a, RecView x, RecView h, RecView grad,
                                                       const typename RecState<T>::type *h0,
                                                       const typename RecState<T>::type *grad_state, RecView ga,
                                                       RecView gx, typename RecState<T>::type *grad_h0,
                                                       long long chains, long long steps, long long inner) {
  typedef typename RecState<T>::type S;
  const long long ch = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (ch >= chains) return;
  const long long o = ch / inner, i = ch - o * inner;
  const T *pa = (const T *)a.p + o * a.so + i;
  const T *px = GATED ? (const T *)x.p + o * x.so + i : nullptr;
  const T *ph = (const T *)h.p + o * h.so + i;
  const T *pg = (const T *)grad.p + o * grad.so + i;
  T *pga = (T *)ga.p + o * ga.so + i;
  T *pgx = (T *)gx.p + o * gx.so + i;
  S c = grad_state ? grad_state[ch] : S(0);
  for (long long t = steps - 1; t >= 0; --t) {
    S f = rec_load(pa + t * a.st);
    const S g = rec_load(pg + t * grad.st) + c;
    const S hp = t ? rec_load(ph + (t - 1) * h.st) : h0 ? h0[ch] : S(0);
    if (GATED) {
      S rest;
      rec_gate(f, f, rest);
      rec_store(pga + t * ga.st, g * (hp - rec_load(px + t * x.st)) * (f * rest));
      rec_store(pgx + t * gx.st, g * rest);
    } else {
      rec_store(pga + t * ga.st, g * hp);
      rec_store(pgx + t * gx.st, g);
    }
    c = f * g;
  }
  if (grad_h0) grad_h0[ch] = c;
}

}  // namespace mmpd

namespace {

using mmpd::RecView;

// Sizes that a launch and the kernels' 64-bit offsets can address.
int rec_sizes(const char *what, int dtype, int64_t outer, int64_t steps, int64_t inner) {
  if (outer < 0 || steps < 0 || inner < 0) return mmp::set_error(MMP_E_ARG, std::string(what) + ": negative size");
  if (dtype != MMP_FLOAT16 && dtype != MMP_FLOAT32 && dtype != MMP_FLOAT64)
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": needs a floating dtype");
  if (inner && outer > (INT64_C(1) << 36) / inner)
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": more than 2^36 chains");
  return MMP_OK;
}

template <class T, bool G>
int run_fwd(RecView a, RecView x, const void *h0, RecView h, void *state, long long chains, long long steps,
            long long inner) {
  typedef typename mmpd::RecState<T>::type S;
  mmpd::rec_kernel<T, G><<<(unsigned)((chains + 127) / 128), 128, 0, mmp::stream()>>>(
      a, x, (const S *)h0, h, (S *)state, chains, steps, inner);
  MMP_LAUNCH_CHECK("recurrence");
  return MMP_OK;
}

template <class T, bool G>
int run_bwd(RecView a, RecView x, RecView h, RecView grad, const void *h0, const void *grad_state, RecView ga,
            RecView gx, void *grad_h0, long long chains, long long steps, long long inner) {
  typedef typename mmpd::RecState<T>::type S;
  mmpd::rec_grad_kernel<T, G><<<(unsigned)((chains + 127) / 128), 128, 0, mmp::stream()>>>(
      a, x, h, grad, (const S *)h0, (const S *)grad_state, ga, gx, (S *)grad_h0, chains, steps, inner);
  MMP_LAUNCH_CHECK("recurrence_grad");
  return MMP_OK;
}

}  // namespace

extern "C" {

int mmp_recurrence(int dtype, int gated, int64_t outer, int64_t steps, int64_t inner, const void *a, int64_t a_so,
                   int64_t a_st, const void *x, int64_t x_so, int64_t x_st, const void *h0, void *h, int64_t h_so,
                   int64_t h_st, void *state) {
  int rc = rec_sizes("recurrence", dtype, outer, steps, inner);
  if (rc) return rc;
  const long long chains = outer * inner;
  if (chains == 0) return MMP_OK;
  if (steps > 0 && (!a || !x || !h)) return mmp::set_error(MMP_E_ARG, "recurrence: null pointer");
  if (!mmp::stream()) return mmp::set_error(MMP_E_CUDA, "no CUDA device available");
  const RecView va{a, a_so, a_st}, vx{x, x_so, x_st}, vh{h, h_so, h_st};
#define MMP_REC(T) \
  return gated ? run_fwd<T, true>(va, vx, h0, vh, state, chains, steps, inner) \
               : run_fwd<T, false>(va, vx, h0, vh, state, chains, steps, inner)
  if (dtype == MMP_FLOAT16) MMP_REC(__half);
  if (dtype == MMP_FLOAT32) MMP_REC(float);
  MMP_REC(double);
#undef MMP_REC
}

int mmp_recurrence_grad(int dtype, int gated, int64_t outer, int64_t steps, int64_t inner, const void *a, int64_t a_so,
                        int64_t a_st, const void *x, int64_t x_so, int64_t x_st, const void *h, int64_t h_so,
                        int64_t h_st, const void *grad, int64_t g_so, int64_t g_st, const void *h0,
                        const void *grad_state, void *grad_a, int64_t ga_so, int64_t ga_st, void *grad_x,
                        int64_t gx_so, int64_t gx_st, void *grad_h0) {
  int rc = rec_sizes("recurrence_grad", dtype, outer, steps, inner);
  if (rc) return rc;
  const long long chains = outer * inner;
  if (chains == 0) return MMP_OK;
  if (steps > 0 && (!a || (gated && !x) || !h || !grad || !grad_a || !grad_x))
    return mmp::set_error(MMP_E_ARG, "recurrence_grad: null pointer");
  if (!mmp::stream()) return mmp::set_error(MMP_E_CUDA, "no CUDA device available");
  const RecView va{a, a_so, a_st}, vx{x, x_so, x_st}, vh{h, h_so, h_st}, vg{grad, g_so, g_st},
      vga{grad_a, ga_so, ga_st}, vgx{grad_x, gx_so, gx_st};
#define MMP_REC(T)                                                                                            \
  return gated ? run_bwd<T, true>(va, vx, vh, vg, h0, grad_state, vga, vgx, grad_h0, chains, steps, inner)   \
               : run_bwd<T, false>(va, vx, vh, vg, h0, grad_state, vga, vgx, grad_h0, chains, steps, inner)
  if (dtype == MMP_FLOAT16) MMP_REC(__half);
  if (dtype == MMP_FLOAT32) MMP_REC(float);
  MMP_REC(double);
#undef MMP_REC
}

}  // extern "C"
