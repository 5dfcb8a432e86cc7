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
// Both directions are one scan of affine maps s -> f s + u (backward: u = f
// grad, from the last step to the first).  A span of steps composes to
// s -> A s + H with A the product of its f and H its result from s = 0, so
// spans are worked on side by side and joined by their (A, H):
//   lane     one group of VEC neighbouring chains (a chain: one (outer, inner))
//   warp     a span of S steps of its 32 groups
//   block    `warps` spans after one another, joined through shared memory
//   cluster  its blocks' spans after one another, joined through each
//            other's shared memory; then the cluster moves on along the axis
// Every input is read once and every output written once; no block waits for
// one outside its cluster, nothing is allocated, and the order of all
// operations is fixed by the sizes.  What bounds it is HBM traffic, so the
// loads run ahead: each thread copies the steps of its next spans with
// cp.async into a ring in shared memory that only it reads.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "mmp_device.cuh"
#include "mmp_internal.h"

namespace mmpd {

namespace cg = cooperative_groups;

// Element strides of a 3-D operand over (outer, step); inner has stride 1.
struct RecView {
  const void *p;
  long long so, st;
};

template <class T> struct RecState { typedef float type; };
template <> struct RecState<double> { typedef double type; };

// f = sigmoid(z) and 1 - f from e = exp(-|z|) in (0, 1], so that neither
// cancels and z = +-inf gives exactly 1 and 0 (e = 0): a gate of +inf keeps
// the state as it is, one of -inf replaces it.  A NaN goes to both.  float16
// gates use __expf, whose error of 2 + 1.2 |z| ulp is far below theirs.
template <class T> __device__ __forceinline__ float rec_exp(float z) { return expf(z); }
template <> __device__ __forceinline__ float rec_exp<__half>(float z) { return __expf(z); }
template <class T> __device__ __forceinline__ void rec_gate(float z, float &f, float &rest) {
  const float e = rec_exp<T>(-fabsf(z));
  const float r = __fdividef(1.0f, 1.0f + e);
  const float q = e * r;
  f = z < 0.0f ? q : r;
  rest = z < 0.0f ? r : q;
}
template <class T> __device__ __forceinline__ void rec_gate(double z, double &f, double &rest) {
  const double e = exp(-fabs(z));
  const double r = 1.0 / (1.0 + e);
  const double q = e * r;
  f = z < 0.0 ? q : r;
  rest = z < 0.0 ? r : q;
}

// s -> A s + H.  A state of exactly zero stays out of the product: A may
// have overflowed (decays above 1), and the steps themselves give 0 there.
template <class S> __device__ __forceinline__ S rec_apply(S A, S H, S s) { return s == S(0) ? H : fma(A, s, H); }

template <class T, int VEC> struct alignas(sizeof(T) * VEC) RecVec { T v[VEC]; };

template <int BYTES> __device__ __forceinline__ void rec_cp_async(void *dst, const void *src) {
  const unsigned d = (unsigned)__cvta_generic_to_shared(dst);
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void rec_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `n` of this thread's newest groups are still on the way.
__device__ __forceinline__ void rec_wait(int n) {
  if (n >= 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

struct RecArgs {
  RecView in[4];   // forward: a, x; backward: a, grad, h, x
  RecView out[2];  // forward: h; backward: grad_a, grad_x
  const void *h0;
  const void *seed;  // the state before the first span: h0 / grad_state
  void *last;        // the state after the last span: state / grad_h0
  long long groups, steps, per;  // per: groups along inner
  int iters, stages;
};

constexpr int kRecWarps = 8;

// Steps of one warp's span: 16 forward, 8 backward (its ring holds more
// arrays).
template <bool GRAD> struct RecSpan { static constexpr int value = GRAD ? 8 : 16; };

template <class T, int VEC, bool GRAD, bool GATED, bool CLUSTER>
__global__ void __launch_bounds__(32 * kRecWarps, 2) rec_kernel(const __grid_constant__ RecArgs g) {
  typedef typename RecState<T>::type S;
  typedef RecVec<T, VEC> V;
  constexpr int N = RecSpan<GRAD>::value;
  constexpr int NA = GRAD ? (GATED ? 4 : 3) : 2;
  constexpr bool ASYNC = sizeof(V) >= 4;  // cp.async copies 4, 8 or 16 bytes
  extern __shared__ __align__(16) unsigned char s_ring[];
  __shared__ S s_a[2][kRecWarps][32 * VEC], s_h[2][kRecWarps][32 * VEC];
  __shared__ S s_ca[CLUSTER ? 2 : 1][CLUSTER ? 8 : 1][32 * VEC], s_ch[CLUSTER ? 2 : 1][CLUSTER ? 8 : 1][32 * VEC];
  const int lane = threadIdx.x, w = threadIdx.y, warps = blockDim.y;
  const int threads = 32 * warps, tid = w * 32 + lane;
  int rank = 0, ranks = 1;
  long long blk = blockIdx.x;
  if (CLUSTER) {
    rank = (int)cg::this_cluster().block_rank();
    ranks = (int)cg::this_cluster().num_blocks();
    blk = blockIdx.x / ranks;
    // every block of the cluster has to run before its shared memory is written
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  }
  const long long grp = blk * 32 + lane;
  const bool active = grp < g.groups;
  const long long o = active ? grp / g.per : 0;
  const long long i = active ? (grp - o * g.per) * VEC : 0;
  const T *in[NA];
#pragma unroll
  for (int q = 0; q < NA; ++q) in[q] = (const T *)g.in[q].p + o * g.in[q].so + i;
  T *out[2];
#pragma unroll
  for (int q = 0; q < (GRAD ? 2 : 1); ++q) out[q] = (T *)const_cast<void *>(g.out[q].p) + o * g.out[q].so + i;
  V *ring = reinterpret_cast<V *>(s_ring);
  const long long span = (long long)ranks * warps * N;  // steps of the cluster
  const long long mine = ((long long)rank * warps + w) * N;
  S carry[VEC];  // the state before the cluster's present span
#pragma unroll
  for (int v = 0; v < VEC; ++v) carry[v] = active && g.seed ? ((const S *)g.seed)[grp * VEC + v] : S(0);

  // step k in the order of work lies at t = k forward, steps - 1 - k backward;
  // h is read one step before, so at t = 0 (where h0 stands in) not at all
  V pre[ASYNC ? 1 : NA][ASYNC ? 1 : N];
  auto issue = [&](int it) {
    const long long k0 = it * span + mine;
    const long long left = active ? g.steps - k0 : 0;
    if (left <= 0) return;
    V *slot = ring + (size_t)(ASYNC ? it % g.stages : 0) * NA * N * threads + tid;
#pragma unroll
    for (int q = 0; q < NA; ++q) {
      const long long st = GRAD ? -g.in[q].st : g.in[q].st;
      const T *p = in[q] + (GRAD ? g.steps - 1 - k0 : k0) * g.in[q].st;
      const long long n = GRAD && q == 2 ? left - 1 : left;
      if (GRAD && q == 2) p += st;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (j < n) {
          if constexpr (ASYNC) rec_cp_async<(int)sizeof(V)>(slot + (q * N + j) * threads, p);
          else pre[q][j] = *reinterpret_cast<const V *>(p);
        }
        p += st;
      }
    }
  };
  auto commit = [&]() {
    if constexpr (ASYNC) rec_commit();
  };
  const int ahead = ASYNC ? g.stages - 1 : 0;
  if constexpr (ASYNC) {
    for (int it = 0; it < ahead; ++it) {
      issue(it);
      commit();
    }
  } else {
    issue(0);
  }
  if (CLUSTER) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");

  for (int it = 0; it < g.iters; ++it) {
    if constexpr (ASYNC) {
      if (it + ahead < g.iters) issue(it + ahead);
      commit();
      rec_wait(ahead);
    } else {
#pragma unroll
      for (int q = 0; q < NA; ++q)
#pragma unroll
        for (int j = 0; j < N; ++j) ring[(q * N + j) * threads + tid] = pre[q][j];
      if (it + 1 < g.iters) issue(it + 1);
    }
    const long long k0 = it * span + mine;
    const long long left = active ? g.steps - k0 : 0;
    const V *slot = ring + (size_t)(ASYNC ? it % g.stages : 0) * NA * N * threads + tid;
    auto raw = [&](int q, int j, int v) -> S { return Cvt<S, T>::f(slot[(q * N + j) * threads].v[v]); };

    // the span's composition, from a state of zero.  Gates are evaluated once
    // and kept: f and u forward, f and 1 - f backward.
    S F[GATED ? N : 1][VEC], U[GATED ? N : 1][VEC], A[VEC], H[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A[v] = S(1);
      H[v] = S(0);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j < left) {
        const V va = slot[j * threads], vb = slot[(N + j) * threads];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          S f = Cvt<S, T>::f(va.v[v]), u = Cvt<S, T>::f(vb.v[v]);
          if constexpr (GATED) {
            S rest;
            rec_gate<T>(f, f, rest);
            F[j][v] = f;
            U[j][v] = GRAD ? rest : rest * u;
            if (!GRAD) u = U[j][v];
          }
          H[v] = GRAD ? f * (u + H[v]) : fma(f, H[v], u);
          A[v] *= f;
        }
      }
    }

    // join the block's warps, then the cluster's blocks
    const int par = it & 1;
    S s[VEC];
    if (warps > 1 || CLUSTER) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        s_a[par][w][lane * VEC + v] = A[v];
        s_h[par][w][lane * VEC + v] = H[v];
      }
      __syncthreads();
      if (CLUSTER) {
        // this block's composition to every block of the cluster, one warp a block
        for (int r = w; r < ranks; r += warps) {
          S *pa = cg::this_cluster().map_shared_rank(&s_ca[par][rank][0], r);
          S *ph = cg::this_cluster().map_shared_rank(&s_ch[par][rank][0], r);
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            S a = S(1), h = S(0);
            for (int b = 0; b < warps; ++b) {
              const S ab = s_a[par][b][lane * VEC + v];
              h = rec_apply(ab, s_h[par][b][lane * VEC + v], h);
              a *= ab;
            }
            pa[lane * VEC + v] = a;
            ph[lane * VEC + v] = h;
          }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        S c = carry[v];
        if (CLUSTER) {
          S start = c;
          for (int r = 0; r < ranks; ++r) {
            if (r == rank) start = c;
            c = rec_apply(s_ca[par][r][lane * VEC + v], s_ch[par][r][lane * VEC + v], c);
          }
          carry[v] = c;
          c = start;
        }
        s[v] = c;
        for (int b = 0; b < warps; ++b) {
          if (b == w) s[v] = c;
          if (b >= w && CLUSTER) break;
          c = rec_apply(s_a[par][b][lane * VEC + v], s_h[par][b][lane * VEC + v], c);
        }
        if (!CLUSTER) carry[v] = c;
      }
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        s[v] = carry[v];
        carry[v] = rec_apply(A[v], H[v], carry[v]);
      }
    }

    // the span's steps again, from the state before it
    T *po[2];
#pragma unroll
    for (int q = 0; q < (GRAD ? 2 : 1); ++q) po[q] = out[q] + (GRAD ? g.steps - 1 - k0 : k0) * g.out[q].st;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (j < left) {
        V r0, r1;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const S f = GATED ? F[GATED ? j : 0][v] : raw(0, j, v);
          if (!GRAD) {
            s[v] = fma(f, s[v], GATED ? U[GATED ? j : 0][v] : raw(1, j, v));
            r0.v[v] = Cvt<T, S>::f(s[v]);
          } else {
            const S gt = raw(1, j, v) + s[v];
            S hp = S(0);
            if (j + 1 < left) hp = raw(2, j, v);
            else if (g.h0) hp = ((const S *)g.h0)[grp * VEC + v];
            if constexpr (GATED) {
              const S rest = U[j][v];
              r0.v[v] = Cvt<T, S>::f(gt * (hp - raw(3, j, v)) * (f * rest));
              r1.v[v] = Cvt<T, S>::f(gt * rest);
            } else {
              r0.v[v] = Cvt<T, S>::f(gt * hp);
              r1.v[v] = Cvt<T, S>::f(gt);
            }
            s[v] = f * gt;
          }
        }
        *reinterpret_cast<V *>(po[0]) = r0;
        if (GRAD) *reinterpret_cast<V *>(po[1]) = r1;
        if (k0 + j + 1 == g.steps && g.last) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) ((S *)g.last)[grp * VEC + v] = s[v];
        }
      }
      po[0] += GRAD ? -g.out[0].st : g.out[0].st;
      if (GRAD) po[1] -= g.out[1].st;
    }
  }
  if (g.steps == 0 && g.last && active && w == 0) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) ((S *)g.last)[grp * VEC + v] = carry[v];
  }
}

}  // namespace mmpd

namespace {

using mmpd::RecArgs;
using mmpd::RecView;

// Sizes that a launch and the kernels' 64-bit offsets can address.
int rec_sizes(const char *what, int dtype, int64_t outer, int64_t steps, int64_t inner) {
  if (outer < 0 || steps < 0 || inner < 0) return mmp::set_error(MMP_E_ARG, std::string(what) + ": negative size");
  if (dtype != MMP_FLOAT16 && dtype != MMP_FLOAT32 && dtype != MMP_FLOAT64)
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": needs a floating dtype");
  if (inner && outer > (INT64_C(1) << 32) / inner)
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": more than 2^32 chains");
  if (steps > INT32_MAX) return mmp::set_error(MMP_E_ARG, std::string(what) + ": more than 2^31 - 1 steps");
  return MMP_OK;
}

template <class T, int VEC, bool GRAD, bool GATED, bool CLUSTER>
int rec_launch(const RecArgs &g, unsigned blocks, int warps, int ranks, size_t smem) {
  auto fn = mmpd::rec_kernel<T, VEC, GRAD, GATED, CLUSTER>;
  if (smem > 32 * 1024)  // together with the static part this can pass the default 48 KB
    MMP_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks * ranks);
  cfg.blockDim = dim3(32, warps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = mmp::stream();
  cudaLaunchAttribute at[1];
  if (CLUSTER) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)ranks;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  MMP_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, g));
  return MMP_OK;
}

template <class T, int VEC, bool GRAD, bool GATED>
int rec_run(RecArgs g, long long chains, long long inner) {
  constexpr int N = mmpd::RecSpan<GRAD>::value;
  constexpr int NA = GRAD ? (GATED ? 4 : 3) : 2;
  g.groups = chains / VEC;
  g.per = inner / VEC;
  const long long blocks = (g.groups + 31) / 32;
  // as many warps a block and blocks a cluster as there are spans for, until
  // two blocks an SM are there
  const long long spans = (g.steps + N - 1) / N;
  int warps = 1, ranks = 1;
  while (warps < mmpd::kRecWarps && warps < spans) warps *= 2;
  while (ranks < 8 && blocks * ranks < 2 * mmp::sm_count() && (long long)ranks * warps < spans) ranks *= 2;
  if (blocks * ranks > INT32_MAX) return mmp::set_error(MMP_E_ARG, "recurrence: too many chains");
  g.iters = (int)((spans + (long long)warps * ranks - 1) / ((long long)warps * ranks));
  constexpr bool async = sizeof(T) * VEC >= 4;
  g.stages = async ? (g.iters < 3 ? (g.iters > 0 ? g.iters : 1) : 3) : 1;
  const size_t smem = (size_t)g.stages * NA * N * warps * 32 * sizeof(T) * VEC;
  return ranks > 1 ? rec_launch<T, VEC, GRAD, GATED, true>(g, (unsigned)blocks, warps, ranks, smem)
                   : rec_launch<T, VEC, GRAD, GATED, false>(g, (unsigned)blocks, warps, ranks, smem);
}

// Whether every operand can be moved in pieces of `bytes` (e: element size).
bool rec_aligned(const RecArgs &g, int nin, int nout, long long inner, size_t bytes, size_t e) {
  const long long vec = (long long)(bytes / e);
  if (inner % vec) return false;
  auto ok = [&](const RecView &v) { return (uintptr_t)v.p % bytes == 0 && v.so % vec == 0 && v.st % vec == 0; };
  for (int i = 0; i < nin; ++i)
    if (!ok(g.in[i])) return false;
  for (int i = 0; i < nout; ++i)
    if (!ok(g.out[i])) return false;
  return true;
}

template <bool GRAD, bool GATED>
int rec_dispatch(int dtype, const RecArgs &g, long long chains, long long inner) {
  constexpr int nin = GRAD ? (GATED ? 4 : 3) : 2, nout = GRAD ? 2 : 1;
  if (dtype == MMP_FLOAT16) {
    if (rec_aligned(g, nin, nout, inner, 4, 2)) return rec_run<__half, 2, GRAD, GATED>(g, chains, inner);
    return rec_run<__half, 1, GRAD, GATED>(g, chains, inner);
  }
  if (dtype == MMP_FLOAT32) return rec_run<float, 1, GRAD, GATED>(g, chains, inner);
  return rec_run<double, 1, GRAD, GATED>(g, chains, inner);
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
  RecArgs g = {};
  g.in[0] = RecView{a, a_so, a_st};
  g.in[1] = RecView{x, x_so, x_st};
  g.out[0] = RecView{h, h_so, h_st};
  g.h0 = g.seed = h0;
  g.last = state;
  g.steps = steps;
  return gated ? rec_dispatch<false, true>(dtype, g, chains, inner) : rec_dispatch<false, false>(dtype, g, chains, inner);
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
  RecArgs r = {};
  r.in[0] = RecView{a, a_so, a_st};
  r.in[1] = RecView{grad, g_so, g_st};
  r.in[2] = RecView{h, h_so, h_st};
  r.in[3] = RecView{x, x_so, x_st};
  r.out[0] = RecView{grad_a, ga_so, ga_st};
  r.out[1] = RecView{grad_x, gx_so, gx_st};
  r.h0 = h0;
  r.seed = grad_state;
  r.last = grad_h0;
  r.steps = steps;
  return gated ? rec_dispatch<true, true>(dtype, r, chains, inner) : rec_dispatch<true, false>(dtype, r, chains, inner);
}

}  // extern "C"
