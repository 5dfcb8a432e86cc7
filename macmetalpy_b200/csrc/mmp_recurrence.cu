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
// gates take ex2.approx and rcp.approx (relative errors 2^-22.5 + |z| 2^-24 and
// 2^-23, far below the gates' own rounding of 2^-11): the kernel issues some
// 20 instructions an element, and expf and the division would add as many.
__device__ __forceinline__ float rec_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rec_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <class T> __device__ __forceinline__ void rec_gate(float z, float &f, float &rest) {
  constexpr bool half = sizeof(T) == 2;
  const float e = half ? rec_ex2(fabsf(z) * -1.4426950408889634f) : expf(-fabsf(z));
  const float r = rec_rcp(1.0f + e);
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

template <int BYTES> __device__ __forceinline__ void rec_cp_async(unsigned dst, const void *src) {
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void rec_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most `n` of this thread's newest groups are still on the way.
__device__ __forceinline__ void rec_wait(int n) {
  if (n >= 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The cluster's exchange: st.async writes into the other blocks' shared memory
// and counts its bytes on a barrier there.  A fence in its place (the release
// of barrier.cluster) waits for this block's own loads and stores on the way,
// the ring's loads ahead among them: 314 us against 302 for 1 x 65521 x 1000
// float32.
__device__ __forceinline__ unsigned rec_map(const void *p, int rank) {
  unsigned r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void rec_send(unsigned dst, unsigned bar, float a, float h) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(dst),
               "f"(a), "f"(h), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void rec_send(unsigned dst, unsigned bar, double a, double h) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f64 [%0], {%1, %2}, [%3];" ::"r"(dst),
               "d"(a), "d"(h), "r"(bar)
               : "memory");
}
// Waits for the barrier's phase; false if it has not come after a second or so.
__device__ __forceinline__ bool rec_arrived(unsigned bar, unsigned phase) {
  for (unsigned n = 0; n < (1u << 23); ++n) {
    unsigned ok;
    asm volatile(
        "{\n.reg .pred p;\nmbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
        "selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(phase)
        : "memory");
    if (ok) return true;
    if (n > 256) __nanosleep(64);
  }
  return false;
}

struct RecArgs {
  RecView in[4];   // forward: a, x; backward: a, grad, h, x
  RecView out[2];  // forward: h; backward: grad_a, grad_x
  const void *h0;
  const void *seed;  // the state before the first span: h0 / grad_state
  void *last;        // the state after the last span: state / grad_h0
  long long groups, per;  // per: groups along inner
  int steps, iters, stages;
  int near;  // every step stride is below 2^31 bytes
  int *err;
};

constexpr int kRecWarps = 8;

// Steps of one warp's span, by the bytes that a lane moves a step: 32 KB of
// ring a stage and block of 8 warps, so that two blocks of three stages fit an
// SM.
template <int BYTES, bool GRAD> struct RecSpan { static constexpr int value = (GRAD ? 8 : 16) / (BYTES == 8 ? 2 : 1); };

template <class S> struct alignas(2 * sizeof(S)) RecMap {
  S a, h;
};

// How a span's rows reach the ring.  kWide: the warp copies them in 16-byte
// pieces, several rows an instruction, past L1 (the others take 4 or 8 bytes a
// lane, whose lines on the way are held in what the ring leaves of L1).
enum { kPlain, kLane, kWide };

template <class T, int VEC, int COPY, bool GRAD, bool GATED, bool CLUSTER>
__global__ void __launch_bounds__(32 * kRecWarps, 2) rec_kernel(const __grid_constant__ RecArgs g) {
  typedef typename RecState<T>::type S;
  typedef RecVec<T, VEC> V;
  constexpr int N = RecSpan<(int)sizeof(V), GRAD>::value;
  constexpr int NA = GRAD ? (GATED ? 4 : 3) : 2;
  constexpr int NO = GRAD ? 2 : 1;
  constexpr int NC = 32 * VEC;            // chains of the block
  constexpr bool ASYNC = COPY != kPlain;
  constexpr int PIECE = 16 / (int)sizeof(T);             // elements
  constexpr int PER = NC / PIECE, ROWS = 32 / PER;        // pieces a row, rows an instruction
  extern __shared__ __align__(16) unsigned char s_ring[];
  __shared__ RecMap<S> s_map[kRecWarps][NC];                         // the warps' spans
  __shared__ RecMap<S> s_blk[CLUSTER ? 2 : 1][CLUSTER ? 8 : 1][NC];  // the cluster's blocks' spans
  __shared__ S s_start[kRecWarps][NC], s_carry[NC];
  __shared__ __align__(8) unsigned long long s_bar[2];
  const int lane = threadIdx.x, w = threadIdx.y, warps = blockDim.y;
  int rank = 0, ranks = 1;
  long long blk = blockIdx.x;
  if (CLUSTER) {
    rank = (int)cg::this_cluster().block_rank();
    ranks = (int)cg::this_cluster().num_blocks();
    blk = blockIdx.x / ranks;
    // every block of the cluster has to run, its barriers set up, before it is sent anything
    if (w == 0 && lane < 2)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((unsigned)__cvta_generic_to_shared(&s_bar[lane]))
                   : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  const long long grp = blk * 32 + lane;
  const bool active = grp < g.groups;
  const long long o = active ? grp / g.per : 0;
  const long long i = active ? (grp - o * g.per) * VEC : 0;
  // where this lane copies from: its own chains, or its piece of the warp's
  const long long cg0 = COPY == kWide ? blk * 32 * VEC + lane % PER * PIECE : 0;  // first chain of the piece
  const bool copies = COPY == kWide ? cg0 < g.groups * VEC : active;
  const T *in[NA];
  if (COPY == kWide) {
    const long long co = copies ? cg0 / (g.per * VEC) : 0, ci = copies ? cg0 - co * (g.per * VEC) : 0;
#pragma unroll
    for (int q = 0; q < NA; ++q) in[q] = (const T *)g.in[q].p + co * g.in[q].so + ci;
  } else {
#pragma unroll
    for (int q = 0; q < NA; ++q) in[q] = (const T *)g.in[q].p + o * g.in[q].so + i;
  }
  T *out[NO];
#pragma unroll
  for (int q = 0; q < NO; ++q) out[q] = (T *)const_cast<void *>(g.out[q].p) + o * g.out[q].so + i;
  // this thread's slots: [stage][array][step], a row of 32 lanes each
  V *const ring = reinterpret_cast<V *>(s_ring) + (size_t)w * g.stages * (NA * N * 32) + lane;
  const int span = ranks * warps * N;  // steps of the cluster
  const int mine = (rank * warps + w) * N;
  S carry[VEC];  // the state before the present span of a block of one warp
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    carry[v] = active && g.seed ? ((const S *)g.seed)[grp * VEC + v] : S(0);
    if (w == 0) s_carry[lane * VEC + v] = carry[v];
  }

  // step k in the order of work lies at t = k forward, steps - 1 - k backward;
  // h is read one step before, so at t = 0 (where h0 stands in) not at all
  V pre[ASYNC ? 1 : NA][ASYNC ? 1 : N];
  auto issue = [&](int it) {
    const int k0 = it * span + mine;
    const int left = copies ? g.steps - k0 : 0;
    if (left <= 0) return;
    const unsigned slot = (unsigned)__cvta_generic_to_shared(ring + (ASYNC ? it % g.stages : 0) * (NA * N * 32));
    const long long t0 = GRAD ? g.steps - 1 - k0 : k0;
    if constexpr (COPY == kWide) {
      const int row = lane / PER;
      const unsigned dst = slot - lane * (int)sizeof(V) + row * (NC * (int)sizeof(T)) + lane % PER * 16;
#pragma unroll
      for (int q = 0; q < NA; ++q) {
        const long long st = (GRAD ? -g.in[q].st : g.in[q].st) * ROWS;
        const T *p = in[q] + ((GRAD && q == 2 ? t0 - 1 : t0) + (GRAD ? -row : row)) * g.in[q].st;
        const int n = (GRAD && q == 2 ? left - 1 : left) - row;
#pragma unroll
        for (int j = 0; j < N; j += ROWS) {
          if (j < n) rec_cp_async<16>(dst + (q * N + j) * (NC * (int)sizeof(T)), p);
          p += st;
        }
      }
      return;
    }
    if (left > N && g.near) {  // a whole span with one address instruction a step
#pragma unroll
      for (int q = 0; q < NA; ++q) {
        const int st = (int)(GRAD ? -g.in[q].st : g.in[q].st) * (int)sizeof(T);
        const char *p = (const char *)(in[q] + (GRAD && q == 2 ? t0 - 1 : t0) * g.in[q].st);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const char *pj = p + (long long)st * j;
          if constexpr (ASYNC) rec_cp_async<(int)sizeof(V)>(slot + (q * N + j) * 32 * (int)sizeof(V), pj);
          else pre[q][j] = *reinterpret_cast<const V *>(pj);
        }
      }
      return;
    }
#pragma unroll
    for (int q = 0; q < NA; ++q) {
      const long long st = GRAD ? -g.in[q].st : g.in[q].st;
      const T *p = in[q] + (GRAD && q == 2 ? t0 - 1 : t0) * g.in[q].st;
      const int n = GRAD && q == 2 ? left - 1 : left;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (j < n) {
          if constexpr (ASYNC) rec_cp_async<(int)sizeof(V)>(slot + (q * N + j) * 32 * (int)sizeof(V), p);
          else pre[q][j] = *reinterpret_cast<const V *>(p);
        }
        p += st;
      }
    }
  };
  const int ahead = ASYNC ? g.stages - 1 : 0;
  if constexpr (ASYNC) {
    for (int it = 0; it < ahead; ++it) {
      issue(it);
      rec_commit();
    }
  } else {
    issue(0);
  }
  if (CLUSTER) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  bool heard = true;

  for (int it = 0; it < g.iters; ++it) {
    if constexpr (ASYNC) {
      if (COPY == kWide) __syncwarp();  // every lane is done with the stage that is filled next
      if (it + ahead < g.iters) issue(it + ahead);
      rec_commit();
      rec_wait(ahead);
      if (COPY == kWide) __syncwarp();  // the other lanes' pieces too
    } else {
#pragma unroll
      for (int q = 0; q < NA; ++q)
#pragma unroll
        for (int j = 0; j < N; ++j) ring[(q * N + j) * 32] = pre[q][j];
      if (it + 1 < g.iters) issue(it + 1);
    }
    const int k0 = it * span + mine;
    const int left = active ? g.steps - k0 : 0;
    const V *const slot = ring + (ASYNC ? it % g.stages : 0) * (NA * N * 32);

    // the span's composition, from a state of zero.  Gates are evaluated once
    // and kept: f and u forward, f and 1 - f backward.
    S F[GATED ? N : 1][VEC], U[GATED ? N : 1][VEC], A[VEC], H[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A[v] = S(1);
      H[v] = S(0);
    }
    auto compose = [&](int j) {
      const V va = slot[j * 32], vb = slot[(N + j) * 32];
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
    };
    if (left >= N) {
#pragma unroll
      for (int j = 0; j < N; ++j) compose(j);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < left) compose(j);
    }

    // join the block's warps, then the cluster's blocks: one thread a chain
    S s[VEC];
    if (warps > 1 || CLUSTER) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) s_map[w][lane * VEC + v] = RecMap<S>{A[v], H[v]};
      __syncthreads();
      const int tid = w * 32 + lane, par = it & 1;
      if (CLUSTER) {
        const unsigned bar = (unsigned)__cvta_generic_to_shared(&s_bar[par]);
        if (tid == 0)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
                       "r"(ranks * NC * (int)sizeof(RecMap<S>))
                       : "memory");
        for (int c = tid; c < NC; c += 32 * warps) {
          RecMap<S> m = s_map[0][c];
          for (int b = 1; b < warps; ++b) {
            const RecMap<S> n = s_map[b][c];
            m.h = rec_apply(n.a, n.h, m.h);
            m.a *= n.a;
          }
          for (int r = 0; r < ranks; ++r) rec_send(rec_map(&s_blk[par][rank][c], r), rec_map(&s_bar[par], r), m.a, m.h);
        }
        if (tid < NC && heard) {
          heard = rec_arrived(bar, (it >> 1) & 1);
          if (!heard) atomicExch(g.err, 9);
        }
      }
      for (int c = tid; c < NC; c += 32 * warps) {
        S st = s_carry[c];
        if (CLUSTER) {
          S at = st;
          for (int r = 0; r < ranks; ++r) {
            if (r == rank) at = st;
            st = rec_apply(s_blk[par][r][c].a, s_blk[par][r][c].h, st);
          }
          s_carry[c] = st;
          st = at;
        }
        for (int b = 0; b < warps; ++b) {
          s_start[b][c] = st;
          st = rec_apply(s_map[b][c].a, s_map[b][c].h, st);
        }
        if (!CLUSTER) s_carry[c] = st;
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < VEC; ++v) s[v] = s_start[w][lane * VEC + v];
    } else {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        s[v] = carry[v];
        carry[v] = rec_apply(A[v], H[v], carry[v]);
      }
    }

    // the span's steps again, from the state before it
    auto replay = [&](int j, bool first, V &r0, V &r1) {
      V va, vb, vh, vx;
      if (GRAD || !GATED) vb = slot[(N + j) * 32];
      if (!GATED) va = slot[j * 32];
      if (GRAD && !first) vh = slot[(2 * N + j) * 32];
      if (GRAD && GATED) vx = slot[((NA - 1) * N + j) * 32];
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        const S f = GATED ? F[GATED ? j : 0][v] : Cvt<S, T>::f(va.v[v]);
        if (!GRAD) {
          s[v] = fma(f, s[v], GATED ? U[GATED ? j : 0][v] : Cvt<S, T>::f(vb.v[v]));
          r0.v[v] = Cvt<T, S>::f(s[v]);
        } else {
          const S gt = Cvt<S, T>::f(vb.v[v]) + s[v];
          const S hp = !first ? Cvt<S, T>::f(vh.v[v]) : g.h0 ? ((const S *)g.h0)[grp * VEC + v] : S(0);
          if constexpr (GATED) {
            const S rest = U[j][v];
            r0.v[v] = Cvt<T, S>::f(gt * (hp - Cvt<S, T>::f(vx.v[v])) * (f * rest));
            r1.v[v] = Cvt<T, S>::f(gt * rest);
          } else {
            r0.v[v] = Cvt<T, S>::f(gt * hp);
            r1.v[v] = Cvt<T, S>::f(gt);
          }
          s[v] = f * gt;
        }
      }
    };
    const long long t0 = GRAD ? g.steps - 1 - k0 : k0;
    if (left > N && g.near) {  // whole, and not the last span
#pragma unroll
      for (int j = 0; j < N; ++j) {
        V r[2];
        replay(j, false, r[0], r[1]);
#pragma unroll
        for (int q = 0; q < NO; ++q) {
          const int st = (int)(GRAD ? -g.out[q].st : g.out[q].st) * (int)sizeof(T);
          *reinterpret_cast<V *>((char *)(out[q] + t0 * g.out[q].st) + (long long)st * j) = r[q];
        }
      }
    } else if (left > 0) {
      T *po[NO];
#pragma unroll
      for (int q = 0; q < NO; ++q) po[q] = out[q] + t0 * g.out[q].st;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (j < left) {
          V r[2];
          replay(j, GRAD && j + 1 == left, r[0], r[1]);
#pragma unroll
          for (int q = 0; q < NO; ++q) {
            *reinterpret_cast<V *>(po[q]) = r[q];
            po[q] += GRAD ? -g.out[q].st : g.out[q].st;
          }
        }
      }
      if (left <= N && g.last) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) ((S *)g.last)[grp * VEC + v] = s[v];
      }
    }
  }
  if (CLUSTER) {  // no block ends while it may still be sent to
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
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
  if (steps > INT64_C(1) << 30) return mmp::set_error(MMP_E_ARG, std::string(what) + ": more than 2^30 steps");
  return MMP_OK;
}

template <class T, int VEC, int COPY, bool GRAD, bool GATED, bool CLUSTER>
int rec_launch(const RecArgs &g, unsigned blocks, int warps, int ranks, size_t smem) {
  auto fn = mmpd::rec_kernel<T, VEC, COPY, GRAD, GATED, CLUSTER>;
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

template <class T, int VEC, int COPY, bool GRAD, bool GATED>
int rec_run(RecArgs g, long long chains, long long inner) {
  constexpr int N = mmpd::RecSpan<(int)sizeof(T) * VEC, GRAD>::value;
  constexpr int NA = GRAD ? (GATED ? 4 : 3) : 2;
  g.groups = chains / VEC;
  g.per = inner / VEC;
  g.err = mmp::device_error_word();
  g.near = 1;
  for (const RecView &v : g.in) g.near &= v.st * (long long)sizeof(T) == (int)(v.st * (long long)sizeof(T));
  for (const RecView &v : g.out) g.near &= v.st * (long long)sizeof(T) == (int)(v.st * (long long)sizeof(T));
  const long long blocks = (g.groups + 31) / 32;
  // as many warps a block and blocks a cluster as there are spans for, while
  // all blocks fit at two an SM: 8 x 2048 x 2048 float16 (256 blocks) takes 46
  // us in blocks alone and 59 in clusters of two, which run in two waves;
  // 1 x 65521 x 1000 float32 (32 blocks) 606 alone and 186 in clusters of eight
  const long long spans = ((long long)g.steps + N - 1) / N;
  int warps = 1, ranks = 1;
  while (warps < mmpd::kRecWarps && warps < spans) warps *= 2;
  while (ranks < 8 && blocks * ranks * 2 <= 2 * mmp::sm_count() && (long long)ranks * warps < spans) ranks *= 2;
  if (blocks * ranks > INT32_MAX) return mmp::set_error(MMP_E_ARG, "recurrence: too many chains");
  g.iters = (int)((spans + (long long)warps * ranks - 1) / ((long long)warps * ranks));
  g.stages = COPY != mmpd::kPlain ? (g.iters < 3 ? (g.iters > 0 ? g.iters : 1) : 3) : 1;
  const size_t smem = (size_t)g.stages * NA * N * warps * 32 * sizeof(T) * VEC;
  return ranks > 1 ? rec_launch<T, VEC, COPY, GRAD, GATED, true>(g, (unsigned)blocks, warps, ranks, smem)
                   : rec_launch<T, VEC, COPY, GRAD, GATED, false>(g, (unsigned)blocks, warps, ranks, smem);
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
  using namespace mmpd;
  const size_t e = mmp_dtype_size(dtype);
  const bool wide = rec_aligned(g, nin, nout, inner, 16, e);
  if (dtype == MMP_FLOAT16) {
    if (wide) return rec_run<__half, 2, kWide, GRAD, GATED>(g, chains, inner);
    if (rec_aligned(g, nin, nout, inner, 4, e)) return rec_run<__half, 2, kLane, GRAD, GATED>(g, chains, inner);
    return rec_run<__half, 1, kPlain, GRAD, GATED>(g, chains, inner);
  }
  if (dtype == MMP_FLOAT32)
    return wide ? rec_run<float, 1, kWide, GRAD, GATED>(g, chains, inner)
                : rec_run<float, 1, kLane, GRAD, GATED>(g, chains, inner);
  return rec_run<double, 1, kLane, GRAD, GATED>(g, chains, inner);
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
  g.steps = (int)steps;
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
  r.steps = (int)steps;
  return gated ? rec_dispatch<true, true>(dtype, r, chains, inner) : rec_dispatch<true, false>(dtype, r, chains, inner);
}

}  // extern "C"
