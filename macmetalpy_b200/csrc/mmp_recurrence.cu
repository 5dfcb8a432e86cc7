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
// A span's steps run twice, once to compose it and once, from the state then
// known, for the outputs.  One more warp of the block joins the spans; where
// the gates do not stay in registers in between (HOLD), the others compose
// the next span before they replay the last and do not wait for it.
// Every input is read once and every output written once; no block waits for
// one outside its cluster, nothing is allocated, and the order of all
// operations is fixed by the sizes and the way rows are copied.  What bounds
// it is HBM traffic, so the loads run ahead: each warp copies the rows of its
// next spans into a ring in shared memory that only it reads.
// Whole calls: 1 x 65521 x 1000 float32 121 to 131 us (6.0 to 6.5 TB/s); 8 x
// 2048 x 2048 float16 gated 44 us (4.6 TB/s; latency, and 256 blocks on 148
// SMs), its gradient 75 to 80 (5.0 to 5.4); 2 x 16383 x 1536 float32 gradient
// 172 to 180 (5.6 to 5.9).
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "mmp_chain.cuh"
#include "mmp_device.cuh"
#include "mmp_internal.h"

namespace mmp {
void *driver_fn(const char *name);
}

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
// the state as it is, one of -inf replaces it.  A NaN goes to both.  Gates in
// 32 bits take rcp.approx in the place of a division (relative error 2^-23
// against 2^-24), those of float16 arrays ex2.approx besides (2^-22.5 + 1.2 |z|
// 2^-24, of which |z| 2^-24 and the constant's part come from the argument; far
// below the gates' own rounding of 2^-11): the kernel issues some 20
// instructions an element, and expf and the division would add as many.
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

// A store that the compiler knows to be global (its pointer comes out of a
// structure), so that it does not hold back the loads from the ring after it.
template <class V> __device__ __forceinline__ void rec_store(void *p, const V &v) {
  if constexpr (sizeof(V) == 2)
    asm volatile("st.global.b16 [%0], %1;" ::"l"(p), "h"(*reinterpret_cast<const unsigned short *>(&v)));
  else if constexpr (sizeof(V) == 4)
    asm volatile("st.global.b32 [%0], %1;" ::"l"(p), "r"(*reinterpret_cast<const unsigned *>(&v)));
  else
    asm volatile("st.global.b64 [%0], %1;" ::"l"(p), "l"(*reinterpret_cast<const unsigned long long *>(&v)));
}

template <int BYTES> __device__ __forceinline__ void rec_cp_async(unsigned dst, const void *src) {
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
// the ring's loads ahead among them (1 x 65521 x 1000 float32 with two stages
// of 4-byte copies: 231 us against 216).
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

// Named barriers of the block: 1 and 2, a span's compositions are there; 3
// and 4, the states before them are.
__device__ __forceinline__ void rec_bar_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
__device__ __forceinline__ void rec_bar_arrive(int id, int threads) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

struct RecArgs {
  RecView in[4];   // forward: a, x; backward: a, grad, h, x
  RecView out[2];  // forward: h; backward: grad_a, grad_x
  const void *h0;
  const void *seed;  // the state before the first span: h0 / grad_state
  void *last;        // the state after the last span: state / grad_h0
  long long outer, inner, tiles;  // tiles: of 32 VEC chains along inner
  int steps, iters, stages, warps;
  int near;  // every step stride is below 2^31 bytes
  int *err;
};

constexpr int kRecWarps = 7;  // and one that joins them: 8 warps of 128 registers, two blocks an SM

// How a span's rows reach the ring.  kTma: one tensor copy an array, by one
// lane of the warp.  kLane: cp.async of each lane's own 4 or 8 bytes (any
// strides; issuing these takes a third of the warps' time, and their lines on
// the way are held in what the ring leaves of L1).  kPlain: loads of 2 bytes,
// for float16 in rows of odd width.
enum { kPlain, kLane, kTma };

// Steps of one warp's span, by the bytes that a lane moves a step: 28 KB of
// ring a stage and block of 7 warps, so that two blocks of three stages fit
// an SM.  kLane has half of that backward, which leaves its lines more of L1 (8
// x 2048 x 2050 float16 gated 105 us, 113 with whole spans; 8 x 2048 x 1025
// float32 plain 78, 81).  Forward it has whole spans (1 x 65521 x 1001 float32
// 252 us, 306 with half ones; 8 x 2048 x 2050 float16 plain 53, 65, gated 61,
// 59).
template <int BYTES, int COPY, bool GRAD> struct RecSpan {
  static constexpr int value = (GRAD ? 8 : 16) / (BYTES == 8 ? 2 : 1) / (COPY == kLane && GRAD ? 2 : 1);
};

template <class S> struct alignas(2 * sizeof(S)) RecMap {
  S a, h;
};

template <int COPY> struct RecMaps {};
struct alignas(64) RecMap3 {
  CUtensorMap m;
  int swap;  // (inner, outer, steps) in place of (inner, steps, outer)
};
template <> struct RecMaps<kTma> {
  RecMap3 in[4];
};

__device__ __forceinline__ void rec_tma(unsigned dst, const RecMap3 &map, unsigned bar, int i, int t, int o) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          dst),
      "l"(&map.m), "r"(bar), "r"(i), "r"(map.swap ? o : t), "r"(map.swap ? t : o)
      : "memory");
}

// HOLD: gates of a span stay in registers from compose to replay, which then
// follow one another; else they are evaluated twice, and a span is composed
// while the one before it is joined.
template <class T, int VEC, int COPY, bool GRAD, bool GATED, bool CLUSTER, bool HOLD>
__global__ void __launch_bounds__(32 * (kRecWarps + 1), 2) rec_kernel(
    const __grid_constant__ RecArgs g, const __grid_constant__ RecMaps<COPY> maps) {
  typedef typename RecState<T>::type S;
  typedef RecVec<T, VEC> V;
  constexpr int N = RecSpan<(int)sizeof(V), COPY, GRAD>::value;
  constexpr int NA = GRAD ? (GATED ? 4 : 3) : 2;
  constexpr int NO = GRAD ? 2 : 1;
  constexpr int NC = 32 * VEC;            // chains of the block
  constexpr bool ASYNC = COPY == kLane;
  constexpr int kStages = 3;
  extern __shared__ __align__(128) unsigned char s_ring[];
  constexpr int LAG = HOLD ? 0 : 1;  // spans between compose and replay
  __shared__ __align__(16) RecMap<S> s_map[2][kRecWarps][NC];                      // the warps' spans
  __shared__ __align__(16) RecMap<S> s_blk[CLUSTER ? 2 : 1][CLUSTER ? 8 : 1][NC];  // the cluster's blocks' spans
  __shared__ __align__(16) S s_start[2][kRecWarps][NC];                            // states before the warps' spans
  __shared__ __align__(8) unsigned long long s_bar[2], s_full[kRecWarps][kStages];
  const int lane = threadIdx.x, w = threadIdx.y, warps = g.warps;
  int rank = 0, ranks = 1;
  long long blk = blockIdx.x;
  if (CLUSTER) {
    rank = (int)cg::this_cluster().block_rank();
    ranks = (int)cg::this_cluster().num_blocks();
    blk = blockIdx.x / ranks;
  }
  // the lane's chains: of a row of tiles for tensor copies, else of all groups in a row
  long long o, i;
  bool active;
  if constexpr (COPY == kTma) {
    o = blk / g.tiles;
    i = (blk - o * g.tiles) * NC + lane * VEC;
    active = i < g.inner;
  } else {
    const long long grp = blk * 32 + lane, per = g.inner / VEC;
    active = grp < g.outer * per;
    o = active ? grp / per : 0;
    i = active ? (grp - o * per) * VEC : 0;
  }
  const long long chain = o * g.inner + i;
  const T *in[NA];
#pragma unroll
  for (int q = 0; q < NA; ++q) in[q] = (const T *)g.in[q].p + o * g.in[q].so + i;
  T *out[NO];
#pragma unroll
  for (int q = 0; q < NO; ++q) out[q] = (T *)const_cast<void *>(g.out[q].p) + o * g.out[q].so + i;
  // this thread's slots: [stage][array][step], a row of 32 lanes each
  // (tensor copies go to multiples of 128 bytes)
  const unsigned skew = (unsigned)(-(int)__cvta_generic_to_shared(s_ring)) & 127u;
  V *const ring = reinterpret_cast<V *>(s_ring + skew) + (size_t)w * g.stages * (NA * N * 32) + lane;
  chain_wait();
  chain_next();
  const int span = ranks * warps * N;  // steps of the cluster
  const int mine = (rank * warps + w) * N;
  S carry[VEC];  // the joining warp's: the state before the cluster's present span
#pragma unroll
  for (int v = 0; v < VEC; ++v)
    carry[v] = w == warps && active && g.seed ? ((const S *)g.seed)[chain + v] : S(0);
  if (CLUSTER) {
    // Every block of the cluster has to run, its barriers set up, before it is
    // sent anything, and to have read the first state, whose place the last
    // one may be written to.
    if (w == 0 && lane < 2)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((unsigned)__cvta_generic_to_shared(&s_bar[lane]))
                   : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  if (w == warps) {
    // The joining warp, beside the warps that compose and replay: a lane has
    // the chains of its group.
    if (CLUSTER) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    bool heard = true;
    for (int it = 0; it < g.iters; ++it) {
      const int par = it & 1;
      rec_bar_sync(1 + par, 32 * (warps + 1));
      RecMap<S> m[kRecWarps][VEC];
#pragma unroll
      for (int b = 0; b < kRecWarps; ++b)
#pragma unroll
        for (int v = 0; v < VEC; ++v) m[b][v] = b < warps ? s_map[par][b][lane * VEC + v] : RecMap<S>{S(1), S(0)};
      S st[VEC];
      if (CLUSTER) {
        // This block's composition to every block of the cluster, and theirs
        // back.  Two places are enough: a block sends for it + 2 once it has
        // everyone's of it + 1, which each sent after reading it's.
        RecMap<S> all[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          all[v] = m[0][v];
#pragma unroll
          for (int b = 1; b < kRecWarps; ++b) {
            all[v].h = rec_apply(m[b][v].a, m[b][v].h, all[v].h);
            all[v].a *= m[b][v].a;
          }
        }
        const unsigned bar = (unsigned)__cvta_generic_to_shared(&s_bar[par]);
        if (lane == 0)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
                       "r"(ranks * NC * (int)sizeof(RecMap<S>))
                       : "memory");
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          if (r < ranks) {
            const unsigned to = rec_map(&s_blk[par][rank][lane * VEC], r), tob = rec_map(&s_bar[par], r);
#pragma unroll
            for (int v = 0; v < VEC; ++v) rec_send(to + v * (int)sizeof(RecMap<S>), tob, all[v].a, all[v].h);
          }
        }
        if (heard) {
          heard = rec_arrived(bar, (it >> 1) & 1);
          if (!heard) atomicExch(g.err, 9);
        }
        RecMap<S> n[8][VEC];
#pragma unroll
        for (int r = 0; r < 8; ++r)
#pragma unroll
          for (int v = 0; v < VEC; ++v)
            n[r][v] = r < ranks ? s_blk[par][CLUSTER ? r : 0][lane * VEC + v] : RecMap<S>{S(1), S(0)};
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (r == rank) st[v] = carry[v];
            carry[v] = rec_apply(n[r][v].a, n[r][v].h, carry[v]);
          }
        }
      } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) st[v] = carry[v];
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
#pragma unroll
        for (int b = 0; b < kRecWarps; ++b) {
          if (b < warps) s_start[par][b][lane * VEC + v] = st[v];
          st[v] = rec_apply(m[b][v].a, m[b][v].h, st[v]);
        }
        if (!CLUSTER) carry[v] = st[v];
      }
      rec_bar_arrive(3 + par, 32 * (warps + 1));
    }
    if (CLUSTER) {
      asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    }
    return;
  }

  // step k in the order of work lies at t = k forward, steps - 1 - k backward;
  // h is read one step before, so at t = 0 (where h0 stands in) not at all
  V pre[ASYNC ? 1 : NA][ASYNC ? 1 : N];
  auto issue = [&](int it, int stage) {
    const int k0 = it * span + mine;
    const int left = active || COPY == kTma ? g.steps - k0 : 0;
    if (left <= 0) return;
    const unsigned slot = (unsigned)__cvta_generic_to_shared(ring + stage * (NA * N * 32));
    if constexpr (COPY == kTma) {  // called by lane 0; rows in order of time, steps outside the axis read as zeros
      const unsigned full = (unsigned)__cvta_generic_to_shared(&s_full[w][stage]);
      const int t0 = GRAD ? g.steps - k0 - N : k0;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full),
                   "r"(NA * N * 32 * (int)sizeof(V))
                   : "memory");
#pragma unroll
      for (int q = 0; q < NA; ++q)
        rec_tma(slot + q * N * 32 * (int)sizeof(V), maps.in[q], full, (int)(i / NC) * NC, GRAD && q == 2 ? t0 - 1 : t0,
                (int)o);
      return;
    }
    const long long t0 = GRAD ? g.steps - 1 - k0 : k0;
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
  // stages that are filled ahead: all but the one in work and, with a lag,
  // the one that is replayed (unless every span has its own)
  const int ahead = COPY == kPlain ? 0 : g.stages - (LAG && g.stages < g.iters ? 2 : 1);
  bool heard = true;
  if constexpr (COPY == kTma) {
    if (lane == 0) {
      for (int q = 0; q < kStages; ++q)
        asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((unsigned)__cvta_generic_to_shared(&s_full[w][q]))
                     : "memory");
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      for (int it = 0; it < ahead; ++it) issue(it, it);
    }
    __syncwarp();
  } else if constexpr (ASYNC) {
    for (int it = 0; it < ahead; ++it) {
      issue(it, it);
      rec_commit();
    }
  } else {
    issue(0, 0);
  }
  if (CLUSTER) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  auto row = [](int j) { return COPY == kTma && GRAD ? N - 1 - j : j; };  // where the ring has a step
  constexpr int M = N < 8 ? N : 8;  // steps whose ring entries are read at once
  S F[HOLD ? N : 1][VEC], U[HOLD ? N : 1][VEC];  // f and u forward, f and 1 - f backward
  S A[VEC], H[VEC], s[VEC];

  // the composition of a span's steps: the state after them, from zero
  auto compose = [&](int it, int stage) {
    const int left = active ? g.steps - (it * span + mine) : 0;
    const V *const slot = ring + stage * (NA * N * 32);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
      A[v] = S(1);
      H[v] = S(0);
    }
    auto step = [&](int j, const V &va, const V &vb) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        S f = Cvt<S, T>::f(va.v[v]), u = Cvt<S, T>::f(vb.v[v]), rest;
        if (GATED) {
          rec_gate<T>(f, f, rest);
          if (!GRAD) u *= rest;
        }
        if constexpr (HOLD) {
          F[j][v] = f;
          U[j][v] = GRAD ? rest : u;
        }
        H[v] = GRAD ? f * (u + H[v]) : fma(f, H[v], u);
        A[v] *= f;
      }
    };
    if (left >= N) {
#pragma unroll
      for (int j0 = 0; j0 < N; j0 += M) {
        V va[M], vb[M];
#pragma unroll
        for (int j = 0; j < M; ++j) {
          va[j] = slot[row(j0 + j) * 32];
          vb[j] = slot[(N + row(j0 + j)) * 32];
        }
#pragma unroll
        for (int j = 0; j < M; ++j) step(j0 + j, va[j], vb[j]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < left) step(j, slot[row(j) * 32], slot[(N + row(j)) * 32]);
    }
  };

  // its steps again, from the state s before them, with the outputs
  auto replay = [&](int it, int stage) {
    const int k0 = it * span + mine;
    const int left = active ? g.steps - k0 : 0;
    const V *const slot = ring + stage * (NA * N * 32);
    struct Row {
      V a, b, h, x;
    };
    auto read = [&](int j, bool first) {
      Row w;
      if (!HOLD) w.a = slot[row(j) * 32];
      if (GRAD || !HOLD) w.b = slot[(N + row(j)) * 32];
      if (GRAD && !first) w.h = slot[(2 * N + row(j)) * 32];
      if (GRAD && GATED) w.x = slot[((NA - 1) * N + row(j)) * 32];
      return w;
    };
    auto step = [&](int j, const Row &w, bool first, V &r0, V &r1) {
      const V &va = w.a, &vb = w.b, &vh = w.h, &vx = w.x;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        S f, rest, u;
        if constexpr (HOLD) {
          f = F[j][v];
          rest = u = U[j][v];
        } else {
          f = Cvt<S, T>::f(va.v[v]);
          if (GATED) rec_gate<T>(f, f, rest);
          if (!GRAD) u = GATED ? rest * Cvt<S, T>::f(vb.v[v]) : Cvt<S, T>::f(vb.v[v]);
        }
        if (!GRAD) {
          s[v] = fma(f, s[v], u);
          r0.v[v] = Cvt<T, S>::f(s[v]);
        } else {
          const S gt = Cvt<S, T>::f(vb.v[v]) + s[v];
          const S hp = !first ? Cvt<S, T>::f(vh.v[v]) : g.h0 ? ((const S *)g.h0)[chain + v] : S(0);
          r0.v[v] = Cvt<T, S>::f(GATED ? gt * (hp - Cvt<S, T>::f(vx.v[v])) * (f * rest) : gt * hp);
          r1.v[v] = Cvt<T, S>::f(GATED ? gt * rest : gt);
          s[v] = f * gt;
        }
      }
    };
    const long long t0 = GRAD ? g.steps - 1 - k0 : k0;
    Row rows[M];
    if (left > N && g.near) {  // whole, and not the last span
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (j % M == 0) {
#pragma unroll
          for (int i = 0; i < M; ++i) rows[i] = read(j + i, false);
        }
        V r[2];
        step(j, rows[j % M], false, r[0], r[1]);
#pragma unroll
        for (int q = 0; q < NO; ++q) {
          const int st = (int)(GRAD ? -g.out[q].st : g.out[q].st) * (int)sizeof(T);
          rec_store((char *)(out[q] + t0 * g.out[q].st) + (long long)st * j, r[q]);
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
          const bool first = GRAD && j + 1 == left;
          step(j, read(j, first), first, r[0], r[1]);
#pragma unroll
          for (int q = 0; q < NO; ++q) {
            rec_store(po[q], r[q]);
            po[q] += GRAD ? -g.out[q].st : g.out[q].st;
          }
        }
      }
      if (left <= N && g.last) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) ((S *)g.last)[chain + v] = s[v];
      }
    }
  };

  // stages in turn: of the span filled next, composed next, replayed next
  int fill = ahead % g.stages, next = 0, last = 0;
  unsigned phase = 0;
  for (int it = 0; it < g.iters + LAG; ++it) {
    if (it < g.iters) {
      if constexpr (COPY == kTma) {
        __syncwarp();  // every lane is done with the stage that is filled next
        if (lane == 0 && it + ahead < g.iters) issue(it + ahead, fill);
        if (heard && it * span + mine < g.steps) {
          heard = rec_arrived((unsigned)__cvta_generic_to_shared(&s_full[w][next]), phase);
          if (!heard) atomicExch(g.err, 9);
        }
      } else if constexpr (ASYNC) {
        if (it + ahead < g.iters) issue(it + ahead, fill);
        rec_commit();
        rec_wait(ahead);
      } else {
        V *const slot = ring + next * (NA * N * 32);
#pragma unroll
        for (int q = 0; q < NA; ++q)
#pragma unroll
          for (int j = 0; j < N; ++j) slot[(q * N + j) * 32] = pre[q][j];
        if (it + 1 < g.iters) issue(it + 1, 0);
      }
      compose(it, next);
      if (++fill == g.stages) fill = 0;
      if (++next == g.stages) {
        next = 0;
        phase ^= 1;
      }
    }
    if (it < g.iters) {
#pragma unroll
      for (int v = 0; v < VEC; ++v) s_map[it & 1][w][lane * VEC + v] = RecMap<S>{A[v], H[v]};
      rec_bar_arrive(1 + (it & 1), 32 * (warps + 1));
    }
    if (it >= LAG) {
      const int par = (it - LAG) & 1;
      rec_bar_sync(3 + par, 32 * (warps + 1));
#pragma unroll
      for (int v = 0; v < VEC; ++v) s[v] = s_start[par][w][lane * VEC + v];
      replay(it - LAG, last);
      if (++last == g.stages) last = 0;
    }
  }
  if (CLUSTER) {  // no block ends while it may still be sent to
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  }
}

// A few steps (a decode step's one, a short segment): a thread has VEC
// neighbouring chains and walks their steps, B of them loaded at once.
template <class T, int VEC, bool GRAD, bool GATED>
__global__ void __launch_bounds__(128) rec_short_kernel(const __grid_constant__ RecArgs g) {
  typedef typename RecState<T>::type S;
  typedef RecVec<T, VEC> V;
  constexpr int SV = VEC * (int)sizeof(S) > 16 ? 16 / (int)sizeof(S) : VEC;  // states move 16 bytes at a time
  typedef RecVec<S, SV> VS;
  constexpr int NA = GRAD ? (GATED ? 4 : 3) : 2, NO = GRAD ? 2 : 1, B = 4;
  const long long grp = blockIdx.x * 128ll + threadIdx.x, per = g.inner / VEC;
  if (grp >= g.outer * per) return;
  const long long o = grp / per, i = (grp - o * per) * VEC, chain = o * g.inner + i;
  const T *in[NA];
#pragma unroll
  for (int q = 0; q < NA; ++q) in[q] = (const T *)g.in[q].p + o * g.in[q].so + i;
  T *out[NO];
#pragma unroll
  for (int q = 0; q < NO; ++q) out[q] = (T *)const_cast<void *>(g.out[q].p) + o * g.out[q].so + i;
  auto states = [&](const void *p, S *to) {
#pragma unroll
    for (int v = 0; v < VEC; v += SV) {
      VS r;
#pragma unroll
      for (int e = 0; e < SV; ++e) r.v[e] = S(0);
      if (p) r = *reinterpret_cast<const VS *>((const S *)p + chain + v);
#pragma unroll
      for (int e = 0; e < SV; ++e) to[v + e] = r.v[e];
    }
  };
  S s[VEC];
  chain_wait();
  chain_next();
  states(g.seed, s);
  for (int k0 = 0; k0 < g.steps; k0 += B) {
    V raw[B][NA];
#pragma unroll
    for (int j = 0; j < B; ++j) {
      const long long t = GRAD ? g.steps - 1 - (k0 + j) : k0 + j;
#pragma unroll
      for (int q = 0; q < NA; ++q)
        if (k0 + j < g.steps && (!GRAD || q != 2 || t > 0))
          raw[j][q] = *reinterpret_cast<const V *>(in[q] + (GRAD && q == 2 ? t - 1 : t) * g.in[q].st);
    }
#pragma unroll
    for (int j = 0; j < B; ++j) {
      if (k0 + j >= g.steps) break;
      const long long t = GRAD ? g.steps - 1 - (k0 + j) : k0 + j;
      S hp[GRAD ? VEC : 1];
      if constexpr (GRAD) {
        if (t > 0) {
#pragma unroll
          for (int v = 0; v < VEC; ++v) hp[v] = Cvt<S, T>::f(raw[j][2].v[v]);
        } else {
          states(g.h0, hp);
        }
      }
      V r0, r1;
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        S f = Cvt<S, T>::f(raw[j][0].v[v]), rest = S(1);
        const S x = Cvt<S, T>::f(raw[j][1].v[v]);  // grad in the backward pass
        if (GATED) rec_gate<T>(f, f, rest);
        if (!GRAD) {
          s[v] = fma(f, s[v], GATED ? rest * x : x);
          r0.v[v] = Cvt<T, S>::f(s[v]);
        } else {
          const S gt = x + s[v];
          r0.v[v] = Cvt<T, S>::f(GATED ? gt * (hp[GRAD ? v : 0] - Cvt<S, T>::f(raw[j][NA - 1].v[v])) * (f * rest)
                                       : gt * hp[GRAD ? v : 0]);
          r1.v[v] = Cvt<T, S>::f(GATED ? gt * rest : gt);
          s[v] = f * gt;
        }
      }
      *reinterpret_cast<V *>(out[0] + t * g.out[0].st) = r0;
      if (GRAD) *reinterpret_cast<V *>(out[NO - 1] + t * g.out[NO - 1].st) = r1;
    }
  }
  if (g.last) {
#pragma unroll
    for (int v = 0; v < VEC; v += SV) {
      VS r;
#pragma unroll
      for (int e = 0; e < SV; ++e) r.v[e] = s[v + e];
      *reinterpret_cast<VS *>((S *)g.last + chain + v) = r;
    }
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

// Bytes of the ring of `warps` warps.
template <class T, int VEC, int COPY, bool GRAD, bool GATED> constexpr size_t rec_ring(int stages, int warps) {
  constexpr int N = mmpd::RecSpan<(int)sizeof(T) * VEC, COPY, GRAD>::value, NA = GRAD ? (GATED ? 4 : 3) : 2;
  return 128 + (size_t)stages * NA * N * warps * 32 * sizeof(T) * VEC;
}
template <int COPY> constexpr int kRecStages = COPY != mmpd::kPlain ? 3 : 2;  // at most

template <class T, int VEC, int COPY, bool GRAD, bool GATED, bool CLUSTER, bool HOLD>
int rec_launch(const RecArgs &g, const mmpd::RecMaps<COPY> &maps, unsigned blocks, int ranks) {
  auto fn = mmpd::rec_kernel<T, VEC, COPY, GRAD, GATED, CLUSTER, HOLD>;
  static mmp::SmemLimit limit;
  const int rc = limit.raise(fn, rec_ring<T, VEC, COPY, GRAD, GATED>(kRecStages<COPY>, mmpd::kRecWarps));
  if (rc) return rc;
  const size_t smem = rec_ring<T, VEC, COPY, GRAD, GATED>(g.stages, g.warps);
  // the composing warps and the joining one
  return mmp::launch_after(fn, blocks * ranks, dim3(32, g.warps + 1), smem, ranks, g, maps);
}

// Byte strides of the second and third axis of a tensor map, as its
// documentation wants them: multiples of 16 below 2^40, the first at least a
// row, the second a multiple of the first.  An axis of one entry takes one
// that fits.
struct RecStrides {
  long long s1, s2;
  bool swap;
};
bool rec_strides(const RecView &v, const RecArgs &g, long long e, RecStrides *s) {
  const long long most = 1ll << 40, row = g.inner * e;
  if (v.st >= most / e || v.so >= most / e) return false;
  long long st = v.st * e, so = v.so * e;
  if (g.outer == 1) so = (g.steps == 1 ? (row + 15) / 16 * 16 : st) * g.steps;
  if (g.steps == 1) st = g.outer == 1 ? (row + 15) / 16 * 16 : so;
  s->swap = so < st;
  s->s1 = s->swap ? so : st;
  s->s2 = s->swap ? st : so;
  return s->s1 >= row && s->s1 > 0 && s->s1 % 16 == 0 && s->s2 % s->s1 == 0 && s->s2 < most;
}

typedef CUresult (*PFN_Encode)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                               const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A map over (inner, steps, outer), or (inner, outer, steps) where the steps
// lie further apart, with boxes of chains x steps.
int rec_map_of(mmpd::RecMap3 *map, const RecView &v, const RecArgs &g, int e, int chains, int steps) {
  static const PFN_Encode enc = (PFN_Encode)mmp::driver_fn("cuTensorMapEncodeTiled");
  if (!enc) return mmp::set_error(MMP_E_CUDA, "cuTensorMapEncodeTiled unavailable");
  RecStrides s;
  if (!rec_strides(v, g, e, &s)) return mmp::set_error(MMP_E_ARG, "recurrence: strides of a tensor copy");
  const bool swap = map->swap = s.swap;
  const cuuint64_t dims[3] = {(cuuint64_t)g.inner, (cuuint64_t)(swap ? g.outer : g.steps),
                              (cuuint64_t)(swap ? g.steps : g.outer)};
  const cuuint64_t strides[2] = {(cuuint64_t)s.s1, (cuuint64_t)s.s2};
  const cuuint32_t box[3] = {(cuuint32_t)chains, (cuuint32_t)(swap ? 1 : steps), (cuuint32_t)(swap ? steps : 1)};
  const cuuint32_t one[3] = {1, 1, 1};
  const CUresult r = enc(&map->m,
                         e == 2   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                         : e == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : CU_TENSOR_MAP_DATA_TYPE_FLOAT64,
                         3,
                         const_cast<void *>(v.p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return mmp::set_error(MMP_E_CUDA, "recurrence: cuTensorMapEncodeTiled failed");
  return MMP_OK;
}

template <class T, int VEC, int COPY, bool GRAD, bool GATED>
int rec_run(RecArgs g) {
  constexpr int N = mmpd::RecSpan<(int)sizeof(T) * VEC, COPY, GRAD>::value;
  constexpr int NA = GRAD ? (GATED ? 4 : 3) : 2;
  constexpr int NC = 32 * VEC;
  g.err = mmp::device_error_word();
  g.near = 1;
  for (const RecView &v : g.in) g.near &= v.st * (long long)sizeof(T) == (int)(v.st * (long long)sizeof(T));
  for (const RecView &v : g.out) g.near &= v.st * (long long)sizeof(T) == (int)(v.st * (long long)sizeof(T));
  g.tiles = (g.inner + NC - 1) / NC;
  const long long blocks = COPY == mmpd::kTma ? g.outer * g.tiles : (g.outer * (g.inner / VEC) + 31) / 32;
  // As many warps a block as there are spans for, and blocks a cluster while
  // all fit at two an SM: 1 x 65521 x 1000 float32 (32 blocks) takes 590 us in
  // blocks alone and 123 in clusters of eight.  Where the blocks are up to one
  // and a half times the SMs, clusters of four, in more than one wave, even out
  // what one wave leaves idle (whole calls: 96 blocks float16 gated 114 us in
  // twos and 93 in fours, its gradient 165 and 136; 160 blocks float32 99 alone
  // and 94, 192 blocks' gradient 192 and 172; but 128 blocks 113 and 116).  From
  // there on blocks alone: 256 of 8 x 2048 x 2048 float16 46 us, in fours 71.
  const long long spans = ((long long)g.steps + N - 1) / N;
  const int warps = spans < mmpd::kRecWarps ? (int)spans : mmpd::kRecWarps, sms = mmp::sm_count();
  int ranks = 1;
  while (ranks < 8 && blocks * ranks * 2 <= 2 * sms && (long long)ranks * warps < spans) ranks *= 2;
  if (ranks < 4 && blocks * 2 <= 3 * sms && spans >= 8 * warps)  // two rounds of spans at least
    ranks = spans >= 192 * warps ? 8 : 4;
  if (blocks * ranks > INT32_MAX) return mmp::set_error(MMP_E_ARG, "recurrence: too many chains");
  g.iters = (int)((spans + (long long)warps * ranks - 1) / ((long long)warps * ranks));
  g.warps = warps;
  g.stages = g.iters < kRecStages<COPY> ? g.iters : kRecStages<COPY>;
  mmpd::RecMaps<COPY> maps;
  if constexpr (COPY == mmpd::kTma) {
    for (int q = 0; q < NA; ++q) {
      const int rc = rec_map_of(&maps.in[q], g.in[q], g, (int)sizeof(T), NC, N);
      if (rc) return rc;
    }
  }
  // Gates are held where blocks stand alone (8 x 2048 x 2048 float16 44 us,
  // evaluated twice 63).  In clusters that leaves the exchange uncovered: it
  // pays forward and for float64 where SMs have two blocks (1 x 16384 x 2048
  // float16 58 us against 66, its gradient 107 against 93; 1 x 65536 x 512, 64
  // blocks, 154 against 134; 1 x 8192 x 1024 float64 57 against 75, its gradient
  // 87 against 96).
  constexpr bool can_hold = GATED && (!GRAD || sizeof(T) == 8);
  if (ranks == 1) return rec_launch<T, VEC, COPY, GRAD, GATED, false, GATED>(g, maps, (unsigned)blocks, 1);
  if constexpr (can_hold)
    if (blocks * ranks > sms) return rec_launch<T, VEC, COPY, GRAD, GATED, true, true>(g, maps, (unsigned)blocks, ranks);
  return rec_launch<T, VEC, COPY, GRAD, GATED, true, false>(g, maps, (unsigned)blocks, ranks);
}

// Whether every operand can be moved in pieces of `bytes` (e: element size).
bool rec_aligned(const RecArgs &g, int nin, int nout, size_t bytes, size_t e) {
  const long long vec = (long long)(bytes / e);
  if (g.inner % vec) return false;
  auto ok = [&](const RecView &v) { return (uintptr_t)v.p % bytes == 0 && v.so % vec == 0 && v.st % vec == 0; };
  for (int i = 0; i < nin; ++i)
    if (!ok(g.in[i])) return false;
  for (int i = 0; i < nout; ++i)
    if (!ok(g.out[i])) return false;
  return true;
}

// Whether tensor copies can take the inputs, and their tiles of `chains` along
// inner are at least three quarters full.
bool rec_tensors(const RecArgs &g, int nin, int chains, long long e) {
  if (g.inner * 4 < (g.inner + chains - 1) / chains * chains * 3) return false;
  if (g.inner > INT32_MAX || g.outer > INT32_MAX) return false;
  RecStrides s;
  for (int i = 0; i < nin; ++i)
    if ((uintptr_t)g.in[i].p % 16 || !rec_strides(g.in[i], g, e, &s)) return false;
  return true;
}

template <class T, int VEC, bool GRAD, bool GATED>
int rec_short(const RecArgs &g) {
  const long long blocks = (g.outer * (g.inner / VEC) + 127) / 128;
  if (blocks > INT32_MAX) return mmp::set_error(MMP_E_ARG, "recurrence: too many chains");
  return mmp::launch_after(mmpd::rec_short_kernel<T, VEC, GRAD, GATED>, (unsigned)blocks, 128, 0, 1, g);
}

template <bool GRAD, bool GATED>
int rec_dispatch(int dtype, const RecArgs &g) {
  using namespace mmpd;
  constexpr int nin = GRAD ? (GATED ? 4 : 3) : 2, nout = GRAD ? 2 : 1;
  // Up to 32 steps (backward 16) the chains alone are worked on side by side:
  // 32 x 1 x 2048 float16 takes 7.0 us by the spans' kernel, 3.7 here; whole
  // calls at 8 x 24 x 1024 12.0 and 9.0, 64 x 32 x 4096 23.4 and 19.1, but 16 x
  // 64 x 4096 12.8 and 19.2, backward 8 x 32 x 1024 13.5 and 17.4.
  if (g.steps <= (GRAD ? 16 : 32)) {
    const bool states = ((uintptr_t)g.h0 | (uintptr_t)g.seed | (uintptr_t)g.last) % 16 == 0;
    const bool wide = states && rec_aligned(g, nin, nout, 16, mmp_dtype_size(dtype));
    if (dtype == MMP_FLOAT16) {
      if (wide) return rec_short<__half, 8, GRAD, GATED>(g);
      return states && rec_aligned(g, nin, nout, 4, 2) ? rec_short<__half, 2, GRAD, GATED>(g)
                                                       : rec_short<__half, 1, GRAD, GATED>(g);
    }
    if (dtype == MMP_FLOAT32) return wide ? rec_short<float, 4, GRAD, GATED>(g) : rec_short<float, 1, GRAD, GATED>(g);
    return wide ? rec_short<double, 2, GRAD, GATED>(g) : rec_short<double, 1, GRAD, GATED>(g);
  }
  if (dtype == MMP_FLOAT16) {
    if (!rec_aligned(g, nin, nout, 4, 2)) return rec_run<__half, 1, kPlain, GRAD, GATED>(g);
    return rec_tensors(g, nin, 64, 2) ? rec_run<__half, 2, kTma, GRAD, GATED>(g)
                                      : rec_run<__half, 2, kLane, GRAD, GATED>(g);
  }
  if (dtype == MMP_FLOAT32)
    return rec_tensors(g, nin, 32, 4) ? rec_run<float, 1, kTma, GRAD, GATED>(g)
                                      : rec_run<float, 1, kLane, GRAD, GATED>(g);
  return rec_tensors(g, nin, 32, 8) ? rec_run<double, 1, kTma, GRAD, GATED>(g)
                                    : rec_run<double, 1, kLane, GRAD, GATED>(g);
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
  if (!mmp::device_error_word()) return mmp::set_error(MMP_E_CUDA, "no CUDA device available");
  RecArgs g = {};
  g.in[0] = RecView{a, a_so, a_st};
  g.in[1] = RecView{x, x_so, x_st};
  g.out[0] = RecView{h, h_so, h_st};
  g.h0 = g.seed = h0;
  g.last = state;
  g.steps = (int)steps;
  g.outer = outer;
  g.inner = inner;
  return gated ? rec_dispatch<false, true>(dtype, g) : rec_dispatch<false, false>(dtype, g);
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
  if (!mmp::device_error_word()) return mmp::set_error(MMP_E_CUDA, "no CUDA device available");
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
  r.outer = outer;
  r.inner = inner;
  return gated ? rec_dispatch<true, true>(dtype, r) : rec_dispatch<true, false>(dtype, r);
}

}  // extern "C"
