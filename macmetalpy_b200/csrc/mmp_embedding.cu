// mmp_embedding / mmp_embedding_grad: rows of a table by token id, times a
// scale, and the gradient of the table,
//   out[n, :] = scale * weight[ids[n], :]
//   grad_weight[v, :] = scale * sum over n with ids[n] = v of grad[n, :].
// The reference has take (indexing.py:24-60; numpy on the host) without a
// scale or a gradient.  Products and sums are in float32 (float64 for
// float64 tables) and each output is rounded once.  An id outside [0, rows)
// gives a row of zeros in the lookup, adds nothing in the gradient, and sets
// device error 5, as mmp_gather does for an offset.
//
// Both are bound by HBM traffic.  The gradient reads each row of grad once
// and writes each row of the table once, zeros included, whatever the ids:
//   few tokens   one launch: a block a token, which adds its id's rows if it
//                is the first with that id; other blocks write the zeros of
//                the rows without a token.
//   more         the tokens are sorted by id (stable, so the order of every
//                sum is the ids' alone) by one cluster; then equal shares of
//                the sorted tokens are added run by run, and the few runs over
//                several shares are joined.  The zeros are written beside the
//                sort and beside the sums: writes alone reach 3.9 TB/s here
//                (a plain fill), with reads next to them 6.5 in all.
// No float is added atomically, so equal calls give equal bits.  Inputs are
// not marked __restrict__: a kernel launched by launch_after is resident while
// the one before it still writes them, and a load that passes for one of
// constant memory need not stay behind chain_wait.
// Whole calls: lookup of 16384 of 128000 x 1024 float32 17 us (writes alone take
// 17 at the fill rate); gradient of 512 tokens, 8192 x 768 float32 8.4 us, of
// 16384 tokens, 50257 x 2048 float16 69 us (fill rate 52, copy rate 42), of
// 131072 tokens, 50257 x 768 float16 145 us.
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>
#include <utility>

#include "mmp_chain.cuh"
#include "mmp_device.cuh"
#include "mmp_embedding_plan.h"
#include "mmp_internal.h"

namespace mmpd {

namespace cg = cooperative_groups;

template <class T> struct EmbAcc { typedef float type; };
template <> struct EmbAcc<double> { typedef double type; };

template <class T, int VEC> struct alignas(sizeof(T) * VEC) EmbVec { T v[VEC]; };

// ---- lookup: a thread moves U vectors; vectors of a row are neighbours.
template <class T, class I, int VEC, int U>
__global__ void __launch_bounds__(256) emb_kernel(const T *w, long long rows, FastDiv per,
                                                  long long w_stride, const I *ids, unsigned total,
                                                  typename EmbAcc<T>::type scale, T *__restrict__ out, int *err) {
  typedef typename EmbAcc<T>::type S;
  typedef EmbVec<T, VEC> V;
  const unsigned i0 = blockIdx.x * (256u * U) + threadIdx.x;
  chain_wait();
  chain_next();
  unsigned col[U];
  long long id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned i = i0 + u * 256u;
    const unsigned r = per.div(i);
    col[u] = i - r * per.d;
    id[u] = i < total ? (long long)ids[r] : -1;
  }
  V v[U];
  bool bad = false;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool ok = id[u] >= 0 && id[u] < rows;
    bad |= !ok && i0 + u * 256u < total;
    if (ok) {
      v[u] = *reinterpret_cast<const V *>(w + id[u] * w_stride + (long long)col[u] * VEC);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[u].v[e] = Cvt<T, S>::f(S(0));
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned i = i0 + u * 256u;
    if (i >= total) break;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[u].v[e] = Cvt<T, S>::f(Cvt<S, T>::f(v[u].v[e]) * scale);
    *reinterpret_cast<V *>(out + (long long)i * VEC) = v[u];
  }
  if (bad) atomicExch(err, 5);
}

// ---- ids alone, of a call that has no element to write.
template <class I>
__global__ void __launch_bounds__(256) emb_ids_kernel(const I *ids, unsigned n, long long rows, int *err) {
  chain_wait();
  chain_next();
  bool bad = false;
  for (unsigned i = blockIdx.x * 256u + threadIdx.x; i < n; i += gridDim.x * 256u) {
    const long long id = (long long)ids[i];
    bad |= id < 0 || id >= rows;
  }
  if (bad) atomicExch(err, 5);
}

// Zeros to `n` elements by one warp: 16-byte pieces, the ends element by
// element.
template <class T> __device__ __forceinline__ void emb_zero(T *p, long long n) {
  constexpr int PE = 16 / (int)sizeof(T);
  const T zero = Cvt<T, float>::f(0.0f);
  const int lane = threadIdx.x & 31;
  long long head = (long long)((16 - ((uintptr_t)p & 15)) & 15) / (long long)sizeof(T);
  if (head > n) head = n;
  if (lane < head) p[lane] = zero;  // at most 7
  p += head;
  n -= head;
  uint4 *q = reinterpret_cast<uint4 *>(p);
  const long long pieces = n / PE;
#pragma unroll 4
  for (long long i = lane; i < pieces; i += 32) q[i] = make_uint4(0, 0, 0, 0);
  if (lane < n - pieces * PE) p[pieces * PE + lane] = zero;
}

// ---- zeros of the rows [r0, r1) that no token has, by one block.  s_seen: a
// bitmap of at least r1 - r0 bits.  A warp takes `unit` rows of one word of
// it; neighbouring rows without a token are one stretch of memory.
template <class T, class I>
__device__ void emb_zero_rows(const I *ids, unsigned n, long long rows, long long padding, long long r0,
                              long long r1, unsigned width, T *__restrict__ out, unsigned *s_seen, int *err) {
  const unsigned tid = threadIdx.x, nt = blockDim.x;
  const unsigned count = (unsigned)(r1 - r0);
  __syncthreads();
  for (unsigned i = tid; i < (count + 31) / 32; i += nt) s_seen[i] = 0;
  __syncthreads();
#pragma unroll 4
  for (unsigned i = tid; i < n; i += nt) {
    const long long id = (long long)ids[i];
    if (id >= r0 && id < r1 && id != padding) {
      unsigned *word = s_seen + ((id - r0) >> 5);
      const unsigned bit = 1u << ((id - r0) & 31);
      if (!(*(volatile unsigned *)word & bit)) atomicOr(word, bit);  // frequent ids do not queue up
    }
    if (err && r0 == 0 && (id < 0 || id >= rows)) atomicExch(err, 5);
  }
  __syncthreads();
  // four units a warp at least, where there are rows enough
  unsigned unit = 32;
  while (unit > 1 && count / unit < nt / 32 * 4) unit /= 2;
  for (unsigned r = tid / 32 * unit; r < count; r += nt / 32 * unit) {
    const unsigned m = count - r < unit ? count - r : unit;
    unsigned open = ~(s_seen[r >> 5] >> (r & 31)) & (m == 32 ? 0xffffffffu : (1u << m) - 1);
    while (open) {
      const unsigned lo = __ffs(open) - 1, over = ~(open >> lo);
      const unsigned len = over ? __ffs(over) - 1 : 32;
      emb_zero(out + (r0 + r + lo) * width, (long long)len * width);
      open &= len == 32 ? 0u : ~(((1u << len) - 1) << lo);
    }
  }
}

// This block's part of the rows, in stretches of at most `bits` rows.
template <class T, class I>
__device__ __forceinline__ void emb_zero_share(const I *ids, unsigned n, long long rows, long long padding, unsigned part,
                                               unsigned parts, unsigned bits, unsigned width, T *out, unsigned *s_seen,
                                               int *err) {
  const long long share = (rows + parts - 1) / parts;
  const long long a = share * part, b = a + share < rows ? a + share : rows;
  for (long long r = a; r < b; r += bits)
    emb_zero_rows<T, I>(ids, n, rows, padding, r, r + bits < b ? r + bits : b, width, out, s_seen, err);
}

constexpr unsigned kEmbFew = 1024;       // tokens up to which no sort is made
constexpr unsigned kEmbFewBits = 16384;  // rows a block of that path marks at once

// Zeros of the rows [r0, rows) whose bit in `seen` is not set, by warps
// `warp`, `warp` + `warps`, ..., `unit` rows of a word at a time: r0 is a
// multiple of `unit`, a power of two up to 32, so that no unit reaches into
// the next word (EmbZeroPlan).
template <class T>
__device__ __forceinline__ void emb_zero_marked(const unsigned *seen, unsigned r0, unsigned rows,
                                                unsigned width, T *__restrict__ out, unsigned unit, unsigned warp,
                                                unsigned warps) {
  for (unsigned long long r = r0 + (unsigned long long)warp * unit; r < rows; r += (unsigned long long)warps * unit) {
    const unsigned m = rows - r < unit ? rows - (unsigned)r : unit;
    unsigned open = ~(seen[r >> 5] >> (r & 31)) & (m == 32 ? 0xffffffffu : (1u << m) - 1);
    while (open) {
      const unsigned lo = __ffs(open) - 1, over = ~(open >> lo);
      const unsigned len = over ? __ffs(over) - 1 : 32;
      emb_zero(out + (size_t)(r + lo) * width, (long long)len * width);
      open &= len == 32 ? 0u : ~(((1u << len) - 1) << lo);
    }
  }
}

// Sets the bits of a warp's ids (`want`: this lane has one).  Frequent ids
// share words: the warp's bits of one word go in one atomic, and none goes
// where they are set already.
__device__ __forceinline__ void emb_mark(unsigned *seen, unsigned id, bool want) {
  const unsigned word = want ? id >> 5 : 0xffffffffu;
  const unsigned mates = __match_any_sync(0xffffffffu, word);
  const unsigned bits = __reduce_or_sync(mates, 1u << (id & 31));
  if (!want || (unsigned)__ffs(mates) - 1 != (threadIdx.x & 31)) return;
  if (~*(volatile unsigned *)(seen + word) & bits) atomicOr(seen + word, bits);
}

// ---- few tokens, one launch.  Blocks [0, n): token blockIdx.x, if it is the
// first of its id, adds all of them in the order of n.  The others: zeros.
template <class T, class I, int VEC>
__global__ void __launch_bounds__(256) emb_grad_few(const I *ids, unsigned n, const T *grad,
                                                    long long g_stride, long long rows, unsigned width,
                                                    typename EmbAcc<T>::type scale, long long padding,
                                                    T *__restrict__ out, int *err) {
  typedef typename EmbAcc<T>::type S;
  typedef EmbVec<T, VEC> V;
  __shared__ unsigned s_buf[kEmbFew];  // the list of tokens, or the bitmap
  __shared__ unsigned s_sum[8];
  const unsigned tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  chain_wait();
  chain_next();
  if (blockIdx.x >= n) {
    emb_zero_share<T, I>(ids, n, rows, padding, blockIdx.x - n, gridDim.x - n, kEmbFewBits, width, out, s_buf, err);
    return;
  }
  const unsigned me = blockIdx.x;
  const long long id = (long long)ids[me];
  if (id < 0 || id >= rows) {
    if (tid == 0) atomicExch(err, 5);
    return;
  }
  if (id == padding) return;
  // the tokens of this id in order, 4 places a thread
  unsigned hit = 0, count = 0;
  bool earlier = false;
#pragma unroll
  for (unsigned u = 0; u < kEmbFew / 256; ++u) {
    const unsigned i = tid * (kEmbFew / 256) + u;
    if (i < n && (long long)ids[i] == id) {
      hit |= 1u << u;
      ++count;
      earlier |= i < me;
    }
  }
  if (__syncthreads_or(earlier)) return;
  unsigned before = count;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned t = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += t;
  }
  if (lane == 31) s_sum[w] = before;
  __syncthreads();
  unsigned total = 0;
  before -= count;
#pragma unroll
  for (unsigned v = 0; v < 8; ++v) {
    if (v < w) before += s_sum[v];
    total += s_sum[v];
  }
#pragma unroll
  for (unsigned u = 0; u < kEmbFew / 256; ++u)
    if (hit >> u & 1) s_buf[before++] = tid * (kEmbFew / 256) + u;
  __syncthreads();
  for (unsigned c = tid * VEC; c < width; c += 256 * VEC) {
    S acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = S(0);
    unsigned k = 0;
    for (; k + 8 <= total; k += 8) {
      V v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = *reinterpret_cast<const V *>(grad + s_buf[k + j] * g_stride + c);
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += Cvt<S, T>::f(v[j].v[e]);
    }
    for (; k < total; ++k) {
      const V v = *reinterpret_cast<const V *>(grad + s_buf[k] * g_stride + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += Cvt<S, T>::f(v.v[e]);
    }
    V r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r.v[e] = Cvt<T, S>::f(acc[e] * scale);
    *reinterpret_cast<V *>(out + id * width + c) = r;
  }
}

// ---- the sort of up to kEmbCluster tokens by one cluster, beside the zeros.
constexpr int kSortThreads = 1024, kSortRanks = 8, kSortItems = 8;
constexpr unsigned kEmbCluster = kSortThreads * kSortRanks * kSortItems;  // 65536
constexpr int kSortBits = 9, kSortBins = 1 << kSortBits;  // of a digit at most
struct EmbSortSmem {
  unsigned short count[32][kSortBins];    // a warp's keys of each digit, then those of the warps before it
  unsigned total[kSortRanks][kSortBins];  // each block's
  unsigned local[kSortBins];              // the digit's first place in the block's order
  unsigned base[kSortBins];               // and in the whole order, for this block's keys
  unsigned sum[2][kSortBins / 32];
  unsigned long long key[2][1];  // E * 1024 each: id << 32 | token
};

__device__ __forceinline__ unsigned emb_lanemask_lt() {
  unsigned m;
  asm("mov.u32 %0, %%lanemask_lt;" : "=r"(m));
  return m;
}

// Inclusive sums over the first kSortBins threads (s_sum: one word a warp).
__device__ __forceinline__ unsigned emb_scan_bins(unsigned v, unsigned *s_sum) {
  const unsigned lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  if (lane == 31) s_sum[w] = v;
  asm volatile("bar.sync 1, %0;" ::"n"(kSortBins) : "memory");
#pragma unroll
  for (unsigned u = 0; u < kSortBins / 32; ++u)
    if (u < w) v += s_sum[u];
  return v;
}

// Cluster 0 sorts (LSD radix: a block has E * 1024 neighbouring keys in its
// shared memory, a warp E * 32 of them; a pass puts them in the block's order
// first, so that neighbouring threads then send neighbouring keys to their
// place in the cluster's shared memory: sent one by one, a pass of 30,000 keys
// took 13 us).  A key that counts for no row
// (padding, out of range) is `rows`.  It also marks the ids in the bitmap
// `seen`.  The other clusters write the zeros of the rows below `zeros`.
template <class T, class I>
__global__ void __cluster_dims__(kSortRanks, 1, 1) __launch_bounds__(kSortThreads, 1)
    emb_sort_kernel(const I *ids, unsigned n, long long rows, long long padding, int items, int passes,
                    int digit, unsigned *__restrict__ keys, unsigned *__restrict__ order, unsigned width,
                    T *__restrict__ out, unsigned zeros, unsigned bits, unsigned *__restrict__ seen,
                    unsigned *__restrict__ runs, int *err) {
  extern __shared__ __align__(16) unsigned char s_raw[];
  chain_wait();
  chain_next();
  if (blockIdx.x >= kSortRanks) {
    emb_zero_share<T, I>(ids, n, zeros, padding, blockIdx.x - kSortRanks, gridDim.x - kSortRanks, bits, width, out,
                         (unsigned *)s_raw, nullptr);
    return;
  }
  EmbSortSmem &s = *reinterpret_cast<EmbSortSmem *>(s_raw);
  cg::cluster_group cl = cg::this_cluster();
  // No block may reach into another's shared memory before that one runs:
  // what the first pass sends waits for this barrier, the ids' loads do not.
  auto running = cl.barrier_arrive();
  const unsigned rank = cl.block_rank();
  const unsigned tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const unsigned tile = items * kSortThreads;
  unsigned long long *const buf[2] = {s.key[0], s.key[0] + tile};
  if (rank == 0 && tid == 0) *runs = 0;
  for (long long i = rank * kSortThreads + tid; i < (rows + 31) / 32; i += kSortRanks * kSortThreads) seen[i] = 0;
  const unsigned place = w * items * 32 + lane;  // this thread's keys: place + 32 e
  const unsigned lt = emb_lanemask_lt();
  long long id[kSortItems];
#pragma unroll
  for (int e = 0; e < kSortItems; ++e) {
    const unsigned i = rank * tile + place + e * 32;
    id[e] = e < items && i < n ? (long long)ids[i] : padding;
  }
#pragma unroll
  for (int e = 0; e < kSortItems; ++e) {
    const unsigned p = place + e * 32, i = rank * tile + p;
    if (e < items && i < n) {
      const bool ok = id[e] >= 0 && id[e] < rows;
      if (!ok) atomicExch(err, 5);
      buf[0][p] = (unsigned long long)(ok && id[e] != padding ? id[e] : rows) << 32 | i;
    }
  }
  cl.barrier_wait(std::move(running));
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = 32 + pass * digit;
    const unsigned mask = (1u << digit) - 1;
    unsigned long long *from = buf[pass & 1];
    for (unsigned j = tid; j < sizeof(s.count) / 4; j += kSortThreads) reinterpret_cast<unsigned *>(s.count)[j] = 0;
    __syncthreads();
    unsigned long long k[kSortItems];
    unsigned at[kSortItems];
#pragma unroll
    for (int e = 0; e < kSortItems; ++e) {
      if (e < items) {
        const bool valid = rank * tile + place + e * 32 < n;
        k[e] = valid ? from[place + e * 32] : 0;
        const unsigned d = (unsigned)(k[e] >> shift) & mask;
        unsigned peers = __ballot_sync(0xffffffffu, valid);
        for (int b = 0; b < digit; ++b) {
          const bool bit = (d >> b) & 1u;
          const unsigned bal = __ballot_sync(0xffffffffu, bit);
          peers &= bit ? bal : ~bal;
        }
        const unsigned c = valid ? s.count[w][d] : 0u, before = __popc(peers & lt);
        __syncwarp();
        if (valid && before == 0) s.count[w][d] = (unsigned short)(c + __popc(peers));
        __syncwarp();
        at[e] = c + before;
      }
    }
    __syncthreads();
    // thread = digit: each warp's first place among the block's keys of the
    // digit, the digit's first place in the block
    unsigned mine = 0, inc = 0;
    if (tid < kSortBins) {
      unsigned short c[32];
#pragma unroll
      for (int v = 0; v < 32; ++v) c[v] = s.count[v][tid];
#pragma unroll
      for (int v = 0; v < 32; ++v) {
        s.count[v][tid] = (unsigned short)mine;
        mine += c[v];
      }
      for (int r = 0; r < kSortRanks; ++r) *cl.map_shared_rank(&s.total[rank][tid], r) = mine;
      inc = emb_scan_bins(mine, s.sum[0]);
      s.local[tid] = inc - mine;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kSortItems; ++e) {
      if (e < items && rank * tile + place + e * 32 < n) {
        const unsigned d = (unsigned)(k[e] >> shift) & mask;
        const unsigned q = s.local[d] + s.count[w][d] + at[e];
        if (q < tile) from[q] = k[e];
        else atomicExch(err, 4);  // inconsistent counts: report, never write out of bounds
      }
    }
    cl.sync();
    if (tid < kSortBins) {
      unsigned all = 0, below = 0;
#pragma unroll
      for (int r = 0; r < kSortRanks; ++r) {
        const unsigned t = s.total[r][tid];
        if (r < (int)rank) below += t;
        all += t;
      }
      s.base[tid] = emb_scan_bins(all, s.sum[1]) - all + below;
    }
    __syncthreads();
    const bool final = pass + 1 == passes;
    unsigned long long *to = buf[(pass & 1) ^ 1];
    const unsigned have = n > rank * tile ? (n - rank * tile < tile ? n - rank * tile : tile) : 0;
#pragma unroll
    for (int e = 0; e < kSortItems; ++e) {
      const unsigned j = e * kSortThreads + tid;
      if (final && e < items) {
        // the block's keys are in order now: the first of each id in the warp marks it
        const unsigned id = j < have ? (unsigned)(from[j] >> 32) : 0xffffffffu;
        const unsigned left = __shfl_up_sync(0xffffffffu, id, 1);
        if (id < (unsigned)rows && (lane == 0 || left != id)) atomicOr(&seen[id >> 5], 1u << (id & 31));
      }
      if (j < have) {
        const unsigned long long key = from[j];
        const unsigned d = (unsigned)(key >> shift) & mask;
        const unsigned dst = s.base[d] + j - s.local[d];
        if (dst >= n) {
          atomicExch(err, 4);
        } else if (final) {
          keys[dst] = (unsigned)(key >> 32);
          order[dst] = (unsigned)key;
        } else {
          const unsigned r = dst / tile;
          *cl.map_shared_rank(&to[dst - r * tile], r) = key;
        }
      }
    }
    cl.sync();
  }
}

// ---- more tokens than a cluster holds: keys for sort_pairs, and the marks.
template <class I>
__global__ void __launch_bounds__(256) emb_prep_kernel(const I *ids, unsigned n, long long rows,
                                                       long long padding, unsigned *__restrict__ keys,
                                                       unsigned *__restrict__ order, unsigned *__restrict__ seen,
                                                       int *err) {
  for (unsigned i0 = blockIdx.x * 256u; i0 < n; i0 += gridDim.x * 256u) {
    const unsigned i = i0 + threadIdx.x;
    const long long id = i < n ? (long long)ids[i] : padding;
    const bool ok = id >= 0 && id < rows;
    if (i < n) {
      if (!ok) atomicExch(err, 5);
      keys[i] = (unsigned)(ok && id != padding ? id : rows);
      order[i] = i;
    }
    emb_mark(seen, (unsigned)id, i < n && ok && id != padding);
  }
}

// ---- sums over the sorted tokens.  Shares of `share` tokens; a group of
// `lanes` threads has one share and the columns of its vectors.  The share
// where a run of one id begins adds it whole, into the next share if it ends
// there.  A run of further shares is left in parts, part[share][0] (what
// continues from the share before) and part[share][1] (what begins here),
// and listed in `list` for the next kernel (in any order).
struct EmbRun {
  unsigned share, more, id;  // begins in `share` and goes on through `more` others
};

template <class T, int VEC>
__global__ void __launch_bounds__(256) emb_sum_kernel(const unsigned *keys,
                                                      const unsigned *order, unsigned n, unsigned share,
                                                      unsigned shares, unsigned lanes, const T *grad,
                                                      long long g_stride, unsigned rows, unsigned width,
                                                      typename EmbAcc<T>::type scale, T *__restrict__ out,
                                                      typename EmbAcc<T>::type *__restrict__ part,
                                                      unsigned *__restrict__ runs, EmbRun *__restrict__ list,
                                                      const unsigned *seen, unsigned zeros,
                                                      unsigned zeros_end, unsigned unit, unsigned zero_blocks) {
  typedef typename EmbAcc<T>::type S;
  typedef EmbVec<T, VEC> V;
  chain_wait();
  chain_next();
  if (blockIdx.x < zero_blocks) {  // the zeros of the rows [zeros, zeros_end)
    emb_zero_marked(seen, zeros, zeros_end, width, out, unit,
                    (blockIdx.y * zero_blocks + blockIdx.x) * 8 + threadIdx.x / 32, gridDim.y * zero_blocks * 8);
    return;
  }
  const unsigned grp = threadIdx.x / lanes, groups = 256 / lanes;
  const unsigned s = (blockIdx.x - zero_blocks) * groups + grp;
  const unsigned c = (blockIdx.y * lanes + threadIdx.x % lanes) * VEC;
  if (s >= shares || grp >= groups || c >= width) return;
  unsigned i = s * share;
  const unsigned i0 = i, i1 = n - i < share ? n : i + share;
  unsigned cur = keys[i];
  if (cur >= rows) return;  // sorted last: nothing from here on counts
  bool head = i > 0 && keys[i - 1] == cur;
  if (head && (i == share || keys[i - share - 1] != cur) && (i1 == n || keys[i1] != cur)) {
    // the share before has this run
    head = false;
    while (i < i1 && keys[i] == cur) ++i;
    if (i == i1) return;
    cur = keys[i];
    if (cur >= rows) return;
  }
  // the last run: to its end if that lies in the next share
  const unsigned after = i1 < n ? keys[i1] : rows;  // a key that goes on behind this share
  const bool goes = after < rows && keys[i1 - 1] == after;
  // (a run that comes from the share before and goes on is longer than that)
  const bool from = goes && keys[i0] == after && i0 > 0 && keys[i0 - 1] == after;
  const bool far = goes && (from || (i1 + share < n && keys[i1 + share] == after));
  const unsigned stop = goes && !far ? (i1 + share < n ? i1 + share : n) : i1;
  S acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = S(0);
  auto flush = [&](bool on) {
    if (head || on) {
      S *p = part + ((size_t)s * 2 + (head ? 0 : 1)) * width + c;
#pragma unroll
      for (int e = 0; e < VEC; ++e) p[e] = acc[e];
      if (!head && c == 0) {
        // the share where it ends: doubling steps, then halving
        unsigned step = 2;
        while ((s + step) * (unsigned long long)share < n && keys[(s + step) * share] == cur) step *= 2;
        unsigned lo = step / 2, hi = step;  // share s + lo begins with the id, s + hi does not
        while (lo + 1 < hi) {
          const unsigned mid = lo + (hi - lo) / 2;
          if ((s + mid) * (unsigned long long)share < n && keys[(s + mid) * share] == cur) lo = mid;
          else hi = mid;
        }
        list[atomicAdd(runs, 1u)] = EmbRun{s, lo, cur};
      }
    } else {
      V r;
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.v[e] = Cvt<T, S>::f(acc[e] * scale);
      *reinterpret_cast<V *>(out + (size_t)cur * width + c) = r;
    }
  };
  auto turn = [&](unsigned key) {  // the next token's id
    if (key != cur) {
      flush(false);
      head = false;
      cur = key;
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] = S(0);
    }
  };
  auto add = [&](const V &v) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] += Cvt<S, T>::f(v.v[e]);
  };
  // B tokens at a time from a multiple of B on (keys and order have that many
  // entries; what lies outside [i, stop) is passed over): eight, or four where
  // eight would take more registers than four blocks an SM have
  constexpr int B = VEC >= 8 ? 4 : 8;
  for (unsigned b = i / B * B; b < stop; b += B) {
    unsigned key[B], at[B];
#pragma unroll
    for (int j = 0; j < B; j += 4) {
      *reinterpret_cast<uint4 *>(key + j) = *reinterpret_cast<const uint4 *>(keys + b + j);
      *reinterpret_cast<uint4 *>(at + j) = *reinterpret_cast<const uint4 *>(order + b + j);
    }
    V v[B];
    if (b >= i && b + B <= i1 && key[B - 1] < rows) {
#pragma unroll
      for (int j = 0; j < B; ++j) v[j] = *reinterpret_cast<const V *>(grad + (long long)at[j] * g_stride + c);
      if (key[0] == cur && key[B - 1] == cur) {
#pragma unroll
        for (int j = 0; j < B; ++j) add(v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < B; ++j) {
          turn(key[j]);
          add(v[j]);
        }
      }
    } else {
      unsigned use = 0;
#pragma unroll
      for (int j = 0; j < B; ++j) {
        const unsigned q = b + j;
        // behind this share only the run that goes on from it
        if (q >= i && q < stop && key[j] < rows && (q < i1 || key[j] == after)) {
          use |= 1u << j;
          v[j] = *reinterpret_cast<const V *>(grad + (long long)at[j] * g_stride + c);
        }
      }
#pragma unroll
      for (int j = 0; j < B; ++j) {
        if (use >> j & 1) {
          turn(key[j]);
          add(v[j]);
        }
      }
    }
  }
  flush(far);
}

// Listed runs: the parts of one in order, a warp an eighth of them, then the
// warps' sums in order.
template <class T, int JV>
__global__ void __launch_bounds__(256) emb_join_kernel(unsigned width, typename EmbAcc<T>::type scale,
                                                       const typename EmbAcc<T>::type *part,
                                                       const unsigned *runs,
                                                       const EmbRun *list, T *__restrict__ out,
                                                       const unsigned *seen, unsigned zeros, unsigned rows,
                                                       unsigned unit, unsigned join_blocks) {
  typedef typename EmbAcc<T>::type S;
  typedef EmbVec<S, JV> V;
  __shared__ V s_part[8][32];
  chain_wait();
  if (blockIdx.x >= join_blocks) {  // the zeros of the rows from `zeros` on
    const unsigned blocks = gridDim.x - join_blocks;
    emb_zero_marked(seen, zeros, rows, width, out, unit,
                    (blockIdx.y * blocks + blockIdx.x - join_blocks) * 8 + threadIdx.x / 32, gridDim.y * blocks * 8);
    return;
  }
  const unsigned lane = threadIdx.x & 31, w = threadIdx.x >> 5, count = *runs;
  for (unsigned k = blockIdx.x; k < count; k += join_blocks) {
    const EmbRun run = list[k];
    const unsigned s = run.share, more = run.more, key = run.id, eighth = (more + 7) / 8;
    const unsigned a = s + 1 + w * eighth, b = a + eighth < s + 1 + more ? a + eighth : s + 1 + more;
    for (unsigned c0 = blockIdx.y * 32 * JV; c0 < width; c0 += gridDim.y * 32 * JV) {
      const unsigned c = c0 + lane * JV;
      V acc;
#pragma unroll
      for (int e = 0; e < JV; ++e) acc.v[e] = S(0);
      if (c < width) {
        if (w == 0) acc = *reinterpret_cast<const V *>(part + ((size_t)s * 2 + 1) * width + c);
#pragma unroll 8
        for (unsigned t = a; t < b; ++t) {
          const V v = *reinterpret_cast<const V *>(part + (size_t)t * 2 * width + c);
#pragma unroll
          for (int e = 0; e < JV; ++e) acc.v[e] += v.v[e];
        }
      }
      s_part[w][lane] = acc;
      __syncthreads();
      if (w == 0 && c < width) {
        for (int v = 1; v < 8; ++v)
#pragma unroll
          for (int e = 0; e < JV; ++e) acc.v[e] += s_part[v][lane].v[e];
#pragma unroll
        for (int e = 0; e < JV; ++e) out[(size_t)key * width + c + e] = Cvt<T, S>::f(acc.v[e] * scale);
      }
      __syncthreads();
    }
  }
}

}  // namespace mmpd

namespace {

using mmpd::FastDiv;

FastDiv emb_div(unsigned d) {
  unsigned l = 0;
  while (l < 32 && (1ull << l) < d) ++l;
  FastDiv f;
  f.d = d;
  f.m = (unsigned)(((1ull << 32) * ((1ull << l) - d)) / d + 1);
  f.s = l;
  return f;
}

int emb_check(const char *what, int dtype, int ids_dtype, int64_t rows, int64_t width, int64_t n) {
  if (rows < 0 || width < 0 || n < 0) return mmp::set_error(MMP_E_ARG, std::string(what) + ": negative size");
  if (dtype != MMP_FLOAT16 && dtype != MMP_FLOAT32 && dtype != MMP_FLOAT64)
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": needs a floating dtype");
  if (ids_dtype != MMP_INT32 && ids_dtype != MMP_INT64)
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": ids must be int32 or int64");
  if (rows > (1 << 30) || n > (1 << 30) || width > (1 << 30))
    return mmp::set_error(MMP_E_ARG, std::string(what) + ": a size passes 2^30");
  return MMP_OK;
}

// Elements that every row can be moved in at once: 16, 8 or 4 bytes where
// width, strides and pointers allow it, else one.
template <class T> int emb_vec(const void *p, const void *q, long long width, long long stride) {
  for (int bytes = 16; bytes > (int)sizeof(T); bytes /= 2) {
    const int vec = bytes / (int)sizeof(T);
    if ((uintptr_t)p % bytes == 0 && (uintptr_t)q % bytes == 0 && width % vec == 0 && stride % vec == 0) return vec;
  }
  return 1;
}

// f(std::integral_constant<int, vec>) for the vec that emb_vec gave.
template <class T, class F> int emb_with_vec(int vec, F f) {
  constexpr int most = 16 / (int)sizeof(T);
  if (vec == most) return f(std::integral_constant<int, most>());
  if constexpr (most >= 4)
    if (vec == most / 2) return f(std::integral_constant<int, most / 2>());
  if constexpr (most >= 8)
    if (vec == most / 4) return f(std::integral_constant<int, most / 4>());
  return f(std::integral_constant<int, 1>());
}

template <class T, class I, int VEC>
int emb_launch(const T *w, int64_t rows, int64_t width, int64_t w_stride, const I *ids, int64_t n, double scale,
               T *out) {
  typedef typename mmpd::EmbAcc<T>::type S;
  const int64_t per = width / VEC;
  // in parts whose vectors 32 bits count
  const int64_t most = (INT64_C(1) << 31) / per > 0 ? (INT64_C(1) << 31) / per : 1;
  for (int64_t r = 0; r < n; r += most) {
    const int64_t m = n - r < most ? n - r : most;
    const unsigned total = (unsigned)(m * per);
    int *err = mmp::device_error_word();
    // four vectors a thread where that leaves every SM its blocks
    const bool four = total >= 1024u * 4 * (unsigned)mmp::sm_count();
    const int rc = mmp::launch_after(four ? mmpd::emb_kernel<T, I, VEC, 4> : mmpd::emb_kernel<T, I, VEC, 1>,
                                     four ? (total + 1023) / 1024 : (total + 255) / 256, 256, 0, 1, w, rows,
                                     emb_div((unsigned)per), w_stride, ids + r, total, (S)scale, out + r * width, err);
    if (rc) return rc;
  }
  return MMP_OK;
}

template <class T, class I>
int run_emb(const void *w, int64_t rows, int64_t width, int64_t w_stride, const void *ids, int64_t n, double scale,
            void *out) {
  return emb_with_vec<T>(emb_vec<T>(w, out, width, w_stride), [&](auto vec) {
    return emb_launch<T, I, decltype(vec)::value>((const T *)w, rows, width, w_stride, (const I *)ids, n, scale, (T *)out);
  });
}

int emb_ids(int ids_dtype, const void *ids, int64_t n, int64_t rows) {
  const int64_t most = (int64_t)mmp::sm_count() * 8, want = (n + 255) / 256;
  const unsigned grid = (unsigned)(want < most ? want : most);
  int *err = mmp::device_error_word();
  if (ids_dtype == MMP_INT32)
    return mmp::launch_after(mmpd::emb_ids_kernel<int>, grid, 256, 0, 1, (const int *)ids, (unsigned)n, rows, err);
  return mmp::launch_after(mmpd::emb_ids_kernel<long long>, grid, 256, 0, 1, (const long long *)ids, (unsigned)n, rows,
                           err);
}

// Device memory of one call, from the stream-ordered pool.
struct EmbBuf {
  void *p = nullptr;
  int alloc(size_t bytes) {
    MMP_CUDA_TRY(cudaMallocAsync(&p, bytes, mmp::stream()));
    return MMP_OK;
  }
  ~EmbBuf() {
    if (p) cudaFreeAsync(p, mmp::stream());
  }
};

template <class T, class I, int VEC>
int emb_few(const I *ids, unsigned n, const T *grad, int64_t g_stride, int64_t rows, int64_t width, double scale,
            int64_t padding, T *out) {
  // a block a token, and eight an SM for the zeros while they have a 64 KB each
  const int64_t most = (int64_t)mmp::sm_count() * 8, want = rows * width * (int64_t)sizeof(T) / 65536 + 1;
  const unsigned zero = (unsigned)(want < most ? want : most);
  return mmp::launch_after(mmpd::emb_grad_few<T, I, VEC>, n + zero, 256, 0, 1, ids, n, grad, g_stride, rows, (unsigned)width,
                           (typename mmpd::EmbAcc<T>::type)scale, padding, out, mmp::device_error_word());
}

// How the sums are shared out.
struct EmbShares {
  unsigned lanes, slices, groups, share, shares;
};
EmbShares emb_shares(unsigned n, int64_t width, int vec) {
  EmbShares r;
  r.lanes = 1;
  while (r.lanes < 256 && r.lanes * vec < width) r.lanes *= 2;
  r.slices = (unsigned)((width + (int64_t)r.lanes * vec - 1) / ((int64_t)r.lanes * vec));
  r.groups = 256 / r.lanes;
  // shares of 32 tokens: fewer where that leaves SMs without blocks, more
  // where it makes more than sixteen blocks an SM (each share may leave two
  // parts to join)
  const unsigned sms = (unsigned)mmp::sm_count();
  r.share = 32;
  auto blocks = [&] { return ((uint64_t)n + r.share - 1) / r.share * r.slices / r.groups; };
  while (r.share > 8 && blocks() < 4u * sms) r.share /= 2;
  while (blocks() > 16u * sms) r.share *= 2;
  r.shares = (n + r.share - 1) / r.share;
  return r;
}

struct EmbSorted {
  unsigned *keys, *order, *runs, *seen;
  mmpd::EmbRun *list;
  void *part;
  unsigned n;
  mmp::EmbZeroPlan zeros;
  EmbShares sh;
};

template <class T, int VEC>
int emb_sum(const EmbSorted &e, const T *grad, int64_t g_stride, int64_t rows, int64_t width, double scale, T *out) {
  typedef typename mmpd::EmbAcc<T>::type S;
  const unsigned n = e.n, lanes = e.sh.lanes, slices = e.sh.slices, groups = e.sh.groups, share = e.sh.share,
                 shares = e.sh.shares;
  // beside them two blocks an SM that write zeros
  const unsigned zeros = e.zeros.first, zeros_end = e.zeros.second, unit = e.zeros.unit;
  auto zero_grid = [&](unsigned from, unsigned to, unsigned most) {
    const uint64_t want = ((uint64_t)(to - from + unit - 1) / unit + 7) / 8;
    return (unsigned)(want < most ? want : most);
  };
  const unsigned zero_blocks = zero_grid(zeros, zeros_end, 2 * (unsigned)mmp::sm_count());
  const int rc = mmp::launch_after(mmpd::emb_sum_kernel<T, VEC>, dim3(zero_blocks + (shares + groups - 1) / groups, slices), 256, 0, 1, e.keys,
                        e.order, n, share, shares, lanes, grad, g_stride, (unsigned)rows, (unsigned)width, (S)scale, out,
                        (S *)e.part, e.runs, e.list, e.seen, zeros, zeros_end, unit, zero_blocks);
  if (rc) return rc;
  constexpr int JV = VEC >= 4 ? 4 : 1;
  const unsigned cols = (unsigned)((width + 32 * JV - 1) / (32 * JV));
  const unsigned join = shares < 128 ? shares : 128, slots = cols < 32 ? cols : 32;
  const unsigned last = zero_grid(zeros_end, (unsigned)rows, (4 * (unsigned)mmp::sm_count() + slots - 1) / slots);
  return mmp::launch_after(mmpd::emb_join_kernel<T, JV>, dim3(join + last, slots), 256, 0, 1, (unsigned)width, (S)scale,
                          (const S *)e.part, e.runs, e.list, out, e.seen, zeros_end, (unsigned)rows, unit, join);
}

template <class T, class I>
int run_emb_grad(const void *ids_, int64_t n, const void *grad_, int64_t g_stride, int64_t rows, int64_t width,
                 double scale, int64_t padding, void *out_) {
  const I *ids = (const I *)ids_;
  const T *grad = (const T *)grad_;
  T *out = (T *)out_;
  const int vec = emb_vec<T>(grad, out, width, g_stride);
  if (n <= mmpd::kEmbFew)
    return emb_with_vec<T>(vec, [&](auto v) {
      return emb_few<T, I, decltype(v)::value>(ids, (unsigned)n, grad, g_stride, rows, width, scale, padding, out);
    });
  int bits = 1;
  while ((INT64_C(1) << bits) <= rows) ++bits;  // the key `rows` included
  int *err = mmp::device_error_word();
  EmbBuf mem;
  EmbSorted e;
  e.n = (unsigned)n;
  e.sh = emb_shares(e.n, width, vec);
  // keys, order (a second time each for sort_pairs), parts, list, then what
  // sort_pairs wants zeroed with them: its state, bitmap, count
  const bool cluster = n <= mmpd::kEmbCluster;
  e.zeros = mmp::emb_zero_plan(rows, width * (int64_t)sizeof(T), cluster);
  const size_t np = ((size_t)n + 7) & ~(size_t)7, words = ((size_t)rows + 31) / 32;
  const size_t parts = (size_t)e.sh.shares * 2 * width * sizeof(typename mmpd::EmbAcc<T>::type);
  const size_t sorted = np * (cluster ? 8 : 16), lists = ((size_t)e.sh.shares * sizeof(mmpd::EmbRun) + 15) / 16 * 16;
  const size_t state = cluster ? 0 : mmp::sort_pairs_state((unsigned)n, bits);
  int rc = mem.alloc(sorted + (parts + 15) / 16 * 16 + lists + state + words * 4 + 16);
  if (rc) return rc;
  e.keys = (unsigned *)mem.p;
  e.order = e.keys + np;
  e.part = (char *)mem.p + sorted;
  e.list = (mmpd::EmbRun *)((char *)e.part + (parts + 15) / 16 * 16);
  char *const zeroed = (char *)e.list + lists;
  e.seen = (unsigned *)(zeroed + state);
  e.runs = e.seen + words;
  if (cluster) {
    const int items = (int)((n + mmpd::kSortThreads * mmpd::kSortRanks - 1) / (mmpd::kSortThreads * mmpd::kSortRanks));
    const int passes = (bits + mmpd::kSortBits - 1) / mmpd::kSortBits, digit = (bits + passes - 1) / passes;
    const int64_t zeros = e.zeros.first, row = width * (int64_t)sizeof(T);
    // one block an SM in clusters of eight, with 64 KB of zeros each at least
    const int64_t all = mmp::sm_count() / mmpd::kSortRanks - 1;
    const int64_t want = zeros * row / (65536 * mmpd::kSortRanks) + 1;
    const unsigned clusters = 1 + (unsigned)(want < all ? want : all);
    const int64_t share = (zeros + (clusters - 1) * mmpd::kSortRanks - 1) / ((clusters - 1) * mmpd::kSortRanks);
    auto bytes = [](int items) { return sizeof(mmpd::EmbSortSmem) + (size_t)items * mmpd::kSortThreads * 16; };
    constexpr size_t kSeen = 65536;  // of bitmap a block at most
    const size_t seen = share < (int64_t)kSeen * 8 ? (size_t)(share + 31) / 32 * 4 : kSeen;
    const size_t smem = bytes(items) < seen ? seen : bytes(items);
    auto fn = mmpd::emb_sort_kernel<T, I>;
    static mmp::SmemLimit limit;
    static_assert(sizeof(mmpd::EmbSortSmem) + mmpd::kSortItems * mmpd::kSortThreads * 16 >= kSeen, "the limit");
    rc = limit.raise(fn, bytes(mmpd::kSortItems));
    if (rc) return rc;
    rc = mmp::launch_after(fn, dim3(clusters * mmpd::kSortRanks), mmpd::kSortThreads, smem, 1, ids, (unsigned)n, rows, padding,
                          items, passes, digit, e.keys, e.order, (unsigned)width, out, (unsigned)zeros, (unsigned)(seen * 8),
                          e.seen, e.runs, err);
    if (rc) return rc;
  } else {
    unsigned *const kb[2] = {e.keys, e.keys + 2 * np}, *const ob[2] = {e.order, e.order + 2 * np};
    MMP_CUDA_TRY(cudaMemsetAsync(zeroed, 0, state + words * 4 + 4, mmp::stream()));
    mmpd::emb_prep_kernel<I><<<mmp::sm_count() * 2, 256, 0, mmp::stream()>>>(ids, (unsigned)n, rows, padding, kb[0],
                                                                             ob[0], e.seen, err);
    MMP_LAUNCH_CHECK("embedding_grad keys");
    int cur = 0;
    rc = mmp::sort_pairs(kb, ob, (unsigned)n, bits, zeroed, &cur);
    if (rc) return rc;
    e.keys = kb[cur];
    e.order = ob[cur];
  }
  return emb_with_vec<T>(
      vec, [&](auto v) { return emb_sum<T, decltype(v)::value>(e, grad, g_stride, rows, width, scale, out); });
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
  if (n == 0) return MMP_OK;
  if (!ids || (width && (!out || (rows && !weight)))) return mmp::set_error(MMP_E_ARG, "embedding: null pointer");
  if (!mmp::device_error_word()) return mmp::set_error(MMP_E_CUDA, "no CUDA device available");
  if (width == 0) return emb_ids(ids_dtype, ids, n, rows);
  MMP_EMB_DISPATCH(run_emb, weight, rows, width, w_stride, ids, n, scale, out);
}

int mmp_embedding_grad(int dtype, int ids_dtype, const void *ids, int64_t n, const void *grad, int64_t g_stride,
                       int64_t rows, int64_t width, double scale, int64_t padding_idx, void *grad_weight) {
  int rc = emb_check("embedding_grad", dtype, ids_dtype, rows, width, n);
  if (rc) return rc;
  const bool empty = rows == 0 || width == 0;
  if (empty && n == 0) return MMP_OK;
  if ((n && !ids) || (!empty && ((n && !grad) || !grad_weight)))
    return mmp::set_error(MMP_E_ARG, "embedding_grad: null pointer");
  if (!mmp::device_error_word()) return mmp::set_error(MMP_E_CUDA, "no CUDA device available");
  if (empty) return emb_ids(ids_dtype, ids, n, rows);
  MMP_EMB_DISPATCH(run_emb_grad, ids, n, grad, g_stride, rows, width, scale, padding_idx, grad_weight);
}

}  // extern "C"
