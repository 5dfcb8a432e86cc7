// Kernels that follow one another on the library stream: a kernel launched by
// launch_after may be set up while the one before it in the stream ends.  It
// calls chain_wait before it touches memory, which waits until that one is
// done and its writes are there, and chain_next to let the one behind it be
// set up in turn.  Its inputs are no `const __restrict__`, which would promise
// the compiler that nothing writes them while the kernel runs.
#pragma once
#include <cuda_runtime.h>

#include <atomic>

#include "mmp_internal.h"

namespace mmpd {

__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace mmpd

namespace mmp {

// `ranks`: blocks a cluster (1: none, or the kernel's own).
template <class... P, class... A>
int launch_after(void (*fn)(P...), dim3 grid, dim3 block, size_t smem, int ranks, const A &...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream();
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)ranks;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = ranks > 1 ? 2 : 1;
  MMP_CUDA_TRY(cudaLaunchKernelEx(&cfg, fn, P(args)...));
  return MMP_OK;
}

// A kernel's limit of dynamic shared memory, raised once per device to the most
// that any of its launches asks for.  (A limit set to each call's own size
// could be lowered by another thread between that and the launch.)  One
// object per kernel.
struct SmemLimit {
  std::atomic<bool> set[64];
  template <class... P>
  int raise(void (*fn)(P...), size_t most) {
    const int dev = current_device();
    if (dev < 0 || dev >= 64) return set_error(MMP_E_ARG, "device out of range");
    if (!set[dev].load(std::memory_order_acquire)) {
      MMP_CUDA_TRY(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
      set[dev].store(true, std::memory_order_release);
    }
    return MMP_OK;
  }
};

}  // namespace mmp
