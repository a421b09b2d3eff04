// Kernels of one call that follow one another in a stream: the next one's CTAs may start, and
// do what does not depend on the one before, while that one's last CTAs still run.  It saves 1 to 3 us a
// launch (the eight of a training step of 4 x 1900 tokens x 6 heads of 128: 163 -> 148 us).
#pragma once
#include <cuda_runtime.h>

namespace atlas {

// In the earlier kernel: the next one's CTAs may take the places that become free (they do
// once every CTA of this kernel has come here or has ended).  A kernel that allocates tensor
// memory comes here after that: a waiting CTA of the next kernel keeps what it has allocated.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// In a kernel launched with follow(): waits until the kernel before it has ended and its writes
// are visible.  Every CTA waits before it reads anything that an earlier kernel of the call writes, and
// before it writes anything that one of them reads; each kernel that follows has to call this, so that
// the end of one is also the end of all before it.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <class... P, class... A>
cudaError_t follow(void (*kernel)(P...), unsigned grid, unsigned block, size_t smem, cudaStream_t stream, A&&... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(block);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  c.attrs = &at;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}

}  // namespace atlas
