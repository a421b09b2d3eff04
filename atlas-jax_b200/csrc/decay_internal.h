// Shared by the decay attention kernels (decay_attn.cu, decay_scan.cu, decay_grad.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "atlas_decay.h"
#include "follow.cuh"
#include "scan_internal.h"

namespace atlas {
namespace decay {

constexpr int CH = 64;  // tokens of a chunk: a state is kept for each, on every path

struct Args {
  AtlasDecayParams p;
  const void *q, *k, *v, *dy;
  const float* log_decay;
  void *y, *dq, *dk, *dv;
  float* states;   // (B * H, chunks, D, D): the state entering each chunk
  float* dstates;  // the same shape: the cotangent of the state leaving each chunk
  float* dg_part;  // (B * H, dg_parts): partial sums of dlog_decay
  int dg_parts;
  int* status;
};

__host__ __device__ inline int chunks(const AtlasDecayParams& p) { return (p.T + CH - 1) / CH; }  // T <= 2^30
__host__ __device__ inline int64_t chains(const AtlasDecayParams& p) { return (int64_t)p.B * p.H; }
__host__ __device__ inline int chunk_len(const AtlasDecayParams& p, int c) {
  const int left = p.T - c * CH;
  return left < CH ? left : CH;
}

// Lets a kernel use `bytes` of dynamic shared memory; asked of the driver once per device.
template <auto Kernel>
cudaError_t allow_smem(size_t bytes) {
  static DeviceCache done;
  cudaError_t e = cudaSuccess;
  done.get([&] {
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == cudaSuccess ? 0 : -1;
  });
  return e;
}

// tcgen05 path: bf16, D a multiple of 8, 16-byte aligned rows.
namespace tcore {
bool mappable(const AtlasDecayParams& p, const int64_t* strides);  // whether TMA can address such a tensor
// The walk along the sequences (decay_scan.cu): forward y and states, or (bwd) the cotangent
// states.  saves: (chains, chunks, D, D), the state entering every chunk in the order of the
// walk, or NULL.  sums: sums_bytes() of scratch.
size_t sums_bytes(const AtlasDecayParams& p, bool bwd);
cudaError_t launch_seq(const Args& a, bool bwd, const float* in, float* out, float* saves, float* sums,
                       cudaStream_t s);
// dq, dk, dv and the parts of dlog_decay, chunk by chunk, from a.states and a.dstates (decay_grad.cu)
cudaError_t launch_grads(const Args& a, cudaStream_t s);
}  // namespace tcore

}  // namespace decay
}  // namespace atlas
