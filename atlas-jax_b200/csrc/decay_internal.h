// Shared by the decay attention kernels (decay_attn.cu, decay_tc.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "atlas_decay.h"
#include "scan_internal.h"

namespace atlas {
namespace decay {

constexpr int CH = 128;  // tokens of a chunk: a state is kept for each, on every path

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

// tcgen05 path (decay_tc.cu): bf16, D a multiple of 8, 16-byte aligned rows.
namespace tc {
// Per-chunk state sums into a.states (fwd: sum l^(L-1-s) k_s v_s^T) or a.dstates
// (bwd: scale * sum l^(t+1) q_t dy_t^T).
cudaError_t launch_chunk_states(const Args& a, bool bwd, cudaStream_t s);
cudaError_t launch_out(const Args& a, cudaStream_t s);
cudaError_t launch_grads(const Args& a, cudaStream_t s);
}  // namespace tc

}  // namespace decay
}  // namespace atlas
