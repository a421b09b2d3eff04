// Shared by the tcgen05 kernels of decay attention (decay_scan.cu, decay_grad.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cudaTypedefs.h>

#include "common.cuh"
#include "decay_internal.h"
#include "f32x2.cuh"
#include "tc_ops.cuh"

namespace atlas {
namespace decay {
namespace tcore {

using namespace tcx;
typedef __nv_bfloat16 bf16;

constexpr int C = CH;  // tokens of a block
constexpr int BOX = C * 128;  // bytes of a TMA box: 64 tokens x 64 channels

// ---- PTX ----
__device__ __forceinline__ void arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tma_load(void* dst, const CUtensorMap* map, int x, int h, int t, int b, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(h), "r"(t), "r"(b), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int x, int h, int t, int b, const void* src) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(map),
               "r"(x), "r"(h), "r"(t), "r"(b), "r"(smem_u32(src))
               : "memory");
}
// a box into L2 ahead of its load
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* map, int x, int h, int t, int b) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(map), "r"(x), "r"(h),
               "r"(t), "r"(b)
               : "memory");
}
// 16 lanes x 16 or 32 columns: v[4 j + 2 i + k] = row lane / 4 + 8 i, column 8 j + 2 (lane % 4) + k
__device__ __forceinline__ void tmem_frag16(uint32_t addr, float* v) {
  uint32_t* r = (uint32_t*)v;
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_frag32(uint32_t addr, float* v) {
  uint32_t* r = (uint32_t*)v;
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
// K-major operand of a TMA tile (64 channels of K a box); 16 channels on: +32 bytes
__device__ __forceinline__ uint64_t desc_tile(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// MN-major operand of a TMA tile (tokens are K, a box per 64 channels of N); 16 tokens on: +2048 bytes
__device__ __forceinline__ uint64_t desc_tile_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(BOX >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// Eight float32 values as three bf16 parts whose sum holds all 24 bits, 16-byte groups `stride`
// apart.  The upper parts are cut off, not rounded: 8 bits each leave 8 for the last (and the
// kernels run as fast as with rounding conversions).
__device__ __forceinline__ void put_parts3(uint8_t* dst, uint32_t stride, F2* v) {
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    uint4 pk;
    uint32_t* h = (uint32_t*)&pk;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[j] = bf2_cut(v[j]);
      if (p < 2) v[j] = v[j] - bf2_unpack(h[j]);
    }
    *(uint4*)(dst + p * stride) = pk;
  }
}
__device__ __forceinline__ float powd(float g, int n) { return n == 0 ? 1.f : expf((float)n * g); }

// The tensor map of (B, T, H, D) bf16 activations with element strides s (batch, token,
// head); false where the driver refuses it (decay_scan.cu).
bool make_map(CUtensorMap* m, const void* x, const AtlasDecayParams& p, const int64_t* s);

}  // namespace tcore
}  // namespace decay
}  // namespace atlas
