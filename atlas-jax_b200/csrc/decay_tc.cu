// Decay attention (include/atlas_decay.h): the gradients of q, k and v on the tcgen05 tensor
// cores.  bf16 activations, D a multiple of 8 up to 128 (zero-padded to DP = 64 or 128
// channels in shared memory).
//
// One CTA owns one 128-token chunk of one (batch, head); the states between chunks come
// from the walks along the sequence (decay_scan.cu), so chunks are independent here.  Operand tiles are bf16 in the core-matrix layout of tc_ops.cuh, which
// serves as K-major and as MN-major operand, so no tile is transposed; accumulators are
// float32 in TMEM.
//
// Precision.  Products of two bf16 inputs are exact in float32.  A float32 operand (a
// state, or k and q times their decay) is split into bf16 parts whose sum holds 24 bits
// (three parts) where a float32 output depends on it, and 16 bits (two parts) where only
// bf16 outputs do.  The smaller parts are accumulated first: the tensor core truncates each
// accumulation step to the accumulator's exponent, so it is the steps after the leading
// part that cost bits.  The decayed scores are rounded once to bf16.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "decay_internal.h"
#include "scan_internal.h"
#include "tc_ops.cuh"

namespace atlas {
namespace decay {
namespace tcore {

using namespace tcx;
typedef __nv_bfloat16 bf16;

template <int DP>
constexpr int TILE = CH * DP * 2;  // bytes of a 128-token tile
template <int DP>
constexpr int STILE = DP * DP * 2;       // bytes of one part of a state
constexpr int PTILE = CH * CH * 2;       // bytes of a tile of scores

__device__ __forceinline__ uint8_t* align128(uint8_t* p) {
  return (uint8_t*)(((uintptr_t)p + 127) & ~(uintptr_t)127);
}
__device__ __forceinline__ void cp_async16(void* sdst, const void* gsrc) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(sdst)), "l"(gsrc) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ void cta_sync() {
  fence_before();
  __syncthreads();
  fence_after();
}

// Copies rows [t0, t0 + L) of a head (row r at x + r * st) into a 128 x DP core-matrix
// tile, zero beyond L rows and D channels.  Lanes run along the 8 rows of a core matrix
// first: a warp writes 512 consecutive bytes and reads 64 of each of 8 rows.
template <int DP>
__device__ void load_tile(uint8_t* tile, const bf16* x, int64_t st, int L, int D) {
  for (int u = threadIdx.x; u < CH * DP / 8; u += blockDim.x) {
    const int r = (u & 7) | (u / DP << 3), c = ((u >> 3) % (DP / 8)) * 8;
    if (r < L && c < D)
      cp_async16(tile + u * 16, x + r * st + c);
    else
      *(uint4*)(tile + u * 16) = make_uint4(0, 0, 0, 0);
  }
}

// Splits 8 float32 values into NP bf16 parts (each the rounding of what the ones before
// left) and stores them as 16-byte groups `stride` bytes apart.
template <int NP>
__device__ __forceinline__ void store_parts(uint8_t* dst, uint32_t stride, float* v) {
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    uint4 pk;
    __nv_bfloat162* h = (__nv_bfloat162*)&pk;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      if (p + 1 < NP) {
        const float2 f = __bfloat1622float2(h[j]);
        v[2 * j] -= f.x;
        v[2 * j + 1] -= f.y;
      }
    }
    *(uint4*)(dst + p * stride) = pk;
  }
}

// A float32 D x D state into NP parts, DP x DP tiles (row = key channel) STILE apart.
template <int DP, int NP>
__device__ void load_state(uint8_t* dst, const float* S, int D) {
  for (int u = threadIdx.x; u < DP * DP / 8; u += blockDim.x) {
    const int d = (u & 7) | (u / DP << 3), e = ((u >> 3) % (DP / 8)) * 8;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (d < D && e < D) {
      *(float4*)v = *(const float4*)(S + (int64_t)d * D + e);
      *(float4*)(v + 4) = *(const float4*)(S + (int64_t)d * D + e + 4);
    }
    store_parts<NP>(dst + u * 16, STILE<DP>, v);
  }
}

// D (+)= A B over K, issued by one warp.  A: M x K (a tile of a_cols columns whose rows are
// the M index, or with a_mn the K index); B likewise with N.
__device__ __forceinline__ void mma(uint32_t tmd, const uint8_t* A, int a_cols, bool a_mn, const uint8_t* B,
                                    int b_cols, bool b_mn, int M, int N, int K, bool accumulate) {
  const uint32_t id = idesc_bf16(M, N, a_mn, b_mn);
  const uint32_t sa = a_mn ? (uint32_t)a_cols * 32 : 256, sb = b_mn ? (uint32_t)b_cols * 32 : 256;
  for (int ks = 0; ks < K / 16; ++ks) {
    const uint32_t pa = smem_u32(A) + ks * sa, pb = smem_u32(B) + ks * sb;
    mma_kf16(tmd, a_mn ? desc_mnmajor(pa, a_cols) : desc_kmajor(pa, a_cols),
             b_mn ? desc_mnmajor(pb, b_cols) : desc_kmajor(pb, b_cols), id, (accumulate || ks) ? 1u : 0u);
  }
}

struct Ctl {
  float pw[CH + 1];  // decay^n
  float red[16];
  uint64_t bar;
  uint32_t tmem;
  volatile int bad;
};

// every thread waits for the committed MMAs (bounded); false after a timeout, uniformly
__device__ __forceinline__ bool wait_mma(Ctl& c, uint32_t& phase, int* status) {
  const bool ok = c.bad || mbar_wait(&c.bar, phase);
  phase ^= 1;
  if (!ok) {
    set_status(status, ATLAS_ERR_DEVICE_TIMEOUT);
    c.bad = 1;
  }
  cta_sync();
  return !c.bad;
}

// TMEM allocation, barrier, the table of decay powers
__device__ __forceinline__ void setup(Ctl& c, uint32_t cols, float g) {
  const int tid = threadIdx.x;
  if (tid < 32) {
    tmem_alloc(&c.tmem, cols);
    tmem_relinquish();
  }
  if (tid == 0) {
    mbar_init(&c.bar, 1);
    fence_mbar_init();
    c.bad = 0;
  }
  for (int n = tid; n <= CH; n += blockDim.x) c.pw[n] = n == 0 ? 1.f : expf((float)n * g);
}

struct Pos {
  int64_t chain, chunk_index;
  int b, h, c, L, t0;
};
__device__ __forceinline__ Pos position(const AtlasDecayParams& P) {
  Pos z;
  const int nc = chunks(P);
  z.chunk_index = blockIdx.x;
  z.chain = blockIdx.x / nc;
  z.c = (int)(blockIdx.x % nc);
  z.b = (int)(z.chain / P.H);
  z.h = (int)(z.chain % P.H);
  z.L = chunk_len(P, z.c);
  z.t0 = z.c * CH;
  return z;
}
__device__ __forceinline__ const bf16* head(const void* x, const int64_t* s, const Pos& z) {
  return (const bf16*)x + z.b * s[0] + (int64_t)z.t0 * s[1] + z.h * s[2];
}
__device__ __forceinline__ int64_t flat_row(const AtlasDecayParams& P, const Pos& z, int r) {
  return (((int64_t)z.b * P.T + z.t0 + r) * P.H + z.h) * P.D;
}

// n consecutive TMEM columns (a multiple of 16) of this warp's lane quadrant
template <int n>
__device__ __forceinline__ void tmem_ld(uint32_t addr, float* v) {
#pragma unroll
  for (int j = 0; j < n; j += 16) tmem_ld16(addr + j, v + j);
  tmem_wait_ld();
}

// this thread's n columns from c0 of an output row, bf16; columns from D on are padding
template <int n>
__device__ __forceinline__ void store_row(bf16* row, int c0, int D, const float* v) {
#pragma unroll
  for (int g = 0; g < n / 8; ++g) {
    if (c0 + 8 * g >= D) break;
    uint4 pk;
    __nv_bfloat162* h = (__nv_bfloat162*)&pk;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[8 * g + 2 * j], v[8 * g + 2 * j + 1]);
    *(uint4*)(row + c0 + 8 * g) = pk;
  }
}
__device__ __forceinline__ void store8(uint8_t* dst, const float* v) {
  uint4 pk;
  __nv_bfloat162* h = (__nv_bfloat162*)&pk;
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
  *(uint4*)dst = pk;
}

// ---------------------------------------------------------------------------
// gradients
// ---------------------------------------------------------------------------
// 16 warps: warp w reads lane quadrant w % 4, column quarter w / 4.  TMEM: A = Q K^T in
// columns 0-127, O V^T in 128-255 (O = dy), and the products of DP columns with the states
// from 256 on.  The region R holds in turn the three parts of S, those of the cotangent
// state, and the two tiles of decayed scores.
template <int DP>
__device__ __forceinline__ float dot_tile(const uint8_t* tile, int r, int c0, const float* v) {
  float s = 0.f;
#pragma unroll
  for (int g = 0; g < DP / 32; ++g) {  // DP / 4 columns in groups of 8
    const uint4 pk = *(const uint4*)(tile + cm_off(r, c0 + 8 * g, DP));
    const __nv_bfloat162* h = (const __nv_bfloat162*)&pk;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __bfloat1622float2(h[j]);
      s = fmaf(f.x, v[8 * g + 2 * j], fmaf(f.y, v[8 * g + 2 * j + 1], s));
    }
  }
  return s;
}

template <int DP>
__global__ void __launch_bounds__(512, 1) grads_kernel(Args a) {
  extern __shared__ uint8_t raw[];
  constexpr int RB = 3 * STILE<DP> > 2 * PTILE ? 3 * STILE<DP> : 2 * PTILE;
  constexpr int NC = DP / 4;  // columns of an output row that a thread holds
  constexpr uint32_t X0 = 256, X1 = 256 + DP, X2 = DP == 64 ? 384 : 256;
  uint8_t* Q = align128(raw);
  uint8_t* K = Q + TILE<DP>;
  uint8_t* V = K + TILE<DP>;
  uint8_t* O = V + TILE<DP>;
  uint8_t* R = O + TILE<DP>;
  Ctl& ctl = *(Ctl*)(R + RB);
  const AtlasDecayParams& P = a.p;
  const Pos z = position(P);
  const int D = P.D, w = threadIdx.x >> 5, qd = w & 3, cq = w >> 2, t = 32 * qd + (threadIdx.x & 31);
  const int c0 = cq * NC;
  const int64_t so = z.chunk_index * (int64_t)D * D;
  load_tile<DP>(Q, head(a.q, P.q_stride, z), P.q_stride[1], z.L, D);
  load_tile<DP>(K, head(a.k, P.k_stride, z), P.k_stride[1], z.L, D);
  load_tile<DP>(V, head(a.v, P.v_stride, z), P.v_stride[1], z.L, D);
  load_tile<DP>(O, (const bf16*)a.dy + flat_row(P, z, 0), (int64_t)P.H * D, z.L, D);
  load_state<DP, 3>(R, a.states + so, D);
  setup(ctl, 512, a.log_decay[z.h]);
  cp_async_wait_all();
  fence_async_smem();
  cta_sync();
  const uint32_t tm = ctl.tmem, lane = (uint32_t)(32 * qd) << 16;
  uint32_t phase = 0;
  float dq[NC], dk[NC], dv[NC], dg = 0.f;
  if (w == 0) {
    for (int p = 2; p >= 0; --p)
      mma(tm + X0, O, DP, false, R + p * STILE<DP>, DP, false, CH, DP, DP, p < 2);  // O S^T
    mma(tm, Q, DP, false, K, DP, false, CH, CH, DP, false);
    mma(tm + 128, O, DP, false, V, DP, false, CH, CH, DP, false);
    mma_commit(&ctl.bar);
  }
  __syncwarp();
  bool ok = wait_mma(ctl, phase, a.status);
  if (ok) {
    tmem_ld<NC>(tm + lane + X0 + c0, dq);
    const float wi = P.scale * ctl.pw[t + 1];
#pragma unroll
    for (int j = 0; j < NC; ++j) dq[j] *= wi;
    dg += (float)(t + 1) * dot_tile<DP>(Q, t, c0, dq);
    load_state<DP, 3>(R, a.dstates + so, D);
    {  // L l^L <R, S> of the chunk
      float rs = 0.f;
      for (int u = threadIdx.x; u < D * D / 4; u += 512) {
        const float4 x = *(const float4*)(a.states + so + 4 * u), y = *(const float4*)(a.dstates + so + 4 * u);
        rs += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
      }
      dg += (float)z.L * ctl.pw[z.L] * rs;
    }
    fence_async_smem();
    cta_sync();
    if (w == 0) {
      for (int p = 2; p >= 0; --p)
        mma(tm + X1, V, DP, false, R + p * STILE<DP>, DP, false, CH, DP, DP, p < 2);  // V R^T
      for (int p = 1; p >= 0; --p)
        mma(tm + X2, K, DP, false, R + p * STILE<DP>, DP, true, CH, DP, DP, p < 1);   // K R
      mma_commit(&ctl.bar);
    }
    __syncwarp();
    ok = wait_mma(ctl, phase, a.status);
  }
  if (ok) {
    const float wo = t < z.L ? ctl.pw[z.L - 1 - t] : 0.f;
    tmem_ld<NC>(tm + lane + X1 + c0, dk);
    tmem_ld<NC>(tm + lane + X2 + c0, dv);
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      dk[j] *= wo;
      dv[j] *= wo;
    }
    if (t < z.L) dg += (float)(z.L - 1 - t) * dot_tile<DP>(K, t, c0, dk);
    // scores: P = scale l^(t-s) A into R, scale l^(t-s) O V^T behind it
#pragma unroll
    for (int cb = 0; cb < 32; cb += 16) {
      const int s0 = 32 * cq + cb;
      float p[16], x[16];
      tmem_ld<16>(tm + lane + s0, p);
      tmem_ld<16>(tm + lane + 128 + s0, x);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int lag = t - s0 - j;
        const float f = P.scale * ctl.pw[max(lag, 0)];
        x[j] = lag >= 0 ? f * x[j] : 0.f;
        dg = lag > 0 ? fmaf((float)lag * p[j], x[j], dg) : dg;
        p[j] = lag >= 0 ? f * p[j] : 0.f;
      }
      store8(R + cm_off(t, s0, CH), p);
      store8(R + cm_off(t, s0 + 8, CH), p + 8);
      store8(R + PTILE + cm_off(t, s0, CH), x);
      store8(R + PTILE + cm_off(t, s0 + 8, CH), x + 8);
    }
    fence_async_smem();
    cta_sync();
    if (w == 0) {
      mma(tm + X0, R + PTILE, CH, false, K, DP, true, CH, DP, CH, false);  // dq += dA K
      mma(tm + X1, R + PTILE, CH, true, Q, DP, true, CH, DP, CH, false);   // dk += dA^T Q
      mma(tm, R, CH, true, O, DP, true, CH, DP, CH, false);                // dv += P^T O
      mma_commit(&ctl.bar);
    }
    __syncwarp();
    ok = wait_mma(ctl, phase, a.status);
  }
  if (ok) {
    const int64_t row = flat_row(P, z, t);
    float v[NC];
    tmem_ld<NC>(tm + lane + X0 + c0, v);
#pragma unroll
    for (int j = 0; j < NC; ++j) v[j] += dq[j];
    if (t < z.L) store_row<NC>((bf16*)a.dq + row, c0, D, v);
    tmem_ld<NC>(tm + lane + X1 + c0, v);
#pragma unroll
    for (int j = 0; j < NC; ++j) v[j] += dk[j];
    if (t < z.L) store_row<NC>((bf16*)a.dk + row, c0, D, v);
    tmem_ld<NC>(tm + lane + c0, v);
#pragma unroll
    for (int j = 0; j < NC; ++j) v[j] += dv[j];
    if (t < z.L) store_row<NC>((bf16*)a.dv + row, c0, D, v);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dg += __shfl_xor_sync(0xffffffffu, dg, o);
    if ((threadIdx.x & 31) == 0) ctl.red[w] = dg;
    cta_sync();
    if (threadIdx.x == 0) {
      float s = 0.f;
      for (int i = 0; i < 16; ++i) s += ctl.red[i];
      a.dg_part[z.chunk_index] = s;
    }
  }
  cta_sync();
  if (w == 0) tmem_dealloc(tm, 512);
}

// ---------------------------------------------------------------------------

static unsigned grid(const Args& a) { return (unsigned)(chains(a.p) * chunks(a.p)); }

template <int DP>
static cudaError_t grads(const Args& a, cudaStream_t s) {
  const size_t sm = 4 * TILE<DP> + std::max(3 * STILE<DP>, 2 * PTILE) + sizeof(Ctl) + 128;
  cudaError_t e = allow_smem<grads_kernel<DP>>(sm);
  if (e != cudaSuccess) return e;
  grads_kernel<DP><<<grid(a), 512, sm, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_grads(const Args& a, cudaStream_t s) { return a.p.D <= 64 ? grads<64>(a, s) : grads<128>(a, s); }

}  // namespace tcore
}  // namespace decay
}  // namespace atlas
