// Decay attention (include/atlas_decay.h): the gradients of q, k and v and the parts of
// dlog_decay on the tcgen05 tensor cores, from the states that the walks along the sequence
// keep in front of every block (decay_scan.cu).  With O = dy, S the state entering a block
// of L <= 64 tokens, R the cotangent of the state leaving it, M_ts = l^(t-s) for s <= t:
//
//     A = Q K^T,  P = M o A,  B = O V^T,  dA = M o B
//     dq = scale (dA K + l^(t+1) O S^T)
//     dk = scale dA^T Q + l^(L-1-s) V R^T
//     dv = scale P^T O + l^(L-1-s) K R
//     dlog_decay += scale sum (t-s) A dA + sum (t+1) q . dq_S + sum (L-1-s) k . dk_R + L l^L <R, S>
//     (dq_S, dk_R: the terms with S and R)
//
// Blocks are independent: one CTA each.  q, k, v, dy arrive by TMA and leave as dq, dk, dv
// through the same tiles (straight from registers: no faster); S and R are split into three bf16 parts
// (dlog_decay is a float32 output; K R reads two of R's, 16 bits, since dv rounds to bf16's 8).  P and dA
// are rounded to bf16 as operands of dq, dk and dv, whose relative error goes from the 1.66e-3 of
// their own rounding to 1.8e-3; dlog_decay takes A and dA from before that rounding.  All accumulators
// have M = 64 (decay_tc.cuh); warp w reads lane quadrant w % 4 and its half (D <= 64) or quarter w / 4 of the
// columns.
//
// D <= 64: 256 TMEM columns (dA K, P^T O, dA^T Q and K R take the places of A, B, O S^T and
// V R^T), 97 KB of shared memory: two CTAs share an SM, and one's loads and float32 work
// run during the other's MMAs.  D <= 128: the parts of S and R take turns in one region and
// K R has columns of its own; one CTA an SM.
//
// What bounds it: the latency of one block's steps (loads, splits, five groups of MMAs, stores: about
// 13,000 cycles at D = 64, 22,000 at D = 128) with two blocks or one in flight an SM; the tensor pipe is
// busy for a fifth of the time, the schedulers for 29 % (D = 64) and 23 %.  Measured: 16 x 4096 tokens x 8 heads of 64 about
// 200 us (88 KB a block: 3.6 TB/s); 4 x 1900 x 6 heads of 128 67 us.  A CTA an SM that walks over the blocks, the next
// one's tiles on their way (D = 64) or its state in registers (D = 128), took as long.
#include <algorithm>

#include "decay_tc.cuh"

namespace atlas {
namespace decay {
namespace tcore {

template <int DP>
struct GCfg {
  // Threads, and warps of a TMEM lane quadrant, with 1 / HF of the columns each.  (D = 64 with 512: 16 x
  // 4096 tokens x 8 heads 5 us longer; D = 128 with 256: 4 x 1900 x 6 2 us longer.)
  static constexpr int NT = DP == 64 ? 256 : 512, HF = NT / 128;
  static constexpr int NB = DP / 64, TILE = NB * BOX, ST = DP * DP * 2, PT = C * C * 2;
  static constexpr int OFF_PARTS = 4 * TILE;
  static constexpr int OFF_P = OFF_PARTS + (DP == 64 ? 6 : 3) * ST;
  static constexpr int OFF_CTL = OFF_P + 2 * PT;
  // TMEM columns of A, B and the products with S and R, and of those that take their places
  static constexpr uint32_t COLS = DP == 64 ? 256 : 512;
  static constexpr uint32_t T_A = 0, T_B = 64, T_OS = 128, T_VR = 128 + DP;
  static constexpr uint32_t T_DQ = DP == 64 ? 0 : 128, T_DV = DP == 64 ? 64 : 0, T_DK = DP == 64 ? 128 : 256,
                            T_KR = DP == 64 ? 192 : 384;
};
struct GCtl {
  float pw[C + 1];
  float red[16];  // a warp's part of dlog_decay
  uint64_t loaded, done[5];
  uint32_t tmem;
  volatile int bad;
};
template <int DP>
constexpr size_t GRAD_SMEM = GCfg<DP>::OFF_CTL + sizeof(GCtl) + 1024;

struct Maps {
  CUtensorMap q, k, v, o, dq, dk, dv;
};

__device__ __forceinline__ void cta_sync() {
  fence_before();
  __syncthreads();
  fence_after();
}
// Waits (bounded).  After a timeout the CTA goes through its remaining steps without waiting
// and stores nothing.
__device__ __forceinline__ void wait_for(GCtl& c, uint64_t* bar, int* status) {
  if (!c.bad && !mbar_wait(bar, 0, 4000000u)) {
    set_status(status, ATLAS_ERR_DEVICE_TIMEOUT);
    c.bad = 1;
  }
  fence_after();
}
// one warp: D (+)= A B, descriptors stepping by sa and sb per 16 of K
template <int N>
__device__ __forceinline__ void mma_steps(uint32_t d, uint64_t A, uint64_t sa, uint64_t B, uint64_t sb, uint32_t id,
                                          bool accumulate) {
#pragma unroll
  for (int k = 0; k < N; ++k) mma_kf16(d, A + k * sa, B + k * sb, id, accumulate || k > 0);
}
template <int NV>
__device__ __forceinline__ void frag(uint32_t addr, float* v) {
  static_assert(NV == 8 || NV == 16, "fragments of 16 or 32 columns");
  if constexpr (NV == 8)
    tmem_frag16(addr, v);
  else
    tmem_frag32(addr, v);
}

template <int DP>
__global__ void __launch_bounds__(GCfg<DP>::NT, DP == 64 ? 2 : 1) grads_kernel(const __grid_constant__ Maps maps, const Args a) {
  using G = GCfg<DP>;
  constexpr int NT = G::NT, CW = DP / G::HF, SC = C / G::HF;  // columns of a warp, of outputs and of scores
  constexpr int NV = CW / 2;                                 // values of a thread's fragment: 2 rows x CW / 4 columns
  extern __shared__ uint8_t raw[];
  uint8_t* sm = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  GCtl& ctl = *(GCtl*)(sm + G::OFF_CTL);
  const AtlasDecayParams& P = a.p;
  const int tid = threadIdx.x, w = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, D = P.D;
  const int nc = chunks(P);
  const int64_t chain = blockIdx.x / nc;
  const int c = (int)(blockIdx.x % nc), b = (int)(chain / P.H), h = (int)(chain % P.H), L = chunk_len(P, c);
  const int q = w & 3, hf = w >> 2, r = lane >> 2, c2 = 2 * (lane & 3), t0 = 16 * q + r;
  const float g = a.log_decay[h];
  const uint32_t base = smem_u32(sm);
  // S and R (float32, D x D) -> three parts each; <R, S>.  Their loads go out first.
  const float* Sg = a.states + (int64_t)blockIdx.x * D * D;
  const float* Rg = a.dstates + (int64_t)blockIdx.x * D * D;
  float rs = 0.f;
  auto load8 = [&](const float* M, int u, F2* v) {
    const int d = (u & 7) | (u / DP << 3), e = ((u >> 3) % (DP / 8)) * 8;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
    if (d < D && e < D) {
      x = *(const float4*)(M + d * D + e);
      y = *(const float4*)(M + d * D + e + 4);
    }
    v[0] = f2(x.x, x.y), v[1] = f2(x.z, x.w), v[2] = f2(y.x, y.y), v[3] = f2(y.z, y.w);
  };
  auto dot8 = [&](const F2* x, const F2* y) {
    const F2 s = fma2(x[0], y[0], fma2(x[1], y[1], fma2(x[2], y[2], x[3] * y[3])));
    const float2 t = f2_get(s);
    rs += t.x + t.y;
  };
  uint8_t* parts = sm + G::OFF_PARTS;
  constexpr int NU = DP * DP / 8 / NT;  // groups of 8 of a state a thread
  F2 x[NU][4], y[NU][4];
#pragma unroll
  for (int i = 0; i < NU; ++i) load8(Sg, tid + NT * i, x[i]);
  if (tid == 0) {
    mbar_init(&ctl.loaded, 1);
    for (int i = 0; i < 5; ++i) mbar_init(&ctl.done[i], 1);
    fence_mbar_init();
    ctl.bad = 0;
    const int nbox = D > 64 ? 2 : 1;
    mbar_expect_tx(&ctl.loaded, (uint32_t)(4 * nbox * BOX));
    for (int i = 0; i < nbox; ++i) {
      tma_load(sm + i * BOX, &maps.q, 64 * i, h, c * C, b, &ctl.loaded);
      tma_load(sm + G::TILE + i * BOX, &maps.k, 64 * i, h, c * C, b, &ctl.loaded);
      tma_load(sm + 2 * G::TILE + i * BOX, &maps.v, 64 * i, h, c * C, b, &ctl.loaded);
      tma_load(sm + 3 * G::TILE + i * BOX, &maps.o, 64 * i, h, c * C, b, &ctl.loaded);
    }
  }
  // Into L2 for the CTA that will run here next: with its data on the way already, a CTA's first
  // phase is short (two CTAs an SM hide only part of it).
  const int64_t nb = (int64_t)blockIdx.x + (DP == 64 ? 2 : 1) * 148;
  if (tid == 64 && nb < gridDim.x) {
    const int64_t nchain = nb / nc;
    const int nt = (int)(nb % nc) * C, nbat = (int)(nchain / P.H), nh = (int)(nchain % P.H);
    for (int i = 0; i < (D > 64 ? 2 : 1); ++i) {
      tma_prefetch(&maps.q, 64 * i, nh, nt, nbat);
      tma_prefetch(&maps.k, 64 * i, nh, nt, nbat);
      tma_prefetch(&maps.v, 64 * i, nh, nt, nbat);
      tma_prefetch(&maps.o, 64 * i, nh, nt, nbat);
    }
    bulk_prefetch_l2(a.states + nb * D * D, D * D * 4);
    bulk_prefetch_l2(a.dstates + nb * D * D, D * D * 4);
  }
  if (w == 1) {
    tmem_alloc(&ctl.tmem, G::COLS);
    tmem_relinquish();
  }
  if (tid >= 64 && tid <= 64 + C) ctl.pw[tid - 64] = powd(g, tid - 64);

  after_previous();  // R: loaded while S is split
#pragma unroll
  for (int i = 0; i < NU; ++i) load8(Rg, tid + NT * i, y[i]);
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    if (DP == 64) dot8(x[i], y[i]);
    F2 t[4] = {x[i][0], x[i][1], x[i][2], x[i][3]};
    put_parts3(parts + (tid + NT * i) * 16, G::ST, t);
  }
  if (DP == 64) {
#pragma unroll
    for (int i = 0; i < NU; ++i) put_parts3(parts + 3 * G::ST + (tid + NT * i) * 16, G::ST, y[i]);
  }
  fence_async_smem();
  cta_sync();
  let_next_start();  // (after the allocation of tensor memory)
  const uint32_t tm = ctl.tmem, tmu = __shfl_sync(0xffffffffu, tm, 0), at = tm + ((uint32_t)(32 * q) << 16);
  const uint64_t pd = desc_mnmajor(base + G::OFF_PARTS, DP), pk = desc_kmajor(base + G::OFF_PARTS, DP);
  constexpr uint64_t STEP_K = 256 / 16, STEP_MN = DP * 32 / 16, PART = G::ST / 16, TSTEP_MN = 2048 / 16;
  const uint32_t id_ss = idesc_bf16(64, 64, false, false), id_kk = idesc_bf16(64, DP, false, false),
                 id_kn = idesc_bf16(64, DP, false, true), id_nn = idesc_bf16(64, DP, true, true);
  const uint32_t tq = base, tk = base + G::TILE, tv = base + 2 * G::TILE, to = base + 3 * G::TILE;  // tiles
  const uint32_t sp = base + G::OFF_P, sa = sp + G::PT;                                             // P, dA
  // a tile (K-major, boxes of 64 channels) times a state's parts, K- or MN-major
  auto times_parts = [&](uint32_t d, uint32_t tile, uint64_t part0, bool mn, int np) {
    const uint64_t x = desc_tile(tile);
#pragma unroll 1
    for (int p = np - 1; p >= 0; --p) {
#pragma unroll
      for (int bx = 0; bx < G::NB; ++bx)
        mma_steps<4>(d, x + bx * (BOX / 16), 2, part0 + p * PART + bx * 4 * (mn ? STEP_MN : STEP_K), mn ? STEP_MN : STEP_K,
                     mn ? id_kn : id_kk, p < np - 1 || bx > 0);
    }
  };
  auto issue_dq = [&] { mma_steps<4>(tmu + G::T_DQ, desc_kmajor(sa, C), 256 / 16, desc_tile_mn(tk), TSTEP_MN, id_kn, false); };
  auto issue_dk = [&] { mma_steps<4>(tmu + G::T_DK, desc_mnmajor(sa, C), C * 32 / 16, desc_tile_mn(tq), TSTEP_MN, id_nn, false); };
  auto issue_dv = [&] { mma_steps<4>(tmu + G::T_DV, desc_mnmajor(sp, C), C * 32 / 16, desc_tile_mn(to), TSTEP_MN, id_nn, false); };

  // The products are issued in the order in which their operands come, each step's float32 work
  // running during the next one's MMAs:
  //   A, B | products with S (and R) | scores | P and dA products that have room | the rest
  if (w == 0) {
    wait_for(ctl, &ctl.loaded, a.status);
#pragma unroll
    for (int bx = 0; bx < G::NB; ++bx) {
      mma_steps<4>(tmu + G::T_A, desc_tile(tq + bx * BOX), 2, desc_tile(tk + bx * BOX), 2, id_ss, bx > 0);
      mma_steps<4>(tmu + G::T_B, desc_tile(to + bx * BOX), 2, desc_tile(tv + bx * BOX), 2, id_ss, bx > 0);
    }
    mma_commit(&ctl.done[0]);
    times_parts(tmu + G::T_OS, to, pk, false, 3);                               // O S^T
    if (DP == 64) times_parts(tmu + G::T_VR, tv, pk + 3 * PART, false, 3);      // V R^T
    mma_commit(&ctl.done[1]);
  }
  __syncwarp();
  if (DP != 64) {
#pragma unroll
    for (int i = 0; i < NU; ++i) dot8(x[i], y[i]);
  }
  float dg = 0.f;
  // ---- scores ----
  wait_for(ctl, &ctl.done[0], a.status);
  {
    float xa[SC / 2], xb[SC / 2];
    frag<SC / 2>(at + G::T_A + SC * hf, xa);
    frag<SC / 2>(at + G::T_B + SC * hf, xb);
    tmem_wait_ld();
    F2 gl = f2(0.f, 0.f);
    uint8_t* pt = sm + G::OFF_P + cm_off(t0, SC * hf + c2, C);
#pragma unroll
    for (int j = 0; j < SC / 8; ++j)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int lag = t0 + 8 * k - (SC * hf + 8 * j + c2);  // of the pair's first column
        const F2 M = f2(lag >= 0 ? ctl.pw[lag] : 0.f, lag >= 1 ? ctl.pw[lag - 1] : 0.f);
        // masked scores are dropped, not multiplied by 0
        const F2 A = f2(lag >= 0 ? xa[4 * j + 2 * k] : 0.f, lag >= 1 ? xa[4 * j + 2 * k + 1] : 0.f);
        const F2 B = f2(lag >= 0 ? xb[4 * j + 2 * k] : 0.f, lag >= 1 ? xb[4 * j + 2 * k + 1] : 0.f);
        const F2 dA = M * B;
        gl = fma2(f2((float)lag, (float)(lag - 1)) * A, dA, gl);
        *(uint32_t*)(pt + k * C * 16 + j * 128) = bf2_pack(M * A);
        *(uint32_t*)(pt + G::PT + k * C * 16 + j * 128) = bf2_pack(dA);
      }
    const float2 gg = f2_get(gl);
    dg = P.scale * (gg.x + gg.y);
  }
  if constexpr (DP != 64) {  // the parts of R in the place of S's
    wait_for(ctl, &ctl.done[1], a.status);
#pragma unroll
    for (int i = 0; i < NU; ++i) put_parts3(parts + (tid + NT * i) * 16, G::ST, y[i]);
  }
  fence_async_smem();
  cta_sync();
  if (w == 0) {
    if (DP == 64) {
      issue_dq();
      issue_dv();
    } else {
      times_parts(tmu + G::T_VR, tv, pk, false, 3);
      times_parts(tmu + G::T_KR, tk, pd, true, 2);
      issue_dv();
    }
    mma_commit(&ctl.done[2]);
  }
  __syncwarp();
  // ---- the terms with S and R ----
  F2 dq[NV / 2], dk[NV / 2];  // [2 j]: row t0, columns 8 j + c2 and the next of this warp's; [2 j + 1]: row t0 + 8
  const float wo0 = t0 < L ? ctl.pw[L - 1 - t0] : 0.f, wo1 = t0 + 8 < L ? ctl.pw[L - 9 - t0] : 0.f;
  const F2 o0 = f2(wo0, wo0), o1 = f2(wo1, wo1);
  // rows t0 and t0 + 8 of a tile . a fragment
  auto dot_rows = [&](int which, const F2* v, float f0, float f1) {
    F2 s0 = f2(0.f, 0.f), s1 = s0;
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) {
      const int col = hf * CW + 8 * j, bx = col >> 6, jj = (col >> 3) & 7;
      const uint8_t* y = sm + which * G::TILE + bx * BOX + t0 * 128 + ((jj ^ r) << 4) + 2 * c2;
      s0 = fma2(bf2_unpack(*(const uint32_t*)y), v[2 * j], s0);
      s1 = fma2(bf2_unpack(*(const uint32_t*)(y + 8 * 128)), v[2 * j + 1], s1);
    }
    const float2 u = f2_get(s0), v1 = f2_get(s1);
    return f0 * (u.x + u.y) + f1 * (v1.x + v1.y);
  };
  // fragment of columns `col` on, row t0 times f0, row t0 + 8 times f1
  auto scaled = [&](uint32_t col, F2 f0, F2 f1, F2* v) {
    float t[NV];
    frag<NV>(at + col + hf * CW, t);
    tmem_wait_ld();
#pragma unroll
    for (int j = 0; j < NV / 2; ++j) v[j] = (j & 1 ? f1 : f0) * f2(t[2 * j], t[2 * j + 1]);
  };
  auto scaled_dk = [&] {
    scaled(G::T_VR, o0, o1, dk);
    dg += dot_rows(1, dk, (float)max(L - 1 - t0, 0), (float)max(L - 9 - t0, 0)) + (float)L * ctl.pw[L] * rs;
  };
  wait_for(ctl, &ctl.loaded, a.status);  // (long over: this thread is about to read the tiles itself)
  wait_for(ctl, &ctl.done[1], a.status);
  scaled(G::T_OS, f2(ctl.pw[t0 + 1], ctl.pw[t0 + 1]), f2(ctl.pw[t0 + 9], ctl.pw[t0 + 9]), dq);
  dg += P.scale * dot_rows(0, dq, (float)(t0 + 1), (float)(t0 + 9));
  if (DP == 64) scaled_dk();
  cta_sync();
  if (w == 0) {
    if (DP == 64) {
      issue_dk();
      times_parts(tmu + G::T_KR, tk, pd + 3 * PART, true, 2);
    } else {
      issue_dq();
    }
    mma_commit(&ctl.done[3]);
  }
  __syncwarp();
  wait_for(ctl, &ctl.done[2], a.status);
  if (DP != 64) {
    scaled_dk();
    cta_sync();
    if (w == 0) {
      issue_dk();
      mma_commit(&ctl.done[4]);
    }
    __syncwarp();
    wait_for(ctl, &ctl.done[3], a.status);
  }
  // ---- outputs, through tiles that no product reads any more ----
  const F2 sc = f2(P.scale, P.scale);
  auto put = [&](int which, const F2* v) {
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) {
      const int col = hf * CW + 8 * j, bx = col >> 6, jj = (col >> 3) & 7;
      uint8_t* y = sm + which * G::TILE + bx * BOX + t0 * 128 + ((jj ^ r) << 4) + 2 * c2;
      *(uint32_t*)y = bf2_pack(v[2 * j]);
      *(uint32_t*)(y + 8 * 128) = bf2_pack(v[2 * j + 1]);
    }
  };
  float v[NV];
  frag<NV>(at + G::T_DQ + hf * CW, v);
  tmem_wait_ld();
#pragma unroll
  for (int j = 0; j < NV / 2; ++j) dq[j] = sc * (dq[j] + f2(v[2 * j], v[2 * j + 1]));
  put(3, dq);  // dy's tile: dV, its last reader, is done (done[2])
  wait_for(ctl, &ctl.done[DP == 64 ? 3 : 4], a.status);
  frag<NV>(at + G::T_DK + hf * CW, v);
  tmem_wait_ld();
#pragma unroll
  for (int j = 0; j < NV / 2; ++j) dk[j] = fma2(sc, f2(v[2 * j], v[2 * j + 1]), dk[j]);
  put(0, dk);
  F2 dv[NV / 2];
  scaled(G::T_KR, o0, o1, dv);
  frag<NV>(at + G::T_DV + hf * CW, v);
  tmem_wait_ld();
#pragma unroll
  for (int j = 0; j < NV / 2; ++j) dv[j] = fma2(sc, f2(v[2 * j], v[2 * j + 1]), dv[j]);
  put(1, dv);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dg += __shfl_xor_sync(0xffffffffu, dg, o);
  if (lane == 0) ctl.red[w] = dg;
  fence_async_smem();
  cta_sync();
  if (tid == 0 && !ctl.bad) {
    for (int i = 0; i < (D > 64 ? 2 : 1); ++i) {
      tma_store(&maps.dq, 64 * i, h, c * C, b, sm + 3 * G::TILE + i * BOX);
      tma_store(&maps.dk, 64 * i, h, c * C, b, sm + i * BOX);
      tma_store(&maps.dv, 64 * i, h, c * C, b, sm + G::TILE + i * BOX);
    }
    bulk_commit();
    float s = 0.f;
    for (int i = 0; i < NT / 32; ++i) s += ctl.red[i];
    a.dg_part[blockIdx.x] = s;
    bulk_wait_read0();
  }
  if (w == 1) tmem_dealloc(tm, G::COLS);
}

template <int DP>
static cudaError_t launch(const Maps& m, const Args& a, cudaStream_t s) {
  cudaError_t e = allow_smem<grads_kernel<DP>>(GRAD_SMEM<DP>);
  if (e != cudaSuccess) return e;
  return follow(grads_kernel<DP>, (unsigned)(chains(a.p) * chunks(a.p)), GCfg<DP>::NT, GRAD_SMEM<DP>, s, m, a);
}

cudaError_t launch_grads(const Args& a, cudaStream_t s) {
  const AtlasDecayParams& p = a.p;
  const int64_t flat[3] = {(int64_t)p.T * p.H * p.D, (int64_t)p.H * p.D, p.D};
  Maps m;
  if (!make_map(&m.q, a.q, p, p.q_stride) || !make_map(&m.k, a.k, p, p.k_stride) || !make_map(&m.v, a.v, p, p.v_stride) ||
      !make_map(&m.o, a.dy, p, flat) || !make_map(&m.dq, a.dq, p, flat) || !make_map(&m.dk, a.dk, p, flat) ||
      !make_map(&m.dv, a.dv, p, flat))
    return cudaErrorInvalidValue;
  return p.D <= 64 ? launch<64>(m, a, s) : launch<128>(m, a, s);
}

}  // namespace tcore
}  // namespace decay
}  // namespace atlas
