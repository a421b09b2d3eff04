// Decay attention (include/atlas_decay.h), the pass along the sequence on the tcgen05
// tensor cores: outputs and states of the forward, and the cotangent states of the backward.
//
// One CTA walks a segment of one (batch, head) in blocks of C = 64 tokens with the state
// S in registers (float32).  Per block of L tokens, l = exp(log_decay):
//
//     A  = Q K^T               dS = K'^T V,  k'_s = l^(L-1-s) k_s       QS = Q S
//     P  = l^(t-s) o A         S <- l^L S + dS                          O  = P V
//     y_t = scale (O_t + l^(t+1) QS_t)
//
// Only QS and the update of S depend on the block before, so the CTA is a pipeline of
// groups that hand blocks on through mbarriers:
//
//     4 warps       k' split into three bf16 parts (float32 accuracy of the state)
//     4 warps       scores: A from TMEM, decayed, masked, rounded to bf16
//     4 warps       outputs: O and QS from TMEM, y to memory, 64 bytes of a row at a time
//     4 (16) warps  the state: dS from TMEM, S in registers, two bf16 parts of S for QS
//     3 warps       issue the MMAs;  one warp issues the TMA loads of q, k, v
//
// The same kernel without q's side gives the states alone: the sums of a segment (first
// pass of a split sequence), and with (q, scale dy, l^(t+1)) for (k, v, l^(L-1-s)) and the blocks
// taken from the last to the first, the cotangent states of the backward.
//
// A sequence is split into segments where there are fewer (batch, head) pairs than SMs: the
// segments' sums first, then every segment, from a state put together from the sums before
// it.
//
// What bounds it: the latency of a block's two chains, S -> parts -> QS -> y and k' -> dS -> S, each step
// of which waits for the group before.  No unit is full: a block is about 5,300 warp instructions at
// D = 64, 1,340 of the 2,200 cycles that it takes on each of four schedulers (61 %), and 15,000 at D = 128,
// 3,770 of 5,900 (64 %); the tensor pipe is busy for 37 % and 20 %.  Measured: 8 x 8192 tokens x 12 heads
// of 64 149 us (96 CTAs, one a chain: 2.7 TB/s); 65536 x 16 heads of 128, in nine segments, 494 us, 144 of
// them sums; the cotangent states of 16 x 4096 x 8 heads of 64 58 us (4.6 TB/s).  A prefetch of the blocks to come into
// L2 and a fourth stage change nothing; O and QS handed on in halves of 64 columns (D = 128) cost 12 %.
//
// Layout: q, k, v tiles as TMA writes them (rows of 128 bytes, 128-byte swizzle, a box per
// 64 channels); k', scores and S in the core-matrix layout of tc_ops.cuh.  All M = 64
// accumulators sit in 16 lanes of each TMEM lane quadrant and are read with 16x256b loads,
// which spread them over all 32 lanes of a warp: lane holds rows lane / 4 and lane / 4 + 8,
// columns 8 j + 2 (lane % 4) and the next one.
#include <algorithm>
#include <mutex>

#include "decay_tc.cuh"

namespace atlas {
namespace decay {
namespace tcore {

template <int DP, bool FWD>
struct Cfg {
  static constexpr int NB = DP / 64;                    // boxes of a tile
  static constexpr int TILE = NB * BOX;                 // 64 tokens x DP channels
  static constexpr int TILES = FWD ? 3 : 2;             // of a stage: (q,) k, v
  static constexpr int STAGES = FWD ? (DP == 64 ? 3 : 2) : (DP == 64 ? 4 : 3);
  static constexpr int DBL = FWD && DP == 128 ? 1 : 2;  // buffers of k', scores, S and the accumulators
  // Warps of the k' and of the state group.  Few, with more values each, where the registers allow: the
  // schedulers are shared with the groups that wait (D = 64, 8 x 8192 tokens x 12 heads, 8 and 8: 164 us;
  // 4 and 8: 156; 4 and 4: 150).  D = 128 with a state group of 8 spills.
  static constexpr int KWARPS = FWD ? 4 : 8, SWARPS = DP == 64 ? 4 : 16;
  static constexpr int MWARPS = FWD ? 3 : 1;            // warps that issue MMAs
  static constexpr int W_P = KWARPS, W_Y = W_P + (FWD ? 4 : 0), W_S = W_Y + (FWD ? 4 : 0), W_MMA = W_S + SWARPS;  // first warps of the groups
  static constexpr int W_LOAD = W_MMA + MWARPS, NT = 32 * (W_LOAD + 1);
  static constexpr int PT = C * C * 2;                  // a tile of scores
  static constexpr int ST = DP * DP * 2;                // one part of a state
  static constexpr int OFF_KP = STAGES * TILES * TILE;
  static constexpr int OFF_P = OFF_KP + DBL * 3 * TILE;
  static constexpr int OFF_S = OFF_P + (FWD ? DBL * PT : 0);
  static constexpr int OFF_CTL = OFF_S + (FWD ? DBL * 2 * ST : 0);
  // TMEM columns
  static constexpr uint32_t T_A = 0, T_DS = FWD ? DBL * 64 : 0, T_QS = T_DS + DBL * DP, T_O = T_QS + DBL * DP;
  static constexpr uint32_t COLS = FWD ? 512 : DBL * DP;
  static_assert(!FWD || T_O + DBL * DP <= 512, "TMEM");
};

struct Ctl {
  F2 w[2 * C];                       // w[C + lag] = (l^lag, l^(lag - 1)), clamped at exponent 0
  uint64_t full[4], empty[4];        // stages
  uint64_t a_full[2], a_free[2];     // A in TMEM
  uint64_t kp_full[2], kp_free[2];   // k' parts
  uint64_t ds_full[2], ds_free[2];   // dS in TMEM
  uint64_t s_full[2], s_free[2];     // parts of S
  uint64_t p_full[2], p_free[2];     // scores
  uint64_t o_full[2], o_free[2];     // O and QS in TMEM
  uint64_t fin;
  uint32_t tmem;
  volatile int bad;
};
template <int DP, bool FWD>
constexpr size_t SEQ_SMEM = Cfg<DP, FWD>::OFF_CTL + sizeof(Ctl) + 1024;

struct SeqArgs {
  AtlasDecayParams p;
  const float* log_decay;
  const float* in;  // (chains, D, D) entering the first segment of the walk, or NULL: zeros
  float* out;       // leaving the last one
  // What enters segments 0 and 1 of every chain's walk and the sums of segments 1 .. segs - 2, written
  // by the sums' pass.  Segment 0's is a copy, so that `out` may be `in`.
  float* sums;
  bf16* y;
  float* saves;    // state entering every block, in the order of the walk; or NULL
  int segs;        // segments of a sequence
  int seg_blocks;  // blocks of a segment
  int joined;      // join_kernel has made the sums the states that enter their segments
  int sums_pass;   // segments 0 .. segs - 2, all but the first from zeros, to `sums`
  int* status;
};
__device__ __forceinline__ float* sum_at(const SeqArgs& a, int64_t chain, int i) {
  return a.sums + (chain * a.segs + i) * a.p.D * a.p.D;
}

// Waits for completion number n (from 0) of a barrier.  Bounded; a timeout anywhere in the
// CTA is recorded and lets every group leave its loop.  Only the first poll is inline: the
// groups share the schedulers' instruction caches, and their loops together are about as
// large as those (unrolled further, the kernel ran 20 to 40 % longer).
__device__ __noinline__ bool wait_on(Ctl& c, uint64_t* bar, uint32_t parity, int* status) {
  for (uint32_t i = 0; i < 4000000u; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 15) == 15 && c.bad) return false;
  }
  c.bad = 1;
  set_status(status, ATLAS_ERR_DEVICE_TIMEOUT);
  return false;
}
__device__ __forceinline__ bool wait(Ctl& c, uint64_t* bar, int n, int* status) {
  return mbar_try_wait(bar, (uint32_t)n & 1) || wait_on(c, bar, (uint32_t)n & 1, status);
}
// one arrival for a whole warp, after its shared-memory writes / TMEM reads
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) arrive(bar);
}

// Lanes 4 n .. 4 n + 3: v[j] of lane c and v[c] of lane j change places.
__device__ __forceinline__ void quad_transpose(uint32_t* v, int c) {
#pragma unroll
  for (int m = 1; m <= 2; m *= 2)
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int j = m == 1 ? 2 * n : n;  // pair (j, j + m)
      const uint32_t x = __shfl_xor_sync(0xffffffffu, c & m ? v[j] : v[j + m], m);
      v[j] = c & m ? x : v[j];
      v[j + m] = c & m ? v[j + m] : x;
    }
}

struct Walk {  // one CTA's blocks: first, first + step, ..., n of them
  int64_t chain;
  int b, h, seg, first, step, n;
};

template <int DP, bool FWD>
__global__ void __launch_bounds__(Cfg<DP, FWD>::NT, 1)
    seq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_x,
               const __grid_constant__ CUtensorMap map_y, const SeqArgs a,
               bool reversed) {
  using K = Cfg<DP, FWD>;
  extern __shared__ uint8_t raw[];
  uint8_t* sm = (uint8_t*)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
  Ctl& ctl = *(Ctl*)(sm + K::OFF_CTL);
  const AtlasDecayParams& P = a.p;
  // the warp's number as a uniform value: each role's branch is then known not to diverge
  const int w = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int D = P.D, nblk = (P.T + C - 1) / C;
  Walk z;
  const int per_chain = a.segs - a.sums_pass;
  z.chain = blockIdx.x / per_chain;
  z.seg = (int)(blockIdx.x % per_chain);  // in the order of the walk
  z.b = (int)(z.chain / P.H);
  z.h = (int)(z.chain % P.H);
  {
    const int at = reversed ? a.segs - 1 - z.seg : z.seg;
    const int lo = at * a.seg_blocks, hi = min(nblk, lo + a.seg_blocks);
    z.n = hi - lo;
    z.first = reversed ? hi - 1 : lo;
    z.step = reversed ? -1 : 1;
  }
  const int nbox = D > 64 ? 2 : 1;
  auto load_block = [&](int i) {  // one thread
    const int st = i % K::STAGES, blk = z.first + i * z.step;
    mbar_expect_tx(&ctl.full[st], (uint32_t)(K::TILES * nbox * BOX));
    uint8_t* t = sm + (st + 1) * K::TILES * K::TILE;
    for (int hb = 0; hb < nbox; ++hb) {
      if (FWD) tma_load(t - 3 * K::TILE + hb * BOX, &map_q, 64 * hb, z.h, blk * C, z.b, &ctl.full[st]);
      tma_load(t - 2 * K::TILE + hb * BOX, &map_x, 64 * hb, z.h, blk * C, z.b, &ctl.full[st]);
      tma_load(t - K::TILE + hb * BOX, &map_y, 64 * hb, z.h, blk * C, z.b, &ctl.full[st]);
    }
  };
  if (w == K::W_LOAD && lane == 0) {
    for (int i = 0; i < K::STAGES; ++i) {
      mbar_init(&ctl.full[i], 1);
      mbar_init(&ctl.empty[i], K::MWARPS + K::KWARPS);  // the issuing warps' last MMAs, and the warps that read k
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.a_full[i], 1);
      mbar_init(&ctl.a_free[i], 4);
      mbar_init(&ctl.kp_full[i], K::KWARPS);
      mbar_init(&ctl.kp_free[i], 1);
      mbar_init(&ctl.p_full[i], 4);
      mbar_init(&ctl.p_free[i], 1);
      mbar_init(&ctl.o_full[i], 2);  // O and QS
      mbar_init(&ctl.o_free[i], 4);
      mbar_init(&ctl.ds_full[i], 1);
      mbar_init(&ctl.ds_free[i], K::SWARPS);
      mbar_init(&ctl.s_full[i], K::SWARPS);
      mbar_init(&ctl.s_free[i], 1);
    }
    mbar_init(&ctl.fin, K::MWARPS);
    ctl.bad = 0;
    fence_mbar_init();
    for (int i = 0; i < min(K::STAGES, z.n); ++i) load_block(i);  // on their way while the rest is set up
  }
  if (w == K::W_MMA) {
    tmem_alloc(&ctl.tmem, K::COLS);
    tmem_relinquish();
  }
  const float g = a.log_decay[z.h];
  for (int u = threadIdx.x; u < 2 * C; u += K::NT) ctl.w[u] = f2(powd(g, max(u - C, 0)), powd(g, max(u - C - 1, 0)));
  if (FWD)  // score blocks above the diagonal are written here once and never again
    for (int u = threadIdx.x; u < K::DBL * K::PT / 16; u += K::NT) *(uint4*)(sm + K::OFF_P + u * 16) = make_uint4(0, 0, 0, 0);
  fence_async_smem();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tm = ctl.tmem;
  let_next_start();  // this CTA has its tensor memory: the next kernel cannot take it away

  if (w < K::KWARPS) {
    // ---- k' : thread (token row, every KP-th 16-byte group) ----
    constexpr int KP = K::KWARPS / 2;
    const int r = threadIdx.x & 63, first = threadIdx.x >> 6;
    const float wfull = reversed ? powd(g, r + 1) : powd(g, C - 1 - r);
    for (int i = 0; i < z.n; ++i) {
      const int st = i % K::STAGES, b = i % K::DBL, blk = z.first + i * z.step;
      const int L = min(C, P.T - blk * C);
      if (!wait(ctl, &ctl.full[st], i / K::STAGES, a.status)) break;
      if (i >= K::DBL && !wait(ctl, &ctl.kp_free[b], i / K::DBL - 1, a.status)) break;
      const float wr = reversed || L == C ? wfull : r < L ? powd(g, L - 1 - r) : 0.f;
      const F2 w2 = f2(wr, wr);
      const uint8_t* x = sm + (st * K::TILES + K::TILES - 2) * K::TILE + r * 128;
      uint8_t* kp = sm + K::OFF_KP + b * 3 * K::TILE + cm_off(r, 0, DP);
#pragma unroll 1
      for (int jj = 0; jj < DP / 8 / KP; ++jj) {
        const int j = first + KP * jj;
        const uint4 pk = *(const uint4*)(x + (j >> 3) * BOX + (((j & 7) ^ (r & 7)) << 4));
        F2 v[4] = {w2 * bf2_unpack(pk.x), w2 * bf2_unpack(pk.y), w2 * bf2_unpack(pk.z), w2 * bf2_unpack(pk.w)};
        put_parts3(kp + j * 128, K::TILE, v);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        arrive(&ctl.kp_full[b]);
        arrive(&ctl.empty[st]);
      }
    }
  } else if (FWD && w < K::W_Y) {
    // ---- scores ----
    // Rounded to bf16, as P V's operand: y's relative error goes from the 1.66e-3 of its own rounding to
    // 1.8e-3.  (A second part would be as many MMAs again and a tile more, for digits that y's type drops.)
    if (FWD) {
      const int q = w & 3, r = lane >> 2, c2 = 2 * (lane & 3), t0 = 16 * q + r;
      uint8_t* prow = sm + K::OFF_P + cm_off(t0, c2, C);
      for (int i = 0; i < z.n; ++i) {
        const int b = i % K::DBL, n = i / K::DBL;
        if (!wait(ctl, &ctl.a_full[b], n, a.status)) break;
        if (i >= K::DBL && !wait(ctl, &ctl.p_free[b], n - 1, a.status)) break;
        fence_after();
#pragma unroll 1
        for (int hc = 0; hc < 2; ++hc) {  // 32 columns; those beyond the warp's diagonal stay zero
          if (2 * hc <= q) {
            float v[16];
            tmem_frag32(tm + K::T_A + 64 * b + 32 * hc + ((uint32_t)(32 * q) << 16), v);
            tmem_wait_ld();
            uint8_t* p = prow + b * K::PT + hc * 512;
            int lag = t0 - (32 * hc + c2);  // of the first column of block j = 0, row t0
#pragma unroll
            for (int j = 0; j < 4; ++j, lag -= 8) {
              // masked entries are dropped, not multiplied by 0
              const F2 m = f2(lag >= 0 ? v[4 * j] : 0.f, lag >= 1 ? v[4 * j + 1] : 0.f);
              const F2 o = f2(lag >= -8 ? v[4 * j + 2] : 0.f, lag >= -7 ? v[4 * j + 3] : 0.f);
              const F2* wt = ctl.w + lag + C;
              *(uint32_t*)(p + j * 128) = bf2_pack(m * wt[0]);
              *(uint32_t*)(p + C * 16 + j * 128) = bf2_pack(o * wt[8]);  // 8 rows on
            }
          }
        }
        fence_before();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          arrive(&ctl.a_free[b]);
          arrive(&ctl.p_full[b]);
        }
      }
    }
  } else if (FWD && w < K::W_S) {
    // ---- outputs ----
    if (FWD) {
      const int q = w & 3, r = lane >> 2, cq = lane & 3, t0 = 16 * q + r;
      const float i0 = P.scale * powd(g, t0 + 1), i1 = P.scale * powd(g, t0 + 9);
      const F2 i02 = f2(i0, i0), i12 = f2(i1, i1), sc2 = f2(P.scale, P.scale);
      const int64_t row = (int64_t)P.H * D;
      bf16* y0 = a.y + (((int64_t)z.b * P.T + t0) * P.H + z.h) * D + 8 * cq;
      for (int i = 0; i < z.n; ++i) {
        const int b = i % K::DBL, blk = z.first + i * z.step, L = P.T - blk * C;
        if (!wait(ctl, &ctl.o_full[b], i / K::DBL, a.status)) break;
        fence_after();
        const uint32_t at = tm + ((uint32_t)(32 * q) << 16) + b * DP;
#pragma unroll 1
        for (int col = 0; col < DP; col += 32) {
          float v[16], x[16];
          tmem_frag32(at + K::T_O + col, v);
          tmem_frag32(at + K::T_QS + col, x);
          tmem_wait_ld();
          if (col == DP - 32) {
            fence_before();
            warp_arrive(&ctl.o_free[b]);
          }
          uint32_t e[4], f[4];  // rows t0 and t0 + 8, columns 8 j + 2 cq and the next
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            e[j] = bf2_pack(fma2(i02, f2(x[4 * j], x[4 * j + 1]), sc2 * f2(v[4 * j], v[4 * j + 1])));
            f[j] = bf2_pack(fma2(i12, f2(x[4 * j + 2], x[4 * j + 3]), sc2 * f2(v[4 * j + 2], v[4 * j + 3])));
          }
          // now columns 8 cq .. 8 cq + 7: 16 bytes a lane, 64 in a row for the four lanes of one
          quad_transpose(e, cq);
          quad_transpose(f, cq);
          bf16* y = y0 + (int64_t)blk * C * row + col;
          if (col + 8 * cq < D) {
            if (t0 < L) *(uint4*)y = make_uint4(e[0], e[1], e[2], e[3]);
            if (t0 + 8 < L) *(uint4*)(y + 8 * row) = make_uint4(f[0], f[1], f[2], f[3]);
          }
        }
      }
    }
  } else if (w < K::W_MMA) {
    // ---- the state ----
    // DP = 64: 16 rows in lanes 0-15 of the quadrant.  DP = 128: rows are lanes.  A warp has 16 rows and
    // half of the columns.
    constexpr int NJ = DP == 64 ? 32 / K::SWARPS : 8;  // 8-column blocks of a warp
    const int sub = (w - K::W_S) >> 2, q = w & 3, r = lane >> 2, c2 = 2 * (lane & 3);
    const int hf = DP == 64 ? 0 : sub & 1, e0 = (DP == 64 ? sub : sub >> 1) * 8 * NJ;
    const int d0 = DP == 64 ? 16 * q + r : 32 * q + 16 * hf + r;
    const uint32_t at = tm + K::T_DS + e0 + ((uint32_t)(32 * q + 16 * hf) << 16);
    after_previous();            // (no other warp reads or writes what an earlier kernel of the call does)
    F2 S[2 * NJ];                // [2 j]: row d0, columns e0 + 8 j + c2 and the next; [2 j + 1]: row d0 + 8
    const int64_t DD = (int64_t)D * D;
    const bool in0 = d0 < D, in1 = d0 + 8 < D;
    {
      // S = f s + S for the state at s (or zeros); f as a float pair
      auto add_state = [&](const float* s, double f, bool first) {
        const float fh = (float)f, fl = (float)(f - (double)fh);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int e = e0 + 8 * j + c2;
          float2 x = make_float2(0.f, 0.f), y = x;
          if (s && e < D) {
            if (in0) x = *(const float2*)(s + (int64_t)d0 * D + e);
            if (in1) y = *(const float2*)(s + (int64_t)(d0 + 8) * D + e);
          }
          const F2 h2 = f2(fh, fh), l2 = f2(fl, fl);
          S[2 * j] = first ? f2(x.x, x.y) : fma2(S[2 * j], h2, fma2(S[2 * j], l2, f2(x.x, x.y)));
          S[2 * j + 1] = first ? f2(y.x, y.y) : fma2(S[2 * j + 1], h2, fma2(S[2 * j + 1], l2, f2(y.x, y.y)));
        }
      };
      const float* in = a.in ? a.in + z.chain * DD : nullptr;
      if (a.sums_pass || a.segs == 1) {
        add_state(z.seg == 0 ? in : nullptr, 0., true);
      } else if (z.seg == 0) {
        add_state(in ? sum_at(a, z.chain, 0) : nullptr, 0., true);
      } else {
        const double f = exp((double)g * ((double)a.seg_blocks * C));
        const int j0 = a.joined ? z.seg : 1;
        for (int j = j0; j <= z.seg; ++j) add_state(sum_at(a, z.chain, j), f, j == j0);
      }
    }
    auto put_state = [&](float* out) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int e = e0 + 8 * j + c2;
        if (e < D) {
          if (in0) *(float2*)(out + (int64_t)d0 * D + e) = f2_get(S[2 * j]);
          if (in1) *(float2*)(out + (int64_t)(d0 + 8) * D + e) = f2_get(S[2 * j + 1]);
        }
      }
    };
    if (a.sums_pass && z.seg == 0 && a.in) put_state(sum_at(a, z.chain, 0));
    // decay over a block as a float pair: its rounding would be multiplied in again every block
    const double fd = exp((double)g * C);
    const float fh = (float)fd, fl = (float)(fd - (double)fh), sc = reversed ? P.scale : 1.f;
    for (int i = 0; i < z.n; ++i) {
      const int blk = z.first + i * z.step, b = i % K::DBL, n = i / K::DBL;
      if (a.saves) put_state(a.saves + (z.chain * nblk + blk) * DD);
      if (FWD) {  // two parts for QS: 16 bits of S, an error of 2^-17 where y rounds by 2^-9 (S itself stays float32)
        if (i >= K::DBL && !wait(ctl, &ctl.s_free[b], n - 1, a.status)) break;
        uint8_t* s = sm + K::OFF_S + b * 2 * K::ST + cm_off(d0, e0 + c2, DP);
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const F2 x = S[2 * j + k];
            const uint32_t hi = bf2_pack(x);
            uint8_t* d = s + j * 128 + k * DP * 16;  // 8 rows on
            *(uint32_t*)d = hi;
            *(uint32_t*)(d + K::ST) = bf2_pack(x - bf2_unpack(hi));
          }
        fence_async_smem();
        warp_arrive(&ctl.s_full[b]);
      }
      float fbh = fh, fbl = fl;
      if ((blk + 1) * C > P.T) {
        const double f = exp((double)g * (P.T - blk * C));
        fbh = (float)f, fbl = (float)(f - (double)fbh);
      }
      if (!wait(ctl, &ctl.ds_full[b], n, a.status)) break;
      fence_after();
      const F2 h2 = f2(fbh, fbh), l2 = f2(fbl, fbl), c = f2(sc, sc);
#pragma unroll
      for (int j = 0; j < 2 * NJ; j += 8) {  // 32 columns at a time: the registers of 1024 threads hold no more
        float v[16];
        tmem_frag32(at + b * DP + 4 * j, v);
        tmem_wait_ld();
        if (j == 2 * NJ - 8) {
          fence_before();
          warp_arrive(&ctl.ds_free[b]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          F2 x = f2(v[2 * k], v[2 * k + 1]);
          if (!FWD) x = x * c;
          S[j + k] = fma2(S[j + k], h2, fma2(S[j + k], l2, x));
        }
      }
    }
    if (a.sums_pass)
      put_state(sum_at(a, z.chain, z.seg + 1));
    else if (a.out && z.seg == a.segs - 1)
      put_state(a.out + z.chain * DD);
  } else if (w < K::W_MMA + K::MWARPS) {
    // ---- MMAs ----
    // Issuing blocks while the tensor pipe is busy, and a wait costs its latency even when it
    // is over at once; with one warp for all of them the pipe idled through every wait.
    // Descriptors step through a tile by adding to their start address (bytes / 16).
    const uint32_t base = smem_u32(sm);
    const uint32_t tmu = __shfl_sync(0xffffffffu, tm, 0);
    auto tile = [&](int i, int which) { return base + ((i % K::STAGES + 1) * K::TILES - which) * K::TILE; };  // 1: v, 2: k, 3: q
    if (w == K::W_MMA) {  // dS = K'^T V
      const uint32_t id = idesc_bf16(DP, DP, true, true);
      for (int i = 0; i < z.n; ++i) {
        const int b = i % K::DBL, n = i / K::DBL;
        if (!(wait(ctl, &ctl.full[i % K::STAGES], i / K::STAGES, a.status) && wait(ctl, &ctl.kp_full[b], n, a.status) &&
              (i < K::DBL || wait(ctl, &ctl.ds_free[b], n - 1, a.status))))
          break;
        fence_after();
        const uint64_t v = desc_tile_mn(tile(i, 1)), kp = desc_mnmajor(base + K::OFF_KP + b * 3 * K::TILE, DP);
#pragma unroll 1
        for (int p = 2; p >= 0; --p)  // small parts first: each step truncates to the accumulator's exponent
#pragma unroll
          for (int ks = 0; ks < C / 16; ++ks)
            mma_kf16(tmu + K::T_DS + b * DP, kp + (p * K::TILE + ks * DP * 32) / 16, v + ks * (2048 / 16), id,
                     p < 2 || ks > 0);
        mma_commit(&ctl.kp_free[b]);
        mma_commit(&ctl.ds_full[b]);
        mma_commit(&ctl.empty[i % K::STAGES]);
      }
    } else if (FWD && w == K::W_MMA + 1) {  // A = Q K^T of the next block, O = P V
      const uint32_t id = idesc_bf16(64, 64, false, false), ido = idesc_bf16(64, DP, false, true);
      auto scores = [&](int i) {
        const uint64_t q = desc_tile(tile(i, 3)), k = desc_tile(tile(i, 2));
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          const uint64_t o = ((ks >> 2) * BOX + (ks & 3) * 32) / 16;
          mma_kf16(tmu + K::T_A + 64 * (i % K::DBL), q + o, k + o, id, ks > 0);
        }
        mma_commit(&ctl.a_full[i % K::DBL]);
      };
      bool ok = wait(ctl, &ctl.full[0], 0, a.status);
      if (ok) scores(0);
      for (int i = 0; i < z.n && ok; ++i) {
        const int b = i % K::DBL, n = i / K::DBL;
        if (i + 1 < z.n) {
          const int b1 = (i + 1) % K::DBL;
          ok = wait(ctl, &ctl.full[(i + 1) % K::STAGES], (i + 1) / K::STAGES, a.status) &&
               (i + 1 < K::DBL || wait(ctl, &ctl.a_free[b1], (i + 1) / K::DBL - 1, a.status));
          if (!ok) break;
          fence_after();
          scores(i + 1);
        }
        ok = wait(ctl, &ctl.p_full[b], n, a.status) && (i < K::DBL || wait(ctl, &ctl.o_free[b], n - 1, a.status));
        if (!ok) break;
        fence_after();
        const uint64_t v = desc_tile_mn(tile(i, 1)), pt = desc_kmajor(base + K::OFF_P + b * K::PT, C);
#pragma unroll
        for (int ks = 0; ks < C / 16; ++ks)
          mma_kf16(tmu + K::T_O + b * DP, pt + ks * (256 / 16), v + ks * (2048 / 16), ido, ks > 0);
        mma_commit(&ctl.p_free[b]);
        mma_commit(&ctl.o_full[b]);
        mma_commit(&ctl.empty[i % K::STAGES]);
      }
    } else if (FWD) {  // QS
      const uint32_t id = idesc_bf16(64, DP, false, true);
      for (int i = 0; i < z.n; ++i) {
        const int b = i % K::DBL, n = i / K::DBL;
        if (!(wait(ctl, &ctl.full[i % K::STAGES], i / K::STAGES, a.status) && wait(ctl, &ctl.s_full[b], n, a.status) &&
              (i < K::DBL || wait(ctl, &ctl.o_free[b], n - 1, a.status))))
          break;
        fence_after();
        const uint64_t q = desc_tile(tile(i, 3)), S = desc_mnmajor(base + K::OFF_S + b * 2 * K::ST, DP);
#pragma unroll 1
        for (int p = 1; p >= 0; --p)
#pragma unroll
          for (int ks = 0; ks < DP / 16; ++ks)
            mma_kf16(tmu + K::T_QS + b * DP, q + ((ks >> 2) * BOX + (ks & 3) * 32) / 16,
                     S + (p * K::ST + ks * DP * 32) / 16, id, p < 1 || ks > 0);
        mma_commit(&ctl.s_free[b]);
        mma_commit(&ctl.o_full[b]);
        mma_commit(&ctl.empty[i % K::STAGES]);
      }
    }
    if (FWD || w == K::W_MMA) {
      mma_commit(&ctl.fin);  // nothing of this CTA is in flight on the tensor core when its TMEM is freed
      wait(ctl, &ctl.fin, 0, a.status);
    }
  } else if (lane == 0) {
    // ---- loads ----
    int i = min(K::STAGES, z.n);
    for (; i < z.n; ++i) {
      if (!wait(ctl, &ctl.empty[i % K::STAGES], i / K::STAGES - 1, a.status)) break;
      load_block(i);
    }
    if (ctl.bad)  // let the copies land before the CTA goes
      for (int k = max(0, i - K::STAGES); k < i; ++k)
        for (int n = 0; n < 1000000 && !mbar_try_wait(&ctl.full[k % K::STAGES], (uint32_t)(k / K::STAGES) & 1); ++n) {
        }
  }
  fence_before();
  __syncthreads();
  if (w == K::W_MMA) tmem_dealloc(tm, K::COLS);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// (B, T, H, D) activations with element strides s (batch, token, head) as boxes of 64 tokens x
// 64 channels of one head, 128-byte swizzle; elements outside read as zero and are not written.
// An axis of length 1 takes the row size as its stride (its own is never used).
bool make_map(CUtensorMap* m, const void* x, const AtlasDecayParams& p, const int64_t* s) {
  auto enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)p.D, (cuuint64_t)p.H, (cuuint64_t)p.T, (cuuint64_t)p.B};
  const cuuint64_t row = (cuuint64_t)p.D * 2;
  const cuuint64_t strides[3] = {p.H > 1 ? (cuuint64_t)s[2] * 2 : row, p.T > 1 ? (cuuint64_t)s[1] * 2 : row,
                                 p.B > 1 ? (cuuint64_t)s[0] * 2 : row};
  const cuuint32_t box[4] = {64, 1, C, 1}, es[4] = {1, 1, 1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(x), dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The strides that a tensor map holds: multiples of 16 bytes below 2^40, none of them 0.
bool mappable(const AtlasDecayParams& p, const int64_t* s) {
  const int64_t n[3] = {p.B, p.T, p.H};
  for (int i = 0; i < 3; ++i)
    if (n[i] > 1 && (s[i] <= 0 || s[i] % 8 != 0 || s[i] >= (int64_t)1 << 39)) return false;
  return encode_fn() != nullptr;
}

template <int DP, bool FWD>
static cudaError_t launch(const CUtensorMap& q, const CUtensorMap& x, const CUtensorMap& y, const SeqArgs& a,
                          bool reversed, cudaStream_t s) {
  cudaError_t e = allow_smem<seq_kernel<DP, FWD>>(SEQ_SMEM<DP, FWD>);
  if (e != cudaSuccess) return e;
  const unsigned grid = (unsigned)(chains(a.p) * (a.segs - a.sums_pass));
  if (a.segs > 1 && !a.sums_pass)
    return follow(seq_kernel<DP, FWD>, grid, Cfg<DP, FWD>::NT, SEQ_SMEM<DP, FWD>, s, q, x, y, a, reversed);
  seq_kernel<DP, FWD><<<grid, Cfg<DP, FWD>::NT, SEQ_SMEM<DP, FWD>, s>>>(q, x, y, a, reversed);
  return cudaGetLastError();
}

// Whether the sums are joined by a kernel of their own, and not by the segments' CTAs, which read them one
// after the other at about 0.7 us (D = 64) or 2.5 us (D = 128, with few registers left for loads) each.
// 4 x 1900 tokens x 6 heads of 128, six segments: 26.7 + 4.8 us against 38.7; 3 x 777 x 12 heads of 64, four:
// 10.2 + 3.0 us against 10.4; 32768 x 2 heads of 64, 64 segments, the whole forward: 37 us against 116.
static bool join_first(const AtlasDecayParams& p, int segs) { return segs > (p.D > 64 ? 2 : 4); }

// How many segments to cut a sequence into, and their blocks: the least time by what was measured (us).
// A CTA an SM, in rounds; a round is a CTA's start and end, and its blocks.
struct Split {
  int segs, blocks;
};
static Split split(const AtlasDecayParams& p, bool bwd) {
  const bool wide = p.D > 64;
  const double start = wide ? 9 : 5, start_sum = wide ? 7.5 : 3;  // (the sums' end runs beside the next start)
  const double sum = wide ? 1.3 : 0.9, full = wide ? (bwd ? 1.9 : 3.1) : bwd ? 0.9 : 1.15;  // a block
  const int nblk = (p.T + C - 1) / C;
  const int64_t n = chains(p), sms = 148;
  auto rounds = [&](int64_t ctas) { return (double)((ctas + sms - 1) / sms); };
  Split best{1, nblk};
  double cost = rounds(n) * (start + nblk * full);
  for (int k = 2; k <= 64 && k <= nblk; ++k) {
    const int len = (nblk + k - 1) / k, segs = (nblk + len - 1) / len;
    if (segs != k) continue;
    const double c = rounds(n * k) * (start + len * full) + rounds(n * (k - 1)) * (start_sum + len * sum) +
                     (join_first(p, k) ? 4 + 0.1 * k : 0.7 * (k - 2));
    if (c < 0.95 * cost) cost = c, best = Split{k, len};
  }
  return best;
}

// What enters segments 2, 3, ..: S <- l^len S + sum, in place, len tokens each.  One thread per 4
// elements of a chain's state; the loads of UN segments are in flight together.
__global__ void __launch_bounds__(256) join_kernel(SeqArgs a) {
  constexpr int UN = 8;
  const int per = a.p.D * a.p.D / 4;
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  let_next_start();
  after_previous();
  if (u >= chains(a.p) * per) return;
  const int64_t chain = u / per;
  float4* m = (float4*)sum_at(a, chain, 1) + (u - chain * per);
  const double f = exp((double)a.log_decay[chain % a.p.H] * ((double)a.seg_blocks * C));
  const float fh = (float)f, fl = (float)(f - (double)fh);
  float4 S = m[0];
  for (int s0 = 1; s0 < a.segs - 1; s0 += UN) {
    float4 x[UN];
#pragma unroll
    for (int i = 0; i < UN; ++i)
      if (s0 + i < a.segs - 1) x[i] = m[(int64_t)(s0 + i) * per];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      if (s0 + i >= a.segs - 1) break;
      S.x = fmaf(S.x, fh, fmaf(S.x, fl, x[i].x));
      S.y = fmaf(S.y, fh, fmaf(S.y, fl, x[i].y));
      S.z = fmaf(S.z, fh, fmaf(S.z, fl, x[i].z));
      S.w = fmaf(S.w, fh, fmaf(S.w, fl, x[i].w));
      m[(int64_t)(s0 + i) * per] = S;
    }
  }
}

size_t sums_bytes(const AtlasDecayParams& p, bool bwd) {
  const int segs = split(p, bwd).segs;
  return segs > 1 ? (size_t)chains(p) * segs * p.D * p.D * sizeof(float) : 0;
}

cudaError_t launch_seq(const Args& a, bool bwd, const float* in, float* out, float* saves, float* sums,
                       cudaStream_t s) {
  const AtlasDecayParams& p = a.p;
  const int64_t flat[3] = {(int64_t)p.T * p.H * p.D, (int64_t)p.H * p.D, p.D};
  CUtensorMap mq{}, mx{}, my{};
  bool ok;
  if (bwd)
    ok = make_map(&mx, a.q, p, p.q_stride) && make_map(&my, a.dy, p, flat);
  else
    ok = make_map(&mq, a.q, p, p.q_stride) && make_map(&mx, a.k, p, p.k_stride) && make_map(&my, a.v, p, p.v_stride);
  if (!ok) return cudaErrorInvalidValue;
  const Split z = split(p, bwd);
  const bool wide = p.D > 64;
  SeqArgs q{};
  q.p = p;
  q.log_decay = a.log_decay;
  q.in = in;
  q.out = out;
  q.y = (bf16*)a.y;
  q.saves = nullptr;
  q.segs = z.segs;
  q.seg_blocks = z.blocks;
  q.status = a.status;
  q.sums = sums;
  if (z.segs > 1) {
    q.sums_pass = 1;
    cudaError_t e = wide ? launch<128, false>(mq, mx, my, q, bwd, s) : launch<64, false>(mq, mx, my, q, bwd, s);
    if (e != cudaSuccess) return e;
    q.sums_pass = 0;
    if (join_first(p, z.segs)) {
      q.joined = 1;
      const int64_t n = chains(p) * p.D * p.D / 4;
      e = follow(join_kernel, (unsigned)((n + 255) / 256), 256, 0, s, q);
      if (e != cudaSuccess) return e;
    }
  }
  q.saves = saves;
  if (bwd) return wide ? launch<128, false>(mq, mx, my, q, true, s) : launch<64, false>(mq, mx, my, q, true, s);
  return wide ? launch<128, true>(mq, mx, my, q, false, s) : launch<64, true>(mq, mx, my, q, false, s);
}

}  // namespace tcore
}  // namespace decay
}  // namespace atlas
