// Decay attention (include/atlas_decay.h): entry points, the float32 CUDA-core kernels for
// the calls outside the tensor path (decay_scan.cu, decay_grad.cu), and the recurrent
// single-token form.
//
// A sequence is cut into chunks of CH = 64 tokens.  With L tokens in a chunk, local
// positions t, s and l = exp(log_decay):
//
//   forward   dS[c]     = sum_s l^(L-1-s) k_s v_s^T                   every chunk by itself
//             S[c+1]    = l^L S[c] + dS[c]                            recurrence over chunks
//             y_t       = scale [ sum_{s<=t} l^(t-s) (q_t.k_s) v_s + l^(t+1) q_t^T S[c] ]
//   backward  (o = scale dy)  QO[c] = sum_t l^(t+1) q_t o_t^T,  R[c-1] = l^L R[c] + QO[c]
//             (R[c]: cotangent of the state leaving chunk c)
//             dq_t = sum_{s<=t} l^(t-s) (o_t.v_s) k_s + l^(t+1) S[c] o_t
//             dk_s = sum_{t>=s} l^(t-s) (o_t.v_s) q_t + l^(L-1-s) R[c] v_s
//             dv_s = sum_{t>=s} l^(t-s) (q_t.k_s) o_t + l^(L-1-s) R[c]^T k_s
//             dlog_decay = sum_{s<=t} (t-s) l^(t-s) (q_t.k_s)(o_t.v_s) + sum_t (t+1) q_t.dq_t^inter
//                          + sum_s (L-1-s) k_s.dk_s^inter + L l^L <R[c], S[c]>, over all chunks
//             (the terms of dq and dk that go through S and R are "inter").
//
// Every power of l has an exponent >= 0, so no decay, however strong, overflows.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "decay_internal.h"
#include "scan_internal.h"

namespace atlas {
namespace decay {

// l^n for n >= 0 (l^0 = 1 also for log_decay = -infinity)
__device__ __forceinline__ float pow_decay(float g, int n) { return n == 0 ? 1.f : expf((float)n * g); }

// ---------------------------------------------------------------------------
// recurrence over chunks
// ---------------------------------------------------------------------------
// One thread per 4 (VEC) state elements walks the chunks (backward: from the last one) and
// replaces each chunk's sum by the running state in front of it.  Pure streaming: the loads
// of UN chunks are in flight together, since only the add depends on the previous chunk.
// The per-chunk factor l^L is applied as a float pair (its rounding error would otherwise
// be multiplied in again at every chunk).
template <int VEC>
__global__ void __launch_bounds__(256) scan_kernel(Args a, const float* in, float* out, float* buf, bool bwd) {
  constexpr int UN = 8;
  const AtlasDecayParams& P = a.p;
  let_next_start();
  after_previous();
  const int nc = chunks(P), DD = P.D * P.D, per = DD / VEC;
  const int64_t total = chains(P) * per;
  const int64_t u = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (u >= total) return;
  const int64_t chain = u / per;
  const int e = (int)(u - chain * per) * VEC;
  const double g = (double)a.log_decay[chain % P.H];
  const double f64 = exp(g * CH), fl64 = exp(g * chunk_len(P, nc - 1));
  float S[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) S[j] = in ? in[chain * DD + e + j] : 0.f;
  float* base = buf + chain * nc * DD + e;
  for (int c0 = 0; c0 < nc; c0 += UN) {
    float x[UN][VEC];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int c = bwd ? nc - 1 - (c0 + i) : c0 + i;
      if (c0 + i < nc) {
        if constexpr (VEC == 4)
          *(float4*)x[i] = *(const float4*)(base + (int64_t)c * DD);
        else
          x[i][0] = base[(int64_t)c * DD];
      }
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      if (c0 + i >= nc) break;
      const int c = bwd ? nc - 1 - (c0 + i) : c0 + i;
      const double f = c == nc - 1 ? fl64 : f64;
      const float fh = (float)f, fl = (float)(f - (double)fh);
      if constexpr (VEC == 4)
        *(float4*)(base + (int64_t)c * DD) = *(const float4*)S;
      else
        base[(int64_t)c * DD] = S[0];
#pragma unroll
      for (int j = 0; j < VEC; ++j) S[j] = fmaf(S[j], fh, fmaf(S[j], fl, x[i][j]));
    }
  }
  if (out) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[chain * DD + e + j] = S[j];
  }
}

// dlog_decay[h] = sum over batches and parts, in a fixed order
__global__ void __launch_bounds__(256) dg_kernel(Args a, float* dg) {
  const AtlasDecayParams& P = a.p;
  const int h = blockIdx.x;
  const int64_t n = (int64_t)P.B * a.dg_parts;
  after_previous();
  double acc = 0;
  for (int64_t i = threadIdx.x; i < n; i += 256) {
    const int64_t b = i / a.dg_parts, c = i - b * a.dg_parts;
    acc += (double)a.dg_part[(b * P.H + h) * a.dg_parts + c];
  }
  __shared__ double red[256];
  red[threadIdx.x] = acc;
  __syncthreads();
  for (int k = 128; k > 0; k >>= 1) {
    if (threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) dg[h] = (float)red[0];
}

// ---------------------------------------------------------------------------
// float32 CUDA-core kernels (any D <= 128, strides and alignment; float32 activations)
// ---------------------------------------------------------------------------
// 256 threads as 16 x 16 over token tiles of TT = 32 rows in shared memory, D zero-padded to
// DP.  Thread (ty, tx) owns rows ty and ty + 16 of a tile's product and NJ groups of VW
// consecutive columns; it reads its operands as 16-byte groups (rows along the summed axis,
// columns along the output), so a multiply-add costs a quarter of a shared-memory load or less.
constexpr int TT = 32;
constexpr int LP = TT + 4;  // row pitch of a tile of scores: 16-byte aligned rows

template <int DP>
struct Tile {
  static constexpr int LD = DP + 4;  // row pitch: 16-byte aligned, 8 rows apart in different banks
  static constexpr int VW = DP == 32 ? 2 : 4, NJ = DP / 16 / VW, NC = VW * NJ;  // columns of a thread
  float x[TT][LD];
  static __device__ __forceinline__ int col(int tx, int j) { return VW * tx + 16 * VW * j; }
};

struct View {
  const void* p;
  int64_t sb, st, sh;
};
__device__ __forceinline__ View view(const void* p, const int64_t* s) { return View{p, s[0], s[1], s[2]}; }
__device__ __forceinline__ View flat(const void* p, const AtlasDecayParams& P) {
  return View{p, (int64_t)P.T * P.H * P.D, (int64_t)P.H * P.D, (int64_t)P.D};
}

// rows [t0, t0 + TT) of head (b, h) into a tile; rows from t_end on and columns from D on are
// 0.  vec: groups of four channels can be loaded at once.
template <typename TA, int DP>
__device__ void load_rows(Tile<DP>& tile, const View& x, int b, int h, int t0, int t_end, int D, bool vec) {
  const TA* base = (const TA*)x.p + b * x.sb + h * x.sh;
#pragma unroll
  for (int i = 0; i < TT * DP / 4 / 256; ++i) {
    const int u = threadIdx.x + 256 * i, r = u / (DP / 4), c = 4 * (u % (DP / 4)), t = t0 + r;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (t < t_end && c < D) {
      const TA* p = base + (int64_t)t * x.st + c;
      if (vec) {
        if constexpr (sizeof(TA) == 4) {
          *(float4*)v = *(const float4*)p;
        } else {
          const uint2 k = *(const uint2*)p;
          const __nv_bfloat16* e = (const __nv_bfloat16*)&k;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = __bfloat162float(e[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (c + j < D) v[j] = ld_act(p, (size_t)j);
      }
    }
    *(float4*)&tile.x[r][c] = *(const float4*)v;
  }
}
// columns tx owns, of row r
template <int DP>
__device__ __forceinline__ void row_cols(float* v, const Tile<DP>& t, int r, int tx) {
  using L = Tile<DP>;
#pragma unroll
  for (int j = 0; j < L::NJ; ++j) {
    if constexpr (L::VW == 4)
      *(float4*)(v + 4 * j) = *(const float4*)&t.x[r][L::col(tx, j)];
    else
      *(float2*)v = *(const float2*)&t.x[r][L::col(tx, j)];
  }
}

// per-chunk sums of weight * X^T Y (forward: k, v, l^(L-1-s); bwd: q, scale dy, l^(t+1)).
// 2 x 500 tokens x 8 heads of 48: 6.6 us, the latency of two loads and a chunk's products.
// Thread (ty, tx): rows NR ty + i and its columns.
template <typename TA, int DP>
__global__ void __launch_bounds__(256) sums_kernel(Args a, bool bwd, bool vec) {
  using L = Tile<DP>;
  constexpr int NR = DP / 16;
  __shared__ L X, Y;
  __shared__ float w[CH];
  const AtlasDecayParams& P = a.p;
  let_next_start();
  const int nc = chunks(P), D = P.D;
  const int64_t chain = blockIdx.x / nc;
  const int c = (int)(blockIdx.x % nc), b = (int)(chain / P.H), h = (int)(chain % P.H);
  const int len = chunk_len(P, c), tc = c * CH;
  const float g = a.log_decay[h];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const View xv = bwd ? view(a.q, P.q_stride) : view(a.k, P.k_stride);
  const View yv = bwd ? flat(a.dy, P) : view(a.v, P.v_stride);
  if (threadIdx.x < CH)
    w[threadIdx.x] = bwd ? P.scale * pow_decay(g, threadIdx.x + 1)
                         : (int)threadIdx.x < len ? pow_decay(g, len - 1 - threadIdx.x) : 0.f;
  float acc[NR][L::NC];
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int j = 0; j < L::NC; ++j) acc[i][j] = 0.f;
  for (int s0 = 0; s0 < len; s0 += TT) {
    __syncthreads();
    load_rows<TA>(X, xv, b, h, tc + s0, tc + len, D, vec);
    load_rows<TA>(Y, yv, b, h, tc + s0, tc + len, D, vec);
    __syncthreads();
#pragma unroll 4
    for (int r = 0; r < TT; ++r) {  // rows beyond the chunk are 0
      const float wr = w[s0 + r];
      float xr[NR], yr[L::NC];
#pragma unroll
      for (int i = 0; i < NR; i += 2) {
        const float2 t = *(const float2*)&X.x[r][NR * ty + i];
        xr[i] = wr * t.x;
        xr[i + 1] = wr * t.y;
      }
      row_cols(yr, Y, r, tx);
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < L::NC; ++j) acc[i][j] = fmaf(xr[i], yr[j], acc[i][j]);
    }
  }
  float* out = (bwd ? a.dstates : a.states) + (chain * nc + c) * (int64_t)D * D;
#pragma unroll
  for (int i = 0; i < NR; ++i)
#pragma unroll
    for (int j = 0; j < L::NC; ++j) {
      const int d = NR * ty + i, e = L::col(tx, j / L::VW) + j % L::VW;
      if (d < D && e < D) out[d * D + e] = acc[i][j];
    }
}

// acc (rows ty, ty + 16; the thread's columns) += w_r * sum_m A[r][m] M(m, column) over a D x D
// matrix in global memory; transposed: M(m, c) = M[c][m].  `stage`: two free tiles, SR rows.
template <int DP>
__device__ void times_state(float (*acc)[Tile<DP>::NC], const Tile<DP>& A, const float* M, bool transposed, int D,
                            const float* w, Tile<DP>* stage) {
  using L = Tile<DP>;
  constexpr int SR = DP < 2 * TT ? DP : 2 * TT;
  float(*st)[L::LD] = stage->x;  // the second tile follows the first
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float part[2][L::NC];
#pragma unroll
  for (int j = 0; j < L::NC; ++j) part[0][j] = part[1][j] = 0.f;
  for (int m0 = 0; m0 < D; m0 += SR) {
    if (m0) __syncthreads();
#pragma unroll
    for (int i = 0; i < SR * DP / 256; ++i) {
      const int u = threadIdx.x + 256 * i;
      // consecutive threads along the contiguous axis of M
      const int m = transposed ? u % SR : u / DP, c = transposed ? u / SR : u % DP;
      float x = 0.f;
      if (m0 + m < D && c < D) x = transposed ? M[(int64_t)c * D + m0 + m] : M[(int64_t)(m0 + m) * D + c];
      st[m][c] = x;
    }
    __syncthreads();
    const int n = min(SR, (D - m0 + 3) & ~3);
#pragma unroll 4
    for (int m = 0; m < n; m += 4) {  // rows beyond D are 0
      const float4 a0 = *(const float4*)&A.x[ty][m0 + m], a1 = *(const float4*)&A.x[ty + 16][m0 + m];
      const float p0[4] = {a0.x, a0.y, a0.z, a0.w}, p1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float x[L::NC];
        row_cols(x, stage[(m + k) / TT], (m + k) % TT, tx);
#pragma unroll
        for (int j = 0; j < L::NC; ++j) {
          part[0][j] = fmaf(p0[k], x[j], part[0][j]);
          part[1][j] = fmaf(p1[k], x[j], part[1][j]);
        }
      }
    }
  }
#pragma unroll
  for (int j = 0; j < L::NC; ++j) {
    acc[0][j] = fmaf(w[0], part[0][j], acc[0][j]);
    acc[1][j] = fmaf(w[1], part[1][j], acc[1][j]);
  }
}

__device__ __forceinline__ float dot4(float4 x, float4 y, float s) {
  return fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s))));
}
// (row ty + 16 i) . (row tx + 16 j) for i, j < 2, of two tiles
template <int DP>
__device__ __forceinline__ void dots(float (*p)[2], const Tile<DP>& A, const Tile<DP>& B) {
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  p[0][0] = p[0][1] = p[1][0] = p[1][1] = 0.f;
#pragma unroll 8
  for (int m = 0; m < DP; m += 4) {
    const float4 a0 = *(const float4*)&A.x[ty][m], a1 = *(const float4*)&A.x[ty + 16][m];
    const float4 b0 = *(const float4*)&B.x[tx][m], b1 = *(const float4*)&B.x[tx + 16][m];
    p[0][0] = dot4(a0, b0, p[0][0]);
    p[0][1] = dot4(a0, b1, p[0][1]);
    p[1][0] = dot4(a1, b0, p[1][0]);
    p[1][1] = dot4(a1, b1, p[1][1]);
  }
}
// acc += Pm (32 x 32) B
template <int DP>
__device__ __forceinline__ void times_tile(float (*acc)[Tile<DP>::NC], const float (*Pm)[LP], const Tile<DP>& B) {
  using L = Tile<DP>;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int m = 0; m < TT; m += 4) {
    const float4 a0 = *(const float4*)&Pm[ty][m], a1 = *(const float4*)&Pm[ty + 16][m];
    const float p0[4] = {a0.x, a0.y, a0.z, a0.w}, p1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float x[L::NC];
      row_cols(x, B, m + k, tx);
#pragma unroll
      for (int j = 0; j < L::NC; ++j) {
        acc[0][j] = fmaf(p0[k], x[j], acc[0][j]);
        acc[1][j] = fmaf(p1[k], x[j], acc[1][j]);
      }
    }
  }
}
template <typename TA, int DP>
__device__ void store_rows(void* x, const float (*acc)[Tile<DP>::NC], const AtlasDecayParams& P, int b, int h, int t0,
                           int t_end, float scale) {
  using L = Tile<DP>;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int t = t0 + ty + 16 * i;
    if (t >= t_end) continue;
    TA* row = (TA*)x + (((int64_t)b * P.T + t) * P.H + h) * P.D;
#pragma unroll
    for (int j = 0; j < L::NC; ++j) {
      const int e = L::col(tx, j / L::VW) + j % L::VW;
      if (e < P.D) st_act(row, (size_t)e, scale * acc[i][j]);
    }
  }
}

__device__ __forceinline__ float cta_sum(float v) {  // every thread gets the sum
  __shared__ float red[8];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += red[i];
  return s;
}

struct TilePos {
  int64_t chain;
  int tile, b, h, c, L, tc, r0;  // r0: first row of the tile within its chunk
};
__device__ __forceinline__ TilePos tile_pos(const AtlasDecayParams& P, int64_t index, int tiles) {
  TilePos t;
  t.chain = index / tiles;
  t.tile = (int)(index % tiles);
  t.b = (int)(t.chain / P.H);
  t.h = (int)(t.chain % P.H);
  t.c = t.tile / (CH / TT);
  t.L = chunk_len(P, t.c);
  t.tc = t.c * CH;
  t.r0 = (t.tile % (CH / TT)) * TT;
  return t;
}

// y of one tile of 32 tokens.  2 x 500 tokens x 8 heads of 48: 13 us, the latency of three or four
// loads one after the other and their products.
template <typename TA, int DP>
__global__ void __launch_bounds__(256) out_kernel(Args a, int tiles, bool vec) {
  using L = Tile<DP>;
  extern __shared__ float sm[];
  L &A = *(L*)sm, &K = *(&A + 1), &V = *(&A + 2);
  float(*Pm)[LP] = (float(*)[LP])(&A + 3);
  __shared__ float pw[CH + 1];
  const AtlasDecayParams& P = a.p;
  const TilePos z = tile_pos(P, blockIdx.x, tiles);
  const int D = P.D, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, tend = z.tc + z.L;
  if (threadIdx.x <= CH) pw[threadIdx.x] = pow_decay(a.log_decay[z.h], threadIdx.x);
  load_rows<TA>(A, view(a.q, P.q_stride), z.b, z.h, z.tc + z.r0, tend, D, vec);
  float acc[2][L::NC];
#pragma unroll
  for (int j = 0; j < L::NC; ++j) acc[0][j] = acc[1][j] = 0.f;
  after_previous();  // the states
  __syncthreads();   // pw
  const float w[2] = {pw[z.r0 + ty + 1], pw[z.r0 + ty + 17]};
  times_state<DP>(acc, A, a.states + (z.chain * chunks(P) + z.c) * (int64_t)D * D, false, D, w, &K);
  for (int s0 = 0; s0 <= z.r0; s0 += TT) {
    __syncthreads();
    load_rows<TA>(K, view(a.k, P.k_stride), z.b, z.h, z.tc + s0, tend, D, vec);
    load_rows<TA>(V, view(a.v, P.v_stride), z.b, z.h, z.tc + s0, tend, D, vec);
    __syncthreads();
    float p[2][2];
    dots(p, A, K);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int lag = z.r0 + ty + 16 * i - (s0 + tx + 16 * j);
        Pm[ty + 16 * i][tx + 16 * j] = lag >= 0 ? p[i][j] * pw[lag] : 0.f;
      }
    __syncthreads();
    times_tile<DP>(acc, Pm, V);
  }
  store_rows<TA, DP>(a.y, acc, P, z.b, z.h, z.tc + z.r0, tend, P.scale);
}

// One gradient of one tile of 32 tokens: a product with S or R, and masked scores x with the other
// tokens' rows:
//
//     out = w (X M) + sum over tiles of (weights o X W^T) U      dq: X = dy, M = S^T, W = v,  U = k
//                                                                dk: X = v,  M = R^T, W = dy, U = q
//                                                                dv: X = k,  M = R,   W = q,  U = dy
//
// Three CTAs a tile, each with one accumulator; dk and dv share no product, and a CTA that made both
// was the launch's longest (2 x 500 tokens x 8 heads of 48: 45 us, with three 38).  8 us of that are
// multiply-adds at the full rate, about half of its issue slots; the rest is the latency of four loads, one
// after the other, with five CTAs an SM.  (128 threads of four rows, six CTAs an SM: 32 us with all
// data in L2, but 8 us longer where it comes from memory.)  dq's and dk's CTAs also sum their terms of
// dlog_decay, with Y = q and k.
enum Grad { DK, DV, DQ };
template <typename TA, int DP>
__global__ void __launch_bounds__(256, DP == 128 ? 2 : 4) grads_kernel(Args a, int tiles, bool vec) {
  using L = Tile<DP>;
  extern __shared__ float sm[];
  __shared__ float pw[CH + 1];
  L *const t = (L*)sm, &X = t[0], &Y = t[1], &U = t[2], &W = t[3];
  float(*Pm)[LP] = (float(*)[LP])(t + 4);
  const AtlasDecayParams& P = a.p;
  const TilePos z = tile_pos(P, blockIdx.x / 3, tiles);
  const int kind = blockIdx.x % 3;
  const int D = P.D, tx = threadIdx.x & 15, ty = threadIdx.x >> 4, tend = z.tc + z.L;
  const View q = view(a.q, P.q_stride), k = view(a.k, P.k_stride), v = view(a.v, P.v_stride), o = flat(a.dy, P);
  const View xs = kind == DQ ? o : kind == DK ? v : k, us = kind == DQ ? k : kind == DK ? q : o,
             ws = kind == DQ ? v : kind == DK ? o : q;
  load_rows<TA>(X, xs, z.b, z.h, z.tc + z.r0, tend, D, vec);
  if (kind != DV) load_rows<TA>(Y, kind == DQ ? q : k, z.b, z.h, z.tc + z.r0, tend, D, vec);
  if (threadIdx.x <= CH) pw[threadIdx.x] = pow_decay(a.log_decay[z.h], threadIdx.x);
  let_next_start();
  after_previous();  // R
  __syncthreads();
  float acc[2][L::NC], dg = 0.f;
#pragma unroll
  for (int j = 0; j < L::NC; ++j) acc[0][j] = acc[1][j] = 0.f;
  // steps from the rows to the chunk's start (dq) or end
  const int n0 = kind == DQ ? z.r0 + ty + 1 : z.L - 1 - z.r0 - ty, n1 = kind == DQ ? n0 + 16 : n0 - 16;
  const float s = kind == DQ ? P.scale : 1.f, w[2] = {n0 >= 0 ? s * pw[n0] : 0.f, n1 >= 0 ? s * pw[n1] : 0.f};
  const int64_t so = (z.chain * chunks(P) + z.c) * (int64_t)D * D;
  const float *R = a.dstates + so, *S = a.states + so;
  times_state<DP>(acc, X, kind == DQ ? S : R, kind != DV, D, w, &U);
  if (kind != DV) {  // columns from D on are 0 in Y
    float y0[L::NC], y1[L::NC];
    row_cols(y0, Y, ty, tx);
    row_cols(y1, Y, ty + 16, tx);
#pragma unroll
    for (int j = 0; j < L::NC; ++j) {
      if (n0 > 0) dg += (float)n0 * y0[j] * acc[0][j];
      if (n1 > 0) dg += (float)n1 * y1[j] * acc[1][j];
    }
  }
  if (kind == DQ && z.r0 == 0) {  // once for each chunk, where the loop below is short
    float rs = 0.f;
#pragma unroll 4
    for (int u = threadIdx.x; u < D * D; u += 256) rs = fmaf(R[u], S[u], rs);
    dg += (float)z.L * pw[z.L] * rs;
  }
  for (int s0 = kind == DQ ? 0 : z.r0; s0 < (kind == DQ ? z.r0 + 1 : z.L); s0 += TT) {
    __syncthreads();
    load_rows<TA>(U, us, z.b, z.h, z.tc + s0, tend, D, vec);
    load_rows<TA>(W, ws, z.b, z.h, z.tc + s0, tend, D, vec);
    __syncthreads();
    float x[2][2], p[2][2];
    dots(x, X, W);
    if (kind == DQ) dots(p, Y, U);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int d = z.r0 + ty + 16 * i - (s0 + tx + 16 * j), lag = kind == DQ ? d : -d;
        const float f = lag >= 0 ? P.scale * pw[lag] * x[i][j] : 0.f;
        if (kind == DQ && lag > 0) dg += (float)lag * p[i][j] * f;
        Pm[ty + 16 * i][tx + 16 * j] = f;
      }
    __syncthreads();
    times_tile<DP>(acc, Pm, U);
  }
  store_rows<TA, DP>(kind == DQ ? a.dq : kind == DK ? a.dk : a.dv, acc, P, z.b, z.h, z.tc + z.r0, tend, 1.f);
  if (kind == DV) return;
  dg = cta_sum(dg);
  if (threadIdx.x == 0) a.dg_part[z.chain * a.dg_parts + (kind == DQ ? 0 : tiles) + z.tile] = dg;
}

// ---------------------------------------------------------------------------
// recurrent form
// ---------------------------------------------------------------------------
// One CTA per (sequence, head, slice of SL value columns): the columns of the state are
// independent, so a slice needs no exchange with the others.  Thread (row group rg, column
// group cg) keeps rows rg, rg + RG, ... of VEC consecutive columns in registers from the
// first token to the last; y's sum over rows goes through shared memory.  The decay is applied as a
// float pair, as along a sequence: rounded to one float32 its error would be multiplied in again at
// every token, for as long as the state is kept (2.1e-5 of the state after 4096 at 1 - 2^-9).  Bound by the state's
// bytes where there are many sequences: SL = 64 then moves four 16-byte groups a thread
// (DP = 64), 32 twice as many CTAs for few sequences (256 x 12 heads of 64: 27 us with SL = 32).
// 256 sequences x 12 heads of 64: 21 us, 4.8 TB/s; one sequence: 2.5 us, most of it the launch.  Several
// tokens wait for their q, k and v one after the other: 128 sequences x 4 heads of 128 in float32, two
// tokens 18 us, five 26 (floor 11).
template <typename TA, int DP, int SL, int VEC>
__global__ void __launch_bounds__(256) step_kernel(Args a, const float* in, const int32_t* slots, int32_t n_slots,
                                                   float* out) {
  constexpr int CG = SL / VEC, RG = 256 / CG, NR = DP / RG;  // column groups, row groups, rows a thread
  static_assert(CG <= 32 && NR >= 1, "a warp holds whole rows of a slice");
  __shared__ float red[8][SL + 1], qs[DP], ks[DP];
  __shared__ float2 decay;
  const AtlasDecayParams& P = a.p;
  const int D = P.D, slices = (D + SL - 1) / SL;
  const int chain = blockIdx.x / slices, sl = blockIdx.x % slices, b = chain / P.H, h = chain % P.H;
  const int cg = threadIdx.x % CG, rg = threadIdx.x / CG, e0 = SL * sl + cg * VEC;
  const int32_t row = slots ? slots[b] : b;
  TA* y = (TA*)a.y + ((int64_t)b * P.T * P.H + h) * D;
  if (slots && (row < 0 || row >= n_slots)) {  // idle
    for (int u = threadIdx.x; u < P.T * SL; u += 256) {
      const int t = u / SL, e = SL * sl + u % SL;
      if (e < D) st_act(y + (int64_t)t * P.H * D, (size_t)e, 0.f);
    }
    return;
  }
  const int64_t off = ((int64_t)row * P.H + h) * D * D + rg * D + e0;
  if (threadIdx.x == 255) {
    const double l = exp((double)a.log_decay[h]);
    const float lh = (float)l;
    decay = make_float2(lh, (float)(l - (double)lh));
  }
  const TA* q = (const TA*)a.q + b * P.q_stride[0] + h * P.q_stride[2];
  const TA* k = (const TA*)a.k + b * P.k_stride[0] + h * P.k_stride[2];
  const TA* v = (const TA*)a.v + b * P.v_stride[0] + h * P.v_stride[2];
  float S[NR][VEC];
#pragma unroll
  for (int i = 0; i < NR; ++i) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) S[i][j] = 0.f;
    if (in && rg + i * RG < D && e0 < D) {
      if constexpr (VEC == 4)
        *(float4*)S[i] = *(const float4*)(in + off + i * RG * D);
      else
        S[i][0] = in[off + i * RG * D];
    }
  }
  for (int t = 0; t < P.T; ++t) {
    if (threadIdx.x < DP)
      qs[threadIdx.x] = (int)threadIdx.x < D ? ld_act(q + t * P.q_stride[1], (size_t)threadIdx.x) : 0.f;
    else if (threadIdx.x < 2 * DP)
      ks[threadIdx.x - DP] =
          (int)threadIdx.x - DP < D ? ld_act(k + t * P.k_stride[1], (size_t)(threadIdx.x - DP)) : 0.f;
    float vv[VEC], acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      vv[j] = e0 + j < D ? ld_act(v + t * P.v_stride[1], (size_t)(e0 + j)) : 0.f;
      acc[j] = 0.f;
    }
    __syncthreads();
    const float lh = decay.x, ll = decay.y;
#pragma unroll
    for (int i = 0; i < NR; ++i) {  // rows from D on: k = q = 0
      const float kd = ks[rg + i * RG], qd = qs[rg + i * RG];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        S[i][j] = fmaf(lh, S[i][j], fmaf(ll, S[i][j], kd * vv[j]));
        acc[j] = fmaf(qd, S[i][j], acc[j]);
      }
    }
    // rows of this warp (lanes CG apart), then warps through shared memory
#pragma unroll
    for (int o = CG; o < 32; o <<= 1)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
    if ((threadIdx.x & 31) < CG) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) red[threadIdx.x >> 5][cg * VEC + j] = acc[j];
    }
    __syncthreads();
    if (threadIdx.x < SL) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s += red[i][threadIdx.x];
      const int e = SL * sl + threadIdx.x;
      if (e < D) st_act(y + (int64_t)t * P.H * D, (size_t)e, P.scale * s);
    }
  }
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    if (rg + i * RG < D && e0 < D) {
      if constexpr (VEC == 4)
        *(float4*)(out + off + i * RG * D) = *(const float4*)S[i];
      else
        out[off + i * RG * D] = S[i][0];
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
static int check(const AtlasDecayParams* p) {
  if (!p) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "params is NULL");
  if (p->abi_version != ATLAS_ABI_VERSION) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "abi_version mismatch");
  if (p->B < 0 || p->T < 0 || p->H < 0 || p->D < 1)
    return report_error(ATLAS_ERR_INVALID_ARGUMENT, "B, T and H must not be negative and D must be positive");
  if (p->D > 128) return report_error(ATLAS_ERR_UNSUPPORTED, "decay attention: head_dim D must be at most 128");
  if (p->act_dtype != ATLAS_F32 && p->act_dtype != ATLAS_BF16)
    return report_error(ATLAS_ERR_INVALID_ARGUMENT, "act_dtype must be ATLAS_F32 or ATLAS_BF16");
  if (!std::isfinite(p->scale)) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "scale must be finite");
  for (const int64_t* s : {p->q_stride, p->k_stride, p->v_stride})
    if (s[0] < 0 || s[1] < 0 || s[2] < 0)
      return report_error(ATLAS_ERR_INVALID_ARGUMENT, "strides must not be negative");
  if (p->T > 1 << 30) return report_error(ATLAS_ERR_UNSUPPORTED, "decay attention: T must be at most 2^30");
  // grids are one-dimensional: (batch, head, 32-token tile, gradient) and (batch, head, state element / 256)
  if (chains(*p) > INT32_MAX / std::max(6 * chunks(*p), 64))  // (a product of the three could pass 2^63)
    return report_error(ATLAS_ERR_UNSUPPORTED, "decay attention: B * H * T is too large for one call");
  clear_error();
  return ATLAS_OK;
}

static size_t state_bytes(const AtlasDecayParams& p) {
  return (size_t)chains(p) * chunks(p) * p.D * p.D * sizeof(float);
}
static int parts(const AtlasDecayParams& p) { return 2 * chunks(p) * (CH / TT); }  // of dlog_decay per chain
static int status_of(cudaError_t e) {
  return e == cudaSuccess ? ATLAS_OK : report_error(ATLAS_ERR_CUDA, cudaGetErrorString(e));
}
static bool empty(const AtlasDecayParams& p) { return chains(p) == 0; }

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
// The tensor path moves 16-byte groups of 8 channels by TMA.  Params alone decide.
static bool tensor_path(const AtlasDecayParams& p) {
  return p.act_dtype == ATLAS_BF16 && p.D % 8 == 0 && p.aligned16 && tcore::mappable(p, p.q_stride) &&
         tcore::mappable(p, p.k_stride) && tcore::mappable(p, p.v_stride);
}
// workspaces: the sums of a split walk (tensor path); the chunks' states, where they are not kept
static size_t fwd_bytes(const AtlasDecayParams& p, bool saved) {
  return tensor_path(p) ? tcore::sums_bytes(p, false) : saved ? 0 : state_bytes(p);
}
// the chunks' cotangent states, the sums of their walk, the parts of dlog_decay
static size_t bwd_states(const AtlasDecayParams& p) { return state_bytes(p) + (tensor_path(p) ? tcore::sums_bytes(p, true) : 0); }
static size_t bwd_bytes(const AtlasDecayParams& p) {
  return bwd_states(p) + (size_t)chains(p) * parts(p) * sizeof(float);
}
// the pointers that a call promises to be 16-byte aligned
template <class... T>
static int check_aligned(const AtlasDecayParams& p, T... ptr) {
  if (!p.aligned16) return ATLAS_OK;
  for (const void* x : {(const void*)ptr...})
    if (!aligned16(x)) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "aligned16 is set, but a buffer is not 16-byte aligned");
  return ATLAS_OK;
}

static cudaError_t scan(const Args& a, const float* in, float* out, bool bwd, cudaStream_t s) {
  float* buf = bwd ? a.dstates : a.states;
  const bool v4 = a.p.D % 2 == 0 && aligned16(in) && aligned16(out) && aligned16(buf);  // D * D % 4 == 0
  const int64_t n = chains(a.p) * a.p.D * a.p.D / (v4 ? 4 : 1);
  const unsigned grid = (unsigned)((n + 255) / 256);
  return follow(v4 ? scan_kernel<4> : scan_kernel<1>, grid, 256, 0, s, a, in, out, buf, bwd);
}

// whether groups of four channels of every tensor can be loaded at once
static bool vec4(const Args& a) {
  const AtlasDecayParams& p = a.p;
  const int64_t bytes = p.act_dtype == ATLAS_BF16 ? 2 : 4;
  int64_t all = p.D * bytes;
  for (const int64_t* s : {p.q_stride, p.k_stride, p.v_stride}) all |= s[0] * bytes | s[1] * bytes | s[2] * bytes;
  for (const void* x : {a.q, a.k, a.v, a.dy}) all |= (int64_t)(uintptr_t)x;
  return all % (4 * bytes) == 0;
}
// the CUDA-core kernels for one activation type and padded head size
enum Phase { SUMS_FWD, SUMS_BWD, OUT, GRADS };
template <typename TA, int DP>
static cudaError_t plain_dp(const Args& a, Phase f, cudaStream_t s) {
  const int tiles = (a.p.T + TT - 1) / TT;
  const bool vec = vec4(a);
  const auto smem = [](int n, int squares) { return n * sizeof(Tile<DP>) + (size_t)squares * TT * LP * sizeof(float); };
  if (f == OUT) {
    const cudaError_t e = allow_smem<out_kernel<TA, DP>>(smem(3, 1));
    if (e != cudaSuccess) return e;
    return follow(out_kernel<TA, DP>, (unsigned)(chains(a.p) * tiles), 256, smem(3, 1), s, a, tiles, vec);
  } else if (f == GRADS) {
    const cudaError_t e = allow_smem<grads_kernel<TA, DP>>(smem(4, 1));
    if (e != cudaSuccess) return e;
    return follow(grads_kernel<TA, DP>, (unsigned)(chains(a.p) * tiles * 3), 256, smem(4, 1), s, a, tiles, vec);
  } else {
    sums_kernel<TA, DP><<<(unsigned)(chains(a.p) * chunks(a.p)), 256, 0, s>>>(a, f == SUMS_BWD, vec);
  }
  return cudaGetLastError();
}
template <typename TA>
static cudaError_t plain_t(const Args& a, Phase f, cudaStream_t s) {
  return a.p.D <= 32 ? plain_dp<TA, 32>(a, f, s) : a.p.D <= 64 ? plain_dp<TA, 64>(a, f, s) : plain_dp<TA, 128>(a, f, s);
}
static cudaError_t plain(const Args& a, Phase f, cudaStream_t s) {
  return a.p.act_dtype == ATLAS_BF16 ? plain_t<__nv_bfloat16>(a, f, s) : plain_t<float>(a, f, s);
}
// the states entering every chunk (bwd: leaving), from the chunks' sums
static cudaError_t plain_states(const Args& a, const float* in, float* out, bool bwd, cudaStream_t s) {
  const cudaError_t e = plain(a, bwd ? SUMS_BWD : SUMS_FWD, s);
  return e == cudaSuccess ? scan(a, in, out, bwd, s) : e;
}

// out = in (or zeros): what an empty sequence leaves
static cudaError_t pass_state(const AtlasDecayParams& p, const float* in, float* out, cudaStream_t s) {
  if (!out || in == out) return cudaSuccess;
  const size_t n = (size_t)chains(p) * p.D * p.D * sizeof(float);
  return in ? cudaMemcpyAsync(out, in, n, cudaMemcpyDeviceToDevice, s) : cudaMemsetAsync(out, 0, n, s);
}

template <typename TA, int DP, int SL, int VEC>
static cudaError_t step_go(const Args& a, const float* in, const int32_t* slots, int32_t n, float* out, cudaStream_t s) {
  step_kernel<TA, DP, SL, VEC><<<(unsigned)(chains(a.p) * ((a.p.D + SL - 1) / SL)), 256, 0, s>>>(a, in, slots, n, out);
  return cudaGetLastError();
}
template <typename TA, int DP>
static cudaError_t step_dp(const Args& a, const float* in, const int32_t* slots, int32_t n, float* out, cudaStream_t s) {
  if (a.p.D % 4 != 0 || !aligned16(in) || !aligned16(out)) return step_go<TA, DP, 32, 1>(a, in, slots, n, out, s);
  return chains(a.p) < 2 * 148 ? step_go<TA, DP, 32, 4>(a, in, slots, n, out, s)
                               : step_go<TA, DP, 64, 4>(a, in, slots, n, out, s);
}
template <typename TA>
static cudaError_t step_t(const Args& a, const float* in, const int32_t* slots, int32_t n, float* out, cudaStream_t s) {
  return a.p.D <= 64 ? step_dp<TA, 64>(a, in, slots, n, out, s) : step_dp<TA, 128>(a, in, slots, n, out, s);
}

}  // namespace decay
}  // namespace atlas

using namespace atlas;
using namespace atlas::decay;

extern "C" size_t atlas_decay_saved_bytes(const AtlasDecayParams* p) {
  if (check(p) != ATLAS_OK) return 0;
  return state_bytes(*p);
}

extern "C" size_t atlas_decay_fwd_workspace_bytes(const AtlasDecayParams* p) {
  if (check(p) != ATLAS_OK) return 0;
  return fwd_bytes(*p, false);
}

extern "C" size_t atlas_decay_saved_workspace_bytes(const AtlasDecayParams* p) {
  if (check(p) != ATLAS_OK) return 0;
  return fwd_bytes(*p, true);
}

extern "C" size_t atlas_decay_bwd_workspace_bytes(const AtlasDecayParams* p) {
  if (check(p) != ATLAS_OK) return 0;
  return bwd_bytes(*p);
}

extern "C" int atlas_decay_fwd(const AtlasDecayParams* p, const void* q, const void* k, const void* v,
                               const float* log_decay, const float* state_in, void* y, float* state_out, void* saved,
                               void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(p);
  if (rc) return rc;
  if (empty(*p)) return ATLAS_OK;
  cudaStream_t s = (cudaStream_t)stream;
  if (!state_out || !log_decay) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  if (p->T == 0) return status_of(pass_state(*p, state_in, state_out, s));
  if (!q || !k || !v || !y) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  const size_t need = fwd_bytes(*p, saved != nullptr);
  if (need && (!workspace || workspace_bytes < need))
    return report_error(ATLAS_ERR_WORKSPACE, "workspace smaller than atlas_decay_fwd_workspace_bytes() (with saved: "
                                             "atlas_decay_saved_workspace_bytes())");
  rc = check_aligned(*p, q, k, v, y, state_in, state_out, saved, need ? workspace : nullptr);
  if (rc) return rc;
  Args a{};
  a.p = *p;
  a.q = q, a.k = k, a.v = v;
  a.log_decay = log_decay;
  a.y = y;
  a.states = (float*)(saved ? saved : workspace);
  a.status = device_status_ptr();
  if (tensor_path(*p)) return status_of(tcore::launch_seq(a, false, state_in, state_out, (float*)saved, (float*)workspace, s));
  cudaError_t e = plain_states(a, state_in, state_out, false, s);
  if (e == cudaSuccess) e = plain(a, OUT, s);
  return status_of(e);
}

extern "C" int atlas_decay_bwd(const AtlasDecayParams* p, const void* q, const void* k, const void* v,
                               const float* log_decay, const void* saved, const void* dy, const float* dstate_out,
                               void* dq, void* dk, void* dv, float* dlog_decay, float* dstate_in, void* workspace,
                               size_t workspace_bytes, void* stream) {
  int rc = check(p);
  if (rc) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  if (empty(*p) || p->T == 0) {
    if (p->H > 0 && dlog_decay) {
      // an empty sequence passes the state through: no decay is applied
      cudaError_t e = cudaMemsetAsync(dlog_decay, 0, (size_t)p->H * sizeof(float), s);
      if (e != cudaSuccess) return status_of(e);
    }
    return empty(*p) ? ATLAS_OK : status_of(pass_state(*p, dstate_out, dstate_in, s));
  }
  if (!q || !k || !v || !log_decay || !saved || !dy || !dq || !dk || !dv)
    return report_error(ATLAS_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  if (!workspace || workspace_bytes < bwd_bytes(*p))
    return report_error(ATLAS_ERR_WORKSPACE, "workspace smaller than atlas_decay_bwd_workspace_bytes()");
  rc = check_aligned(*p, q, k, v, dy, dq, dk, dv, saved, dstate_out, dstate_in, workspace);
  if (rc) return rc;
  Args a{};
  a.p = *p;
  a.q = q, a.k = k, a.v = v, a.dy = dy;
  a.log_decay = log_decay;
  a.dq = dq, a.dk = dk, a.dv = dv;
  a.states = (float*)const_cast<void*>(saved);
  a.dstates = (float*)workspace;
  a.dg_part = (float*)((uint8_t*)workspace + bwd_states(*p));
  a.status = device_status_ptr();
  const bool tensor = tensor_path(*p);
  a.dg_parts = tensor ? chunks(*p) : 2 * ((p->T + TT - 1) / TT);
  cudaError_t e = tensor ? tcore::launch_seq(a, true, dstate_out, dstate_in, a.dstates, (float*)workspace + state_bytes(*p) / sizeof(float), s)
                         : plain_states(a, dstate_out, dstate_in, true, s);
  if (e == cudaSuccess) e = tensor ? tcore::launch_grads(a, s) : plain(a, GRADS, s);
  if (e == cudaSuccess && dlog_decay) {
    e = follow(dg_kernel, p->H, 256, 0, s, a, dlog_decay);
  }
  return status_of(e);
}

extern "C" int atlas_decay_step(const AtlasDecayParams* p, const void* q, const void* k, const void* v,
                                const float* log_decay, const float* state_in, const int32_t* slots, int32_t n_slots,
                                void* y, float* state_out, void* stream) {
  int rc = check(p);
  if (rc) return rc;
  if (empty(*p)) return ATLAS_OK;
  if (!state_in || !state_out || !log_decay)
    return report_error(ATLAS_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  if (slots && n_slots < 0) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "n_slots must not be negative");
  if (p->T > 0 && (!q || !k || !v || !y)) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  Args a{};
  a.p = *p;
  a.q = q, a.k = k, a.v = v, a.y = y;
  a.log_decay = log_decay;
  cudaStream_t s = (cudaStream_t)stream;
  return status_of(p->act_dtype == ATLAS_BF16 ? step_t<__nv_bfloat16>(a, state_in, slots, n_slots, state_out, s)
                                              : step_t<float>(a, state_in, slots, n_slots, state_out, s));
}
