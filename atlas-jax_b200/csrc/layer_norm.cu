// Layer norm with a fused residual add (include/atlas_norm.h).
//
// Bound by memory: forward and backward each read every input element once and write every
// output element once; a vector stays in registers between the statistics and the output.
// The variance is summed from (h - mean)^2 over those registers.
//
// A team of lanes owns a vector; lane i holds CHN groups of VEC consecutive channels (16
// bytes where the rows allow it), group j at (j * lanes + i) * VEC.  Teams:
//   SUB    a power of two of lanes (4 .. 32) inside a warp, one group each: short vectors
//          (heads).  The weights repeat every G * N channels, so a thread whose position
//          advances by whole rows keeps its channels: the weight gradients stay in registers.
//   WARP   one warp, CHN groups: up to 32 * VEC * CHN channels
//   BLOCK  all warps of a block: longer vectors
//   BIG    vectors beyond that: the block reads the vector once for each sum
//   TINY   up to 8 channels: one thread in float64.  The gradient of so short a vector
//          cancels (for two channels it is of the order eps / var: the normalised pair is
//          always near +-1), and float32 statistics would leave few of its digits.
// The backward runs a fixed number of blocks; each adds up its rows' weight gradients in
// registers and leaves one partial row, and a second kernel adds those in a fixed order.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "atlas_norm.h"
#include "common.cuh"
#include "scan_internal.h"

namespace atlas {
namespace norm {

typedef __nv_bfloat16 bf16;

struct Args {
  int64_t rows, vecs;  // vecs = rows * G
  int G, N;
  float eps;
  const void *x, *res, *dy, *dh;
  const float *w, *b;
  void *y, *h, *dx;
  float* stats;
  const float* cstats;
  float* part;  // partial rows: dw then db
  int width;    // channels of a partial row
};

// VEC consecutive elements as one load / store
template <typename TA, int VEC>
struct alignas(sizeof(TA) * VEC) Pack {
  TA v[VEC];
};
template <typename TA, int VEC>
__device__ __forceinline__ void load(float* f, const TA* p) {
  const Pack<TA, VEC> k = *(const Pack<TA, VEC>*)p;
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = ld_act(k.v, (size_t)j);
}
template <typename TA, int VEC>
__device__ __forceinline__ void store(TA* p, const float* f) {
  Pack<TA, VEC> k;
#pragma unroll
  for (int j = 0; j < VEC; ++j) st_act(k.v, (size_t)j, f[j]);
  *(Pack<TA, VEC>*)p = k;
}
template <typename TA>
__device__ __forceinline__ float round_to(float x) {
  TA t[1];
  st_act(t, 0, x);
  return ld_act(t, 0);
}
// parameters: float32 rows, VEC at a time where VEC is a multiple of 4 (16-byte aligned then)
template <int VEC>
__device__ __forceinline__ void load_param(float* f, const float* p, float missing) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = missing;
  } else if constexpr (VEC % 4 == 0) {
#pragma unroll
    for (int j = 0; j < VEC; j += 4) *(float4*)(f + j) = *(const float4*)(p + j);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = p[j];
  }
}

enum Team { SUB, WARP, BLOCK };

// Sums of K values over a team; every lane gets them.  BLOCK: `red` holds 2 x 32 x K floats,
// used alternately so that one barrier per call is enough.
template <Team TEAM, int LANES, int K>
__device__ __forceinline__ void team_sum(float* v, float* red, int& turn) {
  constexpr int W = TEAM == SUB ? LANES : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TEAM == BLOCK) {
    float* r = red + turn * 32 * K;
    turn ^= 1;
    const int w = threadIdx.x >> 5, nw = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) r[w * K + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = 0.f;
    for (int i = 0; i < nw; ++i)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += r[i * K + k];
  }
}

// Where this thread's team works: its vectors are first, first + stride, ... and lane /
// lanes place it in the team.  SUB: the position inside a row is fixed, rows advance.
template <Team TEAM, int LANES>
struct Place {
  int64_t first, stride;
  int lane, lanes;
  __device__ __forceinline__ Place(const Args& a, int rows_per_block) {
    if constexpr (TEAM == SUB) {
      const int per_row = a.G * LANES, slot = threadIdx.x / per_row, in_row = threadIdx.x % per_row;
      lane = in_row % LANES;
      lanes = LANES;
      first = ((int64_t)blockIdx.x * rows_per_block + slot) * a.G + in_row / LANES;
      if (slot >= rows_per_block) first = a.vecs;  // spare threads of the last warp
      stride = (int64_t)gridDim.x * rows_per_block * a.G;
    } else if constexpr (TEAM == WARP) {
      lane = threadIdx.x & 31;
      lanes = 32;
      first = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
      stride = (int64_t)gridDim.x * (blockDim.x >> 5);
    } else {
      lane = threadIdx.x;
      lanes = blockDim.x;
      first = blockIdx.x;
      stride = gridDim.x;
    }
  }
};

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
template <typename TA, Team TEAM, int LANES, int VEC, int CHN>
__global__ void __launch_bounds__(TEAM == BLOCK ? 512 : 256) fwd_kernel(Args a, int rows_per_block) {
  __shared__ float red[2 * 32];
  int turn = 0;
  const Place<TEAM, LANES> z(a, rows_per_block);
  const TA *x = (const TA*)a.x, *res = (const TA*)a.res;
  const float inv = 1.f / (float)a.N;
  // every lane of a warp runs the same number of rounds (the shuffles need them all)
  for (int64_t v0 = z.first;; v0 += z.stride) {
    const bool on = v0 < a.vecs;
    if (TEAM == BLOCK ? !on : !__any_sync(0xffffffffu, on)) break;
    const int64_t base = v0 * a.N;
    float f[CHN][VEC], s[1] = {0.f};
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      const int n = (c * z.lanes + z.lane) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[c][j] = 0.f;
      if (on && n < a.N) load<TA, VEC>(f[c], x + base + n);
    }
    if (res) {
#pragma unroll
      for (int c = 0; c < CHN; ++c) {
        const int n = (c * z.lanes + z.lane) * VEC;
        if (on && n < a.N) {
          float r[VEC];
          load<TA, VEC>(r, res + base + n);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[c][j] = round_to<TA>(f[c][j] + r[j]);
          store<TA, VEC>((TA*)a.h + base + n, f[c]);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < CHN; ++c)
#pragma unroll
      for (int j = 0; j < VEC; ++j) s[0] += f[c][j];
    team_sum<TEAM, LANES, 1>(s, red, turn);
    const float mean = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      const int n = (c * z.lanes + z.lane) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        f[c][j] -= mean;
        if (n < a.N) s[0] = fmaf(f[c][j], f[c][j], s[0]);
      }
    }
    team_sum<TEAM, LANES, 1>(s, red, turn);
    const float rstd = 1.f / sqrtf(fmaf(s[0], inv, a.eps));
    if (on && z.lane == 0 && a.stats) *(float2*)(a.stats + 2 * v0) = make_float2(mean, rstd);
    const int g = a.G == 1 ? 0 : (int)(v0 % a.G);
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      const int n = (c * z.lanes + z.lane) * VEC;
      if (on && n < a.N) {
        float w[VEC], b[VEC];
        load_param<VEC>(w, a.w ? a.w + (int64_t)g * a.N + n : nullptr, 1.f);
        load_param<VEC>(b, a.b ? a.b + (int64_t)g * a.N + n : nullptr, 0.f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[c][j] = fmaf(f[c][j] * rstd, w[j], b[j]);
        store<TA, VEC>((TA*)a.y + base + n, f[c]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// With z = (h - mean) rstd and u = dy w:  dx = rstd (u - mean(u) - z mean(u z)) + dh,
// dw += dy z, db += dy.
template <typename TA, Team TEAM, int LANES, int VEC, int CHN>
__global__ void __launch_bounds__(TEAM == BLOCK ? 512 : 256) bwd_kernel(Args a, int rows_per_block) {
  extern __shared__ float acc_sm[];  // WARP, SUB: 2 x width
  __shared__ float red[2 * 32 * 2];
  int turn = 0;
  const Place<TEAM, LANES> z(a, rows_per_block);
  const TA *h = (const TA*)a.h, *dy = (const TA*)a.dy, *dh = (const TA*)a.dh;
  const float inv = 1.f / (float)a.N;
  const int g = a.G == 1 ? 0 : (int)(z.first % a.G);  // the stride is a multiple of G
  float w[CHN][VEC], dw[CHN][VEC], db[CHN][VEC];
#pragma unroll
  for (int c = 0; c < CHN; ++c) {
    const int n = (c * z.lanes + z.lane) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[c][j] = dw[c][j] = db[c][j] = 0.f;
    if (n < a.N) load_param<VEC>(w[c], a.w ? a.w + (int64_t)g * a.N + n : nullptr, 1.f);
  }
  for (int64_t v0 = z.first;; v0 += z.stride) {
    const bool on = v0 < a.vecs;
    if (TEAM == BLOCK ? !on : !__any_sync(0xffffffffu, on)) break;
    const int64_t base = v0 * a.N;
    float f[CHN][VEC], d[CHN][VEC];
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      const int n = (c * z.lanes + z.lane) * VEC;
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[c][j] = d[c][j] = 0.f;
      if (on && n < a.N) {
        load<TA, VEC>(f[c], h + base + n);
        load<TA, VEC>(d[c], dy + base + n);
      }
    }
    float2 st = on ? *(const float2*)(a.cstats + 2 * v0) : make_float2(0.f, 0.f);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      const int n = (c * z.lanes + z.lane) * VEC;
      if (n < a.N) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float zz = (f[c][j] - st.x) * st.y;
          dw[c][j] = fmaf(d[c][j], zz, dw[c][j]);
          db[c][j] += d[c][j];
          const float u = d[c][j] * w[c][j];
          s[0] += u;
          s[1] = fmaf(u, zz, s[1]);
          f[c][j] = zz;
          d[c][j] = u;
        }
      }
    }
    team_sum<TEAM, LANES, 2>(s, red, turn);
    const float m1 = s[0] * inv, m2 = s[1] * inv;
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      const int n = (c * z.lanes + z.lane) * VEC;
      if (on && n < a.N) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[c][j] = st.y * (d[c][j] - m1 - f[c][j] * m2);
        if (dh) {
          load<TA, VEC>(f[c], dh + base + n);
#pragma unroll
          for (int j = 0; j < VEC; ++j) d[c][j] += f[c][j];
        }
        store<TA, VEC>((TA*)a.dx + base + n, d[c]);
      }
    }
  }
  if (!a.part) return;
  float* pw = a.part + (int64_t)blockIdx.x * 2 * a.width;
  float* pb = pw + a.width;
  if constexpr (TEAM == BLOCK) {
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      const int n = (c * z.lanes + z.lane) * VEC;
      if (n < a.N) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          pw[n + j] = dw[c][j];
          pb[n + j] = db[c][j];
        }
      }
    }
  } else {
    // teams of one block with the same channels add up in turn
    float *aw = acc_sm, *ab = acc_sm + a.width;
    const int turns = TEAM == SUB ? rows_per_block : blockDim.x >> 5;
    const int mine = TEAM == SUB ? threadIdx.x / (a.G * LANES) : threadIdx.x >> 5;
    const int off = TEAM == SUB ? g * a.N : 0;
    for (int i = 0; i < turns; ++i) {
      if (i == mine) {
#pragma unroll
        for (int c = 0; c < CHN; ++c) {
          const int n = (c * z.lanes + z.lane) * VEC;
          if (n < a.N) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const int o = off + n + j;
              aw[o] = i == 0 ? dw[c][j] : aw[o] + dw[c][j];
              ab[o] = i == 0 ? db[c][j] : ab[o] + db[c][j];
            }
          }
        }
      }
      __syncthreads();
    }
    for (int o = threadIdx.x; o < a.width; o += blockDim.x) {
      pw[o] = aw[o];
      pb[o] = ab[o];
    }
  }
}

// dw, db (G, N) from the partial rows: channel (g, n) is column (g * N + n) % width of the
// rows p with p % groups == group, groups = G * N / width.
__global__ void __launch_bounds__(1024) param_kernel(Args a, int parts, float* dw, float* db) {
  __shared__ float red[2][32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, col = blockIdx.x * 32 + tx, total = a.G * a.N;
  const int groups = total / a.width;
  float sw = 0.f, sb = 0.f;
  if (col < total) {
    const int grp = col / a.width, n = col % a.width;
    for (int p = grp + ty * groups; p < parts; p += 32 * groups) {
      const float* r = a.part + (int64_t)p * 2 * a.width + n;
      sw += r[0];
      sb += r[a.width];
    }
  }
  red[0][ty][tx] = sw;
  red[1][ty][tx] = sb;
  __syncthreads();
  if (ty < 2) {
    float s = 0.f;
    for (int i = 0; i < 32; ++i) s += red[ty][i][tx];
    float* out = ty ? db : dw;
    if (col < total && out) out[col] = s;
  }
}

// ---------------------------------------------------------------------------
// vectors that do not fit a block's registers
// ---------------------------------------------------------------------------
template <typename TA>
__global__ void __launch_bounds__(512) big_fwd_kernel(Args a) {
  __shared__ float red[2 * 32];
  int turn = 0;
  const float inv = 1.f / (float)a.N;
  for (int64_t v = blockIdx.x; v < a.vecs; v += gridDim.x) {
    const TA *x = (const TA*)a.x + v * a.N, *res = a.res ? (const TA*)a.res + v * a.N : nullptr;
    TA* hh = res ? (TA*)a.h + v * a.N : nullptr;
    const int g = (int)(v % a.G);
    float s[1] = {0.f};
    for (int n = threadIdx.x; n < a.N; n += 512) {  // a thread re-reads only what it wrote to h
      float f = ld_act(x, (size_t)n);
      if (res) {
        f = round_to<TA>(f + ld_act(res, (size_t)n));
        st_act(hh, (size_t)n, f);
      }
      s[0] += f;
    }
    const TA* h = res ? hh : x;
    team_sum<BLOCK, 32, 1>(s, red, turn);
    const float mean = s[0] * inv;
    s[0] = 0.f;
    for (int n = threadIdx.x; n < a.N; n += 512) {
      const float f = ld_act(h, (size_t)n) - mean;
      s[0] = fmaf(f, f, s[0]);
    }
    team_sum<BLOCK, 32, 1>(s, red, turn);
    const float rstd = 1.f / sqrtf(fmaf(s[0], inv, a.eps));
    if (threadIdx.x == 0 && a.stats) *(float2*)(a.stats + 2 * v) = make_float2(mean, rstd);
    for (int n = threadIdx.x; n < a.N; n += 512) {
      const float w = a.w ? a.w[(int64_t)g * a.N + n] : 1.f, b = a.b ? a.b[(int64_t)g * a.N + n] : 0.f;
      st_act((TA*)a.y + v * a.N, (size_t)n, fmaf((ld_act(h, (size_t)n) - mean) * rstd, w, b));
    }
  }
}

// dx; the weight gradients are summed by columns in big_param_kernel, which runs first (dx
// may be the buffer of dy)
template <typename TA>
__global__ void __launch_bounds__(512) big_bwd_kernel(Args a) {
  __shared__ float red[2 * 32 * 2];
  int turn = 0;
  const float inv = 1.f / (float)a.N;
  for (int64_t v = blockIdx.x; v < a.vecs; v += gridDim.x) {
    const TA *h = (const TA*)a.h + v * a.N, *dy = (const TA*)a.dy + v * a.N;
    const TA* dh = a.dh ? (const TA*)a.dh + v * a.N : nullptr;
    const float* w = a.w ? a.w + (v % a.G) * (int64_t)a.N : nullptr;
    const float2 st = *(const float2*)(a.cstats + 2 * v);
    float s[2] = {0.f, 0.f};
    for (int n = threadIdx.x; n < a.N; n += 512) {
      const float u = ld_act(dy, (size_t)n) * (w ? w[n] : 1.f);
      s[0] += u;
      s[1] = fmaf(u, (ld_act(h, (size_t)n) - st.x) * st.y, s[1]);
    }
    team_sum<BLOCK, 32, 2>(s, red, turn);
    for (int n = threadIdx.x; n < a.N; n += 512) {
      const float u = ld_act(dy, (size_t)n) * (w ? w[n] : 1.f), zz = (ld_act(h, (size_t)n) - st.x) * st.y;
      const float d = st.y * (u - s[0] * inv - zz * (s[1] * inv));
      st_act((TA*)a.dx + v * a.N, (size_t)n, d + (dh ? ld_act(dh, (size_t)n) : 0.f));
    }
  }
}
// grid (columns / 256, parts): one thread per channel over every parts-th row
template <typename TA>
__global__ void __launch_bounds__(256) big_param_kernel(Args a) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int total = a.G * a.N;
  if (col >= total) return;
  const int g = (int)(col / a.N);
  float sw = 0.f, sb = 0.f;
  for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const float2 st = *(const float2*)(a.cstats + 2 * (r * a.G + g));
    const float d = ld_act((const TA*)a.dy + r * total, (size_t)col);
    sw = fmaf(d, (ld_act((const TA*)a.h + r * total, (size_t)col) - st.x) * st.y, sw);
    sb += d;
  }
  float* p = a.part + (int64_t)blockIdx.y * 2 * a.width + col;
  p[0] = sw;
  p[a.width] = sb;
}

// ---------------------------------------------------------------------------
// vectors of at most 8 channels; stats holds 1 / deviation as a float pair (the mean is summed again)
// ---------------------------------------------------------------------------
constexpr int TINY = 8;

template <typename TA>
__device__ __forceinline__ double tiny_mean(const TA* h, int N) {
  double s = 0;
  for (int n = 0; n < N; ++n) s += (double)ld_act(h, (size_t)n);
  return s / N;
}
template <typename TA>
__global__ void __launch_bounds__(256) tiny_fwd_kernel(Args a) {
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < a.vecs; v += (int64_t)gridDim.x * 256) {
    const TA* h = (const TA*)a.x + v * a.N;
    if (a.res) {
      TA* hh = (TA*)a.h + v * a.N;
      for (int n = 0; n < a.N; ++n)
        st_act(hh, (size_t)n, ld_act(h, (size_t)n) + ld_act((const TA*)a.res + v * a.N, (size_t)n));
      h = hh;
    }
    const double mean = tiny_mean(h, a.N);
    double s = 0;
    for (int n = 0; n < a.N; ++n) {
      const double d = (double)ld_act(h, (size_t)n) - mean;
      s += d * d;
    }
    const double rstd = 1.0 / sqrt(s / a.N + (double)a.eps);
    if (a.stats) {
      const float hi = (float)rstd;
      *(float2*)(a.stats + 2 * v) = make_float2(hi, isfinite(hi) ? (float)(rstd - (double)hi) : 0.f);
    }
    const int64_t g = v % a.G;
    for (int n = 0; n < a.N; ++n) {
      const double z = ((double)ld_act(h, (size_t)n) - mean) * rstd;
      st_act((TA*)a.y + v * a.N, (size_t)n,
             (float)(z * (a.w ? a.w[g * a.N + n] : 1.f) + (a.b ? a.b[g * a.N + n] : 0.f)));
    }
  }
}
template <typename TA>
__global__ void __launch_bounds__(256) tiny_bwd_kernel(Args a) {
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < a.vecs; v += (int64_t)gridDim.x * 256) {
    const TA *h = (const TA*)a.h + v * a.N, *dy = (const TA*)a.dy + v * a.N;
    const float* w = a.w ? a.w + (v % a.G) * (int64_t)a.N : nullptr;
    const float2 st = *(const float2*)(a.cstats + 2 * v);
    const double mean = tiny_mean(h, a.N), rstd = (double)st.x + (double)st.y;
    double m1 = 0, m2 = 0;
    for (int n = 0; n < a.N; ++n) {
      const double u = (double)ld_act(dy, (size_t)n) * (w ? w[n] : 1.f);
      m1 += u;
      m2 += u * (((double)ld_act(h, (size_t)n) - mean) * rstd);
    }
    m1 /= a.N, m2 /= a.N;
    double d[TINY];  // dx may be the buffer of dy: read all of it first
    for (int n = 0; n < a.N; ++n) {
      const double u = (double)ld_act(dy, (size_t)n) * (w ? w[n] : 1.f);
      d[n] = rstd * (u - m1 - ((double)ld_act(h, (size_t)n) - mean) * rstd * m2);
      if (a.dh) d[n] += (double)ld_act((const TA*)a.dh + v * a.N, (size_t)n);
    }
    for (int n = 0; n < a.N; ++n) st_act((TA*)a.dx + v * a.N, (size_t)n, (float)d[n]);
  }
}
// grid (columns / 256, parts), like big_param_kernel
template <typename TA>
__global__ void __launch_bounds__(256) tiny_param_kernel(Args a) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int total = a.G * a.N;
  if (col >= total) return;
  const int64_t g = col / a.N;
  double sw = 0, sb = 0;
  for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const TA* h = (const TA*)a.h + r * total + g * a.N;
    const float2 st = *(const float2*)(a.cstats + 2 * (r * a.G + g));
    const double d = (double)ld_act((const TA*)a.dy + r * total, (size_t)col);
    sw += d * (((double)ld_act(h, (size_t)(col - g * a.N)) - tiny_mean(h, a.N)) * ((double)st.x + (double)st.y));
    sb += d;
  }
  float* p = a.part + (int64_t)blockIdx.y * 2 * a.width + col;
  p[0] = (float)sw;
  p[a.width] = (float)sb;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int PARTS = 592;  // most blocks of the backward (and partial rows): 4 per SM
constexpr int BIG_PARTS = 64;
constexpr int MAX_GN = 1 << 20;

static int check(const AtlasNormParams* p) {
  if (!p) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "params is NULL");
  if (p->abi_version != ATLAS_ABI_VERSION) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "abi_version mismatch");
  if (p->act_dtype != ATLAS_F32 && p->act_dtype != ATLAS_BF16)
    return report_error(ATLAS_ERR_INVALID_ARGUMENT, "act_dtype must be ATLAS_F32 or ATLAS_BF16");
  if (p->rows < 0 || p->G < 1 || p->N < 1)
    return report_error(ATLAS_ERR_INVALID_ARGUMENT, "rows must not be negative, G and N must be positive");
  if ((int64_t)p->G * p->N > MAX_GN)
    return report_error(ATLAS_ERR_UNSUPPORTED, "layer norm: G * N must be at most 2^20");
  if (p->rows > ((int64_t)1 << 50) / ((int64_t)p->G * p->N))
    return report_error(ATLAS_ERR_UNSUPPORTED, "layer norm: rows * G * N must be at most 2^50");
  if (!(p->eps >= 0.f) || !std::isfinite(p->eps))
    return report_error(ATLAS_ERR_INVALID_ARGUMENT, "eps must be finite and not negative");
  clear_error();
  return ATLAS_OK;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static int status_of(cudaError_t e) {
  return e == cudaSuccess ? ATLAS_OK : report_error(ATLAS_ERR_CUDA, cudaGetErrorString(e));
}

// How a problem runs.  VEC: channels per load; SUB for vectors of 2 to 32 aligned groups,
// a power of two, where the row of G vectors fits a block; TINY for up to 8 channels; else WARP up to 4 groups (16
// bytes) or 8 single channels a lane; else BLOCK up to 2 bf16 groups, 4 float32 groups or 8
// single channels a thread (what the backward holds without spilling); else BIG.
struct Plan {
  bool big, tiny;
  Team team;
  int vec, lanes, chn, threads, rows_per_block, width, parts;
  int64_t grid;
};
static Plan plan(const Args& a, int act_dtype, bool vec_ok, bool bwd) {
  Plan z{};
  const int full = act_dtype == ATLAS_BF16 ? 8 : 4;
  z.vec = vec_ok && a.N % full == 0 ? full : 1;
  const int groups = (a.N + z.vec - 1) / z.vec;
  const bool pow2 = (groups & (groups - 1)) == 0;
  z.rows_per_block = 1;
  int64_t units;  // blocks' worth of work
  if (a.N <= TINY) {
    z.tiny = true;
    z.width = a.G * a.N;
    units = (a.vecs + 255) / 256;
  } else if (z.vec > 1 && pow2 && groups >= 4 && groups <= 32 && (int64_t)a.G * groups <= 256) {
    z.team = SUB;
    z.lanes = groups;
    z.chn = 1;
    z.rows_per_block = 256 / (a.G * groups);
    z.threads = (z.rows_per_block * a.G * groups + 31) / 32 * 32;
    z.width = a.G * a.N;
    units = (a.rows + z.rows_per_block - 1) / z.rows_per_block;
  } else if (groups <= (z.vec > 1 ? 128 : 256) && (a.G == 1 || !bwd)) {
    z.team = WARP;
    z.lanes = 32;
    z.chn = (groups + 31) / 32;
    z.threads = 256;
    z.width = a.N;
    units = (a.vecs + 7) / 8;
  } else if (groups <= 512 * (z.vec == 8 ? 2 : z.vec == 4 ? 4 : 8)) {
    z.team = BLOCK;
    z.lanes = 0;
    z.chn = (groups + 511) / 512;
    z.width = a.N;
    units = a.vecs;
  } else {
    z.big = true;
    z.width = a.G * a.N;
    units = a.vecs;
  }
  if (!z.big && !z.tiny) {
    if (z.vec == 1) z.chn = z.chn <= 4 ? 4 : 8;
    if (z.team == BLOCK) z.threads = ((groups + z.chn - 1) / z.chn + 31) / 32 * 32;
  }
  const int64_t most = bwd ? PARTS : 148 * 16;
  z.grid = std::max<int64_t>(1, std::min(units, most));
  if (bwd && !z.big && !z.tiny && z.team == BLOCK) {  // a multiple of G: each block keeps one group's weights
    z.grid = std::min<int64_t>(units, std::max<int64_t>(a.G, z.grid / a.G * a.G));
  }
  z.parts = (int)(z.big || z.tiny ? std::min<int64_t>(z.big ? BIG_PARTS : PARTS, std::max<int64_t>(1, a.rows)) : z.grid);
  return z;
}

// partial rows of the backward, over either alignment
static size_t ws_bytes(const AtlasNormParams& p) {
  Args a{};
  a.rows = p.rows, a.vecs = p.rows * p.G, a.G = p.G, a.N = p.N;
  size_t n = 0;
  for (bool v : {false, true}) {
    const Plan z = plan(a, p.act_dtype, v, true);
    n = std::max(n, (size_t)z.parts * 2 * z.width * sizeof(float));
  }
  return n;
}

template <typename TA, Team TEAM, int LANES, int VEC, int CHN>
static cudaError_t go(const Args& a, const Plan& z, bool bwd, cudaStream_t s) {
  if (bwd) {
    const size_t sm = TEAM == BLOCK ? 0 : (size_t)2 * z.width * sizeof(float);
    bwd_kernel<TA, TEAM, LANES, VEC, CHN><<<(unsigned)z.grid, z.threads, sm, s>>>(a, z.rows_per_block);
  } else {
    fwd_kernel<TA, TEAM, LANES, VEC, CHN><<<(unsigned)z.grid, z.threads, 0, s>>>(a, z.rows_per_block);
  }
  return cudaGetLastError();
}
template <typename TA, Team TEAM, int VEC>
static cudaError_t by_chn(const Args& a, const Plan& z, bool bwd, cudaStream_t s) {
  if constexpr (VEC > 1) {
    if (z.chn == 1) return go<TA, TEAM, 32, VEC, 1>(a, z, bwd, s);
    if constexpr (TEAM == BLOCK && VEC == 8) {
      return go<TA, TEAM, 32, VEC, 2>(a, z, bwd, s);
    } else {
      if (z.chn == 2) return go<TA, TEAM, 32, VEC, 2>(a, z, bwd, s);
      if (z.chn == 3) return go<TA, TEAM, 32, VEC, 3>(a, z, bwd, s);
      return go<TA, TEAM, 32, VEC, 4>(a, z, bwd, s);
    }
  } else {
    return z.chn == 4 ? go<TA, TEAM, 32, 1, 4>(a, z, bwd, s) : go<TA, TEAM, 32, 1, 8>(a, z, bwd, s);
  }
}
template <typename TA, int FULL>
static cudaError_t run(const Args& a, const Plan& z, bool bwd, cudaStream_t s) {
  if (z.tiny) {
    if (!bwd) {
      tiny_fwd_kernel<TA><<<(unsigned)z.grid, 256, 0, s>>>(a);
    } else {
      if (a.part) {
        tiny_param_kernel<TA><<<dim3((a.G * a.N + 255) / 256, z.parts), 256, 0, s>>>(a);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
      }
      tiny_bwd_kernel<TA><<<(unsigned)z.grid, 256, 0, s>>>(a);
    }
    return cudaGetLastError();
  }
  if (z.big) {
    if (!bwd) {
      big_fwd_kernel<TA><<<(unsigned)z.grid, 512, 0, s>>>(a);
    } else {
      if (a.part) {
        big_param_kernel<TA><<<dim3((a.G * a.N + 255) / 256, z.parts), 256, 0, s>>>(a);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
      }
      big_bwd_kernel<TA><<<(unsigned)z.grid, 512, 0, s>>>(a);
    }
    return cudaGetLastError();
  }
  if (z.team == SUB) {
    switch (z.lanes) {
      case 4: return go<TA, SUB, 4, FULL, 1>(a, z, bwd, s);
      case 8: return go<TA, SUB, 8, FULL, 1>(a, z, bwd, s);
      case 16: return go<TA, SUB, 16, FULL, 1>(a, z, bwd, s);
      default: return go<TA, SUB, 32, FULL, 1>(a, z, bwd, s);
    }
  }
  if (z.team == WARP)
    return z.vec > 1 ? by_chn<TA, WARP, FULL>(a, z, bwd, s) : by_chn<TA, WARP, 1>(a, z, bwd, s);
  return z.vec > 1 ? by_chn<TA, BLOCK, FULL>(a, z, bwd, s) : by_chn<TA, BLOCK, 1>(a, z, bwd, s);
}
static cudaError_t launch(const Args& a, const AtlasNormParams& p, const Plan& z, bool bwd, cudaStream_t s) {
  return p.act_dtype == ATLAS_BF16 ? run<bf16, 8>(a, z, bwd, s) : run<float, 4>(a, z, bwd, s);
}

}  // namespace norm
}  // namespace atlas

using namespace atlas;
using namespace atlas::norm;

extern "C" size_t atlas_layernorm_workspace_bytes(const AtlasNormParams* p) {
  if (check(p) != ATLAS_OK) return 0;
  return ws_bytes(*p);
}

extern "C" int atlas_layernorm_fwd(const AtlasNormParams* p, const void* x, const void* residual, const float* weight,
                                   const float* bias, void* y, void* h, float* stats, void* stream) {
  int rc = check(p);
  if (rc) return rc;
  if (p->rows == 0) return ATLAS_OK;
  if (!x || !y || (residual && !h)) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  if ((uintptr_t)stats & 7) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "stats must be 8-byte aligned");
  Args a{};
  a.rows = p->rows, a.vecs = p->rows * p->G, a.G = p->G, a.N = p->N;
  a.eps = p->eps;
  a.x = x, a.res = residual, a.y = y, a.h = h;
  a.w = weight, a.b = bias;
  a.stats = stats;
  const bool v = aligned16(x) && aligned16(y) && aligned16(weight) && aligned16(bias) &&
                 (!residual || (aligned16(residual) && aligned16(h)));
  const Plan z = plan(a, p->act_dtype, v, false);
  a.width = z.width;
  return status_of(launch(a, *p, z, false, (cudaStream_t)stream));
}

extern "C" int atlas_layernorm_bwd(const AtlasNormParams* p, const void* dy, const void* h, const float* weight,
                                   const float* stats, const void* dh, void* dx, float* dweight, float* dbias,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check(p);
  if (rc) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  if (p->rows == 0) {  // no rows: zero parameter gradients
    for (float* g : {dweight, dbias})
      if (g) {
        cudaError_t e = cudaMemsetAsync(g, 0, (size_t)p->G * p->N * sizeof(float), s);
        if (e != cudaSuccess) return status_of(e);
      }
    return ATLAS_OK;
  }
  if (!dy || !h || !stats || !dx) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "a required pointer is NULL");
  if ((uintptr_t)stats & 7) return report_error(ATLAS_ERR_INVALID_ARGUMENT, "stats must be 8-byte aligned");
  const bool params = dweight || dbias;
  if (params && (!workspace || workspace_bytes < ws_bytes(*p)))
    return report_error(ATLAS_ERR_WORKSPACE, "workspace smaller than atlas_layernorm_workspace_bytes()");
  Args a{};
  a.rows = p->rows, a.vecs = p->rows * p->G, a.G = p->G, a.N = p->N;
  a.dy = dy, a.h = const_cast<void*>(h), a.dh = dh, a.dx = dx;
  a.w = weight;
  a.cstats = stats;
  a.part = params ? (float*)workspace : nullptr;
  const bool v = aligned16(dy) && aligned16(h) && aligned16(dx) && aligned16(weight) && (!dh || aligned16(dh));
  const Plan z = plan(a, p->act_dtype, v, true);
  a.width = z.width;
  cudaError_t e = launch(a, *p, z, true, s);
  if (e == cudaSuccess && params) {
    param_kernel<<<(unsigned)((p->G * p->N + 31) / 32), 1024, 0, s>>>(a, z.parts, dweight, dbias);
    e = cudaGetLastError();
  }
  return status_of(e);
}
