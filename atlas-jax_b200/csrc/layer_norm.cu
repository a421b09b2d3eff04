// Layer norm with a fused residual add (include/atlas_norm.h).
//
// Bound by memory: forward and backward each read every input element once and write every
// output element once; a vector stays in registers between the statistics and the output.
// The variance is summed from (h - mean)^2 over those registers; a mean far above the deviation is
// corrected once (far() below).
//
// A team of lanes owns a vector; lane i holds CHN groups of VEC consecutive channels (16
// bytes where the rows allow it), group j at (j * lanes + i) * VEC.  Teams:
//   SUB    a power of two of lanes (4 .. 32) inside a warp, one group each: short vectors
//          (heads).  The weights repeat every G * N channels, so a thread whose position
//          advances by whole rows keeps its channels: the weight gradients stay in registers.
//   WARPS  1 to 16 whole warps; several teams share a block while they fit 8 warps, each with
//          a named barrier of its own for its sums
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
#include "f32x2.cuh"
#include "follow.cuh"
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
// A group as pairs (the backward is as near to the issue limit as to the memory's); a single
// channel is a pair with a zero.
template <int VEC>
constexpr int PAIRS = (VEC + 1) / 2;
template <typename TA, int VEC>
__device__ __forceinline__ void unpack2(F2* f, const Pack<TA, VEC>& k) {
  if constexpr (sizeof(TA) == 2 && VEC > 1) {
    const uint32_t* h = (const uint32_t*)&k;
#pragma unroll
    for (int j = 0; j < PAIRS<VEC>; ++j) f[j] = bf2_unpack(h[j]);
  } else if constexpr (VEC > 1) {
    const uint64_t* h = (const uint64_t*)&k;
#pragma unroll
    for (int j = 0; j < PAIRS<VEC>; ++j) f[j].v = h[j];
  } else {
    f[0] = f2(ld_act(k.v, 0), 0.f);
  }
}
template <typename TA, int VEC>
__device__ __forceinline__ void store2(TA* p, const F2* f) {
  if constexpr (VEC > 1) {
    Pack<TA, VEC> k;
#pragma unroll
    for (int j = 0; j < PAIRS<VEC>; ++j) {
      if constexpr (sizeof(TA) == 2)
        ((uint32_t*)&k)[j] = bf2_pack(f[j]);
      else
        ((uint64_t*)&k)[j] = f[j].v;
    }
    *(Pack<TA, VEC>*)p = k;
  } else {
    st_act(p, 0, f2_get(f[0]).x);
  }
}
// 16 bytes from global to this thread's own slot in shared memory, without registers
__device__ __forceinline__ void copy16(void* slot, const void* g) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(slot)), "l"(g)
               : "memory");
}
enum Team { SUB, ONE, MANY };  // MANY: WARPS teams of more than one warp

// n elements from element o on of a tensor of `total`, at any alignment, into a slot of shared memory: the
// aligned 16-byte pieces that hold them, copied by the lanes of a team (which have to meet before they
// read).  Pieces reach into the neighbouring vectors, but not beyond the tensor: at its ends
// single elements.  The vector starts at offset span_shift() of the slot.
template <typename TA>
__device__ __forceinline__ int span_shift(const TA* t, int64_t o) {
  return (int)((uintptr_t)(t + o) & 15) / (int)sizeof(TA);
}
template <typename TA>
__device__ __forceinline__ void copy_span(uint8_t* slot, const TA* t, int64_t o, int n, int64_t total, int lane,
                                          int lanes) {
  const uintptr_t lo = (uintptr_t)(t + o), hi = (uintptr_t)(t + o + n), a0 = lo & ~(uintptr_t)15;
  for (uintptr_t a = a0 + 16 * lane; a < hi; a += 16 * lanes) {
    uint8_t* d = slot + (a - a0);
    if (a >= (uintptr_t)t && a + 16 <= (uintptr_t)(t + total)) {
      copy16(d, (const void*)a);
    } else {
      for (int j = 0; j < 16 / (int)sizeof(TA); ++j) {
        const uintptr_t e = a + j * sizeof(TA);
        if (e >= lo && e < hi) ((TA*)d)[j] = *(const TA*)e;
      }
    }
  }
}
static __host__ __device__ __forceinline__ int span_bytes(int n, int size) { return (n * size + 30) / 16 * 16; }
// the lanes of a team meet
template <Team TEAM>
__device__ __forceinline__ void team_sync(int warps, int barrier) {
  if constexpr (TEAM == MANY)
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
  else
    __syncwarp();
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

// Sums of K values over a team; every lane gets them.  MANY: `red` holds 2 x 16 x K floats of
// the team, used alternately so that one barrier per call is enough.
template <Team TEAM, int LANES, int K>
__device__ __forceinline__ void team_sum(float* v, float* red, int& turn, int warps, int barrier) {
  constexpr int W = TEAM == SUB ? LANES : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TEAM == MANY) {
    float* r = red + turn * 16 * K;
    turn ^= 1;
    const int w = (threadIdx.x >> 5) % warps;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) r[w * K + k] = v[k];
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(warps * 32) : "memory");
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = 0.f;
    for (int i = 0; i < warps; ++i)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += r[i * K + k];
  }
}

// The rounding of a float32 mean is some 2^-23 of it: beyond FAR deviations it would show in y, and the
// forward then sums h - mean once more (the differences are exact there) and takes off what the mean
// missed.  Other vectors keep their results and pay for a comparison (20000 x 787 bf16 with a residual, forward: 83 -> 87 us;
// other sizes nothing; summed for every vector 91, and 3 to 8 % at other sizes).
constexpr float FAR = 4.f;
__device__ __forceinline__ bool far(float mean, float rstd) {  // alike in a warp, and in a team
  return __any_sync(0xffffffffu, fabsf(mean) * rstd > FAR);
}
// `missed`: mean of h - mean; var: mean of its square.  1 / deviation about the mean itself.
__device__ __forceinline__ float far_rstd(float missed, float var, float eps) {
  const float v = fmaf(-missed, missed, var);
  return 1.f / sqrtf((v < 0.f ? 0.f : v) + eps);  // (below 0: rounding, where all channels are equal)
}

// Where this thread's team works: its vectors are first, first + stride, ... and lane /
// lanes place it in the team.  SUB: the position inside a row is fixed, rows advance.
// WARPS: `per_block` teams of a block take consecutive vectors.
template <Team TEAM, int LANES>
struct Place {
  int64_t first, stride;
  int lane, lanes, team, warps;
  __device__ __forceinline__ Place(const Args& a, int per_block) {
    if constexpr (TEAM == SUB) {
      const int per_row = a.G * LANES, slot = threadIdx.x / per_row, in_row = threadIdx.x % per_row;
      lane = in_row % LANES;
      lanes = LANES;
      warps = 1;
      team = slot;
      first = ((int64_t)blockIdx.x * per_block + slot) * a.G + in_row / LANES;
      if (slot >= per_block) first = a.vecs;  // spare threads of the last warp
      stride = (int64_t)gridDim.x * per_block * a.G;
    } else {
      lanes = TEAM == ONE ? 32 : blockDim.x / per_block;
      warps = lanes >> 5;
      team = threadIdx.x / lanes;
      lane = threadIdx.x % lanes;
      first = (int64_t)blockIdx.x * per_block + team;
      stride = (int64_t)gridDim.x * per_block;
    }
  }
  // every lane of a warp (SUB) or team runs the same number of rounds
  __device__ __forceinline__ bool done(int64_t v, int64_t vecs) const {
    return TEAM == SUB ? !__any_sync(0xffffffffu, v < vecs) : v >= vecs;
  }
};

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
// The vectors to come are copied into a ring in shared memory, `stages` - 1 of them ahead; every
// thread copies the groups that it will work on itself, so the ring needs no barrier and holds no
// registers.  Where rows are not aligned (VEC = 1) a team copies the aligned span that holds its vector,
// meets, and each lane picks its channels (51739 x 183 bf16: 35 us, 99 with direct loads
// of single channels).  Bound by memory: about 140 KB an SM are on
// their way with a residual (half of it without: the residual's slots then stay empty), and the weights stay
// in registers (read again for every row they were as many bytes as the row, through an L1 that was then
// 72 % busy).  65536 x 768 bf16 with a residual: 77 us, 5.2 TB/s, 14 us less than with direct loads and 32
// warps an SM.
template <typename TA, Team TEAM, int LANES, int VEC, int CHN>
__global__ void __launch_bounds__(TEAM == MANY ? 512 : 256, TEAM == MANY ? 1 : VEC * CHN <= 8 ? 4 : 2)
    fwd_kernel(Args a, int per_block, int stages) {
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ float red_all[8][2 * 16];
  constexpr bool OWN = VEC > 1;  // a thread copies what it uses; otherwise the team copies a span
  constexpr int NP = PAIRS<VEC>;
  typedef Pack<TA, VEC> Raw;
  int turn = 0;
  const Place<TEAM, LANES> z(a, per_block);
  float* red = red_all[TEAM == MANY ? z.team : 0];
  const float inv = 1.f / (float)a.N;
  const int n0 = z.lane * VEC, dn = z.lanes * VEC, left = a.N - n0;  // this thread's groups start at n0 + c * dn
  const TA *x = (const TA*)a.x + n0, *res = a.res ? (const TA*)a.res + n0 : nullptr;
  F2 w[CHN][NP], b[CHN][NP];
  auto params = [&](int64_t g) {
#pragma unroll
    for (int c = 0; c < CHN; ++c)
      if (c * dn < left) {
        const int64_t k = g * a.N + n0 + c * dn;
        float u[2 * NP], v[2 * NP];
        u[2 * NP - 1] = v[2 * NP - 1] = 0.f;
        load_param<VEC>(u, a.w ? a.w + k : nullptr, 1.f);
        load_param<VEC>(v, a.b ? a.b + k : nullptr, 0.f);
#pragma unroll
        for (int j = 0; j < NP; ++j) w[c][j] = f2(u[2 * j], u[2 * j + 1]), b[c][j] = f2(v[2 * j], v[2 * j + 1]);
      }
  };
  const bool fixed = TEAM == SUB || a.G == 1;  // one group's weights in every round
  if (fixed) params(TEAM == SUB ? z.first % a.G : 0);
  Raw* ring = (Raw*)dyn + threadIdx.x;  // slot (stage, stream, c): 2 streams
  const int pitch = blockDim.x, bytes = span_bytes(a.N, sizeof(TA));
  uint8_t* spans = dyn + (size_t)z.team * stages * 2 * bytes;  // slot (stage, stream) of the team
  auto fetch = [&](int64_t v, int st) {
    if (v < a.vecs) {
      const int64_t o = v * a.N;
      if constexpr (OWN) {
        Raw* r = ring + st * 2 * CHN * pitch;
#pragma unroll
        for (int c = 0; c < CHN; ++c)
          if (c * dn < left) {
            copy16(r + c * pitch, x + o + c * dn);
            if (res) copy16(r + (CHN + c) * pitch, res + o + c * dn);
          }
      } else {
        copy_span(spans + st * 2 * bytes, (const TA*)a.x, o, a.N, a.vecs * a.N, z.lane, z.lanes);
        if (res) copy_span(spans + (st * 2 + 1) * bytes, (const TA*)a.res, o, a.N, a.vecs * a.N, z.lane, z.lanes);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int at = 0;  // stage of the current vector
  for (int i = 0; i < 3; ++i) fetch(i < stages - 1 ? z.first + i * z.stride : a.vecs, i);  // 3 groups always
  for (int64_t v0 = z.first; !z.done(v0, a.vecs); v0 += z.stride) {
    const bool on = v0 < a.vecs;
    const int64_t o = v0 * a.N;
    if (!fixed) params(v0 % a.G);
    // the group of this vector is the (stages - 1)-th newest
    if (stages == 4)
      asm volatile("cp.async.wait_group 2;" ::: "memory");
    else
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (!OWN) team_sync<TEAM>(z.warps, 1 + z.team);
    const Raw* slot = OWN ? ring + at * 2 * CHN * pitch
                          : (const Raw*)(spans + at * 2 * bytes) + span_shift((const TA*)a.x, o) + n0;
    const Raw* slot_r = OWN ? slot + CHN * pitch
                            : (const Raw*)(spans + (at * 2 + 1) * bytes) + span_shift((const TA*)a.res, o) + n0;
    const int step = OWN ? pitch : dn;
    F2 f[CHN][NP], s2 = f2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      if (on && c * dn < left) {
        unpack2<TA, VEC>(f[c], slot[c * step]);
        if (res) {
          F2 r[NP];
          unpack2<TA, VEC>(r, slot_r[c * step]);
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            f[c][j] = f[c][j] + r[j];
            if (sizeof(TA) == 2) f[c][j] = bf2_unpack(bf2_pack(f[c][j]));  // the stream's type: what h holds
          }
          store2<TA, VEC>((TA*)a.h + o + n0 + c * dn, f[c]);
        }
#pragma unroll
        for (int j = 0; j < NP; ++j) s2 = s2 + f[c][j];
      }
    }
    {  // into the slot of the vector before
      const int to = at == 0 ? stages - 1 : at - 1;
      fetch(v0 + (stages - 1) * z.stride, to);
      at = at + 1 == stages ? 0 : at + 1;
    }
    float2 t = f2_get(s2);
    float s[1] = {t.x + t.y};
    team_sum<TEAM, LANES, 1>(s, red, turn, z.warps, 1 + z.team);
    const float mean = s[0] * inv;
    const F2 nmean = f2(-mean, VEC == 1 ? 0.f : -mean);
    s2 = f2(0.f, 0.f);
#pragma unroll
    for (int c = 0; c < CHN; ++c)
      if (on && c * dn < left) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          f[c][j] = f[c][j] + nmean;
          s2 = fma2(f[c][j], f[c][j], s2);
        }
      }
    t = f2_get(s2);
    s[0] = t.x + t.y;
    team_sum<TEAM, LANES, 1>(s, red, turn, z.warps, 1 + z.team);
    float rstd = 1.f / sqrtf(fmaf(s[0], inv, a.eps)), missed = 0.f;
    if (far(mean, rstd)) {
      const float var = s[0] * inv;
      if constexpr (OWN) {
        s2 = f2(0.f, 0.f);
#pragma unroll
        for (int c = 0; c < CHN; ++c)
          if (on && c * dn < left) {
#pragma unroll
            for (int j = 0; j < NP; ++j) s2 = s2 + f[c][j];
          }
        t = f2_get(s2);
        s[0] = t.x + t.y;
      } else {  // from memory (this thread wrote h): fewer registers
        const TA* hv = (res ? (const TA*)a.h + n0 : x) + o;
        s[0] = 0.f;
#pragma unroll 1
        for (int n = 0; on && n < left; n += dn) s[0] += ld_act(hv, (size_t)n) - mean;
      }
      team_sum<TEAM, LANES, 1>(s, red, turn, z.warps, 1 + z.team);
      missed = s[0] * inv;
      rstd = far_rstd(missed, var, a.eps);
      const F2 m2 = f2(-missed, VEC == 1 ? 0.f : -missed);
#pragma unroll
      for (int c = 0; c < CHN; ++c)
#pragma unroll
        for (int j = 0; j < NP; ++j) f[c][j] = f[c][j] + m2;
    }
    if (on && z.lane == 0 && a.stats) *(float2*)(a.stats + 2 * v0) = make_float2(mean + missed, rstd);
    const F2 r2 = f2(rstd, rstd);
#pragma unroll
    for (int c = 0; c < CHN; ++c)
      if (on && c * dn < left) {
#pragma unroll
        for (int j = 0; j < NP; ++j) f[c][j] = fma2(f[c][j] * r2, w[c][j], b[c][j]);
        store2<TA, VEC>((TA*)a.y + o + n0 + c * dn, f[c]);
      }
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
// With z = (h - mean) rstd and u = dy w:  dx = rstd (u - mean(u) - z mean(u z)) + dh,
// dw += dy z, db += dy.
// A ring as in the forward (a register prefetch spilled, which made every copy wait for its
// load: 325 us at 65536 x 768 bf16 with dh; the ring 79, 5.1 TB/s, and 4 for the sum of the partial rows).  The
// sums of the weights' gradients take the registers that the forward has for the weights, and leave 16
// warps an SM.  Three groups of 8 bf16 with their sums are more than 128 registers: 80 (one warp a
// vector) and 136 bytes (more) of each thread's are kept in local memory and read again.
template <typename TA, Team TEAM, int LANES, int VEC, int CHN>
__global__ void __launch_bounds__(TEAM == MANY ? 512 : 256, TEAM == MANY ? 1 : TEAM == SUB ? 4 : VEC * CHN <= 8 ? 3 : 2)
    bwd_kernel(Args a, int per_block, int stages) {
  extern __shared__ __align__(16) uint8_t dyn[];  // the ring; after it the teams' sums, 2 x width each
  __shared__ float red_all[8][2 * 16 * 2];
  constexpr bool OWN = VEC > 1;  // as in the forward
  constexpr int NP = PAIRS<VEC>;
  typedef Pack<TA, VEC> Raw;
  let_next_start();
  int turn = 0;
  const Place<TEAM, LANES> z(a, per_block);
  float* red = red_all[TEAM == MANY ? z.team : 0];
  const float inv = 1.f / (float)a.N;
  const int g = a.G == 1 ? 0 : (int)(z.first % a.G);  // the stride is a multiple of G
  const int n0 = z.lane * VEC, dn = z.lanes * VEC;    // this thread's groups start at n0 + c * dn
  const float* wg = a.w ? a.w + (int64_t)g * a.N + n0 : nullptr;
  const TA *h = (const TA*)a.h + n0, *dy = (const TA*)a.dy + n0, *dh = a.dh ? (const TA*)a.dh + n0 : nullptr;
  F2 dw[CHN][NP], db[CHN][NP];
#pragma unroll
  for (int c = 0; c < CHN; ++c)
#pragma unroll
    for (int j = 0; j < NP; ++j) dw[c][j] = db[c][j] = f2(0.f, 0.f);
  Raw* ring = (Raw*)dyn + threadIdx.x;  // slot (stage, stream, c): 3 streams
  const int pitch = blockDim.x, bytes = span_bytes(a.N, sizeof(TA));
  uint8_t* spans = dyn + (size_t)z.team * stages * 3 * bytes;  // slot (stage, stream) of the team
  auto fetch = [&](int64_t v, int st) {
    if (v < a.vecs) {
      const int64_t o = v * a.N;
      if constexpr (OWN) {
        Raw* r = ring + st * 3 * CHN * pitch;
#pragma unroll
        for (int c = 0; c < CHN; ++c)
          if (n0 + c * dn < a.N) {
            copy16(r + c * pitch, h + o + c * dn);
            copy16(r + (CHN + c) * pitch, dy + o + c * dn);
            if (dh) copy16(r + (2 * CHN + c) * pitch, dh + o + c * dn);
          }
      } else {
        uint8_t* r = spans + st * 3 * bytes;
        copy_span(r, (const TA*)a.h, o, a.N, a.vecs * a.N, z.lane, z.lanes);
        copy_span(r + bytes, (const TA*)a.dy, o, a.N, a.vecs * a.N, z.lane, z.lanes);
        if (dh) copy_span(r + 2 * bytes, (const TA*)a.dh, o, a.N, a.vecs * a.N, z.lane, z.lanes);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int at = 0;  // stage of the current vector
  auto span = [&](int st, int k, const void* t, int64_t o) {  // this thread's first channel in stream k of a stage
    return (const Raw*)(spans + (st * 3 + k) * bytes) + span_shift((const TA*)t, o) + n0;
  };
  for (int i = 0; i < 3; ++i) fetch(i < stages - 1 ? z.first + i * z.stride : a.vecs, i);  // 3 groups always
  float2 nst = z.first < a.vecs ? *(const float2*)(a.cstats + 2 * z.first) : make_float2(0.f, 0.f);
  for (int64_t v0 = z.first; !z.done(v0, a.vecs); v0 += z.stride) {
    const bool on = v0 < a.vecs;
    const float2 st = nst;
    if (v0 + z.stride < a.vecs) nst = *(const float2*)(a.cstats + 2 * (v0 + z.stride));
    // the group of this vector is the (stages - 1)-th newest
    if (stages == 4)
      asm volatile("cp.async.wait_group 2;" ::: "memory");
    else
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (!OWN) team_sync<TEAM>(z.warps, 1 + z.team);
    F2 f[CHN][NP], d[CHN][NP], s0 = f2(0.f, 0.f), s1 = f2(0.f, 0.f);
    const F2 nmean = f2(-st.x, -st.x), rstd = f2(st.y, st.y);
    const int cur = at;
    const Raw* slot = ring + cur * 3 * CHN * pitch;
    const int64_t o = v0 * a.N;
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      if (on && n0 + c * dn < a.N) {
        if constexpr (OWN) {
          unpack2<TA, VEC>(f[c], slot[c * pitch]);
          unpack2<TA, VEC>(d[c], slot[(CHN + c) * pitch]);
        } else {
          unpack2<TA, VEC>(f[c], span(cur, 0, a.h, o)[c * dn]);
          unpack2<TA, VEC>(d[c], span(cur, 1, a.dy, o)[c * dn]);
        }
        float w[2 * NP];
        w[2 * NP - 1] = 0.f;
        load_param<VEC>(w, wg ? wg + c * dn : nullptr, 1.f);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          f[c][j] = (f[c][j] + nmean) * rstd;
          dw[c][j] = fma2(d[c][j], f[c][j], dw[c][j]);
          db[c][j] = db[c][j] + d[c][j];
          d[c][j] = d[c][j] * f2(w[2 * j], w[2 * j + 1]);
          s0 = s0 + d[c][j];
          s1 = fma2(d[c][j], f[c][j], s1);
        }
      }
    }
    {  // into the slot of the vector before
      const int to = at == 0 ? stages - 1 : at - 1;
      fetch(v0 + (stages - 1) * z.stride, to);
      at = at + 1 == stages ? 0 : at + 1;
    }
    const float2 t0 = f2_get(s0), t1 = f2_get(s1);
    float s[2] = {t0.x + t0.y, t1.x + t1.y};
    team_sum<TEAM, LANES, 2>(s, red, turn, z.warps, 1 + z.team);
    const float m1 = -st.y * (s[0] * inv), m2 = -st.y * (s[1] * inv);
    const F2 c1 = f2(m1, m1), c2 = f2(m2, m2);
#pragma unroll
    for (int c = 0; c < CHN; ++c) {
      if (on && n0 + c * dn < a.N) {
#pragma unroll
        for (int j = 0; j < NP; ++j) d[c][j] = fma2(rstd, d[c][j], fma2(f[c][j], c2, c1));
        if (dh) {
          if constexpr (OWN)
            unpack2<TA, VEC>(f[c], slot[(2 * CHN + c) * pitch]);
          else
            unpack2<TA, VEC>(f[c], span(cur, 2, a.dh, o)[c * dn]);
#pragma unroll
          for (int j = 0; j < NP; ++j) d[c][j] = d[c][j] + f[c][j];
        }
        store2<TA, VEC>((TA*)a.dx + o + n0 + c * dn, d[c]);
      }
    }
  }
  if (!a.part) return;
  float* pw = a.part + (int64_t)blockIdx.x * 2 * a.width;
  // the teams of the block side by side, where the ring was, then added up in order
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  const bool alone = TEAM != SUB && per_block == 1;  // one team: straight to its partial row
  float* aw = alone ? pw : (float*)dyn + z.team * 2 * a.width;
  const int off = (TEAM == SUB ? g * a.N : 0) + n0;
  if (z.team < per_block) {
#pragma unroll
    for (int c = 0; c < CHN; ++c)
      if (n0 + c * dn < a.N) {
        float* k = aw + off + c * dn;
        if constexpr (VEC % 4 == 0) {
#pragma unroll
          for (int j = 0; j < NP; j += 2) {
            const float2 x = f2_get(dw[c][j]), y = f2_get(dw[c][j + 1]), u = f2_get(db[c][j]), v = f2_get(db[c][j + 1]);
            *(float4*)(k + 2 * j) = make_float4(x.x, x.y, y.x, y.y);
            *(float4*)(k + a.width + 2 * j) = make_float4(u.x, u.y, v.x, v.y);
          }
        } else {
          k[0] = f2_get(dw[c][0]).x;
          k[a.width] = f2_get(db[c][0]).x;
        }
      }
  }
  if (alone) return;
  __syncthreads();
  for (int k = threadIdx.x; k < 2 * a.width; k += blockDim.x) {
    float s = 0.f;
    for (int i = 0; i < per_block; ++i) s += ((const float*)dyn)[i * 2 * a.width + k];
    pw[k] = s;
  }
}

// dw, db (G, N) from the partial rows: channel (g, n) is column (g * N + n) % width of the
// rows p with p % groups == group, groups = G * N / width.
// A block adds up 8 channels (a 32-byte sector of each row), 64 rows side by side.
constexpr int PCOL = 8, PROW = 64;
__global__ void __launch_bounds__(PCOL * PROW) param_kernel(Args a, int parts, float* dw, float* db) {
  __shared__ float red[2][PROW][PCOL];
  const int tx = threadIdx.x % PCOL, ty = threadIdx.x / PCOL, col = blockIdx.x * PCOL + tx, total = a.G * a.N;
  const int groups = total / a.width;
  float sw = 0.f, sb = 0.f;
  after_previous();
  if (col < total) {
    const int grp = col / a.width, n = col % a.width;
#pragma unroll 4
    for (int p = grp + ty * groups; p < parts; p += PROW * groups) {
      const float* r = a.part + (int64_t)p * 2 * a.width + n;
      sw += r[0];
      sb += r[a.width];
    }
  }
  red[0][ty][tx] = sw;
  red[1][ty][tx] = sb;
  __syncthreads();
  if (ty < 16) {
    const int which = ty >> 3, part = ty & 7;  // 8 threads a sum, neighbours 8 lanes apart in one warp
    float s = 0.f;
    for (int i = part; i < PROW; i += 8) s += red[which][i][tx];
    __syncwarp();
    red[which][part][tx] = s;
  }
  __syncthreads();
  if (ty < 2) {
    float s = 0.f;
    for (int i = 0; i < 8; ++i) s += red[ty][i][tx];
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
    team_sum<MANY, 32, 1>(s, red, turn, 16, 1);
    const float mean = s[0] * inv;
    s[0] = 0.f;
    for (int n = threadIdx.x; n < a.N; n += 512) {
      const float f = ld_act(h, (size_t)n) - mean;
      s[0] = fmaf(f, f, s[0]);
    }
    team_sum<MANY, 32, 1>(s, red, turn, 16, 1);
    float rstd = 1.f / sqrtf(fmaf(s[0], inv, a.eps)), missed = 0.f;
    if (far(mean, rstd)) {
      const float var = s[0] * inv;
      s[0] = 0.f;
      for (int n = threadIdx.x; n < a.N; n += 512) s[0] += ld_act(h, (size_t)n) - mean;
      team_sum<MANY, 32, 1>(s, red, turn, 16, 1);
      missed = s[0] * inv;
      rstd = far_rstd(missed, var, a.eps);
    }
    if (threadIdx.x == 0 && a.stats) *(float2*)(a.stats + 2 * v) = make_float2(mean + missed, rstd);
    for (int n = threadIdx.x; n < a.N; n += 512) {
      const float w = a.w ? a.w[(int64_t)g * a.N + n] : 1.f, b = a.b ? a.b[(int64_t)g * a.N + n] : 0.f;
      st_act((TA*)a.y + v * a.N, (size_t)n, fmaf((ld_act(h, (size_t)n) - mean - missed) * rstd, w, b));
    }
  }
}

// Loads of BU elements 512 apart are in flight together (the compiler cannot move them over the stores):
// 9000 x 4099 bf16 with dh 237 -> 144 us.
constexpr int BU = 4;
template <typename TA>
__device__ __forceinline__ void load_apart(float* f, const TA* p, int n0, int n) {
#pragma unroll
  for (int i = 0; i < BU; ++i) f[i] = n0 + 512 * i < n ? ld_act(p, (size_t)(n0 + 512 * i)) : 0.f;
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
    const float* wg = a.w ? a.w + (v % a.G) * (int64_t)a.N : nullptr;
    const float2 st = *(const float2*)(a.cstats + 2 * v);
    float s[2] = {0.f, 0.f};
    for (int n0 = threadIdx.x; n0 < a.N; n0 += 512 * BU) {
      float f[BU], d[BU], w[BU];
      load_apart<TA>(f, h, n0, a.N);
      load_apart<TA>(d, dy, n0, a.N);
      if (wg) load_apart<float>(w, wg, n0, a.N);
#pragma unroll
      for (int i = 0; i < BU; ++i) {
        const float u = wg ? d[i] * w[i] : d[i];  // 0 beyond the vector
        s[0] += u;
        s[1] = fmaf(u, (f[i] - st.x) * st.y, s[1]);
      }
    }
    team_sum<MANY, 32, 2>(s, red, turn, 16, 1);
    for (int n0 = threadIdx.x; n0 < a.N; n0 += 512 * BU) {
      float f[BU], d[BU], w[BU], e[BU];
      load_apart<TA>(f, h, n0, a.N);
      load_apart<TA>(d, dy, n0, a.N);
      if (wg) load_apart<float>(w, wg, n0, a.N);
      if (dh) load_apart<TA>(e, dh, n0, a.N);
#pragma unroll
      for (int i = 0; i < BU; ++i) {
        const float u = wg ? d[i] * w[i] : d[i], zz = (f[i] - st.x) * st.y;
        const float g = st.y * (u - s[0] * inv - zz * (s[1] * inv));
        if (n0 + 512 * i < a.N) st_act((TA*)a.dx + v * a.N, (size_t)(n0 + 512 * i), dh ? g + e[i] : g);
      }
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
#pragma unroll 4
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
constexpr int SMS = 148;
constexpr int MAX_SMEM = 208 << 10;  // dynamic, of a backward block: 2 stages of 512 threads x 4 groups x 3 streams + sums
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

// How a problem runs.  VEC: channels per load.  SUB for vectors of 4 to 32 aligned groups, a
// power of two, where the row of G vectors fits a block; TINY for up to 8 channels; WARPS
// while a thread holds at most 3 groups of 8 bf16, 4 groups of 4 float32 or 8 single
// channels (what the backward keeps in 128 registers, but for 80 to 136 bytes at 3 groups of
// bf16; single channels of one warp spill more, in 64 and 80 registers); else BIG.  As few warps as hold
// the vector: the shuffles and address arithmetic of a vector are paid once for each warp.
struct Plan {
  bool big, tiny;
  Team team;
  int vec, lanes, chn, threads, per_block, width, parts;
  int64_t grid;
};
// single channels: BIG from here on (bf16 training, WARPS and BIG: 14000 x 1301 240 and 312 us, 9000 x 2051 310 and 235)
constexpr int SINGLES = 1600;
static Plan plan(const Args& a, int act_dtype, bool vec_ok, bool bwd) {
  Plan z{};
  const int full = act_dtype == ATLAS_BF16 ? 8 : 4;
  z.vec = vec_ok && a.N % full == 0 ? full : 1;
  const int groups = (a.N + z.vec - 1) / z.vec, most = z.vec == 8 ? 3 : z.vec == 4 ? 4 : 8;  // groups a thread
  const bool pow2 = (groups & (groups - 1)) == 0;
  z.per_block = 1;
  z.threads = 256;
  int64_t units;  // blocks' worth of work
  if (a.N <= TINY) {
    z.tiny = true;
    z.width = a.G * a.N;
    units = (a.vecs + 255) / 256;
  } else if (z.vec > 1 && pow2 && groups >= 4 && groups <= 32 && (int64_t)a.G * groups <= 256) {
    z.team = SUB;
    z.lanes = groups;
    z.chn = 1;
    z.per_block = 256 / (a.G * groups);
    z.threads = (z.per_block * a.G * groups + 31) / 32 * 32;
    z.width = a.G * a.N;
    units = (a.rows + z.per_block - 1) / z.per_block;
  } else if (groups <= (z.vec == 1 ? SINGLES : 512 * most)) {
    const int per_lane = z.vec == 8 ? 3 : z.vec == 4 ? 4 : 8;  // (single channels, 4 a lane: 20000 x 787 234 us, 8: 189)
    const int warps = std::min(16, (groups + 32 * per_lane - 1) / (32 * per_lane));
    z.team = warps == 1 ? ONE : MANY;
    z.chn = (groups + 32 * warps - 1) / (32 * warps);
    if (z.vec == 1) z.chn = z.chn <= 4 ? 4 : 8;
    // a block's teams share channels; with weights for each group that needs one team
    z.per_block = bwd && a.G > 1 ? 1 : std::max(1, 8 / warps);
    z.threads = 32 * warps * z.per_block;
    z.width = a.N;
    units = (a.vecs + z.per_block - 1) / z.per_block;
  } else {
    z.big = true;
    z.threads = 512;
    z.width = a.G * a.N;
    units = a.vecs;
  }
  // Blocks are what an SM holds at its register use (each keeps sums, or weights); the forward's
  // fewer where that makes their numbers of rounds equal.
  const int64_t blocks = SMS * (!bwd && (z.big || z.tiny) ? 8 : z.threads * z.chn * z.vec <= 2048 ? 4 : 2);
  const int64_t rounds = std::max<int64_t>(1, (units + blocks - 1) / blocks);
  z.grid = std::max<int64_t>(1, bwd ? std::min(units, blocks) : (units + rounds - 1) / rounds);
  if (bwd && !z.big && !z.tiny && z.team != SUB && a.G > 1)  // a multiple of G: a block keeps one group's weights
    z.grid = std::min<int64_t>(units, std::max<int64_t>(a.G, z.grid / a.G * a.G));
  z.parts = (int)(z.big ? std::min<int64_t>(BIG_PARTS, std::max<int64_t>(1, a.rows))
                  : z.tiny ? std::min<int64_t>(4 * SMS, std::max<int64_t>(1, a.rows)) : z.grid);
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

// A kernel's dynamic shared memory above 48 KB, asked of the driver once per device.
template <auto Kernel>
static cudaError_t allow_smem() {
  static DeviceCache done;
  cudaError_t e = cudaSuccess;
  done.get([&] {
    e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
    return e == cudaSuccess ? 0 : -1;
  });
  return e;
}
template <typename TA, Team TEAM, int LANES, int VEC, int CHN>
static cudaError_t go(const Args& a, const Plan& z, bool bwd, cudaStream_t s) {
  // as many stages, up to 4, as the blocks that an SM's registers hold have room for
  const int stage = (bwd ? 3 : 2) * (VEC > 1 ? CHN * z.threads * 16 : z.per_block * span_bytes(a.N, sizeof(TA)));
  const int room = (VEC == 1 && z.threads > 256 ? 200 : bwd || VEC * CHN <= 8 ? 50 : z.threads <= 256 ? 100 : 200) << 10;
  const int stages = 4 * stage <= room ? 4 : 2;
  if (bwd) {
    const size_t sums = TEAM == SUB || z.per_block > 1 ? (size_t)z.per_block * 2 * z.width * sizeof(float) : 0;
    const size_t sm = std::max((size_t)(stages * stage), sums);
    cudaError_t e = allow_smem<bwd_kernel<TA, TEAM, LANES, VEC, CHN>>();
    if (e != cudaSuccess) return e;
    bwd_kernel<TA, TEAM, LANES, VEC, CHN><<<(unsigned)z.grid, z.threads, sm, s>>>(a, z.per_block, stages);
  } else {
    cudaError_t e = allow_smem<fwd_kernel<TA, TEAM, LANES, VEC, CHN>>();
    if (e != cudaSuccess) return e;
    fwd_kernel<TA, TEAM, LANES, VEC, CHN><<<(unsigned)z.grid, z.threads, stages * stage, s>>>(a, z.per_block, stages);
  }
  return cudaGetLastError();
}
template <typename TA, Team TEAM, int VEC>
static cudaError_t by_chn(const Args& a, const Plan& z, bool bwd, cudaStream_t s) {
  if constexpr (VEC > 1) {
    if (z.chn == 1) return go<TA, TEAM, 32, VEC, 1>(a, z, bwd, s);
    if (z.chn == 2) return go<TA, TEAM, 32, VEC, 2>(a, z, bwd, s);
    if constexpr (VEC == 8) {
      return go<TA, TEAM, 32, VEC, 3>(a, z, bwd, s);
    } else {
      return z.chn == 3 ? go<TA, TEAM, 32, VEC, 3>(a, z, bwd, s) : go<TA, TEAM, 32, VEC, 4>(a, z, bwd, s);
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
  if (z.team == ONE)
    return z.vec > 1 ? by_chn<TA, ONE, FULL>(a, z, bwd, s) : by_chn<TA, ONE, 1>(a, z, bwd, s);
  return z.vec > 1 ? by_chn<TA, MANY, FULL>(a, z, bwd, s) : by_chn<TA, MANY, 1>(a, z, bwd, s);
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
    e = follow(param_kernel, (unsigned)((p->G * p->N + PCOL - 1) / PCOL), PCOL * PROW, 0, s, a, z.parts, dweight, dbias);
  }
  return status_of(e);
}
