// Memory-bound sm_100a kernels that stand around the fused projections of an attention layer: rotary
// positions with the normalisation of query and key heads in front of them, and the norm around a block
// with its gate, residual sum, scale and shift. Forward and backward, C ABI at the end of the file.
//
// All of them are byte movers: 16-byte accesses, every element of the large tensors read and written
// once, sums in FP32, one rounding to BF16 at the end. Reductions over tokens (gradients of weights and
// of per-sample vectors) go through FP32 partial sums in caller-provided scratch and are finished in a
// fixed order, so results do not depend on scheduling.
#include <cstdint>
#include <type_traits>
#include <cuda_bf16.h>
#include "../../include/fga.h"
#include "common.cuh"
#include "f32x2.cuh"
#include "ptx.cuh"
#include "seq_bounds.cuh"

namespace fga {
namespace {

constexpr int kHeadDim = 128;

__device__ __forceinline__ void unpack8(uint4 v, F2 (&f)[4]) {
  f[0] = f2_of_bf16(v.x);
  f[1] = f2_of_bf16(v.y);
  f[2] = f2_of_bf16(v.z);
  f[3] = f2_of_bf16(v.w);
}
__device__ __forceinline__ uint4 pack8(const F2 (&f)[4]) {
  return make_uint4(bf16_of_f2(f[0]), bf16_of_f2(f[1]), bf16_of_f2(f[2]), bf16_of_f2(f[3]));
}
__device__ __forceinline__ uint4 load16(const uint16_t* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ void store16(uint16_t* p, uint4 v) { *reinterpret_cast<uint4*>(p) = v; }

// 16 bytes global -> shared without passing through registers; groups are per thread.
__device__ __forceinline__ void copy16_async(uint32_t dst, const uint16_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

// =============================================================================================
// Rotary positions. Pair i of a head turns by angle pos[axis(i)] * inv_freq[i]; interleaved pairs are
// elements (2i, 2i+1), half-split pairs (i, i+64). With a weight w the head is first divided by its root
// mean square and multiplied by w:  y = R(x * rstd * w).
//
// Angles: a position of 10^6 times a frequency of 1 leaves an FP32 product with errors of 0.06 rad. The
// angle is only needed modulo one turn, so the frequency is held as a 64-bit fixed-point number of turns
// (2^-64 each, rounded once from twice FP64's precision), the product with the integer position wraps modulo
// 2^64 exactly, and only the top 32 bits become a float. The frequency's rounding is off by |position| * 2^-64
// turns, the float by 2^-28: together below 2^-27 turns at every position below 2^36, whatever the frequency.
//
// Mapping: one warp per token (several when tokens are few), which computes the token's 64 sines and
// cosines once for all heads. Eight lanes hold a head row, each 8 elements of its lower and 8 of its upper
// half, so both kinds of pairs turn inside a lane; a warp takes four head rows at a time. The first version
// (16 lanes a row, scalar arithmetic) issued 870 instructions per token of 8 heads and was bound by that, at
// 3.7 TB/s. Now 131072 tokens x (4 + 4) heads with head norms take 101 us forward (5.3 TB/s) and 162 us
// backward (5.0 TB/s; its registers hold it to 16 warps an SM), 16384 x (32 + 8) without norms 55 us
// (6.1 TB/s, where a plain copy measures 6.55). At the 80 registers of three blocks an SM the forward kernels with
// norms spill 32 and 44 bytes a thread.
// =============================================================================================
constexpr int kRotaryWarps = 8;

struct RotaryParams {
  const uint16_t* x[2];       // forward: inputs; backward: the forward's inputs (only read where w is set)
  const uint16_t* dy[2];      // backward: incoming gradients, contiguous
  uint16_t* out[2];           // forward: outputs; backward: gradients of x; contiguous
  const uint16_t* w[2];       // [128] or null
  long long x_tok[2];         // strides in elements
  int x_head[2];
  int heads[2];
  const void* pos;            // [tokens, axes]
  int pos64;
  int axes;
  int ends[4];                // pairs of axis a are ends[a-1] .. ends[a]-1
  const void* freq;           // [64]
  int freq64;
  int tokens;
  int splits;                 // warps per token
  float eps;
  float* partial;             // backward with weights: [grid][2][128]
};

// A lane's share of the angles: pairs lane and lane + 32.
struct LaneAngle {
  unsigned long long turns[2];  // 2^-64 turns per position
  int axis[2];
};
__device__ __forceinline__ LaneAngle lane_angle(const RotaryParams& P, int lane) {
  LaneAngle a;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int pair = lane + 32 * i;
    const double f = P.freq64 ? __ldg(static_cast<const double*>(P.freq) + pair)
                              : static_cast<double>(__ldg(static_cast<const float*>(P.freq) + pair));
    // turns per position: f / (2 pi) as the sum of two FP64 numbers, 1 / (2 pi) being one as well; whole turns go
    const double per_turn = 0.15915494309189535, per_turn_rest = -9.839338337591243e-18;
    const double t = f * per_turn, rest = fma(f, per_turn, -t) + f * per_turn_rest;
    a.turns[i] = static_cast<unsigned long long>(__double2ll_rn((t - rint(t)) * 18446744073709551616.0)) +
                 static_cast<unsigned long long>(__double2ll_rn(rest * 18446744073709551616.0));
    a.axis[i] = (P.axes > 1 && pair >= P.ends[0]) + (P.axes > 2 && pair >= P.ends[1]) + (P.axes > 3 && pair >= P.ends[2]);
  }
  return a;
}
// Sine and cosine of both of a lane's angles. The nearest quarter turn is taken off the fixed-point angle,
// which leaves |r| <= 1/8 turn; there sin(2 pi r) = r (s0 + s1 r^2 + s2 r^4 + s3 r^6) to a relative 3.3e-9 and
// cos(2 pi r) = 1 + r^2 (c1 + c2 r^2 + c3 r^4) to 3.3e-8 (fitted by iteratively reweighted least squares), so
// FP32 rounding dominates. Both angles go through as one packed pair; the general sincospif took a quarter
// of the kernel's instructions.
__device__ __forceinline__ void warp_rotation(const RotaryParams& P, const LaneAngle& a, int token, int lane,
                                              float* cosines, float* sines) {
  float rest[2], c[2], s[2];
  uint32_t quarter[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const long long at = static_cast<long long>(token) * P.axes + a.axis[i];
    const long long pos = P.pos64 ? __ldg(static_cast<const long long*>(P.pos) + at)
                                  : static_cast<long long>(__ldg(static_cast<const int*>(P.pos) + at));
    const uint32_t turn = static_cast<uint32_t>((a.turns[i] * static_cast<unsigned long long>(pos)) >> 32);
    quarter[i] = (turn + 0x20000000u) >> 30;
    rest[i] = static_cast<float>(static_cast<int>(turn - (quarter[i] << 30))) * 2.3283064365386963e-10f;  // 2^-32
  }
  const F2 r = f2(rest[0], rest[1]), u = r * r;
  const F2 sine = r * fma2(fma2(fma2(u, f2(-75.3935558f), f2(81.59235342f)), u, f2(-41.34166145f)), u, f2(6.28318529f));
  const F2 cosine = fma2(fma2(fma2(u, f2(-83.66591204f), f2(64.92322849f)), u, f2(-19.73916726f)), u, f2(1.f));
  split(cosine, c[0], c[1]);
  split(sine, s[0], s[1]);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool odd = quarter[i] & 1;
    const float cs = odd ? s[i] : c[i], sn = odd ? c[i] : s[i];
    cosines[lane + 32 * i] = (quarter[i] + 1) & 2 ? -cs : cs;  // quarters 1 and 2
    sines[lane + 32 * i] = quarter[i] & 2 ? -sn : sn;          // quarters 2 and 3
  }
  __syncwarp();
}

// Turns a lane's 16 elements (f[0..3] from the lower half of the head, f[4..7] from the upper). Interleaved:
// pair i of f is (lo, hi) of f[i], with cosine c[i>>1] half i&1. Half-split: f[i] turns with f[i + 4], with
// cosines c[i].
template <bool kInterleaved>
__device__ __forceinline__ void rotate16(F2 (&f)[8], const F2 (&c)[4], const F2 (&s)[4]) {
  if constexpr (kInterleaved) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float a, b, c0, c1, s0, s1;
      split(f[i], a, b);
      split(c[i >> 1], c0, c1);
      split(s[i >> 1], s0, s1);
      const float cc = i & 1 ? c1 : c0, ss = i & 1 ? s1 : s0;
      f[i] = f2(a * cc - b * ss, b * cc + a * ss);
    }
  } else {
    const F2 minus = f2(-1.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const F2 a = f[i], b = f[i + 4];
      f[i] = fma2(b * minus, s[i], a * c[i]);
      f[i + 4] = fma2(a, s[i], b * c[i]);
    }
  }
}

__device__ __forceinline__ float eight_lane_sum(float v) {
#pragma unroll
  for (int o = 4; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void unpack16(uint4 lower, uint4 upper, F2 (&f)[8]) {
  F2 a[4], b[4];
  unpack8(lower, a);
  unpack8(upper, b);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = a[i];
    f[i + 4] = b[i];
  }
}

template <bool kInterleaved, bool kBackward, bool kNorm>
__global__ void __launch_bounds__(32 * kRotaryWarps, kBackward && kNorm ? 2 : 3) rotary_kernel(const RotaryParams P) {
  __shared__ float tables[kRotaryWarps][2][64];
  __shared__ float reduce[kBackward && kNorm ? kRotaryWarps : 1][2][kHeadDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane & 7, quarter = lane >> 3;
  const LaneAngle angle = lane_angle(P, lane);
  __shared__ uint4 weights[2][kHeadDim / 8];  // registers are short
  F2 dw[2][8];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[t][i] = f2(0.f);
    if (kNorm && P.w[t] != nullptr && threadIdx.x < kHeadDim / 8) weights[t][threadIdx.x] = load16(P.w[t] + threadIdx.x * 8);
  }
  if (kNorm) __syncthreads();
  // A trip takes four head rows of q, or four of k. The loads of the first trip of both are in flight before
  // the angles are worked out, and of two trips of a tensor before the first is used.
  struct Trip {
    uint4 raw[2], x[2];
  };
  const int units = P.tokens * P.splits;  // below 2^31: there is more than one split only with few tokens
  for (int u = blockIdx.x * kRotaryWarps + warp; u < units; u += gridDim.x * kRotaryWarps) {
    const int token = P.splits == 1 ? u : u / P.splits, split_at = u - token * P.splits;
    F2 c[4], s[4];
    const float *ct = tables[warp][0], *st = tables[warp][1];
    auto angles = [&]() {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // interleaved: pairs sub*4 .. +3 of the lower half, 32 + sub*4 .. +3 of the upper; else sub*8 .. +7
        const int at = kInterleaved ? sub * 4 + (i & 1) * 2 + (i >> 1) * 32 : sub * 8 + 2 * i;
        c[i] = f2(ct[at], ct[at + 1]);
        s[i] = kBackward ? f2(-st[at], -st[at + 1]) : f2(st[at], st[at + 1]);
      }
    };
    // `tensor` is a compile-time 0 (q) or 1 (k), which keeps the parameters immediate
    auto load = [&](auto tensor, int trip) {
      constexpr int t = decltype(tensor)::value;
      Trip v;
      v.raw[0] = v.raw[1] = v.x[0] = v.x[1] = make_uint4(0, 0, 0, 0);
      const int h = 4 * trip + quarter;
      if (h < P.heads[t]) {
        const uint16_t* xp = P.x[t] + token * P.x_tok[t] + static_cast<long long>(h) * P.x_head[t] + sub * 8;
        if constexpr (kBackward) {
          const uint16_t* gp = P.dy[t] + (static_cast<long long>(token) * P.heads[t] + h) * kHeadDim + sub * 8;
          v.raw[0] = load16(gp);
          v.raw[1] = load16(gp + 64);
          if (kNorm && P.w[t] != nullptr) {
            v.x[0] = load16(xp);
            v.x[1] = load16(xp + 64);
          }
        } else {
          v.raw[0] = load16(xp);
          v.raw[1] = load16(xp + 64);
        }
      }
      return v;
    };
    auto turn = [&](auto tensor, int trip, const Trip& v) {
      constexpr int t = decltype(tensor)::value;
      const int h = 4 * trip + quarter;
      const bool normed = kNorm && P.w[t] != nullptr;
      F2 f[8];
      unpack16(v.raw[0], v.raw[1], f);
      if constexpr (!kBackward) {
        if (normed) {
          F2 sq = f[0] * f[0], wt[8];
#pragma unroll
          for (int i = 1; i < 8; ++i) sq = fma2(f[i], f[i], sq);
          unpack16(weights[t][sub], weights[t][8 + sub], wt);
          const F2 rstd = f2(rsqrtf(eight_lane_sum(sum(sq)) * (1.f / kHeadDim) + P.eps));
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = f[i] * rstd * wt[i];
        }
        rotate16<kInterleaved>(f, c, s);
      } else {
        if constexpr (kNorm) angles();  // from shared memory every time: registers are short
        rotate16<kInterleaved>(f, c, s);
        if (normed) {
          // n = x * rstd, g the gradient behind the norm: dw += g * n, dx = rstd * (g*w - n * mean(g*w*n)).
          // Rows that do not exist hold zeros and add nothing: their rstd, which eps = 0 would make infinite, is 0.
          F2 x[8], g[8], sq = f2(0.f), dot = f2(0.f);
          unpack16(v.x[0], v.x[1], x);
          unpack16(weights[t][sub], weights[t][8 + sub], g);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            g[i] = g[i] * f[i];
            sq = fma2(x[i], x[i], sq);
            dot = fma2(g[i], x[i], dot);
          }
          const float square = eight_lane_sum(sum(sq)) * (1.f / kHeadDim) + P.eps;
          const float rstd = h < P.heads[t] ? rsqrtf(square) : 0.f;
          const F2 r = f2(rstd), mean = f2(-eight_lane_sum(sum(dot)) * rstd * (1.f / kHeadDim));
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = x[i] * r;
            dw[t][i] = fma2(f[i], x[i], dw[t][i]);
            f[i] = r * fma2(x[i], mean, g[i]);
          }
        }
      }
      if (h < P.heads[t]) {
        uint16_t* op = P.out[t] + (static_cast<long long>(token) * P.heads[t] + h) * kHeadDim + sub * 8;
        store16(op, make_uint4(bf16_of_f2(f[0]), bf16_of_f2(f[1]), bf16_of_f2(f[2]), bf16_of_f2(f[3])));
        store16(op + 64, make_uint4(bf16_of_f2(f[4]), bf16_of_f2(f[5]), bf16_of_f2(f[6]), bf16_of_f2(f[7])));
      }
    };
    auto rest = [&](auto tensor, Trip v) {
      constexpr int t = decltype(tensor)::value;
      const int trips = (P.heads[t] + 3) >> 2;
      int trip = split_at;
      if constexpr (kBackward && kNorm) {  // no registers for a second trip: it reads two tensors
        if (trip < trips) turn(tensor, trip, v);
        for (trip += P.splits; trip < trips; trip += P.splits) turn(tensor, trip, load(tensor, trip));
      } else {
        for (; trip + P.splits < trips; trip += 2 * P.splits) {
          const Trip next = load(tensor, trip + P.splits);
          turn(tensor, trip, v);
          v = load(tensor, trip + 2 * P.splits);
          turn(tensor, trip + P.splits, next);
        }
        if (trip < trips) turn(tensor, trip, v);
      }
    };
    const std::integral_constant<int, 0> q{};
    const std::integral_constant<int, 1> k{};
    const Trip q0 = load(q, split_at);
    Trip k0;
    if constexpr (!(kBackward && kNorm)) k0 = load(k, split_at);
    __syncwarp();  // the table of the last token has been read
    warp_rotation(P, angle, token, lane, tables[warp][0], tables[warp][1]);
    if constexpr (!(kBackward && kNorm)) angles();
    rest(q, q0);
    if constexpr (kBackward && kNorm) k0 = load(k, split_at);
    rest(k, k0);
  }
  if constexpr (kBackward && kNorm) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v[2];
        split(dw[t][i], v[0], v[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          v[e] += __shfl_xor_sync(0xffffffffu, v[e], 8);
          v[e] += __shfl_xor_sync(0xffffffffu, v[e], 16);
          if (quarter == 0) reduce[warp][t][(i >> 2) * 64 + sub * 8 + 2 * (i & 3) + e] = v[e];
        }
      }
    __syncthreads();
    const int t = threadIdx.x >> 7, col = threadIdx.x & 127;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < kRotaryWarps; ++k) v += reduce[k][t][col];
    P.partial[(static_cast<long long>(blockIdx.x) * 2 + t) * kHeadDim + col] = v;
  }
}

// =============================================================================================
// Column sums of FP32 partials: out[s][col] (=|+=) sum over slots first(s) .. last(s) of part[slot][col].
// 128 columns a block (four a lane), 16 warps that each take every 16th slot, joined in order. Widths are
// multiples of four.
// =============================================================================================
struct FinishParams {
  const float* part;       // slot pitch `pitch`
  long long pitch;
  int width;
  int slots;               // samples == 0: slots 0 .. slots-1 go into one row
  const int* cu;           // samples > 0: the slots of sample s are c + s for its row chunks c
  int samples, tokens, chunk_rows;
  void* out[3];            // up to three results whose partials lie `width` floats apart in a slot
  int out_f32[3], accumulate[3];
};

__global__ void __launch_bounds__(512) finish_sums_kernel(const __grid_constant__ FinishParams P) {
  __shared__ float4 sums[16][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int col = blockIdx.x * 128 + lane * 4, which = blockIdx.y, sample = blockIdx.z;
  if (P.out[which] == nullptr) return;
  int first = 0, last = P.slots;
  if (P.samples > 0) {
    const int a = seq_bound(P.cu, sample, P.samples, P.tokens), b = seq_bound(P.cu, sample + 1, P.samples, P.tokens);
    first = a / P.chunk_rows + sample;
    last = b > a ? (b - 1) / P.chunk_rows + sample + 1 : first;
  }
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < P.width) {
    const float* p = P.part + static_cast<long long>(which) * P.width + col;
#pragma unroll 8
    for (int i = first + slice; i < last; i += 16) {
      const float4 x = __ldcs(reinterpret_cast<const float4*>(p + i * P.pitch));
      v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
    }
  }
  sums[slice][lane] = v;
  __syncthreads();
  if (slice == 0 && col < P.width) {
#pragma unroll
    for (int k = 1; k < 16; ++k) {
      const float4 x = sums[k][lane];
      v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
    }
    const long long at = static_cast<long long>(sample) * P.width + col;
    if (P.out_f32[which]) {
      float* o = static_cast<float*>(P.out[which]) + at;
      const bool add = P.accumulate[which];
      o[0] = add ? o[0] + v.x : v.x;
      o[1] = add ? o[1] + v.y : v.y;
      o[2] = add ? o[2] + v.z : v.z;
      o[3] = add ? o[3] + v.w : v.w;
    } else {
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(P.out[which]) + at) =
          make_uint2(bf16_of_f2(f2(v.x, v.y)), bf16_of_f2(f2(v.z, v.w)));
    }
  }
}

// =============================================================================================
// Norm around a block.  r = x + gate * branch;  n = (r - mean) * rstd (mean only when centred);
// y = n * weight * (1 + scale) + shift.  gate, scale and shift are one row per packed sample.
//
// A block takes a chunk of consecutive rows, a thread the same 8 * kVec columns of each, so weight,
// scale, shift and gate stay on the SM from row to row (forward in registers; backward in shared memory, because
// the column sums, register sums over the chunk, leave no registers for them: 156 -> 134 us at 16384 x 4096
// with gate, scale and shift). Slot chunk + sample of the partial sums is unique: walking down the rows
// either of the two grows. The next rows are on their way to shared memory meanwhile, each thread fetching
// what it will read itself, so a row costs one barrier (two when centred) for its sums.
//
// Bound by memory: 8191 x 5120 with a residual sum 53 us (6.3 TB/s), 16384 x 4096 centred with gate, scale
// and shift 89 us forward (6.0 TB/s) and 132 to 135 us backward (6.0 TB/s: six streams, 48 FP32 column sums a
// thread). Narrow rows are bound by latency: norm_chunk_rows() counts on the same four blocks an SM for all widths up
// to 1024, whose warps are then few (32768 rows backward: 71 us at 64 columns as at 512, 75 us at 1024).
// =============================================================================================
struct NormParams {
  const uint16_t *x, *branch, *weight, *gate, *scale, *shift;
  const int* cu;
  int samples, tokens, hidden, chunk_rows, center;
  float eps;
  uint16_t *y, *r;            // forward outputs (r may be null: no branch)
  float *rstd, *mean;         // [tokens]: written by forward (may be null), read by backward
  const uint16_t *dy, *dr;    // backward: either may be null
  uint16_t *dx, *dbranch;     // dbranch only with a gate
  float* part_weight;         // [chunks][hidden] or null
  float* part_mod;            // [chunks + samples][3][hidden]: gate, scale, shift; or null
};

// Sum of N values over the block; `buf` alternates between two halves so that one barrier is enough.
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float* buf, int warps) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) buf[i * 32 + warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = lane < warps ? buf[i * 32 + lane] : 0.f;
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    v[i] = s;
  }
}

struct RowRange {
  int sample, end;  // current sample (or P.samples: padding) and the row at which it ends
};

__device__ __forceinline__ RowRange range_of(const NormParams& P, int row) {
  RowRange s;
  s.sample = P.cu == nullptr ? 0 : seq_of_row(P.cu, P.samples, P.tokens, row);
  s.end = s.sample < P.samples ? seq_bound(P.cu, s.sample + 1, P.samples, P.tokens) : P.tokens;
  if (s.end <= row) s.end = row + 1;  // offsets that do not ascend
  return s;
}

constexpr int kRowsAhead = 2;  // rows in flight: more (3 or 4) cost up to a fifth, their shared memory costs a block

template <int kVec>
__global__ void __launch_bounds__(256 * kVec) norm_forward_kernel(const NormParams P) {
  __shared__ float buf[2][64];
  extern __shared__ uint4 ring[];  // every thread's own pieces: [row][x, branch][kVec][thread]
  const int warps = blockDim.x >> 5;
  const int row0 = blockIdx.x * P.chunk_rows, row1 = min(row0 + P.chunk_rows, P.tokens);
  const int vecs = P.hidden >> 3;
  const float inv_h = 1.f / P.hidden;
  uint4 wt[kVec], gt[kVec], sc[kVec], sh[kVec];
  bool on[kVec];
  int col[kVec];
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    const int v = threadIdx.x + k * blockDim.x;
    on[k] = v < vecs;
    col[k] = v * 8;
    wt[k] = gt[k] = sc[k] = sh[k] = make_uint4(0, 0, 0, 0);
    if (on[k] && P.weight != nullptr) wt[k] = load16(P.weight + col[k]);
  }
  const uint32_t mine = smem_u32(ring) + threadIdx.x * 16, piece = blockDim.x * 16;
  auto fetch = [&](int row) {  // a group per row, also when there is none left
    if (row < row1) {
      const uint32_t at = mine + (row % kRowsAhead) * 2 * kVec * piece;
#pragma unroll
      for (int k = 0; k < kVec; ++k)
        if (on[k]) {
          const long long from = static_cast<long long>(row) * P.hidden + col[k];
          copy16_async(at + k * piece, P.x + from);
          if (P.branch != nullptr) copy16_async(at + (kVec + k) * piece, P.branch + from);
        }
    }
    copy_commit();
  };
  for (int i = 0; i < kRowsAhead; ++i) fetch(row0 + i);
  RowRange s{0, 0};
  int parity = 0;
  for (int row = row0; row < row1; ++row) {
    if (row == row0 || row >= s.end) {
      s = range_of(P, row);
      if (s.sample < P.samples) {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (on[k]) {
            const long long at = static_cast<long long>(s.sample) * P.hidden + col[k];
            if (P.gate != nullptr) gt[k] = load16(P.gate + at);
            if (P.scale != nullptr) sc[k] = load16(P.scale + at);
            if (P.shift != nullptr) sh[k] = load16(P.shift + at);
          }
      }
    }
    const bool padding = s.sample >= P.samples;
    F2 r[kVec][4];
    copy_wait<kRowsAhead - 1>();
    const uint32_t slot = mine + (row % kRowsAhead) * 2 * kVec * piece;
    F2 total = f2(0.f);
#pragma unroll
    for (int k = 0; k < kVec; ++k) {
      unpack8(on[k] ? shared16(slot + k * piece) : make_uint4(0, 0, 0, 0), r[k]);  // columns beyond the row hold zeros
      if (on[k] && P.branch != nullptr && !(padding && P.gate != nullptr)) {
        F2 b[4], g[4];
        unpack8(shared16(slot + (kVec + k) * piece), b);
        unpack8(gt[k], g);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[k][i] = P.gate != nullptr ? fma2(g[i], b[i], r[k][i]) : r[k][i] + b[i];
        store16(P.r + static_cast<long long>(row) * P.hidden + col[k], pack8(r[k]));
      } else if (on[k] && P.r != nullptr) {
        store16(P.r + static_cast<long long>(row) * P.hidden + col[k], pack8(r[k]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) total = total + r[k][i];
    }
    float mean = 0.f;
    if (P.center) {
      float t[1] = {sum(total)};
      block_sum(t, buf[parity], warps);
      parity ^= 1;
      mean = t[0] * inv_h;
      const F2 minus = f2(-mean);
#pragma unroll
      for (int k = 0; k < kVec; ++k)
        if (on[k])
#pragma unroll
          for (int i = 0; i < 4; ++i) r[k][i] = r[k][i] + minus;
    }
    total = f2(0.f);
#pragma unroll
    for (int k = 0; k < kVec; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) total = fma2(r[k][i], r[k][i], total);
    float t[1] = {sum(total)};
    block_sum(t, buf[parity], warps);
    parity ^= 1;
    fetch(row + kRowsAhead);  // this row's pieces are in registers
    const float rstd = rsqrtf(t[0] * inv_h + P.eps);
    if (threadIdx.x == 0 && P.rstd != nullptr) {
      P.rstd[row] = rstd;
      if (P.mean != nullptr) P.mean[row] = mean;
    }
    const F2 scaled = f2(rstd);
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      if (on[k]) {
        F2 y[4], e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = r[k][i] * scaled;
        if (P.weight != nullptr) {
          unpack8(wt[k], e);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = y[i] * e[i];
        }
        if (P.scale != nullptr) {
          unpack8(sc[k], e);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = fma2(y[i], e[i], y[i]);
        }
        if (P.shift != nullptr) {
          unpack8(sh[k], e);
#pragma unroll
          for (int i = 0; i < 4; ++i) y[i] = y[i] + e[i];
        }
        store16(P.y + static_cast<long long>(row) * P.hidden + col[k], padding ? make_uint4(0, 0, 0, 0) : pack8(y));
      }
  }
}

// dz = dy * (1 + scale);  dn = dz * weight;  dc = rstd * (dn - n * mean(dn * n)) (- its mean when centred)
// dx = dr + dc;  dbranch = gate * dx;  sums over the rows of a sample: dgate = sum dx * branch,
// dshift = sum dy, a = sum dy * n, from which dscale = a * weight and dweight gets (1 + scale) * a. The
// mean over a centred row of dc is rstd * mean(dn), because the mean of n is zero up to rounding.
//
// With a gate, whose gradient needs the branch anyway, r is computed again from x and the branch, exactly as
// the forward pass did. So it is where the norm is centred: r as it was stored is off by up to 2^-8 of r, which
// beside r - mean is anything (a mean of 40 deviations: 10 % of n). An RMS norm without a gate reads the stored
// r, whose rounding is then at most 2^-8 of n: gradients are 2.4e-3 from 64 bits in the 2-norm, where rounding
// them alone gives 1.7e-3, and computing r again would be five streams instead of four in a pass bound by memory.
template <int kVec, bool kMod, bool kRebuild>
__global__ void __launch_bounds__(256 * kVec) norm_backward_kernel(const NormParams P) {
  __shared__ float buf[2][64];
  extern __shared__ uint4 ring[];  // every thread's own pieces: [row][r or x, dy, dr, branch][kVec][thread]
  static_assert(kMod || !kRebuild, "the branch has a place in the ring only there");
  constexpr int kParts = kMod ? 4 : 3;
  const int warps = blockDim.x >> 5;
  const int row0 = blockIdx.x * P.chunk_rows, row1 = min(row0 + P.chunk_rows, P.tokens);
  const int vecs = P.hidden >> 3;
  const float inv_h = 1.f / P.hidden;
  F2 sa[kVec][4], dg[kVec][4], dh[kVec][4];
  bool on[kVec];
  int col[kVec];
  auto clear = [&]() {
#pragma unroll
    for (int k = 0; k < kVec; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[k][i] = dg[k][i] = dh[k][i] = f2(0.f);
  };
#pragma unroll
  for (int k = 0; k < kVec; ++k) {
    const int v = threadIdx.x + k * blockDim.x;
    on[k] = v < vecs;
    col[k] = v * 8;
  }
  clear();
  const uint32_t mine = smem_u32(ring) + threadIdx.x * 16, piece = blockDim.x * 16;
  // weight, gate and scale of this thread's columns, behind the rows in flight: registers are short
  const uint32_t kept = mine + kRowsAhead * kParts * kVec * piece;
  auto keep = [&](int which, int k, const uint16_t* from) {
    const uint4 v = load16(from);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(kept + (which * kVec + k) * piece), "r"(v.x), "r"(v.y),
                 "r"(v.z), "r"(v.w)
                 : "memory");
  };
  auto kept_row = [&](int which, int k) { return shared16(kept + (which * kVec + k) * piece); };
  if (P.weight != nullptr)
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      if (on[k]) keep(0, k, P.weight + col[k]);
  if (kRebuild && P.gate == nullptr)  // a gate of 1: the sum comes out as an addition's
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(kept + (kVec + k) * piece), "r"(0x3f803f80) : "memory");
  auto fetch = [&](int row) {  // a group per row, also when there is none left
    if (row < row1) {
      const uint32_t at = mine + (row % kRowsAhead) * kParts * kVec * piece;
#pragma unroll
      for (int k = 0; k < kVec; ++k)
        if (on[k]) {
          const long long from = static_cast<long long>(row) * P.hidden + col[k];
          copy16_async(at + k * piece, P.x + from);
          if (P.dy != nullptr) copy16_async(at + (kVec + k) * piece, P.dy + from);
          if (P.dr != nullptr) copy16_async(at + (2 * kVec + k) * piece, P.dr + from);
          if (kMod && P.branch != nullptr) copy16_async(at + (3 * kVec + k) * piece, P.branch + from);
        }
    }
    copy_commit();
  };
  // Leaves the sums of the rows of `sample` behind. `fresh`: the first flush of this block.
  auto flush = [&](int sample, bool fresh) {
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      if (on[k]) {
        const uint4 none = make_uint4(0, 0, 0, 0);
        F2 w[4], a[4];
        unpack8(P.weight != nullptr ? kept_row(0, k) : none, w);
        unpack8(kMod && P.scale != nullptr ? kept_row(2, k) : none, a);
        auto put = [&](float* at, const F2(&v)[4], bool add) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float4 o, *p = reinterpret_cast<float4*>(at) + i;
            split(v[2 * i], o.x, o.y);
            split(v[2 * i + 1], o.z, o.w);
            if (add) {
              const float4 q = *p;
              o = make_float4(o.x + q.x, o.y + q.y, o.z + q.z, o.w + q.w);
            }
            *p = o;
          }
        };
        F2 v[4];
        if (kMod && P.part_mod != nullptr) {
          float* base = P.part_mod + static_cast<long long>(blockIdx.x + sample) * 3 * P.hidden + col[k];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = P.weight != nullptr ? sa[k][i] * w[i] : sa[k][i];
          put(base, dg[k], false);
          put(base + P.hidden, v, false);
          put(base + 2 * P.hidden, dh[k], false);
        }
        if (P.part_weight != nullptr) {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = kMod && P.scale != nullptr ? fma2(sa[k][i], a[i], sa[k][i]) : sa[k][i];
          put(P.part_weight + static_cast<long long>(blockIdx.x) * P.hidden + col[k], v, !fresh);
        }
      }
    clear();
  };
  for (int i = 0; i < kRowsAhead; ++i) fetch(row0 + i);
  float next_rstd = row0 < row1 ? __ldg(P.rstd + row0) : 0.f;
  float next_mean = row0 < row1 && P.mean != nullptr ? __ldg(P.mean + row0) : 0.f;
  RowRange s{P.samples, 0};
  int parity = 0;
  bool fresh = true;
  for (int row = row0; row < row1; ++row) {
    if (row == row0 || row >= s.end) {
      if (row != row0 && s.sample < P.samples) {
        flush(s.sample, fresh);
        fresh = false;
      }
      s = range_of(P, row);
      if (kMod && s.sample < P.samples) {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (on[k]) {
            const long long at = static_cast<long long>(s.sample) * P.hidden + col[k];
            if (P.gate != nullptr) keep(1, k, P.gate + at);
            if (P.scale != nullptr) keep(2, k, P.scale + at);
          }
      }
    }
    const bool padding = s.sample >= P.samples;
    const float rstd = next_rstd, mean = next_mean;
    if (row + 1 < row1) {  // a trip to memory ahead
      next_rstd = __ldg(P.rstd + row + 1);
      if (P.mean != nullptr) next_mean = __ldg(P.mean + row + 1);
    }
    F2 n[kVec][4], dn[kVec][4], dot2 = f2(0.f), sum2 = f2(0.f);
    copy_wait<kRowsAhead - 1>();
    const uint32_t slot = mine + (row % kRowsAhead) * kParts * kVec * piece;
    const F2 scaled = f2(rstd), offset = f2(-mean * rstd);
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      if (!padding && on[k]) {
        F2 e[4];
        unpack8(shared16(slot + k * piece), n[k]);
        if constexpr (kRebuild) {
          F2 g[4];
          unpack8(shared16(slot + (3 * kVec + k) * piece), e);
          unpack8(kept_row(1, k), g);
#pragma unroll
          for (int i = 0; i < 4; ++i) n[k][i] = fma2(g[i], e[i], n[k][i]);
        }
        unpack8(P.dy != nullptr ? shared16(slot + (kVec + k) * piece) : make_uint4(0, 0, 0, 0), dn[k]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          n[k][i] = fma2(n[k][i], scaled, offset);
          sa[k][i] = fma2(dn[k][i], n[k][i], sa[k][i]);
          if (kMod) dh[k][i] = dh[k][i] + dn[k][i];
        }
        if (kMod && P.scale != nullptr) {
          unpack8(kept_row(2, k), e);
#pragma unroll
          for (int i = 0; i < 4; ++i) dn[k][i] = fma2(dn[k][i], e[i], dn[k][i]);
        }
        if (P.weight != nullptr) {
          unpack8(kept_row(0, k), e);
#pragma unroll
          for (int i = 0; i < 4; ++i) dn[k][i] = dn[k][i] * e[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          dot2 = fma2(dn[k][i], n[k][i], dot2);
          sum2 = sum2 + dn[k][i];
        }
      }
    float t[2] = {sum(dot2), sum(sum2)};
    block_sum(t, buf[parity], warps);
    parity ^= 1;
    const F2 dot = f2(-t[0] * inv_h), avg = f2(P.center ? -t[1] * inv_h : 0.f);
#pragma unroll
    for (int k = 0; k < kVec; ++k)
      if (on[k]) {
        const long long at = static_cast<long long>(row) * P.hidden + col[k];
        F2 d[4];
        unpack8(P.dr != nullptr ? shared16(slot + (2 * kVec + k) * piece) : make_uint4(0, 0, 0, 0), d);
        if (!padding)
#pragma unroll
          for (int i = 0; i < 4; ++i) d[i] = fma2(scaled, fma2(n[k][i], dot, dn[k][i] + avg), d[i]);
        store16(P.dx + at, pack8(d));
        if (kMod && P.dbranch != nullptr) {
          F2 b[4], g[4];
          unpack8(shared16(slot + (3 * kVec + k) * piece), b);
          unpack8(kept_row(1, k), g);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!padding) dg[k][i] = fma2(d[i], b[i], dg[k][i]);
            g[i] = g[i] * d[i];
          }
          store16(P.dbranch + at, padding ? make_uint4(0, 0, 0, 0) : pack8(g));
        }
      }
    fetch(row + kRowsAhead);  // what it overwrites this thread has read and used
  }
  if (row0 < row1) {
    if (s.sample < P.samples) {
      flush(s.sample, fresh);
    } else if (fresh && P.part_weight != nullptr) {
      float* base = P.part_weight + static_cast<long long>(blockIdx.x) * P.hidden;  // nothing but padding
      for (int i = threadIdx.x; i < P.hidden; i += blockDim.x) base[i] = 0.f;
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// Rows a norm block walks: as many blocks as are taken to be resident at once (four on an SM up to 1024 columns,
// else two) share the rows evenly; at least one row. A forward pass that has no per-sample rows to load takes a
// fourth of that, so that SMs which are ahead take more (8191 x 5120: 62.5 -> 55.2 us; with gate, scale and
// shift loaded four times as often 16384 x 4096 went from 90 to 94 us). In the backward pass every block
// leaves its sums behind.
int norm_chunk_rows(long long tokens, int hidden, int sms) {
  return static_cast<int>(ceil_div(tokens, (hidden <= 1024 ? 4ll : 2ll) * sms));
}

struct NormShape {
  int vec, threads;
};
// 8 columns a thread up to 2048 columns, 16 above: a block of at most 256 threads for 2048 columns and
// 512 for 8192. The modulated backward kernels have 126 registers at 16 columns, so two blocks share an SM up to
// 4096 columns; above, one does, and the grid of two an SM takes two rounds there.
NormShape norm_shape(int hidden) {
  const int vecs = hidden / 8, vec = hidden <= 2048 ? 1 : 2;
  return {vec, static_cast<int>(ceil_div(ceil_div(vecs, vec), 32) * 32)};
}

// Bytes of the rows in flight, `parts` tensors each, and of `kept` rows beside them: 16 bytes a thread and vector.
uint32_t norm_smem(NormShape s, int parts, int kept) { return 16u * s.vec * s.threads * (kRowsAhead * parts + kept); }

// `done`: the kernel's own, for allow_smem().
int run_norm(void (*kernel)(NormParams), uint64_t& done, int grid, NormShape shape, int parts, int kept,
             const NormParams& P, cudaStream_t st) {
  const NormShape widest = norm_shape(shape.vec == 1 ? 2048 : 8192);
  const int rc = allow_smem(kernel, norm_smem(widest, parts, kept), done);
  if (rc != kSuccess) return rc;
  kernel<<<grid, shape.threads, norm_smem(shape, parts, kept), st>>>(P);
  return kSuccess;
}
uint64_t g_norm_smem[8];  // forward, backward, modulated, with r built again; each with 8 and 16 columns a thread

int rotary_grid(long long units, bool sums, int sms) {
  // With sums every block leaves a row of partials behind, so the grid is what is resident at once.
  const long long blocks = ceil_div(units, kRotaryWarps), most = sums ? 2ll * sms : 8ll * sms;
  return static_cast<int>(blocks < most ? blocks : most);
}

// Warps a token's heads are spread over: as many as it takes to give every SM 16 warps.
int rotary_splits(long long tokens, int heads, int sms) {
  const long long want = ceil_div(16ll * sms, tokens), most = (heads + 3) / 4;
  return static_cast<int>(want < most ? want : most);
}

int launch_rotary(const RotaryParams& P, int interleaved, bool backward, bool norm, int grid, cudaStream_t st) {
  const dim3 g(grid), b(32 * kRotaryWarps);
  if (interleaved) {
    if (!backward) {
      if (norm) rotary_kernel<true, false, true><<<g, b, 0, st>>>(P);
      else rotary_kernel<true, false, false><<<g, b, 0, st>>>(P);
    } else {
      if (norm) rotary_kernel<true, true, true><<<g, b, 0, st>>>(P);
      else rotary_kernel<true, true, false><<<g, b, 0, st>>>(P);
    }
  } else {
    if (!backward) {
      if (norm) rotary_kernel<false, false, true><<<g, b, 0, st>>>(P);
      else rotary_kernel<false, false, false><<<g, b, 0, st>>>(P);
    } else {
      if (norm) rotary_kernel<false, true, true><<<g, b, 0, st>>>(P);
      else rotary_kernel<false, true, false><<<g, b, 0, st>>>(P);
    }
  }
  FGA_LAUNCHED();
  return kSuccess;
}

int check_rotary(const FgaRotary* a, bool backward, RotaryParams& P) {
  FGA_REQUIRE(a != nullptr, "rotary: null arguments");
  FGA_REQUIRE(a->tokens >= 1 && a->tokens <= 0x7fff0000, "rotary: tokens must be in [1, 2^31 - 2^16]");
  FGA_REQUIRE(a->positions != nullptr && a->inv_freq != nullptr, "rotary: null pointer");
  FGA_REQUIRE(a->axes >= 1 && a->axes <= 4, "rotary: one to four axes");
  int at = 0;
  for (int i = 0; i < a->axes; ++i) {
    FGA_REQUIRE(a->sections[i] >= 0 && a->sections[i] <= 64, "rotary: a section has 0 to 64 pairs");
    at += a->sections[i];
    P.ends[i] = at;
  }
  FGA_REQUIRE(at == 64, "rotary: the sections must add up to 64 pairs, not %d", at);
  for (int t = 0; t < 2; ++t) {
    FGA_REQUIRE(a->heads[t] >= 1 && a->heads[t] <= 65536, "rotary: 1 to 65536 heads");
    const bool reads_x = !backward || a->weight[t] != nullptr;
    FGA_REQUIRE(a->out[t] != nullptr && (a->x[t] != nullptr || !reads_x) && (a->dy[t] != nullptr || !backward),
                "rotary: null pointer");
    FGA_REQUIRE(aligned16(a->x[t]) && aligned16(a->dy[t]) && aligned16(a->out[t]) && aligned16(a->weight[t]),
                "rotary: pointers must be 16-byte aligned");
    FGA_REQUIRE(a->dweight_f32[t] || aligned16(a->dweight[t]), "rotary: pointers must be 16-byte aligned");
    FGA_REQUIRE(a->x_token_stride[t] % 8 == 0 && a->x_head_stride[t] % 8 == 0,
                "rotary: strides must be multiples of 8 elements");
    P.x[t] = static_cast<const uint16_t*>(a->x[t]);
    P.dy[t] = static_cast<const uint16_t*>(a->dy[t]);
    P.out[t] = static_cast<uint16_t*>(a->out[t]);
    P.w[t] = static_cast<const uint16_t*>(a->weight[t]);
    P.x_tok[t] = a->x_token_stride[t];
    FGA_REQUIRE(a->x_head_stride[t] >= 0 && a->x_head_stride[t] <= 0x7fffffff, "rotary: head stride out of range");
    P.x_head[t] = static_cast<int>(a->x_head_stride[t]);
    P.heads[t] = a->heads[t];
  }
  P.pos = a->positions;
  P.pos64 = a->positions_int64;
  P.axes = a->axes;
  P.freq = a->inv_freq;
  P.freq64 = a->inv_freq_f64;
  P.tokens = static_cast<int>(a->tokens);
  P.eps = a->eps;
  P.splits = rotary_splits(a->tokens, a->heads[0] > a->heads[1] ? a->heads[0] : a->heads[1], sm_count());
  return kSuccess;
}

int check_norm(const FgaNorm* a, bool backward, NormParams& P) {
  FGA_REQUIRE(a != nullptr, "norm: null arguments");
  // 2^16 rows of room: a chunk's end and the rows fetched ahead of it are 32-bit sums
  FGA_REQUIRE(a->tokens >= 1 && a->tokens <= 0x7fff0000, "norm: tokens must be in [1, 2^31 - 2^16]");
  FGA_REQUIRE(a->hidden >= 8 && a->hidden % 8 == 0 && a->hidden <= 8192, "norm: hidden must be a multiple of 8 up to 8192");
  FGA_REQUIRE(a->samples >= 1 && a->samples <= 65535, "norm: 1 to 65535 samples");
  FGA_REQUIRE(a->cu_seqlens != nullptr || a->samples == 1, "norm: several samples need cu_seqlens");
  FGA_REQUIRE(a->gate == nullptr || a->branch != nullptr, "norm: a gate needs a branch");
  const void* all[] = {a->x,  a->branch, a->weight,  a->gate,  a->scale, a->shift,  a->y,       a->r,
                       a->dy, a->dr,     a->dx,      a->dbranch, a->dgate, a->dscale, a->dshift, a->scratch,
                       a->dweight_f32 ? nullptr : a->dweight};
  for (const void* p : all) FGA_REQUIRE(aligned16(p), "norm: pointers must be 16-byte aligned");
  P.x = static_cast<const uint16_t*>(a->x);
  P.branch = static_cast<const uint16_t*>(a->branch);
  P.weight = static_cast<const uint16_t*>(a->weight);
  P.gate = static_cast<const uint16_t*>(a->gate);
  P.scale = static_cast<const uint16_t*>(a->scale);
  P.shift = static_cast<const uint16_t*>(a->shift);
  P.cu = a->cu_seqlens;
  P.center = a->center;
  P.eps = a->eps;
  P.y = static_cast<uint16_t*>(a->y);
  P.r = static_cast<uint16_t*>(a->r);
  P.rstd = a->rstd;
  P.mean = a->center ? a->mean : nullptr;
  P.dy = static_cast<const uint16_t*>(a->dy);
  P.dr = static_cast<const uint16_t*>(a->dr);
  P.dx = static_cast<uint16_t*>(a->dx);
  P.dbranch = static_cast<uint16_t*>(a->dbranch);
  P.tokens = static_cast<int>(a->tokens);
  P.hidden = a->hidden;
  P.samples = a->samples;
  const int rows = norm_chunk_rows(a->tokens, a->hidden, sm_count());
  P.chunk_rows = backward || a->gate || a->scale || a->shift ? rows : (rows + 3) / 4;
  return kSuccess;
}

}  // namespace
}  // namespace fga

using namespace fga;

extern "C" {

int fga_rotary_forward(const FgaRotary* args, void* stream) {
  RotaryParams P = {};
  const int rc = check_rotary(args, false, P);
  if (rc != kSuccess) return rc;
  const int grid = rotary_grid(static_cast<long long>(P.tokens) * P.splits, false, sm_count());
  return launch_rotary(P, args->interleaved, false, P.w[0] || P.w[1], grid, static_cast<cudaStream_t>(stream));
}

int64_t fga_rotary_scratch_floats(int64_t tokens, int q_heads, int k_heads) {
  if (tokens < 1 || q_heads < 1 || k_heads < 1) return 0;
  const int sms = sm_count();
  const int splits = rotary_splits(tokens, q_heads > k_heads ? q_heads : k_heads, sms);
  return static_cast<int64_t>(rotary_grid(tokens * splits, true, sms)) * 2 * kHeadDim;
}

int fga_rotary_backward(const FgaRotary* args, void* stream) {
  RotaryParams P = {};
  int rc = check_rotary(args, true, P);
  if (rc != kSuccess) return rc;
  const bool norm = P.w[0] || P.w[1];
  FGA_REQUIRE(args->dweight[0] == nullptr || args->dweight[0] != args->dweight[1] ||
                  (args->dweight_f32[0] && args->dweight_f32[1] && args->dweight_accumulate[1]),
              "rotary: one weight gradient for both tensors must be FP32 and accumulate");
  FGA_REQUIRE(!norm || (args->scratch != nullptr && aligned16(args->scratch)), "rotary: weight gradients need scratch");
  P.partial = args->scratch;
  const int grid = rotary_grid(static_cast<long long>(P.tokens) * P.splits, norm, sm_count());
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = launch_rotary(P, args->interleaved, true, norm, grid, st);
  if (rc != kSuccess || !norm || (!args->dweight[0] && !args->dweight[1])) return rc;
  FinishParams F = {};
  F.part = args->scratch;
  F.pitch = 2 * kHeadDim;
  F.width = kHeadDim;
  F.slots = grid;
  for (int t = 0; t < 2; ++t) {
    F.out[t] = args->weight[t] ? args->dweight[t] : nullptr;
    F.out_f32[t] = args->dweight_f32[t];
    F.accumulate[t] = args->dweight_accumulate[t];
  }
  const bool shared = F.out[0] != nullptr && F.out[0] == F.out[1];
  if (shared) F.out[1] = nullptr;
  finish_sums_kernel<<<dim3(1, 2, 1), 512, 0, st>>>(F);
  FGA_LAUNCHED();
  if (shared) {  // one gradient for both weights: k's sums are added when q's are there
    F.out[1] = F.out[0];
    F.out[0] = nullptr;
    finish_sums_kernel<<<dim3(1, 2, 1), 512, 0, st>>>(F);
    FGA_LAUNCHED();
  }
  return kSuccess;
}

int fga_norm_forward(const FgaNorm* args, void* stream) {
  NormParams P = {};
  const int rc = check_norm(args, false, P);
  if (rc != kSuccess) return rc;
  FGA_REQUIRE(P.x != nullptr && P.y != nullptr && (P.branch == nullptr) == (P.r == nullptr),
              "norm: x, y, and r exactly where there is a branch");
  FGA_REQUIRE(P.rstd == nullptr || !P.center || P.mean != nullptr, "norm: a centred norm keeps its means beside rstd");
  const NormShape shape = norm_shape(P.hidden);
  const int grid = static_cast<int>(ceil_div(P.tokens, P.chunk_rows));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc2 = shape.vec == 1 ? run_norm(norm_forward_kernel<1>, g_norm_smem[0], grid, shape, 2, 0, P, st)
                                 : run_norm(norm_forward_kernel<2>, g_norm_smem[1], grid, shape, 2, 0, P, st);
  if (rc2 != kSuccess) return rc2;
  FGA_LAUNCHED();
  return kSuccess;
}

int64_t fga_norm_scratch_floats(int64_t tokens, int hidden, int samples, int has_weight, int modulated) {
  if (tokens < 1 || hidden < 1 || samples < 1) return 0;
  const int64_t chunks = ceil_div(tokens, norm_chunk_rows(tokens, hidden, sm_count()));
  return (has_weight ? chunks * hidden : 0) + (modulated ? (chunks + samples) * 3 * hidden : 0);
}

int fga_norm_backward(const FgaNorm* args, void* stream) {
  NormParams P = {};
  int rc = check_norm(args, true, P);
  if (rc != kSuccess) return rc;
  const bool rebuild = P.x != nullptr && P.branch != nullptr;
  if (!rebuild) P.x = P.r;  // what the forward normalised: the residual sum, or x itself where there is no branch
  if (!rebuild && P.gate == nullptr) P.branch = nullptr;
  const bool modulated = args->dgate || args->dscale || args->dshift;
  FGA_REQUIRE(P.x != nullptr && P.dx != nullptr && P.rstd != nullptr && (!P.center || P.mean != nullptr),
              "norm: null pointer");
  FGA_REQUIRE((P.gate == nullptr) == (P.dbranch == nullptr), "norm: dbranch exactly where there is a gate");
  FGA_REQUIRE(args->scratch != nullptr || (!modulated && args->dweight == nullptr), "norm: sums over rows need scratch");
  const long long chunks = ceil_div(P.tokens, P.chunk_rows);
  if (args->dweight != nullptr) P.part_weight = args->scratch;
  if (modulated) P.part_mod = args->scratch + (args->dweight != nullptr ? chunks * P.hidden : 0);
  const NormShape shape = norm_shape(P.hidden);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = static_cast<int>(chunks);
  const bool mod = P.branch || P.scale || modulated;
  if (shape.vec == 1)
    rc = rebuild ? run_norm(norm_backward_kernel<1, true, true>, g_norm_smem[6], grid, shape, 4, 3, P, st)
         : mod   ? run_norm(norm_backward_kernel<1, true, false>, g_norm_smem[4], grid, shape, 4, 3, P, st)
                 : run_norm(norm_backward_kernel<1, false, false>, g_norm_smem[2], grid, shape, 3, 1, P, st);
  else
    rc = rebuild ? run_norm(norm_backward_kernel<2, true, true>, g_norm_smem[7], grid, shape, 4, 3, P, st)
         : mod   ? run_norm(norm_backward_kernel<2, true, false>, g_norm_smem[5], grid, shape, 4, 3, P, st)
                 : run_norm(norm_backward_kernel<2, false, false>, g_norm_smem[3], grid, shape, 3, 1, P, st);
  if (rc != kSuccess) return rc;
  FGA_LAUNCHED();
  const int blocks = static_cast<int>(ceil_div(P.hidden, 128));
  if (args->dweight != nullptr) {
    FinishParams F = {};
    F.part = P.part_weight;
    F.pitch = P.hidden;
    F.width = P.hidden;
    F.slots = static_cast<int>(chunks);
    F.out[0] = args->dweight;
    F.out_f32[0] = args->dweight_f32;
    F.accumulate[0] = args->dweight_accumulate;
    finish_sums_kernel<<<dim3(blocks, 1, 1), 512, 0, st>>>(F);
    FGA_LAUNCHED();
  }
  if (modulated) {
    FinishParams F = {};
    F.part = P.part_mod;
    F.pitch = 3ll * P.hidden;
    F.width = P.hidden;
    F.cu = P.cu;
    F.samples = P.samples;
    F.tokens = P.tokens;
    F.chunk_rows = P.chunk_rows;
    F.out[0] = args->dgate;
    F.out[1] = args->dscale;
    F.out[2] = args->dshift;
    finish_sums_kernel<<<dim3(blocks, 3, P.samples), 512, 0, st>>>(F);
    FGA_LAUNCHED();
  }
  return kSuccess;
}

}  // extern "C"
