// Attention over packed sequences on tcgen05 tensor cores (sm_100a): softmax(scale Q K^T) V for each
// sequence and head, optionally causal, with shared key/value heads; forward and backward, BF16 operands,
// FP32 accumulation and statistics. Head dimension 128.
//
// Common to the kernels: one block per SM, which works alone except in the dK/dV kernel, where a cluster of two
// or four may share a tile. Operand tiles are 128 rows x 128
// columns, 32 KiB in two 64-column halves with the 128-byte swizzle, TMA-loaded from a 3-D map [tokens,
// heads, 128], so any row may start a tile and rows behind the tensor read as zero. The same tile serves as
// K-major operand (reduction over its columns) and as MN-major one (reduction over its rows): only the
// descriptor differs. Products accumulate in TMEM, where a thread of the four warps of a warpgroup owns a
// row; probabilities go back to TMEM as the BF16 A operand of the next product and never touch shared
// memory.
//
// A tile that ends behind its sequence holds rows of the next one, or of nothing at all. They are masked in
// the softmax, but 0 * NaN is NaN in a matrix product, so the loading warp overwrites such rows with zeros
// in shared memory before it hands the tile over.
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>
#include "../../include/fga.h"
#include "common.cuh"
#include "f32x2.cuh"
#include "ptx.cuh"
#include "seq_bounds.cuh"
#include "wait.cuh"

namespace fga {
namespace {

constexpr int kTile = 128;                // rows of an operand tile
constexpr int kDim = 128;                 // head dimension
constexpr uint32_t kHalfBytes = 16384;    // 128 rows x 128 bytes
constexpr uint32_t kTileBytes = 2 * kHalfBytes;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Range of the scores. The exponent of a probability is fma(s, scale * log2(e), -top) with `top`, the row's largest
// product, rounded to FP32. All of a row's probabilities are off by the same factor then, which their sum
// undoes, as long as it stays inside FP32: half a step is 16 at 2^29. The backward pass starts from the
// logarithm of the sum, rounded twice, and nothing undoes that: probabilities are off by about 2^-23 of the score,
// half a BF16 step at 2^15 and an eighth at 2^20. Rows beyond come out as NaN, not as plausible values.
constexpr float kMaxTop = 536870912.f;  // 2^29, in units of log2
constexpr float kMaxLse = 1048576.f;    // 2^20
__device__ __forceinline__ float exponent_of_lse(float lse) {
  return fabsf(lse) <= kMaxLse ? -kLog2e * lse : __int_as_float(0x7fffffff);
}

struct AttentionParams {
  const int* cu;
  int samples, tokens, heads, kv_heads, group;  // group = heads / kv_heads
  int causal;
  float scale_log2;                             // scale * log2(e)
  uint16_t* o;                                  // forward: [tokens, heads, 128]
  float* lse;                                   // [heads, tokens], natural logarithm
  const uint16_t* d_o;                          // backward: gradient of o, contiguous
  uint16_t *dq, *dk, *dv;
  float* delta;                                 // [heads, tokens]: rowwise sums of d_o * o
  float scale;
  int tiles;                                    // work tiles per head in the grid (an upper bound)
  int parts;                                    // dK/dV: blocks (one cluster) that share the queries of a tile
  int* status;
  int* host_status;                             // a copy of the status word in pinned host memory, or null
  unsigned long long timeout_ns;
};

// Shared-memory matrix descriptors of a tile (128-byte swizzle, 8-row groups 1024 bytes apart): a constant
// high word and a low word of address and leading stride. K-major, and MN-major with the 64-column halves
// 16384 bytes apart.
constexpr uint32_t kDescHigh = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k_major(uint32_t addr) { return ((addr >> 4) & 0x3fffu) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_mn_major(uint32_t addr) {
  return ((addr >> 4) & 0x3fffu) | ((kHalfBytes >> 4) << 16);
}
// Instruction descriptors: BF16 x BF16 -> FP32, M = N = 128, B K-major or MN-major.
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((kTile >> 3) << 17) | ((kTile >> 4) << 24);
constexpr uint32_t kIdescMn = kIdesc | (1u << 16);

// The products below are issued by one elected lane of a converged warp.
// D[128, 128] = A B^T over the 128 columns of two K-major tiles.
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a_tile, uint32_t b_tile) {
  const uint32_t a = desc_k_major(a_tile), b = desc_k_major(b_tile);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t step = (k >> 2) * (kHalfBytes >> 4) + (k & 3) * 2;
    mma_bf16<kDescHigh, kIdesc>(d, a + step, b + step, k != 0);
  }
}
// D[128, 128] (+)= A B over 16 * kSteps rows of B from row 16 * step on: A from TMEM (BF16, 8 columns a
// step), B a tile read MN-major.
template <int kSteps>
__device__ __forceinline__ void mma_weighted_part(uint32_t d, uint32_t a_tmem, uint32_t b_tile, int step, bool accumulate) {
  const uint32_t b = desc_mn_major(b_tile) + step * 128;
#pragma unroll
  for (int k = 0; k < kSteps; ++k)
    mma_bf16_ta<kDescHigh, kIdescMn>(d, a_tmem + k * 8, b + k * 128, k != 0 ? 1u : accumulate);
}
// Over all 128 rows, with the halves of A 64 columns apart.
__device__ __forceinline__ void mma_weighted(uint32_t d, uint32_t a_tmem, uint32_t b_tile, bool accumulate) {
  mma_weighted_part<4>(d, a_tmem, b_tile, 0, accumulate);
  mma_weighted_part<4>(d, a_tmem + 64, b_tile, 4, true);
}

// Work tile `t` of `rows` rows: tiles are numbered sequence by sequence, the rows behind the last
// sequence last. Executed by whole warps. Every block walks over the offsets, 32 a step, and every sequence has
// blocks of its own however short it is: packs of a thousand sequences cost more for that than for their
// products (16 tokens each, 8 heads, forward: 100 sequences 40 us, 1000 575 us, 5000 7.7 ms).
struct WorkTile {
  int first, len;  // rows of the sequence
  int row0;        // first row of the tile within the sequence
  bool padding;    // belongs to no sequence
};
__device__ __forceinline__ bool find_tile(const AttentionParams& P, int rows, int t, WorkTile& w) {
  const int lane = threadIdx.x & 31;
  const int n = P.cu == nullptr ? 1 : P.samples;
  int before = 0;
  for (int base = 0; base <= n; base += 32) {
    const int s = base + lane;
    int a = 0, b = 0;
    if (s <= n) {
      a = seq_bound(P.cu, s, n, P.tokens);
      b = s < n ? seq_bound(P.cu, s + 1, n, P.tokens) : P.tokens;
    }
    const int count = b > a ? (b - a + rows - 1) / rows : 0;
    int upto = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, before + upto > t);
    if (hit != 0) {
      const int src = __ffs(hit) - 1;
      w.first = __shfl_sync(0xffffffffu, a, src);
      w.len = __shfl_sync(0xffffffffu, b, src) - w.first;
      w.row0 = (t - before - __shfl_sync(0xffffffffu, upto - count, src)) * rows;
      w.padding = base + src == n;
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int head, int row) {
  tma_load_3d(dst, map, bar, 0, head, row);
  tma_load_3d(dst + kHalfBytes, map, bar, 64, head, row);
}

// Whole warp: load a tile of which only `valid` < 128 rows belong to the sequence, through a barrier of
// the loading warp's own, clear the others and hand the tile over with a plain arrival on `full`.
__device__ __forceinline__ bool load_tail(uint32_t dst, const CUtensorMap* map, uint32_t full, uint32_t own, uint32_t& phase,
                                          int head, int row, int valid, int lane, WaitCtx& w) {
  bool ok = true;
  if (lane == 0) {
    mbar_arrive_expect_tx(own, kTileBytes);
    load_tile(dst, map, own, head, row);
    ok = wait_small(own, phase, w, 62);
  }
  phase ^= 1;
  ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
  if (!ok) {
    w.dead = true;
    return false;
  }
  // whole 128-byte rows: the swizzle only permutes 16-byte pieces inside a row
  for (uint32_t at = valid * 128 + lane * 16; at < kHalfBytes; at += 512) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + at), "r"(0u) : "memory");
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst + kHalfBytes + at), "r"(0u) : "memory");
  }
  fence_proxy_async_shared();
  __syncwarp();
  if (lane == 0) mbar_arrive_local(full);
  return true;
}

// A place in a ring of buffers and the parity of its barriers there.
struct Slot {
  int at;
  uint32_t phase;
  template <int kSlots>
  __device__ __forceinline__ void next() {
    if (++at == kSlots) {
      at = 0;
      phase ^= 1;
    }
  }
};

__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// 64 columns of a row of an FP32 accumulator, times `factor`, as BF16 to global memory: thread = row. They
// are staged in the thread's own 144-byte slot (a skew of 16 bytes keeps 16-byte stores free of bank
// conflicts) and leave with one bulk copy. Whole warps.
constexpr uint32_t kSlotPitch = 144;
__device__ __forceinline__ void store_piece(uint32_t tmem, uint32_t slot, uint16_t* dst, float factor, bool valid) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t r[32];
    tmem_ld_32x32(tmem + c * 32, r);
    tmem_ld_wait();
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      uint32_t p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        p[e] = pack_pair(__uint_as_float(r[v * 8 + 2 * e]) * factor, __uint_as_float(r[v * 8 + 2 * e + 1]) * factor);
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot + c * 64 + v * 16), "r"(p[0]), "r"(p[1]),
                   "r"(p[2]), "r"(p[3])
                   : "memory");
    }
  }
  fence_proxy_async_shared();
  if (valid) {
    bulk_store(dst, slot, 128);
    bulk_commit();
  }
  __syncwarp();
}
__device__ __forceinline__ void store_row(uint32_t tmem, uint32_t slot, uint16_t* dst, float factor, bool valid) {
  store_piece(tmem, slot, dst, factor, valid);
  bulk_wait_read_all();
  store_piece(tmem + 64, slot, dst + 64, factor, valid);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void shared_pairs(uint32_t at, F2 (&v)[2]) {
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(v[0].v), "=l"(v[1].v) : "r"(at) : "memory");
}
__device__ __forceinline__ F2 f2_of_bits(uint32_t lo, uint32_t hi) { return f2(__uint_as_float(lo), __uint_as_float(hi)); }
// 2^x of both halves.
__device__ __forceinline__ F2 exp2_pair(F2 x) {
  float lo, hi;
  split(x, lo, hi);
  return f2(exp2_approx(lo), exp2_approx(hi));
}

// Every thread of the block: zero rows [row, end) of one head.
__device__ __forceinline__ void zero_rows(uint16_t* base, int heads, int head, int row, int end) {
  for (int i = threadIdx.x; i < (end - row) * 16; i += blockDim.x)
    *reinterpret_cast<uint4*>(base + (static_cast<long long>(row + (i >> 4)) * heads + head) * kDim + (i & 15) * 8) =
        make_uint4(0, 0, 0, 0);
}

// An error that this block met, its own or an earlier kernel's: to where the host sees it without asking the
// device. The code goes last.
__device__ __forceinline__ void tell_host(const AttentionParams& P) {
  if (P.host_status == nullptr) return;
  volatile int* to = P.host_status;
  to[1] = ld_relaxed_sys_s32(P.status + 1);
  to[2] = ld_relaxed_sys_s32(P.status + 2);
  __threadfence_system();
  to[0] = ld_relaxed_sys_s32(P.status);
}

// Teardown shared by the kernels: copies that were issued but never consumed after an abort may still be
// landing in this block's shared memory.
__device__ __forceinline__ void settle(WaitCtx& w, const AttentionParams& P) {
  uint32_t aborted;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(aborted) : "r"(w.abort_flag) : "memory");
  if (aborted != 0 || w.dead) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) nanosleep(1000);
    if (w.dead && (threadIdx.x & 31) == 0) tell_host(P);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
}

// First thing in a kernel: what takes a trip to global memory and is needed a little later. The answer is the
// same for the lanes of a warp, which go on to wait together.
__device__ __forceinline__ bool begin(const AttentionParams& P, const CUtensorMap* a, const CUtensorMap* b,
                                      const CUtensorMap* c, const CUtensorMap* d) {
  if (threadIdx.x == 0) {
    tma_prefetch_desc(a);
    tma_prefetch_desc(b);
    tma_prefetch_desc(c);
    if (d != nullptr) tma_prefetch_desc(d);
  }
  return __any_sync(0xffffffffu, ld_relaxed_sys_s32(P.status) != 0);  // an error of an earlier kernel is sticky
}

// =============================================================================================
// Forward. A block owns 256 query rows of one head as two tiles; each has a warpgroup for its softmax
// (thread = row, the row's 128 scores in registers), S in 128 TMEM columns, which its probabilities then
// overlay as BF16, and its output in 128 more. While one tile is in the softmax the tensor cores work on
// the other: S_a(j+1) follows P_a(j) V directly, then the same for tile b.
//
// The running maximum is only moved when it grows by more than 8 (in powers of two): until then
// probabilities are at most 2^8 too large, which the final division by the equally scaled sum undoes, and
// the output accumulator need not be touched.
//
// What bounds it: an iteration (256 queries x 128 keys) takes 3150 cycles where its products take 2048. A
// tile's softmax is 1690 of them (1024 for 16384 exponentials at 16 per cycle), then come the rest of P V and
// the next S (640) and the latencies of two hand-overs; both tiles run that chain half a period apart. An
// issuing warp for each tile (263 against 247 us for the packed prompts below), key tiles of 64 with two score
// buffers per query tile (271 us), one hand-over instead of two (the same) and a polynomial in place of a
// quarter of the exponentials (258 us) do not shorten it. 16383 tokens x 8 heads: 0.94 ms in a few calls, 1.07 ms
// (1.03 PFLOP/s) at the 1.6 GHz that the power limit leaves in longer runs; its 512 blocks are 3.46 rounds of 148
// SMs and take the time of 4. 8192 tokens of packed causal prompts, 32 heads on 8: 225 to 248 us, 0.81 to 0.90
// PFLOP/s. Nothing splits the keys of a block, so few heads on a long sequence leave SMs idle (4097 causal tokens:
// 65 us for 1 head as for 4; 8191: 118 us).
// =============================================================================================
constexpr int kFwdThreads = 384;
constexpr uint32_t kFwdStageBytes = 2 * kTileBytes;  // V(j) and K(j + 1): the operands of one iteration
constexpr uint32_t kFwdSmem = 3 * kTileBytes + 2 * kFwdStageBytes + 256 + 1024;

__global__ void __launch_bounds__(kFwdThreads, 1)
    attention_forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                             const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttentionParams P) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_smem = base, k0_smem = base + 2 * kTileBytes, ring = base + 3 * kTileBytes;
  const uint32_t bars = ring + 2 * kFwdStageBytes;
  const uint32_t q_full = bars, k0_full = bars + 16, full = k0_full + 8, empty = full + 16, s_full = empty + 16,
                 p_full = s_full + 16 /* [tile][part] */, pv_done = p_full + 32, own_bar = pv_done + 16,
                 tmem_slot = own_bar + 8, abort_word = tmem_slot + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const bool sticky = begin(P, &map_q, &map_k, &map_v, nullptr);
  const int head = blockIdx.x % P.heads, kv_head = head / P.group;
  WorkTile wt;
  // the last tiles first: under a causal mask they are the longest
  if (!find_tile(P, 2 * kTile, P.tiles - 1 - static_cast<int>(blockIdx.x / P.heads), wt)) return;
  if (wt.padding) {
    const int row = wt.first + wt.row0, end = min(row + 2 * kTile, wt.first + wt.len);
    zero_rows(P.o, P.heads, head, row, end);
    if (P.lse != nullptr)
      for (int r = row + threadIdx.x; r < end; r += blockDim.x)
        P.lse[static_cast<long long>(head) * P.tokens + r] = -INFINITY;
    return;
  }
  // key tiles of the two query tiles; a second tile that starts behind the sequence has none
  const int all_tiles = (wt.len + kTile - 1) / kTile;
  const int n0 = P.causal ? min(all_tiles, wt.row0 / kTile + 1) : all_tiles;
  const int n1 = wt.row0 + kTile >= wt.len ? 0 : P.causal ? min(all_tiles, wt.row0 / kTile + 2) : all_tiles;
  const int n_max = max(n0, n1);

  WaitCtx w{P.status, P.timeout_ns, abort_word, sticky};
  if (warp == 8 && lane == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 16 * i, 4);
      mbar_init(p_full + 16 * i + 8, 4);
      mbar_init(pv_done + 8 * i, 1);
    }
    mbar_init(k0_full, 1);
    mbar_init(own_bar, 1);
    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort_word), "r"(0u) : "memory");
    fence_mbar_init();
    if (!w.dead) {  // Q and K(0) are on their way while the block sets up
      mbar_arrive_expect_tx(q_full, kTileBytes);
      load_tile(q_smem, &map_q, q_full, head, wt.first + wt.row0);
      mbar_arrive_expect_tx(k0_full, kTileBytes);
      load_tile(k0_smem, &map_k, k0_full, kv_head, wt.first);
      if (n1 > 0) {
        mbar_arrive_expect_tx(q_full + 8, kTileBytes);
        load_tile(q_smem + kTileBytes, &map_q, q_full + 8, head, wt.first + wt.row0 + kTile);
      }
    }
  }
  __syncwarp();
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot) : "memory");

  if (warp >= 8) {
    regs_down<80>();
    if (warp == 8) {
      // ---------------------------------------------------------------- loads: V(j) with K(j + 1)
      uint32_t own_phase = 0;
      for (int j = 0; j < n_max && !w.dead; ++j) {
        if (j >= 2 && !warp_wait(empty + 8 * (j & 1), ((j >> 1) & 1) ^ 1, w, 60)) break;
        const int row = j * kTile, valid = wt.len - row;
        const uint32_t dst = ring + (j & 1) * kFwdStageBytes, bar = full + 8 * (j & 1);
        if (valid < kTile) {  // the last tile: no K follows
          if (!load_tail(dst, &map_v, bar, own_bar, own_phase, kv_head, wt.first + row, valid, lane, w)) break;
        } else if (lane == 0) {
          const bool more = j + 1 < n_max;
          mbar_arrive_expect_tx(bar, more ? 2 * kTileBytes : kTileBytes);
          load_tile(dst, &map_v, bar, kv_head, wt.first + row);
          if (more) load_tile(dst + kTileBytes, &map_k, bar, kv_head, wt.first + row + kTile);
        }
        __syncwarp();
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------------- products
      auto scores = [&](int i, uint32_t k_tile) {
        if (elect_one()) {
          mma_rows(tmem + i * 128, q_smem + i * kTileBytes, k_tile);
          tc_commit(s_full + 8 * i);
        }
        __syncwarp();
      };
      // P(j) V(j) of tile i, the first 96 keys and the last 32, as its warpgroup hands them over
      auto weighted = [&](int i, uint32_t v, int j, bool last) {
        const uint32_t o = tmem + 256 + i * 128, p = tmem + i * 128;
        if (!warp_wait(p_full + 16 * i, j & 1, w, 66)) return;
        tc_fence_after();
        if (elect_one()) mma_weighted_part<6>(o, p, v, 0, j > 0);
        __syncwarp();
        if (!warp_wait(p_full + 16 * i + 8, j & 1, w, 66)) return;
        tc_fence_after();
        if (elect_one()) {
          mma_weighted_part<2>(o, p + 48, v, 6, true);
          if (last) tc_commit(pv_done + 8 * i);
        }
        __syncwarp();
      };
      if (warp_wait(k0_full, 0, w, 63) && warp_wait(q_full, 0, w, 64)) {
        tc_fence_after();
        scores(0, k0_smem);
        if (n1 > 0 && warp_wait(q_full + 8, 0, w, 64)) {
          tc_fence_after();
          scores(1, k0_smem);
        }
      }
#pragma unroll 1
      for (int j = 0; j < n_max && !w.dead; ++j) {
        if (!warp_wait(full + 8 * (j & 1), (j >> 1) & 1, w, 65)) break;
        const uint32_t v = ring + (j & 1) * kFwdStageBytes;
#pragma unroll 1
        for (int i = 0; i < 2; ++i) {
          const int n = i ? n1 : n0;
          if (j < n && !w.dead) weighted(i, v, j, j + 1 == n);
          if (j + 1 < n && !w.dead) scores(i, v + kTileBytes);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax: warpgroup = query tile
    regs_up<208>();
    const int i = warp >> 2, row_in_tile = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + i * 128 + lanes, o_tmem = tmem + 256 + i * 128 + lanes;
    const int row = wt.row0 + i * kTile + row_in_tile;  // within the sequence
    const float c = P.scale_log2;
    const int tiles = i ? n1 : n0;
    const bool releases = warp == (n1 > 0 ? 4 : 0);
    float m = 0.f, l = 0.f;
    bool alive = true;
    for (int j = 0; j < tiles; ++j) {
      if (!warp_wait(s_full + 8 * i, j & 1, w, 70)) {
        w.dead = true;
        alive = false;
        break;
      }
      tc_fence_after();
      // The scores of the tile that has the most keys are the last product of an iteration to be issued:
      // their arrival frees the operands of the iteration before.
      if (releases && lane == 0 && j > 0) mbar_arrive_local(empty + 8 * ((j - 1) & 1));
      uint32_t s[4][32];
#pragma unroll
      for (int q = 0; q < 4; ++q) tmem_ld_32x32(s_tmem + q * 32, s[q]);
      tmem_ld_wait();
      if (j == tiles - 1) {  // keys behind the sequence, and behind the row under a causal mask
        const int limit = min(wt.len, P.causal ? row + 1 : wt.len) - j * kTile;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (q * 32 + e >= limit) s[q][e] = 0xff800000u;  // -inf
      }
      auto row_max = [&]() {
        float mx[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) mx[q] = fmaxf(__uint_as_float(s[q][0]), __uint_as_float(s[q][1]));
#pragma unroll
        for (int e = 2; e < 32; e += 2)
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = max3(mx[q], __uint_as_float(s[q][e]), __uint_as_float(s[q][e + 1]));
        return max3(mx[0], mx[1], fmaxf(mx[2], mx[3]));
      };
      const F2 c2 = f2(c);
      uint32_t p[2][16];
      // 32 probabilities, all from the special function unit: a quarter of them by a polynomial of degree four
      // instead, to relieve it, made the kernel 5 % slower (8192 tokens of packed prompts: 258 against 246 us).
      // One rounding to BF16, the type the products take; their sum stays FP32 and unrounded.
      auto probabilities = [&](int q, F2 shift, F2& total, uint32_t (&out)[16]) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const F2 x = fma2(f2_of_bits(s[q][2 * e], s[q][2 * e + 1]), c2, shift);
          const F2 y = exp2_pair(x);
          total = total + y;
          out[e] = bf16_of_f2(y);
        }
      };
      auto hand_over = [&](int part) {
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(p_full + 16 * i + 8 * part);
      };
      const float top = row_max();
      if (j == 0) {
        m = top == -INFINITY ? 0.f : top;
      } else if (__any_sync(0xffffffffu, row < wt.len && (top - m) * c > 8.f)) {  // rows behind the sequence have no say
        // S(j) was issued behind the product that last wrote the output: its arrival covers both
        const float up = fmaxf(m, top), f = exp2_approx((m - up) * c);
        m = up;
        l *= f;
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          uint32_t o[32];
          tmem_ld_32x32(o_tmem + q * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st_32x32(o_tmem + q * 32, o);
        }
      }
      const F2 shift = f2(-m * c);
      F2 sum2[2] = {f2(0.f), f2(0.f)};
      probabilities(0, shift, sum2[0], p[0]);
      probabilities(1, shift, sum2[1], p[1]);
      tmem_st_32x16(s_tmem, p[0]);
      tmem_st_32x16(s_tmem + 16, p[1]);
      probabilities(2, shift, sum2[0], p[0]);
      tmem_st_32x16(s_tmem + 32, p[0]);
      hand_over(0);
      probabilities(3, shift, sum2[1], p[1]);
      tmem_st_32x16(s_tmem + 48, p[1]);
      hand_over(1);
      l += sum(sum2[0] + sum2[1]);
    }
    if (alive && tiles > 0 && warp_wait(pv_done + 8 * i, 0, w, 72)) {
      tc_fence_after();
      const bool valid = row < wt.len;
      const long long at = wt.first + row;
      const float invalid = fabsf(m * c) <= kMaxTop ? 0.f : __int_as_float(0x7fffffff);  // see the range of the scores
      // The query tile has been read by its last product: its shared memory stages the output.
      store_row(o_tmem, q_smem + i * kTileBytes + row_in_tile * kSlotPitch, P.o + (at * P.heads + head) * kDim,
                (l > 0.f || l != l ? 1.f / l : 0.f) + invalid, valid);
      if (valid && P.lse != nullptr)
        P.lse[static_cast<long long>(head) * P.tokens + at] = (m * c + log2f(l)) * kLn2 + invalid;
      bulk_wait_read_all();  // shared memory may go; the writes complete with the kernel
    }
  }
  settle(w, P);
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// =============================================================================================
// Backward. With P = exp(scale S - lse) and delta = rowsum(dO * O):
//   dV = P^T dO,   dS = P * (dO V^T - delta),   dQ = scale dS K,   dK = scale dS^T Q.
// Two kernels recompute S and dP: the first owns query rows and walks over the keys for dQ, and finds delta of
// its rows on the way; the second owns key/value rows and walks over the queries (of all query heads that
// share them, so a shared head's gradient is one sum in one accumulator). That is 7 tile products where a
// single kernel would need 5, but dQ is then not summed by atomics across blocks: every run gives the same
// bits, and no FP32 copy of dQ is kept.
//
// In both kernels two warpgroups share a 128 x 128 tile of scores, thread = row, 64 columns each. They
// write their halves of P or dS as BF16 over their own halves of the scores, 64 columns apart. (Four
// warpgroups of 32 columns each were 3 % slower.)
//
// 16383 tokens x 8 heads: 1.15 ms for dQ (2070 cycles per tile, 1536 of products) and 1.56 ms for dK and dV
// (2790, 2048 of products) in a few calls, together 1.42 PFLOP/s of tensor work; 1.26 and 1.70 ms, 1.30 PFLOP/s,
// under the power limit of longer runs. The dK/dV kernel spills 8 bytes a thread at its 168 registers.
// =============================================================================================
constexpr int kBwdThreads = 384;

// ---- dK, dV: S^T and dP^T tiles, rows = keys, columns = queries. TMEM: S^T (then P^T) 0, dP^T (then
// dS^T) 128, dV 256, dK 384. The tensor cores run dV(i) and S(i+1) while the warps compute dS(i), and
// dK(i) and dP(i+1) while they compute P(i+1).
//
// Q(i + 1) is needed first and Q(i) is let go last, so Q has three slots and dO two: with two pairs the
// products waited 2100 cycles per tile for Q. The row values (lse, delta) have a warp and a ring of their own.
// All of an SM's shared memory is in use: row values and barriers lie in the 3 KiB in front of the tiles.
//
// With few key/value tiles and heads, two or four blocks of a cluster share the (head, query tile) list of a
// tile in equal consecutive pieces. Their sums meet in shared memory: of the four pieces of 128 x 64 values
// (dV, dK, two halves each) every block finishes 4 / parts, adding what the others send it in the order of
// their ranks, so the result does not depend on who is first.
constexpr int kQSlots = 3, kDoSlots = 2, kRowSlots = 2;
constexpr uint32_t kPiecePitch = 272;  // bytes of 64 FP32 values and a skew against bank conflicts
constexpr uint32_t kDkvSmem = (2 + kQSlots + kDoSlots) * kTileBytes + 3 * 1024;
static_assert(kDkvSmem <= 227 * 1024 && kRowSlots * 1024 + 256 <= 3 * 1024, "shared memory");

__global__ void __launch_bounds__(kBwdThreads, 1)
    attention_dkv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                         const __grid_constant__ AttentionParams P) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t front = smem_u32(smem_raw), base = front + 3 * 1024;
  const uint32_t k_smem = base, v_smem = base + kTileBytes, q_ring = base + 2 * kTileBytes,
                 do_ring = q_ring + kQSlots * kTileBytes;
  const uint32_t rows_smem = front;  // per slot: -lse * log2(e) [128], delta [128]
  const uint32_t bars = rows_smem + kRowSlots * 1024;
  const uint32_t kv_full = bars, q_full = bars + 8, q_empty = q_full + 8 * kQSlots, do_full = q_empty + 8 * kQSlots,
                 do_empty = do_full + 8 * kDoSlots, rows_full = do_empty + 8 * kDoSlots,
                 rows_empty = rows_full + 8 * kRowSlots, s_full = rows_empty + 8 * kRowSlots, dp_full = s_full + 8,
                 p_full = dp_full + 8, ds_full = p_full + 16, acc_done = ds_full + 8, own_bar = acc_done + 8,
                 tmem_slot = own_bar + 8, abort_word = tmem_slot + 8;
  static_assert(8 + 16 * (kQSlots + kDoSlots + kRowSlots) + 56 + 16 <= 256, "barrier area");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const bool sticky = begin(P, &map_q, &map_k, &map_v, &map_do);
  const int part = P.parts > 1 ? static_cast<int>(cluster_ctarank()) : 0, unit = blockIdx.x / P.parts;
  const int kv_head = unit % P.kv_heads;
  WorkTile wt;
  // the first tiles first: under a causal mask they have the most queries behind them
  if (!find_tile(P, kTile, unit / P.kv_heads, wt)) return;  // the whole cluster
  if (wt.padding) {
    const int row = wt.first + wt.row0, end = min(row + kTile, wt.first + wt.len);
    zero_rows(P.dk, P.kv_heads, kv_head, row, end);
    zero_rows(P.dv, P.kv_heads, kv_head, row, end);
    return;
  }
  const int q_tiles = (wt.len + kTile - 1) / kTile;
  const int q_first = P.causal ? wt.row0 / kTile : 0;
  const int per_head = q_tiles - q_first, all = per_head * P.group;
  const int begin_at = static_cast<int>(static_cast<long long>(all) * part / P.parts);
  const int total = static_cast<int>(static_cast<long long>(all) * (part + 1) / P.parts) - begin_at;

  WaitCtx w{P.status, P.timeout_ns, abort_word, sticky};
  if ((front & 1023u) != 0) {  // the tiles would not be where their swizzle needs them
    if (threadIdx.x == 0) {
      if (atomicCAS(P.status, 0, kErrPipelineTimeout) == 0) P.status[1] = 78;
      tell_host(P);
    }
    return;
  }
  if (warp == 8 && lane == 0) {
    mbar_init(kv_full, 1);
    for (int i = 0; i < kQSlots; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(q_empty + 8 * i, 1);
    }
    for (int i = 0; i < kDoSlots; ++i) {
      mbar_init(do_full + 8 * i, 1);
      mbar_init(do_empty + 8 * i, 1);
    }
    for (int i = 0; i < kRowSlots; ++i) {
      mbar_init(rows_full + 8 * i, 1);
      mbar_init(rows_empty + 8 * i, 8);
    }
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_full, 8);
    mbar_init(p_full + 8, 8);
    mbar_init(ds_full, 8);
    mbar_init(acc_done, 1);
    mbar_init(own_bar, 1);
    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort_word), "r"(0u) : "memory");
    fence_mbar_init();
    if (!w.dead && total > 0) {  // on their way while the block sets up
      mbar_arrive_expect_tx(kv_full, 2 * kTileBytes);
      load_tile(k_smem, &map_k, kv_full, kv_head, wt.first + wt.row0);
      load_tile(v_smem, &map_v, kv_full, kv_head, wt.first + wt.row0);
    }
  }
  __syncwarp();
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot) : "memory");

  if (warp >= 8) {
    regs_down<80>();
    // ------------------------------------------------------------------ loads
    if (warp == 8) {
      uint32_t own_phase = 0;
      Slot qs{0, 0}, ds{0, 0};
      // rows behind the sequence are operands of the sums over queries here, so short tiles are cleared
      auto load = [&](const CUtensorMap* map, uint32_t dst, uint32_t full, int head, int row) {
        const int valid = wt.len - row;
        if (valid < kTile) return load_tail(dst, map, full, own_bar, own_phase, head, wt.first + row, valid, lane, w);
        if (lane == 0) {
          mbar_arrive_expect_tx(full, kTileBytes);
          load_tile(dst, map, full, head, wt.first + row);
        }
        __syncwarp();
        return true;
      };
      for (int i = 0; i < total && !w.dead; ++i) {
        const int head = kv_head * P.group + (begin_at + i) / per_head,
                  row = (q_first + (begin_at + i) % per_head) * kTile;
        if (i >= kQSlots && !warp_wait(q_empty + 8 * qs.at, qs.phase ^ 1, w, 80)) break;
        if (!load(&map_q, q_ring + qs.at * kTileBytes, q_full + 8 * qs.at, head, row)) break;
        if (i >= kDoSlots && !warp_wait(do_empty + 8 * ds.at, ds.phase ^ 1, w, 80)) break;
        if (!load(&map_do, do_ring + ds.at * kTileBytes, do_full + 8 * ds.at, head, row)) break;
        qs.next<kQSlots>();
        ds.next<kDoSlots>();
      }
    } else if (warp == 10) {
      // ------------------------------------------------------------------ row values of the queries
      Slot rs{0, 0};
      for (int i = 0; i < total; ++i) {
        const int head = kv_head * P.group + (begin_at + i) / per_head,
                  row = (q_first + (begin_at + i) % per_head) * kTile;
        const long long at = static_cast<long long>(head) * P.tokens + wt.first + row;
        float neg[4], delta[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int q = c * 32 + lane;
          neg[c] = -INFINITY;  // a probability of 0 behind the sequence
          delta[c] = 0.f;
          if (row + q < wt.len) {
            neg[c] = exponent_of_lse(__ldg(P.lse + at + q));
            delta[c] = __ldg(P.delta + at + q);
          }
        }
        if (i >= kRowSlots && !warp_wait(rows_empty + 8 * rs.at, rs.phase ^ 1, w, 79)) break;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t to = rows_smem + rs.at * 1024 + (c * 32 + lane) * 4;
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(to), "f"(neg[c]) : "memory");
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + 512), "f"(delta[c]) : "memory");
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_local(rows_full + 8 * rs.at);
        rs.next<kRowSlots>();
      }
    } else if (warp == 9) {
      // ------------------------------------------------------------------ products
      if (total > 0 && warp_wait(kv_full, 0, w, 81) && warp_wait(q_full, 0, w, 82) && warp_wait(do_full, 0, w, 82)) {
        tc_fence_after();
        if (elect_one()) {
          mma_rows(tmem, k_smem, q_ring);
          tc_commit(s_full);
          mma_rows(tmem + 128, v_smem, do_ring);
          tc_commit(dp_full);
        }
        __syncwarp();
        Slot qs{0, 0}, ds{0, 0};
#pragma unroll 1
        for (int i = 0; i < total; ++i) {
          const int q_at = qs.at, do_at = ds.at;
          qs.next<kQSlots>();
          ds.next<kDoSlots>();
          const bool more = i + 1 < total;
          const uint32_t do_tile = do_ring + do_at * kTileBytes;
          if (more && !warp_wait(q_full + 8 * qs.at, qs.phase, w, 84)) break;
          if (!warp_wait(p_full, i & 1, w, 83)) break;
          tc_fence_after();
          if (elect_one()) {
            mma_weighted_part<2>(tmem + 256, tmem, do_tile, 0, i > 0);
            mma_weighted_part<2>(tmem + 256, tmem + 64, do_tile, 4, true);
          }
          __syncwarp();
          if (!warp_wait(p_full + 8, i & 1, w, 83)) break;
          tc_fence_after();
          if (elect_one()) {
            mma_weighted_part<2>(tmem + 256, tmem + 16, do_tile, 2, true);
            mma_weighted_part<2>(tmem + 256, tmem + 80, do_tile, 6, true);
            if (i + kDoSlots < total) tc_commit(do_empty + 8 * do_at);
            if (more) {
              mma_rows(tmem, k_smem, q_ring + qs.at * kTileBytes);
              tc_commit(s_full);
            }
          }
          __syncwarp();
          if (!warp_wait(ds_full, i & 1, w, 85)) break;
          if (more && !warp_wait(do_full + 8 * ds.at, ds.phase, w, 84)) break;
          tc_fence_after();
          if (elect_one()) {
            mma_weighted(tmem + 384, tmem + 128, q_ring + q_at * kTileBytes, i > 0);
            if (i + kQSlots < total) tc_commit(q_empty + 8 * q_at);
            if (more) {
              mma_rows(tmem + 128, v_smem, do_ring + ds.at * kTileBytes);
              tc_commit(dp_full);
            }
          }
          __syncwarp();
        }
        if (!w.dead && elect_one()) tc_commit(acc_done);
        __syncwarp();
      }
    }
    if (P.parts > 1) {  // the block's part in the two meetings below
      __syncwarp();
      cluster_sync();
      cluster_sync();
    }
  } else {
    regs_up<208>();  // 2 * 128 * 208 + 128 * 80 of the 384 * 168 registers at launch
    // ------------------------------------------------------------------ P and dS
    const int g = warp >> 2, key = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + g * 64, dp_tmem = s_tmem + 128;
    const float c = P.scale_log2;
    Slot rs{0, 0};
    bool alive = true;
#pragma unroll 1
    for (int i = 0; i < total; ++i) {
      const uint32_t rows = rows_smem + rs.at * 1024 + g * 256;
      if (!warp_wait(rows_full + 8 * rs.at, rs.phase, w, 89) || !warp_wait(s_full, i & 1, w, 86)) {
        alive = false;
        break;
      }
      tc_fence_after();
      F2 p[32];
      const F2 c2 = f2(c);
      const bool diagonal = P.causal && (begin_at + i) % per_head == 0;
      // 32 columns as BF16 to TMEM; half of the queries at a time, so that their product may begin
      auto hand_over = [&](int h) {
        if (diagonal) {  // queries in front of the key do not see it
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int q = g * 64 + h * 32 + 2 * e;
            float lo, hi;
            split(p[h * 16 + e], lo, hi);
            p[h * 16 + e] = f2(q < key ? 0.f : lo, q + 1 < key ? 0.f : hi);
          }
        }
        uint32_t b[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) b[e] = bf16_of_f2(p[h * 16 + e]);
        tmem_st_32x16(s_tmem + h * 16, b);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(p_full + 8 * h);
      };
      {
        uint32_t s[2][32];
        tmem_ld_32x32(s_tmem, s[0]);
        tmem_ld_32x32(s_tmem + 32, s[1]);
        tmem_ld_wait();
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          F2 n[2];
          shared_pairs(rows + v * 16, n);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t* x = &s[v >> 3][(v & 7) * 4 + 2 * e];
            p[v * 2 + e] = exp2_pair(fma2(f2_of_bits(x[0], x[1]), c2, n[e]));
          }
          if (v == 7) hand_over(0);
        }
        hand_over(1);
      }
      if (!warp_wait(dp_full, i & 1, w, 87)) {
        alive = false;
        break;
      }
      tc_fence_after();
      const F2 minus = f2(-1.f);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t d[32], b[16];
        tmem_ld_32x32(dp_tmem + h * 32, d);
        tmem_ld_wait();
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          F2 n[2];
          shared_pairs(rows + 512 + h * 128 + v * 16, n);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            b[2 * v + e] = bf16_of_f2(p[h * 16 + v * 2 + e] *
                                      fma2(n[e], minus, f2_of_bits(d[v * 4 + 2 * e], d[v * 4 + 2 * e + 1])));
        }
        // columns [0, 32) of this warpgroup's half have been read when h = 1 is stored to [16, 32), and
        // h = 0 goes to [0, 16), which it has just read itself
        tmem_st_32x16(dp_tmem + h * 16, b);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive_local(ds_full);
        mbar_arrive_local(rows_empty + 8 * rs.at);
      }
      rs.next<kRowSlots>();
    }
    if (P.parts == 1 && alive && warp_wait(acc_done, 0, w, 88)) {
      tc_fence_after();
      const bool valid = wt.row0 + key < wt.len;
      const long long at = (static_cast<long long>(wt.first + wt.row0 + key) * P.kv_heads + kv_head) * kDim;
      // one warpgroup stores dV, the other dK; K and V have been read for the last time
      store_row(tmem + lanes + 256 + g * 128, (g ? k_smem : v_smem) + key * kSlotPitch, (g ? P.dk : P.dv) + at,
                g ? P.scale : 1.f, valid);
      bulk_wait_read_all();  // shared memory may go; the writes complete with the kernel
    }
    if (P.parts > 1) {
      // Each warpgroup takes every second piece. A block without queries has sums of zero; one that gave up
      // leaves its pieces unsent, and what is stored then is as invalid as the status word says.
      const int mine = 4 / P.parts;
      const bool worker = alive && !w.dead && (total == 0 || warp_wait(acc_done, 0, w, 88));
      tc_fence_before();
      __syncwarp();
      cluster_sync();  // all products of all blocks are done: the tiles' memory is free
      if (worker) {
        tc_fence_after();
        for (int piece = g; piece < 4; piece += 2) {
          const int owner = piece / mine;
          if (owner == part) continue;
          // slot of this block among the owner's senders, and of the piece among the owner's
          const int from = part - (part > owner ? 1 : 0);
          const uint32_t to = mapa(k_smem, owner) + ((from * mine + piece % mine) * 128 + key) * kPiecePitch;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t v[32];
            if (total > 0) {
              tmem_ld_32x32(tmem + lanes + 256 + piece * 64 + c * 32, v);
              tmem_ld_wait();
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = 0;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + c * 128 + e * 16), "r"(v[4 * e]),
                           "r"(v[4 * e + 1]), "r"(v[4 * e + 2]), "r"(v[4 * e + 3])
                           : "memory");
          }
        }
      }
      __syncwarp();
      cluster_sync();
      if (worker) {
        const bool valid = wt.row0 + key < wt.len;
        const long long at = (static_cast<long long>(wt.first + wt.row0 + key) * P.kv_heads + kv_head) * kDim;
        for (int piece = g; piece < 4; piece += 2) {
          if (piece / mine != part) continue;
          const uint32_t slot = q_ring + 2 * kTileBytes + (g * 128 + key) * kSlotPitch;  // behind what was received
          bulk_wait_read_all();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t own[32];
            F2 v[16];
            if (total > 0) {
              tmem_ld_32x32(tmem + lanes + 256 + piece * 64 + c * 32, own);
              tmem_ld_wait();
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) own[e] = 0;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = f2(0.f);
            for (int rank = 0; rank < P.parts; ++rank) {
              if (rank == part) {
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = v[e] + f2_of_bits(own[2 * e], own[2 * e + 1]);
              } else {
                const int from = rank - (rank > part ? 1 : 0);
                const uint32_t at_smem = k_smem + ((from * mine + piece % mine) * 128 + key) * kPiecePitch + c * 128;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                  F2 x[2];
                  shared_pairs(at_smem + e * 16, x);
                  v[2 * e] = v[2 * e] + x[0];
                  v[2 * e + 1] = v[2 * e + 1] + x[1];
                }
              }
            }
            const F2 factor = f2(piece >= 2 ? P.scale : 1.f);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(slot + c * 64 + e * 16),
                           "r"(bf16_of_f2(v[4 * e] * factor)), "r"(bf16_of_f2(v[4 * e + 1] * factor)),
                           "r"(bf16_of_f2(v[4 * e + 2] * factor)), "r"(bf16_of_f2(v[4 * e + 3] * factor))
                           : "memory");
          }
          fence_proxy_async_shared();
          if (valid) {
            bulk_store((piece >= 2 ? P.dk : P.dv) + at + (piece & 1) * 64, slot, 128);
            bulk_commit();
          }
          __syncwarp();
        }
        bulk_wait_read_all();
      }
    }
  }
  settle(w, P);
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- dQ: S and dP tiles, rows = queries, columns = keys. TMEM: S (then dS) in two buffers 0 and 128, dP
// 256, dQ 384. The tensor cores run S(j+1) and dP(j+1) while the warps compute dS(j).
// K has three slots and V two for the same reason as above.
constexpr int kKSlots = 3, kVSlots = 2;
constexpr uint32_t kDqSmem = (2 + kKSlots + kVSlots) * kTileBytes + 1024 + 256 + 1024;

__global__ void __launch_bounds__(kBwdThreads, 1)
    attention_dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                        const __grid_constant__ AttentionParams P) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_smem = base, do_smem = base + kTileBytes, k_ring = base + 2 * kTileBytes,
                 v_ring = k_ring + kKSlots * kTileBytes;
  const uint32_t sums_smem = v_ring + kVSlots * kTileBytes;  // halves of the rows' delta
  const uint32_t bars = sums_smem + 1024;
  const uint32_t q_full = bars, k_full = bars + 8, k_empty = k_full + 8 * kKSlots, v_full = k_empty + 8 * kKSlots,
                 v_empty = v_full + 8 * kVSlots, s_full = v_empty + 8 * kVSlots, dp_full = s_full + 16,
                 dp_read = dp_full + 8, ds_full = dp_read + 8, acc_done = ds_full + 8, own_bar = acc_done + 8,
                 sums_full = own_bar + 8, tmem_slot = sums_full + 8, abort_word = tmem_slot + 8;
  static_assert(8 + 16 * (kKSlots + kVSlots) + 64 + 16 <= 256, "barrier area");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const bool sticky = begin(P, &map_q, &map_k, &map_v, &map_do);
  const int head = blockIdx.x % P.heads, kv_head = head / P.group;
  WorkTile wt;
  if (!find_tile(P, kTile, P.tiles - 1 - static_cast<int>(blockIdx.x / P.heads), wt)) return;
  if (wt.padding) {
    const int row = wt.first + wt.row0;
    zero_rows(P.dq, P.heads, head, row, min(row + kTile, wt.first + wt.len));
    return;
  }
  const int all_tiles = (wt.len + kTile - 1) / kTile;
  const int n = P.causal ? min(all_tiles, wt.row0 / kTile + 1) : all_tiles;

  WaitCtx w{P.status, P.timeout_ns, abort_word, sticky};
  if (warp == 8 && lane == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < kKSlots; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(k_empty + 8 * i, 1);
    }
    for (int i = 0; i < kVSlots; ++i) {
      mbar_init(v_full + 8 * i, 1);
      mbar_init(v_empty + 8 * i, 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_full + 8, 1);
    mbar_init(dp_full, 1);
    mbar_init(dp_read, 8);
    mbar_init(ds_full, 8);
    mbar_init(acc_done, 1);
    mbar_init(own_bar, 1);
    mbar_init(sums_full, 8);
    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort_word), "r"(0u) : "memory");
    fence_mbar_init();
    if (!w.dead) {  // on their way while the block sets up
      mbar_arrive_expect_tx(q_full, 2 * kTileBytes);
      load_tile(q_smem, &map_q, q_full, head, wt.first + wt.row0);
      load_tile(do_smem, &map_do, q_full, head, wt.first + wt.row0);
    }
  }
  __syncwarp();
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot) : "memory");

  if (warp >= 8) {
    regs_down<80>();
    // ------------------------------------------------------------------ loads
    if (warp == 8) {
      uint32_t own_phase = 0;
      Slot ks{0, 0}, vs{0, 0};
      for (int j = 0; j < n && !w.dead; ++j) {
        const int row = j * kTile, valid = wt.len - row;
        const uint32_t k_dst = k_ring + ks.at * kTileBytes, k_bar = k_full + 8 * ks.at;
        if (j >= kKSlots && !warp_wait(k_empty + 8 * ks.at, ks.phase ^ 1, w, 90)) break;
        if (valid < kTile) {  // K is also summed over, V only makes scores that are masked
          if (!load_tail(k_dst, &map_k, k_bar, own_bar, own_phase, kv_head, wt.first + row, valid, lane, w)) break;
        } else if (lane == 0) {
          mbar_arrive_expect_tx(k_bar, kTileBytes);
          load_tile(k_dst, &map_k, k_bar, kv_head, wt.first + row);
        }
        __syncwarp();
        if (j >= kVSlots && !warp_wait(v_empty + 8 * vs.at, vs.phase ^ 1, w, 90)) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(v_full + 8 * vs.at, kTileBytes);
          load_tile(v_ring + vs.at * kTileBytes, &map_v, v_full + 8 * vs.at, kv_head, wt.first + row);
        }
        __syncwarp();
        ks.next<kKSlots>();
        vs.next<kVSlots>();
      }
    } else if (warp == 9) {
      // ------------------------------------------------------------------ products
      if (warp_wait(q_full, 0, w, 91) && warp_wait(k_full, 0, w, 92) && warp_wait(v_full, 0, w, 92)) {
        tc_fence_after();
        if (elect_one()) {
          mma_rows(tmem, q_smem, k_ring);
          tc_commit(s_full);
          mma_rows(tmem + 256, do_smem, v_ring);
          tc_commit(dp_full);
          if (kVSlots < n) tc_commit(v_empty);
        }
        __syncwarp();
        Slot ks{0, 0}, vs{0, 0};
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
          const int k_at = ks.at;
          ks.next<kKSlots>();
          vs.next<kVSlots>();
          if (j + 1 < n) {
            if (!warp_wait(k_full + 8 * ks.at, ks.phase, w, 93)) break;
            tc_fence_after();
            if (elect_one()) {
              mma_rows(tmem + ((j + 1) & 1) * 128, q_smem, k_ring + ks.at * kTileBytes);
              tc_commit(s_full + 8 * ((j + 1) & 1));
            }
            __syncwarp();
            if (!warp_wait(v_full + 8 * vs.at, vs.phase, w, 93)) break;
            if (!warp_wait(dp_read, j & 1, w, 94)) break;
            tc_fence_after();
            if (elect_one()) {
              mma_rows(tmem + 256, do_smem, v_ring + vs.at * kTileBytes);
              tc_commit(dp_full);
              if (j + 1 + kVSlots < n) tc_commit(v_empty + 8 * vs.at);
            }
            __syncwarp();
          }
          if (!warp_wait(ds_full, j & 1, w, 95)) break;
          tc_fence_after();
          if (elect_one()) {
            mma_weighted(tmem + 384, tmem + (j & 1) * 128, k_ring + k_at * kTileBytes, j > 0);
            if (j + kKSlots < n) tc_commit(k_empty + 8 * k_at);
          }
          __syncwarp();
        }
        if (!w.dead && elect_one()) tc_commit(acc_done);
        __syncwarp();
      }
    }
  } else {
    regs_up<208>();  // 2 * 128 * 208 + 128 * 80 of the 384 * 168 registers at launch
    // ------------------------------------------------------------------ dS
    const int g = warp >> 2, row_in_tile = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const int row = wt.row0 + row_in_tile;
    const bool valid = row < wt.len;
    const long long at = wt.first + (valid ? row : 0);
    const F2 c2 = f2(P.scale_log2);
    const F2 neg = f2(exponent_of_lse(__ldg(P.lse + static_cast<long long>(head) * P.tokens + at)));
    // delta of the rows, kept for the dK/dV kernel. Where all keys lie in one tile it is the sum of P * dP, which
    // needs no rounded output: a row that sees a single key then gets dS = 0, not the rounding error of its
    // output. (That error is 2^-9 |o| |dO|; beside the spread of dP it vanishes with the root of the number of
    // keys.)
    const bool one_tile = n == 1;
    auto keep_delta = [&](float all) {
      if (g == 0 && valid) P.delta[static_cast<long long>(head) * P.tokens + at] = all;
      return f2(-all);
    };
    auto shared_float = [&](int i) {
      float v;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(sums_smem + i * 4) : "memory");
      return v;
    };
    F2 delta = f2(0.f);
    if (!one_tile) {  // o * dO, half a warp per row
      uint4 o[8], d[8];
      const int half = lane >> 4, sub = lane & 15;
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        const int r = wt.row0 + warp * 16 + 2 * v + half;
        const long long from = (static_cast<long long>(wt.first + min(r, wt.len - 1)) * P.heads + head) * kDim + sub * 8;
        o[v] = __ldg(reinterpret_cast<const uint4*>(P.o + from));
        d[v] = __ldg(reinterpret_cast<const uint4*>(P.d_o + from));
      }
#pragma unroll
      for (int v = 0; v < 8; ++v) {
        F2 partial = f2_of_bf16(o[v].x) * f2_of_bf16(d[v].x);
        partial = fma2(f2_of_bf16(o[v].y), f2_of_bf16(d[v].y), partial);
        partial = fma2(f2_of_bf16(o[v].z), f2_of_bf16(d[v].z), partial);
        partial = fma2(f2_of_bf16(o[v].w), f2_of_bf16(d[v].w), partial);
        float all = sum(partial);
#pragma unroll
        for (int m = 8; m; m >>= 1) all += __shfl_xor_sync(0xffffffffu, all, m);
        if (sub == 0)
          asm volatile("st.shared.f32 [%0], %1;" ::"r"(sums_smem + (warp * 16 + 2 * v + half) * 4), "f"(all) : "memory");
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");  // all eight warps: none has waited for anything yet
      delta = keep_delta(shared_float(row_in_tile));
    }
    bool alive = true;
    for (int j = 0; j < n; ++j) {
      const uint32_t s_tmem = tmem + lanes + (j & 1) * 128 + g * 64, dp_tmem = tmem + lanes + 256 + g * 64;
      if (!warp_wait(s_full + 8 * (j & 1), (j >> 1) & 1, w, 96)) {
        alive = false;
        break;
      }
      tc_fence_after();
      F2 p[32];
      {
        uint32_t s[2][32];
        tmem_ld_32x32(s_tmem, s[0]);
        tmem_ld_32x32(s_tmem + 32, s[1]);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e)
          p[e] = exp2_pair(fma2(f2_of_bits(s[e >> 4][2 * (e & 15)], s[e >> 4][2 * (e & 15) + 1]), c2, neg));
      }
      if (!warp_wait(dp_full, j & 1, w, 97)) {
        alive = false;
        break;
      }
      tc_fence_after();
      uint32_t d[2][32];
      tmem_ld_32x32(dp_tmem, d[0]);
      tmem_ld_32x32(dp_tmem + 32, d[1]);
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(dp_read);
      if (j == n - 1) {  // keys behind the sequence, and behind the row under a causal mask
        const int limit = min(wt.len, P.causal ? row + 1 : wt.len) - j * kTile - g * 64;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          float lo, hi;
          split(p[e], lo, hi);
          p[e] = f2(2 * e >= limit ? 0.f : lo, 2 * e + 1 >= limit ? 0.f : hi);
          if (2 * e >= limit) d[e >> 4][2 * (e & 15)] = 0;  // may be anything, NaN included
          if (2 * e + 1 >= limit) d[e >> 4][2 * (e & 15) + 1] = 0;
        }
      }
      if (one_tile) {
        F2 partial = f2(0.f);
#pragma unroll
        for (int e = 0; e < 32; ++e)
          partial = fma2(p[e], f2_of_bits(d[e >> 4][2 * (e & 15)], d[e >> 4][2 * (e & 15) + 1]), partial);
        const float own = sum(partial);  // the other 64 columns are the other warpgroup's
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(sums_smem + (g * 128 + row_in_tile) * 4), "f"(own) : "memory");
        // a barrier with a limit: a warp that gave up on a wait above never comes here
        __syncwarp();
        if (lane == 0) mbar_arrive_local(sums_full);
        if (!warp_wait(sums_full, 0, w, 99)) {
          alive = false;
          break;
        }
        delta = keep_delta(shared_float(row_in_tile) + shared_float(128 + row_in_tile));
      }
#pragma unroll
      for (int e = 0; e < 32; ++e)
        p[e] = p[e] * (f2_of_bits(d[e >> 4][2 * (e & 15)], d[e >> 4][2 * (e & 15) + 1]) + delta);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t b[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) b[e] = bf16_of_f2(p[h * 16 + e]);
        tmem_st_32x16(s_tmem + h * 16, b);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(ds_full);
    }
    if (alive && warp_wait(acc_done, 0, w, 98)) {
      tc_fence_after();
      // each warpgroup stores half of the columns; Q and dO have been read for the last time
      store_piece(tmem + lanes + 384 + g * 64, (g ? do_smem : q_smem) + row_in_tile * kSlotPitch,
                  P.dq + (static_cast<long long>(wt.first + row) * P.heads + head) * kDim + g * 64, P.scale, valid);
      bulk_wait_read_all();  // shared memory may go; the writes complete with the kernel
    }
  }
  settle(w, P);
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

// 3-D map [tokens, heads, 128] with boxes of 128 tokens x one head x 64 columns, 128-byte swizzle.
static int encode_heads(CUtensorMap* map, const void* base, int tokens, int heads, int64_t token_stride,
                        int64_t head_stride) {
  return encode_tmap_3d(map, base, tokens, heads, kDim, token_stride, head_stride, kTile, 64);
}

static int check_attention(const FgaAttention* a, AttentionParams& P) {
  FGA_REQUIRE(a != nullptr, "attention: null arguments");
  FGA_REQUIRE(a->tokens >= 1 && a->tokens <= 0x7ffffe00, "attention: tokens must be in [1, 2^31 - 512]");
  FGA_REQUIRE(a->kv_heads >= 1 && a->heads >= a->kv_heads && a->heads % a->kv_heads == 0 && a->heads <= 65536,
              "attention: query heads must be a multiple of key/value heads");
  FGA_REQUIRE(a->samples >= 1 && a->samples <= 65535, "attention: 1 to 65535 sequences");
  FGA_REQUIRE(a->cu_seqlens != nullptr || a->samples == 1, "attention: several sequences need cu_seqlens");
  // far from where scale * log2(e) would overflow, or flush to 0 and make 0 * -inf of a masked score
  FGA_REQUIRE(a->scale >= 1e-30f && a->scale <= 1e30f, "attention: scale must be from 1e-30 to 1e30");
  FGA_REQUIRE(a->q && a->k && a->v && a->o && a->status, "attention: null pointer");
  for (const void* p : {a->q, a->k, a->v, const_cast<const void*>(a->o)})
    FGA_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "attention: pointers must be 16-byte aligned");
  for (int t = 0; t < 3; ++t)
    FGA_REQUIRE(a->token_stride[t] > 0 && a->token_stride[t] % 8 == 0 && a->head_stride[t] > 0 && a->head_stride[t] % 8 == 0,
                "attention: strides must be positive multiples of 8 elements");
  P.cu = a->cu_seqlens;
  P.samples = a->samples;
  P.tokens = static_cast<int>(a->tokens);
  P.heads = a->heads;
  P.kv_heads = a->kv_heads;
  P.group = a->heads / a->kv_heads;
  P.causal = a->causal;
  P.scale_log2 = a->scale * kLog2e;
  P.scale = a->scale;
  P.o = static_cast<uint16_t*>(a->o);
  P.lse = a->lse;
  P.status = a->status;
  P.host_status = a->host_status;
  P.timeout_ns = a->timeout_ns;
  return kSuccess;
}

static uint64_t g_smem_forward, g_smem_dkv, g_smem_dq;

// Upper bound of the work tiles of `rows` rows: each sequence, and the rows behind the last, ends in one
// that may be short.
static long long tile_bound(const AttentionParams& P, int rows) {
  return P.cu == nullptr ? (P.tokens + static_cast<long long>(rows) - 1) / rows
                         : P.tokens / rows + static_cast<long long>(P.samples) + 1;
}

// Blocks of a cluster that share a key/value tile: four while there are fewer tiles than SMs, two while
// there are fewer than four per SM, to fill the SMs and to even out tiles of unequal length, but only where
// the mean tile has 16 query tiles or more to walk over (the lengths are not known here, their mean is): a
// meeting costs about 8 us. 8191 causal tokens in five sequences, 32 heads on 4: 551 us alone, 466 us in
// twos; 512 tokens, 8 heads, four query tiles each: 13.7 us alone, 19.4 us in fours.
static int sharing_blocks(const AttentionParams& P, long long units) {
  const long long sms = sm_count();
  const long long walk = P.group * ((P.tokens / P.samples + kTile - 1ll) / kTile) / (P.causal ? 2 : 1);
  if (walk < 16 || units >= 4 * sms) return 1;
  return units < sms ? 4 : 2;
}

}  // namespace fga

using namespace fga;

extern "C" {

int fga_attention_forward(const FgaAttention* args, void* stream) {
  AttentionParams P = {};
  int rc = check_attention(args, P);
  if (rc != kSuccess) return rc;
  CUtensorMap q, k, v;
  if ((rc = encode_heads(&q, args->q, P.tokens, P.heads, args->token_stride[0], args->head_stride[0])) != kSuccess) return rc;
  if ((rc = encode_heads(&k, args->k, P.tokens, P.kv_heads, args->token_stride[1], args->head_stride[1])) != kSuccess) return rc;
  if ((rc = encode_heads(&v, args->v, P.tokens, P.kv_heads, args->token_stride[2], args->head_stride[2])) != kSuccess) return rc;
  const long long tiles = tile_bound(P, 2 * kTile), blocks = tiles * P.heads;
  FGA_REQUIRE(blocks <= 0x7fffffff, "attention: too many heads and sequences for one launch");
  P.tiles = static_cast<int>(tiles);
  if ((rc = allow_smem(attention_forward_kernel, kFwdSmem, g_smem_forward)) != kSuccess) return rc;
  attention_forward_kernel<<<static_cast<unsigned>(blocks), kFwdThreads, kFwdSmem, static_cast<cudaStream_t>(stream)>>>(q, k, v, P);
  FGA_LAUNCHED();
  return kSuccess;
}

int fga_attention_backward(const FgaAttention* args, void* stream) {
  AttentionParams P = {};
  int rc = check_attention(args, P);
  if (rc != kSuccess) return rc;
  FGA_REQUIRE(args->lse && args->d_o && args->dq && args->dk && args->dv && args->delta, "attention: null pointer");
  for (const void* p : {args->d_o, const_cast<const void*>(args->dq), const_cast<const void*>(args->dk),
                        const_cast<const void*>(args->dv)})
    FGA_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "attention: pointers must be 16-byte aligned");
  P.d_o = static_cast<const uint16_t*>(args->d_o);
  P.dq = static_cast<uint16_t*>(args->dq);
  P.dk = static_cast<uint16_t*>(args->dk);
  P.dv = static_cast<uint16_t*>(args->dv);
  P.delta = args->delta;
  CUtensorMap q, k, v, d;
  if ((rc = encode_heads(&q, args->q, P.tokens, P.heads, args->token_stride[0], args->head_stride[0])) != kSuccess) return rc;
  if ((rc = encode_heads(&k, args->k, P.tokens, P.kv_heads, args->token_stride[1], args->head_stride[1])) != kSuccess) return rc;
  if ((rc = encode_heads(&v, args->v, P.tokens, P.kv_heads, args->token_stride[2], args->head_stride[2])) != kSuccess) return rc;
  if ((rc = encode_heads(&d, args->d_o, P.tokens, P.heads, static_cast<int64_t>(P.heads) * kDim, kDim)) != kSuccess) return rc;
  const long long tiles = tile_bound(P, kTile), blocks = tiles * P.heads;
  FGA_REQUIRE(blocks <= 0x7fffffff, "attention: too many heads and sequences for one launch");
  P.tiles = static_cast<int>(tiles);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = allow_smem(attention_dq_kernel, kDqSmem, g_smem_dq)) != kSuccess) return rc;
  attention_dq_kernel<<<static_cast<unsigned>(blocks), kBwdThreads, kDqSmem, st>>>(q, k, v, d, P);
  FGA_LAUNCHED();
  if ((rc = allow_smem(attention_dkv_kernel, kDkvSmem, g_smem_dkv)) != kSuccess) return rc;
  const long long units = tiles * P.kv_heads;
  P.parts = sharing_blocks(P, units);
  FGA_REQUIRE(units * P.parts <= 0x7fffffff, "attention: too many heads and sequences for one launch");
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(units * P.parts));
  config.blockDim = dim3(kBwdThreads);
  config.dynamicSmemBytes = kDkvSmem;
  config.stream = st;
  cudaLaunchAttribute cluster;
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = static_cast<unsigned>(P.parts);
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  FGA_CUDA(cudaLaunchKernelEx(&config, attention_dkv_kernel, q, k, v, d, P));
  FGA_LAUNCHED();
  return kSuccess;
}

}  // extern "C"
