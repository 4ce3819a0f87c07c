// Attention over packed sequences on tcgen05 tensor cores (sm_100a): softmax(scale Q K^T) V for each
// sequence and head, optionally causal, with shared key/value heads; forward and backward, BF16 operands,
// FP32 accumulation and statistics. Head dimension 128.
//
// Common to the kernels: one block per SM works alone (no cluster). Operand tiles are 128 rows x 128
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

struct AttentionParams {
  const int* cu;
  int samples, tokens, heads, kv_heads, group;  // group = heads / kv_heads
  int causal;
  float scale_log2;                             // scale * log2(e)
  uint16_t* o;                                  // forward: [tokens, heads, 128]
  float* lse;                                   // [heads, tokens], natural logarithm
  int tiles;                                    // work tiles per head in the grid (an upper bound)
  int* status;
  unsigned long long timeout_ns;
};

// Shared-memory matrix descriptors of a tile (128-byte swizzle, 8-row groups 1024 bytes apart).
constexpr uint64_t kDescHigh = static_cast<uint64_t>(64u | (1u << 14) | (2u << 29)) << 32;
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) { return kDescHigh | ((addr >> 4) & 0x3fffu) | (1u << 16); }
// MN-major: the 64-column halves are 16384 bytes apart.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr) {
  return kDescHigh | ((addr >> 4) & 0x3fffu) | ((kHalfBytes >> 4) << 16);
}
// Instruction descriptors: BF16 x BF16 -> FP32, M = N = 128, B K-major or MN-major.
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((kTile >> 3) << 17) | ((kTile >> 4) << 24);
constexpr uint32_t kIdescMn = kIdesc | (1u << 16);

// D[128, 128] = A B^T over the 128 columns of two K-major tiles.
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a_tile, uint32_t b_tile) {
  const uint64_t a = desc_k_major(a_tile), b = desc_k_major(b_tile);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t step = (k >> 2) * (kHalfBytes >> 4) + (k & 3) * 2;
    mma_bf16(d, a + step, b + step, kIdesc, k != 0);
  }
}
// D[128, 128] (+)= A B over the 128 rows of B: A from TMEM (BF16, 64 columns), B a tile read MN-major.
__device__ __forceinline__ void mma_weighted(uint32_t d, uint32_t a_tmem, uint32_t b_tile, bool accumulate) {
  const uint64_t b = desc_mn_major(b_tile);
#pragma unroll
  for (int k = 0; k < 8; ++k) mma_bf16_ta(d, a_tmem + k * 8, b + k * 128, kIdescMn, accumulate || k != 0);
}

// Work tile `t` of `rows` rows: tiles are numbered sequence by sequence, the rows behind the last
// sequence last. Executed by whole warps.
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
    ok = mbar_wait(own, phase, w, 62);
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

__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Rows of a 128 x 128 FP32 accumulator, times `factor`, as BF16 to global memory: thread = row. Each
// 64-column piece is staged in the thread's own 144-byte slot (a skew of 16 bytes keeps 16-byte stores free
// of bank conflicts) and leaves with one bulk copy.
constexpr uint32_t kSlotPitch = 144;
__device__ __forceinline__ void store_row(uint32_t tmem, uint32_t slot, uint16_t* dst, float factor, bool valid) {
#pragma unroll
  for (int piece = 0; piece < 2; ++piece) {
    if (piece) bulk_wait_read_all();
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint32_t r[32];
      tmem_ld_32x32(tmem + piece * 64 + c * 32, r);
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
      bulk_store(dst + piece * 64, slot, 128);
      bulk_commit();
    }
    __syncwarp();
  }
}

// Every thread of the block: zero rows [row, end) of one head.
__device__ __forceinline__ void zero_rows(uint16_t* base, int heads, int head, int row, int end) {
  for (int i = threadIdx.x; i < (end - row) * 16; i += blockDim.x)
    *reinterpret_cast<uint4*>(base + (static_cast<long long>(row + (i >> 4)) * heads + head) * kDim + (i & 15) * 8) =
        make_uint4(0, 0, 0, 0);
}

// Teardown shared by the kernels: copies that were issued but never consumed after an abort may still be
// landing in this block's shared memory.
__device__ __forceinline__ void settle(WaitCtx& w) {
  __syncwarp();
  if (should_abort(w)) {
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) nanosleep(1000);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
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
// =============================================================================================
constexpr int kFwdSlots = 5;
constexpr int kFwdThreads = 384;
constexpr uint32_t kFwdSmem = 2 * kTileBytes + kFwdSlots * kTileBytes + 256 + 1024;

__global__ void __launch_bounds__(kFwdThreads, 1)
    attention_forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                             const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttentionParams P) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_smem = base, ring = base + 2 * kTileBytes;
  const uint32_t bars = ring + kFwdSlots * kTileBytes;
  const uint32_t q_full = bars, kv_full = bars + 16, kv_empty = kv_full + 8 * kFwdSlots,
                 s_full = kv_empty + 8 * kFwdSlots, p_full = s_full + 16, pv_done = p_full + 16, own_bar = pv_done + 16,
                 tmem_slot = own_bar + 8, abort_word = tmem_slot + 8;
  static_assert(16 + 16 * kFwdSlots + 48 + 8 + 16 <= 256, "barrier area");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const int head = blockIdx.x % P.heads;
  WorkTile wt;
  // the last tiles first: under a causal mask they are the longest
  if (!find_tile(P, 2 * kTile, P.tiles - 1 - static_cast<int>(blockIdx.x / P.heads), wt)) return;
  if (wt.padding) {
    const int row = wt.first + wt.row0, end = min(row + 2 * kTile, wt.first + wt.len);
    zero_rows(P.o, P.heads, head, row, end);
    for (int r = row + threadIdx.x; r < end; r += blockDim.x)
      P.lse[static_cast<long long>(head) * P.tokens + r] = -INFINITY;
    return;
  }
  // key tiles of the two query tiles; a second tile that starts behind the sequence has none
  const int all_tiles = (wt.len + kTile - 1) / kTile;
  int n[2];
  n[0] = P.causal ? min(all_tiles, wt.row0 / kTile + 1) : all_tiles;
  n[1] = wt.row0 + kTile >= wt.len ? 0 : P.causal ? min(all_tiles, wt.row0 / kTile + 2) : all_tiles;
  const int n_max = max(n[0], n[1]);

  WaitCtx w{P.status, P.timeout_ns, abort_word, ld_relaxed_sys_s32(P.status) != 0};
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);
      mbar_init(pv_done + 8 * i, 1);
    }
    for (int i = 0; i < kFwdSlots; ++i) {
      mbar_init(kv_full + 8 * i, 1);
      mbar_init(kv_empty + 8 * i, 1);
    }
    mbar_init(own_bar, 1);
    asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort_word), "r"(0u) : "memory");
    fence_mbar_init();
  }
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
      // ---------------------------------------------------------------- loads: Q, then K0 V0 K1 V1 ...
      const int kv_head = head / P.group;
      if (lane == 0 && !w.dead)
        for (int i = 0; i < 2; ++i)
          if (n[i] > 0) {
            mbar_arrive_expect_tx(q_full + 8 * i, kTileBytes);
            load_tile(q_smem + i * kTileBytes, &map_q, q_full + 8 * i, head, wt.first + wt.row0 + i * kTile);
          }
      int slot = 0;
      uint32_t phase = 0, own_phase = 0;
      for (int j = 0; j < 2 * n_max && !w.dead; ++j) {
        bool ok = true;
        if (lane == 0) ok = mbar_wait(kv_empty + 8 * slot, phase ^ 1, w, 60);
        if (__shfl_sync(0xffffffffu, ok ? 1 : 0, 0) == 0) {
          w.dead = true;
          break;
        }
        const int row = (j >> 1) * kTile, valid = wt.len - row;
        const uint32_t dst = ring + slot * kTileBytes, full = kv_full + 8 * slot;
        if ((j & 1) && valid < kTile) {
          if (!load_tail(dst, &map_v, full, own_bar, own_phase, kv_head, wt.first + row, valid, lane, w)) break;
        } else if (lane == 0) {
          mbar_arrive_expect_tx(full, kTileBytes);
          load_tile(dst, (j & 1) ? &map_v : &map_k, full, kv_head, wt.first + row);
        }
        if (++slot == kFwdSlots) {
          slot = 0;
          phase ^= 1;
        }
      }
    } else if (warp == 9 && lane == 0) {
      // ---------------------------------------------------------------- products
      int k_slot = 0;                 // slot of K(j); V(j) is in the next one
      uint32_t k_phase = 0;
      auto advance = [](int& slot, uint32_t& phase) {
        if (++slot == kFwdSlots) {
          slot = 0;
          phase ^= 1;
        }
      };
      if (mbar_wait(kv_full, 0, w, 63)) {
        for (int i = 0; i < 2; ++i)
          if (n[i] > 0) {
            if (!mbar_wait(q_full + 8 * i, 0, w, 64)) break;
            tc_fence_after();
            mma_rows(tmem + i * 128, q_smem + i * kTileBytes, ring);
            tc_commit(s_full + 8 * i);
          }
        if (kFwdSlots < 2 * n_max) tc_commit(kv_empty);
      }
      for (int j = 0; j < n_max && !w.dead; ++j) {
        int v_slot = k_slot;
        uint32_t v_phase = k_phase;
        advance(v_slot, v_phase);
        int next = v_slot;
        uint32_t next_phase = v_phase;
        advance(next, next_phase);
        if (!mbar_wait(kv_full + 8 * v_slot, v_phase, w, 65)) break;
        bool have_next = false;
        for (int i = 0; i < 2; ++i) {
          if (j < n[i]) {
            if (!mbar_wait(p_full + 8 * i, j & 1, w, 66)) break;
            tc_fence_after();
            mma_weighted(tmem + 256 + i * 128, tmem + i * 128, ring + v_slot * kTileBytes, j > 0);
            tc_commit(pv_done + 8 * i);
          }
          if (j + 1 < n[i]) {
            if (!have_next) {
              if (!mbar_wait(kv_full + 8 * next, next_phase, w, 67)) break;
              tc_fence_after();
              have_next = true;
            }
            mma_rows(tmem + i * 128, q_smem + i * kTileBytes, ring + next * kTileBytes);
            tc_commit(s_full + 8 * i);
          }
        }
        if (w.dead) break;
        // A slot is only released to a load that will take it, so that no arrival is in flight at the end.
        if (2 * j + 1 + kFwdSlots < 2 * n_max) tc_commit(kv_empty + 8 * v_slot);
        if (2 * j + 2 + kFwdSlots < 2 * n_max) tc_commit(kv_empty + 8 * next);
        k_slot = next;
        k_phase = next_phase;
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
    const int tiles = n[i];
    float m = 0.f, l = 0.f;
    bool alive = true;
    for (int j = 0; j < tiles; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(s_full + 8 * i, j & 1, w, 70))) {
        w.dead = true;
        alive = false;
        break;
      }
      tc_fence_after();
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
      float mx[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        mx[q] = __uint_as_float(s[q][0]);
#pragma unroll
        for (int e = 1; e < 32; ++e) mx[q] = fmaxf(mx[q], __uint_as_float(s[q][e]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      if (j == 0) {
        m = top == -INFINITY ? 0.f : top;
      } else if (__any_sync(0xffffffffu, (top - m) * c > 8.f)) {
        if (!__all_sync(0xffffffffu, mbar_wait(pv_done + 8 * i, (j - 1) & 1, w, 71))) {
          w.dead = true;
          alive = false;
          break;
        }
        tc_fence_after();
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
      const float shift = -m * c;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float a = exp2_approx(fmaf(__uint_as_float(s[q][2 * e]), c, shift));
          const float b = exp2_approx(fmaf(__uint_as_float(s[q][2 * e + 1]), c, shift));
          sum[(2 * e) & 3] += a;
          sum[(2 * e + 1) & 3] += b;
          // One rounding of the probabilities to BF16, the type the products take; their sum stays FP32.
          p[e] = pack_pair(a, b);
        }
        tmem_st_32x16(s_tmem + q * 16, p);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_local(p_full + 8 * i);
    }
    if (alive && tiles > 0 && __all_sync(0xffffffffu, mbar_wait(pv_done + 8 * i, (tiles - 1) & 1, w, 72))) {
      tc_fence_after();
      const bool valid = row < wt.len;
      const long long at = wt.first + row;
      // The query tile has been read by its last product: its shared memory stages the output.
      store_row(o_tmem, q_smem + i * kTileBytes + row_in_tile * kSlotPitch, P.o + (at * P.heads + head) * kDim,
                l > 0.f || l != l ? 1.f / l : 0.f, valid);
      if (valid) P.lse[static_cast<long long>(head) * P.tokens + at] = (m * c + log2f(l)) * kLn2;
      bulk_wait_all();
    }
  }
  settle(w);
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
  FGA_REQUIRE(a->scale > 0.f && a->scale < INFINITY, "attention: scale must be positive and finite");
  FGA_REQUIRE(a->q && a->k && a->v && a->o && a->lse && a->status, "attention: null pointer");
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
  P.o = static_cast<uint16_t*>(a->o);
  P.lse = a->lse;
  P.status = a->status;
  P.timeout_ns = a->timeout_ns;
  return kSuccess;
}

// Upper bound of the work tiles of `rows` rows: each sequence, and the rows behind the last, ends in one
// that may be short.
static long long tile_bound(const AttentionParams& P, int rows) {
  return P.cu == nullptr ? (P.tokens + static_cast<long long>(rows) - 1) / rows
                         : P.tokens / rows + static_cast<long long>(P.samples) + 1;
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
  FGA_CUDA(cudaFuncSetAttribute(attention_forward_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFwdSmem));
  attention_forward_kernel<<<static_cast<unsigned>(blocks), kFwdThreads, kFwdSmem, static_cast<cudaStream_t>(stream)>>>(q, k, v, P);
  FGA_LAUNCHED();
  return kSuccess;
}

}  // extern "C"
