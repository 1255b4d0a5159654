// Causal attention of a prompt's tokens over a paged key-value cache, with or without a sliding window and first tokens that stay
// visible: tcgen05 MMAs on tiles that TMA brings from the pages.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "attention.cuh"
#include "paged.cuh"

namespace b2 {
namespace {

constexpr int kTile = 128;  // rows of a query tile (TMEM lanes), slots of a key tile

struct PromptArgs {
  PagedArgs c;
  const void* q;
  std::int64_t q_row, q_head, tokens;
  void* out;
  std::int64_t o_row, o_head;
  float* lse;
  const std::int32_t* cu;
  int q_heads, group, max_q;
  float scale_log2;  // scale * log2(e)
  int window, sinks;
};

template <typename T, int D, int kTiles>
struct Shape {
  static constexpr int kThreads = 128 + 128 * kTiles;  // a warpgroup of TMA warp, MMA warp and two that sleep; a softmax thread per query row
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 8;
  static constexpr int kSmem = kTileBytes * (kTiles + kStages) + 1024;  // Q, the ring of K and V tiles, alignment slack
  static constexpr int kColumns = kTiles * (kTile + D) <= 256 ? 256 : 512;
};

// A tile in shared memory: D / 64 parts of 128 rows of 128 bytes (64 elements), 128-byte swizzle. As an operand whose rows run along
// K of the product (Q, K) every part is a K-major tile; as V (rows are K) a part is 64 columns of an MN-major operand, its 8-row
// groups 1024 bytes apart and the parts 128 * 128 bytes.
constexpr int kPartBytes = kTile * 128;
__device__ __forceinline__ std::uint64_t value_desc(std::uint32_t smem_addr) {
  return (umma_desc_sw128(smem_addr) & ~(static_cast<std::uint64_t>(0x3FFF) << 16)) | static_cast<std::uint64_t>(kPartBytes >> 4) << 16;
}
// The halves of a word whose exponent is all ones (infinities and NaN).
template <typename T>
__device__ __forceinline__ std::uint32_t nonfinite_halves(std::uint32_t w) {
  constexpr std::uint32_t e = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
  return ((w & e) == e ? 0xFFFFu : 0u) | ((w >> 16 & e) == e ? 0xFFFF0000u : 0u);
}

// Which of the 32 slots from `at` (relative to the tile) a row sees: slot <= hi, and slot > lo or slot < first.
__device__ __forceinline__ std::uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
__device__ __forceinline__ std::uint32_t seen_mask(int at, int hi, int lo, int first) {
  return below(hi + 1 - at) & (~below(lo + 1 - at) | below(first - at));
}

// One CTA per (kTiles * 128 rows, key head, sequence). A row is a (token, query head of the group) pair, the group's heads of a token
// side by side: they share their keys, and a tile has few tokens, so little of the causal edge is computed for nothing. The key
// tiles go from the sinks' to the newest:
//   TMA warp      K and V tiles of 128 slots into one ring, a box per page
//   MMA warp      for each query tile: O += P V, then the next S = Q K^T into the columns that held S and P. (tcgen05.mma of different
//                 shape need not keep their order, so the scores wait until P V has landed; the other tile's MMAs fill the time.)
//   softmax warps one thread per row: P = exp2(c s - m), 16 bits wide, over the first half of S's columns in tensor memory. m is the
//                 first tile's maximum, and stays: P, its sum and O are floating point, so what matters is only that nothing overflows. That is
//                 seen from the tile's sum; the pass is then done again under a new maximum, with O scaled. So no maximum is taken in
//                 an ordinary tile.
template <typename T, int D, int kTiles>
__global__ void __launch_bounds__(Shape<T, D, kTiles>::kThreads, 1)
prompt_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PromptArgs a) {
  using S = Shape<T, D, kTiles>;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  // fp16 ends at 2^16 and loses bits below 2^-14: P starts at up to 2^6 and may grow to 2^15. bf16 has fp32's range.
  constexpr float kShift = kHalf ? 6.0f : 0.0f, kLimit = kHalf ? 32768.0f : 1.0e12f;
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const int h = blockIdx.x, b = blockIdx.y, bq = static_cast<int>(gridDim.z - 1 - blockIdx.z);  // the longest rows first
  int first_token, n;
  paged_tokens(a.c, a.cu, b, a.tokens, first_token, n);
  if (n > a.max_q) {
    if (threadIdx.x == 0) atomicOr(a.c.status, kPagedBadTokens);
    n = a.max_q;
  }
  const int len = paged_len(a.c, b), rows = n * a.group, row0 = bq * (kTiles * kTile);
  if (row0 >= rows) return;  // uniform per CTA, before any barrier or allocation
  const int row_last = min(row0 + kTiles * kTile, rows) - 1;
  const int p_lo = len - n + row0 / a.group, p_hi = len - n + row_last / a.group;  // slots of the first and the last token
  const auto out_row = [&](int row) {
    return static_cast<T*>(a.out) + static_cast<std::int64_t>(first_token + row / a.group) * a.o_row + (h * a.group + row % a.group) * a.o_head;
  };
  const auto lse_at = [&](int row) { return static_cast<std::int64_t>(first_token + row / a.group) * a.q_heads + h * a.group + row % a.group; };
  if (p_hi < 0) {
    // Nothing to see for any row.
    for (int i = threadIdx.x; i < (row_last + 1 - row0) * (D / 8); i += S::kThreads) {
      const int row = row0 + i / (D / 8);
      *reinterpret_cast<uint4*>(out_row(row) + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
      if (i % (D / 8) == 0 && a.lse != nullptr) a.lse[lse_at(row)] = -INFINITY;
    }
    return;
  }
  // The key tiles: the sinks' first, then from `from` to the last token's.
  const int from = a.window > 0 && max(p_lo, 0) - a.window + 1 > 0 ? (max(p_lo, 0) - a.window + 1) / kTile : 0;
  const int sink_tiles = min((min(a.sinks, p_hi + 1) + kTile - 1) / kTile, from);
  const int count = sink_tiles + p_hi / kTile + 1 - from;
  const auto tile_slot = [&](int j) { return (j < sink_tiles ? j : j - sink_tiles + from) * kTile; };
  // Whether every row from slot lo to slot hi sees all of the tile.
  const auto all_seen = [&](int slot0, int lo, int hi) {
    return slot0 + kTile - 1 <= lo && (a.window == 0 || slot0 + kTile <= a.sinks || slot0 > hi - a.window);
  };

  extern __shared__ std::uint8_t smem_raw[];
  __shared__ __align__(8) std::uint64_t s_q_full, s_full[S::kStages], s_empty[S::kStages], s_scores[kTiles], s_p[kTiles], s_pv[kTiles];
  __shared__ std::uint32_t s_tmem_base;
  __shared__ int s_abort, s_nonfinite;
  const std::uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const auto q_smem = [&](int i) { return base + i * S::kTileBytes; };
  const auto stage = [&](int s) { return base + (kTiles + s) * S::kTileBytes; };
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&s_q_full), 4 * kTiles);
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(smem_u32(&s_full[s]), 1);
      mbar_init(smem_u32(&s_empty[s]), 1);
    }
    for (int i = 0; i < kTiles; ++i) {
      mbar_init(smem_u32(&s_scores[i]), 1);
      mbar_init(smem_u32(&s_p[i]), 4);
      mbar_init(smem_u32(&s_pv[i]), 1);
    }
    s_abort = 0, s_nonfinite = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&s_tmem_base), S::kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const auto tmem_s = [&](int i) { return s_tmem_base + static_cast<std::uint32_t>(i * kTile); };
  const auto tmem_o = [&](int i) { return s_tmem_base + static_cast<std::uint32_t>(kTiles * kTile + i * D); };
  volatile int* abort_word = &s_abort;
  const auto warp_wait = [&](std::uint32_t bar, std::uint32_t parity) {
    const bool ok = wait_bar(bar, parity, abort_word);
    return !__any_sync(0xffffffffu, !ok);
  };

  // 168 registers a thread (65536 over 384, in eights) become 208 for the softmax and 88 for the others.
  if (warp < 4) {
   if constexpr (kTiles == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
   if (warp == 0) {
    // Item 2 j is K of tile j, item 2 j + 1 its V. A lane per (box of a page's rows, part).
    constexpr int kParts = D / 64;
    const int box_rows = min(1 << a.c.page_shift, kTile), boxes = kTile / box_rows * kParts;
    const int my_row = lane / kParts * box_rows, my_part = lane % kParts;
    const bool mine = lane < boxes;
    const auto find_page = [&](int j) {
      const int slot = tile_slot(j) + my_row;
      return j < count && mine && slot < len ? paged_page(a.c, b, slot) : -1;
    };
    int page = find_page(0);
    bool ok = true;
    for (int j = 0; ok && j < count; ++j) {
      const int next = find_page(j + 1);
      const int slot = tile_slot(j) + my_row, row = slot & ((1 << a.c.page_shift) - 1);
      const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
      for (int kv = 0; kv < 2; ++kv) {
        const int item = 2 * j + kv, s = item % S::kStages;
        const bool got = wait_bar_relaxed<100>(smem_u32(&s_empty[s]), (item / S::kStages & 1u) ^ 1u, abort_word);
        ok = !__any_sync(0xffffffffu, !got);
        if (!ok) break;
        const std::uint32_t dst = stage(s) + my_part * kPartBytes + my_row * 128, bar = smem_u32(&s_full[s]);
        if (mine && page < 0 && slot < len) {  // a page outside the pool reads as zeros
          for (int i = 0; i < box_rows * 8; ++i) st_shared(dst + i * 16, make_uint4(0, 0, 0, 0));
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_expect_tx(bar, static_cast<std::uint32_t>(__popc(there) * box_rows * 128));
        __syncwarp();
        if (page >= 0) tma_load_4d(dst, kv == 0 ? &map_k : &map_v, bar, my_part * 64, row, h, page);
      }
      page = next;
    }
    __syncwarp();
   } else if (warp == 1) {
    // The whole warp walks the loop (uniform control flow, every lane takes the waits); one elected lane issues.
    constexpr int kFormat = kHalf ? 0 : 1;
    constexpr std::uint32_t idesc_qk = umma_idesc(/*f32*/ 1, kFormat, kFormat, 0, 0, kTile, kTile);
    constexpr std::uint32_t idesc_pv = umma_idesc(/*f32*/ 1, kFormat, kFormat, 0, /*B MN-major*/ 1, kTile, D);
    const auto issue_scores = [&](int i, int s) {  // S = Q K^T; 16 channels are 32 bytes of a row
      const std::uint64_t dq = umma_desc_sw128(q_smem(i)), dk = umma_desc_sw128(stage(s));
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const std::uint32_t at = static_cast<std::uint32_t>(k / 4 * (kPartBytes >> 4) + k % 4 * 2);
        umma_f16(tmem_s(i), dq + at, dk + at, idesc_qk, k != 0 ? 1u : 0u);
      }
    };
    const auto issue_values = [&](int i, int s, bool more) {  // O (+)= P V; 16 slots are 8 columns of P and 16 rows of V
      const std::uint64_t dv = value_desc(stage(s));
#pragma unroll
      for (int k = 0; k < kTile / 16; ++k) umma_f16_ts(tmem_o(i), tmem_s(i) + 8u * k, dv + 128u * k, idesc_pv, more || k != 0 ? 1u : 0u);
    };
    const auto full = [&](int item) { return warp_wait(smem_u32(&s_full[item % S::kStages]), item / S::kStages & 1u); };
    bool ok = warp_wait(smem_u32(&s_q_full), 0u) && full(0);
    tc_fence_after();
    if (ok && elect_one()) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        issue_scores(i, 0);
        tc_commit(smem_u32(&s_scores[i]));
      }
      tc_commit(smem_u32(&s_empty[0]));
    }
    __syncwarp();
    for (int j = 0; ok && j < count; ++j) {
      const bool more = j + 1 < count;
      const int sv = (2 * j + 1) % S::kStages, sk = (2 * j + 2) % S::kStages;
      ok = full(2 * j + 1);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        ok = ok && warp_wait(smem_u32(&s_p[i]), j & 1u);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          issue_values(i, sv, j != 0);
          tc_commit(smem_u32(&s_pv[i]));
          if (i == kTiles - 1) tc_commit(smem_u32(&s_empty[sv]));
        }
        __syncwarp();
        if (!more) continue;
        if (i == 0) ok = full(2 * j + 2);
        ok = ok && warp_wait(smem_u32(&s_pv[i]), j & 1u);
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          issue_scores(i, sk);
          tc_commit(smem_u32(&s_scores[i]));
          if (i == kTiles - 1) tc_commit(smem_u32(&s_empty[sk]));
        }
        __syncwarp();
      }
    }
   }
  } else {
    if constexpr (kTiles == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int i = (warp - 4) / 4, quarter = warp & 3;  // a warp may touch TMEM lanes [32 (warp % 4), +32)
    const int r_local = quarter * 32 + lane, row = row0 + i * kTile + r_local;
    const std::uint32_t lane_off = static_cast<std::uint32_t>(quarter * 32) << 16;
    const bool live = row < rows;
    // Q: 16 bytes a thread, a row's chunks side by side; zeros past the last row.
    for (int at = static_cast<int>(threadIdx.x) - 128; at < kTiles * kTile * (D / 8); at += 128 * kTiles) {
      const int r = at / (D / 8), c = at % (D / 8), of = row0 + r;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (of < rows) {
        v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + static_cast<std::int64_t>(first_token + of / a.group) * a.q_row +
                                            (h * a.group + of % a.group) * a.q_head + c * 8);
      }
      st_shared(q_smem(r / kTile) + c / 8 * kPartBytes + r % kTile * 128 + ((c % 8 ^ (r & 7)) << 4), v);
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&s_q_full));

    // The slot of this thread's token; rows past the last take the last one's (they are not stored). Of the warp: first and last.
    const int p = len - n + min(row, row_last) / a.group;
    const int warp_lo = len - n + min(row - lane, row_last) / a.group, warp_hi = len - n + min(row - lane + 31, row_last) / a.group;
    const float c = a.scale_log2;
    float m = -INFINITY, l = 0.f;  // reference in binades, sum
    bool dead = false;
    const std::uint32_t s_cols = tmem_s(i) + lane_off;
    const auto rescale_o = [&](float factor) {
#pragma unroll 1
      for (int cc = 0; cc < D / 32; ++cc) {
        std::uint32_t r[32];
        tmem_ld_32x32(tmem_o(i) + lane_off + cc * 32, r);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * factor);
        tmem_st_32x32(tmem_o(i) + lane_off + cc * 32, r);
      }
      tmem_st_wait();
    };
    for (int j = 0; j < count; ++j) {
      const int slot0 = tile_slot(j);
      const bool masked = !all_seen(slot0, warp_lo, warp_hi);
      const int hi = p - slot0, lo = a.window > 0 ? hi - a.window : -1, first = a.sinks - slot0;
      if (!warp_wait(smem_u32(&s_scores[i]), j & 1u)) {
        dead = true;
        break;
      }
      tc_fence_after();
      // The largest score this row sees in the tile.
      const auto tile_max = [&]() {
        float top = -INFINITY;
#pragma unroll 1
        for (int cc = 0; cc < 4; ++cc) {
          std::uint32_t r[32];
          tmem_ld_32x32(s_cols + cc * 32, r);
          const std::uint32_t seen = masked ? seen_mask(cc * 32, hi, lo, first) : 0xffffffffu;
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) top = fmaxf(top, (seen >> e & 1u) != 0u ? __uint_as_float(r[e]) : -INFINITY);
        }
        return top * c;
      };
      if (__any_sync(0xffffffffu, m == -INFINITY)) {  // (the row's first tile with something to see)
        const float top = tile_max();
        if (m == -INFINITY && top > -INFINITY) m = top - kShift;
      }
      std::uint32_t pw[64];  // P of this row, stored once the pass stands: it takes the place of the scores
      float sum;
      const auto pass = [&](auto with_mask) {
        constexpr bool kMask = decltype(with_mask)::value;
        const std::uint64_t c2 = pack2(c, c), m2 = pack2(-m, -m);
        std::uint64_t sum_a = pack2(0.f, 0.f), sum_b = sum_a;
        std::uint32_t buf[2][32];
        tmem_ld_32x32(s_cols, buf[0]);
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          tmem_ld_wait();
          if (cc < 3) tmem_ld_32x32(s_cols + (cc + 1) * 32, buf[(cc + 1) & 1]);
          const std::uint32_t(&r)[32] = buf[cc & 1];
          const std::uint32_t seen = kMask ? seen_mask(cc * 32, hi, lo, first) : 0xffffffffu;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            float x[4];
            unpack2(fma2(pack2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), c2, m2), x[0], x[1]);
            unpack2(fma2(pack2(__uint_as_float(r[e + 2]), __uint_as_float(r[e + 3])), c2, m2), x[2], x[3]);
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              x[f] = ex2(x[f]);
              if (kMask && (seen >> (e + f) & 1u) == 0u) x[f] = 0.f;
            }
            sum_a = add2(sum_a, pack2(x[0], x[1]));
            sum_b = add2(sum_b, pack2(x[2], x[3]));
            pw[cc * 16 + e / 2] = pack16<T>(x[0], x[1]);
            pw[cc * 16 + e / 2 + 1] = pack16<T>(x[2], x[3]);
          }
        }
        float s0, s1, s2, s3;
        unpack2(sum_a, s0, s1);
        unpack2(sum_b, s2, s3);
        sum = (s0 + s1) + (s2 + s3);
      };
      for (bool again = false;; again = true) {
        if (masked) {
          pass(std::true_type{});
        } else {
          pass(std::false_type{});
        }
        // Over the limit, or NaN (a row that has become NaN stays so).
        const bool over = !(sum <= kLimit) && l == l;
        if (again || !__any_sync(0xffffffffu, over)) break;
        const float top = tile_max();
        float alpha = 1.0f;
        if (over && top - kShift > m) {
          alpha = ex2(m - (top - kShift));
          m = top - kShift, l *= alpha;
        }
        if (j > 0) {  // O is scaled once every P V so far has landed
          if (!warp_wait(smem_u32(&s_pv[i]), (j - 1) & 1u)) {
            dead = true;
            break;
          }
          tc_fence_after();
          rescale_o(alpha);
        }
      }
      if (dead) break;
      l += sum;
      {
        const std::uint32_t(&lower)[32] = *reinterpret_cast<const std::uint32_t(*)[32]>(&pw[0]);
        const std::uint32_t(&upper)[32] = *reinterpret_cast<const std::uint32_t(*)[32]>(&pw[32]);
        tmem_st_32x32(s_cols, lower);
        tmem_st_32x32(s_cols + 32, upper);
      }
      if (i == 0 && !all_seen(slot0, p_lo, p_hi)) {
        // Some row of the CTA does not see all of this tile, and its zeros in P would make NaN of an infinity or a NaN in V: slots behind
        // the last become zeros here, and so do such values of slots that other rows see, which get them back at the end.
        const int item = 2 * j + 1, s = item % S::kStages;
        if (!warp_wait(smem_u32(&s_full[s]), item / S::kStages & 1u)) {
          dead = true;
          break;
        }
        bool found = false;
        for (int at = lane; at < 32 * (D / 8); at += 32) {  // this warp's 32 slots, 16 bytes a lane
          const int slot = quarter * 32 + at / 8 % 32;
          const std::uint32_t addr = stage(s) + at / 256 * kPartBytes + slot * 128 + at % 8 * 16;
          if (slot0 + slot >= len) {
            st_shared(addr, make_uint4(0, 0, 0, 0));
            continue;
          }
          uint4 v = ld_shared(addr);
          const std::uint32_t x = nonfinite_halves<T>(v.x), y = nonfinite_halves<T>(v.y), z = nonfinite_halves<T>(v.z), w = nonfinite_halves<T>(v.w);
          if ((x | y | z | w) != 0u) {
            found = true;
            v.x &= ~x, v.y &= ~y, v.z &= ~z, v.w &= ~w;
            st_shared(addr, v);
          }
        }
        if (found) s_nonfinite = 1;
        fence_proxy_async_smem();
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s_p[i]));
    }
    if (!dead && warp_wait(smem_u32(&s_pv[i]), (count - 1) & 1u)) {
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.0f / l;
      T* const out = live ? out_row(row) : nullptr;
      const bool repair = *const_cast<volatile int*>(&s_nonfinite) != 0;
#pragma unroll 1
      for (int cc = 0; cc < D / 32; ++cc) {
        std::uint32_t r[32];
        tmem_ld_32x32(tmem_o(i) + lane_off + cc * 32, r);
        tmem_ld_wait();
        float o[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(r[e]) * inv;
        if (repair && live) {
          for (int j = 0; j < count; ++j) {
            const int slot0 = tile_slot(j);
            if (all_seen(slot0, p_lo, p_hi)) continue;
            for (int slot = slot0; slot <= min(slot0 + kTile - 1, p); ++slot) {
              if (a.window > 0 && slot >= a.sinks && slot <= p - a.window) continue;
              const int page = paged_page(a.c, b, slot);
              if (page < 0) continue;
              const T* v = static_cast<const T*>(a.c.v) + paged_row(a.c, page, h, slot) + cc * 32;
#pragma unroll
              for (int e = 0; e < 32; e += 8) {
                float x[8];
                load8<T>(*reinterpret_cast<const uint4*>(v + e), x);
#pragma unroll
                for (int f = 0; f < 8; ++f) o[e + f] += isfinite(x[f]) ? 0.f : x[f];
              }
            }
          }
        }
        if (live) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            *reinterpret_cast<uint4*>(out + cc * 32 + e) = make_uint4(pack16<T>(o[e], o[e + 1]), pack16<T>(o[e + 2], o[e + 3]),
                                                                      pack16<T>(o[e + 4], o[e + 5]), pack16<T>(o[e + 6], o[e + 7]));
          }
        }
      }
      if (live && a.lse != nullptr) a.lse[lse_at(row)] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (s_abort != 0) {
    if (threadIdx.x == 0) atomicOr(a.c.status, kPagedWait);
    const std::uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) {
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(s_tmem_base, S::kColumns);
  }
}

template <typename T, int D, int kTiles>
int launch(const char* op, const PromptArgs& a, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t st) {
  using S = Shape<T, D, kTiles>;
  const auto kernel = prompt_kernel<T, D, kTiles>;
  if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem); e != cudaSuccess) {
    cudaGetLastError();
    return fail_cuda(op, e);
  }
  const std::int64_t tiles = (static_cast<std::int64_t>(a.max_q) * a.group + kTiles * kTile - 1) / (kTiles * kTile);
  if (tiles > 65535) return fail_invalid(op, "too many tokens of one sequence in a call");
  return enqueue(op, kernel, dim3(static_cast<unsigned>(a.c.kv_heads), static_cast<unsigned>(a.c.batch), static_cast<unsigned>(tiles)), S::kThreads,
                 S::kSmem, st, 1, map_k, map_v, a);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_attention_paged(const b2_paged_cache* cache, const b2_view3* q, const b2_view3* out, float* lse, const int32_t* cu_seqlens,
                       int max_q, float scale, int window, int sinks, void* stream) {
  constexpr const char* op = "attention_paged";
  PromptArgs a{};
  if (q == nullptr || out == nullptr) return fail_invalid(op, "null q or out");
  if (const int rc = check_paged_cache(op, cache, &a.c)) return rc;
  if (q->heads <= 0 || q->heads > 65535 || q->heads % cache->kv_heads != 0) return fail_invalid(op, "q must have a multiple of kv_heads heads, at most 65535");
  if (q->tokens < 0 || q->tokens > INT_MAX || out->tokens != q->tokens || out->heads != q->heads) return fail_invalid(op, "q and out must have the same tokens and heads");
  if (!std::isfinite(scale) || !(scale > 0.0f)) return fail_invalid(op, "scale must be finite and positive");
  if (const int rc = check_window(op, a.c, &window, &sinks)) return rc;
  if (max_q < 0) return fail_invalid(op, "max_q must not be negative");
  if (q->tokens == 0 || cache->batch == 0 || max_q == 0) return q->tokens == 0 ? B2_OK : fail_invalid(op, "tokens without a sequence, or max_q 0");
  if (cu_seqlens == nullptr) return fail_invalid(op, "null cu_seqlens");
  if (!rows_ok(q->data, q->row_stride, q->head_stride) || !rows_ok(out->data, out->row_stride, out->head_stride)) {
    return fail_invalid(op, "q and out need a 16-byte aligned base and strides that are multiples of 8");
  }
  if (cache->num_pages == 0) return fail_invalid(op, "the pool has no pages");
  a.q = q->data, a.q_row = q->row_stride, a.q_head = q->head_stride, a.tokens = q->tokens;
  a.out = out->data, a.o_row = out->row_stride, a.o_head = out->head_stride, a.lse = lse, a.cu = cu_seqlens;
  a.q_heads = static_cast<int>(q->heads), a.group = a.q_heads / cache->kv_heads;
  a.max_q = static_cast<int>(std::min<std::int64_t>(max_q, q->tokens));
  if (q->tokens * a.group > INT_MAX / 2) return fail_invalid(op, "too many tokens for one call");
  a.scale_log2 = scale * 1.4426950408889634f, a.window = window, a.sinks = sinks;
  CUtensorMap map_k, map_v;
  const int box = std::min(cache->page_size, kTile);
  if (!make_tensor_map_pages(&map_k, cache, false, box, op) || !make_tensor_map_pages(&map_v, cache, true, box, op)) return B2_ERR_CUDA;
  if (const int rc = paged_status_word(op, &a.c)) return rc;
  const cudaStream_t st = as_stream(stream);
  const bool wide = cache->head_dim == 128;
  if (cache->dtype == B2_DTYPE_BF16) {
    return wide ? launch<__nv_bfloat16, 128, 2>(op, a, map_k, map_v, st) : launch<__nv_bfloat16, 64, 2>(op, a, map_k, map_v, st);
  }
  return wide ? launch<__half, 128, 2>(op, a, map_k, map_v, st) : launch<__half, 64, 2>(op, a, map_k, map_v, st);
}

}  // extern "C"
