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
  int q_tma;         // a box of the map of q is whole tokens (the group divides 128)
  int tiles, splits, works;  // 256-row tiles of the longest sequence; parts of each one's keys; all of them, for all sequences and key heads
  // Of a part, by [part, token, query head]: maximum and sum; O before the division.
  float2* part_ml;
  float* part_o;
};

template <int D>
struct Shape {
  static constexpr int kThreads = 384;  // TMA, MMA, V and Q warp; two softmax warpgroups
  static constexpr int kQBytes = kTile * D * 2, kKBytes = kTile / 2 * D * 2, kVBytes = kTile * D;  // of one CTA of the pair
  static constexpr int kStages = D == 128 ? 4 : 8;
  static constexpr int kSmem = 2 * kQBytes + kStages * (kKBytes + kVBytes) + 1024;  // and what aligns it
};

// Tensor memory columns: O, the scores of two tiles, P of two tiles (two values to a column).
constexpr std::uint32_t kColumns = 512, kColO = 0, kColS = 128, kColP = 384;

constexpr int kPartBytes = kTile * 128;  // 64 channels of Q: 128 rows of 128 bytes
// V is an MN-major operand: rows are K of the product. A CTA's half of the channels is one swizzled row: 64 channels in 128 bytes, or 32 in
// 64 (layout type 4); 8-row groups follow one another.
template <int D>
__device__ __forceinline__ std::uint64_t value_desc(std::uint32_t smem_addr) {
  if constexpr (D == 128) return umma_desc_sw128(smem_addr);
  std::uint64_t d = static_cast<std::uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<std::uint64_t>(1) << 16;
  d |= static_cast<std::uint64_t>(512 >> 4) << 32;
  d |= static_cast<std::uint64_t>(1) << 46;
  d |= static_cast<std::uint64_t>(4) << 61;
  return d;
}
// The top bit of each half of a word is set if its exponent is all ones (infinities and NaN): adding one to the exponent carries there.
template <typename T>
__device__ __forceinline__ std::uint32_t full_exponent(std::uint32_t w) {
  constexpr std::uint32_t e = std::is_same<T, __half>::value ? 0x7C007C00u : 0x7F807F80u, one = std::is_same<T, __half>::value ? 0x04000400u : 0x00800080u;
  return (w & e) + one;
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

// Pairs of exponentials, of every 8, that exp2_fma computes: 8192 tokens, 32 / 8 heads of 128, and 509 over 8192 slots, 14 / 2 of 64: none
// 494 and 51.3 us, one 488 and 49.4, two 493 and 49.0, three 517 and 51.2.
constexpr int kFmaPairs = 1;
// 2^x for a pair of x on the FMA unit, which the softmax leaves half idle while the hardware's exponential has 16
// results a clock and SM: x = n + f with n whole and f in [-1/2, 1/2] (the sum with 1.5 * 2^23 rounds), 2^f by the polynomial
// of degree 4 with the least largest relative error on that interval (2.6e-6; Remez exchange), n added to its exponent. Below
// -126.5 what is left is a subnormal number, and below -127 one that is 0 in 16 bits: kFloor is the float above -127, where the polynomial is
// just above 1 and the exponent's field just empty. (2^-126 for what is not seen, times the largest bf16, would be 4.) What is past
// 127 or NaN gives nonsense: the caller looks at the largest x.
__device__ __forceinline__ void exp2_fma(std::uint64_t x, float& a, float& b) {
  constexpr float kFloor = -127.0f + 0x1p-17f;
  float x0, x1;
  unpack2(x, x0, x1);
  const std::uint64_t low = pack2(fmaxf(x0, kFloor), fmaxf(x1, kFloor));
  const std::uint64_t t = add2(low, pack2(12582912.0f, 12582912.0f)), n = add2(t, pack2(-12582912.0f, -12582912.0f));
  const std::uint64_t f = fma2(n, pack2(-1.0f, -1.0f), low);
  std::uint64_t p = fma2(f, pack2(0.009570102207362652f, 0.009570102207362652f), pack2(0.05591785907745361f, 0.05591785907745361f));
  p = fma2(p, f, pack2(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, pack2(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(p, f, pack2(0.9999992847442627f, 0.9999992847442627f));
  float p0, p1, t0, t1;
  unpack2(p, p0, p1);
  unpack2(t, t0, t1);
  a = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
  b = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if any is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 256 rows of one (sequence, key head) for a CTA pair, and the key tiles they see: the sinks' first, then from `from` to the last token's.
struct __align__(16) Work {
  int index, t0, u0;   // number of this work among the pair's (-1: no more); of its first even and its first odd tile among all such
  int h, b, first_token, n, len;
  int row0, row_last;  // rows of the sequence: (token, query head of the group)
  int p_lo, p_hi;      // slots of the first and the last token
  int from, sink_tiles, part, first_tile, count;  // a part has some of the key tiles; count 0: none
  __device__ __forceinline__ void set(const PromptArgs& a, int id, int first, int tokens, int slots) {
    const int heads = a.c.kv_heads;
    part = id % a.splits, id /= a.splits;
    h = id % heads, b = id / heads % a.c.batch;
    first_token = first, n = tokens, len = slots;
    row0 = (a.tiles - 1 - id / heads / a.c.batch) * (2 * kTile);
    row_last = min(row0 + 2 * kTile, n * a.group) - 1;
    p_lo = len - n + row0 / a.group, p_hi = len - n + row_last / a.group;
    from = a.window > 0 && max(p_lo, 0) - a.window + 1 > 0 ? (max(p_lo, 0) - a.window + 1) / kTile : 0;
    sink_tiles = min((min(a.sinks, p_hi + 1) + kTile - 1) / kTile, from);
    const long long all = p_hi < 0 ? 0 : sink_tiles + p_hi / kTile + 1 - from;
    first_tile = static_cast<int>(part * all / a.splits), count = static_cast<int>((part + 1) * all / a.splits) - first_tile;
  }
  __device__ __forceinline__ int slot(int j) const {
    j += first_tile;
    return (j < sink_tiles ? j : j - sink_tiles + from) * kTile;
  }
  // Whether every row from slot lo to slot hi sees all of a tile.
  __device__ __forceinline__ static bool all_seen(const PromptArgs& a, int slot0, int lo, int hi) {
    return slot0 + kTile - 1 <= lo && (a.window == 0 || slot0 + kTile <= a.sinks || slot0 > hi - a.window);
  }
  __device__ __forceinline__ bool seen_by_all(const PromptArgs& a, int slot0) const { return all_seen(a, slot0, p_lo, p_hi); }
};

// The works of this pair, one after the other. All works in the order of their length (the last rows of a sequence first), dealt to the
// pairs to and fro, so that nobody has the longer of every round; 32 rounds at a time, a lane each. What is dealt is numbers of works that each
// sequence would have if it were as long as the longest: those of a shorter one that do not exist leave their pair with less than others (5
// prompts of 104 to 297 tokens, 16 / 8 heads: of 120 numbers 88 exist; 30 pairs of 74 get two, 16 none). One warp of a CTA walks them and
// leaves them in shared memory for the others: with this in line wherever a role takes its next work the kernel was 179 KB of instructions,
// and its warps spent a quarter of their time waiting for them.
struct Walk {
  int round = 0, id = 0, first = 0, n = 0, len = 0, index = 0, t = 0, u = 0;
  unsigned left = 0;
  // Called by a whole warp; false: no more works.
  __device__ __forceinline__ bool next(const PromptArgs& a, int lane, Work& w) {
#pragma unroll 1
    while (left == 0u) {
      const int pairs = static_cast<int>(gridDim.x) / 2, pair = static_cast<int>(blockIdx.x) / 2;
      if (static_cast<long long>(round) * pairs >= a.works) return false;
      const int mine_round = round + lane;
      const long long mine_id = static_cast<long long>(mine_round) * pairs + ((mine_round & 1) != 0 ? pairs - 1 - pair : pair);
      bool mine = mine_id < a.works;
      if (mine) {
        id = static_cast<int>(mine_id);
        const int tile_id = id / a.splits / a.c.kv_heads, b = tile_id % a.c.batch;
        paged_tokens(a.c, a.cu, b, a.tokens, first, n);
        if (n > a.max_q) {
          atomicOr(a.c.status, kPagedBadTokens);
          n = a.max_q;
        }
        len = paged_len(a.c, b);
        mine = (a.tiles - 1 - tile_id / a.c.batch) * (2 * kTile) < n * a.group;
      }
      left = __ballot_sync(0xffffffffu, mine);
      round += 32;
    }
    const int from = __ffs(left) - 1;
    left &= left - 1u;
    w.set(a, __shfl_sync(0xffffffffu, id, from), __shfl_sync(0xffffffffu, first, from), __shfl_sync(0xffffffffu, n, from), __shfl_sync(0xffffffffu, len, from));
    w.index = index, w.t0 = t, w.u0 = u;
    index += w.count > 0, t += (w.count + 1) / 2, u += w.count / 2;
    return true;
  }
};

// The list of works in shared memory, kList of them, written one after the other by the Q warp.
constexpr int kList = 8;
struct List {
  Work work[kList];
  std::uint64_t here[kList];  // barriers
};
// A reader's place in it.
struct Reader {
  List* list;
  volatile int* abort_word;
  int at = 0;
  // The next work (into w); false: no more, or a wait expired. Called by whole warps.
  __device__ __forceinline__ bool next(Work& w) {
    if (!warp_wait_bar(smem_u32(&list->here[at % kList]), static_cast<std::uint32_t>(at / kList) & 1u, abort_word)) return false;
    w = list->work[at % kList];
    ++at;
    return w.index >= 0;
  }
};
// The key tiles of the works, one after the other.
struct Tiles {
  Reader reader;
  Work w;
  int j = 0;
  __device__ __forceinline__ Tiles(List* list, volatile int* abort_word) : reader{list, abort_word} { w.count = 0; }
  __device__ __forceinline__ bool next(int step = 1) {
    j += step;
#pragma unroll 1
    while (__builtin_expect(j >= w.count, 0)) {
      if (!reader.next(w)) return false;
      j = 0;
    }
    return true;
  }
};

// What infinities and NaN of V that some row does not see did not reach (see the V warp), for one row that has been stored: channels
// [from, to) of `out`.
template <typename T, typename Out>
__device__ __forceinline__ void add_nonfinite(const PromptArgs& a, const Work& w, int p, Out* out, int from, int to) {
#pragma unroll 1
  for (int j = 0; j < w.count; ++j) {
    const int slot0 = w.slot(j);
    if (w.seen_by_all(a, slot0)) continue;
#pragma unroll 1
    for (int slot = slot0; slot <= min(slot0 + kTile - 1, p); ++slot) {
      if (a.window > 0 && slot >= a.sinks && slot <= p - a.window) continue;
      const int page = paged_page(a.c, w.b, slot);
      if (page < 0) continue;
      const T* v = static_cast<const T*>(a.c.v) + paged_row(a.c, page, w.h, slot);
#pragma unroll 1
      for (int d = from; d < to; ++d) {
        const float x = to_float(v[d]);
        if (!isfinite(x)) out[d] = static_cast<Out>(static_cast<float>(out[d]) + x);
      }
    }
  }
}

// The same for tiles that all rows of the pair see, where an infinity of V has met every weight, those among them that are 0 in 16 bits: it is the output.
// 32 * kEach channels from `from` on, of the rows of a whole warp; `sums`: shared memory for as many. 16 bytes a lane, eight in flight (131072 slots
// take 2.4 ms; 2 bytes a lane 5.5): the other warps wait for this one, 200 ms at most.
template <typename T, int kEach, typename Out>
__device__ __forceinline__ void take_nonfinite(const PromptArgs& a, const Work& w, int from, int lane, float* sums, Out* out, bool live, bool empty) {
  constexpr int kChunks = 4 * kEach, kSlots = 32 / kChunks, kBatch = 8;  // lanes to a row; rows to a load
  const T* const v = static_cast<const T*>(a.c.v) + from + lane % kChunks * 8;
  float odd[8] = {};
#pragma unroll 1
  for (int j = 0; j < w.count; ++j) {
    const int slot0 = w.slot(j);
    if (!w.seen_by_all(a, slot0)) continue;
#pragma unroll 1
    for (int i0 = lane / kChunks; i0 < kTile; i0 += kBatch * kSlots) {
      uint4 x[kBatch];
      std::uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int slot = slot0 + i0 + i * kSlots, page = paged_page(a.c, w.b, slot);
        x[i] = page < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(v + paged_row(a.c, page, w.h, slot));
      }
#pragma unroll
      for (int i = 0; i < kBatch; ++i) any |= full_exponent<T>(x[i].x) | full_exponent<T>(x[i].y) | full_exponent<T>(x[i].z) | full_exponent<T>(x[i].w);
      if (__builtin_expect((any & 0x80008000u) == 0u, 1)) continue;
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        float y[8];
        load8<T>(x[i], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (!isfinite(y[e])) odd[e] += y[e];
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
#pragma unroll
    for (int m = kChunks; m < 32; m *= 2) odd[e] += __shfl_xor_sync(0xffffffffu, odd[e], m);
    if (lane < kChunks) sums[lane * 8 + e] = odd[e];
  }
  __syncwarp();
#pragma unroll 1
  for (int d = 0; d < 32 * kEach; ++d) {
    if (live && (empty || !isfinite(sums[d]))) out[from + d] = static_cast<Out>(empty ? 0.f : sums[d]);
  }
  __syncwarp();
}

// Persistent CTA pairs; a work is 256 rows of a (sequence, key head). A row is a (token, query head of the group) pair, the group's heads of a
// token side by side: they share their keys, and 256 rows have few tokens, so little of the causal edge is computed for nothing. Each
// CTA has 128 rows; tcgen05.mma.cta_group::2 multiplies both CTAs' rows with one K or V tile of 128 slots, of which each CTA holds half (64
// slots of K, half of V's channels), so a tile's bytes come from L2 once for 256 rows and shared memory feeds the tensor core with
// time to spare (768 of 1024 clocks a tile; a CTA by itself with 128 rows would need 1280).
//   warp 0      K and V tiles, a box per page; what is not in the pool reads as zeros (a box outside it)
//   warp 1      of CTA 0: S(t + 2) = Q K^T once S(t) has been read, O += P(t) V(t) once P(t) is there
//   warp 2      V's arrival, and in tiles that some row does not see whole what would make NaN of a 0 in P (see below)
//   warp 3      the list of works; Q of the next one
//   warps 4-7   softmax of the even tiles, one thread per row: S into registers, the row's maximum, P = exp2(c S - m), 16 bits wide, into
//               tensor memory columns of its own, so that neither S nor P ever waits for an MMA that still reads the other
//   warps 8-11  the same for the odd tiles, at the same time
// Both warpgroups refer a row's exponentials to one m: they swap the row's maximum of an even and the odd tile behind it. P, its sum
// and O are floating point, so m only has to keep P in range, and stays until a score is kRaise binades above the one it was made from; then the even tile's
// warpgroup scales O, once the P.V before have landed. P is rounded to the cache's type: both operands of an MMA
// have one type, and what the rounding leaves, as a second operand, would double the products P.V. The output's error against 64 bits is 1.2
// to 1.4 times that of its own rounding. The sum is of P before that rounding, in fp32. Tiles are counted through all works (t), so that loads, scores and the first
// softmax of a work go on while the one before is stored; a CTA per work spent 22 of 80 thousand clocks on its start and its end.
// Bound by the softmax: about 3750 clocks for two tiles, 2230 of them the exponentials with what goes with them (two warps of a scheduler; the
// unit for exponentials alone 1800), the rest loads, maxima and barriers, under which that unit idles; the MMAs need 2050. 8192 tokens, 32 / 8
// heads of 128: 488 us, 1.13 PFLOP/s (568 us under the power cap of a long run). Measured and slower: a warpgroup per 128 rows, P over
// S's columns (657 us); the warpgroups by turns, m handed on tile by tile (613); the maximum checked after the exponentials, which are
// repeated if it has grown too much, warpgroups not in step (593); two threads a row, 16 warps (529); S a quarter at a time
// from tensor memory in a loop a fourth as long (608); two threads a row and the groups by turns (532: the warp that issues the MMAs is then
// busy all the time, 2100 clocks a tile, half of them waits and instructions between the MMAs); P.V issued by a warp of its own (695).
template <typename T, int D>
__global__ void __launch_bounds__(Shape<D>::kThreads, 1)
prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
              const __grid_constant__ PromptArgs a) {
  using S = Shape<D>;
  constexpr bool kHalf = std::is_same<T, __half>::value;
  // m is the row's largest score so far less kShift, and moves once a score is kRaise above that. bf16 has fp32's range. fp16 ends at 2^16 and
  // loses bits below 2^-14: the largest of P is kept from 2^13 to 2^15, so that weights are whole to 2^-27 of the largest and held to 2^-38 of it
  // (from 2^6 to 2^8, weights of 2^-25 were off by a fiftieth).
  constexpr float kShift = kHalf ? 13.0f : 0.0f, kRaise = kHalf ? 2.0f : 30.0f;
  constexpr int kMarks = 32;  // works that the V warp can be ahead of the stores, at most: a stage each and two
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  const std::uint32_t rank = cluster_ctarank();

  extern __shared__ std::uint8_t smem_raw[];
  // Barriers of the leader (CTA 0 of the pair): Q, K, V, P, "S is read" and "O is read", by both CTAs; in each CTA: what the MMAs have done.
  __shared__ __align__(8) std::uint64_t s_q[2], s_k[S::kStages], s_v[S::kStages], s_read[2], s_p[2], s_o_free;
  __shared__ __align__(8) std::uint64_t s_q_free[2], s_k_free[S::kStages], s_v_free[S::kStages], s_v_here[S::kStages], s_scores[2], s_pv[2], s_q_here, s_left[kList];
  __shared__ List s_list;
  __shared__ float s_top[2][2][kTile], s_last[2][2][kTile][2];  // the largest scores of a pair of tiles; by work the warpgroups' sums and m
  __shared__ std::uint32_t s_tmem_base, s_nonfinite[kMarks];
  __shared__ __align__(16) std::uint8_t s_out[8][2048];  // of a softmax warp: 32 rows of 32 channels on their way out
  __shared__ int s_abort;
  const std::uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const auto q_smem = [&](int i) { return base + i * S::kQBytes; };
  const auto k_smem = [&](int s) { return base + 2 * S::kQBytes + s * S::kKBytes; };
  const auto v_smem = [&](int s) { return base + 2 * S::kQBytes + S::kStages * S::kKBytes + s * S::kVBytes; };
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(smem_u32(&s_k[s]), 1);
      mbar_init(smem_u32(&s_v[s]), 2);
      mbar_init(smem_u32(&s_k_free[s]), 1);
      mbar_init(smem_u32(&s_v_free[s]), 1);
      mbar_init(smem_u32(&s_v_here[s]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&s_q[i]), 2);
      mbar_init(smem_u32(&s_q_free[i]), 1);
      mbar_init(smem_u32(&s_read[i]), 8);
      mbar_init(smem_u32(&s_p[i]), 8);
      mbar_init(smem_u32(&s_scores[i]), 1);
      mbar_init(smem_u32(&s_pv[i]), 1);
    }
    mbar_init(smem_u32(&s_o_free), 16);
    mbar_init(smem_u32(&s_q_here), 1);
    for (int i = 0; i < kList; ++i) {
      mbar_init(smem_u32(&s_list.here[i]), 1);
      mbar_init(smem_u32(&s_left[i]), 8);
    }
    s_abort = 0;
    for (int i = 0; i < kMarks; ++i) s_nonfinite[i] = 0;
    fence_mbar_init();
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
  }
  Walk walk;
  Work first_work;
  bool has_work = false;
  if (warp == 3) has_work = walk.next(a, lane, first_work);
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(&s_tmem_base), kColumns);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers exist before anything arrives on them
  tc_fence_after();
  const std::uint32_t tmem = s_tmem_base;
  volatile int* abort_word = &s_abort;
  const auto warp_wait = [&](std::uint32_t bar, std::uint32_t parity) { return warp_wait_bar(bar, parity, abort_word); };
  const auto at_leader = [&](const std::uint64_t& bar) { return map_to_cta(smem_u32(&bar), 0u); };
  const auto stage = [](int t) { return t % S::kStages; };
  const auto stage_phase = [](int t) { return static_cast<std::uint32_t>(t / S::kStages) & 1u; };

  // 168 registers a thread (65536 over 384, in eights) become 208 for the softmax and 88 for the others.
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      // K: this CTA's 64 of the tile's slots; V: its half of the channels. A lane per (box of a page's rows, 64 channels).
      constexpr int kParts = D / 64;
      const int page_rows = 1 << a.c.page_shift, k_rows = min(page_rows, kTile / 2), v_rows = min(page_rows, kTile);
      const int k_row = lane / kParts * k_rows + static_cast<int>(rank) * (kTile / 2), k_part = lane % kParts, v_row = lane * v_rows;
      const bool has_k = lane < kTile / 2 / k_rows * kParts, has_v = lane < kTile / v_rows;
      // A tile's entries of the block table are fetched a tile ahead, and checked where they are used.
      constexpr int kNone = -1 << 30;
      const auto fetch = [&](const Work& w, int slot, bool mine) { return mine && slot < w.len ? a.c.table[w.b * a.c.table_ld + (slot >> a.c.page_shift)] : kNone; };
      const auto page_of = [&](int entry) {
        if (entry >= 0 && entry < a.c.num_pages) return entry;
        if (entry != kNone) atomicOr(a.c.status, kPagedBadPage);
        return static_cast<int>(a.c.num_pages);  // outside the pool: zeros
      };
      Tiles k(&s_list, abort_word), v(&s_list, abort_word);
      bool more_k = true, more_v = true;
      int k_entry = 0, v_entry = 0, k_slot = 0, v_slot = 0, k_head = 0, v_head = 0;
#pragma unroll 1
      for (int t = -1; more_k || more_v; ++t) {  // in the order of use: K of tile t, V of tile t - 2
        if (more_k) {
          const int entry = k_entry, slot = k_slot, h = k_head, s = stage(t);
          more_k = k.next();
          if (more_k) k_slot = k.w.slot(k.j) + k_row, k_head = k.w.h, k_entry = fetch(k.w, k_slot, has_k);
          if (t >= 0) {
            if (!warp_wait(smem_u32(&s_k_free[s]), stage_phase(t) ^ 1u)) break;
            if (rank == 0 && lane == 0) mbar_expect_tx(smem_u32(&s_k[s]), 2 * S::kKBytes);  // the pair's copies complete here
            __syncwarp();
            if (has_k) {
              tma_load_4d_pair(k_smem(s) + k_part * (kPartBytes / 2) + lane / kParts * k_rows * 128, &map_k, at_leader(s_k[s]), k_part * 64,
                               slot & (page_rows - 1), h, page_of(entry));
            }
          }
        }
        if (t >= 1 && more_v) {
          const int tv = t - 2, entry = v_entry, slot = v_slot, h = v_head, s = stage(tv);
          more_v = v.next();
          if (more_v) v_slot = v.w.slot(v.j) + v_row, v_head = v.w.h, v_entry = fetch(v.w, v_slot, has_v);
          if (tv >= 0) {
            if (!warp_wait(smem_u32(&s_v_free[s]), stage_phase(tv) ^ 1u)) break;
            if (lane == 0) mbar_expect_tx(smem_u32(&s_v_here[s]), S::kVBytes);
            __syncwarp();
            if (has_v) {
              tma_load_4d(v_smem(s) + v_row * D, &map_v, smem_u32(&s_v_here[s]), static_cast<int>(rank) * (D / 2), slot & (page_rows - 1), h, page_of(entry));
            }
          }
        }
      }
      __syncwarp();
    } else if (warp == 1 && rank == 0) {
      // The whole warp walks the loop (uniform control flow, every lane takes the waits); one elected lane issues.
      constexpr int kFormat = kHalf ? 0 : 1;
      constexpr std::uint32_t idesc_qk = umma_idesc(/*f32*/ 1, kFormat, kFormat, 0, 0, 2 * kTile, kTile);
      constexpr std::uint32_t idesc_pv = umma_idesc(/*f32*/ 1, kFormat, kFormat, 0, /*B MN-major*/ 1, 2 * kTile, D);
      constexpr std::uint16_t kBoth = 3;
      // Two tiles at a time, an even one and the odd one behind it (which a work's last may lack).
      Tiles ahead(&s_list, abort_word), now(&s_list, abort_word);  // whose scores come next, whose P.V
      bool more = ahead.next(2), ok = true, first = true;
      int k_tile = 0, v_tile = 0;
#pragma unroll 1
      for (;; first = false) {
        if (more) {  // S = Q K^T; 16 channels are 32 bytes of a row
          const int q = ahead.w.index & 1;
          if (__builtin_expect(ahead.j == 0, 0)) ok = warp_wait(smem_u32(&s_q[q]), static_cast<std::uint32_t>(ahead.w.index) >> 1 & 1u);
#pragma unroll 1
          for (int g = 0; g < 2 && ahead.j + g < ahead.w.count; ++g, ++k_tile) {
            const int s = stage(k_tile), nth = (g == 0 ? ahead.w.t0 : ahead.w.u0) + ahead.j / 2;
            ok = ok && warp_wait(smem_u32(&s_k[s]), stage_phase(k_tile)) && warp_wait(smem_u32(&s_read[g]), static_cast<std::uint32_t>(nth - 1) & 1u);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const std::uint32_t d = tmem + kColS + static_cast<std::uint32_t>(g) * kTile;
              std::uint64_t dq = umma_desc_sw128(q_smem(q)), dk = umma_desc_sw128(k_smem(s));
#pragma unroll 1
              for (std::uint32_t k = 0; k < D / 64; ++k, dq += kPartBytes >> 4, dk += kPartBytes >> 5) {
#pragma unroll
                for (std::uint32_t i = 0; i < 4; ++i) umma_f16_pair(d, dq + 2 * i, dk + 2 * i, idesc_qk, k + i);
              }
              tc_commit_pair(smem_u32(&s_scores[g]), kBoth);
              tc_commit_pair(smem_u32(&s_k_free[s]), kBoth);
              if (ahead.j + g + 1 == ahead.w.count) tc_commit_pair(smem_u32(&s_q_free[q]), kBoth);
            }
            __syncwarp();
          }
          if (!ok) break;
          more = ahead.next(2);
        }
        if (first) continue;
        if (!now.next(2)) break;
        const bool both = now.j + 1 < now.w.count;
        if (__builtin_expect(now.j == 0 && now.w.index > 0, 0)) ok = warp_wait(smem_u32(&s_o_free), static_cast<std::uint32_t>(now.w.index - 1) & 1u);
#pragma unroll 1
        for (int g = 0; g <= static_cast<int>(both); ++g, ++v_tile) {
          const int s = stage(v_tile);
          ok = ok && warp_wait(smem_u32(&s_v[s]), stage_phase(v_tile)) && warp_wait(smem_u32(&s_p[g]), static_cast<std::uint32_t>((g == 0 ? now.w.t0 : now.w.u0) + now.j / 2) & 1u);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {  // O (+)= P V; 16 slots are 8 columns of P and 16 rows of V
            std::uint64_t dv = value_desc<D>(v_smem(s));
            std::uint32_t at = tmem + kColP + static_cast<std::uint32_t>(g) * (kTile / 2), more_o = static_cast<std::uint32_t>(now.j + g);
#pragma unroll 1
            for (int k = 0; k < kTile / 64; ++k, at += 32, dv += 4 * D) {
#pragma unroll
              for (std::uint32_t i = 0; i < 4; ++i) {
                umma_f16_ts_pair(tmem + kColO, at + 8 * i, dv + i * D, idesc_pv, more_o);
                more_o = 1;
              }
            }
            tc_commit_pair(smem_u32(&s_pv[g]), kBoth);
            tc_commit_pair(smem_u32(&s_v_free[s]), kBoth);
          }
          __syncwarp();
        }
        if (!ok) break;
      }
    } else if (warp == 2) {
      // V is here: on to the leader. Where some row of the pair does not see all of a tile, its zeros in P would make NaN of an infinity
      // or a NaN in V: slots behind the last become zeros, and so do such values of slots that other rows see, which get them back
      // at the end.
      Tiles v(&s_list, abort_word);
      for (int t = 0; v.next(); ++t) {
        const int slot0 = v.w.slot(v.j), s = stage(t);
        if (!warp_wait(smem_u32(&s_v_here[s]), stage_phase(t))) break;
        if (__builtin_expect(!v.w.seen_by_all(a, slot0), 0)) {
          constexpr int kRowChunks = D / 16, kBatch = 8;  // 16-byte chunks of a row of this CTA's half; looked at at a time
          const int rows = min(v.w.len - slot0, kTile);
          for (int i = rows * kRowChunks + lane; i < kTile * kRowChunks; i += 32) st_shared(v_smem(s) + i * 16, make_uint4(0, 0, 0, 0));
          bool found = false;
#pragma unroll 1
          for (int i0 = lane; i0 < rows * kRowChunks; i0 += 32 * kBatch) {
            uint4 x[kBatch];
            std::uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) x[i] = ld_shared(v_smem(s) + (i0 + 32 * i) * 16 % S::kVBytes);  // (past the rows: some others again)
#pragma unroll
            for (int i = 0; i < kBatch; ++i) any |= full_exponent<T>(x[i].x) | full_exponent<T>(x[i].y) | full_exponent<T>(x[i].z) | full_exponent<T>(x[i].w);
            if (__builtin_expect((any & 0x80008000u) == 0u, 1)) continue;
#pragma unroll 1
            for (int i = i0; i < min(i0 + 32 * kBatch, rows * kRowChunks); i += 32) {
              uint4 y = ld_shared(v_smem(s) + i * 16);
              const std::uint32_t bx = nonfinite_halves<T>(y.x), by = nonfinite_halves<T>(y.y), bz = nonfinite_halves<T>(y.z), bw = nonfinite_halves<T>(y.w);
              if ((bx | by | bz | bw) == 0u) continue;
              found = true;
              y.x &= ~bx, y.y &= ~by, y.z &= ~bz, y.w &= ~bw;
              st_shared(v_smem(s) + i * 16, y);
            }
          }
          if (found) {  // the mark of this work, in both CTAs
            st_cluster_u32(map_to_cta(smem_u32(&s_nonfinite[v.w.index % kMarks]), 0u), static_cast<std::uint32_t>(v.w.index) + 1u);
            st_cluster_u32(map_to_cta(smem_u32(&s_nonfinite[v.w.index % kMarks]), 1u), static_cast<std::uint32_t>(v.w.index) + 1u);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(at_leader(s_v[s]));
      }
      __syncwarp();
    } else if (warp == 3) {
      // Q of this CTA's 128 rows, 16 bytes a lane and a few rows at a time; zeros past the last row.
      constexpr int kChunks = D / 8, kStep = 32 / kChunks;
      Work w = first_work;
      bool more = has_work;
      for (int at = 0;; ++at) {
        for (; more && w.count == 0; more = walk.next(a, lane, w)) {
          // Nothing to see for any row: their zeros (or an empty part), and no place in the list.
          for (int i = lane; i < kTile * kChunks; i += 32) {
            const int row = w.row0 + static_cast<int>(rank) * kTile + i / kChunks, token = row / a.group;
            if (row > w.row_last) break;
            const int head = w.h * a.group + row - token * a.group;
            if (a.splits > 1) {
              if (i % kChunks == 0) a.part_ml[(w.part * a.tokens + w.first_token + token) * a.q_heads + head] = make_float2(-INFINITY, 0.f);
              continue;
            }
            *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + static_cast<std::int64_t>(w.first_token + token) * a.o_row + head * a.o_head + i % kChunks * 8) = make_uint4(0, 0, 0, 0);
            if (i % kChunks == 0 && a.lse != nullptr) a.lse[static_cast<std::int64_t>(w.first_token + token) * a.q_heads + head] = -INFINITY;
          }
        }
        // The place in the list is free once the softmax has left the work that was there.
        if (at >= kList && !warp_wait(smem_u32(&s_left[at % kList]), static_cast<std::uint32_t>(at / kList - 1) & 1u)) break;
        if (!more) w.index = -1, w.count = 0;
        if (lane == 0) {
          s_list.work[at % kList] = w;
          mbar_arrive(smem_u32(&s_list.here[at % kList]));
        }
        __syncwarp();
        if (!more) break;
        const int q = w.index & 1, c = lane % kChunks;
        if (!warp_wait(smem_u32(&s_q_free[q]), (static_cast<std::uint32_t>(w.index) >> 1 & 1u) ^ 1u)) break;
        const int row0 = w.row0 + static_cast<int>(rank) * kTile;
        if (a.q_tma != 0) {
          // Whole tokens: rows behind the last are the next sequence's, or zeros, and are not stored.
          if (lane == 0) {
            mbar_expect_tx(smem_u32(&s_q_here), S::kQBytes);
            for (int part = 0; part < D / 64; ++part) tma_load_3d(q_smem(q) + part * kPartBytes, &map_q, smem_u32(&s_q_here), part * 64, w.h * a.group, w.first_token + row0 / a.group);
          }
          __syncwarp();
          if (!warp_wait(smem_u32(&s_q_here), static_cast<std::uint32_t>(w.index) & 1u)) break;
        } else {
          // 16 bytes a lane, a few rows at a time.
          int row = row0 + lane / kChunks, token = row / a.group, g = row - token * a.group;
          const T* src = static_cast<const T*>(a.q) + c * 8 + static_cast<std::int64_t>(w.first_token + token) * a.q_row + (w.h * a.group + g) * a.q_head;
#pragma unroll 4
          for (int r = lane / kChunks; r < kTile; r += kStep) {
            const bool there = row <= w.row_last;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q_smem(q) + c / 8 * kPartBytes + r * 128 + ((c % 8 ^ (r & 7)) << 4)),
                         "l"(there ? static_cast<const void*>(src) : a.q), "r"(there ? 16 : 0) : "memory");
            row += kStep, g += kStep, src += kStep * a.q_head;
            while (g >= a.group) g -= a.group, src += a.q_row - a.group * a.q_head;
          }
          asm volatile("cp.async.wait_all;" ::: "memory");
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(at_leader(s_q[q]));
        more = walk.next(a, lane, w);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int group = (warp - 4) / 4, quarter = warp & 3;  // a warp may touch TMEM lanes [32 (warp % 4), +32)
    const int r_local = quarter * 32 + lane;
    const std::uint32_t lane_off = static_cast<std::uint32_t>(quarter * 32) << 16;
    const std::uint32_t s_cols = tmem + lane_off + kColS + static_cast<std::uint32_t>(group) * kTile, p_cols = tmem + lane_off + kColP + static_cast<std::uint32_t>(group) * (kTile / 2);
    const float c = a.scale_log2;
    bool dead = false;
    // The two warps that have the same rows meet at a barrier of their own (496 us where mbarriers took 510). One that gives up, having set the abort word, arrives there once
    // more: the other leaves its meeting and sees the word.
    const auto meet = [&] {
      asm volatile("barrier.sync.aligned %0, 64;" ::"r"(1 + quarter) : "memory");
      return *abort_word == 0;
    };
    Reader reader{&s_list, abort_word};
    for (;;) {
      Work w;
      const int place = reader.at % kList;
      if (dead || !reader.next(w)) break;
      const int index = w.index;
      const int row = w.row0 + static_cast<int>(rank) * kTile + r_local;
      const bool live = row <= w.row_last;
      // (Rows past the last take the last one's token; they are not stored.)
      const int token = min(row, w.row_last) / a.group, p = w.len - w.n + token;
      T* const out = static_cast<T*>(a.out) + static_cast<std::int64_t>(w.first_token + token) * a.o_row + (w.h * a.group + min(row, w.row_last) - token * a.group) * a.o_head;
      const std::int64_t lse_at = static_cast<std::int64_t>(w.first_token + token) * a.q_heads + w.h * a.group + min(row, w.row_last) - token * a.group;
      const int warp_lo = __shfl_sync(0xffffffffu, p, 0), warp_hi = __shfl_sync(0xffffffffu, p, 31);
      float m = -INFINITY, l = 0.f;  // reference in binades, this warpgroup's part of the sum
#pragma unroll 1
      for (int j = group; j < w.count; j += 2) {
        const int nth = (group == 0 ? w.t0 : w.u0) + j / 2, odd = w.u0 + j / 2;  // number of this tile among its warpgroup's, of its pair's odd one
        const std::uint32_t phase = static_cast<std::uint32_t>(nth) & 1u;
        const bool both = (j | 1) < w.count;
        const int slot0 = w.slot(j);
        const bool masked = !Work::all_seen(a, slot0, warp_lo, warp_hi);
        if (!warp_wait(smem_u32(&s_scores[group]), phase)) {
          dead = true;
          break;
        }
        tc_fence_after();
        std::uint32_t r[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld_32x32(s_cols + i * 32, r[i]);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_tensor(at_leader(s_read[group]));
        if (__builtin_expect(masked, 0)) {  // what the row does not see is minus infinity, whatever it was
          const int hi = p - slot0, lo = a.window > 0 ? hi - a.window : -1, first = a.sinks - slot0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const std::uint32_t seen = seen_mask(i * 32, hi, lo, first);
#pragma unroll
            for (int e = 0; e < 32; ++e) r[i][e] = (seen >> e & 1u) != 0u ? r[i][e] : 0xFF800000u;
          }
        }
        // The row's largest score, NaN if one is. In binades.
        float top;
        {
          float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) x[i] = max3_nan(x[i], __uint_as_float(r[i][e]), __uint_as_float(r[i][e + 1]));
          }
          top = max3_nan(max3_nan(x[0], x[1], x[2]), x[3], x[3]);
        }
        top *= c;
        if (both) {  // of both tiles
          float(&tops)[2][kTile] = s_top[odd & 1];
          tops[group][r_local] = top;
          if (!meet()) {
            dead = true;
            break;
          }
          const float other = tops[group ^ 1][r_local];
          top = max3_nan(top, other, other);
        }
        if (__builtin_expect(!(top < INFINITY), 0)) l = __int_as_float(0x7FC00000), top = -INFINITY;  // NaN or infinity: so is the row, for good
        const bool raise = m == -INFINITY ? top > -INFINITY : top > m + (kShift + kRaise);
        float alpha = 1.0f;
        if (raise) {
          alpha = m == -INFINITY ? 0.f : ex2(m - (top - kShift));  // (nothing seen yet: O is 0)
          m = top - kShift, l *= alpha;
        }
        if (!warp_wait(smem_u32(&s_pv[group]), phase ^ 1u)) {  // the P before this one has been read
          dead = true;
          break;
        }
        tc_fence_after();
        if (__builtin_expect(group == 0 && j > 1 && __any_sync(0xffffffffu, raise), 0)) {
          // O times alpha, once the P.V of the tiles before have landed and ahead of this warpgroup's P, whose P.V comes first. (The wait above
          // has seen to it that the odd tile's barrier is at most one phase behind.)
          if (!warp_wait(smem_u32(&s_pv[1]), static_cast<std::uint32_t>(odd - 1) & 1u)) {
            dead = true;
            break;
          }
          tc_fence_after();
          const std::uint32_t o_cols = tmem + lane_off + kColO;
#pragma unroll 1
          for (int cc = 0; cc < D; cc += 16) {
            std::uint32_t o[16];
            tmem_ld_32x16(o_cols + cc, o);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st_32x16(o_cols + cc, o);
          }
        }
        const float bias = m == -INFINITY ? 0.f : -m;  // (a row that has seen nothing: 2^-infinity)
        const std::uint64_t c2 = pack2(c, c), m2 = pack2(bias, bias);
        std::uint64_t sum_a = pack2(0.f, 0.f), sum_b = sum_a;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          std::uint32_t pw[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float x, y;
            const std::uint64_t xy = fma2(pack2(__uint_as_float(r[i][e]), __uint_as_float(r[i][e + 1])), c2, m2);
            if (e / 2 % 8 < kFmaPairs) {
              exp2_fma(xy, x, y);
            } else {
              unpack2(xy, x, y);
              x = ex2(x), y = ex2(y);
            }
            if (e % 4 == 0) sum_a = add2(sum_a, pack2(x, y));
            else sum_b = add2(sum_b, pack2(x, y));
            pw[e / 2] = pack16<T>(x, y);
          }
          tmem_st_32x16(p_cols + i * 16, pw);
        }
        float s0, s1, s2, s3;
        unpack2(sum_a, s0, s1);
        unpack2(sum_b, s2, s3);
        l += (s0 + s1) + (s2 + s3);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_tensor(at_leader(s_p[group]));
      }
      if (dead) break;
      float(&last)[2][kTile][2] = s_last[index & 1];
      last[group][r_local][0] = l, last[group][r_local][1] = m;
      if (!meet()) break;
      const int last_group = (w.count - 1) & 1, last_nth = (last_group == 0 ? w.t0 : w.u0) + (w.count - 1) / 2;
      if (!warp_wait(smem_u32(&s_pv[last_group]), static_cast<std::uint32_t>(last_nth) & 1u)) {
        dead = true;
        break;
      }
      tc_fence_after();
      m = fmaxf(last[0][r_local][1], last[1][r_local][1]);  // (a last even tile may have raised it alone)
      // A row that has seen nothing still has m at minus infinity; so has one with a NaN or an infinity among the scores of every pair of tiles,
      // whose sums say so. (What the polynomial leaves of an unseen score is in the sums too: they are no sign of the former.)
      const bool undefined = isnan(last[0][r_local][0]) || isnan(last[1][r_local][0]), empty = m == -INFINITY && !undefined;
      l = undefined ? __int_as_float(0x7FC00000) : 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) l += last[i][r_local][0] == 0.f ? 0.f : last[i][r_local][0] * ex2(last[i][r_local][1] - m);
      const float inv = empty ? 0.f : 1.0f / l;
      const bool repair = *const_cast<volatile std::uint32_t*>(&s_nonfinite[index % kMarks]) == static_cast<std::uint32_t>(index) + 1u;
      // Half of the channels a warpgroup; O is free for the next work once they are in registers.
      std::uint32_t x[D / 2];
#pragma unroll
      for (int i = 0; i < D / 64; ++i) tmem_ld_32x32(tmem + lane_off + kColO + group * (D / 2) + i * 32, *reinterpret_cast<std::uint32_t(*)[32]>(&x[i * 32]));
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_tensor(at_leader(s_o_free));
      // A weight that is 0 in 16 bits makes NaN of an infinity in V, and so does a row whose scores are all minus infinity.
      float most[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < D / 2; i += 2) most[i / 2 % 4] = max3_nan(most[i / 2 % 4], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
      const bool spoilt = __any_sync(0xffffffffu, isnan(max3_nan(max3_nan(most[0], most[1], most[2]), most[3], most[3])) && !undefined);
      // The warp's rows, 64 bytes of each at a time, through shared memory, so that four lanes store them: a lane storing its own row touches 32
      // lines an instruction, and the eight warps kept each other waiting for 4500 clocks a work.
      const std::uint32_t at = smem_u32(&s_out[warp - 4][0]);
      const auto put = [&](int e, const uint4& v) { st_shared(at + lane * 64 + ((e ^ (lane >> 1 & 3)) << 4), v); };
      const auto store = [&](void* row_at, int byte) {
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int of = (lane >> 2) + 8 * e;  // row of the warp
          const std::uint64_t to = __shfl_sync(0xffffffffu, reinterpret_cast<std::uint64_t>(row_at), of);
          const uint4 v = ld_shared(at + of * 64 + (((lane & 3) ^ (of >> 1 & 3)) << 4));
          if (w.row0 + static_cast<int>(rank) * kTile + quarter * 32 + of <= w.row_last) *reinterpret_cast<uint4*>(reinterpret_cast<std::uint8_t*>(to) + byte + (lane & 3) * 16) = v;
        }
        __syncwarp();
      };
      if (__builtin_expect(a.splits > 1, 0)) {
        const std::int64_t part_at = static_cast<std::int64_t>(w.part) * a.tokens * a.q_heads + lse_at;
        float* const part_o = a.part_o + part_at * D;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) put(e, make_uint4(x[i * 16 + e * 4], x[i * 16 + e * 4 + 1], x[i * 16 + e * 4 + 2], x[i * 16 + e * 4 + 3]));
          store(part_o, (group * (D / 2) + i * 16) * 4);
        }
        if (__builtin_expect(spoilt, 0)) take_nonfinite<T, D / 64>(a, w, group * (D / 2), lane, reinterpret_cast<float*>(s_out[warp - 4]), part_o, live, empty);
        if (live) {
          if (repair && !empty) add_nonfinite<T>(a, w, p, part_o, group * (D / 2), (group + 1) * (D / 2));
          if (group == 0) a.part_ml[part_at] = make_float2(m, empty ? 0.f : l);
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float o[8];
#pragma unroll
            for (int f = 0; f < 8; ++f) o[f] = __uint_as_float(x[i * 32 + e * 8 + f]) * inv;
            put(e, store8<T>(o));
          }
          store(out, (group * (D / 2) + i * 32) * 2);
        }
        if (__builtin_expect(spoilt, 0)) take_nonfinite<T, D / 64>(a, w, group * (D / 2), lane, reinterpret_cast<float*>(s_out[warp - 4]), out, live, empty);
        if (live) {
          if (repair && !empty) add_nonfinite<T>(a, w, p, out, group * (D / 2), (group + 1) * (D / 2));
          if (group == 0 && a.lse != nullptr) a.lse[lse_at] = empty ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&s_left[place]));
    }
    if (__any_sync(0xffffffffu, *abort_word != 0)) asm volatile("barrier.arrive.aligned %0, 64;" ::"r"(1 + quarter) : "memory");
  }

  tc_fence_before();
  __syncthreads();
  if (s_abort != 0) {
    if (threadIdx.x == 0) atomicOr(a.c.status, kPagedWait);
    const std::uint64_t at = global_ns();
    while (global_ns() - at < 2000000ull) {
    }
    __syncthreads();
  }
  cluster_sync_all();  // nothing of the pair is in flight towards this CTA any more
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, kColumns);
  }
}

constexpr int kJoinWarps = 8;

// The parts of a row's keys joined, a warp per row: blockIdx.x is (tile, sequence, key head), blockIdx.y its rows.
template <typename T, int D>
__global__ void __launch_bounds__(32 * kJoinWarps) prompt_join_kernel(const PromptArgs a) {
  constexpr int kEach = D / 32;  // channels of a lane
  const int lane = static_cast<int>(threadIdx.x) & 31, id = blockIdx.x, h = id % a.c.kv_heads, b = id / a.c.kv_heads % a.c.batch;
  int first, n;  // (no kernel of the call writes cu_seqlens: read ahead of the wait)
  paged_tokens(a.c, a.cu, b, a.tokens, first, n);
  const int row = (a.tiles - 1 - id / a.c.kv_heads / a.c.batch) * (2 * kTile) + static_cast<int>(blockIdx.y) * kJoinWarps + static_cast<int>(threadIdx.x) / 32;
  if (row >= min(n, a.max_q) * a.group) return;
  const int token = first + row / a.group, head = h * a.group + row % a.group;
  const std::int64_t at = static_cast<std::int64_t>(token) * a.q_heads + head, step = a.tokens * a.q_heads;
  wait_for_predecessors();
  float m = -INFINITY, l = 0.f, o[kEach] = {};
#pragma unroll 4
  for (int i = 0; i < a.splits; ++i) {
    const float2 ml = a.part_ml[i * step + at];
    if (ml.y == 0.f) continue;  // nothing seen
    const float* part = a.part_o + (i * step + at) * D + lane * kEach;
    const float top = fmaxf(m, ml.x), f = ex2(ml.x - top), keep = l == 0.f ? 0.f : ex2(m - top);
    m = top, l = fmaf(f, ml.y, keep * l);
#pragma unroll
    for (int e = 0; e < kEach; ++e) o[e] = joined(f, part[e], keep, o[e]);
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  std::uint32_t packed[kEach / 2];
#pragma unroll
  for (int e = 0; e < kEach; e += 2) packed[e / 2] = pack16<T>(o[e] * inv, o[e + 1] * inv);
  T* out = static_cast<T*>(a.out) + static_cast<std::int64_t>(token) * a.o_row + head * a.o_head + lane * kEach;
  if constexpr (kEach == 4) {
    *reinterpret_cast<uint2*>(out) = make_uint2(packed[0], packed[1]);
  } else {
    *reinterpret_cast<std::uint32_t*>(out) = packed[0];
  }
  if (lane == 0 && a.lse != nullptr) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// How many parts the keys of 256 rows are cut into: as many as there are pairs without a work, but of kShortestPart tiles each.
// (509 tokens over 8192 slots, 14 / 2 heads of 64, 28 works for 74 pairs: 74 us in one part, 49 in two.)
constexpr int kShortestPart = 4;
struct PromptPlan {
  int tiles, splits;
  std::int64_t works;
  std::size_t ml, total;
};
PromptPlan plan(const PagedArgs& c, std::int64_t tokens, int q_heads, int head_dim, int max_q, int window, int sinks) {
  PromptPlan p{};
  const std::int64_t tiles = (static_cast<std::int64_t>(max_q) * (q_heads / c.kv_heads) + 2 * kTile - 1) / (2 * kTile), works = tiles * c.batch * c.kv_heads;
  std::int64_t keys = c.most;
  if (window > 0) keys = std::min<std::int64_t>(keys, static_cast<std::int64_t>(window) + max_q + sinks);
  const std::int64_t most = std::max<std::int64_t>(1, keys / (kTile * kShortestPart)), idle = std::max<std::int64_t>(1, sm_count() / 2 / std::max<std::int64_t>(1, works));
  p.splits = static_cast<int>(std::min(most, idle));
  p.tiles = static_cast<int>(std::min<std::int64_t>(tiles, INT_MAX)), p.works = works * p.splits;
  if (p.splits > 1) {
    const std::size_t rows = static_cast<std::size_t>(tokens) * q_heads * p.splits;
    p.ml = (rows * sizeof(float2) + 255) / 256 * 256;
    p.total = p.ml + rows * head_dim * sizeof(float);
  }
  return p;
}

template <typename T, int D>
int launch(const char* op, const PromptArgs& a, const CUtensorMap& map_q, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t st) {
  using S = Shape<D>;
  const auto kernel = prompt_kernel<T, D>;
  static std::atomic<std::uint64_t> allowed{0};
  if (const int rc = allow_shared(op, kernel, S::kSmem, allowed)) return rc;
  const LaunchChain chain(st);
  // As many pairs as fit at once, or as there are works.
  const unsigned pairs = static_cast<unsigned>(std::max(1, std::min(sm_count() / 2, a.works)));
  if (const int rc = enqueue(op, kernel, dim3(2 * pairs), S::kThreads, S::kSmem, st, 2, map_q, map_k, map_v, a)) return rc;
  if (a.splits == 1) return B2_OK;
  return enqueue(op, prompt_join_kernel<T, D>, dim3(static_cast<unsigned>(a.works / a.splits), 2 * kTile / kJoinWarps), 32 * kJoinWarps, 0, st, 1, a);
}

int check(const char* op, const b2_paged_cache* cache, PagedArgs* c, std::int64_t tokens, std::int64_t q_heads, int max_q, int* window, int* sinks) {
  if (const int rc = check_paged_cache(op, cache, c)) return rc;
  if (q_heads <= 0 || q_heads > 65535 || q_heads % cache->kv_heads != 0) return fail_invalid(op, "q must have a multiple of kv_heads heads, at most 65535");
  if (tokens < 0 || tokens > INT_MAX || max_q < 0) return fail_invalid(op, "tokens and max_q must not be negative");
  return check_window(op, *c, window, sinks);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

size_t b2_attention_paged_workspace_bytes(const b2_paged_cache* cache, int64_t tokens, int q_heads, int max_q, int window, int sinks) {
  PagedArgs c{};
  if (check("attention_paged", cache, &c, tokens, q_heads, max_q, &window, &sinks) != B2_OK) return 0;
  return std::max<std::size_t>(plan(c, tokens, q_heads, cache->head_dim, static_cast<int>(std::min<std::int64_t>(max_q, tokens)), window, sinks).total, 256);
}

int b2_attention_paged(const b2_paged_cache* cache, const b2_view3* q, const b2_view3* out, float* lse, const int32_t* cu_seqlens,
                       int max_q, float scale, int window, int sinks, void* workspace, size_t workspace_bytes, void* stream) {
  constexpr const char* op = "attention_paged";
  PromptArgs a{};
  if (q == nullptr || out == nullptr) return fail_invalid(op, "null q or out");
  if (const int rc = check(op, cache, &a.c, q->tokens, q->heads, max_q, &window, &sinks)) return rc;
  if (out->tokens != q->tokens || out->heads != q->heads) return fail_invalid(op, "q and out must have the same tokens and heads");
  if (!std::isfinite(scale) || !(scale > 0.0f)) return fail_invalid(op, "scale must be finite and positive");
  if (q->tokens == 0) return B2_OK;
  if (cache->batch == 0 || max_q == 0) return fail_invalid(op, "tokens without a sequence, or max_q 0");
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
  const PromptPlan p = plan(a.c, a.tokens, a.q_heads, cache->head_dim, a.max_q, window, sinks);
  if (p.works > INT_MAX / 2) return fail_invalid(op, "too many tokens for one call");
  a.tiles = p.tiles, a.splits = p.splits, a.works = static_cast<int>(p.works);
  if (const int rc = check_workspace(op, workspace, workspace_bytes, p.splits > 1 ? p.total : 0)) return rc;
  if (p.splits > 1) {
    a.part_ml = static_cast<float2*>(workspace), a.part_o = reinterpret_cast<float*>(static_cast<std::uint8_t*>(workspace) + p.ml);
  }
  a.scale_log2 = scale * 1.4426950408889634f, a.window = window, a.sinks = sinks;
  a.q_tma = kTile % a.group == 0 && q->row_stride > 0 && q->head_stride > 0;
  CUtensorMap map_q{}, map_k, map_v;
  if ((a.q_tma != 0 && !make_tensor_map_rows(&map_q, q, cache->head_dim, a.group, kTile / a.group, op)) ||
      !make_tensor_map_pages(&map_k, cache, false, std::min(cache->page_size, kTile / 2), 64, op) ||
      !make_tensor_map_pages(&map_v, cache, true, std::min(cache->page_size, kTile), cache->head_dim / 2, op)) {
    return B2_ERR_CUDA;
  }
  if (const int rc = paged_status_word(op, &a.c)) return rc;
  const cudaStream_t st = as_stream(stream);
  const bool wide = cache->head_dim == 128;
  if (cache->dtype == B2_DTYPE_BF16) {
    return wide ? launch<__nv_bfloat16, 128>(op, a, map_q, map_k, map_v, st) : launch<__nv_bfloat16, 64>(op, a, map_q, map_k, map_v, st);
  }
  return wide ? launch<__half, 128>(op, a, map_q, map_k, map_v, st) : launch<__half, 64>(op, a, map_q, map_k, map_v, st);
}

}  // extern "C"
