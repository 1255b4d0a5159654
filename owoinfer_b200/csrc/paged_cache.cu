// What goes into and out of a paged key-value cache: per-head norm + rotation + append, and eviction by accumulated attention weight.
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <mutex>

#include "attention.cuh"
#include "paged.cuh"

namespace b2 {
namespace {

__device__ unsigned g_paged_status = 0;

// ---------------------------------------------------------------------------------------------------------------
// Norm, rotation, append.
// ---------------------------------------------------------------------------------------------------------------
struct AppendArgs {
  PagedArgs c;
  const void* qkv;
  std::int64_t ld, tokens;
  const std::int32_t* cu;
  const std::int32_t* positions;
  const void* q_norm;
  const void* k_norm;
  const float* rope;
  std::int64_t rope_rows;
  void* q_out;
  std::int64_t q_row, q_head;
  float eps;
  int q_heads, half;          // half: rotated pairs
  std::int64_t padded;        // tokens, up to a whole number of warps
  int chunks, chunk_heads;    // a token's heads are cut into chunks of chunk_heads, each for one group of lanes
};

constexpr int kAppendHeads = 4;  // heads a group of lanes loads at a time
constexpr int kAppendThreads = 128;

// A lane's 8 channels of a head: the first elements of four rotation pairs and the second ones, so that norm, rotation and rounding
// need no other lane (the sum of squares apart). Pairs (i, i + half): two pieces of 4 channels; pairs (2 i, 2 i + 1), and the
// channels that are not rotated: one piece of 8.
template <bool kInterleaved>
struct Pieces {
  int first, second;  // channels of the pieces
  __device__ __forceinline__ Pieces(int lane, int half) {
    const bool turns = lane * 8 < 2 * half;
    first = !kInterleaved && turns ? lane * 4 : lane * 8;
    second = !kInterleaved && turns ? half + lane * 4 : lane * 8 + 4;
  }
  template <typename T>
  __device__ __forceinline__ uint4 load(const T* row) const {
    if constexpr (kInterleaved) return __ldcs(reinterpret_cast<const uint4*>(row + first));
    const uint2 x = __ldcs(reinterpret_cast<const uint2*>(row + first)), y = __ldcs(reinterpret_cast<const uint2*>(row + second));
    return make_uint4(x.x, x.y, y.x, y.y);
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const uint4& v) const {
    if constexpr (kInterleaved) {
      *reinterpret_cast<uint4*>(row + first) = v;
    } else {
      *reinterpret_cast<uint2*>(row + first) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2*>(row + second) = make_uint2(v.z, v.w);
    }
  }
  // The pieces' values as the (a, b) of the four rotation pairs, two pairs to a packed pair of fp32, and back.
  template <typename T>
  __device__ __forceinline__ static void split(const uint4& v, std::uint64_t (&a)[2], std::uint64_t (&b)[2]) {
    float x[8];
    load8<T>(v, x);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      a[i] = kInterleaved ? pack2(x[4 * i], x[4 * i + 2]) : pack2(x[2 * i], x[2 * i + 1]);
      b[i] = kInterleaved ? pack2(x[4 * i + 1], x[4 * i + 3]) : pack2(x[4 + 2 * i], x[5 + 2 * i]);
    }
  }
  template <typename T>
  __device__ __forceinline__ static uint4 merge(const std::uint64_t (&pa)[2], const std::uint64_t (&pb)[2]) {
    float a[4], b[4];
    unpack2(pa[0], a[0], a[1]), unpack2(pa[1], a[2], a[3]);
    unpack2(pb[0], b[0], b[1]), unpack2(pb[1], b[2], b[3]);
    if constexpr (kInterleaved) return make_uint4(pack16<T>(a[0], b[0]), pack16<T>(a[1], b[1]), pack16<T>(a[2], b[2]), pack16<T>(a[3], b[3]));
    return make_uint4(pack16<T>(a[0], a[1]), pack16<T>(a[2], a[3]), pack16<T>(b[0], b[1]), pack16<T>(b[2], b[3]));
  }
};

// A group of D / 8 lanes per (token, chunk of its heads). What a token needs once (its sequence, slot, page and angles: four loads one
// after the other) is found while its first heads are on their way; the norm's weights are folded into the angles once per token, so that a
// head costs its loads, a sum of squares over the group, four multiplications or additions a pair, the factor and the rounding.
// With a lane holding 8 neighbouring channels (the other half of a pair 8 shuffles away) and addresses worked out per head it was 230 instructions
// per head and warp, and the issue rate bound it at half the memory's. 7 prompts of up to 4096 tokens, 32 / 8 heads of 128: 83 us, 5.5 TB/s of
// rows read and written (0.84 of what a copy reaches; the issue rate is next, 64 % of it used). One token: the launch and four dependent loads.
template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
  constexpr int kLanes = D / 8;
  const int lane = static_cast<int>(threadIdx.x) % kLanes;
  // A warp's groups have neighbouring tokens and the same heads, so that every branch below that a shuffle depends on is the warp's; a
  // group without a token goes along.
  const std::int64_t unit = (static_cast<std::int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x) / kLanes;
  const std::int64_t chunk = unit / a.padded, at_token = unit - chunk * a.padded;
  if (chunk >= a.chunks) return;  // (padded is a multiple of a warp's groups)
  const bool there = at_token < a.tokens;
  const std::int64_t token = there ? at_token : a.tokens - 1;
  const int head0 = static_cast<int>(chunk) * a.chunk_heads;
  const Pieces<kInterleaved> pieces(lane, a.half);
  const T* row = static_cast<const T*>(a.qkv) + token * a.ld;

  const int last = min(head0 + a.chunk_heads, a.q_heads + 2 * a.c.kv_heads);
  uint4 raw[kAppendHeads], next[kAppendHeads];
  const auto load = [&](int from) {
#pragma unroll
    for (int i = 0; i < kAppendHeads; ++i) {
      if (from + i < last) next[i] = pieces.load(row + (from + i) * D);
    }
  };
  const auto take = [&](int then) {  // the heads that were on their way; those from `then` on take their place
#pragma unroll
    for (int i = 0; i < kAppendHeads; ++i) raw[i] = next[i];
    load(then);
  };
  load(head0);

  // The sequence of this token: the lanes of the group try kLanes places of cu_seqlens at a time.
  int lo = 0, hi = a.c.batch;  // cu[lo] <= token < cu[hi] (what lies outside shows up below)
  while (__any_sync(0xffffffffu, hi - lo > 1)) {
    const int step = max(1, (hi - lo + kLanes - 1) / kLanes), at = lo + (lane + 1) * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && a.cu[at] <= token) >> (threadIdx.x % 32 / kLanes * kLanes);
    const int n = __popc(below & ((1u << kLanes) - 1u));
    hi = min(hi, lo + (n + 1) * step);
    lo += n * step;
  }
  const int b = lo;
  int first, n;
  paged_tokens(a.c, a.cu, b, a.tokens, first, n);
  const int slot = paged_len(a.c, b) - n + static_cast<int>(token - first);
  const bool in_sequence = token >= first && token < first + n;
  if (!in_sequence || slot < 0) atomicOr(a.c.status, kPagedBadTokens);
  const int page = !there || !in_sequence || slot < 0 ? -1 : paged_page(a.c, b, slot);
  const bool stores = there && in_sequence;

  // sin and cos of this lane's pairs; 0 and 1 past the rotation.
  const bool turns = lane * 8 < 2 * a.half;
  std::uint64_t sn[2] = {pack2(0.f, 0.f), pack2(0.f, 0.f)}, cs[2] = {pack2(1.f, 1.f), pack2(1.f, 1.f)};
  if (turns) {
    std::int64_t position = a.positions != nullptr ? a.positions[token] : max(slot, 0);
    if (position < 0 || position >= a.rope_rows) {
      if (in_sequence) atomicOr(a.c.status, kPagedBadPosition);
      position = position < 0 ? 0 : a.rope_rows - 1;
    }
    const float* t = a.rope + position * (2 * a.half) + lane * 4;
    const float4 s4 = *reinterpret_cast<const float4*>(t), c4 = *reinterpret_cast<const float4*>(t + a.half);
    sn[0] = pack2(s4.x, s4.y), sn[1] = pack2(s4.z, s4.w);
    cs[0] = pack2(c4.x, c4.y), cs[1] = pack2(c4.z, c4.w);
  }

  // Heads [from, to) normalised and rotated; head `from` goes to `out`, the next ones `step` elements apart (nullptr: nowhere).
  const auto rotate = [&](int from, int to, const void* norm, T* out, std::int64_t step) {
    std::uint64_t ac[2], as[2], bc[2], bs[2];  // weight times cos and sin (bs: minus), for the first and the second of a pair
    {
      std::uint64_t wa[2] = {pack2(1.f, 1.f), pack2(1.f, 1.f)}, wb[2] = {wa[0], wa[0]};
      if (norm != nullptr) Pieces<kInterleaved>::template split<T>(pieces.load(static_cast<const T*>(norm)), wa, wb);
      const std::uint64_t minus = pack2(-1.f, -1.f);
#pragma unroll
      for (int i = 0; i < 2; ++i) ac[i] = mul2(wa[i], cs[i]), as[i] = mul2(wa[i], sn[i]), bc[i] = mul2(wb[i], cs[i]), bs[i] = mul2(mul2(wb[i], sn[i]), minus);
    }
    for (; from < to; from += kAppendHeads) {
      take(min(from + kAppendHeads, to));
#pragma unroll
      for (int i = 0; i < kAppendHeads; ++i) {
        if (from + i >= to) break;
        std::uint64_t x[2], y[2], u[2], v[2];
        Pieces<kInterleaved>::template split<T>(raw[i], x, y);
        float r = 1.0f;
        if (norm != nullptr) {
          float even, odd;
          unpack2(fma2(y[1], y[1], fma2(x[1], x[1], fma2(y[0], y[0], mul2(x[0], x[0])))), even, odd);
          float sum = even + odd;
#pragma unroll
          for (int m = kLanes / 2; m > 0; m /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
          r = rsqrtf(sum * (1.0f / D) + a.eps);
        }
        const std::uint64_t r2 = pack2(r, r);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u[j] = mul2(x[j], ac[j]), v[j] = mul2(y[j], bc[j]);
          if (turns) u[j] = fma2(y[j], bs[j], u[j]), v[j] = fma2(x[j], as[j], v[j]);
          u[j] = mul2(u[j], r2), v[j] = mul2(v[j], r2);
        }
        if (out != nullptr) {
          pieces.store(out, Pieces<kInterleaved>::template merge<T>(u, v));
          out += step;
        }
      }
    }
  };
  const int q_end = min(a.q_heads, last);
  if (head0 < q_end) rotate(head0, q_end, a.q_norm, stores ? static_cast<T*>(a.q_out) + token * a.q_row + head0 * a.q_head : nullptr, a.q_head);
  const int k_begin = max(head0, a.q_heads), k_end = min(a.q_heads + a.c.kv_heads, last);
  if (k_begin < k_end) {
    T* out = page < 0 ? nullptr : static_cast<T*>(a.c.k) + paged_row(a.c, page, k_begin - a.q_heads, slot);
    rotate(k_begin, k_end, a.k_norm, out, a.c.head_stride);
  }
  const int v_begin = max(head0, a.q_heads + a.c.kv_heads), v_end = min(a.q_heads + 2 * a.c.kv_heads, last);
  if (v_begin < v_end && page >= 0) {
    T* out = static_cast<T*>(a.c.v) + paged_row(a.c, page, v_begin - a.q_heads - a.c.kv_heads, slot);
    for (int from = v_begin; from < v_end; from += kAppendHeads) {
      take(min(from + kAppendHeads, v_end));
#pragma unroll
      for (int i = 0; i < kAppendHeads; ++i) {
        if (from + i >= v_end) break;
        pieces.store(out, raw[i]);
        out += a.c.head_stride;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Eviction.
// ---------------------------------------------------------------------------------------------------------------
struct EvictArgs {
  PagedArgs c;
  const float* weights;
  std::int64_t weights_ld;
  const std::int32_t* table_out;
  std::int64_t table_out_ld;
  std::int32_t* kept;
  std::int32_t* lens_out;
  float* weights_out;
  std::int64_t weights_out_ld;
  int sinks, recent, budget;
};

constexpr int kSelectThreads = 1024, kSelectWarps = kSelectThreads / 32;
constexpr int kSelectItems = 8;  // most slots of a thread in a round: a warp has neighbouring ones, a lane every 32nd of them
constexpr int kSelectRound = kSelectThreads * kSelectItems;
constexpr int kMostSelectCtas = 8;
constexpr int kBins = 2048, kThreadBins = kBins / kSelectThreads;

// The order of the weights as the order of unsigned numbers: -0 counts as 0, NaN comes below everything.
__device__ __forceinline__ unsigned weight_key(float w) {
  if (isnan(w)) return 0u;
  const unsigned u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint2 ld_cluster_v2(std::uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
// Sum of `v` over the CTA's threads before this one, and over all of them. Two barriers; s_warp is free again behind the next one.
__device__ __forceinline__ unsigned sum_before(unsigned v, unsigned (&s_warp)[kSelectWarps], int warp, int lane, unsigned& total) {
  unsigned upto = v;
#pragma unroll
  for (int m = 1; m < 32; m *= 2) {
    const unsigned o = __shfl_up_sync(0xffffffffu, upto, m);
    if (lane >= m) upto += o;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = upto;
  __syncthreads();
  const unsigned mine = lane < kSelectWarps ? s_warp[lane] : 0u;
  unsigned warps = mine;  // of the warps up to this lane's
#pragma unroll
  for (int m = 1; m < kSelectWarps; m *= 2) {
    const unsigned o = __shfl_up_sync(0xffffffffu, warps, m);
    if (lane >= m) warps += o;
  }
  total = __shfl_sync(0xffffffffu, warps, kSelectWarps - 1);
  return __shfl_sync(0xffffffffu, warps - mine, warp) + upto - v;
}

// A CTA per (sequence, key head), or a cluster of up to 8 where a head can have more than kSelectRound slots (16384 slots of 64 heads: 64 us for
// the call with two CTAs a head, 66 with one of twice the slots a thread, 76 with four: what a cluster waits for is more than what it shares). A
// CTA's share of the slots between the first and the last ones stays in registers (past 65536 slots a head it is read again for every pass).
// The weight of the last slot that stays is found from the top bits down, 11, 11 and 10 of them: a histogram over the cluster, and the bin in
// which the running count from above reaches what may stay. (Bytes put the weights of a cache into a dozen bins of the first
// histogram, where a warp's additions to one word wait for one another.) Then every CTA counts what stays of its share, and
// writes it behind what the CTAs before it keep. Bound by the latency of its dozen steps between barriers, not by the weights' bytes.
__device__ __forceinline__ void select(const EvictArgs& a, int h, int b, int len, int ctas, int rank) {
  __shared__ __align__(16) unsigned s_hist[2][kBins];
  __shared__ unsigned s_warp[kSelectWarps];
  __shared__ __align__(8) uint2 s_count;
  __shared__ unsigned s_pick[2];
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32;
  const std::int64_t row = static_cast<std::int64_t>(b) * a.c.kv_heads + h;
  const float* w = a.weights + row * a.weights_ld;
  float* w_out = a.weights_out == nullptr ? nullptr : a.weights_out + row * a.weights_out_ld;
  std::int32_t* kept = a.kept + row * a.budget;
  if (rank == 0 && h == 0 && tid == 0) a.lens_out[b] = min(len, a.budget);
  if (len <= a.budget) {  // (the same for the whole cluster)
    for (int i = rank * kSelectThreads + tid; i < a.budget; i += ctas * kSelectThreads) {
      kept[i] = i < len ? i : -1;
      if (i < len && w_out != nullptr) w_out[i] = w[i];
    }
    return;
  }
  for (int i = rank * kSelectThreads + tid; i < a.sinks + a.recent; i += ctas * kSelectThreads) {
    const int to = i < a.sinks ? i : a.budget - a.recent + i - a.sinks, from = i < a.sinks ? i : len - a.recent + i - a.sinks;
    kept[to] = from;
    if (w_out != nullptr) w_out[to] = w[from];
  }
  const int room = a.budget - a.sinks - a.recent;
  if (room == 0) return;
  const int middle = len - a.recent - a.sinks, share = (middle + ctas - 1) / ctas;
  const int begin = a.sinks + min(middle, rank * share), end = a.sinks + min(middle, (rank + 1) * share);
  const int rounds = max(1, (share + kSelectRound - 1) / kSelectRound);
  const int items = rounds > 1 ? kSelectItems : (share + kSelectThreads - 1) / kSelectThreads;  // of a thread in a round

  float mine[kSelectItems];
  const auto slot_of = [&](int round, int i) { return begin + round * kSelectRound + (warp * items + i) * 32 + lane; };
  const auto load = [&](int round) {
#pragma unroll
    for (int i = 0; i < kSelectItems; ++i) {
      if (i >= items) break;
      const int slot = slot_of(round, i);
      mine[i] = slot < end ? w[slot] : 0.f;
    }
  };
  if (rounds == 1) load(0);

  unsigned prefix = 0, wanted = static_cast<unsigned>(room);  // of the slots whose upper bits are `prefix`, how many stay
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, above_shift = pass == 0 ? 32 : pass == 1 ? 21 : 10;
    const unsigned mask = pass == 2 ? 1023u : 2047u;
    unsigned(&hist)[kBins] = s_hist[pass & 1];
    *reinterpret_cast<uint2*>(&hist[tid * kThreadBins]) = make_uint2(0, 0);
    __syncthreads();
    for (int round = 0; round < rounds; ++round) {
      if (rounds > 1) load(round);
#pragma unroll
      for (int i = 0; i < kSelectItems; ++i) {
        if (i >= items) break;
        const unsigned key = weight_key(mine[i]);
        if (slot_of(round, i) < end && (pass == 0 || key >> above_shift == prefix)) atomicAdd(&hist[key >> shift & mask], 1u);
      }
    }
    // (The other half of s_hist is cleared for the next pass only after this barrier: by then every CTA has read it.)
    uint2 bins;  // this thread's bins, the largest ones thread 0's
    const int bin0 = kBins - (tid + 1) * kThreadBins;
    if (ctas == 1) {
      __syncthreads();
      bins = *reinterpret_cast<const uint2*>(&hist[bin0]);
    } else {
      cluster_sync_all();
      bins = make_uint2(0, 0);
      for (int c = 0; c < ctas; ++c) {
        const uint2 x = ld_cluster_v2(map_to_cta(smem_u32(&hist[bin0]), c));
        bins.x += x.x, bins.y += x.y;
      }
    }
    unsigned total;
    unsigned before = sum_before(bins.x + bins.y, s_warp, warp, lane, total);
    const unsigned n[kThreadBins] = {bins.y, bins.x};
#pragma unroll
    for (int i = 0; i < kThreadBins; ++i) {
      if (before < wanted && before + n[i] >= wanted) s_pick[0] = static_cast<unsigned>(bin0 + kThreadBins - 1 - i), s_pick[1] = wanted - before;
      before += n[i];
    }
    __syncthreads();
    prefix = prefix << (pass == 2 ? 10 : 11) | s_pick[0];
    wanted = s_pick[1];
  }

  // `prefix` is the key of the last one that stays, and `wanted` of its equals stay. What lies above it and level with it in the shares ahead.
  unsigned above_before = 0, equal_before = 0;
  if (ctas > 1) {
    unsigned above = 0, equal = 0;
    for (int round = 0; round < rounds; ++round) {
      if (rounds > 1) load(round);
#pragma unroll
      for (int i = 0; i < kSelectItems; ++i) {
        if (i >= items) break;
        const unsigned key = weight_key(mine[i]);
        const bool there = slot_of(round, i) < end;
        above += there && key > prefix, equal += there && key == prefix;
      }
    }
    unsigned all_above, all_equal;
    sum_before(above, s_warp, warp, lane, all_above);
    sum_before(equal, s_warp, warp, lane, all_equal);
    if (tid == 0) s_count = make_uint2(all_above, all_equal);
    cluster_sync_all();
    for (int c = 0; c < rank; ++c) {
      const uint2 x = ld_cluster_v2(map_to_cta(smem_u32(&s_count), c));
      above_before += x.x, equal_before += x.y;
    }
    cluster_sync_all();  // nobody reads another CTA's shared memory from here on
  }

  const unsigned lower = (1u << lane) - 1u;
  for (int round = 0; round < rounds; ++round) {
    if (rounds > 1) load(round);
    // Of 32 slots side by side a bit each: above, level.
    const auto compare = [&](int i, unsigned& above, unsigned& equal) {
      const unsigned key = weight_key(mine[i]);
      const bool there = slot_of(round, i) < end;
      above = __ballot_sync(0xffffffffu, there && key > prefix), equal = __ballot_sync(0xffffffffu, there && key == prefix);
    };
    unsigned n_above = 0, n_equal = 0, above, equal;
#pragma unroll
    for (int i = 0; i < kSelectItems; ++i) {
      if (i >= items) break;
      compare(i, above, equal);
      n_above += __popc(above), n_equal += __popc(equal);
    }
    // (A lane's share of its warp's counts, so that the sums over threads are those over warps.)
    unsigned all_above, all_equal;
    unsigned ra = sum_before(lane == 0 ? n_above : 0u, s_warp, warp, lane, all_above);
    unsigned re = sum_before(lane == 0 ? n_equal : 0u, s_warp, warp, lane, all_equal);
    ra = above_before + __shfl_sync(0xffffffffu, ra, 0), re = equal_before + __shfl_sync(0xffffffffu, re, 0);
    above_before += all_above, equal_before += all_equal;
#pragma unroll
    for (int i = 0; i < kSelectItems; ++i) {
      if (i >= items) break;
      compare(i, above, equal);
      const unsigned mine_above = ra + __popc(above & lower), mine_equal = re + __popc(equal & lower);
      if ((above >> lane & 1u) != 0u || ((equal >> lane & 1u) != 0u && mine_equal < wanted)) {
        const unsigned to = static_cast<unsigned>(a.sinks) + mine_above + min(mine_equal, wanted);
        kept[to] = slot_of(round, i);
        if (w_out != nullptr) w_out[to] = mine[i];
      }
      ra += __popc(above), re += __popc(equal);
    }
  }
}

// Rows row0, row0 + step, … of the new pages from the slots in `kept`, kRows of K and of V in flight: a group of D / 8 lanes, 16 bytes each.
template <int D, int kRows>
__device__ __forceinline__ void move_rows(const EvictArgs& a, int b, int h, int row0, int step, int len) {
  const int lane = static_cast<int>(threadIdx.x) % (D / 8);
  const std::int32_t* kept = a.kept + (static_cast<std::int64_t>(b) * a.c.kv_heads + h) * a.budget;
  const std::uint16_t *k = static_cast<const std::uint16_t*>(a.c.k), *v = static_cast<const std::uint16_t*>(a.c.v);
  uint4 kr[kRows], vr[kRows];
  std::int64_t to[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int r = row0 + i * step;
    to[i] = -1;
    if (r >= len) continue;
    const int slot = kept[r], page = paged_page(a.c, b, slot), page_to = a.table_out[b * a.table_out_ld + (r >> a.c.page_shift)];
    if (page_to < 0 || page_to >= a.c.num_pages) atomicOr(a.c.status, kPagedBadPage);
    if (page < 0 || page_to < 0 || page_to >= a.c.num_pages) continue;
    const std::int64_t from = paged_row(a.c, page, h, slot) + lane * 8;
    to[i] = paged_row(a.c, page_to, h, r) + lane * 8;
    kr[i] = *reinterpret_cast<const uint4*>(k + from);
    vr[i] = *reinterpret_cast<const uint4*>(v + from);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    if (to[i] < 0) continue;
    *reinterpret_cast<uint4*>(static_cast<std::uint16_t*>(a.c.k) + to[i]) = kr[i];
    *reinterpret_cast<uint4*>(static_cast<std::uint16_t*>(a.c.v) + to[i]) = vr[i];
  }
}

__global__ void __launch_bounds__(kSelectThreads) select_kernel(const EvictArgs a) {
  dependents_may_start();
  select(a, blockIdx.y, blockIdx.z, paged_len(a.c, blockIdx.z), gridDim.x, blockIdx.x);
}

constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 4;  // rows of K and of V that a group of lanes has in flight

// kept -> the new pages. 64 heads of 4096 kept slots of 128: 46 us, 5.8 TB/s.
template <int D>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const EvictArgs a) {
  constexpr int kGroups = kMoveThreads / (D / 8);
  const int h = blockIdx.y, b = blockIdx.z;
  wait_for_predecessors();
  move_rows<D, kMoveRows>(a, b, h, static_cast<int>(blockIdx.x) * (kGroups * kMoveRows) + static_cast<int>(threadIdx.x) / (D / 8), kGroups,
                          min(paged_len(a.c, b), a.budget));
}

// Both at once for a few heads: the first CTA of a cluster selects, all of them move. One launch less, 2 us of the host's time; on the device
// 8 heads of 1100 slots to 512 10.3 us (two kernels 10.9), 2000 to 1024 12.4 (12.4). Past two rows a group of lanes the move wants more
// SMs (4000 to 2048: 16.5 and 14.4), and 16 heads are more clusters than fit at a time (1000 to 512: 19.8 and 12.4).
constexpr int kEvictCtas = 8, kEvictRows = 2;
template <int D>
__global__ void __launch_bounds__(kSelectThreads) evict_kernel(const EvictArgs a) {
  const int h = blockIdx.y, b = blockIdx.z, len = paged_len(a.c, b);
  if (blockIdx.x == 0) select(a, h, b, len, 1, 0);
  cluster_sync_all();  // (releases and acquires what the first CTA wrote, too)
  constexpr int kGroups = kSelectThreads / (D / 8);
  move_rows<D, kEvictRows>(a, b, h, static_cast<int>(blockIdx.x) * kGroups + static_cast<int>(threadIdx.x) / (D / 8), kEvictCtas * kGroups, min(len, a.budget));
}

template <typename T, int D>
int launch_append(const char* op, const AppendArgs& a, bool interleaved, cudaStream_t st) {
  const std::int64_t units = a.padded * a.chunks, per_block = kAppendThreads / (D / 8);
  const auto kernel = interleaved ? append_kernel<T, D, true> : append_kernel<T, D, false>;
  return enqueue(op, kernel, dim3(static_cast<unsigned>((units + per_block - 1) / per_block)), kAppendThreads, 0, st, 1, a);
}

}  // namespace

int check_paged_cache(const char* op, const b2_paged_cache* c, PagedArgs* a) {
  if (c == nullptr || c->struct_size < sizeof(b2_paged_cache)) return fail_invalid(op, "null cache, or a struct_size that is not b2_paged_cache's");
  if (c->dtype != B2_DTYPE_BF16 && c->dtype != B2_DTYPE_F16) return fail_invalid(op, "the cache's dtype must be B2_DTYPE_BF16 or B2_DTYPE_F16");
  if (c->head_dim != 64 && c->head_dim != 128) return fail_invalid(op, "head_dim must be 64 or 128");
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)) != 0) {
    return fail_invalid(op, "page_size must be a power of two from 16 to 1024");
  }
  if (c->batch < 0 || c->batch > 65535 || c->kv_heads <= 0 || c->kv_heads > 65535) return fail_invalid(op, "batch and kv_heads must be at most 65535, kv_heads positive");
  if (c->num_pages < 0 || c->num_pages > INT_MAX || c->table_width < 0 || static_cast<std::int64_t>(c->table_width) * c->page_size > kMostSlots ||
      c->table_ld < c->table_width) {
    return fail_invalid(op, "num_pages must be below 2^31, table_width * page_size at most 2^31 - 2^21, table_ld at least table_width");
  }
  if (c->page_stride % 8 != 0 || c->head_stride % 8 != 0 || c->row_stride % 8 != 0 || c->row_stride < c->head_dim || c->page_stride < 0 || c->head_stride < 0) {
    return fail_invalid(op, "the pools' strides must be multiples of 8 elements, a row's at least head_dim");
  }
  if (c->num_pages > 0 && (!rows_ok(c->k, 0, 0) || !rows_ok(c->v, 0, 0))) return fail_invalid(op, "null or not 16-byte aligned pool");
  if (c->batch > 0 && (c->seq_lens == nullptr || (c->table_width > 0 && c->block_table == nullptr))) return fail_invalid(op, "null seq_lens or block_table");
  *a = PagedArgs{};
  a->k = c->k, a->v = c->v;
  a->page_stride = c->page_stride, a->head_stride = c->head_stride, a->row_stride = c->row_stride, a->num_pages = c->num_pages;
  a->table = c->block_table, a->table_ld = c->table_ld, a->lens = c->seq_lens;
  a->most = c->table_width * c->page_size, a->batch = c->batch, a->kv_heads = c->kv_heads;
  for (a->page_shift = 4; (1 << a->page_shift) < c->page_size;) ++a->page_shift;
  return B2_OK;
}

int check_window(const char* op, const PagedArgs& c, int* window, int* sinks) {
  if (*window < 0 || *sinks < 0) return fail_invalid(op, "window and sinks must not be negative");
  if (*window >= c.most) *window = 0;
  if (*window > 1 << 30) return fail_invalid(op, "window must be at most 2^30");
  *sinks = std::min(*sinks, c.most);
  return B2_OK;
}

int paged_status_word(const char* op, PagedArgs* a) {
  static std::atomic<unsigned*> cached[64] = {};  // by device
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) device = 64;
  a->status = device < 64 ? cached[device].load(std::memory_order_relaxed) : nullptr;
  if (a->status != nullptr) return B2_OK;
  void* word = nullptr;
  if (const cudaError_t e = cudaGetSymbolAddress(&word, g_paged_status); e != cudaSuccess) {
    cudaGetLastError();
    return fail_cuda(op, e);
  }
  a->status = static_cast<unsigned*>(word);
  if (device < 64) cached[device].store(a->status, std::memory_order_relaxed);
  return B2_OK;
}

namespace {
// A map of 16-bit elements: sizes and boxes from the inner dimension out, strides of the outer ones in elements.
bool encode_map(CUtensorMap* map, const void* base, int rank, const std::int64_t* sizes, const std::int64_t* strides, const int* box, bool narrow, const char* op) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) {
      encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }
  });
  if (encode == nullptr) {
    fail_status(B2_ERR_CUDA, op, "cuTensorMapEncodeTiled is not available from this driver");
    return false;
  }
  cuuint64_t dims[4], bytes[3];
  cuuint32_t boxes[4], elem[4];
  for (int i = 0; i < rank; ++i) dims[i] = static_cast<cuuint64_t>(sizes[i]), boxes[i] = static_cast<cuuint32_t>(box[i]), elem[i] = 1;
  for (int i = 0; i + 1 < rank; ++i) bytes[i] = static_cast<cuuint64_t>(strides[i]) * 2;
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, bytes, boxes, elem,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, narrow ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return true;
  fail_status(B2_ERR_CUDA, op, "cuTensorMapEncodeTiled failed with code " + std::to_string(static_cast<int>(r)));
  return false;
}
}  // namespace

bool make_tensor_map_pages(CUtensorMap* map, const b2_paged_cache* c, bool values, int box_rows, int box_columns, const char* op) {
  const std::int64_t sizes[4] = {c->head_dim, c->page_size, c->kv_heads, c->num_pages}, strides[3] = {c->row_stride, c->head_stride, c->page_stride};
  const int box[4] = {box_columns, box_rows, 1, 1};
  return encode_map(map, values ? c->v : c->k, 4, sizes, strides, box, box_columns == 32, op);
}

bool make_tensor_map_rows(CUtensorMap* map, const b2_view3* v, int head_dim, int box_heads, int box_tokens, const char* op) {
  const std::int64_t sizes[3] = {head_dim, v->heads, v->tokens}, strides[2] = {v->head_stride, v->row_stride};
  const int box[3] = {64, box_heads, box_tokens};
  return encode_map(map, v->data, 3, sizes, strides, box, false, op);
}

}  // namespace b2

using namespace b2;

extern "C" {

int b2_qk_norm_rope_append(const b2_paged_cache* cache, const void* qkv, int64_t ld, int64_t tokens, int q_heads,
                           const int32_t* cu_seqlens, const int32_t* positions, const void* q_norm, const void* k_norm, float eps,
                           const float* rope, int64_t rope_rows, int rot_dim, int interleaved, void* q_out, int64_t q_row_stride,
                           int64_t q_head_stride, void* stream) {
  constexpr const char* op = "qk_norm_rope_append";
  AppendArgs a{};
  if (const int rc = check_paged_cache(op, cache, &a.c)) return rc;
  if (tokens < 0 || tokens > INT_MAX || q_heads <= 0 || q_heads > 65535) return fail_invalid(op, "tokens and q_heads must not be negative, q_heads from 1 to 65535");
  if (rot_dim < 0 || rot_dim > cache->head_dim || rot_dim % 16 != 0) return fail_invalid(op, "rot_dim must be a multiple of 16 up to head_dim");
  if ((q_norm == nullptr) != (k_norm == nullptr)) return fail_invalid(op, "q_norm and k_norm: both or neither");
  if (!(eps >= 0.0f) || std::isinf(eps)) return fail_invalid(op, "eps must be finite and not negative");
  if (tokens == 0) return B2_OK;
  const std::int64_t heads = q_heads + 2 * static_cast<std::int64_t>(cache->kv_heads);
  if (cache->batch == 0 || cu_seqlens == nullptr) return fail_invalid(op, "tokens without a sequence, or null cu_seqlens");
  if (!rows_ok(qkv, ld, 0) || ld < heads * cache->head_dim) return fail_invalid(op, "qkv must be 16-byte aligned, its rows at least (q_heads + 2 kv_heads) * head_dim elements and a multiple of 8 apart");
  if (!rows_ok(q_out, q_row_stride, q_head_stride)) return fail_invalid(op, "q_out needs a 16-byte aligned base and strides that are multiples of 8");
  if (q_norm != nullptr && (!aligned_to(q_norm, 16) || !aligned_to(k_norm, 16))) return fail_invalid(op, "q_norm and k_norm must be 16-byte aligned");
  if (rot_dim > 0 && (rope == nullptr || !aligned_to(rope, 16) || rope_rows <= 0)) return fail_invalid(op, "rope must be a 16-byte aligned table of at least one row");
  a.qkv = qkv, a.ld = ld, a.tokens = tokens, a.cu = cu_seqlens, a.positions = positions, a.q_norm = q_norm, a.k_norm = k_norm;
  a.rope = rope, a.rope_rows = rope_rows, a.q_out = q_out, a.q_row = q_row_stride, a.q_head = q_head_stride, a.eps = eps;
  a.q_heads = q_heads, a.half = rot_dim / 2;
  // Few tokens: four heads to a group of lanes, so that the whole GPU works. From 16 tokens per SM on all of a token's heads, so that what
  // a token needs is found once (32 / 8 heads of 128: 9000 tokens 47 us, with four heads 66; 4000 25 against 32; 2300 both 21; 1500 23
  // against 14).
  const bool whole = tokens >= 16 * static_cast<std::int64_t>(sm_count());
  a.chunk_heads = whole ? static_cast<int>(heads) : kAppendHeads;
  a.chunks = static_cast<int>((heads + a.chunk_heads - 1) / a.chunk_heads);
  a.padded = (tokens + 3) / 4 * 4;
  if (a.padded * a.chunks > INT_MAX) return fail_invalid(op, "too many tokens for one call");
  if (const int rc = paged_status_word(op, &a.c)) return rc;
  const bool wide = cache->head_dim == 128;
  if (cache->dtype == B2_DTYPE_BF16) {
    return wide ? launch_append<__nv_bfloat16, 128>(op, a, interleaved != 0, as_stream(stream)) : launch_append<__nv_bfloat16, 64>(op, a, interleaved != 0, as_stream(stream));
  }
  return wide ? launch_append<__half, 128>(op, a, interleaved != 0, as_stream(stream)) : launch_append<__half, 64>(op, a, interleaved != 0, as_stream(stream));
}

int b2_kv_evict(const b2_paged_cache* cache, const float* weights, int64_t weights_ld, int sinks, int recent, int budget,
                const int32_t* table_out, int64_t table_out_ld, int table_out_width, int32_t* kept, int32_t* lens_out,
                float* weights_out, int64_t weights_out_ld, void* stream) {
  constexpr const char* op = "kv_evict";
  EvictArgs a{};
  if (const int rc = check_paged_cache(op, cache, &a.c)) return rc;
  if (sinks < 0 || recent < 0 || budget <= 0 || static_cast<std::int64_t>(sinks) + recent > budget) {
    return fail_invalid(op, "budget must be positive, sinks and recent not negative and together at most budget");
  }
  if (budget > kMostSlots) return fail_invalid(op, "budget must be at most 2^31 - 2^21");
  if (table_out_width < 0 || table_out_ld < table_out_width || static_cast<std::int64_t>(table_out_width) * cache->page_size < budget) {
    return fail_invalid(op, "table_out must name pages for budget slots");
  }
  const std::int64_t slots = static_cast<std::int64_t>(cache->table_width) * cache->page_size;
  if (weights_ld < slots || (weights_out != nullptr && weights_out_ld < budget)) {
    return fail_invalid(op, "weights must have a place for every slot of the block table, weights_out for budget slots");
  }
  if (cache->batch == 0) return B2_OK;
  if (weights == nullptr || table_out == nullptr || kept == nullptr || lens_out == nullptr) return fail_invalid(op, "null weights, table_out, kept or lens_out");
  if (weights == weights_out) return fail_invalid(op, "weights_out must not be weights");
  // (Every CTA reads the old lengths while the first ones write the new.)
  if (lens_out < cache->seq_lens + cache->batch && cache->seq_lens < lens_out + cache->batch) return fail_invalid(op, "lens_out must not be the cache's seq_lens");
  a.weights = weights, a.weights_ld = weights_ld, a.table_out = table_out, a.table_out_ld = table_out_ld, a.kept = kept;
  a.lens_out = lens_out, a.weights_out = weights_out, a.weights_out_ld = weights_out_ld;
  a.sinks = sinks, a.recent = recent, a.budget = budget;
  if (const int rc = paged_status_word(op, &a.c)) return rc;
  const cudaStream_t st = as_stream(stream);
  const LaunchChain chain(st);
  int ctas = 1;
  while (ctas < kMostSelectCtas && static_cast<std::int64_t>(ctas) * kSelectRound < slots) ctas *= 2;
  const unsigned heads = static_cast<unsigned>(cache->kv_heads), batch = static_cast<unsigned>(cache->batch);
  const std::int64_t most = std::min<std::int64_t>(budget, slots);
  if (ctas == 1 && most <= kEvictCtas * kEvictRows * (kSelectThreads / (cache->head_dim / 8)) &&
      static_cast<std::int64_t>(heads) * batch * kEvictCtas <= sm_count() * 5 / 8) {
    const dim3 grid(kEvictCtas, heads, batch);
    return cache->head_dim == 128 ? enqueue(op, evict_kernel<128>, grid, kSelectThreads, 0, st, kEvictCtas, a)
                                  : enqueue(op, evict_kernel<64>, grid, kSelectThreads, 0, st, kEvictCtas, a);
  }
  if (const int rc = enqueue(op, select_kernel, dim3(static_cast<unsigned>(ctas), heads, batch), kSelectThreads, 0, st, ctas, a)) return rc;
  const int rows = kMoveThreads / (cache->head_dim / 8) * kMoveRows;
  if (most == 0) return B2_OK;
  const dim3 grid(static_cast<unsigned>((most + rows - 1) / rows), heads, batch);
  return cache->head_dim == 128 ? enqueue(op, move_kernel<128>, grid, kMoveThreads, 0, st, 1, a) : enqueue(op, move_kernel<64>, grid, kMoveThreads, 0, st, 1, a);
}

int b2_paged_cache_status(unsigned* host_value, int clear) {
  constexpr const char* op = "paged_cache_status";
  if (host_value == nullptr) return fail_invalid(op, "null host_value");
  if (const cudaError_t e = cudaMemcpyFromSymbol(host_value, g_paged_status, sizeof(unsigned)); e != cudaSuccess) return fail_cuda(op, e);
  if (clear != 0) {
    const unsigned zero = 0;
    if (const cudaError_t e = cudaMemcpyToSymbol(g_paged_status, &zero, sizeof(unsigned)); e != cudaSuccess) return fail_cuda(op, e);
  }
  return B2_OK;
}

}  // extern "C"
