// Log probabilities of given tokens under a row of logits, with rank, entropy and the most probable alternatives, in one pass over the logits.
#include <algorithm>
#include <cmath>

#include "attention.cuh"
#include "text.cuh"

namespace b2 {
namespace {

constexpr int kThreads = 128;
constexpr int kWarps = kThreads / 32;
// A lane's loads at a time, units (what a warp copies at a time) in shared memory, CTAs to an SM. Eight loads cost less around them, four leave more CTAs,
// which is what short rows want: their ends cannot hide behind another row's middle otherwise. 2400 rows in bf16 with one alternative: of 150000
// 146 us with eight and 166 with four, of 32000 62 and 59, of 4000 34 and 23. (256 threads, eight loads, 2 CTAs: 177, 94, 73; 64 threads,
// 9 CTAs: 142, 54, 21, but with 20 alternatives 203 for 179, and a few long rows a fifth slower.)
template <bool kLong>
struct Shape {
  static constexpr int kBatch = kLong ? 8 : 4, kStages = kLong ? 2 : 3, kPerSm = kLong ? 5 : 6;
  static constexpr int kUnit = 32 * kBatch, kRing = kStages * kThreads * kBatch * 16;
};
constexpr int kMostStages = 3;
constexpr int kMostTop = 32;
constexpr int kMostCluster = 8;
constexpr int kCandidates = 512;  // elements at or above the bound that are sorted
constexpr int kMostPicked = 64;    // threads whose elements are looked through again

struct LogprobArgs {
  const void* logits;
  std::int64_t ld;
  const std::int64_t* targets;
  float* logprobs;
  std::int32_t* ranks;
  float* entropy;
  float* lse;
  float* top_logprobs;
  std::int32_t* top_tokens;
  std::int64_t rows;
  unsigned* status;
  float scale, scale_log2;  // scale * log2(e)
  int vocab, top, ctas;
};

__device__ __forceinline__ void st_cluster_u64(std::uint32_t cluster_addr, std::uint64_t x) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_addr), "l"(x) : "memory");
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The order of values as unsigned numbers of the type's own size, 1 for NaN, 0 for none. (The lowest value, -infinity, is 0x3FF, 0x7F or 0x7FFFFF.)
template <typename T>
constexpr int kOrderBits = 8 * sizeof(T);
template <typename T>
__device__ __forceinline__ std::uint32_t order_of(float x) {  // (x: a value of T)
  if constexpr (sizeof(T) == 4) {
    const std::uint32_t u = __float_as_uint(x + 0.0f);  // (-0 is 0)
    return isnan(x) ? 1u : static_cast<std::int32_t>(u) < 0 ? ~u : u | 0x80000000u;
  } else {
    const std::uint32_t u = pack16<T>(x + 0.0f, 0.f) & 0xffffu;
    return isnan(x) ? 1u : (u & 0x8000u) != 0u ? ~u & 0xffffu : u | 0x8000u;
  }
}
template <typename T>
__device__ __forceinline__ float value_of(std::uint32_t order) {
  if (order == 1u) return __int_as_float(0x7fc00000);
  constexpr std::uint32_t kSign = 1u << (kOrderBits<T> - 1);
  const std::uint32_t u = (order & kSign) != 0u ? order & ~kSign : ~order & (kSign | (kSign - 1u));
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(u);
  } else {
    float lo, hi;
    unpack16<T>(u, lo, hi);
    return lo;
  }
}

template <typename T>
constexpr float kLowest = std::is_same<T, __half>::value ? -65504.f : std::is_same<T, float>::value ? -3.4028234e38f : -3.3895314e38f;
template <typename T>
constexpr int kChunk = 16 / sizeof(T);  // elements of a 16-byte load

// A 16-byte load's elements, as they are compared and as fp32.
template <typename T>
struct Chunk {
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&x)[kChunk<T>]) const {
    if constexpr (sizeof(T) == 2) {
      load8<T>(raw, x);
    } else {
      x[0] = __uint_as_float(raw.x), x[1] = __uint_as_float(raw.y), x[2] = __uint_as_float(raw.z), x[3] = __uint_as_float(raw.w);
    }
  }
};
// The largest (NaN if nothing else is there), and how many are at least some value.
template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
};
template <>
struct Pair<__half> {
  using type = __half2;
};
template <typename T>
__device__ __forceinline__ typename Pair<T>::type pair_of(std::uint32_t w) { return *reinterpret_cast<const typename Pair<T>::type*>(&w); }
template <typename T, int n>
__device__ __forceinline__ float top_of(const Chunk<T> (&v)[n]) {
  if constexpr (sizeof(T) == 4) {
    float m[4] = {__uint_as_float(v[0].raw.x), __uint_as_float(v[0].raw.y), __uint_as_float(v[0].raw.z), __uint_as_float(v[0].raw.w)};
#pragma unroll
    for (int u = 1; u < n; ++u) {
      m[0] = fmaxf(m[0], __uint_as_float(v[u].raw.x)), m[1] = fmaxf(m[1], __uint_as_float(v[u].raw.y));
      m[2] = fmaxf(m[2], __uint_as_float(v[u].raw.z)), m[3] = fmaxf(m[3], __uint_as_float(v[u].raw.w));
    }
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  } else {
    typename Pair<T>::type m[4] = {pair_of<T>(v[0].raw.x), pair_of<T>(v[0].raw.y), pair_of<T>(v[0].raw.z), pair_of<T>(v[0].raw.w)};
#pragma unroll
    for (int u = 1; u < n; ++u) {
      m[0] = __hmax2(m[0], pair_of<T>(v[u].raw.x)), m[1] = __hmax2(m[1], pair_of<T>(v[u].raw.y));
      m[2] = __hmax2(m[2], pair_of<T>(v[u].raw.z)), m[3] = __hmax2(m[3], pair_of<T>(v[u].raw.w));
    }
    m[0] = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
    return fmaxf(__low2float(m[0]), __high2float(m[0]));
  }
}
template <typename T>
__device__ __forceinline__ float top_of(const Chunk<T>& c) {
  const Chunk<T> v[1] = {c};
  return top_of(v);
}
// Nothing but -infinity.
template <typename T, int n>
__device__ __forceinline__ bool blank(const Chunk<T> (&v)[n]) {
  constexpr std::uint32_t kNone = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  std::uint32_t other = 0;
#pragma unroll
  for (int u = 0; u < n; ++u) other |= (v[u].raw.x ^ kNone) | (v[u].raw.y ^ kNone) | (v[u].raw.z ^ kNone) | (v[u].raw.w ^ kNone);
  return other == 0;
}
// (Four times as many; least: a value of T.)
template <typename T>
__device__ __forceinline__ int count_from(const Chunk<T>& c, float least) {
  if constexpr (sizeof(T) == 4) {
    return 4 * ((__uint_as_float(c.raw.x) >= least) + (__uint_as_float(c.raw.y) >= least) + (__uint_as_float(c.raw.z) >= least) + (__uint_as_float(c.raw.w) >= least));
  } else {
    const auto both = pair_of<T>(pack16<T>(least, least));
    // Masks of the halves that count: four bits of each half of each.
    const std::uint32_t t = (__hge2_mask(pair_of<T>(c.raw.x), both) & 0x0f0f0f0fu) | (__hge2_mask(pair_of<T>(c.raw.y), both) & 0xf0f0f0f0u);
    const std::uint32_t s = (__hge2_mask(pair_of<T>(c.raw.z), both) & 0x0f0f0f0fu) | (__hge2_mask(pair_of<T>(c.raw.w), both) & 0xf0f0f0f0u);
    return __popc((t & 0x00ff00ffu) | (s & 0xff00ff00u));
  }
}
// The value of T above x: a number, or NaN of infinity.
template <typename T>
__device__ __forceinline__ float next_of(float x) {
  return value_of<T>(order_of<T>(x) + 1u);
}

// (a - b) c, which may be a number where a - b is none.
__device__ __forceinline__ float apart(float a, float b, float c) { return fmaf(a, 0.5f, -0.5f * b) * (2.f * c); }

// Sums over part of a row against a reference `ref` near its largest logit: s = sum 2^x, w = sum x 2^x with x = (l - ref) c, c = scale log2(e).
// The reference is the largest of what came first and follows once something is kAhead binades above it.
struct Sums {
  float ref, s, w;  // (-infinity, 0, 0: nothing)
  __device__ __forceinline__ Sums moved(float to, float c) const {
    Sums r{to, 0.f, 0.f};
    if (s != 0.f) {  // (nothing, or only what weighs nothing, so far: nothing to scale, and -infinity times 0 to avoid)
      const float d = apart(ref, to, c), f = ex2(d);
      r.s = s * f;
      r.w = f == 0.f ? 0.f : f * fmaf(d, s, w);
    }
    return r;
  }
  // All lanes' sums (those of the first `width` lanes, a power of two, and of each such group), against the largest reference.
  __device__ __forceinline__ void join_lanes(int width, float c) {
    float to = ref;
    for (int m = width / 2; m > 0; m /= 2) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, m));
    *this = moved(to, c);
    for (int m = width / 2; m > 0; m /= 2) s += __shfl_xor_sync(0xffffffffu, s, m), w += __shfl_xor_sync(0xffffffffu, w, m);
  }
};
// A thread's sums while it reads. x = l c - base is one fma of a pair, base = ref c as it is rounded: what that is off is put right at the end. That is 64
// binades at most below kWide, where different logits are as far apart; a reference beyond is subtracted first. (2000 rows of 150000 in bf16, one in 500 allowed,
// the others at -1e9: 165 us; at -1e10, beyond: 244.)
struct Running {
  static constexpr float kAhead = 8.f, kWide = 2147483648.f;
  float ref = -INFINITY, base = 0.f;
  float limit = -INFINITY;  // up to it a load's largest element lets the sums go on as they are
  float least = -INFINITY;  // what is below it weighs nothing and may be cut to it (-infinity: not known)
  bool cuts = false;        // elements are cut as they come: there have been some that had to be, or the reference is wide
  std::uint64_t s[2] = {0, 0}, w[2] = {0, 0};  // (pairs, in two chains)
  __device__ __forceinline__ Sums finished(float c) const {
    float s0, s1, w0, w1;
    unpack2(add2(s[0], s[1]), s0, s1);
    unpack2(add2(w[0], w[1]), w0, w1);
    Sums r{ref, s0 + s1, w0 + w1};
    if (wide() || r.s == 0.f) return r;
    const float d = fmaf(ref, c, -base), f = ex2(-d);  // x above is (l - ref) c + d
    r.w = f * fmaf(-d, r.s, r.w), r.s *= f;
    return r;
  }
  __device__ __forceinline__ bool wide() const { return !(fabsf(base) < kWide); }
  // Ahead of elements of which `top` is the largest (NaN: no number among them).
  template <typename T>
  __device__ __forceinline__ void rise(float top, float c) {
    if (!(top > ref) || (ref > -INFINITY && apart(top, ref, c) <= kAhead)) return;
    Sums m = finished(c).moved(top, c);
    const bool was_wide = wide();
    ref = top, base = top * c;
    if (wide() != was_wide) cuts = !was_wide;
    if (!wide() && m.s != 0.f) {  // (what finished() will undo)
      const float d = fmaf(ref, c, -base), f = ex2(d);
      m.w = f * fmaf(d, m.s, m.w), m.s *= f;
    }
    s[0] = pack2(m.s, 0.f), w[0] = pack2(m.w, 0.f), s[1] = w[1] = pack2(0.f, 0.f);
    limit = wide() ? -INFINITY : top + kAhead / c;
    least = fmaxf(kLowest<T>, -2.9e38f / c);
    if (wide() || !(apart(least, top, c) < -200.f)) least = -INFINITY;
  }
  // The sums of 2^x and x 2^x go on over loads, the elements cut to `least` where that is asked for.
  template <typename T, int count, bool kCut>
  __device__ __forceinline__ void go_on(const Chunk<T> (&v)[count], float c, std::uint64_t (&s2)[2], std::uint64_t (&w2)[2]) const {
    const std::uint64_t minus = pack2(-base, -base), cc = pack2(c, c);
#pragma unroll
    for (int i = 0; i < 2; ++i) s2[i] = s[i], w2[i] = w[i];
#pragma unroll
    for (int u = 0; u < count; ++u) {
      float l[kChunk<T>];
      v[u].get(l);
#pragma unroll
      for (int i = 0; i < kChunk<T>; i += 2) {
        if (kCut) l[i] = max_nan(l[i], least), l[i + 1] = max_nan(l[i + 1], least);
        float x, y;
        const std::uint64_t xy = fma2(pack2(l[i], l[i + 1]), cc, minus);
        unpack2(xy, x, y);
        const std::uint64_t e = pack2(ex2(x), ex2(y));
        s2[i / 2 % 2] = add2(s2[i / 2 % 2], e), w2[i / 2 % 2] = fma2(e, xy, w2[i / 2 % 2]);
      }
    }
  }
  __device__ __forceinline__ void take(const std::uint64_t (&s2)[2], const std::uint64_t (&w2)[2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) s[i] = s2[i], w[i] = w2[i];
  }
  // The loads v, which lie at `from` too, 32 apart, with `top` the largest of their elements; behind `valid` of them such as hold `least`. Nearly always
  // the reference stands and all elements are numbers that x holds: what is not shows as NaN in the sum of x 2^x, -infinity times 0 among it. Then it is
  // done again, cut to `least`, and so are the loads that follow. (`top` is not waited for, nor every element looked at.)
  template <typename T, int count>
  __device__ __forceinline__ void add(const Chunk<T> (&v)[count], const uint4* from, int valid, float top, float c) {
    std::uint64_t s2[2], w2[2];
    if (!cuts) {
      go_on<T, count, false>(v, c, s2, w2);
      float w0, w1;
      unpack2(add2(w2[0], w2[1]), w0, w1);
      const bool odd = isnan(w0 + w1);
      if (!(top > limit) && !odd && (valid == count || least > -INFINITY)) {
        take(s2, w2);
        return;
      }
      if (ref == -INFINITY && top == -INFINITY) {  // nothing that weighs anything so far
        float s0, s1;
        unpack2(add2(s2[0], s2[1]), s0, s1);
        if (!isnan(s0 + s1)) return;
      }
      cuts = odd;
    }
    rise<T>(top, c);
    if (least > -INFINITY) {
      go_on<T, count, true>(v, c, s2, w2);
      take(s2, w2);
      return;
    }
#pragma unroll 1
    for (int u = 0; u < valid; ++u) {
      Chunk<T> one;
      float l[kChunk<T>];
      one.raw = from[u * 32];
      one.get(l);
#pragma unroll
      for (int i = 0; i < kChunk<T>; i += 2) add_two(l[i], l[i + 1], c);
    }
  }
  // Any elements: what is 2^-200 and less of the reference is 2^-200, 0 in fp32 and times x no NaN.
  __device__ __forceinline__ void add_two(float l, float m, float c) {
    const float by = wide() ? 0.5f : c, less = wide() ? 0.5f * ref : base, times = wide() ? 2.f * c : 1.f;  // (as apart() does)
    float x, y;
    unpack2(mul2(fma2(pack2(l, m), pack2(by, by), pack2(-less, -less)), pack2(times, times)), x, y);
    x = max_nan(x, -200.f), y = max_nan(y, -200.f);
    const std::uint64_t e = pack2(ex2(x), ex2(y));
    s[0] = add2(s[0], e), w[0] = fma2(e, pack2(x, y), w[0]);
  }
};

struct Shared {
  std::uint32_t best[kThreads];     // order of a thread's largest element
  std::uint32_t falling[kThreads];  // the same of each warp, the largest first
  std::uint32_t second[kThreads];   // order of its largest one outside the batch of loads that has the largest
  int best_at[kThreads];
  Sums warp_sums[kWarps];
  unsigned warp_before[kWarps];
  std::uint64_t found[kCandidates];
  std::uint64_t first[kMostCluster * kMostTop];  // of each CTA of the cluster: its first `top`, in order (in the first CTA)
  Sums sums[kMostCluster];
  unsigned before[kMostCluster];
  int picked[kMostPicked];
  int num_picked, num_found;
  std::uint32_t bound, above, place_bound;
  std::uint64_t full[kWarps][kMostStages];
  int abort;
};

// A warp's keys, the largest first.
__device__ __forceinline__ std::uint32_t sorted(std::uint32_t key, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k *= 2) {
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2) {
      const std::uint32_t other = __shfl_xor_sync(0xffffffffu, key, j);
      key = ((lane & k) == 0) == ((lane & j) == 0) ? max(key, other) : min(key, other);
    }
  }
  return key;
}
// The 32 largest of two such warps' keys, the largest first.
template <typename K>
__device__ __forceinline__ K merged(K a, K b, int lane) {
  K key = max(a, __shfl_sync(0xffffffffu, b, 31 - lane));
#pragma unroll
  for (int j = 16; j > 0; j /= 2) {
    const K other = __shfl_xor_sync(0xffffffffu, key, j);
    key = (lane & j) == 0 ? max(key, other) : min(key, other);
  }
  return key;
}
// The largest bound that at least `count` of the keys reach; a whole warp. 0 where fewer than `count` keys are above 0.
template <int kPer>
__device__ __forceinline__ std::uint32_t bound_of(const std::uint32_t (&key)[kPer], int count) {
  std::uint32_t bound = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const std::uint32_t t = bound | 1u << bit;
    unsigned n = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) n += key[i] >= t;
    if (__reduce_add_sync(0xffffffffu, n) >= static_cast<unsigned>(count)) bound = t;
  }
  return bound;
}
// A token and its place in the order as one number: falling in the order, unlike for every token.
__device__ __forceinline__ std::uint64_t entry(std::uint32_t order, std::uint32_t token) { return static_cast<std::uint64_t>(order) << 32 | (0xFFFFFFFFu - token); }

__device__ __forceinline__ void bulk_load(std::uint32_t dst, const void* src, std::uint32_t bytes, std::uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// A row as `head` elements up to the first 16-byte boundary, whole loads, and the rest; of the loads the run [begin, end) is the CTA's.
template <typename T>
struct Row {
  const T* logits;
  const uint4* body;
  int head, chunks, begin, end;
  __device__ __forceinline__ Row(const LogprobArgs& a, std::int64_t row, int rank) {
    logits = static_cast<const T*>(a.logits) + row * a.ld;
    head = min(a.vocab, static_cast<int>((16u - (reinterpret_cast<std::uintptr_t>(logits) & 15u)) % 16u / sizeof(T)));
    chunks = (a.vocab - head) / kChunk<T>;
    body = reinterpret_cast<const uint4*>(logits + head);
    const int per_cta = a.ctas == 1 ? chunks : (chunks + a.ctas - 1) / a.ctas;
    begin = min(rank * per_cta, chunks), end = min(begin + per_cta, chunks);
  }
};

// What a row's sums make of a logit, and the outputs.
template <typename T>
struct RowOutputs {
  const LogprobArgs& a;
  std::int64_t at;
  Sums sums;
  float log_s;
  bool nothing;
  __device__ __forceinline__ RowOutputs(const LogprobArgs& args, std::int64_t row, const Sums& s) : a(args), at(row), sums(s), log_s(logf(s.s)) {
    nothing = s.ref == -INFINITY && !isnan(s.s);
  }
  __device__ __forceinline__ float logprob(float l) const {
    return nothing ? -INFINITY : isnan(sums.s) ? __int_as_float(0x7fc00000) : apart(l, sums.ref, a.scale) - log_s;
  }
  __device__ __forceinline__ void row(std::int64_t target, float logit, unsigned before) const {  // (before: four times)
    const bool has_target = target >= 0 && target < a.vocab;
    if (a.lse != nullptr) a.lse[at] = nothing ? -INFINITY : fmaf(sums.ref, a.scale, log_s);
    if (a.entropy != nullptr) {
      const float h = log_s - sums.w / sums.s * 0.6931471805599453f;
      a.entropy[at] = nothing || h < 0.f ? 0.f : h;
    }
    if (a.logprobs != nullptr) a.logprobs[at] = has_target ? logprob(logit) : target < 0 ? 0.f : __int_as_float(0x7fc00000);
    if (a.ranks != nullptr) a.ranks[at] = has_target ? static_cast<int>(before / 4u) + 1 : 0;
  }
  __device__ __forceinline__ void token(int place, std::uint64_t e) const {
    a.top_tokens[at * a.top + place] = static_cast<std::int32_t>(0xFFFFFFFFu - static_cast<std::uint32_t>(e));
    a.top_logprobs[at * a.top + place] = logprob(value_of<T>(static_cast<std::uint32_t>(e >> 32)));
  }
};

// A CTA per row, or where rows are few a cluster, each CTA with a run of it; one pass over the logits. Every thread keeps its sums against its own
// reference, how many of its elements come before the target, and its largest element. The alternatives come from what the threads saw: the `top`-th
// largest of their largest elements is a bound that `top` elements reach, so that only the threads whose largest one reaches it can hold one of the first
// `top`: their elements are read once more (the batches of loads that have those, from L2), and those at or above the bound sorted by counting.
// A warp's loads are bulk copies into shared memory, units ahead of the one that it works on.
// Exponentials bound it after memory: 4096 rows of 160000 in bf16 with one alternative take 242 us, 83 % of a copy's rate, the exponentials' unit 67 % busy. Few rows take
// a chain of latencies: one row of 150001 with 5 alternatives 12 us, 6 of them for its sums, 2 for the target, 4 for the alternatives.
template <typename T, bool kLong>
__global__ void __launch_bounds__(kThreads, Shape<kLong>::kPerSm) logprobs_kernel(const LogprobArgs a) {
  constexpr int n = kChunk<T>, kBatch = Shape<kLong>::kBatch, kStages = Shape<kLong>::kStages, kUnit = Shape<kLong>::kUnit;
  constexpr unsigned kAll = 0xffffffffu;
  extern __shared__ __align__(128) std::uint8_t s_ring[];
  __shared__ __align__(16) Shared sh;
  const int ctas = a.ctas, rank = static_cast<int>(blockIdx.x % static_cast<unsigned>(ctas));
  const std::int64_t row = blockIdx.x / static_cast<unsigned>(ctas);
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32;
  const float c = a.scale_log2, nan = __int_as_float(0x7fc00000);
  const std::int64_t target64 = a.targets != nullptr ? __ldg(a.targets + row) : -1;
  if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // (the others are there: waited for ahead of the first store to one)
  const Row<T> r(a, row, rank);
  const T* const body = r.logits + r.head + static_cast<std::int64_t>(r.begin) * n;
  const int first_token = r.head + r.begin * n, loads = r.end - r.begin, edges = a.vocab - r.chunks * n;

  const std::uint32_t own_ring = smem_u32(s_ring) + warp * (kStages * kUnit * 16), own_bars = smem_u32(&sh.full[warp][0]);
  const auto copy_unit = [&](int unit, int stage) {  // (of this warp's: lane 0)
    if (unit * kUnit >= loads) return;
    const std::uint32_t bytes = static_cast<std::uint32_t>(min(kUnit, loads - unit * kUnit)) * 16u;
    mbar_expect_tx(own_bars + stage * 8, bytes);
    bulk_load(own_ring + stage * (kUnit * 16), reinterpret_cast<const uint4*>(body) + static_cast<std::int64_t>(unit) * kUnit, bytes, own_bars + stage * 8);
  };
  if (lane == 0) {  // (a warp's barriers are its own)
#pragma unroll
    for (int i = 0; i < kStages; ++i) mbar_init(own_bars + i * 8, 1);
    fence_mbar_init();
#pragma unroll
    for (int i = 0; i < kStages; ++i) copy_unit(warp + i * kWarps, i);
  }
  if (tid == 0) sh.abort = 0;
  const bool has_target = target64 >= 0 && target64 < a.vocab;
  const int target = has_target ? static_cast<int>(target64) : -1;
  const float mine = has_target ? to_float(r.logits[target]) : 0.f;
  // The elements outside whole loads, one to a thread of the first CTA.
  const int edge_token = tid < r.head ? tid : r.head + r.chunks * n + tid - r.head;
  const bool has_edge = rank == 0 && tid < edges;
  const float edge = has_edge ? to_float(r.logits[edge_token]) : 0.f;
  __syncthreads();  // (no wait looks at the abort word before it is cleared)
  int stage = 0;
  std::uint32_t parity = 0;
  bool lost = false;  // a wait expired

  const auto falling_of = [&](std::uint32_t key) {
    if (a.top > 1) return sorted(key, lane);
    for (int m = 16; m > 0; m /= 2) key = max(key, __shfl_xor_sync(kAll, key, m));
    return key;
  };
  Running sums;
  unsigned before = 0;
  // The thread's largest element and the first of the batch of loads that has it first, counted from the CTA's first (NaN and -infinity: not yet).
  float best_top = -INFINITY, second_top = -INFINITY;  // (second_top: outside that batch)
  int best_at = -1;
  const bool mine_nan = isnan(mine);
  const auto is_before = [&](float l, int token) { return l > mine || (l == mine && token < target) || (mine_nan && (!isnan(l) || token < target)); };
  const bool counts = has_target && a.ranks != nullptr;
  const float next = counts && !mine_nan ? next_of<T>(mine) : nan;  // what is behind the target comes before it from here on (of infinity NaN: nothing does)
  // The loads v, which lie at `from` too: first, first + 32, ...; behind `valid` of them the first again.
  const auto see = [&](Chunk<T>(&v)[kBatch], const uint4* from, int first, int valid) {
    const float top = top_of(v);
    if (sums.ref == -INFINITY) sums.template rise<T>(top, c);
    if (valid < kBatch) {
      std::uint32_t least = __float_as_uint(sums.least);
      if constexpr (sizeof(T) == 2) least = pack16<T>(sums.least, sums.least);
#pragma unroll
      for (int u = 1; u < kBatch; ++u) {
        if (u >= valid) v[u].raw = make_uint4(least, least, least, least);
      }
    }
    if (kLong || !(sums.cuts && top == -INFINITY && blank(v))) sums.add(v, from, valid, top, c);
    if (counts && (top >= mine || mine_nan)) {
      const int token = first_token + first * n;
      const bool ahead = token + ((kBatch - 1) * 32 + 1) * n <= target;
      if (!mine_nan && (ahead || token > target)) {
        const float least = ahead ? mine : next;
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (u < valid) before += count_from(v[u], least);
        }
      } else {
#pragma unroll 1
        for (int u = 0; u < valid; ++u) {
          Chunk<T> one;
          float l[n];
          one.raw = from[u * 32];
          one.get(l);
#pragma unroll
          for (int i = 0; i < n; ++i) before += is_before(l[i], token + u * 32 * n + i) ? 4u : 0u;
        }
      }
    }
    second_top = fmaxf(second_top, fminf(top, best_top));
    if (top > best_top) best_top = top, best_at = first;
  };
  for (int unit = warp; unit * kUnit < loads; unit += kWarps) {
    if (!lost && !mbar_try_wait(own_bars + stage * 8, parity)) lost = !wait_bar(own_bars + stage * 8, parity, &sh.abort);
    const uint4* const from = reinterpret_cast<const uint4*>(s_ring) + (warp * kStages + stage) * kUnit + lane;
    const int first = unit * kUnit + lane;
    Chunk<T> v[kBatch];
    if (!lost && (unit + 1) * kUnit <= loads) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) v[u].raw = from[u * 32];
      see(v, from, first, kBatch);
    } else if (!lost && first < loads) {
      const int valid = min(kBatch, (loads - first + 31) / 32);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) v[u].raw = from[u < valid ? u * 32 : 0];
      see(v, from, first, valid);
    }
    lost = __any_sync(kAll, lost);  // (the unit is read)
    // What a lane has to cut is a mask's, mostly, and then all cut: lanes that go on differently would take turns. (509 rows of 32003 in fp16 of which one in 500
    // is allowed: 24.5 us without this and the look at whole loads, 21.2 with. Long rows without a mask would take 5 % more: 4096 of 160000 238 and 250;
    // with one 2000 of 150000 181 and 139.)
    if constexpr (!kLong) sums.cuts = __any_sync(kAll, sums.cuts);
    if (!lost && lane == 0) copy_unit(unit + kStages * kWarps, stage);
    stage = stage == kStages - 1 ? 0 : stage + 1;
    parity ^= stage == 0 ? 1u : 0u;
  }
  std::uint32_t best = best_at >= 0 ? order_of<T>(best_top) : 0u;
  if (has_edge) {
    sums.template rise<T>(edge, c);
    sums.add_two(edge, -INFINITY, c);
    if (counts) before += is_before(edge, edge_token) ? 4u : 0u;
  }

  // The warp's sums, and the order of its threads' largest elements.
  Sums all = sums.finished(c);
  if (lost) all.s = nan;
  all.join_lanes(32, c);
  for (int m = 16; m > 0; m /= 2) before += __shfl_xor_sync(kAll, before, m);
  if (lane == 0) sh.warp_sums[warp] = all, sh.warp_before[warp] = before;
  if (a.top > 0) {
    sh.best[tid] = best, sh.second[tid] = second_top > -INFINITY ? order_of<T>(second_top) : 0u, sh.best_at[tid] = best_at;
    sh.falling[tid] = falling_of(best);
  }
  __syncthreads();
  if (ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");

  Sums row_sums = lane < kWarps ? sh.warp_sums[lane] : Sums{-INFINITY, 0.f, 0.f};
  row_sums.join_lanes(kWarps, c);
  unsigned row_before = lane < kWarps ? sh.warp_before[lane] : 0u;
  for (int m = kWarps / 2; m > 0; m /= 2) row_before += __shfl_xor_sync(kAll, row_before, m);
  row_before = __shfl_sync(kAll, row_before, 0);
  row_sums.ref = __shfl_sync(kAll, row_sums.ref, 0), row_sums.s = __shfl_sync(kAll, row_sums.s, 0), row_sums.w = __shfl_sync(kAll, row_sums.w, 0);
  const RowOutputs<T> put(a, row, row_sums);
  if (ctas == 1) {
    if (tid == 0) put.row(target64, mine, row_before);
  } else if (tid == 0) {
    const std::uint32_t at = map_to_cta(smem_u32(sh.sums + rank), 0);
    st_cluster_u32(at, __float_as_uint(row_sums.ref)), st_cluster_u32(at + 4, __float_as_uint(row_sums.s)), st_cluster_u32(at + 8, __float_as_uint(row_sums.w));
    st_cluster_u32(map_to_cta(smem_u32(sh.before + rank), 0), row_before);
  }
  if (a.top > 0) {
    const std::uint32_t to = ctas > 1 ? map_to_cta(smem_u32(sh.first + rank * kMostTop), 0) : 0u;
    const auto put_one = [&](int place, std::uint64_t e) {  // (0: there are not that many)
      if (ctas > 1) st_cluster_u64(to + place * 8, e);
      else if (e != 0) put.token(place, e);
    };
    // The bound, how many threads are above it, and who reaches it: by the first warp.
    std::uint32_t key[kWarps];
    const auto pick = [&](const auto& is_one) {
      int num = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        const bool one = is_one(i);
        const unsigned those = __ballot_sync(kAll, one);
        const int at = num + __popc(those & ((1u << lane) - 1u));
        if (one && at < kMostPicked) sh.picked[at] = lane + 32 * i;
        num += __popc(those);
      }
      if (lane == 0) sh.num_picked = num;
    };
    const auto find_bound = [&] {
      if (warp == 0) {
        std::uint32_t bound, above = 0;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) key[i] = sh.falling[lane + 32 * i];
        if (a.top > 1) {
#pragma unroll
          for (int m = 1; m < kWarps; m *= 2) {
#pragma unroll
            for (int i = 0; i < kWarps; i += 2 * m) key[i] = merged(key[i], key[i + m], lane);
          }
          bound = __shfl_sync(kAll, key[0], a.top - 1);
          above = static_cast<std::uint32_t>(__popc(__ballot_sync(kAll, key[0] > bound)));
        } else {
          bound = key[0];
#pragma unroll
          for (int i = 1; i < kWarps; ++i) bound = max(bound, key[i]);
        }
        pick([&](int i) { return sh.best[lane + 32 * i] >= bound && sh.best[lane + 32 * i] > 0u; });
        if (lane == 0) sh.bound = bound, sh.above = above, sh.num_found = 0;
      }
      __syncthreads();
    };
    // The i-th load of a thread, and how many units a warp has at most.
    const auto load_of = [&](int thread, int i) { return (thread / 32 + i / kBatch * kWarps) * kUnit + i % kBatch * 32 + thread % 32; };
    const int units_each = (loads + kWarps * kUnit - 1) / (kWarps * kUnit);
    const auto load = [&](int at) {
      Chunk<T> v;
      v.load(body + static_cast<std::int64_t>(at) * n);
      return v;
    };
    find_bound();
    if (sh.bound == 0u) {
      // Fewer than `top` threads have seen anything above -infinity: for the others their first -infinity, or NaN. (The bound may be one of these
      // then. Of a thread with a number it is not known whether another of its batches reaches that: it is looked through.)
      if (sh.second[tid] == 0u) sh.second[tid] = order_of<T>(-INFINITY);
      if (best == 0u) {
        int where = -1;
        for (int j = 0; j < units_each * kBatch && best <= 1u; ++j) {
          const int at = load_of(tid, j);
          if (at >= loads) continue;
          const std::uint32_t o = order_of<T>(top_of(load(at)));
          if (o > best) best = o, where = at - j % kBatch * 32;
        }
        sh.best[tid] = sh.second[tid] = best, sh.best_at[tid] = where;
      }
      sh.falling[tid] = falling_of(best);
      __syncthreads();
      find_bound();
    }
    const std::uint32_t bound = sh.bound;
    // Where many threads' largest elements equal the bound (a mask that leaves fewer than `top` tokens, a constant row), only the first
    // places can hold an alternative: the bound on places is that of as many loads as are wanted.
    std::uint32_t place_bound = 0xffffffffu;
    if (sh.num_picked > kMostPicked) {
      __syncthreads();  // (the number is read)
      if (warp == 0) {
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
          const int thread = lane + 32 * i;
          key[i] = 0u;
          if (sh.best[thread] == bound) {
            Chunk<T> v[kBatch];
            const int at = sh.best_at[thread];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) v[u] = load(at + u * 32 < loads ? at + u * 32 : at);
#pragma unroll
            for (int u = kBatch - 1; u >= 0; --u) {  // (the first load of the batch that has it)
              if (at + u * 32 < loads && order_of<T>(top_of(v[u])) == bound) key[i] = 0x7fffffffu - static_cast<std::uint32_t>(at + u * 32);
            }
          }
        }
        const std::uint32_t least = bound_of(key, a.top - static_cast<int>(sh.above));
        if (lane == 0) sh.place_bound = 0x7fffffffu - least;
        pick([&](int i) { return sh.best[lane + 32 * i] > bound || key[i] >= least; });  // (`top` threads)
      }
      __syncthreads();
      place_bound = sh.place_bound;
    }
    const int num_picked = sh.num_picked;
    const auto push = [&](std::uint64_t e) {
      const int i = atomicAdd(&sh.num_found, 1);
      if (i < kCandidates) sh.found[i] = e;
    };
    const std::uint64_t edge_entry = has_edge ? entry(order_of<T>(edge), static_cast<std::uint32_t>(edge_token)) : 0;
    if (edge_entry != 0) push(edge_entry);
    const auto look = [&](const Chunk<T>& v, int at) {
      const std::uint32_t order = order_of<T>(top_of(v));
      if (order < bound || (order == bound && static_cast<std::uint32_t>(at) > place_bound)) return;
      float l[n];
      v.get(l);
#pragma unroll
      for (int e = 0; e < n; ++e) {
        const std::uint32_t o = order_of<T>(l[e]);
        if (o > bound || (o == bound && static_cast<std::uint32_t>(at) <= place_bound)) push(entry(o, static_cast<std::uint32_t>(first_token + at * n + e)));
      }
    };
    // `count` loads, where(i) says which (what is not below `loads` is none), several of a thread on their way.
    const auto look_through = [&](int count, const auto& where) {
      constexpr int kAhead = 2;
      for (int i = tid; i < count; i += kAhead * kThreads) {
        Chunk<T> v[kAhead];
        int at[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
          at[q] = i + kThreads * q < count ? where(i + kThreads * q) : loads;
          if (at[q] < loads) v[q] = load(at[q]);
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
          if (at[q] < loads) look(v[q], at[q]);
        }
      }
    };
    // The batches that have the picked threads' largest elements; of the threads that have such elements elsewhere too, the rest.
    look_through(num_picked * kBatch, [&](int i) { return sh.best_at[sh.picked[i / kBatch]] + i % kBatch * 32; });
    for (int i = 0; i < num_picked; ++i) {
      const int thread = sh.picked[i], seen = sh.best_at[thread] / kUnit;
      if (sh.second[thread] < bound) continue;
      look_through(units_each * kBatch, [&](int j) { return thread / 32 + j / kBatch * kWarps == seen ? loads : load_of(thread, j); });
    }
    __syncthreads();
    // In order: an entry's place is the number of entries above it.
    const int found = sh.num_found;
    if (found <= kCandidates) {
      for (int i = tid; i < found; i += kThreads) {
        const std::uint64_t e = sh.found[i];
        int larger = 0;
        for (int j = 0; j < found; ++j) larger += sh.found[j] > e;
        if (larger < a.top) put_one(larger, e);
      }
      for (int i = found + tid; i < a.top; i += kThreads) put_one(i, 0);
    } else if (warp == 0) {
      // More than fit (a few threads that have hundreds of large values each): one alternative after the other, a pass over the run for each.
      std::uint64_t last_one = ~0ull;
      for (int k = 0; k < a.top; ++k) {
        std::uint64_t best = edge_entry < last_one ? edge_entry : 0;
#pragma unroll 4
        for (int at = lane; at < loads; at += 32) {
          const Chunk<T> v = load(at);
          float l[n];
          v.get(l);
#pragma unroll
          for (int e = 0; e < n; ++e) {
            const std::uint64_t one = entry(order_of<T>(l[e]), static_cast<std::uint32_t>(first_token + at * n + e));
            if (one < last_one && one > best) best = one;
          }
        }
        for (int m = 16; m > 0; m /= 2) best = max(best, static_cast<std::uint64_t>(__shfl_xor_sync(kAll, static_cast<unsigned long long>(best), m)));
        last_one = best;
        if (lane == 0) put_one(k, best);
      }
    }
  }
  if (ctas > 1) {
    cluster_sync_all();
    if (rank == 0 && warp == 0) {
      Sums row_sums = lane < ctas ? sh.sums[lane] : Sums{-INFINITY, 0.f, 0.f};
      row_sums.join_lanes(kMostCluster, c);
      row_sums.ref = __shfl_sync(kAll, row_sums.ref, 0), row_sums.s = __shfl_sync(kAll, row_sums.s, 0), row_sums.w = __shfl_sync(kAll, row_sums.w, 0);
      unsigned row_before = lane < ctas ? sh.before[lane] : 0u;
      for (int m = kMostCluster / 2; m > 0; m /= 2) row_before += __shfl_xor_sync(kAll, row_before, m);
      const RowOutputs<T> put(a, row, row_sums);
      if (lane == 0) put.row(target64, mine, row_before);
      if (a.top > 0) {
        unsigned long long e[kMostCluster];
#pragma unroll
        for (int i = 0; i < kMostCluster; ++i) e[i] = i < ctas && lane < a.top ? sh.first[i * kMostTop + lane] : 0ull;
#pragma unroll
        for (int m = 1; m < kMostCluster; m *= 2) {
#pragma unroll
          for (int i = 0; i < kMostCluster; i += 2 * m) {
            if (i + m < ctas) e[i] = merged(e[i], e[i + m], lane);
          }
        }
        if (lane < a.top) put.token(lane, e[0]);
      }
    }
  }
  if (lost) {  // give the copies on their way time to land
    if (lane == 0) atomicOr(a.status, kPagedWait);
    const std::uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) {
    }
  }
}

template <typename T, bool kLong>
int launch(const char* op, LogprobArgs a, cudaStream_t stream) {
  using S = Shape<kLong>;
  static std::atomic<std::uint64_t> done{0};
  if (const int s = allow_shared(op, logprobs_kernel<T, kLong>, S::kRing, done); s != B2_OK) return s;
  // CTAs to a row: as many as the GPU has room for, each with two loads a thread at least.
  while (a.ctas < kMostCluster && a.rows * a.ctas * 2 <= static_cast<std::int64_t>(S::kPerSm) * sm_count() && a.vocab / kChunk<T> >= a.ctas * 4 * kThreads) a.ctas *= 2;
  return enqueue(op, logprobs_kernel<T, kLong>, dim3(static_cast<unsigned>(a.rows * a.ctas)), dim3(kThreads), S::kRing, stream, a.ctas, a);
}
template <typename T>
int launch(const char* op, const LogprobArgs& a, cudaStream_t stream) {
  return a.vocab / kChunk<T> > 64 * kThreads ? launch<T, true>(op, a, stream) : launch<T, false>(op, a, stream);
}

}  // namespace
}  // namespace b2

extern "C" int b2_token_logprobs(const b2_logprobs* p, void* stream) {
  using namespace b2;
  const char* const op = "token_logprobs";
  if (p == nullptr || p->struct_size != sizeof(b2_logprobs)) return fail_invalid(op, "struct_size does not match");
  if (!dtype_known(p->dtype)) return fail_invalid(op, "dtype is not a type that this call takes");
  if (p->rows < 0 || p->rows >= (1LL << 31)) return fail_invalid(op, "rows must be from 0 to 2^31 - 1");
  if (p->vocab <= 0 || p->vocab > (1 << 30)) return fail_invalid(op, "vocab must be from 1 to 2^30");
  if (p->top < 0 || p->top > kMostTop || p->top > p->vocab) return fail_invalid(op, "top must be from 0 to 32 and at most vocab");
  if (!(p->scale > 0.0f) || p->scale > 1e30f) return fail_invalid(op, "scale must be above 0 and at most 1e30");
  if (p->rows == 0) return B2_OK;
  if (p->logits == nullptr || !aligned_to(p->logits, static_cast<std::uintptr_t>(dtype_bytes(p->dtype))) || p->ld < p->vocab)
    return fail_invalid(op, "logits must be rows of at least vocab elements");
  if (p->top > 0 && (p->top_logprobs == nullptr || p->top_tokens == nullptr)) return fail_invalid(op, "top_logprobs and top_tokens are missing");
  const void* const fours[] = {p->logprobs, p->ranks, p->entropy, p->lse, p->top_logprobs, p->top_tokens};
  for (const void* q : fours) {
    if (!aligned_to(q, 4)) return fail_invalid(op, "an output is not aligned");
  }
  if (!aligned_to(p->targets, 8)) return fail_invalid(op, "targets must be 8-byte aligned");
  PagedArgs status{};
  if (const int s = paged_status_word(op, &status); s != B2_OK) return s;
  const LogprobArgs a{p->logits, p->ld, p->targets, p->logprobs, p->ranks, p->entropy, p->lse, p->top_logprobs, p->top_tokens, p->rows, status.status,
                      p->scale, p->scale * 1.4426950408889634f, p->vocab, p->top, 1};
  const cudaStream_t s = as_stream(stream);
  if (p->dtype == B2_DTYPE_F32) return launch<float>(op, a, s);
  return p->dtype == B2_DTYPE_F16 ? launch<__half>(op, a, s) : launch<__nv_bfloat16>(op, a, s);
}
