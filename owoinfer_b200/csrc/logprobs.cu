// Log probabilities of given tokens under a row of logits, with rank, entropy and the most probable alternatives, in one pass over the logits.
#include <algorithm>
#include <cmath>

#include "attention.cuh"
#include "text.cuh"

namespace b2 {
namespace {

constexpr int kThreads = 512;
constexpr int kMostTop = 32;
constexpr int kMostCluster = 8;
constexpr int kCandidates = 1024;  // elements at or above the bound that are sorted
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
  float scale, scale_log2;  // scale * log2(e)
  int vocab, top, ctas;
};

__device__ __forceinline__ void st_cluster_u64(std::uint32_t cluster_addr, std::uint64_t x) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_addr), "l"(x) : "memory");
}

// The order of values as unsigned numbers, 1 for NaN, 0 for none: of a value as fp32 the bits that tell the values of T apart.
template <typename T>
constexpr int kOrderBits = std::is_same<T, float>::value ? 32 : std::is_same<T, __half>::value ? 19 : 16;
template <typename T>
__device__ __forceinline__ std::uint32_t order_of(float x) {
  const std::uint32_t u = __float_as_uint(x + 0.0f);  // (-0 is 0)
  const std::uint32_t order = (static_cast<std::int32_t>(u) < 0 ? ~u : u | 0x80000000u) >> (32 - kOrderBits<T>);
  return isnan(x) ? 1u : order;
}
template <typename T>
__device__ __forceinline__ float value_of(std::uint32_t order) {
  if (order == 1u) return __int_as_float(0x7fc00000);
  constexpr int kDrop = 32 - kOrderBits<T>;
  const std::uint32_t u = order << kDrop;
  return __uint_as_float((u & 0x80000000u) != 0u ? u & 0x7fffffffu : ~(u | ((1u << kDrop) - 1u)));
}

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
__device__ __forceinline__ float top_of(const Chunk<float>& c) {
  return fmaxf(fmaxf(__uint_as_float(c.raw.x), __uint_as_float(c.raw.y)), fmaxf(__uint_as_float(c.raw.z), __uint_as_float(c.raw.w)));
}
__device__ __forceinline__ float top_of(const Chunk<__nv_bfloat16>& c) {
  const auto h = [](std::uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
  const __nv_bfloat162 m = __hmax2(__hmax2(h(c.raw.x), h(c.raw.y)), __hmax2(h(c.raw.z), h(c.raw.w)));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float top_of(const Chunk<__half>& c) {
  const auto h = [](std::uint32_t w) { return *reinterpret_cast<const __half2*>(&w); };
  const __half2 m = __hmax2(__hmax2(h(c.raw.x), h(c.raw.y)), __hmax2(h(c.raw.z), h(c.raw.w)));
  return fmaxf(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sums over part of a row against a reference `ref` near its largest logit: s = sum 2^x, w = sum x 2^x with x = (l - ref) scale log2(e).
// The reference is the largest of what came first and follows once something is kAhead binades above it.
struct Sums {
  static constexpr float kAhead = 8.f;
  float ref, s, w;  // (-infinity, 0, 0: nothing)
  __device__ __forceinline__ void rise(float top, float c) {
    if (!(top > ref) || (ref > -INFINITY && (top - ref) * c <= kAhead)) return;
    *this = moved(top, c);
  }
  __device__ __forceinline__ Sums moved(float to, float c) const {
    Sums r{to, 0.f, 0.f};
    if (s != 0.f) {  // (nothing, or only what weighs nothing, so far: nothing to scale, and -infinity times 0 to avoid)
      const float d = (ref - to) * c, f = ex2(d);
      r.s = s * f;
      r.w = f == 0.f ? 0.f : f * fmaf(d, s, w);
    }
    return r;
  }
  // The elements of one load. What is 2^-200 and less of the reference is 2^-200: 0 in fp32, and times x no NaN.
  template <int n>
  __device__ __forceinline__ void add(const float (&l)[n], float c) {
    const float from = ref > -INFINITY ? ref : 0.f;
    const std::uint64_t minus = pack2(-from, -from), cc = pack2(c, c);
    std::uint64_t s2 = pack2(0.f, 0.f), w2 = s2;
#pragma unroll
    for (int i = 0; i < n; i += 2) {
      float x, y;
      unpack2(mul2(add2(pack2(l[i], l[i + 1]), minus), cc), x, y);
      x = max_nan(x, -200.f), y = max_nan(y, -200.f);
      const std::uint64_t e = pack2(ex2(x), ex2(y));
      s2 = add2(s2, e), w2 = fma2(e, pack2(x, y), w2);
    }
    float a, b;
    unpack2(s2, a, b);
    s += a + b;
    unpack2(w2, a, b);
    w += a + b;
  }
  __device__ __forceinline__ void join(const Sums& o, float c) {
    const float to = fmaxf(ref, o.ref);
    const Sums p = moved(to, c), q = o.moved(to, c);
    ref = to, s = p.s + q.s, w = p.w + q.w;
  }
};

struct Shared {
  std::uint32_t best[kThreads];  // order of a thread's largest element, then that of where it stands
  std::uint32_t place[kThreads];
  std::uint64_t found[kCandidates];
  std::uint64_t first[kMostCluster * kMostTop];  // of each CTA of the cluster: its first `top`, in order (in the first CTA)
  Sums sums[kMostCluster];
  int before[kMostCluster];
  Sums warp_sums[kThreads / 32];
  int warp_before[kThreads / 32];
  int picked[kMostPicked];
  int num_picked, num_found;
  std::uint32_t bound, above, ties, place_bound;
  std::uint64_t last;
};

// The largest bound (of `bits` bits) that at least `count` of the keys reach; a whole warp. 0 where fewer than `count` keys are above 0.
template <int kPer>
__device__ __forceinline__ std::uint32_t bound_of(const std::uint32_t (&key)[kPer], int bits, int count) {
  std::uint32_t bound = 0;
  for (int bit = bits - 1; bit >= 0; --bit) {
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

// A cluster of CTAs per row, each with a run of it; one pass over the logits. Every thread keeps its sums against its own reference, how many of its
// elements come before the target, and its largest element. The alternatives come from what the threads saw: the `top`-th largest of their
// largest elements is a bound that `top` elements reach, so that only the threads whose largest one reaches it can hold one of the first `top`:
// their elements are read once more (top / 512 of the row, from L2), and those at or above the bound sorted by counting.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) logprobs_kernel(const LogprobArgs a) {
  constexpr int n = kChunk<T>, kBatch = 4;
  __shared__ __align__(16) Shared sh;
  const int ctas = a.ctas, rank = static_cast<int>(blockIdx.x % static_cast<unsigned>(ctas));
  const std::int64_t row = blockIdx.x / static_cast<unsigned>(ctas);
  const int tid = static_cast<int>(threadIdx.x);
  if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // (the others are there: waited for ahead of the first store to one)
  const T* const logits = static_cast<const T*>(a.logits) + row * a.ld;
  const float c = a.scale_log2;

  // The row as `head` elements up to the first 16-byte boundary, whole loads, and the rest.
  const int head = min(a.vocab, static_cast<int>((16u - (reinterpret_cast<std::uintptr_t>(logits) & 15u)) % 16u / sizeof(T)));
  const int chunks = (a.vocab - head) / n, edges = a.vocab - chunks * n;
  const T* const body = logits + head;
  const int per_cta = (chunks + ctas - 1) / ctas, begin = min(rank * per_cta, chunks), end = min(begin + per_cta, chunks);

  const std::int64_t target64 = a.targets != nullptr ? a.targets[row] : -1;
  const bool has_target = target64 >= 0 && target64 < a.vocab;
  const int target = has_target ? static_cast<int>(target64) : -1;
  const float mine = has_target ? to_float(logits[target]) : 0.f;
  const bool mine_nan = isnan(mine);
  const auto is_before = [&](float l, int token) { return l > mine || (l == mine && token < target) || (mine_nan && (!isnan(l) || token < target)); };

  Sums sums{-INFINITY, 0.f, 0.f};
  int before = 0;
  std::uint32_t best = 0;
  int best_at = -1;  // the load that has it first, relative to `begin`, or the first of a batch
  const auto see = [&](const Chunk<T>(&v)[kBatch], int first, int count) {  // loads first, first + kThreads, ...
    float top = top_of(v[0]);
#pragma unroll
    for (int u = 1; u < kBatch; ++u) {
      if (u < count) top = fmaxf(top, top_of(v[u]));
    }
    sums.rise(top, c);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (u >= count) continue;
      float l[n];
      v[u].get(l);
      sums.add(l, c);
    }
    if (has_target && (top >= mine || mine_nan)) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (u >= count) continue;
        float l[n];
        v[u].get(l);
#pragma unroll
        for (int i = 0; i < n; ++i) before += is_before(l[i], head + (first + u * kThreads) * n + i);
      }
    }
    const std::uint32_t order = order_of<T>(top);
    if (order > best) best = order, best_at = first - begin;
  };
  int at = begin + tid;
  for (; at + (kBatch - 1) * kThreads < end; at += kBatch * kThreads) {
    Chunk<T> v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) v[u].load(body + static_cast<std::int64_t>(at + u * kThreads) * n);
    see(v, at, kBatch);
  }
  if (at < end) {
    Chunk<T> v[kBatch];
    const int left = (end - at + kThreads - 1) / kThreads;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      v[u].raw = make_uint4(0, 0, 0, 0);
      if (u < left) v[u].load(body + static_cast<std::int64_t>(at + u * kThreads) * n);
    }
    see(v, at, left);
  }
  // The elements outside whole loads, one to a thread of the first CTA.
  const int edge_token = tid < head ? tid : head + chunks * n + tid - head;
  const bool has_edge = rank == 0 && tid < edges;
  const float edge = has_edge ? to_float(logits[edge_token]) : 0.f;
  if (has_edge) {
    const float l[2] = {edge, -INFINITY};
    sums.rise(edge, c);
    sums.add(l, c);
    if (has_target) before += is_before(edge, edge_token);
  }

  // The CTA's sums.
#pragma unroll
  for (int m = 16; m > 0; m /= 2) {
    Sums o;
    o.ref = __shfl_xor_sync(0xffffffffu, sums.ref, m), o.s = __shfl_xor_sync(0xffffffffu, sums.s, m), o.w = __shfl_xor_sync(0xffffffffu, sums.w, m);
    sums.join(o, c);
  }
  before = static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(before)));
  if (tid % 32 == 0) sh.warp_sums[tid / 32] = sums, sh.warp_before[tid / 32] = before;
  sh.best[tid] = best;
  if (tid == 0) sh.num_picked = 0, sh.num_found = 0;
  __syncthreads();
  if (ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");

  if (a.top > 0) {
    if (tid < 32) {
      std::uint32_t key[kThreads / 32];
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) key[i] = sh.best[tid + 32 * i];
      const std::uint32_t bound = bound_of(key, kOrderBits<T>, a.top);
      unsigned above = 0, ties = 0;
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) above += key[i] > bound, ties += bound > 0u && key[i] == bound;
      above = __reduce_add_sync(0xffffffffu, above), ties = __reduce_add_sync(0xffffffffu, ties);
      if (tid == 0) sh.bound = bound, sh.above = above, sh.ties = ties;
    }
    __syncthreads();
    const std::uint32_t bound = sh.bound;
    // Where many threads' largest elements equal the bound (a mask that leaves fewer than `top` tokens, a constant row), only the first
    // places can hold an alternative: the bound on places is that of as many loads as are wanted.
    std::uint32_t place_bound = 0xffffffffu, place = 0;
    if (sh.above + sh.ties > kMostPicked) {
      if (best == bound && best_at >= 0) {
        for (int u = kBatch - 1; u >= 0; --u) {  // the first load of the batch that has it
          const int at = begin + best_at + u * kThreads;
          if (at >= end) continue;
          Chunk<T> v;
          v.load(body + static_cast<std::int64_t>(at) * n);
          if (order_of<T>(top_of(v)) == bound) place = static_cast<std::uint32_t>(at - begin);
        }
        place = 0x7fffffffu - place;
      }
      sh.place[tid] = place;
      __syncthreads();
      if (tid < 32) {
        std::uint32_t key[kThreads / 32];
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) key[i] = sh.place[tid + 32 * i];
        const std::uint32_t b = bound_of(key, 31, a.top - static_cast<int>(sh.above));
        if (tid == 0) sh.place_bound = b == 0u ? 0xffffffffu : 0x7fffffffu - b;
      }
      __syncthreads();
      place_bound = sh.place_bound;
    }
    const bool picked = best_at >= 0 && (best > bound || (best == bound && (place_bound == 0xffffffffu || 0x7fffffffu - place <= place_bound)));
    if (picked) {
      const int i = atomicAdd(&sh.num_picked, 1);
      sh.picked[i] = tid;  // (at most kMostPicked, or `top` by the bound on places)
    }
    const auto push = [&](std::uint64_t e) {
      const int i = atomicAdd(&sh.num_found, 1);
      if (i < kCandidates) sh.found[i] = e;
    };
    if (has_edge) push(entry(order_of<T>(edge), static_cast<std::uint32_t>(edge_token)));
    __syncthreads();
    const int threads = sh.num_picked, loads = (end - begin + kThreads - 1) / kThreads;
    for (int i = tid; i < threads * loads; i += kThreads) {
      const int at = begin + sh.picked[i % threads] + i / threads * kThreads;
      if (at >= end) continue;
      Chunk<T> v;
      v.load(body + static_cast<std::int64_t>(at) * n);
      const std::uint32_t order = order_of<T>(top_of(v));
      if (order < bound || (order == bound && static_cast<std::uint32_t>(at - begin) > place_bound)) continue;
      float l[n];
      v.get(l);
#pragma unroll
      for (int e = 0; e < n; ++e) {
        const std::uint32_t o = order_of<T>(l[e]);
        if (o > bound || (o == bound && static_cast<std::uint32_t>(at - begin) <= place_bound)) push(entry(o, static_cast<std::uint32_t>(head + at * n + e)));
      }
    }
    __syncthreads();
    // In order, to the first CTA: an entry's place is the number of entries above it.
    const std::uint32_t to = map_to_cta(smem_u32(sh.first + rank * kMostTop), 0);
    const int found = sh.num_found;
    if (found <= kCandidates) {
      for (int i = tid; i < found; i += kThreads) {
        const std::uint64_t e = sh.found[i];
        int larger = 0;
        for (int j = 0; j < found; ++j) larger += sh.found[j] > e;
        if (larger < a.top) st_cluster_u64(to + larger * 8, e);
      }
      for (int i = found + tid; i < a.top; i += kThreads) st_cluster_u64(to + i * 8, 0);
    } else {
      // More than fit (hundreds of threads that share a few large values in turn): one alternative after the other, a pass over the CTA's run for each.
      std::uint64_t last = ~0ull;
      for (int k = 0; k < a.top; ++k) {
        std::uint64_t next = 0;
        const auto look = [&](std::uint64_t e) {
          if (e < last && e > next) next = e;
        };
        for (int at = begin + tid; at < end; at += kThreads) {
          Chunk<T> v;
          v.load(body + static_cast<std::int64_t>(at) * n);
          float l[n];
          v.get(l);
#pragma unroll
          for (int e = 0; e < n; ++e) look(entry(order_of<T>(l[e]), static_cast<std::uint32_t>(head + at * n + e)));
        }
        if (has_edge) look(entry(order_of<T>(edge), static_cast<std::uint32_t>(edge_token)));
        __syncthreads();  // (the last round's is read)
        if (tid == 0) sh.last = 0;
        __syncthreads();
        atomicMax(reinterpret_cast<unsigned long long*>(&sh.last), static_cast<unsigned long long>(next));
        __syncthreads();
        last = sh.last;
        if (tid == 0) st_cluster_u64(to + k * 8, last);
      }
    }
  }
  if (tid == 0) {
    Sums all = sh.warp_sums[0];
    int b = sh.warp_before[0];
    for (int i = 1; i < kThreads / 32; ++i) all.join(sh.warp_sums[i], c), b += sh.warp_before[i];
    const std::uint32_t at = map_to_cta(smem_u32(sh.sums + rank), 0);
    st_cluster_u32(at, __float_as_uint(all.ref)), st_cluster_u32(at + 4, __float_as_uint(all.s)), st_cluster_u32(at + 8, __float_as_uint(all.w));
    st_cluster_u32(map_to_cta(smem_u32(sh.before + rank), 0), static_cast<std::uint32_t>(b));
  }
  if (ctas > 1) cluster_sync_all();
  else __syncthreads();
  if (rank != 0) return;

  Sums all = sh.sums[0];
  int b = sh.before[0];
  for (int i = 1; i < ctas; ++i) all.join(sh.sums[i], c), b += sh.before[i];
  const float log_s = logf(all.s);
  const bool nothing = all.ref == -INFINITY && !isnan(all.s);
  const float nan = __int_as_float(0x7fc00000);
  const auto logprob = [&](float l) { return nothing ? -INFINITY : isnan(all.s) ? nan : (l - all.ref) * a.scale - log_s; };
  if (tid == 0) {
    if (a.lse != nullptr) a.lse[row] = nothing ? -INFINITY : fmaf(all.ref, a.scale, log_s);
    if (a.entropy != nullptr) {
      const float h = log_s - all.w / all.s * 0.6931471805599453f;
      a.entropy[row] = nothing || h < 0.f ? 0.f : h;
    }
    if (a.logprobs != nullptr) a.logprobs[row] = has_target ? logprob(mine) : target64 < 0 ? 0.f : nan;
    if (a.ranks != nullptr) a.ranks[row] = has_target ? b + 1 : 0;
  }
  if (a.top > 0) {
    for (int i = tid; i < ctas * a.top; i += kThreads) {
      const std::uint64_t e = sh.first[i / a.top * kMostTop + i % a.top];
      int larger = 0;
      for (int j = 0; j < ctas * a.top; ++j) larger += sh.first[j / a.top * kMostTop + j % a.top] > e;
      if (larger >= a.top || e == 0) continue;
      const std::uint32_t token = 0xFFFFFFFFu - static_cast<std::uint32_t>(e);
      a.top_tokens[row * a.top + larger] = static_cast<std::int32_t>(token);
      a.top_logprobs[row * a.top + larger] = logprob(value_of<T>(static_cast<std::uint32_t>(e >> 32)));
    }
  }
}

template <typename T>
int launch(const char* op, LogprobArgs a, std::int64_t rows, cudaStream_t stream) {
  // CTAs to a row: as many as the GPU has room for (two of 512 threads to an SM), each with two loads a thread at least.
  a.ctas = 1;
  while (a.ctas < kMostCluster && rows * a.ctas * 2 <= 2 * sm_count() && a.vocab / kChunk<T> >= a.ctas * 2 * 2 * kThreads) a.ctas *= 2;
  return enqueue(op, logprobs_kernel<T>, dim3(static_cast<unsigned>(rows * a.ctas)), dim3(kThreads), 0, stream, a.ctas, a);
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
  const LogprobArgs a{p->logits, p->ld, p->targets, p->logprobs, p->ranks, p->entropy, p->lse, p->top_logprobs, p->top_tokens,
                      p->scale, p->scale * 1.4426950408889634f, p->vocab, p->top, 1};
  const cudaStream_t s = as_stream(stream);
  if (p->dtype == B2_DTYPE_F32) return launch<float>(op, a, p->rows, s);
  return p->dtype == B2_DTYPE_F16 ? launch<__half>(op, a, p->rows, s) : launch<__nv_bfloat16>(op, a, p->rows, s);
}
