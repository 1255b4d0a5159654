// Attention of one new token per sequence over a paged key-value cache, split over the cache's length and joined, with the
// attention that each cached slot got added up.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "attention.cuh"
#include "paged.cuh"

namespace b2 {
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kKeys = 16;       // slots of a step of a warp: a page holds a multiple of it
constexpr int kStages = 2;      // steps of a warp in shared memory: the one it works on and the one on its way
constexpr int kRows = 16;       // query heads of a CTA: the rows of an MMA
constexpr int kMostCluster = 8, kClusterSteps = 24;  // CTAs that join their parts in shared memory; steps of each at most
constexpr int kJoinThreads = 256;
constexpr int kJoinSlots = 4, kJoinHeads = 4, kJoinPerSm = 8;
constexpr int kMostGroup = 4096;  // (a float each in shared memory)

struct DecodeArgs {
  PagedArgs c;
  const void* q;
  std::int64_t q_row, q_head;
  void* out;
  std::int64_t o_row, o_head;
  float* lse;
  int q_heads, group;           // query heads; query heads to a key head
  float scale_log2;             // scale * log2(e)
  int window, sinks;            // window 0: none
  int chunk, splits;            // steps of a CTA; CTAs to a (sequence, key head) at most
  float2* part_ml;              // [batch, q_heads, splits] maximum and sum of a part
  float* part_o;                // [batch, q_heads, splits, D]
  float* scores;                // [batch, q_heads, scores_ld] scaled scores in binades, or NULL
  std::int64_t scores_ld;
  const float* weights;
  float* weights_out;
  std::int64_t weights_ld;
};

// The steps of kKeys slots that the newest of `len` tokens sees some slot of: first the sinks', then from `from` on.
struct Steps {
  int sinks, from, count;
  __device__ __forceinline__ Steps(const DecodeArgs& a, int len) {
    const int all = (len + kKeys - 1) / kKeys;
    from = a.window > 0 && len > a.window ? (len - a.window) / kKeys : 0;
    sinks = min((min(a.sinks, len) + kKeys - 1) / kKeys, from);
    count = sinks + all - from;
  }
  __device__ __forceinline__ int slot(int i) const { return (i < sinks ? i : i - sinks + from) * kKeys; }
};
__device__ __forceinline__ bool sees(const DecodeArgs& a, int len, int slot) {
  return slot < len && (a.window == 0 || slot < a.sinks || slot >= len - a.window);
}

__device__ __forceinline__ void ldsm4(std::uint32_t addr, std::uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(std::uint32_t addr, std::uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ float2 ld_cluster_f32x2(std::uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(std::uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], const std::uint32_t (&a)[4], std::uint32_t b0, std::uint32_t b1);
template <>
__device__ __forceinline__ void mma16<__nv_bfloat16>(float (&d)[4], const std::uint32_t (&a)[4], std::uint32_t b0, std::uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16<__half>(float (&d)[4], const std::uint32_t (&a)[4], std::uint32_t b0, std::uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The reference of a row's exponentials is its first step's maximum less kShift binades, moved up once a score is kRaise binades above that
// maximum. bf16 has fp32's range: P keeps its relative precision however large it is. fp16 ends at 2^16 and loses bits below 2^-14, P in two
// parts below 2^-25 all of it: the largest of P is kept from 2^13 to 2^15, so that weights are held to 2^-38 of the largest. (From 1 to
// 2^8, weights of 2^-18 lost a hundredth, and of 2^-25 everything.)
template <typename T>
struct Reference {
  static constexpr bool kHalf = std::is_same<T, __half>::value;
  static constexpr float kShift = kHalf ? 13.0f : 0.0f, kRaise = kHalf ? 2.0f : 8.0f;
};

// Four channels of an output in which something is not finite: where the token sees infinities or NaN of V in steps [begin, end), they are
// the output, whatever their weights. P in two parts makes NaN of them, the second part being 0 or negative.
template <typename T>
__device__ __forceinline__ void take_nonfinite(const DecodeArgs& a, const Steps& steps, int begin, int end, int len, int b, int h, int d, float4& sum) {
  float odd[4] = {};
  unsigned found = 0;
#pragma unroll 1
  for (int i = begin * kKeys; i < end * kKeys; ++i) {
    const int slot = steps.slot(i / kKeys) + i % kKeys;
    const int page = sees(a, len, slot) ? paged_page(a.c, b, slot) : -1;
    if (page < 0) continue;
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.c.v) + paged_row(a.c, page, h, slot) + d);
    float x[4];
    unpack16<T>(v.x, x[0], x[1]);
    unpack16<T>(v.y, x[2], x[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!isfinite(x[e])) odd[e] += x[e], found |= 1u << e;
    }
  }
  if ((found & 1u) != 0u) sum.x = odd[0];
  if ((found & 2u) != 0u) sum.y = odd[1];
  if ((found & 4u) != 0u) sum.z = odd[2];
  if ((found & 8u) != 0u) sum.w = odd[3];
}

// softmax(scale q·K^T)·V of one query row per head: o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s in binades, m a running
// reference. A CTA per (part of the cache, key head and block of 16 query heads, sequence). Its warps work apart: each has TMA
// bring its own steps of 16 slots (whose 16 rows a page holds in one piece) and keeps its own maxima, sums and output rows in
// registers; they meet at the end. Q·K^T and P·V are 16-row MMAs with the group's query heads as rows: the cache is read once
// for all of them. At one byte of cache to every group / 2 multiply-adds the memory bounds it; 128-row tensor tiles would be
// filled to group / 128. 64 sequences of up to 8101 slots, 32 / 8 heads of 128, with weights: 200 us, 6.3 TB/s (the
// call 222); one of 131001, 32 / 4 heads in fp16: 50 us, 5.3 TB/s (59).
template <typename T, int D, bool kScores, bool kCluster>
__global__ void __launch_bounds__(kThreads, 3)
decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const DecodeArgs a) {
  dependents_may_start();
  extern __shared__ std::uint8_t smem_raw[];
  __shared__ __align__(8) std::uint64_t s_full[kWarps][kStages];
  __shared__ int s_abort;
  // A step in shared memory: K, then V, each D / 64 parts of 16 rows of 128 bytes with the 128-byte swizzle.
  constexpr int kParts = D / 64, kPartBytes = kKeys * 128, kHalfBytes = kParts * kPartBytes, kStageBytes = 2 * kHalfBytes;
  const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32;
  const int blocks = (a.group + kRows - 1) / kRows;
  const int split = blockIdx.x, h = blockIdx.y / blocks, g0 = (blockIdx.y % blocks) * kRows, b = blockIdx.z;
  const int rows = min(kRows, a.group - g0), q_head0 = h * a.group + g0;
  if (threadIdx.x == 0) s_abort = 0;
  // Pages of 32 steps at a time, a lane each. Without a window a step's slots do not go by the length, so the first 32 entries of the block
  // table are on their way along with it.
  const std::int32_t* const table = a.c.table + b * a.c.table_ld;
  const int early_slot = (split * a.chunk + warp + lane * kWarps) * kKeys;
  int entry = a.window == 0 && early_slot < a.c.most ? table[early_slot >> a.c.page_shift] : -1;
  const int len = paged_len(a.c, b);
  const Steps steps(a, len);
  const int begin = split * a.chunk, end = min(steps.count, begin + a.chunk);
  // (Part 0 of an empty sequence goes on: it writes the zeros, or the empty part that the join finds. So does all of a cluster.)
  if (!kCluster && begin >= end && split > 0) return;
  const int mine = begin + warp < end ? (end - begin - warp + kWarps - 1) / kWarps : 0;  // this warp's steps
  const auto checked = [&](int page, int i) {
    if (i >= mine) return -1;
    if (page < 0 || page >= a.c.num_pages) {
      atomicOr(a.c.status, kPagedBadPage);
      return -1;
    }
    return page;
  };
  const auto fetch_pages = [&](int n) {
    const int i = n + lane;
    return i < mine ? checked(table[steps.slot(begin + warp + i * kWarps) >> a.c.page_shift], i) : -1;
  };
  int pages = a.window == 0 ? checked(entry, lane) : fetch_pages(0), pages_next = fetch_pages(32);

  std::uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  // In a cluster the scores stay here, [rows][chunk * kKeys], behind the rings.
  float* const own_scores = reinterpret_cast<float*>(smem + kWarps * kStages * kStageBytes);
  const int own_ld = a.chunk * kKeys;
  const std::uint32_t ring = smem_u32(smem) + static_cast<std::uint32_t>(warp) * (kStages * kStageBytes);
  const auto bar = [&](int n) { return smem_u32(&s_full[warp][n % kStages]); };
  if (lane == 0) {  // (a warp's barriers are its own: no other waits for them)
#pragma unroll
    for (int i = 0; i < kStages; ++i) mbar_init(bar(i), 1);
    fence_mbar_init();
  }
  __syncwarp();
  const auto issue = [&](int n) {  // step n of this warp into its stage
    if (n >= mine) return;
    if (n > 0 && n % 32 == 0) {
      pages = pages_next;
      pages_next = fetch_pages(n + 32);
    }
    const int page = __shfl_sync(0xffffffffu, pages, n % 32);
    const std::uint32_t stage = ring + static_cast<std::uint32_t>(n % kStages) * kStageBytes;
    if (page < 0) {  // a page outside the pool reads as zeros
      for (int i = lane; i < kStageBytes / 16; i += 32) st_shared(stage + i * 16, make_uint4(0, 0, 0, 0));
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(n));
    } else if (lane == 0) {
      const int row = steps.slot(begin + warp + n * kWarps) & ((1 << a.c.page_shift) - 1);
      mbar_expect_tx(bar(n), kStageBytes);
#pragma unroll
      for (int i = 0; i < kParts; ++i) {
        tma_load_4d(stage + i * kPartBytes, &map_k, bar(n), i * 64, row, h, page);
        tma_load_4d(stage + kHalfBytes + i * kPartBytes, &map_v, bar(n), i * 64, row, h, page);
      }
    }
  };
#pragma unroll
  for (int n = 0; n < kStages; ++n) issue(n);

  // Q as the A operand: rows lane / 4 and + 8 (zeros past the group), two neighbouring channels to a register.
  std::uint32_t qf[D / 16][4];
  {
    const T* q = static_cast<const T*>(a.q) + b * a.q_row + (lane % 4) * 2;
    const int r0 = lane / 4, r1 = r0 + 8;
    const auto at = [&](int r, int d) { return r < rows ? *reinterpret_cast<const std::uint32_t*>(q + (q_head0 + r) * a.q_head + d) : 0u; };
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      qf[d][0] = at(r0, d * 16), qf[d][1] = at(r1, d * 16);
      qf[d][2] = at(r0, d * 16 + 8), qf[d][3] = at(r1, d * 16 + 8);
    }
  }
  __syncthreads();  // s_abort is cleared before any wait looks at it (the copies and Q are on their way meanwhile)
  float o[D / 8][4] = {};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

  for (int n = 0; n < mine; ++n) {
    const bool got = wait_bar(bar(n), n / kStages & 1u, &s_abort);
    if (__any_sync(0xffffffffu, !got)) break;
    const std::uint32_t k_rows = ring + static_cast<std::uint32_t>(n % kStages) * kStageBytes, v_rows = k_rows + kHalfBytes;
    const int slot0 = steps.slot(begin + warp + n * kWarps);
    const bool all = sees(a, len, slot0) && sees(a, len, slot0 + kKeys - 1) && (a.window == 0 || slot0 + kKeys <= a.sinks || slot0 >= len - a.window);
    if (!all) {  // 0 times what a hidden slot of V holds has to be 0
      for (int i = lane; i < kKeys * kParts * 8; i += 32) {
        if (!sees(a, len, slot0 + i / 8 % kKeys)) st_shared(v_rows + i * 16, make_uint4(0, 0, 0, 0));
      }
      fence_proxy_async_smem();  // (ahead of the TMA that fills the stage next)
      __syncwarp();
    }

    float s[2][4] = {};  // slots 0..7 and 8..15 of the step
    {
      const int r = (lane >> 4) * 8 + lane % 8, half = lane >> 3 & 1;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        std::uint32_t kf[4];
        ldsm4(k_rows + d / 4 * kPartBytes + r * 128 + (((2 * d + half) % 8 ^ (r & 7)) << 4), kf);
        mma16<T>(s[0], qf[d], kf[0], kf[1]);
        mma16<T>(s[1], qf[d], kf[2], kf[3]);
      }
    }
    // In binades; what is not seen is minus infinity.
    const int key = slot0 + (lane % 4) * 2;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[t][i] *= a.scale_log2;
        if (!all && !sees(a, len, key + t * 8 + (i & 1))) s[t][i] = -INFINITY;
      }
    }
    if constexpr (kScores) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = lane / 4 + 8 * i;
        if (r < rows) {
          float* row = kCluster ? own_scores + r * own_ld + (warp + n * kWarps) * kKeys + (lane % 4) * 2
                                : a.scores + (static_cast<std::int64_t>(b) * a.q_heads + q_head0 + r) * a.scores_ld + key;
          *reinterpret_cast<float2*>(row) = make_float2(s[0][2 * i], s[0][2 * i + 1]);
          *reinterpret_cast<float2*>(row + 8) = make_float2(s[1][2 * i], s[1][2 * i + 1]);
        }
      }
    }
    float top[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
    }
    const auto above = [&](int i) { return m[i] == -INFINITY ? top[i] > -INFINITY : top[i] > m[i] + (Reference<T>::kShift + Reference<T>::kRaise); };
    if (__any_sync(0xffffffffu, above(0) || above(1))) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!above(i)) continue;
        const float to = top[i] - Reference<T>::kShift, grow = ex2(m[i] - to);  // 0 the first time
        m[i] = to, l[i] *= grow;
#pragma unroll
        for (int d = 0; d < D / 8; ++d) o[d][2 * i] *= grow, o[d][2 * i + 1] *= grow;
      }
    }
    float p[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ref = m[i >> 1];
        p[t][i] = ref == -INFINITY && s[t][i] == -INFINITY ? 0.f : ex2(s[t][i] - ref);
        l[i >> 1] += p[t][i];
      }
    }
    // P for the tensor core. What its rounding to 8 (11) bits leaves goes in as a second operand: P·V is then as exact as the values
    // are, for 16 more MMAs in a kernel that waits for memory.
    std::uint32_t hi[4], lo[4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = p[t][2 * i], y = p[t][2 * i + 1];
        hi[2 * t + i] = pack16<T>(x, y);
        float xh, yh;
        unpack16<T>(hi[2 * t + i], xh, yh);
        lo[2 * t + i] = pack16<T>(x - xh, y - yh);
      }
    }
    const int r = (lane >> 3 & 1) * 8 + lane % 8, half = lane >> 4;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      std::uint32_t vf[4];
      ldsm4_trans(v_rows + d / 4 * kPartBytes + r * 128 + (((2 * d + half) % 8 ^ (r & 7)) << 4), vf);
      mma16<T>(o[2 * d], hi, vf[0], vf[1]);
      mma16<T>(o[2 * d + 1], hi, vf[2], vf[3]);
      mma16<T>(o[2 * d], lo, vf[0], vf[1]);
      mma16<T>(o[2 * d + 1], lo, vf[2], vf[3]);
    }
    __syncwarp();  // the stage is read
    issue(n + kStages);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
  }

  // The warps' parts meet in the rings' place.
  __syncthreads();
  if (s_abort != 0) {  // a wait expired: give the copies on their way time to land
    if (threadIdx.x == 0) atomicOr(a.c.status, kPagedWait);
    const std::uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) {
    }
    if constexpr (!kCluster) return;
  }
  float* s_o = reinterpret_cast<float*>(smem);           // [kWarps][kRows][D + 4]
  constexpr int kLd = D + 4;
  float* s_ml = s_o + kWarps * kRows * kLd;              // [kWarps][kRows][2]
  float* s_part = s_ml + kWarps * kRows * 2;             // [kRows][2] of this CTA
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = warp * kRows + lane / 4 + 8 * i;
    if (lane % 4 == 0) s_ml[2 * row] = m[i], s_ml[2 * row + 1] = l[i];
#pragma unroll
    for (int d = 0; d < D / 8; ++d) *reinterpret_cast<float2*>(s_o + row * kLd + d * 8 + (lane % 4) * 2) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
  }
  __syncthreads();
  constexpr int kQuads = D / 4;
  for (int at = threadIdx.x; at < rows * kQuads; at += kThreads) {
    const int row = at / kQuads, d = (at % kQuads) * 4;
    float mm = -INFINITY, ll = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_ml[2 * (w * kRows + row)]);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float lw = s_ml[2 * (w * kRows + row) + 1];
      const float f = lw == 0.f ? 0.f : ex2(s_ml[2 * (w * kRows + row)] - mm);  // (a warp that saw nothing has nothing to add)
      const float4 x = *reinterpret_cast<const float4*>(s_o + (w * kRows + row) * kLd + d);
      ll = fmaf(f, lw, ll);
      sum.x = fmaf(f, x.x, sum.x), sum.y = fmaf(f, x.y, sum.y), sum.z = fmaf(f, x.z, sum.z), sum.w = fmaf(f, x.w, sum.w);
    }
    if (__builtin_expect(!isfinite(sum.x + sum.y + sum.z + sum.w), 0)) {
      if (ll == 0.f) sum = make_float4(0.f, 0.f, 0.f, 0.f);  // every score minus infinity
      else take_nonfinite<T>(a, steps, begin, end, len, b, h, d, sum);
    }
    const std::int64_t head = static_cast<std::int64_t>(b) * a.q_heads + q_head0 + row;
    if constexpr (kCluster) {
      *reinterpret_cast<float4*>(s_o + row * kLd + d) = sum;  // (in the place of warp 0's, which only this thread reads)
      if (d == 0) s_part[2 * row] = mm, s_part[2 * row + 1] = ll;
    } else if (a.part_o == nullptr) {
      const float inv = ll == 0.f ? 0.f : 1.0f / ll;
      T* out = static_cast<T*>(a.out) + b * a.o_row + (q_head0 + row) * a.o_head + d;
      *reinterpret_cast<uint2*>(out) = make_uint2(pack16<T>(sum.x * inv, sum.y * inv), pack16<T>(sum.z * inv, sum.w * inv));
      if (d == 0 && a.lse != nullptr) a.lse[head] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * 0.6931471805599453f;
    } else {
      *reinterpret_cast<float4*>(a.part_o + (head * a.splits + split) * D + d) = sum;
      if (d == 0) a.part_ml[head * a.splits + split] = make_float2(mm, ll);
    }
  }
  if constexpr (kCluster) {
    // The parts are the cluster's CTAs: each joins some of the output, and adds up what its own slots got.
    __shared__ float s_lse[kRows];
    cluster_sync_all();
    const auto all_parts = [&](int row, float2(&ml)[kMostCluster]) {
#pragma unroll
      for (int i = 0; i < kMostCluster; ++i) ml[i] = i < a.splits ? ld_cluster_f32x2(map_to_cta(smem_u32(s_part + 2 * row), static_cast<std::uint32_t>(i))) : make_float2(-INFINITY, 0.f);
    };
    const auto sum_of = [&](const float2(&ml)[kMostCluster], float& mm, float& ll) {
      mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int i = 0; i < kMostCluster; ++i) mm = fmaxf(mm, ml[i].x);
#pragma unroll
      for (int i = 0; i < kMostCluster; ++i) ll += ml[i].y == 0.f ? 0.f : ml[i].y * ex2(ml[i].x - mm);
    };
    for (int at = split * kThreads + static_cast<int>(threadIdx.x); at < rows * kQuads; at += a.splits * kThreads) {
      const int row = at / kQuads, d = (at % kQuads) * 4;
      float2 ml[kMostCluster];
      float4 x[kMostCluster];
      all_parts(row, ml);
#pragma unroll
      for (int i = 0; i < kMostCluster; ++i) {
        if (i < a.splits) x[i] = ld_cluster_f32x4(map_to_cta(smem_u32(s_o + row * kLd + d), static_cast<std::uint32_t>(i)));
      }
      float mm, ll;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      sum_of(ml, mm, ll);
#pragma unroll
      for (int i = 0; i < kMostCluster; ++i) {
        if (ml[i].y == 0.f) continue;
        const float f = ex2(ml[i].x - mm);
        sum.x = joined(f, x[i].x, 1.f, sum.x), sum.y = joined(f, x[i].y, 1.f, sum.y), sum.z = joined(f, x[i].z, 1.f, sum.z), sum.w = joined(f, x[i].w, 1.f, sum.w);
      }
      const float inv = ll == 0.f ? 0.f : 1.0f / ll;
      T* out = static_cast<T*>(a.out) + b * a.o_row + (q_head0 + row) * a.o_head + d;
      *reinterpret_cast<uint2*>(out) = make_uint2(pack16<T>(sum.x * inv, sum.y * inv), pack16<T>(sum.z * inv, sum.w * inv));
      if (d == 0 && a.lse != nullptr) a.lse[static_cast<std::int64_t>(b) * a.q_heads + q_head0 + row] = ll == 0.f ? -INFINITY : (mm + log2f(ll)) * 0.6931471805599453f;
    }
    if constexpr (kScores) {
      if (static_cast<int>(threadIdx.x) < rows) {
        float2 ml[kMostCluster];
        float mm, ll;
        all_parts(static_cast<int>(threadIdx.x), ml);
        sum_of(ml, mm, ll);
        s_lse[threadIdx.x] = ll == 0.f ? INFINITY : mm + log2f(ll);
      }
      __syncthreads();
      const std::int64_t at = (static_cast<std::int64_t>(b) * a.c.kv_heads + h) * a.weights_ld;
      for (int i = threadIdx.x; i < (end - begin) * kKeys; i += kThreads) {
        const int slot = steps.slot(begin + i / kKeys) + i % kKeys;
        if (slot >= len) continue;
        float got = 0.f;
        if (sees(a, len, slot)) {
          for (int g = 0; g < rows; ++g) got += ex2(own_scores[g * own_ld + i] - s_lse[g]);
        }
        a.weights_out[at + slot] = (slot < len - 1 ? a.weights[at + slot] : 0.f) + got;
      }
      // Slots of steps that the window hides.
      for (int slot = steps.sinks * kKeys + split * kThreads + static_cast<int>(threadIdx.x); slot < steps.from * kKeys; slot += a.splits * kThreads) {
        a.weights_out[at + slot] = a.weights[at + slot];
      }
    }
    cluster_sync_all();  // nobody reads another CTA's shared memory from here on
  }
}

// The maximum and the logarithm of the sum of all parts of a query head, in binades (infinity where nothing is seen). Whole warps.
__device__ __forceinline__ float joined_lse(const float2* ml, int parts, int lane) {
  float mm = -INFINITY;
  for (int i = lane; i < parts; i += 32) mm = fmaxf(mm, ml[i].x);
#pragma unroll
  for (int w = 16; w > 0; w /= 2) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, w));
  float ll = 0.f;
  for (int i = lane; i < parts; i += 32) ll += ml[i].y == 0.f ? 0.f : ml[i].y * ex2(ml[i].x - mm);
#pragma unroll
  for (int w = 16; w > 0; w /= 2) ll += __shfl_xor_sync(0xffffffffu, ll, w);
  return ll == 0.f ? INFINITY : mm + log2f(ll);
}

// The parts of a (sequence, key head) joined: the first CTAs have its query heads, the others ranges of its slots, which add up what those
// got: ex2 of the scores that the first kernel left minus the row's logarithm. Bound by latency (lengths, parts, scores one after the
// other): 64 sequences of up to 8101 slots, 32 / 8 heads, 20 us behind the first kernel for 50 MB; as a CTA per 1024 slots and head, 27.
template <typename T, int D, bool kScores>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const DecodeArgs a, int head_ctas, int slices) {
  extern __shared__ __align__(16) float s_lse[];  // [group]
  __shared__ __align__(16) float4 s_sum[kJoinThreads];
  __shared__ float2 s_ml[kJoinThreads];
  const int h = blockIdx.y, b = blockIdx.z, warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32;
  const int len = paged_len(a.c, b);  // (no kernel of the call writes the lengths: read ahead of the wait)
  const Steps steps(a, len);
  const int parts = max(1, (steps.count + a.chunk - 1) / a.chunk);
  const std::int64_t head0 = static_cast<std::int64_t>(b) * a.q_heads + h * a.group;

  if (static_cast<int>(blockIdx.x) < head_ctas) {
    // Four channels a thread, a slice of a head's parts each: one pass with a running maximum, so that no load waits for another.
    constexpr int kQuads = D / 4;
    const int quad = static_cast<int>(threadIdx.x) % kQuads, unit = static_cast<int>(threadIdx.x) / kQuads, slice = unit % slices;
    const int heads = kJoinThreads / kQuads / slices;  // of a CTA at a time
    wait_for_predecessors();
    for (int g0 = static_cast<int>(blockIdx.x) * heads; g0 < a.group; g0 += head_ctas * heads) {
      const int g = min(g0 + unit / slices, a.group - 1);  // (behind the last: the last again, not stored)
      const float2* ml = a.part_ml + (head0 + g) * a.splits;
      const float* part = a.part_o + (head0 + g) * a.splits * D + quad * 4;
      float m = -INFINITY, l = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      const auto add = [&](float mi, float li, const float4& x) {
        if (li == 0.f) return;  // nothing seen
        const float top = fmaxf(m, mi), f = ex2(mi - top), keep = l == 0.f ? 0.f : ex2(m - top);
        m = top, l = fmaf(f, li, keep * l);
        sum.x = joined(f, x.x, keep, sum.x), sum.y = joined(f, x.y, keep, sum.y);
        sum.z = joined(f, x.z, keep, sum.z), sum.w = joined(f, x.w, keep, sum.w);
      };
      for (int i0 = slice; i0 < parts; i0 += 4 * slices) {
        float2 of[4];
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = i0 + i * slices;
          of[i] = at < parts ? ml[at] : make_float2(0.f, 0.f);
          if (at < parts) x[i] = *reinterpret_cast<const float4*>(part + static_cast<std::int64_t>(at) * D);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) add(of[i].x, of[i].y, x[i]);
      }
      if (slices > 1) {
        __syncthreads();  // (the slices of the heads before are read)
        s_sum[threadIdx.x] = sum, s_ml[threadIdx.x] = make_float2(m, l);
        __syncthreads();
      }
      if (slice == 0 && g0 + unit / slices < a.group) {
        for (int i = 1; i < min(slices, parts); ++i) add(s_ml[threadIdx.x + i * kQuads].x, s_ml[threadIdx.x + i * kQuads].y, s_sum[threadIdx.x + i * kQuads]);
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T* out = static_cast<T*>(a.out) + b * a.o_row + (h * a.group + g) * a.o_head + quad * 4;
        *reinterpret_cast<uint2*>(out) = make_uint2(pack16<T>(sum.x * inv, sum.y * inv), pack16<T>(sum.z * inv, sum.w * inv));
        if (quad == 0 && a.lse != nullptr) a.lse[head0 + g] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      }
    }
    return;
  }

  if constexpr (kScores) {
    // kJoinSlots slots of a thread at a time, a CTA's width apart: their loads do not wait for one another.
    constexpr int kRange = kJoinThreads * kJoinSlots;
    const int first = (static_cast<int>(blockIdx.x) - head_ctas) * kRange;
    if (first >= len) return;
    const std::int64_t row = (static_cast<std::int64_t>(b) * a.c.kv_heads + h) * a.weights_ld;
    wait_for_predecessors();
    // The scores of kJoinHeads heads and the sums so far are on their way while the heads' logarithms are made.
    float sum[kJoinSlots], early[kJoinHeads][kJoinSlots];
    bool seen[kJoinSlots];
    const auto fetch = [&](int j0) {
#pragma unroll
      for (int i = 0; i < kJoinSlots; ++i) {
        const int j = j0 + i * kJoinThreads;
        seen[i] = sees(a, len, j);
        sum[i] = j < len - 1 ? a.weights[row + j] : 0.f;
#pragma unroll
        for (int g = 0; g < kJoinHeads; ++g) early[g][i] = seen[i] && g < a.group ? a.scores[(head0 + g) * a.scores_ld + j] : 0.f;
      }
    };
    fetch(first + static_cast<int>(threadIdx.x));
    for (int g = warp; g < a.group; g += kJoinThreads / 32) {
      const float lse2 = joined_lse(a.part_ml + (head0 + g) * a.splits, parts, lane);
      if (lane == 0) s_lse[g] = lse2;
    }
    __syncthreads();
    const int step = (static_cast<int>(gridDim.x) - head_ctas) * kRange;
    for (int j0 = first + static_cast<int>(threadIdx.x); j0 < len; j0 += step) {
      float got[kJoinSlots] = {};
#pragma unroll
      for (int g = 0; g < kJoinHeads; ++g) {
        if (g >= a.group) break;
#pragma unroll
        for (int i = 0; i < kJoinSlots; ++i) {
          if (seen[i]) got[i] += ex2(early[g][i] - s_lse[g]);
        }
      }
      const float* s = a.scores + head0 * a.scores_ld + j0;
#pragma unroll 4
      for (int g = kJoinHeads; g < a.group; ++g) {
#pragma unroll
        for (int i = 0; i < kJoinSlots; ++i) {
          if (seen[i]) got[i] += ex2(s[g * a.scores_ld + i * kJoinThreads] - s_lse[g]);
        }
      }
#pragma unroll
      for (int i = 0; i < kJoinSlots; ++i) {
        if (j0 + i * kJoinThreads < len) a.weights_out[row + j0 + i * kJoinThreads] = sum[i] + got[i];
      }
      if (j0 + step < len) fetch(j0 + step);
    }
  }
}

// How a call is cut into CTAs, by their number per SM, of which three fit at a time. One sequence: two equal CTAs per SM (131001
// slots, 4 key heads, this kernel: 53 us; three per SM 58, six 76). Several, whose lengths differ: eighteen, handed out as SMs come free (64 of up to 8101, 8
// key heads: 196 us; three per SM 233), but of kLongEnough steps at least, since each has its start and its part to join
// (4 of up to 30001: 76 us; as eighteen per SM 79). The lengths are on the device, so the rule goes by the number of sequences: equal ones do
// better as two per SM (the whole call behind a flushed L2, 32 / 4 heads of 128 in fp16: two of 65000 70.7 us, as eighteen 78.8; three of 43000
// 70.7 and 76.8; two of 130000 130 both ways), uneven ones worse by more (65000, 20000 and 5000: 69.6, as eighteen 60.4).
// Short ones are joined by the CTAs of a cluster in shared memory (by one CTA, where there are enough of them): one launch instead of two and
// no workspace, some 2 us of the host's time. Slots, and us with the second kernel and so: 6 sequences, 32 / 8 heads of 128: 500 15.8 and
// 10.8, 2000 18.5 and 16.7, 2600 19.2 and 19.9; 16: 500 16.5 and 12.6; 30, 14 / 2 of 64: 1000 16.0 and 11.0, 2000 16.6 and 14.4; so up to
// kClusterSteps a CTA. Five sixths of what fits on the SMs by shared memory, since a cluster wants its SMs side by side (60 clusters of
// seven at 3 CTAs an SM: 21 us, of six 14.4; 55 of six where 2 fit on an SM: 30.5, with the second kernel 20.6). One sequence has too few
// CTAs that way sooner (160 slots: 6.9 and 8.3; 517: 8.3 and 8.3; 1000: 9.8 and 8.3) and ends at a third of the steps.
constexpr std::int64_t kSharedOfSm = 228 * 1024;
constexpr int ring_bytes(int d) { return kWarps * kStages * 2 * kKeys * d * 2; }
constexpr int kOneSequence = 2, kSeveral = 18, kLongEnough = 32, kShortest = kWarps;

struct Plan {
  int chunk, splits;
  std::int64_t scores_ld;
  std::size_t ml, o, scores, total;
  bool parts, cluster;  // parts in the workspace; or in the CTAs of a cluster
};
Plan plan(const PagedArgs& c, int q_heads, int head_dim, int window, int sinks, bool weights) {
  Plan p{};
  p.scores_ld = (static_cast<std::int64_t>(c.most) + kKeys - 1) / kKeys * kKeys;
  const std::int64_t group = q_heads / c.kv_heads, units = std::max<std::int64_t>(1, c.batch * c.kv_heads * ((group + kRows - 1) / kRows));
  std::int64_t steps = p.scores_ld / kKeys;
  if (window > 0) steps = std::min<std::int64_t>(steps, (static_cast<std::int64_t>(window) + kKeys - 1) / kKeys + 1 + (static_cast<std::int64_t>(sinks) + kKeys - 1) / kKeys);
  const std::int64_t ctas = static_cast<std::int64_t>(sm_count()) * (c.batch <= 1 ? kOneSequence : kSeveral);
  std::int64_t chunk = (steps * units + ctas - 1) / ctas;
  if (c.batch > 1) chunk = std::max<std::int64_t>(chunk, kLongEnough);
  chunk = std::max<std::int64_t>(chunk, kShortest);
  const std::int64_t at_once = 5LL * sm_count() / 6, each = std::max<std::int64_t>(1, std::min<std::int64_t>(kMostCluster, 3 * at_once / units));
  const std::int64_t share = std::max<std::int64_t>((steps + each - 1) / each, kShortest);
  const std::int64_t per_sm = kSharedOfSm / (ring_bytes(head_dim) + (weights ? group * share * kKeys * 4 : 0) + 4096);
  p.cluster = group <= kRows && share <= (c.batch <= 1 ? kClusterSteps / 3 : kClusterSteps) && (per_sm >= 3 || units * each <= per_sm * at_once);
  if (p.cluster) chunk = share;
  p.chunk = static_cast<int>(std::min<std::int64_t>(chunk, INT_MAX / 2));
  p.splits = static_cast<int>(std::max<std::int64_t>(1, (steps + p.chunk - 1) / p.chunk));
  p.parts = !p.cluster && (p.splits > 1 || weights);
  const auto align = [](std::size_t n) { return (n + 255) / 256 * 256; };
  const std::size_t heads = static_cast<std::size_t>(c.batch) * q_heads;
  if (p.parts) {
    p.ml = 0;
    p.o = align(heads * p.splits * sizeof(float2));
    p.scores = p.o + align(heads * p.splits * head_dim * 4);
    p.total = p.scores + (weights ? align(heads * p.scores_ld * 4) : 0);
  }
  return p;
}

int check(const char* op, const b2_paged_cache* cache, PagedArgs* c, int q_heads, int max_len, int* window, int* sinks) {
  if (const int rc = check_paged_cache(op, cache, c)) return rc;
  if (q_heads <= 0 || q_heads > 65535 || q_heads % cache->kv_heads != 0) return fail_invalid(op, "q_heads must be a multiple of kv_heads, at most 65535");
  if (max_len < 0 || max_len > c->most) return fail_invalid(op, "max_len must lie within the block table");
  if (max_len > 0) c->most = max_len;
  if (const int rc = check_window(op, *c, window, sinks)) return rc;
  if (q_heads / cache->kv_heads > kMostGroup) return fail_invalid(op, "at most 4096 query heads to a key head");
  return B2_OK;
}

template <typename T, int D, bool kScores>
int launch(const char* op, const DecodeArgs& a, const Plan& p, const CUtensorMap& map_k, const CUtensorMap& map_v, cudaStream_t st) {
  constexpr int ring = ring_bytes(D), meet = (kWarps * kRows * (D + 4 + 2) + 2 * kRows) * 4;
  static_assert(meet <= ring);
  const LaunchChain chain(st);
  const unsigned blocks = static_cast<unsigned>((a.group + kRows - 1) / kRows), batch = static_cast<unsigned>(a.c.batch);
  const dim3 grid(static_cast<unsigned>(p.splits), static_cast<unsigned>(a.c.kv_heads) * blocks, batch);
  if (p.cluster) {
    constexpr int most = ring + 1024 + kRows * kClusterSteps * kKeys * 4;
    static std::atomic<std::uint64_t> allowed{0};
    if (const int rc = allow_shared(op, decode_kernel<T, D, kScores, true>, most, allowed)) return rc;
    const int smem = ring + 1024 + (kScores ? a.group * p.chunk * kKeys * 4 : 0);
    return enqueue(op, decode_kernel<T, D, kScores, true>, grid, kThreads, static_cast<std::size_t>(smem), st, p.splits, map_k, map_v, a);
  }
  constexpr int smem = ring + 1024;  // and what aligns it
  const auto kernel = decode_kernel<T, D, kScores, false>;
  static std::atomic<std::uint64_t> allowed{0};
  if (const int rc = allow_shared(op, kernel, smem, allowed)) return rc;
  if (const int rc = enqueue(op, kernel, grid, kThreads, smem, st, 1, map_k, map_v, a)) return rc;
  if (!p.parts) return B2_OK;
  // A slice has four parts in flight at once. Slot CTAs: eight per SM, so that the lengths of a batch even out.
  constexpr int units = kJoinThreads / (D / 4), range = kJoinThreads * kJoinSlots;
  int slices = 1;
  while (slices < units && 4 * slices < p.splits) slices *= 2;
  const int heads = units / slices, head_ctas = std::min((a.group + heads - 1) / heads, 64);
  const std::int64_t most = (static_cast<std::int64_t>(a.c.most) + range - 1) / range, pairs = static_cast<std::int64_t>(a.c.kv_heads) * a.c.batch;
  const int slot_ctas = kScores ? static_cast<int>(std::min(most, (static_cast<std::int64_t>(kJoinPerSm) * sm_count() + pairs - 1) / pairs)) : 0;
  return enqueue(op, join_kernel<T, D, kScores>, dim3(static_cast<unsigned>(head_ctas + slot_ctas), static_cast<unsigned>(a.c.kv_heads), batch), kJoinThreads,
                 kScores ? static_cast<std::size_t>(a.group) * 4 : 0, st, 1, a, head_ctas, slices);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

size_t b2_attention_paged_decode_workspace_bytes(const b2_paged_cache* cache, int q_heads, int max_len, int window, int sinks, int with_weights) {
  PagedArgs c{};
  if (check("attention_paged_decode", cache, &c, q_heads, max_len, &window, &sinks) != B2_OK) return 0;
  return std::max<std::size_t>(plan(c, q_heads, cache->head_dim, window, sinks, with_weights != 0).total, 256);
}

int b2_attention_paged_decode(const b2_paged_cache* cache, const b2_view3* q, const b2_view3* out, float* lse, int max_len,
                              float scale, int window, int sinks, const float* weights, float* weights_out, int64_t weights_ld,
                              void* workspace, size_t workspace_bytes, void* stream) {
  constexpr const char* op = "attention_paged_decode";
  DecodeArgs a{};
  if (q == nullptr || out == nullptr) return fail_invalid(op, "null q or out");
  if (q->heads <= 0 || q->heads > 65535) return fail_invalid(op, "q must have from 1 to 65535 heads");
  if (const int rc = check(op, cache, &a.c, static_cast<int>(q->heads), max_len, &window, &sinks)) return rc;
  if (q->tokens != cache->batch || out->tokens != q->tokens || out->heads != q->heads) return fail_invalid(op, "q and out must have one token per sequence and the same heads");
  if (!std::isfinite(scale) || !(scale > 0.0f)) return fail_invalid(op, "scale must be finite and positive");
  if ((weights == nullptr) != (weights_out == nullptr)) return fail_invalid(op, "weights and weights_out: both or neither");
  if (weights != nullptr && weights_ld < a.c.most) return fail_invalid(op, "weights need a place for every slot");
  if (cache->batch == 0) return B2_OK;
  if (!rows_ok(q->data, q->row_stride, q->head_stride) || !rows_ok(out->data, out->row_stride, out->head_stride)) {
    return fail_invalid(op, "q and out need a 16-byte aligned base and strides that are multiples of 8");
  }
  a.q = q->data, a.q_row = q->row_stride, a.q_head = q->head_stride, a.out = out->data, a.o_row = out->row_stride, a.o_head = out->head_stride;
  a.lse = lse, a.q_heads = static_cast<int>(q->heads), a.group = a.q_heads / cache->kv_heads;
  if (static_cast<std::int64_t>(cache->kv_heads) * ((a.group + kRows - 1) / kRows) > 65535) return fail_invalid(op, "too many heads");
  const bool scores = weights != nullptr;
  const Plan p = plan(a.c, a.q_heads, cache->head_dim, window, sinks, scores);
  if (const int rc = check_workspace(op, workspace, workspace_bytes, p.total)) return rc;
  a.scores_ld = p.scores_ld;
  a.scale_log2 = scale * 1.4426950408889634f, a.window = window, a.sinks = sinks, a.chunk = p.chunk, a.splits = p.splits;
  if (p.parts) {
    std::uint8_t* ws = static_cast<std::uint8_t*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(ws + p.ml), a.part_o = reinterpret_cast<float*>(ws + p.o);
    if (scores) a.scores = reinterpret_cast<float*>(ws + p.scores);
  }
  a.weights = weights, a.weights_out = weights_out, a.weights_ld = weights_ld;
  const cudaStream_t st = as_stream(stream);
  if (const int rc = paged_status_word(op, &a.c)) return rc;
  if (cache->num_pages == 0) return fail_invalid(op, "the pool has no pages");
  CUtensorMap map_k, map_v;
  if (!make_tensor_map_pages(&map_k, cache, false, kKeys, 64, op) || !make_tensor_map_pages(&map_v, cache, true, kKeys, 64, op)) return B2_ERR_CUDA;
  const bool wide = cache->head_dim == 128;
  if (cache->dtype == B2_DTYPE_BF16) {
    using T = __nv_bfloat16;
    if (scores) return wide ? launch<T, 128, true>(op, a, p, map_k, map_v, st) : launch<T, 64, true>(op, a, p, map_k, map_v, st);
    return wide ? launch<T, 128, false>(op, a, p, map_k, map_v, st) : launch<T, 64, false>(op, a, p, map_k, map_v, st);
  }
  using T = __half;
  if (scores) return wide ? launch<T, 128, true>(op, a, p, map_k, map_v, st) : launch<T, 64, true>(op, a, p, map_k, map_v, st);
  return wide ? launch<T, 128, false>(op, a, p, map_k, map_v, st) : launch<T, 64, false>(op, a, p, map_k, map_v, st);
}

}  // extern "C"
