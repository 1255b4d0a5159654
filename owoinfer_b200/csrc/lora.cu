// Low-rank adapters of many requests at once beside a projection that they share: the tokens sorted by adapter once for a step, then for each
// projection x A^T of every tile of tokens, split over the channels, and its product with B^T added to the projection's output.
#include <algorithm>
#include <cmath>

#include "text.cuh"

namespace b2 {
namespace {

__device__ unsigned g_lora_status = 0;
enum LoraFault : unsigned { kLoraBadAdapter = 1, kLoraBadRank = 2 };

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kPlanThreads = 1024;
constexpr int kMostAdapters = 4096, kMostRank = 128;
constexpr int kMostSplits = 16;

// Tokens of a tile: one warp's rows where few tokens share an adapter (its warps divide the channels then), four warps' where many do, for A and B to
// be read once for more of them.
inline int tile_rows(std::int64_t tokens) { return tokens <= 1024 ? 16 : 64; }
inline std::int64_t most_tiles(std::int64_t tokens, int adapters) {
  const int rows = tile_rows(tokens);
  return std::min(tokens, tokens / rows + adapters + 1);
}

// A plan: how many tiles there are, the tiles, the tokens in the order of their adapters.
struct PlanHead {
  int tiles, pad[3];
};
struct Tile {
  int adapter, first, count, pad;  // -1: tokens without an adapter
};
struct Plan {
  const PlanHead* head;
  const Tile* tiles;
  const std::int32_t* order;
};
inline std::size_t plan_bytes(std::int64_t tokens, int adapters) {
  const std::size_t bytes = sizeof(PlanHead) + static_cast<std::size_t>(most_tiles(tokens, adapters)) * sizeof(Tile) + static_cast<std::size_t>(tokens) * 4;
  return (bytes + 255) / 256 * 256;
}
inline Plan plan_at(const void* p, std::int64_t tokens, int adapters) {
  const char* at = static_cast<const char*>(p);
  const Tile* tiles = reinterpret_cast<const Tile*>(at + sizeof(PlanHead));
  return {reinterpret_cast<const PlanHead*>(at), tiles, reinterpret_cast<const std::int32_t*>(tiles + most_tiles(tokens, adapters))};
}

// A CTA per adapter, and one for the tokens without: each counts all tokens by adapter (a thread a run of neighbouring tokens, which mostly have
// the same one), and puts its own in their places, in their order.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const std::int32_t* ids, int tokens, int adapters, int rows, PlanHead* head, Tile* tiles,
                                                            std::int32_t* order) {
  extern __shared__ int s_count[];  // [adapters + 1]
  __shared__ int s_warp[kPlanThreads / 32], s_before[2];
  const int tid = static_cast<int>(threadIdx.x), own = static_cast<int>(blockIdx.x);
  for (int i = tid; i <= adapters; i += kPlanThreads) s_count[i] = 0;
  if (tid < 2) s_before[tid] = 0;
  __syncthreads();
  const int per = (tokens + kPlanThreads - 1) / kPlanThreads, begin = static_cast<int>(min(static_cast<long long>(tid) * per, static_cast<long long>(tokens)));
  const int end = min(tokens, begin + per);
  const auto id_of = [&](int token) {
    const int id = ids[token];
    return id >= 0 && id < adapters ? id : adapters;
  };
  int run = -1, length = 0, mine = 0;
  for (int i = begin; i < end; ++i) {
    const int id = id_of(i);
    if (own == 0 && ids[i] >= adapters) atomicOr(&g_lora_status, kLoraBadAdapter);
    mine += id == own;
    if (id != run) {
      if (length > 0) atomicAdd(&s_count[run], length);
      run = id, length = 0;
    }
    ++length;
  }
  if (length > 0) atomicAdd(&s_count[run], length);
  __syncthreads();
  // Tokens and tiles of the adapters before this one.
  int tokens_before = 0, tiles_before = 0;
  for (int i = tid; i < own; i += kPlanThreads) tokens_before += s_count[i], tiles_before += (s_count[i] + rows - 1) / rows;
  if (tokens_before > 0) atomicAdd(&s_before[0], tokens_before), atomicAdd(&s_before[1], tiles_before);
  // This thread's place among the CTA's tokens.
  const int lane = tid % 32;
  int sum = mine;
#pragma unroll
  for (int m = 1; m < 32; m *= 2) {
    const int v = __shfl_up_sync(0xffffffffu, sum, m);
    if (lane >= m) sum += v;
  }
  if (lane == 31) s_warp[tid / 32] = sum;
  __syncthreads();
  int place = s_before[0] + sum - mine;
  for (int i = 0; i < tid / 32; ++i) place += s_warp[i];
  if (mine > 0) {
    for (int i = begin; i < end; ++i) {
      if (id_of(i) == own) order[place++] = i;
    }
  }
  const int count = s_count[own], num = (count + rows - 1) / rows;
  for (int i = tid; i < num; i += kPlanThreads) tiles[s_before[1] + i] = Tile{own < adapters ? own : -1, s_before[0] + i * rows, min(rows, count - i * rows), 0};
  if (own == adapters && tid == 0) head->tiles = s_before[1] + num;
}

struct LoraArgs {
  Plan plan;
  const void* a;
  const void* b;
  std::int64_t a_adapter, a_row, b_adapter, b_row;
  const float* scales;
  const std::int32_t* ranks;
  const void* x;
  const void* y;
  void* out;
  std::int64_t ldx, ldy, ldo;
  float* part;  // [splits, tiles * rows, rank padded]
  std::int64_t part_split;
  int adapters, rank, dim, width;
  int splits, slice;  // parts of the channels, channels of each (a multiple of 32)
  int columns;        // columns of an output CTA
};

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], std::uint32_t a0, std::uint32_t a1, std::uint32_t a2, std::uint32_t a3, std::uint32_t b0, std::uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ uint4 load16(const void* p) { return *reinterpret_cast<const uint4*>(p); }

__device__ __forceinline__ int rank_of(const LoraArgs& a, int adapter) {
  if (a.ranks == nullptr) return a.rank;
  const int r = a.ranks[adapter];
  if (r >= 0 && r <= a.rank) return r;
  atomicOr(&g_lora_status, kLoraBadRank);
  return r < 0 ? 0 : a.rank;
}

// x A^T of a tile's tokens over a part of the channels, in 16-row MMAs with the ranks as columns. Which channels a place of an MMA's K stands for does
// not matter as long as x and A agree: a lane takes 8 neighbouring ones of each, straight from memory in one load, as the K of two MMAs.
// kNT: ranks / 8, up to a power of two. kFew: the warps divide the channels, not the rows.
template <typename T, int kNT, bool kFew>
__global__ void __launch_bounds__(kThreads) shrink_kernel(const LoraArgs a) {
  dependents_may_start();
  constexpr int kRows = kFew ? 16 : 64, kRanks = kNT * 8;
  __shared__ float s_sum[kFew ? kWarps : 1][kFew ? 16 * kRanks : 1];
  if (static_cast<int>(blockIdx.x) >= a.plan.head->tiles) return;
  const Tile tile = a.plan.tiles[blockIdx.x];
  if (tile.adapter < 0) return;
  const int rank = rank_of(a, tile.adapter);
  const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32, g = lane / 4, c = lane % 4;
  const int row0 = kFew ? 0 : warp * 16;
  if (!kFew && row0 >= tile.count) return;
  const T* x[2];
  bool there[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = row0 + g + 8 * i;
    there[i] = r < tile.count;
    x[i] = static_cast<const T*>(a.x) + (there[i] ? a.plan.order[tile.first + r] : 0) * a.ldx + c * 8;
  }
  const T* const w = static_cast<const T*>(a.a) + tile.adapter * a.a_adapter + g * a.a_row + c * 8;
  const int from = static_cast<int>(blockIdx.y) * a.slice, to = min(a.dim, from + a.slice);
  float acc[kNT][4] = {};
  constexpr int kStep = kFew ? 32 * kWarps : 32, kUnroll = kNT <= 2 ? 4 : kNT <= 4 ? 2 : 1;
  const auto block = [&](int k, bool in, uint4 (&xv)[2], uint4 (&wv)[kNT]) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 2; ++i) xv[i] = in && there[i] ? load16(x[i] + k) : zero;
#pragma unroll
    for (int j = 0; j < kNT; ++j) wv[j] = in && j * 8 + g < rank ? load16(w + j * 8 * a.a_row + k) : zero;
  };
  for (int k = from + (kFew ? warp * 32 : 0); k < to; k += kStep * kUnroll) {
    uint4 xv[kUnroll][2], wv[kUnroll][kNT];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) block(k + u * kStep, k + u * kStep + c * 8 < to, xv[u], wv[u]);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        mma<T>(acc[j], xv[u][0].x, xv[u][1].x, xv[u][0].y, xv[u][1].y, wv[u][j].x, wv[u][j].y);
        mma<T>(acc[j], xv[u][0].z, xv[u][1].z, xv[u][0].w, xv[u][1].w, wv[u][j].z, wv[u][j].w);
      }
    }
  }
  float* const out = a.part + blockIdx.y * a.part_split + static_cast<std::int64_t>(blockIdx.x) * kRows * kRanks;
  if constexpr (kFew) {
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) *reinterpret_cast<float2*>(&s_sum[warp][(g + 8 * i) * kRanks + j * 8 + c * 2]) = make_float2(acc[j][2 * i], acc[j][2 * i + 1]);
    }
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < 16 * kRanks; i += kThreads) {
      float sum = s_sum[0][i];
#pragma unroll
      for (int v = 1; v < kWarps; ++v) sum += s_sum[v][i];
      out[i] = sum;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) *reinterpret_cast<float2*>(out + (row0 + g + 8 * i) * kRanks + j * 8 + c * 2) = make_float2(acc[j][2 * i], acc[j][2 * i + 1]);
    }
  }
}

// Ranks of an MMA's K go to lanes as the channels above: 8 neighbouring ones of 32 for two MMAs, or (16 ranks and fewer) 4 of 16 for one.
template <typename T, int kNT>
struct Low {  // t = x A^T of a warp's 16 rows as A operands: in two parts, which hold 16 (bf16) or 22 (fp16) bits of it
  static constexpr int kSteps = kNT <= 2 ? 1 : kNT / 2, kPer = kNT <= 2 ? 4 : 8, kBlocks = kNT <= 2 ? 1 : kNT / 4;
  std::uint32_t hi[kSteps][4], lo[kSteps][4];
  float back[2];  // what a row's values were divided by
  __device__ __forceinline__ void load(const float* part, std::int64_t part_split, int splits, int g, int c, int rank, float scale) {
    constexpr int kRanks = kNT * 8;
    float t[2][kBlocks * kPer];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int q = 0; q < kBlocks * kPer; ++q) t[i][q] = 0.f;
      for (int s = 0; s < splits; ++s) {
#pragma unroll
        for (int q = 0; q < kBlocks * kPer; q += 4) {
          const int at = q / kPer * 32 + c * kPer + q % kPer;
          if (at >= kRanks) continue;  // (8 ranks: the upper lanes have none)
          const float4 v = *reinterpret_cast<const float4*>(part + s * part_split + (g + 8 * i) * kRanks + at);
          t[i][q] += v.x, t[i][q + 1] += v.y, t[i][q + 2] += v.z, t[i][q + 3] += v.w;
        }
      }
      float top = 0.f;
#pragma unroll
      for (int q = 0; q < kBlocks * kPer; ++q) {
        // (infinities of x have made NaN of what lies behind the rank)
        t[i][q] = q / kPer * 32 + c * kPer + q % kPer < rank ? t[i][q] * scale : 0.f;
        top = fmaxf(top, fabsf(t[i][q]));
      }
      back[i] = 1.f;
      if constexpr (std::is_same<T, __half>::value) {
        // fp16 ends at 2^16 and loses bits below 2^-14: a row's largest value is brought between 2^14 and 2^15 by a power of two.
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = top < INFINITY ? max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14, -100) : 0;
        const float f = __uint_as_float(static_cast<unsigned>(127 - e) << 23);
        back[i] = __uint_as_float(static_cast<unsigned>(127 + e) << 23);
#pragma unroll
        for (int q = 0; q < kBlocks * kPer; ++q) t[i][q] *= f;
      }
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {  // registers of an A operand: rows g and g + 8, the first two of four ranks, then the other two
        const float x = t[r & 1][s * 4 + (r >> 1) * 2], y = t[r & 1][s * 4 + (r >> 1) * 2 + 1];
        hi[s][r] = pack16<T>(x, y);
        float xh, yh;
        unpack16<T>(hi[s][r], xh, yh);
        lo[s][r] = pack16<T>(isfinite(xh) ? x - xh : 0.f, isfinite(yh) ? y - yh : 0.f);
      }
    }
  }
};
// The elements of a word (two neighbouring ranks from `at`) that are used.
__device__ __forceinline__ std::uint32_t used(std::uint32_t w, int at, int rank) {
  return at + 1 < rank ? w : at < rank ? w & 0xffffu : 0u;
}

// t B^T of a tile added to the projection's output, for some of the columns. A warp's 16 rows x 32 columns at a time: of the four MMAs
// beside one another each takes every other pair of the columns, so that a lane ends up with 8 neighbouring columns of two rows, one load and one
// store each. What bounds it is memory: y is read and out written once, t and B come from L2.
template <typename T, int kNT, bool kFew>
__global__ void __launch_bounds__(kThreads) expand_kernel(const LoraArgs a) {
  using L = Low<T, kNT>;
  constexpr int kRows = kFew ? 16 : 64, kRanks = kNT * 8;
  const bool exists = static_cast<int>(blockIdx.x) < a.plan.head->tiles;
  const Tile tile = exists ? a.plan.tiles[blockIdx.x] : Tile{-1, 0, 0, 0};
  if (!exists || (tile.adapter < 0 && a.y == a.out)) {
    wait_for_predecessors();  // (this kernel is not done before the one that it follows)
    return;
  }
  const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32, g = lane / 4, c = lane % 4;
  const int row0 = kFew ? 0 : warp * 16;
  if (!kFew && row0 >= tile.count) return;
  const T* y[2];
  T* out[2];
  bool there[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = row0 + g + 8 * i;
    there[i] = r < tile.count;
    const std::int64_t token = there[i] ? a.plan.order[tile.first + r] : 0;
    y[i] = static_cast<const T*>(a.y) + token * a.ldy + c * 8, out[i] = static_cast<T*>(a.out) + token * a.ldo + c * 8;
  }
  const int from = static_cast<int>(blockIdx.y) * a.columns + (kFew ? warp * 32 : 0), to = min(a.width, (static_cast<int>(blockIdx.y) + 1) * a.columns);
  constexpr int kStep = kFew ? 32 * kWarps : 32;
  if (tile.adapter < 0) {
    for (int n = from; n < to; n += kStep) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (there[i] && n + c * 8 < to) *reinterpret_cast<uint4*>(out[i] + n) = load16(y[i] + n);
      }
    }
    wait_for_predecessors();
    return;
  }
  const int rank = rank_of(a, tile.adapter);
  const float scale = a.scales != nullptr ? a.scales[tile.adapter] : 1.f;
  wait_for_predecessors();
  L low;
  low.load(a.part + (static_cast<std::int64_t>(blockIdx.x) * kRows + row0) * kRanks, a.part_split, a.splits, g, c, rank, scale);
  const T* const w = static_cast<const T*>(a.b) + tile.adapter * a.b_adapter + (g / 2 * 8 + g % 2) * a.b_row + c * L::kPer;
  for (int n = from; n < to; n += kStep) {
    uint4 yv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (there[i] && n + c * 8 < to) yv[i] = load16(y[i] + n);
      else yv[i] = make_uint4(0, 0, 0, 0);
    }
    float acc[4][4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = n + g / 2 * 8 < to;  // (columns come in eights)
      const T* const row = w + (n + 2 * j) * a.b_row;
#pragma unroll
      for (int q = 0; q < L::kBlocks; ++q) {
        const int at = q * 32 + c * L::kPer;
        std::uint32_t v[4] = {};
        if (in && at < rank) {
          if constexpr (L::kPer == 8) {
            const uint4 r = load16(row + q * 32);
            v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w;
          } else {
            const uint2 r = *reinterpret_cast<const uint2*>(row);
            v[0] = r.x, v[1] = r.y;
          }
        }
        if (rank < at + L::kPer) {
#pragma unroll
          for (int e = 0; e < L::kPer / 2; ++e) v[e] = used(v[e], at + 2 * e, rank);
        }
#pragma unroll
        for (int e = 0; e < L::kPer / 4; ++e) {
          const int s = q * (L::kPer / 4) + e;
          mma<T>(acc[j], low.hi[s][0], low.hi[s][1], low.hi[s][2], low.hi[s][3], v[2 * e], v[2 * e + 1]);
          mma<T>(acc[j], low.lo[s][0], low.lo[s][1], low.lo[s][2], low.lo[s][3], v[2 * e], v[2 * e + 1]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float v[8];
      load8<T>(yv[i], v);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = fmaf(acc[j][2 * i], low.back[i], v[2 * j]);
        v[2 * j + 1] = fmaf(acc[j][2 * i + 1], low.back[i], v[2 * j + 1]);
      }
      if (there[i] && n + c * 8 < to) *reinterpret_cast<uint4*>(out[i] + n) = store8<T>(v);
    }
  }
}

inline int padded_tiles(int rank) {  // ranks / 8, up to a power of two
  int n = 1;
  while (n * 8 < rank) n *= 2;
  return n;
}
// Parts of the channels: CTAs for the whole GPU twice over, of 256 channels at least.
inline int splits_of(std::int64_t tokens, int adapters, std::int64_t dim) {
  const std::int64_t tiles = std::max<std::int64_t>(1, most_tiles(tokens, adapters));
  const std::int64_t wanted = (2 * 148 + tiles - 1) / tiles, most = std::max<std::int64_t>(1, dim / 256);
  return static_cast<int>(std::min<std::int64_t>({wanted, most, kMostSplits}));
}
inline std::size_t workspace_bytes(std::int64_t tokens, int adapters, std::int64_t dim, int rank) {
  const std::size_t rows = static_cast<std::size_t>(most_tiles(tokens, adapters)) * tile_rows(tokens);
  return std::max<std::size_t>(256, rows * padded_tiles(rank) * 8 * 4 * splits_of(tokens, adapters, dim));
}

template <typename T, int kNT, bool kFew>
int launch(const char* op, LoraArgs a, std::int64_t tokens, cudaStream_t stream) {
  const unsigned tiles = static_cast<unsigned>(most_tiles(tokens, a.adapters));
  const LaunchChain chain(stream);
  const unsigned parts = static_cast<unsigned>((a.dim + a.slice - 1) / a.slice);
  a.splits = static_cast<int>(parts);
  if (const int s = enqueue(op, shrink_kernel<T, kNT, kFew>, dim3(tiles, parts), dim3(kThreads), 0, stream, 1, a); s != B2_OK) return s;
  // Columns of a CTA: as many as leave 8 CTAs to an SM, 128 at least.
  const std::int64_t most = std::max<std::int64_t>(1, 8LL * sm_count() / tiles);
  a.columns = static_cast<int>(std::max<std::int64_t>(128, ((a.width + most - 1) / most + 127) / 128 * 128));
  return enqueue(op, expand_kernel<T, kNT, kFew>, dim3(tiles, static_cast<unsigned>((a.width + a.columns - 1) / a.columns)), dim3(kThreads), 0, stream, 1, a);
}
template <typename T, int kNT>
int launch(const char* op, const LoraArgs& a, std::int64_t tokens, cudaStream_t stream) {
  return tile_rows(tokens) == 16 ? launch<T, kNT, true>(op, a, tokens, stream) : launch<T, kNT, false>(op, a, tokens, stream);
}
template <typename T>
int launch(const char* op, const LoraArgs& a, std::int64_t tokens, cudaStream_t stream) {
  switch (padded_tiles(a.rank)) {
    case 1: return launch<T, 1>(op, a, tokens, stream);
    case 2: return launch<T, 2>(op, a, tokens, stream);
    case 4: return launch<T, 4>(op, a, tokens, stream);
    case 8: return launch<T, 8>(op, a, tokens, stream);
    default: return launch<T, 16>(op, a, tokens, stream);
  }
}

int check_sizes(const char* op, std::int64_t tokens, int adapters) {
  if (tokens < 0 || tokens > (1LL << 30)) return fail_invalid(op, "tokens must be from 0 to 2^30");
  if (adapters < 1 || adapters > kMostAdapters) return fail_invalid(op, "adapters must be from 1 to 4096");
  return B2_OK;
}
int check_shape(const char* op, std::int64_t dim, int rank) {
  if (dim <= 0 || dim % 8 != 0 || dim > (1LL << 30)) return fail_invalid(op, "dim must be a multiple of 8 from 8 to 2^30");
  if (rank <= 0 || rank % 8 != 0 || rank > kMostRank) return fail_invalid(op, "rank must be a multiple of 8 from 8 to 128");
  return B2_OK;
}

}  // namespace
}  // namespace b2

extern "C" {

size_t b2_lora_plan_bytes(int64_t tokens, int adapters) {
  if (b2::check_sizes("lora_plan", tokens, adapters) != B2_OK) return 0;
  return b2::plan_bytes(tokens, adapters);
}

int b2_lora_plan(const int32_t* token_adapters, int64_t tokens, int adapters, void* plan, size_t bytes, void* stream) {
  using namespace b2;
  const char* const op = "lora_plan";
  if (const int s = check_sizes(op, tokens, adapters); s != B2_OK) return s;
  if (plan == nullptr || !aligned_to(plan, 256) || bytes < plan_bytes(tokens, adapters)) return fail_invalid(op, "plan is missing, too small or not 256-byte aligned");
  if (tokens == 0) return B2_OK;
  if (token_adapters == nullptr || !aligned_to(token_adapters, 4)) return fail_invalid(op, "token_adapters is missing or not aligned");
  const Plan p = plan_at(plan, tokens, adapters);
  return enqueue(op, plan_kernel, dim3(static_cast<unsigned>(adapters + 1)), dim3(kPlanThreads), static_cast<std::size_t>(adapters + 1) * 4, as_stream(stream), 1,
                 token_adapters, static_cast<int>(tokens), adapters, tile_rows(tokens), const_cast<PlanHead*>(p.head), const_cast<Tile*>(p.tiles),
                 const_cast<std::int32_t*>(p.order));
}

size_t b2_lora_workspace_bytes(int64_t tokens, int adapters, int64_t dim, int rank) {
  using namespace b2;
  const char* const op = "lora_add";
  if (check_sizes(op, tokens, adapters) != B2_OK || check_shape(op, dim, rank) != B2_OK) return 0;
  return workspace_bytes(tokens, adapters, dim, rank);
}

int b2_lora_add(const b2_lora* l, const void* plan, size_t bytes, int64_t tokens, const void* x, int64_t ldx, const void* y, int64_t ldy, void* out, int64_t ldo,
                void* workspace, size_t ws_bytes, void* stream) {
  using namespace b2;
  const char* const op = "lora_add";
  if (l == nullptr || l->struct_size != sizeof(b2_lora)) return fail_invalid(op, "struct_size does not match");
  if (l->dtype != B2_DTYPE_BF16 && l->dtype != B2_DTYPE_F16) return fail_invalid(op, "dtype must be bf16 or fp16");
  if (const int s = check_sizes(op, tokens, l->adapters); s != B2_OK) return s;
  if (const int s = check_shape(op, l->dim, l->rank); s != B2_OK) return s;
  if (l->width <= 0 || l->width % 8 != 0 || l->width > (1LL << 30)) return fail_invalid(op, "width must be a multiple of 8 from 8 to 2^30");
  const auto strides_ok = [](std::int64_t adapter, std::int64_t row, std::int64_t least) { return adapter >= 0 && adapter % 8 == 0 && row >= least && row % 8 == 0; };
  if (l->a == nullptr || !aligned_to(l->a, 16) || !strides_ok(l->a_adapter_stride, l->a_row_stride, l->dim)) return fail_invalid(op, "a must be 16-byte aligned rows of dim elements");
  if (l->b == nullptr || !aligned_to(l->b, 16) || !strides_ok(l->b_adapter_stride, l->b_row_stride, l->rank)) return fail_invalid(op, "b must be 16-byte aligned rows of rank elements");
  if (!aligned_to(l->scales, 4) || !aligned_to(l->ranks, 4)) return fail_invalid(op, "scales and ranks must be aligned");
  if (tokens == 0) return B2_OK;
  if (plan == nullptr || !aligned_to(plan, 256) || bytes < plan_bytes(tokens, l->adapters)) return fail_invalid(op, "plan is missing, too small or not 256-byte aligned");
  if (!matrix_ok(x, ldx, l->dim, 2)) return fail_invalid(op, "x must be 16-byte aligned rows of at least dim elements");
  if (!matrix_ok(y, ldy, l->width, 2)) return fail_invalid(op, "y must be 16-byte aligned rows of at least width elements");
  if (!matrix_ok(out, ldo, l->width, 2)) return fail_invalid(op, "out must be 16-byte aligned rows of at least width elements");
  if (out == y && ldo != ldy) return fail_invalid(op, "out in y's place must have y's rows");
  if (const int s = check_workspace(op, workspace, ws_bytes, workspace_bytes(tokens, l->adapters, l->dim, l->rank)); s != B2_OK) return s;
  LoraArgs a{};
  a.plan = plan_at(plan, tokens, l->adapters);
  a.a = l->a, a.b = l->b, a.a_adapter = l->a_adapter_stride, a.a_row = l->a_row_stride, a.b_adapter = l->b_adapter_stride, a.b_row = l->b_row_stride;
  a.scales = l->scales, a.ranks = l->ranks, a.x = x, a.y = y, a.out = out, a.ldx = ldx, a.ldy = ldy, a.ldo = ldo;
  a.adapters = l->adapters, a.rank = l->rank, a.dim = static_cast<int>(l->dim), a.width = static_cast<int>(l->width);
  a.part = static_cast<float*>(workspace);
  a.part_split = most_tiles(tokens, l->adapters) * tile_rows(tokens) * padded_tiles(l->rank) * 8;
  const int splits = splits_of(tokens, l->adapters, l->dim);
  a.slice = static_cast<int>(((l->dim + splits - 1) / splits + 31) / 32 * 32);
  return l->dtype == B2_DTYPE_F16 ? launch<__half>(op, a, tokens, as_stream(stream)) : launch<__nv_bfloat16>(op, a, tokens, as_stream(stream));
}

int b2_lora_status(unsigned* host_value, int clear) {
  using namespace b2;
  const char* const op = "lora_status";
  if (host_value == nullptr) return fail_invalid(op, "host_value is missing");
  if (cudaError_t e = cudaDeviceSynchronize(); e != cudaSuccess) return fail_cuda(op, e);
  if (cudaError_t e = cudaMemcpyFromSymbol(host_value, g_lora_status, sizeof(unsigned)); e != cudaSuccess) return fail_cuda(op, e);
  if (clear != 0) {
    const unsigned zero = 0;
    if (cudaError_t e = cudaMemcpyToSymbol(g_lora_status, &zero, sizeof zero); e != cudaSuccess) return fail_cuda(op, e);
  }
  return B2_OK;
}

}  // extern "C"
