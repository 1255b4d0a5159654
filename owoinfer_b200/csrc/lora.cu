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
constexpr int kMostParts = 8;  // CTAs of a cluster that divide the channels

// Tokens of a tile: one warp's rows of few tokens, eight warps' of many, for A and B to be read once for more of them.
constexpr int kFewTokens = 256, kFewRows = 16, kManyRows = 128;
inline int tile_rows(std::int64_t tokens) { return tokens <= kFewTokens ? kFewRows : kManyRows; }
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
  // t = scale x A^T by [tile, row of the tile]: in two 16-bit parts [ranks, padded] each, and what a row was divided by.
  void* t_hi;
  void* t_lo;
  float* t_back;
  int adapters, rank, dim, width;
  int parts, slice;  // parts of the channels, channels of each (a multiple of 64)
  int columns;        // columns of an output CTA
};

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint4& a, std::uint32_t b0, std::uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  }
}
// K of 32: 8 neighbouring elements of a lane in each operand.
template <typename T>
__device__ __forceinline__ void mma_twice(float (&d)[4], const uint4& a0, const uint4& a1, const uint4& b) {
  mma<T>(d, make_uint4(a0.x, a1.x, a0.y, a1.y), b.x, b.y);
  mma<T>(d, make_uint4(a0.z, a1.z, a0.w, a1.w), b.z, b.w);
}
__device__ __forceinline__ uint4 load16(const void* p) { return *reinterpret_cast<const uint4*>(p); }

__device__ __forceinline__ int rank_of(const LoraArgs& a, int adapter) {
  if (a.ranks == nullptr) return a.rank;
  const int r = a.ranks[adapter];
  if (r >= 0 && r <= a.rank) return r;
  atomicOr(&g_lora_status, kLoraBadRank);
  return r < 0 ? 0 : a.rank;
}

// Where t's ranks r and r + 1 of a row lie, r + 2 and r + 3 two words on (r a multiple of 4): in the order of an MMA's A operands, four words of a lane
// for each 16 rows and K of 16. Ranks of a K go to lanes as they come from B in one load: 8 neighbouring ones of 32 for two MMAs, or (16 ranks and fewer)
// 4 of 16 for one.
template <int kRanks>
__device__ __forceinline__ std::int64_t low_word(std::int64_t row, int r) {
  constexpr int kSteps = kRanks <= 16 ? 1 : kRanks / 16;
  const int step = kRanks <= 16 ? 0 : r / 32 * 2 + r % 8 / 4, c = kRanks <= 16 ? r / 4 : r % 32 / 8;
  return ((row / 16 * kSteps + step) * 32 + row % 8 * 4 + c) * 4 + row % 16 / 8;
}

// Sums of x A^T over the channels' parts, [rows][ranks] in the shared memory of each CTA of a cluster at `sums`, joined, scaled and left for the product with
// B: a row by ranks / 4 neighbouring lanes, every CTA some of the rows. In two 16-bit parts t keeps 16 (bf16) or 22 (fp16) of its bits.
template <typename T, int kRanks, int kRows>
__device__ __forceinline__ void leave_sums(const LoraArgs& a, const Tile& tile, std::int64_t tile_number, int rank, const float* sums) {
  constexpr int kLanes = kRanks / 4;
  if (a.parts > 1) cluster_sync_all();
  else __syncthreads();
  const int part = static_cast<int>(blockIdx.x) % a.parts, lane = static_cast<int>(threadIdx.x) % kLanes;
  const float scale = a.scales != nullptr ? a.scales[tile.adapter] : 1.f;
  const std::uint32_t own = smem_u32(sums);
  for (int first = part * (kThreads / kLanes); first < kRows; first += a.parts * (kThreads / kLanes)) {  // (the same number of rounds for a warp's lanes)
    const int row = first + static_cast<int>(threadIdx.x) / kLanes;
    float v[4] = {};
    if (row < kRows) {
      const std::uint32_t at = own + (row * kRanks + lane * 4) * 4;
      for (int p = 0; p < a.parts; ++p) {
        const float4 s = a.parts > 1 ? ld_cluster_f32x4(map_to_cta(at, static_cast<std::uint32_t>(p))) : *reinterpret_cast<const float4*>(sums + row * kRanks + lane * 4);
        v[0] += s.x, v[1] += s.y, v[2] += s.z, v[3] += s.w;
      }
    }
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = lane * 4 + e < rank ? v[e] * scale : 0.f;  // (infinities of x have made NaN of what lies behind the rank)
      top = fmaxf(top, fabsf(v[e]));
    }
    float by = 1.f, back = 1.f;
    if constexpr (std::is_same<T, __half>::value) {
      // fp16 ends at 2^16 and loses bits below 2^-14: a row's largest value is brought between 2^14 and 2^15 by a power of two.
#pragma unroll
      for (int m = kLanes / 2; m > 0; m /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
      const int e = top < INFINITY ? max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14, -100) : 0;
      by = __uint_as_float(static_cast<unsigned>(127 - e) << 23), back = __uint_as_float(static_cast<unsigned>(127 + e) << 23);
    }
    if (row >= kRows) continue;
    std::uint32_t hi[2], lo[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float x = v[2 * e] * by, y = v[2 * e + 1] * by;
      hi[e] = pack16<T>(x, y);
      float xh, yh;
      unpack16<T>(hi[e], xh, yh);
      lo[e] = pack16<T>(isfinite(xh) ? x - xh : 0.f, isfinite(yh) ? y - yh : 0.f);
    }
    const std::int64_t to = low_word<kRanks>(tile_number * kRows + row, lane * 4);
    static_cast<std::uint32_t*>(a.t_hi)[to] = hi[0], static_cast<std::uint32_t*>(a.t_hi)[to + 2] = hi[1];
    static_cast<std::uint32_t*>(a.t_lo)[to] = lo[0], static_cast<std::uint32_t*>(a.t_lo)[to + 2] = lo[1];
    if (lane == 0) a.t_back[tile_number * kRows + row] = back;
  }
  if (a.parts > 1) cluster_sync_all();  // (nobody leaves while others read its sums)
}

// x A^T of a tile's tokens over a part of the channels, in 16-row MMAs with the ranks as columns. Which channels a place of an MMA's K stands for does
// not matter as long as x and A agree: a lane takes 8 neighbouring ones of each, in one load, as the K of two MMAs. kNT: ranks / 8, up to a
// power of two. Few tokens: a tile's warps divide the part's channels and are added up in shared memory.
template <typename T, int kNT>
__global__ void __launch_bounds__(kThreads) shrink_few_kernel(const LoraArgs a) {
  dependents_may_start();
  constexpr int kRanks = kNT * 8;
  __shared__ __align__(16) float s_sum[kWarps][kFewRows * kRanks];
  const int tile_number = static_cast<int>(blockIdx.x) / a.parts, part = static_cast<int>(blockIdx.x) % a.parts;
  if (tile_number >= a.plan.head->tiles) return;
  const Tile tile = a.plan.tiles[tile_number];
  if (tile.adapter < 0) return;
  const int rank = rank_of(a, tile.adapter);
  const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32, g = lane / 4, c = lane % 4;
  const T* x[2];
  bool there[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = g + 8 * i;
    there[i] = r < tile.count;
    x[i] = static_cast<const T*>(a.x) + (there[i] ? a.plan.order[tile.first + r] : 0) * a.ldx + c * 8;
  }
  const T* const w = static_cast<const T*>(a.a) + tile.adapter * a.a_adapter + g * a.a_row + c * 8;
  const int from = part * a.slice, to = min(a.dim, from + a.slice);
  float acc[kNT][4] = {};
  constexpr int kStep = 32 * kWarps, kUnroll = kNT <= 2 ? 4 : kNT <= 4 ? 2 : 1;
  const auto block = [&](int k, bool in, uint4 (&xv)[2], uint4 (&wv)[kNT]) {
    const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < kNT; ++j) wv[j] = in && j * 8 + g < rank ? load16(w + j * 8 * a.a_row + k) : zero;
#pragma unroll
    for (int i = 0; i < 2; ++i) xv[i] = in && there[i] ? load16(x[i] + k) : zero;
  };
  for (int k = from + warp * 32; k < to; k += kStep * kUnroll) {
    uint4 xv[kUnroll][2], wv[kUnroll][kNT];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) block(k + u * kStep, k + u * kStep + c * 8 < to, xv[u], wv[u]);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int j = 0; j < kNT; ++j) mma_twice<T>(acc[j], xv[u][0], xv[u][1], wv[u][j]);
    }
  }
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<float2*>(&s_sum[warp][(g + 8 * i) * kRanks + j * 8 + c * 2]) = make_float2(acc[j][2 * i], acc[j][2 * i + 1]);
  }
  __syncthreads();
  for (int i = static_cast<int>(threadIdx.x); i < kFewRows * kRanks; i += kThreads) {
    float sum = s_sum[0][i];
#pragma unroll
    for (int v = 1; v < kWarps; ++v) sum += s_sum[v][i];
    s_sum[0][i] = sum;
  }
  leave_sums<T, kRanks, kFewRows>(a, tile, tile_number, rank, s_sum[0]);
}

__device__ __forceinline__ void copy16(std::uint32_t to, const void* from, bool there) {  // (zeros where there is nothing)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_are_one_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void wait_for_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
// Four 8 x 8 matrices of 16-bit elements, the rows of matrix i from the addresses of lanes 8 i to 8 i + 7.
__device__ __forceinline__ uint4 matrices(std::uint32_t addr) {
  uint4 r;
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
  return r;
}

// The same for many tokens: four warps of 32 rows each with all ranks, 64 channels at a time through three stages of shared memory, rows of 128 bytes whose
// 16-byte pieces are permuted by the row. (With the lanes' own pieces as operands, as above, each MMA had four moves beside it to bring its
// registers together: 8191 tokens, 4096 channels, rank 64: 30 us.)
template <int kNT>
constexpr int kShrinkStage = kManyRows * 128 + kNT * 8 * 128;
constexpr int kShrinkStages = 3;
template <typename T, int kNT>
__global__ void __launch_bounds__(kThreads) shrink_many_kernel(const LoraArgs a) {
  dependents_may_start();
  constexpr int kRanks = kNT * 8;
  extern __shared__ __align__(128) std::uint8_t smem[];
  const int tile_number = static_cast<int>(blockIdx.x) / a.parts, part = static_cast<int>(blockIdx.x) % a.parts;
  if (tile_number >= a.plan.head->tiles) return;
  const Tile tile = a.plan.tiles[tile_number];
  if (tile.adapter < 0) return;
  const int rank = rank_of(a, tile.adapter);
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32, g = lane / 4, c = lane % 4;
  // A thread copies piece tid % 8 of rows tid / 8, tid / 8 + 16, ...
  const int piece = tid % 8;
  const T* x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = tid / 8 + i * 16;
    x[i] = r < tile.count ? static_cast<const T*>(a.x) + a.plan.order[tile.first + r] * a.ldx + piece * 8 : nullptr;
  }
  const T* const w = static_cast<const T*>(a.a) + tile.adapter * a.a_adapter;
  const int from = part * a.slice, to = min(a.dim, from + a.slice), stages = max(0, (to - from + 63) / 64);
  const std::uint32_t ring = smem_u32(smem);
  const auto copy_stage = [&](int n) {
    if (n < stages) {
      const std::uint32_t at = ring + n % kShrinkStages * kShrinkStage<kNT> + (tid / 8) * 128 + ((piece ^ (tid / 8 & 7)) << 4);
      const int k = from + n * 64;
      const bool in = k + piece * 8 < to;
#pragma unroll
      for (int i = 0; i < 8; ++i) copy16(at + i * 2048, x[i] != nullptr && in ? x[i] + k : a.x, x[i] != nullptr && in);
#pragma unroll
      for (int i = 0; i < (kRanks + 15) / 16; ++i) {
        const int row = tid / 8 + i * 16;
        if (kRanks < 16 && row >= kRanks) continue;
        const bool there = in && row < rank;
        copy16(at + kManyRows * 128 + i * 2048, there ? w + row * a.a_row + k + piece * 8 : w, there);
      }
    }
    copies_are_one_group();
  };
#pragma unroll
  for (int i = 0; i < kShrinkStages - 1; ++i) copy_stage(i);
  float acc[2][kNT][4] = {};
  // Lane addresses within a stage: x as A operands (rows 0..7, 8..15, then the next 8 channels), A as B operands of two MMAs (8 channels, the next 8, then
  // the next 8 ranks).
  const int xr = warp * 32 + (lane & 15), xp = lane >> 4, wr = (lane >> 4) * 8 + (lane & 7), wp = lane >> 3 & 1;
  for (int n = 0; n < stages; ++n) {
    wait_for_copies<kShrinkStages - 2>();
    __syncthreads();  // (everybody's pieces of this stage are there, and the stage before is read)
    copy_stage(n + kShrinkStages - 1);
    const std::uint32_t at = ring + n % kShrinkStages * kShrinkStage<kNT>;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      uint4 xv[2];
#pragma unroll
      for (int m = 0; m < 2; ++m) xv[m] = matrices(at + (xr + m * 16) * 128 + (((2 * s + xp) ^ (xr & 7)) << 4));
#pragma unroll
      for (int j = 0; j < (kNT + 1) / 2; ++j) {
        const uint4 wv = matrices(at + kManyRows * 128 + ((kNT == 1 ? wr & 7 : wr) + j * 16) * 128 + (((2 * s + wp) ^ (wr & 7)) << 4));
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          mma<T>(acc[m][2 * j], xv[m], wv.x, wv.y);
          if constexpr (kNT > 1) mma<T>(acc[m][2 * j + 1], xv[m], wv.z, wv.w);
        }
      }
    }
  }
  __syncthreads();  // (the last stage is read)
  float* const sums = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int m = 0; m < 2; ++m) {
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<float2*>(sums + (warp * 32 + m * 16 + g + 8 * i) * kRanks + j * 8 + c * 2) = make_float2(acc[m][j][2 * i], acc[m][j][2 * i + 1]);
      }
    }
  }
  leave_sums<T, kRanks, kManyRows>(a, tile, tile_number, rank, sums);
}

// t of a warp's 16 rows as A operands.
template <typename T, int kNT>
struct Low {
  static constexpr int kPer = kNT <= 2 ? 4 : 8, kBlocks = kNT <= 2 ? 1 : kNT / 4, kSteps = kNT <= 2 ? 1 : kNT / 2;
  uint4 hi[kSteps], lo[kSteps];
  float back[2];
  __device__ __forceinline__ Low(const LoraArgs& a, std::int64_t row0, int g, int c) {
#pragma unroll
    for (int i = 0; i < 2; ++i) back[i] = a.t_back[row0 + g + 8 * i];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const std::int64_t at = (row0 / 16 * kSteps + s) * 32 + g * 4 + c;
      hi[s] = lo[s] = make_uint4(0, 0, 0, 0);
      if (c * kPer < kNT * 8) hi[s] = static_cast<const uint4*>(a.t_hi)[at], lo[s] = static_cast<const uint4*>(a.t_lo)[at];  // (8 ranks: the upper lanes have none)
    }
  }
};
// The elements of a word (two neighbouring ranks from `at`) that are used.
__device__ __forceinline__ std::uint32_t used(std::uint32_t w, int at, int rank) {
  return at + 1 < rank ? w : at < rank ? w & 0xffffu : 0u;
}

// t B^T added to 16 rows x 32 columns of the projection's output. Of the four MMAs beside one another each takes every other pair of the columns, so that a
// lane ends up with 8 neighbouring columns of two rows, one load and one store each. b(j, q): the lane's ranks of block q of column `column_of(j)`.
__device__ __forceinline__ int column_of(int j, int g) { return g / 2 * 8 + 2 * j + g % 2; }
// kRagged: the last piece of 8 ranks that are used has others behind them.
template <typename T, int kNT, bool kRagged, typename B>
__device__ __forceinline__ void add_block(const Low<T, kNT>& low, int c, int rank, const uint4 (&y)[2], const B& b, uint4 (&out)[2]) {
  using L = Low<T, kNT>;
  float acc[4][4] = {};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int q = 0; q < L::kBlocks; ++q) {
      uint4 v = b(j, q);
      if constexpr (kRagged) {  // (pieces of 8 ranks that are not used at all are zeros)
        const int at = q * 32 + c * L::kPer;
        v.x = used(v.x, at, rank), v.y = used(v.y, at + 2, rank);
        if constexpr (L::kPer == 8) v.z = used(v.z, at + 4, rank), v.w = used(v.w, at + 6, rank);
      }
      mma<T>(acc[j], low.hi[q * (L::kPer / 4)], v.x, v.y);
      mma<T>(acc[j], low.lo[q * (L::kPer / 4)], v.x, v.y);
      if constexpr (L::kPer == 8) {
        mma<T>(acc[j], low.hi[2 * q + 1], v.z, v.w);
        mma<T>(acc[j], low.lo[2 * q + 1], v.z, v.w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float v[8];
    load8<T>(y[i], v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[2 * j] = fmaf(acc[j][2 * i], low.back[i], v[2 * j]);
      v[2 * j + 1] = fmaf(acc[j][2 * i + 1], low.back[i], v[2 * j + 1]);
    }
    out[i] = store8<T>(v);
  }
}
// A warp's 16 rows of y and out, for a lane; rows of tokens without an adapter only move.
template <typename T>
struct OutRows {
  const T* y[2];
  T* out[2];
  bool there[2];
  __device__ __forceinline__ OutRows(const LoraArgs& a, const Tile& tile, int row0, int g, int c) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = row0 + g + 8 * i;
      there[i] = r < tile.count;
      const std::int64_t token = there[i] ? a.plan.order[tile.first + r] : 0;
      y[i] = static_cast<const T*>(a.y) + token * a.ldy + c * 8, out[i] = static_cast<T*>(a.out) + token * a.ldo + c * 8;
    }
  }
  __device__ __forceinline__ void move(int from, int to, int step, int c) const {
    for (int n = from; n < to; n += step) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (there[i] && n + c * 8 < to) *reinterpret_cast<uint4*>(out[i] + n) = load16(y[i] + n);
      }
    }
  }
};
// The tile of a CTA; one that has nothing to do says so.
__device__ __forceinline__ bool tile_to_add(const LoraArgs& a, Tile& tile) {
  const bool exists = static_cast<int>(blockIdx.x) < a.plan.head->tiles;
  if (exists) tile = a.plan.tiles[blockIdx.x];
  return exists && (tile.adapter >= 0 || a.y != a.out);
}

// Few tokens: a tile's warps take columns in turn, B comes straight from memory.
template <typename T, int kNT>
__global__ void __launch_bounds__(kThreads) expand_few_kernel(const LoraArgs a) {
  using L = Low<T, kNT>;
  constexpr int kStep = 32 * kWarps;
  Tile tile;
  if (!tile_to_add(a, tile)) {
    wait_for_predecessors();  // (this kernel is not done before the one that it follows)
    return;
  }
  const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32, g = lane / 4, c = lane % 4;
  const OutRows<T> rows(a, tile, 0, g, c);
  const int from = static_cast<int>(blockIdx.y) * a.columns + warp * 32, to = min(a.width, (static_cast<int>(blockIdx.y) + 1) * a.columns);
  if (tile.adapter < 0) {
    rows.move(from, to, kStep, c);
    wait_for_predecessors();
    return;
  }
  const int rank = rank_of(a, tile.adapter);
  const T* const w = static_cast<const T*>(a.b) + tile.adapter * a.b_adapter + c * L::kPer;
  wait_for_predecessors();
  const L low(a, static_cast<std::int64_t>(blockIdx.x) * kFewRows, g, c);
  const auto add_all = [&](auto ragged) {
    for (int n = from; n < to; n += kStep) {
      uint4 y[2], out[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) y[i] = rows.there[i] && n + c * 8 < to ? load16(rows.y[i] + n) : make_uint4(0, 0, 0, 0);
      add_block<T, kNT, decltype(ragged)::value>(low, c, rank, y, [&](int j, int q) {
        uint4 v = make_uint4(0, 0, 0, 0);
        const int column = n + column_of(j, g);
        if (column >= to || q * 32 + c * L::kPer >= rank) return v;
        const T* const p = w + column * a.b_row + q * 32;
        if constexpr (L::kPer == 8) {
          v = load16(p);
        } else {
          const uint2 r = *reinterpret_cast<const uint2*>(p);
          v.x = r.x, v.y = r.y;
        }
        return v;
      }, out);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (rows.there[i] && n + c * 8 < to) *reinterpret_cast<uint4*>(rows.out[i] + n) = out[i];
      }
    }
  };
  if (rank % 8 != 0) add_all(std::true_type{});
  else add_all(std::false_type{});
}

// Where a 16-byte piece of a row of 128 bytes lies so that eight lanes, four pieces of two rows, meet no bank twice: rows alike but for the
// bits that `fold` takes.
__device__ __forceinline__ int folded(int piece, int fold) { return (piece & ~7) | ((piece & 7) ^ fold); }

// Many: eight warps of 16 rows each, 32 columns at a time through four stages of shared memory: a lane copies the pieces of y that it adds to, B is
// everybody's. What bounds it is memory: y is read and out written once.
constexpr int kManyThreads = 256, kExpandStages = 4;
template <int kNT>
constexpr int kExpandStage = 32 * kNT * 16 + kManyRows * 64;
template <typename T, int kNT>
__global__ void __launch_bounds__(kManyThreads, kNT <= 8 ? 3 : 2) expand_many_kernel(const LoraArgs a) {
  using L = Low<T, kNT>;
  constexpr int kRanks = kNT * 8, kBBytes = 32 * kNT * 16;
  extern __shared__ __align__(128) std::uint8_t smem[];
  Tile tile;
  if (!tile_to_add(a, tile)) {
    wait_for_predecessors();  // (this kernel is not done before the one that it follows)
    return;
  }
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32, g = lane / 4, c = lane % 4;
  const OutRows<T> rows(a, tile, warp * 16, g, c);
  const int from = static_cast<int>(blockIdx.y) * a.columns, to = min(a.width, from + a.columns), steps = (to - from + 31) / 32;
  if (tile.adapter < 0) {
    rows.move(from, to, 32, c);
    wait_for_predecessors();
    return;
  }
  const int rank = rank_of(a, tile.adapter);
  const auto fold_of = [](int column) { return kNT >= 8 ? (column & 1) << 2 | (column >> 3 & 3) : 0; };
  // What this thread copies of B at each step: piece tid % kNT of column tid / kNT and of those kColumns on; where its own operands lie.
  constexpr int kColumns = kManyThreads / kNT < 32 ? kManyThreads / kNT : 32, kCopies = 32 / kColumns;
  const int column = tid / kNT, piece = tid % kNT;
  const bool copies = column < 32 && piece * 8 < rank;
  const T* w[kCopies];
  std::uint32_t w_to[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    w[i] = static_cast<const T*>(a.b) + tile.adapter * a.b_adapter + (from + column + i * kColumns) * a.b_row + piece * 8;
    w_to[i] = (column + i * kColumns) * (kNT * 16) + folded(piece, fold_of(column + i * kColumns)) * 16;
  }
  const std::int64_t w_step = 32 * a.b_row;
  const std::uint32_t ring = smem_u32(smem);
  const T* y_from[2] = {rows.y[0] + from, rows.y[1] + from};
  int to_copy = 0;
  const auto copy_step = [&] {
    if (to_copy < steps) {
      const std::uint32_t at = ring + to_copy % kExpandStages * kExpandStage<kNT>;
      const int left = to - from - to_copy * 32;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        copy16(at + kBBytes + ((warp * 2 + i) * 32 + lane) * 16, y_from[i], rows.there[i] && c * 8 < left);
        y_from[i] += 32;
      }
      if (column < 32) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          copy16(at + w_to[i], w[i], copies && column + i * kColumns < left);
          w[i] += w_step;
        }
      }
      ++to_copy;
    }
    copies_are_one_group();
  };
#pragma unroll
  for (int i = 0; i < kExpandStages - 1; ++i) copy_step();
  wait_for_predecessors();
  const L low(a, static_cast<std::int64_t>(blockIdx.x) * kManyRows + warp * 16, g, c);
  std::uint32_t b_from[4][L::kBlocks];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int q = 0; q < L::kBlocks; ++q) {
      const int n = column_of(j, g);
      b_from[j][q] = n * (kNT * 16) + (L::kPer == 8 ? folded(q * 4 + c, fold_of(n)) * 16 : c * 8);
    }
  }
  T* out_to[2] = {rows.out[0] + from, rows.out[1] + from};
  const auto add_all = [&](auto ragged) {
    for (int s = 0; s < steps; ++s) {
      wait_for_copies<kExpandStages - 2>();
      __syncthreads();  // (everybody's pieces of this step are there, and the step before is read)
      copy_step();
      const std::uint8_t* const at = smem + s % kExpandStages * kExpandStage<kNT>;
      uint4 y[2], out[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) y[i] = load16(at + kBBytes + ((warp * 2 + i) * 32 + lane) * 16);
      add_block<T, kNT, decltype(ragged)::value>(low, c, rank, y, [&](int j, int q) {
        if constexpr (L::kPer == 8) {
          return load16(at + b_from[j][q]);
        } else {
          if (c * 4 >= kRanks) return make_uint4(0, 0, 0, 0);
          const uint2 r = *reinterpret_cast<const uint2*>(at + b_from[j][q]);
          return make_uint4(r.x, r.y, 0, 0);
        }
      }, out);
      const bool in = c * 8 < to - from - s * 32;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (rows.there[i] && in) *reinterpret_cast<uint4*>(out_to[i]) = out[i];
        out_to[i] += 32;
      }
    }
  };
  if (rank % 8 != 0) add_all(std::true_type{});
  else add_all(std::false_type{});
}

inline int padded_tiles(int rank) {  // ranks / 8, up to a power of two
  int n = 1;
  while (n * 8 < rank) n *= 2;
  return n;
}
// Parts of the channels (a power of two): CTAs for the whole GPU twice (of few tokens) or three times over, of 256 channels at least.
inline int parts_of(std::int64_t tokens, int adapters, std::int64_t dim) {
  const std::int64_t tiles = most_tiles(tokens, adapters), room = (tokens <= kFewTokens ? 2 : 3) * 148;
  int parts = 1;
  while (parts < kMostParts && tiles * parts * 2 <= room && dim >= parts * 2 * 256) parts *= 2;
  return parts;
}
inline std::size_t rows_of(std::int64_t tokens, int adapters) { return static_cast<std::size_t>(most_tiles(tokens, adapters)) * tile_rows(tokens); }
inline std::size_t part_bytes(std::int64_t tokens, int adapters, int rank) {  // (an operand has 16 ranks at least)
  return (rows_of(tokens, adapters) * std::max(2, padded_tiles(rank)) * 16 + 255) / 256 * 256;
}
inline std::size_t workspace_bytes(std::int64_t tokens, int adapters, int rank) {
  return std::max<std::size_t>(256, 2 * part_bytes(tokens, adapters, rank) + rows_of(tokens, adapters) * 4);
}

template <typename T, int kNT>
int launch(const char* op, LoraArgs a, std::int64_t tokens, cudaStream_t stream) {
  const unsigned tiles = static_cast<unsigned>(most_tiles(tokens, a.adapters));
  const LaunchChain chain(stream);
  // Columns of a CTA: as many as leave 8 small or 4 large CTAs to an SM, 128 at least.
  const bool few = tokens <= kFewTokens;
  const std::int64_t most = std::max<std::int64_t>(1, (few ? 8LL : 4LL) * sm_count() / tiles);
  a.columns = static_cast<int>(std::max<std::int64_t>(128, ((a.width + most - 1) / most + 127) / 128 * 128));
  const dim3 grid(tiles, static_cast<unsigned>((a.width + a.columns - 1) / a.columns));
  if (few) {
    if (const int s = enqueue(op, shrink_few_kernel<T, kNT>, dim3(tiles * a.parts), dim3(kThreads), 0, stream, a.parts, a); s != B2_OK) return s;
    return enqueue(op, expand_few_kernel<T, kNT>, grid, dim3(kThreads), 0, stream, 1, a);
  }
  static std::atomic<std::uint64_t> shrink_done{0}, expand_done{0};
  constexpr int kShrinkBytes = kShrinkStages * kShrinkStage<kNT>, kExpandBytes = kExpandStages * kExpandStage<kNT>;
  if (const int s = allow_shared(op, shrink_many_kernel<T, kNT>, kShrinkBytes, shrink_done); s != B2_OK) return s;
  if (const int s = allow_shared(op, expand_many_kernel<T, kNT>, kExpandBytes, expand_done); s != B2_OK) return s;
  if (const int s = enqueue(op, shrink_many_kernel<T, kNT>, dim3(tiles * a.parts), dim3(kThreads), kShrinkBytes, stream, a.parts, a); s != B2_OK) return s;
  return enqueue(op, expand_many_kernel<T, kNT>, grid, dim3(kManyThreads), kExpandBytes, stream, 1, a);
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
  return workspace_bytes(tokens, adapters, rank);
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
  if (const int s = check_workspace(op, workspace, ws_bytes, workspace_bytes(tokens, l->adapters, l->rank)); s != B2_OK) return s;
  LoraArgs a{};
  a.plan = plan_at(plan, tokens, l->adapters);
  a.a = l->a, a.b = l->b, a.a_adapter = l->a_adapter_stride, a.a_row = l->a_row_stride, a.b_adapter = l->b_adapter_stride, a.b_row = l->b_row_stride;
  a.scales = l->scales, a.ranks = l->ranks, a.x = x, a.y = y, a.out = out, a.ldx = ldx, a.ldy = ldy, a.ldo = ldo;
  a.adapters = l->adapters, a.rank = l->rank, a.dim = static_cast<int>(l->dim), a.width = static_cast<int>(l->width);
  char* const at = static_cast<char*>(workspace);
  const std::size_t part = part_bytes(tokens, l->adapters, l->rank);
  a.t_hi = at, a.t_lo = at + part, a.t_back = reinterpret_cast<float*>(at + 2 * part);
  a.parts = parts_of(tokens, l->adapters, l->dim);
  a.slice = static_cast<int>(((l->dim + a.parts - 1) / a.parts + 63) / 64 * 64);
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
