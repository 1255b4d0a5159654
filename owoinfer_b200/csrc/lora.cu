// Low-rank adapters of many requests at once beside a projection that they share: the tokens sorted by adapter once for a step, then for each
// projection x A^T of every tile of tokens, split over the channels, and its product with B^T added to the projection's output.
#include <algorithm>
#include <cmath>

#include "attention.cuh"
#include "text.cuh"

namespace b2 {
namespace {

__device__ unsigned g_lora_status = 0;
enum LoraFault : unsigned { kLoraBadAdapter = 1, kLoraBadRank = 2, kLoraWait = 4, kLoraOtherPlan = 8 };  // (4: a bounded wait expired)

constexpr int kThreads = 128, kWarps = kThreads / 32;
constexpr int kPlanThreads = 1024;
constexpr int kMostAdapters = 4096, kMostRank = 128;
constexpr int kMostParts = 8, kMostManyParts = 4;  // CTAs of a cluster that divide the channels, of few and of many tokens

// A plan sorts the tokens by adapter and cuts them into tiles, of one warp's rows, where there are few tokens, and of eight warps', for A and B to be
// read once for more of them: [0] and [1] below.
constexpr int kFewRows = 16, kManyRows = 128, kFewTokens = 4096;
inline std::int64_t most_tiles(std::int64_t tokens, int adapters, int rows) {
  return rows == kFewRows && tokens > kFewTokens ? 0 : std::min(tokens, tokens / rows + adapters + 1);
}
struct alignas(16) PlanHead {
  int tiles[2], tokens, adapters;
};
struct Tile {
  int adapter, first, count, pad;  // -1: tokens without an adapter
};
struct Plan {
  PlanHead* head;
  Tile* tiles[2];
  std::int32_t* order;
};
inline std::size_t plan_bytes(std::int64_t tokens, int adapters) {
  const std::size_t tiles = static_cast<std::size_t>(most_tiles(tokens, adapters, kFewRows) + most_tiles(tokens, adapters, kManyRows));
  return (sizeof(PlanHead) + tiles * sizeof(Tile) + static_cast<std::size_t>(tokens) * 4 + 255) / 256 * 256;
}
inline Plan plan_at(void* p, std::int64_t tokens, int adapters) {
  char* at = static_cast<char*>(p);
  Tile* tiles = reinterpret_cast<Tile*>(at + sizeof(PlanHead));
  Tile* large = tiles + most_tiles(tokens, adapters, kFewRows);
  return {reinterpret_cast<PlanHead*>(at), {tiles, large}, reinterpret_cast<std::int32_t*>(large + most_tiles(tokens, adapters, kManyRows))};
}
// What a kernel reads of it: one kind of tiles.
struct Tiles {
  const PlanHead* head;
  const Tile* tiles;
  const std::int32_t* order;
  int tokens, adapters, kind;  // kind: which tiles
  // How many; none of a plan of other tokens or adapters, whose tiles lie elsewhere.
  __device__ __forceinline__ int count() const {
    const int4 h = *reinterpret_cast<const int4*>(head);
    if (h.z == tokens && h.w == adapters) return kind == 0 ? h.x : h.y;
    atomicOr(&g_lora_status, kLoraOtherPlan);
    return 0;
  }
};

// A CTA per adapter, and one for the tokens without: each counts all tokens by adapter (a thread a run of neighbouring tokens, which mostly have
// the same one), and puts its own in their places, in their order.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const std::int32_t* ids, int tokens, int adapters, const Plan plan) {
  extern __shared__ int s_count[];  // [adapters + 1]
  __shared__ int s_warp[kPlanThreads / 32], s_before[3];
  const int tid = static_cast<int>(threadIdx.x), own = static_cast<int>(blockIdx.x);
  for (int i = tid; i <= adapters; i += kPlanThreads) s_count[i] = 0;
  if (tid < 3) s_before[tid] = 0;
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
  int tokens_before = 0, tiles_before[2] = {};
  for (int i = tid; i < own; i += kPlanThreads) {
    tokens_before += s_count[i], tiles_before[0] += (s_count[i] + kFewRows - 1) / kFewRows, tiles_before[1] += (s_count[i] + kManyRows - 1) / kManyRows;
  }
  if (tokens_before > 0) atomicAdd(&s_before[0], tokens_before), atomicAdd(&s_before[1], tiles_before[0]), atomicAdd(&s_before[2], tiles_before[1]);
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
      if (id_of(i) == own) plan.order[place++] = i;
    }
  }
  const int count = s_count[own];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int rows = k == 0 ? kFewRows : kManyRows, num = (count + rows - 1) / rows;
    if (k == 0 && tokens > kFewTokens) continue;
    for (int i = tid; i < num; i += kPlanThreads) {
      plan.tiles[k][s_before[1 + k] + i] = Tile{own < adapters ? own : -1, s_before[0] + i * rows, min(rows, count - i * rows), 0};
    }
    if (own == adapters && tid == 0) plan.head->tiles[k] = s_before[1 + k] + num, plan.head->tokens = tokens, plan.head->adapters = adapters;
  }
}

struct LowWords {
  std::uint32_t* hi;
  std::uint32_t* lo;
  float* back;
};
struct LoraArgs {
  Tiles plan;
  const void* a;
  const void* b;
  std::int64_t a_adapter, a_row, b_adapter, b_row;
  const float* scales;
  const std::int32_t* ranks;
  const void* x;
  const void* y;
  void* out;
  std::int64_t ldx, ldy, ldo;
  // Of several tokens: t = scale x A^T, by [tile, row of the tile], in two 16-bit parts in operand order, and what a row was divided by.
  LowWords low;
  int rank, dim, width;
  int parts, slice;  // parts of the channels, channels of each (a multiple of 64)
  int columns;        // columns of an output CTA
  int groups;         // clusters to a tile
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
__device__ __forceinline__ uint4 load16(const void* p) { return *reinterpret_cast<const uint4*>(p); }

__device__ __forceinline__ int rank_of(const LoraArgs& a, int adapter) {
  if (a.ranks == nullptr) return a.rank;
  const int r = a.ranks[adapter];
  if (r >= 0 && r <= a.rank) return r;
  atomicOr(&g_lora_status, kLoraBadRank);
  return r < 0 ? 0 : a.rank;
}

// fp32 values of a row, the largest of them `top`, as two 16-bit parts. fp16 ends at 2^16 and loses bits below 2^-14: there the largest is brought between
// 2^14 and 2^15 by a power of two, which `back` undoes. (Where it is an infinity the others may be any number: 2^-114 keeps them below one.)
template <typename T>
struct Halves {
  float by = 1.f, back = 1.f;
  __device__ __forceinline__ explicit Halves(float top) {
    if constexpr (std::is_same<T, __half>::value) {
      const int e = max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14, -100);
      by = __uint_as_float(static_cast<unsigned>(127 - e) << 23), back = __uint_as_float(static_cast<unsigned>(127 + e) << 23);
    }
  }
  __device__ __forceinline__ void split(float x, float y, std::uint32_t& hi, std::uint32_t& lo) const {
    if constexpr (std::is_same<T, __half>::value) x *= by, y *= by;
    hi = pack16<T>(x, y);
    float xh, yh;
    unpack16<T>(hi, xh, yh);
    lo = pack16<T>(isfinite(xh) ? x - xh : 0.f, isfinite(yh) ? y - yh : 0.f);
  }
};

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
// B, as rows from `to_row` of an operand: a row by ranks / 4 neighbouring lanes, rows first, first + step, ... (Rows behind the tile's tokens are left out: what
// t has there ends up in rows that nobody stores.) In two 16-bit parts t keeps 16 (bf16) or 22 (fp16) of its bits.
template <typename T, int kRanks>
__device__ __forceinline__ void leave_sums(const LoraArgs& a, const Tile& tile, int rank, const float* sums, int first, int step, const LowWords& to, std::int64_t to_row) {
  constexpr int kLanes = kRanks / 4;
  const int lane = static_cast<int>(threadIdx.x) % kLanes;
  const float scale = a.scales != nullptr ? a.scales[tile.adapter] : 1.f;
  const std::uint32_t own = smem_u32(sums);
  for (; first < tile.count; first += step) {  // (the same number of rounds for a warp's lanes)
    const int row = first + static_cast<int>(threadIdx.x) / kLanes;
    float v[4] = {};
    if (row < tile.count) {
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
    if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int m = kLanes / 2; m > 0; m /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    }
    if (row >= tile.count) continue;
    const Halves<T> by(top);
    std::uint32_t hi[2], lo[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) by.split(v[2 * e], v[2 * e + 1], hi[e], lo[e]);
    const std::int64_t word = low_word<kRanks>(to_row + row, lane * 4);
    to.hi[word] = hi[0], to.hi[word + 2] = hi[1], to.lo[word] = lo[0], to.lo[word + 2] = lo[1];
    if (lane == 0) to.back[to_row + row] = by.back;
  }
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

// Several tokens: x A^T of a tile over a part of the channels, the ranks as columns, kNT: ranks / 8, up to a power of two. Four warps of 32 rows each with all ranks, 64
// channels at a time through three stages of shared memory, rows of 128 bytes whose 16-byte pieces are permuted by the row. (With operands straight
// from memory each MMA had four moves beside it to bring its registers together: 8191 tokens, 4096 channels, rank 64: 30 us.) What bounds it is memory and, between
// its copies and its last MMA, latency: 3000 tokens of 4 adapters, 4096 to 4096, rank 32 take 24 us with the kernel behind it, twice what their bytes take.
template <int kNT>
constexpr int kShrinkStage = kManyRows * 128 + kNT * 8 * 128;
constexpr int kShrinkStages = 3;
template <typename T, int kNT>
__global__ void __launch_bounds__(kThreads) shrink_several_kernel(const LoraArgs a) {
  dependents_may_start();
  constexpr int kRanks = kNT * 8;
  extern __shared__ __align__(128) std::uint8_t smem[];
  const int tile_number = static_cast<int>(blockIdx.x) / a.parts, part = static_cast<int>(blockIdx.x) % a.parts;
  if (tile_number >= a.plan.count()) return;
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
  if (a.parts > 1) cluster_sync_all();
  else __syncthreads();
  constexpr int kRound = kThreads / (kRanks / 4);
  leave_sums<T, kRanks>(a, tile, rank, sums, part * kRound, a.parts * kRound, a.low, static_cast<std::int64_t>(tile_number) * kManyRows);
  if (a.parts > 1) cluster_sync_all();  // (nobody leaves while others read its sums)
}

// t of a warp's 16 rows as A operands.
template <typename T, int kNT>
struct Low {
  static constexpr int kPer = kNT <= 2 ? 4 : 8, kBlocks = kNT <= 2 ? 1 : kNT / 4, kSteps = kNT <= 2 ? 1 : kNT / 2;
  uint4 hi[kSteps], lo[kSteps];
  float back[2];
  __device__ __forceinline__ Low(const LowWords& from, std::int64_t row0, int g, int c) {
#pragma unroll
    for (int i = 0; i < 2; ++i) back[i] = from.back[row0 + g + 8 * i];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const std::int64_t at = (row0 / 16 * kSteps + s) * 32 + g * 4 + c;
      hi[s] = lo[s] = make_uint4(0, 0, 0, 0);
      if (c * kPer < kNT * 8) hi[s] = reinterpret_cast<const uint4*>(from.hi)[at], lo[s] = reinterpret_cast<const uint4*>(from.lo)[at];  // (8 ranks: the upper lanes have none)
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
  const bool exists = static_cast<int>(blockIdx.x) < a.plan.count();
  if (exists) tile = a.plan.tiles[blockIdx.x];
  return exists && (tile.adapter >= 0 || a.y != a.out);
}

// Where a 16-byte piece of a row of 128 bytes lies so that eight lanes, four pieces of two rows, meet no bank twice: rows alike but for the
// bits that `fold` takes.
__device__ __forceinline__ int folded(int piece, int fold) { return (piece & ~7) | ((piece & 7) ^ fold); }

// Of 16 bytes of 8 ranks of a column, of 32 columns.
template <int kNT>
__device__ __forceinline__ int fold_of(int column) { return kNT >= 8 ? (column & 1) << 2 | (column >> 3 & 3) : 0; }
// Where a lane's operands of a step lie among its B.
template <typename T, int kNT>
__device__ __forceinline__ void place_operands(int g, int c, std::uint32_t (&at)[4][Low<T, kNT>::kBlocks]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int q = 0; q < Low<T, kNT>::kBlocks; ++q) {
      const int n = column_of(j, g);
      at[j][q] = n * (kNT * 16) + (Low<T, kNT>::kPer == 8 ? folded(q * 4 + c, fold_of<kNT>(n)) * 16 : c * 8);
    }
  }
}
template <typename T, int kNT>
__device__ __forceinline__ uint4 operand(const std::uint8_t* p, int c) {
  if constexpr (Low<T, kNT>::kPer == 8) {
    return load16(p);
  } else {
    if (c * 4 >= kNT * 8) return make_uint4(0, 0, 0, 0);
    const uint2 r = *reinterpret_cast<const uint2*>(p);
    return make_uint4(r.x, r.y, 0, 0);
  }
}

// Few tokens: 16 of a tile in one kernel. A cluster of CTAs divides the channels, then the columns; a CTA's warps take 64 of its channels each in turn, are
// added up with each other and with the other CTAs' through distributed shared memory, and take 32 of its columns each in turn. A, x, B and y come through
// stages of shared memory of each warp, the first of B and y ahead of A's last. What bounds it is latency, and how much of A and B is on its way.
// Where tiles are few several clusters share one: each makes the tile's sums and has some of the columns. One token of rank 16, 2048 to 2048, takes 4.1 us, 64 of as many
// users, 48 adapters, 4096 to 6144, 7.3, from memory 11 (their bytes: 1.2). (As two kernels 1.7 from memory more, and another launch of 2.5 us for the host.)
template <int kNT>
struct FewShape {
  static constexpr int kRanks = kNT * 8;
  static constexpr int kStageA = (kFewRows + kRanks) * 128, kStagesA = kNT <= 4 ? 3 : kNT <= 8 ? 2 : 1, kRingA = kStagesA * kStageA;
  // Of B's stages so many are its own, the others lie where A's were: two CTAs fit an SM. (With more on its way but one CTA to an SM, us: 64 users of 32 ranks
  // 17 for 11, 300 tokens of 3 adapters of 128 ranks 31 for 21.)
  static constexpr int kBBytes = 32 * kNT * 16, kStageB = kBBytes + 1024, kStagesB = kNT <= 8 ? 4 : 2, kOwnB = kNT <= 2 ? 4 : kNT <= 4 ? 2 : kNT <= 8 ? 1 : 0, kRingB = kOwnB * kStageB;
  static constexpr int kSumBytes = kFewRows * kRanks * 4, kLowBytes = kFewRows * (kRanks < 16 ? 16 : kRanks) * 2;  // of the sums, of one of t's parts
  static constexpr int kSums = kWarps * (kRingA + kRingB), kLow = kSums + kSumBytes, kBytes = kLow + 2 * kLowBytes + kFewRows * 4;
  static_assert((kStagesB - kOwnB) * kStageB <= kRingA && kSumBytes <= kRingA, "some of B's stages, and a warp's sums, lie in its stages of A");
};
template <typename T, int kNT>
__global__ void __launch_bounds__(kThreads) few_kernel(const LoraArgs a) {
  using S = FewShape<kNT>;
  constexpr int kRanks = S::kRanks;
  extern __shared__ __align__(128) std::uint8_t smem[];
  const int part = static_cast<int>(blockIdx.x) % a.parts, group = static_cast<int>(blockIdx.x) / a.parts % a.groups;
  const int tile_number = static_cast<int>(blockIdx.x) / a.parts / a.groups;
  if (tile_number >= a.plan.count()) return;
  const Tile tile = a.plan.tiles[tile_number];
  if (tile.adapter < 0 && a.y == a.out) return;
  const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32, g = lane / 4, c = lane % 4;
  constexpr int kStep = 32 * kWarps;
  const OutRows<T> rows(a, tile, 0, g, c);
  const int first = min(a.width, (group * a.parts + part) * a.columns), from = first + warp * 32, to = min(a.width, first + a.columns);
  if (tile.adapter < 0) {
    rows.move(from, to, kStep, c);
    return;
  }
  const int rank = rank_of(a, tile.adapter);

  // Of A and x a lane copies piece lane % 8 of rows lane / 8, lane / 8 + 4, ...: 64 channels, rows of 128 bytes whose pieces are permuted by the row.
  const int piece = lane % 8;
  const T* x[kFewRows / 4];
#pragma unroll
  for (int i = 0; i < kFewRows / 4; ++i) {
    const int r = lane / 8 + i * 4;
    x[i] = r < tile.count ? static_cast<const T*>(a.x) + a.plan.order[tile.first + r] * a.ldx + piece * 8 : nullptr;
  }
  const T* const wa = static_cast<const T*>(a.a) + tile.adapter * a.a_adapter + lane / 8 * a.a_row + piece * 8;
  const int from_k = part * a.slice, to_k = min(a.dim, from_k + a.slice);
  const std::uint32_t ring_a = smem_u32(smem) + warp * S::kRingA;
  int next_k = from_k + warp * 64, copied_a = 0;
  const auto copy_a = [&] {
    if (next_k < to_k) {
      const std::uint32_t at = ring_a + copied_a * S::kStageA + lane / 8 * 128;
      const bool in = next_k + piece * 8 < to_k;
      const auto piece_at = [&](int i) { return at + i * 512 + ((piece ^ (lane / 8 + i * 4 & 7)) << 4); };
#pragma unroll
      for (int i = 0; i < kRanks / 4; ++i) {
        const bool there = in && lane / 8 + i * 4 < rank;
        copy16(piece_at(i), there ? wa + i * 4 * a.a_row + next_k : wa, there);
      }
#pragma unroll
      for (int i = 0; i < kFewRows / 4; ++i) copy16(piece_at(kRanks / 4 + i), x[i] != nullptr && in ? x[i] + next_k : a.x, x[i] != nullptr && in);
      next_k += 64 * kWarps;
      copied_a = copied_a == S::kStagesA - 1 ? 0 : copied_a + 1;
    }
    copies_are_one_group();
  };
  // Of B piece lane % kNT of column lane / kNT and of those kColumns on, of y the pieces that it adds to.
  constexpr int kColumns = 32 / kNT;
  const int b_column = lane / kNT, b_piece = lane % kNT;
  const T* const wb = static_cast<const T*>(a.b) + tile.adapter * a.b_adapter + b_column * a.b_row + b_piece * 8;
  std::uint8_t* const rings[2] = {smem + kWarps * S::kRingA + warp * S::kRingB, smem + warp * S::kRingA};
  const auto stage_b = [&](int i) { return i < S::kOwnB ? rings[0] + i * S::kStageB : rings[1] + (i - S::kOwnB) * S::kStageB; };
  int next_n = from, copied_b = 0;
  const auto copy_b = [&] {
    if (next_n < to) {
      const std::uint32_t at = smem_u32(stage_b(copied_b));
#pragma unroll
      for (int i = 0; i < kNT; ++i) {
        const int n = b_column + i * kColumns;
        const bool in = b_piece * 8 < rank && next_n + n < to;
        copy16(at + n * (kNT * 16) + folded(b_piece, fold_of<kNT>(n)) * 16, in ? wb + (next_n + i * kColumns) * a.b_row : a.b, in);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const bool in = rows.there[i] && next_n + c * 8 < to;
        copy16(at + S::kBBytes + (i * 32 + lane) * 16, in ? rows.y[i] + next_n : a.y, in);
      }
      next_n += kStep;
      copied_b = copied_b == S::kStagesB - 1 ? 0 : copied_b + 1;
    }
    copies_are_one_group();
  };
#pragma unroll
  for (int i = 0; i < S::kStagesA; ++i) copy_a();
#pragma unroll
  for (int i = 0; i < S::kOwnB; ++i) copy_b();

  float acc[kNT][4] = {};
  {
    // Lane addresses within a stage: A as B operands of two MMAs (8 channels, the next 8, then the next 8 ranks), x as A operands (rows 0..7, 8..15, then
    // the next 8 channels).
    const int wr = (lane >> 4) * 8 + (lane & 7), wp = lane >> 3 & 1, xr = lane & 15, xp = lane >> 4;
    int stage = 0, number = 0;
    for (int k = from_k + warp * 64; k < to_k; k += 64 * kWarps, ++number) {
      if (number < S::kStagesA) wait_for_copies<S::kStagesA + S::kOwnB - 1>();  // (B's first stages are behind these)
      else wait_for_copies<S::kStagesA - 1>();
      __syncwarp();  // (the warp's pieces of this stage are there)
      const std::uint32_t at = ring_a + stage * S::kStageA;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint4 xv = matrices(at + kRanks * 128 + xr * 128 + (((2 * s + xp) ^ (xr & 7)) << 4));
#pragma unroll
        for (int j = 0; j < (kNT + 1) / 2; ++j) {
          const uint4 wv = matrices(at + ((kNT == 1 ? wr & 7 : wr) + j * 16) * 128 + (((2 * s + wp) ^ (wr & 7)) << 4));
          mma<T>(acc[2 * j], xv, wv.x, wv.y);
          if constexpr (kNT > 1) mma<T>(acc[2 * j + 1], xv, wv.z, wv.w);
        }
      }
      __syncwarp();  // (the stage is read)
      copy_a();
      stage = stage == S::kStagesA - 1 ? 0 : stage + 1;
    }
  }
  wait_for_copies<0>();
  __syncwarp();
  constexpr int kNext = S::kRingA / 4;  // floats from a warp's sums to the next one's
  float* const own = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int j = 0; j < kNT; ++j) {
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<float2*>(own + warp * kNext + (g + 8 * i) * kRanks + j * 8 + c * 2) = make_float2(acc[j][2 * i], acc[j][2 * i + 1]);
  }
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(smem + S::kSums);
  for (int i = static_cast<int>(threadIdx.x); i < tile.count * kRanks; i += kThreads) {
    float sum = own[i];
#pragma unroll
    for (int v = 1; v < kWarps; ++v) sum += own[v * kNext + i];
    sums[i] = sum;
  }
  if (a.parts > 1) cluster_sync_all();
  else __syncthreads();
#pragma unroll
  for (int i = S::kOwnB; i < S::kStagesB; ++i) copy_b();
  std::uint8_t* const t = smem + S::kLow;
  const LowWords words{reinterpret_cast<std::uint32_t*>(t), reinterpret_cast<std::uint32_t*>(t + S::kLowBytes), reinterpret_cast<float*>(t + 2 * S::kLowBytes)};
  leave_sums<T, kRanks>(a, tile, rank, sums, 0, kThreads / (kRanks / 4), words, 0);
  __syncthreads();
  if (a.parts > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // (it has read the others' sums)

  const Low<T, kNT> low(words, 0, g, c);
  std::uint32_t b_from[4][Low<T, kNT>::kBlocks];
  place_operands<T, kNT>(g, c, b_from);
  const auto add_all = [&](auto ragged) {
    int stage = 0;
    for (int n = from; n < to; n += kStep) {
      wait_for_copies<S::kStagesB - 1>();
      __syncwarp();  // (the warp's pieces of this step are there)
      const std::uint8_t* const at = stage_b(stage);
      uint4 y[2], out[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) y[i] = load16(at + S::kBBytes + (i * 32 + lane) * 16);
      add_block<T, kNT, decltype(ragged)::value>(low, c, rank, y, [&](int j, int q) { return operand<T, kNT>(at + b_from[j][q], c); }, out);
      __syncwarp();  // (the stage is read)
      copy_b();
      stage = stage == S::kStagesB - 1 ? 0 : stage + 1;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (rows.there[i] && n + c * 8 < to) *reinterpret_cast<uint4*>(rows.out[i] + n) = out[i];
      }
    }
  };
  if (rank % 8 != 0) add_all(std::true_type{});
  else add_all(std::false_type{});
  wait_for_copies<0>();
  if (a.parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // (nobody leaves while others read its sums)
}

// Several: eight warps of 16 rows each, 32 columns at a time through four stages of shared memory: a lane copies the pieces of y that it adds to, B is
// everybody's. What bounds it is memory: y is read and out written once.
constexpr int kManyThreads = 256, kExpandStages = 4;
template <int kNT>
constexpr int kExpandStage = 32 * kNT * 16 + kManyRows * 64;
template <typename T, int kNT>
__global__ void __launch_bounds__(kManyThreads, kNT <= 8 ? 3 : 2) expand_several_kernel(const LoraArgs a) {
  using L = Low<T, kNT>;
  constexpr int kBBytes = 32 * kNT * 16;
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
  // What this thread copies of B at each step: piece tid % kNT of column tid / kNT and of those kColumns on; where its own operands lie.
  constexpr int kColumns = kManyThreads / kNT < 32 ? kManyThreads / kNT : 32, kCopies = 32 / kColumns;
  const int column = tid / kNT, piece = tid % kNT;
  const bool copies = column < 32 && piece * 8 < rank;
  const T* w[kCopies];
  std::uint32_t w_to[kCopies];
#pragma unroll
  for (int i = 0; i < kCopies; ++i) {
    w[i] = static_cast<const T*>(a.b) + tile.adapter * a.b_adapter + (from + column + i * kColumns) * a.b_row + piece * 8;
    w_to[i] = (column + i * kColumns) * (kNT * 16) + folded(piece, fold_of<kNT>(column + i * kColumns)) * 16;
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
  const L low(a.low, static_cast<std::int64_t>(blockIdx.x) * kManyRows + warp * 16, g, c);
  std::uint32_t b_from[4][L::kBlocks];
  place_operands<T, kNT>(g, c, b_from);
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
      add_block<T, kNT, decltype(ragged)::value>(low, c, rank, y, [&](int j, int q) { return operand<T, kNT>(at + b_from[j][q], c); }, out);
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

// What the kernels of many tokens share: a bounded wait that gave up, barriers of MMAs, where the accumulators are.
struct Tensor {
  std::uint64_t done[4];
  std::uint32_t memory;
  int abort;
};
template <int kColumns>
__device__ __forceinline__ void begin_tensor(Tensor& s) {
  if (threadIdx.x / 32 == 0) {
    tmem_alloc(smem_u32(&s.memory), kColumns);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    s.abort = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&s.done[i]), 1);
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
// Frees the tensor memory once everybody is done with it. A wait that expired is reported; what was issued has had time to end by then.
template <int kColumns>
__device__ __forceinline__ void end_tensor(Tensor& s) {
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (s.abort != 0) {
    if (threadIdx.x == 0) atomicOr(&g_lora_status, kLoraWait);
    const std::uint64_t t0 = global_ns();
    while (global_ns() - t0 < 2000000ull) {
    }
  }
  if (threadIdx.x / 32 == 0) tmem_dealloc(s.memory, kColumns);
}

// Many tokens: 128 of a tile in one kernel, both products by tcgen05. A cluster of CTAs divides the channels, then the columns: each adds up x A^T over its
// own channels (64 at a time), they exchange the sums through distributed shared memory, and each adds t B^T to its own columns of y (64 at a time), t in
// tensor memory in its two 16-bit parts. Both kinds of steps run through the same stages of shared memory, rows of 128 bytes with the 128-byte swizzle,
// so that y and B are on their way while the sums are exchanged. A tile's tokens need not be neighbours, so that the threads copy the rows, piece by
// piece. Where tiles are few several clusters share one: each makes the tile's sums and has some of the columns. Memory should bound it (x and y are read, out written):
// 8191 tokens of 6 adapters, 4096 to 4096, rank 64 take 64 us, half of a copy's rate; a CTA's parts, the exchange among them, do not overlap each other.
// (As two kernels, x A^T left in global memory: 8191 tokens, 4096 to 4096, rank 64: 71 us, on mma.sync, whose rate is a quarter, 69.)
template <int kNT>
struct ManyShape {
  static_assert(kNT >= 8, "ranks above 32 only: way_of()");
  static constexpr int kN = kNT * 8;                                              // ranks of an MMA
  static constexpr int kOperand = kN > 64 ? 128 * 128 : 64 * 128;                 // of a step: A's ranks by 64 channels, or B's 64 columns by its ranks
  static constexpr int kStage = kOperand + kManyRows * 128, kStages = kN > 64 ? 3 : 4;
  // Tensor memory: accumulators (of x A^T, then of two steps' t B^T), from kLow on t. Two CTAs of an SM have all of it; a kernel of the framework that
  // allocates some and waits for its neighbours has more than half of the shared memory, and does not fit beside one: no two wait for one another.
  static constexpr int kLow = 128, kColumns = 256;
  static constexpr int kBytes = kStages * kStage + 1024;                          // and what aligns it
  // The sums that are exchanged: blocks of ranks, 16 KB each, as many to a stage as two stages take them all.
  static constexpr int kBlock = 32, kBlocks = kN / kBlock, kPerStage = kBlocks / 2;
  static_assert(kManyRows * kBlock * 4 * kPerStage <= kStage && kManyRows * kN * 2 <= kStage, "the sums, then t's parts, lie in two stages' places");
};
template <typename T, int kNT>
__global__ void __launch_bounds__(kManyThreads, 2) many_kernel(const LoraArgs a) {
  using S = ManyShape<kNT>;
  extern __shared__ std::uint8_t smem_raw[];
  __shared__ Tensor sh;
  __shared__ float s_back[kManyRows];
  const int part = static_cast<int>(blockIdx.x) % a.parts, group = static_cast<int>(blockIdx.x) / a.parts % a.groups;
  const int tile_number = static_cast<int>(blockIdx.x) / a.parts / a.groups;
  if (tile_number >= a.plan.count()) return;
  const Tile tile = a.plan.tiles[tile_number];
  if (tile.adapter < 0 && a.y == a.out) return;
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32;
  const int from_k = part * a.slice, to_k = min(a.dim, from_k + a.slice), k_steps = a.slice / 64;  // (as many for every part)
  const int from = min(a.width, (group * a.parts + part) * a.columns), to = min(a.width, from + a.columns), steps = k_steps + (to - from + 63) / 64;
  // A warp has 32 rows of the tile and one half of a step's 128 bytes of each. Lane l moves piece l % 4 of rows l / 4, l / 4 + 8, l / 4 + 16, l / 4 + 24.
  const int row0 = warp % 4 * 32, half = warp / 4, column = half * 32 + lane % 4 * 8;
  const T* x_from[4];
  const T* y_from[4];
  T* out_to[4];
  bool there[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = row0 + lane / 4 + i * 8;
    there[i] = r < tile.count;
    const std::int64_t token = there[i] ? a.plan.order[tile.first + r] : 0;
    x_from[i] = static_cast<const T*>(a.x) + token * a.ldx + from_k + column;
    y_from[i] = static_cast<const T*>(a.y) + token * a.ldy + from + column, out_to[i] = static_cast<T*>(a.out) + token * a.ldo + from + column;
  }
  if (tile.adapter < 0) {  // (they only move)
    for (int n = 0; n < to - from; n += 64) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (there[i] && n + column < to - from) *reinterpret_cast<uint4*>(out_to[i] + n) = load16(y_from[i] + n);
      }
    }
    return;
  }
  const int rank = rank_of(a, tile.adapter);
  std::uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const std::uint32_t ring = smem_u32(smem);
  const T* const wa = static_cast<const T*>(a.a) + tile.adapter * a.a_adapter + from_k;
  const T* const wb = static_cast<const T*>(a.b) + tile.adapter * a.b_adapter + from * a.b_row;
  const auto at_piece = [](int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); };
  constexpr int kPieces = S::kN / 8;
  const auto copy_step = [&](int s) {
    if (s < steps) {
      const std::uint32_t at = ring + s % S::kStages * S::kStage;
      const bool first = s < k_steps;
      const int n = (first ? s : s - k_steps) * 64, left = (first ? to_k - from_k : to - from) - n;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = there[i] && column < left;
        copy16(at + S::kOperand + at_piece(row0 + lane / 4 + i * 8, half * 4 + lane % 4), in ? (first ? x_from[i] : y_from[i]) + n : a.x, in);
      }
      if (first) {
#pragma unroll
        for (int i = 0; i < S::kN * 8 / kManyThreads; ++i) {
          const int row = tid / 8 + i * (kManyThreads / 8), piece = tid % 8;
          const bool in = row < rank && piece * 8 < left;
          copy16(at + at_piece(row, piece), in ? wa + row * a.a_row + n + piece * 8 : wa, in);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 64 * kPieces / kManyThreads; ++i) {
          const int j = tid + i * kManyThreads, row = j / kPieces, piece = j % kPieces;
          const bool in = row < left && piece * 8 < rank;
          copy16(at + piece / 8 * (64 * 128) + at_piece(row, piece & 7), in ? wb + (n + row) * a.b_row + piece * 8 : wb, in);
        }
      }
    }
    copies_are_one_group();
  };
  // The two stages that are free last ahead of the exchange stay free until it is over.
  const int held = k_steps + S::kStages - 2;
#pragma unroll
  for (int i = 0; i < S::kStages; ++i) {
    if (i < held) copy_step(i);
  }
  begin_tensor<S::kColumns>(sh);
  const std::uint32_t lanes = static_cast<std::uint32_t>(row0) << 16, accumulators = sh.memory, low = sh.memory + S::kLow;
  constexpr int kFormat = std::is_same<T, __half>::value ? 0 : 1;
  constexpr std::uint32_t idesc_a = umma_idesc(/*f32*/ 1, kFormat, kFormat, 0, 0, kManyRows, S::kN), idesc_b = umma_idesc(1, kFormat, kFormat, 0, 0, kManyRows, 64);
  bool lost = false;
  const auto wait_done = [&](int s) {  // the MMAs of step s
    if (!lost) lost = !warp_wait_bar(smem_u32(&sh.done[s % S::kStages]), static_cast<std::uint32_t>(s / S::kStages) & 1u, &sh.abort);
    tc_fence_after();
  };
  const auto copies_are_there = [&] {  // of the step that is next; everybody's
    wait_for_copies<S::kStages - 2>();
    fence_proxy_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  };
  for (int s = 0; s < k_steps; ++s) {
    copies_are_there();
    if (warp == 0 && elect_one()) {
      const std::uint32_t at = ring + s % S::kStages * S::kStage;
      const std::uint64_t dx = umma_desc_sw128(at + S::kOperand), dw = umma_desc_sw128(at);
#pragma unroll
      for (std::uint32_t i = 0; i < 4; ++i) umma_f16(accumulators, dx + 2 * i, dw + 2 * i, idesc_a, static_cast<std::uint32_t>(s) + i);
      tc_commit(smem_u32(&sh.done[s % S::kStages]));
    }
    if (s > 0) {
      wait_done(s - 1);
      if (s - 1 + S::kStages < held) copy_step(s - 1 + S::kStages);
    }
  }
  wait_done(k_steps - 1);

  // The sums of all parts, joined by every CTA for itself: lanes side by side read a row's neighbouring ranks. (A thread a row, 144 bytes from the next
  // thread's, took 25 us of reads from the other CTAs' shared memory.)
  float back;
  {
    constexpr int kRowBytes = S::kBlock * 4, kLanes = S::kBlock / 4, kRows = kManyThreads / kLanes, kRounds = kManyRows / kRows;
    const auto stage_of = [&](int i) { return smem + (k_steps + S::kStages - 1 - i) % S::kStages * S::kStage; };
    const auto sum_at = [&](int b, int row, int piece) { return stage_of(b / S::kPerStage) + b % S::kPerStage * (kManyRows * kRowBytes) + row * kRowBytes + (piece ^ (row & 7)) * 16; };
#pragma unroll
    for (int b = half; b < S::kBlocks; b += 2) {
      std::uint32_t r[S::kBlock];
      tmem_ld_32x32(accumulators + lanes + b * S::kBlock, r);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < kLanes; ++i) *reinterpret_cast<uint4*>(sum_at(b, row0 + lane, i)) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
    }
    if (a.parts > 1) cluster_sync_all();
    else __syncthreads();
    const float scale = a.scales != nullptr ? a.scales[tile.adapter] : 1.f;
    const int piece = tid % kLanes;
    float v[kRounds][S::kBlocks][4];
    const auto gather = [&](auto parts) {  // (the parts' number at compile time: all of a block's loads are on their way together)
      constexpr int kParts = decltype(parts)::value;
#pragma unroll
      for (int i = 0; i < kRounds; ++i) {
        const int row = tid / kLanes + i * kRows;
#pragma unroll
        for (int b = 0; b < S::kBlocks; ++b) {
          const std::uint32_t at = smem_u32(sum_at(b, row, piece));
          float4 o[kParts] = {};
          if (row < tile.count) {
#pragma unroll
            for (int q = 0; q < kParts; ++q) o[q] = ld_cluster_f32x4(map_to_cta(at, static_cast<std::uint32_t>(q)));
          }
#pragma unroll
          for (int q = 1; q < kParts; ++q) o[0].x += o[q].x, o[0].y += o[q].y, o[0].z += o[q].z, o[0].w += o[q].w;
          v[i][b][0] = o[0].x, v[i][b][1] = o[0].y, v[i][b][2] = o[0].z, v[i][b][3] = o[0].w;
        }
      }
    };
    if (a.parts == 1) gather(std::integral_constant<int, 1>{});
    else if (a.parts == 2) gather(std::integral_constant<int, 2>{});
    else gather(std::integral_constant<int, kMostManyParts>{});
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
#pragma unroll
      for (int b = 0; b < S::kBlocks; ++b) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i][b][e] = b * S::kBlock + piece * 4 + e < rank ? v[i][b][e] * scale : 0.f;  // (infinities of x have made NaN of the others)
      }
    }
    if (a.parts > 1) cluster_sync_all();  // (read by all)
    else __syncthreads();
    // Its two parts as rows, in the same place, then a row to a thread and into tensor memory.
    constexpr int kTRow = S::kN * 2;
    const auto t_at = [&](int which, int row, int at) { return stage_of(which) + row * kTRow + folded(at, row & 7) * 16; };
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
      const int row = tid / kLanes + i * kRows;
      float top = 0.f;
      if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
        for (int b = 0; b < S::kBlocks; ++b) {
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(v[i][b][e]));
        }
#pragma unroll
        for (int m = kLanes / 2; m > 0; m /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
      }
      const Halves<T> by(top);
#pragma unroll
      for (int b = 0; b < S::kBlocks; ++b) {
        uint2 hi, lo;
        by.split(v[i][b][0], v[i][b][1], hi.x, lo.x), by.split(v[i][b][2], v[i][b][3], hi.y, lo.y);
        const int at = b * S::kBlock + piece * 4;  // (the rank)
        *reinterpret_cast<uint2*>(t_at(0, row, at / 8) + at % 8 * 2) = hi, *reinterpret_cast<uint2*>(t_at(1, row, at / 8) + at % 8 * 2) = lo;
      }
      if (std::is_same<T, __half>::value && piece == 0) s_back[row] = by.back;
    }
    __syncthreads();
    back = std::is_same<T, __half>::value ? s_back[row0 + lane] : 1.f;
#pragma unroll
    for (int i = 0; i < S::kN / 8; ++i) {
      const uint4 p = load16(t_at(half, row0 + lane, i));
      const std::uint32_t r[4] = {p.x, p.y, p.z, p.w};
      tmem_st_32x4(low + lanes + half * (S::kN / 2) + i * 4, r);
    }
    tmem_st_wait();
    __syncthreads();  // (read by all)
  }
  copy_step(held);

  for (int s = k_steps; s <= steps; ++s) {
    if (s < steps) {
      if (rank % 8 != 0) {  // the last piece that is used has ranks behind the last one: whatever they hold, they are zeros
        wait_for_copies<S::kStages - 2>();
        __syncthreads();
        const int piece = rank / 8;
        for (int r = tid; r < 64; r += kManyThreads) {
          std::uint16_t* const p = reinterpret_cast<std::uint16_t*>(smem + s % S::kStages * S::kStage + piece / 8 * (64 * 128) + at_piece(r, piece & 7));
          for (int e = rank % 8; e < 8; ++e) p[e] = 0;
        }
      }
      copies_are_there();  // (and the accumulator of the step before the last has been read)
      if (warp == 0 && elect_one()) {
        const std::uint32_t at = ring + s % S::kStages * S::kStage, d = accumulators + (s & 1) * 64;
#pragma unroll
        for (int i = 0; i < S::kN / 16; ++i) {
          const std::uint64_t db = umma_desc_sw128(at + i / 4 * (64 * 128)) + 2 * (i % 4);
          umma_f16_ts(d, low + i * 8, db, idesc_b, static_cast<std::uint32_t>(i));
          umma_f16_ts(d, low + S::kN / 2 + i * 8, db, idesc_b, 1u);
        }
        tc_commit(smem_u32(&sh.done[s % S::kStages]));
      }
    }
    const int e = s - 1;  // the step that is added
    if (e >= k_steps) {
      wait_done(e);
      if (row0 < tile.count) {
        std::uint32_t v[32];
        tmem_ld_32x32(accumulators + (e & 1) * 64 + lanes + half * 32, v);
        tmem_ld_wait();
        std::uint8_t* const at = smem + e % S::kStages * S::kStage + S::kOperand;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4* const p = reinterpret_cast<uint4*>(at + at_piece(row0 + lane, half * 4 + i));
          float f[8];
          load8<T>(*p, f);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = fmaf(__uint_as_float(v[8 * i + j]), back, f[j]);
          *p = store8<T>(f);
        }
        __syncwarp();
        const int n = (e - k_steps) * 64;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 p = load16(at + at_piece(row0 + lane / 4 + i * 8, half * 4 + lane % 4));
          if (there[i] && n + column < to - from) *reinterpret_cast<uint4*>(out_to[i] + n) = p;
        }
        __syncwarp();  // (this warp's pieces of the stage are read: it is the next to be copied into)
      }
    }
    copy_step(e + S::kStages);
  }
  wait_for_copies<0>();
  end_tensor<S::kColumns>(sh);
}

inline int padded_tiles(int rank) {  // ranks / 8, up to a power of two
  int n = 1;
  while (n * 8 < rank) n *= 2;
  return n;
}
// Which kernels a call runs. Small tiles read A and B again every 16 tokens, large ones are mostly empty where adapters are many: small ones go by their number
// times the ranks for each large tile. Of large tiles, the kernel of many tokens wins by its products (mma.sync's rate is a quarter) and has more to set up. With
// 4096 channels and columns from memory, few / several / many tokens' kernels, us (in brackets small tiles times ranks for each large tile): 64 tokens of as many
// adapters, rank 64 (64) 16 / 44 / 37; 300 of 3, rank 128 (470) 21 / 24 / 25; 1000 of 6, rank 64 (320) 17 / 21 / 29, rank 128 (630) 31 / 28 / 39; 1500 of 4, rank 64
// (390) 26 / 23 / 30; 3000 of 4, rank 16 (110) 25 / 23 / 31, rank 128 88 / 52 / 49; 3000 of 60, rank 64 (190) 46 / 58 / 59, rank 128 (380) 91 / 94 / 73; 5000 of 6, rank
// 16 (110; a wave and a bit of CTAs, each a tile's whole work) 45 / 32 / 44; 8191 of 6, rank 64 85 / 68 / 59; 16000 of 60, 2048 channels and columns, rank 32 63 / 51 / 69.
enum class Way { kFew, kSeveral, kMany };
inline Way way_of(std::int64_t tokens, int adapters, int rank) {
  const std::int64_t large = most_tiles(tokens, adapters, kManyRows);
  if (tokens <= kFewTokens && most_tiles(tokens, adapters, kFewRows) * rank <= large * (tokens <= 1024 ? 500 : 200)) return Way::kFew;
  return rank > 32 && large * rank >= 3500 ? Way::kMany : Way::kSeveral;
}
inline int rows_of(Way way) { return way == Way::kFew ? kFewRows : kManyRows; }
// Small tiles that a plan is likely to have, where requests take their adapters at random: one for each adapter that somebody has, and more where they
// have more than 16 tokens.
inline std::int64_t likely_tiles(std::int64_t tokens, int adapters) {
  const double n = adapters + 1.0;
  return static_cast<std::int64_t>(std::ceil(n * (1.0 - std::exp(-static_cast<double>(tokens) / n)) + std::max(0.0, tokens / 16.0 - n / 2.0)));
}
// Parts of the channels (a power of two): CTAs for the whole GPU twice over (thrice of several tokens), of 256 channels at least. (Of few tokens by the tiles
// that are likely; by those that there may be, 300 tokens of 60 adapters of 128 ranks took 42 us for 31.)
inline int parts_of(Way way, std::int64_t tokens, int adapters, std::int64_t dim) {
  const std::int64_t room = (way == Way::kSeveral ? 3LL : 2LL) * sm_count(), most = way == Way::kMany ? kMostManyParts : kMostParts;
  const std::int64_t tiles = way == Way::kFew ? likely_tiles(tokens, adapters) : most_tiles(tokens, adapters, kManyRows);
  int parts = 1;
  while (parts < most && tiles * parts * 2 <= room && dim >= parts * 2 * 256) parts *= 2;
  return parts;
}
// Of several tokens: one of t's two parts (an operand has 16 ranks at least).
inline std::size_t part_bytes(std::int64_t rows, int rank) { return (static_cast<std::size_t>(rows) * std::max(2, padded_tiles(rank)) * 16 + 255) / 256 * 256; }
inline std::size_t workspace_bytes(std::int64_t tokens, int adapters, int rank) {
  const Way way = way_of(tokens, adapters, rank);
  if (way != Way::kSeveral) return 0;
  const std::int64_t rows = most_tiles(tokens, adapters, kManyRows) * kManyRows;
  return 2 * part_bytes(rows, rank) + static_cast<std::size_t>(rows) * 4;
}

template <typename T, int kNT>
int launch(const char* op, LoraArgs a, Way way, unsigned tiles, cudaStream_t stream) {
  if (way == Way::kSeveral) {
    const LaunchChain chain(stream);
    // Columns of a CTA: as many as leave 4 CTAs to an SM, 128 at least.
    const std::int64_t most = std::max<std::int64_t>(1, 4LL * sm_count() / tiles);
    a.columns = static_cast<int>(std::max<std::int64_t>(128, ((a.width + most - 1) / most + 127) / 128 * 128));
    const dim3 grid(tiles, static_cast<unsigned>((a.width + a.columns - 1) / a.columns));
    static std::atomic<std::uint64_t> shrink_done{0}, expand_done{0};
    constexpr int kShrinkBytes = kShrinkStages * kShrinkStage<kNT>, kExpandBytes = kExpandStages * kExpandStage<kNT>;
    if (const int s = allow_shared(op, shrink_several_kernel<T, kNT>, kShrinkBytes, shrink_done); s != B2_OK) return s;
    if (const int s = allow_shared(op, expand_several_kernel<T, kNT>, kExpandBytes, expand_done); s != B2_OK) return s;
    if (const int s = enqueue(op, shrink_several_kernel<T, kNT>, dim3(tiles * a.parts), dim3(kThreads), kShrinkBytes, stream, a.parts, a); s != B2_OK) return s;
    return enqueue(op, expand_several_kernel<T, kNT>, grid, dim3(kManyThreads), kExpandBytes, stream, 1, a);
  }
  // Clusters to a tile: as many as the GPU has room for (2 CTAs to an SM), of 128 columns a CTA at least. One where x is out: all of a cluster's channels are
  // read before one of its columns is written, those of another cluster may not be.
  const std::int64_t room = a.x == a.out ? 1 : std::max<std::int64_t>(1, 2LL * sm_count() / (static_cast<std::int64_t>(tiles) * a.parts));
  a.groups = static_cast<int>(std::max<std::int64_t>(1, std::min<std::int64_t>(room, a.width / (128 * a.parts))));
  a.columns = (a.width + a.parts * a.groups - 1) / (a.parts * a.groups);
  a.columns = way == Way::kFew ? (a.columns + 31) / 32 * 32 : (a.columns + 63) / 64 * 64;
  const dim3 grid(tiles * a.parts * a.groups);
  if constexpr (kNT >= 8) {
    if (way == Way::kMany) {
      static std::atomic<std::uint64_t> many_done{0};
      if (const int s = allow_shared(op, many_kernel<T, kNT>, ManyShape<kNT>::kBytes, many_done); s != B2_OK) return s;
      return enqueue(op, many_kernel<T, kNT>, grid, dim3(kManyThreads), ManyShape<kNT>::kBytes, stream, a.parts, a);
    }
  }
  static std::atomic<std::uint64_t> few_done{0};
  if (const int s = allow_shared(op, few_kernel<T, kNT>, FewShape<kNT>::kBytes, few_done); s != B2_OK) return s;
  return enqueue(op, few_kernel<T, kNT>, grid, dim3(kThreads), FewShape<kNT>::kBytes, stream, a.parts, a);
}
template <typename T>
int launch(const char* op, const LoraArgs& a, Way way, unsigned tiles, cudaStream_t stream) {
  switch (padded_tiles(a.rank)) {
    case 1: return launch<T, 1>(op, a, way, tiles, stream);
    case 2: return launch<T, 2>(op, a, way, tiles, stream);
    case 4: return launch<T, 4>(op, a, way, tiles, stream);
    case 8: return launch<T, 8>(op, a, way, tiles, stream);
    default: return launch<T, 16>(op, a, way, tiles, stream);
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
  return enqueue(op, plan_kernel, dim3(static_cast<unsigned>(adapters + 1)), dim3(kPlanThreads), static_cast<std::size_t>(adapters + 1) * 4, as_stream(stream), 1,
                 token_adapters, static_cast<int>(tokens), adapters, plan_at(plan, tokens, adapters));
}

size_t b2_lora_workspace_bytes(int64_t tokens, int adapters, int64_t dim, int rank) {
  using namespace b2;
  const char* const op = "lora_add";
  if (check_sizes(op, tokens, adapters) != B2_OK || check_shape(op, dim, rank) != B2_OK) return 0;
  return std::max<std::size_t>(256, workspace_bytes(tokens, adapters, rank));
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
  if (out == x && ldo != ldx && tokens > 1) return fail_invalid(op, "out in x's place must have x's rows");
  if (const int s = check_workspace(op, workspace, ws_bytes, workspace_bytes(tokens, l->adapters, l->rank)); s != B2_OK) return s;
  LoraArgs a{};
  const Way way = way_of(tokens, l->adapters, l->rank);
  const std::int64_t tiles = most_tiles(tokens, l->adapters, rows_of(way));
  const Plan p = plan_at(const_cast<void*>(plan), tokens, l->adapters);
  a.plan = Tiles{p.head, p.tiles[way != Way::kFew], p.order, static_cast<int>(tokens), l->adapters, way != Way::kFew};
  a.a = l->a, a.b = l->b, a.a_adapter = l->a_adapter_stride, a.a_row = l->a_row_stride, a.b_adapter = l->b_adapter_stride, a.b_row = l->b_row_stride;
  a.scales = l->scales, a.ranks = l->ranks, a.x = x, a.y = y, a.out = out, a.ldx = ldx, a.ldy = ldy, a.ldo = ldo;
  a.rank = l->rank, a.dim = static_cast<int>(l->dim), a.width = static_cast<int>(l->width);
  char* const at = static_cast<char*>(workspace);
  const std::size_t part = part_bytes(tiles * rows_of(way), l->rank);
  a.low = LowWords{reinterpret_cast<std::uint32_t*>(at), reinterpret_cast<std::uint32_t*>(at + part), reinterpret_cast<float*>(at + 2 * part)};
  a.parts = parts_of(way, tokens, l->adapters, l->dim);
  a.slice = static_cast<int>(((l->dim + a.parts - 1) / a.parts + 63) / 64 * 64);
  return l->dtype == B2_DTYPE_F16 ? launch<__half>(op, a, way, static_cast<unsigned>(tiles), as_stream(stream)) : launch<__nv_bfloat16>(op, a, way, static_cast<unsigned>(tiles), as_stream(stream));
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
