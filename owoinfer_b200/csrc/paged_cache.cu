// What goes into and out of a paged key-value cache: per-head norm + rotation + append, and eviction by accumulated attention weight.
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <mutex>

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
  int q_heads, half, chunks;  // half: rotated pairs; chunks: groups of kHeads heads of a token
};

constexpr int kAppendHeads = 4;  // heads a group of lanes works on at a time, their loads issued together
constexpr int kAppendThreads = 256;

// One group of D / 8 lanes (8 channels each) per (token, four heads): the sum of squares is a butterfly within the group, and
// the other element of a rotation pair is in the same lane (interleaved) or half a rotation's lanes away.
template <typename T, int D, bool kInterleaved>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendArgs a) {
  constexpr int kLanes = D / 8;
  const int lane = static_cast<int>(threadIdx.x) % kLanes;
  const unsigned group_mask = (kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u)) << (threadIdx.x % 32 / kLanes * kLanes);
  const std::int64_t unit = (static_cast<std::int64_t>(blockIdx.x) * kAppendThreads + threadIdx.x) / kLanes;
  const std::int64_t token = unit / a.chunks;
  if (token >= a.tokens) return;
  const int head0 = static_cast<int>(unit - token * a.chunks) * kAppendHeads, heads = a.q_heads + 2 * a.c.kv_heads;

  uint4 raw[kAppendHeads];
  const T* row = static_cast<const T*>(a.qkv) + token * a.ld + lane * 8;
#pragma unroll
  for (int i = 0; i < kAppendHeads; ++i) {
    if (head0 + i < heads) raw[i] = *reinterpret_cast<const uint4*>(row + static_cast<std::int64_t>(head0 + i) * D);
  }

  // The sequence of this token: the lanes of the group try kLanes places of cu_seqlens at a time.
  int lo = 0, hi = a.c.batch;  // cu[lo] <= token < cu[hi] (what lies outside shows up below)
  while (hi - lo > 1) {
    const int step = (hi - lo + kLanes - 1) / kLanes, at = lo + (lane + 1) * step;
    const bool below = at < hi && a.cu[at] <= token;
    const int n = __popc(__ballot_sync(group_mask, below) & group_mask);
    hi = min(hi, lo + (n + 1) * step);
    lo += n * step;
  }
  const int b = lo;
  int first, n;
  paged_tokens(a.c, a.cu, b, a.tokens, first, n);
  const int slot = paged_len(a.c, b) - n + static_cast<int>(token - first);
  const bool in_sequence = token >= first && token < first + n;
  if (!in_sequence || slot < 0) {
    atomicOr(a.c.status, kPagedBadTokens);
    if (!in_sequence) return;
  }

  float sn[8], cs[8];
  // Which pair of the rotation this lane's first channel belongs to; lanes past the rotation keep their values.
  const bool turns = lane * 8 < 2 * a.half;
  if (turns) {
    std::int64_t position = a.positions != nullptr ? a.positions[token] : max(slot, 0);
    if (position < 0 || position >= a.rope_rows) {
      atomicOr(a.c.status, kPagedBadPosition);
      position = position < 0 ? 0 : a.rope_rows - 1;
    }
    const float* t = a.rope + position * (2 * a.half);
    if constexpr (kInterleaved) {
      const float4 s4 = *reinterpret_cast<const float4*>(t + lane * 4), c4 = *reinterpret_cast<const float4*>(t + a.half + lane * 4);
      sn[0] = sn[1] = s4.x, sn[2] = sn[3] = s4.y, sn[4] = sn[5] = s4.z, sn[6] = sn[7] = s4.w;
      cs[0] = cs[1] = c4.x, cs[2] = cs[3] = c4.y, cs[4] = cs[5] = c4.z, cs[6] = cs[7] = c4.w;
    } else {
      const int pair = lane * 8 < a.half ? lane * 8 : lane * 8 - a.half;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 s4 = *reinterpret_cast<const float4*>(t + pair + i), c4 = *reinterpret_cast<const float4*>(t + a.half + pair + i);
        sn[i] = s4.x, sn[i + 1] = s4.y, sn[i + 2] = s4.z, sn[i + 3] = s4.w;
        cs[i] = c4.x, cs[i + 1] = c4.y, cs[i + 2] = c4.z, cs[i + 3] = c4.w;
      }
    }
  }
  const int page = slot < 0 ? -1 : paged_page(a.c, b, slot);
  const int away = a.half / 8, partner = !turns ? lane : lane < away ? lane + away : lane - away;

#pragma unroll
  for (int i = 0; i < kAppendHeads; ++i) {
    const int head = head0 + i;
    if (head >= heads) break;
    if (head >= a.q_heads + a.c.kv_heads) {
      if (page >= 0) {
        T* v = static_cast<T*>(a.c.v) + paged_row(a.c, page, head - a.q_heads - a.c.kv_heads, slot) + lane * 8;
        *reinterpret_cast<uint4*>(v) = raw[i];
      }
      continue;
    }
    const bool is_q = head < a.q_heads;
    float x[8];
    load8<T>(raw[i], x);
    if (a.q_norm != nullptr) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
#pragma unroll
      for (int m = kLanes / 2; m > 0; m /= 2) sum += __shfl_xor_sync(group_mask, sum, m);
      const float r = rsqrtf(sum * (1.0f / D) + a.eps);
      float w[8];
      load8<T>(__ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(is_q ? a.q_norm : a.k_norm) + lane * 8)), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * r * w[j];
    }
    if (a.half > 0) {
      if constexpr (kInterleaved) {
        if (turns) {
#pragma unroll
          for (int j = 0; j < 8; j += 2) {
            const float u = x[j], v = x[j + 1];
            x[j] = u * cs[j] - v * sn[j];
            x[j + 1] = v * cs[j] + u * sn[j];
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float other = __shfl_sync(group_mask, x[j], partner, kLanes);
          if (turns) x[j] = lane < away ? x[j] * cs[j] - other * sn[j] : x[j] * cs[j] + other * sn[j];
        }
      }
    }
    if (is_q) {
      *reinterpret_cast<uint4*>(static_cast<T*>(a.q_out) + token * a.q_row + head * a.q_head + lane * 8) = store8<T>(x);
    } else if (page >= 0) {
      *reinterpret_cast<uint4*>(static_cast<T*>(a.c.k) + paged_row(a.c, page, head - a.q_heads, slot) + lane * 8) = store8<T>(x);
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

constexpr int kSelectThreads = 512;
constexpr int kSelectItems = 16;  // consecutive slots of a thread in a round
constexpr int kSelectRound = kSelectThreads * kSelectItems;
constexpr int kMostSelectCtas = 8;

// The order of the weights as the order of unsigned numbers: -0 counts as 0, NaN comes below everything.
__device__ __forceinline__ unsigned weight_key(float w) {
  if (isnan(w)) return 0u;
  const unsigned u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned ld_cluster_u32(std::uint32_t addr) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// A cluster per (sequence, key head), each CTA with its share of the slots between the first and the last ones. The weight of
// the last slot that stays is found bit by bit from the top (8 at a time, a histogram over the cluster for each byte); then
// every CTA counts what stays in its share, and writes it behind what the CTAs before it keep.
__global__ void __launch_bounds__(kSelectThreads) select_kernel(const EvictArgs a) {
  dependents_may_start();
  __shared__ unsigned s_hist[2][256];
  __shared__ unsigned s_total[256];
  __shared__ unsigned s_warp[2][kSelectThreads / 32];
  __shared__ unsigned s_count[2];
  __shared__ unsigned s_pick[2];
  const int ctas = gridDim.x, rank = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int tid = static_cast<int>(threadIdx.x), warp = tid / 32, lane = tid % 32;
  const int len = paged_len(a.c, b);
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
  // This CTA's share, a multiple of 4 slots.
  const int middle = len - a.recent - a.sinks;
  const int share = ((middle + ctas - 1) / ctas + 3) / 4 * 4;
  const int begin = a.sinks + min(middle, rank * share), end = a.sinks + min(middle, (rank + 1) * share);

  unsigned prefix = 0, wanted = static_cast<unsigned>(room);  // of the slots whose upper bits are `prefix`, how many stay
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    unsigned(&hist)[256] = s_hist[pass & 1];
    for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    for (int i = begin + tid; i < end; i += kSelectThreads) {
      const unsigned key = weight_key(w[i]);
      if (pass == 0 || key >> (shift + 8) == prefix) atomicAdd(&hist[key >> shift & 255u], 1u);
    }
    // (The other half of s_hist is cleared for the next pass only after this barrier: by then every CTA has read it.)
    cluster_sync_all();
    if (tid < 256) {
      unsigned sum = 0;
      for (int c = 0; c < ctas; ++c) sum += ld_cluster_u32(map_to_cta(smem_u32(&hist[tid]), c));
      s_total[tid] = sum;
    }
    __syncthreads();
    if (warp == 0) {  // from the largest byte down: where the running count reaches what is wanted
      unsigned mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += s_total[255 - lane * 8 - i];
      unsigned upto = mine;
#pragma unroll
      for (int m = 1; m < 32; m *= 2) {
        const unsigned o = __shfl_up_sync(0xffffffffu, upto, m);
        if (lane >= m) upto += o;
      }
      unsigned before = upto - mine;
      if (before < wanted && upto >= wanted) {
        for (int i = 0; i < 8; ++i) {
          const unsigned n = s_total[255 - lane * 8 - i];
          if (before + n >= wanted) {
            s_pick[0] = static_cast<unsigned>(255 - lane * 8 - i), s_pick[1] = wanted - before;
            break;
          }
          before += n;
        }
      }
    }
    __syncthreads();
    prefix = prefix << 8 | s_pick[0];
    wanted = s_pick[1];
  }

  // `prefix` is the key of the last one that stays, and `wanted` of its equals stay. Counts of this CTA's share: above, equal.
  unsigned above = 0, equal = 0;
  for (int i = begin + tid; i < end; i += kSelectThreads) {
    const unsigned key = weight_key(w[i]);
    above += key > prefix, equal += key == prefix;
  }
  if (tid < 2) s_count[tid] = 0;
  __syncthreads();
  above = __reduce_add_sync(0xffffffffu, above), equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) atomicAdd(&s_count[0], above), atomicAdd(&s_count[1], equal);
  cluster_sync_all();
  unsigned above_before = 0, equal_before = 0;
  for (int c = 0; c < rank; ++c) {
    above_before += ld_cluster_u32(map_to_cta(smem_u32(&s_count[0]), c));
    equal_before += ld_cluster_u32(map_to_cta(smem_u32(&s_count[1]), c));
  }
  cluster_sync_all();  // nobody reads another CTA's shared memory from here on

  for (int at = begin; at < end; at += kSelectRound) {
    const int mine = at + tid * kSelectItems;
    unsigned key[kSelectItems], n_above = 0, n_equal = 0;
#pragma unroll
    for (int i = 0; i < kSelectItems; ++i) {
      key[i] = mine + i < end ? weight_key(w[mine + i]) : 0u;
      n_above += mine + i < end && key[i] > prefix, n_equal += mine + i < end && key[i] == prefix;
    }
    unsigned upto_above = n_above, upto_equal = n_equal;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
      const unsigned oa = __shfl_up_sync(0xffffffffu, upto_above, m), oe = __shfl_up_sync(0xffffffffu, upto_equal, m);
      if (lane >= m) upto_above += oa, upto_equal += oe;
    }
    __syncthreads();  // (s_warp of the round before is read)
    if (lane == 31) s_warp[0][warp] = upto_above, s_warp[1][warp] = upto_equal;
    __syncthreads();
    unsigned ra = above_before + upto_above - n_above, re = equal_before + upto_equal - n_equal;
    for (int i = 0; i < kSelectThreads / 32; ++i) {
      if (i < warp) ra += s_warp[0][i], re += s_warp[1][i];
      above_before += s_warp[0][i], equal_before += s_warp[1][i];
    }
#pragma unroll
    for (int i = 0; i < kSelectItems; ++i) {
      if (mine + i >= end) break;
      const bool up = key[i] > prefix, level = key[i] == prefix;
      if (up || (level && re < wanted)) {
        const unsigned to = static_cast<unsigned>(a.sinks) + ra + min(re, wanted);
        kept[to] = mine + i;
        if (w_out != nullptr) w_out[to] = w[mine + i];
      }
      ra += up, re += level;
    }
  }
}

constexpr int kMoveThreads = 256;
constexpr int kMoveRows = 4;  // rows of K and of V that a group of lanes has in flight

// kept -> the new pages: a group of D / 8 lanes moves kMoveRows rows of K and of V, 16 bytes a lane.
template <int D>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(const EvictArgs a) {
  constexpr int kLanes = D / 8, kGroups = kMoveThreads / kLanes;
  const int h = blockIdx.y, b = blockIdx.z, lane = static_cast<int>(threadIdx.x) % kLanes, group = static_cast<int>(threadIdx.x) / kLanes;
  wait_for_predecessors();
  const int len = min(paged_len(a.c, b), a.budget);
  const int row0 = static_cast<int>(blockIdx.x) * (kGroups * kMoveRows) + group;
  if (row0 >= len) return;
  const std::int32_t* kept = a.kept + (static_cast<std::int64_t>(b) * a.c.kv_heads + h) * a.budget;
  const std::uint16_t *k = static_cast<const std::uint16_t*>(a.c.k), *v = static_cast<const std::uint16_t*>(a.c.v);
  uint4 kr[kMoveRows], vr[kMoveRows];
  std::int64_t to[kMoveRows];
#pragma unroll
  for (int i = 0; i < kMoveRows; ++i) {
    const int r = row0 + i * kGroups;
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
  for (int i = 0; i < kMoveRows; ++i) {
    if (to[i] < 0) continue;
    *reinterpret_cast<uint4*>(static_cast<std::uint16_t*>(a.c.k) + to[i]) = kr[i];
    *reinterpret_cast<uint4*>(static_cast<std::uint16_t*>(a.c.v) + to[i]) = vr[i];
  }
}

template <typename T, int D>
int launch_append(const char* op, const AppendArgs& a, bool interleaved, cudaStream_t st) {
  const std::int64_t units = a.tokens * a.chunks, per_block = kAppendThreads / (D / 8);
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
  if (c->num_pages < 0 || c->num_pages > INT_MAX || c->table_width < 0 || static_cast<std::int64_t>(c->table_width) * c->page_size > INT_MAX ||
      c->table_ld < c->table_width) {
    return fail_invalid(op, "num_pages and table_width * page_size must be below 2^31, table_ld at least table_width");
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
  void* word = nullptr;
  if (const cudaError_t e = cudaGetSymbolAddress(&word, g_paged_status); e != cudaSuccess) {
    cudaGetLastError();
    return fail_cuda(op, e);
  }
  a->status = static_cast<unsigned*>(word);
  return B2_OK;
}

bool make_tensor_map_pages(CUtensorMap* map, const b2_paged_cache* c, bool values, int box_rows, const char* op) {
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
  const auto u = [](std::int64_t v) { return static_cast<cuuint64_t>(v); };
  const cuuint64_t dims[4] = {u(c->head_dim), u(c->page_size), u(c->kv_heads), u(c->num_pages)};
  const cuuint64_t strides[3] = {u(c->row_stride) * 2, u(c->head_stride) * 2, u(c->page_stride) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1}, elem[4] = {1, 1, 1, 1};
  const CUresult r = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, values ? c->v : c->k, dims, strides, box, elem,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r == CUDA_SUCCESS) return true;
  fail_status(B2_ERR_CUDA, op, "cuTensorMapEncodeTiled failed with code " + std::to_string(static_cast<int>(r)) + " for the pages' pool");
  return false;
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
  a.chunks = static_cast<int>((heads + kAppendHeads - 1) / kAppendHeads);
  if (tokens * a.chunks > INT_MAX) return fail_invalid(op, "too many tokens for one call");
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
  a.weights = weights, a.weights_ld = weights_ld, a.table_out = table_out, a.table_out_ld = table_out_ld, a.kept = kept;
  a.lens_out = lens_out, a.weights_out = weights_out, a.weights_out_ld = weights_out_ld;
  a.sinks = sinks, a.recent = recent, a.budget = budget;
  if (const int rc = paged_status_word(op, &a.c)) return rc;
  const cudaStream_t st = as_stream(stream);
  const LaunchChain chain(st);
  int ctas = 1;
  while (ctas < kMostSelectCtas && static_cast<std::int64_t>(ctas) * kSelectRound < slots) ctas *= 2;
  const unsigned heads = static_cast<unsigned>(cache->kv_heads), batch = static_cast<unsigned>(cache->batch);
  if (const int rc = enqueue(op, select_kernel, dim3(static_cast<unsigned>(ctas), heads, batch), kSelectThreads, 0, st, ctas, a)) return rc;
  const int rows = kMoveThreads / (cache->head_dim / 8) * kMoveRows;
  const std::int64_t most = std::min<std::int64_t>(budget, slots);
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
