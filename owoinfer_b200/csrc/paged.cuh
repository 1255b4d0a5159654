// A key-value cache in pages, as the kernels on it see it: argument checks, slot arithmetic with bounds, the status word, and
// what the 16-bit types need. No counterpart in the reference.
#pragma once

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace b2 {

// Why b2_paged_cache_status is not 0.
enum PagedFault : unsigned {
  kPagedBadPage = 1,      // a page of the block table outside the pool
  kPagedBadLength = 2,    // seq_lens below 0 or past the block table or max_len
  kPagedBadTokens = 4,    // cu_seqlens that fall or leave [0, the call's tokens]; in the append also tokens without a sequence or a slot
  kPagedBadPosition = 8,  // a position outside the rotation table
  kPagedWait = 16,        // a bounded wait expired
};

// Slots of a block table, at most: a slot is an int, and so is a loop's stride past the last one (the longest: 8 CTAs an SM of 1024 slots
// each, in the join of single-token attention, 1.2 million).
constexpr std::int64_t kMostSlots = (1LL << 31) - (1LL << 21);

struct PagedArgs {
  void* k;
  void* v;
  std::int64_t page_stride, head_stride, row_stride, num_pages;  // elements
  const std::int32_t* table;
  std::int64_t table_ld;
  const std::int32_t* lens;
  unsigned* status;
  int most, page_shift, batch, kv_heads;  // most: slots a sequence can have
};

// Checks the cache of a call and fills `a` but for its status word (head_dim 64 or 128, a page size that is a power of two from 16 to
// 1024). Makes no CUDA call.
int check_paged_cache(const char* op, const b2_paged_cache* c, PagedArgs* a);
// The current device's status word into `a`.
int paged_status_word(const char* op, PagedArgs* a);
// Where a call may write or read rows of `row` elements: 16-byte aligned, strides in multiples of 8 elements.
inline bool rows_ok(const void* p, std::int64_t row, std::int64_t head) { return p != nullptr && aligned_to(p, 16) && row % 8 == 0 && head % 8 == 0; }
// A kernel's dynamic shared memory, set once per device (`done`: a static of the caller's, a bit for each device).
template <typename Kernel>
int allow_shared(const char* op, Kernel kernel, int bytes, std::atomic<std::uint64_t>& done) {
  int device = 0;
  if (cudaGetDevice(&device) == cudaSuccess && device < 64 && (done.load(std::memory_order_relaxed) >> device & 1u) != 0u) return B2_OK;
  if (const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); e != cudaSuccess) {
    cudaGetLastError();
    return fail_cuda(op, e);
  }
  if (device < 64) done.fetch_or(1ull << device, std::memory_order_relaxed);
  return B2_OK;
}
// cuTensorMapEncodeTiled for the cache's keys or values, [pages, heads, rows, head_dim]: boxes of box_rows rows of box_columns
// elements, 64 with the 128-byte swizzle or 32 with the 64-byte one. Returns false (and sets the last error) on failure.
bool make_tensor_map_pages(CUtensorMap* map, const b2_paged_cache* c, bool values, int box_rows, int box_columns, const char* op);
// The same for a view [tokens, heads, head_dim] of 16-bit elements: boxes of 64 elements of box_heads heads of box_tokens tokens.
bool make_tensor_map_rows(CUtensorMap* map, const b2_view3* v, int head_dim, int box_heads, int box_tokens, const char* op);
// A window that reaches every slot is none; sinks past the last slot are all slots.
int check_window(const char* op, const PagedArgs& c, int* window, int* sinks);
// A workspace of `need` bytes. One that is given is looked at even where none is needed: what a caller sized wrongly shows at
// its first call, whatever that call's lengths.
inline int check_workspace(const char* op, const void* workspace, std::size_t bytes, std::size_t need) {
  if (workspace == nullptr ? bytes == 0 && need == 0 : aligned_to(workspace, 256) && bytes >= std::max<std::size_t>(need, 256)) return B2_OK;
  return fail_invalid(op, "workspace is missing, too small (its _workspace_bytes call has the size) or not 256-byte aligned");
}

#ifdef __CUDACC__
// Slots of sequence b, at least 0 and at most what its row of the block table (or the call) allows.
__device__ __forceinline__ int paged_len(const PagedArgs& a, int b) {
  const int len = a.lens[b];
  if (len >= 0 && len <= a.most) return len;
  atomicOr(a.status, kPagedBadLength);
  return len < 0 ? 0 : a.most;
}
// The page with slot `slot` (which lies in the block table) of sequence b, or -1.
__device__ __forceinline__ int paged_page(const PagedArgs& a, int b, int slot) {
  const int page = a.table[b * a.table_ld + (slot >> a.page_shift)];
  if (page >= 0 && page < a.num_pages) return page;
  atomicOr(a.status, kPagedBadPage);
  return -1;
}
// Offset in elements of a slot's row of one head.
__device__ __forceinline__ std::int64_t paged_row(const PagedArgs& a, int page, int head, int slot) {
  return page * a.page_stride + head * a.head_stride + (slot & ((1 << a.page_shift) - 1)) * a.row_stride;
}
// The call's tokens of sequence b: [first, first + n) of `tokens`.
__device__ __forceinline__ void paged_tokens(const PagedArgs& a, const std::int32_t* cu, int b, std::int64_t tokens, int& first, int& n) {
  const int from = cu[b], to = cu[b + 1];
  first = from, n = to - from;
  if (from >= 0 && to >= from && to <= tokens) return;
  atomicOr(a.status, kPagedBadTokens);
  first = 0, n = 0;
}

// f x + keep sum, the join of a part of an output: an infinity is one however small the part's factor, 0 included.
__device__ __forceinline__ float joined(float f, float x, float keep, float sum) {
  const float y = fmaf(f, x, keep * sum);
  if (__builtin_expect(!isnan(y), 1)) return y;
  return (isinf(x) ? x : f * x) + (isinf(sum) ? sum : keep * sum);
}

template <typename T>
__device__ __forceinline__ float to_float(T v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ std::uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ std::uint32_t pack16<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const std::uint32_t*>(&h);
}
template <>
__device__ __forceinline__ std::uint32_t pack16<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const std::uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void unpack16(std::uint32_t w, float& lo, float& hi);
template <>
__device__ __forceinline__ void unpack16<__nv_bfloat16>(std::uint32_t w, float& lo, float& hi) {
  lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void unpack16<__half>(std::uint32_t w, float& lo, float& hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  lo = f.x, hi = f.y;
}
template <typename T>
__device__ __forceinline__ void load8(const uint4& raw, float (&x)[8]) {
  unpack16<T>(raw.x, x[0], x[1]);
  unpack16<T>(raw.y, x[2], x[3]);
  unpack16<T>(raw.z, x[4], x[5]);
  unpack16<T>(raw.w, x[6], x[7]);
}
template <typename T>
__device__ __forceinline__ uint4 store8(const float (&x)[8]) {
  return make_uint4(pack16<T>(x[0], x[1]), pack16<T>(x[2], x[3]), pack16<T>(x[4], x[5]), pack16<T>(x[6], x[7]));
}
#endif

}  // namespace b2
