// The residual stream takes up a layer's output, and its root-mean-square norm leaves in 8 bits for the projection that follows.
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>

#include "text.cuh"

namespace b2 {
namespace {

struct NormArgs {
  const void* x;
  std::int64_t ldx;
  const void* residual;
  std::int64_t ld_residual;
  void* residual_out;
  std::int64_t ld_residual_out;
  const void* weight;
  int weight_dtype;
  void* norm_out;
  std::int64_t ld_norm;
  int norm_f16;
  void* q;
  std::int64_t ldq;
  float* scale;
  std::int64_t tokens;
  int dim, group, row_threads;
  float eps;
};

constexpr int kMostDim = 32768;
constexpr float kSmallestScale = 1e-30f;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int m = 16; m > 0; m /= 2) v += __shfl_xor_sync(0xffffffffu, v, m);
  return v;
}
__device__ __forceinline__ float warp_max(float v, int width = 32) {
#pragma unroll
  for (int m = 16; m > 0; m /= 2) {
    if (m < width) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, m));
  }
  return v;
}
template <bool kE4m3>
__device__ __forceinline__ uint2 codes8(const float (&v)[8], float by) {
  std::uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (kE4m3) {
      const std::uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * by, v[4 * i + 1] * by), __NV_SATFINITE, __NV_E4M3);
      const std::uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * by, v[4 * i + 3] * by), __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | hi << 16;
    } else {  // (NaN converts to 0; nothing is past 127.5: the largest of a row is 127 within a few roundings)
      int c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] = __float2int_rn(v[4 * i + e] * by);
      w[i] = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    }
  }
  return make_uint2(w[0], w[1]);
}

// s = x + residual; y = s rsqrt(mean s^2 + eps) w; codes round(y / scale). A row's threads hold 8 neighbouring channels each, kPer times over, from
// the load to the codes: one pass over memory, and one block barrier, for the sum of squares and the largest |s w| (the scale of a
// whole row does not need the norm's factor first) are reduced together. What bounds it is memory: 16384 x 8192, bf16 with its residual to
// e4m3, takes 142 us, as long as a copy of as many bytes (a scale per 128 channels: 192); a row alone takes the 2.4 us of a launch, a load and a store.
template <typename X, typename R, bool kE4m3, int kPer, int kThreads>
__global__ void __launch_bounds__(kThreads) norm_kernel(const NormArgs a) {
  __shared__ float2 s_part[32];
  const int row_in_block = static_cast<int>(threadIdx.x) / a.row_threads, lane = static_cast<int>(threadIdx.x) % a.row_threads;
  const std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * (blockDim.x / a.row_threads) + row_in_block;
  const bool there = row < a.tokens;
  const int chunks = a.dim / 8;
  const bool adds = a.residual != nullptr;

  Raw8<X> x[kPer];
  Raw8<R> res[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int c = lane + i * a.row_threads;
    x[i].zero(), res[i].zero();
    if (!there || c >= chunks) continue;
    x[i].load(static_cast<const X*>(a.x) + row * a.ldx + c * 8);
    if (adds) res[i].load(static_cast<const R*>(a.residual) + row * a.ld_residual + c * 8);
  }
  float v[kPer][8];  // s, then s w
  float sum = 0.f, top = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int c = lane + i * a.row_threads;
    float r[8];
    x[i].get(v[i]);
    res[i].get(r);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[i][e] += r[e];
      sum = fmaf(v[i][e], v[i][e], sum);
    }
    if (!there || c >= chunks) continue;
    if (a.residual_out != nullptr) put8(static_cast<R*>(a.residual_out) + row * a.ld_residual_out + c * 8, v[i]);
    if (a.weight != nullptr) {
      float w[8];
      if (a.weight_dtype == B2_DTYPE_F32) {
        Raw8<float> raw;
        raw.load(static_cast<const float*>(a.weight) + c * 8);
        raw.get(w);
      } else {
        const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const std::uint16_t*>(a.weight) + c * 8);
        if (a.weight_dtype == B2_DTYPE_F16) load8<__half>(raw, w);
        else load8<__nv_bfloat16>(raw, w);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] *= w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[i][e]));
  }
  sum = warp_sum(sum), top = warp_max(top);
  if (a.row_threads > 32) {
    const int warps = a.row_threads / 32, first = row_in_block * warps;
    if (threadIdx.x % 32 == 0) s_part[threadIdx.x / 32] = make_float2(sum, top);
    __syncthreads();
    sum = 0.f, top = 0.f;
    for (int i = 0; i < warps; ++i) {
      const float2 p = s_part[first + i];
      sum += p.x, top = fmaxf(top, p.y);
    }
  }
  // A row with a NaN or an infinity, or whose squares pass fp32, has NaN for its scales (rsqrt of infinity would make zeros of the rest), and so
  // has one of zeros without an eps.
  const float square = sum / static_cast<float>(a.dim) + a.eps;
  const float r = square > 0.f && square < INFINITY ? rsqrtf(square) : __int_as_float(0x7fc00000);
  constexpr float kLargest = kE4m3 ? 448.f : 127.f;
  const auto scale_of = [&](float most) { return isnan(r) ? r : fmaxf(most * r / kLargest, kSmallestScale); };
  // y / scale is s w times Q / max|s w|: the norm's factor is in both, and its roundings would move what lies between two codes. Where that passes fp32, or
  // the scale is the smallest one (or NaN): y itself, then times 1 / scale.
  const auto by_largest = [](float most, float scale) { return scale > kSmallestScale && most > kLargest / 3e38f; };
  float scale = 0.f, by = 0.f, rest = r;  // (rest: of y = v rest)
  if (a.group == 0) {
    scale = scale_of(top), by = kLargest / top;
    if (!by_largest(top, scale)) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= r;
      }
      by = 1.f / scale, rest = 1.f;
    }
    if (there && lane == 0) a.scale[row] = scale;
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int c = lane + i * a.row_threads;
    const bool mine = there && c < chunks;
    if (a.group != 0) {  // (a group's lanes are neighbours in a warp: the shuffles are the whole warp's)
      float most = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[i][e]));
      most = warp_max(most, a.group / 8), scale = scale_of(most), by = kLargest / most, rest = r;
      if (!by_largest(most, scale)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] *= r;
        by = 1.f / scale, rest = 1.f;
      }
      if (mine && c * 8 % a.group == 0) a.scale[row * (a.dim / a.group) + c * 8 / a.group] = scale;
    }
    if (!mine) continue;
    *reinterpret_cast<uint2*>(static_cast<std::uint8_t*>(a.q) + row * a.ldq + c * 8) = codes8<kE4m3>(v[i], by);
    if (a.norm_out != nullptr) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = v[i][e] * rest;
      std::uint16_t* const p = static_cast<std::uint16_t*>(a.norm_out) + row * a.ld_norm + c * 8;
      *reinterpret_cast<uint4*>(p) = a.norm_f16 != 0 ? store8<__half>(y) : store8<__nv_bfloat16>(y);
    }
  }
}

template <typename X, typename R, bool kE4m3>
int launch(const char* op, NormArgs a, cudaStream_t stream) {
  // Few rows: a thread per 8 channels, for the latency. Many: up to four times as much a thread, whose loads are on their way together, and
  // as few threads behind a row's barrier. Once, twice, four times, us on B200 (bf16, INT8): 200 x 4096: 3.7, 3.6, 4.5;
  // 400 x 4096: 5.0, 4.6, 5.4; 1500 x 4096: 13.8, 11.4, 12.4; 2011 x 4096 (fp32 residual): 19.2, 17.7, 19.6; 2011 x 8192: 36.9, 29.9, 24.8;
  // 8000 x 8192: 132, 100, 74.
  const int chunks = a.dim / 8;
  int per = a.tokens <= sm_count() ? 1 : a.tokens * chunks <= 1 << 20 ? 2 : 4;
  while (per < 4 && (chunks + per - 1) / per > 1024) per *= 2;
  while (per > 1 && chunks <= 32 * (per / 2)) per /= 2;
  a.row_threads = ((chunks + per - 1) / per + 31) / 32 * 32;
  const int rows = std::max(1, 128 / a.row_threads);
  const std::int64_t blocks = (a.tokens + rows - 1) / rows;
  const dim3 grid(static_cast<unsigned>(blocks)), block(static_cast<unsigned>(rows * a.row_threads));
  if (per == 1) return enqueue(op, norm_kernel<X, R, kE4m3, 1, 1024>, grid, block, 0, stream, 1, a);
  if (per == 2) return enqueue(op, norm_kernel<X, R, kE4m3, 2, 1024>, grid, block, 0, stream, 1, a);
  // (Four times 8 channels of x and an fp32 residual do not quite fit the registers that 1024 threads leave a thread.)
  if (block.x <= 256) return enqueue(op, norm_kernel<X, R, kE4m3, 4, 256>, grid, block, 0, stream, 1, a);
  return enqueue(op, norm_kernel<X, R, kE4m3, 4, 1024>, grid, block, 0, stream, 1, a);
}

}  // namespace
}  // namespace b2

extern "C" int b2_add_rms_norm_quantize(const b2_norm_quantize* p, void* stream) {
  using namespace b2;
  const char* const op = "add_rms_norm_quantize";
  if (p == nullptr || p->struct_size != sizeof(b2_norm_quantize)) return fail_invalid(op, "struct_size does not match");
  if (p->tokens < 0 || p->tokens >= (1LL << 31)) return fail_invalid(op, "tokens must be from 0 to 2^31 - 1");
  if (p->dim <= 0 || p->dim > kMostDim || p->dim % 8 != 0) return fail_invalid(op, "dim must be a multiple of 8 from 8 to 32768");
  if (p->group != 0 && ((p->group != 32 && p->group != 64 && p->group != 128 && p->group != 256) || p->dim % p->group != 0))
    return fail_invalid(op, "group must be 0, 32, 64, 128 or 256 and divide dim");
  if (!(p->eps >= 0.0f) || std::isinf(p->eps)) return fail_invalid(op, "eps must be a finite number of at least 0");
  if (p->codes != B2_CODES_INT8 && p->codes != B2_CODES_E4M3) return fail_invalid(op, "codes must be B2_CODES_INT8 or B2_CODES_E4M3");
  if (!dtype_known(p->x_dtype)) return fail_invalid(op, "x_dtype is not a type that this call takes");
  if (p->residual == nullptr && p->residual_out != nullptr) return fail_invalid(op, "residual_out needs a residual");
  if (p->residual != nullptr && p->residual_dtype != p->x_dtype && p->residual_dtype != B2_DTYPE_F32)
    return fail_invalid(op, "the residual must have x's type or be fp32");
  if (p->weight != nullptr && !dtype_known(p->weight_dtype)) return fail_invalid(op, "weight_dtype is not a type that this call takes");
  if (p->norm_out != nullptr && (!dtype_known(p->norm_dtype) || p->norm_dtype == B2_DTYPE_F32)) return fail_invalid(op, "norm_out must be bf16 or fp16");
  if (p->tokens == 0) return B2_OK;
  const int r_dtype = p->residual != nullptr ? p->residual_dtype : p->x_dtype;
  if (!matrix_ok(p->x, p->ldx, p->dim, dtype_bytes(p->x_dtype))) return fail_invalid(op, "x must be 16-byte aligned rows of at least dim elements");
  if (p->residual != nullptr && !matrix_ok(p->residual, p->ld_residual, p->dim, dtype_bytes(r_dtype)))
    return fail_invalid(op, "residual must be 16-byte aligned rows of at least dim elements");
  if (p->residual_out != nullptr && !matrix_ok(p->residual_out, p->ld_residual_out, p->dim, dtype_bytes(r_dtype)))
    return fail_invalid(op, "residual_out must be 16-byte aligned rows of at least dim elements");
  if (p->norm_out != nullptr && !matrix_ok(p->norm_out, p->ld_norm, p->dim, 2)) return fail_invalid(op, "norm_out must be 16-byte aligned rows of at least dim elements");
  if (p->weight != nullptr && !aligned_to(p->weight, 16)) return fail_invalid(op, "weight must be 16-byte aligned");
  if (p->q == nullptr || !aligned_to(p->q, 8) || p->ldq < p->dim || p->ldq % 8 != 0) return fail_invalid(op, "q must be 8-byte aligned rows of at least dim codes");
  if (p->scale == nullptr || !aligned_to(p->scale, 4)) return fail_invalid(op, "scale is missing or not aligned");
  // A row is read by its own threads alone: what is written in a tensor's place has its rows where that has them.
  const auto in_place = [&](const void* out, std::int64_t ld_out, int out_dtype, const void* in, std::int64_t ld, int dtype) {
    return out != in || (dtype_bytes(out_dtype) == dtype_bytes(dtype) && (ld_out == ld || p->tokens == 1));
  };
  if (p->residual_out != nullptr && (!in_place(p->residual_out, p->ld_residual_out, r_dtype, p->x, p->ldx, p->x_dtype) ||
                                     !in_place(p->residual_out, p->ld_residual_out, r_dtype, p->residual, p->ld_residual, r_dtype)))
    return fail_invalid(op, "residual_out in the place of x or of the residual must have its rows and its type");
  if (p->norm_out != nullptr && !in_place(p->norm_out, p->ld_norm, p->norm_dtype, p->x, p->ldx, p->x_dtype))
    return fail_invalid(op, "norm_out in x's place must have x's rows, of 16 bits");
  if (p->norm_out != nullptr && p->norm_out == p->residual_out) return fail_invalid(op, "norm_out and residual_out must be two matrices");
  NormArgs a{p->x, p->ldx, p->residual, p->ld_residual, p->residual_out, p->ld_residual_out, p->weight, p->weight_dtype, p->norm_out, p->ld_norm,
             p->norm_dtype == B2_DTYPE_F16, p->q, p->ldq, p->scale, p->tokens, p->dim, p->group, 0, p->eps};
  const cudaStream_t s = as_stream(stream);
  const auto go = [&](auto x, auto r) {
    using X = decltype(x);
    using R = decltype(r);
    return p->codes == B2_CODES_E4M3 ? launch<X, R, true>(op, a, s) : launch<X, R, false>(op, a, s);
  };
  if (p->x_dtype == B2_DTYPE_F32) return go(float{}, float{});
  if (p->x_dtype == B2_DTYPE_F16) return r_dtype == B2_DTYPE_F32 ? go(__half{}, float{}) : go(__half{}, __half{});
  return r_dtype == B2_DTYPE_F32 ? go(__nv_bfloat16{}, float{}) : go(__nv_bfloat16{}, __nv_bfloat16{});
}
