// What the operators around a text decoder's attention share (norm_quantize.cu, lora.cu, logprobs.cu): element types, eight neighbouring elements as
// fp32 and back. No counterpart in the reference.
#pragma once

#include <type_traits>

#include "paged.cuh"

namespace b2 {

inline int dtype_bytes(int dtype) { return dtype == B2_DTYPE_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype == B2_DTYPE_BF16 || dtype == B2_DTYPE_F16 || dtype == B2_DTYPE_F32; }
// Rows of a matrix that are read and written 16 bytes at a time.
inline bool matrix_ok(const void* p, std::int64_t ld, std::int64_t width, int bytes) {
  return p != nullptr && aligned_to(p, 16) && ld >= width && ld * bytes % 16 == 0;
}

#ifdef __CUDACC__
// Eight elements at p (16-byte aligned).
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (unsigned i = 0; i < sizeof(T) / 2; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    if constexpr (sizeof(T) == 2) {
      load8<T>(v[0], x);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[4 * i] = __uint_as_float(v[i].x), x[4 * i + 1] = __uint_as_float(v[i].y);
        x[4 * i + 2] = __uint_as_float(v[i].z), x[4 * i + 3] = __uint_as_float(v[i].w);
      }
    }
  }
};
template <typename T>
__device__ __forceinline__ void put8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = store8<T>(x);
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}
#endif

}  // namespace b2
