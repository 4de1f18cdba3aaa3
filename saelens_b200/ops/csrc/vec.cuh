// Loads and stores of VEC consecutive elements of fp32, bf16 or fp16 as fp32 values.  The pointer
// is aligned to the access (VEC * sizeof(T), at most 16 bytes); wider vectors are split into
// 16-byte accesses.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace sb {
namespace vec {

template <class T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }

template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// the value that T holds for v
template <class T>
__device__ __forceinline__ float rounded(float v) { return to_f<T>(from_f<T>(v)); }

template <int BYTES>
struct Raw;
template <>
struct Raw<2> { using type = uint16_t; };
template <>
struct Raw<4> { using type = uint32_t; };
template <>
struct Raw<8> { using type = uint2; };
template <>
struct Raw<16> { using type = uint4; };

// VEC elements as they lie in memory
template <class T, int VEC>
struct Pack {
  static constexpr int kBytes = VEC * int(sizeof(T));
  static constexpr int kAccess = kBytes > 16 ? 16 : kBytes;
  static constexpr int kN = kBytes / kAccess;
  using R = typename Raw<kAccess>::type;
  R r[kN];

  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kN; ++i) r[i] = reinterpret_cast<const R*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kN; ++i) reinterpret_cast<R*>(p)[i] = r[i];
  }
  __device__ __forceinline__ void zero() {
    uint32_t* w = reinterpret_cast<uint32_t*>(r);
    if (kBytes < 4) {
      reinterpret_cast<uint16_t*>(r)[0] = 0;
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 4; ++i) w[i] = 0u;
    }
  }
  __device__ __forceinline__ float get(int j) const { return to_f<T>(reinterpret_cast<const T*>(r)[j]); }
  __device__ __forceinline__ void set(int j, float v) { reinterpret_cast<T*>(r)[j] = from_f<T>(v); }
};

}  // namespace vec
}  // namespace sb
