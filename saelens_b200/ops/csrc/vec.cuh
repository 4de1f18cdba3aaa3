// Loads and stores of VEC consecutive elements of fp32, bf16 or fp16 as fp32 values.  The pointer
// is aligned to the access (VEC * sizeof(T), at most 16 bytes); wider vectors are split into
// 16-byte accesses.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

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

// two 16-bit values in one word
template <class T>
__device__ __forceinline__ float2 pair_to_f(uint32_t w) {
  if constexpr (sizeof(T) != 2) return make_float2(0.f, 0.f);
  else if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <class T>
__device__ __forceinline__ uint32_t pair_from_f(float lo, float hi) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

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
  // All values at once: 16-bit ones are converted in pairs, one instruction for two on the way back.
  __device__ __forceinline__ void unpack(float (&f)[VEC]) const {
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(r);
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) {
        const float2 p = pair_to_f<T>(w[j]);
        f[2 * j] = p.x;
        f[2 * j + 1] = p.y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = get(j);
    }
  }
  __device__ __forceinline__ void pack(const float (&f)[VEC]) {
    if constexpr (sizeof(T) == 2 && VEC % 2 == 0) {
      uint32_t* w = reinterpret_cast<uint32_t*>(r);
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j) w[j] = pair_from_f<T>(f[2 * j], f[2 * j + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) set(j, f[j]);
    }
  }
  __device__ __forceinline__ float get(int j) const { return to_f<T>(reinterpret_cast<const T*>(r)[j]); }
  __device__ __forceinline__ void set(int j, float v) { reinterpret_cast<T*>(r)[j] = from_f<T>(v); }
};

}  // namespace vec
}  // namespace sb
