// Element types, vector accesses and small reductions shared by the token operators (layer norm, rotary positions,
// cross attention).  All arithmetic is fp32; a 16-bit value is rounded once, when it is stored.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "d2c_common.cuh"

namespace d2c {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N elements moved by one access (N * sizeof(T) bytes, aligned to that; 32 bytes is sm_100's widest).
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load_vec(const T* p) {
  Vec<T, N> r;
  constexpr int bytes = sizeof(T) * N;
  if constexpr (bytes == 32) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
  } else {
    r = *reinterpret_cast<const Vec<T, N>*>(p);
  }
  return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const Vec<T, N>& r) {
  constexpr int bytes = sizeof(T) * N;
  if constexpr (bytes == 32) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    *reinterpret_cast<Vec<T, N>*>(p) = r;
  }
}

// Pairs of floats: one instruction for two operations.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_split(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Two 16-bit values of one word, and back (one conversion for both).
template <typename T>
__device__ __forceinline__ F2 unpack_word(uint32_t w) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  } else {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return f2(h.x, h.y);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack_word(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

inline size_t token_dtype_size(int dtype) { return dtype == D2C_F32 ? 4 : 2; }
inline bool token_dtype_ok(int dtype) { return dtype == D2C_F32 || dtype == D2C_F16 || dtype == D2C_BF16; }
inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Refuses a call (once) whose device reported that a bounded wait gave up; clears the report.
int take_device_status();

}  // namespace d2c
