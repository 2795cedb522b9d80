// Storage types of the trainable block's operators (layernorm.hip, linear16.hip, gradclip.hip): fp32, bf16 or fp16 in memory, fp32 in
// registers.  A vector access moves 16 bytes per lane from any element address: global memory takes 16-byte accesses at every
// alignment of the element type, so rows that start anywhere (odd widths, slices) need no path of their own.
#pragma once
#include "common.h"

#include <atomic>

namespace hopmi {

constexpr int T_F32 = 0, T_BF16 = 1, T_F16 = 2;      // dtype codes of the C ABI

typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes at any element address
typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));

template <typename T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };

template <typename T> __device__ __forceinline__ u32x4_t ld16(const T* p) { return *reinterpret_cast<const u32x4_any*>(p); }
template <typename T> __device__ __forceinline__ void st16(T* p, u32x4_t v) { *reinterpret_cast<u32x4_any*>(p) = v; }

// element e (a compile-time constant after unrolling) of a 16-byte vector, widened
__device__ __forceinline__ float vget(const u32x4_t& v, int e, const float*) { return __uint_as_float(v[e]); }
__device__ __forceinline__ float vget(const u32x4_t& v, int e, const __bf16*) {
  const unsigned w = v[e >> 1];
  return __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
}
__device__ __forceinline__ float vget(const u32x4_t& v, int e, const _Float16*) {
  const unsigned w = v[e >> 1];
  return (float)__builtin_bit_cast(_Float16, (unsigned short)((e & 1) ? (w >> 16) : (w & 0xffffu)));
}

// two values rounded to nearest even and packed, element 0 in the low half
__device__ __forceinline__ unsigned pk2(float a, float b, const __bf16*) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  const b2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ unsigned pk2(float a, float b, const _Float16*) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const h2 v = {(_Float16)a, (_Float16)b};
  return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ u32x4_t vpack(const float* f, const float*) {
  return u32x4_t{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
}
template <typename T> __device__ __forceinline__ u32x4_t vpack(const float* f, const T* t) {
  return u32x4_t{pk2(f[0], f[1], t), pk2(f[2], f[3], t), pk2(f[4], f[5], t), pk2(f[6], f[7], t)};
}

// Lets a kernel have `bytes` of dynamic LDS on the current device; `done` (one per kernel) holds the devices that have been told.
inline void allow_lds(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return;              // (the launch reports it)
  const unsigned long long bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  else (void)hipGetLastError();
}

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

// N consecutive elements from any element address, widened (N * sizeof(T) = 16 or 32 bytes)
template <int N, typename T> __device__ __forceinline__ void ldf(const T* p, float (&f)[N]) {
  constexpr int V = Vec<T>::N;
  static_assert(N % V == 0, "whole 16-byte vectors");
#pragma unroll
  for (int i = 0; i < N / V; ++i) {
    const u32x4_t v = ld16(p + i * V);
#pragma unroll
    for (int e = 0; e < V; ++e) f[i * V + e] = vget(v, e, p);
  }
}

// The sum over a wave's 64 lanes, in every lane, without the LDS pipe: lane exchanges within 16 lanes (DPP), then between the 16-lane rows
// and the halves (gfx950's row swaps).  Each exchange adds two values that both partners hold, so all lanes end with the same bits.
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = dpp_add<0xb1>(v);                            // lanes 1, 0, 3, 2
  v = dpp_add<0x4e>(v);                            // 2, 3, 0, 1
  v = dpp_add<0x141>(v);                           // mirrored within 8
  v = dpp_add<0x140>(v);                           // mirrored within 16
  const auto h = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(h[0]) + __uint_as_float(h[1]);
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(w[0]) + __uint_as_float(w[1]);
}

}  // namespace hopmi
