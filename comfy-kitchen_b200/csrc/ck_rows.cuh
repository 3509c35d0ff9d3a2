// What the row-wise training kernels (layer norm, GELU) share: vectors of a row in registers, sums over a warp, and the
// MXFP8 copy of a row (E4M3 codes, tiled E8M0 scales) written and read beside the arithmetic.
#pragma once

#include <type_traits>

#include "ck_common.cuh"
#include "ck_quant_math.cuh"

namespace ck {
namespace rows {

// kVec consecutive elements as they stand in memory.
template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Raw {
  T v[kVec];
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return __float2bfloat16_rn(v);
  } else if constexpr (std::is_same<T, __half>::value) {
    return __float2half_rn(v);
  } else {
    return v;
  }
}

template <typename T, int kVec>
__device__ __forceinline__ void unpack(const Raw<T, kVec>& r, float (&f)[kVec]) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value && kVec % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  } else if constexpr (std::is_same<T, __half>::value && kVec % 2 == 0) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) {
      const float2 p = __half22float2(h[i]);
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) f[i] = to_float(r.v[i]);
  }
}

template <typename T, int kVec>
__device__ __forceinline__ Raw<T, kVec> pack(const float (&f)[kVec]) {
  Raw<T, kVec> r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value && kVec % 2 == 0) {
    __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&r);
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) p[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
  } else if constexpr (std::is_same<T, __half>::value && kVec % 2 == 0) {
    __half2* p = reinterpret_cast<__half2*>(&r);
#pragma unroll
    for (int i = 0; i < kVec / 2; ++i) p[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) r.v[i] = from_float<T>(f[i]);
  }
  return r;
}

template <typename T, int kVec>
__device__ __forceinline__ Raw<T, kVec> zeros() {
  Raw<T, kVec> r;
#pragma unroll
  for (int i = 0; i < kVec; ++i) r.v[i] = from_float<T>(0.0f);
  return r;
}

// A vector of a row that this SM reads once (16 bytes: no line in L1).  Coherent loads: the row may come from the kernel before
// this one, behind whose end the caller has waited.
template <typename T, int kVec>
__device__ __forceinline__ Raw<T, kVec> load_once(const T* p) {
  Raw<T, kVec> r;
  if constexpr (sizeof(T) * kVec == 16) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p) : "memory");
  } else {
    r = *reinterpret_cast<const Raw<T, kVec>*>(p);
  }
  return r;
}

template <typename T, int kVec>
__device__ __forceinline__ void store(T* p, const Raw<T, kVec>& r) {
  *reinterpret_cast<Raw<T, kVec>*>(p) = r;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Factor of an E8M0 byte, as the dequantizer has it: byte 0 stands for zero.
__device__ __forceinline__ float e8m0_factor(uint32_t byte) { return __uint_as_float(byte << 23); }

// Two E4M3 codes (low half of `pair`) -> their values.
__device__ __forceinline__ float2 e4m3_pair(uint32_t pair) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(pair)));
  return __half22float2(*reinterpret_cast<const __half2*>(&h2));
}

// Four codes of one scale block -> the values they stand for.
__device__ __forceinline__ void e4m3_four(uint32_t word, float factor, float* f) {
  const float2 lo = e4m3_pair(word & 0xFFFFu), hi = e4m3_pair(word >> 16);
  f[0] = lo.x * factor;
  f[1] = lo.y * factor;
  f[2] = hi.x * factor;
  f[3] = hi.y * factor;
}

// Rows in two levels: row r is row r % inner of outer index r / inner.
struct RowStrides {
  int64_t outer_stride;  // elements
  int64_t inner_stride;
  uint32_t inner;
  __device__ __forceinline__ int64_t offset(uint32_t row) const {
    const uint32_t o = row / inner;
    return static_cast<int64_t>(o) * outer_stride + static_cast<int64_t>(row - o * inner) * inner_stride;
  }
};

}  // namespace rows
}  // namespace ck
