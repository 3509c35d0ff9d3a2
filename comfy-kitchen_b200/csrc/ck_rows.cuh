// What the row-wise training kernels (layer norm, GELU) share: vectors of a row in registers, sums over a warp, and the
// MXFP8 copy of a row (E4M3 codes, tiled E8M0 scales) written and read beside the arithmetic.
#pragma once

#include <type_traits>

#include "ck_quant_math.cuh"
#include "ck_sm100.cuh"

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

// The same as pairs of fp32 numbers, the form that one instruction computes on.
template <typename T, int kVec>
__device__ __forceinline__ void unpack(const Raw<T, kVec>& r, float2 (&f)[kVec / 2]) {
  float v[kVec];
  unpack(r, v);
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i) f[i] = make_float2(v[2 * i], v[2 * i + 1]);
}
template <typename T, int kVec>
__device__ __forceinline__ Raw<T, kVec> pack(const float2 (&f)[kVec / 2]) {
  float v[kVec];
#pragma unroll
  for (int i = 0; i < kVec / 2; ++i) {
    v[2 * i] = f[i].x;
    v[2 * i + 1] = f[i].y;
  }
  return pack<T, kVec>(v);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// 1 / sqrt(v): the hardware's estimate and a Newton step.  Where the step would meet infinities the estimate is the value.
__device__ __forceinline__ float inverse_root(float v) {
  const float r = rsqrtf(v);
  const float better = r * fmaf(-0.5f * v * r, r, 1.5f);
  return v > 0.0f && v < 3e38f ? better : r;
}

// The scale of an MXFP8 block as quant::mxfp8_scale has it, by integers where neither the byte nor its factor is special: with
// amax = m 2^E and 448 = 1.75 2^8 the exponent is E - 8, and one more where m > 1.75.  (The rounded quotient amax / 448 that the definition
// takes the logarithm of says the same: the fp32 number above 1.75 2^E gives 1 + 2^-23.8, which rounds to 1 + 2^-23, not to 1.)
__device__ __forceinline__ quant::Mxfp8Scale block_scale(float amax) {
  const uint32_t e = ((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 8u;
  if (e - 1u < 250u && __float_as_uint(amax) < 0x7F800000u) return {__uint_as_float((254u - e) << 23), e, false};
  return quant::mxfp8_scale(amax);
}

// Four values of a block -> four codes.
__device__ __forceinline__ uint32_t block_codes(float2 a, float2 b, const quant::Mxfp8Scale& s) {
  a = mul_x2(a, both(s.inv));
  b = mul_x2(b, both(s.inv));
  const uint32_t w = quant::f32x2_to_e4m3x2(a.y, a.x) | (quant::f32x2_to_e4m3x2(b.y, b.x) << 16);
  return s.dead ? 0u : w;
}

// Rows in two levels: row r is row r % inner of outer index r / inner.
struct RowStrides {
  int64_t outer_stride;  // elements
  int64_t inner_stride;
  uint32_t inner;
  __device__ __forceinline__ int64_t offset(uint32_t row) const {
    const uint32_t o = row < inner ? 0u : row / inner;
    return static_cast<int64_t>(o) * outer_stride + static_cast<int64_t>(row - o * inner) * inner_stride;
  }
};

}  // namespace rows
}  // namespace ck
