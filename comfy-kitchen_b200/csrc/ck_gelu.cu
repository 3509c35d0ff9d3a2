// GELU (tanh form) whose input is kept as an MXFP8 copy, for sm_100a: the forward pass writes the result and the copy, the
// backward pass reads the copy.
//
//   y  = u s,   s = 1 / (1 + exp(-2 z)),   z = sqrt(2/pi) (u + 0.044715 u^3)      (u s = u/2 (1 + tanh z))
//   du = dy (s + 2 u s (1 - s) z'),   z' = sqrt(2/pi) (1 + 3 * 0.044715 u^2),   u the value that stands in the copy
//
// Both are bound by HBM: 2 bytes read and 3.03 written, 3.03 read and 2 written, for an element of a 16-bit type.  A thread takes
// one block of 32 elements of a row, as the MXFP8 quantizer does: its scale needs no exchange between lanes.  4608 x 12288 bf16: 45 and 46 us,
// 6.2 TB/s, 95 % of what a copy reaches.
#include "ck_rows.cuh"

namespace ck {
namespace {

using namespace rows;

constexpr int kBlocksOfRow = 64, kRowsOfGrid = 4;  // scale blocks and rows of a thread block
constexpr float kRoot = 0.7978845608028654f;       // sqrt(2 / pi)
constexpr float kCubic = 0.044715f;

// 2^-8 exp(-2 z) and 2^8 s = 1 / (2^-8 + 2^-8 exp(-2 z)) for two elements at a time: a product for u^2, two fused steps for the exponent to the base
// of two, the chip's power and reciprocal (2 and 1 units in the last place).  The factor of 2^8 keeps the reciprocal a normal number until s is below
// 2^-126; where u is so negative that the power is infinite, s is zero.  With exact divisions and their range
// checks the kernels were bound by instructions: 58 and 70 us at 4608 x 12288 bf16 against 45 and 46.
struct Gate {
  float2 t, r;
};
__device__ __forceinline__ Gate gate(float2 u, float2 squares) {
  constexpr float kLog2e = 1.4426950408889634f;
  const float2 p = fma_x2(squares, both(-2.0f * kRoot * kLog2e * kCubic), both(-2.0f * kRoot * kLog2e));
  const float2 e = fma_x2(u, p, both(-8.0f));
  Gate g;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(g.t.x) : "f"(e.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(g.t.y) : "f"(e.y));
  const float2 d = add_x2(g.t, both(0x1p-8f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g.r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(g.r.y) : "f"(d.y));
  return g;
}

__device__ __forceinline__ float2 gelu(float2 u) { return mul_x2(u, mul_x2(gate(u, mul_x2(u, u)).r, both(0x1p-8f))); }

// s + 2 u s (1 - s) z', with 1 - s as exp(-2 z) s, which keeps its digits where s is close to one.  Beyond +-10 the gate is
// within 1e-37 of 0 or 1 and u times its slope within 1e-35 of 0, while u^2 could overflow: the limits stand for all such u.  NaN stays NaN.
__device__ __forceinline__ float2 gelu_slope(float2 u) {
  asm("min.NaN.f32 %0, %0, 0f41200000;" : "+f"(u.x));
  asm("min.NaN.f32 %0, %0, 0f41200000;" : "+f"(u.y));
  asm("max.NaN.f32 %0, %0, 0fC1200000;" : "+f"(u.x));
  asm("max.NaN.f32 %0, %0, 0fC1200000;" : "+f"(u.y));
  const float2 squares = mul_x2(u, u);
  const Gate g = gate(u, squares);
  const float2 s = mul_x2(g.r, both(0x1p-8f)), slope = mul_x2(u, fma_x2(squares, both(6.0f * kRoot * kCubic), both(2.0f * kRoot)));
  return fma_x2(slope, mul_x2(mul_x2(g.t, g.r), s), s);
}

template <typename T>
__device__ __forceinline__ void load_block(const T* p, float2 (&f)[16]) {
  constexpr int kVec = 32 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 32 / kVec; ++i) {
    const Vec256 w = ld_global_stream_256(p + i * kVec);
    float2 part[kVec / 2];
    unpack(*reinterpret_cast<const Raw<T, kVec>*>(&w), part);
#pragma unroll
    for (int j = 0; j < kVec / 2; ++j) f[i * (kVec / 2) + j] = part[j];
  }
}

template <typename T>
__device__ __forceinline__ void store_block(T* p, const float2 (&f)[16]) {
  constexpr int kVec = 32 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 32 / kVec; ++i) {
    float2 part[kVec / 2];
#pragma unroll
    for (int j = 0; j < kVec / 2; ++j) part[j] = f[i * (kVec / 2) + j];
    const Raw<T, kVec> r = pack<T, kVec>(part);
    st_global_256(p + i * kVec, *reinterpret_cast<const Vec256*>(&r));
  }
}

template <typename T>
__global__ void __launch_bounds__(kBlocksOfRow * kRowsOfGrid)
gelu_mxfp8_forward_kernel(const T* x, T* y, uint8_t* codes, uint8_t* scales, int64_t rows, int64_t cols, int64_t blocks_padded) {
  pdl_launch_dependents();
  const int64_t block = static_cast<int64_t>(blockIdx.y) * kBlocksOfRow + threadIdx.x;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsOfGrid + threadIdx.y;
  pdl_wait();
  uint32_t byte = 0;
  if (row < rows && block < cols >> 5) {
    const int64_t at = row * cols + block * 32;
    float2 u[16];
    load_block(x + at, u);
    if (codes != nullptr) {
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fmaxf(fabsf(u[i].x), fabsf(u[i].y)));
      const quant::Mxfp8Scale s = block_scale(amax);
      Vec256 out;
#pragma unroll
      for (int i = 0; i < 8; ++i) out.w[i] = block_codes(u[2 * i], u[2 * i + 1], s);
      st_global_256(codes + at, out);
      byte = s.byte;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) u[i] = gelu(u[i]);
    store_block(y + at, u);
  }
  if (codes == nullptr) return;
  // four bytes of a row are one store; padding rows and blocks are zero
  uint32_t word = byte | (__shfl_xor_sync(0xFFFFFFFFu, byte, 1) << 8);
  word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2) << 16;
  if (block < blocks_padded && (block & 3) == 0) {
    *reinterpret_cast<uint32_t*>(scales + swizzled_scale_offset(row, block, blocks_padded >> 2)) = word;
  }
}

template <typename T>
__global__ void __launch_bounds__(kBlocksOfRow * kRowsOfGrid)
gelu_mxfp8_backward_kernel(const T* dy, const uint8_t* codes, const uint8_t* scales, T* dx, int64_t rows, int64_t cols, int64_t blocks_padded) {
  pdl_launch_dependents();
  const int64_t block = static_cast<int64_t>(blockIdx.y) * kBlocksOfRow + threadIdx.x;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowsOfGrid + threadIdx.y;
  pdl_wait();
  if (row >= rows || block >= cols >> 5) return;
  const int64_t at = row * cols + block * 32;
  const Vec256 held = ld_global_stream_256(codes + at);
  const float factor = e8m0_factor(ld_global_u8(scales + swizzled_scale_offset(row, block, blocks_padded >> 2)));
  float2 d[16];
  load_block(dy + at, d);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float2 u = mul_x2(e4m3_pair((held.w[i / 2] >> (16 * (i & 1))) & 0xFFFFu), both(factor));
    d[i] = mul_x2(d[i], gelu_slope(u));
  }
  store_block(dx + at, d);
}

int check(const char* op, const void* in, const void* out, const void* codes, const void* scales, int dtype, int64_t rows, int64_t cols) {
  CK_REQUIRE(in && out, "%s: null pointer", op);
  CK_REQUIRE(dtype == CK_DTYPE_F32 || dtype == CK_DTYPE_F16 || dtype == CK_DTYPE_BF16, "%s: unsupported dtype code %d", op, dtype);
  CK_REQUIRE(rows > 0 && cols > 0 && cols % 32 == 0, "%s: bad shape [%lld, %lld]", op, (long long)rows, (long long)cols);
  CK_REQUIRE(reinterpret_cast<uintptr_t>(in) % 32 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0 && reinterpret_cast<uintptr_t>(codes) % 32 == 0 &&
                 reinterpret_cast<uintptr_t>(scales) % 4 == 0,
             "%s: tensors have to be aligned to 32 bytes, scales to 4", op);
  CK_REQUIRE(round_up(rows, 128) / kRowsOfGrid <= 0x7FFFFFFF && ceil_div(cols, 32 * kBlocksOfRow) <= 65535, "%s: tensor too large", op);
  return CK_OK;
}

template <typename T>
int launch_forward(const void* x, void* y, void* codes, void* scales, int64_t rows, int64_t cols, cudaStream_t s) {
  const int64_t padded = round_up(cols / 32, 4);
  const dim3 grid(static_cast<unsigned>(round_up(rows, 128) / kRowsOfGrid), static_cast<unsigned>(ceil_div(padded, kBlocksOfRow)));
  CK_CUDA(launch_pdl(gelu_mxfp8_forward_kernel<T>, grid, dim3(kBlocksOfRow, kRowsOfGrid), 0, s, static_cast<const T*>(x), static_cast<T*>(y),
                     static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), rows, cols, padded));
  return CK_OK;
}

template <typename T>
int launch_backward(const void* dy, const void* codes, const void* scales, void* dx, int64_t rows, int64_t cols, cudaStream_t s) {
  const int64_t padded = round_up(cols / 32, 4);
  const dim3 grid(static_cast<unsigned>(ceil_div(rows, kRowsOfGrid)), static_cast<unsigned>(ceil_div(padded, kBlocksOfRow)));
  CK_CUDA(launch_pdl(gelu_mxfp8_backward_kernel<T>, grid, dim3(kBlocksOfRow, kRowsOfGrid), 0, s, static_cast<const T*>(dy),
                     static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<T*>(dx), rows, cols, padded));
  return CK_OK;
}

}  // namespace
}  // namespace ck

extern "C" int ck_gelu_mxfp8_forward(const void* x, int dtype, void* y, void* codes, void* block_scales, int64_t rows, int64_t cols,
                                     void* stream) {
  using namespace ck;
  CK_REQUIRE((codes == nullptr) == (block_scales == nullptr), "gelu_mxfp8_forward: codes and block_scales go together");
  if (int rc = check("gelu_mxfp8_forward", x, y, codes, block_scales, dtype, rows, cols)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CK_DTYPE_BF16: return launch_forward<__nv_bfloat16>(x, y, codes, block_scales, rows, cols, s);
    case CK_DTYPE_F16: return launch_forward<__half>(x, y, codes, block_scales, rows, cols, s);
    default: return launch_forward<float>(x, y, codes, block_scales, rows, cols, s);
  }
}

extern "C" int ck_gelu_mxfp8_backward(const void* dy, int dtype, const void* codes, const void* block_scales, void* dx, int64_t rows, int64_t cols,
                                      void* stream) {
  using namespace ck;
  CK_REQUIRE(codes && block_scales, "gelu_mxfp8_backward: null pointer");
  if (int rc = check("gelu_mxfp8_backward", dy, dx, codes, block_scales, dtype, rows, cols)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CK_DTYPE_BF16: return launch_backward<__nv_bfloat16>(dy, codes, block_scales, dx, rows, cols, s);
    case CK_DTYPE_F16: return launch_backward<__half>(dy, codes, block_scales, dx, rows, cols, s);
    default: return launch_backward<float>(dy, codes, block_scales, dx, rows, cols, s);
  }
}
