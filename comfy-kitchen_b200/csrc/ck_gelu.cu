// GELU (tanh form) whose input is kept as an MXFP8 copy, for sm_100a: the forward pass writes the result and the copy, the
// backward pass reads the copy.
//
//   y  = u s,   s = 1 / (1 + exp(-2 z)),   z = sqrt(2/pi) (u + 0.044715 u^3)      (u s = u/2 (1 + tanh z))
//   du = dy (s + 2 u s (1 - s) z'),   z' = sqrt(2/pi) (1 + 3 * 0.044715 u^2),   u the value that stands in the copy
//
// Both are bound by HBM: 2 bytes read and 3.03 written, 3.03 read and 2 written, for an element of a 16-bit type.  A thread takes
// one block of 32 elements of a row, as the MXFP8 quantizer does: its scale needs no exchange between lanes.
#include "ck_rows.cuh"

namespace ck {
namespace {

using namespace rows;

constexpr int kBlocksOfRow = 64, kRowsOfGrid = 4;  // scale blocks and rows of a thread block
constexpr float kRoot = 0.7978845608028654f;       // sqrt(2 / pi)
constexpr float kCubic = 0.044715f;

// exp(-2 z): infinite for a large negative u, whose gate 1 / (1 + exp(-2 z)) is zero
__device__ __forceinline__ float gelu_exp(float u) { return __expf(-2.0f * kRoot * fmaf(kCubic * u * u, u, u)); }

__device__ __forceinline__ float gelu(float u) { return u / (1.0f + gelu_exp(u)); }

// s + 2 u s (1 - s) z', with 1 - s as exp(-2 z) s, which keeps its digits where s is close to one.  Beyond +-10 the gate is
// within 1e-37 of 0 or 1 and u times its slope within 1e-35 of 0, while u^2 could overflow: the limits stand for all such u.  NaN stays NaN.
__device__ __forceinline__ float gelu_slope(float u) {
  u = u > 10.0f ? 10.0f : (u < -10.0f ? -10.0f : u);
  const float t = gelu_exp(u), s = 1.0f / (1.0f + t);
  return fmaf(u * 2.0f * kRoot * fmaf(3.0f * kCubic * u, u, 1.0f), t * s * s, s);
}

template <typename T>
__device__ __forceinline__ void load_block(const T* p, float (&f)[32]) {
  constexpr int kVec = 32 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 32 / kVec; ++i) {
    const Vec256 w = ld_global_stream_256(p + i * kVec);
    float part[kVec];
    unpack(*reinterpret_cast<const Raw<T, kVec>*>(&w), part);
#pragma unroll
    for (int j = 0; j < kVec; ++j) f[i * kVec + j] = part[j];
  }
}

template <typename T>
__device__ __forceinline__ void store_block(T* p, const float (&f)[32]) {
  constexpr int kVec = 32 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 32 / kVec; ++i) {
    float part[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) part[j] = f[i * kVec + j];
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
    float u[32];
    load_block(x + at, u);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(u[i]));
    const quant::Mxfp8Scale s = block_scale(amax);
    Vec256 out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out.w[i] = block_codes(make_float2(u[4 * i], u[4 * i + 1]), make_float2(u[4 * i + 2], u[4 * i + 3]), s);
    st_global_256(codes + at, out);
    byte = s.byte;
#pragma unroll
    for (int i = 0; i < 32; ++i) u[i] = gelu(u[i]);
    store_block(y + at, u);
  }
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
  float d[32];
  load_block(dy + at, d);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float u[4];
    e4m3_four(held.w[i], factor, u);
#pragma unroll
    for (int j = 0; j < 4; ++j) d[4 * i + j] *= gelu_slope(u[j]);
  }
  store_block(dx + at, d);
}

int check(const char* op, const void* in, const void* out, const void* codes, const void* scales, int dtype, int64_t rows, int64_t cols) {
  CK_REQUIRE(in && out && codes && scales, "%s: null pointer", op);
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
  if (int rc = check("gelu_mxfp8_backward", dy, dx, codes, block_scales, dtype, rows, cols)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CK_DTYPE_BF16: return launch_backward<__nv_bfloat16>(dy, codes, block_scales, dx, rows, cols, s);
    case CK_DTYPE_F16: return launch_backward<__half>(dy, codes, block_scales, dx, rows, cols, s);
    default: return launch_backward<float>(dy, codes, block_scales, dx, rows, cols, s);
  }
}
