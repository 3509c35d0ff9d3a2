// Layer norm over the last dimension for sm_100a: forward, optionally with an MXFP8 copy of the input, and backward from the
// input or from that copy.
//
//   m = mean_k x,  v = mean_k (x - m)^2,  i = 1 / sqrt(v + eps),  h = (x - m) i
//   y = h f + b,   f = offset + w (1 without a weight)
//   g = dy f,      dx = i (g - mean_k g - h mean_k(g h)),   dw = sum_rows dy h,   db = sum_rows dy
//
// w and b belong to groups of consecutive rows (one group: the learned weight of a layer; one for each sample: modulation).
// Rows are taken in two levels of strides, so that a slice of the tokens of a longer buffer needs no copy.  All
// sums and statistics are fp32; a row stays in registers between its passes, so its mean is subtracted before
// squares are taken.  Results are rounded to their types once.
#include "ck_rows.cuh"

namespace ck {
namespace {

using namespace rows;

struct ForwardArgs {
  const void* x;
  RowStrides x_rows;
  const void* weight;  // null: 1
  const void* bias;    // null: 0
  int64_t weight_stride, bias_stride;  // between groups
  uint32_t rows_per_group;
  float offset, eps;
  void* y;
  float* mean;  // null: not wanted (inference)
  float* rstd;
  uint8_t* codes;  // null: no copy
  uint8_t* scales;
  uint32_t rows, rows_padded;
  int64_t cols;
  int* status;  // for waits that give up (ck_gemm_status)
  bool params_f32;      // else of x's type
  bool params_aligned;  // weights and biases start on vectors
};

template <typename W, int kVec>
__device__ __forceinline__ void load_param_of(const W* p, bool aligned, float (&f)[kVec]) {
  Raw<W, kVec> r;
  if (kVec > 1 && aligned) {
    r = *reinterpret_cast<const Raw<W, kVec>*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < kVec; ++i) r.v[i] = p[i];
  }
  unpack(r, f);
}

// kVec weights or biases from element `at` on: fp32 or of the type T.
template <typename T, int kVec>
__device__ __forceinline__ void load_param(const void* base, int64_t at, bool f32, bool aligned, float (&f)[kVec]) {
  if (!std::is_same<T, float>::value && f32) {
    if constexpr (kVec == 8) {  // two 16-byte loads
      float lo[4], hi[4];
      load_param_of<float, 4>(static_cast<const float*>(base) + at, aligned, lo);
      load_param_of<float, 4>(static_cast<const float*>(base) + at + 4, aligned, hi);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] = lo[i];
        f[4 + i] = hi[i];
      }
    } else {
      load_param_of<float, kVec>(static_cast<const float*>(base) + at, aligned, f);
    }
  } else {
    load_param_of<T, kVec>(static_cast<const T*>(base) + at, aligned, f);
  }
}

template <typename T>
__device__ __forceinline__ float param(const void* base, int64_t at, bool f32) {
  return f32 ? static_cast<const float*>(base)[at] : to_float(static_cast<const T*>(base)[at]);
}

template <typename T>
__device__ __forceinline__ void store_param(void* base, int64_t at, bool f32, float v) {
  if (f32) {
    static_cast<float*>(base)[at] = v;
  } else {
    static_cast<T*>(base)[at] = from_float<T>(v);
  }
}

// Sum over the warps of one row (threadIdx.y); `buf`: a slot for each warp of the block, another one for each sum of a kernel.
template <int kSlot>
__device__ __forceinline__ float row_sum(float v, float* buf) {
  v = warp_sum(v);
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  float* mine = buf + kSlot * 32 + threadIdx.y * warps;
  if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (int i = 0; i < warps; ++i) s += mine[i];
  return s;
}

// The MXFP8 copy of a row of which each lane holds kVec elements: codes beside the arithmetic's registers, a scale byte for
// every 32 elements, four of them in one 4-byte store.  Bits as ck_quantize_mxfp8 writes them.  All lanes of a warp come here.
template <int kVec>
__device__ __forceinline__ void store_mxfp8(const float2 (&f)[kVec / 2], bool inside, const ForwardArgs& a, uint32_t row, int64_t vec) {
  constexpr int kLanes = 32 / kVec;  // lanes of a block
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < kVec / 2; ++j) amax = fmaxf(amax, fmaxf(fabsf(f[j].x), fabsf(f[j].y)));
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
  const quant::Mxfp8Scale s = block_scale(amax);
  if (inside) {
    uint32_t words[kVec / 4];
#pragma unroll
    for (int j = 0; j < kVec / 4; ++j) words[j] = block_codes(f[2 * j], f[2 * j + 1], s);
    uint8_t* to = a.codes + static_cast<int64_t>(row) * a.cols + vec * kVec;
    if constexpr (kVec == 8) {
      *reinterpret_cast<uint2*>(to) = make_uint2(words[0], words[1]);
    } else {
      *reinterpret_cast<uint32_t*>(to) = words[0];
    }
  }
  uint32_t word = inside ? s.byte : 0u;
  word |= __shfl_down_sync(0xFFFFFFFFu, word, kLanes) << 8;
  word |= __shfl_down_sync(0xFFFFFFFFu, word, 2 * kLanes) << 16;
  if (inside && (threadIdx.x & (4 * kLanes - 1)) == 0) {
    const int64_t block = vec * kVec >> 5;
    *reinterpret_cast<uint32_t*>(a.scales + swizzled_scale_offset(row, block, ceil_div(a.cols >> 5, 4))) = word;
  }
}

// Rows past the last one: the scale layout's tiles are 128 rows high, and their padding reads as zeros.
__device__ __forceinline__ void clear_scales_of_row(const ForwardArgs& a, uint32_t row) {
  const int64_t quads = ceil_div(a.cols >> 5, 4);
  for (int64_t q = threadIdx.x; q < quads; q += blockDim.x) {
    *reinterpret_cast<uint32_t*>(a.scales + swizzled_scale_offset(row, q * 4, quads)) = 0u;
  }
}

// blockDim = (threads of a row, rows of a block); a thread holds kNum vectors, a row's thread count apart.
template <typename T, int kVec, int kNum, bool kCopy, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) layer_norm_forward_kernel(const ForwardArgs a) {
  __shared__ float buf[64];
  pdl_launch_dependents();
  const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < a.rows;
  const int64_t vecs = a.cols / kVec;
  pdl_wait();
  const T* x = static_cast<const T*>(a.x) + (live ? a.x_rows.offset(row) : 0);
  Raw<T, kVec> raw[kNum];
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
    const int64_t v = threadIdx.x + i * blockDim.x;
    raw[i] = live && v < vecs ? load_once<T, kVec>(x + v * kVec) : zeros<T, kVec>();
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
    float f[kVec];
    unpack(raw[i], f);
#pragma unroll
    for (int j = 0; j < kVec; ++j) sum += f[j];
  }
  const float mean = row_sum<0>(sum, buf) / static_cast<float>(a.cols);
  float square = 0.0f;
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
    float f[kVec];
    unpack(raw[i], f);
    if (threadIdx.x + i * blockDim.x < vecs) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) square = fmaf(f[j] - mean, f[j] - mean, square);
    }
  }
  const float rstd = inverse_root(row_sum<1>(square, buf) / static_cast<float>(a.cols) + a.eps);
  if constexpr (kCopy) {
    if (!live && row < a.rows_padded) clear_scales_of_row(a, row);
  }
  if (live && threadIdx.x == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  const int64_t group = live ? row / a.rows_per_group : 0;
  T* y = static_cast<T*>(a.y) + static_cast<int64_t>(row) * a.cols;
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
    const int64_t v = threadIdx.x + i * blockDim.x;
    const bool inside = live && v < vecs;
    if constexpr (kCopy) {
      float2 pairs[kVec / 2];
      unpack(raw[i], pairs);
      store_mxfp8<kVec>(pairs, inside, a, row, v);
    }
    float f[kVec];
    unpack(raw[i], f);
    if (inside) {
      float w[kVec], b[kVec];
      if (a.weight != nullptr) load_param<T, kVec>(a.weight, group * a.weight_stride + v * kVec, a.params_f32, a.params_aligned, w);
      if (a.bias != nullptr) load_param<T, kVec>(a.bias, group * a.bias_stride + v * kVec, a.params_f32, a.params_aligned, b);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const float h = (f[j] - mean) * rstd;
        f[j] = fmaf(h, a.weight != nullptr ? a.offset + w[j] : 1.0f, a.bias != nullptr ? b[j] : 0.0f);
      }
      store(y + v * kVec, pack<T, kVec>(f));
    }
  }
}

// ---- rows that come through shared memory
// A block's row is a bulk copy into a ring of stages, issued that many rows ahead by one thread, so that what is in flight
// does not depend on registers or on where the warps stand.  Barriers of the ring are mbarriers whose waits are bounded (mbar_wait).
struct Ring {
  uint32_t full;        // shared address of the stages' barriers
  volatile int* abort;  // a wait gave up
};
constexpr int kMaxRing = 4;

// A team of blockDim.x threads takes a row at a time; the block's rows are of one group, whose factors f and biases stand in shared memory
// as fp32 (`shared_params`) where there is room.  A row is unpacked once and stays in registers as fp32.  Mean and variance take one
// meeting of the team's warps: each brings the mean of what it holds and the squares about that.
template <typename T, int kVec, int kNum, bool kCopy>
__global__ void __launch_bounds__(1024) layer_norm_forward_ring_kernel(const ForwardArgs a, const uint32_t chunks, const uint32_t chunk_rows,
                                                                       const int stages, const bool shared_params) {
  constexpr int kPairs = kVec / 2;
  extern __shared__ __align__(128) uint8_t shared_bytes[];  // factors, biases, the teams' rings
  __shared__ __align__(8) uint64_t full[32][kMaxRing];
  __shared__ float2 buf[2][32];   // [turn][warp of the block]: mean and squares
  __shared__ float counts[32];    // elements that a team's warp holds
  __shared__ int abort_flag;
  pdl_launch_dependents();
  const int team = threadIdx.y, teams = blockDim.y, width = blockDim.x, warps = width >> 5, warp = threadIdx.x >> 5;
  const uint32_t group = blockIdx.x / chunks, chunk = blockIdx.x - group * chunks;
  const uint32_t begin = chunk * chunk_rows, end = min(a.rows_per_group, begin + chunk_rows), row0 = group * a.rows_per_group;
  const int vecs = static_cast<int>(a.cols / kVec);
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const uint32_t row_bytes = static_cast<uint32_t>(a.cols) * sizeof(T), stage_bytes = (row_bytes + 127) & ~127u;
  const uint32_t param_bytes = (static_cast<uint32_t>(a.cols) * 4 + 127) & ~127u;
  const bool weight = a.weight != nullptr, bias = a.bias != nullptr;
  float* const factor_buf = reinterpret_cast<float*>(shared_bytes);
  float* const bias_buf = reinterpret_cast<float*>(shared_bytes + (shared_params && weight ? param_bytes : 0u));
  const uint8_t* const ring = shared_bytes + (shared_params ? ((weight ? param_bytes : 0u) + (bias ? param_bytes : 0u)) : 0u) + team * stages * stage_bytes;
  const uint32_t ring_at = sm100::smem_u32(ring), full_at = sm100::smem_u32(full[team]);
  const auto load_row = [&](uint32_t r, int s) {  // by one thread of the team
    sm100::mbar_arrive_expect_tx(full_at + s * 8, row_bytes);
    sm100::bulk_load_1d(ring_at + s * stage_bytes, static_cast<const T*>(a.x) + a.x_rows.offset(row0 + r), row_bytes, full_at + s * 8);
  };
  int held = 0;
#pragma unroll
  for (int i = 0; i < kNum; ++i) held += max(0, min(32, vecs - warp * 32 - i * width)) * kVec;
  const float inv_held = held > 0 ? 1.0f / static_cast<float>(held) : 0.0f;
  if (team == 0 && (threadIdx.x & 31) == 0) counts[warp] = static_cast<float>(held);
  if (threadIdx.x == 0) {
    if (team == 0) abort_flag = 0;
    for (int s = 0; s < stages; ++s) sm100::mbar_init(&full[team][s], 1);
    sm100::fence_barrier_init();
    pdl_wait();
    for (int s = 0; s < stages; ++s) {
      const uint32_t r = begin + team + s * teams;
      if (r < end) load_row(r, s);
    }
  }
  pdl_wait();
  constexpr int kPart = 4;  // four of a vector lie together and the vectors 16 bytes apart: a warp's 16-byte loads meet no bank twice
  const int part_stride = vecs * kPart;
  if (shared_params) {
    for (int v = team * width + threadIdx.x; v < vecs; v += width * teams) {
      float f[kVec];
      if (weight) {
        load_param<T, kVec>(a.weight, group * a.weight_stride + static_cast<int64_t>(v) * kVec, a.params_f32, a.params_aligned, f);
#pragma unroll
        for (int j = 0; j < kVec; ++j) factor_buf[j / kPart * part_stride + v * kPart + j % kPart] = a.offset + f[j];
      }
      if (bias) {
        load_param<T, kVec>(a.bias, group * a.bias_stride + static_cast<int64_t>(v) * kVec, a.params_f32, a.params_aligned, f);
#pragma unroll
        for (int j = 0; j < kVec; ++j) bias_buf[j / kPart * part_stride + v * kPart + j % kPart] = f[j];
      }
    }
  }
  __syncthreads();
  const auto read_params = [&](const float* from, int v, float2(&f)[kPairs]) {
#pragma unroll
    for (int q = 0; q < kVec / kPart; ++q) {
      const float4 part = *reinterpret_cast<const float4*>(from + q * part_stride + v * kPart);
      f[2 * q] = make_float2(part.x, part.y);
      f[2 * q + 1] = make_float2(part.z, part.w);
    }
  };
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  for (uint32_t r = begin + team; r < end; r += teams, turn ^= 1) {
    if (!sm100::mbar_wait(full_at + stage * 8, phase, &abort_flag)) break;
    float2 f[kNum][kPairs];
    float2 sum = both(0.0f);
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const int v = threadIdx.x + i * width;
      if (v < vecs) {
        unpack(*reinterpret_cast<const Raw<T, kVec>*>(ring + stage * stage_bytes + v * 16), f[i]);
      } else {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) f[i][j] = both(0.0f);
      }
#pragma unroll
      for (int j = 0; j < kPairs; ++j) sum = add_x2(sum, f[i][j]);
    }
    const float mine = warp_sum(sum.x + sum.y) * inv_held;
    float2 square = both(0.0f);
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      if (static_cast<int>(threadIdx.x) + i * width < vecs) {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          const float2 d = add_x2(f[i][j], both(-mine));
          square = fma_x2(d, d, square);
        }
      }
    }
    float mean = mine, squares = warp_sum(square.x + square.y);
    if (warps > 1) {
      float2* const slots = buf[turn] + team * warps;
      if ((threadIdx.x & 31) == 0) slots[warp] = make_float2(mine, squares);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(width) : "memory");
      mean = 0.0f;
      for (int w = 0; w < warps; ++w) mean = fmaf(slots[w].x, counts[w], mean);
      mean *= inv_cols;
      squares = 0.0f;
      for (int w = 0; w < warps; ++w) {
        const float d = slots[w].x - mean;
        squares += fmaf(d * d, counts[w], slots[w].y);
      }
    } else {
      __syncwarp();
    }
    const float rstd = inverse_root(squares * inv_cols + a.eps);
    const uint32_t row = row0 + r;
    if (threadIdx.x == 0) {
      if (r + stages * teams < end) load_row(r + stages * teams, stage);  // all have read the stage
      if (a.mean != nullptr) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
      }
    }
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
    T* const y = static_cast<T*>(a.y) + static_cast<int64_t>(row) * a.cols;
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const int v = threadIdx.x + i * width;
      if constexpr (kCopy) store_mxfp8<kVec>(f[i], v < vecs, a, row, v);
      if (v >= vecs) continue;
      float2 w[kPairs], b[kPairs];
      if (shared_params) {
        if (weight) read_params(factor_buf, v, w);
        if (bias) read_params(bias_buf, v, b);
      } else {
        float p[kVec];
        if (weight) {
          load_param<T, kVec>(a.weight, group * a.weight_stride + static_cast<int64_t>(v) * kVec, a.params_f32, a.params_aligned, p);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) w[j] = make_float2(a.offset + p[2 * j], a.offset + p[2 * j + 1]);
        }
        if (bias) {
          load_param<T, kVec>(a.bias, group * a.bias_stride + static_cast<int64_t>(v) * kVec, a.params_f32, a.params_aligned, p);
#pragma unroll
          for (int j = 0; j < kPairs; ++j) b[j] = make_float2(p[2 * j], p[2 * j + 1]);
        }
      }
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        // in one step for 16-bit types, where a mean of that many times the deviation leaves no digits in x anyway
        f[i][j] = sizeof(T) == 2 ? fma_x2(f[i][j], both(rstd), both(-mean * rstd)) : mul_x2(add_x2(f[i][j], both(-mean)), both(rstd));
        if (weight && bias) {
          f[i][j] = fma_x2(f[i][j], w[j], b[j]);
        } else if (weight) {
          f[i][j] = mul_x2(f[i][j], w[j]);
        } else if (bias) {
          f[i][j] = add_x2(f[i][j], b[j]);
        }
      }
      store(y + static_cast<int64_t>(v) * kVec, pack<T, kVec>(f[i]));
    }
  }
  if constexpr (kCopy) {  // the scales' padding rows
    if (blockIdx.x == gridDim.x - 1) {
      for (uint32_t row = a.rows + team; row < a.rows_padded; row += teams) clear_scales_of_row(a, row);
    }
  }
  if (abort_flag) {
    if (threadIdx.x == 0 && team == 0) atomicExch(a.status, 1);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
  }
}

// Rows of any width, which do not stay in registers: a block goes over its row three times.
template <typename T>
__global__ void __launch_bounds__(512) layer_norm_forward_wide_kernel(const ForwardArgs a) {
  __shared__ float buf[64];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + a.x_rows.offset(row);
  float sum = 0.0f;
  for (int64_t k = threadIdx.x; k < a.cols; k += blockDim.x) sum += to_float(x[k]);
  const float mean = row_sum<0>(sum, buf) / static_cast<float>(a.cols);
  float square = 0.0f;
  for (int64_t k = threadIdx.x; k < a.cols; k += blockDim.x) {
    const float d = to_float(x[k]) - mean;
    square = fmaf(d, d, square);
  }
  const float rstd = inverse_root(row_sum<1>(square, buf) / static_cast<float>(a.cols) + a.eps);
  if (threadIdx.x == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  const int64_t group = row / a.rows_per_group;
  T* y = static_cast<T*>(a.y) + static_cast<int64_t>(row) * a.cols;
  for (int64_t k = threadIdx.x; k < a.cols; k += blockDim.x) {
    const float h = (to_float(x[k]) - mean) * rstd;
    y[k] = from_float<T>(fmaf(h, a.weight != nullptr ? a.offset + param<T>(a.weight, group * a.weight_stride + k, a.params_f32) : 1.0f,
                                  a.bias != nullptr ? param<T>(a.bias, group * a.bias_stride + k, a.params_f32) : 0.0f));
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
struct BackwardArgs {
  const void* dy;
  RowStrides dy_rows;
  const void* x;  // the input, or null: `codes` and `scales` stand for it
  RowStrides x_rows;
  const uint8_t* codes;
  const uint8_t* scales;
  const float* mean;
  const float* rstd;
  const void* weight;  // null: 1
  int64_t weight_stride;
  float offset;
  bool params_f32, params_aligned;
  void* dx;
  void* dweight;  // [groups, cols], null: not wanted
  void* dbias;
  float* partials;  // [groups * chunks][2][cols], where a group's rows are several blocks'
  uint32_t rows_per_group, groups, chunks, chunk_rows;
  int64_t cols;
  int* status;  // for waits that give up (ck_gemm_status)
};

// The input's vector v of `row` in fp32, from the type it was given in or from its copy.
template <typename T, int kVec>
struct InputVec {
  Raw<T, kVec> raw;
};
template <int kVec>
struct CopyVec {
  uint32_t words[kVec / 4 > 0 ? kVec / 4 : 1];
  uint32_t byte;
};

// A team of blockDim.x threads takes kRows rows at a time, every thread the same columns of all of them: a row's two sums go through
// shared memory once for all kRows, and the column sums for dw and db stay in registers until the block's rows are
// done.  Then the teams' sums are added in a fixed order and written: as results where the block has all rows of its group, else as
// partial sums that a second kernel adds.
template <typename T, int kVec, int kNum, int kRows, bool kCopy>
__global__ void __launch_bounds__(512) layer_norm_backward_kernel(const BackwardArgs a) {
  constexpr int kMaxWarps = 16;
  __shared__ __align__(16) float row_buf[2][kMaxWarps][2 * kRows];  // [turn][warp of the block][sums]
  extern __shared__ __align__(16) float shared_buf[];               // first the factors f, later the teams' column sums
  pdl_launch_dependents();
  const int team = threadIdx.y, teams = blockDim.y, width = blockDim.x, warps = width >> 5;
  const uint32_t group = blockIdx.x / a.chunks, chunk = blockIdx.x - group * a.chunks;
  const uint32_t begin = chunk * a.chunk_rows, end = min(a.rows_per_group, begin + a.chunk_rows);
  const int64_t vecs = a.cols / kVec;
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  pdl_wait();
  // The factors as fp32 in shared memory, all teams': in registers they would be a third of what a thread holds.  Four of a vector lie
  // together and the vectors 16 bytes apart, so that a warp's 16-byte loads meet no bank twice.
  constexpr int kPart = kVec < 4 ? kVec : 4;
  const int part_stride = static_cast<int>(vecs) * kPart;
  if (a.weight != nullptr) {
    for (int v = team * width + threadIdx.x; v < vecs; v += width * teams) {
      float f[kVec];
      load_param<T, kVec>(a.weight, group * a.weight_stride + static_cast<int64_t>(v) * kVec, a.params_f32, a.params_aligned, f);
#pragma unroll
      for (int j = 0; j < kVec; ++j) shared_buf[j / kPart * part_stride + v * kPart + j % kPart] = a.offset + f[j];
    }
    __syncthreads();
  }
  const auto factors = [&](int i, float(&f)[kVec]) {
    if (a.weight == nullptr) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) f[j] = 1.0f;
      return;
    }
    const int v = min(threadIdx.x + i * width, static_cast<int>(vecs) - 1);
#pragma unroll
    for (int q = 0; q < kVec / kPart; ++q) {
      const Raw<float, kPart> part = *reinterpret_cast<const Raw<float, kPart>*>(shared_buf + q * part_stride + v * kPart);
#pragma unroll
      for (int j = 0; j < kPart; ++j) f[q * kPart + j] = part.v[j];
    }
  };
  float dw[kNum][kVec], db[kNum][kVec];
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) dw[i][j] = db[i][j] = 0.0f;
  }
  int turn = 0;
  for (uint32_t r0 = begin + team * kRows; r0 < end; r0 += teams * kRows, turn ^= 1) {
    Raw<T, kVec> dy[kRows][kNum];
    std::conditional_t<kCopy, CopyVec<kVec>, InputVec<T, kVec>> in[kRows][kNum];
    float mean[kRows], rstd[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const bool live = r0 + r < end;
      const uint32_t row = group * a.rows_per_group + (live ? r0 + r : begin);
      const T* dy_row = static_cast<const T*>(a.dy) + a.dy_rows.offset(row);
      const T* x_row = kCopy ? nullptr : static_cast<const T*>(a.x) + a.x_rows.offset(row);
#pragma unroll
      for (int i = 0; i < kNum; ++i) {
        const int64_t v = threadIdx.x + i * width;
        const bool inside = live && v < vecs;
        dy[r][i] = inside ? load_once<T, kVec>(dy_row + v * kVec) : zeros<T, kVec>();
        if constexpr (kCopy) {
          in[r][i].byte = inside ? a.scales[swizzled_scale_offset(row, v * kVec >> 5, ceil_div(a.cols >> 5, 4))] : 0u;
#pragma unroll
          for (int j = 0; j < kVec / 4; ++j) {
            in[r][i].words[j] = inside ? reinterpret_cast<const uint32_t*>(a.codes + static_cast<int64_t>(row) * a.cols + v * kVec)[j] : 0u;
          }
        } else {
          in[r][i].raw = inside ? load_once<T, kVec>(x_row + v * kVec) : zeros<T, kVec>();
        }
      }
      rstd[r] = live ? a.rstd[row] : 0.0f;
      mean[r] = live ? a.mean[row] : 0.0f;
    }
    const auto values = [&](int r, int i, float(&h)[kVec]) {
      if constexpr (kCopy) {
        const float s = e8m0_factor(in[r][i].byte);
#pragma unroll
        for (int j = 0; j < kVec / 4; ++j) e4m3_four(in[r][i].words[j], s, h + 4 * j);
      } else {
        unpack(in[r][i].raw, h);
      }
#pragma unroll
      for (int j = 0; j < kVec; ++j) h[j] = (h[j] - mean[r]) * rstd[r];
    };
    float sums[2 * kRows];  // of g and of g h, row after row
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
      for (int i = 0; i < kNum; ++i) {
        float h[kVec], d[kVec], f[kVec];
        values(r, i, h);
        unpack(dy[r][i], d);
        factors(i, f);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float g = d[j] * f[j];
          s1 += g;
          s2 = fmaf(g, h[j], s2);
          dw[i][j] = fmaf(d[j], h[j], dw[i][j]);
          db[i][j] += d[j];
        }
      }
      sums[2 * r] = warp_sum(s1);
      sums[2 * r + 1] = warp_sum(s2);
    }
    if (warps > 1) {  // the team's warps meet; two buffers in turn, so that one meeting a round is enough
      const int warp0 = team * warps;
      if ((threadIdx.x & 31) == 0) {
#pragma unroll
        for (int s = 0; s < 2 * kRows; ++s) row_buf[turn][warp0 + (threadIdx.x >> 5)][s] = sums[s];
      }
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(width) : "memory");
#pragma unroll
      for (int s = 0; s < 2 * kRows; ++s) sums[s] = 0.0f;
      for (int w = 0; w < warps; ++w) {
#pragma unroll
        for (int s = 0; s < 2 * kRows; ++s) sums[s] += row_buf[turn][warp0 + w][s];
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r0 + r >= end) break;
      const float c1 = sums[2 * r] * inv_cols, c2 = sums[2 * r + 1] * inv_cols;
      T* dx = static_cast<T*>(a.dx) + (static_cast<int64_t>(group) * a.rows_per_group + r0 + r) * a.cols;
#pragma unroll
      for (int i = 0; i < kNum; ++i) {
        const int64_t v = threadIdx.x + i * width;
        if (v < vecs) {
          float h[kVec], d[kVec], f[kVec];
          values(r, i, h);
          unpack(dy[r][i], d);
          factors(i, f);
#pragma unroll
          for (int j = 0; j < kVec; ++j) d[j] = (fmaf(d[j], f[j], -c1) - h[j] * c2) * rstd[r];
          store(dx + v * kVec, pack<T, kVec>(d));
        }
      }
    }
  }
  if (a.dweight == nullptr && a.dbias == nullptr) return;
  // the teams' column sums
  float* column_buf = shared_buf;  // [2 * kVec][threads]
  const int threads = width * teams, at = team * width + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      column_buf[j * threads + at] = dw[i][j];
      column_buf[(kVec + j) * threads + at] = db[i][j];
    }
    __syncthreads();
    const int64_t v = threadIdx.x + i * width;
    if (v >= vecs) continue;
    for (int j = team; j < 2 * kVec; j += teams) {
      float s = 0.0f;
      for (int t = 0; t < teams; ++t) s += column_buf[j * threads + t * width + threadIdx.x];
      const int64_t k = v * kVec + j % kVec;
      if (a.partials != nullptr) {
        a.partials[(static_cast<int64_t>(blockIdx.x) * 2 + j / kVec) * a.cols + k] = s;
      } else {
        void* to = j < kVec ? a.dweight : a.dbias;
        if (to != nullptr) store_param<T>(to, group * a.cols + k, a.params_f32, s);
      }
    }
  }
}

// The same where rows are long enough to come through shared memory (see the forward pass): a team's rows of dy and of x or its codes are
// bulk copies into its own ring, a few rows ahead, and what a thread holds of a row is read from there once.
template <typename T, int kVec, int kNum, bool kCopy>
__global__ void __launch_bounds__(512) layer_norm_backward_ring_kernel(const BackwardArgs a, const int stages) {
  constexpr int kMaxTeams = 15, kPairs = kVec / 2;
  extern __shared__ __align__(128) uint8_t shared_bytes[];  // factors f, then the teams' rings; the teams' column sums in the end
  __shared__ __align__(8) uint64_t full[kMaxTeams][kMaxRing];
  __shared__ float2 row_buf[2][16];  // [turn][warp of the block]
  __shared__ int abort_flag;
  pdl_launch_dependents();
  const int team = threadIdx.y, teams = blockDim.y, width = blockDim.x, warps = width >> 5, lane = threadIdx.x & 31;
  const uint32_t group = blockIdx.x / a.chunks, chunk = blockIdx.x - group * a.chunks;
  const uint32_t begin = chunk * a.chunk_rows, end = min(a.rows_per_group, begin + a.chunk_rows), row0 = group * a.rows_per_group;
  const int vecs = static_cast<int>(a.cols / kVec);
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const uint32_t dy_bytes = static_cast<uint32_t>(a.cols) * sizeof(T), x_bytes = static_cast<uint32_t>(a.cols) * (kCopy ? 1 : sizeof(T));
  const uint32_t x_at = (dy_bytes + 127) & ~127u, stage_bytes = x_at + ((x_bytes + 127) & ~127u);
  const uint32_t factor_bytes = a.weight != nullptr ? (static_cast<uint32_t>(a.cols) * 4 + 127) & ~127u : 0u;
  float* const shared_buf = reinterpret_cast<float*>(shared_bytes);
  uint8_t* const ring = shared_bytes + factor_bytes + team * stages * stage_bytes;
  const uint32_t ring_at = sm100::smem_u32(ring), full_at = sm100::smem_u32(full[team]);
  const auto load_row = [&](uint32_t r, int s) {  // by one thread of the team
    const uint32_t row = row0 + r, to = ring_at + s * stage_bytes, bar = full_at + s * 8;
    sm100::mbar_arrive_expect_tx(bar, dy_bytes + x_bytes);
    sm100::bulk_load_1d(to, static_cast<const T*>(a.dy) + a.dy_rows.offset(row), dy_bytes, bar);
    const void* x = kCopy ? static_cast<const void*>(a.codes + static_cast<int64_t>(row) * a.cols)
                          : static_cast<const void*>(static_cast<const T*>(a.x) + a.x_rows.offset(row));
    sm100::bulk_load_1d(to + x_at, x, x_bytes, bar);
  };
  if (threadIdx.x == 0) {
    if (team == 0) abort_flag = 0;
    for (int s = 0; s < stages; ++s) sm100::mbar_init(&full[team][s], 1);
    sm100::fence_barrier_init();
    pdl_wait();
    for (int s = 0; s < stages; ++s) {
      const uint32_t r = begin + team + s * teams;
      if (r < end) load_row(r, s);
    }
  }
  pdl_wait();
  // factors in shared memory, as above
  constexpr int kPart = 4;
  const int part_stride = vecs * kPart;
  if (a.weight != nullptr) {
    for (int v = team * width + threadIdx.x; v < vecs; v += width * teams) {
      float f[kVec];
      load_param<T, kVec>(a.weight, group * a.weight_stride + static_cast<int64_t>(v) * kVec, a.params_f32, a.params_aligned, f);
#pragma unroll
      for (int j = 0; j < kVec; ++j) shared_buf[j / kPart * part_stride + v * kPart + j % kPart] = a.offset + f[j];
    }
  }
  __syncthreads();
  const auto factors = [&](int i, float2(&f)[kPairs]) {
    if (a.weight == nullptr) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) f[j] = both(1.0f);
      return;
    }
    const int v = min(static_cast<int>(threadIdx.x) + i * width, vecs - 1);
#pragma unroll
    for (int q = 0; q < kVec / kPart; ++q) {
      const float4 part = *reinterpret_cast<const float4*>(shared_buf + q * part_stride + v * kPart);
      f[2 * q] = make_float2(part.x, part.y);
      f[2 * q + 1] = make_float2(part.z, part.w);
    }
  };
  float2 dw[kNum][kPairs], db[kNum][kPairs];
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j) dw[i][j] = db[i][j] = both(0.0f);
  }
  // what comes beside a row, read a row ahead
  float next_mean = 0.0f, next_rstd = 0.0f;
  uint32_t next_byte[kNum] = {};
  const int64_t quads = ceil_div(a.cols >> 5, 4);
  const auto beside = [&](uint32_t r) {
    if (r >= end) return;
    next_mean = a.mean[row0 + r];
    next_rstd = a.rstd[row0 + r];
    if constexpr (kCopy) {
#pragma unroll
      for (int i = 0; i < kNum; ++i) {
        const int v = threadIdx.x + i * width;
        if (v < vecs) next_byte[i] = a.scales[swizzled_scale_offset(row0 + r, v * kVec >> 5, quads)];
      }
    }
  };
  beside(begin + team);
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  for (uint32_t r = begin + team; r < end; r += teams, turn ^= 1) {
    const float mean = next_mean, rstd = next_rstd;
    float factor[kNum];
#pragma unroll
    for (int i = 0; i < kNum; ++i) factor[i] = e8m0_factor(next_byte[i]);
    beside(r + teams);
    if (!sm100::mbar_wait(full_at + stage * 8, phase, &abort_flag)) break;
    const uint8_t* const from = ring + stage * stage_bytes;
    // unpacked once: dy and h stay in registers for both passes
    float2 d[kNum][kPairs], h[kNum][kPairs];
    const float2 rstd2 = both(rstd), shift = both(sizeof(T) == 2 ? -mean * rstd : -mean);
    float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const int v = min(static_cast<int>(threadIdx.x) + i * width, vecs - 1);
      Raw<T, kVec> raw = *reinterpret_cast<const Raw<T, kVec>*>(from + v * 16);
      if (static_cast<int>(threadIdx.x) + i * width >= vecs) raw = zeros<T, kVec>();  // past the row's end: dy = 0, whatever h
      unpack(raw, d[i]);
      if constexpr (kCopy) {
        const auto codes = *reinterpret_cast<const Raw<uint32_t, kVec / 4>*>(from + x_at + v * kVec);
#pragma unroll
        for (int j = 0; j < kVec / 4; ++j) {
          h[i][2 * j] = mul_x2(e4m3_pair(codes.v[j] & 0xFFFFu), both(factor[i]));
          h[i][2 * j + 1] = mul_x2(e4m3_pair(codes.v[j] >> 16), both(factor[i]));
        }
      } else {
        unpack(*reinterpret_cast<const Raw<T, kVec>*>(from + x_at + v * 16), h[i]);
      }
      float2 f[kPairs];
      factors(i, f);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        // (x - mean) / std; in one step for 16-bit types, where a mean of that many times the deviation leaves no digits in x anyway
        h[i][j] = sizeof(T) == 2 ? fma_x2(h[i][j], rstd2, shift) : mul_x2(add_x2(h[i][j], shift), rstd2);
        const float2 g = mul_x2(d[i][j], f[j]);
        s1 = add_x2(s1, g);
        s2 = fma_x2(g, h[i][j], s2);
        dw[i][j] = fma_x2(d[i][j], h[i][j], dw[i][j]);
        db[i][j] = add_x2(db[i][j], d[i][j]);
      }
    }
    // both sums in five exchanges: the lower half of a warp goes on with one, the upper with the other
    float sum = (lane < 16 ? s1.x + s1.y : s2.x + s2.y) + __shfl_xor_sync(0xFFFFFFFFu, lane < 16 ? s2.x + s2.y : s1.x + s1.y, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    float c1, c2;
    if (warps > 1) {  // the team's warps meet; two buffers in turn, so that one meeting a row is enough
      float2* const slots = row_buf[turn] + team * warps;
      if ((lane & 15) == 0) reinterpret_cast<float*>(slots + (threadIdx.x >> 5))[lane >> 4] = sum;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(width) : "memory");
      float2 all = both(0.0f);
      for (int w = 0; w < warps; ++w) all = add_x2(all, slots[w]);
      c1 = all.x * inv_cols;
      c2 = all.y * inv_cols;
    } else {
      c1 = __shfl_sync(0xFFFFFFFFu, sum, 0) * inv_cols;
      c2 = __shfl_sync(0xFFFFFFFFu, sum, 16) * inv_cols;
    }
    if (threadIdx.x == 0 && r + stages * teams < end) load_row(r + stages * teams, stage);  // all have read the stage
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
    T* const dx = static_cast<T*>(a.dx) + static_cast<int64_t>(row0 + r) * a.cols;
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const int v = threadIdx.x + i * width;
      if (v < vecs) {
        float2 f[kPairs];
        factors(i, f);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          d[i][j] = mul_x2(fma_x2(h[i][j], both(-c2), fma_x2(d[i][j], f[j], both(-c1))), rstd2);
        }
        store(dx + v * kVec, pack<T, kVec>(d[i]));
      }
    }
  }
  __syncthreads();  // the ring is the column sums' now
  if (abort_flag) {
    if (threadIdx.x == 0 && team == 0) atomicExch(a.status, 1);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
    return;
  }
  if (a.dweight == nullptr && a.dbias == nullptr) return;
  const int threads = width * teams, at = team * width + threadIdx.x;
  const auto put = [&](int j, int v, float s) {  // sum j (of kVec for dw, then of kVec for db) of vector v
    const int64_t k = static_cast<int64_t>(v) * kVec + j % kVec;
    if (a.partials != nullptr) {
      a.partials[(static_cast<int64_t>(blockIdx.x) * 2 + j / kVec) * a.cols + k] = s;
    } else {
      void* const to = j < kVec ? a.dweight : a.dbias;
      if (to != nullptr) store_param<T>(to, group * a.cols + k, a.params_f32, s);
    }
  };
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
    const int v = threadIdx.x + i * width;
    if (teams == 1) {
      if (v < vecs) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          put(j, v, j % 2 == 0 ? dw[i][j / 2].x : dw[i][j / 2].y);
          put(kVec + j, v, j % 2 == 0 ? db[i][j / 2].x : db[i][j / 2].y);
        }
      }
      continue;
    }
    if (i > 0) __syncthreads();
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      shared_buf[(2 * j) * threads + at] = dw[i][j].x;
      shared_buf[(2 * j + 1) * threads + at] = dw[i][j].y;
      shared_buf[(kVec + 2 * j) * threads + at] = db[i][j].x;
      shared_buf[(kVec + 2 * j + 1) * threads + at] = db[i][j].y;
    }
    __syncthreads();
    if (v < vecs) {
      for (int j = team; j < 2 * kVec; j += teams) {
        float s = 0.0f;
        for (int t = 0; t < teams; ++t) s += shared_buf[j * threads + t * width + threadIdx.x];
        put(j, v, s);
      }
    }
  }
}

// Rows of any width: dx by blocks that go over their row twice, then the column sums by blocks of 32 columns.
template <typename T>
__device__ __forceinline__ float normalized(const BackwardArgs& a, uint32_t row, int64_t k) {
  float v;
  if (a.x != nullptr) {
    v = to_float(static_cast<const T*>(a.x)[a.x_rows.offset(row) + k]);
  } else {
    v = e4m3_pair(a.codes[static_cast<int64_t>(row) * a.cols + k]).x *
        e8m0_factor(a.scales[swizzled_scale_offset(row, k >> 5, ceil_div(a.cols >> 5, 4))]);
  }
  return (v - a.mean[row]) * a.rstd[row];
}

template <typename T>
__global__ void __launch_bounds__(512) layer_norm_backward_wide_kernel(const BackwardArgs a) {
  __shared__ float buf[64];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t row = blockIdx.x, group = row / a.rows_per_group;
  const T* dy = static_cast<const T*>(a.dy) + a.dy_rows.offset(row);
  const int64_t w0 = group * a.weight_stride;
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t k = threadIdx.x; k < a.cols; k += blockDim.x) {
    const float g = to_float(dy[k]) * (a.weight != nullptr ? a.offset + param<T>(a.weight, w0 + k, a.params_f32) : 1.0f);
    s1 += g;
    s2 = fmaf(g, normalized<T>(a, row, k), s2);
  }
  const float c1 = row_sum<0>(s1, buf) / static_cast<float>(a.cols), c2 = row_sum<1>(s2, buf) / static_cast<float>(a.cols);
  const float rstd = a.rstd[row];
  T* dx = static_cast<T*>(a.dx) + static_cast<int64_t>(row) * a.cols;
  for (int64_t k = threadIdx.x; k < a.cols; k += blockDim.x) {
    const float g = to_float(dy[k]) * (a.weight != nullptr ? a.offset + param<T>(a.weight, w0 + k, a.params_f32) : 1.0f);
    dx[k] = from_float<T>((g - c1 - normalized<T>(a, row, k) * c2) * rstd);
  }
}

template <typename T>
__global__ void __launch_bounds__(512) layer_norm_columns_wide_kernel(const BackwardArgs a) {
  __shared__ float buf[2][16][33];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t group = blockIdx.x / a.chunks, chunk = blockIdx.x - group * a.chunks;
  const uint32_t begin = chunk * a.chunk_rows, end = min(a.rows_per_group, begin + a.chunk_rows);
  const int64_t k = static_cast<int64_t>(blockIdx.y) * 32 + threadIdx.x;
  float dw = 0.0f, db = 0.0f;
  if (k < a.cols) {
    for (uint32_t r = begin + threadIdx.y; r < end; r += 16) {
      const uint32_t row = group * a.rows_per_group + r;
      const float d = to_float(static_cast<const T*>(a.dy)[a.dy_rows.offset(row) + k]);
      dw = fmaf(d, normalized<T>(a, row, k), dw);
      db += d;
    }
  }
  buf[0][threadIdx.y][threadIdx.x] = dw;
  buf[1][threadIdx.y][threadIdx.x] = db;
  __syncthreads();
  if (threadIdx.y < 2 && k < a.cols) {
    float s = 0.0f;
#pragma unroll
    for (int t = 0; t < 16; ++t) s += buf[threadIdx.y][t][threadIdx.x];
    if (a.partials != nullptr) {
      a.partials[(static_cast<int64_t>(blockIdx.x) * 2 + threadIdx.y) * a.cols + k] = s;
    } else {
      void* to = threadIdx.y == 0 ? a.dweight : a.dbias;
      if (to != nullptr) store_param<T>(to, group * a.cols + k, a.params_f32, s);
    }
  }
}

// The chunks' partial sums of a group, added in their order: 32 columns a block, the chunks over its warps.
template <typename T>
__global__ void __launch_bounds__(512) layer_norm_join_kernel(const float* partials, uint32_t chunks, int64_t cols, void* dweight, void* dbias, bool f32) {
  __shared__ float buf[16][33];
  pdl_launch_dependents();
  const uint32_t group = blockIdx.y >> 1, which = blockIdx.y & 1;
  void* to = which == 0 ? dweight : dbias;
  if (to == nullptr) return;
  const int64_t k = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
  pdl_wait();
  float s = 0.0f;
  if (k < cols) {
#pragma unroll 8
    for (uint32_t c = threadIdx.y; c < chunks; c += 16) s += partials[((static_cast<int64_t>(group) * chunks + c) * 2 + which) * cols + k];
  }
  buf[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && k < cols) {
    s = 0.0f;
#pragma unroll
    for (int t = 0; t < 16; ++t) s += buf[t][threadIdx.x];
    store_param<T>(to, group * cols + k, f32, s);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <typename T>
constexpr int kVecOf = 16 / static_cast<int>(sizeof(T));

bool on_vectors(const void* p, int64_t elements, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && elements * size % 16 == 0;
}
bool on_vectors(const void* p, const RowStrides& r, int size) {
  return on_vectors(p, r.outer_stride, size) && r.inner_stride * size % 16 == 0;
}

template <typename T, int kVec, int kNum, bool kCopy>
int launch_forward_num(const ForwardArgs& a, int warps, cudaStream_t s) {
  const int threads = warps * 32, rows_of_block = warps >= 8 ? 1 : 8 / warps;
  const dim3 grid(static_cast<unsigned>(ceil_div(kCopy ? a.rows_padded : a.rows, rows_of_block))), block(threads, rows_of_block);
  auto kernel = warps <= 8 ? layer_norm_forward_kernel<T, kVec, kNum, kCopy, 256> : layer_norm_forward_kernel<T, kVec, kNum, kCopy, 1024>;
  CK_CUDA(launch_pdl(kernel, grid, block, 0, s, a));
  return CK_OK;
}

template <typename T, int kVec, int kNum, bool kCopy>
int launch_forward_ring_num(ForwardArgs a, int warps, cudaStream_t s) {
  constexpr int64_t kRoom = 216 * 1024;
  const int64_t stage = round_up(a.cols * static_cast<int64_t>(sizeof(T)), 128), param = round_up(a.cols * 4, 128);
  int64_t params = (a.weight != nullptr ? param : 0) + (a.bias != nullptr ? param : 0);
  const bool shared_params = params + 2 * stage <= kRoom;
  if (!shared_params) params = 0;
  int64_t teams = 32 / warps;
  if (warps > 1 && teams > 15) teams = 15;  // named barriers 1 to 15
  while (teams > 1 && params + 2 * teams * stage > kRoom) --teams;
  int64_t stages = (kRoom - params) / (teams * stage);
  if (stages > kMaxRing) stages = kMaxRing;
  // one block an SM, and no block with less than a row for each team
  const int64_t groups = a.rows / a.rows_per_group;
  int64_t chunks = sm_count() / groups;
  if (chunks > ceil_div(a.rows_per_group, teams)) chunks = ceil_div(a.rows_per_group, teams);
  if (chunks < 1) chunks = 1;
  const uint32_t chunk_rows = static_cast<uint32_t>(ceil_div(a.rows_per_group, chunks));
  chunks = ceil_div(a.rows_per_group, chunk_rows);
  const int smem = static_cast<int>(params + teams * stages * stage);
  auto kernel = layer_norm_forward_ring_kernel<T, kVec, kNum, kCopy>;
  CK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (int rc = gemm_status_word(&a.status)) return rc;
  CK_CUDA(launch_pdl(kernel, dim3(static_cast<unsigned>(groups * chunks)), dim3(32 * warps, static_cast<unsigned>(teams)), smem, s, a,
                     static_cast<uint32_t>(chunks), chunk_rows, static_cast<int>(stages), shared_params));
  return CK_OK;
}

// 24 elements a thread
template <typename T, int kVec, bool kCopy>
int launch_forward_ring(const ForwardArgs& a, cudaStream_t s) {
  constexpr int kUnit = 8 / kVec;
  const int64_t vecs = a.cols / kVec;
  const int warps = static_cast<int>(ceil_div(vecs, 32 * 3 * kUnit));
  const int64_t num = ceil_div(vecs, 32 * warps * kUnit);
  if (num == 1) return launch_forward_ring_num<T, kVec, kUnit, kCopy>(a, warps, s);
  if (num == 2) return launch_forward_ring_num<T, kVec, 2 * kUnit, kCopy>(a, warps, s);
  return launch_forward_ring_num<T, kVec, 3 * kUnit, kCopy>(a, warps, s);
}

// Warps of a row: as few as hold it, eight vectors a lane (no barrier crosses a warp then, and a lane has its loads in flight
// together); where the rows alone do not fill the chip, as many as leave one vector a lane, up to 32.
template <typename T, int kVec, bool kCopy>
int launch_forward(const ForwardArgs& a, cudaStream_t s) {
  const int64_t vecs = ceil_div(a.cols, kVec);
  if (vecs > 32 * 32 * 8) return fail(CK_ERR_UNSUPPORTED, "layer_norm_forward: a copy of rows of %lld is not supported", (long long)a.cols);
  if constexpr (kVec > 1) {
    if (a.cols <= 32 * 32 * 24 && a.rows > 2 * sm_count() && a.rows_per_group >= 16) return launch_forward_ring<T, kVec, kCopy>(a, s);
  }
  int warps = static_cast<int>(ceil_div(vecs, 32 * 8));
  while (warps < 32 && static_cast<int64_t>(warps) * 32 < vecs && static_cast<int64_t>(a.rows) * warps < 8 * sm_count()) ++warps;
  const int num = static_cast<int>(ceil_div(vecs, 32 * warps));
  if (num == 1) return launch_forward_num<T, kVec, 1, kCopy>(a, warps, s);
  if (num == 2) return launch_forward_num<T, kVec, 2, kCopy>(a, warps, s);
  if (num <= 4) return launch_forward_num<T, kVec, 4, kCopy>(a, warps, s);
  if (num <= 6) return launch_forward_num<T, kVec, 6, kCopy>(a, warps, s);
  return launch_forward_num<T, kVec, 8, kCopy>(a, warps, s);
}

template <typename T>
int forward_typed(const ForwardArgs& given, cudaStream_t s) {
  ForwardArgs a = given;
  constexpr int kVec = kVecOf<T>;
  const int param_size = a.params_f32 ? 4 : sizeof(T);
  a.params_aligned = (a.weight == nullptr || on_vectors(a.weight, a.weight_stride, param_size)) &&
                     (a.bias == nullptr || on_vectors(a.bias, a.bias_stride, param_size));
  const bool vectors = a.cols % kVec == 0 && on_vectors(a.x, a.x_rows, sizeof(T)) && reinterpret_cast<uintptr_t>(a.y) % 16 == 0;
  if (a.codes != nullptr) {
    CK_REQUIRE(vectors, "layer_norm_forward: rows with a copy have to start on 16-byte boundaries");
    return launch_forward<T, kVec, true>(a, s);
  }
  if (vectors && a.cols <= int64_t{32} * 32 * 8 * kVec) return launch_forward<T, kVec, false>(a, s);
  if (a.cols <= 32 * 32 * 8) return launch_forward<T, 1, false>(a, s);
  CK_CUDA(launch_pdl(layer_norm_forward_wide_kernel<T>, dim3(a.rows), dim3(512), 0, s, a));
  return CK_OK;
}

// ---- backward: how the rows are shared out
struct Plan {
  bool wide;      // rows that a block's threads do not hold
  bool ring;      // rows that come through shared memory
  int num;        // vectors of a thread
  int warps;      // of a team
  int teams;      // of a block
  int rows;       // that a team takes at a time
  int stages;     // of a team's ring
  int smem;       // bytes
  uint32_t chunks, chunk_rows;  // blocks of a group, rows of each
};

// size: of an element; weight: whether there is one.
Plan plan_backward(int64_t cols, int size, int vec, bool copy, bool weight, int64_t groups, int64_t rows_per_group) {
  Plan p = {};
  const int64_t vecs = ceil_div(cols, vec);
  const int unit = vec == 4 ? 2 : 1;  // 24 elements a thread, or up to 32 (one by one: 4, up to 8)
  p.wide = vecs > 512 * (vec == 1 ? 8 : vec == 4 ? 6 : 4);
  p.ring = vec > 1 && vecs >= 64 && !p.wide;
  int64_t step = 64;
  if (!p.wide) {
    p.warps = static_cast<int>(ceil_div(vecs, 32 * (vec == 1 ? 4 : 3 * unit)));
    if (p.warps > 16) p.warps = 16;
    p.num = static_cast<int>(ceil_div(vecs, 32 * p.warps * unit)) * unit;
    p.teams = 16 / p.warps;
    if (p.teams > 15) p.teams = 15;  // named barriers 1 to 15
    p.rows = !p.ring && p.num <= 2 ? 2 : 1;
    step = static_cast<int64_t>(p.teams) * p.rows;
    const int64_t sums = 2 * vec * 32 * p.warps * p.teams * 4, factors = weight ? round_up(cols * 4, 128) : 0;
    if (p.ring) {
      const int64_t stage = round_up(cols * size, 128) + round_up(cols * (copy ? 1 : size), 128);
      int64_t stages = (208 * 1024 - factors) / (p.teams * stage);
      p.stages = static_cast<int>(stages > kMaxRing ? kMaxRing : stages);
      p.wide = p.stages < 2;
      p.smem = static_cast<int>(factors + p.teams * p.stages * stage);
      if (sums > p.smem) p.smem = static_cast<int>(sums);
    } else {
      p.smem = static_cast<int>(sums > factors ? sums : factors);
    }
  }
  // one block an SM, and no block with less than one round of its teams
  int64_t chunks = sm_count() / groups;
  if (chunks > ceil_div(rows_per_group, step)) chunks = ceil_div(rows_per_group, step);
  if (chunks < 1) chunks = 1;
  p.chunk_rows = static_cast<uint32_t>(ceil_div(rows_per_group, chunks));
  p.chunks = static_cast<uint32_t>(ceil_div(rows_per_group, p.chunk_rows));
  return p;
}

template <typename T, int kVec, int kNum, int kRows, bool kCopy>
int launch_backward_num(const BackwardArgs& a, const Plan& p, cudaStream_t s) {
  auto kernel = layer_norm_backward_kernel<T, kVec, kNum, kRows, kCopy>;
  if (p.smem > 32 * 1024) CK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem));
  CK_CUDA(launch_pdl(kernel, dim3(a.groups * a.chunks), dim3(32 * p.warps, p.teams), p.smem, s, a));
  return CK_OK;
}

template <typename T, int kVec, int kNum, bool kCopy>
int launch_backward_ring(BackwardArgs a, const Plan& p, cudaStream_t s) {
  if (int rc = gemm_status_word(&a.status)) return rc;
  auto kernel = layer_norm_backward_ring_kernel<T, kVec, kNum, kCopy>;
  if (p.smem > 32 * 1024) CK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, p.smem));
  CK_CUDA(launch_pdl(kernel, dim3(a.groups * a.chunks), dim3(32 * p.warps, p.teams), p.smem, s, a, p.stages));
  return CK_OK;
}

template <typename T, int kVec, bool kCopy>
int launch_backward(const BackwardArgs& a, const Plan& p, cudaStream_t s) {
  if constexpr (kVec == 1) {
    switch (p.num) {
      case 1: return launch_backward_num<T, 1, 1, 2, false>(a, p, s);
      case 2: return launch_backward_num<T, 1, 2, 2, false>(a, p, s);
      case 3: case 4: return launch_backward_num<T, 1, 4, 1, false>(a, p, s);
      default: return launch_backward_num<T, 1, 8, 1, false>(a, p, s);
    }
  } else if (p.ring) {
    if constexpr (kVec == 4) {
      switch (p.num) {
        case 2: return launch_backward_ring<T, 4, 2, kCopy>(a, p, s);
        case 4: return launch_backward_ring<T, 4, 4, kCopy>(a, p, s);
        default: return launch_backward_ring<T, 4, 6, kCopy>(a, p, s);
      }
    } else {
      switch (p.num) {
        case 1: case 2: return launch_backward_ring<T, 8, 2, kCopy>(a, p, s);
        case 3: return launch_backward_ring<T, 8, 3, kCopy>(a, p, s);
        default: return launch_backward_ring<T, 8, 4, kCopy>(a, p, s);
      }
    }
  } else {  // fewer than 64 vectors
    return p.num == 1 ? launch_backward_num<T, kVec, 1, 2, kCopy>(a, p, s) : launch_backward_num<T, kVec, 2, 2, kCopy>(a, p, s);
  }
}

int backward_vec(const BackwardArgs& a, int dtype) {
  const int size = dtype == CK_DTYPE_F32 ? 4 : 2, vec = 16 / size;
  const bool vectors = a.cols % vec == 0 && on_vectors(a.dy, a.dy_rows, size) && reinterpret_cast<uintptr_t>(a.dx) % 16 == 0 &&
                       (a.x != nullptr ? on_vectors(a.x, a.x_rows, size) : reinterpret_cast<uintptr_t>(a.codes) % 16 == 0);
  return vectors ? vec : 1;
}

template <typename T>
int backward_typed(const BackwardArgs& given, int dtype, void* workspace, int64_t workspace_bytes, cudaStream_t s) {
  BackwardArgs a = given;
  a.params_aligned = a.weight == nullptr || on_vectors(a.weight, a.weight_stride, a.params_f32 ? 4 : sizeof(T));
  const int vec = backward_vec(a, dtype);
  Plan p = plan_backward(a.cols, sizeof(T), vec, a.x == nullptr, a.weight != nullptr, a.groups, a.rows_per_group);
  p.wide = p.wide || (vec == 1 && a.x == nullptr);
  a.chunks = p.chunks;
  a.chunk_rows = p.chunk_rows;
  const bool sums = a.dweight != nullptr || a.dbias != nullptr;
  const int64_t need = static_cast<int64_t>(a.groups) * p.chunks * 2 * a.cols * 4;
  if (sums && p.chunks > 1) {
    CK_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 4 == 0,
               "layer_norm_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    a.partials = static_cast<float*>(workspace);
  }
  constexpr int kVec = kVecOf<T>;
  int rc = CK_OK;
  if (p.wide) {
    CK_CUDA(launch_pdl(layer_norm_backward_wide_kernel<T>, dim3(a.groups * a.rows_per_group), dim3(512), 0, s, a));
    if (sums) {
      const dim3 grid(a.groups * p.chunks, static_cast<unsigned>(ceil_div(a.cols, 32)));
      CK_CUDA(launch_pdl(layer_norm_columns_wide_kernel<T>, grid, dim3(32, 16), 0, s, a));
    }
  } else if (vec == 1) {
    rc = launch_backward<T, 1, false>(a, p, s);
  } else if (a.x != nullptr) {
    rc = launch_backward<T, kVec, false>(a, p, s);
  } else {
    rc = launch_backward<T, kVec, true>(a, p, s);
  }
  if (rc != CK_OK) return rc;
  if (a.partials != nullptr) {
    const dim3 grid(static_cast<unsigned>(ceil_div(a.cols, 32)), 2 * a.groups);
    CK_CUDA(launch_pdl(layer_norm_join_kernel<T>, grid, dim3(32, 16), 0, s, static_cast<const float*>(a.partials), a.chunks, a.cols,
                       a.dweight, a.dbias, a.params_f32));
  }
  return CK_OK;
}

bool is_float_code(int dtype) { return dtype == CK_DTYPE_F32 || dtype == CK_DTYPE_F16 || dtype == CK_DTYPE_BF16; }

int check_shapes(const char* op, int dtype, int param_dtype, int64_t rows, int64_t inner, int64_t cols, int64_t groups) {
  CK_REQUIRE(is_float_code(dtype), "%s: unsupported dtype code %d", op, dtype);
  CK_REQUIRE(param_dtype == dtype || param_dtype == CK_DTYPE_F32, "%s: parameters are fp32 or of the input's type, got dtype code %d", op, param_dtype);
  CK_REQUIRE(rows > 0 && cols > 0 && inner > 0 && groups > 0, "%s: empty input [%lld, %lld]", op, (long long)rows, (long long)cols);
  CK_REQUIRE(rows <= 0x7FFFFF00 && cols <= 0x7FFFFFFF && inner <= rows, "%s: input too large [%lld, %lld]", op, (long long)rows, (long long)cols);
  CK_REQUIRE(rows % groups == 0, "%s: %lld rows do not form %lld groups", op, (long long)rows, (long long)groups);
  CK_REQUIRE(groups <= 32767, "%s: %lld groups, at most 32767", op, (long long)groups);
  return CK_OK;
}

}  // namespace
}  // namespace ck

extern "C" int ck_layer_norm_forward(const void* x, int dtype, int64_t rows, int64_t cols, int64_t inner, int64_t x_outer_stride,
                                     int64_t x_inner_stride, const void* weight, const void* bias, int param_dtype, int64_t groups,
                                     int64_t weight_stride, int64_t bias_stride, float weight_offset, float eps, void* y, float* mean, float* rstd,
                                     void* codes, void* block_scales, void* stream) {
  using namespace ck;
  if (int rc = check_shapes("layer_norm_forward", dtype, param_dtype, rows, inner, cols, groups)) return rc;
  CK_REQUIRE(x && y, "layer_norm_forward: null pointer");
  CK_REQUIRE((mean == nullptr) == (rstd == nullptr), "layer_norm_forward: mean and rstd go together");
  CK_REQUIRE((codes == nullptr) == (block_scales == nullptr), "layer_norm_forward: codes and block_scales go together");
  if (codes != nullptr) {
    CK_REQUIRE(cols % 32 == 0, "layer_norm_forward: a copy needs rows of a multiple of 32, got %lld", (long long)cols);
    CK_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 8 == 0 && reinterpret_cast<uintptr_t>(block_scales) % 4 == 0,
               "layer_norm_forward: codes and block_scales have to be aligned to 8 and 4 bytes");
  }
  ForwardArgs a = {};
  a.x = x;
  a.x_rows = {x_outer_stride, x_inner_stride, static_cast<uint32_t>(inner)};
  a.weight = weight;
  a.bias = bias;
  a.weight_stride = weight_stride;
  a.bias_stride = bias_stride;
  a.rows_per_group = static_cast<uint32_t>(rows / groups);
  a.offset = weight_offset;
  a.params_f32 = param_dtype == CK_DTYPE_F32;
  a.eps = eps;
  a.y = y;
  a.mean = mean;
  a.rstd = rstd;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(block_scales);
  a.rows = static_cast<uint32_t>(rows);
  a.rows_padded = static_cast<uint32_t>(round_up(rows, 128));
  a.cols = cols;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CK_DTYPE_BF16: return forward_typed<__nv_bfloat16>(a, s);
    case CK_DTYPE_F16: return forward_typed<__half>(a, s);
    default: return forward_typed<float>(a, s);
  }
}

extern "C" int64_t ck_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols, int64_t groups) {
  using namespace ck;
  if (rows <= 0 || cols <= 0 || groups <= 0 || rows % groups != 0) return 0;
  int64_t most = 0;  // over the forms that alignment decides between
  for (int form = 0; form < 12; ++form) {
    const int vec = form % 3 == 0 ? 1 : form % 3 == 1 ? 4 : 8;
    const Plan p = plan_backward(cols, vec == 4 ? 4 : 2, vec, form / 3 % 2 != 0, form / 6 != 0, groups, rows / groups);
    const int64_t need = p.chunks > 1 ? groups * p.chunks * 2 * cols * 4 : 0;
    if (need > most) most = need;
  }
  return most;
}

extern "C" int ck_layer_norm_backward(const void* dy, int dtype, int64_t rows, int64_t cols, int64_t dy_inner, int64_t dy_outer_stride,
                                      int64_t dy_inner_stride, const void* x, int64_t x_inner, int64_t x_outer_stride, int64_t x_inner_stride,
                                      const void* codes, const void* block_scales, const float* mean, const float* rstd, const void* weight,
                                      int param_dtype, int64_t groups, int64_t weight_stride, float weight_offset, void* dx, void* dweight,
                                      void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ck;
  if (int rc = check_shapes("layer_norm_backward", dtype, param_dtype, rows, dy_inner, cols, groups)) return rc;
  CK_REQUIRE(dy && dx && mean && rstd, "layer_norm_backward: null pointer");
  CK_REQUIRE((x != nullptr) != (codes != nullptr && block_scales != nullptr), "layer_norm_backward: either the input or its copy");
  CK_REQUIRE(x == nullptr || (x_inner > 0 && x_inner <= rows), "layer_norm_backward: bad row count of the input");
  CK_REQUIRE(x != nullptr || cols % 32 == 0, "layer_norm_backward: a copy has rows of a multiple of 32, got %lld", (long long)cols);
  BackwardArgs a = {};
  a.dy = dy;
  a.dy_rows = {dy_outer_stride, dy_inner_stride, static_cast<uint32_t>(dy_inner)};
  a.x = x;
  a.x_rows = {x_outer_stride, x_inner_stride, static_cast<uint32_t>(x != nullptr ? x_inner : 1)};
  a.codes = static_cast<const uint8_t*>(codes);
  a.scales = static_cast<const uint8_t*>(block_scales);
  a.mean = mean;
  a.rstd = rstd;
  a.weight = weight;
  a.weight_stride = weight_stride;
  a.offset = weight_offset;
  a.params_f32 = param_dtype == CK_DTYPE_F32;
  a.dx = dx;
  a.dweight = dweight;
  a.dbias = dbias;
  a.rows_per_group = static_cast<uint32_t>(rows / groups);
  a.groups = static_cast<uint32_t>(groups);
  a.cols = cols;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CK_DTYPE_BF16: return backward_typed<__nv_bfloat16>(a, dtype, workspace, workspace_bytes, s);
    case CK_DTYPE_F16: return backward_typed<__half>(a, dtype, workspace, workspace_bytes, s);
    default: return backward_typed<float>(a, dtype, workspace, workspace_bytes, s);
  }
}
