// Root-mean-square norm over the last dimension, for sm_100a, forward and backward:
//
//   h = x + r (rounded to their type; r may be absent),  rstd = 1 / sqrt(mean_k(h^2) + eps),  y = h * rstd * f,  f = weight_offset + weight
//   dh' = dh + rstd * (g - u * mean_k(g * u)),  g = dy * f,  u = h * rstd;   dweight = sum over rows of dy * u
//
// Bound by memory: each tensor is read or written once.  A team of threads has a row in registers: its lanes take neighbouring vectors, kVecs
// each, all fetched before the first is used; teams of up to 32 lanes share warps, wider rows have a block to themselves.
// The result can be MXFP8 (the values rounded to x's type, then as ck_quantize_mxfp8 has them): the lanes that share a block of 32 elements
// find its maximum, those that share four blocks write a word of scales.
// Backward, the blocks stay: each takes every so-manieth row, fetches the next one before it works on the one it has, and adds dweight's
// terms of its columns in registers; a second kernel adds the blocks' sums in order.
#include <atomic>

#include "ck_rows.cuh"

namespace ck {
namespace {

using rows::RowStrides;

struct RmsArgs {
  const void* x;
  const void* residual;  // or null
  const void* weight;    // or null: 1
  void* y;               // null where codes are written
  void* h;               // with a residual
  float* rstd;           // or null
  uint8_t* codes;
  uint8_t* scales;
  int64_t rows, cols;
  RowStrides x_strides, r_strides;
  float eps, offset;
  bool weight_f32;
  int lanes;             // of a team
};

struct RmsBackwardArgs {
  const void* dy;
  const void* h;
  const void* dh;      // or null
  const float* rstd;
  const void* weight;  // or null
  void* dx;
  float* partials;     // [blocks][cols], or null
  int64_t rows, cols;
  RowStrides dy_strides, h_strides, dh_strides;
  float offset;
  bool weight_f32;
  int lanes;
};

// Vectors of a lane.  A row of up to kVecs * 1024 vectors is one that a block holds; wider ones are walked twice.
constexpr int vecs_of(int bytes) { return bytes == 32 ? 2 : bytes == 16 ? 4 : 8; }
constexpr int kMostLanes = 1024, kMostBackwardLanes = 512;

template <typename T, int kEl>
__device__ __forceinline__ rows::Raw<T, kEl> load_vec(const T* p) {
  if constexpr (sizeof(T) * kEl == 32) {
    rows::Raw<T, kEl> r;
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
    asm volatile("ld.global.L1::no_allocate.v8.u32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p)
                 : "memory");
    return r;
  } else {
    return rows::load_once<T, kEl>(p);
  }
}
template <typename T, int kEl>
__device__ __forceinline__ void store_vec(T* p, const rows::Raw<T, kEl>& r) {
  if constexpr (sizeof(T) * kEl == 32) {
    st_global_256_no_allocate(p, *reinterpret_cast<const Vec256*>(&r));
  } else {
    rows::store(p, r);
  }
}

// kEl factors from column c on.
template <typename T, int kEl>
__device__ __forceinline__ void load_factors(const void* weight, bool f32, float offset, int64_t c, float (&f)[kEl]) {
  if (weight == nullptr) {
#pragma unroll
    for (int i = 0; i < kEl; ++i) f[i] = 1.0f;
    return;
  }
  if (sizeof(T) == 4 || f32) {
    const float* w = static_cast<const float*>(weight) + c;
    constexpr int kVec = kEl % 4 == 0 ? 4 : 1;  // the row's vectors begin at multiples of kEl
#pragma unroll
    for (int i = 0; i < kEl / kVec; ++i) {
      float part[kVec];
      rows::unpack(*reinterpret_cast<const rows::Raw<float, kVec>*>(w + i * kVec), part);
#pragma unroll
      for (int j = 0; j < kVec; ++j) f[i * kVec + j] = part[j];
    }
  } else {
    const T* w = static_cast<const T*>(weight) + c;
    constexpr int kVec = kEl % 8 == 0 ? 8 : kEl;
#pragma unroll
    for (int i = 0; i < kEl / kVec; ++i) {
      float part[kVec];
      rows::unpack(*reinterpret_cast<const rows::Raw<T, kVec>*>(w + i * kVec), part);
#pragma unroll
      for (int j = 0; j < kVec; ++j) f[i * kVec + j] = part[j];
    }
  }
#pragma unroll
  for (int i = 0; i < kEl; ++i) f[i] += offset;
}

// Sum over a team.  Teams of whole warps are whole blocks: `buf` holds a value for each warp, and `twice` says that it may still be read.
__device__ __forceinline__ float team_sum(float v, int lanes, float* buf) {
  if (lanes <= 32) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
  }
  v = rows::warp_sum(v);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float sum = 0.0f;
  const int warps = lanes >> 5;
  for (int i = 0; i < warps; ++i) sum += buf[i];
  return sum;
}

template <typename T, int kBytes, bool kCodes>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const RmsArgs a) {
  constexpr int kEl = kBytes / static_cast<int>(sizeof(T)), kVecs = vecs_of(kBytes);
  __shared__ float buf[32];
  pdl_launch_dependents();
  const int team = threadIdx.x / a.lanes, lane = threadIdx.x - team * a.lanes, teams = blockDim.x / a.lanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * teams + team;
  const int64_t blocks = a.cols >> 5, col_tiles = ceil_div(blocks, 4);
  const bool live = row < a.rows;  // other teams share warps with such, or write the scales' padding rows
  pdl_wait();
  rows::Raw<T, kEl> raw[kVecs], add[kVecs];
  bool have[kVecs];
  const T* x = static_cast<const T*>(a.x) + (live ? a.x_strides.offset(static_cast<uint32_t>(row)) : 0);
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int64_t c = (static_cast<int64_t>(j) * a.lanes + lane) * kEl;
    have[j] = live && c < a.cols;
    raw[j] = have[j] ? load_vec<T, kEl>(x + c) : rows::zeros<T, kEl>();
  }
  if (a.residual != nullptr) {
    const T* r = static_cast<const T*>(a.residual) + (live ? a.r_strides.offset(static_cast<uint32_t>(row)) : 0);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      if (have[j]) add[j] = load_vec<T, kEl>(r + (static_cast<int64_t>(j) * a.lanes + lane) * kEl);
    }
    T* h = static_cast<T*>(a.h) + row * a.cols;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      if (!have[j]) continue;
      float u[kEl], v[kEl];
      rows::unpack(raw[j], u);
      rows::unpack(add[j], v);
#pragma unroll
      for (int i = 0; i < kEl; ++i) u[i] += v[i];
      raw[j] = rows::pack<T, kEl>(u);  // the norm is of what stands in h
      store_vec(h + (static_cast<int64_t>(j) * a.lanes + lane) * kEl, raw[j]);
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    float u[kEl];
    rows::unpack(raw[j], u);
#pragma unroll
    for (int i = 0; i < kEl; ++i) sum = fmaf(u[i], u[i], sum);
  }
  sum = team_sum(sum, a.lanes, buf);
  const float rstd = rows::inverse_root(sum / static_cast<float>(a.cols) + a.eps);
  if (a.rstd != nullptr && live && lane == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int64_t c = (static_cast<int64_t>(j) * a.lanes + lane) * kEl;
    float u[kEl], f[kEl];
    if (have[j]) {
      rows::unpack(raw[j], u);
      load_factors<T, kEl>(a.weight, a.weight_f32, a.offset, c, f);
#pragma unroll
      for (int i = 0; i < kEl; ++i) u[i] = u[i] * rstd * f[i];
    } else {
#pragma unroll
      for (int i = 0; i < kEl; ++i) u[i] = 0.0f;
    }
    const rows::Raw<T, kEl> out = rows::pack<T, kEl>(u);
    if constexpr (!kCodes) {
      if (have[j]) store_vec(static_cast<T*>(a.y) + row * a.cols + c, out);
    } else {
      // what a call of the norm and one of the quantizer would give: the values rounded to T
      rows::unpack(out, u);
      float amax = 0.0f;
#pragma unroll
      for (int i = 0; i < kEl; ++i) amax = fmaxf(amax, fabsf(u[i]));
      constexpr int kShare = 32 / kEl;  // lanes of a block of 32 elements
#pragma unroll
      for (int o = 1; o < kShare; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
      const quant::Mxfp8Scale s = rows::block_scale(amax);
      uint32_t w[kEl / 4];
#pragma unroll
      for (int i = 0; i < kEl / 4; ++i) w[i] = rows::block_codes(make_float2(u[4 * i], u[4 * i + 1]), make_float2(u[4 * i + 2], u[4 * i + 3]), s);
      if (have[j]) {
        uint8_t* to = a.codes + row * a.cols + c;
        if constexpr (kEl == 16) {
          *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
          *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
        }
      }
      uint32_t word = (s.byte & 0xFFu) << (8 * ((lane / kShare) & 3));
      word |= __shfl_xor_sync(0xFFFFFFFFu, word, kShare);
      word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2 * kShare);
      const int64_t block = c >> 5;
      if ((lane & (4 * kShare - 1)) == 0 && block < blocks && row < round_up(a.rows, 128)) {
        *reinterpret_cast<uint32_t*>(a.scales + swizzled_scale_offset(row, block, col_tiles)) = word;
      }
    }
  }
}

// Rows that no block holds: walked twice.
template <typename T>
__global__ void __launch_bounds__(1024) rms_norm_wide_kernel(const RmsArgs a) {
  __shared__ float buf[32];
  pdl_launch_dependents();
  pdl_wait();
  const int64_t row = blockIdx.x, blocks = a.cols >> 5, col_tiles = ceil_div(blocks, 4);
  const bool live = row < a.rows;
  const T* x = static_cast<const T*>(a.x) + (live ? a.x_strides.offset(static_cast<uint32_t>(row)) : 0);
  const T* r = a.residual == nullptr ? nullptr : static_cast<const T*>(a.residual) + (live ? a.r_strides.offset(static_cast<uint32_t>(row)) : 0);
  T* h = static_cast<T*>(a.h) + row * a.cols;
  float sum = 0.0f;
  if (live) {
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
      float v = rows::to_float(x[c]);
      if (r != nullptr) {
        const T t = rows::from_float<T>(v + rows::to_float(r[c]));
        h[c] = t;
        v = rows::to_float(t);
      }
      sum = fmaf(v, v, sum);
    }
  }
  sum = team_sum(sum, 1024, buf);
  const float rstd = rows::inverse_root(sum / static_cast<float>(a.cols) + a.eps);
  if (a.rstd != nullptr && live && threadIdx.x == 0) a.rstd[row] = rstd;
  const T* from = r != nullptr ? h : x;  // each thread reads what it wrote
  const int64_t end = round_up(a.cols, 1024);
  for (int64_t c = threadIdx.x; c < end; c += 1024) {
    T y = rows::from_float<T>(0.0f);
    if (live && c < a.cols) {
      float f[1];
      load_factors<T, 1>(a.weight, a.weight_f32, a.offset, c, f);
      y = rows::from_float<T>(rows::to_float(from[c]) * rstd * f[0]);
    }
    if (a.codes == nullptr) {
      if (live && c < a.cols) static_cast<T*>(a.y)[row * a.cols + c] = y;
      continue;
    }
    const float v = rows::to_float(y);  // a warp has a block of 32 elements
    float amax = fabsf(v);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    const quant::Mxfp8Scale s = rows::block_scale(amax);
    if (live && c < a.cols) a.codes[row * a.cols + c] = static_cast<uint8_t>(rows::block_codes(make_float2(v, 0.0f), make_float2(0.0f, 0.0f), s));
    const int64_t block = c >> 5;
    if ((threadIdx.x & 31) == 0 && block < col_tiles * 4) a.scales[swizzled_scale_offset(row, block, col_tiles)] = static_cast<uint8_t>(s.byte);
  }
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
template <typename T, int kEl, int kVecs>
struct BackwardRow {
  rows::Raw<T, kEl> dy[kVecs], h[kVecs];
  float rstd;
};

template <typename T, int kBytes, int kThreads>
__global__ void __launch_bounds__(kThreads) rms_norm_backward_kernel(const RmsBackwardArgs a) {
  constexpr int kEl = kBytes / static_cast<int>(sizeof(T)), kVecs = vecs_of(kBytes);
  __shared__ float buf[2][32];
  extern __shared__ float sums[];  // [teams][cols], where teams share a block
  pdl_launch_dependents();
  const int team = threadIdx.x / a.lanes, lane = threadIdx.x - team * a.lanes, teams = blockDim.x / a.lanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
  bool have[kVecs];
#pragma unroll
  for (int j = 0; j < kVecs; ++j) have[j] = (static_cast<int64_t>(j) * a.lanes + lane) * kEl < a.cols;
  const auto fetch = [&](int64_t row) {
    BackwardRow<T, kEl, kVecs> b;
    const bool live = row < a.rows;
    const uint32_t r = live ? static_cast<uint32_t>(row) : 0u;
    const T* dy = static_cast<const T*>(a.dy) + a.dy_strides.offset(r);
    const T* h = static_cast<const T*>(a.h) + a.h_strides.offset(r);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int64_t c = (static_cast<int64_t>(j) * a.lanes + lane) * kEl;
      const bool get = live && have[j];
      b.dy[j] = get ? load_vec<T, kEl>(dy + c) : rows::zeros<T, kEl>();
      b.h[j] = get ? load_vec<T, kEl>(h + c) : rows::zeros<T, kEl>();
    }
    b.rstd = live ? ld_f32_dependent(a.rstd + row) : 0.0f;
    return b;
  };
  pdl_wait();
  float acc[kVecs][kEl] = {};
  const float over = 1.0f / static_cast<float>(a.cols);
  int64_t first = static_cast<int64_t>(blockIdx.x) * teams;  // the block's first team's row: all teams take the same number of turns
  BackwardRow<T, kEl, kVecs> next = fetch(first + team);
  for (int turn = 0; first < a.rows; first += step, turn ^= 1) {
    const BackwardRow<T, kEl, kVecs> b = next;
    const int64_t row = first + team;
    rows::Raw<T, kEl> more[kVecs];  // dh, which is added behind the sum
    if (a.dh != nullptr) {
      const T* dh = static_cast<const T*>(a.dh) + a.dh_strides.offset(row < a.rows ? static_cast<uint32_t>(row) : 0u);
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        if (row < a.rows && have[j]) more[j] = load_vec<T, kEl>(dh + (static_cast<int64_t>(j) * a.lanes + lane) * kEl);
      }
    }
    next = fetch(first + step + team);
    float along = 0.0f;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      float f[kEl], dy[kEl], h[kEl];
      if (have[j]) {
        load_factors<T, kEl>(a.weight, a.weight_f32, a.offset, (static_cast<int64_t>(j) * a.lanes + lane) * kEl, f);
        rows::unpack(b.dy[j], dy);
        rows::unpack(b.h[j], h);
#pragma unroll
        for (int i = 0; i < kEl; ++i) {
          const float u = h[i] * b.rstd;
          along = fmaf(dy[i] * f[i], u, along);
          acc[j][i] = fmaf(dy[i], u, acc[j][i]);
        }
      }
    }
    along = team_sum(along, a.lanes, buf[turn]) * over;
    if (row < a.rows) {
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        if (!have[j]) continue;
        const int64_t c = (static_cast<int64_t>(j) * a.lanes + lane) * kEl;
        float f[kEl], dy[kEl], h[kEl], dh[kEl];
        load_factors<T, kEl>(a.weight, a.weight_f32, a.offset, c, f);
        rows::unpack(b.dy[j], dy);
        rows::unpack(b.h[j], h);
        if (a.dh != nullptr) {
          rows::unpack(more[j], dh);
        } else {
#pragma unroll
          for (int i = 0; i < kEl; ++i) dh[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kEl; ++i) dh[i] = fmaf(b.rstd, fmaf(-(h[i] * b.rstd), along, dy[i] * f[i]), dh[i]);
        store_vec(static_cast<T*>(a.dx) + row * a.cols + c, rows::pack<T, kEl>(dh));
      }
    }
  }
  if (a.partials == nullptr) return;
  float* to = a.partials + static_cast<int64_t>(blockIdx.x) * a.cols;
  if (teams == 1) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int64_t c = (static_cast<int64_t>(j) * a.lanes + lane) * kEl;
#pragma unroll
      for (int i = 0; i < kEl; ++i) {
        if (have[j]) to[c + i] = acc[j][i];
      }
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int64_t c = (static_cast<int64_t>(j) * a.lanes + lane) * kEl;
#pragma unroll
    for (int i = 0; i < kEl; ++i) {
      if (have[j]) sums[team * a.cols + c + i] = acc[j][i];
    }
  }
  __syncthreads();
  for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
    float s = 0.0f;
    for (int t = 0; t < teams; ++t) s += sums[t * a.cols + c];
    to[c] = s;
  }
}

// Rows that no block holds.
template <typename T>
__global__ void __launch_bounds__(1024) rms_norm_backward_wide_kernel(const RmsBackwardArgs a) {
  __shared__ float buf[32];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t row = blockIdx.x;
  const T* dy = static_cast<const T*>(a.dy) + a.dy_strides.offset(row);
  const T* h = static_cast<const T*>(a.h) + a.h_strides.offset(row);
  const T* dh = a.dh == nullptr ? nullptr : static_cast<const T*>(a.dh) + a.dh_strides.offset(row);
  const float rstd = ld_f32_dependent(a.rstd + row);
  float along = 0.0f;
#pragma unroll 4
  for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
    float f[1];
    load_factors<T, 1>(a.weight, a.weight_f32, a.offset, c, f);
    along = fmaf(rows::to_float(dy[c]) * f[0], rows::to_float(h[c]) * rstd, along);
  }
  along = team_sum(along, 1024, buf) / static_cast<float>(a.cols);
#pragma unroll 4
  for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
    float f[1];
    load_factors<T, 1>(a.weight, a.weight_f32, a.offset, c, f);
    const float u = rows::to_float(h[c]) * rstd, old = dh == nullptr ? 0.0f : rows::to_float(dh[c]);
    static_cast<T*>(a.dx)[static_cast<int64_t>(row) * a.cols + c] = rows::from_float<T>(fmaf(rstd, fmaf(-u, along, rows::to_float(dy[c]) * f[0]), old));
  }
}

// Their part of dweight: a column a thread, a chunk of the rows a block.
template <typename T>
__global__ void __launch_bounds__(256) rms_norm_columns_kernel(const RmsBackwardArgs a, int64_t chunk) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (c >= a.cols) return;
  float sum = 0.0f;
  const int64_t end = min(a.rows, (blockIdx.y + 1) * chunk);
#pragma unroll 4
  for (int64_t r = blockIdx.y * chunk; r < end; ++r) {
    const T* dy = static_cast<const T*>(a.dy) + a.dy_strides.offset(static_cast<uint32_t>(r));
    const T* h = static_cast<const T*>(a.h) + a.h_strides.offset(static_cast<uint32_t>(r));
    sum = fmaf(rows::to_float(dy[c]), rows::to_float(h[c]) * ld_f32_dependent(a.rstd + r), sum);
  }
  a.partials[blockIdx.y * a.cols + c] = sum;
}

// The blocks' sums of a column, in order: eight threads above one another take every eighth, then they are added.
template <typename P>
__global__ void __launch_bounds__(256) rms_norm_add_kernel(const float* partials, int blocks, int64_t cols, P* out) {
  __shared__ float buf[8][33];
  pdl_launch_dependents();
  pdl_wait();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + x;
  float sum = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (int b = y; b < blocks; b += 8) sum += ld_f32_dependent(partials + b * cols + c);
  }
  buf[y][x] = sum;
  __syncthreads();
  if (y != 0 || c >= cols) return;
  sum = buf[0][x];
#pragma unroll
  for (int i = 1; i < 8; ++i) sum += buf[i][x];
  out[c] = rows::from_float<P>(sum);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool is_float(int dtype) { return dtype == CK_DTYPE_F32 || dtype == CK_DTYPE_F16 || dtype == CK_DTYPE_BF16; }
int size_of(int dtype) { return dtype == CK_DTYPE_F32 ? 4 : 2; }

struct Rows {
  const void* base;
  int64_t inner, outer_stride, inner_stride;
};

// Bytes of a vector: the widest that every row of every tensor starts on, of which a row has a whole number.
int vector_bytes(int dtype, int64_t cols, const void* weight, int param_dtype, std::initializer_list<Rows> tensors) {
  const int size = size_of(dtype);
  for (int bytes : {32, 16, 4}) {
    if (bytes < size || cols * size % bytes != 0) continue;
    const int factor_bytes = bytes / size * size_of(param_dtype) < 16 ? bytes / size * size_of(param_dtype) : 16;
    bool ok = weight == nullptr || reinterpret_cast<uintptr_t>(weight) % factor_bytes == 0;
    for (const Rows& t : tensors) {
      ok = ok && (t.base == nullptr || (reinterpret_cast<uintptr_t>(t.base) % bytes == 0 && t.outer_stride * size % bytes == 0 && t.inner_stride * size % bytes == 0));
    }
    if (ok) return bytes;
  }
  return size;
}

// Lanes of a team, 0 for rows that no block holds.
int lanes_of(int dtype, int bytes, int64_t cols, int least, int most) {
  const int64_t vecs = ceil_div(cols * size_of(dtype), bytes), lanes = ceil_div(vecs, vecs_of(bytes));
  if (lanes > most) return 0;
  if (lanes > 32) return static_cast<int>(round_up(lanes, 32));
  int pow2 = least;
  while (pow2 < lanes) pow2 *= 2;
  return pow2;
}

RowStrides strides_of(const Rows& r) { return {r.outer_stride, r.inner_stride, static_cast<uint32_t>(r.inner)}; }
bool rows_ok(const Rows& r, int64_t rows) { return r.inner > 0 && r.inner <= 0xFFFFFFFFll && (r.inner >= rows || rows % r.inner == 0); }

template <typename T>
int launch_forward(const RmsArgs& args, int bytes, cudaStream_t s) {
  RmsArgs a = args;
  const int64_t rows = a.codes != nullptr ? round_up(a.rows, 128) : a.rows;
  // four blocks of scales are a word: a team has the lanes that write one at least
  a.lanes = lanes_of(sizeof(T) == 4 ? CK_DTYPE_F32 : CK_DTYPE_BF16, bytes, a.cols, a.codes != nullptr ? 128 * static_cast<int>(sizeof(T)) / 32 : 1, kMostLanes);
  if (a.lanes == 0) {
    CK_CUDA(launch_pdl(rms_norm_wide_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(1024), 0, s, a));
    return CK_OK;
  }
  const int threads = a.lanes > 32 ? a.lanes : 128;
  const dim3 grid(static_cast<unsigned>(ceil_div(rows, threads / a.lanes))), block(threads);
  if (a.codes != nullptr) {
    CK_CUDA(launch_pdl(rms_norm_kernel<T, 32, true>, grid, block, 0, s, a));
    return CK_OK;
  }
  switch (bytes) {
    case 32: CK_CUDA(launch_pdl(rms_norm_kernel<T, 32, false>, grid, block, 0, s, a)); break;
    case 16: CK_CUDA(launch_pdl(rms_norm_kernel<T, 16, false>, grid, block, 0, s, a)); break;
    case 4: CK_CUDA(launch_pdl(rms_norm_kernel<T, 4, false>, grid, block, 0, s, a)); break;
    default: CK_CUDA(launch_pdl(rms_norm_kernel<T, sizeof(T), false>, grid, block, 0, s, a));
  }
  return CK_OK;
}

// Blocks that share the rows, and so dweight's partial sums: two of 512 threads an SM, four rows a team at least.
constexpr int kBackwardThreads = 128;
struct BackwardPlan {
  int lanes, threads, blocks;
  int64_t chunk;  // wide rows: rows of a chunk
};
BackwardPlan backward_plan(int dtype, int bytes, int64_t rows, int64_t cols) {
  BackwardPlan p = {};
  p.lanes = lanes_of(dtype, bytes, cols, 1, kMostBackwardLanes);
  if (p.lanes == 0) {
    const int64_t strips = ceil_div(cols, 256);
    int64_t chunks = ceil_div(4 * sm_count(), strips);
    if (chunks > rows) chunks = rows;
    p.chunk = ceil_div(rows, chunks);
    p.blocks = static_cast<int>(ceil_div(rows, p.chunk));
    return p;
  }
  p.threads = p.lanes > 32 ? p.lanes : kBackwardThreads;
  const int64_t teams = p.threads / p.lanes, resident = static_cast<int64_t>(sm_count()) * (p.threads >= 512 ? 1 : 512 / p.threads);
  int64_t blocks = ceil_div(rows, teams * 4);
  if (blocks < sm_count()) blocks = ceil_div(rows, teams) < sm_count() ? ceil_div(rows, teams) : sm_count();
  p.blocks = static_cast<int>(blocks < resident ? blocks : resident);
  return p;
}

template <typename T, int kBytes>
int launch_backward_vec(const RmsBackwardArgs& a, const BackwardPlan& p, cudaStream_t s) {
  const int teams = p.threads / p.lanes;
  const size_t smem = teams > 1 && a.partials != nullptr ? teams * a.cols * 4 : 0;
  if (p.threads <= 256) {
    CK_CUDA(launch_pdl(rms_norm_backward_kernel<T, kBytes, 256>, dim3(p.blocks), dim3(p.threads), smem, s, a));
  } else {
    CK_CUDA(launch_pdl(rms_norm_backward_kernel<T, kBytes, 512>, dim3(p.blocks), dim3(p.threads), smem, s, a));
  }
  return CK_OK;
}

template <typename T>
int launch_backward(RmsBackwardArgs a, const BackwardPlan& p, int bytes, cudaStream_t s) {
  a.lanes = p.lanes;
  if (p.lanes == 0) {
    CK_CUDA(launch_pdl(rms_norm_backward_wide_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, s, a));
    if (a.partials == nullptr) return CK_OK;
    CK_CUDA(launch_pdl(rms_norm_columns_kernel<T>, dim3(static_cast<unsigned>(ceil_div(a.cols, 256)), p.blocks), dim3(256), 0, s, a, p.chunk));
    return CK_OK;
  }
  switch (bytes) {
    case 32: return launch_backward_vec<T, 32>(a, p, s);
    case 16: return launch_backward_vec<T, 16>(a, p, s);
    case 4: return launch_backward_vec<T, 4>(a, p, s);
    default: return launch_backward_vec<T, sizeof(T)>(a, p, s);
  }
}

template <typename P>
int launch_add(const float* partials, int blocks, int64_t cols, void* out, cudaStream_t s) {
  CK_CUDA(launch_pdl(rms_norm_add_kernel<P>, dim3(static_cast<unsigned>(ceil_div(cols, 32))), dim3(256), 0, s, partials, blocks, cols, static_cast<P*>(out)));
  return CK_OK;
}

int check_rms(const char* op, int dtype, int param_dtype, int64_t rows, int64_t cols) {
  CK_REQUIRE(is_float(dtype), "%s: unsupported dtype code %d", op, dtype);
  CK_REQUIRE(param_dtype == dtype || param_dtype == CK_DTYPE_F32, "%s: the weight must be of the input's type or fp32", op);
  CK_REQUIRE(rows > 0 && cols > 0 && rows < (1ll << 31) - 128 && cols < (1ll << 31), "%s: bad shape [%lld, %lld]", op, (long long)rows, (long long)cols);
  return CK_OK;
}

}  // namespace
}  // namespace ck

extern "C" int ck_rms_norm_forward(const void* x, int dtype, int64_t rows, int64_t cols, int64_t x_inner, int64_t x_outer_stride, int64_t x_inner_stride,
                                   const void* residual, int64_t r_inner, int64_t r_outer_stride, int64_t r_inner_stride, const void* weight,
                                   int param_dtype, float weight_offset, float eps, void* y, void* h, float* rstd, void* codes, void* block_scales,
                                   void* stream) {
  using namespace ck;
  const char* op = "rms_norm_forward";
  if (int rc = check_rms(op, dtype, param_dtype, rows, cols)) return rc;
  CK_REQUIRE(x != nullptr && (y != nullptr) != (codes != nullptr) && (codes != nullptr) == (block_scales != nullptr), "%s: null pointer", op);
  CK_REQUIRE((residual != nullptr) == (h != nullptr), "%s: a residual and the sum's buffer belong together", op);
  const Rows xr = {x, x_inner, x_outer_stride, x_inner_stride}, rr = {residual, r_inner, r_outer_stride, r_inner_stride};
  CK_REQUIRE(rows_ok(xr, rows) && (residual == nullptr || rows_ok(rr, rows)), "%s: bad row strides", op);
  RmsArgs a = {};
  a.x = x;
  a.residual = residual;
  a.weight = weight;
  a.y = y;
  a.h = h;
  a.rstd = rstd;
  a.codes = static_cast<uint8_t*>(codes);
  a.scales = static_cast<uint8_t*>(block_scales);
  a.rows = rows;
  a.cols = cols;
  a.x_strides = strides_of(xr);
  if (residual != nullptr) a.r_strides = strides_of(rr);
  a.eps = eps;
  a.offset = weight == nullptr ? 0.0f : weight_offset;
  a.weight_f32 = param_dtype == CK_DTYPE_F32;
  const Rows out = {y, 1, cols, cols}, sum = {h, 1, cols, cols};
  const int bytes = vector_bytes(dtype, cols, weight, param_dtype, {xr, rr, out, sum});
  if (codes != nullptr) {
    CK_REQUIRE(cols % 32 == 0 && bytes == 32 && reinterpret_cast<uintptr_t>(codes) % 32 == 0 && reinterpret_cast<uintptr_t>(block_scales) % 4 == 0,
               "%s: MXFP8 results need columns of a multiple of 32, rows and codes on 32-byte boundaries, the weight on 16-byte ones", op);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CK_DTYPE_BF16: return launch_forward<__nv_bfloat16>(a, bytes, s);
    case CK_DTYPE_F16: return launch_forward<__half>(a, bytes, s);
    default: return launch_forward<float>(a, bytes, s);
  }
}

namespace {
// The most blocks that any vector width takes: the workspace's size does not depend on addresses.
int64_t rms_backward_blocks(int dtype, int64_t rows, int64_t cols) {
  int64_t most = 1;
  for (int bytes : {32, 16, 4, 2}) {
    if (bytes < ck::size_of(dtype)) continue;
    const int64_t n = ck::backward_plan(dtype, bytes, rows, cols).blocks;
    if (n > most) most = n;
  }
  return most;
}
}  // namespace

extern "C" int64_t ck_rms_norm_backward_workspace_bytes(int dtype, int64_t rows, int64_t cols) {
  if (ck::check_rms("rms_norm_backward", dtype, CK_DTYPE_F32, rows, cols) != CK_OK) return 0;
  return rms_backward_blocks(dtype, rows, cols) * cols * 4;
}

extern "C" int ck_rms_norm_backward(const void* dy, int dtype, int64_t rows, int64_t cols, int64_t dy_inner, int64_t dy_outer_stride,
                                    int64_t dy_inner_stride, const void* h, int64_t h_inner, int64_t h_outer_stride, int64_t h_inner_stride,
                                    const void* dh, int64_t dh_inner, int64_t dh_outer_stride, int64_t dh_inner_stride, const float* rstd,
                                    const void* weight, int param_dtype, float weight_offset, void* dx, void* dweight, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  using namespace ck;
  const char* op = "rms_norm_backward";
  if (int rc = check_rms(op, dtype, param_dtype, rows, cols)) return rc;
  CK_REQUIRE(dy && h && rstd && dx, "%s: null pointer", op);
  const Rows dyr = {dy, dy_inner, dy_outer_stride, dy_inner_stride}, hr = {h, h_inner, h_outer_stride, h_inner_stride};
  const Rows dhr = {dh, dh_inner, dh_outer_stride, dh_inner_stride}, out = {dx, 1, cols, cols};
  CK_REQUIRE(rows_ok(dyr, rows) && rows_ok(hr, rows) && (dh == nullptr || rows_ok(dhr, rows)), "%s: bad row strides", op);
  RmsBackwardArgs a = {};
  a.dy = dy;
  a.h = h;
  a.dh = dh;
  a.rstd = rstd;
  a.weight = weight;
  a.dx = dx;
  a.rows = rows;
  a.cols = cols;
  a.dy_strides = strides_of(dyr);
  a.h_strides = strides_of(hr);
  if (dh != nullptr) a.dh_strides = strides_of(dhr);
  a.offset = weight == nullptr ? 0.0f : weight_offset;
  a.weight_f32 = param_dtype == CK_DTYPE_F32;
  const int bytes = vector_bytes(dtype, cols, weight, param_dtype, {dyr, hr, dhr, out});
  const BackwardPlan p = backward_plan(dtype, bytes, rows, cols);
  if (dweight != nullptr) {
    CK_REQUIRE(workspace != nullptr && workspace_bytes >= p.blocks * cols * 4 && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "%s: workspace of %lld bytes, %lld needed", op, (long long)workspace_bytes, (long long)(p.blocks * cols * 4));
    a.partials = static_cast<float*>(workspace);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc;
  switch (dtype) {
    case CK_DTYPE_BF16: rc = launch_backward<__nv_bfloat16>(a, p, bytes, s); break;
    case CK_DTYPE_F16: rc = launch_backward<__half>(a, p, bytes, s); break;
    default: rc = launch_backward<float>(a, p, bytes, s);
  }
  if (rc != CK_OK || dweight == nullptr) return rc;
  switch (param_dtype) {
    case CK_DTYPE_BF16: return launch_add<__nv_bfloat16>(a.partials, p.blocks, cols, dweight, s);
    case CK_DTYPE_F16: return launch_add<__half>(a.partials, p.blocks, cols, dweight, s);
    default: return launch_add<float>(a.partials, p.blocks, cols, dweight, s);
  }
}
