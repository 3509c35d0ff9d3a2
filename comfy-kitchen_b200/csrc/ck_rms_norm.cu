// Root-mean-square norm over the last dimension, for sm_100a, forward and backward:
//
//   h = x + r (rounded to their type; r may be absent),  rstd = 1 / sqrt(mean_k(h^2) + eps),  y = h * rstd * f,  f = weight_offset + weight
//   dh' = dh + rstd * (g - u * mean_k(g * u)),  g = dy * f,  u = h * rstd;   dweight = sum over rows of dy * u
//
// Bound by memory: each tensor is read or written once.  A team of threads has a row in registers: its lanes take neighbouring vectors, kVecs
// each, all fetched before the first is used; teams of up to 32 lanes share warps, wider rows have a block to themselves.
// The result can be MXFP8 (the values rounded to x's type, then as ck_quantize_mxfp8 has them): the lanes that share a block of 32 elements
// find its maximum, those that share four blocks write a word of scales.
// Backward, the blocks stay: each takes its share of the rows, spread over all, out of a ring in shared memory and adds dweight's terms of its columns in
// registers; a second kernel adds the blocks' sums in order.
// 16384 x 4096 bf16 with a residual: forward 82 us (6.56 TB/s, 1.00 of the copy rate), with an MXFP8 result 83 (5.7), backward 89 (6.0); 20000 x 1001
// 44 and 44; one row of 4096 2.6 and 6.7.
#include <atomic>

#include "ck_rows.cuh"

namespace ck {
namespace {

using sm100::smem_u32;

// rows::RowStrides with another quotient.  Row r is row r % inner of outer index r / inner; the quotient by a product and a shift, made for `inner` on the
// host, is the division by an invariant integer of Granlund and Montgomery (1994): for rows below 2^31, r / d = (high half of m * r + r) >> l with 2^l >= d
// and m = floor(2^32 (2^l - d) / d) + 1.  (The compiler's division, for three tensors a row, kept the conversion unit busy for half of the backward kernel's time.)
struct DividedRows {
  int64_t outer_stride, inner_stride;  // elements
  uint32_t inner, m, l;
  __device__ __forceinline__ int64_t offset(uint32_t row) const {
    const uint32_t o = (__umulhi(m, row) + row) >> l;
    return static_cast<int64_t>(o) * outer_stride + static_cast<int64_t>(row - o * inner) * inner_stride;
  }
};

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
  DividedRows x_strides, r_strides;
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
  DividedRows dy_strides, h_strides, dh_strides;
  float offset;
  bool weight_f32;
  int lanes;
  int batches;         // of the ring
};

// How a row lies: vectors of 32 or 16 bytes on whose boundaries every row starts; vectors of 16 bytes of which a row's first and last
// have elements of its neighbours too (all tensors' rows lie alike); single elements, where tensors' rows lie differently.
enum class Form { k32, k16, kShifted, kSingle };

template <typename T, Form kForm>
constexpr int elements() {
  return kForm == Form::k32 ? 32 / static_cast<int>(sizeof(T)) : kForm == Form::kSingle ? 1 : 16 / static_cast<int>(sizeof(T));
}
// Vectors of a lane.  A row of up to so many times 1024 vectors is one that a block holds; wider ones are walked twice.
constexpr int forward_vecs(Form form) { return form == Form::k32 ? 2 : form == Form::kSingle ? 8 : 4; }
constexpr int kMostLanes = 1024;

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

// Which elements of a shifted vector, whose first element is column c, are the row's own: its neighbours' read as zeros and are not written.
// (The 16 aligned bytes that hold an element of a tensor lie in its allocation.)
template <typename T, Form kForm>
struct Own {
  uint32_t w[kForm == Form::kShifted ? 4 : 1];
  __device__ __forceinline__ void set(int c, int cols) {
    if constexpr (kForm == Form::kShifted) {
      constexpr int kPerWord = 4 / static_cast<int>(sizeof(T));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = c + i * kPerWord;
        w[i] = 0xFFFFFFFFu;
        if (kPerWord == 1) {
          if (at < 0 || at >= cols) w[i] = 0;
        } else {
          if (at < 0 || at >= cols) w[i] &= 0xFFFF0000u;
          if (at + 1 < 0 || at + 1 >= cols) w[i] &= 0x0000FFFFu;
        }
      }
    }
  }
};
template <typename T, Form kForm>
__device__ __forceinline__ rows::Raw<T, elements<T, kForm>()> load_cols(const T* at, const Own<T, kForm>& own) {
  rows::Raw<T, elements<T, kForm>()> r = load_vec<T, elements<T, kForm>()>(at);
  if constexpr (kForm == Form::kShifted) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] &= own.w[i];
  }
  return r;
}
template <typename T, Form kForm>
__device__ __forceinline__ void store_cols(T* row, int c, int cols, const rows::Raw<T, elements<T, kForm>()>& r) {
  constexpr int kEl = elements<T, kForm>();
  if constexpr (kForm == Form::k32) {
    st_global_256_no_allocate(row + c, *reinterpret_cast<const Vec256*>(&r));
  } else {
    if (kForm == Form::kShifted && (c < 0 || c + kEl > cols)) {
#pragma unroll
      for (int i = 0; i < kEl; ++i) {
        if (c + i >= 0 && c + i < cols) row[c + i] = r.v[i];
      }
    } else {
      rows::store(row + c, r);
    }
  }
}

// A vector's numbers, in pairs that one instruction computes on.
template <int kEl>
struct Numbers {
  static constexpr int kPairs = (kEl + 1) / 2;
  float2 p[kPairs];
};
template <typename T, int kEl>
__device__ __forceinline__ Numbers<kEl> numbers_of(const rows::Raw<T, kEl>& r) {
  Numbers<kEl> n;
  float f[kEl];
  rows::unpack(r, f);
#pragma unroll
  for (int i = 0; i < Numbers<kEl>::kPairs; ++i) n.p[i] = make_float2(f[2 * i], 2 * i + 1 < kEl ? f[2 * i + 1] : 0.0f);
  return n;
}
template <typename T, int kEl>
__device__ __forceinline__ rows::Raw<T, kEl> raw_of(const Numbers<kEl>& n) {
  float f[kEl];
#pragma unroll
  for (int i = 0; i < kEl; ++i) f[i] = i % 2 == 0 ? n.p[i / 2].x : n.p[i / 2].y;
  return rows::pack<T, kEl>(f);
}

// The factors of a vector's columns.
template <typename T, Form kForm>
__device__ __forceinline__ void load_factors(const void* weight, bool f32, float offset, int c, int cols, Numbers<elements<T, kForm>()>* out) {
  constexpr int kEl = elements<T, kForm>();
  float f[kEl];
  const auto give = [&]() {
#pragma unroll
    for (int i = 0; i < Numbers<kEl>::kPairs; ++i) out->p[i] = make_float2(f[2 * i], 2 * i + 1 < kEl ? f[2 * i + 1] : 0.0f);
  };
  if (weight == nullptr) {
#pragma unroll
    for (int i = 0; i < kEl; ++i) f[i] = 1.0f;
    return give();
  }
  if constexpr (kForm == Form::kShifted) {
    if (c < 0 || c + kEl > cols) {
#pragma unroll
      for (int i = 0; i < kEl; ++i) {
        const int at = min(max(c + i, 0), cols - 1);
        f[i] = sizeof(T) == 4 || f32 ? static_cast<const float*>(weight)[at] : rows::to_float(static_cast<const T*>(weight)[at]);
      }
    } else if (sizeof(T) == 4 || f32) {
#pragma unroll
      for (int i = 0; i < kEl; ++i) f[i] = static_cast<const float*>(weight)[c + i];
    } else {
#pragma unroll
      for (int i = 0; i < kEl; ++i) f[i] = rows::to_float(static_cast<const T*>(weight)[c + i]);
    }
  } else if (sizeof(T) == 4 || f32) {
    const float* w = static_cast<const float*>(weight) + c;
    constexpr int kVec = kEl % 4 == 0 ? 4 : 1;
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
  give();
}

// Elements of its neighbour in a row's first vector.
template <typename T, Form kForm>
__device__ __forceinline__ int shift_of(const T* row) {
  return kForm == Form::kShifted ? static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15) / static_cast<int>(sizeof(T)) : 0;
}

// Sum over a team.  Teams of whole warps are whole blocks: `buf` holds a value for each warp.
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

template <typename T, Form kForm, bool kCodes>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const RmsArgs a) {
  constexpr int kEl = elements<T, kForm>(), kVecs = forward_vecs(kForm);
  __shared__ float buf[32];
  pdl_launch_dependents();
  const int team = threadIdx.x / a.lanes, lane = threadIdx.x - team * a.lanes, teams = blockDim.x / a.lanes;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * teams + team;
  const int cols = static_cast<int>(a.cols);
  const int64_t blocks = a.cols >> 5, col_tiles = ceil_div(blocks, 4);
  const bool live = row < a.rows;  // other teams share warps with such, or write the scales' padding rows
  pdl_wait();
  rows::Raw<T, kEl> raw[kVecs], add[kVecs];
  Own<T, kForm> own[kVecs];
  bool have[kVecs];
  const T* x = static_cast<const T*>(a.x) + (live ? a.x_strides.offset(static_cast<uint32_t>(row)) : 0);
  const int shift = shift_of<T, kForm>(x);
  const auto col_of = [&](int j) { return (j * a.lanes + lane) * kEl - shift; };
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    have[j] = live && col_of(j) < cols;
    own[j].set(col_of(j), cols);
    raw[j] = have[j] ? load_cols<T, kForm>(x + col_of(j), own[j]) : rows::zeros<T, kEl>();
  }
  if (a.residual != nullptr) {
    const T* r = static_cast<const T*>(a.residual) + (live ? a.r_strides.offset(static_cast<uint32_t>(row)) : 0);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      if (have[j]) add[j] = load_cols<T, kForm>(r + col_of(j), own[j]);
    }
    T* h = static_cast<T*>(a.h) + row * a.cols;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      if (!have[j]) continue;
      Numbers<kEl> u = numbers_of(raw[j]);
      const Numbers<kEl> v = numbers_of(add[j]);
#pragma unroll
      for (int i = 0; i < Numbers<kEl>::kPairs; ++i) u.p[i] = add_x2(u.p[i], v.p[i]);
      raw[j] = raw_of<T>(u);  // the norm is of what stands in h
      store_cols<T, kForm>(h, col_of(j), cols, raw[j]);
    }
  }
  float2 sums = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const Numbers<kEl> u = numbers_of(raw[j]);
#pragma unroll
    for (int i = 0; i < Numbers<kEl>::kPairs; ++i) sums = fma_x2(u.p[i], u.p[i], sums);
  }
  const float sum = team_sum(sums.x + sums.y, a.lanes, buf);
  const float rstd = rows::inverse_root(sum / static_cast<float>(a.cols) + a.eps);
  if (a.rstd != nullptr && live && lane == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int c = col_of(j);
    Numbers<kEl> n = numbers_of(raw[j]);  // zeros where there is nothing
    if (have[j]) {
      Numbers<kEl> f;
      load_factors<T, kForm>(a.weight, a.weight_f32, a.offset, c, cols, &f);
#pragma unroll
      for (int i = 0; i < Numbers<kEl>::kPairs; ++i) n.p[i] = mul_x2(mul_x2(n.p[i], rows::both(rstd)), f.p[i]);
    }
    const rows::Raw<T, kEl> out = raw_of<T>(n);
    if constexpr (!kCodes) {
      if (have[j]) store_cols<T, kForm>(static_cast<T*>(a.y) + row * a.cols, c, cols, out);
    } else {
      // what a call of the norm and one of the quantizer would give: the values rounded to T
      float u[kEl];
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
      Numbers<1> f;
      load_factors<T, Form::kSingle>(a.weight, a.weight_f32, a.offset, static_cast<int>(c), static_cast<int>(a.cols), &f);
      y = rows::from_float<T>(rows::to_float(from[c]) * rstd * f.p[0].x);
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
// 16 bytes of a row on their way to shared memory.
__device__ __forceinline__ void copy_16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copies_wait(int left) {
  switch (left) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
  }
}

// Sums over a team of one number for each of kRows rows, which go through the exchange together.
template <int kRows>
__device__ __forceinline__ void team_sums(float (&v)[kRows], int lanes, float (*buf)[32]) {
  if (lanes <= 32) {
    for (int o = lanes >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) v[r] += __shfl_xor_sync(0xFFFFFFFFu, v[r], o);
    }
    return;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) v[r] += __shfl_xor_sync(0xFFFFFFFFu, v[r], o);
  }
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) buf[r][threadIdx.x >> 5] = v[r];
  }
  __syncthreads();
  const int warps = lanes >> 5;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // at most sixteen warps; what stands behind the last one is zero
      if (4 * i < warps) {
        const float4 q = *reinterpret_cast<const float4*>(&buf[r][4 * i]);
        sum += (q.x + q.y) + (q.z + q.w);
      }
    }
    v[r] = sum;
  }
}

constexpr int kMostBatches = 4;

// kRows rows at a time: waiting, the exchange over lanes and the meeting of warps cost the same for one.  They come
// through a ring in shared memory, a.batches of kRows rows, of which each thread writes and reads its own vectors alone, so that nobody meets for
// them; a batch is asked for as soon as the one in its place has been read for the last time.  (16384 x 4096 bf16: with the next row in
// registers, 49 KiB on their way to an SM, 122 us, so 89; with 32 bytes of a lane, of which a copy takes 16, every sector was asked for twice: 148.)
// kSingle, whose elements cannot be copied so, reads a row when it comes to it.
template <typename T, Form kForm, int kVecs, int kThreads, int kRows>
__global__ void __launch_bounds__(kThreads, 512 / kThreads) rms_norm_backward_kernel(const RmsBackwardArgs a) {
  constexpr int kEl = elements<T, kForm>(), kPairs = Numbers<kEl>::kPairs;
  constexpr bool kRing = kForm != Form::kSingle;
  constexpr int kPieces = kRing ? kVecs * kEl * static_cast<int>(sizeof(T)) / 16 : 1;  // of 16 bytes, of a tensor and thread
  __shared__ __align__(16) float buf[2][kRows][32];
  extern __shared__ __align__(16) uint8_t ring[];  // [batches][rows][tensors][pieces][threads] 16 bytes; then [teams][cols] sums, where teams share a block
  pdl_launch_dependents();
  const int cols = static_cast<int>(a.cols);
  const int team = threadIdx.x / a.lanes, lane = threadIdx.x - team * a.lanes, teams = blockDim.x / a.lanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
  int64_t first = static_cast<int64_t>(blockIdx.x) * teams;  // the block's first team's row: all teams take the same number of turns
  // The host chooses the grid so that all rows of a team begin at the same place of a vector: dweight's terms stay with their columns.
  const int shift = shift_of<T, kForm>(static_cast<const T*>(a.dx) + (first + team) * a.cols);
  const auto col_of = [&](int j) { return (j * a.lanes + lane) * kEl - shift; };
  Own<T, kForm> own[kVecs];
  bool have[kVecs];
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    have[j] = col_of(j) < cols;
    own[j].set(col_of(j), cols);
  }
  if (threadIdx.x < 32) {
#pragma unroll
    for (int r = 0; r < kRows; ++r) buf[0][r][threadIdx.x] = buf[1][r][threadIdx.x] = 0.0f;
  }
  __syncthreads();
  const int tensors = a.dh != nullptr ? 3 : 2;
  const uint32_t slot = blockDim.x * 16, tensor_bytes = kPieces * slot, row_bytes = tensors * tensor_bytes;
  const uint32_t mine = smem_u32(ring) + threadIdx.x * 16;
  const auto fetch = [&](int64_t begin, int batch) {
    if constexpr (kRing) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t row = begin + i * step;
        if (row < a.rows) {
          const uint32_t r = static_cast<uint32_t>(row);
          const T* from[3] = {static_cast<const T*>(a.dy) + a.dy_strides.offset(r), static_cast<const T*>(a.h) + a.h_strides.offset(r),
                              static_cast<const T*>(a.dh) + (tensors == 3 ? a.dh_strides.offset(r) : 0)};
          const uint32_t to = mine + (batch * kRows + i) * row_bytes;
#pragma unroll
          for (int t = 0; t < 3; ++t) {
            if (t == 2 && tensors == 2) break;
#pragma unroll
            for (int j = 0; j < kVecs; ++j) {
              if (!have[j]) continue;
#pragma unroll
              for (int q = 0; q < kPieces / kVecs; ++q) {
                copy_16(to + t * tensor_bytes + (j * (kPieces / kVecs) + q) * slot, from[t] + col_of(j) + q * (16 / static_cast<int>(sizeof(T))));
              }
            }
          }
        }
      }
      copies_end();
    }
  };
  const auto take = [&](const T* direct, uint32_t at, int j) {
    rows::Raw<T, kEl> r;
    if constexpr (kRing) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
      for (int q = 0; q < kPieces / kVecs; ++q) {
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[4 * q]), "=r"(w[4 * q + 1]), "=r"(w[4 * q + 2]), "=r"(w[4 * q + 3])
                     : "r"(at + (j * (kPieces / kVecs) + q) * slot) : "memory");
      }
      if constexpr (kForm == Form::kShifted) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] &= own[j].w[i];
      }
    } else {
      r = load_cols<T, kForm>(direct + col_of(j), own[j]);
    }
    return r;
  };
  pdl_wait();
  Numbers<kEl> acc[kVecs], f[kVecs];
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) acc[j].p[i] = make_float2(0.0f, 0.0f);
    if (have[j]) load_factors<T, kForm>(a.weight, a.weight_f32, a.offset, col_of(j), cols, &f[j]);
  }
  const float over = 1.0f / static_cast<float>(a.cols);
  const int64_t turn_rows = kRows * step;
  for (int s = 0; s < a.batches; ++s) fetch(first + team + s * turn_rows, s);
  const auto rstd_of = [&](int64_t row) { return row < a.rows ? ld_f32_dependent(a.rstd + row) : 0.0f; };
  float next_rstd[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) next_rstd[i] = rstd_of(first + team + i * step);
  int batch = 0;
  for (int turn = 0; first < a.rows; first += turn_rows, turn ^= 1) {
    float rstd[kRows], sum[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      rstd[i] = next_rstd[i];
      next_rstd[i] = rstd_of(first + team + turn_rows + i * step);
    }
    if constexpr (kRing) copies_wait(a.batches - 1);
    const uint32_t from = mine + batch * kRows * row_bytes;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t row = first + team + i * step;
      float2 sums = make_float2(0.0f, 0.0f);
      if (row < a.rows) {
        const T* dy_row = kRing ? nullptr : static_cast<const T*>(a.dy) + a.dy_strides.offset(static_cast<uint32_t>(row));
        const T* h_row = kRing ? nullptr : static_cast<const T*>(a.h) + a.h_strides.offset(static_cast<uint32_t>(row));
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
          if (!have[j]) continue;
          const Numbers<kEl> dy = numbers_of(take(dy_row, from + i * row_bytes, j)), h = numbers_of(take(h_row, from + i * row_bytes + tensor_bytes, j));
#pragma unroll
          for (int q = 0; q < kPairs; ++q) {
            const float2 u = mul_x2(h.p[q], rows::both(rstd[i]));
            sums = fma_x2(mul_x2(dy.p[q], f[j].p[q]), u, sums);
            acc[j].p[q] = fma_x2(dy.p[q], u, acc[j].p[q]);
          }
        }
      }
      sum[i] = sums.x + sums.y;
    }
    team_sums(sum, a.lanes, buf[turn]);
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t row = first + team + i * step;
      if (row >= a.rows) continue;
      // dh + rstd * (g - u * along); the row is read again, from where it stands: in registers it would be a block of the SM less
      const float2 of_g = rows::both(rstd[i]), of_h = rows::both(-rstd[i] * rstd[i] * (sum[i] * over));
      const uint32_t r = static_cast<uint32_t>(row);
      const T* dy_row = kRing ? nullptr : static_cast<const T*>(a.dy) + a.dy_strides.offset(r);
      const T* h_row = kRing ? nullptr : static_cast<const T*>(a.h) + a.h_strides.offset(r);
      const T* dh_row = kRing || tensors == 2 ? nullptr : static_cast<const T*>(a.dh) + a.dh_strides.offset(r);
#pragma unroll
      for (int j = 0; j < kVecs; ++j) {
        if (!have[j]) continue;
        const Numbers<kEl> dy = numbers_of(take(dy_row, from + i * row_bytes, j)), h = numbers_of(take(h_row, from + i * row_bytes + tensor_bytes, j));
        Numbers<kEl> out;
        if (tensors == 3) {
          out = numbers_of(take(dh_row, from + i * row_bytes + 2 * tensor_bytes, j));
        } else {
#pragma unroll
          for (int q = 0; q < kPairs; ++q) out.p[q] = make_float2(0.0f, 0.0f);
        }
#pragma unroll
        for (int q = 0; q < kPairs; ++q) out.p[q] = fma_x2(mul_x2(dy.p[q], f[j].p[q]), of_g, fma_x2(h.p[q], of_h, out.p[q]));
        store_cols<T, kForm>(static_cast<T*>(a.dx) + row * a.cols, col_of(j), cols, raw_of<T>(out));
      }
    }
    fetch(first + team + a.batches * turn_rows, batch);
    batch = batch + 1 == a.batches ? 0 : batch + 1;
  }
  if constexpr (kRing) copies_wait(0);
  if (a.partials == nullptr) return;
  float* to = a.partials + static_cast<int64_t>(blockIdx.x) * a.cols;
  float* sums = reinterpret_cast<float*>(ring);
  if (teams > 1) __syncthreads();  // the ring is done with
  float* own_sums = teams == 1 ? to : sums + team * a.cols;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    const int c = col_of(j);
#pragma unroll
    for (int i = 0; i < kEl; ++i) {
      if (have[j] && (kForm != Form::kShifted || (c + i >= 0 && c + i < cols))) own_sums[c + i] = i % 2 == 0 ? acc[j].p[i / 2].x : acc[j].p[i / 2].y;
    }
  }
  if (teams == 1) return;
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
    Numbers<1> f;
    load_factors<T, Form::kSingle>(a.weight, a.weight_f32, a.offset, static_cast<int>(c), static_cast<int>(a.cols), &f);
    along = fmaf(rows::to_float(dy[c]) * f.p[0].x, rows::to_float(h[c]) * rstd, along);
  }
  along = team_sum(along, 1024, buf) / static_cast<float>(a.cols);
#pragma unroll 4
  for (int64_t c = threadIdx.x; c < a.cols; c += 1024) {
    Numbers<1> f;
    load_factors<T, Form::kSingle>(a.weight, a.weight_f32, a.offset, static_cast<int>(c), static_cast<int>(a.cols), &f);
    const float u = rows::to_float(h[c]) * rstd, old = dh == nullptr ? 0.0f : rows::to_float(dh[c]);
    static_cast<T*>(a.dx)[static_cast<int64_t>(row) * a.cols + c] = rows::from_float<T>(fmaf(rstd, fmaf(-u, along, rows::to_float(dy[c]) * f.p[0].x), old));
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

// The blocks' sums of a column, in order: 32 threads above one another take every 32nd, then they are added.
template <typename P>
__global__ void __launch_bounds__(1024) rms_norm_add_kernel(const float* partials, int blocks, int64_t cols, P* out) {
  __shared__ float buf[32][33];
  pdl_launch_dependents();
  pdl_wait();
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + x;
  float sum = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int b = y; b < blocks; b += 32) sum += ld_f32_dependent(partials + b * cols + c);
  }
  buf[y][x] = sum;
  __syncthreads();
  sum = rows::warp_sum(buf[x][y]);  // column y of the block's 32
  const int64_t own = static_cast<int64_t>(blockIdx.x) * 32 + y;
  if (x == 0 && own < cols) out[own] = rows::from_float<P>(sum);
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

// How the rows of all tensors lie; `out` is contiguous.
Form form_of(int dtype, int64_t rows, int64_t cols, int widest, const void* weight, const void* out, std::initializer_list<Rows> tensors) {
  const int size = size_of(dtype);
  const auto at = [](const void* p) { return reinterpret_cast<uintptr_t>(p); };
  for (int bytes = widest; bytes >= 16; bytes /= 2) {
    bool ok = cols * size % bytes == 0 && at(out) % bytes == 0 && at(weight) % 16 == 0;
    for (const Rows& t : tensors) {
      ok = ok && (t.base == nullptr || (at(t.base) % bytes == 0 && t.outer_stride * size % bytes == 0 && t.inner_stride * size % bytes == 0));
    }
    if (ok) return bytes == 32 ? Form::k32 : Form::k16;
  }
  bool alike = true;
  for (const Rows& t : tensors) {
    if (t.base == nullptr) continue;
    alike = alike && (at(t.base) - at(out)) % 16 == 0 && (t.inner_stride - cols) * size % 16 == 0 &&
            (t.inner >= rows || (t.outer_stride - t.inner * cols) * size % 16 == 0);
  }
  return alike ? Form::kShifted : Form::kSingle;
}

int elements_of(int size, Form form) { return form == Form::k32 ? 32 / size : form == Form::kSingle ? 1 : 16 / size; }

// Lanes of a team, 0 for rows that no block holds.
int lanes_of(int size, Form form, int64_t cols, int vecs, int least, int most) {
  const int el = elements_of(size, form);
  const int64_t lanes = ceil_div(ceil_div(cols + (form == Form::kShifted ? el - 1 : 0), el), vecs);
  if (lanes > most) return 0;
  if (lanes > 32) return static_cast<int>(round_up(lanes, 32));
  int pow2 = least;
  while (pow2 < lanes) pow2 *= 2;
  return pow2;
}

DividedRows strides_of(const Rows& r, int64_t rows) {
  const uint32_t d = static_cast<uint32_t>(r.inner < rows ? r.inner : rows);
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return {r.outer_stride, r.inner_stride, d, static_cast<uint32_t>((((1ull << l) - d) << 32) / d + 1), l};
}
bool rows_ok(const Rows& r, int64_t rows) { return r.inner > 0 && (r.inner >= rows || rows % r.inner == 0); }

template <typename T>
int launch_forward(const RmsArgs& args, Form form, cudaStream_t s) {
  RmsArgs a = args;
  const int64_t rows = a.codes != nullptr ? round_up(a.rows, 128) : a.rows;
  // four blocks of scales are a word: a team has the lanes that write one at least
  a.lanes = lanes_of(sizeof(T), form, a.cols, forward_vecs(form), a.codes != nullptr ? 128 * static_cast<int>(sizeof(T)) / 32 : 1, kMostLanes);
  if (a.lanes == 0) {
    CK_CUDA(launch_pdl(rms_norm_wide_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(1024), 0, s, a));
    return CK_OK;
  }
  const int threads = a.lanes > 32 ? a.lanes : 128;
  const dim3 grid(static_cast<unsigned>(ceil_div(rows, threads / a.lanes))), block(threads);
  if (a.codes != nullptr) {
    CK_CUDA(launch_pdl(rms_norm_kernel<T, Form::k32, true>, grid, block, 0, s, a));
    return CK_OK;
  }
  switch (form) {
    case Form::k32: CK_CUDA(launch_pdl(rms_norm_kernel<T, Form::k32, false>, grid, block, 0, s, a)); break;
    case Form::k16: CK_CUDA(launch_pdl(rms_norm_kernel<T, Form::k16, false>, grid, block, 0, s, a)); break;
    case Form::kShifted: CK_CUDA(launch_pdl(rms_norm_kernel<T, Form::kShifted, false>, grid, block, 0, s, a)); break;
    default: CK_CUDA(launch_pdl(rms_norm_kernel<T, Form::kSingle, false>, grid, block, 0, s, a));
  }
  return CK_OK;
}

// How a backward pass runs: vectors and lanes of a team, and the blocks that share the rows and so dweight's partial sums.
struct BackwardPlan {
  int vecs, lanes, threads, blocks;
  int64_t chunk;  // rows that no block holds: rows of a chunk
};
constexpr int kMostBackwardLanes = 512, kMostBlocksPerSm = 8, kRingBytes = 216 * 1024;
BackwardPlan backward_plan(int size, Form form, int64_t rows, int64_t cols) {
  BackwardPlan p = {};
  // the fewest vectors with which a block holds the row: 32 numbers a lane at most
  for (p.vecs = form == Form::kSingle ? 8 : 2; p.vecs <= (form == Form::kSingle || size == 4 ? 8 : 4); p.vecs *= 2) {
    p.lanes = lanes_of(size, form, cols, p.vecs, 1, kMostBackwardLanes);
    if (p.lanes != 0) break;
  }
  if (p.lanes == 0) {
    const int64_t strips = ceil_div(cols, 256);
    int64_t chunks = ceil_div(4 * sm_count(), strips);
    if (chunks > rows) chunks = rows;
    p.chunk = ceil_div(rows, chunks);
    p.blocks = static_cast<int>(ceil_div(rows, p.chunk));
    return p;
  }
  p.threads = p.lanes > 32 ? p.lanes : 128;
  return p;
}

// The most partial sums of a column that any form of these rows has: what a call needs does not depend on addresses.
int64_t most_backward_blocks(int dtype, int64_t rows, int64_t cols) {
  const BackwardPlan widest = backward_plan(size_of(dtype), Form::k16, rows, cols);
  if (widest.lanes == 0) return widest.blocks;  // then no form has a block that holds a row
  const int64_t most = static_cast<int64_t>(kMostBlocksPerSm) * sm_count(), least = 8;  // the period of rows that lie alike
  return rows < least ? least : rows < most ? rows : most;
}

template <typename T, Form kForm, int kVecs, int kThreads, int kRows>
int launch_backward_as(RmsBackwardArgs a, BackwardPlan* p, cudaStream_t s) {
  auto kernel = rms_norm_backward_kernel<T, kForm, kVecs, kThreads, kRows>;
  const int teams = p->threads / p->lanes;
  // 512 threads of an SM, who share its memory out: as many batches as there is room for
  const int per_sm = 512 / p->threads < kMostBlocksPerSm ? 512 / p->threads : kMostBlocksPerSm;
  size_t smem = 0;
  a.batches = 1;
  if (kForm != Form::kSingle) {
    const int batch = kRows * p->threads * kVecs * elements<T, kForm>() * static_cast<int>(sizeof(T)) * (a.dh != nullptr ? 3 : 2);
    a.batches = kRingBytes / per_sm / batch;
    a.batches = a.batches < 1 ? 1 : a.batches > kMostBatches ? kMostBatches : a.batches;
    smem = static_cast<size_t>(a.batches) * batch;
  }
  if (teams > 1 && a.partials != nullptr && smem < teams * a.cols * 4) smem = teams * a.cols * 4;
  static std::atomic<bool> configured[64];
  int dev = 0;
  CK_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    CK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes));
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  int64_t blocks = static_cast<int64_t>(per_sm) * sm_count();
  if (blocks > ceil_div(a.rows, teams)) blocks = ceil_div(a.rows, teams);
  if (kForm == Form::kShifted) {
    // all rows of a team begin at the same place of a vector: the rows between two of its own are a multiple of eight (four)
    constexpr int kPeriod = 16 / static_cast<int>(sizeof(T));
    const int64_t blocks_of_period = kPeriod / (teams < kPeriod ? teams : kPeriod);  // teams are a power of two
    blocks = blocks >= blocks_of_period ? blocks / blocks_of_period * blocks_of_period : blocks_of_period;
  }
  p->blocks = static_cast<int>(blocks);
  CK_CUDA(launch_pdl(kernel, dim3(p->blocks), dim3(p->threads), smem, s, a));
  return CK_OK;
}

template <typename T, Form kForm, int kVecs>
int launch_backward_vecs(const RmsBackwardArgs& a, BackwardPlan* p, cudaStream_t s) {
  // two rows at a time where two batches of them fit: 32 bytes a lane and tensor
  constexpr int kRows = kForm != Form::kSingle && kVecs * elements<T, kForm>() * sizeof(T) <= 32 ? 2 : 1;
  return p->threads <= 256 ? launch_backward_as<T, kForm, kVecs, 256, kRows>(a, p, s) : launch_backward_as<T, kForm, kVecs, 512, kRows>(a, p, s);
}

template <typename T, Form kForm>
int launch_backward_form(const RmsBackwardArgs& a, BackwardPlan* p, cudaStream_t s) {
  if constexpr (sizeof(T) == 4) {
    if (p->vecs == 8) return launch_backward_vecs<T, kForm, 8>(a, p, s);
  }
  return p->vecs == 2 ? launch_backward_vecs<T, kForm, 2>(a, p, s) : launch_backward_vecs<T, kForm, 4>(a, p, s);
}

template <typename T>
int launch_backward(RmsBackwardArgs a, BackwardPlan* p, Form form, cudaStream_t s) {
  a.lanes = p->lanes;
  if (p->lanes == 0) {
    CK_CUDA(launch_pdl(rms_norm_backward_wide_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, s, a));
    if (a.partials == nullptr) return CK_OK;
    CK_CUDA(launch_pdl(rms_norm_columns_kernel<T>, dim3(static_cast<unsigned>(ceil_div(a.cols, 256)), p->blocks), dim3(256), 0, s, a, p->chunk));
    return CK_OK;
  }
  switch (form) {
    case Form::kShifted: return launch_backward_form<T, Form::kShifted>(a, p, s);
    case Form::kSingle: return launch_backward_vecs<T, Form::kSingle, 8>(a, p, s);
    default: return launch_backward_form<T, Form::k16>(a, p, s);
  }
}

template <typename P>
int launch_add(const float* partials, int blocks, int64_t cols, void* out, cudaStream_t s) {
  CK_CUDA(launch_pdl(rms_norm_add_kernel<P>, dim3(static_cast<unsigned>(ceil_div(cols, 32))), dim3(1024), 0, s, partials, blocks, cols, static_cast<P*>(out)));
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
  a.x_strides = strides_of(xr, rows);
  if (residual != nullptr) a.r_strides = strides_of(rr, rows);
  a.eps = eps;
  a.offset = weight == nullptr ? 0.0f : weight_offset;
  a.weight_f32 = param_dtype == CK_DTYPE_F32;
  const Form form = form_of(dtype, rows, cols, 32, weight, y != nullptr ? y : x, {xr, rr, Rows{h, rows, 0, cols}});
  if (codes != nullptr) {
    CK_REQUIRE(cols % 32 == 0 && form == Form::k32 && reinterpret_cast<uintptr_t>(codes) % 32 == 0 && reinterpret_cast<uintptr_t>(block_scales) % 4 == 0,
               "%s: MXFP8 results need columns of a multiple of 32, rows and codes on 32-byte boundaries, the weight on 16-byte ones", op);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case CK_DTYPE_BF16: return launch_forward<__nv_bfloat16>(a, form, s);
    case CK_DTYPE_F16: return launch_forward<__half>(a, form, s);
    default: return launch_forward<float>(a, form, s);
  }
}

extern "C" int64_t ck_rms_norm_backward_workspace_bytes(int dtype, int64_t rows, int64_t cols) {
  if (ck::check_rms("rms_norm_backward", dtype, CK_DTYPE_F32, rows, cols) != CK_OK) return 0;
  return ck::most_backward_blocks(dtype, rows, cols) * cols * 4;
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
  const Rows dhr = {dh, dh_inner, dh_outer_stride, dh_inner_stride};
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
  a.dy_strides = strides_of(dyr, rows);
  a.h_strides = strides_of(hr, rows);
  if (dh != nullptr) a.dh_strides = strides_of(dhr, rows);
  a.offset = weight == nullptr ? 0.0f : weight_offset;
  a.weight_f32 = param_dtype == CK_DTYPE_F32;
  const Form form = form_of(dtype, rows, cols, 16, weight, dx, {dyr, hr, dhr});
  BackwardPlan p = backward_plan(size_of(dtype), form, rows, cols);
  if (dweight != nullptr) {
    CK_REQUIRE(workspace != nullptr && workspace_bytes >= ck_rms_norm_backward_workspace_bytes(dtype, rows, cols) && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "%s: workspace of %lld bytes, %lld needed", op, (long long)workspace_bytes, (long long)ck_rms_norm_backward_workspace_bytes(dtype, rows, cols));
    a.partials = static_cast<float*>(workspace);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int rc;
  switch (dtype) {
    case CK_DTYPE_BF16: rc = launch_backward<__nv_bfloat16>(a, &p, form, s); break;
    case CK_DTYPE_F16: rc = launch_backward<__half>(a, &p, form, s); break;
    default: rc = launch_backward<float>(a, &p, form, s);
  }
  if (rc != CK_OK || dweight == nullptr) return rc;
  switch (param_dtype) {
    case CK_DTYPE_BF16: return launch_add<__nv_bfloat16>(a.partials, p.blocks, cols, dweight, s);
    case CK_DTYPE_F16: return launch_add<__half>(a.partials, p.blocks, cols, dweight, s);
    default: return launch_add<float>(a.partials, p.blocks, cols, dweight, s);
  }
}
