// What the forward and the backward pass of layer norm share: parameters, sums over a row's warps, a thread's columns, and rows that come through
// a ring in shared memory.
//
//   m = mean_k x,  v = mean_k (x - m)^2,  i = 1 / sqrt(v + eps),  h = (x - m) i
//   y = h f + b,   f = offset + w (1 without a weight)
//   g = dy f,      dx = i (g - mean_k g - h mean_k(g h)),   dw = sum_rows dy h,   db = sum_rows dy
//
// w and b belong to groups of consecutive rows (one group: the learned weight of a layer; one for each sample: modulation).
// Rows are taken in two levels of strides, so that a slice of the tokens of a longer buffer needs no copy.  All
// sums and statistics are fp32; a row stays in registers between its passes, so its mean is subtracted before
// squares are taken.  Results are rounded to their types once.
#pragma once

#include <atomic>

#include "ck_rows.cuh"

namespace ck {
namespace {

using namespace rows;

// ---- parameters: fp32, or of x's type
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

// ---- sums
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

// total / count with one more step than the product with 1 / count: the rounded quotient, so that a row of equal numbers whose sum is exact has that
// number for its mean.  Where eps and not the deviation bounds 1 / std (316 for 1e-5), a unit in the last place of 1000 would be 0.02 in h.
__device__ __forceinline__ float mean_of(float total, float count, float inv_count) {
  const float q = total * inv_count;
  const float better = fmaf(fmaf(-q, count, total), inv_count, q);
  return fabsf(q) < __uint_as_float(0x7F800000u) ? better : q;
}

// What a row's warps hold, joined: `slots` has each one's mean and the squares about it, `counts` its number of elements.
struct Moments {
  float mean, squares;
};
__device__ __forceinline__ Moments join_moments(const float2* slots, const float* counts, int warps, float cols, float inv_cols) {
  Moments m = {0.0f, 0.0f};
  for (int w = 0; w < warps; ++w) m.mean = fmaf(slots[w].x, counts[w], m.mean);
  m.mean = mean_of(m.mean, cols, inv_cols);
  for (int w = 0; w < warps; ++w) {
    const float d = slots[w].x - m.mean;
    m.squares += fmaf(d * d, counts[w], slots[w].y);
  }
  return m;
}

// ---- rows that come through shared memory
// A team's row is a bulk copy into a ring of stages, issued that many rows ahead by one thread, so that what is in flight
// does not depend on registers or on where the warps stand.  Barriers of the ring are mbarriers whose waits are bounded (mbar_wait).
// Two rows of each team: with four, 10000 x 1152 fp16 takes 15.4 us forward instead of 13.9, 36864 x 3072 bf16 from the copy 105 backward instead of 102.
constexpr int kMaxRing = 2;

// A row that does not lie on 16-byte boundaries is copied where it does, at the same place in its 16 bytes; what is before and behind
// (up to 15 bytes each) comes by plain loads of one element a lane, read ahead of a row's arithmetic and stored behind it.
template <typename T>
struct RowInRing {
  uint32_t bytes;  // of a row

  __host__ __device__ static constexpr int64_t stage_bytes(int64_t row_bytes) { return round_up(row_bytes + 15, 128); }

  __device__ __forceinline__ static uint32_t offset(const T* row) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15u); }
  __device__ __forceinline__ uint32_t head(const T* row) const { return min((16u - offset(row)) & 15u, bytes); }
  // what the bulk copy of a row brings
  __device__ __forceinline__ uint32_t bulk_bytes(const T* row) const { return (bytes - head(row)) & ~15u; }
  // by one thread; its bytes are expected by the barrier already
  __device__ __forceinline__ void fetch(const T* row, uint32_t stage, uint32_t bar) const {
    const uint32_t h = head(row), n = bulk_bytes(row);
    if (n > 0) sm100::bulk_load_1d(stage + offset(row) + h, reinterpret_cast<const uint8_t*>(row) + h, n, bar);
  }
  // An element beside the copy.  The bulk copy of a later row, which may lie otherwise in its 16 bytes, writes the same place through the async
  // proxy: the fence puts this store before it, for the thread that issues that copy behind the team's next meeting.
  __device__ __forceinline__ static void put(uint8_t* stage, const T* row, uint32_t at, T v) {
    reinterpret_cast<T*>(stage + offset(row))[at] = v;
    sm100::fence_proxy_async();
  }
  // element `*at` of the row is lane's (of sixteen) to bring: eight before the copy, eight behind it
  __device__ __forceinline__ bool edge(const T* row, int lane, uint32_t* at) const {
    const uint32_t h = head(row), tail = (bytes - h) & 15u, e = static_cast<uint32_t>(lane & 7) * sizeof(T);
    *at = ((lane & 8) != 0 ? bytes - tail + e : e) / sizeof(T);
    return e < ((lane & 8) != 0 ? tail : h);
  }
};

// The columns of a thread of a team that takes such rows, in turns of two columns, which are a pair of fp32 numbers in registers: beside one another
// where rows lie on the boundaries of pairs (kVec = 2), else as far apart as the team is wide.
template <typename T, int kVec>
struct Columns {
  static constexpr int kPairs = 1, kTurn = 2;

  int thread, width, cols;

  // The same, computed again: what a pass over a row knows of its columns' places and ends is not kept in registers for the next one.
  __device__ __forceinline__ Columns again() const {
    Columns c = *this;
    asm volatile("" : "+r"(c.thread), "+r"(c.width), "+r"(c.cols));
    return c;
  }

  __device__ __forceinline__ int column(int turn, int e) const { return kVec == 1 ? thread + (2 * turn + e) * width : 2 * (thread + turn * width) + e; }
  __device__ __forceinline__ bool has(int turn, int e = 0) const { return column(turn, e) < cols; }

  __device__ __forceinline__ void read(const uint8_t* row, int turn, float2 (&f)[kPairs]) const {
    const T* const at = reinterpret_cast<const T*>(row);
    if constexpr (kVec == 1) {
      const T* const p = at + column(turn, 0);
      f[0] = make_float2(has(turn) ? to_float(p[0]) : 0.0f, has(turn, 1) ? to_float(p[width]) : 0.0f);
    } else {  // no branch: a place of the row, or zeros for what was there
      unpack(*reinterpret_cast<const Raw<T, kVec>*>(at + min(column(turn, 0), cols - 2)), f);
      if (!has(turn)) f[0] = both(0.0f);
    }
  }

  __device__ __forceinline__ void write(T* row, int turn, const float2 (&f)[kPairs]) const {
    T* const p = row + column(turn, 0);
    if constexpr (kVec == 1) {
      if (has(turn)) p[0] = from_float<T>(f[0].x);
      if (has(turn, 1)) p[width] = from_float<T>(f[0].y);
    } else if (has(turn)) {
      store(p, pack<T, kVec>(f));
    }
  }

  // parameters as fp32 in shared memory, by all threads of a block
  __device__ __forceinline__ void share(float* to, const void* from, int64_t at, bool f32, float offset, int t, int threads) const {
    for (int c = t; c < cols; c += threads) to[c] = offset + param<T>(from, at + c, f32);
  }
  // a turn of them; past the row's end any that are there
  __device__ __forceinline__ void shared_params(const float* from, int turn, float2 (&f)[kPairs]) const {
    if constexpr (kVec == 2) {
      f[0] = *reinterpret_cast<const float2*>(from + min(column(turn, 0), cols - 2));
    } else {
      f[0] = make_float2(from[min(column(turn, 0), cols - 1)], from[min(column(turn, 1), cols - 1)]);
    }
  }
};

// ---- host side
template <typename T>
constexpr int kVecOf = 16 / static_cast<int>(sizeof(T));

bool on_vectors(const void* p, int64_t elements, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && elements * size % 16 == 0;
}
bool on_bytes(const void* p, const RowStrides& r, int size, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && r.outer_stride * size % bytes == 0 && r.inner_stride * size % bytes == 0;
}
bool on_vectors(const void* p, const RowStrides& r, int size) { return on_bytes(p, r, size, 16); }

constexpr int kRingRoom = 216 * 1024;  // of shared memory, for parameters and rings

// What a kernel may be launched with is state of the function on its device: one bound for all calls, set before the first of them, so that calls of
// several threads, whose plans differ, do not take it from one another.
template <auto kKernel>
int allow_ring_room() {
  static std::atomic<bool> allowed[64];
  int dev = 0;
  CK_CUDA(cudaGetDevice(&dev));
  const bool known = dev >= 0 && dev < 64;
  if (known && allowed[dev].load(std::memory_order_acquire)) return CK_OK;
  CK_CUDA(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingRoom));
  if (known) allowed[dev].store(true, std::memory_order_release);
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
