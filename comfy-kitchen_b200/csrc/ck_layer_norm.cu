// Layer norm over the last dimension for sm_100a, forward pass, optionally with an MXFP8 copy of the input (the mathematics in ck_layer_norm.cuh).
#include "ck_layer_norm.cuh"

namespace ck {
namespace {

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

// The MXFP8 copy of a row that stands in shared memory, by the `width` threads of its team: one block of 32 elements a thread at a time, so that
// its scale needs no exchange.  A block is read in 16-byte pieces, each lane starting with another one (lanes' blocks are 64 or 128 bytes
// apart, which would meet the same banks), and the codes' words are turned back.
template <typename T>
__device__ __forceinline__ void copy_row(const uint8_t* from, int thread, int width, const ForwardArgs& a, uint32_t row) {
  constexpr int kPieces = 2 * static_cast<int>(sizeof(T)), kElements = 32 / kPieces, kWords = 8 / kPieces;
  const int blocks = static_cast<int>(a.cols >> 5), blocks_padded = (blocks + 3) & ~3;
  const int turn = kPieces == 4 ? (thread >> 1) & 3 : thread & 7;
  for (int first = 0; first < blocks_padded; first += width) {
    const int block = first + thread;
    uint32_t byte = 0;
    if (block < blocks) {
      float2 u[kPieces][kElements / 2];
      float amax = 0.0f;
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const int piece = (p + turn) & (kPieces - 1);
        unpack(*reinterpret_cast<const Raw<T, kElements>*>(from + block * (32 * sizeof(T)) + piece * 16), u[p]);
#pragma unroll
        for (int j = 0; j < kElements / 2; ++j) amax = fmaxf(amax, fmaxf(fabsf(u[p][j].x), fabsf(u[p][j].y)));
      }
      const quant::Mxfp8Scale scale = block_scale(amax);
      byte = scale.byte;
      uint32_t words[kPieces][kWords];
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
#pragma unroll
        for (int j = 0; j < kWords; ++j) words[p][j] = block_codes(u[p][2 * j], u[p][2 * j + 1], scale);
      }
#pragma unroll
      for (int bit = 1; bit < kPieces; bit *= 2) {  // by `turn` places
        uint32_t moved[kPieces][kWords];
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
#pragma unroll
          for (int j = 0; j < kWords; ++j) moved[p][j] = (turn & bit) != 0 ? words[(p - bit) & (kPieces - 1)][j] : words[p][j];
        }
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
#pragma unroll
          for (int j = 0; j < kWords; ++j) words[p][j] = moved[p][j];
        }
      }
      Vec256 out;
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
#pragma unroll
        for (int j = 0; j < kWords; ++j) out.w[p * kWords + j] = words[p][j];
      }
      st_global_256(a.codes + static_cast<int64_t>(row) * a.cols + block * 32, out);
    }
    uint32_t word = byte | (__shfl_xor_sync(0xFFFFFFFFu, byte, 1) << 8);
    word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2) << 16;
    if (block < blocks_padded && (block & 3) == 0) {
      *reinterpret_cast<uint32_t*>(a.scales + swizzled_scale_offset(row, block, blocks_padded >> 2)) = word;
    }
  }
}

// Many rows.  A team of blockDim.x threads takes a row at a time out of its ring; the block's rows are of one group, whose factors f and biases stand
// in shared memory as fp32.  A row is unpacked once and stays in registers as fp32, up to 96 columns a thread: waiting, sums over
// lanes and the meeting of a team's warps cost the same for few columns as for many.  36864 x 3072 bf16, a warp a row: 92 us
// (4.9 TB/s) against 109 with four warps a row; with the copy 113 against 155.  Mean and variance take one meeting: each warp brings the mean of what it holds and the squares about that.
// kExact: the columns fill all threads.
template <typename T, int kVec, int kNum, bool kCopy, bool kExact>
__global__ void __launch_bounds__(kVec * kNum <= 16 ? 1024 : 512) layer_norm_forward_ring_kernel(const ForwardArgs a, const uint32_t chunks, const uint32_t chunk_rows,
                                                                      const int stages) {
  constexpr int kPairs = kVec / 2;
  extern __shared__ __align__(128) uint8_t shared_bytes[];  // factors, biases, the teams' rings
  __shared__ __align__(8) uint64_t full[32][kMaxRing];
  __shared__ float2 buf[2][16];   // [turn][warp of the block]: mean and squares, where a team is several warps
  __shared__ float counts[16];    // elements that a team's warp holds
  __shared__ int abort_flag;
  pdl_launch_dependents();
  const int team = threadIdx.y, teams = blockDim.y, width = blockDim.x, warps = width >> 5, warp = threadIdx.x >> 5;
  const uint32_t group = blockIdx.x / chunks, chunk = blockIdx.x - group * chunks;
  const uint32_t begin = chunk * chunk_rows, end = min(a.rows_per_group, begin + chunk_rows), row0 = group * a.rows_per_group;
  const int vecs = static_cast<int>(a.cols / kVec);
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const uint32_t row_bytes = static_cast<uint32_t>(a.cols) * sizeof(T), stage_bytes = (row_bytes + 127) & ~127u;
  const uint32_t param_bytes = (static_cast<uint32_t>(a.cols) * 4 + 127) & ~127u;
  float* const factor_buf = reinterpret_cast<float*>(shared_bytes);
  float* const bias_buf = reinterpret_cast<float*>(shared_bytes + param_bytes);
  const uint8_t* const ring = shared_bytes + 2 * param_bytes + team * stages * stage_bytes;
  const uint32_t ring_at = sm100::smem_u32(ring), full_at = sm100::smem_u32(full[team]);
  const auto load_row = [&](uint32_t r, int s) {  // by one thread of the team
    sm100::mbar_arrive_expect_tx(full_at + s * 8, row_bytes);
    sm100::bulk_load_1d(ring_at + s * stage_bytes, static_cast<const T*>(a.x) + a.x_rows.offset(row0 + r), row_bytes, full_at + s * 8);
  };
  const auto has = [&](int i) { return kExact || static_cast<int>(threadIdx.x) + i * width < vecs; };
  int held = 32 * kNum * kVec;
  if constexpr (!kExact) {
    held = 0;
#pragma unroll
    for (int i = 0; i < kNum; ++i) held += max(0, min(32, vecs - warp * 32 - i * width)) * kVec;
  }
  const float count = static_cast<float>(held), inv_held = held > 0 ? 1.0f / count : 0.0f;
  if (team == 0 && (threadIdx.x & 31) == 0) counts[warp] = count;
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
  for (int v = team * width + threadIdx.x; v < vecs; v += width * teams) {
    float f[kVec], b[kVec];
    if (a.weight != nullptr) load_param<T, kVec>(a.weight, group * a.weight_stride + static_cast<int64_t>(v) * kVec, a.params_f32, a.params_aligned, f);
    if (a.bias != nullptr) load_param<T, kVec>(a.bias, group * a.bias_stride + static_cast<int64_t>(v) * kVec, a.params_f32, a.params_aligned, b);
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      factor_buf[j / kPart * part_stride + v * kPart + j % kPart] = a.weight != nullptr ? a.offset + f[j] : 1.0f;
      bias_buf[j / kPart * part_stride + v * kPart + j % kPart] = a.bias != nullptr ? b[j] : 0.0f;
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
  bool landed = true;  // after a wait that gave up the team still meets for each row, with no more copies, and the result is void
  for (uint32_t r = begin + team; r < end; r += teams, turn ^= 1) {
    landed = sm100::mbar_wait(full_at + stage * 8, phase, &abort_flag) && landed;
    const uint8_t* const from = ring + stage * stage_bytes;
    const uint32_t row = row0 + r;
    if constexpr (kCopy) copy_row<T>(from, threadIdx.x, width, a, row);
    float2 f[kNum][kPairs];
    float2 sum[2] = {both(0.0f), both(0.0f)};
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      if (has(i)) {
        unpack(*reinterpret_cast<const Raw<T, kVec>*>(from + (threadIdx.x + i * width) * 16), f[i]);
      } else {
#pragma unroll
        for (int j = 0; j < kPairs; ++j) f[i][j] = both(0.0f);
      }
#pragma unroll
      for (int j = 0; j < kPairs; ++j) sum[j & 1] = add_x2(sum[j & 1], f[i][j]);
    }
    sum[0] = add_x2(sum[0], sum[1]);
    const float mine = mean_of(warp_sum(sum[0].x + sum[0].y), count, inv_held);
    float2 square[2] = {both(0.0f), both(0.0f)};
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const float2 minus = both(has(i) ? -mine : 0.0f);  // zeros where there is nothing
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const float2 d = add_x2(f[i][j], minus);
        square[j & 1] = fma_x2(d, d, square[j & 1]);
        if constexpr (kCopy) f[i][j] = d;
      }
    }
    square[0] = add_x2(square[0], square[1]);
    float mean = mine, squares = warp_sum(square[0].x + square[0].y);
    if (warps > 1) {
      float2* const slots = buf[turn] + team * warps;
      if ((threadIdx.x & 31) == 0) slots[warp] = make_float2(mine, squares);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(width) : "memory");
      const Moments all = join_moments(slots, counts, warps, static_cast<float>(a.cols), inv_cols);
      mean = all.mean;
      squares = all.squares;
    } else {
      __syncwarp();
    }
    const float rstd = inverse_root(squares * inv_cols + a.eps);
    if (threadIdx.x == 0) {
      if (landed && r + stages * teams < end) load_row(r + stages * teams, stage);  // all have read the stage
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
    // h = (x - mean) / std, the difference first: a product of x and 1 / std would leave its rounding in the result where eps and not the deviation bounds
    // 1 / std.  Or, in one step, from x - mine and what the warp's mean is off, a few deviations at most: beside a copy, where it takes 58.8 us
    // instead of 60.2 (18432 x 3072 bf16); without one 14.1 instead of 13.5 (4096 x 3072).
    const float2 scale = both(rstd), shift = both(kCopy ? (mine - mean) * rstd : -mean);
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      if (!has(i)) continue;
      const int v = threadIdx.x + i * width;
      float2 w[kPairs], b[kPairs];
      read_params(factor_buf, v, w);
      read_params(bias_buf, v, b);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const float2 h = kCopy ? fma_x2(f[i][j], scale, shift) : mul_x2(add_x2(f[i][j], shift), scale);
        f[i][j] = fma_x2(h, w[j], b[j]);
      }
      store(y + static_cast<int64_t>(v) * kVec, pack<T, kVec>(f[i]));
    }
  }
  if constexpr (kCopy) {  // the scales' padding rows
    for (uint32_t row = a.rows + blockIdx.x * teams + team; row < a.rows_padded; row += gridDim.x * teams) clear_scales_of_row(a, row);
  }
  if (!landed) {
    if ((threadIdx.x & 31) == 0) atomicExch(a.status, 1);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
  }
}

// The same for rows that do not lie on 16-byte boundaries (Columns and RowInRing in ck_layer_norm.cuh), without a copy.  36864 x 3071 fp16: 140 us
// against 455 for rows in registers without a ring, an element a load either way.
template <typename T, int kVec, int kNum>
__global__ void __launch_bounds__(512) layer_norm_forward_off_vectors_kernel(const ForwardArgs a, const uint32_t chunks, const uint32_t chunk_rows,
                                                                             const int stages) {
  using Cols = Columns<T, kVec>;
  using Row = RowInRing<T>;
  extern __shared__ __align__(128) uint8_t shared_bytes[];  // factors, biases, the teams' rings
  __shared__ __align__(8) uint64_t full[16][kMaxRing];
  __shared__ float2 buf[2][16];  // [turn][warp of the block]: mean and squares
  __shared__ float counts[16];   // elements that a team's warp holds
  __shared__ int abort_flag;
  pdl_launch_dependents();
  const int team = threadIdx.y, teams = blockDim.y, width = blockDim.x, warps = width >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t group = blockIdx.x / chunks, chunk = blockIdx.x - group * chunks;
  const uint32_t begin = chunk * chunk_rows, end = min(a.rows_per_group, begin + chunk_rows), row0 = group * a.rows_per_group;
  const Cols own = {static_cast<int>(threadIdx.x), width, static_cast<int>(a.cols)};
  const Row in = {static_cast<uint32_t>(a.cols) * static_cast<uint32_t>(sizeof(T))};
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const uint32_t stage_bytes = static_cast<uint32_t>(Row::stage_bytes(in.bytes)), param_bytes = (static_cast<uint32_t>(a.cols) * 4 + 127) & ~127u;
  float* const factor_buf = reinterpret_cast<float*>(shared_bytes);
  float* const bias_buf = reinterpret_cast<float*>(shared_bytes + param_bytes);
  uint8_t* const ring = shared_bytes + 2 * param_bytes + team * stages * stage_bytes;
  const uint32_t ring_at = sm100::smem_u32(ring), full_at = sm100::smem_u32(full[team]);
  const auto row_of = [&](uint32_t r) { return static_cast<const T*>(a.x) + a.x_rows.offset(row0 + r); };
  const auto load_row = [&](uint32_t r, int s) {  // by one thread of the team
    const T* const row = row_of(r);
    sm100::mbar_arrive_expect_tx(full_at + s * 8, in.bulk_bytes(row));
    in.fetch(row, ring_at + s * stage_bytes, full_at + s * 8);
  };
  // sixteen lanes of a team's first warp bring what lies beside the copy
  const auto put_edge = [&](const T* row, int s, uint32_t e, T v) { Row::put(ring + s * stage_bytes, row, e, v); };
  float held = 0.0f;
#pragma unroll
  for (int i = 0; i < kNum; ++i) held += (own.has(i) ? 1.0f : 0.0f) + (own.has(i, 1) ? 1.0f : 0.0f);
  held = warp_sum(held);
  const float inv_held = held > 0.0f ? 1.0f / held : 0.0f;
  if (team == 0 && lane == 0) counts[warp] = held;
  if (threadIdx.x == 0) {
    if (team == 0) abort_flag = 0;
    for (int s = 0; s < stages; ++s) sm100::mbar_init(&full[team][s], 1);
    sm100::fence_barrier_init();
  }
  pdl_wait();
  if (warp == 0) {
    __syncwarp();
    for (int s = 0; s < stages; ++s) {
      const uint32_t r = begin + team + s * teams;
      if (r >= end) break;
      if (lane == 0) load_row(r, s);
      const T* const row = row_of(r);
      uint32_t e;
      if (lane < 16 && in.edge(row, lane, &e)) put_edge(row, s, e, row[e]);
    }
  }
  for (int c = team * width + threadIdx.x; c < own.cols; c += width * teams) {
    factor_buf[c] = a.weight != nullptr ? a.offset + param<T>(a.weight, group * a.weight_stride + c, a.params_f32) : 1.0f;
    bias_buf[c] = a.bias != nullptr ? param<T>(a.bias, group * a.bias_stride + c, a.params_f32) : 0.0f;
  }
  __syncthreads();
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  bool landed = true;  // after a wait that gave up the team still meets for each row, with no more copies, and the result is void
  for (uint32_t r = begin + team; r < end; r += teams, turn ^= 1) {
    const uint32_t next = r + stages * teams;  // the row that comes into this one's stage
    T edge = from_float<T>(0.0f);
    uint32_t edge_at = 0;
    bool has_edge = false;
    if (warp == 0 && lane < 16 && next < end) {
      const T* const row = row_of(next);
      has_edge = in.edge(row, lane, &edge_at);
      if (has_edge) edge = row[edge_at];
    }
    landed = sm100::mbar_wait(full_at + stage * 8, phase, &abort_flag) && landed;
    const uint8_t* const from = ring + stage * stage_bytes + Row::offset(row_of(r));
    float2 f[kNum];
    float2 sum[2] = {both(0.0f), both(0.0f)};
    Cols at = own.again();
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      float2 v[1];
      at.read(from, i, v);  // zeros past the row's end
      f[i] = v[0];
      sum[i & 1] = add_x2(sum[i & 1], f[i]);
    }
    sum[0] = add_x2(sum[0], sum[1]);
    const float mine = mean_of(warp_sum(sum[0].x + sum[0].y), held, inv_held);
    float2 square[2] = {both(0.0f), both(0.0f)};
    at = own.again();
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const float2 d = add_x2(f[i], make_float2(at.has(i) ? -mine : 0.0f, at.has(i, 1) ? -mine : 0.0f));
      square[i & 1] = fma_x2(d, d, square[i & 1]);
    }
    square[0] = add_x2(square[0], square[1]);
    float mean = mine, squares = warp_sum(square[0].x + square[0].y);
    if (warps > 1) {
      float2* const slots = buf[turn] + team * warps;
      if (lane == 0) slots[warp] = make_float2(mine, squares);
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(width) : "memory");
      const Moments all = join_moments(slots, counts, warps, static_cast<float>(a.cols), inv_cols);
      mean = all.mean;
      squares = all.squares;
    } else {
      __syncwarp();
    }
    const float rstd = inverse_root(squares * inv_cols + a.eps);
    const uint32_t row = row0 + r;
    if (threadIdx.x == 0) {
      if (landed && next < end) load_row(next, stage);  // all have read the stage
      if (a.mean != nullptr) {
        a.mean[row] = mean;
        a.rstd[row] = rstd;
      }
    }
    if (has_edge) put_edge(row_of(next), stage, edge_at, edge);  // read behind the team's next meeting
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
    T* const y = static_cast<T*>(a.y) + static_cast<int64_t>(row) * a.cols;
    at = own.again();
    const float2 scale = both(rstd), shift = both(-mean);  // as in the kernel for whole vectors
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      if (!at.has(i)) continue;
      float2 v[1] = {mul_x2(add_x2(f[i], shift), scale)};
      float2 w[1], b[1];
      at.shared_params(factor_buf, i, w);
      at.shared_params(bias_buf, i, b);
      v[0] = fma_x2(v[0], w[0], b[0]);
      at.write(y, i, v);
    }
  }
  if (!landed) {
    if ((threadIdx.x & 31) == 0) atomicExch(a.status, 1);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
  }
}

// Rows of any width and alignment, which do not stay in registers: a block goes over its row three times, the second and third out of L1.
template <typename T, int kVec>
__global__ void __launch_bounds__(512) layer_norm_forward_wide_kernel(const ForwardArgs a) {
  __shared__ float buf[64];
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + a.x_rows.offset(row);
  float sum = 0.0f;
#pragma unroll 4
  for (int64_t k = kVec * threadIdx.x; k < a.cols; k += kVec * blockDim.x) {
    float f[kVec];
    unpack(*reinterpret_cast<const Raw<T, kVec>*>(x + k), f);
#pragma unroll
    for (int i = 0; i < kVec; ++i) sum += f[i];
  }
  const float mean = row_sum<0>(sum, buf) / static_cast<float>(a.cols);
  float square = 0.0f;
#pragma unroll 4
  for (int64_t k = kVec * threadIdx.x; k < a.cols; k += kVec * blockDim.x) {
    float f[kVec];
    unpack(*reinterpret_cast<const Raw<T, kVec>*>(x + k), f);
#pragma unroll
    for (int i = 0; i < kVec; ++i) square = fmaf(f[i] - mean, f[i] - mean, square);
  }
  const float rstd = inverse_root(row_sum<1>(square, buf) / static_cast<float>(a.cols) + a.eps);
  if (threadIdx.x == 0 && a.mean != nullptr) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
  const int64_t group = row / a.rows_per_group;
  T* y = static_cast<T*>(a.y) + static_cast<int64_t>(row) * a.cols;
#pragma unroll 4
  for (int64_t k = kVec * threadIdx.x; k < a.cols; k += kVec * blockDim.x) {
    float f[kVec], w[kVec], b[kVec];
    unpack(*reinterpret_cast<const Raw<T, kVec>*>(x + k), f);
    if (a.weight != nullptr) load_param<T, kVec>(a.weight, group * a.weight_stride + k, a.params_f32, a.params_aligned, w);
    if (a.bias != nullptr) load_param<T, kVec>(a.bias, group * a.bias_stride + k, a.params_f32, a.params_aligned, b);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      f[i] = fmaf((f[i] - mean) * rstd, a.weight != nullptr ? a.offset + w[i] : 1.0f, a.bias != nullptr ? b[i] : 0.0f);
    }
    store(y + k, pack<T, kVec>(f));
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <typename T, int kVec, int kNum, bool kCopy>
int launch_forward_num(const ForwardArgs& a, int warps, cudaStream_t s) {
  const int threads = warps * 32, rows_of_block = warps >= 8 ? 1 : 8 / warps;
  const dim3 grid(static_cast<unsigned>(ceil_div(kCopy ? a.rows_padded : a.rows, rows_of_block))), block(threads, rows_of_block);
  auto kernel = warps <= 8 ? layer_norm_forward_kernel<T, kVec, kNum, kCopy, 256> : layer_norm_forward_kernel<T, kVec, kNum, kCopy, 1024>;
  CK_CUDA(launch_pdl(kernel, grid, block, 0, s, a));
  return CK_OK;
}

struct RingPlan {
  int warps, teams, stages;  // of a row; of a block; of a team's ring
  int smem;                  // 0: no room
};

// A block of up to 16 warps an SM, or of 32 with a short row each.  A row's warps: as few as hold it, and as many more as the rows leave idle: those that
// fit into the ring, or those that an SM gets.
RingPlan plan_ring(int64_t rows, int64_t cols, int64_t size, bool whole) {
  const int64_t stage = round_up(cols * size + (whole ? 0 : 15), 128), params = 2 * round_up(cols * 4, 128), columns = 16 / size * 32;
  RingPlan p = {};
  p.warps = static_cast<int>(ceil_div(cols, 32 * 96));
  if (p.warps > 16 || params + 2 * stage > kRingRoom) return p;
  int64_t teams = cols <= 512 && whole ? 32 : 16 / p.warps;
  if (teams > (kRingRoom - params) / (2 * stage)) teams = (kRingRoom - params) / (2 * stage);
  if (teams > ceil_div(rows, sm_count())) teams = ceil_div(rows, sm_count());
  int64_t warps = teams > 16 ? 1 : 16 / teams;
  if (warps > ceil_div(cols, columns)) warps = ceil_div(cols, columns);
  if (warps > p.warps) p.warps = static_cast<int>(warps);
  p.teams = static_cast<int>(teams);
  const int64_t stages = (kRingRoom - params) / (teams * stage);
  p.stages = static_cast<int>(stages > kMaxRing ? kMaxRing : stages);
  p.smem = static_cast<int>(params + teams * p.stages * stage);
  return p;
}

template <auto kKernel>
int launch_ring(ForwardArgs a, const RingPlan& p, cudaStream_t s) {
  // one block an SM, and no block with less than a row for each team
  const int64_t groups = a.rows / a.rows_per_group;
  int64_t chunks = sm_count() / groups;
  if (chunks > ceil_div(a.rows_per_group, p.teams)) chunks = ceil_div(a.rows_per_group, p.teams);
  if (chunks < 1) chunks = 1;
  const uint32_t chunk_rows = static_cast<uint32_t>(ceil_div(a.rows_per_group, chunks));
  chunks = ceil_div(a.rows_per_group, chunk_rows);
  if (int rc = allow_ring_room<kKernel>()) return rc;
  if (int rc = gemm_status_word(&a.status)) return rc;
  CK_CUDA(launch_pdl(kKernel, dim3(static_cast<unsigned>(groups * chunks)), dim3(32 * p.warps, p.teams), p.smem, s, a, static_cast<uint32_t>(chunks),
                     chunk_rows, p.stages));
  return CK_OK;
}

template <typename T, int kVec, int kNum, bool kCopy>
int launch_forward_ring_num(const ForwardArgs& a, const RingPlan& p, cudaStream_t s) {
  if (a.cols == int64_t{32} * p.warps * kNum * kVec) return launch_ring<layer_norm_forward_ring_kernel<T, kVec, kNum, kCopy, true>>(a, p, s);
  return launch_ring<layer_norm_forward_ring_kernel<T, kVec, kNum, kCopy, false>>(a, p, s);
}

template <typename T, int kVec, bool kCopy>
int launch_forward_ring(const ForwardArgs& a, const RingPlan& p, cudaStream_t s) {
  constexpr int kUnit = 8 / kVec;
  const int64_t num = ceil_div(a.cols, 32 * p.warps * 8);  // eights of columns
  if (num <= 2 && p.warps == 1) return launch_forward_ring_num<T, kVec, 2 * kUnit, kCopy>(a, p, s);
  if (num <= 4) return launch_forward_ring_num<T, kVec, 4 * kUnit, kCopy>(a, p, s);
  if (num <= 8) return launch_forward_ring_num<T, kVec, 8 * kUnit, kCopy>(a, p, s);
  return launch_forward_ring_num<T, kVec, 12 * kUnit, kCopy>(a, p, s);
}

// Warps of a row: as few as hold it, eight vectors a lane (no barrier crosses a warp then, and a lane has its loads in flight
// together); where the rows alone do not fill the chip, as many as leave one vector a lane, up to 32.
template <typename T, int kVec, bool kCopy>
int launch_forward(const ForwardArgs& a, cudaStream_t s) {
  const int64_t vecs = ceil_div(a.cols, kVec);
  CK_REQUIRE(vecs <= 32 * 32 * 8, "layer_norm_forward: a copy of rows of %lld is not supported", (long long)a.cols);
  if constexpr (kVec * sizeof(T) == 16) {
    // (30000 x 256 bf16 with a copy, which gives eight lanes of a warp work: 18.6 us against 15.0; without one 10.6 against 12.1)
    if (a.rows > 2 * sm_count() && a.rows_per_group >= 16 && reinterpret_cast<uintptr_t>(a.codes) % 32 == 0 && (!kCopy || a.cols > 256)) {
      const RingPlan p = plan_ring(a.rows, a.cols, sizeof(T), true);
      if (p.smem > 0 && a.rows / a.rows_per_group <= 2 * sm_count()) return launch_forward_ring<T, kVec, kCopy>(a, p, s);
    }
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
  // x, y and the parameters lie on the boundaries of n elements
  const auto rows_on = [&](int n) {
    return a.cols % n == 0 && on_bytes(a.x, a.x_rows, sizeof(T), n * sizeof(T)) && reinterpret_cast<uintptr_t>(a.y) % (n * sizeof(T)) == 0;
  };
  const auto params_on = [&](int bytes) {
    const auto on = [&](const void* p, int64_t stride) {
      return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * param_size % bytes == 0);
    };
    return on(a.weight, a.weight_stride) && on(a.bias, a.bias_stride);
  };
  const bool vectors = rows_on(kVec), pairs = rows_on(2);
  a.params_aligned = params_on(vectors ? 16 : 2 * param_size);
  if (a.codes != nullptr) {
    CK_REQUIRE(vectors, "layer_norm_forward: rows with a copy have to start on 16-byte boundaries");
    return launch_forward<T, kVec, true>(a, s);
  }
  if (vectors && a.cols <= int64_t{32} * 32 * 8 * kVec) return launch_forward<T, kVec, false>(a, s);
  if (!vectors) {
    if (a.rows > 2 * sm_count() && a.rows_per_group >= 16 && a.cols > 384 && a.rows / a.rows_per_group <= 2 * sm_count()) {
      const RingPlan p = plan_ring(a.rows, a.cols, sizeof(T), false);
      if (p.smem > 0) {
        const auto by_num = [&](auto vec) {
          constexpr int kV = decltype(vec)::value;
          const int64_t num = ceil_div(a.cols, 64 * p.warps);  // pairs
          if (num <= 16) return launch_ring<layer_norm_forward_off_vectors_kernel<T, kV, 16>>(a, p, s);
          if (num <= 32) return launch_ring<layer_norm_forward_off_vectors_kernel<T, kV, 32>>(a, p, s);
          return launch_ring<layer_norm_forward_off_vectors_kernel<T, kV, 48>>(a, p, s);
        };
        return pairs ? by_num(std::integral_constant<int, 2>()) : by_num(std::integral_constant<int, 1>());
      }
    }
    if (pairs && a.cols <= 2 * 32 * 32 * 8) return launch_forward<T, 2, false>(a, s);
    if (a.cols <= 32 * 32 * 8) return launch_forward<T, 1, false>(a, s);
  }
  auto kernel = vectors ? layer_norm_forward_wide_kernel<T, kVec> : pairs ? layer_norm_forward_wide_kernel<T, 2> : layer_norm_forward_wide_kernel<T, 1>;
  const int64_t vecs = a.cols / (vectors ? kVec : pairs ? 2 : 1);
  const unsigned threads = vecs >= 512 ? 512 : static_cast<unsigned>(round_up(vecs, 32));
  CK_CUDA(launch_pdl(kernel, dim3(a.rows), dim3(threads), 0, s, a));
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

