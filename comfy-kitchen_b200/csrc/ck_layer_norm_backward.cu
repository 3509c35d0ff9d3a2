// Layer norm over the last dimension for sm_100a, backward pass, from the input or from its MXFP8 copy (the mathematics in ck_layer_norm.cuh).
#include "ck_layer_norm.cuh"

namespace ck {
namespace {

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

// Short rows, a warp each.  It takes kRows of them at a time, every lane the same columns of all: a row's two sums go over the lanes, and the
// column sums for dw and db stay in registers until the block's rows are done.  Then the warps' sums are added in a fixed order and
// written: as results where the block has all rows of its group, else as partial sums that a second kernel adds.
template <typename T, int kVec, int kNum, int kRows, bool kCopy>
__global__ void __launch_bounds__(512) layer_norm_backward_kernel(const BackwardArgs a) {
  const int width = blockDim.x;  // 32; given as a constant the compiler has fewer loads in flight (20000 x 320 fp32 from the copy: 25.5 us against 22.0)
  extern __shared__ __align__(16) float shared_buf[];  // first the factors f, later the warps' column sums
  pdl_launch_dependents();
  const int team = threadIdx.y, teams = blockDim.y;
  const uint32_t group = blockIdx.x / a.chunks, chunk = blockIdx.x - group * a.chunks;
  const uint32_t begin = chunk * a.chunk_rows, end = min(a.rows_per_group, begin + a.chunk_rows);
  const int64_t vecs = a.cols / kVec;
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  pdl_wait();
  // The factors as fp32 in shared memory, all warps': in registers they would be a third of what a thread holds.  Four of a vector lie
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
  for (uint32_t r0 = begin + team * kRows; r0 < end; r0 += teams * kRows) {
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
  // the warps' column sums
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
// bulk copies into its own ring, a few rows ahead, and what a thread holds of a row is read from there once.  Bound by HBM, and by the instructions
// that a row costs each warp whatever its columns: 256 threads with 48 columns of 255 registers instead of 512 with 24 took 36864 x 3072 bf16
// from 125 us to 112, from the copy from 143 to 110.  As they stand: 111 (6.1 TB/s) and 102 (5.6 TB/s).
template <typename T, int kVec, int kNum, int kThreads, bool kCopy, bool kExact>
__global__ void __launch_bounds__(kThreads) layer_norm_backward_ring_kernel(const BackwardArgs a, const int stages) {
  constexpr int kMaxTeams = 15, kPairs = kVec / 2;
  // g stays in registers for the second pass.  Or dy, and the factors are read again, where a thread holds 48 columns (but for a copy of 16-bit rows):
  // there the compiler's order of reads is worth more (36864 x 3072 bf16: 111 us against 118; 4096 x 12288 fp32 from the copy 86 against 95;
  // 36864 x 3072 bf16 from the copy 102 against 109 the other way round)
  constexpr bool kAgain = kNum * kVec == 48 && !(kCopy && sizeof(T) == 2);
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
  const uint32_t factor_bytes = (static_cast<uint32_t>(a.cols) * 4 + 127) & ~127u;
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
  const auto has = [&](int i) { return kExact || static_cast<int>(threadIdx.x) + i * width < vecs; };
  const auto vec_of = [&](int i) { return kExact ? static_cast<int>(threadIdx.x) + i * width : min(static_cast<int>(threadIdx.x) + i * width, vecs - 1); };
  // factors in shared memory, as above
  constexpr int kPart = 4;
  const int part_stride = vecs * kPart;
  for (int v = team * width + threadIdx.x; v < vecs; v += width * teams) {
    float f[kVec];
    if (a.weight != nullptr) load_param<T, kVec>(a.weight, group * a.weight_stride + static_cast<int64_t>(v) * kVec, a.params_f32, a.params_aligned, f);
#pragma unroll
    for (int j = 0; j < kVec; ++j) shared_buf[j / kPart * part_stride + v * kPart + j % kPart] = a.weight != nullptr ? a.offset + f[j] : 1.0f;
  }
  __syncthreads();
  const auto factors = [&](int i, float2(&f)[kPairs]) {
    const int v = vec_of(i);
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
  const uint8_t* scale_at[kNum];  // in row 0
  if constexpr (kCopy) {
#pragma unroll
    for (int i = 0; i < kNum; ++i) scale_at[i] = a.scales + swizzled_scale_offset(0, vec_of(i) * kVec >> 5, quads);
  }
  const auto beside = [&](uint32_t r) {
    if (r >= end) return;
    next_mean = a.mean[row0 + r];
    next_rstd = a.rstd[row0 + r];
    if constexpr (kCopy) {
      const int64_t row_at = swizzled_scale_offset(row0 + r, 0, quads);
#pragma unroll
      for (int i = 0; i < kNum; ++i) next_byte[i] = scale_at[i][row_at];
    }
  };
  beside(begin + team);
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  bool landed = true;  // after a wait that gave up the team still meets for each row, with no more copies, and the result is void
  for (uint32_t r = begin + team; r < end; r += teams, turn ^= 1) {
    const float mean = next_mean, rstd = next_rstd;
    float factor[kNum];
#pragma unroll
    for (int i = 0; i < kNum; ++i) factor[i] = e8m0_factor(next_byte[i]);
    beside(r + teams);
    landed = sm100::mbar_wait(full_at + stage * 8, phase, &abort_flag) && landed;
    const uint8_t* const from = ring + stage * stage_bytes;
    // unpacked once: g (or dy) and h stay in registers for the second pass
    float2 d[kNum][kPairs], h[kNum][kPairs];
    const float2 rstd2 = both(rstd), minus = both(-mean);
    float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const int v = vec_of(i);
      Raw<T, kVec> raw = *reinterpret_cast<const Raw<T, kVec>*>(from + v * 16);
      if (!has(i)) raw = zeros<T, kVec>();  // past the row's end: dy = 0, whatever h
      unpack(raw, d[i]);
      if constexpr (kCopy) {
        const auto codes = *reinterpret_cast<const Raw<uint32_t, kVec / 4>*>(from + x_at + v * kVec);
#pragma unroll
        for (int j = 0; j < kVec / 4; ++j) {
          h[i][2 * j] = fma_x2(e4m3_pair(codes.v[j] & 0xFFFFu), both(factor[i]), minus);
          h[i][2 * j + 1] = fma_x2(e4m3_pair(codes.v[j] >> 16), both(factor[i]), minus);
        }
      } else {
        unpack(*reinterpret_cast<const Raw<T, kVec>*>(from + x_at + v * 16), h[i]);
      }
      float2 f[kPairs];
      factors(i, f);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        h[i][j] = mul_x2(kCopy ? h[i][j] : add_x2(h[i][j], minus), rstd2);
        dw[i][j] = fma_x2(d[i][j], h[i][j], dw[i][j]);
        db[i][j] = add_x2(db[i][j], d[i][j]);
        const float2 g = mul_x2(d[i][j], f[j]);
        s1 = add_x2(s1, g);
        s2 = fma_x2(g, h[i][j], s2);
        if constexpr (!kAgain) d[i][j] = g;
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
    if (threadIdx.x == 0 && landed && r + stages * teams < end) load_row(r + stages * teams, stage);  // all have read the stage
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
    T* const dx = static_cast<T*>(a.dx) + static_cast<int64_t>(row0 + r) * a.cols;
    const float2 c1r = both(-c1 * rstd), c2r = both(-c2 * rstd);
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      const int v = threadIdx.x + i * width;
      if (has(i)) {
        float2 f[kPairs];
        if constexpr (kAgain) factors(i, f);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          d[i][j] = kAgain ? mul_x2(fma_x2(h[i][j], both(-c2), fma_x2(d[i][j], f[j], both(-c1))), rstd2) : fma_x2(h[i][j], c2r, fma_x2(d[i][j], rstd2, c1r));
        }
        store(dx + v * kVec, pack<T, kVec>(d[i]));
      }
    }
  }
  if (!landed && (threadIdx.x & 31) == 0) atomicExch(a.status, 1);
  __syncthreads();  // the ring is the column sums' now
  if (abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
    return;
  }
  if (a.dweight == nullptr && a.dbias == nullptr) return;
  // The teams' sums of all columns side by side in shared memory, then four columns a thread, added in the teams' order.
  const int threads = width * teams, at = team * width + threadIdx.x, cols = static_cast<int>(a.cols);
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
    if (!has(i)) continue;
    float* const to = shared_buf + team * cols + (threadIdx.x + i * width) * kVec;
#pragma unroll
    for (int j = 0; j < kPairs; j += 2) {
      *reinterpret_cast<float4*>(to + 2 * j) = make_float4(dw[i][j].x, dw[i][j].y, dw[i][j + 1].x, dw[i][j + 1].y);
      *reinterpret_cast<float4*>(to + teams * cols + 2 * j) = make_float4(db[i][j].x, db[i][j].y, db[i][j + 1].x, db[i][j + 1].y);
    }
  }
  __syncthreads();
  for (int which = 0; which < 2; ++which) {
    void* const result = which == 0 ? a.dweight : a.dbias;
#pragma unroll 2
    for (int k = 4 * at; k < cols; k += 4 * threads) {
      float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int t = 0; t < teams; ++t) {
        const float4 f = *reinterpret_cast<const float4*>(shared_buf + (which * teams + t) * cols + k);
        s.x += f.x;
        s.y += f.y;
        s.z += f.z;
        s.w += f.w;
      }
      if (a.partials != nullptr) {
        *reinterpret_cast<float4*>(a.partials + (static_cast<int64_t>(blockIdx.x) * 2 + which) * cols + k) = s;
      } else if (result != nullptr) {
        store_param<T>(result, group * a.cols + k, a.params_f32, s.x);
        store_param<T>(result, group * a.cols + k + 1, a.params_f32, s.y);
        store_param<T>(result, group * a.cols + k + 2, a.params_f32, s.z);
        store_param<T>(result, group * a.cols + k + 3, a.params_f32, s.w);
      }
    }
  }
}

// The same for rows that do not lie on 16-byte boundaries (Columns and RowInRing in ck_layer_norm.cuh): 36864 x 3071 fp16 228 us, against 677 for
// 24 columns a thread whose places the compiler kept in registers over all rows.
template <typename T, int kVec, int kNum, int kThreads>
__global__ void __launch_bounds__(kThreads) layer_norm_backward_off_vectors_kernel(const BackwardArgs a, const int stages) {
  using Cols = Columns<T, kVec>;
  using Row = RowInRing<T>;
  constexpr int kMaxTeams = 15, kPairs = Cols::kPairs, kTurn = Cols::kTurn;
  extern __shared__ __align__(128) uint8_t shared_bytes[];  // factors f, then the teams' rings; the teams' column sums in the end
  __shared__ __align__(8) uint64_t full[kMaxTeams][kMaxRing];
  __shared__ float2 row_buf[2][16];  // [turn][warp of the block]
  __shared__ int abort_flag;
  pdl_launch_dependents();
  const int team = threadIdx.y, teams = blockDim.y, width = blockDim.x, warps = width >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t group = blockIdx.x / a.chunks, chunk = blockIdx.x - group * a.chunks;
  const uint32_t begin = chunk * a.chunk_rows, end = min(a.rows_per_group, begin + a.chunk_rows), row0 = group * a.rows_per_group;
  const Cols own = {static_cast<int>(threadIdx.x), width, static_cast<int>(a.cols)};
  const Row in = {static_cast<uint32_t>(a.cols) * static_cast<uint32_t>(sizeof(T))};
  const float inv_cols = 1.0f / static_cast<float>(a.cols);
  const uint32_t dy_stage = static_cast<uint32_t>(Row::stage_bytes(in.bytes)), stage_bytes = 2 * dy_stage;
  const uint32_t factor_bytes = a.weight != nullptr ? (static_cast<uint32_t>(a.cols) * 4 + 127) & ~127u : 0u;
  float* const shared_buf = reinterpret_cast<float*>(shared_bytes);
  uint8_t* const ring = shared_bytes + factor_bytes + team * stages * stage_bytes;
  const uint32_t ring_at = sm100::smem_u32(ring), full_at = sm100::smem_u32(full[team]);
  const auto dy_row = [&](uint32_t r) { return static_cast<const T*>(a.dy) + a.dy_rows.offset(row0 + r); };
  const auto x_row = [&](uint32_t r) { return static_cast<const T*>(a.x) + a.x_rows.offset(row0 + r); };
  const auto load_row = [&](uint32_t r, int s) {  // by one thread of the team
    const uint32_t to = ring_at + s * stage_bytes, bar = full_at + s * 8;
    const T* const dy = dy_row(r);
    const T* const x = x_row(r);
    sm100::mbar_arrive_expect_tx(bar, in.bulk_bytes(dy) + in.bulk_bytes(x));
    in.fetch(dy, to, bar);
    in.fetch(x, to + dy_stage, bar);
  };
  // Sixteen lanes of a team's first warp bring what lies beside the copies of a row of dy, the others that of x.
  const auto edge_row = [&](uint32_t r) { return lane < 16 ? dy_row(r) : x_row(r); };
  const auto put_edge = [&](const T* row, int s, uint32_t at, T v) { Row::put(ring + s * stage_bytes + (lane < 16 ? 0u : dy_stage), row, at, v); };
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
      const T* const row = edge_row(r);
      uint32_t at;
      if (in.edge(row, lane & 15, &at)) put_edge(row, s, at, row[at]);
    }
  }
  if (a.weight != nullptr) {
    own.share(shared_buf, a.weight, group * a.weight_stride, a.params_f32, a.offset, team * width + threadIdx.x, width * teams);
  }
  __syncthreads();
  Cols at = own;
  const auto factors = [&](int i, float2(&f)[kPairs]) {
    if (a.weight != nullptr) {
      at.shared_params(shared_buf, i, f);
    } else {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) f[j] = both(1.0f);
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
  const auto beside = [&](uint32_t r) {
    if (r >= end) return;
    next_mean = a.mean[row0 + r];
    next_rstd = a.rstd[row0 + r];
  };
  beside(begin + team);
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  bool landed = true;  // after a wait that gave up the team still meets for each row, with no more copies, and the result is void
  for (uint32_t r = begin + team; r < end; r += teams, turn ^= 1) {
    const float mean = next_mean, rstd = next_rstd;
    beside(r + teams);
    const uint32_t next = r + stages * teams;  // the row that comes into this one's stage
    T edge = from_float<T>(0.0f);
    uint32_t edge_at = 0;
    bool has_edge = false;
    if (warp == 0 && next < end) {
      const T* const row = edge_row(next);
      has_edge = in.edge(row, lane & 15, &edge_at);
      if (has_edge) edge = row[edge_at];
    }
    landed = sm100::mbar_wait(full_at + stage * 8, phase, &abort_flag) && landed;
    const uint8_t* const from = ring + stage * stage_bytes;
    const uint8_t* const dy_from = from + Row::offset(dy_row(r));
    const uint8_t* const x_from = from + dy_stage + Row::offset(x_row(r));
    // unpacked once: g and h stay in registers for the second pass
    float2 d[kNum][kPairs], h[kNum][kPairs];
    const float2 rstd2 = both(rstd), minus = both(-mean);
    float2 s1 = both(0.0f), s2 = both(0.0f);
    at = own.again();
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      at.read(dy_from, i, d[i]);  // past the row's end: dy = 0, and h something finite
      at.read(x_from, i, h[i]);
      float2 f[kPairs];
      factors(i, f);
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        h[i][j] = mul_x2(add_x2(h[i][j], minus), rstd2);
        dw[i][j] = fma_x2(d[i][j], h[i][j], dw[i][j]);
        db[i][j] = add_x2(db[i][j], d[i][j]);
        d[i][j] = mul_x2(d[i][j], f[j]);  // g from here on
        s1 = add_x2(s1, d[i][j]);
        s2 = fma_x2(d[i][j], h[i][j], s2);
      }
    }
    // both sums in five exchanges: the lower half of a warp goes on with one, the upper with the other
    float sum = (lane < 16 ? s1.x + s1.y : s2.x + s2.y) + __shfl_xor_sync(0xFFFFFFFFu, lane < 16 ? s2.x + s2.y : s1.x + s1.y, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    float c1, c2;
    if (warps > 1) {  // the team's warps meet; two buffers in turn, so that one meeting a row is enough
      float2* const slots = row_buf[turn] + team * warps;
      if ((lane & 15) == 0) reinterpret_cast<float*>(slots + warp)[lane >> 4] = sum;
      asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(width) : "memory");
      float2 all = both(0.0f);
      for (int w = 0; w < warps; ++w) all = add_x2(all, slots[w]);
      c1 = all.x * inv_cols;
      c2 = all.y * inv_cols;
    } else {
      c1 = __shfl_sync(0xFFFFFFFFu, sum, 0) * inv_cols;
      c2 = __shfl_sync(0xFFFFFFFFu, sum, 16) * inv_cols;
      __syncwarp();
    }
    if (threadIdx.x == 0 && landed && next < end) load_row(next, stage);  // all have read the stage
    if (has_edge) put_edge(edge_row(next), stage, edge_at, edge);  // read behind the team's next meeting
    if (++stage == stages) {
      stage = 0;
      phase ^= 1u;
    }
    T* const dx = static_cast<T*>(a.dx) + static_cast<int64_t>(row0 + r) * a.cols;
    const float2 c1r = both(-c1 * rstd), c2r = both(-c2 * rstd);
    at = own.again();
#pragma unroll
    for (int i = 0; i < kNum; ++i) {
      if (!at.has(i)) continue;
#pragma unroll
      for (int j = 0; j < kPairs; ++j) d[i][j] = fma_x2(h[i][j], c2r, fma_x2(d[i][j], rstd2, c1r));
      at.write(dx, i, d[i]);
    }
  }
  if (!landed && (threadIdx.x & 31) == 0) atomicExch(a.status, 1);
  __syncthreads();  // the ring is the column sums' now
  if (abort_flag) {
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
    return;
  }
  if (a.dweight == nullptr && a.dbias == nullptr) return;
  const int threads = width * teams, place = team * width + threadIdx.x, cols = own.cols;  // as in the kernel for whole vectors
  at = own.again();
#pragma unroll
  for (int i = 0; i < kNum; ++i) {
#pragma unroll
    for (int e = 0; e < kTurn; ++e) {
      if (!at.has(i, e)) continue;
      float* const to = shared_buf + team * cols + at.column(i, e);
      to[0] = e == 0 ? dw[i][0].x : dw[i][0].y;
      to[teams * cols] = e == 0 ? db[i][0].x : db[i][0].y;
    }
  }
  __syncthreads();
  for (int which = 0; which < 2; ++which) {
    void* const result = which == 0 ? a.dweight : a.dbias;
#pragma unroll 4
    for (int k = place; k < cols; k += threads) {
      float s = 0.0f;
      for (int t = 0; t < teams; ++t) s += shared_buf[(which * teams + t) * cols + k];
      if (a.partials != nullptr) {
        a.partials[(static_cast<int64_t>(blockIdx.x) * 2 + which) * cols + k] = s;
      } else if (result != nullptr) {
        store_param<T>(result, group * a.cols + k, a.params_f32, s);
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
  const uint32_t part = blockIdx.y, group = part / a.chunks, chunk = part - group * a.chunks;
  const uint32_t begin = chunk * a.chunk_rows, end = min(a.rows_per_group, begin + a.chunk_rows);
  const int64_t k = static_cast<int64_t>(blockIdx.x) * 32 + threadIdx.x;
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
      a.partials[(static_cast<int64_t>(part) * 2 + threadIdx.y) * a.cols + k] = s;
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

// size: of an element; vec: elements that lie together, of which rows are made (whole vectors of 16 bytes, pairs or one); weight: whether there is one.
Plan plan_backward(int64_t cols, int size, int vec, bool copy, bool weight, int64_t groups, int64_t rows_per_group) {
  Plan p = {};
  const bool whole = vec * size == 16;
  const int turn = vec == 1 ? 2 : vec, unit = 8 / turn;  // turns of eight columns
  p.ring = cols >= (whole ? 512 : 129) && !(copy && !whole);
  p.wide = p.ring ? cols > (whole && size == 2 ? 512 * 32 : 256 * 48) : copy && !whole;
  int64_t step = 64;
  int most = 8;
  if (!p.wide) {
    if (p.ring) {
      // 24 columns a thread of 512, beyond that 48 a thread of 256; whole 16-bit vectors of the widest rows 32 of 512
      p.warps = whole && cols > 256 * 48 ? 16 : static_cast<int>(ceil_div(cols, 32 * 48));
      if (cols <= 32 * 24 || p.warps > 8) most = 16;
      const int64_t eights = ceil_div(cols, 32 * 8 * p.warps);
      if (whole) {
        p.num = static_cast<int>(eights <= 2 ? 2 : eights <= 4 ? eights : 6) * unit;  // as there are kernels
      } else {
        p.num = eights <= 1 ? 4 : eights <= 3 ? 12 : 24;  // pairs
      }
    } else {
      const int64_t vecs = ceil_div(cols, whole ? vec : 1);
      p.warps = 1;
      p.num = static_cast<int>(ceil_div(vecs, 32));
    }
    if (!p.ring) most = 16;
    p.teams = most / p.warps;
    if (p.teams > 15) p.teams = 15;  // named barriers 1 to 15
    p.rows = !p.ring && p.num <= 2 ? 2 : 1;
    step = static_cast<int64_t>(p.teams) * p.rows;
    const int64_t sums = p.ring ? 2 * p.teams * cols * 4 : 2 * (whole ? vec : 2) * 32 * p.warps * p.teams * 4;
    const int64_t factors = weight || (p.ring && whole) ? round_up(cols * 4, 128) : 0;
    if (p.ring) {
      const int64_t dy_stage = round_up(cols * size + (whole ? 0 : 15), 128), stage = dy_stage + (copy ? round_up(cols, 128) : dy_stage);
      while (p.teams > 1 && factors + 2 * p.teams * stage > kRingRoom) --p.teams;
      const int64_t stages = (kRingRoom - factors) / (p.teams * stage);
      p.stages = static_cast<int>(stages > kMaxRing ? kMaxRing : stages);
      p.wide = p.stages < (whole ? 1 : 2);
      p.smem = static_cast<int>(factors + p.teams * p.stages * stage);
      if (sums > p.smem) p.smem = static_cast<int>(sums);
      step = p.teams;
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
  // 480 threads' column sums at most: 30 KB, which needs no leave
  CK_CUDA(launch_pdl(layer_norm_backward_kernel<T, kVec, kNum, kRows, kCopy>, dim3(a.groups * a.chunks), dim3(32, p.teams), p.smem, s, a));
  return CK_OK;
}

template <auto kKernel>
int launch_rows_in_ring(BackwardArgs a, const Plan& p, cudaStream_t s) {
  if (int rc = allow_ring_room<kKernel>()) return rc;
  if (int rc = gemm_status_word(&a.status)) return rc;
  CK_CUDA(launch_pdl(kKernel, dim3(a.groups * a.chunks), dim3(32 * p.warps, p.teams), p.smem, s, a, p.stages));
  return CK_OK;
}

template <typename T, int kVec, int kNum, int kThreads, bool kCopy>
int launch_backward_ring(const BackwardArgs& a, const Plan& p, cudaStream_t s) {
  // Where the columns fill all threads nothing is asked for each vector.  Where a thread reads 48 columns of both dy and x, asking keeps the reads of
  // later vectors behind the arithmetic of earlier ones, which is worth more (36864 x 3072 bf16: 111 us against 114; from the copy 113 against
  // 102); 32 columns of each of 512 threads leave no registers for either.
  constexpr bool kCanFill = kNum * kVec <= 24 || (kThreads == 256 && (kCopy || kNum * kVec <= 32));
  if constexpr (kCanFill) {
    if (a.cols == int64_t{32} * p.warps * kNum * kVec) return launch_rows_in_ring<layer_norm_backward_ring_kernel<T, kVec, kNum, kThreads, kCopy, true>>(a, p, s);
  }
  return launch_rows_in_ring<layer_norm_backward_ring_kernel<T, kVec, kNum, kThreads, kCopy, false>>(a, p, s);
}

template <typename T, int kVec, int kNum, int kThreads>
int launch_backward_off_vectors(const BackwardArgs& a, const Plan& p, cudaStream_t s) {
  return launch_rows_in_ring<layer_norm_backward_off_vectors_kernel<T, kVec, kNum, kThreads>>(a, p, s);
}

template <typename T, int kVec, bool kCopy>
int launch_backward(const BackwardArgs& a, const Plan& p, cudaStream_t s) {
  constexpr bool kWhole = kVec * sizeof(T) == 16;
  constexpr int kUnit = kVec == 1 ? 4 : 8 / kVec;  // turns of eight columns
  if (p.ring) {
    if constexpr (!kWhole) {
      if (p.num == 4) return launch_backward_off_vectors<T, kVec, 4, 512>(a, p, s);
      if (p.num == 12) return launch_backward_off_vectors<T, kVec, 12, 512>(a, p, s);
      return launch_backward_off_vectors<T, kVec, 24, 256>(a, p, s);
    } else {
      if (p.num == 2 * kUnit) return launch_backward_ring<T, kVec, 2 * kUnit, 512, kCopy>(a, p, s);
      if (p.num == 3 * kUnit) return launch_backward_ring<T, kVec, 3 * kUnit, 512, kCopy>(a, p, s);
      if constexpr (sizeof(T) == 2) {
        if (p.warps > 8) return launch_backward_ring<T, kVec, 4 * kUnit, 512, kCopy>(a, p, s);
      }
      if (p.num == 4 * kUnit) return launch_backward_ring<T, kVec, 4 * kUnit, 256, kCopy>(a, p, s);
      return launch_backward_ring<T, kVec, 6 * kUnit, 256, kCopy>(a, p, s);
    }
  }
  if constexpr (kWhole) {  // fewer than 512 columns
    if (p.num == 1) return launch_backward_num<T, kVec, 1, 2, kCopy>(a, p, s);
    if (p.num == 2) return launch_backward_num<T, kVec, 2, 2, kCopy>(a, p, s);
    if constexpr (sizeof(T) == 4) return launch_backward_num<T, kVec, 4, 1, kCopy>(a, p, s);
    return fail(CK_ERR_UNSUPPORTED, "layer_norm_backward: no kernel for %d vectors", p.num);
  } else {  // up to 128, one by one
    if (p.num == 1) return launch_backward_num<T, 1, 1, 2, false>(a, p, s);
    if (p.num == 2) return launch_backward_num<T, 1, 2, 2, false>(a, p, s);
    return launch_backward_num<T, 1, 4, 1, false>(a, p, s);
  }
}

// Elements that lie together in every tensor: 16 bytes of them, two, or one.
int backward_vec(const BackwardArgs& a, int size) {
  for (int vec = 16 / size; vec > 1; vec = vec > 2 ? 2 : 1) {
    const int bytes = vec * size;
    if (a.cols % vec == 0 && on_bytes(a.dy, a.dy_rows, size, bytes) && reinterpret_cast<uintptr_t>(a.dx) % bytes == 0 &&
        (a.x != nullptr ? on_bytes(a.x, a.x_rows, size, bytes) : reinterpret_cast<uintptr_t>(a.codes) % 16 == 0)) {
      return vec;
    }
  }
  return 1;
}

template <typename T>
int backward_typed(const BackwardArgs& given, void* workspace, int64_t workspace_bytes, cudaStream_t s) {
  BackwardArgs a = given;
  a.params_aligned = a.weight == nullptr || on_vectors(a.weight, a.weight_stride, a.params_f32 ? 4 : sizeof(T));
  const int vec = backward_vec(a, sizeof(T));
  const Plan p = plan_backward(a.cols, sizeof(T), vec, a.x == nullptr, a.weight != nullptr, a.groups, a.rows_per_group);
  a.chunks = p.chunks;
  a.chunk_rows = p.chunk_rows;
  const bool sums = a.dweight != nullptr || a.dbias != nullptr;
  const int64_t need = static_cast<int64_t>(a.groups) * p.chunks * 2 * a.cols * 4;
  if (sums && p.chunks > 1) {
    CK_REQUIRE(workspace != nullptr && workspace_bytes >= need && reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
               "layer_norm_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    a.partials = static_cast<float*>(workspace);
  }
  constexpr int kVec = kVecOf<T>;
  int rc = CK_OK;
  if (p.wide) {
    CK_CUDA(launch_pdl(layer_norm_backward_wide_kernel<T>, dim3(a.groups * a.rows_per_group), dim3(512), 0, s, a));
    if (sums) {
      // strips of columns in the dimension that has room for any width; groups are at most 32767, chunks of fewer groups than SMs as many as those
      const dim3 grid(static_cast<unsigned>(ceil_div(a.cols, 32)), a.groups * p.chunks);
      CK_CUDA(launch_pdl(layer_norm_columns_wide_kernel<T>, grid, dim3(32, 16), 0, s, a));
    }
  } else if (vec == 1) {
    rc = launch_backward<T, 1, false>(a, p, s);
  } else if (vec == 2) {
    rc = launch_backward<T, 2, false>(a, p, s);
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

}  // namespace
}  // namespace ck

extern "C" int64_t ck_layer_norm_backward_workspace_bytes(int64_t rows, int64_t cols, int64_t groups) {
  using namespace ck;
  if (rows <= 0 || cols <= 0 || groups <= 0 || rows % groups != 0) return 0;
  int64_t most = 0;  // over the forms that types and alignment decide between
  for (const int size : {2, 4}) {
    for (const int vec : {16 / size, 2, 1}) {
      for (int form = 0; form < 4; ++form) {
        const Plan p = plan_backward(cols, size, vec, (form & 1) != 0, (form & 2) != 0, groups, rows / groups);
        const int64_t need = p.chunks > 1 ? groups * p.chunks * 2 * cols * 4 : 0;
        if (need > most) most = need;
      }
    }
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
    case CK_DTYPE_BF16: return backward_typed<__nv_bfloat16>(a, workspace, workspace_bytes, s);
    case CK_DTYPE_F16: return backward_typed<__half>(a, workspace, workspace_bytes, s);
    default: return backward_typed<float>(a, workspace, workspace_bytes, s);
  }
}
