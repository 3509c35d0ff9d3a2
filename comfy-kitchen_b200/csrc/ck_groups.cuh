// Rows that are grouped by expert: group e has the rows [offsets[e - 1], offsets[e]) of a matrix (the first one from 0 on), ends that
// lie on the device.  What every kernel on such rows shares: the bounds, kept inside the matrix and from decreasing whatever the ends say (so
// no row belongs to two groups, and the tiles are never more than the rows have), and the walk over the groups' tiles, whose number only the device knows.
#pragma once

#include "ck_common.cuh"
#include "ck_rows.cuh"
#include "ck_sm100.cuh"

namespace ck {
namespace groups {

constexpr int kMaxGroups = 1024;  // 8 KiB of shared memory for the table

// A value that the kernel before this one may have written (see ld_f32_dependent).
__device__ __forceinline__ int ld_s32_dependent(const int* p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// First row behind group e, inside the matrix.
__device__ __forceinline__ int group_end(const int* offsets, int e, int rows) {
  return e < 0 ? 0 : min(max(ld_s32_dependent(offsets + e), 0), rows);
}

// Group of a row: the first whose end lies behind it, `count` if none does.  For ends that decrease it is still one whose
// begin is not behind the row.
__device__ __forceinline__ int group_of_row(const int* offsets, int count, int row) {
  int lo = 0, hi = count;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ld_s32_dependent(offsets + mid) > row) {
      hi = mid;
    } else {
      lo = mid + 1;
    }
  }
  return lo;
}

// Where the scale tiles (128 rows by 4 blocks, 512 bytes) of a group's own row blocks begin, in row blocks.  A group's first row is its
// first tile's first row, so groups share no tile: with s and t its begin and end, ceil((t - s) / 128) <= t / 128 - s / 128 + 1
// (whole quotients), which is the distance to the next group's.
__host__ __device__ __forceinline__ int64_t first_scale_block(int begin, int e) { return (begin >> 7) + e; }
__host__ __device__ __forceinline__ int64_t scale_blocks(int64_t rows, int64_t count) { return ceil_div(rows, 128) + count; }

// In shared memory: the groups' bounds, and the numbers of row tiles before each.
struct Table {
  int bound[kMaxGroups + 1];  // group e: rows [bound[e], bound[e + 1])
  int tiles[kMaxGroups + 1];  // row tiles of the groups before e
};

// Filled by all threads of the block, when the ends are there.  An end below an earlier one counts as that one.
__device__ __forceinline__ void fill_table(Table* t, const int* offsets, int count, int rows, int tile_rows) {
  for (int e = threadIdx.x; e <= count; e += blockDim.x) t->bound[e] = group_end(offsets, e - 1, rows);
  __syncthreads();
  if (threadIdx.x < 32) {
    int before = 0;
    for (int first = 0; first < count; first += 32) {
      const int e = first + static_cast<int>(threadIdx.x), from = min(e, count), to = min(e + 1, count);
      if (__any_sync(0xFFFFFFFFu, t->bound[to] < t->bound[from])) {
        if (threadIdx.x == 0) {
          for (int i = first + 1; i <= count; ++i) t->bound[i] = max(t->bound[i], t->bound[i - 1]);
        }
        __syncwarp();
      }
      const int own = (t->bound[to] - t->bound[from] + tile_rows - 1) / tile_rows;
      int sum = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xFFFFFFFFu, sum, o);
        if (static_cast<int>(threadIdx.x) >= o) sum += up;
      }
      if (e < count) t->tiles[e] = before + sum - own;
      before += __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    if (threadIdx.x == 0) t->tiles[count] = before;
  }
  __syncthreads();
}

struct Tile {
  int group;
  int row;        // its first row in the matrix
  int end;        // first row behind the group
  int index;      // row tile within the group
  int tile_n;
};

// Item -> tile.  A group's tiles follow one another, in bands of so many row tiles, down a band's rows first: the tiles that run together share
// operands in L2.
__device__ __forceinline__ Tile place(const Table* t, int count, int tiles_n, int tile_rows, int item) {
  constexpr int kBand = 8;
  int lo = 0, hi = count - 1;  // the last group with tiles[e] * tiles_n <= item
  const int before = item / tiles_n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t->tiles[mid] <= before) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  Tile p;
  p.group = lo;
  const int tiles_m = t->tiles[lo + 1] - t->tiles[lo], in_group = item - t->tiles[lo] * tiles_n;
  const int band = in_group / (kBand * tiles_n), in_band = in_group - band * kBand * tiles_n;
  const int height = min(kBand, tiles_m - band * kBand);
  p.tile_n = in_band / height;
  p.index = band * kBand + in_band - p.tile_n * height;
  p.row = t->bound[lo] + p.index * tile_rows;
  p.end = t->bound[lo + 1];
  return p;
}

// 32 x 32 numbers turned by a warp: a lane writes its feature's, one for each row, and reads 16 bytes of neighbouring features of row 32 / pieces * i + lane / pieces.
// Numbers of 16 bits lie by feature, in pieces of eight rows whose places change with the feature so that neither the writes nor the transposing reads of 8 x 8
// matrices (whose rows are the features 8 j + 2 m and 8 j + 2 m + 1, so that a lane gets eight in a row) meet a bank twice; those of 32 lie by row.
__device__ __forceinline__ uint32_t turn_place(int feature, int piece) {
  return static_cast<uint32_t>(feature * 64 + ((piece ^ (feature >> 1) ^ (feature >> 3)) & 3) * 16);
}
template <typename OutT>
__device__ __forceinline__ void turn_write(uint32_t turn, int lane, const float* v) {
  if constexpr (sizeof(OutT) == 2) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float pair[2] = {v[2 * i], v[2 * i + 1]};
      const rows::Raw<OutT, 2> r = rows::pack<OutT, 2>(pair);
      w[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) sm100::st_shared_128(turn + turn_place(lane, q), w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) asm volatile("st.shared.f32 [%0], %1;" ::"r"(turn + (i * 32 + lane) * 4), "f"(v[i]) : "memory");
  }
}
template <typename OutT>
__device__ __forceinline__ rows::Raw<OutT, 16 / static_cast<int>(sizeof(OutT))> turn_read(uint32_t turn, int lane, int i) {
  rows::Raw<OutT, 16 / static_cast<int>(sizeof(OutT))> r;
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
  if constexpr (sizeof(OutT) == 2) {
    const int feature = (lane & 7) / 2 * 8 + (lane >> 3) * 2 + (lane & 1);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(turn + turn_place(feature, i))
                 : "memory");
  } else {
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(turn + (i * 32 + lane) * 16)
                 : "memory");
  }
  return r;
}

}  // namespace groups
}  // namespace ck
