// Gradients of a linear layer one operand of which is held in MXFP8, for sm_100a:
//
//   weight:  dW[N, K] = sum_m dY[m, n] X[m, k]     X the MXFP8 copy of the layer's input   (and db[N] = sum_m dY[m, n])
//   input:   dX[M, K] = sum_n dY[m, n] W[n, k]     W the layer's MXFP8 weight
//
// Both contract over the rows of the MXFP8 matrix, whose scale blocks lie along its rows: the block-scaled MMA kinds, which
// contract along the blocks, do not apply.  An E4M3 number times a power of two has four significant bits, which bf16 holds
// exactly, so the products run on the bf16 tensor-core path with nothing lost: a first kernel writes the matrix as bf16 to the
// workspace (3 bytes of traffic an element beside 2 * M or 2 * N operations; db's partial sums are made beside it), and a GEMM over both follows.  dY in bf16 is an operand as it
// stands; in fp16 it is the exact sum of two bf16 numbers, in fp32 of three, and the GEMM contracts over all of them.
//
// The GEMM: CTA pairs on 256 x 256 tiles (cta_group::2, each CTA 128 rows of A and 128 columns of B), operands by TMA in
// stages of 64 contraction steps, two accumulators in tensor memory so that a tile's epilogue runs beside the next one's
// main loop.  B is row-major along the result's columns and A, for the weight's gradient, along the result's rows: both are
// read as MN-major operands, without a transposed copy.  Few tiles are split over the contraction, the partial sums going
// through the workspace to a kernel that adds them in a fixed order.
//
// Bound by the tensor pipe and, in a loop, by the power limit: 4608 x 3072 x 12288 bf16 takes 214 us in the GEMM (1.63 PFLOP/s, the pipe 96 % active) and 231
// with the launch before it; 4608 x 12288 x 3072 to fp32 with db 233 (86 %, the sums in parts) and 264 to 300.
//
// Rows that are grouped by expert: dX[i] = dY[i] W_e for the rows i of group e.  The same GEMM over a list of tiles that every CTA makes for itself
// from the groups' ends, the operands' places changed round: W_e's columns are the MMA's 256 rows, dY's rows its columns, of which there may be any multiple of 32, so that the MMAs
// of a group's last tile cost what it has rows for (its loads are a whole tile's); results of 16 bits are turned in shared memory on their way out (us, so / with dY's rows as the MMA's: 64 groups of 2048 x
// 2048, 312 uneven rows each, bf16 285 / 314, fp32 817 / 867; 40 of 1000 x 1056, 300 uneven ones, fp16 105 / 128; eight of 8192 x 4096, 1024 each, in a loop 574 / 576: the power
// limit).  A tile begins at its group's first row, wherever in dY that is, and stores the group's rows alone.  8192 rows of eight groups of 8192 x 4096
// bf16: 372 us cold (1.48 PFLOP/s, the pipe 90 % active), and 118 before it for the weights as bf16 (0.8 GB, 1.04 of the copy rate).  It starts in plain stream order.
#include "ck_gemm_kernel.cuh"
#include "ck_groups.cuh"
#include "ck_rows.cuh"

namespace ck {
namespace {

constexpr int kGradStages = 6;
constexpr int kDeep = 64;                           // contraction steps of a stage: 128 bytes of bf16
constexpr int kOperandBytes = 128 * kDeep * 2;      // of A or B, stage and CTA
constexpr int kPairRows = 256, kPairCols = 256;     // a tile
constexpr int kBoxBytes = 64 * kDeep * 2;           // 64 rows (A) or columns (B) of an MN-major operand
constexpr int kTableBytes = (static_cast<int>(sizeof(groups::Table)) + 15) / 16 * 16, kTurnBytes = 8 * 2048;  // of eight warps, 32 x 32 numbers of 16 bits
constexpr int grad_smem(bool grouped) { return 1024 + kGradStages * 2 * kOperandBytes + 256 + (grouped ? kTableBytes + kTurnBytes : 0); }
static_assert(grad_smem(true) <= 227 * 1024, "shared memory budget exceeded");
static_assert(alone_with_tensor_memory(grad_smem(false)), "no allocation of tensor memory waits");
// Epilogue warps: eight, 128 columns each; for fp32 results, whose sums go on in registers, sixteen of 64.
constexpr int grad_epilogue_warps(bool parts) { return parts ? 16 : 8; }
constexpr int grad_threads(bool parts) { return 64 + 32 * grad_epilogue_warps(parts); }  // beside them producer and issuer
template <typename OutT>
constexpr bool kInParts = std::is_same<OutT, float>::value;

// kind::f16: bf16 operands, fp32 accumulators; bit 15 / 16: A / B are MN-major
constexpr uint32_t grad_idesc(bool a_mn, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((kPairCols >> 3) << 17) | ((kPairRows >> 4) << 24);
}

struct GradParams {
  int rows, cols;       // of the result
  int deep_stages;      // stages of one of A's planes
  int planes;           // bf16 numbers whose sum is an element of dY
  int tiles_m, tiles_n;
  int splits, stages_per_split;
  void* out;            // the result, or fp32 partial sums [splits][rows][cols]
  int* status;
  const float* sum_partials;  // db's partial sums [sum_chunks][sum_cols], to be added beside the first main loop; null: none
  int sum_chunks, sum_cols, sum_dtype;
  void* sum_out;
  const int* offsets;         // grouped rows: the groups' ends
  int groups;
};

__device__ __forceinline__ void store_as(void* out, int dtype, int64_t at, float v) {
  if (dtype == CK_DTYPE_BF16) {
    static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  } else if (dtype == CK_DTYPE_F16) {
    static_cast<__half*>(out)[at] = __float2half_rn(v);
  } else {
    static_cast<float*>(out)[at] = v;
  }
}

__device__ __forceinline__ void mma_bf16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// MN-major operand in boxes of 64 elements x 64 contraction steps with the 128-byte swizzle: groups of eight steps are 1024
// bytes apart, boxes kBoxBytes.
__device__ __forceinline__ uint64_t make_mn_desc(uint32_t smem_addr) { return make_smem_desc(smem_addr, kBoxBytes, 1024, 2); }

// Eight tile rows at a time, down them first: the tiles that run together share operands in L2.
__device__ __forceinline__ void tile_place(const GradParams& p, int tile, int* tile_m, int* tile_n) {
  constexpr int kBand = 8;
  const int band = tile / (kBand * p.tiles_n), in_band = tile - band * kBand * p.tiles_n;
  const int height = min(kBand, p.tiles_m - band * kBand);
  *tile_n = in_band / height;
  *tile_m = band * kBand + in_band - *tile_n * height;
}

// A sum in fp32 leaves tensor memory after at most so many stages and goes on in registers.  The accumulator cuts what it adds to its own
// magnitude, so an error grows with the number of additions: 288 of them (4608 tokens) left 1.9e-6 of the result, in three parts
// 5e-7, in five 2.7e-7.  Each part costs 1 us of a tile's 28, for which the tensor pipe stands still (4608 x 12288 x 3072: 263 us in
// one part, 283 in three, 298 in five).  A result in 16 bits, which rounds at 2e-3 or 2e-4, does without: of 8192 terms
// (8192 rows of eight groups of 8192 x 4096, bf16) 15 of ten thousand results are the neighbour of the nearest number, with sums in fp32 by a library 2 of ten thousand, and both are off by
// 1.66e-3 of the result.
constexpr int kSumStages = 32;
__device__ __forceinline__ int part_stages(int stages) {
  const int parts = (stages + kSumStages - 1) / kSumStages;
  return (stages + parts - 1) / parts;
}

template <typename OutT, bool kMnA, bool kGrouped>
__global__ void __launch_bounds__(grad_threads(kInParts<OutT>), 1)
grad_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GradParams p) {
  // Grouped rows: launched in plain stream order (launch_grad_gemm), so there is nothing to wait for, and what comes behind starts when this ends.
  if constexpr (!kGrouped) pdl_launch_dependents();
  const uint32_t rank = cluster_cta_rank();
  const int worker = blockIdx.x >> 1, workers = gridDim.x >> 1;
  constexpr bool kParts = kInParts<OutT>;
  constexpr int kWarps = grad_epilogue_warps(kParts), kWarpCols = kPairCols / (kWarps / 4), kWarpBoxes = kWarpCols / 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + kGradStages * kOperandBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kGradStages * 2 * kOperandBytes);  // loads -> MMAs
  uint64_t* empty_bar = full_bar + kGradStages;                                              // MMAs -> loads
  uint64_t* acc_full_bar = empty_bar + kGradStages;                                          // MMAs -> epilogue
  uint64_t* acc_empty_bar = acc_full_bar + 2;                                                // epilogue -> MMAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  [[maybe_unused]] groups::Table* table = reinterpret_cast<groups::Table*>(smem + kGradStages * 2 * kOperandBytes + 256);
  static_assert((2 * kGradStages + 4) * 8 + 8 <= 256, "barrier area");
  static_assert(!kGrouped || !kMnA, "the rows of the input's gradient are grouped");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kGradStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full_bar[a], 1);
      mbar_init(&acc_empty_bar[a], kWarps * 2);  // the epilogue warps of both CTAs
    }
    fence_barrier_init();
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_b);
  }
  if (warp == 1) tmem_alloc<2>(tmem_slot, 512);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the other CTA's barriers exist before anything reports to them
  tc_fence_after_sync();
  if constexpr (kGrouped) groups::fill_table(table, p.offsets, p.groups, p.rows, kPairRows);
  const uint32_t tmem = *tmem_slot;

  // How many rows of a grouped tile are computed on: the MMA's columns, in steps of 32.
  [[maybe_unused]] const auto columns_of = [](const groups::Tile& t) { return (min(kPairRows, t.end - t.row) + 31) / 32 * 32; };
  const int tiles = (kGrouped ? table->tiles[p.groups] : p.tiles_m) * p.tiles_n, items = tiles * p.splits, all_stages = p.deep_stages * p.planes;
  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (elect_one()) {
      if constexpr (!kGrouped) pdl_wait();
      const uint32_t full = smem_u32(full_bar), empty = smem_u32(empty_bar), a_addr = smem_u32(smem_a), b_addr = smem_u32(smem_b);
      int s = 0;
      uint32_t ph = 0;
      for (int item = worker; item < items; item += workers) {
        const int split = item / tiles;
        int tile_m, tile_n, group = 0, m0 = static_cast<int>(rank) * 128;
        if constexpr (kGrouped) {
          const groups::Tile t = groups::place(table, p.groups, p.tiles_n, kPairRows, item);
          m0 = t.row + static_cast<int>(rank) * (columns_of(t) / 2);
          tile_n = t.tile_n;
          group = t.group;
        } else {
          tile_place(p, item - split * tiles, &tile_m, &tile_n);
          m0 += tile_m * kPairRows;
        }
        const int n0 = tile_n * kPairCols + static_cast<int>(rank) * 128;
        const int end = min(all_stages, (split + 1) * p.stages_per_split);
        for (int ks = split * p.stages_per_split; ks < end; ++ks) {
          // dY's smallest numbers first: what an accumulator adds is cut to the magnitude that it has reached
          const int behind = ks / p.deep_stages, plane = p.planes - 1 - behind, l0 = (ks - behind * p.deep_stages) * kDeep;
          mbar_wait(empty + s * 8, ph ^ 1, abort_flag);
          const uint32_t bar = full + s * 8, a_to = a_addr + s * kOperandBytes, b_to = b_addr + s * kOperandBytes;
          if (rank == 0) mbar_arrive_expect_tx(bar, 2 * 2 * kOperandBytes);  // both CTAs' loads report to the leader
          if constexpr (kGrouped) {  // the operands' places changed round
            tma_load_3d_pair(a_to, &map_b, bar, n0, l0, group);
            tma_load_3d_pair(a_to + kBoxBytes, &map_b, bar, n0 + 64, l0, group);
            tma_load_3d_pair(b_to, &map_a, bar, l0, m0, plane);
          } else {
            if constexpr (kMnA) {
              tma_load_3d_pair(a_to, &map_a, bar, m0, l0, plane);
              tma_load_3d_pair(a_to + kBoxBytes, &map_a, bar, m0 + 64, l0, plane);
            } else {
              tma_load_3d_pair(a_to, &map_a, bar, l0, m0, plane);
            }
            tma_load_2d_pair(b_to, &map_b, bar, n0, l0);
            tma_load_2d_pair(b_to + kBoxBytes, &map_b, bar, n0 + 64, l0);
          }
          if (++s == kGradStages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs, by the pair's leader
    if (rank == 0) {
      if constexpr (!kGrouped) pdl_wait();  // nothing lands earlier: keeps the bounded waits from running beside a long predecessor
      if (elect_one()) {
        const uint32_t full = smem_u32(full_bar), empty = smem_u32(empty_bar), acc_full = smem_u32(acc_full_bar);
        const uint32_t empty_peer = map_to_cta(empty, 1), acc_full_peer = map_to_cta(acc_full, 1);
        constexpr bool kA = kMnA || kGrouped, kB = !kGrouped;  // MN-major
        const uint64_t a0 = kA ? make_mn_desc(smem_u32(smem_a)) : make_operand_desc_sw128(smem_u32(smem_a));
        const uint64_t b0 = kB ? make_mn_desc(smem_u32(smem_b)) : make_operand_desc_sw128(smem_u32(smem_b));
        uint32_t idesc = grad_idesc(kA, kB);
        constexpr int kStepA = kA ? 2048 >> 4 : 32 >> 4, kStepB = kB ? 2048 >> 4 : 32 >> 4;  // 16 contraction steps: 16 rows of 128 bytes, or 32 bytes
        int s = 0, it = 0;
        uint32_t ph = 0;
        for (int item = worker; item < items; item += workers, ++it) {
          const int split = item / tiles, first = split * p.stages_per_split, last = min(all_stages, first + p.stages_per_split);
          const int part = kParts ? part_stages(last - first) : last - first;
          if constexpr (kGrouped) {
            const groups::Tile t = groups::place(table, p.groups, p.tiles_n, kPairRows, item);
            idesc = (grad_idesc(kA, kB) & ~(0x3Fu << 17)) | (static_cast<uint32_t>(columns_of(t) >> 3) << 17);
          }
          for (int begin = first; begin < last; begin += part) {
            const int end = min(last, begin + part);
            const int acc = it & 1;
            const uint32_t d = tmem + acc * kPairCols;
            mbar_wait(&acc_empty_bar[acc], ((it >> 1) & 1) ^ 1, abort_flag);
            tc_fence_after_sync();
            for (int ks = begin; ks < end; ++ks) {
              mbar_wait(full + s * 8, ph, abort_flag);
              tc_fence_after_sync();
              const uint64_t a = a0 + s * (kOperandBytes >> 4), b = b0 + s * (kOperandBytes >> 4);
#pragma unroll
              for (int k = 0; k < kDeep / 16; ++k) mma_bf16_pair(d, a + k * kStepA, b + k * kStepB, idesc, ks != begin || k != 0);
              tc_commit<2>(empty + s * 8);
              tc_commit<2>(empty_peer + s * 8);
              if (++s == kGradStages) {
                s = 0;
                ph ^= 1u;
              }
            }
            tc_commit<2>(acc_full + acc * 8);
            tc_commit<2>(acc_full_peer + acc * 8);
            if (end != last) ++it;
          }
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue
    if constexpr (!kGrouped) pdl_wait();  // the result's buffer may belong to the kernel before this one
    const int quarter = warp & 3, share = (warp - 2) >> 2;
    const uint32_t acc_empty = map_to_cta(smem_u32(acc_empty_bar), 0);
    // db, whose partial sums the kernel before left: a column a thread, in the chunks' order, while the first tile computes
    if (p.sum_partials != nullptr) {
      for (int c = (blockIdx.x * kWarps - 2) * 32 + threadIdx.x; c < p.sum_cols; c += gridDim.x * kWarps * 32) {
        float sum = 0.0f;
#pragma unroll 4
        for (int i = 0; i < p.sum_chunks; ++i) sum += p.sum_partials[static_cast<int64_t>(i) * p.sum_cols + c];
        store_as(p.sum_out, p.sum_dtype, c, sum);
      }
    }
    int it = 0;
    for (int item = worker; item < items; item += workers, ++it) {
      const int split = item / tiles;
      const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
      const auto wait_for = [&](int acc) {
        mbar_wait(&acc_full_bar[acc], (it >> 1) & 1, abort_flag);
        __syncwarp();
        tc_fence_after_sync();
      };
      const auto give_back = [&](int acc) {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc_empty + acc * 8);
      };
      // this thread's row of the tile, its warp's columns; of a grouped tile its result's column, its warp's rows
      int end = p.rows;
      const auto place = [&](int* row, int* col0) {
        int tile_m, tile_n;
        if constexpr (kGrouped) {
          const groups::Tile t = groups::place(table, p.groups, p.tiles_n, kPairRows, item);
          *row = t.row + share * kWarpCols;
          *col0 = t.tile_n * kPairCols + static_cast<int>(rank) * 128 + quarter * 32;
          end = t.end;
        } else {
          tile_place(p, item - split * tiles, &tile_m, &tile_n);
          *row = tile_m * kPairRows + static_cast<int>(rank) * 128 + quarter * 32 + lane;
          *col0 = tile_n * kPairCols + share * kWarpCols;
        }
      };
      // 32 rows by a lane's column each: fp32 as it is, lines of 128 bytes; 16 bits turned in shared memory on the way
      const auto write_turned = [&](int row0, int col0, const uint32_t(&v)[32]) {
        const int count = end - row0;
        if (count <= 0) return;
        if constexpr (kParts) {
          OutT* out = static_cast<OutT*>(p.out) + static_cast<int64_t>(row0) * p.cols + col0 + lane;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (i < count && col0 + lane < p.cols) out[static_cast<int64_t>(i) * p.cols] = rows::from_float<OutT>(__uint_as_float(v[i]));
          }
        } else {
          const uint32_t turn = smem_u32(smem + kGradStages * 2 * kOperandBytes + 256 + kTableBytes) + (warp - 2) * 2048;
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = __uint_as_float(v[i]);
          groups::turn_write<OutT>(turn, lane, f);
          __syncwarp();
          const int col = col0 + lane % 4 * 8;
          OutT* out = static_cast<OutT*>(p.out) + static_cast<int64_t>(row0 + lane / 4) * p.cols + col;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const auto r = groups::turn_read<OutT>(turn, lane, i);
            if (i * 8 + lane / 4 < count && col < p.cols) rows::store(out + static_cast<int64_t>(i * 8) * p.cols, r);
          }
          __syncwarp();
        }
      };
      const auto write = [&](int row, int col, const uint32_t(&v)[32]) {
        if (row < end && col < p.cols) {
          OutT* out = static_cast<OutT*>(p.out) + (static_cast<int64_t>(split) * p.rows + row) * p.cols + col;
          constexpr int kVec = 32 / static_cast<int>(sizeof(OutT));
#pragma unroll
          for (int i = 0; i < 32 / kVec; ++i) {
            float f[kVec];
#pragma unroll
            for (int j = 0; j < kVec; ++j) f[j] = __uint_as_float(v[i * kVec + j]);
            const rows::Raw<OutT, kVec> r = rows::pack<OutT, kVec>(f);
            st_global_256_no_allocate(out + i * kVec, *reinterpret_cast<const Vec256*>(&r));
          }
        }
        __syncwarp();
      };
      int row, col0;
      if constexpr (kParts) {
        int left = min(all_stages, (split + 1) * p.stages_per_split) - split * p.stages_per_split;
        const int part = part_stages(left);
        float sum[kWarpCols] = {};
        for (bool more = false; left > 0; left -= part, more = true) {
          if (more) ++it;
          const int acc = it & 1;
          wait_for(acc);
          const uint32_t from = tmem + acc * kPairCols + lanes + share * kWarpCols;
#pragma unroll
          for (int c = 0; c < kWarpCols / 16; ++c) {
            uint32_t v[16];
            tmem_load_32x16(from + c * 16, v);
            tmem_load_wait();
#pragma unroll
            for (int j = 0; j < 16; ++j) sum[16 * c + j] += __uint_as_float(v[j]);
          }
          give_back(acc);
        }
        place(&row, &col0);
#pragma unroll
        for (int c = 0; c < kWarpBoxes; ++c) {
          uint32_t v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(sum[32 * c + j]);
          if constexpr (kGrouped) {
            write_turned(row + c * 32, col0, v);
          } else {
            write(row, col0 + c * 32, v);
          }
        }
      } else {
        const int acc = it & 1;
        place(&row, &col0);
        wait_for(acc);
        const uint32_t from = tmem + acc * kPairCols + lanes + share * kWarpCols;
#pragma unroll 1
        for (int c = 0; c < kWarpBoxes; ++c) {
          uint32_t v[32];
          tmem_load_32x32(from + c * 32, v);
          tmem_load_wait();
          if (c == kWarpBoxes - 1) give_back(acc);  // read to the end
          if constexpr (kGrouped) {
            write_turned(row + c * 32, col0, v);
          } else {
            write(row, col0 + c * 32, v);
          }
        }
      }
    }
    if constexpr (kGrouped) {  // rows behind the last group
      constexpr int kVec = 16 / static_cast<int>(sizeof(OutT));
      OutT* out = static_cast<OutT*>(p.out);
      const int64_t first = static_cast<int64_t>(table->bound[p.groups]) * p.cols, n = static_cast<int64_t>(p.rows) * p.cols;
      for (int64_t i = first + (static_cast<int64_t>(blockIdx.x) * (kWarps * 32) + threadIdx.x - 64) * kVec; i < n;
           i += static_cast<int64_t>(gridDim.x) * (kWarps * 32) * kVec) {
        rows::store(out + i, rows::zeros<OutT, kVec>());
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicExch(p.status, 1);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
    __syncthreads();
  }
  cluster_sync_all();  // no CTA leaves while its partner may still signal it
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<2>(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// beside the GEMM
// ---------------------------------------------------------------------------
// The partial sums of a split contraction, added in order.
template <typename OutT>
__global__ void __launch_bounds__(256) add_splits_kernel(const float* partials, int splits, int64_t n, OutT* out) {
  pdl_launch_dependents();
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  pdl_wait();
  if (i >= n) return;
  float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < splits; ++s) {
    float part[4];
    rows::unpack(rows::load_once<float, 4>(partials + s * n + i), part);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] += part[j];
  }
  rows::store(out + i, rows::pack<OutT, 4>(f));
}

// What the GEMM needs, in one launch whose blocks share the work out: the first `held_blocks` write the MXFP8 matrix as bf16, the next
// `plane_blocks` dY as bf16 numbers, the others sum dY's columns.
struct PrepareArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  __nv_bfloat16* held;
  int64_t held_rows, held_cols;
  const void* dy;
  __nv_bfloat16* planes;
  int64_t dy_rows, dy_cols;
  int held_blocks, plane_blocks, sum_strips, sum_chunk;
  float* sum_partials;  // or, where one chunk has all rows, null and the result:
  void* sum_out;
  int sum_dtype;
};

// A block of 32 codes a thread, as ck_dequantize_mxfp8 gives them in bf16.
__device__ __forceinline__ void prepare_held(const PrepareArgs& a, int64_t index) {
  const int64_t blocks = a.held_cols >> 5;
  const int64_t row = index < 0xFFFFFFFFll ? static_cast<uint32_t>(index) / static_cast<uint32_t>(blocks) : index / blocks;
  const int64_t block = index - row * blocks;
  if (row >= a.held_rows) return;
  const Vec256 raw = ld_global_stream_256(a.codes + index * 32);
  const float factor = rows::e8m0_factor(ld_global_u8(a.scales + swizzled_scale_offset(row, block, ceil_div(blocks, 4))));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float f[16];
#pragma unroll
    for (int i = 0; i < 4; ++i) rows::e4m3_four(raw.w[4 * h + i], factor, f + 4 * i);
    const rows::Raw<__nv_bfloat16, 16> r = rows::pack<__nv_bfloat16, 16>(f);
    st_global_256(a.held + index * 32 + 16 * h, *reinterpret_cast<const Vec256*>(&r));
  }
}

// dY as the sum of bf16 numbers: each takes the leading eight bits of what is left, so that three hold an fp32 number and two an
// fp16 one.  Infinities and NaN go into the first alone.
template <typename T>
__device__ __forceinline__ void prepare_planes(const PrepareArgs& a, int64_t i) {
  constexpr int kPlanes = sizeof(T) == 4 ? 3 : 2;
  const int64_t n = a.dy_rows * a.dy_cols;
  if (i >= n) return;
  float left[4];
  rows::unpack(rows::load_once<T, 4>(static_cast<const T*>(a.dy) + i), left);
#pragma unroll
  for (int p = 0; p < kPlanes; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = __float_as_uint(left[j]) & 0xFFFF0000u;
      if (left[j] != left[j]) w[j] = 0x7FC00000u;
      left[j] = isfinite(left[j]) ? left[j] - __uint_as_float(w[j]) : 0.0f;
    }
    *reinterpret_cast<uint2*>(a.planes + p * n + i) = make_uint2((w[0] >> 16) | w[1], (w[2] >> 16) | w[3]);
  }
}

// db: 8 columns a thread, 32 of them beside one another and 8 rows above one another.
template <typename T>
__device__ __forceinline__ void prepare_sums(const PrepareArgs& a, int block, float (*buf)[264]) {
  const int x = threadIdx.x & 31, y = threadIdx.x >> 5, chunk = block / a.sum_strips, strip = block - chunk * a.sum_strips;
  const int64_t col = (static_cast<int64_t>(strip) * 32 + x) * 8;
  const int64_t begin = static_cast<int64_t>(chunk) * a.sum_chunk, end = min(a.dy_rows, begin + a.sum_chunk);
  float sum[8] = {};
  if (col < a.dy_cols) {
    constexpr int kVec = 16 / static_cast<int>(sizeof(T));
    const T* at = static_cast<const T*>(a.dy) + (begin + y) * a.dy_cols + col;
#pragma unroll 8
    for (int64_t r = begin + y; r < end; r += 8, at += 8 * a.dy_cols) {
#pragma unroll
      for (int q = 0; q < 8 / kVec; ++q) {
        float f[kVec];
        rows::unpack(rows::load_once<T, kVec>(at + q * kVec), f);
#pragma unroll
        for (int j = 0; j < kVec; ++j) sum[q * kVec + j] += f[j];
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) buf[y][j * 32 + x] = sum[j];
  __syncthreads();
  const int t = threadIdx.x;
  const int64_t c = (static_cast<int64_t>(strip) * 32 + (t & 31)) * 8 + (t >> 5);
  if (c >= a.dy_cols) return;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += buf[i][t];
  if (a.sum_partials != nullptr) {
    a.sum_partials[chunk * a.dy_cols + c] = s;
  } else {
    store_as(a.sum_out, a.sum_dtype, c, s);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) prepare_kernel(const PrepareArgs a) {
  extern __shared__ float sum_buf[][264];
  // Where columns are summed, in shared memory, the GEMM's blocks, which take most of an SM's, come behind these: with them there three
  // of these blocks had room on an SM (4608 x 3072 x 12288: 260 us, 229 so).
  if (a.sum_chunk == 0) pdl_launch_dependents();
  pdl_wait();
  int block = blockIdx.x;
  if (block < a.held_blocks) return prepare_held(a, static_cast<int64_t>(block) * 256 + threadIdx.x);
  block -= a.held_blocks;
  if constexpr (!std::is_same<T, __nv_bfloat16>::value) {
    if (block < a.plane_blocks) return prepare_planes<T>(a, (static_cast<int64_t>(block) * 256 + threadIdx.x) * 4);
  }
  prepare_sums<T>(a, block - a.plane_blocks, sum_buf);
}

// The same for grouped rows: a matrix [N, K] with scales of its own for each group; those of groups without rows are passed over.
struct GroupedPrepareArgs {
  PrepareArgs args;  // held_rows: of one matrix
  const int* offsets;
  int groups;
};
template <typename T>
__global__ void __launch_bounds__(256) prepare_groups_kernel(const GroupedPrepareArgs g) {
  pdl_launch_dependents();
  const int block = blockIdx.x;
  const PrepareArgs& a = g.args;
  if (block < a.held_blocks) {
    const int64_t each = ceil_div(a.held_rows * (a.held_cols >> 5), 256);  // blocks of one matrix
    const int e = static_cast<int>(block / each);
    pdl_wait();
    if (groups::group_end(g.offsets, e, static_cast<int>(a.dy_rows)) <= groups::group_end(g.offsets, e - 1, static_cast<int>(a.dy_rows))) return;
    PrepareArgs one = a;
    one.codes += e * a.held_rows * a.held_cols;
    one.scales += e * round_up(a.held_rows, 128) * round_up(a.held_cols >> 5, 4);
    one.held += e * a.held_rows * a.held_cols;
    return prepare_held(one, (block - e * each) * 256 + threadIdx.x);
  }
  pdl_wait();
  if constexpr (!std::is_same<T, __nv_bfloat16>::value) prepare_planes<T>(a, (static_cast<int64_t>(block - a.held_blocks) * 256 + threadIdx.x) * 4);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
}  // namespace

// bf16 [planes][rows][cols] row-major, boxes of 64 columns x box_rows rows of one plane, 128-byte swizzle.
int make_plane_map(CUtensorMap* map, const void* base, int64_t planes, int64_t rows, int64_t cols, int box_rows, bool two_dims) {
  return cached_map(map, MapKey{two_dims ? 11 : 10, base, rows, cols, planes, box_rows}, [&](CUtensorMap* m) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(CK_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols) * 2, static_cast<cuuint64_t>(rows) * static_cast<cuuint64_t>(cols) * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
    const cuuint32_t elem_strides[3] = {1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, two_dims ? 2 : 3, const_cast<void*>(base), dims, strides, box, elem_strides,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(CK_ERR_CUDA, "cuTensorMapEncodeTiled (planes) failed with code %d", static_cast<int>(r));
    return static_cast<int>(CK_OK);
  });
}

namespace {

int planes_of(int dtype) { return dtype == CK_DTYPE_F32 ? 3 : dtype == CK_DTYPE_F16 ? 2 : 1; }

// result [rows, cols], contraction of `deep` steps
struct GradShape {
  int64_t rows, cols, deep;
  int planes;
};

int grad_splits(const GradShape& g) {
  const int64_t tiles = ceil_div(g.rows, kPairRows) * ceil_div(g.cols, kPairCols), stages = ceil_div(g.deep, kDeep) * g.planes;
  const int64_t workers = sm_count() / 2;
  int64_t splits = workers / tiles;
  if (splits > stages / 8) splits = stages / 8;  // a split of fewer stages costs more to add than it saves
  if (splits < 1) return 1;
  const int64_t per = ceil_div(stages, splits);
  return static_cast<int>(ceil_div(stages, per));
}

// Workspace: the MXFP8 matrix in bf16 | dY's planes | partial sums of a split | of db
struct GradLayout {
  int64_t held_off, planes_off, partials_off, sums_off, total;
  int splits, sum_chunks;
  bool few_rows;  // the matrix is decoded inside the GEMM (ck_grad_few_rows.cu)
};
GradLayout grad_layout(bool weight, int dtype, bool bias, int64_t M, int64_t N, int64_t K) {
  GradLayout l = {};
  const GradShape g = {weight ? N : M, K, weight ? M : N, planes_of(dtype)};
  l.splits = grad_splits(g);
  l.few_rows = !weight && grad_few_rows_applies(M, N, K, g.planes);
  if (l.few_rows) l.splits = 1;
  l.planes_off = l.few_rows ? 0 : round_up((weight ? M : N) * K * 2, 256);
  l.partials_off = l.planes_off + (g.planes > 1 ? round_up(g.planes * M * N * 2, 256) : 0);
  l.sums_off = l.partials_off + (l.splits > 1 ? round_up(l.splits * g.rows * g.cols * 4, 256) : 0);
  // db: six blocks of 256 threads an SM, of 64 rows at least
  const int64_t strips = ceil_div(N, 256);
  int64_t chunks = ceil_div(6 * sm_count(), strips);
  if (chunks > ceil_div(M, 64)) chunks = ceil_div(M, 64);
  chunks = ceil_div(M, ceil_div(M, chunks));
  l.sum_chunks = static_cast<int>(bias ? chunks : 0);
  l.total = l.sums_off + (l.sum_chunks > 1 ? l.sum_chunks * N * 4 : 0);
  if (l.total == 0) l.total = 256;
  return l;
}

template <typename OutT, bool kMnA, bool kGrouped = false>
int launch_grad_gemm(const CUtensorMap& map_a, const CUtensorMap& map_b, const GradParams& p, cudaStream_t stream) {
  auto kernel = grad_gemm_kernel<OutT, kMnA, kGrouped>;
  int dev = 0;
  CK_CUDA(cudaGetDevice(&dev));
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(grad_threads(kInParts<OutT>));
  cfg.dynamicSmemBytes = grad_smem(kGrouped);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // Grouped rows without programmatic serialization: started beside the end of the long preparing kernel, with its wait in front of the
  // cluster's first barrier, one of some twenty thousand passes did not end.
  cfg.numAttrs = pdl_enabled() && !kGrouped ? 2 : 1;
  // all pairs resident at once: how many there is room for depends on where the SMs lie
  static std::atomic<int> resident_on[64];
  int resident = (dev >= 0 && dev < 64) ? resident_on[dev].load(std::memory_order_acquire) : 0;
  if (resident == 0) {
    CK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, grad_smem(kGrouped)));
    resident = sm_count() / 2;
    cfg.gridDim = dim3(resident * 2);
    int clusters = 0;
    CK_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
    if (clusters > 0 && clusters < resident) resident = clusters;
    if (dev >= 0 && dev < 64) resident_on[dev].store(resident, std::memory_order_release);
  }
  const int64_t items = static_cast<int64_t>(p.tiles_m) * p.tiles_n * p.splits;
  cfg.gridDim = dim3(2 * static_cast<unsigned>(items < resident ? items : resident));
  CK_CUDA(cudaLaunchKernelEx(&cfg, kernel, map_a, map_b, p));
  return CK_OK;
}

template <bool kMnA>
int launch_grad_gemm_typed(const CUtensorMap& map_a, const CUtensorMap& map_b, const GradParams& p, int out_dtype, cudaStream_t s) {
  switch (out_dtype) {
    case CK_DTYPE_BF16: return launch_grad_gemm<__nv_bfloat16, kMnA>(map_a, map_b, p, s);
    case CK_DTYPE_F16: return launch_grad_gemm<__half, kMnA>(map_a, map_b, p, s);
    default: return launch_grad_gemm<float, kMnA>(map_a, map_b, p, s);
  }
}

template <typename OutT>
int launch_add_splits(const float* partials, int splits, int64_t n, void* out, cudaStream_t s) {
  CK_CUDA(launch_pdl(add_splits_kernel<OutT>, dim3(static_cast<unsigned>(ceil_div(n, 1024))), dim3(256), 0, s, partials, splits, n,
                     static_cast<OutT*>(out)));
  return CK_OK;
}

bool is_float(int dtype) { return dtype == CK_DTYPE_F32 || dtype == CK_DTYPE_F16 || dtype == CK_DTYPE_BF16; }

int check_grad(const char* op, const void* dy, int dtype, const void* codes, const void* scales, const void* out, int out_dtype, int64_t M, int64_t N,
               int64_t K, const void* ws) {
  CK_REQUIRE(dy && codes && scales && out && ws, "%s: null pointer", op);
  CK_REQUIRE(is_float(dtype) && is_float(out_dtype), "%s: unsupported dtype code %d or %d", op, dtype, out_dtype);
  CK_REQUIRE(M > 0 && N > 0 && K > 0 && M < (1ll << 30) && N < (1ll << 30) && K < (1ll << 30), "%s: bad shape M=%lld N=%lld K=%lld", op,
             (long long)M, (long long)N, (long long)K);
  CK_REQUIRE(K % 32 == 0 && N % 8 == 0, "%s: K=%lld must be a multiple of 32 and N=%lld of 8", op, (long long)K, (long long)N);
  CK_REQUIRE(ceil_div(M, 256) * ceil_div(K, 256) < (1ll << 24) && ceil_div(N, 256) * ceil_div(K, 256) < (1ll << 24), "%s: too large", op);
  CK_REQUIRE(reinterpret_cast<uintptr_t>(dy) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 32 == 0 && reinterpret_cast<uintptr_t>(scales) % 16 == 0 &&
                 reinterpret_cast<uintptr_t>(out) % 32 == 0 && reinterpret_cast<uintptr_t>(ws) % 256 == 0,
             "%s: dy, codes, block scales, result and workspace have to be aligned to 16, 32, 16, 32 and 256 bytes", op);
  return CK_OK;
}

int linear_grad(bool weight, const char* op, const void* dy, int dtype, const void* codes, const void* scales, void* out, int out_dtype, void* dbias,
                int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, cudaStream_t s) {
  const GradLayout l = grad_layout(weight, dtype, dbias != nullptr, M, N, K);
  CK_REQUIRE(workspace_bytes >= l.total, "%s: workspace of %lld bytes, %lld needed", op, (long long)workspace_bytes, (long long)l.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const GradShape g = {weight ? N : M, K, weight ? M : N, planes_of(dtype)};
  PrepareArgs r = {};
  r.codes = static_cast<const uint8_t*>(codes);
  r.scales = static_cast<const uint8_t*>(scales);
  r.held = reinterpret_cast<__nv_bfloat16*>(ws);
  r.held_rows = g.deep;
  r.held_cols = K;
  r.dy = dy;
  r.planes = reinterpret_cast<__nv_bfloat16*>(ws + l.planes_off);
  r.dy_rows = M;
  r.dy_cols = N;
  const int64_t held_blocks = l.few_rows ? 0 : ceil_div(g.deep * (K / 32), 256), plane_blocks = g.planes > 1 ? ceil_div(M * N, 1024) : 0;
  const int64_t sum_blocks = l.sum_chunks * ceil_div(N, 256);
  CK_REQUIRE(held_blocks + plane_blocks + sum_blocks <= 0x7FFFFFFF, "%s: too large", op);
  r.held_blocks = static_cast<int>(held_blocks);
  r.plane_blocks = static_cast<int>(plane_blocks);
  r.sum_strips = static_cast<int>(ceil_div(N, 256));
  r.sum_chunk = l.sum_chunks > 0 ? static_cast<int>(ceil_div(M, l.sum_chunks)) : 0;
  r.sum_partials = l.sum_chunks > 1 ? reinterpret_cast<float*>(ws + l.sums_off) : nullptr;
  r.sum_out = dbias;
  r.sum_dtype = out_dtype;
  const dim3 grid(static_cast<unsigned>(held_blocks + plane_blocks + sum_blocks));
  auto prepare = dtype == CK_DTYPE_BF16 ? prepare_kernel<__nv_bfloat16> : dtype == CK_DTYPE_F16 ? prepare_kernel<__half> : prepare_kernel<float>;
  if (grid.x > 0) CK_CUDA(launch_pdl(prepare, grid, dim3(256), l.sum_chunks > 0 ? 8 * 264 * 4 : 0, s, r));
  const void* a = g.planes > 1 ? static_cast<const void*>(r.planes) : dy;
  if (l.few_rows) return grad_few_rows(a, g.planes, codes, scales, out, out_dtype, M, N, K, s);
  CUtensorMap map_a, map_b;
  if (int rc = make_plane_map(&map_a, a, g.planes, M, N, weight ? kDeep : 128, false)) return rc;
  if (int rc = make_plane_map(&map_b, ws, 1, g.deep, K, kDeep, true)) return rc;
  GradParams p = {};
  p.rows = static_cast<int>(g.rows);
  p.cols = static_cast<int>(g.cols);
  p.deep_stages = static_cast<int>(ceil_div(g.deep, kDeep));
  p.planes = g.planes;
  p.tiles_m = static_cast<int>(ceil_div(g.rows, kPairRows));
  p.tiles_n = static_cast<int>(ceil_div(g.cols, kPairCols));
  p.splits = l.splits;
  p.stages_per_split = static_cast<int>(ceil_div(static_cast<int64_t>(p.deep_stages) * p.planes, l.splits));
  p.out = l.splits > 1 ? ws + l.partials_off : out;
  p.sum_partials = r.sum_partials;
  p.sum_chunks = l.sum_chunks;
  p.sum_cols = static_cast<int>(N);
  p.sum_dtype = out_dtype;
  p.sum_out = dbias;
  if (int rc = gemm_status_word(&p.status)) return rc;
  const int gemm_type = l.splits > 1 ? CK_DTYPE_F32 : out_dtype;
  if (int rc = weight ? launch_grad_gemm_typed<true>(map_a, map_b, p, gemm_type, s) : launch_grad_gemm_typed<false>(map_a, map_b, p, gemm_type, s)) return rc;
  if (l.splits == 1) return CK_OK;
  const float* partials = reinterpret_cast<const float*>(ws + l.partials_off);
  const int64_t n = g.rows * g.cols;
  switch (out_dtype) {
    case CK_DTYPE_BF16: return launch_add_splits<__nv_bfloat16>(partials, l.splits, n, out, s);
    case CK_DTYPE_F16: return launch_add_splits<__half>(partials, l.splits, n, out, s);
    default: return launch_add_splits<float>(partials, l.splits, n, out, s);
  }
}

// ---- grouped rows --------------------------------------------------------------------------------------------
// Workspace: the groups' matrices in bf16 | dY's planes
struct GroupedGradLayout {
  int64_t planes_off, total;
  bool few_rows;  // the matrices are decoded on their way into the operand (ck_grad_few_rows.cu)
};
GroupedGradLayout grouped_grad_layout(int dtype, int64_t M, int64_t N, int64_t K, int64_t E) {
  GroupedGradLayout l;
  l.few_rows = grouped_few_rows_applies(M, E);
  l.planes_off = l.few_rows ? 0 : round_up(E * N * K * 2, 256);
  l.total = l.planes_off + (planes_of(dtype) > 1 ? planes_of(dtype) * M * N * 2 : 0);
  if (l.total == 0) l.total = 256;
  return l;
}

int check_grouped_grad(const char* op, int dtype, int64_t M, int64_t N, int64_t K, int64_t E) {
  CK_REQUIRE(is_float(dtype), "%s: unsupported dtype code %d", op, dtype);
  CK_REQUIRE(M > 0 && N > 0 && K > 0 && M < (1ll << 30) && N < (1ll << 30) && K < (1ll << 30), "%s: bad shape M=%lld N=%lld K=%lld", op,
             (long long)M, (long long)N, (long long)K);
  CK_REQUIRE(E > 0 && E <= groups::kMaxGroups, "%s: %lld groups, 1 to %d are supported", op, (long long)E, groups::kMaxGroups);
  CK_REQUIRE(K % 32 == 0 && N % 8 == 0, "%s: K=%lld must be a multiple of 32 and N=%lld of 8", op, (long long)K, (long long)N);
  CK_REQUIRE((M / kPairRows + E) * ceil_div(K, kPairCols) < (1ll << 30) && E * ceil_div(N * (K / 32), 256) + ceil_div(M * N, 1024) <= 0x7FFFFFFF,
             "%s: too large", op);
  return CK_OK;
}

int grouped_input_grad(const char* op, const void* dy, int dtype, const void* codes, const void* scales, const int* offsets, void* out, int out_dtype,
                       int64_t M, int64_t N, int64_t K, int64_t E, void* workspace, int64_t workspace_bytes, cudaStream_t s) {
  CK_REQUIRE(dy && codes && scales && offsets && out && workspace, "%s: null pointer", op);
  if (int rc = check_grouped_grad(op, dtype, M, N, K, E)) return rc;
  CK_REQUIRE(is_float(out_dtype), "%s: unsupported dtype code %d", op, out_dtype);
  CK_REQUIRE(reinterpret_cast<uintptr_t>(dy) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 32 == 0 && reinterpret_cast<uintptr_t>(scales) % 16 == 0 &&
                 reinterpret_cast<uintptr_t>(out) % 32 == 0 && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 &&
                 reinterpret_cast<uintptr_t>(offsets) % 4 == 0,
             "%s: dy, codes, block scales, result and workspace have to be aligned to 16, 32, 16, 32 and 256 bytes", op);
  const GroupedGradLayout l = grouped_grad_layout(dtype, M, N, K, E);
  CK_REQUIRE(workspace_bytes >= l.total, "%s: workspace of %lld bytes, %lld needed", op, (long long)workspace_bytes, (long long)l.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int planes = planes_of(dtype);
  GroupedPrepareArgs g = {};
  g.offsets = offsets;
  g.groups = static_cast<int>(E);
  g.args.codes = static_cast<const uint8_t*>(codes);
  g.args.scales = static_cast<const uint8_t*>(scales);
  g.args.held = reinterpret_cast<__nv_bfloat16*>(ws);
  g.args.held_rows = N;
  g.args.held_cols = K;
  g.args.dy = dy;
  g.args.planes = reinterpret_cast<__nv_bfloat16*>(ws + l.planes_off);
  g.args.dy_rows = M;
  g.args.dy_cols = N;
  g.args.held_blocks = l.few_rows ? 0 : static_cast<int>(E * ceil_div(N * (K / 32), 256));
  g.args.plane_blocks = planes > 1 ? static_cast<int>(ceil_div(M * N, 1024)) : 0;
  auto prepare = dtype == CK_DTYPE_BF16 ? prepare_groups_kernel<__nv_bfloat16> : dtype == CK_DTYPE_F16 ? prepare_groups_kernel<__half> : prepare_groups_kernel<float>;
  const unsigned blocks = static_cast<unsigned>(g.args.held_blocks + g.args.plane_blocks);
  if (blocks > 0) CK_CUDA(launch_pdl(prepare, dim3(blocks), dim3(256), 0, s, g));
  if (l.few_rows) return grouped_few_rows(planes > 1 ? g.args.planes : dy, planes, codes, scales, offsets, out, out_dtype, M, N, K, E, s);
  CUtensorMap map_a, map_b;
  if (int rc = make_plane_map(&map_a, planes > 1 ? g.args.planes : dy, planes, M, N, 128, false)) return rc;
  if (int rc = make_plane_map(&map_b, ws, E, N, K, kDeep, false)) return rc;
  GradParams p = {};
  p.rows = static_cast<int>(M);
  p.cols = static_cast<int>(K);
  p.deep_stages = static_cast<int>(ceil_div(N, kDeep));
  p.planes = planes;
  p.tiles_m = static_cast<int>(M / kPairRows + (E < M ? E : M));  // the most that the groups can have
  p.tiles_n = static_cast<int>(ceil_div(K, kPairCols));
  p.splits = 1;
  p.stages_per_split = p.deep_stages * planes;
  p.out = out;
  p.offsets = offsets;
  p.groups = static_cast<int>(E);
  if (int rc = gemm_status_word(&p.status)) return rc;
  switch (out_dtype) {
    case CK_DTYPE_BF16: return launch_grad_gemm<__nv_bfloat16, false, true>(map_a, map_b, p, s);
    case CK_DTYPE_F16: return launch_grad_gemm<__half, false, true>(map_a, map_b, p, s);
    default: return launch_grad_gemm<float, false, true>(map_a, map_b, p, s);
  }
}

}  // namespace
}  // namespace ck

extern "C" int64_t ck_grouped_input_grad_mxfp8_workspace_bytes(int dy_dtype, int64_t M, int64_t N, int64_t K, int64_t E) {
  if (ck::check_grouped_grad("grouped_input_grad_mxfp8", dy_dtype, M, N, K, E) != CK_OK) return 0;
  return ck::grouped_grad_layout(dy_dtype, M, N, K, E).total;
}

extern "C" int ck_grouped_input_grad_mxfp8(const void* dy, int dy_dtype, const void* w_codes, const void* w_block_scales, const int* offsets, void* dx,
                                           int out_dtype, int64_t M, int64_t N, int64_t K, int64_t E, void* workspace, int64_t workspace_bytes,
                                           void* stream) {
  return ck::grouped_input_grad("grouped_input_grad_mxfp8", dy, dy_dtype, w_codes, w_block_scales, offsets, dx, out_dtype, M, N, K, E, workspace,
                                workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t ck_linear_grad_mxfp8_workspace_bytes(int of_weight, int dy_dtype, int with_bias, int64_t M, int64_t N, int64_t K) {
  using namespace ck;
  if (M <= 0 || N <= 0 || K <= 0 || M >= (1ll << 30) || N >= (1ll << 30) || K >= (1ll << 30) || K % 32 != 0 || N % 8 != 0 || !is_float(dy_dtype)) return 0;
  return grad_layout(of_weight != 0, dy_dtype, with_bias != 0, M, N, K).total;
}

extern "C" int ck_linear_weight_grad_mxfp8(const void* dy, int dy_dtype, const void* x_codes, const void* x_block_scales, void* dweight, int out_dtype,
                                           void* dbias, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ck;
  if (int rc = check_grad("linear_weight_grad_mxfp8", dy, dy_dtype, x_codes, x_block_scales, dweight, out_dtype, M, N, K, workspace)) return rc;
  return linear_grad(true, "linear_weight_grad_mxfp8", dy, dy_dtype, x_codes, x_block_scales, dweight, out_dtype, dbias, M, N, K, workspace,
                     workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int ck_linear_input_grad_mxfp8(const void* dy, int dy_dtype, const void* w_codes, const void* w_block_scales, void* dx, int out_dtype,
                                          int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ck;
  if (int rc = check_grad("linear_input_grad_mxfp8", dy, dy_dtype, w_codes, w_block_scales, dx, out_dtype, M, N, K, workspace)) return rc;
  return linear_grad(false, "linear_input_grad_mxfp8", dy, dy_dtype, w_codes, w_block_scales, dx, out_dtype, nullptr, M, N, K, workspace,
                     workspace_bytes, static_cast<cudaStream_t>(stream));
}
