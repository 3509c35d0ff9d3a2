// Products of rows that are grouped by expert with the experts' MXFP8 weights, for sm_100a:
//
//   out[i, :] = cast(x[i, :] . W_e^T + b_e)     for the rows i of group e
//
// x [M, K] in MXFP8 or in float (quantized on the way, as ck_quantize_mxfp8 does), W [E, N, K] in MXFP8, the groups' ends on the device.
//
// A tile is rows of one group by columns: it begins at the group's first row, wherever in x that is (a TMA box may start at any row), and its
// scales come from tiles of 128 rows that begin there too.  A first kernel writes those beside the quantization, or from the scales of x
// as they stand (1/32 of x).  The GEMM is the block-scaled one of ck_gemm_kernel.cuh (TMA producer, one issuing lane, epilogue
// warps, two roles' distance by mbarriers) over a list of tiles that every CTA makes for itself from the groups' ends.  Rows behind the group's end are not stored;
// rows behind the last group are zeros.
//
// CTA pairs, for many rows, compute W_e x^T: the weights' rows are the MMA's 256, x's rows its columns, of which there may be any multiple of 32, so that the MMAs of a
// group's last tile cost what it has rows for; its loads of the weights are a whole tile's.  The results come feature by feature and are turned in shared memory on their way
// out.  (With x's rows as the MMA's 256, last tiles whole, us, so / before: 64 experts of 2048 x 2048, 140 rows each 62 / 69, 188 uneven ones 75 / 81, 256 88 / 92; 8 of
// 8192 x 4096, 1024 uneven rows 215 to 258 / 235 to 267; 8 of 8192 x 512 48.9 / 47.5; all of these with pairs that started beside the kernel in front.  Behind it, as now, from MXFP8 rows:
// 140 each 65, 188 uneven 74, 256 74.)
//
// Many rows: bound by the tensor pipe and, in a loop, by the power limit (8192 x 8192 x 4096 of 8 experts from bf16 234 us, 2.3 PFLOP/s with the quantization;
// one weight for all rows 202).  Few rows: by the weights' bytes (64 experts of 2048 x 2048, 32 rows each, 55 us,
// 5.3 TB/s); one token through eight of 64 experts, 25 MB, 10.4 us: two launches, first loads (11.7 with the weights asked for behind the first kernel's end;
// 777 rows of 40 experts of 1000 x 1056 16.3 and 18.3; a few megabytes of weights gain nothing, 64 rows of 8 experts of 1024 x 1024 7.1 and 6.9).
#include "ck_gemm_kernel.cuh"
#include "ck_groups.cuh"
#include "ck_rows.cuh"

namespace ck {
namespace {

struct GroupedParams {
  const int* offsets;
  const uint8_t* sfa;    // x's scales, in the workspace: the groups' tiles
  const uint8_t* sfb;    // W's: [E][ceil(N / 128)][col_tiles] tiles of 512 bytes
  const void* bias;      // [E, N] or null
  void* out;             // [M, N]
  int bias_dtype;
  int groups, M, N;
  int k_bytes, col_tiles, n_row_blocks_b;
  int tiles_n;
  int* status;
};

// Boxes of x's rows: no more of them are fetched than a tile has, to the next of three heights.
constexpr int box_height(int box) { return box == 2 ? 128 : box == 1 ? 32 : 8; }
struct RowMaps {
  CUtensorMap m[3];
};

__device__ __forceinline__ float bias_at(const void* bias, int dtype, int64_t at) {
  if (dtype == CK_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[at]);
  if (dtype == CK_DTYPE_F16) return __half2float(static_cast<const __half*>(bias)[at]);
  return static_cast<const float*>(bias)[at];
}

template <int TILE_N, int NUM_ACC, int STAGES, int CTAS, int kOutBytes>
struct GroupedConfig : Config<Kind::kMxfp8, TILE_N, NUM_ACC, STAGES, CTAS, 0> {
  using Base = Config<Kind::kMxfp8, TILE_N, NUM_ACC, STAGES, CTAS, 0>;
  static constexpr int kTableBytes = (static_cast<int>(sizeof(groups::Table)) + 15) / 16 * 16, kWarps = epilogue_warps(false, TILE_N);
  // a pair's warps turn 32 rows by 32 features; the others pass their columns' bias round
  static constexpr int kEpilogueBytes = CTAS == 2 ? kWarps * 1024 * kOutBytes : kWarps * (TILE_N / (kWarps / 4)) * 4;
  static constexpr int kSmem = Base::kRingBytes + 1024 + 256 + kTableBytes + kEpilogueBytes;
  static_assert(kSmem <= 227 * 1024, "shared memory budget exceeded");
  static_assert(alone_with_tensor_memory(kSmem), "no allocation of tensor memory waits");
};

template <int TILE_N, int NUM_ACC, int STAGES, int CTAS, typename OutT>
__global__ void __launch_bounds__(num_threads(false, TILE_N), 1)
grouped_gemm_kernel(const __grid_constant__ RowMaps maps_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sfx,
                    const __grid_constant__ CUtensorMap map_sfw, const GroupedParams p) {
  using Cfg = GroupedConfig<TILE_N, NUM_ACC, STAGES, CTAS, static_cast<int>(sizeof(OutT))>;
  constexpr int kWarps = epilogue_warps(false, TILE_N);
  constexpr int kTileCols = CTAS == 2 ? 2 * kTileM : TILE_N;  // output features of a tile
  pdl_launch_dependents();
  const uint32_t cta_rank = CTAS == 2 ? cluster_cta_rank() : 0u;
  const int worker = blockIdx.x / CTAS, workers = gridDim.x / CTAS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem_a + STAGES * Cfg::kABytes;
  uint8_t* smem_sfa = smem_b + STAGES * Cfg::kBBytes;
  uint8_t* smem_sfb = smem_sfa + STAGES * Cfg::kSfaBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::kRingBytes);  // loads -> MMAs
  uint64_t* empty_bar = full_bar + STAGES;                                   // MMAs -> loads
  uint64_t* acc_full_bar = empty_bar + STAGES;                               // MMAs -> epilogue
  uint64_t* acc_empty_bar = acc_full_bar + NUM_ACC;                          // epilogue -> MMAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty_bar + NUM_ACC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  groups::Table* table = reinterpret_cast<groups::Table*>(smem + Cfg::kRingBytes + 256);
  static_assert((2 * STAGES + 2 * NUM_ACC) * 8 + 8 <= 256, "barrier area");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < NUM_ACC; ++a) {
      mbar_init(&acc_full_bar[a], 1);
      mbar_init(&acc_empty_bar[a], kWarps * CTAS);
    }
    fence_barrier_init();
    for (int h = 0; h < 3; ++h) prefetch_tensormap(&maps_x.m[h]);
    prefetch_tensormap(&map_w);
    if constexpr (CTAS == 2) {
      prefetch_tensormap(&map_sfx);
      prefetch_tensormap(&map_sfw);
    }
  }
  if (warp == 1) tmem_alloc<CTAS>(tmem_slot, Cfg::kTmemCols);
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CTAS == 2) cluster_sync_all();  // the other CTA's barriers exist before anything reports to them
  tc_fence_after_sync();
  // The kernel before this one has waited for its own predecessor before it let this one start, so the ends, the weights and their scales are there;
  // x's codes and scales are not, where this is a single CTA.  Its first stages' weights are on their way while that kernel still runs.  (Pairs start behind it.)
  groups::fill_table(table, p.offsets, p.groups, p.M, Cfg::kTileRows);
  const uint32_t tmem = *tmem_slot;

  const int items = table->tiles[p.groups] * p.tiles_n;
  // What of a tile's rows is computed on by a pair: as many of the MMA's columns, in steps of 32; and the box that holds a CTA's share of them.
  const auto columns_of = [&](const groups::Tile& t) { return CTAS == 2 ? (min(256, t.end - t.row) + 31) / 32 * 32 : 0; };
  const auto box_of = [&](const groups::Tile& t) {
    const int need = CTAS == 2 ? columns_of(t) / 2 : t.end - t.row;
    return need > box_height(1) ? 2 : CTAS == 2 || need > box_height(0) ? 1 : 0;
  };
  const int k_stages = (p.k_bytes + kStageKBytes - 1) / kStageKBytes, total_mma = (p.k_bytes + kMmaKBytes - 1) / kMmaKBytes;
  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (elect_one()) {
      const uint32_t full = smem_u32(full_bar), empty = smem_u32(empty_bar);
      const uint32_t a_addr = smem_u32(smem_a), b_addr = smem_u32(smem_b), sfa_addr = smem_u32(smem_sfa), sfb_addr = smem_u32(smem_sfb);
      int s = 0, ahead = 0;  // stages whose weights have been asked for already
      uint32_t ph = 0;
      if (worker < items) {
        const groups::Tile t = groups::place(table, p.groups, p.tiles_n, Cfg::kTileRows, worker);
        const int n0 = t.tile_n * kTileCols, rank = static_cast<int>(cta_rank);
        const int w_row = t.group * p.N + n0 + rank * kTileM, rb_w = t.group * p.n_row_blocks_b + n0 / 128 + rank;
        const uint32_t x_bytes = box_height(box_of(t)) * kStageKBytes;
        ahead = min(STAGES, k_stages);
        for (int ks = 0; ks < ahead; ++ks) {
          const uint32_t bar = full + ks * 8;
          if constexpr (CTAS == 2) {
            if (cta_rank == 0) mbar_arrive_expect_tx(bar, 2 * (Cfg::kABytes + x_bytes + Cfg::kSfaBytes + Cfg::kSfbBytes));  // both CTAs' loads report to the leader
            tma_load_2d_pair(a_addr + ks * Cfg::kABytes, &map_w, bar, ks * kStageKBytes, w_row);
            tma_load_3d_pair(sfa_addr + ks * Cfg::kSfaBytes, &map_sfw, bar, 0, ks, rb_w);
          } else {
            mbar_arrive_expect_tx(bar, x_bytes + Cfg::kBBytes + 512u * 2);
            tma_load_2d(b_addr + ks * Cfg::kBBytes, &map_w, bar, ks * kStageKBytes, w_row);
            bulk_load_1d(sfb_addr + ks * Cfg::kSfbBytes, p.sfb + (static_cast<int64_t>(rb_w) * p.col_tiles + ks) * 512, 512, bar);
          }
        }
      }
      pdl_wait();  // also where there is no tile: this kernel does not end before the one in front of it
      for (int item = worker; item < items; item += workers) {
        const groups::Tile t = groups::place(table, p.groups, p.tiles_n, Cfg::kTileRows, item);
        const int n0 = t.tile_n * kTileCols, rank = static_cast<int>(cta_rank);
        const int w_row = t.group * p.N + n0 + rank * kTileM, rb_w = t.group * p.n_row_blocks_b + n0 / 128 + rank;
        const int x_row = t.row + rank * (columns_of(t) / 2);  // (a pair's: half of the tile's rows each)
        const int rb_x = static_cast<int>(groups::first_scale_block(table->bound[t.group], t.group)) + t.index * CTAS;
        const int box = box_of(t);
        const CUtensorMap* map_x = &maps_x.m[box];
        const uint32_t x_bytes = box_height(box) * kStageKBytes;
        const uint8_t* sfx_src = p.sfa + static_cast<int64_t>(rb_x) * p.col_tiles * 512;
        const uint8_t* sfw_src = p.sfb + static_cast<int64_t>(rb_w) * p.col_tiles * 512;
        for (int ks = 0; ks < k_stages; ++ks) {
          mbar_wait(empty + s * 8, ph ^ 1, abort_flag);
          const uint32_t bar = full + s * 8;
          const bool whole = ahead == 0;
          if (!whole) --ahead;
          if constexpr (CTAS == 2) {
            if (whole) {
              if (cta_rank == 0) mbar_arrive_expect_tx(bar, 2 * (Cfg::kABytes + x_bytes + Cfg::kSfaBytes + Cfg::kSfbBytes));
              tma_load_2d_pair(a_addr + s * Cfg::kABytes, &map_w, bar, ks * kStageKBytes, w_row);
              tma_load_3d_pair(sfa_addr + s * Cfg::kSfaBytes, &map_sfw, bar, 0, ks, rb_w);
            }
            tma_load_2d_pair(b_addr + s * Cfg::kBBytes, map_x, bar, ks * kStageKBytes, x_row);
            tma_load_3d_pair(sfb_addr + s * Cfg::kSfbBytes, &map_sfx, bar, 0, ks, rb_x);
          } else {
            if (whole) {
              mbar_arrive_expect_tx(bar, x_bytes + Cfg::kBBytes + 512u * 2);
              tma_load_2d(b_addr + s * Cfg::kBBytes, &map_w, bar, ks * kStageKBytes, w_row);
              bulk_load_1d(sfb_addr + s * Cfg::kSfbBytes, sfw_src + ks * 512, 512, bar);
            }
            tma_load_2d(a_addr + s * Cfg::kABytes, map_x, bar, ks * kStageKBytes, x_row);
            bulk_load_1d(sfa_addr + s * Cfg::kSfaBytes, sfx_src + ks * 512, 512, bar);
          }
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMAs, by the pair's leader
    if (cta_rank == 0 && elect_one()) {
      pdl_wait();  // nothing is complete earlier: keeps the bounded waits from running beside a long predecessor
      const uint32_t a_lo0 = static_cast<uint32_t>(make_operand_desc_sw128(smem_u32(smem_a)));
      const uint32_t b_lo0 = static_cast<uint32_t>(make_operand_desc_sw128(smem_u32(smem_b)));
      const uint32_t op_hi = static_cast<uint32_t>(make_operand_desc_sw128(0) >> 32);
      const uint32_t sfa_lo0 = static_cast<uint32_t>(make_scale_desc(smem_u32(smem_sfa)));
      const uint32_t sfb_lo0 = static_cast<uint32_t>(make_scale_desc(smem_u32(smem_sfb)));
      const uint32_t sf_hi = static_cast<uint32_t>(make_scale_desc(0) >> 32);
      const uint32_t full = smem_u32(full_bar), empty = smem_u32(empty_bar), acc_full = smem_u32(acc_full_bar);
      const uint32_t empty_peer = CTAS == 2 ? map_to_cta(empty, 1) : 0u, acc_full_peer = CTAS == 2 ? map_to_cta(acc_full, 1) : 0u;
      int s = 0, it = 0;
      uint32_t ph = 0;
      for (int item = worker; item < items; item += workers, ++it) {
        // which half of a 128-row block of B's scales a 64-wide tile reads: its column's place in the band
        const groups::Tile t = groups::place(table, p.groups, p.tiles_n, Cfg::kTileRows, item);
        const uint32_t sfb_shift = CTAS == 2 ? 0u : (t.tile_n * TILE_N % 128) / 32;
        const uint32_t idesc = CTAS == 2 ? (Cfg::kIdesc & ~(0x3Fu << 17)) | (static_cast<uint32_t>(columns_of(t) >> 3) << 17) : Cfg::kIdesc;
        const int acc = it % NUM_ACC;
        const uint32_t d = tmem + acc * Cfg::kAccCols;
        for (int ks = 0; ks < k_stages; ++ks) {
          mbar_wait(full + s * 8, ph, abort_flag);
          tc_fence_after_sync();
          const uint32_t t_sfa = tmem + Cfg::kSfaCol + s * Cfg::kSfColsPerBuf, t_sfb = tmem + Cfg::kSfbCol + s * Cfg::kSfColsPerBuf;
          const uint32_t a_lo = a_lo0 + s * (Cfg::kABytes >> 4), b_lo = b_lo0 + s * (Cfg::kBBytes >> 4);
          tc_copy_scales_32x128b<CTAS>(t_sfa, desc64(sfa_lo0 + s * (Cfg::kSfaBytes >> 4), sf_hi));
#pragma unroll
          for (int r = 0; r < Cfg::kSfbRowBlocks; ++r) {
            tc_copy_scales_32x128b<CTAS>(t_sfb + r * 4, desc64(sfb_lo0 + s * (Cfg::kSfbBytes >> 4) + r * 32, sf_hi));
          }
          if (ks == 0) {
            mbar_wait(&acc_empty_bar[acc], ((it / NUM_ACC) & 1) ^ 1, abort_flag);
            tc_fence_after_sync();
          }
          const auto mma = [&](int kb) {
            mma_mxfp8<CTAS>(d, desc64(a_lo + kb * 2, op_hi), desc64(b_lo + kb * 2, op_hi), idesc_with_scale_ids(idesc, kb), t_sfa, t_sfb + sfb_shift,
                            (ks != 0 || kb != 0) ? 1u : 0u);
          };
          const int n_mma = total_mma - ks * kMmaPerStage;
          if (n_mma >= kMmaPerStage) {
#pragma unroll
            for (int kb = 0; kb < kMmaPerStage; ++kb) mma(kb);
          } else {
            for (int kb = 0; kb < n_mma; ++kb) mma(kb);
          }
          tc_commit<CTAS>(empty + s * 8);
          if constexpr (CTAS == 2) tc_commit<CTAS>(empty_peer + s * 8);
          if (++s == STAGES) {
            s = 0;
            ph ^= 1u;
          }
        }
        tc_commit<CTAS>(acc_full + acc * 8);
        if constexpr (CTAS == 2) tc_commit<CTAS>(acc_full_peer + acc * 8);
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue
    pdl_wait();  // see above
    const int quarter = warp & 3, share = (warp - 2) >> 2;
    constexpr int kWarpCols = TILE_N / (kWarps / 4), kChunks = kWarpCols / 32;
    const uint32_t acc_empty = CTAS == 2 ? map_to_cta(smem_u32(acc_empty_bar), 0) : smem_u32(acc_empty_bar);
    OutT* out = static_cast<OutT*>(p.out);
    float* const bias_s = reinterpret_cast<float*>(smem + Cfg::kRingBytes + 256 + Cfg::kTableBytes) + (warp - 2) * kWarpCols;
    // stores of 32 bytes where rows start on such boundaries, of 16 (N is a multiple of 8) otherwise
    const bool wide = (static_cast<int64_t>(p.N) * sizeof(OutT)) % 32 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0;
    int it = 0;
    if constexpr (CTAS == 2) {
      // a lane has one output feature, a column of tensor memory one row
      const uint32_t turn = smem_u32(smem + Cfg::kRingBytes + 256 + Cfg::kTableBytes) + (warp - 2) * 1024 * static_cast<int>(sizeof(OutT));
      for (int item = worker; item < items; item += workers, ++it) {
        const groups::Tile t = groups::place(table, p.groups, p.tiles_n, Cfg::kTileRows, item);
        const int feature = t.tile_n * kTileCols + static_cast<int>(cta_rank) * kTileM + quarter * 32 + lane;
        const int row0 = t.row + share * kWarpCols, rows = min(kWarpCols, t.end - row0);
        const float bias = p.bias != nullptr && feature < p.N ? bias_at(p.bias, p.bias_dtype, static_cast<int64_t>(t.group) * p.N + feature) : 0.0f;
        const int acc = it % NUM_ACC;
        mbar_wait(&acc_full_bar[acc], (it / NUM_ACC) & 1, abort_flag);
        __syncwarp();
        tc_fence_after_sync();
        const uint32_t from = tmem + acc * Cfg::kAccCols + (static_cast<uint32_t>(quarter * 32) << 16) + share * kWarpCols;
        uint32_t buf[kChunks][32];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          if (c * 32 < rows) tmem_load_32x32(from + c * 32, buf[c]);
        }
        tmem_load_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc_empty + acc * 8);
        // 32 rows at a time are turned in shared memory: stores are 16 bytes of a row's features
        constexpr int kVec = 16 / static_cast<int>(sizeof(OutT)), kPieces = 32 / kVec, kRowsAtOnce = 32 / kPieces;
        const int piece = lane % kPieces, at = t.tile_n * kTileCols + static_cast<int>(cta_rank) * kTileM + quarter * 32 + piece * kVec;
        OutT* dst = out + static_cast<int64_t>(row0 + lane / kPieces) * p.N + at;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          if (c * 32 >= rows) break;
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(buf[c][i]) + bias;
          groups::turn_write<OutT>(turn, lane, v);
          __syncwarp();
          rows::Raw<OutT, kVec> got[kPieces];
#pragma unroll
          for (int i = 0; i < kPieces; ++i) got[i] = groups::turn_read<OutT>(turn, lane, i);
#pragma unroll
          for (int i = 0; i < kPieces; ++i) {
            if (c * 32 + i * kRowsAtOnce + lane / kPieces < rows && at < p.N) rows::store(dst + static_cast<int64_t>(c * 32 + i * kRowsAtOnce) * p.N, got[i]);
          }
          __syncwarp();
        }
      }
    } else {
      for (int item = worker; item < items; item += workers, ++it) {
        const groups::Tile t = groups::place(table, p.groups, p.tiles_n, Cfg::kTileRows, item);
        const int row = t.row + static_cast<int>(cta_rank) * kTileM + quarter * 32 + lane, col0 = t.tile_n * TILE_N + share * kWarpCols;
        const int acc = it % NUM_ACC;
        // the warp's columns' bias, one a lane, fetched while the tile computes and passed round through shared memory
        float bias[kChunks] = {};
        if (p.bias != nullptr) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            const int col = col0 + c * 32 + lane;
            if (col < p.N) bias[c] = bias_at(p.bias, p.bias_dtype, static_cast<int64_t>(t.group) * p.N + col);
          }
        }
        mbar_wait(&acc_full_bar[acc], (it / NUM_ACC) & 1, abort_flag);
        __syncwarp();
        tc_fence_after_sync();
        const uint32_t from = tmem + acc * Cfg::kAccCols + (static_cast<uint32_t>(quarter * 32) << 16) + share * kWarpCols;
        uint32_t buf[kChunks][32];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) tmem_load_32x32(from + c * 32, buf[c]);
        tmem_load_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc_empty + acc * 8);
        if (p.bias != nullptr) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) bias_s[c * 32 + lane] = bias[c];
          __syncwarp();
        }
        if (row >= t.end) continue;
        OutT* dst = out + static_cast<int64_t>(row) * p.N + col0;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          const int valid = min(32, p.N - (col0 + c * 32));
          if (valid <= 0) continue;
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(buf[c][i]);
          if (p.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 q = reinterpret_cast<const float4*>(bias_s + c * 32)[i];
              v[4 * i] += q.x;
              v[4 * i + 1] += q.y;
              v[4 * i + 2] += q.z;
              v[4 * i + 3] += q.w;
            }
          }
          if (wide && valid == 32) {
            store_row_chunk<OutT>(dst + c * 32, v, 32, true);
          } else {
            constexpr int kVec = 16 / static_cast<int>(sizeof(OutT));
#pragma unroll
            for (int i = 0; i < 32 / kVec; ++i) {
              float f[kVec];
#pragma unroll
              for (int j = 0; j < kVec; ++j) f[j] = v[i * kVec + j];
              if (i * kVec < valid) rows::store(dst + c * 32 + i * kVec, rows::pack<OutT, kVec>(f));
            }
          }
        }
      }
    }
    // rows behind the last group
    constexpr int kVec = 16 / static_cast<int>(sizeof(OutT));
    const int64_t first = static_cast<int64_t>(table->bound[p.groups]) * p.N, n = static_cast<int64_t>(p.M) * p.N;
    for (int64_t i = first + (static_cast<int64_t>(blockIdx.x) * (kWarps * 32) + threadIdx.x - 64) * kVec; i < n;
         i += static_cast<int64_t>(gridDim.x) * (kWarps * 32) * kVec) {
      rows::store(out + i, rows::zeros<OutT, kVec>());
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0) atomicExch(p.status, 1);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
    __syncthreads();
  }
  if constexpr (CTAS == 2) cluster_sync_all();  // no CTA leaves while its partner may still signal it
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<CTAS>(tmem, Cfg::kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// in front of the GEMM: x's scales in the groups' tiles
// ---------------------------------------------------------------------------
// A block of 32 elements a thread, four neighbouring threads a word of scales; rows behind the last group are passed over.
template <typename T>
__global__ void __launch_bounds__(256) quantize_groups_kernel(const T* x, const int* offsets, int count, int rows, int64_t cols, uint8_t* codes,
                                                              uint8_t* scales) {
  const int64_t blocks = cols >> 5, col_tiles = ceil_div(blocks, 4);
  const int64_t index = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t row = index / (col_tiles * 4), block = index - row * (col_tiles * 4);
  pdl_wait();
  pdl_launch_dependents();  // not earlier: the GEMM reads the weights and the ends without waiting for this kernel's end
  uint32_t byte = 0;
  if (row < rows && block < blocks) {
    constexpr int kVec = 16 / static_cast<int>(sizeof(T));
    const T* from = x + row * cols + block * 32;
    float2 u[16];
    rows::Raw<T, kVec> raw[32 / kVec];
#pragma unroll
    for (int i = 0; i < 32 / kVec; ++i) raw[i] = rows::load_once<T, kVec>(from + i * kVec);
#pragma unroll
    for (int i = 0; i < 32 / kVec; ++i) {
      float2 part[kVec / 2];
      rows::unpack(raw[i], part);
#pragma unroll
      for (int j = 0; j < kVec / 2; ++j) u[i * (kVec / 2) + j] = part[j];
    }
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fmaxf(fabsf(u[i].x), fabsf(u[i].y)));
    const quant::Mxfp8Scale s = rows::block_scale(amax);
    Vec256 out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out.w[i] = rows::block_codes(u[2 * i], u[2 * i + 1], s);
    st_global_256(codes + row * cols + block * 32, out);
    byte = s.byte;
  }
  uint32_t word = byte | (__shfl_xor_sync(0xFFFFFFFFu, byte, 1) << 8);
  word |= __shfl_xor_sync(0xFFFFFFFFu, word, 2) << 16;
  if (row >= rows || (block & 3) != 0) return;
  const int e = groups::group_of_row(offsets, count, static_cast<int>(row));
  if (e == count) return;
  const int begin = groups::group_end(offsets, e - 1, rows);
  const int64_t to = groups::first_scale_block(begin, e) * 128 + row - begin;
  *reinterpret_cast<uint32_t*>(scales + swizzled_scale_offset(to, block, col_tiles)) = word;
}

// A word (one row, four blocks) a thread; the 128 words of a tile of x's scales beside one another.
__global__ void __launch_bounds__(256) regroup_scales_kernel(const uint8_t* from, const int* offsets, int count, int rows, int64_t col_tiles, uint8_t* scales) {
  const int64_t index = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, tile = index >> 7;
  const int64_t row_block = tile / col_tiles, col = tile - row_block * col_tiles, row = row_block * 128 + (index & 127);
  pdl_wait();
  pdl_launch_dependents();  // not earlier, as above
  if (row >= rows) return;
  const int e = groups::group_of_row(offsets, count, static_cast<int>(row));
  if (e == count) return;
  const int begin = groups::group_end(offsets, e - 1, rows);
  const int64_t to = groups::first_scale_block(begin, e) * 128 + row - begin;
  uint32_t word;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(word) : "l"(from + swizzled_scale_offset(row, col * 4, col_tiles)) : "memory");
  *reinterpret_cast<uint32_t*>(scales + swizzled_scale_offset(to, col * 4, col_tiles)) = word;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <int TILE_N, int NUM_ACC, int STAGES, int CTAS, typename OutT>
int launch_grouped(const void* a, const void* b, GroupedParams p, cudaStream_t stream) {
  using Cfg = GroupedConfig<TILE_N, NUM_ACC, STAGES, CTAS, static_cast<int>(sizeof(OutT))>;
  auto kernel = grouped_gemm_kernel<TILE_N, NUM_ACC, STAGES, CTAS, OutT>;
  int dev = 0;
  CK_CUDA(cudaGetDevice(&dev));
  RowMaps maps_x;
  CUtensorMap map_w, map_sfx = {}, map_sfw = {};
  for (int h = 0; h < 3; ++h) {
    if (int rc = make_operand_map(&maps_x.m[h], a, p.M, p.k_bytes, box_height(h))) return rc;
  }
  const int64_t row_blocks = groups::scale_blocks(p.M, p.groups);
  if (int rc = make_operand_map(&map_w, b, static_cast<int64_t>(p.groups) * p.N, p.k_bytes, CTAS == 2 ? kTileM : TILE_N)) return rc;
  if (CTAS == 2) {
    if (int rc = make_scale_map(&map_sfx, p.sfa, row_blocks, p.col_tiles, 1, Cfg::kSfbRowBlocks)) return rc;
    if (int rc = make_scale_map(&map_sfw, p.sfb, static_cast<int64_t>(p.groups) * p.n_row_blocks_b, p.col_tiles, 1, 1)) return rc;
  }
  p.tiles_n = static_cast<int>(ceil_div(p.N, CTAS == 2 ? 2 * kTileM : TILE_N));
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(num_threads(false, TILE_N));
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CTAS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // Pairs in plain stream order, as the input gradient's (launch_grad_gemm): what has no limit to its wait, the kernel in front, the tensor memory and the
  // cluster's barrier, then has nothing to wait for.
  cfg.numAttrs = pdl_enabled() && CTAS == 1 ? 2 : 1;
  // all workers resident at once; how many pairs there is room for depends on where the SMs lie
  static std::atomic<int> resident_on[64];
  int resident = (dev >= 0 && dev < 64) ? resident_on[dev].load(std::memory_order_acquire) : 0;
  if (resident == 0) {
    CK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
    resident = sm_count() / CTAS;
    if (CTAS > 1) {
      cfg.gridDim = dim3(resident * CTAS);
      int clusters = 0;
      CK_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg));
      if (clusters > 0 && clusters < resident) resident = clusters;
    }
    if (dev >= 0 && dev < 64) resident_on[dev].store(resident, std::memory_order_release);
  }
  // the most tiles that the groups can have; those that there are the device counts
  const int64_t used = p.groups < p.M ? p.groups : p.M;
  const int64_t items = (p.M / Cfg::kTileRows + used) * p.tiles_n;
  cfg.gridDim = dim3(CTAS * static_cast<unsigned>(items < resident ? items : resident));
  CK_CUDA(cudaLaunchKernelEx(&cfg, kernel, maps_x, map_w, map_sfx, map_sfw, p));
  return CK_OK;
}

template <typename OutT>
int launch_grouped_shape(const void* a, const void* b, const GroupedParams& p, cudaStream_t stream) {
  const int64_t used = p.groups < p.M ? p.groups : p.M, rows = ceil_div(p.M, used);  // of a group, if they are alike
  const int64_t tiles = used * ceil_div(rows, 128) * ceil_div(p.N, 128), stages = ceil_div(p.k_bytes, kStageKBytes);
  // Pairs for groups of more than 128 rows on average, where single CTAs would take turns and an SM's share is more than 32 stages: starting behind the
  // first kernel's end costs pairs three microseconds (us, pair / 128 x 128: tiles 1024, 140 rows each of 64 by 2048 x 2048 77 / 95; 640, 200 uneven of 40 by 1000 x
  // 1056 27.8 / 31.8; 256, 150 of 4 by 4096 x 4096 23.4 / 25.6; 512, 140 of 32 by 1024 x 1024 19.1 / 20.0; the other way 256, 1024 of 2 by 2048 x 2048 16.8 / 16.2; 384, 256 of 24 by 1024 x
  // 1024 22.2 / 18.9; 128, 256 of 8 by 1024 x 4096 24.9 / 19.9; fewer rows, 100 of 64 by 2048 x 2048 71 / 65, 113 of 8 by 4096 x 4096 36 / 32).  The average cannot tell uneven groups from
  // even ones: 117 uneven rows of 64 by 2048 x 2048 take 77 / 78.  Half tiles where whole ones leave half of the SMs without one (1 row of 1536 x 2048 8.8 / 9.1; 8 rows
  // of as many experts, 96 tiles, 14.1 / 10.4; 777 of 40 of 1000 x 1056 19.0 / 16.3).
  if (rows > 128 && tiles > sm_count() && tiles * stages > 32 * sm_count()) return launch_grouped<256, 1, 5, 2, OutT>(a, b, p, stream);
  if (tiles * 2 <= sm_count()) return launch_grouped<64, 2, 6, 1, OutT>(a, b, p, stream);
  return launch_grouped<128, 2, 5, 1, OutT>(a, b, p, stream);
}

bool is_float(int dtype) { return dtype == CK_DTYPE_F32 || dtype == CK_DTYPE_F16 || dtype == CK_DTYPE_BF16; }

struct GroupedLayout {
  int64_t codes_off, total;
};
GroupedLayout grouped_layout(int64_t M, int64_t K, int64_t count, bool from_float) {
  GroupedLayout l;
  l.codes_off = round_up(groups::scale_blocks(M, count) * ceil_div(K, 128) * 512, 256);
  l.total = l.codes_off + (from_float ? M * K : 0);
  return l;
}

int check_grouped(const char* op, int64_t M, int64_t N, int64_t K, int64_t E) {
  CK_REQUIRE(M > 0 && N > 0 && K > 0 && M < (1ll << 30) && N < (1ll << 30) && K < (1ll << 30), "%s: bad shape M=%lld N=%lld K=%lld", op,
             (long long)M, (long long)N, (long long)K);
  CK_REQUIRE(E > 0 && E <= groups::kMaxGroups, "%s: %lld groups, 1 to %d are supported", op, (long long)E, groups::kMaxGroups);
  CK_REQUIRE(K % 32 == 0 && N % 8 == 0, "%s: K=%lld must be a multiple of 32 and N=%lld of 8", op, (long long)K, (long long)N);
  CK_REQUIRE(E * round_up(N, 128) < (1ll << 31) && (ceil_div(M, 64) + E) * ceil_div(N > K ? N : K, 64) < (1ll << 30) &&
                 M * ceil_div(K, 128) < (1ll << 37), "%s: too large", op);
  return CK_OK;
}

int grouped_mm(const char* op, const void* x, int x_dtype, const void* x_scales, const void* b, const void* sfb, const int* offsets, const void* bias,
               int bias_dtype, void* out, int out_dtype, int64_t M, int64_t N, int64_t K, int64_t E, void* workspace, int64_t workspace_bytes,
               cudaStream_t s) {
  CK_REQUIRE(x && b && sfb && offsets && out && workspace, "%s: null pointer", op);
  if (int rc = check_grouped(op, M, N, K, E)) return rc;
  CK_REQUIRE(is_float(out_dtype) && (x_scales != nullptr || is_float(x_dtype)) && (bias == nullptr || is_float(bias_dtype)), "%s: unsupported dtype code", op);
  CK_REQUIRE(reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(b) % 16 == 0 && reinterpret_cast<uintptr_t>(sfb) % 16 == 0 &&
                 reinterpret_cast<uintptr_t>(x_scales) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                 reinterpret_cast<uintptr_t>(offsets) % 4 == 0 && reinterpret_cast<uintptr_t>(workspace) % 256 == 0,
             "%s: operands, scales and result have to be aligned to 16 bytes, the workspace to 256", op);
  const bool from_float = x_scales == nullptr;
  const GroupedLayout l = grouped_layout(M, K, E, from_float);
  CK_REQUIRE(workspace_bytes >= l.total, "%s: workspace of %lld bytes, %lld needed", op, (long long)workspace_bytes, (long long)l.total);
  uint8_t* scales = static_cast<uint8_t*>(workspace);
  uint8_t* codes = scales + l.codes_off;
  const int64_t col_tiles = ceil_div(K, 128);
  const int count = static_cast<int>(E), rows = static_cast<int>(M);
  if (from_float) {
    const dim3 grid(static_cast<unsigned>(ceil_div(M * col_tiles * 4, 256)));
    switch (x_dtype) {
      case CK_DTYPE_BF16:
        CK_CUDA(launch_pdl(quantize_groups_kernel<__nv_bfloat16>, grid, dim3(256), 0, s, static_cast<const __nv_bfloat16*>(x), offsets, count, rows, K, codes, scales));
        break;
      case CK_DTYPE_F16:
        CK_CUDA(launch_pdl(quantize_groups_kernel<__half>, grid, dim3(256), 0, s, static_cast<const __half*>(x), offsets, count, rows, K, codes, scales));
        break;
      default:
        CK_CUDA(launch_pdl(quantize_groups_kernel<float>, grid, dim3(256), 0, s, static_cast<const float*>(x), offsets, count, rows, K, codes, scales));
    }
  } else {
    CK_CUDA(launch_pdl(regroup_scales_kernel, dim3(static_cast<unsigned>(ceil_div(ceil_div(M, 128) * col_tiles * 128, 256))), dim3(256), 0, s,
                       static_cast<const uint8_t*>(x_scales), offsets, count, rows, col_tiles, scales));
  }
  GroupedParams p = {};
  p.offsets = offsets;
  p.sfa = scales;
  p.sfb = static_cast<const uint8_t*>(sfb);
  p.bias = bias;
  p.out = out;
  p.bias_dtype = bias_dtype;
  p.groups = count;
  p.M = rows;
  p.N = static_cast<int>(N);
  p.k_bytes = static_cast<int>(K);
  p.col_tiles = static_cast<int>(col_tiles);
  p.n_row_blocks_b = static_cast<int>(ceil_div(N, 128));
  if (int rc = gemm_status_word(&p.status)) return rc;
  const void* a = from_float ? codes : x;
  switch (out_dtype) {
    case CK_DTYPE_BF16: return launch_grouped_shape<__nv_bfloat16>(a, b, p, s);
    case CK_DTYPE_F16: return launch_grouped_shape<__half>(a, b, p, s);
    default: return launch_grouped_shape<float>(a, b, p, s);
  }
}

}  // namespace
}  // namespace ck

extern "C" int64_t ck_grouped_mm_mxfp8_workspace_bytes(int from_float, int64_t M, int64_t K, int64_t E) {
  if (M <= 0 || K <= 0 || E <= 0 || M >= (1ll << 30) || K >= (1ll << 30) || E > ck::groups::kMaxGroups) return 0;
  return ck::grouped_layout(M, K, E, from_float != 0).total;
}

extern "C" int ck_grouped_mm_mxfp8(const void* a, const void* b, const void* block_scale_a, const void* block_scale_b, const int* offsets, const void* bias,
                                   int bias_dtype, void* out, int out_dtype, int64_t M, int64_t N, int64_t K, int64_t E, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  CK_REQUIRE(block_scale_a != nullptr, "grouped_mm_mxfp8: null pointer");
  return ck::grouped_mm("grouped_mm_mxfp8", a, CK_DTYPE_F32, block_scale_a, b, block_scale_b, offsets, bias, bias_dtype, out, out_dtype, M, N, K, E, workspace,
                        workspace_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int ck_grouped_linear_mxfp8(const void* x, int x_dtype, const void* w, const void* w_scales, const int* offsets, const void* bias, int bias_dtype,
                                       void* out, int out_dtype, int64_t M, int64_t N, int64_t K, int64_t E, void* workspace, int64_t workspace_bytes,
                                       void* stream) {
  return ck::grouped_mm("grouped_linear_mxfp8", x, x_dtype, nullptr, w, w_scales, offsets, bias, bias_dtype, out, out_dtype, M, N, K, E, workspace,
                        workspace_bytes, static_cast<cudaStream_t>(stream));
}
