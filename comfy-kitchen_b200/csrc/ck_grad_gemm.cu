// Gradients of a linear layer one operand of which is held in MXFP8, for sm_100a:
//
//   weight:  dW[N, K] = sum_m dY[m, n] X[m, k]     X the MXFP8 copy of the layer's input   (and db[N] = sum_m dY[m, n])
//   input:   dX[M, K] = sum_n dY[m, n] W[n, k]     W the layer's MXFP8 weight
//
// Both contract over the rows of the MXFP8 matrix, whose scale blocks lie along its rows: the block-scaled MMA kinds, which
// contract along the blocks, do not apply.  An E4M3 number times a power of two has four significant bits, which bf16 holds
// exactly, so the products run on the bf16 tensor-core path with nothing lost: a first kernel writes the matrix as bf16 to the
// workspace (3 bytes of traffic an element beside 2 * M or 2 * N operations), and a GEMM over both follows.  dY in bf16 is an operand as it
// stands; in fp16 it is the exact sum of two bf16 numbers, in fp32 of three, and the GEMM contracts over all of them.
//
// The GEMM: CTA pairs on 256 x 256 tiles (cta_group::2, each CTA 128 rows of A and 128 columns of B), operands by TMA in
// stages of 64 contraction steps, two accumulators in tensor memory so that a tile's epilogue runs beside the next one's
// main loop.  B is row-major along the result's columns and A, for the weight's gradient, along the result's rows: both are
// read as MN-major operands, without a transposed copy.  Few tiles are split over the contraction, the partial sums going
// through the workspace to a kernel that adds them in a fixed order.
#include "ck_gemm_kernel.cuh"
#include "ck_rows.cuh"

namespace ck {
namespace {

constexpr int kGradStages = 6;
constexpr int kDeep = 64;                           // contraction steps of a stage: 128 bytes of bf16
constexpr int kOperandBytes = 128 * kDeep * 2;      // of A or B, stage and CTA
constexpr int kPairRows = 256, kPairCols = 256;     // a tile
constexpr int kBoxBytes = 64 * kDeep * 2;           // 64 rows (A) or columns (B) of an MN-major operand
constexpr int kGradSmem = 1024 + kGradStages * 2 * kOperandBytes + 256;
constexpr int kGradThreads = 32 * 10;               // producer, issuer, eight epilogue warps

// kind::f16: bf16 operands, fp32 accumulators; bit 15 / 16: A / B are MN-major
constexpr uint32_t grad_idesc(bool a_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((a_mn ? 1u : 0u) << 15) | (1u << 16) | ((kPairCols >> 3) << 17) | ((kPairRows >> 4) << 24);
}

struct GradParams {
  int rows, cols;       // of the result
  int deep_stages;      // stages of one of A's planes
  int planes;           // bf16 numbers whose sum is an element of dY
  int tiles_m, tiles_n;
  int splits, stages_per_split;
  void* out;            // the result, or fp32 partial sums [splits][rows][cols]
  int* status;
};

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

template <typename OutT, bool kMnA>
__global__ void __launch_bounds__(kGradThreads, 1)
grad_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GradParams p) {
  pdl_launch_dependents();
  const uint32_t rank = cluster_cta_rank();
  const int worker = blockIdx.x >> 1, workers = gridDim.x >> 1;
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
  static_assert((2 * kGradStages + 4) * 8 + 8 <= 256, "barrier area");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kGradStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full_bar[a], 1);
      mbar_init(&acc_empty_bar[a], 8 * 2);  // the epilogue warps of both CTAs
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
  const uint32_t tmem = *tmem_slot;

  const int tiles = p.tiles_m * p.tiles_n, items = tiles * p.splits, all_stages = p.deep_stages * p.planes;
  if (warp == 0) {
    // ---------------------------------------------------------------- loads
    if (elect_one()) {
      pdl_wait();
      const uint32_t full = smem_u32(full_bar), empty = smem_u32(empty_bar), a_addr = smem_u32(smem_a), b_addr = smem_u32(smem_b);
      int s = 0;
      uint32_t ph = 0;
      for (int item = worker; item < items; item += workers) {
        const int split = item / tiles;
        int tile_m, tile_n;
        tile_place(p, item - split * tiles, &tile_m, &tile_n);
        const int m0 = tile_m * kPairRows + static_cast<int>(rank) * 128, n0 = tile_n * kPairCols + static_cast<int>(rank) * 128;
        const int end = min(all_stages, (split + 1) * p.stages_per_split);
        for (int ks = split * p.stages_per_split; ks < end; ++ks) {
          const int plane = ks / p.deep_stages, l0 = (ks - plane * p.deep_stages) * kDeep;
          mbar_wait(empty + s * 8, ph ^ 1, abort_flag);
          const uint32_t bar = full + s * 8, a_to = a_addr + s * kOperandBytes, b_to = b_addr + s * kOperandBytes;
          if (rank == 0) mbar_arrive_expect_tx(bar, 2 * 2 * kOperandBytes);  // both CTAs' loads report to the leader
          if constexpr (kMnA) {
            tma_load_3d_pair(a_to, &map_a, bar, m0, l0, plane);
            tma_load_3d_pair(a_to + kBoxBytes, &map_a, bar, m0 + 64, l0, plane);
          } else {
            tma_load_3d_pair(a_to, &map_a, bar, l0, m0, plane);
          }
          tma_load_2d_pair(b_to, &map_b, bar, n0, l0);
          tma_load_2d_pair(b_to + kBoxBytes, &map_b, bar, n0 + 64, l0);
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
      pdl_wait();  // nothing lands earlier: keeps the bounded waits from running beside a long predecessor
      if (elect_one()) {
        const uint32_t full = smem_u32(full_bar), empty = smem_u32(empty_bar), acc_full = smem_u32(acc_full_bar);
        const uint32_t empty_peer = map_to_cta(empty, 1), acc_full_peer = map_to_cta(acc_full, 1);
        const uint64_t a0 = kMnA ? make_mn_desc(smem_u32(smem_a)) : make_operand_desc_sw128(smem_u32(smem_a));
        const uint64_t b0 = make_mn_desc(smem_u32(smem_b));
        constexpr uint32_t kIdesc = grad_idesc(kMnA);
        constexpr int kStepA = kMnA ? 2048 >> 4 : 32 >> 4, kStepB = 2048 >> 4;  // 16 contraction steps: 16 rows of 128 bytes, or 32 bytes
        int s = 0, it = 0;
        uint32_t ph = 0;
        for (int item = worker; item < items; item += workers, ++it) {
          const int split = item / tiles, begin = split * p.stages_per_split, end = min(all_stages, begin + p.stages_per_split);
          const int acc = it & 1;
          const uint32_t d = tmem + acc * kPairCols;
          mbar_wait(&acc_empty_bar[acc], ((it >> 1) & 1) ^ 1, abort_flag);
          tc_fence_after_sync();
          for (int ks = begin; ks < end; ++ks) {
            mbar_wait(full + s * 8, ph, abort_flag);
            tc_fence_after_sync();
            const uint64_t a = a0 + s * (kOperandBytes >> 4), b = b0 + s * (kOperandBytes >> 4);
#pragma unroll
            for (int k = 0; k < kDeep / 16; ++k) mma_bf16_pair(d, a + k * kStepA, b + k * kStepB, kIdesc, ks != begin || k != 0);
            tc_commit<2>(empty + s * 8);
            tc_commit<2>(empty_peer + s * 8);
            if (++s == kGradStages) {
              s = 0;
              ph ^= 1u;
            }
          }
          tc_commit<2>(acc_full + acc * 8);
          tc_commit<2>(acc_full_peer + acc * 8);
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- epilogue
    pdl_wait();  // the result's buffer may belong to the kernel before this one
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t acc_empty = map_to_cta(smem_u32(acc_empty_bar), 0);
    int it = 0;
    for (int item = worker; item < items; item += workers, ++it) {
      const int split = item / tiles, acc = it & 1;
      int tile_m, tile_n;
      tile_place(p, item - split * tiles, &tile_m, &tile_n);
      const int row = tile_m * kPairRows + static_cast<int>(rank) * 128 + quarter * 32 + lane;
      const int col0 = tile_n * kPairCols + half * 128;
      mbar_wait(&acc_full_bar[acc], (it >> 1) & 1, abort_flag);
      __syncwarp();
      tc_fence_after_sync();
      const uint32_t from = tmem + acc * kPairCols + (static_cast<uint32_t>(quarter * 32) << 16) + half * 128;
      OutT* out = static_cast<OutT*>(p.out) + (static_cast<int64_t>(split) * p.rows + row) * p.cols;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        tmem_load_32x32(from + c * 32, v);
        tmem_load_wait();
        if (c == 3) {  // read to the end: the accumulator goes back
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(acc_empty + acc * 8);
        }
        const int col = col0 + c * 32;
        if (row < p.rows && col < p.cols) {
          constexpr int kVec = 32 / static_cast<int>(sizeof(OutT));
#pragma unroll
          for (int i = 0; i < 32 / kVec; ++i) {
            float f[kVec];
#pragma unroll
            for (int j = 0; j < kVec; ++j) f[j] = __uint_as_float(v[i * kVec + j]);
            const rows::Raw<OutT, kVec> r = rows::pack<OutT, kVec>(f);
            st_global_256_no_allocate(out + col + i * kVec, *reinterpret_cast<const Vec256*>(&r));
          }
        }
        __syncwarp();
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

// dY as the sum of bf16 numbers: each takes the leading eight bits of what is left, so that three hold an fp32 number and two an
// fp16 one.  Infinities and NaN go into the first alone.
template <typename T, int kPlanes>
__global__ void __launch_bounds__(256) split_planes_kernel(const T* x, int64_t n, __nv_bfloat16* planes) {
  pdl_launch_dependents();
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  pdl_wait();
  if (i >= n) return;
  float left[4];
  rows::unpack(rows::load_once<T, 4>(x + i), left);
#pragma unroll
  for (int p = 0; p < kPlanes; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = __float_as_uint(left[j]) & 0xFFFF0000u;
      if (left[j] != left[j]) w[j] = 0x7FC00000u;
      left[j] = isfinite(left[j]) ? left[j] - __uint_as_float(w[j]) : 0.0f;
    }
    *reinterpret_cast<uint2*>(planes + p * n + i) = make_uint2((w[0] >> 16) | w[1], (w[2] >> 16) | w[3]);
  }
}

// db: 8 columns a thread, 32 of them beside one another and 8 rows above one another; `chunk` rows a block.  With one block for all
// rows (out != null) the result itself, else partial sums.
template <typename T, typename OutT>
__global__ void __launch_bounds__(256) column_sums_kernel(const T* x, int rows_, int cols, int chunk, float* partials, OutT* out) {
  __shared__ float buf[8][256 + 8];
  pdl_launch_dependents();
  const int col = (blockIdx.x * 32 + threadIdx.x) * 8, begin = blockIdx.y * chunk, end = min(rows_, begin + chunk);
  pdl_wait();
  float sum[8] = {};
  if (col < cols) {
    constexpr int kVec = 16 / static_cast<int>(sizeof(T));
#pragma unroll 4
    for (int r = begin + threadIdx.y; r < end; r += 8) {
      const T* at = x + static_cast<int64_t>(r) * cols + col;
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
  for (int j = 0; j < 8; ++j) buf[threadIdx.y][j * 32 + threadIdx.x] = sum[j];
  __syncthreads();
  const int t = threadIdx.y * 32 + threadIdx.x, c = (blockIdx.x * 32 + (t & 31)) * 8 + (t >> 5);
  if (c >= cols) return;
  float s = 0.0f;
#pragma unroll
  for (int y = 0; y < 8; ++y) s += buf[y][t];
  if (out != nullptr) {
    out[c] = rows::from_float<OutT>(s);
  } else {
    partials[static_cast<int64_t>(blockIdx.y) * cols + c] = s;
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
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
};
GradLayout grad_layout(bool weight, int dtype, bool bias, int64_t M, int64_t N, int64_t K) {
  GradLayout l = {};
  const GradShape g = {weight ? N : M, K, weight ? M : N, planes_of(dtype)};
  l.splits = grad_splits(g);
  l.planes_off = round_up((weight ? M : N) * K * 2, 256);
  l.partials_off = l.planes_off + (g.planes > 1 ? round_up(g.planes * M * N * 2, 256) : 0);
  l.sums_off = l.partials_off + (l.splits > 1 ? round_up(l.splits * g.rows * g.cols * 4, 256) : 0);
  // enough blocks to fill the chip twice, of 32 rows at least
  const int64_t strips = ceil_div(N, 256);
  int64_t chunks = ceil_div(2 * sm_count(), strips);
  if (chunks > ceil_div(M, 32)) chunks = ceil_div(M, 32);
  l.sum_chunks = static_cast<int>(bias ? chunks : 0);
  l.total = l.sums_off + (l.sum_chunks > 1 ? l.sum_chunks * N * 4 : 0);
  return l;
}

template <typename OutT, bool kMnA>
int launch_grad_gemm(const CUtensorMap& map_a, const CUtensorMap& map_b, const GradParams& p, cudaStream_t stream) {
  auto kernel = grad_gemm_kernel<OutT, kMnA>;
  int dev = 0;
  CK_CUDA(cudaGetDevice(&dev));
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kGradThreads);
  cfg.dynamicSmemBytes = kGradSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  // all pairs resident at once: how many there is room for depends on where the SMs lie
  static std::atomic<int> resident_on[64];
  int resident = (dev >= 0 && dev < 64) ? resident_on[dev].load(std::memory_order_acquire) : 0;
  if (resident == 0) {
    CK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGradSmem));
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

template <typename T, typename OutT>
int launch_column_sums(const void* dy, int64_t M, int64_t N, int chunks, float* partials, void* out, cudaStream_t s) {
  const int chunk = static_cast<int>(ceil_div(M, chunks)), blocks = static_cast<int>(ceil_div(M, chunk));
  const dim3 block(32, 8);
  const unsigned strips = static_cast<unsigned>(ceil_div(N, 256));
  OutT* const result = static_cast<OutT*>(out);
  auto kernel = column_sums_kernel<T, OutT>;
  CK_CUDA(launch_pdl(kernel, dim3(strips, blocks), block, 0, s, static_cast<const T*>(dy), static_cast<int>(M), static_cast<int>(N), chunk, partials,
                     blocks == 1 ? result : nullptr));
  if (blocks == 1) return CK_OK;
  auto join = column_sums_kernel<float, OutT>;
  CK_CUDA(launch_pdl(join, dim3(strips, 1), block, 0, s, static_cast<const float*>(partials), blocks, static_cast<int>(N), blocks,
                     static_cast<float*>(nullptr), result));
  return CK_OK;
}

template <typename T>
int launch_column_sums_typed(const void* dy, int64_t M, int64_t N, int chunks, float* partials, void* out, int out_dtype, cudaStream_t s) {
  switch (out_dtype) {
    case CK_DTYPE_BF16: return launch_column_sums<T, __nv_bfloat16>(dy, M, N, chunks, partials, out, s);
    case CK_DTYPE_F16: return launch_column_sums<T, __half>(dy, M, N, chunks, partials, out, s);
    default: return launch_column_sums<T, float>(dy, M, N, chunks, partials, out, s);
  }
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
  CK_REQUIRE(reinterpret_cast<uintptr_t>(dy) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 32 == 0 && reinterpret_cast<uintptr_t>(ws) % 256 == 0,
             "%s: dy, the result and the workspace have to be aligned to 16, 32 and 256 bytes", op);
  return CK_OK;
}

int linear_grad(bool weight, const char* op, const void* dy, int dtype, const void* codes, const void* scales, void* out, int out_dtype, void* dbias,
                int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, cudaStream_t s) {
  const GradLayout l = grad_layout(weight, dtype, dbias != nullptr, M, N, K);
  CK_REQUIRE(workspace_bytes >= l.total, "%s: workspace of %lld bytes, %lld needed", op, (long long)workspace_bytes, (long long)l.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const GradShape g = {weight ? N : M, K, weight ? M : N, planes_of(dtype)};
  if (int rc = ck_dequantize_mxfp8(codes, scales, ws, CK_DTYPE_BF16, g.deep, K, s)) return rc;
  const void* a = dy;
  if (g.planes > 1) {
    __nv_bfloat16* planes = reinterpret_cast<__nv_bfloat16*>(ws + l.planes_off);
    const int64_t n = M * N;
    const dim3 grid(static_cast<unsigned>(ceil_div(n, 1024)));
    if (dtype == CK_DTYPE_F32) {
      CK_CUDA(launch_pdl(split_planes_kernel<float, 3>, grid, dim3(256), 0, s, static_cast<const float*>(dy), n, planes));
    } else {
      CK_CUDA(launch_pdl(split_planes_kernel<__half, 2>, grid, dim3(256), 0, s, static_cast<const __half*>(dy), n, planes));
    }
    a = planes;
  }
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
  if (int rc = gemm_status_word(&p.status)) return rc;
  const int gemm_type = l.splits > 1 ? CK_DTYPE_F32 : out_dtype;
  if (int rc = weight ? launch_grad_gemm_typed<true>(map_a, map_b, p, gemm_type, s) : launch_grad_gemm_typed<false>(map_a, map_b, p, gemm_type, s)) return rc;
  if (l.splits > 1) {
    const float* partials = reinterpret_cast<const float*>(ws + l.partials_off);
    const int64_t n = g.rows * g.cols;
    int rc = CK_OK;
    switch (out_dtype) {
      case CK_DTYPE_BF16: rc = launch_add_splits<__nv_bfloat16>(partials, l.splits, n, out, s); break;
      case CK_DTYPE_F16: rc = launch_add_splits<__half>(partials, l.splits, n, out, s); break;
      default: rc = launch_add_splits<float>(partials, l.splits, n, out, s);
    }
    if (rc != CK_OK) return rc;
  }
  if (dbias == nullptr) return CK_OK;
  float* sums = reinterpret_cast<float*>(ws + l.sums_off);
  switch (dtype) {
    case CK_DTYPE_BF16: return launch_column_sums_typed<__nv_bfloat16>(dy, M, N, l.sum_chunks, sums, dbias, out_dtype, s);
    case CK_DTYPE_F16: return launch_column_sums_typed<__half>(dy, M, N, l.sum_chunks, sums, dbias, out_dtype, s);
    default: return launch_column_sums_typed<float>(dy, M, N, l.sum_chunks, sums, dbias, out_dtype, s);
  }
}

}  // namespace
}  // namespace ck

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
