// A linear layer's input gradient through its MXFP8 weight for few rows, sm_100a:  dX[M, K] = dY[M, N] . W[N, K].
//
// Bound by the weight's bytes (N K 33/32): the 38.9 MB of a 12288 x 3072 weight take 5.9 us at the copy rate.  The GEMM of ck_grad_gemm.cu would
// have the weight written as bf16 first and read that back (17 + 24 us for 8 rows; 20.6 here, 23.3 for 128 rows).  Here the weight is decoded on its way into the operand: a CTA takes
// 128 columns of W and a range of its rows; codes and scales of 64 rows at a time come by TMA, sixteen warps decode them (exactly, to
// bf16) and write them to shared memory as an MN-major operand, the columns of W being the MMA's 128 rows; dY comes by TMA as the
// other operand, its rows being the MMA's columns (16 to 208 of them); one thread issues the MMAs.  Decoding has no
// exchange between lanes: adjacent codes of a row are adjacent in the operand.
//
// The CTAs of a cluster share a strip's rows and add their sums through distributed shared memory, in their order.
// Warp-wide MMAs (m16n8k16) in place of tcgen05 took 17 to 28 us for these sizes: one takes about 40 cycles here, and its
// fragments want two rows' codes in one register.  dY in fp16 or fp32 enters as two or three bf16 numbers, exactly, as in the GEMM.
//
// Rows that are grouped by expert, few for each: the same stages in a kernel that stays.  A CTA takes tiles of up to a.padded rows of one group by
// 128 columns one after another; its steps are numbered through all of them, so that the rings and their phases go on from tile to tile, and four
// more warps store a tile's result while the others are at the next one.
#include <atomic>

#include "ck_gemm_kernel.cuh"
#include "ck_groups.cuh"
#include "ck_rows.cuh"

namespace ck {
namespace {

using namespace rows;

constexpr int kCols = 128, kDeep = 64;           // of W: columns of a strip, rows of a stage
constexpr int kCodeWarps = 16;                   // warps that decode, and store the result
constexpr int kThreads = 32 * (kCodeWarps + 2);  // beside them the loads of dY and the MMAs
constexpr int kHeldBytes = kDeep * kCols * 2;    // of a stage
constexpr int kBoxBytes = kDeep * 128;           // 64 columns of it
// Four groups of warps decode stages in turn: a stage is a chain of waits, conversions, stores and a fence, which sixteen warps at one stage
// ran through in step (28 us for 8 rows of 12288 x 3072, in turn 20; codes read into registers ahead of their use, 24 whether 5, 8 or 12 stages ahead).
constexpr int kGroups = 4, kGroupWarps = kCodeWarps / kGroups;
// The operands' stages, at least four: a group's wait for its stage to be free goes by the parity of the phase, and what it has waited for
// before must leave no doubt which phase that is.  At its step j it knows that the MMAs of step j - 4 - stages are done (its step before
// waited for them), and has to know that of those of step j - 2 * stages.
constexpr int kMinStages = 4, kMaxStages = 6;
// The ring of codes and scales as they come, four or eight stages: multiples of the groups, so that every use of a stage is the same group's and its
// waits see every phase.
constexpr int kScaleBytes = 512, kRawBytes = kDeep * kCols + kScaleBytes;  // a stage's codes, the tile with its scales
constexpr int kMaxRaw = 8;
static_assert(kMaxRaw % kGroups == 0 && kMinStages >= kGroups, "no wait may take one phase for another");
constexpr int kSmem = 208 * 1024;
static_assert(alone_with_tensor_memory(kSmem), "no allocation of tensor memory waits");

struct FewRowsArgs {
  const uint8_t* codes;
  const uint8_t* scales;
  void* out;
  int out_dtype;
  int M, N, K;
  int padded;  // M as a multiple of 16
  int planes;  // bf16 numbers whose sum is an element of dY
  int parts;   // accumulators that the first of them take in turn; the others have one each, in front of these
  int stages, raw_stages;
  int steps_per_split;  // of 64 rows of W
  int* status;          // for waits that give up (ck_gemm_status)
};

__device__ __forceinline__ void mma_bf16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

template <typename OutT>
__device__ __forceinline__ void store_one(void* out, int64_t at, float v) {
  static_cast<OutT*>(out)[at] = from_float<OutT>(v);
}
__device__ __forceinline__ void store_result(const FewRowsArgs& a, int64_t at, float v) {
  if (a.out_dtype == CK_DTYPE_BF16) {
    store_one<__nv_bfloat16>(a.out, at, v);
  } else if (a.out_dtype == CK_DTYPE_F16) {
    store_one<__half>(a.out, at, v);
  } else {
    store_one<float>(a.out, at, v);
  }
}

// Codes and a scale's byte as they came to shared memory.  They are used behind a wait, and their place is given back in front of it, so nothing but a fence
// between the proxies puts these reads before the next copy's writes: an arrival on a barrier does not.  Without it a warp's reads, held up where the MMAs keep shared memory busy,
// met the codes of four steps later, in 3 to 70 passes of a hundred of one build (200 rows of bf16, 4864 x 256 and 4864 x 8192) and in none of another.  (Giving the place back behind
// the decoding needs no fence and costs 4 % where four stages of codes are all there is room for: 64 experts of 2048 x 2048, 200 rows each, 126.7 us instead of 123.5.)
__device__ __forceinline__ uint4 load_codes(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t load_scale(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// Four codes -> four bf16 numbers times `factor`.
__device__ __forceinline__ uint2 decode_four(uint32_t codes, float2 factor) {
  uint32_t lo, hi;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
  const float2 a = mul_x2(__half22float2(*reinterpret_cast<const __half2*>(&lo)), factor);
  const float2 b = mul_x2(__half22float2(*reinterpret_cast<const __half2*>(&hi)), factor);
  const __nv_bfloat162 p = __floats2bfloat162_rn(a.x, a.y), q = __floats2bfloat162_rn(b.x, b.y);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&p), *reinterpret_cast<const uint32_t*>(&q));
}

__global__ void __launch_bounds__(kThreads)
grad_few_rows_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_codes, const FewRowsArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], raw_full_bar[kMaxRaw], raw_empty_bar[kMaxRaw], done_bar;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  pdl_launch_dependents();
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));  // the operands' stages
  uint8_t* const raw = smem + a.stages * (kHeldBytes + a.planes * a.padded * 128);                                       // the codes' stages
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, splits = gridDim.x, strip = blockIdx.y;
  const int steps = (a.N + kDeep - 1) / kDeep, first = split * a.steps_per_split, last = min(steps, first + a.steps_per_split);
  const int plane_bytes = a.padded * 128, stage_bytes = kHeldBytes + a.planes * plane_bytes;
  const int minor = a.planes - 1, accumulators = minor + min(a.parts, last - first);
  uint32_t tmem_cols = 32;
  while (static_cast<int>(tmem_cols) < (minor + a.parts) * a.padded) tmem_cols *= 2;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full_bar[s], kGroupWarps + 1);  // the decoding warps, the loads of dY
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < a.raw_stages; ++s) {
      mbar_init(&raw_full_bar[s], 1);
      mbar_init(&raw_empty_bar[s], kGroupWarps);
    }
    mbar_init(&done_bar, 1);
    fence_barrier_init();
    prefetch_tensormap(&map_dy);
    prefetch_tensormap(&map_codes);
  }
  if (warp == kCodeWarps + 1) tmem_alloc<1>(&tmem_slot, tmem_cols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const uint32_t full = smem_u32(full_bar), empty = smem_u32(empty_bar), raw_full = smem_u32(raw_full_bar), raw_empty = smem_u32(raw_empty_bar);
  pdl_wait();

  if (warp < kCodeWarps) {
    // ---------------------------------------------------------------- decoding
    // A thread takes 16 columns of four rows, 16 apart.  The eight lanes of a phase of 16-byte accesses have column units 0 to 3 of a row and 4 to 7 of the
    // next, or the other way round: different banks in the codes as they come, and with the 128-byte swizzle in the operand.
    constexpr int kItems = kDeep / (4 * kGroupWarps);
    const int group = warp / kGroupWarps, odd = (lane >> 2) & 1, unit = (lane & 3) + (odd ^ ((lane >> 3) & 1)) * 4;
    const int row0 = warp % kGroupWarps * 4 + odd + (lane >> 4) * 2;
    const uint32_t code_at = smem_u32(raw) + row0 * kCols + unit * 16, scale_at = smem_u32(raw) + kDeep * kCols + (unit >> 1);
    const uint32_t row_at = smem_u32(smem) + (unit >> 2) * kBoxBytes + row0 * 128;
    const uint32_t low = ((unit & 3) * 2) ^ (row0 & 7), high = low ^ 1;  // the same for rows 16 apart
    int stage = group, raw_stage = group;
    uint32_t phase = 0, raw_phase = 0;
    for (int step = first + group; step < last; step += kGroups) {
      mbar_wait(raw_full + raw_stage * 8, raw_phase, &abort_flag);
      uint4 codes[kItems];
      uint32_t byte[kItems];
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int row = row0 + 4 * kGroupWarps * i;
        codes[i] = load_codes(code_at + raw_stage * kRawBytes + 4 * kGroupWarps * i * kCols);
        byte[i] = load_scale(scale_at + raw_stage * kRawBytes + (row & 31) * 16 + (row >> 5) * 4 + (step & 1) * 8);  // a tile of scales is two stages high
      }
      if (const int left = a.N - step * kDeep; left < kDeep) {  // what stands in rows past the last one is nobody's: infinite, it would make NaN of zeros
#pragma unroll
        for (int i = 0; i < kItems; ++i) byte[i] = row0 + 4 * kGroupWarps * i < left ? byte[i] : 0u;
      }
      fence_proxy_async();  // read before the next copy into this place (load_codes)
      __syncwarp();
      if (lane == 0) mbar_arrive(&raw_empty_bar[raw_stage]);
      mbar_wait(empty + stage * 8, phase ^ 1, &abort_flag);
      const uint32_t to = row_at + stage * stage_bytes;
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const float2 factor = both(e8m0_factor(byte[i]));
        const uint2 v0 = decode_four(codes[i].x, factor), v1 = decode_four(codes[i].y, factor);
        const uint2 v2 = decode_four(codes[i].z, factor), v3 = decode_four(codes[i].w, factor);
        st_shared_128(to + 4 * kGroupWarps * i * 128 + (low << 4), v0.x, v0.y, v1.x, v1.y);
        st_shared_128(to + 4 * kGroupWarps * i * 128 + (high << 4), v2.x, v2.y, v3.x, v3.y);
      }
      fence_proxy_async();  // the MMAs read what was written here
      __syncwarp();
      if (lane == 0) mbar_arrive(&full_bar[stage]);
      stage += kGroups;
      if (stage >= a.stages) {
        stage -= a.stages;
        phase ^= 1u;
      }
      raw_stage += kGroups;
      if (raw_stage >= a.raw_stages) {
        raw_stage -= a.raw_stages;
        raw_phase ^= 1u;
      }
    }
    // ---------------------------------------------------------------- result
    // A warp has 32 of the strip's columns, one a lane, and every fourth 16 rows of dX.
    mbar_wait(&done_bar, 0, &abort_flag);
    __syncwarp();
    tc_fence_after_sync();
    const int quarter = warp & 3, k = strip * kCols + quarter * 32 + lane;
    float* const sums = reinterpret_cast<float*>(smem);  // [padded][kCols], where a cluster adds
    for (int m0 = (warp >> 2) * 16; m0 < a.padded; m0 += kCodeWarps * 4) {
      float f[16] = {};
      for (int n = 0; n < accumulators; ++n) {
        uint32_t v[16];
        tmem_load_32x16(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + n * a.padded + m0, v);
        tmem_load_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] += __uint_as_float(v[i]);
      }
      if (splits > 1) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[(m0 + i) * kCols + quarter * 32 + lane] = f[i];
      } else if (k < a.K) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (m0 + i < a.M) store_result(a, static_cast<int64_t>(m0 + i) * a.K + k, f[i]);
        }
      }
      __syncwarp();
    }
    tc_fence_before_sync();
  } else if (warp == kCodeWarps) {
    // ---------------------------------------------------------------- loads: codes and scales as far ahead as their ring goes, dY with its stage
    if (elect_one()) {
      const int64_t col_tiles = (a.K / 32 + 3) >> 2;
      int stage = 0, raw_stage = 0, ahead = first;
      uint32_t phase = 0, raw_phase = 0;
      const auto fetch = [&]() {
        mbar_wait(raw_empty + raw_stage * 8, raw_phase ^ 1, &abort_flag);
        const uint32_t bar = raw_full + raw_stage * 8, to = smem_u32(raw) + raw_stage * kRawBytes;
        mbar_arrive_expect_tx(bar, kRawBytes);
        tma_load_2d(to, &map_codes, bar, strip * kCols, ahead * kDeep);
        bulk_load_1d(to + kDeep * kCols, a.scales + ((ahead >> 1) * col_tiles + strip) * kScaleBytes, kScaleBytes, bar);
        ++ahead;
        if (++raw_stage == a.raw_stages) {
          raw_stage = 0;
          raw_phase ^= 1u;
        }
      };
      while (ahead < last && ahead < first + a.raw_stages) fetch();
      for (int step = first; step < last; ++step) {
        mbar_wait(empty + stage * 8, phase ^ 1, &abort_flag);
        const uint32_t bar = full + stage * 8, to = smem_u32(smem) + stage * stage_bytes + kHeldBytes;
        mbar_arrive_expect_tx(bar, a.planes * plane_bytes);
        for (int p = 0; p < a.planes; ++p) {
          asm volatile(
              "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to + p * plane_bytes),
              "l"(reinterpret_cast<uint64_t>(&map_dy)), "r"(bar), "r"(step * kDeep), "r"(0), "r"(p)
              : "memory");
        }
        if (++stage == a.stages) {
          stage = 0;
          phase ^= 1u;
        }
        if (ahead < last) fetch();
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- MMAs
    if (elect_one()) {
      // kind::f16: bf16 operands, fp32 sums, A (W's columns) MN-major in boxes of 64 columns, B (dY's rows) K-major
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (static_cast<uint32_t>(a.padded >> 3) << 17) | ((kCols >> 4) << 24);
      int stage = 0, part = 0;
      uint32_t phase = 0;
      for (int step = first; step < last; ++step) {
        mbar_wait(full + stage * 8, phase, &abort_flag);
        tc_fence_after_sync();
        const uint32_t at = smem_u32(smem) + stage * stage_bytes;
        const uint64_t held = make_smem_desc(at, kBoxBytes, 1024, 2);
        for (int p = 0; p < a.planes; ++p) {
          const uint32_t to = tmem + (p == 0 ? (minor + part) * a.padded : (minor - p) * a.padded);  // the smallest in front
          const bool begins = step == first + (p == 0 ? part : 0);
          const uint64_t dy = make_operand_desc_sw128(at + kHeldBytes + p * plane_bytes);
#pragma unroll
          for (int i = 0; i < kDeep / 16; ++i) {  // 16 rows of 128 bytes, 32 bytes
            mma_bf16(to, held + i * (2048 >> 4), dy + i * (32 >> 4), idesc, !begins || i != 0);
          }
        }
        tc_commit<1>(empty + stage * 8);
        if (++part == a.parts) part = 0;
        if (++stage == a.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      tc_commit<1>(smem_u32(&done_bar));
    }
    __syncwarp();
  }
  __syncthreads();
  tc_fence_after_sync();
  if (splits > 1) {
    cluster_sync_all();
    // this CTA's share of the tile, over the cluster's CTAs
    const uint32_t own = smem_u32(smem);
    for (int i = split * kThreads + threadIdx.x; i < a.M * (kCols / 4); i += splits * kThreads) {
      float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int r = 0; r < splits; ++r) {
        const float4 p = ld_shared_cluster_f32x4(map_to_cta(own + i * 16, r));
        s.x += p.x;
        s.y += p.y;
        s.z += p.z;
        s.w += p.w;
      }
      const int m = i / (kCols / 4), k = strip * kCols + i % (kCols / 4) * 4;
      if (k >= a.K) continue;
      const int64_t at = static_cast<int64_t>(m) * a.K + k;
      const float f[4] = {s.x, s.y, s.z, s.w};
      if (a.out_dtype == CK_DTYPE_BF16) {
        store(static_cast<__nv_bfloat16*>(a.out) + at, pack<__nv_bfloat16, 4>(f));
      } else if (a.out_dtype == CK_DTYPE_F16) {
        store(static_cast<__half*>(a.out) + at, pack<__half, 4>(f));
      } else {
        store(static_cast<float*>(a.out) + at, pack<float, 4>(f));
      }
    }
    cluster_sync_all();  // no CTA leaves while another may still read its sums
  }
  if (abort_flag) {
    if (threadIdx.x == 0) atomicExch(a.status, 1);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
    __syncthreads();
  }
  if (warp == kCodeWarps + 1) tmem_dealloc<1>(tmem, tmem_cols);
}

// ---- grouped rows --------------------------------------------------------------------------------------------
// dX[i] = dY[i] W_e for the rows i of group e: the same operand, but blocks that stay and take tiles (a group's rows, 128 columns of W_e) in turn, accumulators in two
// sets, so that a tile is stored beside the next one's steps, and loads of dY and of codes by warps of their own.  Bound by the decoding, 2.9 million codes a microsecond: 64
// groups of 32 rows, 2048 x 2048 each, bf16 94 us (fp32, three numbers an element, 143); eight rows of as many groups, 1536 x 2048, 13.6.
constexpr int kRowBox = 16;  // rows of dY in a copy
constexpr int kStoreWarps = 4, kGroupedThreads = kThreads + 32 * (kStoreWarps + 1);  // beside those of the kernel above, and the loads of dY apart from the codes

struct GroupedFewRowsArgs {
  const uint8_t* scales;
  void* out;
  const int* offsets;
  int out_dtype;
  int groups, M, N, K;
  int padded;       // rows of a tile at most, a multiple of kRowBox
  int planes;       // bf16 numbers whose sum is an element of dY
  int parts;        // accumulators that the first of them take in turn; the others have one each, in front of these
  int sets;         // of accumulators: two where tensor memory holds them, so that a tile is stored beside the next one's steps
  int stages, raw_stages;
  int strips;
  int* status;
};

__global__ void __launch_bounds__(kGroupedThreads)
grouped_few_rows_kernel(const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_dy_whole,
                        const __grid_constant__ CUtensorMap map_codes, const GroupedFewRowsArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], raw_full_bar[kMaxRaw], raw_empty_bar[kMaxRaw], acc_full_bar[2], acc_empty_bar[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  pdl_launch_dependents();
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));  // the operands' stages
  uint8_t* const raw = smem + a.stages * (kHeldBytes + a.planes * a.padded * 128);                                       // the codes' stages
  groups::Table* const table = reinterpret_cast<groups::Table*>(raw + a.raw_stages * kRawBytes);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int steps = (a.N + kDeep - 1) / kDeep;
  const int plane_bytes = a.padded * 128, stage_bytes = kHeldBytes + a.planes * plane_bytes;
  const int minor = a.planes - 1, set_cols = (minor + a.parts) * a.padded;
  uint32_t tmem_cols = 32;
  while (static_cast<int>(tmem_cols) < a.sets * set_cols) tmem_cols *= 2;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(&full_bar[s], kGroupWarps + 1);  // the decoding warps, the loads of dY
      mbar_init(&empty_bar[s], 1);
    }
    for (int s = 0; s < a.raw_stages; ++s) {
      mbar_init(&raw_full_bar[s], 1);
      mbar_init(&raw_empty_bar[s], kGroupWarps);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full_bar[s], 1);
      mbar_init(&acc_empty_bar[s], kStoreWarps);
    }
    fence_barrier_init();
    prefetch_tensormap(&map_dy);
    prefetch_tensormap(&map_dy_whole);
    prefetch_tensormap(&map_codes);
  }
  if (warp == kCodeWarps + 1) tmem_alloc<1>(&tmem_slot, tmem_cols);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  const uint32_t full = smem_u32(full_bar), empty = smem_u32(empty_bar), raw_full = smem_u32(raw_full_bar), raw_empty = smem_u32(raw_empty_bar);
  pdl_wait();
  groups::fill_table(table, a.offsets, a.groups, a.M, a.padded);
  // Tiles of this CTA: items worker, worker + workers, ...  Its steps count through them.
  const int items = table->tiles[a.groups] * a.strips, worker = blockIdx.x, workers = gridDim.x;
  const int mine = worker < items ? (items - worker + workers - 1) / workers : 0;
  const auto place = [&](int i) { return groups::place(table, a.groups, a.strips, a.padded, worker + i * workers); };

  if (warp < kCodeWarps) {
    // ---------------------------------------------------------------- decoding
    const int group = warp / kGroupWarps, odd = (lane >> 2) & 1, unit = (lane & 3) + (odd ^ ((lane >> 3) & 1)) * 4;
    const int row0 = warp % kGroupWarps * 4 + odd + (lane >> 4) * 2;
    const uint32_t code_at = smem_u32(raw) + row0 * kCols + unit * 16, scale_at = smem_u32(raw) + kDeep * kCols + (unit >> 1);
    const uint32_t row_at = smem_u32(smem) + (unit >> 2) * kBoxBytes + row0 * 128;
    const uint32_t low = ((unit & 3) * 2) ^ (row0 & 7), high = low ^ 1;  // the same for rows 16 apart
    constexpr int kItems = kDeep / (4 * kGroupWarps);
    int stage = group, raw_stage = group;
    uint32_t phase = 0, raw_phase = 0;
    int step = group;  // within its tile
    for (int left_tiles = mine; left_tiles > 0; step += kGroups) {
      while (step >= steps) {
        step -= steps;
        if (--left_tiles == 0) break;
      }
      if (left_tiles == 0) break;
      mbar_wait(raw_full + raw_stage * 8, raw_phase, &abort_flag);
      uint4 codes[kItems];
      uint32_t byte[kItems];
      const int left = a.N - step * kDeep;  // what stands for rows past the last one is nobody's
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const int row = row0 + 4 * kGroupWarps * i;
        codes[i] = load_codes(code_at + raw_stage * kRawBytes + 4 * kGroupWarps * i * kCols);
        byte[i] = load_scale(scale_at + raw_stage * kRawBytes + (row & 31) * 16 + (row >> 5) * 4 + (step & 1) * 8);  // a tile of scales is two stages high
        if (row >= left) byte[i] = 0;
      }
      fence_proxy_async();  // read before the next copy into this place (load_codes)
      __syncwarp();
      if (lane == 0) mbar_arrive(&raw_empty_bar[raw_stage]);
      mbar_wait(empty + stage * 8, phase ^ 1, &abort_flag);
      const uint32_t to = row_at + stage * stage_bytes;
#pragma unroll
      for (int i = 0; i < kItems; ++i) {
        const float2 factor = both(e8m0_factor(byte[i]));
        const uint2 v0 = decode_four(codes[i].x, factor), v1 = decode_four(codes[i].y, factor);
        const uint2 v2 = decode_four(codes[i].z, factor), v3 = decode_four(codes[i].w, factor);
        st_shared_128(to + 4 * kGroupWarps * i * 128 + (low << 4), v0.x, v0.y, v1.x, v1.y);
        st_shared_128(to + 4 * kGroupWarps * i * 128 + (high << 4), v2.x, v2.y, v3.x, v3.y);
      }
      fence_proxy_async();  // the MMAs read what was written here
      __syncwarp();
      if (lane == 0) mbar_arrive(&full_bar[stage]);
      stage += kGroups;
      if (stage >= a.stages) {
        stage -= a.stages;
        phase ^= 1u;
      }
      raw_stage += kGroups;
      if (raw_stage >= a.raw_stages) {
        raw_stage -= a.raw_stages;
        raw_phase ^= 1u;
      }
    }
  } else if (warp == kCodeWarps) {
    // ---------------------------------------------------------------- loads of codes and scales, as far ahead as their ring goes
    if (elect_one()) {
      const int64_t col_tiles = (a.K / 32 + 3) >> 2, group_tiles = (a.N + 127) / 128 * col_tiles;
      int raw_stage = 0;
      uint32_t raw_phase = 0;
      for (int i = 0; i < mine; ++i) {
        const groups::Tile t = place(i);
        const uint8_t* const scales = a.scales + (t.group * group_tiles + t.tile_n) * kScaleBytes;
        for (int step = 0; step < steps; ++step) {
          mbar_wait(raw_empty + raw_stage * 8, raw_phase ^ 1, &abort_flag);
          const uint32_t bar = raw_full + raw_stage * 8, to = smem_u32(raw) + raw_stage * kRawBytes;
          mbar_arrive_expect_tx(bar, kRawBytes);
          asm volatile(
              "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(to),
              "l"(reinterpret_cast<uint64_t>(&map_codes)), "r"(bar), "r"(t.tile_n * kCols), "r"(step * kDeep), "r"(t.group)
              : "memory");
          bulk_load_1d(to + kDeep * kCols, scales + (step >> 1) * col_tiles * kScaleBytes, kScaleBytes, bar);
          if (++raw_stage == a.raw_stages) {
            raw_stage = 0;
            raw_phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == kCodeWarps + 2) {
    // ---------------------------------------------------------------- loads of dY
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < mine; ++i) {
        const groups::Tile t = place(i);
        // a tile's rows of dY in one box where it has more than half of them, in boxes of 16 otherwise
        const int count = min(a.padded, t.end - t.row);
        const bool whole = 2 * count > a.padded;
        const int boxes = whole ? 1 : (count + kRowBox - 1) / kRowBox, box_rows = whole ? a.padded : kRowBox;
        const CUtensorMap* const map = whole ? &map_dy_whole : &map_dy;
        for (int step = 0; step < steps; ++step) {
          mbar_wait(empty + stage * 8, phase ^ 1, &abort_flag);
          const uint32_t bar = full + stage * 8, to = smem_u32(smem) + stage * stage_bytes + kHeldBytes;
          mbar_arrive_expect_tx(bar, a.planes * boxes * box_rows * 128);
          for (int p = 0; p < a.planes; ++p) {
            for (int b = 0; b < boxes; ++b) {
              asm volatile(
                  "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                      to + p * plane_bytes + b * (kRowBox * 128)),
                  "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(step * kDeep), "r"(t.row + b * kRowBox), "r"(p)
                  : "memory");
            }
          }
          if (++stage == a.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == kCodeWarps + 1) {
    // ---------------------------------------------------------------- MMAs
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; i < mine; ++i) {
        // as many of the MMA's columns as the tile has rows, in sixteens
        const groups::Tile t = place(i);
        const uint32_t columns = (min(a.padded, t.end - t.row) + 15) / 16 * 16;
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | ((columns >> 3) << 17) | ((kCols >> 4) << 24);
        const int set = a.sets == 2 ? i & 1 : 0;
        const uint32_t base = tmem + set * set_cols;
        mbar_wait(&acc_empty_bar[set], ((i / a.sets) & 1) ^ 1, &abort_flag);
        tc_fence_after_sync();
        int part = 0;
        for (int step = 0; step < steps; ++step) {
          mbar_wait(full + stage * 8, phase, &abort_flag);
          tc_fence_after_sync();
          const uint32_t at = smem_u32(smem) + stage * stage_bytes;
          const uint64_t held = make_smem_desc(at, kBoxBytes, 1024, 2);
          for (int p = 0; p < a.planes; ++p) {
            const uint32_t to = base + (p == 0 ? (minor + part) * a.padded : (minor - p) * a.padded);  // the smallest in front
            const bool begins = step == (p == 0 ? part : 0);
            const uint64_t dy = make_operand_desc_sw128(at + kHeldBytes + p * plane_bytes);
#pragma unroll
            for (int q = 0; q < kDeep / 16; ++q) {  // 16 rows of 128 bytes, 32 bytes
              mma_bf16(to, held + q * (2048 >> 4), dy + q * (32 >> 4), idesc, !begins || q != 0);
            }
          }
          tc_commit<1>(empty + stage * 8);
          if (++part == a.parts) part = 0;
          if (++stage == a.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        tc_commit<1>(smem_u32(&acc_full_bar[set]));
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- results: a warp has 32 of the strip's columns, one a lane
    const int quarter = warp & 3, accumulators = minor + min(a.parts, steps);
    for (int i = 0; i < mine; ++i) {
      const groups::Tile t = place(i);
      const int set = a.sets == 2 ? i & 1 : 0, k = t.tile_n * kCols + quarter * 32 + lane, count = min(a.padded, t.end - t.row);
      mbar_wait(&acc_full_bar[set], (i / a.sets) & 1, &abort_flag);
      __syncwarp();
      tc_fence_after_sync();
      for (int m0 = 0; m0 < count; m0 += 16) {
        float f[16] = {};
        for (int n = 0; n < accumulators; ++n) {
          uint32_t v[16];
          tmem_load_32x16(tmem + set * set_cols + (static_cast<uint32_t>(quarter * 32) << 16) + n * a.padded + m0, v);
          tmem_load_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) f[j] += __uint_as_float(v[j]);
        }
        if (m0 + 16 >= count) {  // read to the end
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&acc_empty_bar[set]);
        }
        if (k < a.K) {
          const int64_t at = static_cast<int64_t>(t.row + m0) * a.K + k;
          const auto store_rows = [&](auto* out) {
            using OutT = std::remove_pointer_t<decltype(out)>;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              if (m0 + j < count) out[at + static_cast<int64_t>(j) * a.K] = from_float<OutT>(f[j]);
            }
          };
          if (a.out_dtype == CK_DTYPE_BF16) {
            store_rows(static_cast<__nv_bfloat16*>(a.out));
          } else if (a.out_dtype == CK_DTYPE_F16) {
            store_rows(static_cast<__half*>(a.out));
          } else {
            store_rows(static_cast<float*>(a.out));
          }
        }
        __syncwarp();
      }
    }
    // rows behind the last group, in units of 16 bytes (K is a multiple of 32)
    const int64_t size = a.out_dtype == CK_DTYPE_F32 ? 4 : 2;
    const int64_t begin = static_cast<int64_t>(table->bound[a.groups]) * a.K * size, end = static_cast<int64_t>(a.M) * a.K * size;
    for (int64_t at = begin + (static_cast<int64_t>(blockIdx.x) * (32 * kStoreWarps) + threadIdx.x - (kGroupedThreads - 32 * kStoreWarps)) * 16; at < end;
         at += static_cast<int64_t>(gridDim.x) * (32 * kStoreWarps) * 16) {
      *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.out) + at) = make_uint4(0, 0, 0, 0);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (abort_flag) {
    if (threadIdx.x == 0) atomicExch(a.status, 1);
    for (int i = 0; i < 200; ++i) __nanosleep(1000);  // copies that are in flight land before the memory is released
    __syncthreads();
  }
  if (warp == kCodeWarps + 1) tmem_dealloc<1>(tmem, tmem_cols);
}

int make_code_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols) {
  return cached_map(map, MapKey{12, base, rows, cols, kDeep, 0}, [&](CUtensorMap* m) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(CK_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols)};
    const cuuint32_t box[2] = {kCols, kDeep};
    const cuuint32_t elem_strides[2] = {1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(CK_ERR_CUDA, "cuTensorMapEncodeTiled (codes) failed with code %d", static_cast<int>(r));
    return static_cast<int>(CK_OK);
  });
}

// Clusters of `splits` CTAs that run at once: a cluster has to find its SMs in one part of the chip.
int clusters_at_once(int splits, int* out) {
  static std::atomic<int> known[64][9];
  int dev = 0;
  CK_CUDA(cudaGetDevice(&dev));
  const bool cached = dev >= 0 && dev < 64;
  int n = cached ? known[dev][splits].load(std::memory_order_acquire) : 0;
  if (n == 0) {
    CK_CUDA(cudaFuncSetAttribute(grad_few_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, 148);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    CK_CUDA(cudaOccupancyMaxActiveClusters(&n, grad_few_rows_kernel, &cfg));
    if (n < 1) n = 1;
    if (cached) known[dev][splits].store(n, std::memory_order_release);
  }
  *out = n;
  return CK_OK;
}

}  // namespace

int make_plane_map(CUtensorMap* map, const void* base, int64_t planes, int64_t rows, int64_t cols, int box_rows, bool two_dims);

bool grad_few_rows_applies(int64_t M, int64_t N, int64_t K, int planes) {
  const int64_t stage = kHeldBytes + planes * round_up(M, 16) * 128;
  return round_up(M, 16) <= 256 && kMinStages * stage <= kSmem - 1024 - kGroups * kRawBytes && N < (1 << 30) && ceil_div(K, kCols) <= 65535;
}

// dy: bf16 [planes][M, N].
int grad_few_rows(const void* dy, int planes, const void* codes, const void* scales, void* out, int out_dtype, int64_t M, int64_t N, int64_t K,
                  cudaStream_t stream) {
  FewRowsArgs a = {};
  a.codes = static_cast<const uint8_t*>(codes);
  a.scales = static_cast<const uint8_t*>(scales);
  a.out = out;
  a.out_dtype = out_dtype;
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.padded = static_cast<int>(round_up(M, 16));
  a.planes = planes;
  // An accumulator cuts what it adds to its own magnitude.  So the second and third numbers of dY's elements have their own, and for a result in fp32 four
  // take the first numbers in turn: 9 rows of fp32 through 6208 x 2624 were off by 3.1e-6 of the result with one for all.
  a.parts = 512 / a.padded - (planes - 1);
  if (a.parts > (out_dtype == CK_DTYPE_F32 ? 4 : 1)) a.parts = out_dtype == CK_DTYPE_F32 ? 4 : 1;
  CK_REQUIRE(a.parts >= 1, "linear_input_grad_mxfp8: %d accumulators", a.parts);
  const int stage = kHeldBytes + planes * a.padded * 128, steps = static_cast<int>(ceil_div(N, kDeep)), strips = static_cast<int>(ceil_div(K, kCols));
  a.raw_stages = (kSmem - 1024 - kMaxRaw * kRawBytes) / stage >= kMinStages ? kMaxRaw : kGroups;
  a.stages = (kSmem - 1024 - a.raw_stages * kRawBytes) / stage;
  CK_REQUIRE(a.stages >= kMinStages, "linear_input_grad_mxfp8: %d stages", a.stages);
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  // Ranges of W's rows, eight at most (the portable cluster size): those with the fewest stages one after another, a wave of clusters counting
  // six beside its own (first loads, the exchange of sums).
  int splits = 1, least = 0x7FFFFFFF;
  for (int s = 1; s <= 8 && s <= steps; ++s) {
    int at_once = 0;
    if (int rc = clusters_at_once(s, &at_once)) return rc;
    const int cost = (strips + at_once - 1) / at_once * (6 + (steps + s - 1) / s);
    if (cost < least) {
      least = cost;
      splits = s;
    }
  }
  a.steps_per_split = (steps + splits - 1) / splits;
  splits = (steps + a.steps_per_split - 1) / a.steps_per_split;
  if (int rc = gemm_status_word(&a.status)) return rc;
  CUtensorMap map_dy;
  if (int rc = make_plane_map(&map_dy, dy, planes, M, N, a.padded, false)) return rc;
  // boxes of 128 columns x 64 rows, as they lie in memory; rows past N and columns past K read as zeros
  CUtensorMap map_codes;
  if (int rc = make_code_map(&map_codes, codes, N, K)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, strips);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  CK_CUDA(cudaLaunchKernelEx(&cfg, grad_few_rows_kernel, map_dy, map_codes, a));
  return CK_OK;
}

// ---- grouped rows --------------------------------------------------------------------------------------------
namespace {

constexpr int kGroupedSmem = 226 * 1024 - 1024;  // dynamic, beside the barriers
static_assert(alone_with_tensor_memory(kGroupedSmem), "no allocation of tensor memory waits");

// Rows of a tile at most: as many as there is room for beside the fewest stages and eight of codes, or four where groups of so many rows would need
// more, or less than 64 fitted.  A tile computes and loads what it has rows for, and a group in fewer tiles has its weight decoded less often; codes that are fetched
// four stages ahead come late at times (us, eight / four: 333 uneven rows of 16 experts of 1536 x 2048 in fp32, tiles of 48 / 64, 43.4 / 33.4, even ones 37.1 / 36.2, 64
// experts of 2048 x 2048, 64 uneven rows each, 201 / 203; fp16, 80 / 112, 250 uneven rows each 405 / 415, 19 of 1024 x 1024 41.5 / 42.6; bf16, 160 / 224, 191 / 189).
int grouped_few_rows_tile(int64_t rows, int planes) {
  const auto most = [&](int raw_stages) {
    const int room = (kGroupedSmem - 1024 - raw_stages * kRawBytes - static_cast<int>(sizeof(groups::Table))) / kMinStages - kHeldBytes;
    return room / (planes * kRowBox * 128) * kRowBox;
  };
  return most(kMaxRaw) >= (rows > 64 ? rows : 64) ? most(kMaxRaw) : most(kGroups);
}

// E4M3 [E, N, K], boxes of 128 columns x 64 rows of one matrix, as they lie in memory; rows past N and columns past K read as zeros.
int make_experts_code_map(CUtensorMap* map, const void* base, int64_t E, int64_t N, int64_t K) {
  return cached_map(map, MapKey{13, base, E, N, K, 0}, [&](CUtensorMap* m) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (fn == nullptr) return fail(CK_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(N), static_cast<cuuint64_t>(E)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(K), static_cast<cuuint64_t>(N) * static_cast<cuuint64_t>(K)};
    const cuuint32_t box[3] = {kCols, kDeep, 1};
    const cuuint32_t elem_strides[3] = {1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(CK_ERR_CUDA, "cuTensorMapEncodeTiled (experts' codes) failed with code %d", static_cast<int>(r));
    return static_cast<int>(CK_OK);
  });
}

}  // namespace

// Whether groups of so many rows are decoded here: for each tile of theirs once, where the GEMM of ck_grad_gemm.cu has all matrices
// written as bf16 and reads them back (0.45 us for a million codes).  us, here / there: 64 experts of 2048 x 2048, 256 rows each, bf16 202 / 260, fp16
// 425 / 450 to 490, 8 of 4096 x 2048, 256 rows of fp32, 163 / 208; 512 rows, bf16 16 of 1024 x 8192 251 / 186, fp32 32 of 1024 x 1024 181 / 165.
bool grouped_few_rows_applies(int64_t M, int64_t E) {
  const int64_t used = E < M ? E : M;
  return ceil_div(M, used) <= 256;  // of a group, if they are alike
}

// dy: bf16 [planes][M, N].
int grouped_few_rows(const void* dy, int planes, const void* codes, const void* scales, const int* offsets, void* out, int out_dtype, int64_t M, int64_t N,
                     int64_t K, int64_t E, cudaStream_t stream) {
  GroupedFewRowsArgs a = {};
  a.scales = static_cast<const uint8_t*>(scales);
  a.out = out;
  a.offsets = offsets;
  a.out_dtype = out_dtype;
  a.groups = static_cast<int>(E);
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.padded = grouped_few_rows_tile(ceil_div(M, E < M ? E : M), planes);
  a.planes = planes;
  a.strips = static_cast<int>(ceil_div(K, kCols));
  // accumulators as for one weight: the second and third numbers' own, four for a result in fp32 where there is room for two sets of them
  a.parts = 256 / a.padded - (planes - 1);
  a.sets = a.parts >= 1 ? 2 : 1;
  if (a.sets == 1) a.parts = 512 / a.padded - (planes - 1);
  if (a.parts > (out_dtype == CK_DTYPE_F32 ? 4 : 1)) a.parts = out_dtype == CK_DTYPE_F32 ? 4 : 1;
  CK_REQUIRE(a.padded > 0 && a.parts >= 1, "grouped_input_grad_mxfp8: no room for %d rows", a.padded);
  const int stage = kHeldBytes + planes * a.padded * 128, room = kGroupedSmem - 1024 - static_cast<int>(sizeof(groups::Table));
  a.raw_stages = (room - kMaxRaw * kRawBytes) / stage >= kMinStages ? kMaxRaw : kGroups;
  a.stages = (room - a.raw_stages * kRawBytes) / stage;
  CK_REQUIRE(a.stages >= kMinStages, "grouped_input_grad_mxfp8: %d stages", a.stages);
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  if (int rc = gemm_status_word(&a.status)) return rc;
  CUtensorMap map_dy, map_dy_whole, map_codes;
  if (int rc = make_plane_map(&map_dy, dy, planes, M, N, kRowBox, false)) return rc;
  if (int rc = make_plane_map(&map_dy_whole, dy, planes, M, N, a.padded, false)) return rc;
  if (int rc = make_experts_code_map(&map_codes, codes, E, N, K)) return rc;
  static std::atomic<bool> configured[64];
  int dev = 0;
  CK_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
    CK_CUDA(cudaFuncSetAttribute(grouped_few_rows_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kGroupedSmem));
    if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
  }
  // the most tiles that the groups can have; those that there are the device counts
  const int64_t items = (M / a.padded + (E < M ? E : M)) * a.strips, workers = sm_count();
  CK_CUDA(launch_pdl(grouped_few_rows_kernel, dim3(static_cast<unsigned>(items < workers ? items : workers)), dim3(kGroupedThreads), kGroupedSmem, stream,
                     map_dy, map_dy_whole, map_codes, a));
  return CK_OK;
}

}  // namespace ck
