// Global norm of many gradients, and clipping by it, for sm_100a:
//
//   norm = sqrt(sum over all elements of g^2),  g *= min(1, max_norm / (norm + 1e-6))
//
// Bound by memory (and by latency, where the tensors are small): one read for the norm, and a read and a write more where it is above
// max_norm.  Two launches whatever the number of tensors, up to kMostTensors of them: their places travel in the kernels' arguments, nothing is
// copied to the device.  The elements are cut into chunks of one tensor each, which the blocks of a fixed grid take in turn; a block leaves one partial
// sum, and every block of the second kernel adds them all, in order, before it scales anything, so that the result does not depend on
// who runs when.  The second kernel takes the chunks backwards: it begins with what the first one read last, which L2 still holds.
// 134 million elements of bf16: the norm 41.6 us (6.46 TB/s, 0.99 of the copy rate), with the scaling 148 (5.4); a million elements of fp32 in 300 tensors 5.9, both
// launches, where the host takes 29 to collect the tensors.
#include <algorithm>
#include <new>
#include <utility>

#include "ck_rows.cuh"

namespace ck {
namespace {

constexpr int kMostTensors = 1024;       // of a launch
constexpr int kThreads = 512;
constexpr int kVecsPerThread = 4;        // 32-byte vectors of a chunk
constexpr int kChunkVecs = kThreads * kVecsPerThread;

template <int kMost>
struct Tensors {
  uint64_t data[kMost];    // address; element type in the two highest bits
  int64_t count[kMost];    // elements
  int chunks[kMost + 1];   // chunks of the tensors before
  int tensors;
};

__device__ __forceinline__ int type_of(uint64_t data) { return static_cast<int>(data >> 62); }

struct Place {
  uint64_t at;     // first whole vector of the tensor
  int64_t vecs;    // whole vectors of the tensor
  int64_t first;   // of the chunk
  uint64_t begin;  // address of the tensor
  int64_t head, tail;  // elements in front of the first whole vector and behind the last: the first chunk's
  int type;
};

template <int kMost>
__device__ __forceinline__ Place place_of(const Tensors<kMost>& t, int chunk) {
  int lo = 0, hi = t.tensors - 1;  // the last tensor whose chunks begin at `chunk` or before
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.chunks[mid] <= chunk) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  Place p;
  p.type = type_of(t.data[lo]);
  p.begin = t.data[lo] & ~(3ull << 62);
  const int size = p.type == CK_DTYPE_F32 ? 4 : 2;
  const int64_t n = t.count[lo], to_aligned = static_cast<int64_t>((32 - (p.begin & 31)) & 31) / size;
  p.head = min(n, to_aligned);
  p.at = p.begin + p.head * size;
  p.vecs = (n - p.head) * size / 32;
  p.tail = n - p.head - p.vecs * (32 / size);
  p.first = static_cast<int64_t>(chunk - t.chunks[lo]) * kChunkVecs;
  return p;
}

template <typename T>
__device__ __forceinline__ float squares(const Place& p) {
  constexpr int kEl = 32 / static_cast<int>(sizeof(T));
  using V = rows::Raw<T, kEl>;
  float sum = 0.0f;
  V raw[kVecsPerThread];
#pragma unroll
  for (int j = 0; j < kVecsPerThread; ++j) {
    const int64_t v = p.first + j * kThreads + threadIdx.x;
    if (v < p.vecs) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&raw[j]);
      asm volatile("ld.global.L1::no_allocate.v8.u32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p.at + v * 32)
                   : "memory");
    } else {
      raw[j] = rows::zeros<T, kEl>();
    }
  }
#pragma unroll
  for (int j = 0; j < kVecsPerThread; ++j) {
    float f[kEl];
    rows::unpack(raw[j], f);
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < kEl; ++i) part = fmaf(f[i], f[i], part);
    sum += part;
  }
  if (p.first == 0) {
    // up to 15 elements on each side
    const int i = threadIdx.x;
    const T* from = reinterpret_cast<const T*>(p.begin);
    if (i < p.head) {
      const float f = rows::to_float(rows::load_once<T, 1>(from + i).v[0]);
      sum = fmaf(f, f, sum);
    } else if (i >= 32 && i - 32 < p.tail) {
      const float f = rows::to_float(rows::load_once<T, 1>(reinterpret_cast<const T*>(p.at + p.vecs * 32) + i - 32).v[0]);
      sum = fmaf(f, f, sum);
    }
  }
  return sum;
}

template <typename T>
__device__ __forceinline__ void scale(const Place& p, float factor) {
  constexpr int kEl = 32 / static_cast<int>(sizeof(T));
  using V = rows::Raw<T, kEl>;
  V raw[kVecsPerThread];
#pragma unroll
  for (int j = 0; j < kVecsPerThread; ++j) {
    const int64_t v = p.first + j * kThreads + threadIdx.x;
    if (v < p.vecs) {
      uint32_t* w = reinterpret_cast<uint32_t*>(&raw[j]);
      asm volatile("ld.global.L1::no_allocate.v8.u32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p.at + v * 32)
                   : "memory");
    }
  }
#pragma unroll
  for (int j = 0; j < kVecsPerThread; ++j) {
    const int64_t v = p.first + j * kThreads + threadIdx.x;
    if (v >= p.vecs) continue;
    float f[kEl];
    rows::unpack(raw[j], f);
#pragma unroll
    for (int i = 0; i < kEl; ++i) f[i] *= factor;
    const V out = rows::pack<T, kEl>(f);
    st_global_256_no_allocate(reinterpret_cast<void*>(p.at + v * 32), *reinterpret_cast<const Vec256*>(&out));
  }
  if (p.first == 0) {
    const int i = threadIdx.x;
    T* at = i < p.head ? reinterpret_cast<T*>(p.begin) + i : i >= 32 && i - 32 < p.tail ? reinterpret_cast<T*>(p.at + p.vecs * 32) + i - 32 : nullptr;
    if (at != nullptr) *at = rows::from_float<T>(rows::to_float(*at) * factor);
  }
}

__device__ __forceinline__ float block_sum(float v) {
  __shared__ float buf[kThreads / 32];
  v = rows::warp_sum(v);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = threadIdx.x < kThreads / 32 ? buf[threadIdx.x] : 0.0f;
  return rows::warp_sum(v);  // the first warp's is the block's
}

template <int kMost>
__global__ void __launch_bounds__(kThreads) square_sums_kernel(const __grid_constant__ Tensors<kMost> t, float* partials) {
  pdl_launch_dependents();
  pdl_wait();
  float sum = 0.0f;
  const int chunks = t.chunks[t.tensors];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const Place p = place_of(t, c);
    sum += p.type == CK_DTYPE_BF16 ? squares<__nv_bfloat16>(p) : p.type == CK_DTYPE_F16 ? squares<__half>(p) : squares<float>(p);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

// Every block adds the partial sums in the same order and so has the same norm.
__device__ __forceinline__ float norm_of(const float* partials, int n) {
  __shared__ double buf[kThreads / 32];
  __shared__ float result;
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) sum += ld_f32_dependent(partials + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads / 32; ++i) sum += buf[i];
    result = static_cast<float>(sqrt(sum));
  }
  __syncthreads();
  return result;
}

template <int kMost>
__global__ void __launch_bounds__(kThreads, 2) clip_kernel(const __grid_constant__ Tensors<kMost> t, const float* partials, int n_partials, float max_norm,
                                                        float* norm_out) {
  pdl_launch_dependents();
  pdl_wait();
  const float norm = norm_of(partials, n_partials);
  if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out != nullptr) *norm_out = norm;
  if (max_norm < 0.0f) return;  // the norm alone
  const float factor = max_norm / (norm + 1e-6f);
  if (factor >= 1.0f) return;  // (a norm that is no number makes all of them none)
  for (int c = t.chunks[t.tensors] - 1 - static_cast<int>(blockIdx.x); c >= 0; c -= gridDim.x) {
    const Place p = place_of(t, c);
    if (p.type == CK_DTYPE_BF16) {
      scale<__nv_bfloat16>(p, factor);
    } else if (p.type == CK_DTYPE_F16) {
      scale<__half>(p, factor);
    } else {
      scale<float>(p, factor);
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
constexpr int kBlocksPerSm = 4;
int most_blocks() { return kBlocksPerSm * sm_count(); }

int64_t chunks_of(const void* data, int64_t n, int size) {
  const int64_t head = static_cast<int64_t>((32 - (reinterpret_cast<uintptr_t>(data) & 31)) & 31) / size;
  const int64_t vecs = n > head ? (n - head) * size / 32 : 0;
  return vecs > 0 ? ceil_div(vecs, kChunkVecs) : 1;
}

struct Launch {
  int64_t first, tensors;
};

template <int kMost>
int fill(Tensors<kMost>* t, void* const* grads, const int64_t* counts, const int* dtypes, const Launch& l) {
  t->tensors = 0;
  int64_t chunks = 0;
  for (int64_t i = l.first; i < l.first + l.tensors; ++i) {
    if (counts[i] == 0) continue;
    t->data[t->tensors] = reinterpret_cast<uint64_t>(grads[i]) | (static_cast<uint64_t>(dtypes[i]) << 62);
    t->count[t->tensors] = counts[i];
    t->chunks[t->tensors] = static_cast<int>(chunks);
    chunks += chunks_of(grads[i], counts[i], dtypes[i] == CK_DTYPE_F32 ? 4 : 2);
    CK_REQUIRE(chunks < (1ll << 31), "clip_grad_norm: too many elements");
    ++t->tensors;
  }
  t->chunks[t->tensors] = static_cast<int>(chunks);
  return CK_OK;
}

template <int kMost>
int both(void* const* grads, const int64_t* counts, const int* dtypes, int64_t tensors, float max_norm, float* norm, float* partials, cudaStream_t s) {
  Tensors<kMost> t;
  const int blocks = most_blocks();
  const int64_t launches = tensors > 0 ? ceil_div(tensors, kMost) : 1;  // no tensors: the norm is written all the same
  int n_partials = 0;
  for (int64_t i = 0; i < launches; ++i) {
    const Launch l = {i * kMost, std::min<int64_t>(kMost, tensors - i * kMost)};
    if (int rc = fill(&t, grads, counts, dtypes, l)) return rc;
    if (t.tensors == 0) continue;
    const int used = std::min(blocks, t.chunks[t.tensors]);
    CK_CUDA(launch_pdl(square_sums_kernel<kMost>, dim3(used), dim3(kThreads), 0, s, t, partials + n_partials));
    n_partials += used;
  }
  for (int64_t i = 0; i < launches; ++i) {
    if (launches > 1) {
      const Launch l = {i * kMost, std::min<int64_t>(kMost, tensors - i * kMost)};
      if (int rc = fill(&t, grads, counts, dtypes, l)) return rc;
    }
    const int used = max_norm < 0.0f ? 1 : std::max(1, std::min(blocks, t.tensors > 0 ? t.chunks[t.tensors] : 1));
    CK_CUDA(launch_pdl(clip_kernel<kMost>, dim3(used), dim3(kThreads), 0, s, t, static_cast<const float*>(partials), n_partials, max_norm,
                       i == 0 ? norm : static_cast<float*>(nullptr)));
    if (max_norm < 0.0f) break;
  }
  return CK_OK;
}

}  // namespace
}  // namespace ck

extern "C" int64_t ck_clip_grad_norm_workspace_bytes(int64_t tensors) {
  if (tensors < 0 || tensors > (1ll << 24)) return 0;
  return (ck::ceil_div(tensors, ck::kMostTensors) + 1) * ck::most_blocks() * 4;
}

extern "C" int ck_clip_grad_norm(void* const* grads, const int64_t* counts, const int* dtypes, int64_t tensors, float max_norm, float* norm,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace ck;
  const char* op = "clip_grad_norm";
  CK_REQUIRE(tensors >= 0 && tensors <= (1ll << 24), "%s: %lld tensors", op, (long long)tensors);
  CK_REQUIRE(norm != nullptr && workspace != nullptr && (tensors == 0 || (grads != nullptr && counts != nullptr && dtypes != nullptr)), "%s: null pointer", op);
  CK_REQUIRE(workspace_bytes >= ck_clip_grad_norm_workspace_bytes(tensors) && reinterpret_cast<uintptr_t>(workspace) % 4 == 0,
             "%s: workspace of %lld bytes, %lld needed", op, (long long)workspace_bytes, (long long)ck_clip_grad_norm_workspace_bytes(tensors));
  CK_REQUIRE(max_norm == max_norm, "%s: max_norm is no number", op);
  using Range = std::pair<uint64_t, uint64_t>;
  Range* ranges = new (std::nothrow) Range[tensors > 0 ? tensors : 1];
  CK_REQUIRE(ranges != nullptr, "%s: out of memory", op);
  int64_t used = 0;
  bool ok = true;
  for (int64_t i = 0; i < tensors && ok; ++i) {
    const int size = dtypes[i] == CK_DTYPE_F32 ? 4 : 2;
    const uint64_t at = reinterpret_cast<uint64_t>(grads[i]);
    ok = (dtypes[i] == CK_DTYPE_F32 || dtypes[i] == CK_DTYPE_F16 || dtypes[i] == CK_DTYPE_BF16) && counts[i] >= 0 && counts[i] < (1ll << 48) &&
         at < (1ull << 62) && (counts[i] == 0 || (at != 0 && at % size == 0));
    if (ok && counts[i] > 0) ranges[used++] = Range(at, at + static_cast<uint64_t>(counts[i]) * size);
  }
  bool apart = true;
  if (ok) {
    std::sort(ranges, ranges + used);
    for (int64_t i = 1; i < used; ++i) apart = apart && ranges[i - 1].second <= ranges[i].first;
  }
  delete[] ranges;
  CK_REQUIRE(ok, "%s: a tensor's address, type or size is not supported", op);
  CK_REQUIRE(apart || max_norm < 0.0f, "%s: tensors overlap", op);
  float* partials = static_cast<float*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tensors <= 64) return both<64>(grads, counts, dtypes, tensors, max_norm, norm, partials, s);
  return both<kMostTensors>(grads, counts, dtypes, tensors, max_norm, norm, partials, s);
}
