// Norm of many gradient tensors taken as one vector, and their scaling by one factor.
//   total = (sum over all elements of |g|^p)^(1/p), p = 1 or 2, or max |g|
//   g <- g * min(1, max_norm / (total + 1e-6))
//
// The tensors' addresses and sizes travel in the kernel's parameters (no table in device memory to fill, nothing to
// copy, so the calls can be captured), up to kTensors per launch.  They are cut into chunks of kChunk elements; a
// CTA adds up one chunk and stores one partial sum, and a last CTA adds the partial sums, each in a fixed order: the
// result does not change from run to run.  A thread's 64 elements are added in fp32, everything above that in fp64.
// Memory bounds it: the norm reads every gradient once, the scaling reads and writes it once more and is skipped
// on the device when the factor is 1 (eight gradients of 14336 x 4096 bf16: norm 156 us, 6.0 TB/s, scaling 301 us, 6.2 TB/s,
// single calls with cold caches).  The scaling walks the chunks backwards: the ones the norm read
// last are still in L2.
#include <algorithm>
#include <new>

#include "common.cuh"

namespace f8b200 {
namespace {

constexpr int kTensors = 1024;
constexpr int kThreads = 256;
constexpr int64_t kChunk = 16384;

struct TensorList {
  void* ptr[kTensors];
  int64_t numel[kTensors];
  int32_t first_chunk[kTensors];
  uint8_t dtype[kTensors];
  int32_t n;
};
static_assert(sizeof(TensorList) <= 28 * 1024, "kernel parameters are limited to 32764 bytes");

// index of the tensor that chunk c belongs to (first_chunk ascends; no tensor is empty)
__device__ __forceinline__ int tensor_of(const TensorList& list, int c) {
  int lo = 0, hi = list.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.first_chunk[mid] <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int HP>
__device__ __forceinline__ void widen16(const uint4& q, float* v) {  // 16 bytes
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (HP == F8B200_FP32) {
      v[i] = __uint_as_float(w[i]);
    } else if constexpr (HP == F8B200_BF16) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
template <int HP>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (HP == F8B200_FP32) return static_cast<const float*>(p)[i];
  else if constexpr (HP == F8B200_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  else return __half2float(static_cast<const __half*>(p)[i]);
}
template <int HP>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (HP == F8B200_FP32) static_cast<float*>(p)[i] = v;
  else if constexpr (HP == F8B200_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

// KIND: 0 = max |g| (as bits, NaN above infinity), 1 = sum |g|, 2 = sum g^2
template <int KIND>
struct Acc {
  float s = 0.f;
  uint32_t m = 0;
  __device__ __forceinline__ void add(float v) {
    if constexpr (KIND == 0) m = max(m, __float_as_uint(v) & 0x7FFFFFFFu);
    else if constexpr (KIND == 1) s += fabsf(v);
    else s = fmaf(v, v, s);
  }
};

template <int KIND, int HP>
__device__ __forceinline__ Acc<KIND> chunk_norm(const void* base, int64_t at, int count) {
  constexpr int N = HP == F8B200_FP32 ? 4 : 8, ES = 16 / N;
  Acc<KIND> acc;
  const char* p = static_cast<const char*>(base) + at * ES;
  int done = 0;
  if (reinterpret_cast<uintptr_t>(p) % 16 == 0) {
    const uint4* q = reinterpret_cast<const uint4*>(p);
    const int words = count / N;
    constexpr int U = (int)(kChunk / N / kThreads);  // 8 or 16 words per thread of a full chunk
    if (count == kChunk) {
#pragma unroll
      for (int h = 0; h < U / 8; ++h) {
        uint4 w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __ldg(q + threadIdx.x + (h * 8 + i) * kThreads);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v[N];
          widen16<HP>(w[i], v);
#pragma unroll
          for (int j = 0; j < N; ++j) acc.add(v[j]);
        }
      }
    } else {
      for (int i = threadIdx.x; i < words; i += kThreads) {
        float v[N];
        widen16<HP>(__ldg(q + i), v);
#pragma unroll
        for (int j = 0; j < N; ++j) acc.add(v[j]);
      }
    }
    done = words * N;
  }
  for (int i = done + (int)threadIdx.x; i < count; i += kThreads) acc.add(load1<HP>(p, i));
  return acc;
}

__device__ __forceinline__ double block_sum(double v, double* sm) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (lane == 0) sm[w] = v;
  __syncthreads();
  double t = 0.0;
  if (threadIdx.x == 0)
    for (int i = 0; i < nw; ++i) t += sm[i];
  return t;  // in thread 0
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* sm) {
  v = warp_max_u32(v);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (lane == 0) sm[w] = v;
  __syncthreads();
  uint32_t t = 0;
  if (threadIdx.x == 0)
    for (int i = 0; i < nw; ++i) t = max(t, sm[i]);
  return t;
}

template <int KIND>
__global__ void __launch_bounds__(kThreads) norm_parts_kernel(const __grid_constant__ TensorList list, double* __restrict__ parts) {
  __shared__ double sm[kThreads / 32];
  __shared__ uint32_t smu[kThreads / 32];
  const int t = tensor_of(list, (int)blockIdx.x);
  const int64_t at = (int64_t)((int)blockIdx.x - list.first_chunk[t]) * kChunk;
  const int64_t left = list.numel[t] - at;
  const int count = (int)(left < kChunk ? left : kChunk);
  Acc<KIND> a;
  if (list.dtype[t] == F8B200_BF16) a = chunk_norm<KIND, F8B200_BF16>(list.ptr[t], at, count);
  else if (list.dtype[t] == F8B200_FP16) a = chunk_norm<KIND, F8B200_FP16>(list.ptr[t], at, count);
  else a = chunk_norm<KIND, F8B200_FP32>(list.ptr[t], at, count);
  if constexpr (KIND == 0) {
    const uint32_t m = block_max(a.m, smu);
    if (threadIdx.x == 0) parts[blockIdx.x] = (double)__uint_as_float(m);
  } else {
    const double s = block_sum((double)a.s, sm);
    if (threadIdx.x == 0) parts[blockIdx.x] = s;
  }
}

// `root`: the norm itself; otherwise the sum of powers (or the maximum) that ranks add up among themselves first.
template <int KIND>
__global__ void __launch_bounds__(1024) norm_join_kernel(const double* __restrict__ parts, int64_t n, int root, float* __restrict__ out) {
  __shared__ double sm[32];
  __shared__ uint32_t smu[32];
  if constexpr (KIND == 0) {
    uint32_t m = 0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) m = max(m, __float_as_uint((float)parts[i]) & 0x7FFFFFFFu);
    m = block_max(m, smu);
    if (threadIdx.x == 0) *out = __uint_as_float(m);
  } else {
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) s += parts[i];
    s = block_sum(s, sm);
    if (threadIdx.x == 0) *out = (float)(KIND == 2 && root ? sqrt(s) : s);
  }
}

template <int HP>
__device__ __forceinline__ void chunk_scale(void* base, int64_t at, int count, float f) {
  constexpr int N = HP == F8B200_FP32 ? 4 : 8, ES = 16 / N;
  char* p = static_cast<char*>(base) + at * ES;
  int done = 0;
  if (reinterpret_cast<uintptr_t>(p) % 16 == 0) {
    uint4* q = reinterpret_cast<uint4*>(p);
    const int words = count / N;
    for (int i0 = threadIdx.x; i0 < words; i0 += 4 * kThreads) {
      uint4 w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i0 + u * kThreads < words) w[u] = q[i0 + u * kThreads];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (i0 + u * kThreads >= words) continue;
        float v[N];
        widen16<HP>(w[u], v);
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (HP == F8B200_FP32) {
            o[i] = __float_as_uint(v[i] * f);
          } else if constexpr (HP == F8B200_BF16) {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i] * f, v[2 * i + 1] * f);
            o[i] = *reinterpret_cast<const uint32_t*>(&h);
          } else {
            const __half2 h = __floats2half2_rn(v[2 * i] * f, v[2 * i + 1] * f);
            o[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        q[i0 + u * kThreads] = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    done = words * N;
  }
  for (int i = done + (int)threadIdx.x; i < count; i += kThreads) store1<HP>(p, i, load1<HP>(p, i) * f);
}

__global__ void __launch_bounds__(kThreads)
clip_kernel(const __grid_constant__ TensorList list, int chunks, const float* __restrict__ total, float max_norm) {
  float f = __fdiv_rn(max_norm, __ldg(total) + 1e-6f);
  if (f > 1.0f) f = 1.0f;  // a NaN stays
  if (f == 1.0f) return;
  for (int c = chunks - 1 - (int)blockIdx.x; c >= 0; c -= (int)gridDim.x) {
    const int t = tensor_of(list, c);
    const int64_t at = (int64_t)(c - list.first_chunk[t]) * kChunk;
    const int64_t left = list.numel[t] - at;
    const int count = (int)(left < kChunk ? left : kChunk);
    if (list.dtype[t] == F8B200_BF16) chunk_scale<F8B200_BF16>(list.ptr[t], at, count, f);
    else if (list.dtype[t] == F8B200_FP16) chunk_scale<F8B200_FP16>(list.ptr[t], at, count, f);
    else chunk_scale<F8B200_FP32>(list.ptr[t], at, count, f);
  }
}

int check_list(const void* const* ptrs, const int64_t* numels, const int* hp_dtypes, int n) {
  if (n < 0 || (n > 0 && (ptrs == nullptr || numels == nullptr || hp_dtypes == nullptr))) return F8B200_ERR_BAD_ARG;
  int64_t chunks = 0;
  for (int i = 0; i < n; ++i) {
    if (numels[i] < 0 || hp_dtypes[i] < 0 || hp_dtypes[i] > 2) return F8B200_ERR_BAD_ARG;
    if (numels[i] == 0) continue;
    if (ptrs[i] == nullptr) return F8B200_ERR_BAD_ARG;
    if (reinterpret_cast<uintptr_t>(ptrs[i]) % (uintptr_t)hp_size_of(hp_dtypes[i]) != 0) return F8B200_ERR_ALIGNMENT;
    chunks += (numels[i] + kChunk - 1) / kChunk;
    if (chunks > 0x7FFFFFFFLL) return F8B200_ERR_UNSUPPORTED;
  }
  return F8B200_OK;
}

// Whether two of the tensors have bytes in common: they would be scaled twice, by CTAs that do not wait for each other.
// Tensors that lie in the order of their addresses, as the gradients of one buffer do, need no sorting.
int check_apart(void* const* ptrs, const int64_t* numels, const int* hp_dtypes, int n) {
  struct Span {
    uintptr_t begin, end;
  };
  auto span = [&](int i) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(ptrs[i]);
    return Span{p, p + (uintptr_t)numels[i] * (uintptr_t)hp_size_of(hp_dtypes[i])};
  };
  uintptr_t end = 0;
  bool ascending = true;
  for (int i = 0; i < n && ascending; ++i) {
    if (numels[i] == 0) continue;
    const Span s = span(i);
    ascending = s.begin >= end;
    end = s.end;
  }
  if (ascending) return F8B200_OK;
  Span* spans = new (std::nothrow) Span[n];
  if (spans == nullptr) return F8B200_ERR_UNSUPPORTED;
  int used = 0;
  for (int i = 0; i < n; ++i)
    if (numels[i] != 0) spans[used++] = span(i);
  std::sort(spans, spans + used, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  bool apart = true;
  for (int i = 1; i < used; ++i) apart = apart && spans[i].begin >= spans[i - 1].end;
  delete[] spans;
  return apart ? F8B200_OK : F8B200_ERR_BAD_ARG;
}

// Cuts the tensors into lists of kTensors and calls fn(list, chunks of the list, chunks before it).
template <typename Fn>
int for_each_list(const void* const* ptrs, const int64_t* numels, const int* hp_dtypes, int n, Fn&& fn) {
  TensorList list;
  int i = 0;
  int64_t before = 0;
  while (i < n) {
    list.n = 0;
    int64_t chunks = 0;
    for (; i < n && list.n < kTensors; ++i) {
      if (numels[i] == 0) continue;
      list.ptr[list.n] = const_cast<void*>(ptrs[i]);
      list.numel[list.n] = numels[i];
      list.first_chunk[list.n] = (int32_t)chunks;
      list.dtype[list.n] = (uint8_t)hp_dtypes[i];
      ++list.n;
      chunks += (numels[i] + kChunk - 1) / kChunk;
    }
    if (list.n == 0) break;
    const int rc = fn(list, chunks, before);
    if (rc != F8B200_OK) return rc;
    before += chunks;
  }
  return F8B200_OK;
}

}  // namespace
}  // namespace f8b200

using namespace f8b200;

extern "C" int64_t f8b200_multi_norm_workspace_bytes(const int64_t* numels, int n) {
  int64_t chunks = 0;
  for (int i = 0; numels != nullptr && i < n; ++i)
    if (numels[i] > 0) chunks += (numels[i] + kChunk - 1) / kChunk;
  return chunks * (int64_t)sizeof(double);
}

extern "C" int f8b200_multi_norm(const void* const* ptrs, const int64_t* numels, const int* hp_dtypes, int n, int kind, int root,
                                 float* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (kind < 0 || kind > 2 || out == nullptr) return F8B200_ERR_BAD_ARG;
  int rc = check_list(ptrs, numels, hp_dtypes, n);
  if (rc != F8B200_OK) return rc;
  const int64_t need = f8b200_multi_norm_workspace_bytes(numels, n);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return F8B200_ERR_BAD_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) % 8 != 0 || reinterpret_cast<uintptr_t>(out) % 4 != 0) return F8B200_ERR_ALIGNMENT;
  rc = f8b200_device_check();
  if (rc != F8B200_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  double* parts = static_cast<double*>(workspace);
  rc = for_each_list(ptrs, numels, hp_dtypes, n, [&](const TensorList& list, int64_t chunks, int64_t before) {
    const unsigned grid = (unsigned)chunks;
    if (kind == 0) norm_parts_kernel<0><<<grid, kThreads, 0, st>>>(list, parts + before);
    else if (kind == 1) norm_parts_kernel<1><<<grid, kThreads, 0, st>>>(list, parts + before);
    else norm_parts_kernel<2><<<grid, kThreads, 0, st>>>(list, parts + before);
    return check_launch();
  });
  if (rc != F8B200_OK) return rc;
  const int64_t total = need / (int64_t)sizeof(double);
  if (kind == 0) norm_join_kernel<0><<<1, 1024, 0, st>>>(parts, total, root, out);
  else if (kind == 1) norm_join_kernel<1><<<1, 1024, 0, st>>>(parts, total, root, out);
  else norm_join_kernel<2><<<1, 1024, 0, st>>>(parts, total, root, out);
  return check_launch();
}

extern "C" int f8b200_multi_clip(void* const* ptrs, const int64_t* numels, const int* hp_dtypes, int n, const float* total_norm,
                                 float max_norm, void* stream) {
  if (total_norm == nullptr) return F8B200_ERR_BAD_ARG;
  int rc = check_list(ptrs, numels, hp_dtypes, n);
  if (rc == F8B200_OK) rc = check_apart(ptrs, numels, hp_dtypes, n);
  if (rc != F8B200_OK) return rc;
  if (reinterpret_cast<uintptr_t>(total_norm) % 4 != 0) return F8B200_ERR_ALIGNMENT;
  rc = f8b200_device_check();
  if (rc != F8B200_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return for_each_list(ptrs, numels, hp_dtypes, n, [&](const TensorList& list, int64_t chunks, int64_t) {
    const int64_t cap = (int64_t)sm_count() * 8;
    clip_kernel<<<(unsigned)(chunks < cap ? chunks : cap), kThreads, 0, st>>>(list, (int)chunks, total_norm, max_norm);
    return check_launch();
  });
}
