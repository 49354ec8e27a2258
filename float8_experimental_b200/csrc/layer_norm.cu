// Layer norm over the last dimension, forward and backward.
//   mean = sum(x) / C,  var = sum((x - mean)^2) / C,  rstd = 1 / sqrt(var + eps),  n = (x - mean) * rstd
//   y  = n * w + b
//   dx = rstd * (h - sum(h) / C - n * sum(h * n) / C),  h = g * w
//   dw = sum over rows of g * n,   db = sum over rows of g
// All in fp32 whatever the type of x; y, dx, dw and db are rounded once.  The variance is the second moment about the
// mean that was just found, not a difference of two large sums, so a large mean costs no digits.
// w and b have x's type or fp32; either may be absent (1 and 0).  Sums run in a fixed order.
//
// Memory bounds both directions: x read and y written (4 bytes per 16-bit element), x and g read and dx written (6).
#include <type_traits>

#include "common.cuh"

namespace f8b200 {
namespace {

constexpr int kThreads = 256;

template <int HP>
struct Elem;
template <>
struct Elem<F8B200_BF16> { using type = __nv_bfloat16; };
template <>
struct Elem<F8B200_FP16> { using type = __half; };
template <>
struct Elem<F8B200_FP32> { using type = float; };

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}

// 16 bytes of T as fp32 values
template <typename T>
struct Vec {
  static constexpr int N = 16 / (int)sizeof(T);
  __device__ __forceinline__ static void widen(const uint4& q, float (&v)[N]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
  __device__ __forceinline__ static uint4 narrow(const float (&v)[N]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(v[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// N affine values starting at element i (W is T or fp32; the address is 16-byte aligned); `none` where there are none.
template <typename W, int N>
__device__ __forceinline__ void load_affine(const W* p, int64_t i, float none, float (&v)[N]) {
  if (p == nullptr) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = none;
    return;
  }
  constexpr int M = Vec<W>::N;  // values per 16 bytes: N, or half as many when x is 16 bits wide and w is fp32
#pragma unroll
  for (int h = 0; h < N / M; ++h) {
    float t[M];
    Vec<W>::widen(__ldg(reinterpret_cast<const uint4*>(p + i) + h), t);
#pragma unroll
    for (int j = 0; j < M; ++j) v[h * M + j] = t[j];
  }
}

// Sum over the ROWT threads of a row (a warp, or the whole CTA), the same value in all of them.
template <int ROWT>
__device__ __forceinline__ float row_sum(float v, float* smem) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  if constexpr (ROWT > 32) {
    constexpr int W = ROWT / 32;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (lane == 0) smem[w] = v;
    __syncthreads();
    v = lane < W ? smem[lane] : 0.f;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
    v = __shfl_sync(0xFFFFFFFFu, v, 0);
    __syncthreads();
  }
  return v;
}

// ---- forward, a row in registers --------------------------------------------------------------------
template <typename T, typename W, int ROWT, int CH>
__global__ void __launch_bounds__(kThreads)
ln_fwd_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, const W* __restrict__ weight,
              const W* __restrict__ bias, float eps, T* __restrict__ y, int64_t ld_y, float* __restrict__ mean_out,
              float* __restrict__ rstd_out) {
  constexpr int N = Vec<T>::N, RPB = kThreads / ROWT;
  __shared__ float smem[kThreads / 32];
  const int t = threadIdx.x % ROWT;
  const int chunks = (int)(cols / N);
  const float inv_c = 1.0f / (float)cols;
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / ROWT; r < rows; r += (int64_t)gridDim.x * RPB) {
    const uint4* row = reinterpret_cast<const uint4*>(x + r * ld_x);
    uint4 q[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) q[i] = t + i * ROWT < chunks ? __ldcs(row + t + i * ROWT) : make_uint4(0u, 0u, 0u, 0u);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      float v[N];
      Vec<T>::widen(q[i], v);
#pragma unroll
      for (int j = 0; j < N; ++j) s += v[j];
    }
    const float mean = row_sum<ROWT>(s, smem) * inv_c;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (t + i * ROWT < chunks) {
        float v[N];
        Vec<T>::widen(q[i], v);
#pragma unroll
        for (int j = 0; j < N; ++j) s = fmaf(v[j] - mean, v[j] - mean, s);
      }
    }
    const float rstd = 1.0f / sqrtf(row_sum<ROWT>(s, smem) * inv_c + eps);
    if (t == 0 && mean_out != nullptr) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
    uint4* out = reinterpret_cast<uint4*>(y + r * ld_y);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int c = t + i * ROWT;
      if (c < chunks) {
        float v[N], w[N], b[N];
        Vec<T>::widen(q[i], v);
        load_affine<W, N>(weight, (int64_t)c * N, 1.f, w);
        load_affine<W, N>(bias, (int64_t)c * N, 0.f, b);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = fmaf((v[j] - mean) * rstd, w[j], b[j]);
        __stcs(out + c, Vec<T>::narrow(v));
      }
    }
  }
}

// ---- any width, any alignment -----------------------------------------------------------------------
template <typename T, typename W>
__global__ void __launch_bounds__(kThreads)
ln_fwd_any_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, const W* __restrict__ weight,
                  const W* __restrict__ bias, float eps, T* __restrict__ y, int64_t ld_y, float* __restrict__ mean_out,
                  float* __restrict__ rstd_out) {
  __shared__ float smem[kThreads / 32];
  const float inv_c = 1.0f / (float)cols;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * ld_x;
    float s = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) s += to_f32(row[c]);
    const float mean = row_sum<kThreads>(s, smem) * inv_c;
    s = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      const float d = to_f32(row[c]) - mean;
      s = fmaf(d, d, s);
    }
    const float rstd = 1.0f / sqrtf(row_sum<kThreads>(s, smem) * inv_c + eps);
    if (threadIdx.x == 0 && mean_out != nullptr) {
      mean_out[r] = mean;
      rstd_out[r] = rstd;
    }
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      const float w = weight != nullptr ? to_f32(weight[c]) : 1.f, b = bias != nullptr ? to_f32(bias[c]) : 0.f;
      y[r * ld_y + c] = from_f32<T>(fmaf((to_f32(row[c]) - mean) * rstd, w, b));
    }
  }
}

template <typename T, typename W>
__global__ void __launch_bounds__(kThreads)
ln_dx_any_kernel(const T* __restrict__ x, int64_t ld_x, const T* __restrict__ g, int64_t ld_g, int64_t rows, int64_t cols,
                 const W* __restrict__ weight, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                 T* __restrict__ dx, int64_t ld_dx) {
  __shared__ float smem[kThreads / 32];
  const float inv_c = 1.0f / (float)cols;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * ld_x, *gr = g + r * ld_g;
    const float mean = mean_in[r], rstd = rstd_in[r];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      const float h = to_f32(gr[c]) * (weight != nullptr ? to_f32(weight[c]) : 1.f);
      s1 += h;
      s2 = fmaf(h, (to_f32(xr[c]) - mean) * rstd, s2);
    }
    s1 = row_sum<kThreads>(s1, smem) * inv_c;
    s2 = row_sum<kThreads>(s2, smem) * inv_c;
    for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
      const float h = to_f32(gr[c]) * (weight != nullptr ? to_f32(weight[c]) : 1.f);
      const float nv = (to_f32(xr[c]) - mean) * rstd;
      dx[r * ld_dx + c] = from_f32<T>(rstd * (h - s1 - nv * s2));
    }
  }
}

// Partial sums of dw and db: CTA (x, y) adds up rows y, y + gridDim.y, ... of 64 columns, four rows at a time;
// part[y][0 or 1][col].
template <typename T>
__global__ void __launch_bounds__(kThreads)
ln_dw_any_kernel(const T* __restrict__ x, int64_t ld_x, const T* __restrict__ g, int64_t ld_g, int64_t rows, int64_t cols,
                 const float* __restrict__ mean_in, const float* __restrict__ rstd_in, float* __restrict__ part) {
  __shared__ float sm[2][4][64];
  const int cx = threadIdx.x & 63, ry = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + cx;
  float dw = 0.f, db = 0.f;
  if (c < cols) {
    for (int64_t r = (int64_t)blockIdx.y * 4 + ry; r < rows; r += (int64_t)gridDim.y * 4) {
      const float gv = to_f32(g[r * ld_g + c]);
      dw = fmaf(gv, (to_f32(x[r * ld_x + c]) - mean_in[r]) * rstd_in[r], dw);
      db += gv;
    }
  }
  sm[0][ry][cx] = dw;
  sm[1][ry][cx] = db;
  __syncthreads();
  if (ry < 2 && c < cols) part[((int64_t)blockIdx.y * 2 + ry) * cols + c] = sm[ry][0][cx] + sm[ry][1][cx] + sm[ry][2][cx] + sm[ry][3][cx];
}

// dw and db from `parts` partial sums: 32 columns per CTA, eight threads per column.
template <typename W>
__global__ void __launch_bounds__(kThreads)
ln_dw_join_kernel(const float* __restrict__ part, int parts, int64_t cols, W* __restrict__ dw, W* __restrict__ db) {
  __shared__ float sm[2][8][32];
  const int cx = threadIdx.x & 31, py = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + cx;
  float a = 0.f, b = 0.f;
  if (c < cols) {
    for (int i = py; i < parts; i += 8) {
      a += part[(int64_t)i * 2 * cols + c];
      b += part[((int64_t)i * 2 + 1) * cols + c];
    }
  }
  sm[0][py][cx] = a;
  sm[1][py][cx] = b;
  __syncthreads();
  if (py < 2 && c < cols) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v += sm[py][i][cx];
    W* out = py == 0 ? dw : db;
    if (out != nullptr) out[c] = from_f32<W>(v);
  }
}

constexpr int kMaxParts = 148;  // partial sums of dw and db that the workspace has room for

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

unsigned row_grid(int64_t row_groups) {
  const int64_t cap = (int64_t)sm_count() * 8;
  return (unsigned)(row_groups < cap ? row_groups : cap);
}

template <typename T, typename W>
int ln_fwd(const void* x, int64_t rows, int64_t cols, int64_t ld_x, const void* weight, const void* bias, float eps, void* y,
           int64_t ld_y, float* mean, float* rstd, cudaStream_t st) {
  constexpr int N = Vec<T>::N;
  const T* xp = static_cast<const T*>(x);
  const W *wp = static_cast<const W*>(weight), *bp = static_cast<const W*>(bias);
  T* yp = static_cast<T*>(y);
  const bool vec = cols % N == 0 && ld_x % N == 0 && ld_y % N == 0 && aligned16(x) && aligned16(y) && aligned16(weight) &&
                   aligned16(bias);
  const int64_t chunks = cols / N;
#define F8_LN(ROWT, CH) \
  ln_fwd_kernel<T, W, ROWT, CH><<<row_grid((rows + kThreads / ROWT - 1) / (kThreads / ROWT)), kThreads, 0, st>>>( \
      xp, ld_x, rows, cols, wp, bp, eps, yp, ld_y, mean, rstd)
  if (vec && chunks <= 32) F8_LN(32, 1);
  else if (vec && chunks <= 128) F8_LN(32, 4);
  else if (vec && chunks <= 256) F8_LN(256, 1);
  else if (vec && chunks <= 512) F8_LN(256, 2);
  else if (vec && chunks <= 1024) F8_LN(256, 4);
  else if (vec && chunks <= 2048) F8_LN(256, 8);
  else ln_fwd_any_kernel<T, W><<<row_grid(rows), kThreads, 0, st>>>(xp, ld_x, rows, cols, wp, bp, eps, yp, ld_y, mean, rstd);
#undef F8_LN
  return check_launch();
}

template <typename T, typename W>
int ln_bwd(const void* x, const void* g, int64_t rows, int64_t cols, int64_t ld_x, int64_t ld_g, const void* weight,
           const float* mean, const float* rstd, void* dx, int64_t ld_dx, void* dw, void* db, float* part, cudaStream_t st) {
  const T *xp = static_cast<const T*>(x), *gp = static_cast<const T*>(g);
  if (dx != nullptr)
    ln_dx_any_kernel<T, W><<<row_grid(rows), kThreads, 0, st>>>(xp, ld_x, gp, ld_g, rows, cols, static_cast<const W*>(weight),
                                                                mean, rstd, static_cast<T*>(dx), ld_dx);
  if (dw != nullptr || db != nullptr) {
    const int64_t groups = (rows + 3) / 4;
    const int parts = (int)(groups < kMaxParts ? groups : kMaxParts);
    const dim3 grid((unsigned)((cols + 63) / 64), (unsigned)parts);
    ln_dw_any_kernel<T><<<grid, kThreads, 0, st>>>(xp, ld_x, gp, ld_g, rows, cols, mean, rstd, part);
    ln_dw_join_kernel<W><<<(unsigned)((cols + 31) / 32), kThreads, 0, st>>>(part, parts, cols, static_cast<W*>(dw),
                                                                          static_cast<W*>(db));
  }
  return check_launch();
}

}  // namespace
}  // namespace f8b200

using namespace f8b200;

// Calls fn(T*, W*) with the types that the two codes name: w has x's type or fp32.
template <typename Fn>
static int ln_dispatch(int hp_dtype, int affine_dtype, Fn&& fn) {
  using B = __nv_bfloat16;
  if (hp_dtype == F8B200_FP32) return fn(static_cast<float*>(nullptr), static_cast<float*>(nullptr));
  if (hp_dtype == F8B200_BF16)
    return affine_dtype == F8B200_FP32 ? fn(static_cast<B*>(nullptr), static_cast<float*>(nullptr))
                                       : fn(static_cast<B*>(nullptr), static_cast<B*>(nullptr));
  return affine_dtype == F8B200_FP32 ? fn(static_cast<__half*>(nullptr), static_cast<float*>(nullptr))
                                     : fn(static_cast<__half*>(nullptr), static_cast<__half*>(nullptr));
}

static bool ln_types_ok(int hp_dtype, int affine_dtype) {
  return hp_dtype >= 0 && hp_dtype <= 2 && (affine_dtype == hp_dtype || affine_dtype == F8B200_FP32);
}
static bool ln_aligned(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (uintptr_t)hp_size_of(dtype) == 0; }

extern "C" int f8b200_layer_norm(const void* x, int hp_dtype, int64_t rows, int64_t cols, int64_t ld_x, const void* weight,
                                 const void* bias, int affine_dtype, float eps, void* y, int64_t ld_y, float* mean_out,
                                 float* rstd_out, void* stream) {
  if (!ln_types_ok(hp_dtype, affine_dtype) || rows < 0 || cols <= 0) return F8B200_ERR_BAD_ARG;
  if ((mean_out == nullptr) != (rstd_out == nullptr)) return F8B200_ERR_BAD_ARG;
  if (rows == 0) return F8B200_OK;
  if (x == nullptr || y == nullptr || ld_x < cols || ld_y < cols) return F8B200_ERR_BAD_ARG;
  if (!ln_aligned(x, hp_dtype) || !ln_aligned(y, hp_dtype) || !ln_aligned(weight, affine_dtype) || !ln_aligned(bias, affine_dtype))
    return F8B200_ERR_ALIGNMENT;
  const int rc = f8b200_device_check();
  if (rc != F8B200_OK) return rc;
  return ln_dispatch(hp_dtype, affine_dtype, [&](auto* t, auto* w) {
    return ln_fwd<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(w)>>(
        x, rows, cols, ld_x, weight, bias, eps, y, ld_y, mean_out, rstd_out, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int64_t f8b200_layer_norm_bwd_workspace_bytes(int64_t cols) {
  return cols <= 0 ? 0 : (int64_t)kMaxParts * 2 * cols * (int64_t)sizeof(float);
}

extern "C" int f8b200_layer_norm_bwd(const void* x, const void* grad_y, int hp_dtype, int64_t rows, int64_t cols, int64_t ld_x,
                                     int64_t ld_g, const void* weight, int affine_dtype, const float* mean, const float* rstd,
                                     void* dx, int64_t ld_dx, void* dweight, void* dbias, void* workspace,
                                     int64_t workspace_bytes, void* stream) {
  if (!ln_types_ok(hp_dtype, affine_dtype) || rows <= 0 || cols <= 0) return F8B200_ERR_BAD_ARG;
  if (x == nullptr || grad_y == nullptr || mean == nullptr || rstd == nullptr) return F8B200_ERR_BAD_ARG;
  if (ld_x < cols || ld_g < cols || (dx != nullptr && ld_dx < cols)) return F8B200_ERR_BAD_ARG;
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (sums && (workspace == nullptr || workspace_bytes < f8b200_layer_norm_bwd_workspace_bytes(cols))) return F8B200_ERR_BAD_ARG;
  if (!ln_aligned(x, hp_dtype) || !ln_aligned(grad_y, hp_dtype) || !ln_aligned(dx, hp_dtype) ||
      !ln_aligned(weight, affine_dtype) || !ln_aligned(dweight, affine_dtype) || !ln_aligned(dbias, affine_dtype) ||
      reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return F8B200_ERR_ALIGNMENT;
  const int rc = f8b200_device_check();
  if (rc != F8B200_OK) return rc;
  return ln_dispatch(hp_dtype, affine_dtype, [&](auto* t, auto* w) {
    return ln_bwd<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(w)>>(
        x, grad_y, rows, cols, ld_x, ld_g, weight, mean, rstd, dx, ld_dx, dweight, dbias, static_cast<float*>(workspace),
        static_cast<cudaStream_t>(stream));
  });
}
