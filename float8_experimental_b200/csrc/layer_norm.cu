// Layer norm over the last dimension, forward and backward.
//   mean = sum(x) / C,  var = sum((x - mean)^2) / C,  rstd = 1 / sqrt(var + eps),  n = (x - mean) * rstd
//   y  = n * w + b
//   dx = rstd * (h - sum(h) / C - n * sum(h * n) / C),  h = g * w
//   dw = sum over rows of g * n,   db = sum over rows of g
// All in fp32 whatever the type of x; y, dx, dw and db are rounded once.  The first mean m is off by about |mean| * 2^-24
// (its sum, and 1 / C, are rounded), which is much where the mean is large against the spread, so the second pass adds up
// what it leaves:  d = x - m,  r = sum(d) / C,  var = sum(d^2) / C - r^2,  n = d * rstd - r * rstd.  The forward's n then costs
// no digits to a large mean; the backward takes the mean m + r as it was stored, rounded to fp32.
// w and b have x's type or fp32; either may be absent (1 and 0).  Sums run in a fixed order.
//
// Memory bounds both directions: x read and y written (4 bytes per 16-bit element), x and g read and dx written (6).
// 16384 x 8192 bf16, per call of ten in a replayed graph: forward 93 us, 5.8 TB/s; backward 155 us, 5.2 TB/s.
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

// Sum over the ROWT threads of a row (a warp, several, or the whole CTA), the same value in all of them.  Successive
// calls take two buffers in turn: a buffer is written again only behind the other one's barrier, so one barrier
// per sum is enough.
template <int ROWT>
__device__ __forceinline__ float row_sum(float v, float* smem) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, off);
  if constexpr (ROWT > 32) {
    constexpr int W = ROWT / 32;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, group = threadIdx.x / ROWT;
    if (lane == 0) smem[w] = v;
    if constexpr (ROWT == kThreads) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(ROWT) : "memory");
    v = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += smem[group * W + i];
  }
  return v;
}

// The same of two values at once, behind one barrier.
template <int ROWT>
__device__ __forceinline__ float2 row_sum2(float a, float b, float2* smem) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    a += __shfl_xor_sync(0xFFFFFFFFu, a, off);
    b += __shfl_xor_sync(0xFFFFFFFFu, b, off);
  }
  if constexpr (ROWT > 32) {
    constexpr int W = ROWT / 32;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, group = threadIdx.x / ROWT;
    if (lane == 0) smem[w] = make_float2(a, b);
    if constexpr (ROWT == kThreads) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(ROWT) : "memory");
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float2 v = smem[group * W + i];
      a += v.x;
      b += v.y;
    }
  }
  return make_float2(a, b);
}

// two fp32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 w, x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 w, {%6, %7};\n\tfma.rn.f32x2 z, x, y, w;\n\tmov.b64 {%0, %1}, z;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// r and rstd from the sums of d and d^2 (a rounding below zero is none; a NaN stays)
__device__ __forceinline__ float2 residual_and_rstd(float2 sums, float inv_c, float eps) {
  const float r = sums.x * inv_c, var = fmaf(-r, r, sums.y * inv_c);
  return make_float2(r, 1.0f / sqrtf((var < 0.f ? 0.f : var) + eps));
}

// ---- forward, a row in registers --------------------------------------------------------------------
// As few threads per row as hold it in four 16-byte pieces each: several rows per CTA then wait for their sums at
// different times (16384 x 4096 bf16 with 128 threads per row 53 us, with 256 66 us; 32768 x 2048 with 64 53 us, with 256
// 76 us, with one warp and eight pieces 59 us).  Arithmetic in pairs keeps the second sum of the second pass free
// (16384 x 8192, single calls with cold caches as above: 102 us with it, 100 without, 106 element by element); groups of
// less than a CTA need four CTAs per SM (53 us against 59 with three).
template <typename T, typename W, int ROWT, int CH>
__global__ void __launch_bounds__(kThreads, ROWT < kThreads && CH > 1 ? 4 : 0)
ln_fwd_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, const W* __restrict__ weight,
              const W* __restrict__ bias, float eps, T* __restrict__ y, int64_t ld_y, float* __restrict__ mean_out,
              float* __restrict__ rstd_out) {
  constexpr int N = Vec<T>::N, RPB = kThreads / ROWT;
  __shared__ float smem[kThreads / 32];
  __shared__ float2 smem2[kThreads / 32];
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
    const float first = row_sum<ROWT>(s, smem) * inv_c;
    float2 s2 = make_float2(0.f, 0.f), d2 = s2;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      if (t + i * ROWT < chunks) {
        float v[N];
        Vec<T>::widen(q[i], v);
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const float2 d = add2(make_float2(v[j], v[j + 1]), make_float2(-first, -first));
          d2 = add2(d2, d);
          s2 = fma2(d, d, s2);
        }
      }
    }
    const float2 rest = residual_and_rstd(row_sum2<ROWT>(d2.x + d2.y, s2.x + s2.y, smem2), inv_c, eps);
    const float rstd = rest.y, shift = -rest.x * rstd;
    if (t == 0 && mean_out != nullptr) {
      mean_out[r] = first + rest.x;
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
        for (int j = 0; j < N; j += 2) {
          const float2 d = add2(make_float2(v[j], v[j + 1]), make_float2(-first, -first));
          const float2 n = fma2(d, make_float2(rstd, rstd), make_float2(shift, shift));
          const float2 r2 = fma2(n, make_float2(w[j], w[j + 1]), make_float2(b[j], b[j + 1]));
          v[j] = r2.x, v[j + 1] = r2.y;
        }
        __stcs(out + c, Vec<T>::narrow(v));
      }
    }
  }
}

// ---- backward, rows through a ring of private slots -----------------------------------------------------
// Each thread copies its own 16-byte pieces of the coming rows of x and g to shared memory (cp.async, STAGES - 1 rows
// ahead) and reads back only those: the memory system is kept busy across the row sums without a barrier for the
// data.  dw and db gather in registers over all rows of the CTA, which leaves one partial sum per CTA: x and g are read
// once for all three gradients.
constexpr int kBwdThreads = 512;

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// N affine values held as they lie in memory, so that they cost few registers over the whole loop.
template <typename W, int N>
struct Packed {
  static constexpr int Q = N / Vec<W>::N;
  uint4 q[Q];
  __device__ __forceinline__ void load(const W* p, int64_t i) {
#pragma unroll
    for (int h = 0; h < Q; ++h) q[h] = __ldg(reinterpret_cast<const uint4*>(p + i) + h);
  }
  __device__ __forceinline__ void set_one() {
    float v[Vec<W>::N];
#pragma unroll
    for (int j = 0; j < Vec<W>::N; ++j) v[j] = 1.f;
#pragma unroll
    for (int h = 0; h < Q; ++h) q[h] = Vec<W>::narrow(v);
  }
  __device__ __forceinline__ void get(float (&v)[N]) const {
#pragma unroll
    for (int h = 0; h < Q; ++h) {
      float t[Vec<W>::N];
      Vec<W>::widen(q[h], t);
#pragma unroll
      for (int j = 0; j < Vec<W>::N; ++j) v[h * Vec<W>::N + j] = t[j];
    }
  }
};

template <typename T, typename W, int ROWT, int CH, int R, int STAGES>
__global__ void __launch_bounds__(kBwdThreads, 1)
ln_bwd_kernel(const T* __restrict__ x, int64_t ld_x, const T* __restrict__ g, int64_t ld_g, int64_t rows, int64_t cols,
              const W* __restrict__ weight, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
              T* __restrict__ dx, int64_t ld_dx, float* __restrict__ part) {
  constexpr int N = Vec<T>::N, GROUPS = kBwdThreads / ROWT, WARPS = ROWT / 32;
  extern __shared__ uint4 ring[];  // [STAGES][R rows][x, g][CH][thread]
  __shared__ float sums[2][kBwdThreads / 32][2 * R];
  const int t = threadIdx.x % ROWT, group = threadIdx.x / ROWT, lane = threadIdx.x & 31;
  const int chunks = (int)(cols / N);
  const float inv_c = 1.0f / (float)cols;
  // a group takes R rows at a time: one exchange of sums serves them all
  const int64_t sets = (rows + R - 1) / R, step = (int64_t)gridDim.x * GROUPS;
  auto slot = [&](int stage, int u, int which, int i) {
    return ring + (((stage * R + u) * 2 + which) * CH + i) * kBwdThreads + threadIdx.x;
  };
  auto fetch = [&](int64_t p, int stage) {
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int64_t r = R * p + u;
      if (r < rows) {
        const uint4 *xr = reinterpret_cast<const uint4*>(x + r * ld_x), *gr = reinterpret_cast<const uint4*>(g + r * ld_g);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int c = t + i * ROWT;
          if (c < chunks) {
            cp_async16(slot(stage, u, 0, i), xr + c);
            cp_async16(slot(stage, u, 1, i), gr + c);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto stats = [&](int64_t p, float (&mean)[R], float (&rstd)[R]) {
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const bool in = R * p + u < rows;
      mean[u] = in ? __ldg(mean_in + R * p + u) : 0.f;
      rstd[u] = in ? __ldg(rstd_in + R * p + u) : 0.f;
    }
  };

  float dw[CH][N], db[CH][N];
  Packed<W, N> w[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    if (weight != nullptr && t + i * ROWT < chunks) w[i].load(weight, (int64_t)(t + i * ROWT) * N);
    else w[i].set_one();
#pragma unroll
    for (int j = 0; j < N; ++j) dw[i][j] = db[i][j] = 0.f;
  }

  int64_t p = (int64_t)blockIdx.x * GROUPS + group;
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(p + s * step, s);
  float mean[R], rstd[R];
  stats(p, mean, rstd);
  int stage = 0, flip = 0;
  for (; p < sets; p += step) {
    float mean_next[R], rstd_next[R];
    stats(p + step, mean_next, rstd_next);  // their latency passes behind this set's work
    cp_async_wait<STAGES - 2>();
    float s[2 * R] = {};
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const bool row_in = R * p + u < rows;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const bool in = row_in && t + i * ROWT < chunks;
        float xv[N], gv[N], wv[N];
        Vec<T>::widen(in ? *slot(stage, u, 0, i) : make_uint4(0u, 0u, 0u, 0u), xv);
        Vec<T>::widen(in ? *slot(stage, u, 1, i) : make_uint4(0u, 0u, 0u, 0u), gv);
        w[i].get(wv);
#pragma unroll
        for (int j = 0; j < N; ++j) {  // where there is no element, g is 0 and so is everything below
          const float n = (xv[j] - mean[u]) * rstd[u], h = gv[j] * wv[j];
          s[2 * u] += h;
          s[2 * u + 1] = fmaf(h, n, s[2 * u + 1]);
          dw[i][j] = fmaf(gv[j], n, dw[i][j]);
          db[i][j] += gv[j];
        }
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
#pragma unroll
      for (int q = 0; q < 2 * R; ++q) s[q] += __shfl_xor_sync(0xFFFFFFFFu, s[q], off);
    if constexpr (WARPS > 1) {  // two buffers: the next set's sums may be written while these are read
      if (lane == 0) {
#pragma unroll
        for (int q = 0; q < 2 * R; ++q) sums[flip][threadIdx.x >> 5][q] = s[q];
      }
      if constexpr (ROWT == kBwdThreads) __syncthreads();
      else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(ROWT) : "memory");
#pragma unroll
      for (int q = 0; q < 2 * R; ++q) {
        s[q] = 0.f;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) s[q] += sums[flip][group * WARPS + v][q];
      }
      flip ^= 1;
    }
    fetch(p + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
    if (dx != nullptr) {
#pragma unroll
      for (int u = 0; u < R; ++u) {
        if (R * p + u >= rows) continue;
        const float a = s[2 * u] * inv_c, b = s[2 * u + 1] * inv_c;
        uint4* out = reinterpret_cast<uint4*>(dx + (R * p + u) * ld_dx);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int c = t + i * ROWT;
          if (c < chunks) {
            float xv[N], gv[N], wv[N];
            Vec<T>::widen(*slot(stage, u, 0, i), xv);  // still there: held in registers the rows would cost 32 of them
            Vec<T>::widen(*slot(stage, u, 1, i), gv);
            w[i].get(wv);
#pragma unroll
            for (int j = 0; j < N; ++j) {
              const float n = (xv[j] - mean[u]) * rstd[u];
              gv[j] = rstd[u] * (fmaf(gv[j], wv[j], -a) - n * b);
            }
            __stcs(out + c, Vec<T>::narrow(gv));
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < R; ++u) mean[u] = mean_next[u], rstd[u] = rstd_next[u];
    if (++stage == STAGES) stage = 0;
  }
  if (part == nullptr) return;
  asm volatile("cp.async.wait_all;" ::: "memory");
  // the groups' sums over each other, dw and db in turn, through the ring
  float* sm = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (t + i * ROWT < chunks) {
#pragma unroll
        for (int j = 0; j < N; ++j) sm[group * cols + (int64_t)(t + i * ROWT) * N + j] = which == 0 ? dw[i][j] : db[i][j];
      }
    __syncthreads();
    for (int c = threadIdx.x; c < (int)cols; c += kBwdThreads) {
      float v = 0.f;
#pragma unroll
      for (int q = 0; q < GROUPS; ++q) v += sm[q * cols + c];
      part[((int64_t)blockIdx.x * 2 + which) * cols + c] = v;
    }
  }
}

// ---- any width, any alignment -----------------------------------------------------------------------
// Element by element, neighbours by neighbouring threads, so the accesses still fill whole lines.  A short row stays in
// registers between the sums (up to 16 elements per thread forward, 4 backward: with two rows of values in registers too
// few warps fit, 16384 x 3001 took twice the time); a longer one (E = 0) is read again from the caches.
template <typename T, typename W, int E>
__global__ void __launch_bounds__(kThreads)
ln_fwd_any_kernel(const T* __restrict__ x, int64_t ld_x, int64_t rows, int64_t cols, const W* __restrict__ weight,
                  const W* __restrict__ bias, float eps, T* __restrict__ y, int64_t ld_y, float* __restrict__ mean_out,
                  float* __restrict__ rstd_out) {
  __shared__ float smem[kThreads / 32];
  __shared__ float2 smem2[kThreads / 32];
  const float inv_c = 1.0f / (float)cols;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = x + r * ld_x;
    float v[E > 0 ? E : 1];
    // fn(column, the row's value there)
    auto each = [&](auto&& fn) {
      if constexpr (E > 0) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int c = (int)threadIdx.x + i * kThreads;
          if (c < (int)cols) fn((int64_t)c, v[i]);
        }
      } else {
        for (int64_t c = threadIdx.x; c < cols; c += kThreads) fn(c, to_f32(row[c]));
      }
    };
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = (int)threadIdx.x + i * kThreads;
        v[i] = c < (int)cols ? to_f32(row[c]) : 0.f;
      }
    }
    float s = 0.f;
    each([&](int64_t, float a) { s += a; });
    const float first = row_sum<kThreads>(s, smem) * inv_c;
    s = 0.f;
    float d = 0.f;
    each([&](int64_t, float a) {
      d += a - first;
      s = fmaf(a - first, a - first, s);
    });
    const float2 rest = residual_and_rstd(row_sum2<kThreads>(d, s, smem2), inv_c, eps);
    const float rstd = rest.y, shift = -rest.x * rstd;
    if (threadIdx.x == 0 && mean_out != nullptr) {
      mean_out[r] = first + rest.x;
      rstd_out[r] = rstd;
    }
    each([&](int64_t c, float a) {
      const float w = weight != nullptr ? to_f32(weight[c]) : 1.f, b = bias != nullptr ? to_f32(bias[c]) : 0.f;
      y[r * ld_y + c] = from_f32<T>(fmaf(fmaf(a - first, rstd, shift), w, b));
    });
  }
}

template <typename T, typename W, int E>
__global__ void __launch_bounds__(kThreads)
ln_dx_any_kernel(const T* __restrict__ x, int64_t ld_x, const T* __restrict__ g, int64_t ld_g, int64_t rows, int64_t cols,
                 const W* __restrict__ weight, const float* __restrict__ mean_in, const float* __restrict__ rstd_in,
                 T* __restrict__ dx, int64_t ld_dx) {
  __shared__ float smem[2][kThreads / 32];
  const float inv_c = 1.0f / (float)cols;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * ld_x, *gr = g + r * ld_g;
    const float mean = mean_in[r], rstd = rstd_in[r];
    float n[E > 0 ? E : 1], h[E > 0 ? E : 1];
    auto load = [&](int64_t c, float& nv, float& hv) {
      nv = (to_f32(xr[c]) - mean) * rstd;
      hv = to_f32(gr[c]) * (weight != nullptr ? to_f32(weight[c]) : 1.f);
    };
    auto each = [&](auto&& fn) {
      if constexpr (E > 0) {
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const int c = (int)threadIdx.x + i * kThreads;
          if (c < (int)cols) fn((int64_t)c, n[i], h[i]);
        }
      } else {
        for (int64_t c = threadIdx.x; c < cols; c += kThreads) {
          float nv, hv;
          load(c, nv, hv);
          fn(c, nv, hv);
        }
      }
    };
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int c = (int)threadIdx.x + i * kThreads;
        n[i] = h[i] = 0.f;
        if (c < (int)cols) load(c, n[i], h[i]);
      }
    }
    float s1 = 0.f, s2 = 0.f;
    each([&](int64_t, float nv, float hv) {
      s1 += hv;
      s2 = fmaf(hv, nv, s2);
    });
    s1 = row_sum<kThreads>(s1, smem[0]) * inv_c;
    s2 = row_sum<kThreads>(s2, smem[1]) * inv_c;
    each([&](int64_t c, float nv, float hv) { dx[r * ld_dx + c] = from_f32<T>(rstd * (hv - s1 - nv * s2)); });
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
#pragma unroll 4
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
  else if (vec && chunks <= 256) F8_LN(64, 4);
  else if (vec && chunks <= 512) F8_LN(128, 4);
  else if (vec && chunks <= 1024) F8_LN(256, 4);
  else if (vec && chunks <= 2048) F8_LN(256, 8);
#undef F8_LN
#define F8_LN(E) ln_fwd_any_kernel<T, W, E><<<row_grid(rows), kThreads, 0, st>>>(xp, ld_x, rows, cols, wp, bp, eps, yp, ld_y, mean, rstd)
  else if (cols <= 4 * kThreads) F8_LN(4);
  else if (cols <= 8 * kThreads) F8_LN(8);
  else if (cols <= 16 * kThreads) F8_LN(16);
  else F8_LN(0);
#undef F8_LN
  return check_launch();
}

template <typename T, typename W, int ROWT, int CH, int R, int STAGES>
int ln_bwd_launch(const T* x, int64_t ld_x, const T* g, int64_t ld_g, int64_t rows, int64_t cols, const W* weight,
                  const float* mean, const float* rstd, T* dx, int64_t ld_dx, float* part, int* parts, cudaStream_t st) {
  constexpr int kGroups = kBwdThreads / ROWT;
  constexpr int kSmem = STAGES * R * 2 * CH * kBwdThreads * 16;
  static_assert(kGroups * ROWT * CH * Vec<T>::N * 4 <= kSmem, "the groups' sums have to fit into the ring");
  static PerDeviceOnce setup;
  auto kernel = ln_bwd_kernel<T, W, ROWT, CH, R, STAGES>;
  const cudaError_t e = setup.run([&](int*) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem); });
  if (e != cudaSuccess) return record_cuda_error(e);
  const int64_t need = ((rows + R - 1) / R + kGroups - 1) / kGroups;
  int64_t grid = sm_count() < kMaxParts ? sm_count() : kMaxParts;
  if (need < grid) grid = need;
  kernel<<<(unsigned)grid, kBwdThreads, kSmem, st>>>(x, ld_x, g, ld_g, rows, cols, weight, mean, rstd, dx, ld_dx, part);
  *parts = (int)grid;
  return check_launch();
}

template <typename T, typename W>
int ln_bwd(const void* x, const void* g, int64_t rows, int64_t cols, int64_t ld_x, int64_t ld_g, const void* weight,
           const float* mean, const float* rstd, void* dx, int64_t ld_dx, void* dw, void* db, float* part, cudaStream_t st) {
  const T *xp = static_cast<const T*>(x), *gp = static_cast<const T*>(g);
  constexpr int N = Vec<T>::N;
  const int64_t chunks = cols / N;
  const bool vec = cols % N == 0 && chunks <= 2048 && ld_x % N == 0 && ld_g % N == 0 && (dx == nullptr || ld_dx % N == 0) &&
                   aligned16(x) && aligned16(g) && aligned16(dx) && aligned16(weight);
  if (vec) {
    int parts = 0, rc = F8B200_OK;
    float* sums = dw != nullptr || db != nullptr ? part : nullptr;
#define F8_LN(ROWT, CH, R, STAGES)                                                                                           \
  rc = ln_bwd_launch<T, W, ROWT, CH, R, STAGES>(xp, ld_x, gp, ld_g, rows, cols, static_cast<const W*>(weight), mean, rstd, \
                                             static_cast<T*>(dx), ld_dx, sums, &parts, st)
    // the narrowest group of threads that takes a row in two pieces each: 32 accumulators for 16-bit rows
    if (chunks <= 64) F8_LN(32, 2, 2, 3);
    else if (chunks <= 128) F8_LN(64, 2, 2, 3);
    else if (chunks <= 256) F8_LN(128, 2, 2, 3);
    else if (chunks <= 512) F8_LN(256, 2, 2, 3);
    else if (chunks <= 1024) F8_LN(512, 2, 1, 6);
    else F8_LN(512, 4, 1, 3);
#undef F8_LN
    if (rc != F8B200_OK) return rc;
    if (sums != nullptr)
      ln_dw_join_kernel<W><<<(unsigned)((cols + 31) / 32), kThreads, 0, st>>>(part, parts, cols, static_cast<W*>(dw),
                                                                            static_cast<W*>(db));
    return check_launch();
  }
#define F8_LN(E)                                                                                                      \
  ln_dx_any_kernel<T, W, E><<<row_grid(rows), kThreads, 0, st>>>(xp, ld_x, gp, ld_g, rows, cols, static_cast<const W*>(weight), \
                                                                 mean, rstd, static_cast<T*>(dx), ld_dx)
  if (dx == nullptr) {}
  else if (cols <= 4 * kThreads) F8_LN(4);
  else F8_LN(0);
#undef F8_LN
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
  if (!ln_aligned(x, hp_dtype) || !ln_aligned(y, hp_dtype) || !ln_aligned(weight, affine_dtype) || !ln_aligned(bias, affine_dtype) ||
      !ln_aligned(mean_out, F8B200_FP32) || !ln_aligned(rstd_out, F8B200_FP32))
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
      !ln_aligned(mean, F8B200_FP32) || !ln_aligned(rstd, F8B200_FP32) || !ln_aligned(weight, affine_dtype) || !ln_aligned(dweight, affine_dtype) || !ln_aligned(dbias, affine_dtype) ||
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
