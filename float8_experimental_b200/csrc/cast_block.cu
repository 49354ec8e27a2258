// Casts to fp8 with one scale per block of 128, and the way back.
//
// A block is 1 x 128 (by rows), 128 x 1 (by columns) or 128 x 128.  With a = max(max|x|, 1e-12) over the block and
// e the largest whole number with a * 2^e <= the format's maximum,
//     q = fp8(x * 2^e)  (nearest even),    scale_inv = 2^-e,    the block stands for q * scale_inv.
// A power of two moves the exponent only: neither the product nor its inverse rounds, so the only rounding of the
// cast is the one to fp8, and it costs no accuracy against amax / max: fp8 is a floating format, whose
// relative step does not depend on where in its range a value lies.  A block that holds an infinity
// or a NaN is stored as NaN in every place, with a NaN factor.
//
// One CTA takes a 128 x 128 tile, so every block lies inside one CTA and x is read once for all the forms asked
// for: 256 threads, 8 columns and 8 rows (16 apart) per thread, held in registers.
// Memory bounds it: 16384 x 8192 bf16 by rows 70 us (5.7 TB/s), by columns 73, by squares 72, by rows and columns 118
// (4.6 TB/s), back 71 (5.7), 75 from columns; per call of ten in a replayed graph.
#include "common.cuh"

namespace f8b200 {
namespace {

constexpr int kBlk = 128;
constexpr int kThreads = 256;
enum { kByRow = 1, kByCol = 2, kBySquare = 4 };

struct BlockCastArgs {
  const char* x;
  int64_t rows, cols, ld;  // elements
  uint8_t *out_r, *out_c;  // by rows or squares, by columns
  int64_t ld_r, ld_c;
  float *scale_r, *scale_c;
  int64_t ld_scale_r, ld_scale_c;
  uint8_t *exp_r, *exp_c;  // the factors' exponents as the tensor cores read them (see exponent_at); may be null
  int64_t exp_pitch_r, exp_pitch_c;
  int64_t tiles_k;
};

// Where the exponent byte of operand row `row` and block `kb` of the reduction lies: four blocks make one 32-bit
// word, 128 rows make 512 bytes in which row r has the word (r % 32) * 4 + r / 32 -- the order in which
// tcgen05.cp takes 32 x 16 bytes into tensor memory.  `pitch`: bytes of all rows (a multiple of 1024).
__device__ __forceinline__ int64_t exponent_at(int64_t row, int64_t kb, int64_t pitch) {
  return (kb >> 2) * pitch + (row >> 7) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (kb & 3);
}
__device__ __forceinline__ uint8_t exponent_of(float down) { return (uint8_t)((__float_as_uint(down) >> 23) & 0xFFu); }

// up = 2^e and down = 2^-e of a block whose amax has these fp32 bits
template <int KIND>
__device__ __forceinline__ void block_scale(uint32_t amax_bits, float& up, float& down) {
  if (amax_bits >= 0x7F800000u) {
    up = down = __uint_as_float(0x7FFFFFFFu);
    return;
  }
  const uint32_t a = max(amax_bits, __float_as_uint(kEps));
  // both maxima are 1.75 * 2^kTop: one power less when the amax's fraction exceeds 1.75
  constexpr int kTop = KIND == F8B200_E4M3 ? 8 : 15;
  const int e = kTop - ((int)(a >> 23) - 127) - ((a & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  up = __uint_as_float((uint32_t)(127 + e) << 23);
  down = __uint_as_float((uint32_t)(127 - e) << 23);
}

template <int HP>
__device__ __forceinline__ uint32_t widen_bits(uint32_t h) {  // |x| bits of a 16-bit type -> fp32 bits
  if constexpr (HP == F8B200_BF16) return h << 16;
  else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)h)));
}

// Eight consecutive elements of a row as they lie in memory: 16-bit types stay packed (half the registers, and two
// maxima per instruction).
template <int HP>
struct Eight {
  static constexpr int W = HP == F8B200_FP32 ? 8 : 4;
  uint32_t w[W];

  template <bool VEC>
  __device__ __forceinline__ void load(const char* p, int n) {  // n of them exist
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = 0u;
    if (VEC && n == 8) {
#pragma unroll
      for (int h = 0; h < W / 4; ++h) {
        const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p) + h);
        w[4 * h] = q.x, w[4 * h + 1] = q.y, w[4 * h + 2] = q.z, w[4 * h + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (j < n) {
          if constexpr (HP == F8B200_FP32) w[j] = __ldcs(reinterpret_cast<const uint32_t*>(p) + j);
          else w[j >> 1] |= (uint32_t)__ldcs(reinterpret_cast<const unsigned short*>(p) + j) << (16 * (j & 1));
        }
      }
    }
  }
  // element pair j as fp32
  __device__ __forceinline__ float2 pair(int j) const {
    if constexpr (HP == F8B200_FP32) return make_float2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
    else if constexpr (HP == F8B200_BF16) return make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
  }
  // |x| bits of word j, and the larger of two such words: unsigned order is the order of the values, NaN above infinity
  __device__ __forceinline__ uint32_t abs_word(int j) const { return w[j] & (HP == F8B200_FP32 ? 0x7FFFFFFFu : 0x7FFF7FFFu); }
  __device__ __forceinline__ static uint32_t larger(uint32_t a, uint32_t b) { return HP == F8B200_FP32 ? max(a, b) : __vmaxu2(a, b); }
};

template <bool VEC>
__device__ __forceinline__ void store8(uint8_t* p, int n, uint32_t lo, uint32_t hi) {
  if (VEC && n == 8) {
    *reinterpret_cast<uint2*>(p) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
}

template <int HP, int KIND, int FORMS, bool VEC>
__global__ void __launch_bounds__(kThreads, HP == F8B200_FP32 ? 2 : (FORMS == kByRow || FORMS == kByCol) ? 4 : 3) cast_block_kernel(const BlockCastArgs p) {
  __shared__ __align__(16) uint32_t col_max[kThreads / 32][16 * Eight<HP>::W];
  __shared__ uint32_t warp_max[kThreads / 32];
  __shared__ float factors[2][kBlk];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t tm = blockIdx.x / p.tiles_k, tk = blockIdx.x - tm * p.tiles_k;
  const int64_t row0 = tm * kBlk, col = tk * kBlk + tx * 8;
  const int n = (int)max((int64_t)0, min((int64_t)8, p.cols - col));
  constexpr int kEs = HP == F8B200_FP32 ? 4 : 2;

  using V = Eight<HP>;
  constexpr int W = V::W;
  V v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = row0 + ty + 16 * i;
    v[i].template load<VEC>(p.x + (r * p.ld + col) * kEs, r < p.rows ? n : 0);
  }

  if constexpr (FORMS & kByCol) {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      uint32_t m = v[0].abs_word(j);
#pragma unroll
      for (int i = 1; i < 8; ++i) m = V::larger(m, v[i].abs_word(j));
      m = V::larger(m, __shfl_xor_sync(0xFFFFFFFFu, m, 16));
      if (lane < 16) col_max[warp][tx * W + j] = m;
    }
  }
  uint32_t rmax[8];  // fp32: |x| bits; 16 bits: of rows 2i and 2i + 1 in rmax[i]
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint32_t m = v[i].abs_word(0);
#pragma unroll
    for (int j = 1; j < W; ++j) m = V::larger(m, v[i].abs_word(j));
    if constexpr (HP == F8B200_FP32) {
      rmax[i] = m;
    } else {
      m = max(m & 0xFFFFu, m >> 16);
      if (i & 1) rmax[i >> 1] |= m << 16;
      else rmax[i >> 1] = m;
    }
  }
  constexpr int R = HP == F8B200_FP32 ? 8 : 4;
  float up_sq = 0.f;
  if constexpr (FORMS & kBySquare) {
    uint32_t m = rmax[0];
#pragma unroll
    for (int i = 1; i < R; ++i) m = V::larger(m, rmax[i]);
    if constexpr (HP != F8B200_FP32) m = widen_bits<HP>(max(m & 0xFFFFu, m >> 16));
    m = warp_max_u32(m);
    if (lane == 0) warp_max[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) m = max(m, warp_max[w]);
    float down;
    block_scale<KIND>(m, up_sq, down);
    if (threadIdx.x == 0) p.scale_r[tm * p.ld_scale_r + tk] = down;
    if (p.exp_r != nullptr) {  // one factor for 128 rows of the matrix and of its transpose
      const int t = threadIdx.x & 127;
      if (threadIdx.x < 128) p.exp_r[exponent_at(row0 + t, tk, p.exp_pitch_r)] = exponent_of(down);
      else p.exp_c[exponent_at(tk * kBlk + t, tm, p.exp_pitch_c)] = exponent_of(down);
    }
  }

  if constexpr (FORMS & (kByRow | kBySquare)) {
    if constexpr (FORMS & kByRow) {
#pragma unroll
      for (int off = 8; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < R; ++i) rmax[i] = V::larger(rmax[i], __shfl_xor_sync(0xFFFFFFFFu, rmax[i], off));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = row0 + ty + 16 * i;
      float up = up_sq;
      if constexpr (FORMS & kByRow) {
        float down;
        uint32_t m = rmax[i / (8 / R)];
        if constexpr (HP != F8B200_FP32) m = widen_bits<HP>((i & 1) ? m >> 16 : m & 0xFFFFu);
        block_scale<KIND>(m, up, down);
        if (tx == 0) factors[0][ty + 16 * i] = down;
      }
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = v[i].pair(j);
        w[j] = cvt_pair_raw<KIND>(f.x * up, f.y * up);
      }
      if (r < p.rows) store8<VEC>(p.out_r + r * p.ld_r + col, n, w[0] | (w[1] << 16), w[2] | (w[3] << 16));
    }
  }
  if constexpr (FORMS & kByCol) {
    __syncthreads();  // behind the rows' work: the column maxima of the other warps have had time to arrive
    float up[8];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      uint32_t m = col_max[0][tx * W + j];
#pragma unroll
      for (int w = 1; w < kThreads / 32; ++w) m = V::larger(m, col_max[w][tx * W + j]);
#pragma unroll
      for (int h = 0; h < 8 / W; ++h) {
        const int c = j * (8 / W) + h;
        float down;
        if constexpr (HP == F8B200_FP32) block_scale<KIND>(m, up[c], down);
        else block_scale<KIND>(widen_bits<HP>(h ? m >> 16 : m & 0xFFFFu), up[c], down);
        if (ty == 0) factors[1][tx * 8 + c] = down;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = row0 + ty + 16 * i;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = v[i].pair(j);
        w[j] = cvt_pair_raw<KIND>(f.x * up[2 * j], f.y * up[2 * j + 1]);
      }
      if (r < p.rows) store8<VEC>(p.out_c + r * p.ld_c + col, n, w[0] | (w[1] << 16), w[2] | (w[3] << 16));
    }
  }
  if constexpr ((FORMS & (kByRow | kByCol)) != 0) {
    // the tile's factors leave together, neighbours from neighbouring threads: stored by the threads that found them,
    // one here and one there, they cost as much as the bytes (this step took both forms of 16384 x 8192 bf16 from 330 to
    // 148 us, packed maxima from there to 118)
    __syncthreads();
    const int t = threadIdx.x & 127;
    if (threadIdx.x < 128) {
      const int64_t r = row0 + t;
      if ((FORMS & kByRow) && r < p.rows) {
        p.scale_r[tk * p.ld_scale_r + r] = factors[0][t];
        if (p.exp_r != nullptr) p.exp_r[exponent_at(r, tk, p.exp_pitch_r)] = exponent_of(factors[0][t]);
      }
    } else {
      const int64_t c = tk * kBlk + t;
      if ((FORMS & kByCol) && c < p.cols) {
        p.scale_c[tm * p.ld_scale_c + c] = factors[1][t];
        if (p.exp_c != nullptr) p.exp_c[exponent_at(c, tm, p.exp_pitch_c)] = exponent_of(factors[1][t]);
      }
    }
  }
}

template <int HP, int KIND, bool VEC>
int launch_forms(const BlockCastArgs& p, int forms, int64_t tiles, cudaStream_t st) {
  const unsigned grid = (unsigned)tiles;
  if (forms == kByRow) cast_block_kernel<HP, KIND, kByRow, VEC><<<grid, kThreads, 0, st>>>(p);
  else if (forms == kByCol) cast_block_kernel<HP, KIND, kByCol, VEC><<<grid, kThreads, 0, st>>>(p);
  else if (forms == (kByRow | kByCol)) cast_block_kernel<HP, KIND, kByRow | kByCol, VEC><<<grid, kThreads, 0, st>>>(p);
  else cast_block_kernel<HP, KIND, kBySquare, VEC><<<grid, kThreads, 0, st>>>(p);
  return check_launch();
}

// fp8 -> T: y = q * scale(block), in the tiles of the cast: 8 columns and 8 rows, 16 apart, per thread, so that
// column factors are fetched once for eight rows.
struct BlockUncastArgs {
  const uint8_t* q;
  int64_t rows, cols, ld_q;
  const float* scale;
  int64_t s_row, s_col;      // strides of the factors
  int row_shift, col_shift;  // 7: one factor per 128 rows / columns, 0: per row / column
  char* y;
  int64_t ld_y;
  int64_t tiles_k;
};

template <int HP>
__device__ __forceinline__ void store_hp(char* base, int64_t i, float v) {
  if constexpr (HP == F8B200_BF16) reinterpret_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
  else if constexpr (HP == F8B200_FP16) reinterpret_cast<__half*>(base)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(base)[i] = v;
}

template <int HP, int KIND, bool VEC>
__global__ void __launch_bounds__(kThreads) uncast_block_kernel(const BlockUncastArgs p) {
  constexpr __nv_fp8_interpretation_t kInterp = KIND == F8B200_E4M3 ? __NV_E4M3 : __NV_E5M2;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t tm = blockIdx.x / p.tiles_k, tk = blockIdx.x - tm * p.tiles_k;
  const int64_t row0 = tm * kBlk, col = tk * kBlk + tx * 8;
  const int n = (int)max((int64_t)0, min((int64_t)8, p.cols - col));
  if (n == 0) return;
  uint32_t w[8][2];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = row0 + ty + 16 * i;
    const uint8_t* q = p.q + r * p.ld_q + col;
    w[i][0] = w[i][1] = 0u;
    if (r < p.rows) {
      if (VEC && n == 8) {
        const uint2 t = __ldcs(reinterpret_cast<const uint2*>(q));
        w[i][0] = t.x, w[i][1] = t.y;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < n) w[i][j >> 2] |= (uint32_t)q[j] << (8 * (j & 3));
      }
    }
  }
  float sc[8], sr[8];  // factors of the columns, or, where blocks are 128 columns wide, of the rows
  const bool per_col = p.col_shift == 0, per_row = p.row_shift == 0;
  if (per_col) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sc[j] = j < n ? __ldg(p.scale + (row0 >> p.row_shift) * p.s_row + (col + j) * p.s_col) : 0.f;
  }
  if (!per_col) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int64_t r = row0 + ty + 16 * i;
      sr[i] = r < p.rows ? __ldg(p.scale + (r >> p.row_shift) * p.s_row + (col >> p.col_shift) * p.s_col) : 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = row0 + ty + 16 * i;
    if (r >= p.rows) continue;
    if (!per_col) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sc[j] = sr[i];
    } else if (per_row) {  // one factor per element
#pragma unroll
      for (int j = 0; j < 8; ++j) sc[j] = j < n ? __ldg(p.scale + r * p.s_row + (col + j) * p.s_col) : 0.f;
    }
    float y[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((w[i][j >> 1] >> (16 * (j & 1))) & 0xFFFFu), kInterp);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      y[2 * j] = f.x * sc[2 * j];
      y[2 * j + 1] = f.y * sc[2 * j + 1];
    }
    if (VEC && n == 8) {
      if constexpr (HP == F8B200_FP32) {
        float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.y) + r * p.ld_y + col);
        __stcs(o, make_float4(y[0], y[1], y[2], y[3]));
        __stcs(o + 1, make_float4(y[4], y[5], y[6], y[7]));
      } else {
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (HP == F8B200_BF16) {
            const __nv_bfloat162 t = __floats2bfloat162_rn(y[2 * j], y[2 * j + 1]);
            h[j] = *reinterpret_cast<const uint32_t*>(&t);
          } else {
            const __half2 t = __floats2half2_rn(y[2 * j], y[2 * j + 1]);
            h[j] = *reinterpret_cast<const uint32_t*>(&t);
          }
        }
        __stcs(reinterpret_cast<uint4*>(p.y + (r * p.ld_y + col) * 2), make_uint4(h[0], h[1], h[2], h[3]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) store_hp<HP>(p.y, r * p.ld_y + col + j, y[j]);
    }
  }
}

bool aligned(const void* p, int64_t to) { return p == nullptr || reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace
}  // namespace f8b200

using namespace f8b200;

static int64_t exponent_pitch(int64_t rows) { return (rows + 255) / 256 * 256 * 4; }

extern "C" int64_t f8b200_block_exponent_bytes(int64_t rows, int64_t k) {
  return rows <= 0 || k <= 0 ? 0 : exponent_pitch(rows) * ((k + 511) / 512);
}

extern "C" int f8b200_cast_blockwise(const void* x, int hp_dtype, int64_t rows, int64_t cols, int64_t ld_x, int fp8_kind,
                                     int by_square, void* out_r, int64_t ld_r, float* scale_r, int64_t ld_scale_r,
                                     void* exp_r, void* out_c, int64_t ld_c, float* scale_c, int64_t ld_scale_c,
                                     void* exp_c, void* stream) {
  if (hp_dtype < 0 || hp_dtype > 2 || fp8_kind < 0 || fp8_kind > 1 || rows < 0 || cols < 0) return F8B200_ERR_BAD_ARG;
  if (out_r == nullptr && out_c == nullptr) return F8B200_ERR_BAD_ARG;
  if (by_square != 0 && (out_r == nullptr || out_c != nullptr || (exp_r == nullptr) != (exp_c == nullptr))) return F8B200_ERR_BAD_ARG;
  if ((exp_r != nullptr && out_r == nullptr) || (exp_c != nullptr && out_c == nullptr && by_square == 0)) return F8B200_ERR_BAD_ARG;
  if (rows == 0 || cols == 0) return F8B200_OK;
  const int64_t tiles_m = (rows + kBlk - 1) / kBlk, tiles_k = (cols + kBlk - 1) / kBlk;
  if (x == nullptr || ld_x < cols) return F8B200_ERR_BAD_ARG;
  if (out_r != nullptr && (scale_r == nullptr || ld_r < cols || ld_scale_r < (by_square ? tiles_k : rows))) return F8B200_ERR_BAD_ARG;
  if (out_c != nullptr && (scale_c == nullptr || ld_c < cols || ld_scale_c < cols)) return F8B200_ERR_BAD_ARG;
  if (tiles_m > 0x7FFFFFFFLL / tiles_k) return F8B200_ERR_UNSUPPORTED;
  const int es = hp_size_of(hp_dtype);
  if (!aligned(x, es) || !aligned(scale_r, 4) || !aligned(scale_c, 4) || !aligned(exp_r, 16) || !aligned(exp_c, 16)) return F8B200_ERR_ALIGNMENT;
  int rc = f8b200_device_check();
  if (rc != F8B200_OK) return rc;
  BlockCastArgs p;
  p.x = static_cast<const char*>(x);
  p.rows = rows, p.cols = cols, p.ld = ld_x;
  p.out_r = static_cast<uint8_t*>(out_r), p.out_c = static_cast<uint8_t*>(out_c);
  p.ld_r = ld_r, p.ld_c = ld_c;
  p.scale_r = scale_r, p.scale_c = scale_c;
  p.ld_scale_r = ld_scale_r, p.ld_scale_c = ld_scale_c;
  p.exp_r = static_cast<uint8_t*>(exp_r), p.exp_c = static_cast<uint8_t*>(exp_c);
  p.exp_pitch_r = exponent_pitch(rows), p.exp_pitch_c = exponent_pitch(cols);
  p.tiles_k = tiles_k;
  const int forms = by_square ? kBySquare : (out_r != nullptr ? kByRow : 0) | (out_c != nullptr ? kByCol : 0);
  // rows that allow 16-byte loads and 8-byte stores; the last chunk of a row may be shorter
  const bool vec = (ld_x * es) % 16 == 0 && aligned(x, 16) && aligned(out_r, 8) && aligned(out_c, 8) &&
                   (out_r == nullptr || ld_r % 8 == 0) && (out_c == nullptr || ld_c % 8 == 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t tiles = tiles_m * tiles_k;
#define F8_CAST(HP, KIND) (vec ? launch_forms<HP, KIND, true>(p, forms, tiles, st) : launch_forms<HP, KIND, false>(p, forms, tiles, st))
  if (fp8_kind == F8B200_E4M3) {
    if (hp_dtype == F8B200_BF16) return F8_CAST(F8B200_BF16, F8B200_E4M3);
    if (hp_dtype == F8B200_FP16) return F8_CAST(F8B200_FP16, F8B200_E4M3);
    return F8_CAST(F8B200_FP32, F8B200_E4M3);
  }
  if (hp_dtype == F8B200_BF16) return F8_CAST(F8B200_BF16, F8B200_E5M2);
  if (hp_dtype == F8B200_FP16) return F8_CAST(F8B200_FP16, F8B200_E5M2);
  return F8_CAST(F8B200_FP32, F8B200_E5M2);
#undef F8_CAST
}

extern "C" int f8b200_uncast_blockwise(const void* q, int fp8_kind, int64_t rows, int64_t cols, int64_t ld_q,
                                       const float* scale, int64_t scale_row_stride, int64_t scale_col_stride,
                                       int block_rows, int block_cols, int hp_dtype, void* y, int64_t ld_y, void* stream) {
  if (hp_dtype < 0 || hp_dtype > 2 || fp8_kind < 0 || fp8_kind > 1 || rows < 0 || cols < 0) return F8B200_ERR_BAD_ARG;
  if ((block_rows != 1 && block_rows != kBlk) || (block_cols != 1 && block_cols != kBlk)) return F8B200_ERR_BAD_ARG;
  if (rows == 0 || cols == 0) return F8B200_OK;
  if (q == nullptr || scale == nullptr || y == nullptr || ld_q < cols || ld_y < cols) return F8B200_ERR_BAD_ARG;
  if (scale_row_stride < 0 || scale_col_stride < 0) return F8B200_ERR_BAD_ARG;
  const int es = hp_size_of(hp_dtype);
  if (!aligned(y, es) || !aligned(scale, 4)) return F8B200_ERR_ALIGNMENT;
  int rc = f8b200_device_check();
  if (rc != F8B200_OK) return rc;
  BlockUncastArgs p;
  p.q = static_cast<const uint8_t*>(q);
  p.rows = rows, p.cols = cols, p.ld_q = ld_q;
  p.scale = scale, p.s_row = scale_row_stride, p.s_col = scale_col_stride;
  p.row_shift = block_rows == kBlk ? 7 : 0, p.col_shift = block_cols == kBlk ? 7 : 0;
  p.y = static_cast<char*>(y), p.ld_y = ld_y;
  p.tiles_k = (cols + kBlk - 1) / kBlk;
  const int64_t tiles_m = (rows + kBlk - 1) / kBlk;
  if (tiles_m > 0x7FFFFFFFLL / p.tiles_k) return F8B200_ERR_UNSUPPORTED;
  const bool vec = ld_q % 8 == 0 && aligned(q, 8) && aligned(y, 16) && (ld_y * es) % 16 == 0;
  const unsigned grid = (unsigned)(tiles_m * p.tiles_k);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define F8_UNCAST(HP, KIND)                                                                   \
  (vec ? (void)(uncast_block_kernel<HP, KIND, true><<<grid, kThreads, 0, st>>>(p))            \
       : (void)(uncast_block_kernel<HP, KIND, false><<<grid, kThreads, 0, st>>>(p)))
  if (fp8_kind == F8B200_E4M3) {
    if (hp_dtype == F8B200_BF16) F8_UNCAST(F8B200_BF16, F8B200_E4M3);
    else if (hp_dtype == F8B200_FP16) F8_UNCAST(F8B200_FP16, F8B200_E4M3);
    else F8_UNCAST(F8B200_FP32, F8B200_E4M3);
  } else {
    if (hp_dtype == F8B200_BF16) F8_UNCAST(F8B200_BF16, F8B200_E5M2);
    else if (hp_dtype == F8B200_FP16) F8_UNCAST(F8B200_FP16, F8B200_E5M2);
    else F8_UNCAST(F8B200_FP32, F8B200_E5M2);
  }
#undef F8_UNCAST
  return check_launch();
}
