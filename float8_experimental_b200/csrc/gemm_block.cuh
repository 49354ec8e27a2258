// fp8 GEMM with one scale per block of 128 along K (included by gemm.cu, whose device helpers it uses):
//   out[m,n] = sum_j sa(m,j) * sb(n,j) * (sum_{k in block j} A[m,k] * B[n,k])  (+ bias[n])
// sa has one fp32 factor per row of A or per 128 rows, sb the same for B; both are read through two strides,
// so a transposed or broadcast scale tensor needs no copy.
//
// The scale changes with the 128-wide block of K, so the tensor cores' sum over one block is a value of its
// own: every block's MMAs start a fresh tensor-memory accumulator, and the epilogue warps add it, multiplied by
// its scale, to fp32 sums that stay in registers for the whole tile.  Per block that costs a 128x256 tile's
// CTA 32768 fp32 FMAs (256 cycles of its FMA pipes) and as many tensor-memory words against the 512 cycles of the
// MMAs, and two accumulators alternate so that it can run beside them.  It does not quite: 16384 x 8192 x 8192 takes
// 1.11 ms (1.98 PFLOP/s), and at 4096 x 4096 x 8192 the tensor pipe is active 38 % of the time, the FMA pipe 19 %, so each
// waits for the other's hand-over.  With a factor per row on both sides there is one more multiplication per
// element and a shared-memory read per pair (that pipe 50 % busy, the tensor pipe 22 %): 2.11 ms.
//
// Factors that are powers of two go to a third kernel, below, which leaves them to the tensor cores.  Two kernels here:
//   block pair kernel   two CTAs per 256x256 tile, tcgen05.mma.cta_group::2 as in the pair kernel of gemm.cu;
//                       eight epilogue warps per CTA, one row and 128 columns per thread.
//   few-rows kernel     A has few rows (tokens being served): B's rows take the 128-wide side of the MMA and A's
//                       the narrow one, and the CTAs of a cluster split K and join their sums through
//                       distributed shared memory, so that a product of a few tiles still uses every SM's share
//                       of the memory bandwidth that B's bytes need.
// Both are bounded in every wait like the kernels of gemm.cu.

namespace f8b200 {
namespace gemm {
namespace block {

using namespace pair;

// factor of (row, block j) = p[(row >> shift) * row_stride + j * kb_stride]
struct BlockScale {
  const float* p;
  int64_t row_stride, kb_stride;
  int shift;  // 0: one factor per row, 7: per 128 rows
};

__device__ __forceinline__ void tc_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// two fp32 values in one 64-bit register pair
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  return v;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) { return pack2(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  uint32_t a, b;
  asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
  lo = __uint_as_float(a);
  hi = __uint_as_float(b);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2f(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// TMA warp, MMA warp, two that only make their group whole, 8 epilogue warps.  A thread of the epilogue holds 128 sums,
// more than the 168 registers that 12 warps get each leave room for: the first group hands 128 of its own over
// (40 + 2 * 232 = 3 * 168).
constexpr int BTHREADS = 384;
constexpr int BREGS_FEW = 40, BREGS_MANY = 232;
constexpr int BSTAGES = 6;
constexpr int BSTAGE_BYTES = PA_BYTES + PB_BYTES;

struct __align__(16) BlockBars {
  float col_scale[8][2][128];  // per epilogue warp, two k-blocks: the factors of its 128 columns of B
  uint64_t full[BSTAGES];
  uint64_t empty[BSTAGES];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};
constexpr int BSMEM_BYTES = BSTAGES * BSTAGE_BYTES + 1024 + (int)sizeof(BlockBars);

// PER_COL: B has one factor per row (a column of the output); otherwise one per 128 of them, which is one per
// epilogue thread and k-block because a thread's 128 columns start on a multiple of 128.
template <typename OutT, bool PER_COL>
__global__ void __launch_bounds__(BTHREADS, 1)
gemm_block_pair_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                       const BlockScale scale_a, const BlockScale scale_b, const OutT* __restrict__ bias,
                       OutT* __restrict__ out, int64_t ldo, int m, int n, int k, uint32_t idesc, int out_vec_ok,
                       int raster) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  BlockBars* bars = reinterpret_cast<BlockBars*>(tiles + BSTAGES * BSTAGE_BYTES);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t peer = rank ^ 1u;
  const bool leader = rank == 0;
  const int tiles_m = (m + PBM - 1) / PBM, tiles_n = (n + PBN - 1) / PBN;
  const int64_t num_tiles = (int64_t)tiles_m * tiles_n;
  const int num_kb = (k + BK - 1) / BK;
  const int64_t cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
  const bool a_mn = (raster >> LAYOUT_A_MN_BIT) & 1, b_mn = (raster >> LAYOUT_B_MN_BIT) & 1;
  const uint64_t step_a = desc_k_step(a_mn), step_b = desc_k_step(b_mn);

  if (threadIdx.x == 0) {
    for (int s = 0; s < BSTAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&bars->tmem_full[a], 1);
      mbar_init(&bars->tmem_empty[a], 16);
    }
    bars->abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                 "r"((uint32_t)TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(BREGS_FEW));
    if (warp == 0) {
      // ---------------- TMA producer (one per CTA) ----------------
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int64_t t = cluster_id; ok && t < num_tiles; t += num_clusters) {
          const TileCoord tc = tile_coord(t, tiles_m, tiles_n, raster);
          const int row_a = tc.m * PBM + (int)rank * 128;
          const int row_b = tc.n * PBN + (int)rank * 128;
          for (int kb = 0; kb < num_kb; ++kb) {
            if (!pair_wait(&bars->empty[stage], phase ^ 1u, bars, peer, 1u, 64u)) { ok = false; break; }
            uint8_t* sa = tiles + stage * BSTAGE_BYTES;
            if (leader) mbar_expect_tx(&bars->full[stage], 2 * BSTAGE_BYTES);
            const uint32_t full_in_leader = mapa_u32(smem_u32(&bars->full[stage]), 0u);
            tma_load_2d_pair_plain(sa, &tma_a, a_mn ? row_a : kb * BK, a_mn ? kb * BK : row_a, full_in_leader);
            tma_load_2d_pair_plain(sa + PA_BYTES, &tma_b, b_mn ? row_b : kb * BK, b_mn ? kb * BK : row_b,
                                   full_in_leader);
            if (++stage == BSTAGES) { stage = 0; phase ^= 1u; }
          }
        }
        // tail: every release the leader multicast to this CTA's empty barriers has landed
        for (int s = 0; ok && s < BSTAGES; ++s) {
          if (!pair_wait(&bars->empty[stage], phase ^ 1u, bars, peer, 1u, 64u)) { ok = false; break; }
          if (++stage == BSTAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) {  // give the loads in flight time to land before the CTA leaves
          const long long t0 = clock64();
          while (clock64() - t0 < 2000000LL) {}
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer (leader CTA only) ----------------
      if (leader && lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        uint32_t g = 0;  // k-blocks issued so far: their accumulators alternate
        for (int64_t t = cluster_id; ok && t < num_tiles; t += num_clusters) {
          for (int kb = 0; kb < num_kb; ++kb, ++g) {
            const uint32_t acc = g & 1u;
            if (!pair_wait(&bars->full[stage], phase, bars, peer, 4u)) { ok = false; break; }
            if (!pair_wait(&bars->tmem_empty[acc], ((g >> 1) & 1u) ^ 1u, bars, peer, 2u)) { ok = false; break; }
            tc_fence_after();
            const uint32_t a_addr = smem_u32(tiles + stage * BSTAGE_BYTES);
            const uint64_t da = a_mn ? make_smem_desc_mn(a_addr, PA_BYTES) : make_smem_desc(a_addr);
            const uint64_t db = b_mn ? make_smem_desc_mn(a_addr + PA_BYTES, PB_BYTES) : make_smem_desc(a_addr + PA_BYTES);
            const uint32_t tmem_d = tmem_base + acc * (uint32_t)PBN;
  #pragma unroll
            for (int kk = 0; kk < BK / UMMA_K; ++kk)
              tc_mma_f8_pair(tmem_d, da + (uint64_t)kk * step_a, db + (uint64_t)kk * step_b, idesc, kk != 0 ? 1u : 0u);
            tc_commit_pair(&bars->empty[stage]);
            tc_commit_pair(&bars->tmem_full[acc]);
            if (++stage == BSTAGES) { stage = 0; phase ^= 1u; }
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(BREGS_MANY));
    // ---------------- epilogue (warps 4..11 of both CTAs) ----------------
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t taddr0 = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 128);
    const uint32_t empty_in_leader[2] = {mapa_u32(smem_u32(&bars->tmem_empty[0]), 0u),
                                         mapa_u32(smem_u32(&bars->tmem_empty[1]), 0u)};
    bool ok = true;
    uint32_t g = 0;
    for (int64_t t = cluster_id; ok && t < num_tiles; t += num_clusters) {
      const TileCoord tc = tile_coord(t, tiles_m, tiles_n, raster);
      const int row = tc.m * PBM + (int)rank * 128 + quarter * 32 + lane;
      const int col0 = tc.n * PBN + half * 128;
      const bool row_in = row < m, cols_in = col0 < n;
      const float* pa = scale_a.p + (int64_t)((row_in ? row : 0) >> scale_a.shift) * scale_a.row_stride;
      const float* pb = scale_b.p + (int64_t)((cols_in ? col0 : 0) >> scale_b.shift) * scale_b.row_stride;
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0ull;
      float sa = row_in ? __ldg(pa) : 0.f;
      float sb = 0.f, sc[4] = {0.f, 0.f, 0.f, 0.f};
      auto load_cols = [&](int kb) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = col0 + lane + 32 * j;
          sc[j] = c < n ? __ldg(scale_b.p + (int64_t)(c >> scale_b.shift) * scale_b.row_stride +
                                (int64_t)kb * scale_b.kb_stride) : 0.f;
        }
      };
      if constexpr (PER_COL) load_cols(0); else sb = cols_in ? __ldg(pb) : 0.f;
      for (int kb = 0; kb < num_kb; ++kb, ++g) {
        const uint32_t buf = g & 1u;
        // Alternating over all blocks, not within the tile: before a buffer is written again every lane has passed the
        // barriers of the block between, behind its own reads.
        const float* cs = bars->col_scale[warp - 4][buf];
        if constexpr (PER_COL) {
          float* w = bars->col_scale[warp - 4][buf];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[lane + 32 * j] = sc[j];
          __syncwarp();
        }
        const float s = PER_COL ? sa : sa * sb;
        const uint64_t s2 = pack2(s, s);
        if (kb + 1 < num_kb) {  // the next block's factors travel while this one is added up
          sa = row_in ? __ldg(pa + (int64_t)(kb + 1) * scale_a.kb_stride) : 0.f;
          if constexpr (PER_COL) load_cols(kb + 1);
          else sb = cols_in ? __ldg(pb + (int64_t)(kb + 1) * scale_b.kb_stride) : 0.f;
        }
        if (!pair_wait(&bars->tmem_full[buf], (g >> 1) & 1u, bars, peer, 8u)) { ok = false; break; }
        __syncwarp();
        tc_fence_after();
        const uint32_t taddr = taddr0 + buf * (uint32_t)PBN;
        uint32_t r[2][16];
        tc_ld_32x32b_x16(taddr, r[0]);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          tc_wait_ld();
          if (c < 7) {
            tc_ld_32x32b_x16(taddr + (uint32_t)(16 * (c + 1)), r[(c + 1) & 1]);
          } else {  // everything is in registers: the accumulator is free for the MMAs of the next but one block
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(empty_in_leader[buf]);
          }
          const uint32_t(&v)[16] = r[c & 1];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint64_t f = s2;
            if constexpr (PER_COL) f = mul2f(s2, *reinterpret_cast<const uint64_t*>(cs + c * 16 + 2 * i));
            acc[c * 8 + i] = fma2(pack2(v[2 * i], v[2 * i + 1]), f, acc[c * 8 + i]);
          }
        }
      }
      if (!ok) break;
      if (row_in) {
        OutT* orow = out + (int64_t)row * ldo;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = col0 + c * 32;
          const int ncols = min(32, n - col);
          if (ncols > 0) {
            float v[32];
#pragma unroll
            for (int i = 0; i < 16; ++i) unpack2(acc[c * 16 + i], v[2 * i], v[2 * i + 1]);
            if (bias != nullptr) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (i < ncols) v[i] += static_cast<float>(bias[col + i]);
            }
            store_chunk<OutT>(orow + col, v, ncols, out_vec_ok != 0);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the other may still touch its barriers or TMEM
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)TMEM_COLS)
                 : "memory");
  }
}

// ---------------------------------------------------------------------------------------------------
// Few rows of A.  D[128 rows of B, T rows of A] per CTA, K split over the CTAs of a cluster.
// ---------------------------------------------------------------------------------------------------
// Per CTA and k-block: 16 KB of B, T x 128 bytes of A.  With up to 64 rows two CTAs share an SM, so that one's join
// and start-up lie beside the other's loads; four epilogue warps add up 64 columns each thread, and twice as many do
// for 128 rows.
template <int T>
struct FewCfg {
  static constexpr int kCols = T < 64 ? T : 64;              // accumulator columns per epilogue warp
  static constexpr int kEpiWarps = 4 * (T / kCols);
  static constexpr int kThreads = 64 + 32 * kEpiWarps;       // TMA warp, MMA warp, epilogue
  static constexpr int kCtas = T <= 64 ? 2 : 1;              // per SM
  static constexpr int kXBytes = T * BK;
  static constexpr int kStageBytes = 128 * BK + kXBytes;
  static constexpr int kStages = T <= 32 ? 5 : T <= 64 ? 4 : 6;
  static constexpr int kBufs = 512 / kCtas / T < 4 ? 512 / kCtas / T : 4;  // accumulators that alternate
  static constexpr int kTmemCols = kBufs * T < 32 ? 32 : kBufs * T;
  static constexpr int kJoinBytes = T * 128 * 4;             // fp32 sums handed over at the end, over the stages
  static_assert(kJoinBytes <= kStages * kStageBytes, "the sums have to fit into the stages");
  static_assert((kBufs & (kBufs - 1)) == 0 && kBufs >= 2, "buffers are chosen by the low bits of a counter");
};
template <int T>
struct __align__(16) FewBars {
  using Cfg = FewCfg<T>;
  float x_scale[Cfg::kEpiWarps][2][Cfg::kCols];  // per epilogue warp, two k-blocks: the factors of its columns (A's rows)
  uint64_t full[Cfg::kStages];
  uint64_t empty[Cfg::kStages];
  uint64_t tmem_full[Cfg::kBufs];
  uint64_t tmem_empty[Cfg::kBufs];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};
template <int T>
constexpr int few_smem_bytes() {
  return FewCfg<T>::kStages * FewCfg<T>::kStageBytes + 1024 + (int)sizeof(FewBars<T>);
}
template <typename Bars>
__device__ __forceinline__ bool few_wait(uint64_t* bar, uint32_t parity, Bars* bars, uint32_t who) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (uint32_t it = 0; it < 0x7FFFFFFFu; ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 63u) {
      if (bars->abort_flag != 0u) return false;
      if (clock64() - t0 > WAIT_BUDGET_CYCLES) break;
    }
  }
  bars->abort_flag = 1u;
  atomicOr(&g_device_error, who | 0x200u);
  return false;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr) : "memory");
  return v;
}

constexpr int FEW_MAX_SPLIT = 8;  // the portable cluster size

// grid: x = K split (the cluster), y = tiles of 128 rows of B, z = tiles of T rows of A.  `uniform`: B has one factor
// per 128 rows, i.e. one per CTA and k-block, which then goes into A's factors once per block instead of into every FMA.
template <typename OutT, int T>
__global__ void __launch_bounds__(FewCfg<T>::kThreads, FewCfg<T>::kCtas)
gemm_block_few_kernel(const __grid_constant__ CUtensorMap tma_w, const __grid_constant__ CUtensorMap tma_x,
                      const BlockScale scale_w, const BlockScale scale_x, const OutT* __restrict__ bias,
                      OutT* __restrict__ out, int64_t ldo, int m, int n, int k, uint32_t idesc, int w_mn, int out_vec_ok) {
  using Cfg = FewCfg<T>;
  constexpr int S = Cfg::kStages, C = Cfg::kCols, BUFS = Cfg::kBufs;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  FewBars<T>* bars = reinterpret_cast<FewBars<T>*>(tiles + S * Cfg::kStageBytes);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = (int)gridDim.x;
  const uint32_t rank = split > 1 ? cluster_ctarank() : 0u;
  const int num_kb_all = (k + BK - 1) / BK;
  const int kb0 = (int)((int64_t)num_kb_all * rank / split), kb1 = (int)((int64_t)num_kb_all * (rank + 1) / split);
  const int row_w = (int)blockIdx.y * 128, row_x = (int)blockIdx.z * T;
  // Each tile of B starts at another k-block of its share and wraps around: in step, all CTAs would ask for the same
  // 128 bytes of A's rows and for equal offsets of B's at the same time (72 against 61 us at 37 x 28672 x 8192).
  const int rot = (int)(((int64_t)blockIdx.y * 5) % max(1, kb1 - kb0));
  auto block_of = [&](int i) { const int v = i + rot; return v < kb1 ? v : v - (kb1 - kb0); };
  const uint64_t step_w = desc_k_step(w_mn != 0), step_x = desc_k_step(false);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int a = 0; a < BUFS; ++a) {
      mbar_init(&bars->tmem_full[a], 1);
      mbar_init(&bars->tmem_empty[a], Cfg::kEpiWarps);
    }
    bars->abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                 "r"((uint32_t)Cfg::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;

  bool good = true;
  uint64_t acc[C / 2];
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!few_wait(&bars->empty[stage], phase ^ 1u, bars, 1u)) { ok = false; break; }
        uint8_t* sw = tiles + stage * Cfg::kStageBytes;
        mbar_expect_tx(&bars->full[stage], Cfg::kStageBytes);
        const int at = block_of(kb) * BK;
        tma_load_2d(sw, &tma_w, w_mn ? row_w : at, w_mn ? at : row_w, &bars->full[stage]);
        tma_load_2d(sw + 128 * BK, &tma_x, at, row_x, &bars->full[stage]);
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
      // tail: the MMAs have read every stage (the stages are reused for the sums below)
      for (int s = 0; ok && s < S; ++s) {
        if (!few_wait(&bars->empty[stage], phase ^ 1u, bars, 1u)) { ok = false; break; }
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
      if (!ok) {  // give the loads in flight time to land before the CTA leaves
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {}
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, g = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++g) {
        const uint32_t buf = g & (BUFS - 1);
        if (!few_wait(&bars->full[stage], phase, bars, 4u)) break;
        if (!few_wait(&bars->tmem_empty[buf], ((g / BUFS) & 1u) ^ 1u, bars, 2u)) break;
        tc_fence_after();
        const uint32_t w_addr = smem_u32(tiles + stage * Cfg::kStageBytes);
        const uint64_t dw = w_mn ? make_smem_desc_mn(w_addr, 128 * BK) : make_smem_desc(w_addr);
        const uint64_t dx = make_smem_desc(w_addr + 128 * BK);
#pragma unroll
        for (int kk = 0; kk < BK / UMMA_K; ++kk)
          tc_mma_f8(tmem_base + buf * T, dw + (uint64_t)kk * step_w, dx + (uint64_t)kk * step_x, idesc, kk != 0 ? 1u : 0u);
        tc_commit(&bars->empty[stage]);
        tc_commit(&bars->tmem_full[buf]);
        if (++stage == S) { stage = 0; phase ^= 1u; }
      }
    }
  } else {
    const int quarter = warp & 3, part = (warp - 2) >> 2;  // 32 rows of B, C rows of A
    const int row = row_w + quarter * 32 + lane;
    const bool row_in = row < n;
    const bool uniform = scale_w.shift == 7;
    const float* pw = scale_w.p + (int64_t)((row_in ? row : row_w) >> scale_w.shift) * scale_w.row_stride;
    constexpr int XL = (C + 31) / 32;  // factors of A's rows that one lane fetches per k-block
    const float* px[XL];
    bool px_in[XL];
#pragma unroll
    for (int j = 0; j < XL; ++j) {
      const int r = row_x + part * C + lane + 32 * j;
      px_in[j] = lane + 32 * j < C && r < m;
      px[j] = scale_x.p + (int64_t)((px_in[j] ? r : 0) >> scale_x.shift) * scale_x.row_stride;
    }
    float sx[XL], sw = 0.f;
    auto fetch = [&](int i) {
      const int kb = block_of(i);
      sw = __ldg(pw + (int64_t)kb * scale_w.kb_stride);
#pragma unroll
      for (int j = 0; j < XL; ++j) sx[j] = px_in[j] ? __ldg(px[j] + (int64_t)kb * scale_x.kb_stride) : 0.f;
    };
#pragma unroll
    for (int i = 0; i < C / 2; ++i) acc[i] = 0ull;
    if (kb0 < kb1) fetch(kb0);
    uint32_t g = 0;
    const uint32_t taddr0 = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(part * C);
    for (int kb = kb0; kb < kb1; ++kb, ++g) {
      const uint32_t buf = g & (BUFS - 1);
      float* xs = bars->x_scale[warp - 2][kb & 1];
#pragma unroll
      for (int j = 0; j < XL; ++j)
        if (lane + 32 * j < C) xs[lane + 32 * j] = uniform ? sx[j] * sw : sx[j];
      __syncwarp();
      const float s = sw;
      if (kb + 1 < kb1) fetch(kb + 1);
      if (!few_wait(&bars->tmem_full[buf], (g / BUFS) & 1u, bars, 8u)) { good = false; break; }
      __syncwarp();
      tc_fence_after();
      uint32_t r[C / 16][16];
#pragma unroll
      for (int c = 0; c < C / 16; ++c) tc_ld_32x32b_x16(taddr0 + buf * T + c * 16, r[c]);
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->tmem_empty[buf]);
      if (uniform) {
#pragma unroll
        for (int c = 0; c < C / 4; ++c) {
          const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(xs + 4 * c);
          acc[2 * c] = fma2(pack2(r[c / 4][(4 * c) & 15], r[c / 4][(4 * c + 1) & 15]), f.x, acc[2 * c]);
          acc[2 * c + 1] = fma2(pack2(r[c / 4][(4 * c + 2) & 15], r[c / 4][(4 * c + 3) & 15]), f.y, acc[2 * c + 1]);
        }
      } else {
        const uint64_t s2 = pack2(s, s);
#pragma unroll
        for (int c = 0; c < C / 4; ++c) {
          const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(xs + 4 * c);
          acc[2 * c] = fma2(pack2(r[c / 4][(4 * c) & 15], r[c / 4][(4 * c + 1) & 15]), mul2f(f.x, s2), acc[2 * c]);
          acc[2 * c + 1] = fma2(pack2(r[c / 4][(4 * c + 2) & 15], r[c / 4][(4 * c + 3) & 15]), mul2f(f.y, s2), acc[2 * c + 1]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)Cfg::kTmemCols)
                 : "memory");
  }

  // join: the sums lie as [A's row][128] in every CTA of the cluster; CTA r adds up and stores rows r, r + split, ...
  float* mine = reinterpret_cast<float*>(tiles);
  if (warp >= 2 && good) {
    const int r = (warp & 3) * 32 + lane, first = ((warp - 2) >> 2) * C;
#pragma unroll
    for (int i = 0; i < C / 2; ++i) {
      float lo, hi;
      unpack2(acc[i], lo, hi);
      mine[(first + 2 * i) * 128 + r] = lo;
      mine[(first + 2 * i + 1) * 128 + r] = hi;
    }
  }
  const bool failed = bars->abort_flag != 0u;
  if (split > 1) cluster_sync_all(); else __syncthreads();
  if (!failed) {
    const int rows_x = min(T, m - row_x);
    for (int e = (int)threadIdx.x; ; e += Cfg::kThreads) {
      const int i = (e >> 5) * split + (int)rank, c = (e & 31) * 4, col = row_w + c;
      if (i >= rows_x) break;
      if (col >= n) continue;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (split > 1) {
        const uint32_t addr = smem_u32(mine + i * 128 + c);
        float4 p[FEW_MAX_SPLIT];
#pragma unroll
        for (int q = 0; q < FEW_MAX_SPLIT; ++q)
          if (q < split) p[q] = ld_cluster_f32x4(mapa_u32(addr, (uint32_t)q));
#pragma unroll
        for (int q = 0; q < FEW_MAX_SPLIT; ++q)
          if (q < split) v[0] += p[q].x, v[1] += p[q].y, v[2] += p[q].z, v[3] += p[q].w;
      } else {
        const float4 p = *reinterpret_cast<const float4*>(mine + i * 128 + c);
        v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w;
      }
      const int ncols = min(4, n - col);
      __align__(16) OutT o[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        if (bias != nullptr && h < ncols) v[h] += static_cast<float>(bias[col + h]);
        o[h] = static_cast<OutT>(v[h]);
      }
      OutT* dst = out + (int64_t)(row_x + i) * ldo + col;
      if (out_vec_ok && ncols == 4) {  // rows start on 16-byte boundaries, columns on multiples of four
        if constexpr (sizeof(OutT) == 2) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
        else *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int h = 0; h < 4; ++h)
          if (h < ncols) dst[h] = o[h];
      }
    }
  }
  if (split > 1) cluster_sync_all();  // no CTA leaves while another may still read its sums
}

// ---------------------------------------------------------------------------------------------------
// Factors that are powers of two: the tensor cores apply them.  tcgen05.mma.kind::mxf8f6f4.block_scale multiplies the
// products of 32 consecutive k by 2^(ea + eb - 254), one exponent byte per operand row and 32 k, read from tensor
// memory; a block of 128 is four such steps with the same byte, so the accumulator stays in tensor memory over many
// of them and the epilogue runs once per tile and chunk of K.
//
// The tensor cores cut each new sum of a step of 32 k off towards zero at fp32's last place: the error has one sign and grows
// with the number of steps added to one accumulator (values of one sign, relative to the result: 5e-7 at K = 2048, 3.8e-6 at
// 8192, 1.9e-5 at 28672, 5.9e-5 at 65536; normal values a quarter to an eighth of that).  So K is cut into equal chunks of
// at most XCHUNK_* k-blocks, each with an accumulator of its own; eight epilogue warps per CTA add the chunks, rounding
// to nearest, in registers, one row and 128 columns per thread.  A chunk's hand-over costs half a microsecond per tile
// (16384 x 8192 x 8192: 833 us uncut, 834 with 64 k-blocks per chunk, 848 with 32, 877 with 16, 932 with 8).  16-bit outputs
// take 32: the error stays below 1.4e-6, a hundredth of fp16's half step and less of bf16's; fp32 outputs 16: below 5e-7.
//
// Tensor memory (512 columns): two accumulators of 256 columns that share 64 of them, at 0 and 192, and the
// factors at 448.  The epilogue reads the shared columns first and then lets the next chunk's MMAs start, which go to
// the other accumulator, while it drains the rest.
// Factors: one 32-bit word per operand row holds a group of four k-blocks' bytes.  Per group TMA brings 128 words of A
// (this CTA's rows) and 256 of B (the pair's), tcgen05.cp takes them to tensor memory, and the instruction descriptor
// says which byte an MMA uses.  A group's factors come with the stage of its first k-block
// and are copied right before that block's MMAs, into one of five sets in turn: a set must not be written before the
// MMAs of the group five earlier have finished, at least five k-blocks back, and the stage that the issuing thread has
// just found full means that the k-block XSTAGES earlier has been multiplied.  (Copies one group ahead, behind
// another block's MMAs, cost 2 % more time than copies that the group's own MMAs follow; a ring of their own
// with its own commits cost 9 %.)
// ---------------------------------------------------------------------------------------------------
constexpr int XTHREADS = BTHREADS;  // warps as in the kernel above; 56 + 2 * 224 = 3 * 168 registers
constexpr int XREGS_FEW = 56, XREGS_MANY = 224;  // the MMA warp's loop spills with 40 (1.2 % of the time)
constexpr int XSTAGES = 5;
constexpr int XSF_A = 512, XSF_B = 1024;  // bytes of factors per CTA and four k-blocks
constexpr int XSTAGE_BYTES = PA_BYTES + PB_BYTES;
constexpr int XACC_STEP = 192, XSF_COL = 448, XSF_SET = 12, XSF_SETS = 5;
constexpr int XSF_BYTES = 2048;  // of shared memory per stage, for the group that comes with it
static_assert(XSTAGES <= XSF_SETS && XSF_COL + XSF_SETS * XSF_SET <= TMEM_COLS, "see above");

struct __align__(16) ScaledBars {
  uint64_t full[XSTAGES];
  uint64_t empty[XSTAGES];
  uint64_t tmem_full[2];
  uint64_t tmem_shared_free;  // in the leader: 16 arrivals, the shared columns have been read
  TileRing ring;  // written in both CTAs by the leader's producer thread
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};
constexpr int XSTAGING_BYTES = 8 /*warps*/ * EPI_BOX_BYTES;
constexpr int XSMEM_BYTES = XSTAGES * (XSTAGE_BYTES + XSF_BYTES) + XSTAGING_BYTES + 1024 + (int)sizeof(ScaledBars);
constexpr int XCHUNK_32 = 16, XCHUNK_16 = 32;  // k-blocks per accumulator for fp32 and 16-bit outputs

__device__ __forceinline__ void tc_mma_mx_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                               uint32_t tmem_sa, uint32_t tmem_sb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
          tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(tmem_sa), "r"(tmem_sb), "r"(accumulate)
      : "memory");
}
// 512 bytes of shared memory, as 32 rows of 16, to 4 columns of tensor memory, repeated in the four lane quarters, in
// both CTAs of the pair from the same offset of their own shared memory
__device__ __forceinline__ void tc_copy_factors_pair(uint32_t taddr, uint32_t smem_addr) {
  uint64_t d = 0;  // no swizzle; groups of eight 16-byte rows are 128 bytes apart
  d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)(128 >> 4) << 16;
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

// Bits of the kind::mxf8f6f4 instruction descriptor: B's and A's factor byte at 4 and 29, formats at 7 and 10, MN-major
// at 15 and 16, N / 8 at 17, 8-bit exponent factors at 23, M / 16 at 24.
static uint32_t make_idesc_scaled(int a_kind, int b_kind, int a_mn, int b_mn) {
  return ((uint32_t)a_kind << 7) | ((uint32_t)b_kind << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(PBN >> 3) << 17) | (1u << 23) | ((uint32_t)(PBM >> 4) << 24);
}

// 64 columns of this warp's 32 rows to the output, through one staging box per warp (128 bytes wide).
template <typename OutT>
__device__ __forceinline__ void store_columns(const EpilogueArgs<OutT>& e, const float* v64, int row0, int col, uint32_t& boxes) {
  constexpr int COLS_PER_BOX = 128 / (int)sizeof(OutT);
  const int lane = threadIdx.x & 31, row = row0 + lane;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int c0 = col + 32 * h, ncols = min(32, e.n - c0);
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = v64[32 * h + i];
    if (e.bias != nullptr && ncols > 0) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i < ncols) v[i] += static_cast<float>(e.bias[c0 + i]);
    }
    if (!e.use_tma) {
      if (row < e.m && ncols > 0) store_chunk<OutT>(e.out + (int64_t)row * e.ldo + c0, v, ncols, e.out_vec_ok != 0);
      continue;
    }
    const bool first = COLS_PER_BOX == 32 || h == 0, last = COLS_PER_BOX == 32 || h == 1;
    const int box_col = COLS_PER_BOX == 32 ? c0 : col;
    if (box_col >= e.n || row0 >= e.m) continue;  // the same for the whole warp; partial boxes are clipped by the map
    if (first && boxes != 0u) {  // the store before this one must have read the box
      if (lane == 0) bulk_wait_read<0>();
      __syncwarp();
    }
    uint8_t* rowp = e.staging + lane * 128;  // 16-byte chunk j of row `lane` lives at j ^ (lane & 7)
    if constexpr (sizeof(OutT) == 2) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          OutT lo = static_cast<OutT>(v[q * 8 + 2 * t]), hi = static_cast<OutT>(v[q * 8 + 2 * t + 1]);
          w[t] = (uint32_t)(*reinterpret_cast<unsigned short*>(&lo)) | ((uint32_t)(*reinterpret_cast<unsigned short*>(&hi)) << 16);
        }
        *reinterpret_cast<uint4*>(rowp + (((h * 4 + q) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q)
        *reinterpret_cast<float4*>(rowp + ((q ^ (lane & 7)) << 4)) = make_float4(v[q * 4], v[q * 4 + 1], v[q * 4 + 2], v[q * 4 + 3]);
    }
    if (last) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        tma_store_2d_hint(e.tma_out, e.staging, box_col, row0, l2_policy(1));
        bulk_commit();
      }
      ++boxes;
    }
  }
}

template <typename OutT>
__global__ void __launch_bounds__(XTHREADS, 1)
gemm_block_scaled_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                         const __grid_constant__ CUtensorMap tma_ea, const __grid_constant__ CUtensorMap tma_eb,
                         const __grid_constant__ CUtensorMap tma_out, const OutT* __restrict__ bias,
                         OutT* __restrict__ out, int64_t ldo, int m, int n, int k, uint32_t idesc, int out_vec_ok,
                         int use_tma_store, int raster, int chunk_kb, uint32_t* sched) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* staging = tiles + XSTAGES * XSTAGE_BYTES;
  uint8_t* factors = staging + XSTAGING_BYTES;  // per stage: 512 bytes of A's, 1024 of B's
  ScaledBars* bars = reinterpret_cast<ScaledBars*>(factors + XSTAGES * XSF_BYTES);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t peer = rank ^ 1u;
  const bool leader = rank == 0;
  const int tiles_m = (m + PBM - 1) / PBM, tiles_n = (n + PBN - 1) / PBN;
  const int64_t num_tiles = (int64_t)tiles_m * tiles_n;
  const int num_kb = (k + BK - 1) / BK;
  const int64_t cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
  const bool a_mn = (raster >> LAYOUT_A_MN_BIT) & 1, b_mn = (raster >> LAYOUT_B_MN_BIT) & 1;
  const uint64_t step_a = desc_k_step(a_mn), step_b = desc_k_step(b_mn);

  if (threadIdx.x == 0) {
    for (int s = 0; s < XSTAGES; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    mbar_init(&bars->tmem_full[0], 1);
    mbar_init(&bars->tmem_full[1], 1);
    mbar_init(&bars->tmem_shared_free, 16);
    for (int r = 0; r < RING; ++r) mbar_init(&bars->ring.full[r], 1);
    bars->abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                 "r"((uint32_t)TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(XREGS_FEW));
    if (warp == 0) {
      // ---------------- TMA producer (one per CTA) ----------------
      if (lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        const int claim_kb = num_kb > 4 ? num_kb - 4 : 0;
        uint32_t entry = 0;  // ring entries published (leader) or read (partner) so far
        int64_t t = cluster_id;
        while (ok && t < num_tiles) {
          const TileCoord tc = tile_coord(t, tiles_m, tiles_n, raster);
          const int row_a = tc.m * PBM + (int)rank * 128;
          const int row_b = tc.n * PBN + (int)rank * 128;
          int64_t next = t + num_clusters;
          for (int kb = 0; kb < num_kb; ++kb) {
            if (sched != nullptr && leader && kb == claim_kb) next = num_clusters + (int64_t)atomicAdd(sched, 1u);
            if (!pair_wait(&bars->empty[stage], phase ^ 1u, bars, peer, 1u, 64u)) { ok = false; break; }
            uint8_t* sa = tiles + stage * XSTAGE_BYTES;
            const bool with_factors = (kb & 3) == 0;
            if (leader) mbar_expect_tx(&bars->full[stage], 2 * (XSTAGE_BYTES + (with_factors ? XSF_A + XSF_B : 0)));
            const uint32_t full_in_leader = mapa_u32(smem_u32(&bars->full[stage]), 0u);
            if (with_factors) {
              uint8_t* sf = factors + stage * XSF_BYTES;
              tma_load_2d_pair_plain(sf, &tma_ea, row_a, kb >> 2, full_in_leader);
              tma_load_2d_pair_plain(sf + XSF_A, &tma_eb, tc.n * PBN, kb >> 2, full_in_leader);
            }
            tma_load_2d_pair_plain(sa, &tma_a, a_mn ? row_a : kb * BK, a_mn ? kb * BK : row_a, full_in_leader);
            tma_load_2d_pair_plain(sa + PA_BYTES, &tma_b, b_mn ? row_b : kb * BK, b_mn ? kb * BK : row_b,
                                   full_in_leader);
            if (++stage == XSTAGES) { stage = 0; phase ^= 1u; }
          }
          if (!ok) break;
          if (sched != nullptr) {
            if (leader) {
              const uint32_t e = entry & (RING - 1);
              const int32_t v = next < num_tiles ? (int32_t)next : -1;
              bars->ring.tile[e] = v;
              mbar_arrive(&bars->ring.full[e]);
              st_cluster_u32(mapa_u32(smem_u32(&bars->ring.tile[e]), 1u), (uint32_t)v);
              mbar_arrive_release_cluster(mapa_u32(smem_u32(&bars->ring.full[e]), 1u));
            } else {
              const int32_t v = pair_ring_read(bars, entry, peer, 64u, 32u);
              if (v == -2) { ok = false; break; }
              next = v < 0 ? num_tiles : (int64_t)v;
            }
            ++entry;
          }
          t = next;
        }
        // tail: every release the leader multicast to this CTA's empty barriers has landed
        for (int s = 0; ok && s < XSTAGES; ++s) {
          if (!pair_wait(&bars->empty[stage], phase ^ 1u, bars, peer, 1u, 64u)) { ok = false; break; }
          if (++stage == XSTAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) {
          const long long t0 = clock64();
          while (clock64() - t0 < 2000000LL) {}
        }
      }
    } else if (warp == 1) {
      // ---------------- MMA issuer (leader CTA only) ----------------
      if (leader && lane == 0) {
        int stage = 0;
        uint32_t phase = 0;
        int set = 0;
        bool ok = true;
        uint32_t local = 0, chunk = 0;
        int64_t t = cluster_id;
        for (; ok && t < num_tiles; ++local) {
          for (int kb0 = 0; ok && kb0 < num_kb; kb0 += chunk_kb, ++chunk) {
            const uint32_t acc = chunk & 1u;
            const uint32_t tmem_d = tmem_base + acc * (uint32_t)XACC_STEP;
            // the columns that this accumulator shares with the previous chunk's have been read, and all of the one before
            if (chunk > 0 && !pair_wait(&bars->tmem_shared_free, (chunk - 1) & 1u, bars, peer, 2u)) { ok = false; break; }
            const int blocks = min(chunk_kb, num_kb - kb0);  // kb0 is a multiple of four: groups of factors lie within a chunk
            uint32_t sf = 0;
            for (int kb = 0; kb < blocks; ++kb) {
              if (!pair_wait(&bars->full[stage], phase, bars, peer, 4u)) { ok = false; break; }
              tc_fence_after();
              if ((kb & 3) == 0) {
                const uint32_t f = smem_u32(factors + stage * XSF_BYTES);
                sf = tmem_base + XSF_COL + set * XSF_SET;
                tc_copy_factors_pair(sf, f);
                tc_copy_factors_pair(sf + 4, f + XSF_A);
                tc_copy_factors_pair(sf + 8, f + XSF_A + 512);
                if (++set == XSF_SETS) set = 0;
              }
              const uint32_t a_addr = smem_u32(tiles + stage * XSTAGE_BYTES);
              const uint32_t id = idesc | ((uint32_t)(kb & 3) << 4) | ((uint32_t)(kb & 3) << 29);
              const uint64_t da = a_mn ? make_smem_desc_mn(a_addr, PA_BYTES) : make_smem_desc(a_addr);
              const uint64_t db = b_mn ? make_smem_desc_mn(a_addr + PA_BYTES, PB_BYTES) : make_smem_desc(a_addr + PA_BYTES);
#pragma unroll
              for (int kk = 0; kk < BK / UMMA_K; ++kk)
                tc_mma_mx_pair(tmem_d, da + (uint64_t)kk * step_a, db + (uint64_t)kk * step_b, id, sf, sf + 4,
                               (kb | kk) != 0 ? 1u : 0u);
              tc_commit_pair(&bars->empty[stage]);
              if (++stage == XSTAGES) { stage = 0; phase ^= 1u; }
            }
            if (ok) tc_commit_pair(&bars->tmem_full[acc]);
          }
          if (!ok) break;
          if (sched != nullptr) {
            const int32_t v = pair_ring_read(bars, local, peer, 16u, 0u);
            if (v == -2) { ok = false; break; }
            t = v < 0 ? num_tiles : (int64_t)v;
          } else {
            t += num_clusters;
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(XREGS_MANY));
    // ---------------- epilogue (warps 4..11 of both CTAs) ----------------
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const EpilogueArgs<OutT> ea{bias, out, ldo, m, n, out_vec_ok, use_tma_store, &tma_out,
                                staging + (warp - 4) * EPI_BOX_BYTES, 1.0f, 1, nullptr};
    const uint32_t free_in_leader = mapa_u32(smem_u32(&bars->tmem_shared_free), 0u);
    // The shared columns are the last 64 of accumulator 0, read by half 1, and the first of accumulator 1, read by half 0:
    // half 1 takes its two pieces of 64 columns in the other order.
    const int piece[2] = {half * 64, 64 - half * 64};
    uint32_t boxes = 0, local = 0, chunk = 0;
    int64_t t = cluster_id;
    for (; t < num_tiles; ++local) {
      const TileCoord tc = tile_coord(t, tiles_m, tiles_n, raster);
      float sum[128];
      int got = 1;
      for (int kb = 0; kb < num_kb; kb += chunk_kb, ++chunk) {
        const uint32_t acc = chunk & 1u;
        if (lane == 0) got = pair_wait(&bars->tmem_full[acc], (chunk >> 1) & 1u, bars, peer, 8u, WAIT_BY_HINT | 1000u) ? 1 : 0;
        got = __shfl_sync(0xFFFFFFFFu, got, 0);
        if (got == 0) break;
        tc_fence_after();
        const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * (uint32_t)XACC_STEP + (uint32_t)(half * 128);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          uint32_t r[2][32];
          tc_ld_32x32b_x32(taddr + (uint32_t)piece[p], r[0]);
          tc_ld_32x32b_x32(taddr + (uint32_t)(piece[p] + 32), r[1]);
          tc_wait_ld();
          if (p == 0) {  // also says that this warp has read all of the previous chunk's accumulator
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(free_in_leader);
          }
          if (kb == 0) {
#pragma unroll
            for (int i = 0; i < 64; ++i) sum[p * 64 + i] = __uint_as_float(r[i >> 5][i & 31]);
          } else {
#pragma unroll
            for (int i = 0; i < 64; ++i) sum[p * 64 + i] += __uint_as_float(r[i >> 5][i & 31]);
          }
        }
      }
      if (got == 0) break;
      const int row0 = tc.m * PBM + (int)rank * 128 + quarter * 32;
#pragma unroll
      for (int p = 0; p < 2; ++p)
        store_columns<OutT>(ea, sum + p * 64, row0, tc.n * PBN + half * 128 + piece[p], boxes);
      if (sched != nullptr) {
        int v = 0;
        if (lane == 0) v = pair_ring_read(bars, local, peer, 32u, 64u);
        v = __shfl_sync(0xFFFFFFFFu, v, 0);
        t = v < 0 ? num_tiles : (int64_t)v;  // no more tiles, or gave up
      } else {
        t += num_clusters;
      }
    }
    if (use_tma_store && lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA leaves while the other may still touch its barriers or TMEM
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)TMEM_COLS)
                 : "memory");
  }
}

// ---- host side --------------------------------------------------------------------------------------
static bool strides_ok(const BlockScale& s) { return s.row_stride >= 0 && s.kb_stride >= 0; }

template <typename OutT, bool PER_COL>
static int launch_block_pair(const CUtensorMap& ma, const CUtensorMap& mb, const BlockScale& sa, const BlockScale& sb,
                             const void* bias, void* out, int64_t ldo, int m, int n, int k, uint32_t idesc, int vec_ok,
                             int layouts, cudaStream_t st) {
  static PerDeviceOnce setup;
  int max_clusters = 0;
  auto kernel = gemm_block_pair_kernel<OutT, PER_COL>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(BTHREADS);
  cfg.dynamicSmemBytes = BSMEM_BYTES;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t attr_err = setup.run(
      [&](int* clusters_out) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BSMEM_BYTES);
        cudaFuncAttributes fa;
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, kernel);
        // the registers that the first group hands over have to be there, or the others would wait for them
        if (e == cudaSuccess && fa.numRegs * BTHREADS < 128 * BREGS_FEW + 256 * BREGS_MANY) e = cudaErrorInvalidConfiguration;
        if (e == cudaSuccess) {
          cfg.gridDim = dim3(2 * (sm_count() / 2));
          e = cudaOccupancyMaxActiveClusters(clusters_out, kernel, &cfg);
        }
        return e;
      },
      &max_clusters);
  if (attr_err != cudaSuccess) return record_cuda_error(attr_err);
  if (max_clusters < 1) return F8B200_ERR_UNSUPPORTED;
  const int64_t tiles = (int64_t)((m + PBM - 1) / PBM) * ((n + PBN - 1) / PBN);
  int clusters = max_clusters;
  if (persistent_ctas() / 2 < clusters) clusters = persistent_ctas() / 2;
  if (tiles < clusters) clusters = (int)tiles;
  cfg.gridDim = dim3(2 * clusters);
  return record_cuda_error(cudaLaunchKernelEx(&cfg, kernel, ma, mb, sa, sb, static_cast<const OutT*>(bias),
                                              static_cast<OutT*>(out), ldo, m, n, k, idesc, vec_ok,
                                              choose_raster(m, n, k, PBM, PBN) | layouts));
}

// Exponent bytes of an operand (the layout of cast_block.cu's exponent_at) as a matrix of 32-bit words: one row per four
// k-blocks, box = `words` of one of them.
static int encode_exponent_map(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int words) {
  auto fn = get_encode_fn();
  if (fn == nullptr) return F8B200_ERR_DRIVER;
  const int64_t pitch_words = (rows + 255) / 256 * 256;
  const cuuint64_t gdim[2] = {(cuuint64_t)pitch_words, (cuuint64_t)((k + 511) / 512)};
  const cuuint64_t gstride[1] = {(cuuint64_t)(pitch_words * 4)};
  const cuuint32_t box[2] = {(cuuint32_t)words, 1u};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(base), gdim, gstride, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? F8B200_OK : F8B200_ERR_DRIVER;
}

template <typename OutT>
static int launch_block_scaled(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mea, const CUtensorMap& meb,
                               const CUtensorMap& mo, int use_tma, const void* bias, void* out, int64_t ldo, int m, int n,
                               int k, uint32_t idesc, int vec_ok, int layouts, uint32_t* sched, cudaStream_t st) {
  static PerDeviceOnce setup;
  int max_clusters = 0;
  auto kernel = gemm_block_scaled_kernel<OutT>;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(XTHREADS);
  cfg.dynamicSmemBytes = XSMEM_BYTES;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t attr_err = setup.run(
      [&](int* clusters_out) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, XSMEM_BYTES);
        cudaFuncAttributes fa;
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, kernel);
        // as in launch_block_pair: the registers that the first group hands over have to be there
        if (e == cudaSuccess && fa.numRegs * XTHREADS < 128 * XREGS_FEW + 256 * XREGS_MANY) e = cudaErrorInvalidConfiguration;
        if (e == cudaSuccess) {
          cfg.gridDim = dim3(2 * (sm_count() / 2));
          e = cudaOccupancyMaxActiveClusters(clusters_out, kernel, &cfg);
        }
        return e;
      },
      &max_clusters);
  if (attr_err != cudaSuccess) return record_cuda_error(attr_err);
  if (max_clusters < 1) return F8B200_ERR_UNSUPPORTED;
  const int64_t tiles = (int64_t)((m + PBM - 1) / PBM) * ((n + PBN - 1) / PBN);
  int clusters = max_clusters;
  if (persistent_ctas() / 2 < clusters) clusters = persistent_ctas() / 2;
  if (tiles < clusters) clusters = (int)tiles;
  cfg.gridDim = dim3(2 * clusters);
  sched = usable_sched(sched, tiles, clusters);
  if (sched != nullptr) {
    const cudaError_t e = cudaMemsetAsync(sched, 0, sizeof(uint32_t), st);
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  const int num_kb = (k + BK - 1) / BK, most = sizeof(OutT) == 4 ? XCHUNK_32 : XCHUNK_16;
  const int chunks = (num_kb + most - 1) / most, chunk_kb = ((num_kb + chunks - 1) / chunks + 3) / 4 * 4;  // <= most
  return record_cuda_error(cudaLaunchKernelEx(&cfg, kernel, ma, mb, mea, meb, mo, static_cast<const OutT*>(bias),
                                              static_cast<OutT*>(out), ldo, m, n, k, idesc, vec_ok, use_tma,
                                              choose_raster(m, n, k, PBM, PBN) | layouts, chunk_kb, sched));
}

template <typename OutT, int T>
static int launch_block_few(const CUtensorMap& mw, const CUtensorMap& mx, const BlockScale& sw, const BlockScale& sx,
                            const void* bias, void* out, int64_t ldo, int m, int n, int k, uint32_t idesc, int w_mn,
                            int vec_ok, int split, cudaStream_t st) {
  static PerDeviceOnce setup;
  auto kernel = gemm_block_few_kernel<OutT, T>;
  const cudaError_t attr_err = setup.run([&](int*) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, few_smem_bytes<T>());
  });
  if (attr_err != cudaSuccess) return record_cuda_error(attr_err);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(FewCfg<T>::kThreads);
  cfg.dynamicSmemBytes = few_smem_bytes<T>();
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  cfg.gridDim = dim3(split, (n + 127) / 128, (m + T - 1) / T);
  return record_cuda_error(cudaLaunchKernelEx(&cfg, kernel, mw, mx, sw, sx, static_cast<const OutT*>(bias),
                                              static_cast<OutT*>(out), ldo, m, n, k, idesc, w_mn, vec_ok));
}

// instruction descriptor of one CTA: 128 rows of B's side, `cols` rows of A's side
static uint32_t make_idesc_few(int w_kind, int x_kind, int w_mn, int cols) {
  return (1u << 4) | ((uint32_t)w_kind << 7) | ((uint32_t)x_kind << 10) | ((uint32_t)w_mn << 15) |
         ((uint32_t)(cols >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// CTAs of one cluster that split K: as many as the GPU holds at once and leave each at least four k-blocks, in powers of
// two up to 8.  Measured (us, single calls in a graph with cold caches, split 1 / 2 / 4 / 8): 8 x 8192 x 8192 35 / 27 / 25 / 29,
// 16 x 2048 x 8192 35 / 23 / 16 / 16, 64 x 8192 x 28672 121 / 72 / 61 / 68, 128 x 4096 x 4096 33 / 25 / 21 / 35, 128 x 8192 x
// 8192 55 / 37 / 43 / 68, 37 x 28672 x 8192 61 / 68 / 76 / 88.
static int few_split(int64_t tiles, int num_kb, int ctas_per_sm) {
  int split = 1;
  while (split < FEW_MAX_SPLIT && tiles * split * 2 <= (int64_t)ctas_per_sm * sm_count() && num_kb >= split * 2 * 4) split *= 2;
  return split;
}

}  // namespace block
}  // namespace gemm
}  // namespace f8b200

extern "C" int f8b200_gemm_blockwise(const void* a, int a_kind, int a_layout, int64_t lda, const float* scale_a,
                                     int64_t sa_row_stride, int64_t sa_kb_stride, int a_block_rows,
                                     const void* exp_a, const void* b,
                                     int b_kind, int b_layout, int64_t ldb, const float* scale_b, int64_t sb_row_stride,
                                     int64_t sb_kb_stride, int b_block_rows, const void* exp_b, const void* bias,
                                     int out_dtype, void* out, int64_t ldo, int64_t m, int64_t n, int64_t k,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace gemm::block;
  if ((a_block_rows != 1 && a_block_rows != 128) || (b_block_rows != 1 && b_block_rows != 128)) return F8B200_ERR_BAD_ARG;
  const BlockScale sa{scale_a, sa_row_stride, sa_kb_stride, a_block_rows == 128 ? 7 : 0};
  const BlockScale sb{scale_b, sb_row_stride, sb_kb_stride, b_block_rows == 128 ? 7 : 0};
  if (!strides_ok(sa) || !strides_ok(sb)) return F8B200_ERR_BAD_ARG;
  if (workspace != nullptr && workspace_bytes < F8B200_GEMM_WORKSPACE_BYTES) return F8B200_ERR_BAD_ARG;
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return F8B200_ERR_ALIGNMENT;
  if (reinterpret_cast<uintptr_t>(scale_a) % 4 != 0 || reinterpret_cast<uintptr_t>(scale_b) % 4 != 0) return F8B200_ERR_ALIGNMENT;
  bool empty = false;
  int rc = gemm_fp8_validate(a, a_kind, a_layout, lda, b, b_kind, b_layout, ldb, scale_a, scale_b, bias, out_dtype, out,
                             ldo, m, n, k, &empty);
  if (rc != F8B200_OK || empty) return rc;
  const int osz = out_dtype == F8B200_FP32 ? 4 : 2;
  const int vec_ok = (reinterpret_cast<uintptr_t>(out) % 16 == 0) && ((ldo * osz) % 16 == 0);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int layouts = (a_layout << gemm::LAYOUT_A_MN_BIT) | (b_layout << gemm::LAYOUT_B_MN_BIT);
  CUtensorMap ma, mb;
  // a box of an MN-major operand is 128 rows wide, so the few-rows kernel takes A K-major only
  if (m <= 128 && a_layout == F8B200_K_MAJOR) {
    const int t = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
    rc = gemm::encode_operand_map(&ma, a, m, k, lda, t);
    if (rc == F8B200_OK)
      rc = b_layout ? gemm::encode_operand_map_mn(&mb, b, n, k, ldb) : gemm::encode_operand_map(&mb, b, n, k, ldb, 128);
    if (rc != F8B200_OK) return rc;
    const uint32_t idesc = make_idesc_few(b_kind, a_kind, b_layout, t);
    const int split = few_split((n + 127) / 128, (int)((k + 127) / 128), t <= 64 ? FewCfg<64>::kCtas : FewCfg<128>::kCtas);
    return dispatch_out_dtype(out_dtype, [&](auto* tag) {
      using OutT = std::remove_pointer_t<decltype(tag)>;
      auto go = [&](auto t_const) {
        return launch_block_few<OutT, decltype(t_const)::value>(mb, ma, sb, sa, bias, out, ldo, (int)m, (int)n, (int)k,
                                                                idesc, b_layout, vec_ok, split, st);
      };
      if (t == 16) return go(std::integral_constant<int, 16>{});
      if (t == 32) return go(std::integral_constant<int, 32>{});
      if (t == 64) return go(std::integral_constant<int, 64>{});
      return go(std::integral_constant<int, 128>{});
    });
  }
  rc = a_layout ? gemm::encode_operand_map_mn(&ma, a, m, k, lda) : gemm::encode_operand_map(&ma, a, m, k, lda, 128);
  if (rc == F8B200_OK)
    rc = b_layout ? gemm::encode_operand_map_mn(&mb, b, n, k, ldb) : gemm::encode_operand_map(&mb, b, n, k, ldb, 128);
  if (rc != F8B200_OK) return rc;
  if (exp_a != nullptr && exp_b != nullptr) {  // both sides' factors are powers of two
    if (reinterpret_cast<uintptr_t>(exp_a) % 16 != 0 || reinterpret_cast<uintptr_t>(exp_b) % 16 != 0) return F8B200_ERR_ALIGNMENT;
    CUtensorMap mea, meb, mo;
    rc = encode_exponent_map(&mea, exp_a, m, k, 128);
    if (rc == F8B200_OK) rc = encode_exponent_map(&meb, exp_b, n, k, 256);
    memset(&mo, 0, sizeof(mo));
    if (rc == F8B200_OK && vec_ok) rc = gemm::encode_output_map(&mo, out, m, n, ldo, out_dtype);
    if (rc != F8B200_OK) return rc;
    return dispatch_out_dtype(out_dtype, [&](auto* tag) {
      using OutT = std::remove_pointer_t<decltype(tag)>;
      return launch_block_scaled<OutT>(ma, mb, mea, meb, mo, vec_ok, bias, out, ldo, (int)m, (int)n, (int)k,
                                       make_idesc_scaled(a_kind, b_kind, a_layout, b_layout), vec_ok, layouts,
                                       static_cast<uint32_t*>(workspace), st);
    });
  }
  const uint32_t idesc = gemm::pair::make_idesc_pair(a_kind, b_kind, a_layout, b_layout);
  return dispatch_out_dtype(out_dtype, [&](auto* tag) {
    using OutT = std::remove_pointer_t<decltype(tag)>;
    return b_block_rows == 1
               ? launch_block_pair<OutT, true>(ma, mb, sa, sb, bias, out, ldo, (int)m, (int)n, (int)k, idesc, vec_ok,
                                               layouts, st)
               : launch_block_pair<OutT, false>(ma, mb, sa, sb, bias, out, ldo, (int)m, (int)n, (int)k, idesc, vec_ok,
                                                layouts, st);
  });
}
