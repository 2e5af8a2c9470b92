// tcgen05 products of the output layer whose [T, V] result is consumed on
// the spot: the logits x W^T reduced to a log-sum-exp per row (kLse), the
// logits turned into their softmax gradient (kSoftmaxGrad), and the two
// products with that gradient (kRowsF32: rows of dx, kWeightGrad: dW).
//
// The main loop is that of gemm_pair.cuh without its stream-K tail: CTA
// pairs (cta_group::2), 256 x 256 tiles, 128B-swizzled TMA loads into a
// 6-stage ring, one elected thread issuing the MMAs, fp32 accumulators
// double-buffered in TMEM, 4 epilogue warps per CTA that work on one
// accumulator while the other fills.  The rows are those that the packing
// kernel of logprob.cu kept, so their number is read on the GPU.  Units of
// work are (k range, tile): `splits` > 1 cuts the reduction into ranges whose
// results are separate fp32 planes (kRowsF32 only), so that few tiles still
// fill the GPU and the planes are added in a fixed order afterwards.
#pragma once

#include "gemm_core.cuh"

namespace t1 {
namespace vocab {

using namespace gemm;

constexpr int TILE = 256;   // rows and columns of a pair's tile
constexpr int HALF = 128;   // a CTA's rows of A and of B
constexpr int VSTAGES = 6;
constexpr int V_A_BYTES = HALF * BK * 2;
constexpr int V_STAGE_BYTES = 2 * V_A_BYTES;
constexpr int EPI_BUF = 32 * 128;                // 32 rows x 128 bytes, 128B-swizzled
constexpr int EPI_BYTES = 4 /*warps*/ * 2 * EPI_BUF;
constexpr int V_SMEM_BYTES = VSTAGES * V_STAGE_BYTES + EPI_BYTES + 1024 /*align*/ + 256 /*barriers*/;
static_assert(V_SMEM_BYTES <= 232448, "exceeds 227 KB of shared memory");

enum Mode : int { kLse = 0, kSoftmaxGrad = 1, kRowsF32 = 2, kWeightGrad = 3 };

// What the packing of the batch's rows found out on the GPU.
struct RowsMeta {
  int rows;    // rows that take part
  int splits;  // ranges of k that the rows' product (kRowsF32) is cut into
};

struct VocabParams {
  const RowsMeta* meta;  // its rows are M, or in kWeightGrad the reduction's length
  int M, N;              // rows and columns of the product (M: kWeightGrad only)
  int k_blocks;          // of BK = 64 (not in kWeightGrad)
  int ld_part;           // kLse: rows of a column block in `part`
  int accumulate;        // kRowsF32: add to what the plane holds
  float scale;           // 1 / temperature
  int col0;              // vocabulary index of column 0
  const int* targets;    // [M] vocabulary index
  float2* part;          // kLse: [tiles_n][ld_part] (largest logit, sum of exp(logit - largest)) of a column block
  float* target_logit;   // kLse: [M], unscaled
  const float* lse;      // kSoftmaxGrad: [M]
  int* err;
};

// The product's extents, known once the packing has run.
struct Extents {
  int M, tiles_m, tiles_n, k_blocks, splits;
};

template <int MODE>
__device__ __forceinline__ Extents extents(const VocabParams& p) {
  const int rows = p.meta->rows;
  Extents e;
  e.M = MODE == kWeightGrad ? p.M : rows;
  e.tiles_m = (e.M + TILE - 1) / TILE;
  e.tiles_n = (p.N + TILE - 1) / TILE;
  e.k_blocks = MODE == kWeightGrad ? (rows + BK - 1) / BK : p.k_blocks;
  e.splits = MODE == kRowsF32 ? p.meta->splits : 1;
  return e;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ void vocab_unit(const Extents& e, int u, int& mb, int& nb, int& kb0, int& kb1,
                                           int& split) {
  const int tiles = e.tiles_m * e.tiles_n;
  split = u / tiles;
  raster(u % tiles, e.tiles_m, e.tiles_n, mb, nb);
  kb0 = static_cast<int>(static_cast<long>(split) * e.k_blocks / e.splits);
  kb1 = static_cast<int>(static_cast<long>(split + 1) * e.k_blocks / e.splits);
}

template <bool A_MN, bool B_MN, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(192, 1)
    vocab_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                 const __grid_constant__ CUtensorMap tma_c, const VocabParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sA = smem;
  uint8_t* sB = sA + VSTAGES * V_A_BYTES;
  uint8_t* sE = sB + VSTAGES * V_A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(sE + EPI_BYTES);
  uint64_t* empty = full + VSTAGES;
  uint64_t* tfull = empty + VSTAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();  // 0 = leader
  const int cluster = blockIdx.x >> 1;
  const int nclusters = gridDim.x >> 1;
  const ErrorSlot err{p.err};

  if (threadIdx.x == 0) {
    for (int s = 0; s < VSTAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 8);  // 4 epilogue warps x 2 CTAs
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tma_a);
    prefetch_tensormap(&tma_b);
    if (MODE != kLse) prefetch_tensormap(&tma_c);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, TMEM_COLS);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // barriers of both CTAs initialised, TMEM allocated
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const Extents e = extents<MODE>(p);
  const int num_units = e.tiles_m * e.tiles_n * e.splits;

  if (warp == 0) {
    // ------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int u = cluster; u < num_units && !*abort_flag; u += nclusters) {
        int mb, nb, kb0, kb1, split;
        vocab_unit(e, u, mb, nb, kb0, kb1, split);
        const int row_a = mb * TILE + static_cast<int>(crank) * HALF;
        const int row_b = nb * TILE + static_cast<int>(crank) * HALF;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1)) {
            err.set(121);
            *abort_flag = 1;
            break;
          }
          const uint32_t lfull = mapa_shared(smem_u32(&full[stage]), 0);
          if (crank == 0) mbar_arrive_expect_tx(&full[stage], 2 * V_STAGE_BYTES);
          uint8_t* a = sA + stage * V_A_BYTES;
          uint8_t* b = sB + stage * V_A_BYTES;
          const int k0 = kb * BK;
          if (!A_MN) {
            tma_load_2d_pair(a, &tma_a, lfull, k0, row_a);
          } else {
            tma_load_2d_pair(a, &tma_a, lfull, row_a, k0);
            tma_load_2d_pair(a + 8192, &tma_a, lfull, row_a + 64, k0);
          }
          if (!B_MN) {
            tma_load_2d_pair(b, &tma_b, lfull, k0, row_b);
          } else {
            tma_load_2d_pair(b, &tma_b, lfull, row_b, k0);
            tma_load_2d_pair(b + 8192, &tma_b, lfull, row_b + 64, k0);
          }
          if (++stage == VSTAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------- MMA issuer (leader only)
    if (lane == 0 && crank == 0) {
      constexpr uint32_t IDESC = idesc_bf16_f32(TILE, TILE, A_MN, B_MN);
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      for (int u = cluster; u < num_units && !*abort_flag; u += nclusters, ++local) {
        int mb, nb, kb0, kb1, split;
        vocab_unit(e, u, mb, nb, kb0, kb1, split);
        const int acc = local & 1;
        const uint32_t acc_phase = (local >> 1) & 1;
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1)) {
          err.set(122);
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * TILE;
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full[stage], phase)) {
            err.set(123);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(sA + stage * V_A_BYTES);
          const uint32_t b_addr = smem_u32(sB + stage * V_A_BYTES);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t ad = A_MN ? smem_desc_sw128(a_addr + k * 2048, 8192, 1024)
                                     : smem_desc_sw128(a_addr + k * 32, 16, 1024);
            const uint64_t bd = B_MN ? smem_desc_sw128(b_addr + k * 2048, 8192, 1024)
                                     : smem_desc_sw128(b_addr + k * 32, 16, 1024);
            mma_bf16_pair(d_tmem, ad, bd, IDESC, (kb != kb0 || k != 0) ? 1u : 0u);
          }
          mma_commit_pair(&empty[stage], 0x3);
          if (++stage == VSTAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit_pair(&tfull[acc], 0x3);
      }
    }
  } else {
    // ---------------------------------------------------------- epilogue
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    uint8_t* wbuf = sE + q * 2 * EPI_BUF;
    const uint32_t leader_tempty0 = mapa_shared(smem_u32(&tempty[0]), 0);
    const uint32_t leader_tempty1 = mapa_shared(smem_u32(&tempty[1]), 0);
    int bi = 0;
    int local = 0;
    for (int u = cluster; u < num_units; u += nclusters, ++local) {
      int mb, nb, kb0, kb1, split;
      vocab_unit(e, u, mb, nb, kb0, kb1, split);
      const int acc = local & 1;
      const uint32_t acc_phase = (local >> 1) & 1;
      // one lane waits and the warp follows it, so the warp never diverges
      // around the .sync.aligned TMEM loads below
      int ok = 0;
      if (lane == 0) {
        ok = !*abort_flag;
        if (ok && !mbar_wait(&tfull[acc], acc_phase)) {
          err.set(124);
          *abort_flag = 1;
          ok = 0;
        }
      }
      if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      tc_fence_after();
      const int row0 = mb * TILE + static_cast<int>(crank) * HALF + q * 32;
      const int row = row0 + lane;
      const bool row_ok = row < e.M;
      const int tcol0 = nb * TILE;                       // first column of the tile
      const int cols = min(TILE, p.N - tcol0);           // columns of the tile that exist
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * TILE;

      if (MODE == kLse) {
        // A running (largest, sum) over the tile's columns, kept in the
        // accumulator's own units: (logit - largest) is exact near the
        // largest, which is where the sum comes from.
        const float k2 = p.scale * kLog2e;
        const int t = row_ok ? p.targets[row] - tcol0 : -1;
        const int tcol = t < cols ? t : -1;
        float m = -INFINITY, s = 0.f;
#pragma unroll 1
        for (int c = 0; c < TILE; c += 32) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(taddr + c, r);
          tmem_ld_wait();
          if (c + 32 > cols) {  // columns past the vocabulary
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j >= cols) r[j] = __float_as_uint(-INFINITY);
          }
          float mx = __uint_as_float(r[0]);
#pragma unroll
          for (int j = 1; j < 32; ++j) mx = fmaxf(mx, __uint_as_float(r[j]));
          const float mn = fmaxf(m, mx);
          const float ref = mn == -INFINITY ? 0.f : mn;
          s *= ex2((m - ref) * k2);
#pragma unroll
          for (int j = 0; j < 32; ++j) s += ex2((__uint_as_float(r[j]) - ref) * k2);
          m = mn;
          if (tcol >= c && tcol < c + 32) {
            if (!T1_OOB(row, p.ld_part)) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (tcol - c == j) p.target_logit[row] = __uint_as_float(r[j]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc ? leader_tempty1 : leader_tempty0);
        if (row_ok && !T1_OOB(row, p.ld_part)) p.part[static_cast<size_t>(nb) * p.ld_part + row] = make_float2(m, s);
        continue;
      }

      if (MODE == kRowsF32) {
        // fp32 rows through 32 x 32 slabs (128-byte rows)
#pragma unroll 1
        for (int c = 0; c < TILE; c += 32) {
          uint8_t* buf = wbuf + bi * EPI_BUF;
          const bool live = c < cols && row0 < e.M;  // uniform over the warp
          if (lane == 0) bulk_wait_group_read<1>();
          __syncwarp();
          uint32_t r[32];
          tmem_ld_32x32b_x32(taddr + c, r);
          tmem_ld_wait();
          if (c + 32 == TILE) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc ? leader_tempty1 : leader_tempty0);
          }
          if (!live) continue;
          if (kb0 == kb1) {  // a range of no columns
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = 0;
          }
          uint8_t* rowp = buf + lane * 128;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            *reinterpret_cast<uint4*>(rowp + ((j ^ (lane & 7)) << 4)) =
                make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            const int prow = split * e.tiles_m * TILE + row0;
            if (p.accumulate) tma_reduce_add_2d(&tma_c, buf, tcol0 + c, prow);
            else tma_store_2d(&tma_c, buf, tcol0 + c, prow);
            bulk_commit_group();
          }
          bi ^= 1;
        }
        continue;
      }

      // bf16 results (kSoftmaxGrad, kWeightGrad) through 32 x 64 slabs
      float lse2 = 0.f;
      int tcol = -1;
      const float k2 = p.scale * kLog2e;
      if (MODE == kSoftmaxGrad && row_ok) {
        lse2 = p.lse[row] * kLog2e;
        const int t = p.targets[row] - p.col0 - tcol0;
        tcol = t < cols ? t : -1;
      }
      // u's rows are a reduction's length in kWeightGrad: its last block of
      // BK has to be there, with zeros past the last row
      const int m_end = MODE == kSoftmaxGrad ? (e.M + BK - 1) / BK * BK : e.M;
#pragma unroll 1
      for (int c = 0; c < TILE; c += 64) {
        uint8_t* buf = wbuf + bi * EPI_BUF;
        const bool live = c < cols && row0 < m_end;
        if (lane == 0) bulk_wait_group_read<1>();
        __syncwarp();
        uint32_t r[2][32];
        tmem_ld_32x32b_x32(taddr + c, r[0]);
        tmem_ld_32x32b_x32(taddr + c + 32, r[1]);
        tmem_ld_wait();
        if (c + 64 == TILE) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(acc ? leader_tempty1 : leader_tempty0);
        }
        if (!live) continue;
        uint8_t* rowp = buf + lane * 128;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            f[k] = __uint_as_float(r[j >> 2][(j & 3) * 8 + k]);
            if (MODE == kSoftmaxGrad) {
              f[k] = row_ok ? -ex2(fmaf(f[k], k2, -lse2)) : 0.f;
              if (tcol == c + 8 * j + k) f[k] += 1.f;
            } else if (kb0 == kb1) {  // a sum over no rows
              f[k] = 0.f;
            }
          }
          uint4 ov;
          __nv_bfloat162* oh = reinterpret_cast<__nv_bfloat162*>(&ov);
#pragma unroll
          for (int k = 0; k < 4; ++k) oh[k] = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
          *reinterpret_cast<uint4*>(rowp + ((j ^ (lane & 7)) << 4)) = ov;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tma_c, buf, tcol0 + c, row0);
          bulk_commit_group();
        }
        bi ^= 1;
      }
    }
    // every store of this warp completed before the CTA may exit
    if (lane == 0) bulk_wait_group_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncwarp();
  cluster_sync();  // neither CTA leaves while the pair still uses its smem / TMEM
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

}  // namespace vocab
}  // namespace t1
