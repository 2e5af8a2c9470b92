// tcgen05 products of the output layer whose [T, V] result is consumed on
// the spot.  One kernel, three jobs:
//   kLse          logits x W^T, reduced to (largest, sum of exponentials) per
//                 row and 128-column block, and the target's logit;
//   kSoftmaxGrad  the same logits turned into u = g (onehot - softmax), bf16;
//   kGrads        both products with u in one launch: the rows of dx = u W, and
//                 dW = u^T x.
//
// The main loop is that of gemm_pair.cuh: CTA pairs (cta_group::2), 256 x 256
// tiles, 128B-swizzled TMA loads into a 6-stage ring, one elected thread
// issuing the MMAs, fp32 accumulators double-buffered in TMEM, 8 epilogue warps
// per CTA that work on one accumulator while the other fills (with 4, one per
// SM partition, each waited for its own latencies: a u tile took 8 K cycles,
// more than the 8 K of a mainloop at H = 1024).  The
// rows may be those that the packing kernel of logprob.cu kept, so their
// number is read on the GPU.
//
// What bounds it (B200): with H = 4096 and many rows the tensor cores under the
// power limit, at the speed of a library product of the same shape (log-sum-
// exp of 5888 rows at V = 128256: 4.7 ms, 1320 TFLOP/s); with one or two row
// tiles the operands, 64 bytes a cycle and SM at the tensor peak, of which
// 192 KB in flight cover 1.6 us of latency (tensor pipe 55-60 % active); below
// H = 512 the epilogue's exponentials.
//
// Work of a cluster: kLse and kSoftmaxGrad take tiles in turn.  kGrads has
// units of two lengths, dx tiles (over a range of the vocabulary) and dW
// tiles (over the rows); the long ones are dealt out first and the clusters
// that got one less take short ones meanwhile (grad_unit).
#pragma once

#include "arrivals.cuh"
#include "gemm_core.cuh"

namespace t1 {
namespace vocab {

using namespace gemm;

constexpr int TILE = 256;   // rows and columns of a pair's tile
constexpr int HALF = 128;   // a CTA's rows of A and of B
constexpr int VSTAGES = 6;
constexpr int V_A_BYTES = HALF * BK * 2;
constexpr int V_STAGE_BYTES = 2 * V_A_BYTES;
constexpr int EPI_WARPS = 8;                     // two per SM partition; a warp has 32 rows x 128 columns
constexpr int EPI_BUF = 32 * 128;                // 32 rows x 128 bytes, 128B-swizzled, one per warp
constexpr int EPI_BYTES = EPI_WARPS * EPI_BUF;
constexpr int V_THREADS = 64 + 32 * EPI_WARPS;
constexpr int V_SMEM_BYTES = VSTAGES * V_STAGE_BYTES + EPI_BYTES + 1024 /*align*/ + 256 /*barriers*/;
static_assert(V_SMEM_BYTES <= 232448, "exceeds 227 KB of shared memory");

enum Job : int { kLse = 0, kSoftmaxGrad = 1, kGrads = 2 };

// What the packing of the batch's rows found out on the GPU.
struct RowsMeta {
  int rows;    // rows that take part
  int splits;  // ranges of the vocabulary that dx's product is cut into
};

// Row distances and offsets of one 32-row x 256-column block of fp32 sums:
// [column / 4][row][4], so that a warp (a lane per row) moves 512
// consecutive bytes at a time.
constexpr int PLANE_BLOCK = 32 * TILE;

struct VocabParams {
  const RowsMeta* meta;    // null: `rows` and `splits` as given here
  int rows, splits;
  int N;                   // vocabulary columns of this launch
  int H;
  float scale;             // 1 / temperature
  int col0;                // vocabulary index of column 0
  const int* index;        // [rows] token of a packed row; null: the row itself
  int tokens;              // T
  const int64_t* targets;  // [rows] vocabulary index
  Arrivals tickets;        // kLse with join: arrivals per 32 rows
  int tickets_n;
  // kLse
  int64_t ignore, V;
  int ld_part;
  float2* part;            // [block of 128 columns][ld_part]
  float* target_logit;     // [rows], unscaled
  int join;                // the last block of a row group joins its rows
  float *logp, *lse_out;   // with join
  // kSoftmaxGrad
  const float* lse;        // [rows]
  const float* g;          // [rows] dlogp / tau
  // kGrads
  bf16* dx;                // [T, H]
  float* planes;           // [tile][split][8] blocks of PLANE_BLOCK
  int64_t plane_blocks;    // allocated
  int first, last;         // first / last piece of the vocabulary
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLog2e = 1.4426950408889634f;

// Programmatic launch: the next kernel of the stream may start its prologue,
// and this one touches nothing of the previous kernel's before it has ended.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// The tensor cores drop what falls below the accumulator's last bit at every
// step, which adds up: over 4096 products the logits lose 2e-6 of their size.
// The logits are therefore summed from accumulators of about 16 k blocks each
// (equal parts of k, 1472 products at most), added up in registers, rounded.
// Errors of logp (rms, of the row's largest logit; fp32 library arithmetic in
// brackets): 3.6e-7 (4.2e-7) at H = 4096, for 4 % more time; 3.8e-7 (1.6e-7) at
// 1024; 4.9e-7 (2.0e-7) at 1472, the longest accumulator.  At most 16 blocks
// would give 2.5e-7 there for 1-4 % of the time of H between 1025 and 1472 (839
// rows, H = 1032, V = 50021: 106 us against 102).  kSoftmaxGrad sums them in the same
// order as kLse: where a target is nearly sure, u is what exp(logit - lse)
// leaves of 1, and an error of the logit that lse does not share is all of u
// (one accumulator there put dx rows of targets with p = 0.999 off by a half).
constexpr int kLogitBlocks = 16;

// Running (largest m, sum s of exp((v - m) / tau)); k2 = log2(e) / tau.
__device__ __forceinline__ void lse_join(float& m, float& s, float m2, float s2, float k2) {
  const float mn = fmaxf(m, m2);
  const float ref = mn == -INFINITY ? 0.f : mn;
  s = s * ex2((m - ref) * k2) + s2 * ex2((m2 - ref) * k2);
  m = mn;
}

// log-probability and log-sum-exp of a row.  (target - largest) first: exact
// where the target is likely.
__device__ __forceinline__ void write_logp(const float m, const float s, const float target, const bool valid,
                                           const float scale, float* logp, float* lse) {
  const float ref = m == -INFINITY ? 0.f : m;
  const float log_s = logf(s);
  *logp = valid ? (target - ref) * scale - log_s : 0.f;
  *lse = valid ? ref * scale + log_s : 0.f;
}

// ---------------------------------------------------------- units of work
// Time of a unit in k blocks of 64 (0.27 us of tensor time for a pair): a dx
// tile pays about 12 for its start and drain; a dW tile cannot be faster than
// its 128 KB leave (about 6).
__host__ __device__ inline int dx_unit_cost(int k_blocks, int splits) { return k_blocks / splits + 12; }
__host__ __device__ inline int dw_unit_cost(int tiles_t) {
  const int k = tiles_t * (TILE / BK);
  return k > 6 ? k : 6;
}

struct Shape {
  int rows, tiles_t, tiles_n, tiles_h, k_h, k_n, k_rows, splits;
  int k_acc;  // k blocks of a logit's accumulator
};

__device__ __forceinline__ Shape shape_of(const VocabParams& p, bool splits) {
  Shape e;
  e.rows = p.meta != nullptr ? p.meta->rows : p.rows;
  e.splits = !splits ? 1 : p.meta != nullptr ? p.meta->splits : p.splits;
  e.tiles_t = (e.rows + TILE - 1) / TILE;
  e.tiles_n = (p.N + TILE - 1) / TILE;
  e.tiles_h = (p.H + TILE - 1) / TILE;
  e.k_h = (p.H + BK - 1) / BK;
  e.k_n = (p.N + BK - 1) / BK;
  e.k_rows = (e.rows + BK - 1) / BK;
  const int accs = max(1, (e.k_h + kLogitBlocks / 2) / kLogitBlocks);
  e.k_acc = (e.k_h + accs - 1) / accs;
  return e;
}

struct Unit {
  int mb, nb, kb0, kb1;
  int split;  // kGrads: range of the vocabulary, or -1 for a dW tile
};

// The i-th unit of cluster c out of C; false when there is none.
template <int JOB>
__device__ __forceinline__ bool get_unit(const Shape& e, int i, int c, int C, Unit& u) {
  if (JOB != kGrads) {
    const int64_t t = c + static_cast<int64_t>(i) * C;
    if (t >= static_cast<int64_t>(e.tiles_t) * e.tiles_n) return false;
    raster(static_cast<int>(t), e.tiles_t, e.tiles_n, u.mb, u.nb);
    u.kb0 = 0;
    u.kb1 = e.k_h;
    u.split = 0;
    return true;
  }
  const int tiles = e.tiles_t * e.tiles_h, X = tiles * e.splits, D = e.tiles_n * e.tiles_h;
  const int q = X / C, r = X % C;
  const int mine = q + (c < r);
  if (i < mine) {
    const int x = c + i * C;
    u.split = x / tiles;
    raster(x % tiles, e.tiles_t, e.tiles_h, u.mb, u.nb);
    u.kb0 = static_cast<int>(static_cast<int64_t>(u.split) * e.k_n / e.splits);
    u.kb1 = static_cast<int>(static_cast<int64_t>(u.split + 1) * e.k_n / e.splits);
    return true;
  }
  int j = i - mine;
  // dW tiles that clusters r.. take while the first r work on one more dx tile
  const int uw = dw_unit_cost(e.tiles_t);
  const int rounds = r == 0 ? 0 : (dx_unit_cost(e.k_n, e.splits) + uw / 2) / uw;
  const int early = static_cast<int>(min(static_cast<int64_t>(D), static_cast<int64_t>(rounds) * (C - r)));
  const int before = c < r || early <= c - r ? 0 : (early - (c - r) + (C - r) - 1) / (C - r);
  int64_t d;
  if (j < before) d = static_cast<int64_t>(j) * (C - r) + (c - r);
  else d = early + static_cast<int64_t>(j - before) * C + c;
  if (d >= D) return false;
  raster(static_cast<int>(d), e.tiles_n, e.tiles_h, u.mb, u.nb);
  u.kb0 = 0;
  u.kb1 = e.k_rows;
  u.split = -1;
  return true;
}

// Operands: kLse, kSoftmaxGrad: A = rows of x, B = W.  kGrads, dx: A = u, B =
// W by columns; dW: A2 = u by columns, B2 = x by columns.  tma_c: u
// (kSoftmaxGrad) or dW (kGrads).
template <int JOB>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(V_THREADS, 1)
    vocab_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                 const __grid_constant__ CUtensorMap tma_a2, const __grid_constant__ CUtensorMap tma_b2,
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

  launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < VSTAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * EPI_WARPS);  // of both CTAs
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tma_a);
    prefetch_tensormap(&tma_b);
    if (JOB != kLse) prefetch_tensormap(&tma_c);
    if (JOB == kGrads) {
      prefetch_tensormap(&tma_a2);
      prefetch_tensormap(&tma_b2);
    }
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
  wait_previous();
  if (JOB == kLse) clear_arrivals(p.tickets);
  const Shape e = shape_of(p, JOB == kGrads);
  Unit u;

  if (warp == 0) {
    // ------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      for (int i = 0; !*abort_flag && get_unit<JOB>(e, i, cluster, nclusters, u); ++i) {
        const bool dw = JOB == kGrads && u.split < 0;
        const int row_a = u.mb * TILE + static_cast<int>(crank) * HALF;
        const int row_b = u.nb * TILE + static_cast<int>(crank) * HALF;
        for (int kb = u.kb0; kb < u.kb1; ++kb) {
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
          if (dw) {
            tma_load_2d_pair(a, &tma_a2, lfull, row_a, k0);
            tma_load_2d_pair(a + 8192, &tma_a2, lfull, row_a + 64, k0);
            tma_load_2d_pair(b, &tma_b2, lfull, row_b, k0);
            tma_load_2d_pair(b + 8192, &tma_b2, lfull, row_b + 64, k0);
          } else {
            tma_load_2d_pair(a, &tma_a, lfull, k0, row_a);
            if (JOB == kGrads) {
              tma_load_2d_pair(b, &tma_b, lfull, row_b, k0);
              tma_load_2d_pair(b + 8192, &tma_b, lfull, row_b + 64, k0);
            } else {
              tma_load_2d_pair(b, &tma_b, lfull, k0, row_b);
            }
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
      int stage = 0;
      uint32_t phase = 0;
      int filled = 0;  // accumulators handed over so far
      bool ok = true;
      for (int i = 0; ok && !*abort_flag && get_unit<JOB>(e, i, cluster, nclusters, u); ++i) {
        const bool a_mn = JOB == kGrads && u.split < 0;
        constexpr bool b_mn = JOB == kGrads;
        const uint32_t idesc = a_mn ? idesc_bf16_f32(TILE, TILE, true, b_mn) : idesc_bf16_f32(TILE, TILE, false, b_mn);
        int kb = u.kb0;
        do {  // once per accumulator
          const int acc = filled & 1;
          if (!mbar_wait(&tempty[acc], ((filled >> 1) & 1) ^ 1)) {
            err.set(122);
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t d_tmem = tmem_base + acc * TILE;
          const int first = kb, end = JOB == kGrads ? u.kb1 : min(u.kb1, kb + e.k_acc);
          for (; kb < end; ++kb) {
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
              const uint64_t ad = a_mn ? smem_desc_sw128(a_addr + k * 2048, 8192, 1024)
                                       : smem_desc_sw128(a_addr + k * 32, 16, 1024);
              const uint64_t bd = b_mn ? smem_desc_sw128(b_addr + k * 2048, 8192, 1024)
                                       : smem_desc_sw128(b_addr + k * 32, 16, 1024);
              mma_bf16_pair(d_tmem, ad, bd, idesc, (kb != first || k != 0) ? 1u : 0u);
            }
            mma_commit_pair(&empty[stage], 0x3);
            if (++stage == VSTAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
          if (!ok) break;
          mma_commit_pair(&tfull[acc], 0x3);
          ++filled;
        } while (kb < u.kb1);
      }
    }
  } else {
    // ---------------------------------------------------------- epilogue
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    const int half = (warp - 2) >> 2;  // which 128 columns of the tile
    uint8_t* slab = sE + (warp - 2) * EPI_BUF;
    const uint32_t leader_tempty0 = mapa_shared(smem_u32(&tempty[0]), 0);
    const uint32_t leader_tempty1 = mapa_shared(smem_u32(&tempty[1]), 0);
    const float k2 = p.scale * kLog2e;
    int taken = 0;  // accumulators taken over so far
    // One lane waits and the warp follows it, so the warp never diverges
    // around the .sync.aligned TMEM loads that come after.
    auto take = [&](int& acc) {
      acc = taken & 1;
      int ok = 0;
      if (lane == 0) {
        ok = !*abort_flag;
        if (ok && !mbar_wait(&tfull[acc], (taken >> 1) & 1)) {
          err.set(124);
          *abort_flag = 1;
          ok = 0;
        }
      }
      ++taken;
      if (!__shfl_sync(0xffffffffu, ok, 0)) return false;
      tc_fence_after();
      return true;
    };
    // The accumulator's last read is done.
    auto release = [&](int acc) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc ? leader_tempty1 : leader_tempty0);
    };
    const uint32_t quarter = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
    const int w8 = static_cast<int>(crank) * 4 + q;  // which 32 rows of a tile
    for (int i = 0; get_unit<JOB>(e, i, cluster, nclusters, u); ++i) {
      const int row0 = u.mb * TILE + w8 * 32;
      const int row = row0 + lane;
      const int tcol0 = u.nb * TILE;  // first column of the tile
      int acc;

      // logits of 128 columns of the row, the sum of the tile's accumulators
      auto take_logits = [&](float (&v)[HALF]) {
        if (!take(acc)) return false;
        uint32_t first[HALF / 32][32];
#pragma unroll
        for (int c = 0; c < HALF; c += 32) tmem_ld_32x32b_x32(quarter + acc * TILE + half * HALF + c, first[c / 32]);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < HALF; ++j) v[j] = __uint_as_float(first[j / 32][j % 32]);
        release(acc);
        for (int kb = u.kb0 + e.k_acc; kb < u.kb1; kb += e.k_acc) {
          if (!take(acc)) return false;
#pragma unroll
          for (int c = 0; c < HALF; c += 32) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(quarter + acc * TILE + half * HALF + c, r);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) v[c + j] += __uint_as_float(r[j]);
          }
          release(acc);
        }
        return true;
      };

      if (JOB == kLse) {
        float v[HALF];
        if (!take_logits(v)) break;
        // (largest, sum) in the accumulator's own units: (logit - largest) is
        // exact near the largest, which is where the sum comes from
        const bool row_ok = row < e.rows;
        const int col0 = tcol0 + half * HALF, cols = p.N - col0;
        if (cols < HALF) {  // columns past the vocabulary
#pragma unroll
          for (int j = 0; j < HALF; ++j) v[j] = j < cols ? v[j] : -INFINITY;
        }
        float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int j = 4; j < HALF; ++j) mx[j & 3] = fmaxf(mx[j & 3], v[j]);
        float m = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const float ref = m == -INFINITY ? 0.f : m;
        float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < HALF; ++j) a[j & 3] += ex2((v[j] - ref) * k2);
        float s = (a[0] + a[1]) + (a[2] + a[3]);
        const int64_t t = row_ok ? p.targets[row] - col0 : -1;
        const bool mine = t >= 0 && t < min(cols, HALF) && !T1_OOB(row, p.ld_part);
        if (__any_sync(0xffffffffu, mine)) {
          float x = 0.f;
#pragma unroll
          for (int j = 0; j < HALF; ++j) x = static_cast<int>(t) == j ? v[j] : x;
          if (mine) __stcg(&p.target_logit[row], x);
        }
        if (row_ok && !T1_OOB(row, p.ld_part) && !T1_OOB(2 * u.nb + half, 2 * e.tiles_n))
          __stcg(&p.part[static_cast<size_t>(2 * u.nb + half) * p.ld_part + row], make_float2(m, s));
        if (!p.join) continue;
        // the last of the row group's column blocks joins them all, in order
        __threadfence();
        __syncwarp();
        int last = 0;
        if (lane == 0 && !T1_OOB(u.mb * 8 + w8, p.tickets_n)) last = atomicAdd(&p.tickets.use[u.mb * 8 + w8], 1) == 2 * e.tiles_n - 1;
        if (!__shfl_sync(0xffffffffu, last, 0)) continue;
        __threadfence();
        if (!row_ok) continue;
        m = -INFINITY;
        s = 0.f;
#pragma unroll 4
        for (int b = 0; b < 2 * e.tiles_n; ++b) {
          const float2 w = __ldcg(&p.part[static_cast<size_t>(b) * p.ld_part + row]);
          lse_join(m, s, w.x, w.y, k2);
        }
        const int at = p.index != nullptr ? p.index[row] : row;
        if (T1_OOB(at, p.tokens)) continue;
        const int64_t target = p.targets[row];
        write_logp(m, s, __ldcg(&p.target_logit[row]), target != p.ignore && target >= 0 && target < p.V, p.scale,
                   p.logp + at, p.lse_out + at);
        continue;
      }

      const int col0 = tcol0 + half * HALF;  // this warp's first column
      uint8_t* rowp = slab + lane * 128;
      // 32 columns of the row, rounded, to the slab's left or right half
      auto to_slab = [&](const float (&f)[32], int right, bool zero) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 ov;
          __nv_bfloat162* oh = reinterpret_cast<__nv_bfloat162*>(&ov);
#pragma unroll
          for (int k = 0; k < 4; ++k) oh[k] = __floats2bfloat162_rn(f[8 * j + 2 * k], f[8 * j + 2 * k + 1]);
          if (zero) ov = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(rowp + (((4 * right + j) ^ (lane & 7)) << 4)) = ov;
        }
      };

      // a 32 x 64 slab to the columns c.. of the result, by TMA
      auto store_slab = [&](int c) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tma_c, slab, col0 + c, row0);
          bulk_commit_group();
        }
      };

      if (JOB == kSoftmaxGrad) {
        // u, zeros in the rows past the last that complete kGrads' last block
        // of BK rows (a reduction's length there)
        float v[HALF];
        if (!take_logits(v)) break;
        if (row0 >= e.k_rows * BK) continue;  // uniform over the warp
        const bool row_ok = row < e.rows;
        float lse = 0.f, gr = 0.f;
        int tcol = -1;
        if (row_ok) {
          gr = p.g[row];
          lse = p.lse[row];
          const int64_t t = p.targets[row] - p.col0 - col0;
          tcol = t >= 0 && t < HALF ? static_cast<int>(t) : -1;
        }
#pragma unroll
        for (int c = 0; c < HALF; c += 64) {
          if (col0 + c >= p.N) break;
          // the store issued from the slab before has read it
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
#pragma unroll
          for (int right = 0; right < 2; ++right) {
            float f[32];
            // logit - lse is rounded once, near 0 where the target is sure
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = -gr * ex2(fmaf(v[c + 32 * right + j], p.scale, -lse) * kLog2e);
            if (__any_sync(0xffffffffu, tcol >= c + 32 * right && tcol < c + 32 * right + 32)) {
#pragma unroll
              for (int j = 0; j < 32; ++j) f[j] += tcol == c + 32 * right + j ? gr : 0.f;
            }
            to_slab(f, right, !row_ok);
          }
          store_slab(c);
        }
        continue;
      }

      if (!take(acc)) break;
      const uint32_t taddr = quarter + acc * TILE + half * HALF;
      if (u.split >= 0) {
        // dx: these columns' sums, in fp32 until all of the vocabulary is in
        const bool live = row0 < e.rows;
        const size_t block = (static_cast<size_t>(u.mb * e.tiles_h + u.nb) * e.splits + u.split) * 8 + w8;
        float4* plane = reinterpret_cast<float4*>(p.planes + block * PLANE_BLOCK) + half * (HALF / 4) * 32 + lane;
        const bool dead = row < e.rows && p.g[row] == 0.f;  // its dx is 0, whatever W holds
        const int at = row < e.rows && p.index != nullptr ? p.index[row] : row;
        const bool direct = e.splits == 1 && p.last;  // no other range, no later piece
        // uniform over the warp
        const bool plane_ok = !live || (direct && p.first) || !T1_OOB(block, p.plane_blocks);
        if (lane == 0) bulk_wait_group_read<0>();  // stores of an earlier dW tile have read the slab
        __syncwarp();
#pragma unroll 1
        for (int c = 0; c < HALF; c += 32) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(taddr + c, r);
          tmem_ld_wait();
          if (c + 32 == HALF) release(acc);
          if (!live || !plane_ok || col0 + c >= p.H) continue;
          float f[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = u.kb0 == u.kb1 ? 0.f : __uint_as_float(r[j]);
          if (!p.first) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 v = __ldcg(plane + (c / 4 + j) * 32);
              f[4 * j] += v.x;
              f[4 * j + 1] += v.y;
              f[4 * j + 2] += v.z;
              f[4 * j + 3] += v.w;
            }
          }
          if (!direct) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              __stcg(plane + (c / 4 + j) * 32, make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]));
            continue;
          }
          const int right = (c >> 5) & 1;
          to_slab(f, right, dead);
          if (!right && col0 + c + 32 < p.H) continue;
          // whole 128-byte lines (as far as dx goes) of the rows' tokens
          __syncwarp();
#pragma unroll
          for (int it = 0; it < 8; ++it) {
            const int rr = it * 4 + (lane >> 3), j = lane & 7;
            const int64_t t = __shfl_sync(0xffffffffu, at, rr);
            const uint4 v = *reinterpret_cast<const uint4*>(slab + rr * 128 + ((j ^ (rr & 7)) << 4));
            const int col = col0 + (c & ~63) + 8 * j;
            if (row0 + rr < e.rows && col < p.H && (right || j < 4) && !T1_OOB(t, p.tokens)) *reinterpret_cast<uint4*>(p.dx + t * p.H + col) = v;
          }
          __syncwarp();
        }
        continue;
      }

      // dW through 32 x 64 slabs
#pragma unroll 1
      for (int c = 0; c < HALF; c += 64) {
        uint32_t r[2][32];
        tmem_ld_32x32b_x32(taddr + c, r[0]);
        tmem_ld_32x32b_x32(taddr + c + 32, r[1]);
        // the store issued from the slab before has read it
        if (lane == 0) bulk_wait_group_read<0>();
        __syncwarp();
        tmem_ld_wait();
        if (c + 64 == HALF) release(acc);
        if (col0 + c >= p.H || row0 >= p.N) continue;  // uniform over the warp
#pragma unroll
        for (int right = 0; right < 2; ++right) {
          float f[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) f[j] = __uint_as_float(r[right][j]);
          to_slab(f, right, u.kb0 == u.kb1);  // a sum over no rows is 0
        }
        store_slab(c);
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
