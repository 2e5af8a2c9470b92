// Log-probabilities of the target tokens under the output layer, and their
// gradients, without the [T, V] logits in fp32 or their copy in memory.
//
//   logit[t, v] = x[t, :] . W[v, :] / tau
//   lse[t]      = log sum_v exp(logit[t, v]),  logp[t] = logit[t, target[t]] - lse[t]
//   u[t, v]     = (dlogp[t] / tau) (onehot(target[t])[v] - exp(logit[t, v] - lse[t]))
//   dx[t, :]    = sum_v u[t, v] W[v, :]
//   dW[v, :]    = sum_t u[t, v] x[t, :]
//
// u is the one intermediate that is rounded: to bf16, for the tensor cores.
// Its relative error of 2^-9 at most per element adds to the 2^-9 of the
// results' own rounding; all sums are fp32.  Before that rounding u is as good
// as its formula in fp32: 1 - exp(logit - lse) of a target that is nearly sure
// is off by what fp32 holds of lse (2^-24 of it), which logits summed in the
// forward's order do not add to.
//
// A token whose target is ignored (ignore_index, or outside the vocabulary)
// gives logp = lse = 0 and no gradient, whatever its hidden state holds.
#include "vocab_gemm.cuh"

#include <ATen/cuda/CUDAGraphsUtils.cuh>

#include <optional>
#include <unordered_map>

namespace t1 {

CUtensorMap make_map_any(const void* ptr, int64_t inner, int64_t outer, int64_t ld, int box_outer);
torch::Tensor& gemm_error_word();

using vocab::VocabParams;
using vocab::kLog2e;
using vocab::ex2;

// How many ranges of the vocabulary dx's product is cut into, so that its
// `tiles` long units and the dW tiles fill `clusters` evenly: the smallest
// estimate of the time of the busiest cluster plus the planes' traffic and
// the launch that adds them, in tenths of a k block (0.27 us; a tile's plane
// written and read back is 0.5 MB, 0.08 us of the GPU's bandwidth; the launch
// costs about 3 us).
constexpr int kMaxSplits = 32;
__host__ __device__ inline int64_t splits_cost(int s, int tiles, int k_blocks, int dw_tiles, int tiles_t, int clusters) {
  const int64_t ux = vocab::dx_unit_cost(k_blocks, s), uw = vocab::dw_unit_cost(tiles_t);
  const int64_t units = static_cast<int64_t>(tiles) * s;
  const int64_t even = units * ux + dw_tiles * uw + clusters * uw;  // x clusters, so that nothing is divided
  const int64_t longest = (units < clusters ? 1 : units / clusters + (units % clusters != 0)) * ux * clusters;
  return 10 * (even > longest ? even : longest) + (s > 1 ? (100 + 3 * units) * clusters : 0);
}
// The smallest s of the least cost, on the host and by a warp (a lane per s:
// one thread's 32 turns took 10 us).  Whole numbers: both find the same.
__host__ __device__ inline bool splits_allowed(int s, int k_blocks) { return s == 1 || k_blocks >= 8 * s; }
inline int pick_splits(int tiles, int k_blocks, int dw_tiles, int tiles_t, int clusters) {
  int best = 1;
  for (int s = 2; s <= kMaxSplits && splits_allowed(s, k_blocks); ++s)
    if (splits_cost(s, tiles, k_blocks, dw_tiles, tiles_t, clusters) <
        splits_cost(best, tiles, k_blocks, dw_tiles, tiles_t, clusters))
      best = s;
  return best;
}
__device__ __forceinline__ int pick_splits_warp(int tiles, int k_blocks, int dw_tiles, int tiles_t, int clusters) {
  const int s = static_cast<int>(threadIdx.x & 31) + 1;
  const int64_t cost = splits_allowed(s, k_blocks) ? splits_cost(s, tiles, k_blocks, dw_tiles, tiles_t, clusters) : INT64_MAX;
  int64_t least = cost;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const int64_t other = __shfl_xor_sync(0xffffffffu, static_cast<long long>(least), o);
    least = min(least, other);
  }
  return __ffs(__ballot_sync(0xffffffffu, cost == least));
}

struct PackParams {
  const bf16* x;
  long ldx;
  const int64_t* targets;
  int64_t ignore, V;
  int T, H;
  int per_block;         // tokens of a block
  int per_slice;         // 8-column vectors of a block
  float scale;
  const float* dlogp;    // null in the forward
  const float* lse;      // with dlogp
  int k_blocks, tiles_n, tiles_h, clusters;  // of the products with u, with dlogp
  vocab::RowsMeta* meta;
  int* index;            // [T] the packed row's token
  int64_t* target;       // [T]
  float* g;              // [T] dlogp / tau, with dlogp
  float* lse_packed;     // with dlogp
  bf16* xp;              // [T, with dlogp rounded up to 64; H] the rows of x
  float *zero0, *zero1;  // forward: logp and lse, 0 for the tokens left out
  bf16* dx;              // backward: likewise
};

constexpr int kPackThreads = 256;

// Packs the rows that take part: tokens with a target and, in the backward,
// with a gradient (a clipped token's is exactly 0, and so is all it adds).
// Prompts and padding are often half of a batch, and every product below
// shrinks by them.  A block takes some tokens and some columns; it counts the
// rows before its own tokens itself: T / 2 targets out of L2 on average
// instead of a scan in a launch of its own.  Rows keep their order, so sums
// over rows do not depend on timing.
template <bool BWD>
__global__ void __launch_bounds__(kPackThreads) logprob_pack_kernel(const PackParams p) {
  __shared__ int counts[kPackThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kPackThreads / 32;
  vocab::launch_dependents();
  vocab::wait_previous();
  const int t0 = blockIdx.x * p.per_block, t1 = min(p.T, t0 + p.per_block);
  const bool first_slice = blockIdx.y == 0;
  auto takes_part = [&](int t) {
    const int64_t v = p.targets[t];
    const bool valid = v != p.ignore && v >= 0 && v < p.V;
    return BWD ? valid && p.dlogp[t] != 0.f : valid;
  };
  int n = 0;
#pragma unroll 4
  for (int t = threadIdx.x; t < t0; t += kPackThreads) n += takes_part(t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if (lane == 0) counts[warp] = n;
  __syncthreads();
  int pos = 0;
  for (int w = 0; w < kWarps; ++w) pos += counts[w];

  const int nvec = p.H >> 3;
  const int i0 = blockIdx.y * p.per_slice, i1 = min(nvec, i0 + p.per_slice);
  for (int base = t0; base < t1; base += 32) {
    const bool mine = base + lane < t1 && takes_part(base + lane);
    const unsigned mask = __ballot_sync(0xffffffffu, mine);
    // warp w takes tokens w, w + 8, ... of the 32
    for (int j = warp; j < 32 && base + j < t1; j += kWarps) {
      const int t = base + j;
      if (!(mask >> j & 1)) {
        if (!BWD && lane == 0 && first_slice) p.zero0[t] = p.zero1[t] = 0.f;
        if (BWD)
          for (int i = i0 + lane; i < i1; i += 32)
            reinterpret_cast<uint4*>(p.dx + static_cast<size_t>(t) * p.H)[i] = make_uint4(0, 0, 0, 0);
        continue;
      }
      const int at = pos + __popc(mask & ((1u << j) - 1));
      if (T1_OOB(at, p.T)) continue;
      if (lane == 0 && first_slice) {
        p.index[at] = t;
        p.target[at] = p.targets[t];
        if (BWD) {
          p.g[at] = p.dlogp[t] * p.scale;
          p.lse_packed[at] = p.lse[t];
        }
      }
      const bf16* src = p.x + static_cast<size_t>(t) * p.ldx;
#pragma unroll 4
      for (int i = i0 + lane; i < i1; i += 32) {
        const uint4 v = __ldcs(reinterpret_cast<const uint4*>(src + 8 * i));
        *reinterpret_cast<uint4*>(p.xp + static_cast<size_t>(at) * p.H + 8 * i) = v;
      }
    }
    pos += __popc(mask);
  }
  if (t1 != p.T) return;
  // the last block knows how many there are
  if (warp == 0 && first_slice) {
    const int tiles_t = (pos + vocab::TILE - 1) / vocab::TILE;
    const int splits = BWD ? pick_splits_warp(tiles_t * p.tiles_h, p.k_blocks, p.tiles_n * p.tiles_h, tiles_t, p.clusters) : 1;
    if (lane == 0) {
      p.meta->rows = pos;
      p.meta->splits = splits;
    }
  }
  if (BWD) {  // dW's reduction runs over whole blocks of BK rows
    const int end = (pos + gemm::BK - 1) / gemm::BK * gemm::BK;
    for (int r = pos + warp; r < end; r += kWarps)
      for (int i = i0 + lane; i < i1; i += 32)
        reinterpret_cast<uint4*>(p.xp + static_cast<size_t>(r) * p.H)[i] = make_uint4(0, 0, 0, 0);
  }
}

// Joins the column blocks' (largest, sum) of 32 rows: lanes are rows (a
// block's entries of neighbouring rows are neighbours in memory), warps
// share the column blocks.  `meta` and `index` are null for rows that were
// not packed.
constexpr int kJoinWarps = 32;
__global__ void __launch_bounds__(32 * kJoinWarps) logprob_join_kernel(const VocabParams p, int blocks) {
  __shared__ float sm[kJoinWarps][32], ss[kJoinWarps][32];
  vocab::launch_dependents();
  vocab::wait_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  const int rows = p.meta != nullptr ? p.meta->rows : p.rows;
  if (static_cast<int>(blockIdx.x) * 32 >= rows) return;  // uniform over the block
  const bool in = row < rows && !T1_OOB(row, p.ld_part);
  const float k2 = p.scale * kLog2e;
  float m = -INFINITY, s = 0.f;
  if (in) {
#pragma unroll 4
    for (int b = warp; b < blocks; b += kJoinWarps) {
      const float2 v = p.part[static_cast<size_t>(b) * p.ld_part + row];
      vocab::lse_join(m, s, v.x, v.y, k2);
    }
  }
  sm[warp][lane] = m;
  ss[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || !in) return;
  for (int w = 1; w < kJoinWarps; ++w) m = fmaxf(m, sm[w][lane]);
  const float ref = m == -INFINITY ? 0.f : m;
  s = 0.f;
  for (int w = 0; w < kJoinWarps; ++w) s += ss[w][lane] * ex2((sm[w][lane] - ref) * k2);
  const int t = p.index != nullptr ? p.index[row] : row;
  if (T1_OOB(t, p.tokens)) return;
  const int64_t v = p.targets[row];
  vocab::write_logp(m, s, p.target_logit[row], v != p.ignore && v >= 0 && v < p.V, p.scale, p.logp + t, p.lse_out + t);
}

// dx from the planes of several ranges of the vocabulary, added in their
// order: a block per 32 rows x 64 columns, a lane per row, a warp per four
// columns (512 consecutive bytes of a plane), eight planes' loads in flight.
// Adding them up in the product's own epilogue left it to one warp per 32
// rows, one latency after the other (40 us for 32 planes; here 6).
constexpr int kPlanesThreads = 512;
__global__ void __launch_bounds__(kPlanesThreads) logprob_planes_kernel(const VocabParams p) {
  __shared__ __align__(16) uint8_t slab[32 * 128];
  vocab::launch_dependents();
  vocab::wait_previous();
  const vocab::Shape e = vocab::shape_of(p, true);
  if (e.splits == 1) return;  // written by the product
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tile = blockIdx.x >> 3, w8 = blockIdx.x & 7;
  const int mb = tile / e.tiles_h, nb = tile % e.tiles_h;
  const int row0 = mb * vocab::TILE + w8 * 32, row = row0 + lane;
  const int col0 = nb * vocab::TILE + blockIdx.y * 64;
  if (row0 >= e.rows || col0 >= p.H) return;
  const float4* plane = reinterpret_cast<const float4*>(p.planes + (static_cast<size_t>(tile) * e.splits * 8 + w8) * vocab::PLANE_BLOCK) +
                        (blockIdx.y * 16 + warp) * 32 + lane;
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  const int64_t last_block = (static_cast<int64_t>(tile + 1) * e.splits - 1) * 8 + w8;
  if (col0 + warp * 4 < p.H && !T1_OOB(last_block, p.plane_blocks)) {
    for (int s0 = 0; s0 < e.splits; s0 += 8) {
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = s0 + k < e.splits ? __ldcg(plane + static_cast<size_t>(s0 + k) * (8 * vocab::PLANE_BLOCK / 4))
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        f.x += v[k].x;
        f.y += v[k].y;
        f.z += v[k].z;
        f.w += v[k].w;
      }
    }
  }
  if (row < e.rows && p.g[row] == 0.f) f = make_float4(0.f, 0.f, 0.f, 0.f);  // whatever W holds
  uint2 o;
  __nv_bfloat162* oh = reinterpret_cast<__nv_bfloat162*>(&o);
  oh[0] = __floats2bfloat162_rn(f.x, f.y);
  oh[1] = __floats2bfloat162_rn(f.z, f.w);
  *reinterpret_cast<uint2*>(slab + lane * 128 + (((warp >> 1) ^ (lane & 7)) << 4) + (warp & 1) * 8) = o;
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int rr = threadIdx.x >> 3, j = threadIdx.x & 7, col = col0 + 8 * j;
  if (row0 + rr >= e.rows || col >= p.H) return;
  const int64_t t = p.index != nullptr ? p.index[row0 + rr] : row0 + rr;
  if (T1_OOB(t, p.tokens)) return;
  *reinterpret_cast<uint4*>(p.dx + t * p.H + col) = *reinterpret_cast<const uint4*>(slab + rr * 128 + ((j ^ (rr & 7)) << 4));
}

// -------------------------------------------------------------- few rows
// At most 16 tokens (a decoding step's, a short answer's): all that counts is
// reading W once (the gradient reads it once more for dx, and writes dW: 775 us
// for one token, 830 for 16).  A group of warps takes 16 rows of W at a time and shares
// their columns, as many warps as leave each about 256 columns (8 loads of 16
// bytes per row in flight for a thread, 128 KB for an SM); they read W straight into mma fragments (a thread's 16 bytes are
// the four k's that two m16n8k16 steps give it: the order of a sum is free, so
// no shuffling and no shared memory for W) and keep x in shared memory.  The
// next rows' loads are in flight while a block adds up its warps' parts.
// tcgen05 tiles would spend 256 rows of tensor time on them and read x
// through TMA boxes that are mostly padding (T=1 at V=128256, H=4096: 260 us
// against 175 us here, 6.0 TB/s).
struct FewParams {
  const bf16* x;
  long ldx;
  const bf16* w;
  long ldw;
  const int64_t* targets;
  int64_t ignore;
  int T, H, V;
  int share;             // warps that share a group's columns, a power of two
  float scale;
  // forward
  Arrivals ticket;       // of the blocks
  int blocks;            // that part has room for
  float2* part;          // [block][16]
  float* target_logit;   // [16]
  float *logp, *lse_out;
  // backward
  const float *dlogp, *lse;
  bf16* u;               // [T, ldu]
  long ldu;
  float* g;              // [T] dlogp / tau
  bf16* xz;              // [T, H] x, zeros for tokens without a gradient
};

constexpr int kFewThreads = 512;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewRows = 16;    // rows of W of a group
constexpr int kFewLoads = 8;    // blocks of 32 columns that a warp has in flight

// Distance of two tokens' columns in shared memory: 64 bytes past a multiple
// of 128, so that the 8 threads of a 16-byte read's phase (2 tokens x 4)
// touch every bank once.
__host__ __device__ inline int few_pitch(int H) { return (2 * H + 127) / 128 * 128 + 64; }
inline size_t few_smem(int tokens8, int H) {
  return static_cast<size_t>(tokens8) * few_pitch(H) + 2 * kFewWarps * kFewRows * tokens8 * sizeof(float);
}

__device__ __forceinline__ uint4 ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NT, bool BWD>
__global__ void __launch_bounds__(kFewThreads, 1) logprob_few_kernel(const FewParams p) {
  constexpr int TOK = 8 * NT;
  constexpr int CELLS = kFewRows * TOK;  // a group's logits
  extern __shared__ __align__(16) uint8_t few_raw[];
  uint8_t* xs = few_raw;
  const int pitch = few_pitch(p.H);
  float* red = reinterpret_cast<float*>(few_raw + TOK * pitch);
  __shared__ int last;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, c = lane & 3;
  vocab::launch_dependents();
  vocab::wait_previous();
  if (!BWD) clear_arrivals(p.ticket);

  const int teams = kFewWarps / p.share, team = warp / p.share, part = warp % p.share;
  const int blocks32 = (p.H + 31) / 32;                       // of columns
  const int kb_lo = part * blocks32 / p.share, kb_hi = (part + 1) * blocks32 / p.share;
  const int per_warp = (blocks32 + p.share - 1) / p.share;
  const int chunks = (per_warp + kFewLoads - 1) / kFewLoads;  // the same for every warp
  const int rounds = (p.V + kFewRows * teams - 1) / (kFewRows * teams);  // of all blocks: a group per team
  const int steps = (rounds - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x) * chunks;

  uint4 wa[kFewLoads], wb[kFewLoads];
  auto load = [&](int step) {
    const int group = (static_cast<int>(blockIdx.x) + step / chunks * static_cast<int>(gridDim.x)) * teams + team;
    const int ra = min(p.V - 1, group * kFewRows + g), rb = min(p.V - 1, group * kFewRows + g + 8);
    const bf16* pa = p.w + static_cast<size_t>(ra) * p.ldw;
    const bf16* pb = p.w + static_cast<size_t>(rb) * p.ldw;
#pragma unroll
    for (int i = 0; i < kFewLoads; ++i) {
      const int kb = kb_lo + step % chunks * kFewLoads + i, k = kb * 32 + c * 8;
      const bool in = kb < kb_hi && k < p.H;
      wa[i] = in ? ld_stream(pa + k) : make_uint4(0, 0, 0, 0);
      wb[i] = in ? ld_stream(pb + k) : make_uint4(0, 0, 0, 0);
    }
  };
  if (steps > 0) load(0);

  // x to shared memory, zeros past its columns and tokens
  const int vecs = (pitch - 64) / 16;
  for (int i = tid; i < TOK * vecs; i += kFewThreads) {
    const int t = i / vecs, v = i % vecs;
    uint4 val = make_uint4(0, 0, 0, 0);
    if (t < p.T && 8 * v < p.H) val = *reinterpret_cast<const uint4*>(p.x + static_cast<size_t>(t) * p.ldx + 8 * v);
    *reinterpret_cast<uint4*>(xs + t * pitch + 16 * v) = val;
  }
  // what this thread's cells need to know: all are of one token
  const int token = tid % TOK;
  const bool cell = tid < CELLS * teams && token < p.T;
  const int64_t target = cell ? p.targets[token] : -1;
  const bool valid = cell && target != p.ignore && target >= 0 && target < p.V;
  const float k2 = p.scale * kLog2e;
  float lse = 0.f, gr = 0.f;
  if (BWD && valid) {
    lse = p.lse[token];
    gr = p.dlogp[token] * p.scale;
  }
  if (BWD && blockIdx.x == 0 && cell && tid < TOK && !T1_OOB(token, p.T)) p.g[token] = gr;
  __syncthreads();
  if (BWD) {  // a share of x per block
    const int nvec = p.H / 8;
    for (int i = blockIdx.x * kFewThreads + tid; i < p.T * nvec; i += gridDim.x * kFewThreads) {
      const int t = i / nvec, v = i % nvec;
      if (T1_OOB(t, p.T)) continue;
      const int64_t tt = p.targets[t];
      const bool live = tt != p.ignore && tt >= 0 && tt < p.V && p.dlogp[t] != 0.f;
      *reinterpret_cast<uint4*>(p.xz + static_cast<size_t>(t) * p.H + 8 * v) =
          live ? *reinterpret_cast<const uint4*>(xs + t * pitch + 16 * v) : make_uint4(0, 0, 0, 0);
    }
  }

  float m = -INFINITY, s = 0.f;
  float acc[NT][4] = {};
  int buf = 0;
  for (int step = 0; step < steps; ++step) {
    const int chunk = step % chunks;
#pragma unroll
    for (int i = 0; i < kFewLoads; ++i) {
      const int kb = kb_lo + chunk * kFewLoads + i;
      if (kb >= kb_hi) break;  // uniform over the warp
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 xv = *reinterpret_cast<const uint4*>(xs + (n * 8 + g) * pitch + kb * 64 + c * 16);
        mma_16816(acc[n], wa[i].x, wb[i].x, wa[i].y, wb[i].y, xv.x, xv.y);
        mma_16816(acc[n], wa[i].z, wb[i].z, wa[i].w, wb[i].w, xv.z, xv.w);
      }
    }
    if (step + 1 < steps) load(step + 1);
    if (chunk + 1 < chunks) continue;
    // the warps' parts of 16 x TOK logits
    float* mine = red + (buf * kFewWarps + warp) * CELLS;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      *reinterpret_cast<float2*>(mine + g * TOK + n * 8 + 2 * c) = make_float2(acc[n][0], acc[n][1]);
      *reinterpret_cast<float2*>(mine + (g + 8) * TOK + n * 8 + 2 * c) = make_float2(acc[n][2], acc[n][3]);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[n][k] = 0.f;
    }
    __syncthreads();  // two buffers: the next step's parts go to the other
    const int round = static_cast<int>(blockIdx.x) + step / chunks * static_cast<int>(gridDim.x);
    for (int i = tid; cell && i < CELLS * teams; i += kFewThreads) {
      const int of = i / CELLS, at = i % CELLS;
      const int v = (round * teams + of) * kFewRows + at / TOK;
      if (v >= p.V) continue;
      float l = 0.f;
      for (int w = 0; w < p.share; ++w) l += red[(buf * kFewWarps + of * p.share + w) * CELLS + at];
      if (BWD) {
        const float uv = gr != 0.f ? gr * ((v == target ? 1.f : 0.f) - ex2(fmaf(l, p.scale, -lse) * kLog2e)) : 0.f;
        if (!T1_OOB(token, p.T) && !T1_OOB(v, p.ldu)) p.u[token * p.ldu + v] = __float2bfloat16_rn(uv);
      } else {
        vocab::lse_join(m, s, l, 1.f, k2);
        if (v == target && !T1_OOB(token, 16)) __stcg(&p.target_logit[token], l);
      }
    }
    buf ^= 1;
  }
  if (BWD) return;

  // this block's (largest, sum) per token, then all blocks' by the last one
  float2* cells = reinterpret_cast<float2*>(red);
  __syncthreads();
  cells[tid] = make_float2(m, s);
  __syncthreads();
  if (tid < TOK) {
    for (int r = 1; r < min(kFewThreads, CELLS * teams) / TOK; ++r)
      vocab::lse_join(m, s, cells[r * TOK + tid].x, cells[r * TOK + tid].y, k2);
    if (!T1_OOB(blockIdx.x, p.blocks) && !T1_OOB(tid, 16)) __stcg(&p.part[blockIdx.x * 16 + tid], make_float2(m, s));
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) last = atomicAdd(p.ticket.use, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (warp >= p.T) return;  // a warp per token
  m = -INFINITY;
  s = 0.f;
  for (int b = lane; b < static_cast<int>(gridDim.x); b += 32) {
    const float2 v = __ldcg(&p.part[b * 16 + warp]);
    vocab::lse_join(m, s, v.x, v.y, k2);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
    vocab::lse_join(m, s, m2, s2, k2);
  }
  if (lane == 0) {
    const int64_t t = p.targets[warp];
    vocab::write_logp(m, s, __ldcg(&p.target_logit[warp]), t != p.ignore && t >= 0 && t < p.V, p.scale, p.logp + warp,
                      p.lse_out + warp);
  }
}

// ================================================================ host side
T1_BOUNDS_READER(logprob)

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// A launch whose prologue may overlap the end of the stream's previous
// kernel (every kernel here waits for it before it touches memory).
template <class... P, class... A>
static void launch_after(const char* what, void (*kern)(P...), dim3 grid, int threads, size_t smem, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream();
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
  TORCH_CHECK(e == cudaSuccess, what, " launch failed: ", cudaGetErrorString(e));
  count_launch();
}

// `units`: the most units of work that the launch can have.
template <int JOB>
static void launch_vocab(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& ta2, const CUtensorMap& tb2,
                         const CUtensorMap& tc, VocabParams& p, int64_t units) {
  auto kern = vocab::vocab_kernel<JOB>;
  static DeviceFlags configured;
  if (bool& done = configured.here(); !done) {
    T1_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, vocab::V_SMEM_BYTES));
    done = true;
  }
  p.err = gemm_error_word().data_ptr<int>();
  const int clusters = static_cast<int>(std::min<int64_t>(units, num_sms() / 2));
  launch_after("linear_logprob", kern, dim3(2 * clusters), vocab::V_THREADS, vocab::V_SMEM_BYTES, ta, tb, ta2, tb2, tc, p);
}

static torch::TensorOptions counter_options() {
  int dev = 0;
  cudaGetDevice(&dev);
  return torch::TensorOptions().dtype(torch::kInt32).device(torch::kCUDA, dev);
}

// The current stream's.
static ArrivalSets& arrival_sets() {
  static std::unordered_map<uint64_t, ArrivalSets> all;
  return all[(static_cast<uint64_t>(counter_options().device().index()) << 56) ^ reinterpret_cast<uint64_t>(stream())];
}

ArrivalCounters::ArrivalCounters(int64_t n) : n_(n) {
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None) {
    held_ = torch::zeros({n}, counter_options());
    arrivals.use = held_.data_ptr<int>();
    return;
  }
  ArrivalSets& s = arrival_sets();
  if (s.capacity < n) {
    s.capacity = std::max<int64_t>(4096, n);
    s.counters = torch::zeros({2 * s.capacity}, counter_options());
    s.used = 0;
  }
  arrivals.use = s.counters.data_ptr<int>() + s.next * s.capacity;
  arrivals.clear = s.counters.data_ptr<int>() + (1 - s.next) * s.capacity;
  arrivals.clear_n = static_cast<int>(s.used);
  sets_ = &s;
}

// Leaves the counters of the current stream's last launch at `value`, as a
// launch whose wait expired does.
void fill_last_arrivals(int64_t value) {
  ArrivalSets& s = arrival_sets();
  if (s.used > 0) s.counters.narrow(0, (1 - s.next) * s.capacity, s.used).fill_(value);
}

// A workspace cut into 256-byte aligned pieces.
struct Pieces {
  int64_t used = 0;
  int64_t take(int64_t bytes) {
    const int64_t at = used;
    used += round_up(bytes, 256);
    return at;
  }
};

// Distance of two rows; a single row's own stride says nothing.
static int64_t row_ld(const torch::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

static bool aligned_rows(const torch::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && row_ld(t) % 8 == 0;
}

static void check_logprob(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& targets,
                          double temperature) {
  T1_CHECK_INPUT(x, torch::kBFloat16);
  T1_CHECK_INPUT(w, torch::kBFloat16);
  TORCH_CHECK(targets.is_cuda() && targets.scalar_type() == torch::kInt64, "targets must be int64 CUDA");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1), "x must be [T, H] and w [V, H]");
  TORCH_CHECK(x.size(1) > 0 && x.size(1) % 8 == 0, "H must be a positive multiple of 8");
  TORCH_CHECK(w.size(0) > 0 && w.size(0) < (1ll << 30) && x.size(0) < (1ll << 30) && w.size(1) < (1ll << 30),
              "extents of x and w must lie below 2^30, and V above 0");
  TORCH_CHECK(x.stride(1) == 1 && w.stride(1) == 1 && (x.size(0) < 2 || x.stride(0) >= x.size(1)) &&
                  (w.size(0) < 2 || w.stride(0) >= w.size(1)), "x and w must be row-major");
  TORCH_CHECK(targets.dim() == 1 && targets.size(0) == x.size(0), "targets must have T entries");
  TORCH_CHECK(w.device() == x.device() && targets.device() == x.device(), "operands must be on one device");
  TORCH_CHECK(aligned_rows(x) && aligned_rows(w), "x and w must have 16-byte aligned rows");
  TORCH_CHECK(std::isfinite(temperature) && temperature > 0, "temperature must be positive");
}

static void launch_pack(PackParams& p) {
  // about four blocks per SM: 8 to 32 tokens each and, when these are few,
  // slices of the columns (64 vectors at least, two per lane)
  p.per_block = static_cast<int>(std::min<int64_t>(32, std::max<int64_t>(8, ceil_div(p.T, 4 * num_sms()))));
  const int64_t groups = ceil_div(p.T, p.per_block);
  const int64_t slices = std::max<int64_t>(1, std::min(ceil_div(p.H / 8, 64), 4 * num_sms() / groups));
  p.per_slice = static_cast<int>(ceil_div(p.H / 8, slices));
  const dim3 grid(groups, ceil_div(p.H / 8, p.per_slice));
  if (p.dlogp != nullptr) launch_after("logprob_pack", logprob_pack_kernel<true>, grid, kPackThreads, 0, p);
  else launch_after("logprob_pack", logprob_pack_kernel<false>, grid, kPackThreads, 0, p);
}

// Whether a batch takes the few-rows kernel: x has to fit in shared memory.
constexpr size_t kFewSmem = 200 * 1024;
static bool few_rows(int64_t T, int64_t H) { return T <= 16 && few_smem(T <= 8 ? 8 : 16, H) <= kFewSmem; }

static int few_share(int64_t H) {
  int share = 1;
  while (share < kFewWarps && share * kFewLoads * 32 < H) share *= 2;
  return share;
}

static int few_grid(int64_t V, int64_t H) {
  return static_cast<int>(std::min<int64_t>(ceil_div(V, kFewRows * (kFewWarps / few_share(H))), num_sms()));
}

static FewParams few_params(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& targets, int64_t ignore,
                            double temperature) {
  FewParams p{};
  p.x = (const bf16*)x.data_ptr();
  p.ldx = row_ld(x);
  p.w = (const bf16*)w.data_ptr();
  p.ldw = row_ld(w);
  p.targets = targets.data_ptr<int64_t>();
  p.ignore = ignore;
  p.T = x.size(0);
  p.H = x.size(1);
  p.V = w.size(0);
  p.share = few_share(p.H);
  p.scale = static_cast<float>(1.0 / temperature);
  return p;
}

template <bool BWD>
static void launch_few(const FewParams& p) {
  const int tokens8 = p.T <= 8 ? 8 : 16;
  auto kern = tokens8 == 8 ? logprob_few_kernel<1, BWD> : logprob_few_kernel<2, BWD>;
  static DeviceFlags configured[2];
  if (bool& done = configured[tokens8 / 8 - 1].here(); !done) {
    T1_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewSmem));
    done = true;
  }
  launch_after("logprob_few", kern, dim3(few_grid(p.V, p.H)), kFewThreads, few_smem(tokens8, p.H), p);
}

// Whether the forward packs its rows first.  Below 256 tokens there is one
// row of tiles whatever is left out, and a product of less than about 30 us
// gains less from losing half of its rows than the packing costs (6 us).
static bool packs(int64_t T, int64_t H, int64_t V) {
  return T > vocab::TILE && static_cast<double>(T) * H * V > 2e10;
}

// Tiles of columns up to which the last of them joins the rows' sums itself: a
// launch of its own costs about as much as the 64 reads of 32 tiles.
constexpr int kJoinBlocks = 32;

// Returns (logp [T], lse [T]), fp32.
std::vector<torch::Tensor> linear_logprob_fwd(torch::Tensor x, torch::Tensor w, torch::Tensor targets,
                                              int64_t ignore_index, double temperature) {
  check_logprob(x, w, targets, temperature);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), H = x.size(1), V = w.size(0);
  auto f32 = x.options().dtype(torch::kFloat32);
  auto logp = torch::empty({T}, f32), lse = torch::empty({T}, f32);
  if (T == 0) return {logp, lse};
  auto tg = targets.contiguous();
  if (few_rows(T, H)) {
    FewParams p = few_params(x, w, tg, ignore_index, temperature);
    auto ws = torch::empty({32 * few_grid(V, H) + 16}, f32);
    p.part = reinterpret_cast<float2*>(ws.data_ptr<float>());
    p.blocks = few_grid(V, H);
    p.target_logit = ws.data_ptr<float>() + 32 * few_grid(V, H);
    ArrivalCounters counters(1);
    p.ticket = counters.arrivals;
    p.logp = logp.data_ptr<float>();
    p.lse_out = lse.data_ptr<float>();
    launch_few<false>(p);
    counters.launched();
    return {logp, lse};
  }
  const int64_t blocks = ceil_div(V, vocab::TILE), tiles_t = ceil_div(T, vocab::TILE);
  const bool pack = packs(T, H, V);
  Pieces ws;
  const int64_t o_logit = ws.take(4 * T), o_part = ws.take(2 * 8 * blocks * T);
  const int64_t o_meta = ws.take(sizeof(vocab::RowsMeta)), o_index = ws.take(4 * T), o_target = ws.take(8 * T);
  const int64_t o_x = ws.take(pack ? 2 * T * H : 0);
  auto buf = torch::empty({ws.used}, x.options().dtype(torch::kUInt8));
  uint8_t* base = buf.data_ptr<uint8_t>();

  VocabParams p{};
  p.rows = static_cast<int>(T);
  p.N = static_cast<int>(V);
  p.H = static_cast<int>(H);
  p.scale = static_cast<float>(1.0 / temperature);
  p.targets = tg.data_ptr<int64_t>();
  p.ignore = ignore_index;
  p.V = V;
  p.ld_part = p.tokens = static_cast<int>(T);
  p.part = reinterpret_cast<float2*>(base + o_part);
  p.target_logit = reinterpret_cast<float*>(base + o_logit);
  p.logp = logp.data_ptr<float>();
  p.lse_out = lse.data_ptr<float>();
  p.join = blocks <= kJoinBlocks;
  std::optional<ArrivalCounters> counters;
  if (p.join) {
    counters.emplace(tiles_t * 8);
    p.tickets = counters->arrivals;
    p.tickets_n = static_cast<int>(tiles_t * 8);
  }
  if (pack) {
    PackParams k{};
    k.x = (const bf16*)x.data_ptr();
    k.ldx = row_ld(x);
    k.targets = p.targets;
    k.ignore = ignore_index;
    k.V = V;
    k.T = T;
    k.H = H;
    k.meta = reinterpret_cast<vocab::RowsMeta*>(base + o_meta);
    k.index = reinterpret_cast<int*>(base + o_index);
    k.target = reinterpret_cast<int64_t*>(base + o_target);
    k.xp = reinterpret_cast<bf16*>(base + o_x);
    k.zero0 = p.logp;
    k.zero1 = p.lse_out;
    launch_pack(k);
    p.meta = k.meta;
    p.index = k.index;
    p.targets = k.target;
  }
  CUtensorMap ta = make_map_any(pack ? base + o_x : x.data_ptr(), H, T, pack ? H : row_ld(x), vocab::HALF);
  CUtensorMap tb = make_map_any(w.data_ptr(), H, V, row_ld(w), vocab::HALF);
  launch_vocab<vocab::kLse>(ta, tb, ta, tb, ta, p, tiles_t * blocks);
  if (p.join) counters->launched();
  else launch_after("logprob_join", logprob_join_kernel, dim3(ceil_div(T, 32)), 32 * kJoinWarps, 0, p, 2 * blocks);
  return {logp, lse};
}

// The softmax gradient u exists for as many vocabulary columns at a time as
// fit this many bytes; dW's rows of those columns are then final, and dx
// gathers the pieces' products in fp32.
constexpr int64_t kGradBufferBytes = 1ll << 30;

// Writes dx [T, H] and dw [V, H].
void linear_logprob_bwd(torch::Tensor dlogp, torch::Tensor x, torch::Tensor w, torch::Tensor targets,
                        torch::Tensor lse, torch::Tensor dx, torch::Tensor dw, int64_t ignore_index,
                        double temperature) {
  check_logprob(x, w, targets, temperature);
  T1_CHECK_INPUT(dlogp, torch::kFloat32);
  T1_CHECK_INPUT(lse, torch::kFloat32);
  T1_CHECK_INPUT(dx, torch::kBFloat16);
  T1_CHECK_INPUT(dw, torch::kBFloat16);
  const int64_t T = x.size(0), H = x.size(1), V = w.size(0);
  TORCH_CHECK(dlogp.dim() == 1 && dlogp.size(0) == T && lse.dim() == 1 && lse.size(0) == T,
              "dlogp and lse must have T entries");
  TORCH_CHECK(dx.sizes() == x.sizes() && dx.is_contiguous(), "dx must be contiguous [T, H]");
  TORCH_CHECK(dw.sizes() == w.sizes() && dw.is_contiguous(), "dw must be contiguous [V, H]");
  TORCH_CHECK(dlogp.device() == x.device() && lse.device() == x.device() && dx.device() == x.device() &&
                  dw.device() == x.device(), "operands must be on one device");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(dx.data_ptr()) % 16 == 0, "dx must be 16-byte aligned");
  const c10::cuda::CUDAGuard guard(x.device());
  if (T == 0) {
    dw.zero_();
    return;
  }
  auto tg = targets.contiguous(), up = dlogp.contiguous(), ls = lse.contiguous();
  const int clusters = num_sms() / 2;
  const int64_t tiles_t = ceil_div(T, vocab::TILE), tiles_h = ceil_div(H, vocab::TILE);

  const int64_t most = std::max<int64_t>(vocab::TILE, kGradBufferBytes / (2 * T) / vocab::TILE * vocab::TILE);
  const int64_t pieces = ceil_div(V, most);
  const int64_t width = std::min(V, round_up(ceil_div(V, pieces), vocab::TILE));
  const bool few = few_rows(T, H) && pieces == 1;
  // with few rows nothing is packed: u and x have T rows, and TMA reads zeros
  // past them
  const int64_t ldu = round_up(width, 8), u_rows = few ? T : round_up(T, gemm::BK), k_v = ceil_div(width, gemm::BK);
  const int64_t tiles_v = ceil_div(width, vocab::TILE);
  // the most planes and units that the split rule can ask for, over the
  // numbers of rows that the packing may leave
  int64_t planes = 0, most_units = 0, split_tiles = 0;
  for (int64_t m = 1; m <= tiles_t; ++m) {
    const int64_t tiles = m * tiles_h, n = tiles * pick_splits(tiles, k_v, tiles_v * tiles_h, m, clusters);
    most_units = std::max(most_units, n);
    if (pieces > 1 || n > tiles) planes = std::max(planes, n);
    if (n > tiles) split_tiles = std::max(split_tiles, tiles);
  }
  const bool may_split = split_tiles > 0;
  Pieces ws;
  const int64_t o_meta = ws.take(sizeof(vocab::RowsMeta)), o_index = ws.take(4 * T), o_target = ws.take(8 * T),
                o_g = ws.take(4 * T), o_lse = ws.take(4 * T), o_x = ws.take(2 * u_rows * H),
                o_planes = ws.take(4 * 8 * vocab::PLANE_BLOCK * planes), o_u = ws.take(2 * u_rows * ldu);
  auto buf = torch::empty({ws.used}, x.options().dtype(torch::kUInt8));
  uint8_t* base = buf.data_ptr<uint8_t>();

  VocabParams p{};
  p.H = static_cast<int>(H);
  p.g = reinterpret_cast<float*>(base + o_g);
  p.dx = (bf16*)dx.data_ptr();
  p.planes = reinterpret_cast<float*>(base + o_planes);
  p.plane_blocks = 8 * planes;
  p.tokens = static_cast<int>(T);
  bf16 *u = reinterpret_cast<bf16*>(base + o_u), *xp = reinterpret_cast<bf16*>(base + o_x);
  const CUtensorMap txc = make_map_any(xp, H, u_rows, H, gemm::BK);
  if (few) {
    FewParams f = few_params(x, w, tg, ignore_index, temperature);
    f.dlogp = up.data_ptr<float>();
    f.lse = ls.data_ptr<float>();
    f.u = u;
    f.ldu = ldu;
    f.g = reinterpret_cast<float*>(base + o_g);
    f.xz = xp;
    launch_few<true>(f);
    p.rows = static_cast<int>(T);
    p.splits = pick_splits(tiles_h, k_v, tiles_v * tiles_h, 1, clusters);
    p.N = static_cast<int>(V);
    p.first = p.last = 1;
    launch_vocab<vocab::kGrads>(make_map_any(u, V, T, ldu, vocab::HALF),
                                make_map_any(w.data_ptr(), H, V, row_ld(w), gemm::BK),
                                make_map_any(u, V, T, ldu, gemm::BK), txc,
                                make_map_any(dw.data_ptr(), H, V, H, 32), p, most_units + tiles_v * tiles_h);
    if (p.splits > 1) launch_after("logprob_planes", logprob_planes_kernel, dim3(tiles_h * 8, 4), kPlanesThreads, 0, p);
    return;
  }

  PackParams k{};
  k.x = (const bf16*)x.data_ptr();
  k.ldx = row_ld(x);
  k.targets = tg.data_ptr<int64_t>();
  k.ignore = ignore_index;
  k.V = V;
  k.T = T;
  k.H = H;
  k.scale = static_cast<float>(1.0 / temperature);
  k.dlogp = up.data_ptr<float>();
  k.lse = ls.data_ptr<float>();
  k.k_blocks = k_v;
  k.tiles_n = tiles_v;
  k.tiles_h = tiles_h;
  k.clusters = clusters;
  k.meta = reinterpret_cast<vocab::RowsMeta*>(base + o_meta);
  k.index = reinterpret_cast<int*>(base + o_index);
  k.target = reinterpret_cast<int64_t*>(base + o_target);
  k.g = reinterpret_cast<float*>(base + o_g);
  k.lse_packed = reinterpret_cast<float*>(base + o_lse);
  k.xp = xp;
  k.dx = p.dx;
  launch_pack(k);

  p.meta = k.meta;
  p.scale = k.scale;
  p.index = k.index;
  p.targets = k.target;
  p.lse = k.lse_packed;
  const CUtensorMap tx = make_map_any(xp, H, u_rows, H, vocab::HALF);
  for (int64_t v0 = 0; v0 < V; v0 += width) {
    const int64_t n = std::min(width, V - v0);
    const bf16* wp = (const bf16*)w.data_ptr() + v0 * row_ld(w);
    p.N = static_cast<int>(n);
    p.col0 = static_cast<int>(v0);
    p.first = v0 == 0;
    p.last = v0 + width >= V;
    const CUtensorMap tw = make_map_any(wp, H, n, row_ld(w), vocab::HALF);
    const CUtensorMap twc = make_map_any(wp, H, n, row_ld(w), gemm::BK);
    const CUtensorMap tu = make_map_any(u, n, u_rows, ldu, vocab::HALF);
    const CUtensorMap tuc = make_map_any(u, n, u_rows, ldu, gemm::BK);
    const CUtensorMap tus = make_map_any(u, n, u_rows, ldu, 32);
    const CUtensorMap tdw = make_map_any((bf16*)dw.data_ptr() + v0 * H, H, n, H, 32);
    launch_vocab<vocab::kSoftmaxGrad>(tx, tw, tx, tw, tus, p, tiles_t * ceil_div(n, vocab::TILE));
    launch_vocab<vocab::kGrads>(tu, twc, tuc, txc, tdw, p, most_units + ceil_div(n, vocab::TILE) * tiles_h);
  }
  if (may_split) launch_after("logprob_planes", logprob_planes_kernel, dim3(split_tiles * 8, 4), kPlanesThreads, 0, p);
}

}  // namespace t1
