// The likeliest tokens of a row of logits, and one token drawn from it.
//
// Tokens of a row are ordered by logit, largest first, equals by index.  With
// m the largest logit and w_i = exp((z_i - m) / tau):
//   top     the first k, their log-probabilities (z_i - m) / tau - log sum w
//   sample  top_k keeps the first k; top_p, of these, the ones before which
//           less than top_p of their sum has come; min_p those of w_i >= min_p.
//           Each keeps a prefix of the order.  The token drawn is the lowest
//           kept index whose running sum, in index order, exceeds u times the
//           kept tokens' sum.
// -inf and NaN are no tokens; a logit of +inf outweighs all finite ones.
//
// A scan of the whole row by many CTAs, then what is left of it by one (finish),
// which starts in the scan's tail.  Two kinds of scan:
//   scan_list  top, and top_k of at most 1024.  No r tokens of a stretch can all
//              lie below the r-th largest of the largest logits of its 256 or
//              1024 parts, which a histogram of their distances from the
//              stretch's own largest finds: what lies above, little more than r,
//              is listed.  r is a stretch's share of what is asked for and some
//              more; finish looks once more at those that have held back a
//              token that matters.  The stretches know nothing of each other: as
//              one cluster per row that agreed on m and on the bound, the same
//              work waited in barriers most of the time (1024 rows of 128256,
//              k = 64: 264 us), and with r = k its CTAs spent theirs on listing
//              (172 us).  A warp's stretches of 1024 in registers, without any
//              barrier, are scanned in 106 us where these take 118, and cost
//              finish more than that: it has eight times as many lists.
//   scan_bins  all other draws.  A cluster of CTAs holds the row in shared
//              memory and agrees on m; weights are added up, with top_p by
//              distance from m as well, 16 bins per factor of two, and the tokens
//              of the bin where top_p is reached are listed (a tenth of the
//              vocabulary may fall into one).
// Where a list is too long (many equal logits) or does not hold what is asked
// for, finish finds the cut digit by digit, 8 bits at a time, of the
// order-preserving integer of a logit, reading the row anew each time.  Rows of
// which only some hundred neighbouring tokens are not -inf, or whose masked
// stretches hold a finite lowest value throughout, end there: a draw of 50 in
// 410 to 530 us for one row of 128256, 16 unmasked.
// Measured: the likeliest 64 of 1024 rows of 128256 in 119 to 133 us (4.4 to 4.0
// TB/s; 21 instructions a warp for 32 logits in the scan, 75 % of its issue
// slots); 256 draws with top_p in 162 us, 144 of them scan_bins (81 instructions
// for 32 logits, at 57 % of the issue slots: 54 for the exact weight and its bin,
// the rest behind the cluster's first barrier); one draw with top_k in 12 us,
// latencies of two launches.
//
// Weights are 64-bit whole numbers, round(w 2^s) with V 2^s <= 2^62, from
// exponentials in 64 bits: their sums do not depend on the order of the
// additions, so a draw is the same every time, and where a border falls between
// two tokens is off by less than V 2^-(s + 1) of the largest weight (1.8e-9
// at V = 128256, s = 45, if all roundings went one way; 1e-11 in earnest).  In 32 bits one
// draw in a hundred from a flat distribution over 128256 tokens would take a
// neighbour.
#include "programmatic.cuh"

#include <cooperative_groups.h>

namespace t1 {
namespace rows {

namespace cg = cooperative_groups;

using bf16_t = __nv_bfloat16;
using u64 = unsigned long long;

constexpr int kThreads = 256;     // of scan_list, and of finish behind it
constexpr int kBinThreads = 512;  // of scan_bins, and of finish behind it
constexpr int kBatch = 512;       // columns that a warp of finish looks at at a time
constexpr int kMostCtas = 8;      // of a cluster
constexpr int kMostColumns = 96;  // of a thread of scan_bins: what fits in shared memory next to the rest
constexpr int kStretch = 8192;    // columns of a CTA of scan_list
constexpr int kParts = 4;         // of a thread's columns there
constexpr int kMostList = 512;    // tokens of `top`
constexpr int kMostFirst = kParts * kThreads;  // tokens that a list can be asked for
constexpr int kListSlots = 2048;  // tokens that finish orders
constexpr int kRankSlots = 128;   // up to so many by counting
constexpr int kBinCap = 2048;     // tokens that a CTA of scan_bins lists
constexpr int kDigits = 256;
constexpr int kBins = 256;        // of distances, and parts of a bin of weights
constexpr int kWeightBins = 512;  // of scan_bins
constexpr int kBinSteps = 8;
constexpr int kExps = 128;        // steps of an octave in the table of exponentials

// What scan_bins has found out about a row.
struct RowState {
  float m;
  int bin;    // where top_p is reached; -1: in none, or not asked
  u64 total;  // weight of all tokens
  u64 need;   // weight of the kept ones of that bin that reaches top_p
};

struct Params {
  const void* logits;
  int64_t ld;
  int rows, V;
  bool aligned;    // rows begin on 16 bytes
  float tau;
  float scale;     // 1 / tau
  float scale2;    // log2(e) / tau
  double steps;    // kExps log2(e) / tau
  int first;       // top: k; sample: top_k, 0 for all
  float* logp;     // [rows, k]; sample: [rows]
  int64_t* ids;    // [rows, k]; sample: [rows]
  // sample
  const float* u;
  double top_p;      // 1: all
  double log_min_p;  // in units of 1 / kExps of a factor of two; -inf: all
  int one;           // s: the largest logit's weight is 2^s
  // from the scan
  bool by_list;
  int segments;      // stretches or CTAs of a row
  int per_segment;   // their columns
  int cap;           // tokens that a segment lists at most
  int rank;          // r of scan_list
  float4* part;      // [rows][segments] scan_list: largest, sum of weights, bound
  int* counts;       // [rows][segments] tokens listed; above cap: not all
  u64* lists;        // [rows][segments][cap]
  RowState* states;  // [rows] scan_bins
  u64* weights;      // [rows][segments] scan_bins: kept without top_p, above the bin with it
  // what was allocated, for the bounds-checked build
  int64_t elements;      // of the logits, from the first row's first to the last row's last
  int64_t outputs;       // of ids and logp
  int64_t all_segments;  // of part, counts and weights
  int64_t list_slots;    // of lists
};

__device__ __forceinline__ unsigned held_bytes() {
  unsigned n;
  asm("mov.u32 %0, %%dynamic_smem_size;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ float logit(const float* p) { return __ldg(p); }
__device__ __forceinline__ float logit(const bf16_t* p) {
  return __bfloat162float(__ushort_as_bfloat16(__ldg(reinterpret_cast<const unsigned short*>(p))));
}
__device__ __forceinline__ float held_logit(const float* p) { return *p; }
__device__ __forceinline__ float held_logit(const bf16_t* p) { return __bfloat162float(*p); }
// Four neighbours in shared memory.
__device__ __forceinline__ float4 held_quad(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 held_quad(const bf16_t* p) {
  const uint2 q = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(q.x << 16), __uint_as_float(q.x & 0xffff0000u), __uint_as_float(q.y << 16),
                     __uint_as_float(q.y & 0xffff0000u));
}

// A warp's `all` logits of a row from column col0 on to shared memory, -inf behind the row's last.
template <typename T>
__device__ __forceinline__ void fetch(const Params& p, T* held, int at, int row, int col0, int all, int lane) {
  constexpr int kVec = 16 / sizeof(T);
  const int64_t first = row * p.ld + col0;
  const T* from = static_cast<const T*>(p.logits) + first;
  T* to = held + at;
  int cols = max(0, min(all, p.V - col0));
  if (T1_OOB((at + all) * sizeof(T) - 1, held_bytes())) return;
  if (cols > 0 && T1_OOB(first + cols - 1, p.elements)) cols = 0;
  const int vecs = p.aligned ? cols / kVec : 0;
  for (int i = lane; i < vecs; i += 32)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_at(to + kVec * i)), "l"(from + kVec * i) : "memory");
#pragma unroll 8
  for (int c = vecs * kVec + lane; c < cols; c += 32) {
    if (sizeof(T) == 4)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_at(to + c)), "l"(from + c) : "memory");
    else
      to[c] = from[c];
  }
  for (int c = cols + lane; c < all; c += 32) to[c] = static_cast<T>(-INFINITY);
}
__device__ __forceinline__ void fetched() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Larger logits have larger keys.
__device__ __forceinline__ unsigned key_of(float z) {
  const unsigned b = __float_as_uint(z);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
// The order of tokens as one number: larger ones come first.
__device__ __forceinline__ u64 place_of(float z, int column) {
  return static_cast<u64>(key_of(z + 0.f)) << 32 | ~static_cast<unsigned>(column);  // -0 is 0
}
__device__ __forceinline__ float logit_at(u64 place) { return logit_of(static_cast<unsigned>(place >> 32)); }
__device__ __forceinline__ int column_at(u64 place) { return static_cast<int>(~static_cast<unsigned>(place)); }

__device__ __forceinline__ bool is_token(float z) { return z > -INFINITY; }

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int LANES = 32, typename V>
__device__ __forceinline__ V warp_scan(V v, int lane) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) {
    const V up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
// Sum of the threads' values; every thread gets it, and the sum of the threads
// before it.
template <int WARPS, typename V>
__device__ __forceinline__ V block_scan(V v, V& before, V* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const V upto = warp_scan(v, lane);
  __syncthreads();
  if (lane == 31) red[warp] = upto;
  __syncthreads();
  const V of_warp = lane < WARPS ? red[lane] : V(0), of_warps = warp_scan<WARPS>(of_warp, lane);
  before = __shfl_sync(0xffffffffu, of_warps - of_warp, warp) + upto - v;
  return __shfl_sync(0xffffffffu, of_warps, WARPS - 1);
}

__device__ __forceinline__ float exp2f_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// u times the sum, rounded down; u of NaN is 0.
__device__ __forceinline__ u64 target_of(float u, u64 sum) {
  const double d = fmin(fmax(static_cast<double>(u), 0.0), 1.0 - 0x1p-53);
  return __umul64hi(sum, static_cast<u64>(d * 0x1p64));
}
// In 64-bit floating point, which gives what was meant where 0.9 of equal weights
// is a whole number of them.
__device__ __forceinline__ u64 share_of(double top_p, u64 sum) {
  return max(1ull, static_cast<u64>(top_p * static_cast<double>(sum)));
}

// Where the largest logit is infinite, or its neighbours lie far below it, it
// has all the weight.
__device__ __forceinline__ bool is_sharp(float m, float tau) { return !(fabsf(m) * 0x1p-23f <= 100.f * tau); }

// Distance of a logit from the largest one in steps of a sixteenth of its
// octave, 2^-8 to 2^8, and the least logit of a step (a little lower, for the
// rounding of the distance).
__device__ __forceinline__ int step_of(float from, float z) {
  const int s = static_cast<int>(__float_as_uint(z == from ? 0.f : from - z) >> 19) - (119 << 4);
  return min(max(s, 0), kBins - 1);
}
__device__ __forceinline__ float least_of(float from, int step) {
  return from - __uint_as_float(static_cast<unsigned>(step + 1 + (119 << 4)) << 19) * 1.000001f;
}

// 2^(j / kExps), by the block's threads; a barrier has to follow.
__device__ __forceinline__ void fill_exps(double* exps) {
  if (threadIdx.x < kExps) exps[threadIdx.x] = exp2(threadIdx.x / static_cast<double>(kExps));
}

// Weights of a row's tokens.
struct Weigher {
  float m, low;
  double m64, steps;
  bool sharp;
  int one;
  const double* exps;
  static constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: adding it leaves a whole number in the low bits

  // exp(-350) is no weight in any precision here: below, and NaN, counts as that
  __device__ __forceinline__ Weigher(const Params& p, float largest, const double* table)
      : m(largest), low(largest - 400.f * p.tau), m64(largest), steps(p.steps), sharp(is_sharp(largest, p.tau)), one(p.one), exps(table) {}
  // log2 of the weight, of 1 for m, in steps of 1 / kExps
  __device__ __forceinline__ double blunt_steps(float z) const { return (static_cast<double>(fmaxf(z, low)) - m64) * steps; }
  __device__ __forceinline__ double steps_of(float z) const { return sharp ? (z == m ? 0.0 : -4e4) : blunt_steps(z); }
  // 2^(x / kExps + s): a power from the table, the rest of it (|f| <= 1/2) by the series of the exponential function,
  // whose first term left out is below 5e-15; rounded to a whole number by the last addition
  __device__ __forceinline__ u64 weight_at(double x) const {
    constexpr double L = 0.6931471805599453 / kExps;
    const double y = x + kRound;
    const int j = __double2loint(y);
    const double f = x - (y - kRound);
    double e = fma(f, L * L * L * L / 24, L * L * L / 6);
    e = fma(e, f, L * L / 2);
    e = fma(e, f, L);
    e = fma(e, f, 1.0);
    const double base = exps[j & (kExps - 1)];
    const double scaled = __hiloint2double(__double2hiint(base) + (((j >> 7) + one) << 20), __double2loint(base));
    constexpr double kWhole = 4503599627370496.0;  // 2^52
    return __double_as_longlong(fma(e, scaled, kWhole)) - __double_as_longlong(kWhole);
  }
  __device__ __forceinline__ u64 weight(float z) const { return weight_at(steps_of(z)); }
  // Bins of 8 steps, and 256 parts of one.
  __device__ __forceinline__ static int bin_at(double x) { return -__double2loint(x + kRound) >> 3; }
  __device__ __forceinline__ static int part_at(double x, int bin) {
    return min(max(static_cast<int>((0.5 - x - kBinSteps * bin) * (kBins / kBinSteps)), 0), kBins - 1);
  }
};
static_assert(kBinSteps == 8, "bin_at: >> 3");
static_assert(kExps == 128, "weight_at: j >> 7");

// Bins of weights, 16 bits each: a bin of 2^16 tokens stays below 2^32.
template <int N>
__device__ __forceinline__ void add_to(unsigned (&bins)[3][N], int b, u64 w) {
  const unsigned lo = static_cast<unsigned>(w) & 0xffffu, mid = static_cast<unsigned>(w >> 16) & 0xffffu,
                 hi = static_cast<unsigned>(w >> 32);
  if (T1_OOB(b, N)) return;
  atomicAdd(&bins[0][b], lo);
  atomicAdd(&bins[1][b], mid);
  if (hi != 0) atomicAdd(&bins[2][b], hi);
}
template <int N>
__device__ __forceinline__ u64 bin_sum(const unsigned (&bins)[3][N], int b) {
  return bins[0][b] + (static_cast<u64>(bins[1][b]) << 16) + (static_cast<u64>(bins[2][b]) << 32);
}
static_assert(kBinThreads * kMostColumns <= 65536 && kMostCtas * kBinCap <= 65536, "add_to");

// =============================================================== scan by list
// A CTA takes a stretch of a row: its largest logit, the sum of its weights and
// the tokens that may be among the row's first ones.
struct ListShared {
  unsigned bins[kBins];
  float fred[32];
  int bin;
  unsigned listed;
};

// What a scan by list has found out about a stretch.
struct Scan {
  float m, sum, bound;  // largest logit, sum of weights; no token from `bound` on is missing in the list
  unsigned listed;      // above the list's length: not all
};

// The list is `cap` of the `slots` of `lists`, from list0 on.
template <typename T>
__device__ __forceinline__ Scan scan_stretch(const Params& p, int row, int segment, u64* lists, int64_t list0, int64_t slots,
                                             unsigned cap, ListShared& sh, T* held) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // a warp has 32 n columns in a row, a thread four of every 128
  const int n = p.per_segment / kThreads;
  const int col0 = segment * p.per_segment + warp * 32 * n;
  T* mine = held + warp * 32 * n;
  auto quad = [&](int i) { return held_quad(mine + 4 * (32 * i + lane)); };
  fetch(p, held, warp * 32 * n, row, col0, 32 * n, lane);
  sh.bins[tid] = 0;
  if (tid == 0) sh.listed = 0;
  fetched();
  __syncwarp();
  // the largest logits of the thread's parts (a NaN is never the larger of two)
  float part[kParts] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 8
  for (int i = 0; i < n / 4; ++i) {
    const float4 q = quad(i);
    part[0] = fmaxf(part[0], q.x);
    part[1] = fmaxf(part[1], q.y);
    part[2] = fmaxf(part[2], q.z);
    part[3] = fmaxf(part[3], q.w);
  }
  const float m = block_max(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), sh.fred);
  if (m == -INFINITY) return {m, 0.f, m, 0};
  // few tokens need few parts
  if (p.rank <= kThreads / 4) {
    const float own = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    if (is_token(own) && !T1_OOB(step_of(m, own), kBins)) atomicAdd(&sh.bins[step_of(m, own)], 1u);
  } else {
#pragma unroll
    for (int j = 0; j < kParts; ++j)
      if (is_token(part[j]) && !T1_OOB(step_of(m, part[j]), kBins)) atomicAdd(&sh.bins[step_of(m, part[j])], 1u);
  }
  __syncthreads();
  if (warp == 0) {
    int h[kBins / 32], own = 0, upto = 0, bin = -1;
#pragma unroll
    for (int j = 0; j < kBins / 32; ++j) own += h[j] = sh.bins[kBins / 32 * lane + j];
    upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += up;
    }
    upto -= own;
#pragma unroll
    for (int j = 0; j < kBins / 32; ++j) {
      if (upto < p.rank && upto + h[j] >= p.rank) bin = kBins / 32 * lane + j;
      upto += h[j];
    }
    bin = __reduce_max_sync(0xffffffffu, bin);
    if (lane == 0) sh.bin = bin;
  }
  __syncthreads();
  // where too few parts have a token, all tokens; where they lie too far from the largest, none: the list is given up
  const float bound = sh.bin < 0 ? -INFINITY : sh.bin < kBins - 1 ? least_of(m, sh.bin) : INFINITY;
  auto push = [&](float z, int column) {
    const unsigned to = atomicAdd(&sh.listed, 1u);
    if (to < cap && !T1_OOB(list0 + to, slots)) lists[list0 + to] = place_of(z, column);
  };
  float sum = 0.f;
  if (is_sharp(m, p.tau)) {
    for (int c = lane; c < 32 * n; c += 32) {
      const float z = held_logit(mine + c);
      sum += z == m;
      if (is_token(z) && z >= bound) push(z, col0 + c);
    }
  } else {
    // (z - m) / tau as one operation; what rounds off m / tau is the same for all, and made good in the end
    const float shift = -m * p.scale2, off = fmaf(m, p.scale2, shift);
    float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < n / 4; ++i) {
      const float4 q = quad(i);
      const float z[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) s4[j] += exp2f_fast(fmaf(z[j], p.scale2, shift));
      if (fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)) >= bound) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (is_token(z[j]) && z[j] >= bound) push(z[j], col0 + 4 * (32 * i + lane) + j);
      }
    }
    sum = ((s4[0] + s4[1]) + (s4[2] + s4[3])) * exp2f_fast(-off);
    if (!(sum == sum)) {  // NaN among them, which is no token
      sum = 0.f;
      for (int i = 0; i < n / 4; ++i) {
        const float4 q = quad(i);
        const float z[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += z[j] == z[j] ? exp2f_fast((z[j] - m) * p.scale2) : 0.f;
      }
    }
  }
  sum = block_sum(sum, sh.fred);
  return {m, sum, bound, bound == INFINITY ? cap + 1 : min(sh.listed, cap + 1)};
}

// =============================================================== scan by bins
struct BinShared {
  double exps[kExps];
  union {
    unsigned bins[3][kWeightBins];
    u64 sums[kWeightBins];  // then
  };
  u64 red[kBinThreads / 32];
  unsigned red32[kBinThreads / 32];
  float fred[32];
  // what every CTA of the cluster tells all others, once each
  float max_of[kMostCtas];
  u64 total_of[kMostCtas];
  int bin;
  u64 before64;
};

__device__ __forceinline__ void sync_all(cg::cluster_group& cluster) {
  if (cluster.num_blocks() == 1) __syncthreads();
  else cluster.sync();
}

// Every CTA's value to all of the cluster, in slots[rank]; one barrier.
template <typename V>
__device__ __forceinline__ void tell_all(cg::cluster_group& cluster, V* slots, V value) {
  const unsigned n = cluster.num_blocks();
  if (threadIdx.x < n && !T1_OOB(cluster.block_rank(), kMostCtas)) cluster.map_shared_rank(slots, threadIdx.x)[cluster.block_rank()] = value;
  sync_all(cluster);
}

// What a draw without top_k needs besides the sum of all weights.
enum BinMode : int { kAll = 0, kMinP = 1, kTopP = 2 };

template <typename T, int MODE>
__global__ void __launch_bounds__(kBinThreads, 3) scan_bins_kernel(const Params p) {
  __shared__ BinShared sh;
  extern __shared__ __align__(16) uint8_t held_raw[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / ctas;
  // a warp has 32 n columns in a row, a thread four of every 128
  const int n = p.per_segment / kBinThreads;
  const int warp_col0 = rank * p.per_segment + warp * 32 * n;
  T* mine = reinterpret_cast<T*>(held_raw) + warp * 32 * n;
  auto quad = [&](int i) { return held_quad(mine + 4 * (32 * i + lane)); };
  if (ctas > 1) tell_started();
  launch_dependents();
  wait_previous();
  fetch(p, reinterpret_cast<T*>(held_raw), warp * 32 * n, row, warp_col0, 32 * n, lane);
  for (int i = tid; i < 3 * kWeightBins; i += kBinThreads) sh.bins[0][i] = 0;
  fill_exps(sh.exps);
  fetched();
  __syncwarp();
  float m = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < n / 4; ++i) {
    const float4 q = quad(i);
    m = fmaxf(fmaxf(m, fmaxf(q.x, q.y)), fmaxf(q.z, q.w));
  }
  m = block_max(m, sh.fred);
  if (ctas > 1) wait_started();
  tell_all(cluster, sh.max_of, m);
  for (int r = 0; r < ctas; ++r) m = fmaxf(m, sh.max_of[r]);
  const int64_t at = static_cast<int64_t>(row) * p.segments + rank;
  // the row's state and the segment's numbers are there (by the whole cluster: its barriers stay together)
  if (T1_OOB(static_cast<int64_t>(row) * p.segments + ctas - 1, p.all_segments) || T1_OOB(row, p.rows) || T1_OOB(ctas - 1, kMostCtas)) return;
  const Weigher w(p, m, sh.exps);
  if (m == -INFINITY || w.sharp) {  // finish sees that
    if (rank == 0 && tid == 0) p.states[row] = {m, -1, 0, 0};
    if (tid == 0) p.counts[at] = 0;
    return;
  }

  u64 own = 0, kept = 0, before;  // with top_p: what lies below all bins
#pragma unroll 2
  for (int i = 0; i < n / 4; ++i) {
    const float4 q = quad(i);
    const float z[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double x = w.blunt_steps(z[j]);
      const u64 of = w.weight_at(x);
      if (MODE == kTopP) {
        const int b = Weigher::bin_at(x);
        if (b < kWeightBins) add_to(sh.bins, b, of);
        else own += of;
      } else {
        own += of;
        if (MODE == kMinP && x >= p.log_min_p) kept += of;
      }
    }
  }
  u64 my_bin = 0;
  if (MODE == kTopP) {
    __syncthreads();
    my_bin = bin_sum(sh.bins, tid);
    own += my_bin;
    __syncthreads();
    sh.sums[tid] = my_bin;
  }
  const u64 of_cta = block_scan<kBinThreads / 32>(own, before, sh.red);
  tell_all(cluster, sh.total_of, of_cta);
  u64 total = 0;
  for (int r = 0; r < ctas; ++r) total += sh.total_of[r];
  if (MODE != kTopP) {
    if (MODE == kMinP) kept = block_scan<kBinThreads / 32>(kept, before, sh.red);
    if (tid == 0) p.weights[at] = MODE == kMinP ? kept : of_cta;
    if (rank == 0 && tid == 0) p.states[row] = {m, -1, total, 0};
    return;
  }

  // the bin in which top_p is reached, of all CTAs' weights
  const u64 need = share_of(p.top_p, total);
  u64 here = 0;
  for (int r = 0; r < ctas; ++r) here += cluster.map_shared_rank(sh.sums, r)[tid];
  if (tid == 0) sh.bin = -1;
  block_scan<kBinThreads / 32>(here, before, sh.red);
  if (before < need && before + here >= need) {
    sh.bin = tid;
    sh.before64 = before;
  }
  sync_all(cluster);  // and nobody reads another's bins any more
  const int bin = sh.bin;
  if (rank == 0 && tid == 0) p.states[row] = {m, bin, total, need - (bin < 0 ? 0 : sh.before64)};
  if (bin < 0) return;
  // the CTA's weight above that bin, and its tokens in it
  const u64 above = block_scan<kBinThreads / 32>(tid < bin ? my_bin : 0ull, before, sh.red);
  if (tid == 0) p.weights[at] = above;
  auto column_of = [&](int k) { return 128 * (k / 4) + 4 * lane + k % 4; };  // of the warp's, the thread's k-th
  auto mine_at = [&](int k) { return held_logit(mine + column_of(k)); };
  // between which the bin's logits lie
  const float least = __double2float_rd(w.m64 - kBinSteps * (bin + 1.0) / p.steps), most = __double2float_ru(w.m64 - (kBinSteps * bin - 1.0) / p.steps);
  unsigned in_bin[kMostColumns / 32], count = 0;  // bit 4 i + j: of the thread's i-th four the j-th
#pragma unroll
  for (int b = 0; b < kMostColumns / 32; ++b) {
    in_bin[b] = 0;
#pragma unroll 4
    for (int i = 8 * b; i < min(n / 4, 8 * b + 8); ++i) {
      const float4 q = quad(i);
      const float z[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (z[j] >= least && z[j] <= most) in_bin[b] |= 1u << (4 * (i - 8 * b) + j);
    }
    // few of these lie beyond the bin after all
    for (unsigned left = in_bin[b]; left != 0; left &= left - 1) {
      const int k = __ffs(left) - 1;
      if (Weigher::bin_at(w.blunt_steps(mine_at(32 * b + k))) != bin) in_bin[b] &= ~(1u << k);
    }
    count += __popc(in_bin[b]);
  }
  unsigned to;
  const unsigned listed = block_scan<kBinThreads / 32>(count, to, sh.red32);
  if (tid == 0) p.counts[at] = static_cast<int>(min(listed, p.cap + 1u));
#pragma unroll
  for (int b = 0; b < kMostColumns / 32; ++b) {
    for (; in_bin[b] != 0; in_bin[b] &= in_bin[b] - 1, ++to) {
      const int k = 32 * b + __ffs(in_bin[b]) - 1;
      if (to < p.cap && !T1_OOB(at * p.cap + to, p.list_slots)) p.lists[at * p.cap + to] = place_of(mine_at(k), warp_col0 + column_of(k));
    }
  }
}

// ==================================================================== finish
struct FinishShared {
  double exps[kExps];
  u64 red[kBinThreads / 32];
  float fred[32];
  unsigned bins[3][kBins];
  u64 border[kBinThreads / 32];
  u64 kept_of[kMostCtas];
  union {
    u64 list[kListSlots];
    float kept[kBinThreads / 32][kBatch];  // of a warp's batch, in order
    unsigned hist[kDigits];
    u64 weights[kDigits];
  };
  int bin;
  unsigned listed, digit;
  u64 before64, found;
};

// Descending, slots a power of two.
template <int THREADS>
__device__ __forceinline__ void sort_list(u64* list, unsigned slots) {
  for (unsigned size = 2; size <= slots; size *= 2) {
    for (unsigned step = size / 2; step > 0; step /= 2) {
      __syncthreads();
      for (unsigned q = threadIdx.x; q < slots / 2; q += THREADS) {
        const unsigned i = 2 * q - (q & (step - 1)), j = i + step;
        const u64 a = list[i], b = list[j];
        if ((a < b) == ((i & size) == 0)) {
          list[i] = b;
          list[j] = a;
        }
      }
    }
  }
  __syncthreads();
}

// The same of `listed` tokens; kRankSlots or fewer by counting for each how many
// are larger, two threads to one.
template <int THREADS>
__device__ __forceinline__ void order_list(u64* list, unsigned listed) {
  if (listed <= kRankSlots) {
    __syncthreads();
    const unsigned i = threadIdx.x >> 1, part = threadIdx.x & 1;
    const u64 mine = i < listed ? list[i] : 0ull;
    unsigned larger = 0;
    if ((threadIdx.x & ~31u) < 2 * listed) {  // whole warps
#pragma unroll 8
      for (unsigned j = part; j < listed; j += 2) larger += list[j] > mine;
      larger += __shfl_xor_sync(0xffffffffu, larger, 1);
    }
    __syncthreads();
    if (i < listed && part == 0 && !T1_OOB(larger, kListSlots)) list[larger] = mine;
    __syncthreads();
    return;
  }
  unsigned slots = 1;
  while (slots < listed) slots *= 2;
  if (T1_OOB(slots - 1, kListSlots)) return;  // the same for all threads
  for (unsigned i = listed + threadIdx.x; i < slots; i += THREADS) list[i] = 0;
  sort_list<THREADS>(list, slots);
}
static_assert(kMostCtas <= kBinThreads / 32, "each_listed: a warp or more to a segment of scan_bins");
static_assert(2 * kRankSlots <= kThreads && kBins <= kThreads && kDigits <= kThreads, "a thread each");

// ALONE: the row is one stretch, which this CTA has scanned itself and whose
// list is in place.
template <typename T, bool TOP, int THREADS, bool ALONE>
__device__ __forceinline__ void finish_row(const Params& p, int row, FinishShared& sh, const Scan& scan) {
  constexpr int kWarps = THREADS / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row0 = row * p.ld;
  const T* src = static_cast<const T*>(p.logits) + row0;
  const int64_t seg0 = static_cast<int64_t>(row) * p.segments;
  constexpr int kLowest = sizeof(T) == 2 ? 16 : 0;  // key bits below are the same in all of a type's values
  const unsigned first = p.first;
  if (!TOP) fill_exps(sh.exps);
  for (int i = tid; !ALONE && i < 3 * kBins; i += THREADS) sh.bins[0][i] = 0;
  if (tid == 0) sh.listed = ALONE ? scan.listed : 0;

  // ---- the row's largest logit; by list also the sum of its weights
  float m = -INFINITY, sum = 0.f;
  bool complete = true;  // the lists are
  float bound = -INFINITY;
  if (ALONE) {
    m = scan.m;
    sum = scan.sum;
    bound = scan.bound;
    complete = scan.listed <= kListSlots;
  } else if (p.by_list) {
    for (int s = tid; s < p.segments; s += THREADS) {
      if (T1_OOB(seg0 + s, p.all_segments)) continue;
      const float4 of = p.part[seg0 + s];
      m = fmaxf(m, of.x);
      bound = fmaxf(bound, of.z);
      complete = complete && p.counts[seg0 + s] <= p.cap;
    }
    m = block_max(m, sh.fred);
    bound = block_max(bound, sh.fred);
    for (int s = tid; s < p.segments; s += THREADS) {
      if (T1_OOB(seg0 + s, p.all_segments)) continue;
      const float4 of = p.part[seg0 + s];
      sum += of.x == m ? of.y : of.y * exp2f_fast((of.x - m) * p.scale2);
    }
    sum = block_sum(sum, sh.fred);
  } else {
    if (!T1_OOB(row, p.rows)) m = p.states[row].m;
    for (int s = tid; s < p.segments; s += THREADS) complete = complete && !T1_OOB(seg0 + s, p.all_segments) && p.counts[seg0 + s] <= p.cap;
  }
  complete = __syncthreads_and(complete);
  if (m == -INFINITY) {
    for (int i = tid; i < (TOP ? p.first : 1); i += THREADS) {
      const int64_t at = static_cast<int64_t>(row) * (TOP ? p.first : 1) + i;
      if (T1_OOB(at, p.outputs)) continue;
      p.ids[at] = -1;
      p.logp[at] = 0.f;
    }
    return;
  }
  const Weigher w(p, m, sh.exps);
  float log_sum = logf(sum);  // of all weights
  auto log_p = [&](float z) { return (z == m ? 0.f : m == INFINITY ? -INFINITY : (z - m) * p.scale) - log_sum; };
  auto push = [&](u64 place) {
    const unsigned to = atomicAdd(&sh.listed, 1u);
    if (to < kListSlots) sh.list[to] = place;
  };
  auto write_draw = [&](int column, float z) {
    if (T1_OOB(column, p.V) || T1_OOB(row, p.outputs)) return;
    p.ids[row] = column;
    p.logp[row] = log_p(z);
  };
  // every token that the scan has listed
  const int warps_each = max(1, kWarps / p.segments);  // of a segment
  auto each_listed = [&](auto&& of) {
    for (int s = warp / warps_each; s < p.segments; s += kWarps / warps_each) {
      if (T1_OOB(seg0 + s, p.all_segments)) continue;
      const int n = p.counts[seg0 + s];
      const int64_t list0 = (seg0 + s) * p.cap;
      for (int i = warp % warps_each * 32 + lane; i < n; i += 32 * warps_each)
        if (!T1_OOB(list0 + i, p.list_slots)) of(p.lists[list0 + i]);
    }
  };
  // the thread's bin in which `need` is reached (-1: in none), and in sh.before64 what comes before
  auto reach = [&](u64 here, u64 need) {
    u64 before;
    if (tid == 0) sh.bin = -1;
    block_scan<kWarps>(here, before, sh.red);
    if (before < need && before + here >= need) {
      sh.bin = tid;
      sh.before64 = before;
    }
    __syncthreads();
    return sh.bin;
  };
  // the first `n` of the ordered list
  auto write_top = [&](unsigned n) {
    for (int i = tid; i < p.first; i += THREADS) {
      const bool in = i < static_cast<int>(n);
      const int64_t at = static_cast<int64_t>(row) * p.first + i;
      if (T1_OOB(at, p.outputs) || (in && (T1_OOB(i, kListSlots) || T1_OOB(column_at(sh.list[i]), p.V)))) continue;
      p.logp[at] = in ? log_p(logit_at(sh.list[i])) : 0.f;
      p.ids[at] = in ? column_at(sh.list[i]) : -1;
    }
  };

  // columns of the row, 16 at a time; a warp's in a row
  auto each_column = [&](int lo, int hi, auto&& of) {
    const int per = ((hi - lo + THREADS - 1) / THREADS) * 32;
    const int c0 = lo + warp * per, c1 = min(hi, c0 + per);
    for (int c = c0 + lane; c - lane < c1; c += 16 * 32) {
      float z[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) z[j] = c + 32 * j < c1 && !T1_OOB(row0 + c + 32 * j, p.elements) ? logit(src + c + 32 * j) : -INFINITY;
#pragma unroll
      for (int j = 0; j < 16; ++j) of(z[j] == z[j] ? z[j] + 0.f : -INFINITY, c + 32 * j);
    }
  };
  // ---- by list: the row's first tokens in order
  if (p.by_list && complete && !w.sharp) {
    bool enough = ALONE && bound > -INFINITY;  // not only all that there are
    if (!ALONE) {
      each_listed([&](u64 e) { if (!T1_OOB(step_of(m, logit_at(e)), kBins)) atomicAdd(&sh.bins[0][step_of(m, logit_at(e))], 1u); });
      __syncthreads();
      const int bin = reach(tid < kBins ? sh.bins[0][tid] : 0ull, first);
      enough = bin >= 0;
      each_listed([&](u64 e) {
        if (!enough || step_of(m, logit_at(e)) <= bin) push(e);
      });
      __syncthreads();
    }
    unsigned listed = sh.listed;
    if (listed <= kListSlots && (enough || bound == -INFINITY)) {
      order_list<THREADS>(sh.list, listed);
      if (!ALONE && enough) {
        // stretches that may have held back a token that comes before the last of these
        const float last = logit_at(sh.list[first - 1]);
        if (bound > last) {
          for (int s = 0; s < p.segments; ++s) {
            if (T1_OOB(seg0 + s, p.all_segments)) continue;
            const float of = p.part[seg0 + s].z;
            if (of <= last) continue;
            each_column(s * p.per_segment, min(p.V, (s + 1) * p.per_segment), [&](float z, int c) {
              if (z >= last && z < of) push(place_of(z, c));
            });
          }
          __syncthreads();
          listed = sh.listed;
          if (listed <= kListSlots) order_list<THREADS>(sh.list, listed);
        }
      }
      if (listed <= kListSlots) {
        if (TOP) return write_top(listed);
        // kept by top_p and min_p?  Four neighbours of the order a thread.
        constexpr int kPer = kMostFirst / THREADS;
        const unsigned have = min(first, listed);
        u64 e[kPer], of[kPer], own = 0, before;
        double x[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const unsigned i = kPer * tid + j;
          e[j] = i < have ? sh.list[i] : 0ull;
          x[j] = e[j] != 0 ? w.steps_of(logit_at(e[j])) : 0.0;
          of[j] = e[j] != 0 ? w.weight_at(x[j]) : 0ull;
          own += of[j];
        }
        const u64 need = share_of(p.top_p, block_scan<kWarps>(own, before, sh.red));
        unsigned kept = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const unsigned i = kPer * tid + j;
          const bool in = e[j] != 0 && (p.top_p == 1.0 || before < need) && x[j] >= p.log_min_p;
          before += of[j];
          kept += in;
          // by index, the lowest first: the complement of the column, then the logit's key
          if (i < have) sh.list[i] = in ? e[j] << 32 | e[j] >> 32 : 0ull;
        }
        kept = static_cast<unsigned>(block_scan<kWarps>(static_cast<u64>(kept), before, sh.red));
        order_list<THREADS>(sh.list, kept);  // the tokens kept are a prefix of the list
        own = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const unsigned i = kPer * tid + j;
          e[j] = i < kept ? sh.list[i] : 0ull;
          of[j] = e[j] != 0 ? w.weight(logit_of(static_cast<unsigned>(e[j]))) : 0ull;
          own += of[j];
        }
        const u64 target = target_of(p.u[row], block_scan<kWarps>(own, before, sh.red));
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (before <= target && target < before + of[j])
            write_draw(static_cast<int>(~static_cast<unsigned>(e[j] >> 32)), logit_of(static_cast<unsigned>(e[j])));
          before += of[j];
        }
        return;
      }
    }
    __syncthreads();
    if (tid == 0) sh.listed = 0;
    __syncthreads();
  }

  // ---- the last token kept
  float cut_logit = -INFINITY;  // all are
  int cut_column = 0;
  auto cut_at = [&](float z, int column) {
    cut_logit = z;
    cut_column = column;
  };
  auto in_cut = [&](float z, int column) { return is_token(z) && (z > cut_logit || (z == cut_logit && column <= cut_column)); };
  // A token of weight `target`, from the first of them on, of those kept in columns lo to hi.  A batch's kept tokens
  // are put together first: where one in ten is kept, weights are not worked out ten lanes in vain.
  const float min_logit = p.log_min_p > -INFINITY && !w.sharp ? __double2float_rd(w.m64 + (p.log_min_p - 1.0) / p.steps) : -INFINITY;
  auto is_kept = [&](float z, int column) {
    return in_cut(z, column) && z >= min_logit && (p.log_min_p == -INFINITY || w.steps_of(z) >= p.log_min_p);
  };
  // a batch from column c on, to c1: `put` gets its kept tokens' places in order; their number
  auto batch = [&](int c, int c1, auto&& put) {
    float z[kBatch / 32];
#pragma unroll
    for (int j = 0; j < kBatch / 32; ++j) z[j] = c + 32 * j + lane < c1 && !T1_OOB(row0 + c + 32 * j + lane, p.elements) ? logit(src + c + 32 * j + lane) : -INFINITY;
    int n = 0;
#pragma unroll
    for (int j = 0; j < kBatch / 32; ++j) {
      const bool in = is_kept(z[j], c + 32 * j + lane);
      const unsigned all = __ballot_sync(0xffffffffu, in);
      if (in) put(n + __popc(all & ((1u << lane) - 1)), z[j], c + 32 * j + lane);
      n += __popc(all);
    }
    __syncwarp();
    return n;
  };
  auto draw = [&](int lo, int hi, bool have_target, u64 target) {
    const int per = ((hi - lo + THREADS - 1) / THREADS) * 32;
    const int c0 = lo + warp * per, c1 = min(hi, c0 + per);
    u64 own = 0, before;
    for (int c = c0; c < c1; c += kBatch) {
      const int n = batch(c, c1, [&](int i, float z, int) {
        if (!T1_OOB(i, kBatch)) sh.kept[warp][i] = z;
      });
      for (int i = lane; i < n; i += 32) own += w.weight(sh.kept[warp][i]);
      __syncwarp();
    }
    const u64 of_warp = warp_sum64(own);
    const u64 all = block_scan<kWarps>(own, before, sh.red);
    before = __shfl_sync(0xffffffffu, before, 0);
    if (!have_target) target = target_of(p.u[row], all);
    if (target < before || target >= before + of_warp) return;
    // this warp has it, and the list's place to itself
    for (int c = c0; c < c1; c += kBatch) {
      const int n = batch(c, c1, [&](int i, float z, int column) {
        if (!T1_OOB(i, kListSlots)) sh.list[i] = place_of(z, column);
      });
      for (int i = lane; i - lane < n; i += 32) {
        const u64 e = i < n ? sh.list[i] : 0ull;
        const u64 upto = before + warp_scan(i < n ? w.weight(logit_at(e)) : 0ull, lane);
        const unsigned past = __ballot_sync(0xffffffffu, target < upto);
        if (past != 0) {
          if (lane == __ffs(past) - 1) write_draw(column_at(e), logit_at(e));
          return;
        }
        before = __shfl_sync(0xffffffffu, upto, 31);
      }
      __syncwarp();
    }
  };

  bool found = false;
  if (!TOP && !p.by_list && !w.sharp) log_sum = static_cast<float>(log(ldexp(static_cast<double>(p.states[row].total), -p.one)));
  if (!TOP && !p.by_list && !w.sharp && first == 0) {
    // ---- by bins
    const RowState st = p.states[row];
    int segment = -1;  // the draw's
    u64 of_segments = 0, before_segment = 0;
    if (p.top_p == 1.0) {
      found = true;
      if (tid < p.segments && !T1_OOB(seg0 + tid, p.all_segments) && !T1_OOB(tid, kMostCtas)) sh.kept_of[tid] = p.weights[seg0 + tid];
      __syncthreads();
      segment = 0;
    } else if (st.bin >= 0 && complete) {
      each_listed([&](u64 e) {
        const double x = w.blunt_steps(logit_at(e));
        add_to(sh.bins, Weigher::part_at(x, st.bin), w.weight_at(x));
      });
      __syncthreads();
      // the last token before which less than top_p has come is one of this part
      const int part = reach(tid < kBins ? bin_sum(sh.bins, tid) : 0ull, st.need);
      const u64 need = st.need - sh.before64;
      each_listed([&](u64 e) {
        if (Weigher::part_at(w.blunt_steps(logit_at(e)), st.bin) == part) push(e);
      });
      __syncthreads();
      const unsigned few = sh.listed;
      if (few <= kListSlots) {
        order_list<THREADS>(sh.list, few);
        constexpr int kPer = kListSlots / THREADS;
        u64 own = 0, before;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          const unsigned i = kPer * tid + j;
          own += i < few ? w.weight(logit_at(sh.list[i])) : 0ull;
        }
        block_scan<kWarps>(own, before, sh.red);
        if (before < need && before + own >= need) {
          for (unsigned i = kPer * tid; before < need; ++i) {
            before += w.weight(logit_at(sh.list[i]));
            sh.found = sh.list[i];
          }
        }
        __syncthreads();
        const u64 cut = sh.found;
        cut_at(logit_at(cut), column_at(cut));
        found = true;
        if (w.blunt_steps(cut_logit) >= p.log_min_p) {
          // min_p takes no more away: the segments' kept weights
          u64 kept = 0;
          each_listed([&](u64 e) {
            if (e >= cut) kept += w.weight(logit_at(e));
          });
          kept = warp_sum64(kept);
          if (lane == 0) sh.border[warp] = kept;
          __syncthreads();
          if (tid < p.segments && !T1_OOB(seg0 + tid, p.all_segments) && !T1_OOB((tid + 1) * warps_each - 1, kBinThreads / 32) &&
              !T1_OOB(tid, kMostCtas)) {
            kept = p.weights[seg0 + tid];
            for (int v = 0; v < warps_each; ++v) kept += sh.border[tid * warps_each + v];
            sh.kept_of[tid] = kept;
          }
          __syncthreads();
          segment = 0;
        }
      }
    }
    if (segment == 0) {
      for (int s = 0; s < p.segments; ++s) of_segments += sh.kept_of[s];
      const u64 target = target_of(p.u[row], of_segments);
      while (!T1_OOB(segment, p.segments) && target >= before_segment + sh.kept_of[segment]) before_segment += sh.kept_of[segment++];
      const int lo = segment * p.per_segment, hi = min(p.V, lo + p.per_segment);
      draw(lo, hi, true, target - before_segment);
      return;
    }
  }

  // ---- by digits
  // a key from its digits: the bits below are 0, of a negative logit 1
  auto with_low_bits = [](unsigned prefix) { return kLowest == 0 || prefix & 0x80000000u ? prefix : prefix | ((1u << kLowest) - 1); };
  // the n-th token with that key
  auto cut_at_tie = [&](unsigned key, unsigned n) {
    const float z = logit_of(key);
    unsigned here = 0;
    each_column(0, p.V, [&](float q, int) { here += __popc(__ballot_sync(0xffffffffu, q == z)); });
    u64 before;
    block_scan<kWarps>(static_cast<u64>(lane == 0 ? here : 0u), before, sh.red);
    unsigned tie = __shfl_sync(0xffffffffu, static_cast<unsigned>(before), 0);
    each_column(0, p.V, [&](float q, int c) {
      const unsigned all = __ballot_sync(0xffffffffu, q == z);
      if (q == z && tie + __popc(all & ((1u << lane) - 1)) + 1 == n) sh.digit = c;
      tie += __popc(all);
    });
    __syncthreads();
    cut_at(z, sh.digit);
    __syncthreads();
  };
  if (!TOP && !p.by_list && w.sharp) {
    u64 before, own = 0;
    each_column(0, p.V, [&](float z, int) { own += z == m; });
    log_sum = logf(static_cast<float>(block_scan<kWarps>(own, before, sh.red)));
  }
  unsigned have = 0;
  if (first != 0) {
    u64 before, count = 0;
    each_column(0, p.V, [&](float z, int) { count += is_token(z); });
    const unsigned tokens = static_cast<unsigned>(block_scan<kWarps>(count, before, sh.red));
    have = min(first, tokens);
    if (first < tokens) {
      unsigned need = first, prefix = 0, mask = 0;
      for (int shift = 24; shift >= kLowest; shift -= 8) {
        if (tid < kDigits) sh.hist[tid] = 0;
        __syncthreads();
        each_column(0, p.V, [&](float z, int) {
          const unsigned key = key_of(z);
          if (is_token(z) && (key & mask) == prefix) atomicAdd(&sh.hist[key >> shift & 255], 1u);
        });
        __syncthreads();
        const int digit = 255 - reach(tid < kDigits ? sh.hist[kDigits - 1 - tid] : 0ull, need);
        need -= static_cast<unsigned>(sh.before64);
        prefix |= static_cast<unsigned>(digit) << shift;
        mask |= 255u << shift;
        __syncthreads();
      }
      cut_at_tie(with_low_bits(prefix), need);
    }
  }
  if (TOP) {
    if (tid == 0) sh.listed = 0;
    __syncthreads();
    each_column(0, p.V, [&](float z, int c) {
      if (in_cut(z, c)) push(place_of(z, c));
    });
    __syncthreads();
    order_list<THREADS>(sh.list, have);
    return write_top(have);
  }
  if (p.top_p < 1.0 && !found) {
    u64 own = 0, before;
    each_column(0, p.V, [&](float z, int c) {
      if (in_cut(z, c)) own += w.weight(z);
    });
    u64 need = share_of(p.top_p, block_scan<kWarps>(own, before, sh.red));
    unsigned prefix = 0, mask = 0;
    for (int shift = 24; shift >= kLowest; shift -= 8) {
      if (tid < kDigits) sh.weights[tid] = 0;
      __syncthreads();
      each_column(0, p.V, [&](float z, int c) {
        const unsigned key = key_of(z);
        if (in_cut(z, c) && (key & mask) == prefix) atomicAdd(&sh.weights[key >> shift & 255], w.weight(z));
      });
      __syncthreads();
      const int digit = 255 - reach(tid < kDigits ? sh.weights[kDigits - 1 - tid] : 0ull, need);
      need -= sh.before64;
      prefix |= static_cast<unsigned>(digit) << shift;
      mask |= 255u << shift;
      __syncthreads();
    }
    const unsigned key = with_low_bits(prefix);
    const u64 one = w.weight(logit_of(key));
    cut_at_tie(key, static_cast<unsigned>((need + one - 1) / one));  // of these it takes so many to reach `need`
  }
  draw(0, p.V, false, 0);
}

template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS) finish_kernel(const Params p) {
  __shared__ FinishShared sh;
  launch_dependents();
  wait_previous();
  finish_row<T, TOP, THREADS, false>(p, blockIdx.x, sh, Scan{});
}

// `ALONE`: a row is one stretch, and the CTA that scans it finishes it too.
template <typename T, bool TOP, bool ALONE>
__global__ void __launch_bounds__(kThreads) scan_list_kernel(const Params p) {
  __shared__ ListShared sh;
  extern __shared__ __align__(16) uint8_t held_raw[];
  T* held = reinterpret_cast<T*>(held_raw);
  launch_dependents();
  wait_previous();
  if constexpr (ALONE) {
    __shared__ FinishShared rest;
    const Scan scan = scan_stretch<T>(p, blockIdx.x, 0, rest.list, 0, kListSlots, kListSlots, sh, held);
    __syncthreads();
    finish_row<T, TOP, kThreads, true>(p, blockIdx.x, rest, scan);
  } else {
    const int segment = blockIdx.x % p.segments;
    const Scan scan = scan_stretch<T>(p, blockIdx.x / p.segments, segment, p.lists, static_cast<int64_t>(blockIdx.x) * p.cap,
                                      p.list_slots, p.cap, sh, held);
    if (threadIdx.x == 0 && !T1_OOB(blockIdx.x, p.all_segments)) {
      p.part[blockIdx.x] = make_float4(scan.m, scan.sum, scan.bound, 0.f);
      p.counts[blockIdx.x] = static_cast<int>(scan.listed);
    }
  }
}

}  // namespace rows

// ================================================================ host side
T1_BOUNDS_READER(row_select)

static void check_rows(const torch::Tensor& logits, double temperature) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  TORCH_CHECK(logits.scalar_type() == torch::kFloat32 || logits.scalar_type() == torch::kBFloat16,
              "logits must be float32 or bfloat16, got ", logits.scalar_type());
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) > 0, "logits must be [T, V]");
  TORCH_CHECK(logits.size(1) == 1 || logits.stride(1) == 1, "logits must be row-major");
  TORCH_CHECK(logits.size(0) < 2 || logits.stride(0) >= 0, "logits must not have a negative stride");
  // log2(e) / temperature has to be finite (else a row of largest logit 0 has NaN where it meets 0), and the lowest logit
  // less 400 temperatures (Weigher) where it is not the lowest itself
  TORCH_CHECK(temperature >= 0x1p-126 && temperature <= 0x1p64, "temperature must lie in [2^-126, 2^64]");
}

constexpr int64_t kMostVocab = static_cast<int64_t>(rows::kMostCtas) * rows::kMostColumns * rows::kBinThreads;

// The scan's results, one buffer.
static torch::Tensor scan_space(rows::Params& p, const torch::Tensor& logits) {
  const int64_t segments = static_cast<int64_t>(p.rows) * p.segments;
  const auto piece = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
  const int64_t lists = piece(8 * segments * p.cap), part = piece(16 * segments);  // part, or the weights of scan_bins
  const int64_t states = piece(sizeof(rows::RowState) * static_cast<int64_t>(p.rows));
  auto buf = torch::empty({lists + part + states + 4 * segments}, logits.options().dtype(torch::kUInt8));
  uint8_t* base = buf.data_ptr<uint8_t>();
  p.lists = reinterpret_cast<rows::u64*>(base);
  p.part = reinterpret_cast<float4*>(base + lists);
  p.weights = reinterpret_cast<rows::u64*>(base + lists);
  p.states = reinterpret_cast<rows::RowState*>(base + lists + part);
  p.counts = reinterpret_cast<int*>(base + lists + part + states);
  p.all_segments = segments;
  p.list_slots = lists / 8;
  return buf;
}

template <typename T, bool TOP>
static void launch_rows(rows::Params& p, const torch::Tensor& logits) {
  constexpr const char* what = TOP ? "topk_logprobs" : "sample_tokens";
  const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  if (p.by_list) {
    p.segments = static_cast<int>(up(p.V, rows::kStretch));
    p.per_segment = static_cast<int>(up(up(p.V, p.segments), 4 * rows::kThreads) * 4 * rows::kThreads);
    // A stretch's share and three standard deviations and four more: where the first tokens lie anywhere, one row in
    // two thousand has a stretch that is looked at again (k = 64).  Each token more costs every stretch a store.
    const double share = static_cast<double>(p.first) / p.segments;
    p.rank = p.segments == 1 ? p.first : std::min(p.first, static_cast<int>(share + 3 * std::sqrt(share)) + 4);
    p.cap = std::min(p.per_segment, 2 * p.rank + 64);
    torch::Tensor space;
    if (p.segments > 1) space = scan_space(p, logits);
    const size_t held = sizeof(T) * p.per_segment;
    auto scan = p.segments == 1 ? rows::scan_list_kernel<T, TOP, true> : rows::scan_list_kernel<T, TOP, false>;
    static DeviceFlags configured[2];
    if (bool& done = configured[p.segments == 1].here(); !done) {
      T1_CHECK_CUDA(cudaFuncSetAttribute(scan, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(T) * rows::kStretch));
      done = true;
    }
    launch_after(what, scan, dim3(static_cast<unsigned>(p.rows) * p.segments), rows::kThreads, held, p);
    if (p.segments > 1) launch_after(what, rows::finish_kernel<T, TOP, rows::kThreads>, dim3(p.rows), rows::kThreads, 0, p);
    return;
  }
  if constexpr (!TOP) {
    // 32 columns a thread (64 KB a CTA, so that three CTAs share an SM) as long as 8 CTAs are enough; fewer while there
    // are SMs without a CTA
    p.segments = 1;
    while (p.segments < rows::kMostCtas &&
           (p.segments * 32 * rows::kBinThreads < p.V ||
            (2 * static_cast<int64_t>(p.rows) * p.segments <= num_sms() && p.segments * 8 * rows::kBinThreads < p.V)))
      p.segments *= 2;
    p.per_segment = static_cast<int>(up(up(p.V, p.segments), 4 * rows::kBinThreads) * 4 * rows::kBinThreads);
    p.cap = std::min({rows::kBinCap, p.per_segment, p.V});
    auto space = scan_space(p, logits);
    const int mode = p.top_p < 1.0 ? rows::kTopP : std::isfinite(p.log_min_p) ? rows::kMinP : rows::kAll;
    auto scan = mode == rows::kTopP  ? rows::scan_bins_kernel<T, rows::kTopP>
                : mode == rows::kMinP ? rows::scan_bins_kernel<T, rows::kMinP>
                                      : rows::scan_bins_kernel<T, rows::kAll>;
    static DeviceFlags configured[3];
    if (bool& done = configured[mode].here(); !done) {
      T1_CHECK_CUDA(cudaFuncSetAttribute(scan, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         sizeof(T) * rows::kMostColumns * rows::kBinThreads));
      done = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * p.segments);
    cfg.blockDim = dim3(rows::kBinThreads);
    cfg.dynamicSmemBytes = sizeof(T) * p.per_segment;
    cfg.stream = stream();
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.segments;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, scan, static_cast<const rows::Params>(p));
    TORCH_CHECK(e == cudaSuccess, what, " launch failed: ", cudaGetErrorString(e));
    count_launch();
    launch_after(what, rows::finish_kernel<T, TOP, rows::kBinThreads>, dim3(p.rows), rows::kBinThreads, 0, p);
  }
}

template <bool TOP>
static void run_rows(rows::Params& p, const torch::Tensor& logits, double temperature) {
  TORCH_CHECK(logits.size(1) <= kMostVocab, "at most ", std::to_string(kMostVocab), " tokens, got ", std::to_string(logits.size(1)));
  TORCH_CHECK(logits.size(0) < (1ll << 24), "at most 2^24 rows, got ", std::to_string(logits.size(0)));
  p.logits = logits.data_ptr();
  p.ld = logits.size(0) > 1 ? logits.stride(0) : 0;
  p.rows = static_cast<int>(logits.size(0));
  p.elements = logits.size(0) > 0 ? (logits.size(0) - 1) * p.ld + logits.size(1) : 0;
  p.V = static_cast<int>(logits.size(1));
  p.aligned = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.ld * logits.element_size() % 16 == 0;
  p.tau = static_cast<float>(temperature);
  p.scale = static_cast<float>(1.0 / temperature);
  p.scale2 = static_cast<float>(1.4426950408889634 / temperature);
  p.steps = rows::kExps * 1.4426950408889634 / temperature;
  if (p.rows == 0) return;
  if (logits.scalar_type() == torch::kFloat32) launch_rows<float, TOP>(p, logits);
  else launch_rows<rows::bf16_t, TOP>(p, logits);
}

// Returns (logp [T, k] fp32, ids [T, k] int64).
std::vector<torch::Tensor> topk_logprobs(torch::Tensor logits, int64_t k, double temperature) {
  check_rows(logits, temperature);
  TORCH_CHECK(k >= 1 && k <= std::min<int64_t>(rows::kMostList, logits.size(1)), "k must lie in [1, min(V, ",
              std::to_string(rows::kMostList), ")], got ", std::to_string(k));
  const c10::cuda::CUDAGuard guard(logits.device());
  auto logp = torch::empty({logits.size(0), k}, logits.options().dtype(torch::kFloat32));
  auto ids = torch::empty({logits.size(0), k}, logits.options().dtype(torch::kInt64));
  rows::Params p{};
  p.first = static_cast<int>(k);
  p.by_list = true;
  p.logp = logp.data_ptr<float>();
  p.ids = ids.data_ptr<int64_t>();
  p.outputs = ids.numel();
  run_rows<true>(p, logits, temperature);
  return {logp, ids};
}

// Returns (token [B] int64, logp [B] fp32).
std::vector<torch::Tensor> sample_tokens(torch::Tensor logits, torch::Tensor u, double temperature, int64_t top_k,
                                         double top_p, double min_p) {
  check_rows(logits, temperature);
  T1_CHECK_INPUT(u, torch::kFloat32);
  TORCH_CHECK(u.dim() == 1 && u.size(0) == logits.size(0), "u must have a number for every row");
  TORCH_CHECK(u.device() == logits.device(), "operands must be on one device");
  TORCH_CHECK(top_k >= 0, "top_k must not be negative");
  TORCH_CHECK(top_p > 0 && top_p <= 1, "top_p must lie in (0, 1]");
  TORCH_CHECK(min_p >= 0 && min_p <= 1, "min_p must lie in [0, 1]");
  const c10::cuda::CUDAGuard guard(logits.device());
  auto uc = u.contiguous();
  auto token = torch::empty({logits.size(0)}, logits.options().dtype(torch::kInt64));
  auto logp = torch::empty({logits.size(0)}, logits.options().dtype(torch::kFloat32));
  rows::Params p{};
  p.logp = logp.data_ptr<float>();
  p.ids = token.data_ptr<int64_t>();
  p.outputs = token.numel();
  p.u = uc.data_ptr<float>();
  p.first = static_cast<int>(top_k >= logits.size(1) ? 0 : top_k);
  p.by_list = p.first != 0 && p.first <= rows::kMostFirst;
  p.top_p = top_p;
  p.log_min_p = rows::kExps * std::log2(min_p);
  int bits = 0;
  while ((1ll << bits) < logits.size(1)) ++bits;
  p.one = std::min(51, 62 - bits);  // a weight fits the 52 bits of a double
  run_rows<false>(p, logits, temperature);
  return {token, logp};
}

}  // namespace t1
