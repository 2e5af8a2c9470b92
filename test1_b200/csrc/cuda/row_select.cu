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
// A cluster of CTAs holds one row in shared memory: one read of the logits, and
// every warp keeps to the same stretch of them in every pass.  Three ways to the
// cut, of which the first two look at most logits twice or three times:
//   list   the first n <= 512: no n tokens can all lie below the n-th largest
//          of the threads' own largest ones, which a histogram of their
//          distances from m finds.  What lies above (little more than n) goes to
//          the first CTA, which sorts it and does all the rest.
//   bins   top_p alone: weights added up by distance from m, 8 bins per factor
//          of two.  The tokens of the bin where top_p is reached go to the first
//          CTA, which finds the last one kept (by 256 parts of the bin, then by
//          order) and, since it has every CTA's weight above the bin too, the
//          CTA that the draw falls into.  The others are done.
//   digits where neither applies (more tokens are asked for, or too many are
//          equal): the threshold is found digit by digit, 8 bits at a time, of
//          the order-preserving integer of a logit.
//
// Weights are 64-bit whole numbers, round(w 2^s) with V 2^s <= 2^62, from
// exponentials in 64 bits: their sums do not depend on the order of the
// additions, so a draw is the same every time, and where a border falls between
// two tokens is off by less than V 2^-(s + 1) of the largest weight (4e-9 at
// V = 128256 if all roundings went one way; 1e-11 in earnest).  In 32 bits one
// draw in a hundred from a flat distribution over 128256 tokens would take a
// neighbour.
#include "common.cuh"

#include <cooperative_groups.h>

namespace t1 {
namespace rows {

namespace cg = cooperative_groups;

using bf16_t = __nv_bfloat16;
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMostCtas = 8;      // of a cluster
constexpr int kMostList = 512;    // tokens of `top`
constexpr int kListSlots = 2048;  // tokens that the first CTA takes from all
constexpr int kSortSlots = 1024;  // of bins: tokens of the last part
constexpr int kRankSlots = 128;   // up to so many by counting
constexpr int kMostColumns = 96;  // of a thread: what fits in shared memory next to the rest
constexpr int kDigits = 256;
constexpr int kBins = 256;
constexpr int kExps = 128;        // steps of an octave in the table of exponentials

struct Params {
  const void* logits;
  int64_t ld;
  int rows, V;
  int per_thread;  // columns
  bool aligned;    // rows begin on 16 bytes
  float tau;
  float scale;     // 1 / tau
  float scale2;    // log2(e) / tau
  double steps;    // kExps log2(e) / tau
  // top
  int k;
  float* logp;     // [rows, k]; sample: [rows]
  int64_t* ids;    // [rows, k]; sample: [rows]
  // sample
  const float* u;
  int top_k;         // 0: all
  double top_p;      // 1: all
  double log_min_p;  // in units of 1 / kExps of a factor of two; -inf: all
  int one;           // s: the largest logit's weight is 2^s
};

__device__ __forceinline__ uint32_t smem_at(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// Logits from..from + n to shared memory as fp32, by one warp.
__device__ __forceinline__ void fetch(float* to, const float* from, int n, bool aligned, int lane) {
  if (aligned) {
    const int vecs = n / 4;
    for (int i = lane; i < vecs; i += 32)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_at(to + 4 * i)), "l"(from + 4 * i) : "memory");
    to += 4 * vecs;
    from += 4 * vecs;
    n -= 4 * vecs;
  }
  for (int i = lane; i < n; i += 32)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_at(to + i)), "l"(from + i) : "memory");
}
__device__ __forceinline__ void fetch(float* to, const bf16_t* from, int n, bool aligned, int lane) {
  if (aligned) {
    const int vecs = n / 8;
#pragma unroll 4
    for (int i = lane; i < vecs; i += 32) {
      float f[8];
      load8(from + 8 * i, f);
      reinterpret_cast<float4*>(to)[2 * i] = make_float4(f[0], f[1], f[2], f[3]);
      reinterpret_cast<float4*>(to)[2 * i + 1] = make_float4(f[4], f[5], f[6], f[7]);
    }
    to += 8 * vecs;
    from += 8 * vecs;
    n -= 8 * vecs;
  }
#pragma unroll 8
  for (int i = lane; i < n; i += 32)
    to[i] = __bfloat162float(__ushort_as_bfloat16(__ldcs(reinterpret_cast<const unsigned short*>(from + i))));
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
__device__ __forceinline__ unsigned long long place_of(float z, int column) {
  return static_cast<unsigned long long>(key_of(z)) << 32 | ~static_cast<unsigned>(column);
}
__device__ __forceinline__ float logit_at(unsigned long long place) { return logit_of(static_cast<unsigned>(place >> 32)); }
__device__ __forceinline__ int column_at(unsigned long long place) { return static_cast<int>(~static_cast<unsigned>(place)); }

__device__ __forceinline__ bool is_token(float z) { return z > -INFINITY; }

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ unsigned long long warp_scan64(unsigned long long v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

struct Shared {
  double exps[kExps];              // 2^(j / 128)
  unsigned long long red[kWarps];
  unsigned bins[2][3][kBins];      // counts; of weights 16 bits each; the second of a bin's parts
  unsigned long long border[kWarps][kMostCtas];
  union {
    struct {
      unsigned hist[2][kDigits];
      unsigned long long weights[2][kDigits];
    };
    unsigned long long list[kListSlots];  // of the first CTA
    unsigned long long cells[32][33];     // weights of the warp that holds the drawn token
  };
  // what every CTA of the cluster tells all others, once each
  float max_of[kMostCtas];
  float sum_of[kMostCtas];
  unsigned count_of[kMostCtas], ties_of[kMostCtas];
  unsigned long long total_of[kMostCtas], kept_of[kMostCtas], cut_of[kMostCtas], above_of[kMostCtas];
  // what the first CTA finds
  unsigned long long found_cut, found_before, found_total;
  int found_cta;
  // where a threshold falls
  unsigned digit, before32;
  int bin;
  unsigned long long before64;
  unsigned listed;
};

__device__ __forceinline__ float exp2f_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// u times the sum, rounded down; u of NaN is 0.
__device__ __forceinline__ unsigned long long target_of(float u, unsigned long long sum) {
  const double d = fmin(fmax(static_cast<double>(u), 0.0), 1.0 - 0x1p-53);
  return __umul64hi(sum, static_cast<unsigned long long>(d * 0x1p64));
}

__device__ __forceinline__ void sync_all(cg::cluster_group& cluster) {
  if (cluster.num_blocks() == 1) __syncthreads();
  else cluster.sync();
}

// Every CTA's value to all of the cluster, in slots[rank]; one barrier.
template <typename V>
__device__ __forceinline__ void tell_all(cg::cluster_group& cluster, V* slots, V value) {
  const unsigned n = cluster.num_blocks();
  if (threadIdx.x < n) cluster.map_shared_rank(slots, threadIdx.x)[cluster.block_rank()] = value;
  sync_all(cluster);
}

// Sum of the threads' values; every thread gets it, and the sum of the threads
// before it.
__device__ __forceinline__ unsigned long long block_scan64(unsigned long long v, unsigned long long& before,
                                                           unsigned long long* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned long long upto = warp_scan64(v, lane);
  __syncthreads();
  if (lane == 31) red[warp] = upto;
  __syncthreads();
  unsigned long long sum = 0, of_warps = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) of_warps = sum;
    sum += red[w];
  }
  before = of_warps + upto - v;
  return sum;
}

// Descending, slots a power of two.
__device__ __forceinline__ void sort_list(unsigned long long* list, unsigned slots) {
  for (unsigned size = 2; size <= slots; size *= 2) {
    for (unsigned step = size / 2; step > 0; step /= 2) {
      __syncthreads();
      for (unsigned q = threadIdx.x; q < slots / 2; q += kThreads) {
        const unsigned i = 2 * q - (q & (step - 1)), j = i + step;
        const unsigned long long a = list[i], b = list[j];
        if ((a < b) == ((i & size) == 0)) {
          list[i] = b;
          list[j] = a;
        }
      }
    }
  }
  __syncthreads();
}

// The same; kRankSlots or fewer by counting for each how many are larger, four
// threads to one.  Places differ, except for the zeros that fill the list up.
__device__ __forceinline__ void order_list(unsigned long long* list, unsigned listed) {
  if (listed <= kRankSlots) {
    __syncthreads();
    const unsigned i = threadIdx.x >> 2, part = threadIdx.x & 3;
    const unsigned long long mine = i < listed ? list[i] : 0ull;
    unsigned larger = 0;
    if ((threadIdx.x & ~31u) < 4 * listed) {  // whole warps
#pragma unroll 4
      for (unsigned j = part; j < listed; j += 4) larger += list[j] > mine;
      larger += __shfl_xor_sync(0xffffffffu, larger, 1);
      larger += __shfl_xor_sync(0xffffffffu, larger, 2);
    }
    __syncthreads();
    if (i < listed && part == 0) list[larger] = mine;
    __syncthreads();
    return;
  }
  unsigned slots = 1;
  while (slots < listed) slots *= 2;
  for (unsigned i = listed + threadIdx.x; i < slots; i += kThreads) list[i] = 0;
  sort_list(list, slots);
}

// A prefix of the order: all tokens of a larger key, and the first `ties` of
// those that have it.
struct Cut {
  unsigned key;
  unsigned ties;
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 2) rows_kernel(const Params p) {
  __shared__ Shared sh;
  __shared__ float red[32];
  extern __shared__ __align__(16) float held[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / ctas;
  // a warp has 32 n columns in a row, n a multiple of 4.  A thread has every 32nd of them, v[32 i], or, where only
  // sums count, four at a time, quads[32 i]
  const int n = p.per_thread;
  const int warp_col0 = (rank * kWarps + warp) * 32 * n, col0 = warp_col0 + lane;
  float* v = held + warp * 32 * n + lane;
  const float4* quads = reinterpret_cast<const float4*>(held + warp * 32 * n) + lane;
  constexpr int kLowest = sizeof(T) == 2 ? 16 : 0;  // key bits below are the same in all of a type's values
  if (T1_OOB(row, p.rows)) return;

  {
    const int cols = max(0, min(32 * n, p.V - warp_col0));
    fetch(held + warp * 32 * n, static_cast<const T*>(p.logits) + row * p.ld + warp_col0, cols, p.aligned, lane);
    for (int c = cols + lane; c < 32 * n; c += 32) held[warp * 32 * n + c] = -INFINITY;
  }
  for (int i = tid; i < 6 * kBins; i += kThreads) sh.bins[0][0][i] = 0;
  if (tid == 0) sh.listed = 0;
  if (!TOP && tid < kExps) sh.exps[tid] = exp2(tid / static_cast<double>(kExps));
  fetched();
  __syncwarp();
  // ---- largest logit (a NaN is never the larger of two)
  float own_max = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < n / 4; ++i) {
    const float4 q = quads[32 * i];
    own_max = fmaxf(fmaxf(own_max, fmaxf(q.x, q.y)), fmaxf(q.z, q.w));
  }
  float m = block_max(own_max, red);
  // A token to the first CTA's list.
  unsigned* const list_length = cluster.map_shared_rank(&sh.listed, 0);
  unsigned long long* const first_list = cluster.map_shared_rank(sh.list, 0);
  auto push = [&](float z, int column) {
    const unsigned at = atomicAdd(list_length, 1u);
    if (at < kListSlots) first_list[at] = place_of(z + 0.f, column);  // -0 is 0
  };
  // Distance from a largest logit in steps of a sixteenth of its octave, 2^-8 to 2^8, and the least logit of a step (a
  // little lower, for the rounding of the distance).
  auto step_of = [](float from, float z) {
    const int s = static_cast<int>(__float_as_uint(from - z) >> 19) - (119 << 4);
    return min(max(s, 0), kBins - 1);
  };
  auto least_of = [](float from, int step) {
    return from - __uint_as_float(static_cast<unsigned>(step + 1 + (119 << 4)) << 19) * 1.000001f;
  };
  // Sum of exp((z - from) / tau) over this CTA's logits, and the tokens from `bound` on to the list.  Where `from` is
  // infinite, or its neighbours lie far below it, it has all the weight.
  auto is_sharp = [&](float from) { return !(fabsf(from) * 0x1p-23f <= 100.f * p.tau); };
  auto sum_and_push = [&](float from, float bound) {
    if (is_sharp(from)) {
      float sum = 0.f;
      for (int i = 0; i < n; ++i) sum += v[32 * i] == from;
      if (bound < INFINITY)
        for (int i = 0; i < n; ++i)
          if (is_token(v[32 * i]) && v[32 * i] >= bound) push(v[32 * i], col0 + 32 * i);
      return block_sum(sum, red);
    }
    const float low = from - 400.f * p.tau;  // exp(-350) is no weight here: below, and NaN, counts as that
    float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < n / 4; ++i) {
      const float4 q = quads[32 * i];
      const float z[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) s4[j] += exp2f_fast((fmaxf(z[j], low) - from) * p.scale2);
      if (fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)) >= bound) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (is_token(z[j]) && z[j] >= bound) push(z[j], warp_col0 + 4 * (32 * i + lane) + j);
      }
    }
    return block_sum((s4[0] + s4[1]) + (s4[2] + s4[3]), red);
  };
  // A bin of weights.
  auto bin_sum = [](const unsigned* bins, int b) {
    return bins[b] + (static_cast<unsigned long long>(bins[kBins + b]) << 16) + (static_cast<unsigned long long>(bins[2 * kBins + b]) << 32);
  };
  // The bin in which `need` is reached (-1: in none) of the first `of` CTAs' bins, and in sh.before64 what comes before.
  auto reach = [&](unsigned (*bins)[kBins], bool weights, unsigned long long need, int of) {
    unsigned long long here = 0, before;
    if (tid < kBins) {
      for (int r = 0; r < of; ++r) {
        const unsigned* b = cluster.map_shared_rank(&bins[0][0], r);
        here += weights ? bin_sum(b, tid) : b[tid];
      }
    }
    if (tid == 0) sh.bin = -1;
    block_scan64(here, before, sh.red);
    if (before < need && before + here >= need) {
      sh.bin = tid;
      sh.before64 = before;
    }
    __syncthreads();
    return sh.bin;
  };

  const unsigned first = TOP ? p.k : p.top_k;
  float log_sum = 0.f;  // log of the sum of all weights
  tell_all(cluster, sh.max_of, m);
  for (int r = 0; r < ctas; ++r) m = fmaxf(m, sh.max_of[r]);
  // m is the row's largest from here on
  if (m == -INFINITY) {
    if (rank != 0) return;
    for (int i = tid; i < (TOP ? p.k : 1); i += kThreads) {
      p.ids[static_cast<int64_t>(row) * (TOP ? p.k : 1) + i] = -1;
      p.logp[static_cast<int64_t>(row) * (TOP ? p.k : 1) + i] = 0.f;
    }
    return;
  }
  const bool sharp = is_sharp(m);
  if (!TOP && sharp) {
    for (int i = 0; i < n; ++i) v[32 * i] = v[32 * i] == m ? 0.f : -INFINITY;
    own_max = own_max == m ? 0.f : -INFINITY;
    m = 0.f;
    __syncwarp();
  }
  const float low = m - 400.f * p.tau;
  auto log_p = [&](float z) {
    return (z == m ? 0.f : m == INFINITY ? -INFINITY : (z - m) * p.scale) - log_sum;
  };

  const double m64 = m;
  // log2 of the weight, of 1 for m, in steps of 1 / kExps
  auto steps_of = [&](float z) { return (static_cast<double>(fmaxf(z, low)) - m64) * p.steps; };
  // 2^(x / kExps + s): a power from the table, the rest of it (|f| <= 1/2) by the series of the exponential function,
  // whose first term left out is below 5e-15; rounded to a whole number by the last addition
  constexpr double kRound = 6755399441055744.0;  // 1.5 2^52: adding it leaves a whole number in the low bits
  auto weight_at = [&](double x) -> unsigned long long {
    constexpr double L = 0.6931471805599453 / kExps;
    const double y = x + kRound;
    const int j = __double2loint(y);
    const double f = x - (y - kRound);
    double e = fma(f, L * L * L * L / 24, L * L * L / 6);
    e = fma(e, f, L * L / 2);
    e = fma(e, f, L);
    e = fma(e, f, 1.0);
    const double base = sh.exps[j & (kExps - 1)];
    const double scaled = __hiloint2double(__double2hiint(base) + (((j >> 7) + p.one) << 20), __double2loint(base));
    constexpr double kWhole = 4503599627370496.0;  // 2^52
    return __double_as_longlong(fma(e, scaled, kWhole)) - __double_as_longlong(kWhole);
  };
  static_assert(kExps == 128, "j >> 7");
  auto weight = [&](float z) { return weight_at(steps_of(z)); };
  // Bins of 16 steps of a weight's logarithm, and 256 parts of one.
  auto bin_at = [&](double x) { return -__double2loint(x + kRound) >> 4; };
  auto part_at = [&](double x, int bin) { return min(max(static_cast<int>((0.5 - x - 16 * bin) * 16.0), 0), kBins - 1); };
  auto add_to = [](unsigned (*bins)[kBins], int b, unsigned long long w) {
    const unsigned lo = static_cast<unsigned>(w) & 0xffffu, mid = static_cast<unsigned>(w >> 16) & 0xffffu,
                   hi = static_cast<unsigned>(w >> 32);
    atomicAdd(&bins[0][b], lo);
    atomicAdd(&bins[1][b], mid);
    if (hi != 0) atomicAdd(&bins[2][b], hi);
  };
  unsigned long long total = 0, own = 0;  // own: the thread's kept weight
  unsigned long long before_cta = 0;
  bool alone = false;                     // the other CTAs have left
  bool done = false;                      // the cut is found
  // with done: the last token kept
  float cut_logit = -INFINITY;
  int cut_column = 0;

  if (TOP || first != 0) {
    // ---- list
    const bool by_list = !sharp && first <= kThreads;
    float bound = INFINITY;
    if (by_list) {
      if (is_token(own_max)) atomicAdd(&sh.bins[0][0][step_of(m, own_max)], 1u);
      sync_all(cluster);
      const int bin = reach(sh.bins[0], false, first, ctas);
      if (bin >= 0 && bin < kBins - 1) bound = least_of(m, bin);
    }
    tell_all(cluster, sh.sum_of, sum_and_push(m, bound));
    float sum = 0.f;
    for (int r = 0; r < ctas; ++r) sum += sh.sum_of[r];
    log_sum = logf(sum);
    const unsigned listed = *list_length;
    if (bound < INFINITY && listed <= kListSlots) {
      if (rank != 0) return;  // the first CTA waits for that before it leaves
      order_list(sh.list, listed);
      if (TOP) {
        for (int i = tid; i < p.k; i += kThreads) {
          const bool in = i < static_cast<int>(listed);  // of fewer tokens than k all are listed
          const int64_t at = static_cast<int64_t>(row) * p.k + i;
          p.logp[at] = in ? log_p(logit_at(sh.list[i])) : 0.f;
          p.ids[at] = in ? column_at(sh.list[i]) : -1;
        }
      } else {
        // kept by top_p and min_p?
        unsigned long long before, e = tid < static_cast<int>(min(first, listed)) ? sh.list[tid] : 0ull;
        const double x = e != 0 ? steps_of(logit_at(e)) : 0.0;
        const unsigned long long w = e != 0 ? weight_at(x) : 0ull;
        const unsigned long long sum64 = block_scan64(w, before, sh.red);
        const unsigned long long need = max(1ull, static_cast<unsigned long long>(p.top_p * static_cast<double>(sum64)));
        const bool in = e != 0 && (p.top_p == 1.0 || before < need) && x >= p.log_min_p;
        // by index, the lowest first: the complement of the column, then the logit's key
        if (tid < static_cast<int>(first)) sh.list[tid] = in ? e << 32 | e >> 32 : 0ull;
        const unsigned kept = __syncthreads_count(in);
        // the tokens kept are a prefix of the list
        order_list(sh.list, kept);
        e = tid < static_cast<int>(kept) ? sh.list[tid] : 0ull;
        const float z = logit_of(static_cast<unsigned>(e));
        const unsigned long long w2 = e != 0 ? weight_at(steps_of(z)) : 0ull;
        const unsigned long long all = block_scan64(w2, before, sh.red);
        const unsigned long long target = target_of(p.u[row], all);
        if (before <= target && target < before + w2) {
          p.ids[row] = static_cast<int>(~static_cast<unsigned>(e >> 32));
          p.logp[row] = log_p(z);
        }
      }
      sync_all(cluster);
      return;
    }
  } else {
    // ---- bins
    const bool by_bins = p.top_p < 1.0;
#pragma unroll 2
    for (int i = 0; i < n / 4; ++i) {
      const float4 q = quads[32 * i];
      const float z[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double x = steps_of(z[j]);
        const unsigned long long w = weight_at(x);
        own += w;
        if (by_bins) {
          const int b = bin_at(x);
          if (b < kBins) add_to(sh.bins[0], b, w);
        }
      }
    }
    unsigned long long before;
    tell_all(cluster, sh.total_of, block_scan64(own, before, sh.red));
    for (int r = 0; r < ctas; ++r) total += sh.total_of[r];
    log_sum = static_cast<float>(log(ldexp(static_cast<double>(total), -p.one)));
    if (by_bins) {
      unsigned long long need = max(1ull, static_cast<unsigned long long>(p.top_p * static_cast<double>(total)));
      const int bin = reach(sh.bins[0], true, need, ctas);
      if (bin >= 0) {
        need -= sh.before64;
        // the bin's logits lie between these
        const float least = __double2float_rd(m64 - 16.0 * (bin + 1) / p.steps), most = __double2float_ru(m64 - (16.0 * bin - 1) / p.steps);
        // the CTA's weight above the bin, and its tokens in the bin
        const unsigned long long above = block_scan64(tid < bin ? bin_sum(sh.bins[0][0], tid) : 0ull, before, sh.red);
        if (tid == 0) cluster.map_shared_rank(sh.above_of, 0)[rank] = above;
        unsigned in_bin[kMostColumns / 32], mine = 0;
#pragma unroll
        for (int b = 0; b < kMostColumns / 32; ++b) {
          in_bin[b] = 0;
#pragma unroll 8
          for (int i = 32 * b; i < min(n, 32 * b + 32); ++i) {
            const float z = v[32 * i];
            if (z >= least && z <= most && bin_at(steps_of(z)) == bin) in_bin[b] |= 1u << (i - 32 * b);
          }
          mine += __popc(in_bin[b]);
        }
        const unsigned of_cta = static_cast<unsigned>(block_scan64(mine, before, sh.red));
        if (tid == 0) sh.digit = of_cta == 0 ? 0 : atomicAdd(list_length, of_cta);
        __syncthreads();
        unsigned at = sh.digit + static_cast<unsigned>(before);
#pragma unroll
        for (int b = 0; b < kMostColumns / 32; ++b) {
          for (; in_bin[b] != 0; in_bin[b] &= in_bin[b] - 1, ++at) {
            const int i = 32 * b + __ffs(in_bin[b]) - 1;
            if (at < kListSlots) first_list[at] = place_of(v[32 * i] + 0.f, col0 + 32 * i);  // -0 is 0
          }
        }
        sync_all(cluster);
        if (rank == 0) {
          // -2: not found here, -1: the CTAs go on together
          int found = -2;
          const unsigned listed = sh.listed;
          constexpr int kPer = kListSlots / kThreads;
          unsigned long long e[kPer], w[kPer];
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            const unsigned i = j * kThreads + tid;
            e[j] = listed <= kListSlots && i < listed ? sh.list[i] : 0ull;
            w[j] = e[j] != 0 ? weight(logit_at(e[j])) : 0ull;
            if (e[j] != 0) add_to(sh.bins[1], part_at(steps_of(logit_at(e[j])), bin), w[j]);
          }
          __syncthreads();
          const int part = listed <= kListSlots ? reach(sh.bins[1], true, need, 1) : -1;
          if (part >= 0) {
            // the last token before which less than top_p has come is one of this part
            need -= sh.before64;
            if (tid == 0) sh.listed = 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kPer; ++j)
              if (e[j] != 0 && part_at(steps_of(logit_at(e[j])), bin) == part) push(logit_at(e[j]), column_at(e[j]));
            __syncthreads();
            const unsigned few = sh.listed;
            if (few <= kSortSlots) {
              order_list(sh.list, few);
              unsigned long long f[2], wf[2];
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                f[j] = 2 * tid + j < static_cast<int>(few) ? sh.list[2 * tid + j] : 0ull;
                wf[j] = f[j] != 0 ? weight(logit_at(f[j])) : 0ull;
              }
              block_scan64(wf[0] + wf[1], before, sh.red);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                if (f[j] != 0 && before < need && before + wf[j] >= need) sh.found_cut = f[j];
                before += wf[j];
              }
              __syncthreads();
              const unsigned long long cut = sh.found_cut;
              found = -1;
              if (steps_of(logit_at(cut)) >= p.log_min_p) {
                // min_p takes no more away: the CTAs' kept weights, and whose the draw is
                for (int r = 0; r < ctas; ++r) {
                  unsigned long long kept = 0;
#pragma unroll
                  for (int j = 0; j < kPer; ++j)
                    if (e[j] >= cut && column_at(e[j]) / (kThreads * n) == r) kept += w[j];
                  kept = warp_sum64(kept);
                  if (lane == 0) sh.border[warp][r] = kept;
                }
                __syncthreads();
                if (tid < ctas) {
                  unsigned long long kept = sh.above_of[tid];
                  for (int w = 0; w < kWarps; ++w) kept += sh.border[w][tid];
                  sh.kept_of[tid] = kept;
                }
                __syncthreads();
                unsigned long long all = 0, upto = 0;
                for (int r = 0; r < ctas; ++r) all += sh.kept_of[r];
                const unsigned long long target = target_of(p.u[row], all);
                for (found = 0; target >= upto + sh.kept_of[found]; ++found) upto += sh.kept_of[found];
                if (tid < ctas) {
                  Shared* to = cluster.map_shared_rank(&sh, tid);
                  to->found_before = upto;
                  to->found_total = all;
                }
              }
              if (tid < ctas) cluster.map_shared_rank(&sh, tid)->found_cut = cut;
            }
          }
          if (tid < ctas) cluster.map_shared_rank(&sh, tid)->found_cta = found;
        }
        sync_all(cluster);
        if (sh.found_cta >= 0 && sh.found_cta != rank) return;
        alone = sh.found_cta >= 0;
        done = sh.found_cta >= -1;
        if (done) {
          cut_logit = logit_at(sh.found_cut);
          cut_column = column_at(sh.found_cut);
        }
        if (alone) {
          before_cta = sh.found_before;
          total = sh.found_total;
        }
      }
    }
  }

  // ---- digits
  Cut cut{0u, 0u};  // all tokens
  int pass = 0;     // of both kinds of histogram
  unsigned count = 0;
  // a key from its digits: the bits below are 0, of a negative logit 1
  auto with_low_bits = [](unsigned prefix) { return kLowest == 0 || prefix & 0x80000000u ? prefix : prefix | ((1u << kLowest) - 1); };
  if (first != 0) {
    for (int i = 0; i < n; ++i) {
      const float z = v[32 * i];
      v[32 * i] = z == z ? z + 0.f : -INFINITY;  // -0 is 0
      count += is_token(z);
    }
    unsigned long long before;
    tell_all(cluster, sh.count_of, static_cast<unsigned>(block_scan64(count, before, sh.red)));
    count = 0;
    for (int r = 0; r < ctas; ++r) count += sh.count_of[r];
  }
  if (first != 0 && first < count) {
    unsigned need = first, prefix = 0, mask = 0;
    for (int shift = 24; shift >= kLowest; shift -= 8, ++pass) {
      unsigned* hist = sh.hist[pass & 1];
      if (tid < kDigits) hist[tid] = 0;
      __syncthreads();
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float z = v[32 * i];
        const unsigned key = key_of(z);
        if (is_token(z) && (key & mask) == prefix) atomicAdd(&hist[key >> shift & 255], 1u);
      }
      sync_all(cluster);
      if (warp == 0) {
        // a lane has 8 digits, lane 0 the largest
        unsigned h[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          h[j] = 0;
          for (int r = 0; r < ctas; ++r) h[j] += cluster.map_shared_rank(hist, r)[255 - (8 * lane + j)];
          sum += h[j];
        }
        unsigned before = static_cast<unsigned>(warp_scan64(sum, lane)) - sum;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (before < need && before + h[j] >= need) {
            sh.digit = 255 - (8 * lane + j);
            sh.before32 = before;
          }
          before += h[j];
        }
      }
      __syncthreads();
      need -= sh.before32;
      prefix |= sh.digit << shift;
      mask |= 255u << shift;
      // the next pass writes `digit` after a barrier of its own
    }
    cut = {with_low_bits(prefix), need};
  }
  if (!TOP && p.top_p < 1.0 && !done) {
    // the key where top_p of the sum is reached
    unsigned long long sum = 0, before;
#pragma unroll 2
    for (int i = 0; i < n; ++i) {
      const float z = v[32 * i];
      if (is_token(z) && key_of(z) > cut.key) sum += weight(z);
    }
    tell_all(cluster, sh.cut_of, block_scan64(sum, before, sh.red));
    sum = cut.ties != 0 ? cut.ties * weight(logit_of(cut.key)) : 0ull;
    for (int r = 0; r < ctas; ++r) sum += sh.cut_of[r];
    // in 64-bit floating point, which gives what was meant where 0.9 of equal weights is a whole number of them
    unsigned long long need = max(1ull, static_cast<unsigned long long>(p.top_p * static_cast<double>(sum)));
    unsigned prefix = 0, mask = 0;
    for (int shift = 24; shift >= kLowest; shift -= 8, ++pass) {
      unsigned long long* hist = sh.weights[pass & 1];
      if (tid < kDigits) hist[tid] = 0;
      __syncthreads();
      for (int i = 0; i < n; ++i) {
        const float z = v[32 * i] + 0.f;
        const unsigned key = key_of(z);
        if (is_token(z) && key >= cut.key && (key & mask) == prefix) atomicAdd(&hist[key >> shift & 255], weight(z));
      }
      sync_all(cluster);
      if (warp == 0) {
        unsigned long long h[8], all = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          h[j] = 0;
          for (int r = 0; r < ctas; ++r) h[j] += cluster.map_shared_rank(hist, r)[255 - (8 * lane + j)];
          all += h[j];
        }
        unsigned long long upto = warp_scan64(all, lane) - all;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (upto < need && upto + h[j] >= need) {
            sh.digit = 255 - (8 * lane + j);
            sh.before64 = upto;
          }
          upto += h[j];
        }
      }
      __syncthreads();
      need -= sh.before64;
      prefix |= sh.digit << shift;
      mask |= 255u << shift;
    }
    prefix = with_low_bits(prefix);
    const unsigned long long w = weight(logit_of(prefix));
    const unsigned long long ties = (need + w - 1) / w;  // of these it takes so many to reach `need`
    if (prefix > cut.key) cut = {prefix, static_cast<unsigned>(min(ties, 0xffffffffull))};
    else if (ties < cut.ties) cut.ties = static_cast<unsigned>(ties);
  }

  // ---- which of the tokens with the threshold's key are kept: the first ones
  unsigned tie = 0;  // rank of the warp's first
  if (cut.ties != 0) {
    unsigned here = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i)
      here += __popc(__ballot_sync(0xffffffffu, is_token(v[32 * i]) && key_of(v[32 * i] + 0.f) == cut.key));
    unsigned long long before;
    const unsigned of_cta = static_cast<unsigned>(block_scan64(lane == 0 ? here : 0u, before, sh.red));
    tie = __shfl_sync(0xffffffffu, static_cast<unsigned>(before), 0);
    tell_all(cluster, sh.ties_of, of_cta);
    for (int r = 0; r < rank; ++r) tie += sh.ties_of[r];
  }
  if (cut.key != 0) {
#pragma unroll 2
    for (int i = 0; i < n; ++i) {
      const float z = v[32 * i];
      const unsigned key = key_of(z + 0.f);
      bool in = is_token(z) && key > cut.key;
      if (cut.ties != 0) {
        const bool equal = is_token(z) && key == cut.key;
        const unsigned all = __ballot_sync(0xffffffffu, equal);
        in = in || (equal && tie + __popc(all & ((1u << lane) - 1)) < cut.ties);
        tie += __popc(all);
      }
      if (!in) v[32 * i] = -INFINITY;  // from here on no token
    }
  }

  if (TOP) {
    // ---- the kept tokens to the first CTA, which sorts them
    const unsigned have = min(static_cast<unsigned>(p.k), count);
    sync_all(cluster);  // the list lies where the histograms are
    if (rank == 0 && tid == 0) sh.listed = 0;
    sync_all(cluster);
#pragma unroll 4
    for (int i = 0; i < n; ++i)
      if (is_token(v[32 * i])) push(v[32 * i], col0 + 32 * i);
    sync_all(cluster);
    if (rank != 0) return;
    order_list(sh.list, have);
    for (int i = tid; i < p.k; i += kThreads) {
      const bool in = i < static_cast<int>(have);
      const int64_t at = static_cast<int64_t>(row) * p.k + i;
      p.logp[at] = in ? log_p(logit_at(sh.list[i])) : 0.f;
      p.ids[at] = in ? column_at(sh.list[i]) : -1;
    }
    return;
  }

  // ---- the draw
  const float min_logit = p.log_min_p > -INFINITY ? __double2float_rd(m64 + (p.log_min_p - 1.0) / p.steps) : -INFINITY;
  auto kept_at = [&](float z, int column) {
    if (!is_token(z) || z < min_logit) return false;
    if (done && !(z > cut_logit || (z == cut_logit && column <= cut_column))) return false;
    return p.log_min_p == -INFINITY || steps_of(z) >= p.log_min_p;
  };
  if (first != 0 || done || p.top_p < 1.0 || p.log_min_p > -INFINITY) {
    own = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      // which of 32 are kept, then those alone: a thread's few rather than a warp's many
      unsigned kept = 0;
#pragma unroll 8
      for (int i = 0; i < min(32, n - i0); ++i) kept |= kept_at(v[32 * (i0 + i)], col0 + 32 * (i0 + i)) ? 1u << i : 0u;
      for (; kept != 0; kept &= kept - 1) own += weight(v[32 * (i0 + __ffs(kept) - 1)]);
    }
  }
  unsigned long long before;
  const unsigned long long of_warp = warp_sum64(own), of_cta = block_scan64(own, before, sh.red);
  before = __shfl_sync(0xffffffffu, before, 0);  // the warp's
  if (alone) {
    before += before_cta;
  } else {
    tell_all(cluster, sh.kept_of, of_cta);
    total = 0;
    for (int r = 0; r < ctas; ++r) {
      if (r == rank) before += total;
      total += sh.kept_of[r];
    }
  }
  const unsigned long long target = target_of(p.u[row], total);
  if (target < before || target >= before + of_warp) return;
  // this warp has it: the sums of 32 times 32 columns i, then the lanes of one i
  unsigned long long at = before;
  for (int i0 = 0; i0 < n; i0 += 32) {
    __syncwarp();
    for (int i = 0; i < min(32, n - i0); ++i) {
      const float z = v[32 * (i0 + i)];
      sh.cells[i][lane] = kept_at(z, col0 + 32 * (i0 + i)) ? weight(z) : 0ull;
    }
    __syncwarp();
    unsigned long long s = 0;
    if (i0 + lane < n)
      for (int l = 0; l < 32; ++l) s += sh.cells[lane][l];
    const unsigned long long upto = at + warp_scan64(s, lane);
    const unsigned past = __ballot_sync(0xffffffffu, target < upto);
    if (past == 0) {
      at = __shfl_sync(0xffffffffu, upto, 31);
      continue;
    }
    const int l = __ffs(past) - 1;
    at = __shfl_sync(0xffffffffu, upto - s, l);
    const unsigned long long mine = at + warp_scan64(sh.cells[l][lane], lane);
    if (lane == __ffs(__ballot_sync(0xffffffffu, target < mine)) - 1) {
      p.ids[row] = col0 + 32 * (i0 + l);
      p.logp[row] = log_p(v[32 * (i0 + l)]);
    }
    return;
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
  TORCH_CHECK(std::isfinite(temperature) && temperature > 0, "temperature must be positive");
}

constexpr int64_t kMostVocab = static_cast<int64_t>(rows::kMostCtas) * rows::kMostColumns * rows::kThreads;

template <typename T, bool TOP>
static void launch_rows(rows::Params& p) {
  // 32 columns a thread (64 KB a CTA, so that several rows share an SM) as long as 8 CTAs are enough
  int ctas = 1;
  while (ctas < 8 && ctas * 32 * rows::kThreads < p.V) ctas *= 2;
  p.per_thread = (p.V + 4 * ctas * rows::kThreads - 1) / (4 * ctas * rows::kThreads) * 4;
  auto kern = rows::rows_kernel<T, TOP>;
  static DeviceFlags configured;
  if (bool& done = configured.here(); !done) {
    T1_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * rows::kMostColumns * rows::kThreads));
    done = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * ctas);
  cfg.blockDim = dim3(rows::kThreads);
  cfg.dynamicSmemBytes = 4 * p.per_thread * rows::kThreads;
  cfg.stream = stream();
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<const rows::Params>(p));
  TORCH_CHECK(e == cudaSuccess, TOP ? "topk_logprobs" : "sample_tokens", " launch failed: ", cudaGetErrorString(e));
  count_launch();
}

template <bool TOP>
static void run_rows(rows::Params& p, const torch::Tensor& logits, double temperature) {
  TORCH_CHECK(logits.size(1) <= kMostVocab, "at most ", kMostVocab, " tokens, got ", logits.size(1));
  TORCH_CHECK(logits.size(0) < (1ll << 27), "at most 2^27 rows, got ", logits.size(0));
  p.logits = logits.data_ptr();
  p.ld = logits.size(0) > 1 ? logits.stride(0) : 0;
  p.rows = static_cast<int>(logits.size(0));
  p.V = static_cast<int>(logits.size(1));
  p.aligned = reinterpret_cast<uintptr_t>(p.logits) % 16 == 0 && p.ld * logits.element_size() % 16 == 0;
  p.tau = static_cast<float>(temperature);
  p.scale = static_cast<float>(1.0 / temperature);
  p.scale2 = static_cast<float>(1.4426950408889634 / temperature);
  p.steps = rows::kExps * 1.4426950408889634 / temperature;
  if (p.rows == 0) return;
  if (logits.scalar_type() == torch::kFloat32) launch_rows<float, TOP>(p);
  else launch_rows<rows::bf16_t, TOP>(p);
}

// Returns (logp [T, k] fp32, ids [T, k] int64).
std::vector<torch::Tensor> topk_logprobs(torch::Tensor logits, int64_t k, double temperature) {
  check_rows(logits, temperature);
  TORCH_CHECK(k >= 1 && k <= std::min<int64_t>(rows::kMostList, logits.size(1)), "k must lie in [1, min(V, ",
              rows::kMostList, ")], got ", k);
  const c10::cuda::CUDAGuard guard(logits.device());
  auto logp = torch::empty({logits.size(0), k}, logits.options().dtype(torch::kFloat32));
  auto ids = torch::empty({logits.size(0), k}, logits.options().dtype(torch::kInt64));
  rows::Params p{};
  p.k = static_cast<int>(k);
  p.logp = logp.data_ptr<float>();
  p.ids = ids.data_ptr<int64_t>();
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
  p.u = uc.data_ptr<float>();
  p.top_k = static_cast<int>(top_k >= logits.size(1) ? 0 : top_k);
  p.top_p = top_p;
  p.log_min_p = rows::kExps * std::log2(min_p);
  int bits = 0;
  while ((1ll << bits) < logits.size(1)) ++bits;
  p.one = std::min(51, 62 - bits);  // a weight fits the 52 bits of a double
  run_rows<false>(p, logits, temperature);
  return {token, logp};
}

}  // namespace t1
