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
// every thread keeps to the same few of them in every pass.  Thresholds are found digit by
// digit of the order-preserving integer of a logit (8 bits at a time), with the
// CTAs' histograms added up over distributed shared memory.
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
constexpr int kMostCtas = 16;   // of a cluster
constexpr int kMostList = 512;  // tokens of `top`
constexpr int kDigits = 256;

struct Params {
  const void* logits;
  int64_t ld;
  int rows, V;
  float scale;     // 1 / tau
  double scale64;
  // top
  int k;
  float* logp;     // [rows, k]; sample: [rows]
  int64_t* ids;    // [rows, k]; sample: [rows]
  // sample
  const float* u;
  int top_k;                  // 0: all
  double top_p;               // 1: all
  double log_min_p;           // -inf: all
  double one;                 // the weight of the largest logit, 2^s
  int per_thread;             // columns
};

// A logit to shared memory: 32-bit ones without a stop in a register.
__device__ __forceinline__ void fetch(float* to, const float* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from)
               : "memory");
}
__device__ __forceinline__ void fetch(float* to, const bf16_t* from) {
  *to = __bfloat162float(__ushort_as_bfloat16(__ldcs(reinterpret_cast<const unsigned short*>(from))));
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
  unsigned hist[2][kDigits];
  unsigned long long weights[2][kDigits];
  unsigned long long red[kWarps];
  // what every CTA of the cluster tells all others, once each
  float max_of[kMostCtas];
  float sum_of[kMostCtas];
  unsigned count_of[kMostCtas], ties_of[kMostCtas];
  unsigned long long total_of[kMostCtas], kept_of[kMostCtas];
  // the digit that a threshold falls into
  unsigned digit, before32, in32;
  unsigned long long before64;
  unsigned listed;
  unsigned long long list[kMostList];   // of the first CTA
  unsigned long long cells[32][33];     // weights of the warp that holds the drawn token
};

// Every CTA's value to all of the cluster, in slots[rank]; one barrier.
template <typename V>
__device__ __forceinline__ void tell_all(cg::cluster_group& cluster, V* slots, V value) {
  const unsigned n = cluster.num_blocks();
  if (threadIdx.x < n) cluster.map_shared_rank(slots, threadIdx.x)[cluster.block_rank()] = value;
  cluster.sync();
}

// A prefix of the order: all tokens of a larger key, and the first `ties` of
// those that have it.
struct Cut {
  unsigned key;
  unsigned ties;
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads) rows_kernel(const Params p) {
  __shared__ Shared sh;
  extern __shared__ float held[];
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / ctas;
  // a warp has 32 n columns in a row, a thread every 32nd of them
  const int n = p.per_thread;
  const int col0 = (rank * kWarps + warp) * 32 * n + lane;
  float* v = held + warp * 32 * n + lane;  // v[32 i]: the thread's i-th
  constexpr int kLowest = sizeof(T) == 2 ? 16 : 0;  // key bits below are the same in all of a type's values

  const T* src = static_cast<const T*>(p.logits) + row * p.ld;
#pragma unroll 8
  for (int i = 0; i < n; ++i) {
    const int c = col0 + 32 * i;
    if (c < p.V) fetch(&v[32 * i], src + c);
    else v[32 * i] = -INFINITY;
  }
  fetched();
  float m = -INFINITY;
  unsigned count = 0;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    float z = v[32 * i];
    z = z == z ? z + 0.f : -INFINITY;  // -0 is 0
    v[32 * i] = z;
    m = fmaxf(m, z);
    count += z > -INFINITY;
  }

  // ---- largest logit, number of tokens
  __shared__ float red[32];
  m = block_max(m, red);
  {
    unsigned long long c = warp_sum64(count);
    if (lane == 0) sh.red[warp] = c;
    __syncthreads();
    c = 0;
    for (int w = 0; w < kWarps; ++w) c += sh.red[w];
    count = static_cast<unsigned>(c);
  }
  if (tid < static_cast<unsigned>(ctas)) cluster.map_shared_rank(sh.max_of, tid)[rank] = m;
  tell_all(cluster, sh.count_of, count);
  count = 0;
  for (int r = 0; r < ctas; ++r) {
    m = fmaxf(m, sh.max_of[r]);
    count += sh.count_of[r];
  }

  // ---- log of the sum of all weights
  float sum = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) sum += v[32 * i] == m ? 1.f : __expf((v[32 * i] - m) * p.scale);
  if (m == -INFINITY) sum = 0.f;
  sum = block_sum(sum, red);
  tell_all(cluster, sh.sum_of, sum);
  sum = 0.f;
  for (int r = 0; r < ctas; ++r) sum += sh.sum_of[r];
  const float log_sum = logf(sum);

  auto log_weight = [&](float z) {
    return z == m ? 0.0 : (static_cast<double>(z) - static_cast<double>(m)) * p.scale64;
  };
  auto weight = [&](float z) -> unsigned long long { return __double2ull_rn(exp(log_weight(z)) * p.one); };
  // a key from its digits: the bits below are 0, of a negative logit 1
  auto with_low_bits = [](unsigned prefix) { return kLowest == 0 || prefix & 0x80000000u ? prefix : prefix | ((1u << kLowest) - 1); };
  auto is_token = [](float z) { return z > -INFINITY; };

  Cut cut{0u, 0u};  // all tokens
  int pass = 0;     // of both kinds of histogram

  // ---- the n-th token's key
  const unsigned first = TOP ? p.k : p.top_k;
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
      cluster.sync();
      if (warp == 0) {
        // a lane has 8 digits, lane 0 the largest
        unsigned h[8], own = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          h[j] = 0;
          for (int r = 0; r < ctas; ++r) h[j] += cluster.map_shared_rank(hist, r)[255 - (8 * lane + j)];
          own += h[j];
        }
        unsigned before = static_cast<unsigned>(warp_scan64(own, lane)) - own;
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

  if (!TOP && p.top_p < 1.0 && count > 0) {
    // ---- the key where top_p of the sum is reached
    unsigned long long total = 0;
#pragma unroll 2
    for (int i = 0; i < n; ++i) {
      const float z = v[32 * i];
      if (is_token(z) && key_of(z) > cut.key) total += weight(z);
    }
    total = warp_sum64(total);
    __syncthreads();
    if (lane == 0) sh.red[warp] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kWarps; ++w) total += sh.red[w];
    tell_all(cluster, sh.total_of, total);
    total = cut.ties != 0 ? cut.ties * weight(logit_of(cut.key)) : 0ull;
    for (int r = 0; r < ctas; ++r) total += sh.total_of[r];
    // in 64-bit floating point, which gives what was meant where 0.9 of equal weights is a whole number of them
    unsigned long long need = max(1ull, static_cast<unsigned long long>(p.top_p * static_cast<double>(total)));
    unsigned prefix = 0, mask = 0;
    for (int shift = 24; shift >= kLowest; shift -= 8, ++pass) {
      unsigned long long* hist = sh.weights[pass & 1];
      if (tid < kDigits) hist[tid] = 0;
      __syncthreads();
      for (int i = 0; i < n; ++i) {
        const float z = v[32 * i];
        const unsigned key = key_of(z);
        if (is_token(z) && key >= cut.key && (key & mask) == prefix) atomicAdd(&hist[key >> shift & 255], weight(z));
      }
      cluster.sync();
      if (warp == 0) {
        unsigned long long h[8], own = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          h[j] = 0;
          for (int r = 0; r < ctas; ++r) h[j] += cluster.map_shared_rank(hist, r)[255 - (8 * lane + j)];
          own += h[j];
        }
        unsigned long long before = warp_scan64(own, lane) - own;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (before < need && before + h[j] >= need) {
            sh.digit = 255 - (8 * lane + j);
            sh.before64 = before;
          }
          before += h[j];
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
  unsigned tie = 0, ties_here = 0;  // rank of the warp's first
  if (cut.ties != 0) {
#pragma unroll 4
    for (int i = 0; i < n; ++i)
      ties_here += __popc(__ballot_sync(0xffffffffu, is_token(v[32 * i]) && key_of(v[32 * i]) == cut.key));
    __syncthreads();
    if (lane == 0) sh.red[warp] = ties_here;
    __syncthreads();
    unsigned of_cta = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) tie = of_cta;
      of_cta += static_cast<unsigned>(sh.red[w]);
    }
    tell_all(cluster, sh.ties_of, of_cta);
    for (int r = 0; r < rank; ++r) tie += sh.ties_of[r];
  }
  unsigned long long own = 0;  // weight of the thread's kept tokens
#pragma unroll 2
  for (int i = 0; i < n; ++i) {
    const float z = v[32 * i];
    const unsigned key = key_of(z);
    bool in = is_token(z) && key > cut.key;
    if (cut.ties != 0) {
      const bool equal = is_token(z) && key == cut.key;
      const unsigned all = __ballot_sync(0xffffffffu, equal);
      in = in || (equal && tie + __popc(all & ((1u << lane) - 1)) < cut.ties);
      tie += __popc(all);
    }
    if (!TOP && in) {
      in = log_weight(z) >= p.log_min_p;
      if (in) own += weight(z);
    }
    if (!in) v[32 * i] = -INFINITY;  // from here on no token
  }

  if (TOP) {
    // ---- the kept tokens to the first CTA, which sorts them
    const unsigned have = min(static_cast<unsigned>(p.k), count);
    unsigned slots = 1;
    while (slots < static_cast<unsigned>(p.k)) slots *= 2;
    if (rank == 0) {
      if (tid == 0) sh.listed = 0;
      for (unsigned i = tid; i < slots; i += kThreads) sh.list[i] = 0;
    }
    cluster.sync();
    unsigned* listed = cluster.map_shared_rank(&sh.listed, 0);
    unsigned long long* list = cluster.map_shared_rank(sh.list, 0);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      if (is_token(v[32 * i])) {
        const unsigned at = atomicAdd(listed, 1u);
        if (at < kMostList)
          list[at] = static_cast<unsigned long long>(key_of(v[32 * i])) << 32 | ~static_cast<unsigned>(col0 + 32 * i);
      }
    }
    cluster.sync();
    if (rank != 0) return;
    for (unsigned size = 2; size <= slots; size *= 2) {
      for (unsigned step = size / 2; step > 0; step /= 2) {
        const unsigned i = tid, j = i ^ step;
        if (i < slots && j > i) {
          const unsigned long long a = sh.list[i], b = sh.list[j];
          if ((a < b) == ((i & size) == 0)) {
            sh.list[i] = b;
            sh.list[j] = a;
          }
        }
        __syncthreads();
      }
    }
    if (tid < p.k) {
      const unsigned long long e = sh.list[tid];
      const float z = logit_of(static_cast<unsigned>(e >> 32));
      const bool in = tid < static_cast<int>(have);
      const int64_t at = static_cast<int64_t>(row) * p.k + tid;
      if (!T1_OOB(at, static_cast<int64_t>(p.rows) * p.k)) {
        p.logp[at] = in ? (z == m ? 0.f : (z - m) * p.scale) - log_sum : 0.f;
        p.ids[at] = in ? static_cast<int64_t>(~static_cast<unsigned>(e)) : -1;
      }
    }
    return;
  }

  // ---- the draw
  unsigned long long of_warp = warp_sum64(own);
  __syncthreads();
  if (lane == 0) sh.red[warp] = of_warp;
  __syncthreads();
  unsigned long long before = 0, of_cta = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before = of_cta;
    of_cta += sh.red[w];
  }
  tell_all(cluster, sh.kept_of, of_cta);
  unsigned long long total = 0;
  for (int r = 0; r < ctas; ++r) {
    if (r == rank) before += total;
    total += sh.kept_of[r];
  }
  if (T1_OOB(row, p.rows)) return;
  if (total == 0) {
    if (rank == 0 && tid == 0) {
      p.ids[row] = -1;
      p.logp[row] = 0.f;
    }
    return;
  }
  const double ud = fmin(fmax(static_cast<double>(p.u[row]), 0.0), 1.0 - 0x1p-53);  // NaN: 0
  const unsigned long long target = __umul64hi(total, static_cast<unsigned long long>(ud * 0x1p64));
  if (target < before || target >= before + of_warp) return;
  // this warp has it: the sums of 32 times 32 columns i, then the lanes of one i
  unsigned long long at = before;
  for (int i0 = 0; i0 < n; i0 += 32) {
    __syncwarp();
    for (int i = 0; i < min(32, n - i0); ++i) {
      const float z = v[32 * (i0 + i)];
      sh.cells[i][lane] = is_token(z) ? weight(z) : 0ull;
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
      const float z = v[32 * (i0 + l)];
      p.ids[row] = col0 + 32 * (i0 + l);
      p.logp[row] = (z == m ? 0.f : (z - m) * p.scale) - log_sum;
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

// Columns of a thread that fit in shared memory next to the rest.
constexpr int kMostColumns = 96;
constexpr int64_t kMostVocab = 8ll * kMostColumns * rows::kThreads;

template <typename T, bool TOP>
static void launch_rows(rows::Params& p) {
  // 32 columns a thread (64 KB a CTA, so that several rows share an SM) as long as 8 CTAs are enough
  int ctas = 1;
  while (ctas < 8 && ctas * 32 * rows::kThreads < p.V) ctas *= 2;
  p.per_thread = (p.V + ctas * rows::kThreads - 1) / (ctas * rows::kThreads);
  auto kern = rows::rows_kernel<T, TOP>;
  static DeviceFlags configured;
  if (bool& done = configured.here(); !done) {
    T1_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * kMostColumns * rows::kThreads));
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
  p.scale64 = 1.0 / temperature;
  p.scale = static_cast<float>(p.scale64);
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
  p.log_min_p = std::log(min_p);
  int bits = 0;
  while ((1ll << bits) < logits.size(1)) ++bits;
  p.one = std::ldexp(1.0, 62 - bits);
  run_rows<false>(p, logits, temperature);
  return {token, logp};
}

}  // namespace t1
