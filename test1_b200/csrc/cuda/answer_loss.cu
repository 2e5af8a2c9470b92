// Losses on the log-probabilities of answer tokens, with their gradients:
// the preference loss of paired answers and the clipped policy loss.
//
// Both read [B, S] tokens (sequence after sequence) of which the targets
// mark the answers; entries of other tokens are never used, whatever they
// hold.  Both need numbers per sequence and for the whole batch before the
// first gradient can be written (a pair's margin, the token count).  The
// phases:
//   A  per unit (a piece of a sequence): answer tokens, and for the preference
//      loss the sum of their log ratios
//   B  per pair or sequence, from its units (preference: margin, loss and
//      gradient coefficient; policy: the length, only where sequences of
//      several units have a mean of their own)
//   C  per token: the gradient, and the policy loss's own sums
//   D  the policy loss's totals
// Up to kClusterTokens a single launch runs them all, a cluster of 1 to 8
// blocks whose barrier stands between the phases: such a call is launches and
// latency, and every launch saved is 4 us of the host's time.  A larger batch
// is bound by its bytes and takes a launch per phase over all SMs (D: the
// last block of C).  A unit belongs to a warp or, for sequences shorter than
// 32 tokens, to the fewest lanes that hold one.  Sums are carried in fp64 and
// joined in a fixed order: two runs give the same bits.
#include "common.cuh"
#include "sm100.cuh"

#include <ATen/cuda/CUDAGraphsUtils.cuh>

#include <string>
#include <unordered_map>

namespace t1 {

torch::Tensor arrival_counters(int64_t n);

enum PreferenceKind : int { kSigmoid = 0, kHinge = 1, kIpo = 2 };
enum Phase : int { kA = 1, kB = 2, kC = 4, kD = 8 };

struct LossParams {
  const float *logp, *ref, *old, *adv;
  const int64_t* targets;
  int64_t ignore;
  int64_t B;
  int S;
  int unit, chunks;        // tokens of a unit, units of a sequence
  int lanes;               // lanes of a unit: 32, or the power of two >= S
  int phases;              // of this launch
  int parts;               // entries of `totals` when C starts
  double2* units;          // [B * chunks] (sum of log ratios, answer tokens)
  double2* totals;         // [block] preference: (loss, pairs); policy: (answer tokens, sequences that have one)
  float *loss, *dlogp;
  // preference
  int kind, average;
  double beta, smoothing;
  float* coef;             // [B] dloss/dlogp of the sequence's answer tokens, times the number of pairs
  float* rewards;          // [B]
  // policy
  int adv_per_token, per_sequence;
  float lo, hi, edge_lo, edge_hi, kl_coef;
  int* lengths;            // [B] answer tokens, with phase B
  double* sums;            // [block of C][3] loss, KL, clipped
  int* ticket;             // arrivals of C's blocks, zero between launches
  float* stats;            // [2]
};

constexpr int kLossThreads = 512;
constexpr int kLossWarps = kLossThreads / 32;
constexpr int kAhead = 4;  // tokens of a lane whose loads are issued together

// Block-wide sum in fp64, every thread gets it.
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0;
#pragma unroll
  for (int w = 0; w < kLossWarps; ++w) t += red[w];
  return t;
}

// Sum over the `by` neighbouring lanes that share v's subject.
__device__ __forceinline__ double group_sum(double v, int by) {
  for (int o = by >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// (sum, tokens) of sequence b; `by` lanes share its units.
__device__ __forceinline__ double2 join_units(const LossParams& p, int64_t b, int lane, int by) {
  double2 t = make_double2(0, 0);
  for (int c = lane; c < p.chunks; c += by) {
    const double2 v = __ldcg(&p.units[b * p.chunks + c]);
    t.x += v.x;
    t.y += v.y;
  }
  return make_double2(group_sum(t.x, by), group_sum(t.y, by));
}

__device__ __forceinline__ double2 join_totals(const LossParams& p, double* red) {
  double2 t = make_double2(0, 0);
  for (int i = threadIdx.x; i < p.parts; i += kLossThreads) {
    const double2 v = __ldcg(&p.totals[i]);
    t.x += v.x;
    t.y += v.y;
  }
  return make_double2(block_sum_f64(t.x, red), block_sum_f64(t.y, red));
}

__device__ __forceinline__ void write_totals(const LossParams& p, double x, double y, double* red) {
  x = block_sum_f64(x, red);
  y = block_sum_f64(y, red);
  if (threadIdx.x == 0) __stcg(&p.totals[blockIdx.x], make_double2(x, y));
}

// The warps' walk over units: body(unit, sequence, first token, past the last
// token, lane of the unit), with all lanes of a warp in step; unit is -1 for
// lanes that have none in a warp's last round.
template <class F>
__device__ __forceinline__ void for_units(const LossParams& p, F body) {
  const int per_warp = 32 / p.lanes, in_warp = threadIdx.x & 31;
  const int64_t count = p.B * p.chunks, step = static_cast<int64_t>(gridDim.x) * kLossWarps * per_warp;
  for (int64_t u0 = (static_cast<int64_t>(blockIdx.x) * kLossWarps + (threadIdx.x >> 5)) * per_warp; u0 < count; u0 += step) {
    const int64_t u = u0 + in_warp / p.lanes;
    const int64_t b = u < count ? u / p.chunks : 0;
    const int s0 = u < count ? static_cast<int>(u - b * p.chunks) * p.unit : 0;
    body(u < count ? u : -1, b, b * p.S + s0, u < count ? b * p.S + min(p.S, s0 + p.unit) : s0, in_warp & (p.lanes - 1));
  }
}

// ------------------------------------------------------------------ phase A
template <bool POLICY>
__device__ __forceinline__ void count_phase(const LossParams& p, double* red) {
  double tokens = 0, live = 0;
  for_units(p, [&](int64_t u, int64_t, int64_t i0, int64_t i1, int lane) {
    double sum = 0;
    int n = 0;
    if (u < 0) i1 = i0;
    for (int64_t i = i0 + lane; i < i1; i += kAhead * p.lanes) {
      bool ok[kAhead];
      float v[kAhead], r[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t at = i + k * p.lanes;
        ok[k] = at < i1 && p.targets[at] != p.ignore;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t at = i + k * p.lanes;
        n += ok[k];
        v[k] = !POLICY && ok[k] ? p.logp[at] : 0.f;
        r[k] = !POLICY && ok[k] && p.ref != nullptr ? p.ref[at] : 0.f;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) sum += v[k] - r[k];
    }
    const double cnt = group_sum(n, p.lanes);
    if (!POLICY) sum = group_sum(sum, p.lanes);
    if (u >= 0 && lane == 0) {
      __stcg(&p.units[u], make_double2(sum, cnt));
      tokens += cnt;
      live += cnt > 0 ? 1 : 0;
    }
  });
  if (POLICY) write_totals(p, tokens, live, red);
}

// ------------------------------------------------------------------ phase B
__device__ __forceinline__ void pairs_phase(const LossParams& p, double* red) {
  const int64_t P = p.B / 2;
  // a thread for a pair of few units, a warp for one of many
  const int by = p.chunks <= 4 ? 1 : 32, lane = threadIdx.x & (by - 1);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kLossThreads / by;
  double loss = 0, live = 0;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kLossThreads + threadIdx.x) / by; i < P; i += step) {
    const double2 ch = join_units(p, i, lane, by), rj = join_units(p, i + P, lane, by);
    if (lane != 0) continue;
    const double pc = p.average ? 1 / fmax(1.0, ch.y) : 1, pr = p.average ? 1 / fmax(1.0, rj.y) : 1;
    const double m = ch.x * pc - rj.x * pr, z = p.beta * m;
    double l, d;
    if (p.kind == kSigmoid) {
      const double eps = p.smoothing, tail = log1p(exp(-fabs(z)));
      l = (1 - eps) * (fmax(-z, 0.0) + tail) + eps * (fmax(z, 0.0) + tail);
      d = p.beta * (eps / (1 + exp(-z)) - (1 - eps) / (1 + exp(z)));
    } else if (p.kind == kHinge) {
      l = fmax(1 - z, 0.0);
      d = z < 1 ? -p.beta : 0;
    } else {
      const double e = m - 0.5 / p.beta;
      l = e * e;
      d = 2 * e;
    }
    if (ch.y + rj.y > 0) {
      loss += l;
      live += 1;
    } else {
      d = 0;
    }
    __stcg(&p.coef[i], static_cast<float>(d * pc));
    __stcg(&p.coef[i + P], static_cast<float>(-d * pr));
    p.rewards[i] = static_cast<float>(p.beta * ch.x * pc);
    p.rewards[i + P] = static_cast<float>(p.beta * rj.x * pr);
  }
  write_totals(p, loss, live, red);
}

__device__ __forceinline__ void lengths_phase(const LossParams& p, double* red) {
  const int lane = threadIdx.x & 31;
  double tokens = 0, live = 0;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * kLossWarps + (threadIdx.x >> 5); b < p.B; b += static_cast<int64_t>(gridDim.x) * kLossWarps) {
    const double n = join_units(p, b, lane, 32).y;
    if (lane != 0) continue;
    __stcg(&p.lengths[b], static_cast<int>(n));
    tokens += n;
    live += n > 0 ? 1 : 0;
  }
  write_totals(p, tokens, live, red);
}

// ------------------------------------------------------------------ phase C
__device__ __forceinline__ void preference_grad_phase(const LossParams& p, double* red) {
  const double2 total = join_totals(p, red);
  const double pairs = fmax(1.0, total.y);
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.loss = static_cast<float>(total.x / pairs);
  for_units(p, [&](int64_t u, int64_t b, int64_t i0, int64_t i1, int lane) {
    if (u < 0) return;
    const float d = static_cast<float>(__ldcg(&p.coef[b]) / pairs);
    for (int64_t i = i0 + lane; i < i1; i += kAhead * p.lanes) {
      bool ok[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t at = i + k * p.lanes;
        ok[k] = at < i1 && p.targets[at] != p.ignore;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (i + k * p.lanes < i1) p.dlogp[i + k * p.lanes] = ok[k] ? d : 0.f;
    }
  });
}

__device__ __forceinline__ void policy_grad_phase(const LossParams& p, double* red) {
  const double2 total = join_totals(p, red);
  const double tokens = fmax(1.0, total.x), live = fmax(1.0, total.y);
  double loss = 0, kls = 0;
  int cut = 0;
  for_units(p, [&](int64_t u, int64_t b, int64_t i0, int64_t i1, int lane) {
    if (u < 0) return;
    float w = static_cast<float>(1 / tokens);
    if (p.per_sequence) {
      const double n = p.chunks == 1 ? __ldcg(&p.units[u]).y : static_cast<double>(__ldcg(&p.lengths[b]));
      w = static_cast<float>(1 / (fmax(1.0, n) * live));
    }
    const float seq_adv = p.adv_per_token ? 0.f : p.adv[b];
    double unit_loss = 0;
    for (int64_t i = i0 + lane; i < i1; i += kAhead * p.lanes) {
      bool ok[kAhead];
      float lp[kAhead], od[kAhead], rf[kAhead], a[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t at = i + k * p.lanes;
        ok[k] = at < i1 && p.targets[at] != p.ignore;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t at = i + k * p.lanes;
        lp[k] = ok[k] ? p.logp[at] : 0.f;
        od[k] = ok[k] ? p.old[at] : 0.f;
        rf[k] = ok[k] && p.ref != nullptr ? p.ref[at] : 0.f;
        a[k] = ok[k] && p.adv_per_token ? p.adv[at] : seq_adv;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (i + k * p.lanes >= i1) continue;
        float g = 0.f;
        if (ok[k]) {
          // clipped where the log ratio is past log(1 +- clip): the same
          // token whatever exp's rounding does at the edge
          const float d = lp[k] - od[k], rho = expf(d);
          const bool over = d > p.hi, under = d < p.lo;
          const bool clipped = (a[k] > 0.f && over) || (a[k] < 0.f && under);
          float l = -a[k] * (clipped ? (over ? p.edge_hi : p.edge_lo) : rho);
          g = clipped ? 0.f : -a[k] * rho;
          if (p.ref != nullptr) {
            const float e = rf[k] - lp[k], x = expm1f(e), kl = x - e;
            l += p.kl_coef * kl;
            g -= p.kl_coef * x;
            kls += kl;
          }
          g *= w;
          unit_loss += l;
          cut += clipped;
        }
        p.dlogp[i + k * p.lanes] = g;
      }
    }
    loss += unit_loss * w;
  });
  loss = block_sum_f64(loss, red);
  kls = block_sum_f64(kls, red);
  const double cuts = block_sum_f64(cut, red);
  if (threadIdx.x < 3) __stcg(&p.sums[3 * blockIdx.x + threadIdx.x], threadIdx.x == 0 ? loss : threadIdx.x == 1 ? kls : cuts);
}

// ------------------------------------------------------------------ phase D
__device__ __forceinline__ void policy_total_phase(const LossParams& p, double* red) {
  const double tokens = fmax(1.0, join_totals(p, red).x);
  double v[3] = {0, 0, 0};
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += kLossThreads)
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] += __ldcg(&p.sums[3 * i + k]);
#pragma unroll
  for (int k = 0; k < 3; ++k) v[k] = block_sum_f64(v[k], red);
  if (threadIdx.x == 0) {
    *p.loss = static_cast<float>(v[0]);
    p.stats[0] = static_cast<float>(v[1] / tokens);
    p.stats[1] = static_cast<float>(v[2] / tokens);
  }
}

template <bool POLICY>
__global__ void __launch_bounds__(kLossThreads, 2) answer_loss_kernel(const LossParams p) {
  __shared__ double red[kLossWarps];
  __shared__ int last;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.phases & kA) count_phase<POLICY>(p, red);
  if (p.phases & kB) {
    if (p.phases & kA) sm100::cluster_sync();
    if (POLICY) lengths_phase(p, red);
    else pairs_phase(p, red);
  }
  if (p.phases & kC) {
    if (p.phases & kA) sm100::cluster_sync();
    if (POLICY) policy_grad_phase(p, red);
    else preference_grad_phase(p, red);
  }
  if (!POLICY || !(p.phases & kD)) return;
  if (p.phases & kA) {
    sm100::cluster_sync();
    if (blockIdx.x == 0) policy_total_phase(p, red);
    return;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  if (threadIdx.x == 0) *p.ticket = 0;
  policy_total_phase(p, red);
}

// ================================================================ host side
T1_BOUNDS_READER(answer_loss)

// Tokens up to which one cluster does it all.  Eight SMs read about 1.5 TB/s:
// at 256 K tokens (6 MB) that costs what the launches saved were worth.
constexpr int64_t kClusterTokens = 256 * 1024;

static void check_tokens(const torch::Tensor& t, int64_t T, const torch::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), what, " must be on the device of logp");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32, what, " has dtype ", t.scalar_type(), ", expected Float");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == T, what, " must have ", std::to_string(T), " entries");
}

static int64_t check_batch(const torch::Tensor& logp, const torch::Tensor& targets, int64_t S) {
  TORCH_CHECK(logp.is_cuda(), "logp must be a CUDA tensor");
  TORCH_CHECK(logp.dim() == 1, "logp must be [T]");
  check_tokens(logp, logp.size(0), logp, "logp");
  TORCH_CHECK(targets.is_cuda() && targets.device() == logp.device() && targets.scalar_type() == torch::kInt64,
              "targets must be int64 on the device of logp");
  TORCH_CHECK(targets.dim() == 1 && targets.size(0) == logp.size(0), "targets must have T entries");
  TORCH_CHECK(S > 0 && S < (1ll << 30) && logp.size(0) % S == 0, "tokens must be a multiple of seq_len");
  return logp.size(0) / S;
}

// The units of a batch, and how the phases' launches look.
struct LossPlan {
  int cluster;         // blocks of the single launch, 0: a launch per phase
  int blocks, seq_blocks;  // of the launches over units, over sequences
  int unit, chunks, lanes;

  LossPlan(int64_t B, int64_t S) {
    const int64_t T = B * S;
    cluster = 0;
    int64_t warps = 8 * num_sms() * kLossWarps;
    if (T <= kClusterTokens) {
      cluster = 1;
      while (cluster < 8 && cluster * 4096 < T) cluster *= 2;
      warps = cluster * kLossWarps;
    }
    lanes = 32;
    while (lanes > 1 && lanes / 2 >= S) lanes /= 2;
    const int64_t even = (T + warps - 1) / warps;
    unit = static_cast<int>(std::min<int64_t>(std::max<int64_t>((even + 127) / 128 * 128, 128), 2048));
    if (unit > S) unit = static_cast<int>(S);
    chunks = static_cast<int>((S + unit - 1) / unit);
    const int64_t per_block = kLossWarps * (32 / lanes), units = B * chunks;
    blocks = cluster ? cluster : static_cast<int>(std::min<int64_t>((units + per_block - 1) / per_block, 4 * num_sms()));
    seq_blocks = cluster ? cluster : static_cast<int>(std::min<int64_t>((B + kLossWarps - 1) / kLossWarps, num_sms()));
  }
};

// Workspace of a (device, stream), grown on demand; every launch that uses it
// is on that stream.
static torch::Tensor loss_workspace(int64_t bytes) {
  static std::unordered_map<uint64_t, torch::Tensor> all;
  int dev = 0;
  cudaGetDevice(&dev);
  const auto opts = torch::TensorOptions().dtype(torch::kUInt8).device(torch::kCUDA, dev);
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None)
    return torch::empty({bytes}, opts);  // a graph keeps its own
  torch::Tensor& t = all[(static_cast<uint64_t>(dev) << 56) ^ reinterpret_cast<uint64_t>(stream())];
  if (!t.defined() || t.numel() < bytes) t = torch::empty({std::max<int64_t>(bytes, 1 << 16)}, opts);
  return t;
}

// Lays the phases' workspace out and launches `first` | ... | last.
template <bool POLICY>
static void launch_loss(LossParams& p, const LossPlan& plan) {
  const int64_t units = p.B * plan.chunks, blocks = std::max(plan.blocks, plan.seq_blocks);
  auto pad = [](int64_t n) { return (n + 255) / 256 * 256; };
  const torch::Tensor held = loss_workspace(pad(16 * units) + pad(16 * blocks) + pad(24 * blocks) + pad(4 * p.B));
  uint8_t* ws = held.data_ptr<uint8_t>();
  p.units = reinterpret_cast<double2*>(ws);
  p.totals = reinterpret_cast<double2*>(ws + pad(16 * units));
  p.sums = reinterpret_cast<double*>(ws + pad(16 * units) + pad(16 * blocks));
  uint8_t* per_seq = ws + pad(16 * units) + pad(16 * blocks) + pad(24 * blocks);
  p.coef = reinterpret_cast<float*>(per_seq);
  p.lengths = reinterpret_cast<int*>(per_seq);
  p.unit = plan.unit;
  p.chunks = plan.chunks;
  p.lanes = plan.lanes;
  const bool b_phase = !POLICY || (p.per_sequence && plan.chunks > 1);
  auto launch = [&](int phases, int blocks_, int cluster) {
    p.phases = phases;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks_);
    cfg.blockDim = dim3(kLossThreads);
    cfg.stream = stream();
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, answer_loss_kernel<POLICY>, static_cast<LossParams>(p));
    TORCH_CHECK(e == cudaSuccess, "answer_loss launch failed: ", cudaGetErrorString(e));
    count_launch();
  };
  if (plan.cluster) {
    p.parts = plan.cluster;
    launch(kA | (b_phase ? kB : 0) | kC | (POLICY ? kD : 0), plan.cluster, plan.cluster);
    return;
  }
  torch::Tensor tickets;
  if (POLICY) {
    tickets = arrival_counters(1);
    p.ticket = tickets.data_ptr<int>();
  }
  p.parts = b_phase ? plan.seq_blocks : plan.blocks;
  launch(kA, plan.blocks, 1);
  if (b_phase) launch(kB, plan.seq_blocks, 1);
  launch(kC | (POLICY ? kD : 0), plan.blocks, 1);
}

// Returns (loss [], dlogp [T], rewards [B]).
std::vector<torch::Tensor> preference_loss(torch::Tensor logp, c10::optional<torch::Tensor> ref,
                                           torch::Tensor targets, int64_t S, double beta, int64_t kind,
                                           double smoothing, bool average, int64_t ignore_index) {
  const int64_t B = check_batch(logp, targets, S);
  TORCH_CHECK(B % 2 == 0, "a preference batch needs an even number of sequences");
  TORCH_CHECK(kind >= kSigmoid && kind <= kIpo, "unknown preference loss");
  const c10::cuda::CUDAGuard guard(logp.device());
  auto lp = logp.contiguous(), tg = targets.contiguous();
  torch::Tensor rf;
  if (ref.has_value()) {
    check_tokens(*ref, logp.size(0), logp, "ref_logp");
    rf = ref->contiguous();
  }
  auto loss = torch::empty({}, lp.options()), dlogp = torch::empty_like(lp), rewards = torch::empty({B}, lp.options());
  if (B == 0) return {loss.zero_(), dlogp, rewards};
  LossParams p{};
  p.logp = lp.data_ptr<float>();
  p.ref = rf.defined() ? rf.data_ptr<float>() : nullptr;
  p.targets = tg.data_ptr<int64_t>();
  p.ignore = ignore_index;
  p.B = B;
  p.S = static_cast<int>(S);
  p.loss = loss.data_ptr<float>();
  p.dlogp = dlogp.data_ptr<float>();
  p.kind = static_cast<int>(kind);
  p.average = average;
  p.beta = beta;
  p.smoothing = smoothing;
  p.rewards = rewards.data_ptr<float>();
  launch_loss<false>(p, LossPlan(B, S));
  return {loss, dlogp, rewards};
}

// Returns (loss [], dlogp [T], stats [2]).
std::vector<torch::Tensor> policy_loss(torch::Tensor logp, torch::Tensor old, c10::optional<torch::Tensor> ref,
                                       torch::Tensor advantages, torch::Tensor targets, int64_t S, double clip_low,
                                       double clip_high, double kl_coef, bool per_sequence, int64_t ignore_index) {
  const int64_t B = check_batch(logp, targets, S), T = logp.size(0);
  const c10::cuda::CUDAGuard guard(logp.device());
  check_tokens(old, T, logp, "old_logp");
  auto lp = logp.contiguous(), od = old.contiguous(), tg = targets.contiguous();
  torch::Tensor rf;
  if (ref.has_value()) {
    check_tokens(*ref, T, logp, "ref_logp");
    rf = ref->contiguous();
  }
  const bool per_token = advantages.dim() == 1 && advantages.size(0) == T && T != B;
  check_tokens(advantages, per_token ? T : B, logp, "advantages");
  auto adv = advantages.contiguous();
  auto loss = torch::empty({}, lp.options()), dlogp = torch::empty_like(lp), stats = torch::empty({2}, lp.options());
  if (B == 0) return {loss.zero_(), dlogp, stats.zero_()};
  LossParams p{};
  p.logp = lp.data_ptr<float>();
  p.old = od.data_ptr<float>();
  p.ref = rf.defined() ? rf.data_ptr<float>() : nullptr;
  p.adv = adv.data_ptr<float>();
  p.targets = tg.data_ptr<int64_t>();
  p.ignore = ignore_index;
  p.B = B;
  p.S = static_cast<int>(S);
  p.loss = loss.data_ptr<float>();
  p.dlogp = dlogp.data_ptr<float>();
  p.adv_per_token = per_token;
  p.per_sequence = per_sequence;
  p.lo = static_cast<float>(std::log1p(-clip_low));
  p.hi = static_cast<float>(std::log1p(clip_high));
  p.edge_lo = static_cast<float>(1 - clip_low);
  p.edge_hi = static_cast<float>(1 + clip_high);
  p.kl_coef = static_cast<float>(kl_coef);
  p.stats = stats.data_ptr<float>();
  launch_loss<true>(p, LossPlan(B, S));
  return {loss, dlogp, stats};
}

}  // namespace t1
