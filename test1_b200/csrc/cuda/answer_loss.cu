// Losses on the log-probabilities of answer tokens, with their gradients:
// the preference loss of paired answers and the clipped policy loss.
//
// Both read [B, S] tokens (sequence after sequence) of which the targets
// mark the answers; entries of other tokens are never used, whatever they
// hold.  Both need a number per sequence or for the whole batch before the
// first gradient can be written (a pair's margin, the token count), so each
// is a pass that reduces and a pass that writes.
#include "common.cuh"

namespace t1 {

enum PreferenceKind : int { kSigmoid = 0, kHinge = 1, kIpo = 2 };

constexpr int kLossThreads = 256;
constexpr int kChunk = 4096;  // tokens of one sequence that a block takes

// Block-wide sum in fp64, every thread gets it.  `red` must hold 8 doubles.
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) t += red[w];
  return t;
}

// part[b * chunks + c] = (sum of logp - ref, count) over the chunk's answer
// tokens; ref and logp may be null (count only).
__global__ void __launch_bounds__(kLossThreads)
    answer_partials_kernel(const float* __restrict__ logp, const float* __restrict__ ref,
                           const int64_t* __restrict__ targets, int64_t ignore, int S, int chunks,
                           double2* __restrict__ part) {
  __shared__ double red[8];
  const int64_t b = blockIdx.x / chunks;
  const int c = blockIdx.x % chunks;
  const int s1 = min(S, (c + 1) * kChunk);
  double sum = 0;
  int n = 0;
  for (int s = c * kChunk + threadIdx.x; s < s1; s += kLossThreads) {
    const int64_t i = b * S + s;
    if (targets[i] == ignore) continue;
    ++n;
    if (logp != nullptr) sum += ref != nullptr ? logp[i] - ref[i] : logp[i];
  }
  sum = block_sum_f64(sum, red);
  const double cnt = block_sum_f64(n, red);
  if (threadIdx.x == 0) part[blockIdx.x] = make_double2(sum, cnt);
}

__device__ __forceinline__ double2 join_chunks(const double2* part, int64_t b, int chunks) {
  double2 t = make_double2(0, 0);
  for (int c = 0; c < chunks; ++c) {
    const double2 v = part[b * chunks + c];
    t.x += v.x;
    t.y += v.y;
  }
  return t;
}

// One block: margins, loss, rewards and the gradient coefficient of every
// sequence (its tokens' dlogp).
__global__ void __launch_bounds__(kLossThreads)
    preference_pairs_kernel(const double2* __restrict__ part, int chunks, int64_t P, int kind, double beta,
                            double eps, int average, float* __restrict__ coef, float* __restrict__ rewards,
                            float* __restrict__ loss) {
  __shared__ double red[8];
  double total = 0, live = 0;
  for (int64_t i = threadIdx.x; i < P; i += kLossThreads)
    live += join_chunks(part, i, chunks).y + join_chunks(part, i + P, chunks).y > 0 ? 1 : 0;
  live = fmax(1.0, block_sum_f64(live, red));
  for (int64_t i = threadIdx.x; i < P; i += kLossThreads) {
    const double2 ch = join_chunks(part, i, chunks), rj = join_chunks(part, i + P, chunks);
    const double pc = average ? 1 / fmax(1.0, ch.y) : 1, pr = average ? 1 / fmax(1.0, rj.y) : 1;
    const double m = ch.x * pc - rj.x * pr, z = beta * m;
    double l, d;
    if (kind == kSigmoid) {
      const double tail = log1p(exp(-fabs(z)));
      l = (1 - eps) * (fmax(-z, 0.0) + tail) + eps * (fmax(z, 0.0) + tail);
      d = beta * (eps / (1 + exp(-z)) - (1 - eps) / (1 + exp(z)));
    } else if (kind == kHinge) {
      l = fmax(1 - z, 0.0);
      d = z < 1 ? -beta : 0;
    } else {
      const double e = m - 0.5 / beta;
      l = e * e;
      d = 2 * e;
    }
    const bool counts = ch.y + rj.y > 0;
    if (counts) total += l;
    d = counts ? d / live : 0;
    coef[i] = static_cast<float>(d * pc);
    coef[i + P] = static_cast<float>(-d * pr);
    rewards[i] = static_cast<float>(beta * ch.x * pc);
    rewards[i + P] = static_cast<float>(beta * rj.x * pr);
  }
  total = block_sum_f64(total, red);
  if (threadIdx.x == 0) *loss = static_cast<float>(total / live);
}

__global__ void __launch_bounds__(kLossThreads)
    preference_grad_kernel(const int64_t* __restrict__ targets, int64_t ignore, int S, int chunks,
                           const float* __restrict__ coef, float* __restrict__ dlogp) {
  const int64_t b = blockIdx.x / chunks;
  const int c = blockIdx.x % chunks;
  const int s1 = min(S, (c + 1) * kChunk);
  const float d = coef[b];
  for (int s = c * kChunk + threadIdx.x; s < s1; s += kLossThreads)
    dlogp[b * S + s] = targets[b * S + s] != ignore ? d : 0.f;
}

// One block: weight of a token of sequence b in the loss; total[0] = answer tokens.
__global__ void __launch_bounds__(kLossThreads)
    policy_weights_kernel(const double2* __restrict__ part, int chunks, int64_t B, int per_sequence,
                          float* __restrict__ weight, double* __restrict__ total) {
  __shared__ double red[8];
  double n = 0, live = 0;
  for (int64_t b = threadIdx.x; b < B; b += kLossThreads) {
    const double k = join_chunks(part, b, chunks).y;
    n += k;
    live += k > 0 ? 1 : 0;
  }
  n = fmax(1.0, block_sum_f64(n, red));
  live = fmax(1.0, block_sum_f64(live, red));
  for (int64_t b = threadIdx.x; b < B; b += kLossThreads)
    weight[b] = static_cast<float>(per_sequence ? 1 / (fmax(1.0, join_chunks(part, b, chunks).y) * live) : 1 / n);
  if (threadIdx.x == 0) *total = n;
}

__global__ void __launch_bounds__(kLossThreads)
    policy_grad_kernel(const float* __restrict__ logp, const float* __restrict__ old, const float* __restrict__ ref,
                       const float* __restrict__ adv, int adv_per_token, const int64_t* __restrict__ targets,
                       int64_t ignore, int S, int chunks, float lo, float hi, float edge_lo, float edge_hi,
                       float kl_coef, const float* __restrict__ weight, float* __restrict__ dlogp,
                       double* __restrict__ out) {
  __shared__ double red[8];
  const int64_t b = blockIdx.x / chunks;
  const int c = blockIdx.x % chunks;
  const int s1 = min(S, (c + 1) * kChunk);
  const float w = weight[b];
  double loss = 0, kls = 0, cut = 0;
  for (int s = c * kChunk + threadIdx.x; s < s1; s += kLossThreads) {
    const int64_t i = b * S + s;
    float g = 0.f;
    if (targets[i] != ignore) {
      const float lp = logp[i], d = lp - old[i];
      const float a = adv[adv_per_token ? i : b];
      const float rho = expf(d);
      const bool over = d > hi, under = d < lo;
      const bool clipped = (a > 0.f && over) || (a < 0.f && under);
      float l = -a * (clipped ? (over ? edge_hi : edge_lo) : rho);
      g = clipped ? 0.f : -a * rho;
      if (ref != nullptr) {
        const float e = ref[i] - lp, x = expm1f(e), kl = x - e;
        l += kl_coef * kl;
        g -= kl_coef * x;
        kls += kl;
      }
      g *= w;
      loss += l;
      cut += clipped ? 1 : 0;
    }
    dlogp[i] = g;
  }
  loss = block_sum_f64(loss * w, red);
  kls = block_sum_f64(kls, red);
  cut = block_sum_f64(cut, red);
  if (threadIdx.x == 0) {
    out[3 * static_cast<int64_t>(blockIdx.x)] = loss;
    out[3 * static_cast<int64_t>(blockIdx.x) + 1] = kls;
    out[3 * static_cast<int64_t>(blockIdx.x) + 2] = cut;
  }
}

__global__ void __launch_bounds__(kLossThreads)
    policy_total_kernel(const double* __restrict__ out, int64_t blocks, const double* __restrict__ total,
                        float* __restrict__ loss, float* __restrict__ stats) {
  __shared__ double red[8];
  double v[3] = {0, 0, 0};
  for (int64_t i = threadIdx.x; i < blocks; i += kLossThreads)
    for (int k = 0; k < 3; ++k) v[k] += out[3 * i + k];
  for (int k = 0; k < 3; ++k) v[k] = block_sum_f64(v[k], red);
  if (threadIdx.x == 0) {
    *loss = static_cast<float>(v[0]);
    stats[0] = static_cast<float>(v[1] / *total);
    stats[1] = static_cast<float>(v[2] / *total);
  }
}

// ================================================================ host side
T1_BOUNDS_READER(answer_loss)

static void check_tokens(const torch::Tensor& t, int64_t T, const torch::Tensor& like, const char* what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), what, " must be on the device of logp");
  TORCH_CHECK(t.scalar_type() == torch::kFloat32, what, " has dtype ", t.scalar_type(), ", expected Float");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == T, what, " must have T entries");
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

static int64_t loss_blocks(int64_t B, int64_t S, int* chunks) {
  *chunks = static_cast<int>((S + kChunk - 1) / kChunk);
  const int64_t n = B * *chunks;
  TORCH_CHECK(n < INT32_MAX, "too many sequences");
  return n;
}

// Returns (loss [], dlogp [T], rewards [B]).
std::vector<torch::Tensor> preference_loss(torch::Tensor logp, c10::optional<torch::Tensor> ref,
                                           torch::Tensor targets, int64_t S, double beta, int64_t kind,
                                           double smoothing, bool average, int64_t ignore_index) {
  const int64_t B = check_batch(logp, targets, S);
  const c10::cuda::CUDAGuard guard(logp.device());
  auto lp = logp.contiguous(), tg = targets.contiguous();
  torch::Tensor rf;
  if (ref.has_value()) {
    check_tokens(*ref, logp.size(0), logp, "ref_logp");
    rf = ref->contiguous();
  }
  auto loss = torch::empty({}, lp.options()), dlogp = torch::empty_like(lp), rewards = torch::empty({B}, lp.options());
  if (B == 0) return {loss.zero_(), dlogp, rewards};
  int chunks;
  const int64_t blocks = loss_blocks(B, S, &chunks);
  auto part = torch::empty({2 * blocks}, lp.options().dtype(torch::kFloat64));
  auto coef = torch::empty({B}, lp.options());
  answer_partials_kernel<<<blocks, kLossThreads, 0, stream()>>>(
      lp.data_ptr<float>(), rf.defined() ? rf.data_ptr<float>() : nullptr, tg.data_ptr<int64_t>(), ignore_index, S,
      chunks, reinterpret_cast<double2*>(part.data_ptr<double>()));
  check_launch("answer_partials");
  preference_pairs_kernel<<<1, kLossThreads, 0, stream()>>>(
      reinterpret_cast<double2*>(part.data_ptr<double>()), chunks, B / 2, kind, beta, smoothing, average,
      coef.data_ptr<float>(), rewards.data_ptr<float>(), loss.data_ptr<float>());
  check_launch("preference_pairs");
  preference_grad_kernel<<<blocks, kLossThreads, 0, stream()>>>(tg.data_ptr<int64_t>(), ignore_index, S, chunks,
                                                                coef.data_ptr<float>(), dlogp.data_ptr<float>());
  check_launch("preference_grad");
  count_launch(3);
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
  int chunks;
  const int64_t blocks = loss_blocks(B, S, &chunks);
  auto ws = torch::empty({5 * blocks + 1}, lp.options().dtype(torch::kFloat64));
  auto part = reinterpret_cast<double2*>(ws.data_ptr<double>());
  double *out = ws.data_ptr<double>() + 2 * blocks, *total = out + 3 * blocks;
  auto weight = torch::empty({B}, lp.options());
  answer_partials_kernel<<<blocks, kLossThreads, 0, stream()>>>(nullptr, nullptr, tg.data_ptr<int64_t>(), ignore_index,
                                                                S, chunks, part);
  check_launch("answer_partials");
  policy_weights_kernel<<<1, kLossThreads, 0, stream()>>>(part, chunks, B, per_sequence, weight.data_ptr<float>(), total);
  check_launch("policy_weights");
  policy_grad_kernel<<<blocks, kLossThreads, 0, stream()>>>(
      lp.data_ptr<float>(), od.data_ptr<float>(), rf.defined() ? rf.data_ptr<float>() : nullptr, adv.data_ptr<float>(),
      per_token, tg.data_ptr<int64_t>(), ignore_index, S, chunks, static_cast<float>(std::log1p(-clip_low)),
      static_cast<float>(std::log1p(clip_high)), static_cast<float>(1 - clip_low), static_cast<float>(1 + clip_high),
      static_cast<float>(kl_coef), weight.data_ptr<float>(), dlogp.data_ptr<float>(), out);
  check_launch("policy_grad");
  policy_total_kernel<<<1, kLossThreads, 0, stream()>>>(out, blocks, total, loss.data_ptr<float>(), stats.data_ptr<float>());
  check_launch("policy_total");
  count_launch(4);
  return {loss, dlogp, stats};
}

}  // namespace t1
