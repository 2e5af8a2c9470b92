// Divergence of a student from its teacher on the teacher's likeliest tokens,
// and its gradient for the student's log-probabilities.
//
// Per row, with a_k = log p_k and b_k = log q_k of the listed tokens k and, with
// a tail, p_r = 1 - sum p_k and q_r = 1 - sum q_k of the rest (at least 2^-20):
//   forward  f(p, q) = q log(q / p)                     p f' = -q
//   reverse  f(p, q) = p log(p / q)                     p f' = p (a - b + 1)
//   jensen   f(p, q) = (p log(p/m) + q log(q/m)) / 2    p f' = p (a - log m) / 2,  m = (p + q) / 2
//   L = sum f,  dL/da_k = p_k f'(p_k) - p_k f'(p_r), the second term only above the floor
// Without a tail both are scaled to sum to 1 over the list first:
//   dL/da_k = p_k f'(p_k) - p_k sum_j p_j f'(p_j)
//
// What is left of 1 is the difference of two numbers that nearly agree where
// the list holds nearly all, so p and q are summed in 64 bits there (their
// exponentials too: 2^-24 of a p near 1 would be all of a rest of 1e-7).
//
// A warp per row, one read of the inputs.  The rows that take part are counted
// first, in a launch of its own, because every gradient is divided by their
// number.
#include "common.cuh"

namespace t1 {
namespace distil {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kFloor = 0x1p-20f;

enum Kind : int { kForward = 0, kReverse = 1, kJensen = 2 };

struct Params {
  const float* logp;       // [T, K]
  const void* teacher;     // [T, K]
  const int64_t* ids;      // [T, K]
  int64_t T;
  int K, kind;
  int* count;              // rows that take part
  int* ticket;             // blocks that are done
  double* sums;            // [blocks]
  float* loss;
  float* dlogp;            // [T, K]
  float* each;             // [T]
};

template <typename V>
__device__ __forceinline__ float as_float(const V* p);
template <>
__device__ __forceinline__ float as_float<float>(const float* p) {
  return __ldg(p);
}
template <>
__device__ __forceinline__ float as_float<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename V>
__global__ void __launch_bounds__(kThreads) count_kernel(const Params p) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int n = 0;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp; t < p.T; t += static_cast<int64_t>(gridDim.x) * kWarps) {
    bool any = false;
    for (int k = lane; k < p.K; k += 32)
      any = any || (p.ids[t * p.K + k] >= 0 && as_float(static_cast<const V*>(p.teacher) + t * p.K + k) > -INFINITY);
    n += __any_sync(0xffffffffu, any);
  }
  if (lane == 0 && n > 0) atomicAdd(p.count, n);
}

// f(p, q) and p f'(p) of an outcome, a = log p and b = log q.
__device__ __forceinline__ void divergence(int kind, float p, float q, float a, float b, float& f, float& g) {
  if (kind == kForward) {
    f = q > 0.f ? q * (b - a) : 0.f;
    g = -q;
  } else if (kind == kReverse) {
    f = p > 0.f ? p * (a - b) : 0.f;
    g = f + p;
  } else {
    const float log_m = logf(0.5f * (p + q));
    const float fp = p > 0.f ? 0.5f * p * (a - log_m) : 0.f;
    f = fp + (q > 0.f ? 0.5f * q * (b - log_m) : 0.f);
    g = fp;
  }
}

// PER entries a lane.
template <typename V, int PER, bool TAIL>
__global__ void __launch_bounds__(kThreads) loss_kernel(const Params p) {
  __shared__ double of_warp[kWarps];
  __shared__ int last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float scale = 1.f / static_cast<float>(max(1, *p.count));
  double sum = 0.0;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kWarps + warp; t < p.T; t += static_cast<int64_t>(gridDim.x) * kWarps) {
    float a[PER], b[PER];
    bool keep[PER];
    bool any = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int k = lane + 32 * j;
      const int64_t at = t * p.K + k;
      keep[j] = false;
      a[j] = b[j] = 0.f;
      if (k < p.K) {
        keep[j] = p.ids[at] >= 0;
        b[j] = as_float(static_cast<const V*>(p.teacher) + at);
        a[j] = __ldg(p.logp + at);
      }
      keep[j] = keep[j] && b[j] > -INFINITY;
      any = any || keep[j];
    }
    any = __any_sync(0xffffffffu, any);
    float pk[PER], qk[PER], g[PER];
    float loss = 0.f, rest = 0.f;  // rest: f'(p_r), without a tail sum p f'
    if (TAIL) {
      double ps = 0.0, qs = 0.0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const double pd = keep[j] ? exp(static_cast<double>(a[j])) : 0.0, qd = keep[j] ? exp(static_cast<double>(b[j])) : 0.0;
        ps += pd;
        qs += qd;
        pk[j] = static_cast<float>(pd);
        qk[j] = static_cast<float>(qd);
      }
      ps = 1.0 - warp_sum(ps);
      qs = 1.0 - warp_sum(qs);
      const float pr = fmaxf(static_cast<float>(ps), kFloor), qr = fmaxf(static_cast<float>(qs), kFloor);
      float fr, gr;
      divergence(p.kind, pr, qr, logf(pr), logf(qr), fr, gr);
      rest = ps > kFloor ? gr / pr : 0.f;
      if (lane == 0) loss = fr;
    } else {
      // scaled to sum to 1
      float am = -INFINITY, bm = -INFINITY;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (!keep[j]) continue;
        am = fmaxf(am, a[j]);
        bm = fmaxf(bm, b[j]);
      }
      am = warp_max(am);
      bm = warp_max(bm);
      float as = 0.f, bs = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        if (!keep[j]) continue;
        as += expf(a[j] - am);
        bs += expf(b[j] - bm);
      }
      am += logf(t1::warp_sum(as));
      bm += logf(t1::warp_sum(bs));
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        a[j] -= am;
        b[j] -= bm;
        pk[j] = keep[j] ? expf(a[j]) : 0.f;
        qk[j] = keep[j] ? expf(b[j]) : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      float f = 0.f;
      g[j] = 0.f;
      if (keep[j]) divergence(p.kind, pk[j], qk[j], a[j], b[j], f, g[j]);
      loss += f;
      if (!TAIL) rest += g[j];
    }
    loss = t1::warp_sum(loss);
    if (!TAIL) rest = t1::warp_sum(rest);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int k = lane + 32 * j;
      const int64_t at = t * p.K + k;
      if (k < p.K && !T1_OOB(at, p.T * p.K)) p.dlogp[at] = keep[j] ? (g[j] - pk[j] * rest) * scale : 0.f;
    }
    if (!any) loss = 0.f;
    if (lane == 0 && !T1_OOB(t, p.T)) p.each[t] = loss;
    sum += loss;
  }
  // the blocks' sums in their order, by the last one
  if (lane == 0) of_warp[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int w = 0; w < kWarps; ++w) sum += of_warp[w];
    __stcg(p.sums + blockIdx.x, sum);
    __threadfence();
    last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last || warp != 0) return;
  __threadfence();
  sum = 0.0;
  for (int i = lane; i < static_cast<int>(gridDim.x); i += 32) sum += __ldcg(p.sums + i);
  sum = warp_sum(sum);
  if (lane == 0) *p.loss = static_cast<float>(sum * scale);
}

}  // namespace distil

// ================================================================ host side
T1_BOUNDS_READER(distillation)

template <typename V, int PER>
static void launch_loss(const distil::Params& p, int blocks, bool tail) {
  if (tail) distil::loss_kernel<V, PER, true><<<blocks, distil::kThreads, 0, stream()>>>(p);
  else distil::loss_kernel<V, PER, false><<<blocks, distil::kThreads, 0, stream()>>>(p);
  check_launch("distillation_loss");
  count_launch();
}

template <typename V>
static void run_loss(const distil::Params& p, int blocks, bool tail) {
  distil::count_kernel<V><<<blocks, distil::kThreads, 0, stream()>>>(p);
  check_launch("distillation_loss");
  count_launch();
  if (p.K <= 32) launch_loss<V, 1>(p, blocks, tail);
  else if (p.K <= 64) launch_loss<V, 2>(p, blocks, tail);
  else if (p.K <= 128) launch_loss<V, 4>(p, blocks, tail);
  else launch_loss<V, 16>(p, blocks, tail);
}

// Returns (loss [], dlogp [T, K], divergence of every row [T]), fp32.
std::vector<torch::Tensor> distillation_loss(torch::Tensor logp, torch::Tensor teacher, torch::Tensor ids, int64_t kind,
                                             bool tail) {
  T1_CHECK_INPUT(logp, torch::kFloat32);
  TORCH_CHECK(teacher.is_cuda() && (teacher.scalar_type() == torch::kFloat32 || teacher.scalar_type() == torch::kBFloat16),
              "teacher_logp must be a float32 or bfloat16 CUDA tensor");
  T1_CHECK_INPUT(ids, torch::kInt64);
  TORCH_CHECK(logp.dim() == 2 && teacher.sizes() == logp.sizes() && ids.sizes() == logp.sizes(),
              "logp, teacher_logp and ids must be [T, K]");
  TORCH_CHECK(logp.size(1) >= 1 && logp.size(1) <= 512, "a list has 1 to 512 tokens");
  TORCH_CHECK(logp.size(0) < (1ll << 30), "at most 2^30 rows");
  TORCH_CHECK(teacher.device() == logp.device() && ids.device() == logp.device(), "operands must be on one device");
  TORCH_CHECK(kind >= 0 && kind <= 2, "unknown kind of divergence");
  const c10::cuda::CUDAGuard guard(logp.device());
  const int64_t T = logp.size(0), K = logp.size(1);
  auto f32 = logp.options();
  auto dlogp = torch::empty({T, K}, f32), each = torch::empty({T}, f32), loss = torch::zeros({}, f32);
  if (T == 0) return {loss, dlogp, each};
  auto lp = logp.contiguous(), te = teacher.contiguous(), id = ids.contiguous();
  const int blocks = static_cast<int>(std::min<int64_t>((T + distil::kWarps - 1) / distil::kWarps, 8 * num_sms()));
  auto counters = torch::zeros({2}, f32.dtype(torch::kInt32));
  auto sums = torch::empty({blocks}, f32.dtype(torch::kFloat64));
  distil::Params p{};
  p.logp = lp.data_ptr<float>();
  p.teacher = te.data_ptr();
  p.ids = id.data_ptr<int64_t>();
  p.T = T;
  p.K = static_cast<int>(K);
  p.kind = static_cast<int>(kind);
  p.count = counters.data_ptr<int>();
  p.ticket = p.count + 1;
  p.sums = sums.data_ptr<double>();
  p.loss = loss.data_ptr<float>();
  p.dlogp = dlogp.data_ptr<float>();
  p.each = each.data_ptr<float>();
  if (te.scalar_type() == torch::kFloat32) run_loss<float>(p, blocks, tail);
  else run_loss<__nv_bfloat16>(p, blocks, tail);
  return {loss, dlogp, each};
}

}  // namespace t1
