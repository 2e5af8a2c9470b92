// Divergence of a student from its teacher on the teacher's likeliest tokens,
// and its gradient for the student's log-probabilities.
//
// Per row, with a_k = log p_k and b_k = log q_k of the listed tokens k, d = b - a
// and, with a tail, p_r = 1 - sum p_k and q_r = 1 - sum q_k of the rest (at least
// 2^-20):
//   forward  f(p, q) = q d                                     p f' = -q
//   reverse  f(p, q) = -p d                                    p f' = f + p
//   jensen   f(p, q) = (p log(p/m) + q log(q/m)) / 2           p f' = p log(p/m) / 2
//            with m = (p + q) / 2, log(p/m) = -log((1 + e^d) / 2)
//   L = sum f,  dL/da_k = p_k f'(p_k) - p_k f'(p_r), the second term only above the floor
// Without a tail both are scaled to sum to 1 over the list first:
//   dL/da_k = p_k f'(p_k) - p_k sum_j p_j f'(p_j)
// Everything goes by d, the difference of two inputs, and not by logarithms of
// rounded probabilities: where student and teacher are near each other the
// terms cancel, and 2^-24 of a logarithm of 10 is more than is left of them.
//
// What is left of 1 is the difference of two numbers that nearly agree where
// the list holds nearly all, so p and q are summed in 64 bits there, from
// exponentials that are good to 2^-31 (2^-24 of a p near 1 would be all of a rest
// of 1e-7): a power from a table in 64 bits, times a short series of what is left
// of the exponent, below 0.003, for which 32 bits are enough.  The library's
// 64-bit exponential takes twice the instructions, and instructions bound this.
//
// G lanes have a row, PER entries each; the inputs are read once.  (Asking for
// them a round ahead takes the registers of half of the warps: 46 us for 65600
// rows of 64 against 40.)  65600 rows of 64 take 35 us (symmetric), 28 of them
// here: instructions bound it (19.8 M of warps, 71 % of the issue slots; forward
// 12.6 M, 61 %), not its 84 MB.
// Every gradient is divided by the number of rows that take part.  A batch that
// one cluster of 8 CTAs has in one round waits for the others' counts and then
// writes; a larger one is scaled by a second launch, out of L2.
#include "arrivals.cuh"
#include "programmatic.cuh"

#include <cooperative_groups.h>

namespace t1 {
namespace distil {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kFloor = 0x1p-20f;
constexpr int kExps = 128;  // steps of an octave in the table of exponentials

enum Kind : int { kForward = 0, kReverse = 1, kJensen = 2 };

struct Params {
  const float* logp;       // [T, K]
  const void* teacher;     // [T, K]
  bool teacher_bf16;
  const int64_t* ids;      // [T, K]
  int64_t T;
  int K, kind;
  Arrivals ticket;         // blocks that are done
  double* sums;            // [blocks]
  int* counts;             // [blocks]
  float* scale;            // 1 / rows that take part, for the second launch
  float* loss;
  float* dlogp;            // [T, K]
  float* each;             // [T]
  // what was allocated, for the bounds-checked build
  int64_t entries;         // of the inputs and dlogp
  int64_t rows;            // of each
  int blocks;              // of sums and counts
};

// Sums over G neighbouring lanes.
template <int G, typename V>
__device__ __forceinline__ V lanes_sum(V v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int G>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// log((1 + e^-x) / 2) for x >= 0, to a few 2^-24 of itself however small x is:
// with y = e^-x - 1 it is log(1 + y / 2) = 2 artanh(y / (4 + y)), |y / (4 + y)| < 1/3.
__device__ __forceinline__ float log_half_sum(float x) {
  // e^-x - 1: the exponential's series where the difference would cancel (its first term left out is 0.5^8 / 9!)
  float s = fmaf(x, 1.f / 40320, -1.f / 5040);
  s = fmaf(x, s, 1.f / 720);
  s = fmaf(x, s, -1.f / 120);
  s = fmaf(x, s, 1.f / 24);
  s = fmaf(x, s, -1.f / 6);
  s = fmaf(x, s, 0.5f);
  s = fmaf(x, s, -1.f);
  const float y = x < 0.5f ? x * s : __expf(-x) - 1.f;
  const float z = __fdividef(y, 4.f + y), z2 = z * z;
  float a = fmaf(z2, 2.f / 15, 2.f / 13);
  a = fmaf(z2, a, 2.f / 11);
  a = fmaf(z2, a, 2.f / 9);
  a = fmaf(z2, a, 2.f / 7);
  a = fmaf(z2, a, 2.f / 5);
  a = fmaf(z2, a, 2.f / 3);
  a = fmaf(z2, a, 2.f);
  return z * a;
}

// f(p, q) and p f'(p) of an outcome, d = log(q / p), finite where it is multiplied by 0.
__device__ __forceinline__ void divergence(int kind, float p, float q, float d, float& f, float& g) {
  if (kind == kForward) {
    f = q * d;
    g = -q;
  } else if (kind == kReverse) {
    f = -p * d;
    g = f + p;
  } else {
    const float l = log_half_sum(fabsf(d));
    g = -0.5f * p * (fmaxf(d, 0.f) + l);
    f = fmaf(-0.5f * q, fmaxf(-d, 0.f) + l, g);
  }
}

// ONE: one cluster has the batch in one round.  VEC: four neighbouring entries
// a load (K a multiple of 4, tensors on 16 bytes).
template <int G, int PER, bool VEC, bool TAIL, bool ONE>
__global__ void __launch_bounds__(kThreads, PER > 8 ? 1 : 4) loss_kernel(const Params p) {
  __shared__ double exps[kExps];  // 2^(j / 128)
  __shared__ double of_warp[kWarps];
  __shared__ int live_of_warp[kWarps];
  __shared__ double of_cta[8];    // of the cluster
  __shared__ int live_of_cta[8];
  __shared__ int last;
  constexpr int kRows = 32 / G;   // of a warp
  constexpr int kStep = VEC ? 4 : 1;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, of_row = lane % G;
  if (ONE) tell_started();
  // entry j of the lane
  auto entry = [&](int j) { return VEC ? 4 * of_row + 4 * G * (j / 4) + j % 4 : of_row + G * j; };
  const int64_t t_step = static_cast<int64_t>(gridDim.x) * kWarps * kRows;
  const int64_t t_first = (static_cast<int64_t>(blockIdx.x) * kWarps + warp) * kRows;
  int64_t t0 = t_first;
  float in_a[PER], in_b[PER];
  int64_t in_id[PER];
  auto load = [&] {
    const int64_t row = (t0 + lane / G) * p.K;
    const int cols = t0 + lane / G < p.T ? p.K : 0;
#pragma unroll
    for (int j = 0; j < PER; j += kStep) {
      const int k = entry(j);
      if (VEC) {
        longlong2 i0 = make_longlong2(-1, -1), i1 = i0;
        float4 a4 = make_float4(0.f, 0.f, 0.f, 0.f), b4 = a4;
        if (k < cols && !T1_OOB(row + k + 3, p.entries)) {
          i0 = __ldcs(reinterpret_cast<const longlong2*>(p.ids + row + k));
          i1 = __ldcs(reinterpret_cast<const longlong2*>(p.ids + row + k) + 1);
          a4 = __ldcs(reinterpret_cast<const float4*>(p.logp + row + k));
          if (p.teacher_bf16) {
            const uint2 u = __ldcs(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.teacher) + row + k));
            b4 = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                             __uint_as_float(u.y & 0xffff0000u));
          } else {
            b4 = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(p.teacher) + row + k));
          }
        }
        in_id[j] = i0.x, in_id[j + 1] = i0.y, in_id[j + 2] = i1.x, in_id[j + 3] = i1.y;
        in_a[j] = a4.x, in_a[j + 1] = a4.y, in_a[j + 2] = a4.z, in_a[j + 3] = a4.w;
        in_b[j] = b4.x, in_b[j + 1] = b4.y, in_b[j + 2] = b4.z, in_b[j + 3] = b4.w;
      } else {
        const bool in = k < cols && !T1_OOB(row + k, p.entries);
        in_id[j] = in ? __ldcs(p.ids + row + k) : -1;
        in_a[j] = in ? __ldcs(p.logp + row + k) : 0.f;
        in_b[j] = !in              ? 0.f
                    : p.teacher_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.teacher)[row + k])
                                     : __ldcs(static_cast<const float*>(p.teacher) + row + k);
      }
    }
  };
  if (ONE) load();
  if (TAIL) {
    if (threadIdx.x < kExps) exps[threadIdx.x] = exp2(threadIdx.x / static_cast<double>(kExps));
    __syncthreads();
  }
  if (!ONE) clear_arrivals(p.ticket);

  // exp(v) for v <= about 1
  auto exp64 = [&](float at) {
    constexpr float kRound = 12582912.f;  // 1.5 2^23: adding it leaves a whole number in the low bits
    const float v = at < -600.f ? -600.f : at;  // NaN stays
    const float y = fmaf(v, 1.4426950408889634f * kExps, kRound);
    const int j = __float_as_int(y) - 0x4b400000;
    const float n = y - kRound;
    // v - n ln 2 / 128, the constant in two parts
    const float r = fmaf(n, 1.4880111e-11f, fmaf(n, -0.00541521236f, v));
    const float e = fmaf(fmaf(r, 1.f / 6, 0.5f) * r, r, r);
    const double base = exps[j & (kExps - 1)];
    const double power = __hiloint2double(__double2hiint(base) + ((j >> 7) << 20), __double2loint(base));
    return fma(power, static_cast<double>(e), power);
  };
  static_assert(kExps == 128, "j >> 7");

  double sum = 0.0;
  int rows = 0;
  float g[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) g[j] = 0.f;
  auto store = [&](int64_t t, float scale) {
    const int64_t row = t * p.K;
    const int cols = t < p.T ? p.K : 0;
#pragma unroll
    for (int j = 0; j < PER; j += kStep) {
      const int k = entry(j);
      if (k >= cols || T1_OOB(row + k + kStep - 1, p.entries)) continue;
      if (VEC) *reinterpret_cast<float4*>(p.dlogp + row + k) = make_float4(g[j] * scale, g[j + 1] * scale, g[j + 2] * scale, g[j + 3] * scale);
      else p.dlogp[row + k] = g[j] * scale;
    }
  };
  // An entry left out has the logarithm of no probability at all, in both, and so no part in the sums of a tail.  Without
  // one only differences of logarithms count, which may all lie below this, and `kept` says what takes part.
  constexpr float kNothing = -1e4f;
  while (t0 < p.T) {
    if (!ONE) load();
    const int64_t t = t0 + lane / G;
    float a[PER], b[PER];
    unsigned kept = 0;  // bit j: entry j
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const bool keep = in_id[j] >= 0 && in_b[j] > -INFINITY;
      a[j] = keep ? in_a[j] : kNothing;
      b[j] = keep ? in_b[j] : kNothing;
      kept |= static_cast<unsigned>(keep) << j;
    }
    t0 += t_step;
    const unsigned lanes = __ballot_sync(0xffffffffu, kept != 0);
    const bool live = (G == 32 ? lanes : (lanes >> (lane & ~(G - 1))) & ((1u << (G & 31)) - 1)) != 0;
    float pk[PER], qk[PER];
    float loss = 0.f, rest = 0.f;  // rest: f'(p_r), without a tail sum p f'
    float shift = 0.f;             // of d
    if (TAIL) {
      double ps = 0.0, qs = 0.0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const double pd = exp64(a[j]), qd = exp64(b[j]);
        ps += pd;
        qs += qd;
        pk[j] = static_cast<float>(pd);
        qk[j] = static_cast<float>(qd);
      }
      ps = 1.0 - lanes_sum<G>(ps);
      qs = 1.0 - lanes_sum<G>(qs);
      // a student's NaN is above no floor and below none
      const float pr = ps <= kFloor ? kFloor : static_cast<float>(ps), qr = fmaxf(static_cast<float>(qs), kFloor);
      float fr, gr;
      divergence(p.kind, pr, qr, logf(__fdividef(qr, pr)), fr, gr);
      rest = ps <= kFloor ? 0.f : __fdividef(gr, pr);
      if (of_row == 0) loss = fr;
    } else {
      // scaled to sum to 1
      float am = -INFINITY, bm = -INFINITY, as = 0.f, bs = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const bool in = kept >> j & 1;
        am = fmaxf(am, in ? a[j] : -INFINITY);
        bm = fmaxf(bm, in ? b[j] : -INFINITY);
      }
      am = lanes_max<G>(am);
      bm = lanes_max<G>(bm);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const bool in = kept >> j & 1;
        pk[j] = in ? expf(a[j] - am) : 0.f;
        qk[j] = in ? expf(b[j] - bm) : 0.f;
        as += pk[j];
        bs += qk[j];
      }
      as = lanes_sum<G>(as);
      bs = lanes_sum<G>(bs);
      shift = live ? (bm - am) + logf(bs / as) : 0.f;
      as = live ? 1.f / as : 0.f;
      bs = live ? 1.f / bs : 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        pk[j] *= as;
        qk[j] *= bs;
      }
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      float f, d = (b[j] - a[j]) - shift;
      // of a student's -inf as much as there is where it has no weight; q times it is infinite
      if (d > 3e38f && !(p.kind == kForward && qk[j] > 0.f)) d = 3e38f;
      divergence(p.kind, pk[j], qk[j], d, f, g[j]);
      loss += f;
      if (!TAIL) rest += g[j];
    }
    loss = lanes_sum<G>(loss);
    if (!TAIL) rest = lanes_sum<G>(rest);
#pragma unroll
    for (int j = 0; j < PER; ++j) g[j] = kept >> j & 1 ? fmaf(-pk[j], rest, g[j]) : 0.f;
    if (of_row == 0) {
      if (t < p.T && !T1_OOB(t, p.rows)) p.each[t] = loss;
      sum += loss;
      rows += live;
    }
    if (!ONE) store(t, 1.f);
  }
  sum = lanes_sum<32>(sum);
  rows = __reduce_add_sync(0xffffffffu, rows);
  if (lane == 0) {
    of_warp[warp] = sum;
    live_of_warp[warp] = rows;
  }
  __syncthreads();
  sum = 0.0;
  rows = 0;
  for (int w = 0; w < kWarps; ++w) {
    sum += of_warp[w];
    rows += live_of_warp[w];
  }
  if (ONE) {
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned ctas = cluster.num_blocks();
    wait_started();
    if (threadIdx.x < ctas && !T1_OOB(ctas - 1, 8)) {
      cluster.map_shared_rank(of_cta, threadIdx.x)[cluster.block_rank()] = sum;
      cluster.map_shared_rank(live_of_cta, threadIdx.x)[cluster.block_rank()] = rows;
    }
    cluster.sync();
    sum = 0.0;
    rows = 0;
    for (unsigned r = 0; r < ctas; ++r) {
      sum += of_cta[r];
      rows += live_of_cta[r];
    }
    const float scale = 1.f / static_cast<float>(max(1, rows));
    store(t_first + lane / G, scale);
    if (blockIdx.x == 0 && threadIdx.x == 0) *p.loss = static_cast<float>(sum * scale);
    return;
  }
  // the blocks' sums in their order, by the last one
  if (threadIdx.x == 0) {
    if (!T1_OOB(blockIdx.x, p.blocks)) {
      __stcg(p.sums + blockIdx.x, sum);
      __stcg(p.counts + blockIdx.x, rows);
    }
    __threadfence();
    last = atomicAdd(p.ticket.use, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last || warp != 0) return;
  __threadfence();
  sum = 0.0;
  rows = 0;
  for (int i = lane; i < static_cast<int>(gridDim.x); i += 32) {
    if (T1_OOB(i, p.blocks)) continue;
    sum += __ldcg(p.sums + i);
    rows += __ldcg(p.counts + i);
  }
  sum = lanes_sum<32>(sum);
  rows = __reduce_add_sync(0xffffffffu, rows);
  const float scale = 1.f / static_cast<float>(max(1, rows));
  if (lane == 0) {
    *p.loss = static_cast<float>(sum * scale);
    *p.scale = scale;
  }
}

// dlogp times the scale; dlogp is freshly allocated and so begins on 16 bytes.
__global__ void __launch_bounds__(kThreads) scale_kernel(float* dlogp, int64_t n, int64_t entries, const float* scale) {
  const float s = *scale;
  const int64_t vecs = n / 4, step = static_cast<int64_t>(gridDim.x) * kThreads;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  for (int64_t i = i0; i < vecs; i += step) {
    if (T1_OOB(4 * i + 3, entries)) continue;
    float4 v = reinterpret_cast<float4*>(dlogp)[i];
    v = make_float4(v.x * s, v.y * s, v.z * s, v.w * s);
    reinterpret_cast<float4*>(dlogp)[i] = v;
  }
  if (i0 < n - 4 * vecs && !T1_OOB(4 * vecs + i0, entries)) dlogp[4 * vecs + i0] *= s;
}

}  // namespace distil

// ================================================================ host side
T1_BOUNDS_READER(distillation)

template <int G, int PER, bool VEC>
static void launch_loss(distil::Params& p, bool tail) {
  const int64_t per_block = distil::kWarps * (32 / G), blocks_one = (p.T + per_block - 1) / per_block;
  if (blocks_one <= 8) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks_one);
    cfg.blockDim = dim3(distil::kThreads);
    cfg.stream = stream();
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = blocks_one;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    auto kern = tail ? distil::loss_kernel<G, PER, VEC, true, true> : distil::loss_kernel<G, PER, VEC, false, true>;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<const distil::Params>(p));
    TORCH_CHECK(e == cudaSuccess, "distillation_loss launch failed: ", cudaGetErrorString(e));
    count_launch();
    return;
  }
  const int blocks = static_cast<int>(std::min<int64_t>(blocks_one, 8 * num_sms()));
  auto ws = torch::empty({2 * blocks + 1}, torch::TensorOptions().dtype(torch::kFloat64).device(torch::kCUDA, at::cuda::current_device()));
  p.sums = ws.data_ptr<double>();
  p.counts = reinterpret_cast<int*>(p.sums + blocks);
  p.blocks = blocks;
  p.scale = reinterpret_cast<float*>(p.sums + 2 * blocks);
  ArrivalCounters counters(1);
  p.ticket = counters.arrivals;
  auto kern = tail ? distil::loss_kernel<G, PER, VEC, true, false> : distil::loss_kernel<G, PER, VEC, false, false>;
  kern<<<blocks, distil::kThreads, 0, stream()>>>(p);
  check_launch("distillation_loss");
  counters.launched();
  const int64_t n = p.T * p.K;
  distil::scale_kernel<<<static_cast<int>(std::min<int64_t>((n / 4 + distil::kThreads) / distil::kThreads, 8 * num_sms())),
                         distil::kThreads, 0, stream()>>>(p.dlogp, n, p.entries, p.scale);
  check_launch("distillation_loss");
  count_launch(2);
}

template <int G, int PER>
static void launch_loss(distil::Params& p, bool tail, bool vec) {
  if (vec) launch_loss<G, PER, true>(p, tail);
  else launch_loss<G, PER, false>(p, tail);
}

// Few lanes and many entries each, as far as registers go: what a row costs
// besides its entries is shared by more of them.
static void run_loss(distil::Params& p, bool tail) {
  const auto at = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
  const bool vec = p.K % 4 == 0 && (at(p.logp) | at(p.teacher) | at(p.ids) | at(p.dlogp)) % 16 == 0;
  if (p.K <= 8) launch_loss<8, 1, false>(p, tail);
  else if (p.K <= 32) launch_loss<8, 4>(p, tail, vec);
  else if (p.K <= 64) launch_loss<8, 8>(p, tail, vec);
  else if (p.K <= 128) launch_loss<16, 8>(p, tail, vec);
  else launch_loss<32, 16>(p, tail, vec);
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
  auto dlogp = torch::empty({T, K}, f32), each = torch::empty({T}, f32);
  if (T == 0) return {torch::zeros({}, f32), dlogp, each};
  auto loss = torch::empty({}, f32);
  auto lp = logp.contiguous(), te = teacher.contiguous(), id = ids.contiguous();
  distil::Params p{};
  p.logp = lp.data_ptr<float>();
  p.teacher = te.data_ptr();
  p.ids = id.data_ptr<int64_t>();
  p.T = T;
  p.K = static_cast<int>(K);
  p.kind = static_cast<int>(kind);
  p.loss = loss.data_ptr<float>();
  p.dlogp = dlogp.data_ptr<float>();
  p.each = each.data_ptr<float>();
  p.entries = dlogp.numel();
  p.rows = each.numel();
  p.teacher_bf16 = te.scalar_type() == torch::kBFloat16;
  run_loss(p, tail);
  return {loss, dlogp, each};
}

}  // namespace t1
