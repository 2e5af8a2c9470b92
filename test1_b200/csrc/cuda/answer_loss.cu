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
// One launch runs them all, with a barrier of its blocks between the phases:
// a launch of each phase costs 4 us of the host's time.  Up to 32 K tokens the
// blocks are one cluster, whose barrier is the hardware's; above that they are
// a cooperative grid of at most two blocks per SM (5 us more to launch, 1.5
// us a barrier).  A unit belongs to a warp or, for sequences shorter than 32
// tokens, to the fewest lanes that hold one.  Sums are carried in fp64 and
// joined in a fixed order: two runs give the same bits.
//
// Measured on a B200: 10 us up to 32 K tokens (the host's time), 14-18 us up to
// 1 M (latencies of the phases and barriers), 34 us for 4.2 M policy tokens
// (A 8 us, C 17 us at 4.2 TB/s; all bytes once at the copy rate are 14.5 us).
#include "arrivals.cuh"
#include "common.cuh"
#include "sm100.cuh"

#include <ATen/cuda/CUDAGraphsUtils.cuh>

#include <optional>
#include <string>
#include <unordered_map>

namespace t1 {

torch::Tensor& gemm_error_word();

enum PreferenceKind : int { kSigmoid = 0, kHinge = 1, kIpo = 2 };

struct LossParams {
  const float *logp, *ref, *old, *adv;
  const int64_t* targets;
  int64_t ignore;
  int64_t B;
  int S;
  int unit, chunks;        // tokens of a unit, units of a sequence
  int lanes;               // lanes of a unit: 32, or the power of two >= S
  int vectors;             // 16-byte vectors of tokens
  int lengths_phase;       // policy: phase B takes place
  Arrivals arrivals;       // the grid barrier's counter; none: the blocks are one cluster
  int* err;
  uint8_t* answer;         // [T] phase A's finding, an eighth of the targets to read again
  int64_t units_n;         // units and blocks that the workspace has room for
  int blocks_n;
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
  float* stats;            // [2]
};

constexpr int kLossThreads = 512;
constexpr int kLossWarps = kLossThreads / 32;
constexpr int kLossPerSm = 2;  // blocks of an SM
constexpr int kAhead = 4;  // tokens of a lane whose loads are issued together

// Sum over a warp's lanes, every lane gets it.
__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Sums {
  double v[3];
};

// Block-wide sums in fp64; the first warp gets them.
template <int N>
__device__ __forceinline__ Sums block_sums(Sums s, Sums* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int k = 0; k < N; ++k) s.v[k] = warp_sum_f64(s.v[k]);
  __syncthreads();
  if (lane == 0) red[warp] = s;
  __syncthreads();
  if (warp != 0) return s;
#pragma unroll
  for (int k = 0; k < N; ++k) s.v[k] = warp_sum_f64(lane < kLossWarps ? red[lane].v[k] : 0.0);
  return s;
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
    if (T1_OOB(b * p.chunks + c, p.units_n)) continue;
    const double2 v = __ldcg(&p.units[b * p.chunks + c]);
    t.x += v.x;
    t.y += v.y;
  }
  return make_double2(group_sum(t.x, by), group_sum(t.y, by));
}

// The blocks' totals added up, for every thread.
__device__ __forceinline__ double2 join_totals(const LossParams& p, Sums* red) {
  Sums s{{0, 0, 0}};
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += kLossThreads) {
    const double2 v = __ldcg(&p.totals[i]);
    s.v[0] += v.x;
    s.v[1] += v.y;
  }
  s = block_sums<2>(s, red);
  __syncthreads();
  if (threadIdx.x == 0) red[0] = s;
  __syncthreads();
  return make_double2(red[0].v[0], red[0].v[1]);
}

__device__ __forceinline__ void write_totals(const LossParams& p, double x, double y, Sums* red) {
  const Sums s = block_sums<2>(Sums{{x, y, 0}}, red);
  if (threadIdx.x == 0 && !T1_OOB(blockIdx.x, p.blocks_n)) __stcg(&p.totals[blockIdx.x], make_double2(s.v[0], s.v[1]));
}

// The warps' walk over units: body(unit, sequence, first token, tokens, lane
// of the unit), with all lanes of a warp in step; unit is -1 and tokens 0 for
// lanes that have none in a warp's last round.
template <class F>
__device__ __forceinline__ void for_units(const LossParams& p, F body) {
  const int per_warp = 32 / p.lanes, in_warp = threadIdx.x & 31;
  const int64_t count = p.B * p.chunks, step = static_cast<int64_t>(gridDim.x) * kLossWarps * per_warp;
  for (int64_t u0 = (static_cast<int64_t>(blockIdx.x) * kLossWarps + (threadIdx.x >> 5)) * per_warp; u0 < count; u0 += step) {
    const int64_t u = u0 + in_warp / p.lanes;
    const int64_t b = u / p.chunks;
    const int s0 = static_cast<int>(u - b * p.chunks) * p.unit, len = min(p.unit, p.S - s0);
    if (u < count && !T1_OOB(u, p.units_n) && !T1_OOB(len - 1, p.S) && !T1_OOB(b * p.S + s0 + len - 1, p.B * p.S)) {
      body(u, b, b * p.S + s0, len, in_warp & (p.lanes - 1));
    } else {
      body(-1, 0, 0, 0, in_warp & (p.lanes - 1));
    }
  }
}

// Four tokens of a lane, loaded and stored together.  STEP 1: neighbours in
// 16-byte vectors (sequences and units of a multiple of 4 tokens, aligned
// tensors); 32 and 0: a token per lane and round, the other lanes' between
// them (0: `lanes` of them), past the unit's end skipped unless `full`.
template <int STEP>
struct Four {
  int first, step, len;
  bool full;
  __device__ bool in(int k) const { return STEP == 1 || full || first + k * step < len; }
  __device__ int at(int k) const { return first + k * (STEP > 0 ? STEP : step); }
  __device__ void load(const float* p, float (&v)[kAhead], float other) const {
    if (STEP == 1) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(p + first));
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = in(k) ? __ldg(p + at(k)) : other;
    }
  }
  __device__ void load(const int64_t* p, int64_t (&v)[kAhead], int64_t other) const {
    if (STEP == 1) {
      const longlong2 f = __ldg(reinterpret_cast<const longlong2*>(p + first));
      const longlong2 g = __ldg(reinterpret_cast<const longlong2*>(p + first + 2));
      v[0] = f.x; v[1] = f.y; v[2] = g.x; v[3] = g.y;
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = in(k) ? __ldg(p + at(k)) : other;
    }
  }
  __device__ void load(const uint8_t* p, bool (&v)[kAhead]) const {
    if (STEP == 1) {
      const uchar4 f = *reinterpret_cast<const uchar4*>(p + first);
      v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = in(k) ? p[at(k)] : 0;
    }
  }
  __device__ void store(uint8_t* p, const bool (&v)[kAhead]) const {
    if (STEP == 1) {
      *reinterpret_cast<uchar4*>(p + first) = make_uchar4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (in(k)) p[at(k)] = v[k];
    }
  }
  __device__ void store(float* p, const float (&v)[kAhead]) const {
    if (STEP == 1) {
      *reinterpret_cast<float4*>(p + first) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (in(k)) p[at(k)] = v[k];
    }
  }
};
static_assert(kAhead == 4, "Four");

// Calls body with each four of the lane's tokens of a unit.
template <class F>
__device__ __forceinline__ void for_fours(const LossParams& p, int len, int lane, F body) {
  if (p.vectors) {
    for (int s = 4 * lane; s < len; s += 4 * 32)
      if (!T1_OOB(s + 3, len)) body(Four<1>{s, 1, len, true});
  } else if (p.lanes == 32) {
    int s = lane;
    for (; s - lane + 32 * kAhead <= len; s += 32 * kAhead) body(Four<32>{s, 32, len, true});
    if (s < len) body(Four<32>{s, 32, len, false});
  } else {
    for (int s = lane; s < len; s += kAhead * p.lanes) body(Four<0>{s, p.lanes, len, false});
  }
}

// ------------------------------------------------------------------ phase A
template <bool POLICY>
__device__ __forceinline__ void count_phase(const LossParams& p, Sums* red) {
  double tokens = 0, live = 0;
  for_units(p, [&](int64_t u, int64_t, int64_t i0, int len, int lane) {
    double sum = 0;
    int n = 0;
    const int64_t* targets = p.targets + i0;
    const float *logp = p.logp + i0, *ref = p.ref + i0;
    uint8_t* answer = p.answer + i0;
    for_fours(p, len, lane, [&](const auto& four) {
      int64_t t[kAhead];
      float v[kAhead] = {}, r[kAhead] = {}, part = 0.f;
      bool ok[kAhead];
      four.load(targets, t, p.ignore);
      if (!POLICY) four.load(logp, v, 0.f);
      if (!POLICY && p.ref != nullptr) four.load(ref, r, 0.f);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        ok[k] = t[k] != p.ignore;
        n += ok[k];
        if (!POLICY) part += ok[k] ? v[k] - r[k] : 0.f;
      }
      four.store(answer, ok);
      sum += part;
    });
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
__device__ __forceinline__ void pairs_phase(const LossParams& p, Sums* red) {
  const int64_t P = p.B / 2;
  // a thread for a pair of few units, a warp for one of many
  const int by = p.chunks <= 4 ? 1 : 32, lane = threadIdx.x & (by - 1);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kLossThreads / by;
  double loss = 0, live = 0;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * kLossThreads + threadIdx.x) / by; i < P; i += step) {
    if (T1_OOB(i + P, p.B)) continue;
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

__device__ __forceinline__ void lengths_phase(const LossParams& p, Sums* red) {
  const int lane = threadIdx.x & 31;
  double tokens = 0, live = 0;
  for (int64_t b = static_cast<int64_t>(blockIdx.x) * kLossWarps + (threadIdx.x >> 5); b < p.B; b += static_cast<int64_t>(gridDim.x) * kLossWarps) {
    const double n = join_units(p, b, lane, 32).y;
    if (lane != 0 || T1_OOB(b, p.B)) continue;
    __stcg(&p.lengths[b], static_cast<int>(n));
    tokens += n;
    live += n > 0 ? 1 : 0;
  }
  write_totals(p, tokens, live, red);
}

// ------------------------------------------------------------------ phase C
__device__ __forceinline__ void preference_grad_phase(const LossParams& p, Sums* red) {
  const double2 total = join_totals(p, red);
  const double pairs = fmax(1.0, total.y);
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.loss = static_cast<float>(total.x / pairs);
  for_units(p, [&](int64_t u, int64_t b, int64_t i0, int len, int lane) {
    if (u < 0) return;
    const float d = static_cast<float>(__ldcg(&p.coef[b]) / pairs);
    const uint8_t* answer = p.answer + i0;
    float* dlogp = p.dlogp + i0;
    for_fours(p, len, lane, [&](const auto& four) {
      bool ok[kAhead];
      float g[kAhead];
      four.load(answer, ok);
#pragma unroll
      for (int k = 0; k < kAhead; ++k) g[k] = ok[k] ? d : 0.f;
      four.store(dlogp, g);
    });
  });
}

// A token's clipped term for one advantage: past log(1 +- clip) on the side
// that the advantage pushes to, the loss is flat.  The log ratio decides, so
// the same tokens are clipped whatever exp's rounding does at the edge.
struct Clip {
  float minus_a, sign, past, flat;
  __device__ Clip(const LossParams& p, float a)
      : minus_a(-a), sign(a > 0.f ? 1.f : -1.f), past(a > 0.f ? p.hi : a < 0.f ? -p.lo : INFINITY),
        flat(-a * (a > 0.f ? p.edge_hi : p.edge_lo)) {}
};

// exp(e) - 1 and kl = exp(e) - 1 - e: kl's series up to e^7 for small e, where
// the differences would keep no digit (the first term left out is below 2^-25
// of the sum).  Elsewhere exp(e) - 1 comes first: it is at most 1 in size
// where e is far below 0, and kl + e would not give it back.
__device__ __forceinline__ float kl_term(float e, float& exp_m1) {
  float s = fmaf(e, 1.f / 5040, 1.f / 720);
  s = fmaf(e, s, 1.f / 120);
  s = fmaf(e, s, 1.f / 24);
  s = fmaf(e, s, 1.f / 6);
  s = fmaf(e, s, 0.5f);
  const bool near = fabsf(e) < 0.25f;
  const float kl = s * e * e;
  exp_m1 = near ? kl + e : __expf(e) - 1.f;
  return near ? kl : exp_m1 - e;
}

__device__ __forceinline__ void policy_grad_phase(const LossParams& p, Sums* red) {
  const double2 total = join_totals(p, red);
  const double tokens = fmax(1.0, total.x), live = fmax(1.0, total.y);
  const float token_weight = static_cast<float>(1 / tokens);
  double loss = 0, kls = 0;
  int cut = 0;
  for_units(p, [&](int64_t u, int64_t b, int64_t i0, int len, int lane) {
    if (u < 0) return;
    float w = token_weight;
    if (p.per_sequence) {
      const double n = p.chunks == 1 ? __ldcg(&p.units[u]).y : static_cast<double>(__ldcg(&p.lengths[b]));
      w = static_cast<float>(1 / (fmax(1.0, n) * live));
    }
    Clip clip(p, p.adv_per_token ? 0.f : p.adv[b]);
    double unit_loss = 0;
    const float *logp = p.logp + i0, *old = p.old + i0, *ref = p.ref + i0, *adv = p.adv + i0;
    const uint8_t* answer = p.answer + i0;
    float* dlogp = p.dlogp + i0;
    for_fours(p, len, lane, [&](const auto& four) {
      bool ok[kAhead];
      float lp[kAhead], od[kAhead], rf[kAhead], a[kAhead], part = 0.f, kl_part = 0.f;
      four.load(answer, ok);
      four.load(logp, lp, 0.f);
      four.load(old, od, 0.f);
      if (p.ref != nullptr) four.load(ref, rf, 0.f);
      if (p.adv_per_token) four.load(adv, a, 0.f);
      float g[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (p.adv_per_token) clip = Clip(p, a[k]);
        const float d = lp[k] - od[k], grad = clip.minus_a * __expf(d);
        const bool clipped = clip.sign * d > clip.past;
        float l = clipped ? clip.flat : grad;
        g[k] = clipped ? 0.f : grad;
        if (p.ref != nullptr) {
          float exp_m1;
          const float e = rf[k] - lp[k], kl = kl_term(e, exp_m1);
          l = fmaf(p.kl_coef, kl, l);
          g[k] = fmaf(-p.kl_coef, exp_m1, g[k]);
          if (ok[k]) kl_part += kl;
        }
        if (ok[k]) part += l;
        cut += ok[k] && clipped;
        g[k] = ok[k] ? g[k] * w : 0.f;
      }
      four.store(dlogp, g);
      unit_loss += part;
      kls += kl_part;
    });
    loss += unit_loss * w;
  });
  const Sums s = block_sums<3>(Sums{{loss, kls, static_cast<double>(cut)}}, red);
  if (threadIdx.x == 0 && !T1_OOB(blockIdx.x, p.blocks_n))
    for (int k = 0; k < 3; ++k) __stcg(&p.sums[3 * blockIdx.x + k], s.v[k]);
}

// ------------------------------------------------------------------ phase D
__device__ __forceinline__ void policy_total_phase(const LossParams& p, Sums* red) {
  const double tokens = fmax(1.0, join_totals(p, red).x);
  if (threadIdx.x >= 32) return;
  Sums s{{0, 0, 0}};
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += 32)
#pragma unroll
    for (int k = 0; k < 3; ++k) s.v[k] += __ldcg(&p.sums[3 * i + k]);
#pragma unroll
  for (int k = 0; k < 3; ++k) s.v[k] = warp_sum_f64(s.v[k]);
  if (threadIdx.x == 0) {
    *p.loss = static_cast<float>(s.v[0]);
    p.stats[0] = static_cast<float>(s.v[1] / tokens);
    p.stats[1] = static_cast<float>(s.v[2] / tokens);
  }
}

// Waits until every block has arrived for the `nth` time.  False (and an error
// code) if that takes longer than any launch can.
__device__ __forceinline__ bool grid_barrier(const LossParams& p, int nth) {
  __shared__ int ok;
  __syncthreads();
  if (p.arrivals.use == nullptr) {
    if (gridDim.x > 1) sm100::cluster_sync();
    return true;
  }
  if (threadIdx.x == 0) {
    const int all = nth * static_cast<int>(gridDim.x);
    __threadfence();
    atomicAdd(p.arrivals.use, 1);
    ok = 1;
    const uint64_t t0 = sm100::globaltimer_ns();
    int v, n = 0;
    while (true) {
      asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p.arrivals.use) : "memory");
      if (v >= all) break;
      if ((++n & 255) == 0 && sm100::globaltimer_ns() - t0 > sm100::kWaitLimitNs) {
        sm100::ErrorSlot{p.err}.set(131);
        ok = 0;
        break;
      }
    }
    __threadfence();
  }
  __syncthreads();
  return ok;
}

template <bool POLICY>
__global__ void __launch_bounds__(kLossThreads, kLossPerSm) answer_loss_kernel(const LossParams p) {
  __shared__ Sums red[kLossWarps];
  __shared__ int last;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  clear_arrivals(p.arrivals);
  int barriers = 0;
  count_phase<POLICY>(p, red);
  if (!grid_barrier(p, ++barriers)) return;
  if (!POLICY || p.lengths_phase) {
    if (POLICY) lengths_phase(p, red);
    else pairs_phase(p, red);
    if (!grid_barrier(p, ++barriers)) return;
  }
  if (POLICY) policy_grad_phase(p, red);
  else preference_grad_phase(p, red);
  if (!POLICY) return;
  if (p.arrivals.use == nullptr) {
    if (!grid_barrier(p, ++barriers) || blockIdx.x != 0) return;
  } else {  // the last block to arrive
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last = atomicAdd(p.arrivals.use, 1) == (barriers + 1) * static_cast<int>(gridDim.x) - 1;
    __syncthreads();
    if (!last) return;
    __threadfence();
  }
  policy_total_phase(p, red);
}

// ================================================================ host side
T1_BOUNDS_READER(answer_loss)

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

// Tokens of a cluster's block (8 of a lane, two rounds of loads), and blocks of
// the largest cluster that runs anywhere.
constexpr int64_t kBlockTokens = 4096;
constexpr int kLargestCluster = 8;

// The units of a batch and the blocks that share them.
struct LossPlan {
  bool cluster;
  int blocks, unit, chunks, lanes;

  LossPlan(int64_t B, int64_t S) {
    const int64_t T = B * S;
    int most = kLossPerSm * num_sms();
    lanes = 32;
    while (lanes > 1 && lanes / 2 >= S) lanes /= 2;
    const int64_t per_block = kLossWarps * (32 / lanes);
    // no more than two sequences in a row for a group of lanes, four in the
    // largest cluster
    cluster = T <= kBlockTokens * kLargestCluster && B <= 4 * per_block * kLargestCluster;
    if (cluster)
      for (most = 1; most < kLargestCluster && (most * kBlockTokens < T || most * 2 * per_block < B);) most *= 2;
    const int64_t warps = static_cast<int64_t>(most) * kLossWarps;
    // as many units as there are warps, of equal lengths, but no shorter than
    // one round of a lane's loads
    chunks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(warps / B, (S + 32 * kAhead - 1) / (32 * kAhead))));
    unit = static_cast<int>((S + chunks - 1) / chunks);
    if (S % 4 == 0) unit = (unit + 3) / 4 * 4;
    chunks = static_cast<int>((S + unit - 1) / unit);
    blocks = cluster ? most : static_cast<int>(std::min<int64_t>((B * chunks + per_block - 1) / per_block, most));
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

// Lays the phases' workspace out and launches.
template <bool POLICY>
static void launch_loss(LossParams& p, const LossPlan& plan) {
  const int64_t units = p.B * plan.chunks;
  auto pad = [](int64_t n) { return (n + 255) / 256 * 256; };
  const torch::Tensor held =
      loss_workspace(pad(16 * units) + pad(16 * plan.blocks) + pad(24 * plan.blocks) + pad(4 * p.B) + p.B * p.S);
  uint8_t* ws = held.data_ptr<uint8_t>();
  p.units_n = units;
  p.blocks_n = plan.blocks;
  p.units = reinterpret_cast<double2*>(ws);
  p.totals = reinterpret_cast<double2*>(ws + pad(16 * units));
  p.sums = reinterpret_cast<double*>(ws + pad(16 * units) + pad(16 * plan.blocks));
  uint8_t* per_seq = ws + pad(16 * units) + pad(16 * plan.blocks) + pad(24 * plan.blocks);
  p.coef = reinterpret_cast<float*>(per_seq);
  p.lengths = reinterpret_cast<int*>(per_seq);
  p.answer = per_seq + pad(4 * p.B);
  p.unit = plan.unit;
  p.chunks = plan.chunks;
  p.lanes = plan.lanes;
  auto aligned = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  p.vectors = p.S % 4 == 0 && plan.lanes == 32 && aligned(p.targets) && aligned(p.logp) && aligned(p.old) &&
              aligned(p.ref) && (!p.adv_per_token || aligned(p.adv));
  p.lengths_phase = POLICY && p.per_sequence && plan.chunks > 1;
  p.err = gemm_error_word().data_ptr<int>();
  std::optional<ArrivalCounters> counters;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(plan.blocks);
  cfg.blockDim = dim3(kLossThreads);
  cfg.stream = stream();
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (plan.cluster) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = plan.blocks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
  } else {  // blocks that wait for one another
    counters.emplace(1);
    p.arrivals = counters->arrivals;
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.numAttrs = 1;
  }
  const cudaError_t e = cudaLaunchKernelEx(&cfg, answer_loss_kernel<POLICY>, static_cast<LossParams>(p));
  TORCH_CHECK(e == cudaSuccess, "answer_loss launch failed: ", cudaGetErrorString(e));
  if (counters) counters->launched();
  count_launch();
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
