// Log-probabilities of the target tokens under the output layer, and their
// gradients, without the [T, V] logits in fp32 or their copy in memory.
//
//   logit[t, v] = x[t, :] . W[v, :] / tau
//   lse[t]      = log sum_v exp(logit[t, v]),  logp[t] = logit[t, target[t]] - lse[t]
//   u[t, v]     = onehot(target[t])[v] - exp(logit[t, v] - lse[t])
//   dx[t, :]    = (dlogp[t] / tau) sum_v u[t, v] W[v, :]
//   dW[v, :]    = sum_t u[t, v] (dlogp[t] / tau) x[t, :]
//
// A token whose target is ignored (ignore_index, or outside the vocabulary)
// gives logp = lse = 0 and no gradient, whatever its hidden state holds.
#include "vocab_gemm.cuh"

namespace t1 {

CUtensorMap make_map_any(const void* ptr, bool f32, int64_t inner, int64_t outer, int64_t ld, int box_outer);
torch::Tensor& gemm_error_word();

using vocab::VocabParams;
using vocab::kLog2e;
using vocab::ex2;

// Joins the column blocks' (largest, sum) of 32 rows: lanes are rows (a
// block's entries of neighbouring rows are neighbours in memory), warps
// share the column blocks.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(32 * kJoinWarps)
    logprob_join_kernel(const float2* __restrict__ part, const float* __restrict__ target_logit,
                        const int64_t* __restrict__ targets, int64_t ignore, int64_t V, int T, int blocks,
                        float scale, float* __restrict__ logp, float* __restrict__ lse) {
  __shared__ float sm[kJoinWarps][32], ss[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  const bool in = row < T && !T1_OOB(row, T);
  const float k2 = scale * kLog2e;
  float m = -INFINITY, s = 0.f;
  if (in) {
    for (int b = warp; b < blocks; b += kJoinWarps) {
      const float2 v = part[static_cast<size_t>(b) * T + row];
      const float mn = fmaxf(m, v.x);
      const float ref = mn == -INFINITY ? 0.f : mn;
      s = s * ex2((m - ref) * k2) + v.y * ex2((v.x - ref) * k2);
      m = mn;
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
  const int64_t t = targets[row];
  const bool valid = t != ignore && t >= 0 && t < V;
  const float log_s = logf(s);
  // (target - largest) first: exact where the target is likely
  logp[row] = valid ? (target_logit[row] - ref) * scale - log_s : 0.f;
  lse[row] = valid ? ref * scale + log_s : 0.f;
}

// Per row: g = dlogp / tau (0 for a row without a gradient) and, rounded to
// bf16 for the tensor cores, g x: the rounding is one relative 2^-9 at most
// per element of x, independent from element to element.
__global__ void __launch_bounds__(128)
    logprob_scale_rows_kernel(const bf16* __restrict__ x, long ldx, const float* __restrict__ dlogp,
                              const int64_t* __restrict__ targets, int64_t ignore, int64_t V, int T, int H,
                              float scale, float* __restrict__ g, bf16* __restrict__ gx) {
  const int row = blockIdx.x;
  if (T1_OOB(row, T)) return;
  const int64_t t = targets[row];
  const bool valid = t != ignore && t >= 0 && t < V;
  const float gr = valid ? dlogp[row] * scale : 0.f;
  if (threadIdx.x == 0) g[row] = gr;
  for (int i = threadIdx.x; i < H / 8; i += blockDim.x) {
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (gr != 0.f) {
      load8(x + static_cast<size_t>(row) * ldx + 8 * i, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= gr;
    }
    store8(gx + static_cast<size_t>(row) * H + 8 * i, v);
  }
}

// dx[t, :] = g[t] * (sum of the fp32 planes), in plane order.
__global__ void __launch_bounds__(128)
    logprob_dx_kernel(const float* __restrict__ planes, int n_planes, size_t plane_stride,
                      const float* __restrict__ g, int T, int H, bf16* __restrict__ dx, long lddx) {
  const int row = blockIdx.x;
  if (T1_OOB(row, T)) return;
  const float gr = g[row];
  for (int i = threadIdx.x; i < H / 8; i += blockDim.x) {
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (gr != 0.f) {
      for (int s = 0; s < n_planes; ++s) {
        const float4* p = reinterpret_cast<const float4*>(planes + s * plane_stride + static_cast<size_t>(row) * H + 8 * i);
        const float4 a = p[0], b = p[1];
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= gr;
    }
    store8(dx + static_cast<size_t>(row) * lddx + 8 * i, v);
  }
}

// ================================================================ host side
T1_BOUNDS_READER(logprob)

template <bool A_MN, bool B_MN, int MODE>
static void launch_vocab(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, VocabParams& p) {
  auto kern = vocab::vocab_kernel<A_MN, B_MN, MODE>;
  static bool configured = false;
  if (!configured) {
    T1_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, vocab::V_SMEM_BYTES));
    configured = true;
  }
  p.tiles_m = (p.M + vocab::TILE - 1) / vocab::TILE;
  p.tiles_n = (p.N + vocab::TILE - 1) / vocab::TILE;
  p.err = gemm_error_word().data_ptr<int>();
  const int clusters = std::min(p.tiles_m * p.tiles_n * p.splits, num_sms() / 2);
  kern<<<2 * clusters, 192, vocab::V_SMEM_BYTES, stream()>>>(ta, tb, tc, p);
  check_launch("linear_logprob");
  count_launch();
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
  TORCH_CHECK(std::isfinite(temperature) && temperature > 0, "temperature must be positive");
}

// Row distance for a tensor map: a single row's own stride says nothing.
static int64_t row_ld(const torch::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

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
  const int64_t blocks = (V + vocab::TILE - 1) / vocab::TILE;
  auto ws = torch::empty({2 * blocks * T + T}, f32);
  VocabParams p{};
  p.M = static_cast<int>(T);
  p.N = static_cast<int>(V);
  p.k_blocks = static_cast<int>((H + gemm::BK - 1) / gemm::BK);
  p.splits = 1;
  p.scale = static_cast<float>(1.0 / temperature);
  p.targets = tg.data_ptr<int64_t>();
  p.part = reinterpret_cast<float2*>(ws.data_ptr<float>());
  p.target_logit = ws.data_ptr<float>() + 2 * blocks * T;
  CUtensorMap ta = make_map_any(x.data_ptr(), false, H, T, row_ld(x), vocab::HALF);
  CUtensorMap tb = make_map_any(w.data_ptr(), false, H, V, row_ld(w), vocab::HALF);
  launch_vocab<false, false, vocab::kLse>(ta, tb, ta, p);
  logprob_join_kernel<<<(T + 31) / 32, 32 * kJoinWarps, 0, stream()>>>(
      p.part, p.target_logit, p.targets, ignore_index, V, T, blocks, p.scale, logp.data_ptr<float>(),
      lse.data_ptr<float>());
  check_launch("logprob_join");
  count_launch();
  return {logp, lse};
}

// The softmax gradient u exists for as many vocabulary columns at a time as
// fit this many bytes; dW's rows of those columns are then final, and dx
// gathers the chunks' products in fp32.
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
  const float scale = static_cast<float>(1.0 / temperature);
  auto f32 = x.options().dtype(torch::kFloat32);
  auto g = torch::empty({T}, f32);
  auto gx = torch::empty({T, H}, x.options());
  TORCH_CHECK(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && row_ld(x) % 8 == 0,
              "x must have 16-byte aligned rows");
  logprob_scale_rows_kernel<<<T, 128, 0, stream()>>>((const bf16*)x.data_ptr(), row_ld(x), up.data_ptr<float>(),
                                                     tg.data_ptr<int64_t>(), ignore_index, V, T, H, scale,
                                                     g.data_ptr<float>(), (bf16*)gx.data_ptr());
  check_launch("logprob_scale_rows");
  count_launch();

  const int64_t most = std::max<int64_t>(vocab::TILE, kGradBufferBytes / (2 * T) / vocab::TILE * vocab::TILE);
  const int64_t chunks = (V + most - 1) / most;
  const int64_t width = ((V + chunks - 1) / chunks + vocab::TILE - 1) / vocab::TILE * vocab::TILE;
  const int64_t ldu = (std::min(width, V) + 7) / 8 * 8;
  auto u = torch::empty({T, ldu}, x.options());
  const int64_t plane_rows = (T + vocab::TILE - 1) / vocab::TILE * vocab::TILE;
  const int splits = 1;
  auto planes = torch::empty({splits * plane_rows, (H + 3) / 4 * 4}, f32);

  CUtensorMap tx = make_map_any(x.data_ptr(), false, H, T, row_ld(x), vocab::HALF);
  CUtensorMap tgx = make_map_any(gx.data_ptr(), false, H, T, H, 64);
  CUtensorMap tpl = make_map_any(planes.data_ptr(), true, H, splits * plane_rows, planes.size(1), 32);
  for (int64_t v0 = 0; v0 < V; v0 += width) {
    const int64_t n = std::min(width, V - v0);
    const bf16* wp = (const bf16*)w.data_ptr() + v0 * row_ld(w);
    {  // u = onehot - softmax
      VocabParams p{};
      p.M = T;
      p.N = n;
      p.k_blocks = (H + gemm::BK - 1) / gemm::BK;
      p.splits = 1;
      p.scale = scale;
      p.col0 = v0;
      p.targets = tg.data_ptr<int64_t>();
      p.lse = ls.data_ptr<float>();
      p.drow = g.data_ptr<float>();
      launch_vocab<false, false, vocab::kSoftmaxGrad>(tx, make_map_any(wp, false, H, n, row_ld(w), vocab::HALF),
                                                      make_map_any(u.data_ptr(), false, n, T, ldu, 32), p);
    }
    {  // dx's sums: u W
      VocabParams p{};
      p.M = T;
      p.N = H;
      p.k_blocks = (n + gemm::BK - 1) / gemm::BK;
      p.splits = splits;
      p.plane_rows = plane_rows;
      p.accumulate = v0 > 0;
      launch_vocab<false, true, vocab::kRowsF32>(make_map_any(u.data_ptr(), false, n, T, ldu, vocab::HALF),
                                                 make_map_any(wp, false, H, n, row_ld(w), 64), tpl, p);
    }
    {  // dW: u^T (g x)
      VocabParams p{};
      p.M = n;
      p.N = H;
      p.k_blocks = (T + gemm::BK - 1) / gemm::BK;
      p.splits = 1;
      launch_vocab<true, true, vocab::kWeightGrad>(
          make_map_any(u.data_ptr(), false, n, T, ldu, 64), tgx,
          make_map_any((bf16*)dw.data_ptr() + v0 * H, false, H, n, H, 32), p);
    }
  }
  logprob_dx_kernel<<<T, 128, 0, stream()>>>(planes.data_ptr<float>(), splits, plane_rows * planes.size(1),
                                             g.data_ptr<float>(), T, H, (bf16*)dx.data_ptr(), H);
  check_launch("logprob_dx");
  count_launch();
}

}  // namespace t1
