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

// How many ranges the rows' product u W is cut into (tiles of 256 x 256 on
// `clusters` CTA pairs): the smallest estimate of waves x (k blocks of a
// range + start and drain of a tile) + the planes' traffic, in units of a k
// block (0.13 us of tensor time; a tile's plane written and read back is
// 0.5 MB, 0.08 us of the GPU's bandwidth).
__host__ __device__ inline int pick_splits(int tiles, int k_blocks, int clusters) {
  int best = 1;
  int64_t least = INT64_MAX;  // whole numbers: host and device must agree
  for (int s = 1; s <= 32 && (s == 1 || k_blocks >= 16 * s); ++s) {
    const int64_t waves = (static_cast<int64_t>(tiles) * s + clusters - 1) / clusters;
    const int64_t cost = 10 * waves * ((k_blocks + s - 1) / s + 12) + 6ll * s * tiles;
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}

struct PackParams {
  const bf16* x;
  long ldx;
  const int64_t* targets;
  int64_t ignore, V;
  int T, H;
  int per_block;         // tokens of a block
  float scale;
  const float* dlogp;    // null in the forward
  const float* lse;      // with dlogp
  int k_blocks, tiles_n, clusters;  // of the rows' product, with dlogp
  vocab::RowsMeta* meta;
  int* index;            // [T] the packed row's token
  int* target;           // [T]
  float* g;              // [T] dlogp / tau, with dlogp
  float* lse_packed;     // with dlogp
  bf16* xp;              // [T + 64, H] the rows of x
  bf16* gxp;             // [T + 64, H] g x, with dlogp
  float *zero0, *zero1;  // forward: logp and lse, 0 for the tokens left out
  bf16* dx;              // backward: likewise
};

constexpr int kPackThreads = 256;

// Packs the rows that take part: tokens with a target and, in the backward,
// with a gradient (a clipped token's is exactly 0, and so is all it adds).
// Prompts and padding are often half of a batch, and every product below
// shrinks by them.  Each block counts the rows before its own tokens itself:
// T / 2 targets out of L2 on average instead of a scan in a launch of its
// own.  Rows keep their order, so sums over rows do not depend on timing.
//
// In the backward also g x, rounded to bf16 for the tensor cores: a relative
// error of 2^-9 at most per element of x, independent from element to
// element.  (Scaling the other factor instead, u, would round the one large
// entry of each row, whose error all of a row of dx and dW shares.)
template <bool BWD>
__global__ void __launch_bounds__(kPackThreads) logprob_pack_kernel(const PackParams p) {
  __shared__ int counts[kPackThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kPackThreads / 32;
  const int t0 = blockIdx.x * p.per_block, t1 = min(p.T, t0 + p.per_block);
  auto takes_part = [&](int t) {
    const int64_t v = p.targets[t];
    const bool valid = v != p.ignore && v >= 0 && v < p.V;
    return BWD ? valid && p.dlogp[t] != 0.f : valid;
  };
  int n = 0;
  for (int t = threadIdx.x; t < t0; t += kPackThreads) n += takes_part(t);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if (lane == 0) counts[warp] = n;
  __syncthreads();
  int pos = 0;
  for (int w = 0; w < kWarps; ++w) pos += counts[w];

  const int nvec = p.H >> 3;
  for (int base = t0; base < t1; base += 32) {
    const bool mine = base + lane < t1 && takes_part(base + lane);
    const unsigned mask = __ballot_sync(0xffffffffu, mine);
    // warp w takes tokens w, w + 8, ... of the 32
    for (int j = warp; j < 32 && base + j < t1; j += kWarps) {
      const int t = base + j;
      if (!(mask >> j & 1)) {
        if (!BWD && lane == 0) p.zero0[t] = p.zero1[t] = 0.f;
        if (BWD)
          for (int i = lane; i < nvec; i += 32)
            reinterpret_cast<uint4*>(p.dx + static_cast<size_t>(t) * p.H)[i] = make_uint4(0, 0, 0, 0);
        continue;
      }
      const int at = pos + __popc(mask & ((1u << j) - 1));
      if (T1_OOB(at, p.T)) continue;
      float gr = 0.f;
      if (BWD) gr = p.dlogp[t] * p.scale;
      if (lane == 0) {
        p.index[at] = t;
        p.target[at] = static_cast<int>(p.targets[t]);
        if (BWD) {
          p.g[at] = gr;
          p.lse_packed[at] = p.lse[t];
        }
      }
      const bf16* src = p.x + static_cast<size_t>(t) * p.ldx;
      for (int i = lane; i < nvec; i += 32) {
        const size_t dst = static_cast<size_t>(at) * p.H + 8 * i;
        *reinterpret_cast<uint4*>(p.xp + dst) = *reinterpret_cast<const uint4*>(src + 8 * i);
        if (BWD) {
          float v[8];
          load8(src + 8 * i, v);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] *= gr;
          store8(p.gxp + dst, v);
        }
      }
    }
    pos += __popc(mask);
  }
  if (t1 != p.T) return;
  // the last block knows how many there are
  if (threadIdx.x == 0) {
    p.meta->rows = pos;
    if (BWD) p.meta->splits = pick_splits((pos + vocab::TILE - 1) / vocab::TILE * p.tiles_n, p.k_blocks, p.clusters);
  }
  if (BWD) {  // dW's reduction runs over whole blocks of BK rows
    const int end = (pos + gemm::BK - 1) / gemm::BK * gemm::BK;
    for (int i = threadIdx.x; i < (end - pos) * nvec; i += kPackThreads)
      reinterpret_cast<uint4*>(p.gxp + static_cast<size_t>(pos) * p.H)[i] = make_uint4(0, 0, 0, 0);
  }
}

// Joins the column blocks' (largest, sum) of 32 rows: lanes are rows (a
// block's entries of neighbouring rows are neighbours in memory), warps
// share the column blocks.
constexpr int kJoinWarps = 8;
__global__ void __launch_bounds__(32 * kJoinWarps)
    logprob_join_kernel(const float2* __restrict__ part, const float* __restrict__ target_logit,
                        const vocab::RowsMeta* __restrict__ meta, const int* __restrict__ index, int T, int blocks,
                        float scale, float* __restrict__ logp, float* __restrict__ lse) {
  __shared__ float sm[kJoinWarps][32], ss[kJoinWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x * 32 + lane;
  if (blockIdx.x * 32 >= meta->rows) return;  // uniform over the block
  const bool in = row < meta->rows;
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
  const float log_s = logf(s);
  const int t = index[row];
  if (T1_OOB(t, T)) return;
  // (target - largest) first: exact where the target is likely
  logp[t] = (target_logit[row] - ref) * scale - log_s;
  lse[t] = ref * scale + log_s;
}

// dx[t, :] = g[t] * (sum of the fp32 planes), in plane order, for the packed
// rows (the packing wrote the others' zeros).
__global__ void __launch_bounds__(128)
    logprob_dx_kernel(const float* __restrict__ planes, const vocab::RowsMeta* __restrict__ meta, long ldp,
                      const int* __restrict__ index, const float* __restrict__ g, int T, int H,
                      bf16* __restrict__ dx) {
  const int rows = meta->rows, splits = meta->splits;
  const size_t stride = static_cast<size_t>((rows + vocab::TILE - 1) / vocab::TILE * vocab::TILE) * ldp;
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const float gr = g[row];
    const int t = index[row];
    if (T1_OOB(t, T)) continue;
    for (int i = threadIdx.x; i < H / 8; i += blockDim.x) {
      float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      for (int s = 0; s < splits; ++s) {
        const float4* p = reinterpret_cast<const float4*>(planes + s * stride + static_cast<size_t>(row) * ldp + 8 * i);
        const float4 a = p[0], b = p[1];
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] *= gr;
      store8(dx + static_cast<size_t>(t) * H + 8 * i, v);
    }
  }
}

// ================================================================ host side
T1_BOUNDS_READER(logprob)

// `units`: the most units of work that the launch can have.
template <bool A_MN, bool B_MN, int MODE>
static void launch_vocab(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, VocabParams& p,
                         int64_t units) {
  auto kern = vocab::vocab_kernel<A_MN, B_MN, MODE>;
  static bool configured = false;
  if (!configured) {
    T1_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, vocab::V_SMEM_BYTES));
    configured = true;
  }
  p.err = gemm_error_word().data_ptr<int>();
  const int clusters = static_cast<int>(std::min<int64_t>(units, num_sms() / 2));
  kern<<<2 * clusters, 192, vocab::V_SMEM_BYTES, stream()>>>(ta, tb, tc, p);
  check_launch("linear_logprob");
  count_launch();
}

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// A workspace cut into 256-byte aligned pieces.
struct Pieces {
  int64_t used = 0;
  int64_t take(int64_t bytes) {
    const int64_t at = used;
    used += round_up(bytes, 256);
    return at;
  }
};

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
  const int64_t ldx = x.size(0) > 1 ? x.stride(0) : x.size(1);
  TORCH_CHECK(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && ldx % 8 == 0, "x must have 16-byte aligned rows");
  TORCH_CHECK(std::isfinite(temperature) && temperature > 0, "temperature must be positive");
}

// Distance of two rows; a single row's own stride says nothing.
static int64_t row_ld(const torch::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

static void launch_pack(PackParams& p) {
  // a few blocks per SM, and no more than 32 tokens each where T allows it
  p.per_block = static_cast<int>(std::max<int64_t>(8, ceil_div(p.T, 4 * num_sms())));
  const int blocks = static_cast<int>(ceil_div(p.T, p.per_block));
  if (p.dlogp != nullptr) logprob_pack_kernel<true><<<blocks, kPackThreads, 0, stream()>>>(p);
  else logprob_pack_kernel<false><<<blocks, kPackThreads, 0, stream()>>>(p);
  check_launch("logprob_pack");
  count_launch();
}

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
  const int64_t blocks = ceil_div(V, vocab::TILE);
  Pieces ws;
  const int64_t o_meta = ws.take(sizeof(vocab::RowsMeta)), o_index = ws.take(4 * T), o_target = ws.take(4 * T),
                o_logit = ws.take(4 * T), o_part = ws.take(8 * blocks * T), o_x = ws.take(2 * T * H);
  auto buf = torch::empty({ws.used}, x.options().dtype(torch::kUInt8));
  uint8_t* base = buf.data_ptr<uint8_t>();
  const float scale = static_cast<float>(1.0 / temperature);

  PackParams k{};
  k.x = (const bf16*)x.data_ptr();
  k.ldx = row_ld(x);
  k.targets = tg.data_ptr<int64_t>();
  k.ignore = ignore_index;
  k.V = V;
  k.T = T;
  k.H = H;
  k.meta = reinterpret_cast<vocab::RowsMeta*>(base + o_meta);
  k.index = reinterpret_cast<int*>(base + o_index);
  k.target = reinterpret_cast<int*>(base + o_target);
  k.xp = reinterpret_cast<bf16*>(base + o_x);
  k.zero0 = logp.data_ptr<float>();
  k.zero1 = lse.data_ptr<float>();
  launch_pack(k);

  VocabParams p{};
  p.meta = k.meta;
  p.N = static_cast<int>(V);
  p.k_blocks = static_cast<int>(ceil_div(H, gemm::BK));
  p.ld_part = static_cast<int>(T);
  p.scale = scale;
  p.targets = k.target;
  p.part = reinterpret_cast<float2*>(base + o_part);
  p.target_logit = reinterpret_cast<float*>(base + o_logit);
  CUtensorMap ta = make_map_any(k.xp, false, H, T, H, vocab::HALF);
  CUtensorMap tb = make_map_any(w.data_ptr(), false, H, V, row_ld(w), vocab::HALF);
  launch_vocab<false, false, vocab::kLse>(ta, tb, ta, p, ceil_div(T, vocab::TILE) * blocks);
  logprob_join_kernel<<<ceil_div(T, 32), 32 * kJoinWarps, 0, stream()>>>(p.part, p.target_logit, k.meta, k.index, T,
                                                                       blocks, scale, logp.data_ptr<float>(),
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
  const int clusters = num_sms() / 2;
  const int64_t tiles_t = ceil_div(T, vocab::TILE), tiles_h = ceil_div(H, vocab::TILE), k_h = ceil_div(H, gemm::BK);

  const int64_t most = std::max<int64_t>(vocab::TILE, kGradBufferBytes / (2 * T) / vocab::TILE * vocab::TILE);
  const int64_t chunks = ceil_div(V, most);
  const int64_t width = std::min(V, round_up(ceil_div(V, chunks), vocab::TILE));
  const int64_t ldu = round_up(width, 8), u_rows = round_up(T, gemm::BK), k_v = ceil_div(width, gemm::BK);
  // the planes of the most rows that the split rule can ask for
  int64_t plane_rows = 0, most_units = 0;
  for (int64_t m = 1; m <= tiles_t; ++m) {
    const int64_t s = pick_splits(m * tiles_h, k_v, clusters);
    plane_rows = std::max(plane_rows, s * m * vocab::TILE);
    most_units = std::max(most_units, s * m * tiles_h);
  }
  Pieces ws;
  const int64_t o_meta = ws.take(sizeof(vocab::RowsMeta)), o_index = ws.take(4 * T), o_target = ws.take(4 * T),
                o_g = ws.take(4 * T), o_lse = ws.take(4 * T), o_x = ws.take(2 * T * H),
                o_gx = ws.take(2 * u_rows * H), o_planes = ws.take(4 * plane_rows * H), o_u = ws.take(2 * u_rows * ldu);
  auto buf = torch::empty({ws.used}, x.options().dtype(torch::kUInt8));
  uint8_t* base = buf.data_ptr<uint8_t>();

  PackParams k{};
  k.x = (const bf16*)x.data_ptr();
  k.ldx = row_ld(x);
  k.targets = tg.data_ptr<int64_t>();
  k.ignore = ignore_index;
  k.V = V;
  k.T = T;
  k.H = H;
  k.scale = scale;
  k.dlogp = up.data_ptr<float>();
  k.lse = ls.data_ptr<float>();
  k.k_blocks = k_v;
  k.tiles_n = tiles_h;
  k.clusters = clusters;
  k.meta = reinterpret_cast<vocab::RowsMeta*>(base + o_meta);
  k.index = reinterpret_cast<int*>(base + o_index);
  k.target = reinterpret_cast<int*>(base + o_target);
  k.g = reinterpret_cast<float*>(base + o_g);
  k.lse_packed = reinterpret_cast<float*>(base + o_lse);
  k.xp = reinterpret_cast<bf16*>(base + o_x);
  k.gxp = reinterpret_cast<bf16*>(base + o_gx);
  k.dx = (bf16*)dx.data_ptr();
  launch_pack(k);

  bf16* u = reinterpret_cast<bf16*>(base + o_u);
  float* planes = reinterpret_cast<float*>(base + o_planes);
  CUtensorMap tx = make_map_any(k.xp, false, H, T, H, vocab::HALF);
  CUtensorMap tgx = make_map_any(k.gxp, false, H, u_rows, H, 64);
  CUtensorMap tpl = make_map_any(planes, true, H, plane_rows, H, 32);
  for (int64_t v0 = 0; v0 < V; v0 += width) {
    const int64_t n = std::min(width, V - v0);
    const bf16* wp = (const bf16*)w.data_ptr() + v0 * row_ld(w);
    VocabParams p{};
    p.meta = k.meta;
    // u = onehot - softmax
    p.N = n;
    p.k_blocks = k_h;
    p.scale = scale;
    p.col0 = v0;
    p.targets = k.target;
    p.lse = k.lse_packed;
    launch_vocab<false, false, vocab::kSoftmaxGrad>(tx, make_map_any(wp, false, H, n, row_ld(w), vocab::HALF),
                                                    make_map_any(u, false, n, u_rows, ldu, 32), p,
                                                    tiles_t * ceil_div(n, vocab::TILE));
    // dx's sums: u W
    p.N = H;
    p.k_blocks = ceil_div(n, gemm::BK);
    p.accumulate = v0 > 0;
    launch_vocab<false, true, vocab::kRowsF32>(make_map_any(u, false, n, T, ldu, vocab::HALF),
                                               make_map_any(wp, false, H, n, row_ld(w), 64), tpl, p, most_units);
    // dW: u^T (g x)
    p.M = n;
    launch_vocab<true, true, vocab::kWeightGrad>(make_map_any(u, false, n, u_rows, ldu, 64), tgx,
                                                 make_map_any((bf16*)dw.data_ptr() + v0 * H, false, H, n, H, 32), p,
                                                 ceil_div(n, vocab::TILE) * tiles_h);
  }
  logprob_dx_kernel<<<std::min<int64_t>(T, 16 * num_sms()), 128, 0, stream()>>>(planes, k.meta, H, k.index, k.g, T, H,
                                                                               (bf16*)dx.data_ptr());
  check_launch("logprob_dx");
  count_launch();
}

}  // namespace t1
