"""Logits of the output layer in fp32, log-probabilities at lists of tokens and
their gradients, against the definitions in 64 bits.

Tolerances.  A logit is a sum of H exact products accumulated in fp32, 16 of
them per step: its error is at most (H / 16 + 4) 2^-23 of the largest partial
sum, which |x| |w| bounds; exp, log and the joins add a few more 2^-23 of the
same size.  Gradients round u to bf16 (at most 2^-8, relative, element by
element) and the result once more (2^-8; x and w are bf16 already): the 2-norm
of the error stays below 4 x 2^-9 of the result's."""
import pytest
import torch

import _lists_oracle as oracle

pytestmark = pytest.mark.gpu

#        T, H, V, K
SIZES = [(1, 64, 257, 1), (2, 8, 5, 5), (1, 256, 1, 1), (33, 72, 255, 7), (129, 264, 1000, 33), (300, 520, 4097, 64),
         (513, 256, 20011, 20), (700, 1024, 2048, 129), (257, 2048, 520, 300), (300, 64, 600, 512),
         # packed rows
         (600, 1024, 50021, 40),
         # few tokens: one or two column blocks of 8, x and lists that fit in shared memory or not
         (1, 4096, 5003, 64), (8, 1032, 5003, 16), (9, 4096, 777, 100), (16, 2056, 1500, 512), (16, 4096, 1500, 512),
         (5, 8192, 600, 3), (16, 8192, 300, 8), (17, 4096, 300, 8), (3, 512, 40009, 50)]
GRAD_TOL = 4 * 2.0 ** -9


def _inputs(T, H, V, K, seed=0, masked=True):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + T + H + V + K)
    w = (torch.randn(V, H, device="cuda", generator=g) * 2 / H ** 0.5).bfloat16()
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    ids = torch.rand(T, V, device="cuda", generator=g).topk(min(K, V), 1).indices
    if K > V:
        ids = torch.cat([ids, torch.full((T, K - V), -1, device="cuda")], 1)
    if masked and T > 1:
        ids[torch.rand(T, K, device="cuda", generator=g) < 0.2] = -100
        ids[0, 0] = V            # not a vocabulary index: ignored as well
        ids[T // 2] = -100       # a row that takes no part
        if K > 1:
            ids[-1, :2] = V - 1  # the same token twice
    up = torch.randn(T, K, device="cuda", generator=g) / T
    return x, w, ids, up


def _tol(x, w, temperature):
    H = w.shape[1]
    size = float(x.float().norm(dim=1).nan_to_num(0, 0, 0).max() * w.float().norm(dim=1).max())
    return (H / 16 + 32) * 2.0 ** -23 * (size + 4) / min(1.0, temperature)


def _rel(a, b):
    return float((a.double() - b).norm() / b.norm().clamp_min(1e-30))


@pytest.mark.parametrize("T,H,V", [(1, 64, 257), (2, 8, 5), (16, 4096, 1001), (17, 72, 255), (129, 264, 1000), (300, 520, 4097),
                                   (513, 1024, 20011), (16, 8192, 300), (257, 2048, 1)])
def test_logits(T, H, V, cuda_device):
    from test1_b200 import ops

    x, w, _, _ = _inputs(T, H, V, 1)
    l = ops.linear_logits(x, w)
    assert l.dtype == torch.float32 and l.shape == (T, V)
    assert float((l - x.double() @ w.double().t()).abs().max()) <= _tol(x, w, 1.0)
    wide = torch.full((T, H + 8), float("nan"), dtype=x.dtype, device="cuda")
    wide[:, :H] = x
    assert torch.equal(ops.linear_logits(wide[:, :H], w), l)
    assert ops.linear_logits(x[:0], w).shape == (0, V)


@pytest.mark.parametrize("T,H,V,K", SIZES)
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_forward(T, H, V, K, temperature, cuda_device):
    from test1_b200 import ops
    from test1_b200.ops import native

    x, w, ids, _ = _inputs(T, H, V, K)
    logp, lse = ops.linear_topk_logprob_fwd(x, w, ids, temperature=temperature)
    lp, ls, _, _ = oracle.listed_logprob(x, w, ids, temperature)
    tol = _tol(x, w, temperature)
    assert logp.dtype == lse.dtype == torch.float32 and logp.shape == ids.shape and lse.shape == (T,)
    assert float((logp - lp).abs().max()) <= tol
    assert float((lse - ls).abs().max()) <= tol
    none = (ids < 0) | (ids >= V)
    assert not bool(logp[none].any()) and not bool(lse[none.all(1)].any())
    assert native.gemm_error() == 0


@pytest.mark.parametrize("T,H,V,K", SIZES)
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_backward(T, H, V, K, temperature, cuda_device):
    from test1_b200 import ops
    from test1_b200.ops import native

    x, w, ids, up = _inputs(T, H, V, K, seed=1)
    _, ls, dx64, dw64 = oracle.listed_logprob(x, w, ids, temperature, dlogp=up)
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))  # must be fully written
    ops.linear_topk_logprob_bwd(up, x, w, ids, ls.float(), dx, dw, temperature=temperature)
    if V > 1:
        assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL
    else:  # u is 0 but for the rounding of lse, 2^-22 of it
        assert float(dx.abs().max()) < 1e-4 and float(dw.abs().max()) < 1e-4
    assert native.gemm_error() == 0


@pytest.mark.parametrize("T", [6, 40, 600])
def test_rows_left_out_may_hold_anything(T, cuda_device):
    from test1_b200 import ops

    H, V, K = 512, 80013, 12
    x, w, ids, up = _inputs(T, H, V, K, seed=2)
    ids[3:5] = -1
    up[5] = 0.0  # listed, without a gradient
    clean = x.clone()
    x[3:5] = float("nan")
    up[3] = float("nan")
    lp, ls, dx64, dw64 = oracle.listed_logprob(clean, w, ids, 1.0, dlogp=up)
    logp, lse = ops.linear_topk_logprob_fwd(x, w, ids)
    assert float((logp - lp).abs().max()) <= _tol(clean, w, 1.0)
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))
    ops.linear_topk_logprob_bwd(up, x, w, ids, lse, dx, dw)
    assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL
    assert not bool(dx[3:6].any())
    # nothing takes part at all
    logp, lse = ops.linear_topk_logprob_fwd(x, w, torch.full_like(ids, -1))
    assert not bool(logp.any()) and not bool(lse.any())
    ops.linear_topk_logprob_bwd(up, x, w, torch.full_like(ids, -1), lse, dx, dw)
    assert not bool(dx.any()) and not bool(dw.any())


@pytest.mark.parametrize("T", [7, 300])
def test_gradients_that_add_up_to_nothing(T, cuda_device):
    """sum_k dlogp = 0: the softmax's part vanishes, the listed tokens' does not."""
    from test1_b200 import ops

    x, w, ids, up = _inputs(T, 256, 3001, 2, seed=3, masked=False)
    up[:, 0], up[:, 1] = 0.5, -0.5
    _, ls, dx64, dw64 = oracle.listed_logprob(x, w, ids, 1.0, dlogp=up)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ops.linear_topk_logprob_bwd(up, x, w, ids, ls.float(), dx, dw)
    assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL


def test_neighbouring_tokens(cuda_device):
    """A whole list within one tile of the vocabulary, at its start and end."""
    from test1_b200 import ops

    T, H, V, K = 64, 128, 1030, 100
    x, w, ids, up = _inputs(T, H, V, K, seed=4, masked=False)
    ids[:] = torch.arange(K, device="cuda")
    ids[::2] = V - 1 - torch.arange(K, device="cuda")
    ids[1::4] = 200 + torch.arange(K, device="cuda")  # across the border of two
    logp, lse = ops.linear_topk_logprob_fwd(x, w, ids)
    lp, _, dx64, dw64 = oracle.listed_logprob(x, w, ids, 1.0, dlogp=up)
    assert float((logp - lp).abs().max()) <= _tol(x, w, 1.0)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ops.linear_topk_logprob_bwd(up, x, w, ids, lse, dx, dw)
    assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL


def test_vocabulary_in_pieces(cuda_device):
    """A softmax gradient of more than a GB is made and used in pieces."""
    from test1_b200 import ops

    T, H, V, K = 5000, 64, 120011, 9
    x, w, ids, up = _inputs(T, H, V, K, seed=5)
    _, ls, dx64, dw64 = oracle.listed_logprob(x, w, ids, 1.0, dlogp=up)
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))
    ops.linear_topk_logprob_bwd(up, x, w, ids, ls.float(), dx, dw)
    assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL


def test_a_list_of_the_target_alone(cuda_device):
    from test1_b200 import ops

    x, w, ids, up = _inputs(500, 512, 9001, 1, seed=6)
    logp, lse = ops.linear_topk_logprob_fwd(x, w, ids)
    one, lse1 = ops.linear_logprob_fwd(x, w, ids[:, 0].contiguous())
    assert torch.equal(logp[:, 0], one) and torch.equal(lse, lse1)


@pytest.mark.parametrize("T", [5, 300])
def test_strides_streams_and_a_graph(T, cuda_device):
    from test1_b200 import ops

    H, V, K = 256, 5003, 24
    x, w, ids, up = _inputs(T, H, V, K, seed=7)
    wide_x, wide_w = torch.zeros(T, H + 16, dtype=x.dtype, device="cuda"), torch.zeros(V, H + 8, dtype=x.dtype, device="cuda")
    wide_x[:, :H], wide_w[:, :H] = x, w
    wide_ids = torch.zeros(T, 2 * K, dtype=torch.int64, device="cuda")
    wide_ids[:, ::2] = ids

    def both(x, w, ids):
        logp, lse = ops.linear_topk_logprob_fwd(x, w, ids)
        dx, dw = torch.empty(T, H, dtype=x.dtype, device="cuda"), torch.empty(V, H, dtype=x.dtype, device="cuda")
        ops.linear_topk_logprob_bwd(up, x, w, ids, lse, dx, dw)
        return logp, lse, dx, dw

    want = both(x, w, ids)
    assert all(torch.equal(a, b) for a, b in zip(both(wide_x[:, :H], wide_w[:, :H], wide_ids[:, ::2]), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(x, w, ids)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both(x, w, ids)
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_token_named_many_times(cuda_device):
    from test1_b200 import ops

    for T in (1, 300):
        x, w, _, up = _inputs(T, 64, 1030, 512, seed=8, masked=False)
        ids = torch.full((T, 512), 777, device="cuda")
        ids[:, -1] = 3
        ids[0] = 1029
        lp, ls, dx64, dw64 = oracle.listed_logprob(x, w, ids, 0.7, dlogp=up)
        logp, lse = ops.linear_topk_logprob_fwd(x, w, ids, 0.7)
        assert float((logp - lp).abs().max()) <= _tol(x, w, 0.7) and float((lse - ls).abs().max()) <= _tol(x, w, 0.7)
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        ops.linear_topk_logprob_bwd(up, x, w, ids, lse, dx, dw, 0.7)
        assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL


def test_two_streams_and_two_graphs_at_once(cuda_device):
    """Calls that share no buffer do not wait for one another and do not meet."""
    from test1_b200 import ops

    def run(x, w, ids, up, z, u):
        logp, lse = ops.linear_topk_logprob_fwd(x, w, ids)
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        ops.linear_topk_logprob_bwd(up, x, w, ids, lse, dx, dw)
        return (logp, lse, dx, dw, ops.linear_logits(x, w)) + ops.topk_logprobs(z, 50) + ops.sample_tokens(z, u, top_p=0.9) \
            + ops.sample_tokens(z, u, top_k=40) + ops.distillation_loss_fwd_bwd(logp, logp.roll(1, 0), ids, "jensen") \
            + ops.distillation_loss_fwd_bwd(z.view(-1, 11), z.roll(1, 0).view(-1, 11), index, "reverse", tail=False)

    sets, index = [], torch.arange(11, device="cuda").repeat(40 * 50017 // 11, 1)
    for seed in (9, 10):
        x, w, ids, up = _inputs(300, 256, 9001, 24, seed=seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        sets.append((x, w, ids, up, torch.randn(40, 50017, device="cuda", generator=g),
                     torch.rand(40, device="cuda", generator=g)))
    want = [run(*s) for s in sets]
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(*s)
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for stream, s in zip(streams, sets):
            with torch.cuda.stream(stream):
                got.append(run(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, w in zip(got, want) for a, b in zip(o, w))
        for stream, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for (_, o), w in zip(graphs, want) for a, b in zip(o, w))


def test_more_than_32_bits_of_logits(cuda_device):
    """The rows behind 2^31 logits are what they are by themselves."""
    from test1_b200 import ops

    T, H, V = 17000, 64, 128257
    x, w, _, _ = _inputs(T, H, V, 1, seed=11, masked=False)
    u = torch.rand(T, device="cuda", generator=torch.Generator(device="cuda").manual_seed(11))
    logits = ops.linear_logits(x, w)
    assert logits.stride(0) * (T - 1) > 2 ** 31
    last = slice(T - 200, T)
    assert torch.equal(logits[last], ops.linear_logits(x[last], w))
    alone = logits[last].clone()
    for z, part in ((logits, alone), (logits.bfloat16(), alone.bfloat16())):
        for all_rows, few in ((ops.topk_logprobs(z, 8), ops.topk_logprobs(part, 8)),
                              (ops.sample_tokens(z, u, top_k=8), ops.sample_tokens(part, u[last], top_k=8)),
                              (ops.sample_tokens(z, u, top_p=0.9), ops.sample_tokens(part, u[last], top_p=0.9)),
                              (ops.sample_tokens(z, u, top_k=1500), ops.sample_tokens(part, u[last], top_k=1500))):
            assert all(torch.equal(a[last], b) for a, b in zip(all_rows, few))


def test_refusals(cuda_device):
    from test1_b200 import ops

    x, w, ids, up = _inputs(4, 64, 100, 3)
    with pytest.raises(RuntimeError, match="int64"):
        ops.linear_topk_logprob_fwd(x, w, ids.int())
    with pytest.raises(RuntimeError, match="dtype"):
        ops.linear_topk_logprob_fwd(x.float(), w, ids)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        ops.linear_logits(x[:, :60].contiguous(), w[:, :60].contiguous())
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.linear_topk_logprob_fwd(x, w, ids.cpu())
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.linear_topk_logprob_bwd(up, x, w, ids, up[:, 0], torch.empty(4, 128, dtype=x.dtype, device="cuda")[:, ::2],
                                    torch.empty_like(w))
