"""Log-probabilities of the output layer and their gradients (linear_logprob)
against the definition in 64 bits.

Tolerances.  A logit is a sum of H exact products accumulated in fp32, 16 of
them per step: its error is at most (H / 16 + 4) 2^-23 of the largest partial
sum, which is below the largest |logit| plus a few; exp, log and the joins
add a few more 2^-23 of the same size.  Gradients round u and g x to bf16 (at
most 2^-9 each, relative, element by element) and the result once more: the
2-norm of the error stays below 4 x 2^-9 of the result's."""
import pytest
import torch

from _answer_oracle import logprob as oracle

pytestmark = pytest.mark.gpu

#        T, H, V
SIZES = [(1, 64, 257), (2, 8, 5), (1, 256, 1), (33, 72, 255), (129, 264, 1000), (300, 520, 4097),
         (513, 256, 20011), (700, 1024, 2048), (257, 2048, 520),
         # few tokens: one or two column blocks of 8, x that fits in shared memory or not
         (8, 1032, 5003), (9, 4096, 777), (16, 2056, 1500), (5, 8192, 600), (16, 8192, 300), (17, 4096, 300),
         (3, 512, 40009), (16, 520, 4001)]
GRAD_TOL = 4 * 2.0 ** -9


def _inputs(T, H, V, seed=0, masked=True):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + T + H + V)
    w = (torch.randn(V, H, device="cuda", generator=g) * 2 / H ** 0.5).bfloat16()
    ids = torch.randint(0, V, (T,), device="cuda", generator=g)
    x = torch.randn(T, H, device="cuda", generator=g)
    x = (x + 3 * torch.rand(T, 1, device="cuda", generator=g) * w[ids].float()).bfloat16()
    if masked and T > 1:
        ids[1::3] = -100
        ids[T // 2] = V      # not a vocabulary index: ignored as well
    up = torch.randn(T, device="cuda", generator=g) / T
    return x, w, ids, up


def _logp_tol(H, logits_max, temperature=1.0):
    return (H / 16 + 32) * 2.0 ** -23 * (logits_max + 4) / min(1.0, temperature)


def _check_fwd(x, w, t, logp, lse, temperature=1.0):
    from test1_b200.ops import native

    V, H = w.shape
    lp, ls, _, _ = oracle(x, w, t, V, temperature=temperature)
    tol = _logp_tol(H, float((x.float().norm(dim=1).nan_to_num(0, 0, 0).max() * w.float().norm(dim=1).max())), temperature)
    assert logp.dtype == lse.dtype == torch.float32 and logp.shape == lse.shape == t.shape
    assert float((logp - lp).abs().max()) <= tol
    assert float((lse - ls).abs().max()) <= tol
    assert native.gemm_error() == 0


def _rel(a, b):
    return float((a.double() - b).norm() / b.norm().clamp_min(1e-30))


@pytest.mark.parametrize("T,H,V", SIZES)
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_forward(T, H, V, temperature, cuda_device):
    from test1_b200 import ops

    x, w, t, _ = _inputs(T, H, V)
    logp, lse = ops.linear_logprob_fwd(x, w, t, temperature=temperature)
    _check_fwd(x, w, t, logp, lse, temperature)


@pytest.mark.parametrize("T,H,V", SIZES)
@pytest.mark.parametrize("temperature", [1.0, 0.6])
def test_backward(T, H, V, temperature, cuda_device):
    from test1_b200 import ops
    from test1_b200.ops import native

    x, w, t, up = _inputs(T, H, V, seed=1)
    lp, ls, dx64, dw64 = oracle(x, w, t, V, temperature=temperature, dlogp=up)
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))  # must be fully written
    ops.linear_logprob_bwd(up, x, w, t, ls.float(), dx, dw, temperature=temperature)
    if V > 1:
        assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL
    else:  # one class: its probability is 1, lse and logit differ by rounding alone
        assert float(dx.abs().max()) < 1e-4 and float(dw.abs().max()) < 1e-4
    assert native.gemm_error() == 0


def test_ignored_rows_hold_anything(cuda_device):
    """NaN and infinities in hidden states and upstream gradients of ignored
    tokens reach no output; a whole batch of ignored tokens gives zeros."""
    from test1_b200 import ops

    x, w, t, up = _inputs(200, 128, 1003)
    dead = (t < 0) | (t >= 1003)
    bad_x, bad_up = x.clone(), up.clone()
    bad_x[dead] = torch.tensor([float("nan"), float("inf")] * 64, device="cuda").bfloat16()
    bad_up[dead] = float("nan")
    outs = []
    for xx, uu in ((x, up), (bad_x, bad_up)):
        logp, lse = ops.linear_logprob_fwd(xx, w, t)
        dx, dw = torch.empty_like(x), torch.empty_like(w)
        ops.linear_logprob_bwd(uu, xx, w, t, lse, dx, dw)
        outs.append((logp, lse, dx, dw))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert bool((outs[0][0][dead] == 0).all()) and bool((outs[0][2][dead] == 0).all())
    none = torch.full_like(t, -100)
    logp, lse = ops.linear_logprob_fwd(bad_x, w, none)
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))
    ops.linear_logprob_bwd(bad_up, bad_x, w, none, lse, dx, dw)
    assert not any(bool(v.any()) for v in (logp, lse, dx, dw))


def test_ignore_index_inside_the_vocabulary(cuda_device):
    from test1_b200 import ops

    x, w, t, up = _inputs(150, 64, 40, masked=False)
    lp, ls, dx64, dw64 = oracle(x, w, t, 40, ignore_index=7, dlogp=up)
    logp, lse = ops.linear_logprob_fwd(x, w, t, ignore_index=7)
    assert float((logp - lp).abs().max()) < _logp_tol(64, 40)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ops.linear_logprob_bwd(up, x, w, t, lse, dx, dw, ignore_index=7)
    assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL


def test_zero_upstream_rows_and_no_tokens(cuda_device):
    from test1_b200 import ops

    x, w, t, up = _inputs(260, 96, 700, masked=False)
    up[::2] = 0
    _, ls, dx64, dw64 = oracle(x, w, t, 700, dlogp=up)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ops.linear_logprob_bwd(up, x, w, t, ls.float(), dx, dw)
    assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL and not bool(dx[::2].any())
    logp, lse = ops.linear_logprob_fwd(x[:0], w, t[:0])
    assert logp.shape == lse.shape == (0,)
    ops.linear_logprob_bwd(up[:0], x[:0], w, t[:0], lse, dx[:0], dw)
    assert not bool(dw.any())


def test_strided_operands(cuda_device):
    """Rows of wider buffers, strided targets and upstream gradients, a
    broadcast upstream gradient."""
    from test1_b200 import ops

    x, w, t, up = _inputs(140, 128, 900)
    wide_x = torch.full((140, 200), float("nan"), device="cuda").bfloat16()
    wide_w = torch.full((900, 136), float("nan"), device="cuda").bfloat16()
    wide_x[:, 8:136], wide_w[:, :128] = x, w
    xs, ws = wide_x[:, 8:136], wide_w[:, :128]
    ts = torch.stack([t, t], 1).reshape(-1)[::2]
    ups = torch.stack([up, up], 1).reshape(-1)[::2]
    logp, lse = ops.linear_logprob_fwd(xs, ws, ts)
    want = ops.linear_logprob_fwd(x, w, t)
    assert torch.equal(logp, want[0]) and torch.equal(lse, want[1])
    a, b = [torch.empty_like(x) for _ in "ab"], [torch.empty_like(w) for _ in "ab"]
    ops.linear_logprob_bwd(ups, xs, ws, ts, lse, a[0], b[0])
    ops.linear_logprob_bwd(up, x, w, t, lse, a[1], b[1])
    assert torch.equal(*a) and torch.equal(*b)
    one = torch.full((1,), -0.01, device="cuda")
    ops.linear_logprob_bwd(one.expand(140), x, w, t, lse, a[0], b[0])
    ops.linear_logprob_bwd(one.expand(140).contiguous(), x, w, t, lse, a[1], b[1])
    assert torch.equal(*a) and torch.equal(*b)


def test_vocabulary_in_several_pieces(cuda_device):
    """More [T, V] gradient than is held at a time: dx gathers the pieces'
    products, dW comes piece by piece."""
    from test1_b200 import ops

    T, H, V = 5000, 64, 128256
    x, w, t, up = _inputs(T, H, V)
    _, ls, dx64, dw64 = oracle(x, w, t, V, dlogp=up)
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))
    ops.linear_logprob_bwd(up, x, w, t, ls.float(), dx, dw)
    assert _rel(dx, dx64) < GRAD_TOL and _rel(dw, dw64) < GRAD_TOL


def test_gradient_against_differences(cuda_device):
    """sum(up logp) along a direction of exact bf16 steps, central
    differences: the third-order term is below h^2 = 2^-12 of the second."""
    from test1_b200 import ops

    T, H, V = 40, 64, 300
    g = torch.Generator(device="cuda").manual_seed(5)
    grid = lambda *n: (torch.randint(-24, 25, n, device="cuda", generator=g) / 16)  # noqa: E731
    x, w = grid(T, H), grid(V, H) / 8
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    up = torch.randn(T, device="cuda", generator=g)
    step = lambda n: torch.randint(-1, 2, n, device="cuda", generator=g) / 64.0  # noqa: E731
    f = lambda a, b: float((up.double() * ops.linear_logprob_fwd(a.bfloat16(), b.bfloat16(), t)[0].double()).sum())  # noqa: E731
    _, lse = ops.linear_logprob_fwd(x.bfloat16(), w.bfloat16(), t)
    dx, dw = torch.empty_like(x).bfloat16(), torch.empty_like(w).bfloat16()
    ops.linear_logprob_bwd(up, x.bfloat16(), w.bfloat16(), t, lse, dx, dw)
    ex, ew = step((T, H)), step((V, H)) / 8
    for grad, num in (((dx.double() * ex).sum(), f(x + ex, w) - f(x - ex, w)),
                      ((dw.double() * ew).sum(), f(x, w + ew) - f(x, w - ew))):
        scale = float((dx.double().norm() * ex.norm()) / ex.numel() ** 0.5 + (dw.double().norm() * ew.norm()) / ew.numel() ** 0.5)
        assert abs(float(grad) - num / 2) < 2e-2 * abs(num / 2) + 2e-2 * scale


def test_other_stream_and_repeat(cuda_device):
    """On a stream of its own, right after the inputs are made there; two
    runs give the same bits."""
    from test1_b200 import ops

    x, w, t, up = _inputs(700, 256, 5003)
    want = ops.linear_logprob_fwd(x, w, t)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ops.linear_logprob_bwd(up, x, w, t, want[1], dx, dw)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x2, w2 = x.clone(), w.clone()
        got = ops.linear_logprob_fwd(x2, w2, t)
        dx2, dw2 = torch.empty_like(x), torch.empty_like(w)
        ops.linear_logprob_bwd(up, x2, w2, t, got[1], dx2, dw2)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(dx2, dx) and torch.equal(dw2, dw)


def test_refusals(cuda_device):
    from test1_b200 import ops

    x, w, t, up = _inputs(16, 64, 100)
    lse = torch.zeros(16, device="cuda")
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    for bad in (dict(x=x.float()), dict(w=w.float()), dict(t=t.int()), dict(t=t[:-1]), dict(x=x[:, :56]),
                dict(x=x[:, :60], w=w[:, :60]), dict(x=x.t()[:16, :16].t(), w=w), dict(temperature=0.0),
                dict(temperature=float("nan")), dict(t=t.cpu()), dict(w=w[:0]), dict(x=x.view(-1)[1:961].view(15, 64), t=t[:15])):
        a = {**dict(x=x, w=w, t=t, temperature=1.0), **bad}
        with pytest.raises(RuntimeError):
            ops.linear_logprob_fwd(a["x"], a["w"], a["t"], temperature=a["temperature"])
    for bad in (dict(up=up[:-1]), dict(up=up.double()), dict(lse=lse[:-1]), dict(dx=dx[:-1]), dict(dw=dw.t()),
                dict(dx=dx.float()), dict(dw=dw[:, ::2])):
        a = {**dict(up=up, lse=lse, dx=dx, dw=dw), **bad}
        with pytest.raises(RuntimeError):
            ops.linear_logprob_bwd(a["up"], x, w, t, a["lse"], a["dx"], a["dw"])


@pytest.mark.parametrize("T", [5, 300])
def test_captured_in_a_graph(T, cuda_device):
    """Forward and backward in one graph, replayed on other hidden states."""
    from test1_b200 import ops

    x, w, t, up = _inputs(T, 256, 5003)
    dx, dw = torch.empty_like(x), torch.empty_like(w)

    def f():
        logp, lse = ops.linear_logprob_fwd(x, w, t)
        ops.linear_logprob_bwd(up, x, w, t, lse, dx, dw)
        return logp, lse

    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    for k in range(2):
        x.mul_(1 - 0.25 * k)
        want = f()
        want_dx, want_dw = dx.clone(), dw.clone()
        dx.zero_(), dw.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert torch.equal(dx, want_dx) and torch.equal(dw, want_dw)
