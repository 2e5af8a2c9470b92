"""The likeliest tokens of rows of logits and draws from them, against the
definitions in 64 bits.

Tokens are compared exactly.  Weights are held to 2^-(62 - log2 V) of the
largest and 64-bit exponentials, so a draw whose u lies further than 1e-9 from
a border has to agree; the inputs are fixed.

Log-probabilities: (z - m) / tau has two roundings of 2^-24 relative; the sum
of weights is added up in at most 96 + 16 + 16 steps, and an exponential is off
by 2^-22 and by its argument's rounding, 2^-23 |t| e^t < 2^-24: below
(128 + 32) 2^-24 together.  The last subtraction adds 2^-24 of the result."""
import math

import pytest
import torch

import _lists_oracle as oracle

pytestmark = pytest.mark.gpu
INF = math.inf

#        B, V
SIZES = [(1, 1), (3, 2), (2, 31), (5, 33), (2, 511), (2, 513), (7, 1024), (2, 2049), (2, 16384), (3, 16385), (2, 50021),
         (2, 128256), (1, 131073), (1, 200003), (1, 262145), (1, 393216)]


def _logits(B, V, kind, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(100 * seed + B + V)
    z = 2 * torch.randn(B, V, device="cuda", generator=g)
    if kind == "peaked":
        at = torch.randint(0, V, (B, 20), device="cuda", generator=g)
        z.scatter_add_(1, at, 10 * torch.rand(B, 20, device="cuda", generator=g))
    elif kind == "equal":
        z.fill_(-3.5)
    elif kind == "ties":
        z = z.round()
    elif kind == "masked":
        z.masked_fill_(torch.rand(B, V, device="cuda", generator=g) > 0.02, -INF)
        z[0] = -INF
        if B > 1:
            z[1] = torch.finfo(dtype).min
    elif kind == "nan":
        z[:, ::3] = float("nan")
        z[:, 1::5] = -INF
        z[0, V // 2] = INF
        z[-1, V // 3::V // 3 + 1] = INF
    return z.to(dtype), g


def _check_logp(got, want):
    finite = torch.isfinite(want)
    assert torch.equal(got.cpu().double()[~finite], want[~finite])
    tol = 160 * 2.0 ** -24 + 4 * 2.0 ** -24 * want[finite].abs()
    assert bool(((got.cpu().double()[finite] - want[finite]).abs() <= tol).all())


@pytest.mark.parametrize("B,V", SIZES)
@pytest.mark.parametrize("kind", ["plain", "ties", "masked"])
def test_topk_sizes(B, V, kind, cuda_device):
    from test1_b200 import ops

    z, _ = _logits(B, V, kind, torch.float32)
    for k in {1, min(V, 50), min(V, 512)}:
        logp, ids = ops.topk_logprobs(z, k, temperature=0.7)
        want, at = oracle.topk(z, k, 0.7)
        assert ids.dtype == torch.int64 and logp.dtype == torch.float32 and ids.shape == logp.shape == (B, k)
        assert torch.equal(ids.cpu(), at)
        _check_logp(logp, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["plain", "peaked", "equal", "ties", "masked", "nan"])
@pytest.mark.parametrize("k", [1, 3, 64, 333])
def test_topk_kinds(dtype, kind, k, cuda_device):
    from test1_b200 import ops

    for B, V in ((4, 1000), (2, 20011)):
        z, _ = _logits(B, V, kind, dtype, seed=1)
        logp, ids = ops.topk_logprobs(z, k)
        want, at = oracle.topk(z, k, 1.0)
        assert torch.equal(ids.cpu(), at)
        _check_logp(logp, want)


CUTS = [(0, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (50, 0.95, 0.02), (1, 0.5, 1.0), (700, 0.999, 0.0),
        (10 ** 9, 0.01, 0.0)]


@pytest.mark.parametrize("B,V", SIZES)
@pytest.mark.parametrize("top_k,top_p,min_p", CUTS)
def test_sample_sizes(B, V, top_k, top_p, min_p, cuda_device):
    from test1_b200 import ops

    z, g = _logits(B, V, "plain", torch.float32, seed=2)
    u = torch.rand(B, device="cuda", generator=g)
    token, logp = ops.sample_tokens(z, u, temperature=0.8, top_k=top_k, top_p=top_p, min_p=min_p)
    at, want = oracle.sample(z, u, 0.8, top_k, top_p, min_p)
    assert token.dtype == torch.int64 and logp.dtype == torch.float32
    assert torch.equal(token.cpu(), at)
    _check_logp(logp, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["peaked", "equal", "ties", "masked", "nan"])
@pytest.mark.parametrize("top_k,top_p,min_p", CUTS)
def test_sample_kinds(dtype, kind, top_k, top_p, min_p, cuda_device):
    from test1_b200 import ops

    for B, V in ((33, 1000), (6, 20011)):
        z, g = _logits(B, V, kind, dtype, seed=3)
        u = torch.rand(B, device="cuda", generator=g)
        u[0], u[B - 1] = 0.0, 1 - 2.0 ** -24
        u[2] = float("nan")
        token, logp = ops.sample_tokens(z, u, temperature=1.3, top_k=top_k, top_p=top_p, min_p=min_p)
        at, want = oracle.sample(z, u, 1.3, top_k, top_p, min_p)
        assert torch.equal(token.cpu(), at)
        _check_logp(logp, want)


@pytest.mark.parametrize("tau", [1e-3, 0.05, 30.0])
def test_temperatures(tau, cuda_device):
    from test1_b200 import ops

    z, g = _logits(8, 5003, "plain", torch.float32, seed=4)
    u = torch.rand(8, device="cuda", generator=g)
    token, logp = ops.sample_tokens(z, u, temperature=tau, top_p=0.97)
    at, want = oracle.sample(z, u, tau, 0, 0.97, 0.0)
    assert torch.equal(token.cpu(), at)
    _check_logp(logp, want)
    logp, ids = ops.topk_logprobs(z, 20, temperature=tau)
    want, at = oracle.topk(z, 20, tau)
    assert torch.equal(ids.cpu(), at)
    _check_logp(logp, want)


@pytest.mark.parametrize("tau", [1e-37, 1e-6, 2.0 ** 64])
def test_temperatures_and_logits_at_their_ends(tau, cuda_device):
    """Rows of the type's lowest and largest values, alone and among others, and
    numbers u outside [0, 1), which count as its ends (NaN as 0)."""
    from test1_b200 import ops

    z, _ = _logits(6, 4001, "plain", torch.float32, seed=8)
    least, most = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    z[1], z[2], z[3, ::2], z[4, 7] = least, most, least, -INF
    u = torch.tensor([1.0, float("nan"), -3.0, INF, -INF, 0.5], device="cuda")
    for top_k, top_p, min_p in [(0, 1.0, 0.0), (7, 1.0, 0.0), (0, 0.5, 0.0), (0, 1.0, 0.3), (2000, 0.7, 0.1)]:
        token, logp = ops.sample_tokens(z, u, tau, top_k, top_p, min_p)
        at, want = oracle.sample(z, u, tau, top_k, top_p, min_p)
        assert torch.equal(token.cpu(), at)
        _check_logp(logp, want)
    logp, ids = ops.topk_logprobs(z, 9, tau)
    want, at = oracle.topk(z, 9, tau)
    assert torch.equal(ids.cpu(), at)
    _check_logp(logp, torch.where(want < least, -INF, want))  # fp32 has no such numbers


def test_rows_apart_and_unaligned(cuda_device):
    from test1_b200 import ops

    for dtype in (torch.float32, torch.bfloat16):
        z, g = _logits(5, 4001, "plain", dtype, seed=5)
        u = torch.rand(5, device="cuda", generator=g)
        wide = torch.full((5, 4010), float("nan"), dtype=dtype, device="cuda")
        view = wide[:, 3:4004]
        view.copy_(z)
        for a, b in zip(ops.topk_logprobs(z, 40), ops.topk_logprobs(view, 40)):
            assert torch.equal(a, b)
        for a, b in zip(ops.sample_tokens(z, u, top_p=0.9), ops.sample_tokens(view, u, top_p=0.9)):
            assert torch.equal(a, b)
        same = z[:1].expand(5, -1)  # one row, five draws
        at, _ = oracle.sample(z[:1].repeat(5, 1), u, 1.0, 0, 0.9, 0.0)
        assert torch.equal(ops.sample_tokens(same, u, top_p=0.9)[0].cpu(), at)
        assert torch.equal(ops.sample_tokens(z, u.repeat_interleave(2)[::2], top_p=0.9)[0], ops.sample_tokens(z, u, top_p=0.9)[0])


def test_no_rows(cuda_device):
    from test1_b200 import ops

    z = torch.empty(0, 100, device="cuda")
    assert [t.shape for t in ops.topk_logprobs(z, 7)] == [(0, 7), (0, 7)]
    assert [t.shape for t in ops.sample_tokens(z, z[:, 0])] == [(0,), (0,)]


def test_many_rows(cuda_device):
    from test1_b200 import ops

    z, g = _logits(3000, 300, "ties", torch.float32, seed=6)
    u = torch.rand(3000, device="cuda", generator=g)
    at, _ = oracle.sample(z, u, 1.0, 20, 0.8, 0.0)
    assert torch.equal(ops.sample_tokens(z, u, top_k=20, top_p=0.8)[0].cpu(), at)
    _, ids = oracle.topk(z, 17, 1.0)
    assert torch.equal(ops.topk_logprobs(z, 17)[1].cpu(), ids)


def test_frequencies(cuda_device):
    """Draws of 2^18 evenly spread u: a token's share is its probability to
    within two of the spaces between them (one at either end)."""
    from test1_b200 import ops

    n = 1 << 18
    z = torch.tensor([[1.0, -INF, 0.5, 3.0, 0.5, -2.0]], device="cuda")
    u = torch.arange(n, device="cuda", dtype=torch.float32) / n
    token, _ = ops.sample_tokens(z.expand(n, -1), u)
    share = torch.bincount(token, minlength=6).double() / n
    assert bool(((share - torch.softmax(z[0].double(), 0)).abs() <= 2 / n).all())


def test_another_stream_and_a_graph(cuda_device):
    from test1_b200 import ops

    z, g = _logits(6, 30011, "plain", torch.float32, seed=7)
    u = torch.rand(6, device="cuda", generator=g)
    want = ops.sample_tokens(z, u, top_p=0.9) + ops.topk_logprobs(z, 9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample_tokens(z, u, top_p=0.9) + ops.topk_logprobs(z, 9)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    buf_z, buf_u = torch.zeros_like(z), torch.zeros_like(u)
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.sample_tokens(buf_z, buf_u, top_p=0.9) + ops.topk_logprobs(buf_z, 9)
        graphs.append((graph, out))
    buf_z.copy_(z)
    buf_u.copy_(u)
    for graph, out in graphs + graphs:
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(cuda_device):
    from test1_b200 import ops
    from test1_b200.ops import native

    z = torch.zeros(2, 8, device="cuda")
    with pytest.raises(RuntimeError, match="row-major"):
        ops.topk_logprobs(torch.zeros(8, 2, device="cuda").t(), 2)
    with pytest.raises(RuntimeError, match="one device|CUDA"):
        ops.sample_tokens(z, torch.zeros(2))
    with pytest.raises(RuntimeError, match="at most"):
        ops.topk_logprobs(torch.zeros(1, 393217, device="cuda"), 2)
    with pytest.raises(RuntimeError, match="k must lie"):
        native.topk_logprobs(z, 9)
    with pytest.raises(RuntimeError, match="top_p"):
        native.sample_tokens(z, z[:, 0].contiguous(), top_p=0.0)
    with pytest.raises(RuntimeError, match="temperature"):
        native.topk_logprobs(z, 2, 1e30)
