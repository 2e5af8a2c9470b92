"""Forward passes large enough that their rows are packed first (more than 256
tokens, tokens x H x V above 2e10), and how exact the summed logits are.

A logit is summed from accumulators of at most 23 blocks of 64 products (1472),
to which the tensor cores add 16 products a step and drop what falls below the
sum's last bit: at most 92 steps of 2^-23 of the partial sum, which is no
larger than the row's largest |logit| by more than a small part of it; the
accumulators' sum, the exponentials and the join add 8 x 2^-23.  On average a
step drops 0.36 of a last bit of a sum that grows from nothing: 92 x 0.18 =
17 x 2^-23 of the logit, 20 with the rest.  (One accumulator of 4096 products
would lose 46.)"""
import pytest
import torch

from _answer_oracle import logprob as oracle

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -23
#         T, H, V: column blocks joined by a launch of their own (V > 8192), or by the last of them
PACKED = [(700, 1032, 30011), (1500, 2048, 8001), (1031, 4096, 5003)]


def _inputs(T, H, V):
    g = torch.Generator(device="cuda").manual_seed(T + H + V)
    w = (torch.randn(V, H, device="cuda", generator=g) * 2 / H ** 0.5).bfloat16()
    ids = torch.randint(0, V, (T,), device="cuda", generator=g)
    x = torch.randn(T, H, device="cuda", generator=g) + 3 * torch.rand(T, 1, device="cuda", generator=g) * w[ids].float()
    t = ids.clone()
    t[torch.rand(T, device="cuda", generator=g) < 0.4] = -100
    t[T // 2] = V  # not a vocabulary index
    x = x.bfloat16()
    x[(t < 0) | (t >= V)] = torch.tensor([float("nan"), float("inf")] * (H // 2), device="cuda").bfloat16()
    return x, w, t


def _largest(x, w, t, tau):
    """Largest |logit| of every row that counts."""
    rows = ((t >= 0) & (t < w.shape[0])).nonzero()[:, 0]
    return rows, torch.cat([(x[r].double() @ w.double().t()).abs().max(1).values / tau for r in rows.split(256)])


def _check(x, w, t, logp, lse, tau):
    lp, ls, _, _ = oracle(x, w, t, w.shape[0], temperature=tau)
    rows, size = _largest(x, w, t, tau)
    for got, want in ((logp, lp), (lse, ls)):
        off = (got.double() - want).abs()
        assert float((off[rows] / size).max()) <= (92 + 8) * ULP
        assert float((off[rows] / size).square().mean().sqrt()) <= 20 * ULP
        dead = torch.ones_like(t, dtype=torch.bool).index_fill_(0, rows, False)
        assert not bool(got[dead].any())


@pytest.mark.parametrize("T,H,V", PACKED)
@pytest.mark.parametrize("tau", [1.0, 0.7])
def test_packed_forward(T, H, V, tau, cuda_device):
    from test1_b200 import ops

    assert T > 256 and T * H * V > 2e10
    x, w, t = _inputs(T, H, V)
    first = ops.linear_logprob_fwd(x, w, t, temperature=tau)
    _check(x, w, t, *first, tau)
    assert all(torch.equal(a, b) for a, b in zip(first, ops.linear_logprob_fwd(x, w, t, temperature=tau)))
    assert ops.native.gemm_error() == 0


@pytest.mark.parametrize("T,H,V", [(300, 1024, 5003), (300, 1472, 2000), (300, 4096, 2000), (300, 8192, 1000), (64, 4096, 20011)])
def test_logits_of_unpacked_batches(T, H, V, cuda_device):
    from test1_b200 import ops

    x, w, t = _inputs(T, H, V)
    _check(x, w, t, *ops.linear_logprob_fwd(x, w, t), 1.0)


@pytest.mark.parametrize("T,H,V", PACKED)
def test_packed_forward_of_no_or_one_answer(T, H, V, cuda_device):
    from test1_b200 import ops

    x, w, t = _inputs(T, H, V)
    none = torch.full_like(t, -100)
    assert not any(bool(v.any()) for v in ops.linear_logprob_fwd(x, w, none))
    for at in (int((t >= 0).nonzero()[0]), int((t >= 0).nonzero()[-1])):
        one = none.clone()
        one[at] = t[at]
        _check(x, w, one, *ops.linear_logprob_fwd(x, w, one), 1.0)


@pytest.mark.parametrize("T,H,V", PACKED)
def test_packed_forward_strided_on_another_stream_and_captured(T, H, V, cuda_device):
    from test1_b200 import ops

    x, w, t = _inputs(T, H, V)
    want = ops.linear_logprob_fwd(x, w, t)
    wide = torch.full((T, H + 72), float("nan"), device="cuda").bfloat16()
    wide[:, 8:8 + H] = x
    got = ops.linear_logprob_fwd(wide[:, 8:8 + H], w, torch.stack([t, t], 1)[:, 0])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.linear_logprob_fwd(x.clone(), w.clone(), t.clone())
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear_logprob_fwd(x, w, t)
    for shift in (0, 1):  # other targets, another number of rows
        t.copy_(torch.where(torch.arange(T, device="cuda") % (2 + shift) == 0, -100, t))
        want = ops.linear_logprob_fwd(x, w, t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
