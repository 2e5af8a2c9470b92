"""The distillation loss kernels against the definition in 64 bits.

A term is a product of a probability and a difference of logarithms, each
rounded a few times in fp32: (16 + 8 A) 2^-24 of (p + q) (|log p| + |log q| + 1),
where A, the largest |log| of the row, stands for the roundings of a and b that
exp carries over to p and q.  A gradient is such terms without the sum, over
the number of rows."""
import math

import pytest
import torch

import _lists_oracle as oracle

pytestmark = pytest.mark.gpu
KINDS = ["forward", "reverse", "jensen"]


def _inputs(T, K, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed + 100 * T + K)
    share = 1 - 0.6 * torch.rand(T, 1, generator=g) ** 2 - 1e-3
    b = torch.log_softmax(2 * torch.randn(T, K, generator=g), 1) + share.log()
    a = torch.log_softmax(torch.cat([b, torch.log1p(-share)], 1) + 0.5 * torch.randn(T, K + 1, generator=g), 1)[:, :K]
    b = b.to(dtype)
    ids = torch.arange(K).repeat(T, 1)
    if T > 2:
        ids[torch.rand(T, K, generator=g) < 0.2] = -100
        ids[1] = -1
        b[2] = -math.inf
        a[1], b[1] = float("nan"), float("nan")
        b[-1, 0] = -math.inf
    return a, b, ids


def _check(a, b, ids, kind, tail):
    from test1_b200 import ops

    K = a.shape[1]
    loss, dlogp, each = ops.distillation_loss_fwd_bwd(a.cuda(), b.cuda(), ids.cuda(), kind=kind, tail=tail)
    keep = (ids >= 0) & (b.double() > -math.inf)
    clean = torch.where(keep, a, 0.0)
    want, grad, per, size = oracle.distillation(clean, torch.where(keep, b, -math.inf), ids, kind, tail)
    logs = torch.where(keep, torch.maximum(clean.double().abs(), torch.where(keep, b.double(), 0.0).abs()), 0.0)
    A = max(float(logs.max()) if logs.numel() else 0.0, 14.0 if tail else 0.0)
    eps = (16 + 8 * A) * 2.0 ** -24
    n = max(1, int(keep.any(1).sum()))
    assert loss.shape == () and loss.dtype == dlogp.dtype == each.dtype == torch.float32
    assert bool(((each.cpu().double() - per).abs() <= eps * size).all())
    assert abs(float(loss) - float(want)) <= eps * float(size.sum()) / n + 2.0 ** -24 * abs(float(want))
    # the rest's derivative, of which a gradient has p_k times
    tol = eps * (size[:, None] + 1) / n * (torch.exp(clean.double()) + torch.exp(torch.where(keep, b.double(), 0.0)) + 2.0 ** -20)
    if tail and kind == "forward":  # q_r / p_r
        rest = lambda v: (1 - torch.where(keep, v.double().exp(), 0.0).sum(1, keepdim=True)).clamp(min=2.0 ** -20)  # noqa: E731
        tol = tol * (1 + rest(b) / rest(clean))
    assert bool(((dlogp.cpu().double() - grad).abs() <= tol).all())
    assert not bool(dlogp.cpu()[~keep].any()) and not bool(each.cpu()[~keep.any(1)].any())
    assert dlogp.shape == (a.shape[0], K)


@pytest.mark.parametrize("T,K", [(1, 1), (5, 3), (3, 31), (40, 32), (33, 33), (9, 64), (17, 65), (6, 128), (5, 129), (4, 512)])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tail", [True, False])
def test_against_definition(T, K, kind, tail, cuda_device):
    _check(*_inputs(T, K), kind, tail)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tail", [True, False])
def test_bf16_teacher(kind, tail, cuda_device):
    _check(*_inputs(30, 20, seed=1, dtype=torch.bfloat16), kind, tail)


@pytest.mark.parametrize("kind", KINDS)
def test_rest_below_its_floor(kind, cuda_device):
    """Lists that hold everything, or a little more by rounding."""
    a = torch.tensor([[-1e-9, -30.0], [math.log(0.75), math.log(0.25)], [math.log(0.5), math.log(0.50001)], [-5.0, -6.0]])
    b = torch.tensor([[math.log(0.5), math.log(0.4)], [math.log(0.25), math.log(0.75)], [-1e-7, -20.0], [-1e-7, -20.0]])
    _check(a, b, torch.arange(2).repeat(4, 1), kind, True)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tail", [True, False])
def test_agreement_has_no_gradient(kind, tail, cuda_device):
    from test1_b200 import ops

    _, b, ids = _inputs(2, 16, seed=2)
    loss, dlogp, each = ops.distillation_loss_fwd_bwd(b.cuda(), b.cuda(), ids.cuda(), kind=kind, tail=tail)
    assert float(loss.abs()) < 2e-6 and float(dlogp.abs().max()) < 2e-6


@pytest.mark.parametrize("kind", KINDS)
def test_improbable_tokens(kind, cuda_device):
    """Probabilities of 0: 0 log 0 is 0, and no gradient is NaN."""
    from test1_b200 import ops

    a = torch.tensor([[-0.1, -200.0, -3.0]], device="cuda")
    b = torch.tensor([[-200.0, -1.0, -0.7]], device="cuda")
    loss, dlogp, _ = ops.distillation_loss_fwd_bwd(a, b, torch.arange(3, device="cuda")[None], kind=kind)
    assert bool(torch.isfinite(loss)) and bool(torch.isfinite(dlogp).all())


def test_no_rows_and_no_entries(cuda_device):
    from test1_b200 import ops

    for T in (0, 7):
        a = torch.zeros(T, 4, device="cuda")
        loss, dlogp, each = ops.distillation_loss_fwd_bwd(a, a, torch.full((T, 4), -1, device="cuda"))
        assert float(loss) == 0 and not bool(dlogp.any()) and not bool(each.any()) and each.shape == (T,)


def test_many_rows_repeat_and_strides(cuda_device):
    from test1_b200 import ops

    g = torch.Generator().manual_seed(3)
    T, K = 20011, 5
    b = torch.log_softmax(torch.randn(T, K + 1, generator=g), 1)[:, :K].contiguous()
    a = torch.log_softmax(torch.randn(T, K + 1, generator=g), 1)[:, :K].contiguous()
    ids = torch.arange(K).repeat(T, 1)
    ids[::3] = -1
    args = [t.cuda() for t in (a, b, ids)]
    want = ops.distillation_loss_fwd_bwd(*args, kind="jensen")
    p, q = torch.cat([a.double().exp(), 1 - a.double().exp().sum(1, keepdim=True)], 1), \
        torch.cat([b.double().exp(), 1 - b.double().exp().sum(1, keepdim=True)], 1)
    m = (p + q) / 2
    each = ((p * (p / m).log() + q * (q / m).log()).sum(1) / 2)[ids[:, 0] >= 0]
    assert abs(float(want[0]) - float(each.mean())) <= 128 * 2.0 ** -24 * 10
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(ops.distillation_loss_fwd_bwd(*args, kind="jensen"), want))
    wide = [torch.zeros(T, 2 * K, dtype=t.dtype, device="cuda") for t in args]
    for w, t in zip(wide, args):
        w[:, 1::2] = t
    got = ops.distillation_loss_fwd_bwd(*(w[:, 1::2] for w in wide), kind="jensen")
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.distillation_loss_fwd_bwd(*args, kind="jensen")
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_refusals(cuda_device):
    from test1_b200 import ops

    a = torch.zeros(2, 3, device="cuda")
    ids = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        ops.distillation_loss_fwd_bwd(a, a.half(), ids)
    with pytest.raises(RuntimeError, match="dtype"):
        ops.distillation_loss_fwd_bwd(a, a, ids.int())
    with pytest.raises(RuntimeError, match="dtype"):
        ops.distillation_loss_fwd_bwd(a.bfloat16(), a, ids)
