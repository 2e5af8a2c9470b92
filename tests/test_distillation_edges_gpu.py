"""The distillation loss kernels at inputs that the other tests leave out: NaN
in a student's log-probabilities, log-probabilities far below -1e4, tokens
beyond the student's vocabulary."""
import math

import pytest
import torch

import _lists_oracle as oracle
from test_distillation_gpu import _engine

pytestmark = pytest.mark.gpu
KINDS = ["forward", "reverse", "jensen"]
EPS = 2.0 ** -24


def _lists(T, K, seed=0):
    """Both models' log-probabilities of K tokens of a row, which hold 0.7 of
    the probability, and ids of which a fifth is left out."""
    g = torch.Generator().manual_seed(seed + 100 * T + K)
    a, b = (torch.log_softmax(torch.randn(T, K, generator=g), 1) + math.log(0.7) for _ in range(2))
    ids = torch.where(torch.rand(T, K, generator=g) < 0.2, -1, torch.arange(K))
    ids[:, 0] = 0
    return a, b, ids


@pytest.mark.parametrize("T,K", [(3, 1), (4, 5), (5, 32), (6, 33), (7, 64), (5, 100), (4, 129), (5, 512), (2000, 7), (3000, 32),
                                 (1200, 257)])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tail", [True, False])
def test_nan_of_a_kept_entry_is_not_hidden(T, K, kind, tail, cuda_device):
    """One NaN among a row's kept entries: the row, the loss and that entry's
    gradient are NaN, the other rows and what is left out stay as they are."""
    from test1_b200 import ops

    a, b, ids = _lists(T, K)
    args = [t.cuda() for t in (b, ids)]
    _, clean, each = ops.distillation_loss_fwd_bwd(a.cuda(), *args, kind=kind, tail=tail)
    row, col = T // 2, int((ids[T // 2] >= 0).nonzero()[-1])
    a[row, col] = float("nan")
    loss, grad, got = ops.distillation_loss_fwd_bwd(a.cuda(), *args, kind=kind, tail=tail)
    others = torch.arange(T) != row
    assert math.isnan(float(loss)) and math.isnan(float(got[row]))
    assert math.isnan(float(grad[row, col]))
    assert torch.equal(got.cpu()[others], each.cpu()[others]) and torch.equal(grad.cpu()[others], clean.cpu()[others])
    assert not bool(grad.cpu()[ids < 0].any())


@pytest.mark.parametrize("kind", KINDS)
def test_nan_goes_on_to_the_output_layer(kind, cuda_device):
    """Hidden states that have become NaN are seen in loss and gradients, with
    few rows and with many."""
    from test1_b200 import ops

    for T, H, V, K in ((4, 64, 300, 5), (300, 64, 600, 20)):
        g = torch.Generator(device="cuda").manual_seed(T)
        x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
        w = (torch.randn(V, H, device="cuda", generator=g) / 8).bfloat16()
        teacher, ids = torch.log_softmax(torch.randn(T, V, device="cuda", generator=g), 1).topk(K, 1)
        x[T // 2] = float("nan")
        logp, lse = ops.linear_topk_logprob_fwd(x, w, ids)
        loss, dlogp, _ = ops.distillation_loss_fwd_bwd(logp, teacher, ids, kind=kind)
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        ops.linear_topk_logprob_bwd(dlogp, x, w, ids, lse, dx, dw)
        assert bool(torch.isnan(logp[T // 2]).all()) and bool(torch.isnan(dlogp[T // 2]).all())
        assert math.isnan(float(loss))
        assert bool(torch.isnan(dx[T // 2]).all()) and bool(torch.isnan(dw).any())


@pytest.mark.parametrize("T,K", [(2, 1), (3, 5), (4, 8), (6, 33), (5, 65), (1000, 5)])
@pytest.mark.parametrize("kind", KINDS)
def test_far_below_without_a_tail(T, K, kind, cuda_device):
    """Log-probabilities about -2e4, as a temperature of 1e-3 makes them, and
    lists that leave lanes without an entry.

    d = (b - a) - ((max b - max a) + log of the sums' ratio) has three roundings
    at the size of the largest logarithm, A; a - max a is exact, p and q have the
    relative error of K <= 65 additions and an exponential, below 128 roundings
    with those of divisions and series; a gradient has p df/dp of its own entry and
    of all.  (A left-out entry taken for one of -1e4 is off by about 1e4.)"""
    from test1_b200 import ops

    a, b, ids = _lists(T, K, seed=1)
    a = a - 2e4
    args = [t.cuda() for t in (a, b, ids)]
    loss, dlogp, each = ops.distillation_loss_fwd_bwd(*args, kind=kind, tail=False)
    want, grad, per, _ = oracle.distillation(a, b, ids, kind, False)
    n, A, D = T, 2.0 ** 15, 16.0  # T rows; no logarithm above A, nor a difference of scaled ones above D
    tol = 4 * A * EPS + 128 * EPS * (1 + D)
    assert bool(((each.cpu().double() - per).abs() <= tol).all())
    assert abs(float(loss) - float(want)) <= tol
    assert bool(((dlogp.cpu().double() - grad).abs() <= 2 * tol / n).all())
    # the same as from lists without the shift, whose logarithms are nearer: -2e4 rounds a to 2^-10
    near, _, _ = ops.distillation_loss_fwd_bwd((a + 2e4).cuda(), *args[1:], kind=kind, tail=False)
    assert abs(float(near) - float(loss)) <= 2 * tol


@pytest.mark.parametrize("T,K", [(3, 5), (4, 64), (3, 129), (2000, 7)])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("tail", [True, False])
def test_students_without_any_probability(T, K, kind, tail, cuda_device):
    """A student's -inf: where the teacher has weight the forward divergence is
    infinite, the others stay finite; where the teacher's weight is 0 in fp32 too,
    none changes.

    The divergences sum K + 1 <= 130 terms, of logarithms below 16, and their
    factors have 128 roundings, as in the test above."""
    from test1_b200 import ops
    from test1_b200.ops import reference

    a, b, ids = _lists(T, K, seed=2)
    a[:, 0] = -math.inf
    b[0, 0] = -1000.0  # no weight
    loss, dlogp, each = (t.cpu() for t in ops.distillation_loss_fwd_bwd(a.cuda(), b.cuda(), ids.cuda(), kind=kind, tail=tail))
    want, grad, per = reference.distillation_loss_fwd_bwd(a, b, ids, kind, tail)
    assert torch.equal(torch.isinf(each), torch.isinf(per)) and bool(torch.isinf(each[1:]).all()) == (kind == "forward")
    assert not bool(torch.isinf(each[0])) and bool(torch.isinf(loss)) == (kind == "forward")
    finite = torch.isfinite(per)
    tol = 256 * EPS * 17
    assert bool(((each - per)[finite].abs() <= tol).all())
    assert bool(((dlogp - grad).abs() <= 2 * tol / T).all())


@pytest.mark.parametrize("kind,tail", [("forward", True), ("reverse", True), ("jensen", False)])
def test_teacher_of_a_larger_vocabulary(kind, tail, cuda_device):
    """Ids on the GPU that the student's vocabulary does not have take no part,
    as ids of -1 do not."""
    from test1_b200 import DistillationObjective

    eng, cfg = _engine(5, cuda_device, lr=0.0)
    V = cfg.vocab_size
    try:
        ids = torch.randint(0, V, (2, 64), device=cuda_device)
        g = torch.Generator(device="cuda").manual_seed(6)
        logps, top = torch.log_softmax(torch.randn(2, 64, V + 500, device="cuda", generator=g), -1).topk(24, -1)
        top[0, 0, 0], top[1, 1] = V, torch.arange(V, V + 24, device="cuda")
        outs = []
        for t in (top, torch.where(top < V, top, -1)):
            out = eng(input_ids=ids, labels=ids, objective=DistillationObjective(kind=kind, tail=tail), teacher_logps=logps,
                      teacher_ids=t)
            outs.append((out.loss.clone(), eng.last_objective["divergence"].clone(), eng.last_objective["logps"].clone()))
        assert all(torch.equal(a, b) for a, b in zip(*outs))
        assert not bool(outs[0][1][1, 1].any()) and bool(torch.isfinite(outs[0][0]))
        with pytest.raises(ValueError):
            eng(input_ids=ids, labels=ids, objective=DistillationObjective(), teacher_logps=logps, teacher_ids=top.cpu())
        eng.wait_for_updates()
    finally:
        eng.close()
