"""The distillation loss kernels at inputs that the other tests leave out: NaN
in a student's log-probabilities."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
KINDS = ["forward", "reverse", "jensen"]


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
