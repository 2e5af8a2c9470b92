"""Gradients of tokens that the model is nearly sure of (linear_logprob_bwd).

Their u = g (onehot - softmax) is small only because two large terms cancel:
g (1 - p) at the target.  What p is off by in absolute terms counts, against
1 - p.  Every row of dx is held to its own bound:

  lse is an fp32 number: half a unit in its last place, 2^-24 of the power of
  two above it, for a step between lse's binary ranges twice that; the
  exponential and the difference add 2^-21 at most.  Errors of a logit's sum
  count only where the forward's and the backward's differ, and they add up
  the same products in the same order.
  That error of p moves dx by as much of the target's row of W; u's rounding to
  bf16 moves it by 2^-9 of (1 - p) times that row, and 2^-9 in all for the
  others' rows; dx is rounded once more."""
import pytest
import torch

from _answer_oracle import logprob as oracle

pytestmark = pytest.mark.gpu


def _inputs(T, H, V, tau, tail):
    """Logits of 20 (over tau) and a spread of the others' below 1, targets
    whose probability is 1 - tail."""
    g = torch.Generator(device="cuda").manual_seed(T + H + V)
    rand = lambda *n: torch.randn(*n, device="cuda", generator=g)  # noqa: E731
    common = torch.ones(H, device="cuda") / H ** 0.5
    w = (rand(V, H) * 2 / H ** 0.5 + 4 * common).bfloat16()
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    gap = torch.log(torch.tensor(V / tail, device="cuda")) + 0.5 * torch.rand(T, 1, device="cuda", generator=g)
    own = w[t].float() - 4 * common
    x = ((own * gap / own.square().sum(1, keepdim=True) + 5 * common) * tau).bfloat16()
    return x, w, t, rand(T) / T


@pytest.mark.parametrize("tau", [1.0, 0.7])
@pytest.mark.parametrize("T,H,V", [(300, 4096, 2000), (520, 8192, 1000), (40, 2048, 3001), (300, 1024, 2000),
                                   (12, 4096, 2000), (3, 512, 5000)])
def test_rows_of_confident_targets(T, H, V, tau, cuda_device):
    from test1_b200 import ops

    x, w, t, up = _inputs(T, H, V, tau, 1e-3)
    lp, ls, dx64, _ = oracle(x, w, t, V, temperature=tau, dlogp=up)
    tail = -torch.expm1(lp)
    assert float(tail.max()) < 4e-3 and float(tail.min()) > 2e-4
    _, lse = ops.linear_logprob_fwd(x, w, t, temperature=tau)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ops.linear_logprob_bwd(up, x, w, t, lse, dx, dw, temperature=tau)
    of_p = ls.abs() * 2.0 ** -23 + 2.0 ** -21
    row = w.double().norm(dim=1)
    bound = up.double().abs() / tau * ((of_p + 2.0 ** -9 * tail) * row[t] + 2.0 ** -9 * tail * row.max()) + 2.0 ** -9 * dx64.norm(dim=1)
    off = (dx.double() - dx64).norm(dim=1)
    assert float((off / bound).max()) <= 1.0
