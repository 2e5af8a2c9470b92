"""At most 16 tokens: what ignored tokens and tokens without a gradient hold
reaches no other token and no output."""
import pytest
import torch

from _answer_oracle import logprob as oracle

pytestmark = pytest.mark.gpu

GRAD_TOL = 4 * 2.0 ** -9  # u and the results are rounded to bf16


@pytest.mark.parametrize("T", [2, 8, 9, 16])
@pytest.mark.parametrize("H,V", [(64, 70), (1032, 5003)])
def test_dead_tokens_hold_anything(T, H, V, cuda_device):
    from test1_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(T + H)
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    w = (torch.randn(V, H, device="cuda", generator=g) * 2 / H ** 0.5).bfloat16()
    t = torch.randint(0, V, (T,), device="cuda", generator=g)
    up = torch.randn(T, device="cuda", generator=g)
    t[T // 2:] = -100
    up[0] = 0.0  # a token without a gradient
    x[T // 2:] = torch.tensor([float("nan"), float("inf")] * (H // 2), device="cuda").bfloat16()
    up[T // 2:] = float("nan")
    logp, lse = ops.linear_logprob_fwd(x, w, t)
    lp, ls, dx64, dw64 = oracle(x, w, t, V, dlogp=up)
    assert float((logp - lp).abs().max()) < 1e-4 and float((lse - ls).abs().max()) < 1e-4
    assert not bool(logp[T // 2:].any()) and not bool(lse[T // 2:].any())
    bad = lse.clone()
    bad[T // 2:] = float("nan")
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))
    ops.linear_logprob_bwd(up, x, w, t, bad, dx, dw)
    assert not bool(dx[0].any()) and not bool(dx[T // 2:].any())
    assert float((dx.double() - dx64).norm()) <= GRAD_TOL * float(dx64.norm())
    assert float((dw.double() - dw64).norm()) <= GRAD_TOL * float(dw64.norm())
    w[V // 2] = float("inf")  # dead tokens' gradients are 0 whatever W holds
    ops.linear_logprob_bwd(up, x, w, t, bad, dx, dw)
    assert not bool(dx[0].any()) and not bool(dx[T // 2:].any())
