"""Edges of the preference and policy losses on the GPU."""
import pytest
import torch

import _answer_oracle as oracle

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("S", [1, 4, 8])
def test_policy_gradient_far_below_the_reference(S, cuda_device):
    """e = ref - logp of minus thousands and minus infinity: the KL term grows
    with -e (to infinity), its derivative, 1 - exp(e), ends at 1.  A few fp32
    operations on numbers of about 1: 8 x 2^-24."""
    from test1_b200 import ops

    e = torch.tensor([-INF, -5000.3, -1000.7, -100.1, -20.3, -1.1, -0.26, 0.0], device="cuda", dtype=torch.float64)
    lp = torch.full((8,), -0.5, device="cuda")
    ref = (lp.double() + e).float()
    t = torch.zeros(8, dtype=torch.int64, device="cuda")
    adv = torch.zeros(8 // S, device="cuda")
    loss, d, stats = ops.policy_loss_fwd_bwd(lp, lp, ref, adv, t, S, kl_coef=0.5)
    e = ref.double() - lp.double()
    assert float((d.double() + 0.5 * torch.expm1(e) / 8).abs().max()) <= 8 * 2.0 ** -24 * 0.5 / 8
    assert float(loss) == INF and float(stats[0]) == INF
    loss, d, _ = ops.policy_loss_fwd_bwd(lp[1:], lp[1:], ref[1:], torch.zeros(7, device="cuda"), t[1:], 1, kl_coef=0.5)
    want = oracle.policy(lp[1:], lp[1:], ref[1:], torch.zeros(7, device="cuda"), t[1:], 1, 0.2, 0.2, 0.5, "token")
    assert abs(float(loss) - float(want[0])) <= 1e-6 * float(want[0])
    assert float((d.double() - want[1]).abs().max()) <= 8 * 2.0 ** -24 * 0.5 / 7
