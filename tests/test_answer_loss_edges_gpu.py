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


# many sequences: a grid of blocks, sequences of one unit (their length or count per block
# no longer a cluster's), of fewer tokens than a warp has lanes and of more
@pytest.mark.parametrize("B,S", [(5000, 33), (5000, 8), (4800, 20), (40000, 1), (5002, 32)])
def test_many_sequences(B, S, cuda_device):
    """Tolerances: a handful of fp32 operations per token, sums in fp64."""
    from test1_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(B + S)
    rand = lambda *n: torch.randn(*n, device="cuda", generator=g)  # noqa: E731
    T = B * S
    t = torch.where(torch.rand(T, device="cuda", generator=g) < 0.6, 5, -100)
    lp = torch.where(t >= 0, -torch.rand(T, device="cuda", generator=g), float("nan"))
    old, ref, adv = lp + 0.2 * rand(T), lp + 0.3 * rand(T), rand(B) + 0.3
    for reduction in ("token", "sequence"):
        got = ops.policy_loss_fwd_bwd(lp, old, ref, adv, t, S, kl_coef=0.1, reduction=reduction)
        want = oracle.policy(lp, old, ref, adv, t, S, 0.2, 0.2, 0.1, reduction)
        for a, b, size in zip(got, want, (4.0, float(want[1].abs().max()), 1.0)):
            assert float((a.double() - b).abs().max()) <= 1e-5 * size
    got = ops.preference_loss_fwd_bwd(lp, ref, t, S, beta=0.3)
    ok = (t >= 0).view(B, S)
    r = 0.3 * torch.where(ok, (lp.double() - ref.double()).view(B, S), 0.0).sum(1)
    m, live = r[:B // 2] - r[B // 2:], ok[:B // 2].any(1) | ok[B // 2:].any(1)
    loss = torch.where(live, -torch.nn.functional.logsigmoid(m), 0.0).sum() / live.sum()
    d = torch.where(live, -0.3 * torch.sigmoid(-m), 0.0) / live.sum()
    d = torch.where(ok, torch.cat([d, -d])[:, None], 0.0).reshape(T)
    for a, b in zip(got, (loss, d, r)):
        assert float((a.double() - b).abs().max()) <= 1e-5 * float(b.abs().max())
