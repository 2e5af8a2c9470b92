"""The output layer under an objective, on the kernels: loss and gradients
against 64 bits, at a size whose rows are packed.

Tolerances: the hidden states that the log-probabilities see are those after
the norm, rounded; the gradients of its two operators are within 4 x 2^-9 of
theirs (2-norm), and the norm's backward pass rounds once or twice more."""
from types import SimpleNamespace

import pytest
import torch
from torch import nn

import _answer_oracle as oracle

pytestmark = pytest.mark.gpu


class _Weight(nn.Module):
    def __init__(self, w):
        super().__init__()
        self.weight = nn.Parameter(w, requires_grad=False)


def _rel(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("tau", [1.0, 0.8])
@pytest.mark.parametrize("kind", ["preference", "policy"])
def test_loss_and_gradients(kind, tau, cuda_device):
    from test1_b200 import PolicyObjective, PreferenceObjective, ops
    from test1_b200.objectives import ObjectiveStep
    from test1_b200.slide_fsdp import OutputLayer

    B, S, H, V = 4, 320, 1024, 20000
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *n: torch.randn(*n, device="cuda", generator=g)  # noqa: E731
    h, w_n = rand(B * S, H).bfloat16(), (1 + 0.2 * rand(H)).bfloat16()
    w = (rand(V, H) * 2 / H ** 0.5).bfloat16()
    t = torch.randint(0, V, (B, S), device="cuda", generator=g)
    t[:, :90] = -100
    t[1, 200:] = -100
    t = t.reshape(-1)
    head = OutputLayer(_Weight(w_n), _Weight(w), 1e-5, 256)
    x, _ = ops.rmsnorm_fwd(h, w_n, 1e-5)
    lp, _, _, _ = oracle.logprob(x, w, t, V, temperature=tau)
    ref = (lp + 0.1 * rand(B * S)).float()
    old = (lp + torch.where(rand(B * S) > 0, 0.05, -0.5)).float()
    adv = torch.tensor([1.0, -0.5, 0.7, -1.2], device="cuda")
    shape = (B, S)
    if kind == "preference":
        step = ObjectiveStep.build(PreferenceObjective(beta=0.2, temperature=tau), B, S, cuda_device, ref_logps=ref.view(shape))
        loss64, dlogp, _ = oracle.preference(lp, ref, t, S, 0.2, "sigmoid", 0.0, False)
    else:
        step = ObjectiveStep.build(PolicyObjective(kl_coef=0.1, temperature=tau), B, S, cuda_device, ref_logps=ref.view(shape),
                                   old_logps=old.view(shape), advantages=adv)
        loss64, dlogp, _ = oracle.policy(lp, old, ref, adv, t, S, 0.2, 0.2, 0.1, "token")
    loss, dh = head.loss_and_grad(h, SimpleNamespace(objective=step, targets=t, seq_len=S))
    _, _, dx64, dw64 = oracle.logprob(x, w, t, V, temperature=tau, dlogp=dlogp)
    hd, nd = h.double().requires_grad_(), w_n.double().requires_grad_()
    (hd * torch.rsqrt(hd.square().mean(1, keepdim=True) + 1e-5) * nd).backward(dx64)
    assert abs(float(loss) - float(loss64)) <= 1e-4 * max(1.0, abs(float(loss64)))
    assert _rel(head.lm_head.weight.grad, dw64) < 4 * 2.0 ** -9
    assert _rel(dh, hd.grad) < 6 * 2.0 ** -9
    assert _rel(head.norm.weight.grad, nd.grad) < 6 * 2.0 ** -9
