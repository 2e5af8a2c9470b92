"""Rows of logits at inputs that the other tests leave out: the least temperature
with a largest logit of 0, masks that leave neighbouring tokens alone."""
import math

import pytest
import torch

import _lists_oracle as oracle
from test_row_select_gpu import _check_logp

pytestmark = pytest.mark.gpu
LEAST = 2.0 ** -126


@pytest.mark.parametrize("V", [5, 1000, 8193, 128256])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_least_temperature_with_a_largest_logit_of_zero(V, dtype, cuda_device):
    """A largest logit of 0 is no sharper than its neighbours by its own size,
    whatever the temperature."""
    from test1_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(V)
    z = -torch.rand(4, V, device="cuda", generator=g) - 0.1
    z[1:, V // 3] = 0.0
    z[2, ::4] = 0.0
    z[3, V // 2] = -2.0 ** -120  # as far from 0 as 64 temperatures
    z = z.to(dtype)
    u = torch.rand(4, device="cuda", generator=g)
    logp, ids = ops.topk_logprobs(z, 2, LEAST)
    want, at = oracle.topk(z, 2, LEAST)
    assert torch.equal(ids.cpu(), at)
    _check_logp(logp, torch.where(want < -3.4e38, -math.inf, want))
    for top_k, top_p, min_p in [(0, 1.0, 0.0), (3, 1.0, 0.0), (0, 0.5, 0.0), (0, 1.0, 0.3), (3, 0.7, 0.1)]:
        token, logp = ops.sample_tokens(z, u, LEAST, top_k, top_p, min_p)
        at, want = oracle.sample(z, u, LEAST, top_k, top_p, min_p)
        assert torch.equal(token.cpu(), at)
        _check_logp(logp, want)


@pytest.mark.parametrize("B,V", [(2, 20011), (1, 128256)])
@pytest.mark.parametrize("allowed", [26, 100, 1000, 9000])
@pytest.mark.parametrize("lowest", [-math.inf, "min", -1e9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_neighbouring_tokens_alone(B, V, allowed, lowest, dtype, cuda_device):
    """Masks that leave some neighbours, as a grammar does: whole stretches are
    empty, or equal to the type's lowest value."""
    from test1_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(V + allowed)
    z = 2 * torch.randn(B, V, device="cuda", generator=g)
    z[:, :5000] = z[:, 5000 + allowed:] = torch.finfo(dtype).min if lowest == "min" else lowest
    z = z.to(dtype)
    u = torch.rand(B, device="cuda", generator=g)
    logp, ids = ops.topk_logprobs(z, 64, 0.8)
    want, at = oracle.topk(z, 64, 0.8)
    assert torch.equal(ids.cpu(), at)
    _check_logp(logp, torch.where(want < -3.4e38, -math.inf, want))
    for top_k, top_p, min_p in [(50, 0.95, 0.0), (1000, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05)]:
        token, logp = ops.sample_tokens(z, u, 0.8, top_k, top_p, min_p)
        at, want = oracle.sample(z, u, 0.8, top_k, top_p, min_p)
        assert torch.equal(token.cpu(), at)
        _check_logp(logp, want)


def test_temperatures_below_are_refused(cuda_device):
    from test1_b200 import _native, ops

    z, u = torch.zeros(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    x, ids = torch.zeros(2, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    C = _native.cuda()
    for tau in (1e-38, 1e-40, 1e-310):
        for call in (lambda: ops.topk_logprobs(z, 2, tau), lambda: ops.sample_tokens(z, u, tau),
                     lambda: ops.linear_topk_logprob_fwd(x, x, ids, tau), lambda: C.topk_logprobs(z, 2, tau),
                     lambda: C.sample_tokens(z, u, tau, 0, 1.0, 0.0), lambda: C.linear_topk_logprob_fwd(x, x, ids, tau)):
            with pytest.raises((ValueError, RuntimeError), match="2\\^-126"):
                call()
