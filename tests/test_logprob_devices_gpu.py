"""The log-probability operators on two devices of one process."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs 2 GPUs")
@pytest.mark.parametrize("T", [5, 300])
def test_one_device_after_another(T):
    from test1_b200 import ops

    g = torch.Generator().manual_seed(T)
    x, w = torch.randn(T, 256, generator=g).bfloat16(), (torch.randn(1003, 256, generator=g) / 8).bfloat16()
    t, up = torch.randint(0, 1003, (T,), generator=g), torch.randn(T, generator=g)
    out = []
    for dev in ("cuda:0", "cuda:1"):  # the current device stays cuda:0
        a, b, c, d = x.to(dev), w.to(dev), t.to(dev), up.to(dev)
        logp, lse = ops.linear_logprob_fwd(a, b, c)
        dx, dw = torch.empty_like(a), torch.empty_like(b)
        ops.linear_logprob_bwd(d, a, b, c, lse, dx, dw)
        out.append([v.cpu() for v in (logp, lse, dx, dw)])
    assert all(torch.equal(a, b) for a, b in zip(*out))
