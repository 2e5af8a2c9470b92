"""What follows a launch whose bounded wait expired: its arrival counters are
left half way (here they are set to that, nothing waits), and the next calls
on the stream are right all the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _calls():
    """Calls that count arrivals: few tokens, joined column blocks, the losses'
    grid barriers; of different numbers of counters."""
    from test1_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *n: torch.randn(*n, device="cuda", generator=g)  # noqa: E731
    x, w = rand(2000, 64).bfloat16(), rand(3000, 64).bfloat16()
    t = torch.randint(0, 3000, (2000,), device="cuda", generator=g)
    B, S = 64, 1024
    T = B * S
    lp, old, ref, adv = rand(T), rand(T), rand(T), rand(B)
    ids = torch.randint(0, 10, (T,), device="cuda", generator=g)
    return [lambda: ops.linear_logprob_fwd(x[:5], w, t[:5]), lambda: ops.linear_logprob_fwd(x, w, t),
            lambda: ops.preference_loss_fwd_bwd(lp, ref, ids, S),
            lambda: ops.policy_loss_fwd_bwd(lp, old, ref, adv, ids, S, kl_coef=0.1, reduction="sequence")]


@pytest.mark.parametrize("left", [1, 7, 100000, -3])
@pytest.mark.parametrize("own_stream", [False, True])
def test_calls_after_an_expired_wait(left, own_stream, cuda_device):
    from test1_b200 import _native, ops

    calls = _calls()
    want = [f() for f in calls]
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream() if own_stream else torch.cuda.current_stream()):
        for first in calls:
            for f, ref in list(zip(calls, want)) + list(zip(calls, want))[::-1]:
                first()
                _native.cuda().fill_last_arrivals(left)
                for _ in range(3):
                    assert all(torch.equal(a, b) for a, b in zip(f(), ref))
    torch.cuda.synchronize()
    assert ops.native.gemm_error() == 0
