"""Preference and policy losses on the GPU against their definitions in 64
bits.  Per-token values are a handful of fp32 operations (a few 2^-24,
relative to the terms), sums over tokens are carried in fp64: 1e-5 of the
result's size (of the terms' size, for the loss) leaves an order of magnitude."""
import math

import pytest
import torch

import _answer_oracle as oracle

pytestmark = pytest.mark.gpu

TOL = 1e-5
NAN, INF = float("nan"), float("inf")


def _batch(B, S, seed=0, empty=(), fill=NAN):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * B + S)
    rand = lambda *n: torch.randn(*n, device="cuda", generator=g)  # noqa: E731
    T = B * S
    targets = torch.randint(0, 1000, (B, S), device="cuda", generator=g)
    keep = torch.rand(B, S, device="cuda", generator=g) < 0.7
    for b in empty:
        keep[b] = False
    targets = torch.where(keep, targets, -100).reshape(T)
    base = -torch.rand(T, device="cuda", generator=g) * 5
    near = lambda by: torch.where(targets >= 0, base + by * rand(T), fill)  # noqa: E731
    return targets, near(0.2), near(0.1), near(0.2), rand(B) + 0.3, rand(T) + 0.3


def _close(got, want, size=None):
    want = want.double()
    size = float(want.abs().max()) if size is None else size
    assert got.dtype == torch.float32 and got.shape == want.shape
    assert float((got.double() - want).abs().max() if want.numel() else 0) <= TOL * size + 1e-12


SIZES = [(2, 1), (2, 7), (4, 33), (6, 255), (4, 4097), (2, 20001), (300, 5), (2048, 3)]


@pytest.mark.parametrize("B,S", SIZES)
@pytest.mark.parametrize("kind,smoothing,average,with_ref",
                         [("sigmoid", 0.0, False, True), ("sigmoid", 0.2, True, False), ("hinge", 0.0, True, True),
                          ("ipo", 0.0, True, True), ("hinge", 0.1, False, True)])
def test_preference(B, S, kind, smoothing, average, with_ref, cuda_device):
    from test1_b200 import ops

    # the second pair is padding, of the third one only the chosen answer
    empty = [1, 1 + B // 2, 2] if B >= 6 else []
    targets, logp, ref, _, _, _ = _batch(B, S, empty=empty)
    ref = ref if with_ref else None
    out = ops.preference_loss_fwd_bwd(logp, ref, targets, S, beta=0.3, kind=kind, label_smoothing=smoothing, average=average)
    loss, dlogp, rewards = oracle.preference(logp, ref, targets, S, 0.3, kind, smoothing, average)
    _close(out[0], loss)
    _close(out[1], dlogp)
    _close(out[2], rewards, float(rewards.abs().max()) + (0.3 * (1 if average else math.sqrt(S))))


@pytest.mark.parametrize("B,S", [(1, 1), (3, 1)] + SIZES)
@pytest.mark.parametrize("per_token,with_ref,reduction", [(False, True, "token"), (True, False, "sequence"),
                                                          (True, True, "token"), (False, True, "sequence")])
def test_policy(B, S, per_token, with_ref, reduction, cuda_device):
    from test1_b200 import ops

    empty = [1, 4] if B >= 6 else []
    targets, logp, old, ref, adv_seq, adv_tok = _batch(B, S, seed=3, empty=empty, fill=INF)
    adv, ref, kl = (adv_tok if per_token else adv_seq), ref if with_ref else None, 0.1 if with_ref else 0.0
    out = ops.policy_loss_fwd_bwd(logp, old, ref, adv, targets, S, clip_low=0.15, clip_high=0.25, kl_coef=kl,
                                  reduction=reduction)
    loss, dlogp, stats = oracle.policy(logp, old, ref, adv, targets, S, 0.15, 0.25, kl, reduction)
    _close(out[0], loss, 4.0)
    _close(out[1], dlogp)
    _close(out[2], stats, 1.0)


def test_nothing_to_learn_from(cuda_device):
    """No answer token at all, no sequence at all: zeros, no NaN."""
    from test1_b200 import ops

    targets, logp, old, ref, adv, _ = _batch(4, 50, empty=range(4))
    for out in (ops.preference_loss_fwd_bwd(logp, ref, targets, 50),
                ops.policy_loss_fwd_bwd(logp, old, ref, adv, targets, 50, kl_coef=0.1),
                ops.policy_loss_fwd_bwd(logp, old, ref, adv, targets, 50, kl_coef=0.1, reduction="sequence"),
                ops.preference_loss_fwd_bwd(logp[:0], None, targets[:0], 50),
                ops.policy_loss_fwd_bwd(logp[:0], old[:0], None, adv[:0], targets[:0], 50)):
        assert all(bool((v == 0).all()) for v in out)


def test_extreme_log_ratios(cuda_device):
    """Large margins saturate without NaN; a huge ratio is cut where the
    advantage is positive."""
    from test1_b200 import ops

    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    lp = torch.tensor([-1.0, -2000.0, -1500.0, -1.0], device="cuda")
    loss, d, _ = ops.preference_loss_fwd_bwd(lp, None, t, 1, beta=1.0)
    want = oracle.preference(lp, None, t, 1, 1.0, "sigmoid", 0.0, False)
    _close(loss, want[0])
    _close(d, want[1])
    old = torch.tensor([-200.0, -1.0, -1.0, -50.0], device="cuda")
    adv = torch.tensor([1.0, -1.0, 2.0, 0.5], device="cuda")
    loss, d, stats = ops.policy_loss_fwd_bwd(lp, old, None, adv, t, 1)
    want = oracle.policy(lp, old, None, adv, t, 1, 0.2, 0.2, 0.0, "token")
    _close(loss, want[0])
    _close(d, want[1])
    _close(stats, want[2])


def test_gradient_against_differences(cuda_device):
    """Central differences along random directions; away from the edges of
    the clip the losses are smooth: h^2 of the next term."""
    from test1_b200 import ops

    targets, logp, old, ref, adv, _ = _batch(6, 40, seed=9, fill=0.0)
    old = logp - 0.05 * torch.sign(old)  # inside the trust region, not on its edge
    g = torch.Generator(device="cuda").manual_seed(2)
    losses = [lambda p: ops.preference_loss_fwd_bwd(p, ref, targets, 40, beta=0.5, kind=k)[:2] for k in ("sigmoid", "ipo")]
    losses += [lambda p: ops.policy_loss_fwd_bwd(p, old, ref, adv, targets, 40, kl_coef=0.3, reduction=r)[:2]
               for r in ("token", "sequence")]
    h = 2.0 ** -6
    for f in losses:
        e = torch.randn(logp.shape, device="cuda", generator=g)
        e /= e.abs().max()
        num = (float(f(logp + h * e)[0]) - float(f(logp - h * e)[0])) / (2 * h)
        d = float((f(logp)[1].double() * e).sum())
        assert abs(d - num) < 1e-2 * abs(num) + 1e-3


def test_strides_streams_and_repeat(cuda_device):
    from test1_b200 import ops

    targets, logp, old, ref, adv, _ = _batch(10, 777, seed=4)
    spread = lambda v: torch.stack([v, v.flip(0)], 1)[:, 0]  # noqa: E731
    a = ops.policy_loss_fwd_bwd(logp, old, ref, adv, targets, 777, kl_coef=0.1)
    b = ops.policy_loss_fwd_bwd(spread(logp), spread(old), spread(ref), spread(adv), spread(targets), 777, kl_coef=0.1)
    p = ops.preference_loss_fwd_bwd(logp, ref, targets, 777)
    q = ops.preference_loss_fwd_bwd(spread(logp), spread(ref), spread(targets), 777)
    assert all(torch.equal(u, v) for u, v in zip(a + p, b + q))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c = ops.policy_loss_fwd_bwd(logp + 0, old + 0, ref + 0, adv + 0, targets + 0, 777, kl_coef=0.1)
    s.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(a, c))


def test_refusals(cuda_device):
    from test1_b200 import ops

    targets, logp, old, ref, adv, _ = _batch(4, 8)
    pref = lambda **k: ops.preference_loss_fwd_bwd(**{**dict(logp=logp, ref_logp=ref, targets=targets, seq_len=8), **k})  # noqa: E731
    pol = lambda **k: ops.policy_loss_fwd_bwd(**{**dict(logp=logp, old_logp=old, ref_logp=ref, advantages=adv,  # noqa: E731
                                                        targets=targets, seq_len=8), **k})
    for f, bad in ((pref, dict(ref_logp=ref[:-1])), (pref, dict(ref_logp=ref.cpu())), (pref, dict(logp=logp.double())),
                   (pref, dict(targets=targets.int())), (pol, dict(old_logp=old.half())), (pol, dict(old_logp=old[:8])),
                   (pol, dict(advantages=adv.double())), (pol, dict(ref_logp=ref.cpu()))):
        with pytest.raises(RuntimeError):
            f(**bad)
    for f, bad in ((pref, dict(seq_len=7)), (pref, dict(seq_len=0)), (pref, dict(seq_len=32)), (pref, dict(beta=0.0)),
                   (pref, dict(kind="other")), (pref, dict(label_smoothing=0.5)),
                   (pol, dict(clip_low=1.0)), (pol, dict(clip_high=-0.1)), (pol, dict(reduction="mean")),
                   (pol, dict(kl_coef=-1.0)), (pol, dict(kl_coef=0.1, ref_logp=None)), (pol, dict(advantages=adv[:3]))):
        with pytest.raises(ValueError):
            f(**bad)


@pytest.mark.parametrize("B,S", [(4, 64), (40, 1024)])
@pytest.mark.parametrize("offset", [0, 1, 2])
def test_alignment(B, S, offset, cuda_device):
    """Sequences that 16-byte vectors divide, in tensors that start on such a
    boundary and in ones that do not."""
    from test1_b200 import ops

    targets, logp, old, ref, adv, adv_tok = _batch(B, S, seed=6)
    shift = lambda v: torch.cat([v[:offset], v])[offset:]  # noqa: E731
    t, lp, od, rf = shift(targets), shift(logp), shift(old), shift(ref)
    assert offset == 0 or lp.data_ptr() % 16
    got = ops.preference_loss_fwd_bwd(lp, rf, t, S)
    for a, b in zip(got, oracle.preference(logp, ref, targets, S, 0.1, "sigmoid", 0.0, False)):
        _close(a, b, float(b.abs().max()) + (0.1 * math.sqrt(S) if b.shape == (B,) else 0))
    for a_in, per in ((adv, adv), (shift(adv_tok), adv_tok)):
        got = ops.policy_loss_fwd_bwd(lp, od, rf, a_in, t, S, kl_coef=0.1)
        want = oracle.policy(logp, old, ref, per, targets, S, 0.2, 0.2, 0.1, "token")
        for a, b, size in zip(got, want, (4.0, None, 1.0)):
            _close(a, b, size)


def test_captured_in_a_graph(cuda_device):
    """A graph of the operators, replayed on new values in its inputs; the
    eager calls between leave it alone."""
    from test1_b200 import ops

    targets, logp, old, ref, adv, _ = _batch(40, 1024, seed=7, fill=0.0)
    small = [v[:2048].clone() for v in (targets, logp, old, ref)]
    f = lambda: ops.policy_loss_fwd_bwd(logp, old, ref, adv, targets, 1024, kl_coef=0.1) + \
        ops.preference_loss_fwd_bwd(logp, ref, targets, 1024) + \
        ops.preference_loss_fwd_bwd(small[1], small[3], small[0], 64)  # noqa: E731
    f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    for k in range(2):
        logp.add_(0.01 * k)
        want = f()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
