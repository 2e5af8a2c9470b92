"""Preference and policy training on the CPU: the plain operators against
their 64-bit definitions, one engine step against HF + autograd + AdamW, the
generic model path, the refusals and the example.  fp32 arithmetic: 1e-5 of
the results' size."""
import os
import sys

import pytest
import torch

import _answer_oracle as oracle
from test1_b200 import PolicyObjective, PreferenceObjective, SlideFSDPConfig, ops
from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM
from test1_b200.slide_fsdp import SlideFSDP

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _tokens(B, S, V, seed=0, empty=()):
    g = torch.Generator().manual_seed(seed)
    t = torch.randint(0, V, (B, S), generator=g)
    t[torch.rand(B, S, generator=g) < 0.3] = -100
    for b in empty:
        t[b] = -100
    return t.reshape(-1), g


def _near(a, b, tol=1e-5):
    b = b.to(a.dtype)
    assert float((a - b).abs().max()) <= tol * float(b.abs().max().clamp_min(1e-3))


@pytest.mark.parametrize("T,H,V,tau", [(1, 8, 5, 1.0), (40, 16, 101, 0.7), (30, 24, 1, 1.0)])
def test_logprob_and_gradient(T, H, V, tau):
    t, g = _tokens(1, T, V)
    x, w, up = torch.randn(T, H, generator=g), torch.randn(V, H, generator=g), torch.randn(T, generator=g)
    t[-1] = V  # not a vocabulary index
    up[t < 0] = float("nan")
    logp, lse = ops.linear_logprob_fwd(x, w, t, temperature=tau)
    lp, ls, dx64, dw64 = oracle.logprob(x, w, t, V, temperature=tau, dlogp=up)
    _near(logp, lp)
    _near(lse, ls)
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))
    ops.linear_logprob_bwd(up, x, w, t, lse, dx, dw, temperature=tau)
    _near(dx, dx64, 1e-4 if V == 1 else 1e-5)
    _near(dw, dw64, 1e-4 if V == 1 else 1e-5)


@pytest.mark.parametrize("kind,smoothing,average,with_ref", [("sigmoid", 0.1, False, True), ("hinge", 0.0, True, False),
                                                             ("ipo", 0.2, True, True)])
def test_preference_loss(kind, smoothing, average, with_ref):
    B, S = 6, 17
    t, g = _tokens(B, S, 50, empty=(1, 4, 2))
    lp, ref = -torch.rand(B * S, generator=g), -torch.rand(B * S, generator=g) if with_ref else None
    lp[t < 0] = float("nan")
    got = ops.preference_loss_fwd_bwd(lp, ref, t, S, 0.4, kind, smoothing, average)
    for a, b in zip(got, oracle.preference(lp, ref, t, S, 0.4, kind, smoothing, average)):
        _near(a, b)


@pytest.mark.parametrize("per_token,with_ref,reduction", [(False, True, "token"), (True, False, "sequence")])
def test_policy_loss(per_token, with_ref, reduction):
    B, S = 5, 19
    t, g = _tokens(B, S, 50, seed=1, empty=(3,))
    lp, old = -torch.rand(B * S, generator=g), -torch.rand(B * S, generator=g)
    ref = -torch.rand(B * S, generator=g) if with_ref else None
    adv = torch.randn(B * S if per_token else B, generator=g)
    old[t < 0] = float("inf")
    got = ops.policy_loss_fwd_bwd(lp, old, ref, adv, t, S, 0.1, 0.3, 0.2 if with_ref else 0.0, reduction)
    for a, b in zip(got, oracle.policy(lp, old, ref, adv, t, S, 0.1, 0.3, 0.2 if with_ref else 0.0, reduction)):
        _near(a, b)


def test_refusals():
    lp, t = torch.zeros(8), torch.zeros(8, dtype=torch.int64)
    for bad in (dict(seq_len=3), dict(seq_len=8), dict(beta=0.0), dict(kind="x"), dict(label_smoothing=0.7),
                dict(targets=t[:4])):
        with pytest.raises(ValueError):
            ops.preference_loss_fwd_bwd(**{**dict(logp=lp, ref_logp=None, targets=t, seq_len=4), **bad})
    for bad in (dict(clip_low=1.5), dict(kl_coef=0.1), dict(reduction="sum"), dict(advantages=lp[:3]), dict(seq_len=0)):
        with pytest.raises(ValueError):
            ops.policy_loss_fwd_bwd(**{**dict(logp=lp, old_logp=lp, ref_logp=None, advantages=lp, targets=t, seq_len=4), **bad})
    with pytest.raises(ValueError):
        ops.linear_logprob_fwd(torch.zeros(2, 4), torch.zeros(3, 4), t[:2], temperature=0.0)


def _label_logps(model, ids, labels):
    lp = torch.log_softmax(model(input_ids=ids).logits.float(), -1)
    tg = ops.shift_labels(labels).view_as(labels)
    picked = lp.gather(2, tg.clamp_min(0)[..., None])[..., 0]
    return torch.where(tg >= 0, picked, torch.zeros_like(picked)), tg


def _hf_loss(kind, lp, tg, ref, old, adv):
    valid = tg >= 0
    if kind == "preference":
        r = ((lp - ref) * valid).sum(1)
        m = r[: len(r) // 2] - r[len(r) // 2:]
        return -torch.nn.functional.logsigmoid(0.3 * m).mean()
    rho = torch.exp(lp - old)
    l = -torch.minimum(adv[:, None] * rho, adv[:, None] * rho.clamp(0.8, 1.2)) + 0.1 * (torch.expm1(ref - lp) - (ref - lp))
    return (l * valid).sum() / valid.sum()


@pytest.mark.parametrize("kind", ["preference", "policy"])
@pytest.mark.parametrize("model_type", ["llama", "qwen2"])
def test_engine_step_matches_autograd(kind, model_type):
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(0)
    if model_type == "llama":
        cfg = LlamaConfig.tiny()
        ours = LlamaForCausalLM(cfg)
        hf = transformers.LlamaForCausalLM(cfg.to_hf()).float()
        hf.load_state_dict({n: p.detach().clone() for n, p in ours.named_parameters()})
    else:
        hf_cfg = transformers.Qwen2Config(vocab_size=300, hidden_size=64, intermediate_size=96, num_hidden_layers=2,
                                          num_attention_heads=4, num_key_value_heads=2, tie_word_embeddings=False,
                                          max_position_embeddings=128)
        hf, ours = transformers.Qwen2ForCausalLM(hf_cfg).float(), transformers.Qwen2ForCausalLM(hf_cfg).float()
        ours.load_state_dict(hf.state_dict())
    V = hf.config.vocab_size
    opt = torch.optim.AdamW(hf.parameters(), lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    eng = SlideFSDP(ours, SlideFSDPConfig(dtype=torch.float32, device="cpu", lr=1e-3, weight_decay=0.01))
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, V, (4, 24), generator=g)
    labels = ids.clone()
    labels[:, :7] = -100
    adv = torch.tensor([1.0, -0.5, 0.7, -1.2])
    try:
        ref = eng.token_logprobs(ids, labels)
        with torch.no_grad():
            want, tg = _label_logps(hf, ids, labels)
        assert torch.allclose(ref, want, atol=2e-5)
        old = ref + 0.05 * torch.randn(ref.shape, generator=g)
        for _ in range(2):
            if kind == "preference":
                out = eng(input_ids=ids, labels=labels, objective=PreferenceObjective(beta=0.3), ref_logps=ref)
                assert eng.last_objective["rewards"].shape == (4,)
            else:
                out = eng(input_ids=ids, labels=labels, objective=PolicyObjective(kl_coef=0.1), ref_logps=ref,
                          old_logps=old, advantages=adv)
                assert eng.last_objective["stats"].shape == (2,)
            lp, tg = _label_logps(hf, ids, labels)
            assert torch.allclose(eng.last_objective["logps"], lp.detach(), atol=1e-4)
            loss = _hf_loss(kind, lp, tg, ref, old, adv)
            opt.zero_grad()
            loss.backward()
            opt.step()
            assert abs(float(out.loss) - float(loss.detach())) < 1e-4 * max(1.0, abs(float(loss.detach())))
        eng.wait_for_updates()
        master = dict(eng.named_master_tensors())
        for n, p in hf.named_parameters():
            d = (master[n].view(p.shape) - p.detach()).abs()
            # as in the cross-entropy test: Adam moves an element of ~0
            # gradient by up to lr on rounding noise alone
            assert (d > 1e-4).float().mean().item() < 2e-3, n
    finally:
        eng.close()


def test_engine_refuses_incomplete_objectives():
    cfg = LlamaConfig.tiny()
    eng = SlideFSDP(LlamaForCausalLM(cfg, device="meta"), SlideFSDPConfig(dtype=torch.float32, device="cpu"))
    ids = torch.zeros(2, 8, dtype=torch.int64)
    try:
        for kw in (dict(labels=ids, ref_logps=torch.zeros(2, 8)), dict(objective=PreferenceObjective()),
                   dict(labels=ids, objective=PreferenceObjective(), ref_logps=torch.zeros(2, 7)),
                   dict(labels=ids, objective=PolicyObjective(), advantages=torch.zeros(2)),
                   dict(labels=ids, objective=PolicyObjective(kl_coef=0.1), advantages=torch.zeros(2), old_logps=torch.zeros(2, 8)),
                   dict(labels=ids, objective=PolicyObjective(), advantages=torch.zeros(3), old_logps=torch.zeros(2, 8))):
            with pytest.raises(ValueError):
                eng(input_ids=ids, **kw)
        with pytest.raises(ValueError):
            eng(input_ids=ids[:1], labels=ids[:1], objective=PreferenceObjective())
        for bad in (dict(beta=-1.0), dict(kind="dpo"), dict(temperature=0.0)):
            with pytest.raises(ValueError):
                PreferenceObjective(**bad)
        with pytest.raises(ValueError):
            PolicyObjective(clip_low=1.0)
    finally:
        eng.close()


def test_example_learns():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import preference_tuning

    margins, _ = preference_tuning.run("cpu", steps=4, verbose=False)
    assert margins[0] == pytest.approx(0.0, abs=1e-4) and margins[-1] > 0.5
