"""Answer generation and distillation on the CPU: the plain operators against
their 64-bit definitions, gradients against differences, engine steps against HF
+ autograd + AdamW, generation against the model's own logits, the refusals.
fp32 arithmetic: 1e-5 of the results' size."""
import math

import pytest
import torch

import _lists_oracle as oracle
from test1_b200 import DistillationObjective, PolicyObjective, PreferenceObjective, SlideFSDPConfig, ops
from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM
from test1_b200.slide_fsdp import SlideFSDP

INF = math.inf


def _near(a, b, tol=1e-5):
    b = b.to(a.dtype)
    assert float((a - b).abs().max()) <= tol * float(b.abs().max().clamp_min(1e-3))


def _logits(B, V, kind, seed=0):
    g = torch.Generator().manual_seed(seed + 10 * B + V)
    z = 2 * torch.randn(B, V, generator=g)
    if kind == "ties":
        z = z.round()
    elif kind == "masked":
        z.masked_fill_(torch.rand(B, V, generator=g) > 0.2, -INF)
        z[0] = -INF
        z[1, ::2] = float("nan")
        z[1, 0] = INF
    return z, g


@pytest.mark.parametrize("B,V", [(2, 1), (3, 2), (4, 37), (5, 500)])
@pytest.mark.parametrize("kind", ["plain", "ties", "masked"])
def test_topk(B, V, kind):
    z, _ = _logits(B, V, kind)
    for k in {1, min(5, V), min(V, 100)}:
        logp, ids = ops.topk_logprobs(z, k, temperature=0.7)
        want, at = oracle.topk(z, k, 0.7)
        assert torch.equal(ids, at)
        finite = torch.isfinite(want)
        assert torch.equal(logp.double()[~finite], want[~finite])
        assert torch.allclose(logp.double()[finite], want[finite], atol=1e-5)


@pytest.mark.parametrize("B,V", [(2, 1), (3, 2), (40, 37), (30, 500)])
@pytest.mark.parametrize("kind", ["plain", "ties", "masked"])
@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 1.0, 0.0), (7, 1.0, 0.0), (0, 0.8, 0.0), (0, 1.0, 0.1), (20, 0.9, 0.02),
                                               (1000, 0.3, 1.0)])
def test_sample(B, V, kind, top_k, top_p, min_p):
    z, g = _logits(B, V, kind, seed=1)
    u = torch.rand(B, generator=g)
    token, logp = ops.sample_tokens(z, u, temperature=1.2, top_k=top_k, top_p=top_p, min_p=min_p)
    at, want = oracle.sample(z, u, 1.2, top_k, top_p, min_p)
    assert torch.equal(token, at)
    assert torch.allclose(logp.double(), want, atol=1e-5)


@pytest.mark.parametrize("T,H,V,K,tau", [(1, 8, 5, 5, 1.0), (40, 16, 101, 7, 0.7), (30, 24, 1, 1, 1.0)])
def test_listed_logprobs_and_gradient(T, H, V, K, tau):
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(T, H, generator=g), torch.randn(V, H, generator=g)
    ids, up = torch.randint(0, V, (T, K), generator=g), torch.randn(T, K, generator=g)
    if T > 1:
        ids[torch.rand(T, K, generator=g) < 0.3] = -100
        ids[3], ids[4, 0] = -1, V
        up[3] = float("nan")
    logp, lse = ops.linear_topk_logprob_fwd(x, w, ids, temperature=tau)
    lp, ls, dx64, dw64 = oracle.listed_logprob(x, w, ids, tau, dlogp=up)
    _near(logp, lp)
    _near(lse, ls)
    dx, dw = torch.full_like(x, float("nan")), torch.full_like(w, float("nan"))
    ops.linear_topk_logprob_bwd(up, x, w, ids, lse, dx, dw, temperature=tau)
    _near(dx, dx64, 1e-4 if V == 1 else 1e-5)
    _near(dw, dw64, 1e-4 if V == 1 else 1e-5)
    assert torch.allclose(ops.linear_logits(x, w), x @ w.t(), atol=1e-5)


def _lists(T, K, seed=3):
    g = torch.Generator().manual_seed(seed)
    share = 1 - 0.6 * torch.rand(T, 1, generator=g) - 1e-3
    b = torch.log_softmax(torch.randn(T, K, generator=g), 1) + share.log()
    a = torch.log_softmax(torch.cat([b, torch.log1p(-share)], 1) + 0.5 * torch.randn(T, K + 1, generator=g), 1)[:, :K]
    ids = torch.arange(K).repeat(T, 1)
    if T > 2:
        ids[torch.rand(T, K, generator=g) < 0.2] = -1
        ids[1], b[2] = -1, -INF
    return a, b, ids


@pytest.mark.parametrize("kind", ops.DISTILLATION_KINDS)
@pytest.mark.parametrize("tail", [True, False])
def test_distillation_loss(kind, tail):
    a, b, ids = _lists(20, 9)
    loss, dlogp, each = ops.distillation_loss_fwd_bwd(a, b, ids, kind=kind, tail=tail)
    want, grad, per, _ = oracle.distillation(a, b, ids, kind, tail)
    _near(loss, want)
    _near(dlogp, grad)
    _near(each, per)


@pytest.mark.parametrize("kind", ops.DISTILLATION_KINDS)
@pytest.mark.parametrize("tail", [True, False])
def test_distillation_gradient_against_differences(kind, tail):
    """Central differences of the definition in 64 bits, step 1e-5: their own
    error is below 1e-9."""
    a, b, ids = _lists(5, 4, seed=4)
    _, dlogp, _ = ops.distillation_loss_fwd_bwd(a, b, ids, kind=kind, tail=tail)
    for t in range(5):
        for k in range(4):
            up, down = a.double().clone(), a.double().clone()
            up[t, k] += 1e-5
            down[t, k] -= 1e-5
            d = (oracle.distillation(up, b, ids, kind, tail)[0] - oracle.distillation(down, b, ids, kind, tail)[0]) / 2e-5
            assert abs(float(dlogp[t, k]) - float(d)) <= 1e-6


def test_refusals():
    z, u = torch.zeros(2, 8), torch.zeros(2)
    for kw in (dict(temperature=0.0), dict(top_p=0.0), dict(top_p=1.1), dict(min_p=-0.1), dict(min_p=2.0), dict(top_k=-1),
               dict(top_k=1.5), dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            ops.sample_tokens(z, u, **kw)
    for bad in ((z, u[:1]), (z, u.double()), (z.half(), u), (z[0], u)):
        with pytest.raises(ValueError):
            ops.sample_tokens(*bad)
    for k in (0, 9):
        with pytest.raises(ValueError):
            ops.topk_logprobs(z, k)
    with pytest.raises(ValueError):
        ops.topk_logprobs(torch.zeros(2, 600), 513)
    for tau in (-1.0, 1e30):  # 400 tau added to a logit has to stay finite
        with pytest.raises(ValueError):
            ops.topk_logprobs(z, 2, temperature=tau)
        with pytest.raises(ValueError):
            ops.sample_tokens(z, u, tau)
    ids = torch.zeros(2, 3, dtype=torch.int64)
    for bad in ((z, z[0], ids), (z, z, ids[:1]), (z, z, ids[:, :0]), (z, z, torch.zeros(2, 513, dtype=torch.int64))):
        with pytest.raises(ValueError):
            ops.linear_topk_logprob_fwd(*bad)
    with pytest.raises(ValueError):
        ops.linear_topk_logprob_bwd(z, z, z, ids, u, z, z)
    for bad in ((z, z, ids), (z, z[:, :3], ids), (z[:, :0], z[:, :0], ids[:, :0])):
        with pytest.raises(ValueError):
            ops.distillation_loss_fwd_bwd(*bad)
    with pytest.raises(ValueError):
        ops.distillation_loss_fwd_bwd(z[:, :3], z[:, :3], ids, kind="both")


# ------------------------------------------------------------------ engine
def _engine(model_type, lr=1e-3):
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
    return hf, SlideFSDP(ours, SlideFSDPConfig(dtype=torch.float32, device="cpu", lr=lr, weight_decay=0.01))


def _batch(V, seed=5):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (3, 20), generator=g)
    labels = ids.clone()
    labels[:, :6] = -100
    labels[1, 15:] = -100
    return ids, labels, g


@pytest.mark.parametrize("kind,tail", [("forward", True), ("reverse", True), ("jensen", False)])
@pytest.mark.parametrize("model_type", ["llama", "qwen2"])
def test_distillation_step_matches_autograd(kind, tail, model_type):
    hf, eng = _engine(model_type)
    V, K, tau = hf.config.vocab_size, 12, 1.3
    opt = torch.optim.AdamW(hf.parameters(), lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
    ids, labels, g = _batch(V)
    # a teacher's lists, some shorter, some elsewhere than the student's own
    z = 3 * torch.randn(3, 20, V, generator=g)
    logps, top = torch.log_softmax(z / tau, -1).topk(K, -1)
    top[0, 8, 5:] = -1
    keep = (ops.shift_labels(labels).view(3, 20, 1) >= 0) & (top >= 0)
    try:
        for _ in range(2):
            out = eng(input_ids=ids, labels=labels, objective=DistillationObjective(kind=kind, tail=tail, temperature=tau),
                      teacher_logps=logps, teacher_ids=top)
            lp = torch.log_softmax(hf(input_ids=ids).logits.float() / tau, -1).gather(2, top.clamp_min(0))
            got = eng.last_objective
            assert got["divergence"].shape == (3, 20) and got["logps"].shape == (3, 20, K)
            assert torch.allclose(got["logps"], torch.where(keep, lp.detach(), 0.0), atol=1e-4)
            flat = lp.reshape(-1, K)
            loss, grad, each, _ = oracle.distillation(flat.detach(), logps.view(-1, K),
                                                      torch.where(keep, top, -1).view(-1, K), kind, tail)
            assert abs(float(out.loss) - float(loss)) < 1e-4 * max(1.0, float(loss))
            assert torch.allclose(got["divergence"].double().view(-1), each, atol=1e-4)
            opt.zero_grad()
            flat.backward(grad.float())
            opt.step()
        eng.wait_for_updates()
        master = dict(eng.named_master_tensors())
        for n, p in hf.named_parameters():
            d = (master[n].view(p.shape) - p.detach()).abs()
            # Adam moves an element of ~0 gradient by up to lr on rounding alone
            assert (d > 1e-4).float().mean().item() < 2e-3, n
    finally:
        eng.close()


@pytest.mark.parametrize("model_type", ["llama", "qwen2"])
def test_top_logprobs_are_those_of_the_logits(model_type):
    hf, eng = _engine(model_type)
    ids, _, _ = _batch(hf.config.vocab_size)
    try:
        logps, top = eng.top_logprobs(ids, 7, temperature=0.8)
        logits = eng(input_ids=ids).logits.float()
        want, at = ops.topk_logprobs(logits.view(-1, logits.shape[-1]), 7, 0.8)
        assert top.shape == (3, 20, 7) and torch.equal(top.view(-1, 7), at)
        assert torch.allclose(logps.view(-1, 7), want, atol=1e-5)
        # a model distilled from itself has nothing to learn
        out = eng(input_ids=ids, labels=ids, objective=DistillationObjective(temperature=0.8), teacher_logps=logps, teacher_ids=top)
        assert abs(float(out.loss)) < 1e-5
        for bad in (0, 513):
            with pytest.raises(ValueError):
                eng.top_logprobs(ids, bad)
    finally:
        eng.close()


@pytest.mark.parametrize("model_type", ["llama", "qwen2"])
def test_generation(model_type):
    hf, eng = _engine(model_type)
    V = hf.config.vocab_size
    g = torch.Generator().manual_seed(6)
    prompts = torch.randint(0, V, (3, 9), generator=g)
    lengths = torch.tensor([9, 4, 1])
    try:
        # the likeliest token at every step, from the model's own logits
        out = eng.generate(prompts, 5, lengths, top_k=1)
        assert out.input_ids.shape == out.labels.shape == out.logps.shape == (3, 14)
        assert out.lengths.tolist() == [14, 9, 6]
        for b in range(3):
            seq = prompts[b, :lengths[b]]
            for _ in range(5):
                with torch.no_grad():
                    nxt = hf(input_ids=seq[None]).logits[0, -1].argmax()
                seq = torch.cat([seq, nxt[None]])
            n = len(seq)
            assert torch.equal(out.input_ids[b, :n], seq) and not bool(out.input_ids[b, n:].any())
            assert bool((out.labels[b, :lengths[b]] == -100).all()) and bool((out.labels[b, n:] == -100).all())
            assert torch.equal(out.labels[b, lengths[b]:n], seq[lengths[b]:])
        # draws repeat with the same generator; their log-probabilities are those that training sees
        one = eng.generate(prompts, 6, lengths, temperature=0.9, top_p=0.95, generator=torch.Generator().manual_seed(1))
        two = eng.generate(prompts, 6, lengths, temperature=0.9, top_p=0.95, generator=torch.Generator().manual_seed(1))
        assert torch.equal(one.input_ids, two.input_ids) and torch.equal(one.logps, two.logps)
        assert torch.allclose(one.logps, eng.token_logprobs(one.input_ids, one.labels, temperature=0.9), atol=1e-4)
        step = eng(input_ids=one.input_ids, labels=one.labels, objective=PolicyObjective(temperature=0.9), old_logps=one.logps,
                   advantages=torch.tensor([1.0, -1.0, 0.5]))
        assert torch.isfinite(step.loss)
    finally:
        eng.close()


def test_generation_ends():
    hf, eng = _engine("llama")
    prompts = torch.randint(0, hf.config.vocab_size, (2, 5), generator=torch.Generator().manual_seed(7))
    try:
        free = eng.generate(prompts, 4, top_k=1)
        eos = int(free.input_ids[0, 6])  # the first sequence's second token
        out = eng.generate(prompts, 4, top_k=1, eos_token_id=eos)
        for b in range(2):
            answer = free.input_ids[b, 5:].tolist()
            n = answer.index(eos) + 1 if eos in answer else 4
            assert int(out.lengths[b]) == 5 + n
            assert out.input_ids[b, 5:5 + n].tolist() == answer[:n] and not bool(out.input_ids[b, 5 + n:].any())
            assert bool((out.labels[b, 5 + n:] == -100).all()) and not bool(out.logps[b, 4 + n:].any())
        for kw in (dict(max_new_tokens=0), dict(max_new_tokens=2, lengths=torch.tensor([5])),
                   dict(max_new_tokens=2, lengths=torch.tensor([0, 5])), dict(max_new_tokens=2, lengths=torch.tensor([6, 5])),
                   dict(max_new_tokens=2, top_p=0.0), dict(max_new_tokens=2, temperature=0.0)):
            with pytest.raises(ValueError):
                eng.generate(prompts, **kw)
        with pytest.raises(ValueError):
            eng.generate(prompts[0], 2)
    finally:
        eng.close()


def test_engine_refuses_wrong_lists():
    cfg = LlamaConfig.tiny()
    eng = SlideFSDP(LlamaForCausalLM(cfg, device="meta"), SlideFSDPConfig(dtype=torch.float32, device="cpu"))
    ids = torch.zeros(2, 8, dtype=torch.int64)
    top, logps = torch.zeros(2, 8, 3, dtype=torch.int64), torch.zeros(2, 8, 3)
    d = DistillationObjective()
    try:
        for kw in (dict(objective=d), dict(objective=d, teacher_ids=top), dict(objective=d, teacher_logps=logps),
                   dict(objective=d, teacher_ids=top, teacher_logps=logps[:, :7]),
                   dict(objective=d, teacher_ids=top, teacher_logps=logps[..., :2]),
                   dict(objective=d, teacher_ids=top[..., 0], teacher_logps=logps[..., 0]),
                   dict(objective=d, teacher_ids=logps, teacher_logps=logps),
                   dict(objective=d, teacher_ids=top + cfg.vocab_size, teacher_logps=logps),
                   dict(objective=d, teacher_ids=top, teacher_logps=logps, ref_logps=torch.zeros(2, 8)),
                   dict(objective=PreferenceObjective(), teacher_ids=top, teacher_logps=logps),
                   dict(objective=PolicyObjective(), advantages=torch.zeros(2), old_logps=torch.zeros(2, 8), teacher_ids=top),
                   dict(teacher_ids=top, teacher_logps=logps)):
            with pytest.raises(ValueError):
                eng(input_ids=ids, labels=ids, **kw)
        for bad in (dict(kind="kl"), dict(temperature=0.0)):
            with pytest.raises(ValueError):
                DistillationObjective(**bad)
    finally:
        eng.close()
