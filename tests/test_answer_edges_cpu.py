"""Answer generation and distillation at the ends of what their calls take: the
least temperature, sequences that end inside a tile, on the CPU."""
import math

import pytest
import torch

from test1_b200 import DistillationObjective, PolicyObjective, PreferenceObjective, SlideFSDPConfig, ops
from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM
from test1_b200.slide_fsdp import SlideFSDP

LEAST = 2.0 ** -126


def test_temperatures_whose_inverse_fp32_does_not_have_are_refused():
    z, u, ids = torch.zeros(2, 8), torch.zeros(2), torch.zeros(2, 3, dtype=torch.int64)
    for tau in (LEAST * (1 - 2.0 ** -40), 1e-40, 1e-310):
        for call in (lambda: ops.topk_logprobs(z, 2, tau), lambda: ops.sample_tokens(z, u, tau),
                     lambda: ops.linear_topk_logprob_fwd(z, z, ids, tau),
                     lambda: ops.linear_topk_logprob_bwd(u[:, None].expand(2, 3), z, z, ids, u, z, z, tau),
                     lambda: DistillationObjective(temperature=tau), lambda: PolicyObjective(temperature=tau)):
            with pytest.raises(ValueError, match="2\\^-126"):
                call()


def test_the_least_temperature():
    """The largest logits have all the probability, each the same of it."""
    z = torch.tensor([[0.0, -1.0, 0.0, -1e-30]])
    logp, ids = ops.topk_logprobs(z, 3, LEAST)
    assert ids.tolist() == [[0, 2, 3]] and abs(float(logp[0, 0]) + math.log(2)) < 1e-6
    assert float(logp[0, 0]) == float(logp[0, 1]) and float(logp[0, 2]) < -1e7
    for u, token in ((0.0, 0), (0.49, 0), (0.51, 2), (0.99, 2)):
        assert int(ops.sample_tokens(z, torch.tensor([u]), LEAST)[0]) == token


# ------------------------------------------------------------ sequences of any length
def _engine(tile, **config):
    torch.manual_seed(0)
    cfg = LlamaConfig.tiny()
    eng = SlideFSDP(LlamaForCausalLM(cfg), SlideFSDPConfig(dtype=torch.float32, device="cpu", lr=1e-2, **config))
    eng._tile = tile  # as the attention kernels of the GPU take whole ones
    return eng, cfg


def _run(tile, S):
    eng, cfg = _engine(tile)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, cfg.vocab_size, (2, S), generator=g)
    labels = ids.clone()
    labels[0, :3] = -100
    per_token, logps = -torch.rand(2, S, generator=g), torch.log_softmax(torch.randn(2, S, 6, generator=g), -1)
    top = torch.randint(0, cfg.vocab_size, (2, S, 1), generator=g) + torch.arange(6)
    out = {}
    try:
        out["logits"] = eng(input_ids=ids).logits
        out["token_logprobs"] = eng.token_logprobs(ids, labels, temperature=0.8)
        out["top_logprobs"], out["top_ids"] = eng.top_logprobs(ids, 5)
        for name, kw in {
            "cross-entropy": {},
            "preference": dict(objective=PreferenceObjective(), ref_logps=per_token),
            "policy": dict(objective=PolicyObjective(kl_coef=0.1), old_logps=per_token, ref_logps=per_token,
                           advantages=torch.tensor([1.0, -2.0])),
            "policy of tokens": dict(objective=PolicyObjective(), old_logps=per_token, advantages=per_token),
            "distillation": dict(objective=DistillationObjective(), teacher_logps=logps, teacher_ids=top % cfg.vocab_size),
        }.items():
            out[name] = eng(input_ids=ids, labels=labels, **kw).loss
            if kw:
                out.update({f"{name}, {n}": t for n, t in eng.last_objective.items()})
        eng.wait_for_updates()
        out.update({n: t.clone() for n, t in eng.named_master_tensors()})
    finally:
        eng.close()
    return out


@pytest.mark.parametrize("S", [8, 9, 15])
def test_sequences_that_end_inside_a_tile(S):
    """The same losses, results and weights after five steps as without tiles;
    fp32 sums over other numbers of rows, whose rounding five steps carry on: 1e-4
    of the results' size.  Adam moves a weight of nearly no gradient by up to the
    rate on rounding alone, whichever tensor it is of: 2e-3 of all weights may be
    off.  (2e-3 of each tensor would be half a weight of a norm's 256: none.)"""
    plain, tiled = _run(1, S), _run(8, S)
    assert plain.keys() == tiled.keys()
    off = weights = 0
    for n, want in plain.items():
        got = tiled[n]
        assert got.shape == want.shape and got.is_contiguous(), n
        if n.endswith(".weight"):
            off += int(((got - want).abs() > 1e-4).sum())
            weights += want.numel()
        elif want.is_floating_point():
            assert bool(((got - want).abs() <= 1e-4 * max(1.0, float(want.abs().max()))).all()), n
        else:
            assert torch.equal(got, want), n
    assert 0 < weights and off < 2e-3 * weights


def test_generated_answers_go_back_into_the_engine():
    eng, cfg = _engine(16)
    try:
        a = eng.generate(torch.randint(0, cfg.vocab_size, (2, 6)), 5, generator=torch.Generator().manual_seed(2))
        assert a.input_ids.shape == (2, 11)
        logps = eng.token_logprobs(a.input_ids, a.labels)
        assert torch.allclose(logps, a.logps, atol=1e-4)
        eng(input_ids=a.input_ids, labels=a.labels, objective=PolicyObjective(), old_logps=a.logps, advantages=torch.ones(2))
        assert eng.last_objective["logps"].shape == (2, 11)
        eng.wait_for_updates()
    finally:
        eng.close()


def test_results_of_no_positions_stay_whole():
    """A caller's own objective may give results of other shapes."""
    eng, cfg = _engine(8)

    class Mine(PolicyObjective):
        def loss_and_grad(self, logp, targets, seq_len, inputs):
            loss, dlogp, results = super().loss_and_grad(logp, targets, seq_len, inputs)
            return loss, dlogp, dict(results, table=torch.ones(3, 40))

    ids = torch.zeros(2, 5, dtype=torch.int64)
    try:
        eng(input_ids=ids, labels=ids, objective=Mine(), old_logps=torch.zeros(2, 5), advantages=torch.ones(2))
        assert eng.last_objective["table"].shape == (3, 40) and eng.last_objective["logps"].shape == (2, 5)
        eng.wait_for_updates()
    finally:
        eng.close()


def test_scores_refuse_temperatures_before_the_layers_run():
    eng, cfg = _engine(1)
    ids = torch.zeros(1, 4, dtype=torch.int64)
    ran = []
    eng._forward_only = lambda *args: ran.append(args)
    try:
        for tau in (0.0, 1e-40, 2.0 ** 65, float("inf"), float("nan")):
            with pytest.raises(ValueError):
                eng.top_logprobs(ids, 3, temperature=tau)
            with pytest.raises(ValueError):
                eng.generate(ids, 3, temperature=tau)
        assert not ran
    finally:
        eng.close()
