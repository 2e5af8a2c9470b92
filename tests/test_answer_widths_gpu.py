"""Batches whose sequences end inside an attention tile, on the GPU: answers as
``generate`` gives them go on into a step, and scores of odd widths are those of
the same tokens with more behind them."""
import pytest
import torch

from test_distillation_gpu import _engine

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,new", [(1, 1), (50, 7), (63, 2), (70, 130)])
def test_answers_go_on_into_steps(S, new, cuda_device):
    from test1_b200 import DistillationObjective, PolicyObjective

    eng, cfg = _engine(11, cuda_device, lr=0.0)
    W = S + new
    try:
        g = torch.Generator(device="cuda").manual_seed(S)
        a = eng.generate(torch.randint(0, cfg.vocab_size, (3, S)), new, temperature=0.9, generator=g)
        assert a.input_ids.shape == a.labels.shape == a.logps.shape == (3, W)
        seen = eng.token_logprobs(a.input_ids, a.labels, temperature=0.9)
        # the same weights and tokens, hidden states of batches of other widths: roundings of bf16 through two layers
        assert seen.shape == (3, W) and float((seen - a.logps).abs().max()) < 0.25
        out = eng(input_ids=a.input_ids, labels=a.labels, objective=PolicyObjective(temperature=0.9), old_logps=a.logps,
                  advantages=torch.tensor([1.0, -1.0, 0.5]))
        assert bool(torch.isfinite(out.loss)) and torch.equal(eng.last_objective["logps"], seen)
        logps, top = eng.top_logprobs(a.input_ids, 8)
        assert logps.shape == top.shape == (3, W, 8)
        out = eng(input_ids=a.input_ids, labels=a.labels, objective=DistillationObjective(), teacher_logps=logps, teacher_ids=top)
        got = eng.last_objective
        assert got["divergence"].shape == (3, W) and got["logps"].shape == (3, W, 8)
        # a model distilled from itself: two kernels' roundings of the same fp32 logits, below 2^-10 of a logarithm
        assert abs(float(out.loss)) < 1e-3
        eng.wait_for_updates()
    finally:
        eng.close()


def test_what_lies_behind_changes_nothing(cuda_device):
    """69 tokens a sequence against the caller's own 128 with other tokens behind
    them: the same tiles in the same kernels, so the same bits."""
    eng, cfg = _engine(12, cuda_device, lr=0.0)
    try:
        ids = torch.randint(0, cfg.vocab_size, (2, 128), device=cuda_device)
        labels = torch.full_like(ids, -100)
        labels[:, 5:69] = ids[:, 5:69]
        short, long = (eng.token_logprobs(i, t) for i, t in ((ids[:, :69], labels[:, :69]), (ids, labels)))
        assert torch.equal(short, long[:, :69])
        for a, b in zip(eng.top_logprobs(ids[:, :69], 5), eng.top_logprobs(ids, 5)):
            assert torch.equal(a, b[:, :69])
    finally:
        eng.close()


def test_logits_and_loss_of_odd_widths(cuda_device):
    """bf16 logits and the cross-entropy take vocabularies of a multiple of 8."""
    from test1_b200 import SlideFSDP, SlideFSDPConfig
    from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(13)
    cfg = LlamaConfig(vocab_size=4000, hidden_size=512, intermediate_size=1024, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, initializer_range=0.1)
    eng = SlideFSDP(LlamaForCausalLM(cfg, device="meta"), SlideFSDPConfig(dtype=torch.bfloat16, device=cuda_device, lr=0.0))
    try:
        ids = torch.randint(0, 4000, (2, 128))
        labels = torch.full_like(ids, -100)
        labels[:, 5:69] = ids[:, 5:69]
        short, long = (eng(input_ids=i).logits for i in (ids[:, :69], ids))
        assert short.shape == (2, 69, 4000) and torch.equal(short, long[:, :69])
        short, long = (eng(input_ids=i, labels=t).loss.clone() for i, t in ((ids[:, :69], labels[:, :69]), (ids, labels)))
        assert abs(float(short) - float(long)) <= 1e-5 * float(long)  # a sum of 128 tokens in any order
        eng.wait_for_updates()
    finally:
        eng.close()
