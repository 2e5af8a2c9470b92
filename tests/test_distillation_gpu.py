"""Generation, a teacher's likeliest tokens and distillation steps of the engine
on the GPU, together as they are used: a teacher's answers are drawn, scored by
it and learnt from."""
import pytest
import torch

import _lists_oracle as oracle

pytestmark = pytest.mark.gpu


def _engine(seed, device, hidden=512, std=0.1, **config):
    from test1_b200 import SlideFSDP, SlideFSDPConfig
    from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(seed)
    cfg = LlamaConfig(vocab_size=4001, hidden_size=hidden, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, initializer_range=std)
    return SlideFSDP(LlamaForCausalLM(cfg, device="meta"), SlideFSDPConfig(dtype=torch.bfloat16, device=device, **config)), cfg


def _head_inputs(eng, ids):
    """The output layer's own input of a forward pass and its weight on the GPU."""
    from test1_b200 import ops

    seen, head = [], eng.output_layer
    logits_of = head.logits

    def spy(h):
        seen.extend((ops.rmsnorm_fwd(h, head.norm.weight.data, head.eps)[0], head.lm_head.weight.data.clone()))
        return h

    head.logits = spy
    try:
        eng(input_ids=ids)
    finally:
        head.logits = logits_of
    return seen


@pytest.mark.parametrize("chunk", [2048, 100, 0])
def test_top_logprobs(chunk, cuda_device):
    eng, cfg = _engine(0, cuda_device, lm_head_chunk_tokens=chunk)
    ids = torch.randint(0, cfg.vocab_size, (3, 128))
    try:
        logps, top = eng.top_logprobs(ids, 20, temperature=0.9)
        assert logps.shape == top.shape == (3, 128, 20)
        x, w = _head_inputs(eng, ids)
        lp = torch.log_softmax(x.double() @ w.double().t() / 0.9, -1)
        # fp32 accumulation of 512 products of logits below 100
        tol = 64 * 2.0 ** -23 * 100
        assert float((logps.view(-1, 20) - lp.gather(1, top.view(-1, 20))).abs().max()) < tol
        want = lp.topk(20, 1).values
        assert float((logps.view(-1, 20) - want).abs().max()) < tol  # the likeliest, up to equals
        assert bool((top.sort(-1).values.diff(dim=-1) > 0).all())
    finally:
        eng.close()


def test_generation_and_its_logprobs(cuda_device):
    eng, cfg = _engine(1, cuda_device)
    prompts = torch.randint(0, cfg.vocab_size, (4, 70))
    lengths = torch.tensor([70, 33, 1, 64])
    try:
        g = torch.Generator(device="cuda").manual_seed(3)
        out = eng.generate(prompts, 5, lengths, temperature=0.8, top_k=50, top_p=0.95, generator=g)
        assert out.lengths.tolist() == [75, 38, 6, 69] and out.input_ids.shape == (4, 75)
        g = torch.Generator(device="cuda").manual_seed(3)
        again = eng.generate(prompts, 5, lengths, temperature=0.8, top_k=50, top_p=0.95, generator=g)
        assert torch.equal(out.input_ids, again.input_ids) and torch.equal(out.logps, again.logps)
        # training on the same tokens sees the same log-probabilities: hidden states of another row width in bf16
        pad = torch.zeros(4, 128, dtype=torch.int64, device="cuda")
        labels = torch.full_like(pad, -100)
        pad[:, :75], labels[:, :75] = out.input_ids, out.labels
        seen = eng.token_logprobs(pad, labels, temperature=0.8)[:, :75]
        assert float((out.logps - seen).abs().max()) < 0.25
        assert bool(((out.logps != 0) == (seen != 0)).all())
        # every token is one of the 50 likeliest at its place
        _, top = eng.top_logprobs(pad, 60, temperature=0.8)
        for b in range(4):
            for s in range(int(lengths[b]) - 1, int(out.lengths[b]) - 1):
                assert int(out.input_ids[b, s + 1]) in top[b, s].tolist()
    finally:
        eng.close()


@pytest.mark.parametrize("kind,tail", [("forward", True), ("reverse", True), ("jensen", False)])
def test_a_run_of_them_together(kind, tail, cuda_device):
    from test1_b200 import DistillationObjective
    from test1_b200.ops import native

    teacher, cfg = _engine(2, cuda_device)
    prompts = torch.randint(0, cfg.vocab_size, (4, 32))
    try:
        out = teacher.generate(prompts, 32, temperature=1.0, generator=torch.Generator(device="cuda").manual_seed(4))
        logps, top = teacher.top_logprobs(out.input_ids, 16)
    finally:
        teacher.close()
    student, _ = _engine(3, cuda_device, lr=0.0)
    try:
        x, w = _head_inputs(student, out.input_ids)
        step = student(input_ids=out.input_ids, labels=out.labels, objective=DistillationObjective(kind=kind, tail=tail),
                       teacher_logps=logps, teacher_ids=top)
        got = student.last_objective
        ids = torch.where((torch.cat([out.labels[:, 1:], torch.full_like(out.labels[:, :1], -100)], 1) >= 0)[..., None], top, -1)
        lp, _, _, _ = oracle.listed_logprob(x, w, ids.view(-1, 16), 1.0)
        # fp32 accumulation of 512 products of logits below 100
        assert float((got["logps"].view(-1, 16) - lp).abs().max()) < 64 * 2.0 ** -23 * 100
        loss, _, each, _ = oracle.distillation(lp.float().cpu(), logps.view(-1, 16).cpu(), ids.view(-1, 16).cpu(), kind, tail)
        assert abs(float(step.loss) - float(loss)) < 1e-3 * max(1.0, float(loss))
        assert float((got["divergence"].view(-1).cpu() - each).abs().max()) < 1e-2
        assert native.gemm_error() == 0
        student.wait_for_updates()
    finally:
        student.close()
