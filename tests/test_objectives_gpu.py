"""Preference and policy steps of the engine on the GPU: the label
log-probabilities against those of the model's logits, the steps' launches,
and a run that learns."""
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_token_logprobs_match_logits(cuda_device):
    from test1_b200 import SlideFSDP, SlideFSDPConfig, ops
    from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=4001, hidden_size=512, intermediate_size=1024, num_hidden_layers=2,
                      num_attention_heads=4, num_key_value_heads=2, initializer_range=0.1)
    eng = SlideFSDP(LlamaForCausalLM(cfg, device="meta"), SlideFSDPConfig(dtype=torch.bfloat16, device=cuda_device))
    ids = torch.randint(0, cfg.vocab_size, (3, 128))
    labels = ids.clone()
    labels[:, :40] = -100
    try:
        got = eng.token_logprobs(ids, labels, temperature=0.9)
        # the output layer's own input, so that only the last product differs
        states = []
        head = eng.output_layer
        logits_of = head.logits
        head.logits = lambda h: states.append(ops.rmsnorm_fwd(h, head.norm.weight.data, head.eps)[0]) or h
        eng(input_ids=ids)
        w = dict(eng.named_master_tensors())["lm_head.weight"].view(cfg.vocab_size, -1).bfloat16().float().cuda()
        head.logits = logits_of
        lp = torch.log_softmax(states[0].double() @ w.double().t() / 0.9, -1)
        tg = ops.shift_labels(labels).cuda()
        want = torch.where(tg >= 0, lp.gather(1, tg.clamp_min(0)[:, None])[:, 0], 0.0).view(3, 128)
        # fp32 accumulation of 512 products of logits below 100
        assert float((got - want).abs().max()) < 64 * 2.0 ** -23 * 100
        assert not bool(got[:, -1].any())
    finally:
        eng.close()


def test_example_learns_on_the_kernels(cuda_device):
    from test1_b200.ops import native_launch_count

    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import preference_tuning

    before = native_launch_count()
    margins, policy_losses = preference_tuning.run("cuda:0", steps=4, verbose=False)
    assert native_launch_count() > before
    assert abs(margins[0]) < 1e-3 and margins[-1] > 0.5
    assert all(l == l for l in policy_losses)
