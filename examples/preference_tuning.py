"""Training on preferences and on sampled answers: a tiny Llama-architecture
model on the CPU (no GPU needed) or on cuda:0.

    python examples/preference_tuning.py [--device cuda:0] [--steps 8]

1. The frozen reference's log-probabilities of chosen and rejected answers.
2. Preference steps: the margin between the answers' implicit rewards grows.
3. Policy steps on answers with advantages, clipped against the policy that
   gave them and held to the reference by a KL term.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from test1_b200 import PolicyObjective, PreferenceObjective, SlideFSDPConfig  # noqa: E402
from test1_b200.models.llama import LlamaConfig, LlamaForCausalLM  # noqa: E402
from test1_b200.slide_fsdp import SlideFSDP  # noqa: E402


def run(device: str = "cpu", steps: int = 8, verbose: bool = True):
    dev = torch.device(device)
    cfg = LlamaConfig.tiny()
    if dev.type == "cuda":  # the sm_100a attention kernels take head_dim 128
        cfg = LlamaConfig(vocab_size=4096, hidden_size=512, intermediate_size=1536, num_hidden_layers=2,
                          num_attention_heads=4, num_key_value_heads=2)
    dtype = torch.bfloat16 if dev.type == "cuda" else torch.float32
    torch.manual_seed(0)
    engine = SlideFSDP(LlamaForCausalLM(cfg, device="meta"), SlideFSDPConfig(dtype=dtype, device=dev, lr=5e-4))
    say = print if verbose else (lambda *a: None)
    g = torch.Generator().manual_seed(1)
    pairs, prompt, S = 2, 24, 64
    ids = torch.randint(0, cfg.vocab_size, (2 * pairs, S), generator=g)
    ids[pairs:, :prompt] = ids[:pairs, :prompt]  # the answers of a pair share their prompt
    labels = ids.clone()
    labels[:, :prompt] = -100

    ref = engine.token_logprobs(ids, labels)
    margins, policy_losses = [], []
    for step in range(steps):
        out = engine(input_ids=ids, labels=labels, objective=PreferenceObjective(beta=0.1), ref_logps=ref)
        r = engine.last_objective["rewards"]
        margins.append(float((r[:pairs] - r[pairs:]).mean()))
        say(f"preference step {step}: loss {float(out.loss):.4f}, reward margin {margins[-1]:+.3f}")

    old = engine.token_logprobs(ids, labels)
    advantages = torch.tensor([1.0] * pairs + [-1.0] * pairs)
    for step in range(steps):
        out = engine(input_ids=ids, labels=labels, objective=PolicyObjective(clip_high=0.28, kl_coef=0.02),
                     old_logps=old, ref_logps=ref, advantages=advantages)
        kl, clipped = engine.last_objective["stats"].tolist()
        policy_losses.append(float(out.loss))
        say(f"policy step {step}: loss {policy_losses[-1]:+.4f}, KL {kl:.4f}, clipped {clipped:.2f}")
    engine.close()
    return margins, policy_losses


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--device", default="cpu")
    ap.add_argument("--steps", type=int, default=8)
    a = ap.parse_args()
    run(a.device, a.steps)


if __name__ == "__main__":
    main()
