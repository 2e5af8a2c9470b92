"""Training objectives other than next-token cross-entropy.

An objective is a function of the log-probabilities that the model gives to
the labels.  ``SlideFSDP(..)(input_ids, labels, objective=..)`` runs the same
step as cross-entropy training does; its output layer computes the
log-probabilities, the objective gives the loss and its gradient for them, and
the output layer carries that on to the hidden states and the output weights.
For Llama models it does so without a [tokens, vocabulary] tensor of logits
(``ops.linear_logprob_fwd`` and ``ops.linear_logprob_bwd``); the generic path
of other architectures runs their own head under autograd and holds the logits
in fp32.  On several ranks every rank's loss is that of its own batch, and the
gradients are their mean.  (The reference trains with cross-entropy only.)

``SlideFSDP.token_logprobs`` gives the log-probabilities that an objective
compares with: those of a frozen reference model, and those of the policy
that sampled the answers.
"""
from __future__ import annotations

import warnings
from dataclasses import dataclass, field
from typing import Dict, Optional

import torch

from . import ops


def check_temperature(temperature: float) -> None:
    if not 0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive, got {temperature}")


@dataclass
class PreferenceObjective:
    """Paired answers: the first half of a batch are the chosen ones, the
    second half the rejected ones, in the same order (``labels`` -100 outside
    the answers).  Takes ``ref_logps`` [B, S] (optional) and no other input.  The loss, its kinds
    and the padding rules are those of ``ops.preference_loss_fwd_bwd``.
    Results: ``rewards`` [B], the implicit rewards."""

    beta: float = 0.1
    kind: str = "sigmoid"
    label_smoothing: float = 0.0
    average: bool = False
    temperature: float = 1.0

    def __post_init__(self):
        ops.check_preference(self.beta, self.kind, self.label_smoothing)
        if self.label_smoothing and self.kind != "sigmoid":
            warnings.warn(f"label_smoothing has no effect on the {self.kind} loss", stacklevel=3)
        check_temperature(self.temperature)

    def check(self, inputs, batch: int) -> None:
        if batch % 2:
            raise ValueError(f"a preference batch needs an even number of sequences, got {batch}")
        unused = [n for n in ("old_logps", "advantages") if inputs.get(n) is not None]
        if unused:
            raise ValueError(f"a preference objective does not take {', '.join(unused)}")

    def loss_and_grad(self, logp, targets, seq_len, inputs):
        loss, dlogp, rewards = ops.preference_loss_fwd_bwd(
            logp, inputs.get("ref_logps"), targets, seq_len, self.beta, self.kind, self.label_smoothing, self.average)
        return loss, dlogp, {"rewards": rewards}


@dataclass
class PolicyObjective:
    """Clipped policy optimisation of sampled answers.  Takes ``old_logps``
    [B, S] (of the sampling policy), ``advantages`` [B] or [B, S] and, with
    ``kl_coef`` > 0, ``ref_logps`` [B, S].  ``temperature`` is the sampling
    temperature.  The loss is that of ``ops.policy_loss_fwd_bwd``.  Results:
    ``stats`` [2], mean KL and share of clipped tokens."""

    clip_low: float = 0.2
    clip_high: float = 0.2
    kl_coef: float = 0.0
    reduction: str = "token"
    temperature: float = 1.0

    def __post_init__(self):
        ops.check_policy(self.clip_low, self.clip_high, self.kl_coef, self.reduction)
        check_temperature(self.temperature)

    def check(self, inputs, batch: int) -> None:
        needed = ["old_logps", "advantages"] + (["ref_logps"] if self.kl_coef else [])
        missing = [n for n in needed if inputs.get(n) is None]
        if missing:
            raise ValueError(f"this policy objective needs {', '.join(missing)}")

    def loss_and_grad(self, logp, targets, seq_len, inputs):
        loss, dlogp, stats = ops.policy_loss_fwd_bwd(
            logp, inputs["old_logps"], inputs.get("ref_logps"), inputs["advantages"], targets, seq_len,
            self.clip_low, self.clip_high, self.kl_coef, self.reduction)
        return loss, dlogp, {"stats": stats}


@dataclass
class ObjectiveStep:
    """An objective with one batch's inputs, as the output layer gets it."""

    objective: object
    inputs: Dict[str, Optional[torch.Tensor]]
    results: Dict[str, torch.Tensor] = field(default_factory=dict)

    @classmethod
    def build(cls, objective, batch: int, seq_len: int, device, **inputs) -> "ObjectiveStep":
        """Checks the batch's inputs and moves them to ``device`` as flat fp32
        tensors.  Per-token inputs are [batch, seq_len] as ``token_logprobs``
        returns them: entry [b, s] belongs to labels[b, s + 1]."""
        flat = {}
        for name, t in inputs.items():
            if t is None:
                flat[name] = None
                continue
            if tuple(t.shape) != (batch, seq_len) and not (name == "advantages" and tuple(t.shape) == (batch,)):
                raise ValueError(f"{name} must be [{batch}, {seq_len}], got {tuple(t.shape)}")
            flat[name] = t.to(device=device, dtype=torch.float32, non_blocking=True).reshape(-1)
        objective.check(flat, batch)  # before anything of the step has started
        return cls(objective, flat)

    def loss_and_grad(self, logp: torch.Tensor, targets: torch.Tensor, seq_len: int):
        loss, dlogp, results = self.objective.loss_and_grad(logp, targets, seq_len, self.inputs)
        self.results = dict(results, logps=logp.view(-1, seq_len))
        return loss, dlogp

    @property
    def temperature(self) -> float:
        return float(self.objective.temperature)
