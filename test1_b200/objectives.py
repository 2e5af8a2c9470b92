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
that sampled the answers.  ``SlideFSDP.generate`` samples answers and gives the
latter with them; ``SlideFSDP.top_logprobs`` gives a teacher's likeliest tokens
at every position, from which ``DistillationObjective`` trains.
"""
from __future__ import annotations

import warnings
from dataclasses import dataclass, field
from typing import Dict, Optional

import torch
import torch.nn.functional as F

from . import ops


def check_temperature(temperature: float) -> None:
    # below, fp32 has no inverse of it, and the log-probability of the likeliest token is NaN
    if not ops.MIN_TEMPERATURE <= temperature < float("inf"):
        raise ValueError(f"temperature must be at least 2^-126 and finite, got {temperature}")


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
        unused = [n for n in ("old_logps", "advantages", "teacher_logps", "teacher_ids") if inputs.get(n) is not None]
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
        unused = [n for n in ("teacher_logps", "teacher_ids") if inputs.get(n) is not None]
        if unused:
            raise ValueError(f"a policy objective does not take {', '.join(unused)}")

    def loss_and_grad(self, logp, targets, seq_len, inputs):
        loss, dlogp, stats = ops.policy_loss_fwd_bwd(
            logp, inputs["old_logps"], inputs.get("ref_logps"), inputs["advantages"], targets, seq_len,
            self.clip_low, self.clip_high, self.kl_coef, self.reduction)
        return loss, dlogp, {"stats": stats}


@dataclass
class DistillationObjective:
    """Learning from a teacher's likeliest tokens.  Takes ``teacher_logps`` and
    ``teacher_ids`` [B, S, K] as ``SlideFSDP.top_logprobs`` of the teacher gives
    them (at this ``temperature``, of the same vocabulary); positions whose label
    is -100 take no part, nor do entries of id -1 or, where the lists are on the
    GPU, of an id beyond the student's vocabulary (in host memory it is refused).
    The divergences and ``tail``
    are those of ``ops.distillation_loss_fwd_bwd``.  Results: ``divergence``
    [B, S], of every position; ``logps`` [B, S, K], of the teacher's tokens."""

    kind: str = "forward"
    tail: bool = True
    temperature: float = 1.0

    def __post_init__(self):
        ops.check_distillation(self.kind)
        check_temperature(self.temperature)

    def check(self, inputs, batch: int) -> None:
        missing = [n for n in ("teacher_logps", "teacher_ids") if inputs.get(n) is None]
        if missing:
            raise ValueError(f"a distillation objective needs {', '.join(missing)}")
        unused = [n for n in ("ref_logps", "old_logps", "advantages") if inputs.get(n) is not None]
        if unused:
            raise ValueError(f"a distillation objective does not take {', '.join(unused)}")

    def token_lists(self, targets, inputs):
        """[T, K] tokens whose log-probabilities the loss is a function of."""
        ids = inputs["teacher_ids"]
        return torch.where((targets != -100)[:, None], ids, -1)

    def loss_and_grad(self, logp, targets, seq_len, inputs):
        loss, dlogp, each = ops.distillation_loss_fwd_bwd(logp, inputs["teacher_logps"], self.token_lists(targets, inputs),
                                                          self.kind, self.tail)
        return loss, dlogp, {"divergence": each.view(-1, seq_len)}


@dataclass
class ObjectiveStep:
    """An objective with one batch's inputs, as the output layer gets it."""

    objective: object
    inputs: Dict[str, Optional[torch.Tensor]]
    seq_len: int  # of the caller's batch; the step's own may be longer
    results: Dict[str, torch.Tensor] = field(default_factory=dict)

    @classmethod
    def build(cls, objective, batch: int, seq_len: int, device, behind: int = 0, **inputs) -> "ObjectiveStep":
        """Checks the batch's inputs and moves them to ``device`` as flat fp32
        tensors.  Per-token inputs are [batch, seq_len] as ``token_logprobs``
        returns them: entry [b, s] belongs to labels[b, s + 1].  ``behind``
        positions without a label follow every sequence."""
        flat = {}
        lists = [t.shape for n, t in inputs.items() if n.startswith("teacher_") and t is not None]
        for name, t in inputs.items():
            if t is None:
                flat[name] = None
                continue
            if name.startswith("teacher_"):
                if t.dim() != 3 or t.shape != lists[0] or t.shape[:2] != (batch, seq_len):
                    raise ValueError(f"{name} must be [{batch}, {seq_len}, K], got {tuple(t.shape)}")
                if not 1 <= t.shape[2] <= ops.MAX_LIST:
                    raise ValueError(f"{name} must have 1 to {ops.MAX_LIST} entries a position, got {t.shape[2]}")
                if name == "teacher_ids" and t.is_floating_point():
                    raise ValueError(f"teacher_ids must be whole numbers, got {t.dtype}")
                kept = torch.int64 if name == "teacher_ids" else t.dtype if t.dtype == torch.bfloat16 else torch.float32
                t = F.pad(t.to(device=device, dtype=kept, non_blocking=True), (0, 0, 0, behind))
                flat[name] = t.reshape(-1, t.shape[2])
                continue
            if tuple(t.shape) != (batch, seq_len) and not (name == "advantages" and tuple(t.shape) == (batch,)):
                raise ValueError(f"{name} must be [{batch}, {seq_len}], got {tuple(t.shape)}")
            t = t.to(device=device, dtype=torch.float32, non_blocking=True)
            flat[name] = (F.pad(t, (0, behind)) if t.dim() == 2 else t).reshape(-1)
        objective.check(flat, batch)  # before anything of the step has started
        return cls(objective, flat, seq_len)

    def token_lists(self, targets: torch.Tensor) -> Optional[torch.Tensor]:
        """[T, K] tokens whose log-probabilities the objective takes; None: the
        targets alone."""
        lists = getattr(self.objective, "token_lists", None)
        return None if lists is None else lists(targets, self.inputs)

    def loss_and_grad(self, logp: torch.Tensor, targets: torch.Tensor, seq_len: int):
        loss, dlogp, results = self.objective.loss_and_grad(logp, targets, seq_len, self.inputs)
        results = dict(results, logps=logp.view(-1, seq_len, *logp.shape[1:]))
        # those of positions are [B, S, ..]
        self.results = {n: t[:, :self.seq_len].contiguous() if t.dim() > 1 and t.shape[1] == seq_len else t
                        for n, t in results.items()}
        return loss, dlogp

    @property
    def temperature(self) -> float:
        return float(self.objective.temperature)
