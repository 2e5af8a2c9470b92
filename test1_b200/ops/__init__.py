"""Ops of the Llama training step.

Every function takes and returns plain tensors.  CUDA tensors run the
hand-written sm_100a kernels of ``test1_b200._cuda`` (``ops.native``); CPU
tensors run the PyTorch statements in ``ops.reference`` (the oracle, and the
path of the CPU/gloo tests).  There is no silent fallback on the GPU: if the
CUDA extension is missing, the first op raises.

Setting ``T1_OPS=torch`` runs the PyTorch statements on CUDA tensors too; it
exists only to measure the framework against library kernels and is never
the default.
"""
from __future__ import annotations

import os

from . import reference

_FORCE_TORCH = os.environ.get("T1_OPS", "native").lower() == "torch"


def use_native(t) -> bool:
    return t.is_cuda and not _FORCE_TORCH


def _impl(t):
    if use_native(t):
        from . import native

        return native
    return reference


def rmsnorm_fwd(x, w, eps):
    return _impl(x).rmsnorm_fwd(x, w, eps)


def rmsnorm_bwd(dy, x, w, rstd, residual_grad=None):
    return _impl(x).rmsnorm_bwd(dy, x, w, rstd, residual_grad)


def linear_fwd(x, w, residual=None):
    return _impl(x).linear_fwd(x, w, residual)


def linear_fwd_rope(x, w, cos, sin, seq_len, n_q, n_kv, head_dim):
    """QKV projection with the rotary embedding of the q and k heads applied:
    x @ w^T, then rotate column blocks [0, (n_q + n_kv) head_dim) by position
    t % seq_len (on the GPU fused into the GEMM epilogue when possible)."""
    return _impl(x).linear_fwd_rope(x, w, cos, sin, seq_len, n_q, n_kv, head_dim)


def linear_dgrad(dy, w):
    return _impl(dy).linear_dgrad(dy, w)


def linear_wgrad(dy, x, out=None):
    return _impl(dy).linear_wgrad(dy, x, out)


def rope_qkv_(qkv, n_q, n_kv, head_dim, cos, sin, seq_len, inverse=False):
    """Rotate the q and k column blocks of ``qkv`` [T, (n_q+2 n_kv) D] in place."""
    return _impl(qkv).rope_qkv_(qkv, n_q, n_kv, head_dim, cos, sin, seq_len, inverse)


def attention_fwd(qkv, n_q, n_kv, head_dim, seq_len):
    """Causal GQA attention on the fused qkv buffer -> (o [T, n_q D], lse [n_q, T])."""
    return _impl(qkv).attention_qkv_fwd(qkv, n_q, n_kv, head_dim, seq_len)


def attention_bwd(do, qkv, o, lse, n_q, n_kv, head_dim, seq_len):
    """-> dqkv [T, (n_q + 2 n_kv) D] (gradients of the rotated q, k and of v)."""
    return _impl(qkv).attention_qkv_bwd(do, qkv, o, lse, n_q, n_kv, head_dim, seq_len)


def swiglu_fwd(gu):
    """gu [T, 2I] = [gate | up] -> silu(gate) * up [T, I]."""
    return _impl(gu).swiglu_gu_fwd(gu)


def swiglu_bwd(da, gu):
    """-> dgu [T, 2I] = [dgate | dup]."""
    return _impl(gu).swiglu_gu_bwd(da, gu)


def embedding_fwd(ids, w):
    return _impl(w).embedding_fwd(ids, w)


def embedding_bwd(dh, ids, num_rows, out=None):
    return _impl(dh).embedding_bwd(dh, ids, num_rows, out)


def cross_entropy_fwd_bwd(logits, targets, ignore_index=-100, grad_scale=None):
    return _impl(logits).cross_entropy_fwd_bwd(logits, targets, ignore_index, grad_scale)


def linear_cross_entropy(x, w, targets, dx, dw, chunk_rows, ignore_index=-100):
    """Output layer's lm_head GEMM + cross-entropy forward and backward in
    token chunks (no [T, V] logits kept): writes dx [T, H] and dw [V, H],
    returns (loss fp32 scalar, n_valid)."""
    return _impl(x).linear_cross_entropy(x, w, targets, dx, dw, chunk_rows, ignore_index)


def linear_logprob_fwd(x, w, targets, ignore_index=-100, temperature=1.0):
    """Log-probability of every token's target under the output layer:
    logits = x @ w^T / temperature, of which no [T, V] tensor is kept.
    x [T, H], w [V, H], targets [T] -> (logp [T], lse [T]) in fp32, lse the
    log-sum-exp of the row's logits.  Tokens whose target is ignore_index (or
    no vocabulary index) give 0 in both."""
    return _impl(x).linear_logprob_fwd(x, w, targets, ignore_index, temperature)


def linear_logprob_bwd(dlogp, x, w, targets, lse, dx, dw, ignore_index=-100, temperature=1.0):
    """Gradients of ``linear_logprob_fwd``: from dlogp [T] (fp32) and the
    forward's lse (of the same x and w: its logits' errors then cancel), writes
    dx [T, H] and dw [V, H].  Entries of dlogp at ignored tokens are not used."""
    _impl(x).linear_logprob_bwd(dlogp, x, w, targets, lse, dx, dw, ignore_index, temperature)


PREFERENCE_KINDS = reference.PREFERENCE_KINDS


def preference_loss_fwd_bwd(logp, ref_logp, targets, seq_len, beta=0.1, kind="sigmoid", label_smoothing=0.0,
                            average=False, ignore_index=-100):
    """Loss of answer pairs on their log-probability ratios to a reference.

    The batch holds T / seq_len sequences: the first half chosen answers, the
    second half the rejected ones, in the same order.  r = sum over a
    sequence's answer tokens of logp - ref_logp (``average``: the mean; no
    ref_logp: of logp), m = r_chosen - r_rejected, and per pair
      sigmoid  -(1 - label_smoothing) log s(beta m) - label_smoothing log s(-beta m)
      hinge    max(0, 1 - beta m)
      ipo      (m - 1 / (2 beta))^2
    averaged over the pairs that have an answer token (a pair of padding only
    is left out); label_smoothing is the sigmoid loss's alone.  Returns
    (loss [] fp32, dloss/dlogp [T], rewards [T / seq_len] = beta r)."""
    _check_loss(logp, targets, seq_len)
    if (logp.shape[0] // seq_len) % 2:
        raise ValueError(f"a preference batch needs an even number of sequences, got {logp.shape[0] // seq_len}")
    check_preference(beta, kind, label_smoothing)
    return _impl(logp).preference_loss_fwd_bwd(logp, ref_logp, targets, seq_len, beta, kind, label_smoothing,
                                               average, ignore_index)


def policy_loss_fwd_bwd(logp, old_logp, ref_logp, advantages, targets, seq_len, clip_low=0.2, clip_high=0.2,
                        kl_coef=0.0, reduction="token", ignore_index=-100):
    """Clipped policy loss with a KL penalty, on the answer tokens of
    T / seq_len sequences.  With rho = exp(logp - old_logp), advantages A per
    sequence [T / seq_len] or per token [T], and e = ref_logp - logp:
      -min(A rho, A clip(rho, 1 - clip_low, 1 + clip_high)) + kl_coef (exp(e) - 1 - e)
    per token, averaged over all answer tokens (``reduction="token"``) or over
    the sequences that have one of each sequence's mean ("sequence").
    ref_logp may be None when kl_coef is 0.  Returns (loss [] fp32,
    dloss/dlogp [T], [mean KL term, share of clipped tokens])."""
    _check_loss(logp, targets, seq_len)
    check_policy(clip_low, clip_high, kl_coef, reduction)
    if kl_coef and ref_logp is None:
        raise ValueError("a KL term (kl_coef > 0) needs ref_logp")
    if advantages.dim() != 1 or advantages.shape[0] not in (logp.shape[0], logp.shape[0] // seq_len):
        raise ValueError(f"advantages must be [T] or [T / seq_len], got {tuple(advantages.shape)}")
    return _impl(logp).policy_loss_fwd_bwd(logp, old_logp, ref_logp, advantages, targets, seq_len, clip_low,
                                           clip_high, kl_coef, reduction, ignore_index)


def check_preference(beta, kind, label_smoothing):
    if kind not in PREFERENCE_KINDS:
        raise ValueError(f"kind must be one of {PREFERENCE_KINDS}, got {kind!r}")
    if not (0 < beta < float("inf")):
        raise ValueError(f"beta must be positive, got {beta}")
    if not 0.0 <= label_smoothing < 0.5:
        raise ValueError(f"label_smoothing must lie in [0, 0.5), got {label_smoothing}")


def check_policy(clip_low, clip_high, kl_coef, reduction):
    if not (0 <= clip_low < 1 and 0 <= clip_high < float("inf")):
        raise ValueError(f"clip_low must lie in [0, 1) and clip_high in [0, inf), got {clip_low} and {clip_high}")
    if reduction not in ("token", "sequence"):
        raise ValueError(f"reduction must be 'token' or 'sequence', got {reduction!r}")
    if not (0 <= kl_coef < float("inf")):
        raise ValueError(f"kl_coef must not be negative, got {kl_coef}")


def _check_loss(logp, targets, seq_len):
    if logp.dim() != 1 or targets.shape != logp.shape:
        raise ValueError(f"logp and targets must be [T], got {tuple(logp.shape)} and {tuple(targets.shape)}")
    if seq_len <= 0 or logp.shape[0] % seq_len:
        raise ValueError(f"{logp.shape[0]} tokens are not a multiple of seq_len {seq_len}")


shift_labels = reference.shift_labels
rope_tables = reference.rope_tables


def native_launch_count() -> int:
    """Number of sm_100a kernel launches issued through ``ops.native`` so far."""
    import sys

    mod = sys.modules.get(__name__ + ".native")
    return 0 if mod is None else mod.launch_count()
