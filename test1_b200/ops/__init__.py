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

import torch

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


MAX_LIST = 512  # tokens of a row's list
MIN_TEMPERATURE = 2.0 ** -126  # of rows and lists: fp32 has its inverse, and log2(e) times that
MAX_TEMPERATURE = 2.0 ** 64  # of rows: 400 times as much, added to the lowest logit, stays finite


def linear_logits(x, w):
    """Logits x @ w^T in fp32: x [T, H], w [V, H] -> [T, V].  The rows of the
    result may lie further apart than V."""
    return _impl(x).linear_logits(x, w)


def topk_logprobs(logits, k, temperature=1.0):
    """The k likeliest tokens of every row of ``logits`` [T, V] (fp32 or bf16)
    and their log-probabilities under softmax(logits / temperature):
    (logp [T, k] fp32, ids [T, k] int64), likeliest first, of equals the lowest
    index first.  Logits of -inf and NaN are no tokens; a row that has fewer
    than k ends with ids of -1 and log-probabilities of 0.  k is at most
    MAX_LIST, V on the GPU 393216; temperatures lie in [2^-126, 2^64]."""
    _check_logits(logits, temperature)
    if not 1 <= k <= min(MAX_LIST, logits.shape[1]):
        raise ValueError(f"k must lie in [1, {min(MAX_LIST, logits.shape[1])}], got {k}")
    return _impl(logits).topk_logprobs(logits, int(k), float(temperature))


def sample_tokens(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token of every row of ``logits`` [B, V] (fp32 or bf16), drawn with
    the random numbers u [B] (fp32, in [0, 1)) from softmax(logits /
    temperature) after three cuts, all on the tokens' order by logit (of equals
    the lowest index first): ``top_k`` keeps the first top_k (0: all); ``top_p``
    keeps, of these, the ones before which less than top_p of their probability
    has come (1: all); ``min_p`` keeps those at least min_p times as likely as
    the likeliest.  The draw takes the lowest index whose running sum over the
    kept tokens, in index order, exceeds u times their sum, and is the same for
    the same inputs.  Returns (token [B] int64, logp [B] fp32), logp under the
    tempered distribution before the cuts, as ``linear_logprob_fwd`` gives it.
    Logits of -inf and NaN are no tokens; a row without any gives -1 and 0.  V
    is at most 393216 on the GPU; temperatures lie in [2^-126, 2^64]."""
    _check_logits(logits, temperature)
    check_sampling(temperature, top_k, top_p, min_p)
    if u.dim() != 1 or u.shape[0] != logits.shape[0]:
        raise ValueError(f"u must be [{logits.shape[0]}], got {tuple(u.shape)}")
    if u.dtype != torch.float32:
        raise ValueError(f"u must be float32, got {u.dtype}")
    return _impl(logits).sample_tokens(logits, u, float(temperature), int(top_k), float(top_p), float(min_p))


def linear_topk_logprob_fwd(x, w, ids, temperature=1.0):
    """Log-probabilities of a list of tokens of every row under the output
    layer: logits = x @ w^T / temperature, of which no [T, V] tensor is kept.
    x [T, H], w [V, H], ids [T, K] int64 (a teacher's likeliest tokens; K at
    most MAX_LIST) -> (logp [T, K], lse [T]) in fp32.  Entries outside the
    vocabulary give 0, and rows without any other give 0 in lse too: they take
    no part.  A temperature is at least 2^-126."""
    _check_lists(x, w, ids, temperature)
    return _impl(x).linear_topk_logprob_fwd(x, w, ids, float(temperature))


def linear_topk_logprob_bwd(dlogp, x, w, ids, lse, dx, dw, temperature=1.0):
    """Gradients of ``linear_topk_logprob_fwd``: from dlogp [T, K] (fp32) and
    the forward's lse, writes dx [T, H] and dw [V, H].  A token that a list
    names twice gets both gradients.  Entries of dlogp whose token is outside
    the vocabulary are not used."""
    _check_lists(x, w, ids, temperature)
    if dlogp.shape != ids.shape:
        raise ValueError(f"dlogp must be {tuple(ids.shape)}, got {tuple(dlogp.shape)}")
    _impl(x).linear_topk_logprob_bwd(dlogp, x, w, ids, lse, dx, dw, float(temperature))


DISTILLATION_KINDS = reference.DISTILLATION_KINDS


def distillation_loss_fwd_bwd(logp, teacher_logp, ids, kind="forward", tail=True):
    """Divergence of a student from its teacher on the teacher's likeliest
    tokens.

    logp and teacher_logp [T, K] (fp32; the teacher's also bf16) are both
    models' log-probabilities of the tokens ids [T, K] (int64).  Entries of a
    negative id, or of a teacher's log-probability of -inf, are left out, and
    rows without any entry take no part; a row's ids must differ and lie below
    the vocabulary's size, which is not known here (``linear_topk_logprob_fwd``
    gives other tokens a log-probability of 0, and that is probability 1: make
    their ids negative for both).  With p the
    student's and q the teacher's probabilities of the listed tokens and, with
    ``tail``, of the rest of the vocabulary as one more outcome (at least
    2^-20: less is the rounding of what is listed), without it scaled to sum to
    1 over the list:
      forward  sum q log(q / p)
      reverse  sum p log(p / q)
      jensen   half of sum p log(p / m) + q log(q / m), m = (p + q) / 2
    Returns (loss [] fp32, the mean over the rows that take part; dloss/dlogp
    [T, K]; the divergence of every row [T])."""
    if logp.dim() != 2 or teacher_logp.shape != logp.shape or ids.shape != logp.shape:
        raise ValueError(f"logp, teacher_logp and ids must be [T, K], got {tuple(logp.shape)}, "
                         f"{tuple(teacher_logp.shape)} and {tuple(ids.shape)}")
    if not 1 <= logp.shape[1] <= MAX_LIST:
        raise ValueError(f"a list has 1 to {MAX_LIST} tokens, got {logp.shape[1]}")
    check_distillation(kind)
    return _impl(logp).distillation_loss_fwd_bwd(logp, teacher_logp, ids, kind, bool(tail))


def check_distillation(kind):
    if kind not in DISTILLATION_KINDS:
        raise ValueError(f"kind must be one of {DISTILLATION_KINDS}, got {kind!r}")


def check_sampling(temperature, top_k, top_p, min_p):
    check_row_temperature(temperature)
    if top_k < 0 or top_k != int(top_k):
        raise ValueError(f"top_k must be a whole number, 0 for all tokens, got {top_k}")
    if not 0 < top_p <= 1:
        raise ValueError(f"top_p must lie in (0, 1], got {top_p}")
    if not 0 <= min_p <= 1:
        raise ValueError(f"min_p must lie in [0, 1], got {min_p}")


def _check_logits(logits, temperature):
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [T, V], got {tuple(logits.shape)}")
    if logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"logits must be float32 or bfloat16, got {logits.dtype}")
    check_row_temperature(temperature)


def check_row_temperature(temperature):
    if not MIN_TEMPERATURE <= temperature <= MAX_TEMPERATURE:
        raise ValueError(f"temperature must lie in [2^-126, 2^64], got {temperature}")


def _check_lists(x, w, ids, temperature):
    if x.dim() != 2 or w.dim() != 2 or ids.dim() != 2 or ids.shape[0] != x.shape[0]:
        raise ValueError(f"x must be [T, H], w [V, H] and ids [T, K], got {tuple(x.shape)}, {tuple(w.shape)} and "
                         f"{tuple(ids.shape)}")
    if not 1 <= ids.shape[1] <= MAX_LIST:
        raise ValueError(f"a list has 1 to {MAX_LIST} tokens, got {ids.shape[1]}")
    if not MIN_TEMPERATURE <= temperature < float("inf"):
        raise ValueError(f"temperature must be at least 2^-126 and finite, got {temperature}")


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
