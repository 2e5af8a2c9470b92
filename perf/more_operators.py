"""Operators of answer generation and of distillation, as measured cases.

Policy training needs answers that the model itself has drawn, and a small model
learns most from a large one's whole distribution, of which the few likeliest
tokens are kept.  Both begin at the output layer's logits:

  logits     x W^T in fp32, for what looks at all of them
  top        the k likeliest tokens of every row and their log-probabilities
  sample     one token of every row, drawn with a given random number from the
             tempered distribution cut by top-k, top-p and min-p
  at         log softmax(x W^T / tau) at K given tokens of every row (a
             teacher's likeliest), with the row's log-sum-exp
  at_grad    from dloss/dlogp [rows, K]: the gradients of x and of W
  distill    divergence of teacher and student over those tokens and the rest
             of the vocabulary: loss, dloss/dlogp, each token's divergence

Rows are tokens, ``batch * seq`` of them, sequence after sequence.  A list entry
with a negative token is none; a prompt's or padding's list has only such.
"""
import math

import torch

own = False  # True: the framework's operators; False: their plain form

NONE = -100
VOCAB, HIDDEN = 128256, 4096  # the output layer of the framework's default model configuration


def listed():
    return [
        # the next token of one sequence: W is all that is read
        {"name": "logits 1 v128256", "op": "logits", "rows": 1, "hidden": HIDDEN, "vocab": VOCAB},
        # a teacher's logits for a chunk of tokens, before its likeliest tokens are taken
        {"name": "logits 1024 v128256", "op": "logits", "rows": 1024, "hidden": HIDDEN, "vocab": VOCAB},
        # a short answer under the smallest configuration: latency counts
        {"name": "top 48 v1024 k8", "op": "top", "rows": 48, "vocab": 1024, "k": 8, "tau": 1.0, "dtype": "float32",
         "allowed": 1.0, "empty": 0},
        # a teacher's chunk: bandwidth counts
        {"name": "top 1024 v128256 k64", "op": "top", "rows": 1024, "vocab": VOCAB, "k": 64, "tau": 1.0,
         "dtype": "float32", "allowed": 1.0, "empty": 0},
        # one sequence's next token with the usual cuts: latency counts
        {"name": "sample 1 v128256 k50", "op": "sample", "rows": 1, "vocab": VOCAB, "tau": 0.7, "top_k": 50,
         "top_p": 0.95, "min_p": 0.0, "dtype": "float32", "allowed": 1.0, "empty": 0},
        # answers to a batch of prompts, a nucleus without a limit on its size
        {"name": "sample 256 v128256 p0.9", "op": "sample", "rows": 256, "vocab": VOCAB, "tau": 1.0, "top_k": 0,
         "top_p": 0.9, "min_p": 0.0, "dtype": "float32", "allowed": 1.0, "empty": 0},
        # a small ragged batch: odd length, a vocabulary that no tile divides, lists of several lengths
        {"name": "at 7x211 v50021 k20", "op": "at", "batch": 7, "seq": 211, "hidden": 1032, "vocab": 50021, "k": 20,
         "prompt": 0.3, "empty": 1, "ragged": True, "tau": 0.7},
        # the default training batch (4 x 1024) with prompts of about a third
        {"name": "at 4x1024 v128256 k64", "op": "at", "batch": 4, "seq": 1024, "hidden": HIDDEN, "vocab": VOCAB, "k": 64,
         "prompt": 0.35, "empty": 0, "ragged": False, "tau": 1.0},
        # the smallest configuration's output layer
        {"name": "at_grad 2x48 v1024 k16", "op": "at_grad", "batch": 2, "seq": 48, "hidden": 256, "vocab": 1024, "k": 16,
         "prompt": 0.25, "empty": 0, "ragged": False, "tau": 1.0, "kind": "forward", "tail": True},
        # the default training batch, every token a teacher's: the most that one step's output layer has to do
        {"name": "at_grad 4x1024 v128256 k64", "op": "at_grad", "batch": 4, "seq": 1024, "hidden": HIDDEN, "vocab": VOCAB,
         "k": 64, "prompt": 0.0, "empty": 0, "ragged": False, "tau": 1.0, "kind": "forward", "tail": True},
        # two short answers
        {"name": "distill 2x128 k8", "op": "distill", "batch": 2, "seq": 128, "k": 8, "prompt": 0.3, "empty": 0,
         "ragged": False, "kind": "forward", "tail": True},
        # a large batch of odd length, lists of several lengths, the symmetric divergence
        {"name": "distill 64x1025 k64", "op": "distill", "batch": 64, "seq": 1025, "k": 64, "prompt": 0.1, "empty": 1,
         "ragged": True, "kind": "jensen", "tail": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _vocab(rng):
    return rng.choice([1024, 32000, VOCAB, _log_int(rng, 300, VOCAB), _log_int(rng, 300, VOCAB) | 1])


def draw(rng):
    op = rng.choice(["logits", "top", "sample", "at", "at_grad", "distill"])
    hidden = rng.choice([256, 512, 1024, 2048, HIDDEN, 8 * _log_int(rng, 8, 512)])
    vocab = _vocab(rng)
    if op in ("logits", "top", "sample"):
        rows = _log_int(rng, 1, 256 if op == "sample" else 1024)
        case = {"op": op, "rows": rows, "vocab": vocab}
        if op == "logits":
            return dict(case, hidden=hidden)
        case.update(tau=rng.choice([1.0, 0.7, 1.3]), dtype=rng.choice(["float32", "float32", "bfloat16"]),
                    allowed=rng.choice([1.0, 1.0, 0.02]), empty=rng.choice([0, 1]) if rows > 1 else 0)
        if op == "top":
            return dict(case, k=min(vocab, _log_int(rng, 1, 64)))
        return dict(case, top_k=rng.choice([0, 0, _log_int(rng, 1, 1000)]), top_p=rng.choice([1.0, 0.9, 0.95, 0.5]),
                    min_p=rng.choice([0.0, 0.0, 0.05]))
    k = _log_int(rng, 1, 64)
    prompt, ragged = rng.choice([0.1, 0.3]), rng.choice([False, True])
    batch = _log_int(rng, 1, 64 if op == "distill" else 8)
    seq = _log_int(rng, 1, 1025 if op == "distill" else 2048)
    while op != "distill" and batch * seq > 4096:
        seq = max(1, seq // 2)
    case = {"op": op, "batch": batch, "seq": seq, "k": k, "prompt": prompt, "empty": rng.choice([0, 1]) if batch > 1 else 0,
            "ragged": ragged}
    if op != "distill":
        case.update(hidden=hidden, vocab=vocab, tau=rng.choice([1.0, 0.7, 1.3]), k=min(k, vocab // 2))
    if op != "at":
        # without the rest of the vocabulary a list of one token says nothing
        case.update(kind=rng.choice(["forward", "reverse", "jensen"]), tail=case["k"] < 4 or rng.choice([True, True, False]))
    return case


# ------------------------------------------------------------------ inputs
def _spans(case):
    """[first, last) token of every sequence's answer: by the case alone, so that every seed has as many."""
    B, S = case["batch"], case["seq"]
    out = []
    for b in range(B):
        first = min(S, int(S * case["prompt"] * (0.5 + math.modf(0.618034 * (b + 1))[0])))
        last = S - int(0.3 * S * case["prompt"] * math.modf(0.754878 * (b + 1))[0])
        out.append((first, first) if b >= B - case["empty"] else (first, max(first, last)))
    return out


def _answered(case):
    return sum(b - a for a, b in _spans(case))


def _lengths(case, device="cpu"):
    """Entries of every row's list [T], by the case alone: 0 outside the answers."""
    spans = torch.tensor(_spans(case), device=device)
    pos = torch.arange(case["seq"], device=device)
    valid = ((pos >= spans[:, :1]) & (pos < spans[:, 1:])).reshape(-1)
    n = torch.full_like(valid, case["k"], dtype=torch.int64)
    if case["ragged"]:  # a teacher that keeps only what is likely enough
        n = (case["k"] - torch.arange(n.numel(), device=device) * 7919 % case["k"]).clamp(min=min(2, case["k"]))
    return torch.where(valid, n, 0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *n: torch.rand(*n, generator=g, device="cuda")  # noqa: E731
    randn = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    s = {"case": case}
    if case["op"] in ("logits", "at", "at_grad"):
        H, V = case["hidden"], case["vocab"]
        T = case["rows"] if case["op"] == "logits" else case["batch"] * case["seq"]
        ids = torch.randint(0, V, (T,), generator=g, device="cuda")
        w = torch.randn(V, H, generator=g, device="cuda", dtype=torch.bfloat16).mul_(2 / math.sqrt(H))
        # hidden states of a trained model: of unit size, and leaning towards the next token by an amount that
        # runs from none to enough to make it the likeliest of all
        x = randn(T, H)
        x.addcmul_(w[ids].float(), 3 * rand(T, 1))
        s.update(x=x.bfloat16(), w=w)
        if case["op"] == "logits":
            return s
        # the teacher sees almost the same; its likeliest tokens, likeliest first
        teacher = (x + 0.3 * randn(T, H)).bfloat16()
        K, n = case["k"], _lengths(case, "cuda")
        keep = torch.arange(K, device="cuda") < n[:, None]
        top, lists = [], []
        for part in teacher.split(512):
            l = (part @ w.t()).float() / case["tau"]
            v, i = l.topk(K, dim=1)
            top.append(v - torch.logsumexp(l, dim=1, keepdim=True))
            lists.append(i)
        s["ids"] = torch.where(keep, torch.cat(lists), NONE)
        if case["op"] == "at_grad":
            wf = w.float()
            out = [_at(xc, wf, ic, case["tau"]) for xc, ic in zip(s["x"].split(512), s["ids"].split(512))]
            s["lse"] = torch.cat([o["lse"] for o in out])
            q = torch.where(keep, torch.cat(top), 0.0)
            s["dlogp"] = _divergence(torch.cat([o["logp"] for o in out]), q, s["ids"], case["kind"], case["tail"])["dlogp"]
            s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(w)
        return s
    if case["op"] == "distill":
        K, n = case["k"], _lengths(case, "cuda")
        T = n.numel()
        keep = torch.arange(K, device="cuda") < n[:, None]
        # the listed tokens take from half to nearly all of the teacher's probability; the student is near it
        z = torch.sort(3 * randn(T, K), dim=1, descending=True).values
        share = 1 - 0.5 * rand(T, 1) ** 3 - 1e-3
        q = torch.log_softmax(z, dim=1) + share.log()
        p = torch.log_softmax(torch.cat([q, torch.log1p(-share)], dim=1) + 0.4 * randn(T, K + 1), dim=1)[:, :K]
        s["ids"] = torch.where(keep, (torch.randint(0, VOCAB, (T, 1), generator=g, device="cuda")
                                      + 1009 * torch.arange(K, device="cuda")) % VOCAB, NONE)
        s["teacher"] = torch.where(keep, q, 0.0)
        s["logp"] = torch.where(keep, p, 0.0)
        return s
    T, V = case["rows"], case["vocab"]
    # a broad bulk, and a few dozen tokens far above it in rows that are sure, hardly in those that are not
    z = 2.2 * randn(T, V)
    few = torch.randint(0, V, (T, 40), generator=g, device="cuda")
    z.scatter_add_(1, few, 14 * rand(T, 1) * rand(T, 40) ** 2)
    if case["allowed"] < 1:  # a grammar's mask
        z.masked_fill_(rand(T, V) >= case["allowed"], -math.inf)
    z[:, V - V // 128:] = -math.inf  # entries that stand for no token
    if case["empty"]:
        z[T - case["empty"]:] = -math.inf
    s["logits"] = z.to(getattr(torch, case["dtype"]))
    if case["op"] == "sample":
        s["u"] = rand(T)
    return s


# -------------------------------------------------------------- plain forms
def _weights(z, tau, dtype):
    """exp((z - largest) / tau) in ``dtype``, 0 where z is -inf."""
    z = z.to(dtype)
    m = z.max(dim=1, keepdim=True).values
    none = z == -math.inf
    return torch.where(none, 0.0, torch.exp(torch.where(none, 0.0, (z - m) / tau))), m, none


def _plain_top(s):
    c, z = s["case"], s["logits"].float()
    e, m, _ = _weights(z, c["tau"], torch.float32)
    v, ids = torch.sort(z, dim=1, descending=True, stable=True)
    v, ids = v[:, :c["k"]], ids[:, :c["k"]]
    none = v == -math.inf
    logp = torch.where(none, 0.0, (torch.where(none, 0.0, v - m)) / c["tau"] - e.sum(dim=1, keepdim=True).log())
    return {"logp": logp, "ids": torch.where(none, -1, ids)}


def _plain_sample(s):
    c, z = s["case"], s["logits"].float()
    w, m, _ = _weights(z, c["tau"], torch.float64)  # borders of sums of many terms decide
    total = w.sum(dim=1)
    _, order = torch.sort(z, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    if c["top_k"]:
        ws[:, c["top_k"]:] = 0
    if c["top_p"] < 1:
        before = ws.cumsum(dim=1) - ws
        ws = torch.where(before < c["top_p"] * ws.sum(dim=1, keepdim=True), ws, 0.0)
    ws = torch.where(ws >= c["min_p"], ws, 0.0)
    cdf = torch.zeros_like(w).scatter_(1, order, ws).cumsum(dim=1)
    token = (cdf <= s["u"].double()[:, None] * cdf[:, -1:]).sum(dim=1)
    none = total == 0
    token = torch.where(none, 0, token)
    at = z.gather(1, token[:, None])[:, 0].double()
    logp = torch.where(none, 0.0, torch.where(none, 0.0, at - m[:, 0]) / c["tau"] - torch.where(none, 1.0, total).log())
    return {"token": torch.where(none, -1, token), "logp": logp.float()}


def _at(x, wf, ids, tau):
    keep = ids >= 0
    live = keep.any(dim=1)
    l = (x.float() @ wf.t()).div_(tau)
    picked = l.gather(1, ids.clamp(min=0))
    m = l.max(dim=1, keepdim=True).values
    log_sum = l.sub_(m).exp_().sum(dim=1).log()
    return {"logp": torch.where(keep, (picked - m) - log_sum[:, None], 0.0),
            "lse": torch.where(live, m[:, 0] + log_sum, 0.0)}


def _plain_at_grad(s):
    c, ids, x, w = s["case"], s["ids"], s["x"].float(), s["w"].float()
    keep = ids >= 0
    up = torch.where(keep, s["dlogp"] / c["tau"], 0.0)
    u = (x @ w.t()).div_(c["tau"]).sub_(s["lse"][:, None]).exp_().mul_(-up.sum(dim=1, keepdim=True))
    u.masked_fill_(~keep.any(dim=1, keepdim=True), 0.0)
    u.scatter_add_(1, ids.clamp(min=0), up)
    return {"dx": (u @ w).to(s["x"].dtype), "dw": (u.t() @ x).to(s["w"].dtype)}


FLOOR = 2.0 ** -20  # the rest of the vocabulary counts as no less likely than this


def _divergence(logp, teacher, ids, kind, tail):
    keep = (ids >= 0) & (teacher > -math.inf)
    live = keep.any(dim=1)
    a, b = torch.where(keep, logp, -math.inf), torch.where(keep, teacher, -math.inf)
    if not tail:
        lse = lambda v: torch.where(live, torch.where(keep, v.exp(), 0.0).sum(dim=1).log(), 0.0)[:, None]  # noqa: E731
        a, b = a - lse(a), b - lse(b)
    zero = torch.zeros_like(a)
    a, b = torch.where(keep, a, zero), torch.where(keep, b, zero)
    p, q = torch.where(keep, a.exp(), zero), torch.where(keep, b.exp(), zero)

    def terms(p, q, a, b):
        """f(p, q) and df/dp, with a = log p and b = log q."""
        if kind == "forward":
            return q * (b - a), -torch.exp(b - a)
        if kind == "reverse":
            return p * (a - b), a - b + 1
        log_m = ((p + q) / 2).log()
        return 0.5 * (p * (a - log_m) + q * (b - log_m)), 0.5 * (a - log_m)

    one = torch.ones_like(a)
    f, df = terms(torch.where(keep, p, one), torch.where(keep, q, one), a, b)
    f, df = torch.where(keep, f, zero), torch.where(keep, df, zero)
    loss = f.sum(dim=1)
    if tail:
        # what is left of 1, whose last bits count
        left = lambda v: 1 - torch.where(keep, v.double().exp(), 0.0).sum(dim=1, keepdim=True)  # noqa: E731
        rp, rq = left(a), left(b)
        pr, qr = rp.clamp(min=FLOOR).float(), rq.clamp(min=FLOOR).float()
        fr, dfr = terms(pr, qr, pr.log(), qr.log())
        loss = loss + fr[:, 0]
        d = p * (df - torch.where(rp > FLOOR, dfr, 0.0))
    else:
        d = p * (df - (p * df).sum(dim=1, keepdim=True))
    n = live.sum().clamp(min=1).float()
    loss = torch.where(live, loss, 0.0)
    return {"loss": loss.sum() / n, "dlogp": torch.where(keep, d / n, zero), "each": loss}


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        if op == "logits":
            return {"logits": s["x"].float() @ s["w"].float().t()}
        if op == "at":
            return _at(s["x"], s["w"].float(), s["ids"], c["tau"])
        if op == "distill":
            return _divergence(s["logp"], s["teacher"], s["ids"], c["kind"], c["tail"])
        return {"top": _plain_top, "sample": _plain_sample, "at_grad": _plain_at_grad}[op](s)
    from test1_b200 import ops

    if op == "logits":
        return {"logits": ops.linear_logits(s["x"], s["w"])}
    if op == "top":
        logp, ids = ops.topk_logprobs(s["logits"], c["k"], temperature=c["tau"])
        return {"logp": logp, "ids": ids}
    if op == "sample":
        token, logp = ops.sample_tokens(s["logits"], s["u"], temperature=c["tau"], top_k=c["top_k"], top_p=c["top_p"],
                                        min_p=c["min_p"])
        return {"token": token, "logp": logp}
    if op == "at":
        logp, lse = ops.linear_topk_logprob_fwd(s["x"], s["w"], s["ids"], temperature=c["tau"])
        return {"logp": logp, "lse": lse}
    if op == "at_grad":
        ops.linear_topk_logprob_bwd(s["dlogp"], s["x"], s["w"], s["ids"], s["lse"], s["dx"], s["dw"], temperature=c["tau"])
        return {"dx": s["dx"], "dw": s["dw"]}
    loss, dlogp, each = ops.distillation_loss_fwd_bwd(s["logp"], s["teacher"], s["ids"], kind=c["kind"], tail=c["tail"])
    return {"loss": loss, "dlogp": dlogp, "each": each}


# -------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op in ("top", "sample"):
        T, V = case["rows"], case["vocab"]
        read = T * V * (2 if case["dtype"] == "bfloat16" else 4)
        return {"bytes": read + (12 * T * case["k"] if op == "top" else 16 * T), "flops": 4 * T * V}
    if op == "logits":
        T, V, H = case["rows"], case["vocab"], case["hidden"]
        return {"bytes": 2 * H * (T + V) + 4 * T * V, "flops": 2 * T * V * H}
    T, n, K = case["batch"] * case["seq"], _answered(case), case["k"]
    entries = int(_lengths(case).sum())
    if op == "distill":
        return {"bytes": 8 * T * K + 8 * entries + 4 * T * K + 4 * T, "flops": 30 * entries}
    V, H = case["vocab"], case["hidden"]
    if op == "at":
        return {"bytes": 2 * H * (n + V) + 8 * T * K + 4 * T * K + 4 * T, "flops": 2 * n * V * H + 4 * n * V}
    # the logits again, then the two products with them
    return {"bytes": 2 * H * (n + V) + 8 * T * K + 4 * entries + 4 * n + 2 * H * (T + V), "flops": 6 * n * V * H + 5 * n * V}


# ----------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "logits":
        return {"logits": s["x"].double() @ s["w"].double().t()}
    if op in ("top", "sample"):
        return _exact_rows(case, s)
    if op == "distill":
        return _exact_distill(case, s)
    ids, T, V = s["ids"], case["batch"] * case["seq"], case["vocab"]
    rows = (ids >= 0).any(dim=1).nonzero()[:, 0]
    w = s["w"].double()
    logp, lse = torch.zeros(ids.shape, dtype=torch.float64, device="cuda"), torch.zeros(T, dtype=torch.float64, device="cuda")
    dx, dw = torch.zeros(T, case["hidden"], dtype=torch.float64, device="cuda"), torch.zeros_like(w)
    for part in rows.split(512):
        x = s["x"][part].double()
        l = x @ w.t() / case["tau"]
        log_p = torch.log_softmax(l, dim=1)
        row, slot = (ids[part] >= 0).nonzero(as_tuple=True)
        at = ids[part][row, slot]
        if op == "at":
            lse[part] = torch.logsumexp(l, dim=1)
            logp[part[row], slot] = log_p[row, at]
            continue
        # the chain rule through log softmax, entry by entry
        up = torch.zeros_like(l).index_put_((row, at), s["dlogp"][part][row, slot].double(), accumulate=True)
        dl = (up - log_p.exp() * up.sum(dim=1, keepdim=True)) / case["tau"]
        dx[part] = dl @ w
        dw += dl.t() @ x
    return {"logp": logp, "lse": lse} if op == "at" else {"dx": dx, "dw": dw}


def _exact_rows(case, s):
    out = {"logp": [], "ids": [], "token": []}
    for r, row in enumerate(s["logits"]):
        z = row.double()
        allowed = (z > -math.inf).nonzero()[:, 0]
        log_p = torch.log_softmax(z[allowed] / case["tau"], dim=0)
        order = torch.sort(z[allowed], descending=True, stable=True).indices  # of equals the lowest first
        if case["op"] == "top":
            best = order[:case["k"]]
            ids = torch.full((case["k"],), -1, device="cuda")
            logp = torch.zeros(case["k"], dtype=torch.float64, device="cuda")
            ids[:len(best)], logp[:len(best)] = allowed[best], log_p[best]
            out["ids"].append(ids)
            out["logp"].append(logp)
            continue
        if not len(allowed):
            out["token"].append(torch.tensor(-1, device="cuda"))
            out["logp"].append(torch.zeros((), dtype=torch.float64, device="cuda"))
            continue
        if case["top_k"]:
            order = order[:case["top_k"]]
        if case["top_p"] < 1:
            p = torch.softmax(log_p[order], dim=0)
            order = order[p.cumsum(dim=0) - p < case["top_p"]]
        if case["min_p"]:
            order = order[log_p[order] >= log_p[order[0]] + math.log(case["min_p"])]
        kept = order.sort().values
        cdf = torch.softmax(log_p[kept], dim=0).cumsum(dim=0)
        hit = kept[torch.searchsorted(cdf, s["u"][r].double() * cdf[-1], right=True)]
        out["token"].append(allowed[hit])
        out["logp"].append(log_p[hit])
    keys = ("logp", "ids") if case["op"] == "top" else ("token", "logp")
    return {k: torch.stack(out[k]) for k in keys}


def _exact_distill(case, s):
    keep = (s["ids"] >= 0) & (s["teacher"] > -math.inf)
    live = keep.any(dim=1).nonzero()[:, 0]
    logp = s["logp"].double().requires_grad_()
    dead = ~keep[live]
    listed_p = logp[live].exp().masked_fill(dead, 0)
    listed_q = s["teacher"][live].double().exp().masked_fill(dead, 0)
    if case["tail"]:
        rest = lambda v: (1 - v.sum(dim=1, keepdim=True)).clamp(min=2.0 ** -20)  # noqa: E731
        p, q = torch.cat([listed_p, rest(listed_p)], dim=1), torch.cat([listed_q, rest(listed_q)], dim=1)
    else:
        p, q = (v / v.sum(dim=1, keepdim=True) for v in (listed_p, listed_q))
    kl = lambda a, b: torch.where(a > 0, a * (a.clamp(min=1e-300).log() - b.clamp(min=1e-300).log()), 0.0).sum(dim=1)  # noqa: E731
    if case["kind"] == "jensen":
        m = (p + q) / 2
        each = (kl(p, m) + kl(q, m)) / 2
    else:
        each = kl(q, p) if case["kind"] == "forward" else kl(p, q)
    loss = each.sum() / max(1, len(live))
    loss.backward()
    whole = torch.zeros(len(logp), dtype=torch.float64, device="cuda").index_copy_(0, live, each.detach())
    return {"loss": loss.detach(), "dlogp": logp.grad.nan_to_num(0.0), "each": whole}
