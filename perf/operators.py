"""Operators of preference and policy training, as measured cases.

After supervised fine-tuning the same engine is asked for two more things: the
log-probability that the model gives to the tokens of an answer (for its own
weights and for a frozen reference), and losses that are functions of those
log-probabilities.  Four operators make that step:

  logprob       logp[t] = log softmax(x W^T / tau)[t, target[t]], with the row's
                log-sum-exp; rows whose target is ignored give 0
  logprob_grad  from dloss/dlogp[t]: the gradients of x and of W
  preference    paired log ratios of chosen and rejected answers against a
                reference: loss, dloss/dlogp, the implicit rewards
  policy        clipped importance-weighted policy loss with a KL term:
                loss, dloss/dlogp, [mean KL, share of clipped tokens]

Rows are tokens, ``batch * seq`` of them, sequence after sequence.  Every
sequence has a prompt (ignored), an answer and right padding (ignored).
"""
import math

import torch

own = False  # True: the framework's operators; False: their plain form

IGNORE = -100
VOCAB, HIDDEN = 128256, 4096  # the output layer of the framework's default model configuration


def listed():
    return [
        # one token of a sequence that is being generated, scored by the full-size output layer: W is all that is read
        {"name": "logprob 1x1 v128256", "op": "logprob", "batch": 1, "seq": 1, "hidden": HIDDEN, "vocab": VOCAB,
         "prompt": 0.0, "empty": 0, "tau": 1.0},
        # a small evaluation batch: odd length, a vocabulary that no tile divides, one sequence of padding only
        {"name": "logprob 7x211 v50021", "op": "logprob", "batch": 7, "seq": 211, "hidden": 1032, "vocab": 50021,
         "prompt": 0.3, "empty": 1, "tau": 0.7},
        # reference log-probabilities of four pairs of answers at the default training length
        {"name": "logprob 8x1024 v128256", "op": "logprob", "batch": 8, "seq": 1024, "hidden": HIDDEN, "vocab": VOCAB,
         "prompt": 0.25, "empty": 0, "tau": 1.0},
        # the smallest configuration's output layer: latency counts
        {"name": "grad 2x48 v1024", "op": "logprob_grad", "batch": 2, "seq": 48, "hidden": 256, "vocab": 1024,
         "prompt": 0.25, "empty": 0, "tau": 1.0},
        # a small ragged batch
        {"name": "grad 5x173 v32001", "op": "logprob_grad", "batch": 5, "seq": 173, "hidden": 2048, "vocab": 32001,
         "prompt": 0.3, "empty": 1, "tau": 0.7},
        # the default training batch (4 x 1024) with prompts of about a third
        {"name": "grad 4x1024 v128256", "op": "logprob_grad", "batch": 4, "seq": 1024, "hidden": HIDDEN, "vocab": VOCAB,
         "prompt": 0.35, "empty": 0, "tau": 1.0},
        # four pairs, every token an answer's: the most that one step's output layer has to do
        {"name": "grad 8x1024 v128256", "op": "logprob_grad", "batch": 8, "seq": 1024, "hidden": HIDDEN, "vocab": VOCAB,
         "prompt": 0.0, "empty": 0, "tau": 1.0},
        # one pair of short answers
        {"name": "preference 2x128", "op": "preference", "batch": 2, "seq": 128, "prompt": 0.3, "empty": 0,
         "kind": "sigmoid", "beta": 0.1, "smooth": 0.0, "average": False, "ref": True},
        # a large batch of long pairs of odd length, two of them padding, smoothed labels
        {"name": "preference 128x8191", "op": "preference", "batch": 128, "seq": 8191, "prompt": 0.3, "empty": 2,
         "kind": "sigmoid", "beta": 0.1, "smooth": 0.1, "average": False, "ref": True},
        # one prompt's group of short answers
        {"name": "policy 8x96", "op": "policy", "batch": 8, "seq": 96, "prompt": 0.3, "empty": 0,
         "clip_low": 0.2, "clip_high": 0.2, "kl_coef": 0.04, "per_token": False, "reduction": "token"},
        # an ordinary batch with a critic's advantage at every token and no reference model
        {"name": "policy 64x1025", "op": "policy", "batch": 64, "seq": 1025, "prompt": 0.3, "empty": 3,
         "clip_low": 0.2, "clip_high": 0.28, "kl_coef": 0.0, "per_token": True, "reduction": "sequence"},
        # a large batch of long answers: bandwidth counts
        {"name": "policy 512x8192", "op": "policy", "batch": 512, "seq": 8192, "prompt": 0.1, "empty": 0,
         "clip_low": 0.2, "clip_high": 0.2, "kl_coef": 0.04, "per_token": False, "reduction": "token"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["logprob", "logprob_grad", "preference", "policy"])
    if op in ("logprob", "logprob_grad"):
        hidden = rng.choice([256, 512, 1024, 2048, HIDDEN, 8 * _log_int(rng, 8, 1024)])
        vocab = rng.choice([1024, 32000, VOCAB, _log_int(rng, 300, VOCAB), _log_int(rng, 300, VOCAB) | 1])
        batch, seq = _log_int(rng, 1, 16), _log_int(rng, 1, 2048)
        while batch * seq > 8192 or batch * seq * vocab * hidden > 8192 * VOCAB * HIDDEN:
            seq = max(1, seq // 2)
        return {"op": op, "batch": batch, "seq": seq, "hidden": hidden, "vocab": vocab,
                "prompt": rng.choice([0.0, 0.2, 0.4]), "empty": rng.choice([0, 0, 1]) if batch > 1 else 0,
                "tau": rng.choice([1.0, 0.7, 1.3])}
    tokens, seq = _log_int(rng, 64, 512 * 8192 // (4 if op == "preference" else 1)), _log_int(rng, 8, 16384)
    if op == "preference":
        batch = 2 * max(1, tokens // (2 * seq))
        return {"op": op, "batch": batch, "seq": seq, "prompt": rng.choice([0.1, 0.3]),
                "empty": rng.choice([0, 1]) if batch > 2 else 0, "kind": rng.choice(["sigmoid", "sigmoid", "hinge", "ipo"]),
                "beta": rng.choice([0.05, 0.1, 0.5]), "smooth": rng.choice([0.0, 0.1]),
                "average": rng.choice([False, True]), "ref": rng.choice([True, True, False])}
    batch = max(1, tokens // seq)
    return {"op": op, "batch": batch, "seq": seq, "prompt": rng.choice([0.1, 0.3]),
            "empty": rng.choice([0, 1]) if batch > 1 else 0, "clip_low": 0.2, "clip_high": rng.choice([0.2, 0.28]),
            "kl_coef": rng.choice([0.0, 0.04]), "per_token": rng.choice([False, True]),
            "reduction": rng.choice(["token", "sequence"])}


def draw(rng):
    while True:
        case = _draw(rng)
        if 3072 not in (case["batch"] * case["seq"], case["seq"], case.get("hidden"), case.get("vocab")):
            return case


# ------------------------------------------------------------------ inputs
def _spans(case):
    """[first, last) token of every sequence's answer: by the case alone, so that every seed has as many."""
    B, S = case["batch"], case["seq"]
    groups = B // 2 if case["op"] == "preference" else B  # the two answers of a pair share their prompt
    out = []
    for b in range(B):
        g = b % groups
        first = min(S, int(S * case["prompt"] * (0.5 + math.modf(0.618034 * (g + 1))[0])))
        last = S - int(0.3 * S * case["prompt"] * math.modf(0.754878 * (b + 1))[0])
        out.append((first, first) if g >= groups - case["empty"] else (first, max(first, last)))
    return out


def _answered(case):
    return sum(b - a for a, b in _spans(case))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, S = case["batch"], case["seq"]
    T = B * S
    rand = lambda *n: torch.rand(*n, generator=g, device="cuda")  # noqa: E731
    randn = lambda *n: torch.randn(*n, generator=g, device="cuda")  # noqa: E731
    spans = torch.tensor(_spans(case), device="cuda")
    pos = torch.arange(S, device="cuda")
    valid = ((pos >= spans[:, :1]) & (pos < spans[:, 1:])).reshape(T)
    s = {"case": case}
    if case["op"] in ("logprob", "logprob_grad"):
        H, V = case["hidden"], case["vocab"]
        ids = torch.randint(0, V, (T,), generator=g, device="cuda")
        w = torch.randn(V, H, generator=g, device="cuda", dtype=torch.bfloat16).mul_(2 / math.sqrt(H))
        # hidden states of a trained model: of unit size, and leaning towards the next token by an amount that
        # runs from none to enough to make it the likeliest of all
        x = randn(T, H)
        x.addcmul_(w[ids].float(), 3 * rand(T, 1))
        s.update(x=x.bfloat16(), w=w, targets=torch.where(valid, ids, IGNORE))
        if case["op"] == "logprob_grad":
            s["dlogp"] = torch.where(valid, randn(T) / max(1, _answered(case)), 0.0)
            s["lse"] = torch.where(valid, torch.cat([_plain_lse(c, w, case["tau"]) for c in s["x"].split(1024)]), 0.0)
            s["dx"], s["dw"] = torch.empty_like(s["x"]), torch.empty_like(w)
        return s
    ids = torch.randint(0, VOCAB, (T,), generator=g, device="cuda")
    s["targets"] = torch.where(valid, ids, IGNORE)
    sampled = 2.0 * rand(T).clamp_(min=1e-6).log_()  # log-probabilities of sampled tokens, 0 to about -28
    near = lambda by: torch.where(valid, sampled + by * randn(T), 0.0)  # noqa: E731
    s["logp"] = near(0.15)
    if case["op"] == "preference":
        s["ref"] = near(0.05) if case["ref"] else None
    else:
        s["old"], s["ref"] = near(0.05), near(0.15) if case["kl_coef"] else None
        s["advantages"] = 0.25 + randn(T if case["per_token"] else B)
    return s


# -------------------------------------------------------------- plain forms
def _plain_lse(x, w, tau):
    l = (x.float() @ w.float().t()) / tau
    m = l.max(dim=1, keepdim=True).values
    return m[:, 0] + (l - m).exp_().sum(dim=1).log()


def _plain_logprob(s):
    c, t = s["case"], s["targets"]
    valid = t != IGNORE
    l = (s["x"].float() @ s["w"].float().t()) / c["tau"]
    picked = l.gather(1, t.clamp(min=0)[:, None])[:, 0]
    m = l.max(dim=1, keepdim=True).values
    log_sum = (l - m).exp_().sum(dim=1).log()
    zero = torch.zeros_like(log_sum)
    return {"logp": torch.where(valid, (picked - m[:, 0]) - log_sum, zero), "lse": torch.where(valid, m[:, 0] + log_sum, zero)}


def _plain_logprob_grad(s):
    c, t, x, w = s["case"], s["targets"], s["x"].float(), s["w"].float()
    valid = t != IGNORE
    d = (x @ w.t()).div_(c["tau"]).sub_(s["lse"][:, None]).exp_().neg_()
    d.scatter_add_(1, t.clamp(min=0)[:, None], torch.ones_like(d[:, :1]))
    d.mul_(torch.where(valid, s["dlogp"] / c["tau"], torch.zeros_like(s["dlogp"]))[:, None])
    return {"dx": (d @ w).to(s["x"].dtype), "dw": (d.t() @ x).to(s["w"].dtype)}


def _plain_preference(s):
    c = s["case"]
    B, S, P, beta, eps = c["batch"], c["seq"], c["batch"] // 2, c["beta"], c["smooth"]
    valid = (s["targets"] != IGNORE).view(B, S)
    ratio = s["logp"] if s["ref"] is None else s["logp"] - s["ref"]
    r = torch.where(valid, ratio.view(B, S), 0.0).sum(dim=1)
    n = valid.sum(dim=1)
    per = torch.ones_like(r)
    if c["average"]:
        per = 1.0 / n.clamp(min=1).float()
        r = r * per
    m = r[:P] - r[P:]
    live = (n[:P] + n[P:]) > 0  # pairs of padding are no pairs
    z = beta * m
    if c["kind"] == "sigmoid":
        tail = torch.log1p(torch.exp(-z.abs()))
        loss = (1 - eps) * ((-z).clamp(min=0) + tail) + eps * (z.clamp(min=0) + tail)
        dm = beta * (eps / (1 + torch.exp(-z)) - (1 - eps) / (1 + torch.exp(z)))
    elif c["kind"] == "hinge":
        loss, dm = (1 - z).clamp(min=0), torch.where(z < 1, -beta, 0.0)
    else:
        loss, dm = (m - 0.5 / beta) ** 2, 2 * (m - 0.5 / beta)
    pairs = live.sum().clamp(min=1).float()
    dm = torch.where(live, dm, 0.0) / pairs
    d = torch.cat([dm, -dm]) * per
    return {"loss": torch.where(live, loss, 0.0).sum() / pairs,
            "dlogp": torch.where(valid, d[:, None], 0.0).reshape(B * S), "rewards": beta * r}


def _plain_policy(s):
    c = s["case"]
    B, S = c["batch"], c["seq"]
    valid = (s["targets"] != IGNORE).view(B, S)
    a = s["advantages"].view(B, S if c["per_token"] else 1)
    d = (s["logp"] - s["old"]).view(B, S)
    rho = torch.exp(d)
    # outside the trust region on the side that the advantage pushes to: the loss is flat there
    over, under = d > math.log1p(c["clip_high"]), d < math.log1p(-c["clip_low"])
    clipped = ((a > 0) & over) | ((a < 0) & under)
    edge = torch.where(over, 1 + c["clip_high"], 1 - c["clip_low"])
    loss = -a * torch.where(clipped, edge, rho)
    grad = torch.where(clipped, 0.0, -a * rho)
    kl = torch.zeros_like(d)
    if s["ref"] is not None:
        e = (s["ref"] - s["logp"]).view(B, S)
        kl = torch.expm1(e) - e
        loss = loss + c["kl_coef"] * kl
        grad = grad - c["kl_coef"] * torch.expm1(e)
    n = valid.sum(dim=1)
    tokens = n.sum().clamp(min=1).float()
    if c["reduction"] == "token":
        weight = (1 / tokens).expand(B)
    else:
        weight = 1 / (n.clamp(min=1).float() * (n > 0).sum().clamp(min=1).float())
    loss = (torch.where(valid, loss, 0.0).sum(dim=1) * weight).sum()
    stats = torch.stack([torch.where(valid, kl, 0.0).sum(), (clipped & valid).sum().float()]) / tokens
    return {"loss": loss, "dlogp": torch.where(valid, grad * weight[:, None], 0.0).reshape(B * S), "stats": stats}


def run(s):
    c = s["case"]
    if not own:
        return {"logprob": _plain_logprob, "logprob_grad": _plain_logprob_grad, "preference": _plain_preference,
                "policy": _plain_policy}[c["op"]](s)
    from test1_b200 import ops

    if c["op"] == "logprob":
        logp, lse = ops.linear_logprob_fwd(s["x"], s["w"], s["targets"], temperature=c["tau"])
        return {"logp": logp, "lse": lse}
    if c["op"] == "logprob_grad":
        ops.linear_logprob_bwd(s["dlogp"], s["x"], s["w"], s["targets"], s["lse"], s["dx"], s["dw"], temperature=c["tau"])
        return {"dx": s["dx"], "dw": s["dw"]}
    if c["op"] == "preference":
        loss, dlogp, rewards = ops.preference_loss_fwd_bwd(s["logp"], s["ref"], s["targets"], c["seq"], beta=c["beta"],
                                                           kind=c["kind"], label_smoothing=c["smooth"], average=c["average"])
        return {"loss": loss, "dlogp": dlogp, "rewards": rewards}
    loss, dlogp, stats = ops.policy_loss_fwd_bwd(s["logp"], s["old"], s["ref"], s["advantages"], s["targets"], c["seq"],
                                                 clip_low=c["clip_low"], clip_high=c["clip_high"], kl_coef=c["kl_coef"],
                                                 reduction=c["reduction"])
    return {"loss": loss, "dlogp": dlogp, "stats": stats}


# -------------------------------------------------------------------- work
def work(case):
    T, n = case["batch"] * case["seq"], _answered(case)
    if case["op"] in ("logprob", "logprob_grad"):
        H, V = case["hidden"], case["vocab"]
        if case["op"] == "logprob":
            return {"bytes": 2 * H * (n + V) + 8 * T + 8 * T, "flops": 2 * n * V * H + 4 * n * V}
        # the logits again, then the two products with them
        return {"bytes": 2 * H * (n + V) + (8 + 8) * T + 2 * H * (T + V), "flops": 6 * n * V * H + 5 * n * V}
    if case["op"] == "preference":
        return {"bytes": 8 * T + (8 if case["ref"] else 4) * n + 4 * T + 4 * case["batch"], "flops": 4 * n}
    reads = 8 + (4 if case["kl_coef"] else 0) + (4 if case["per_token"] else 0)
    return {"bytes": 8 * T + reads * n + 4 * T + (0 if case["per_token"] else 4 * case["batch"]), "flops": 24 * n}


# ----------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    t, T = s["targets"], case["batch"] * case["seq"]
    rows = (t != IGNORE).nonzero()[:, 0]
    if case["op"] in ("logprob", "logprob_grad"):
        w = s["w"].double().requires_grad_(case["op"] == "logprob_grad")
        if case["op"] == "logprob":
            logp, lse = torch.zeros(2, T, dtype=torch.float64, device="cuda")
            for part in rows.split(1024):
                l = s["x"][part].double() @ w.t() / case["tau"]
                lse[part] = torch.logsumexp(l, dim=1)
                logp[part] = torch.log_softmax(l, dim=1)[torch.arange(len(part), device="cuda"), t[part]]
            return {"logp": logp, "lse": lse}
        dx = torch.zeros(T, case["hidden"], dtype=torch.float64, device="cuda")
        w.grad = torch.zeros_like(w)
        for part in rows.split(1024):
            x = s["x"][part].double().requires_grad_()
            nll = torch.nn.functional.cross_entropy(x @ w.t() / case["tau"], t[part], reduction="none")
            (-nll * s["dlogp"][part].double()).sum().backward()
            dx[part] = x.grad
        return {"dx": dx, "dw": w.grad}
    logp = s["logp"].double().requires_grad_()
    seq = torch.arange(T, device="cuda") // case["seq"]  # the sequence of every token
    n = torch.zeros(case["batch"], dtype=torch.float64, device="cuda").index_add_(0, seq[rows], torch.ones_like(rows, dtype=torch.float64))
    total = lambda v: torch.zeros_like(n).index_add(0, seq[rows], v)  # noqa: E731
    if case["op"] == "preference":
        r = logp[rows] if s["ref"] is None else logp[rows] - s["ref"].double()[rows]
        r = total(r) / n.clamp(min=1) if case["average"] else total(r)
        chosen, rejected = r.chunk(2)
        keep = (sum(n.chunk(2)) > 0).nonzero()[:, 0]
        m = (chosen - rejected)[keep]
        if case["kind"] == "sigmoid":
            log_sig = torch.nn.functional.logsigmoid
            loss = -(1 - case["smooth"]) * log_sig(case["beta"] * m) - case["smooth"] * log_sig(-case["beta"] * m)
        elif case["kind"] == "hinge":
            loss = torch.relu(1 - case["beta"] * m)
        else:
            loss = (m - 1 / (2 * case["beta"])).square()
        loss = loss.sum() / max(1, len(keep))
        loss.backward()
        return {"loss": loss.detach(), "dlogp": logp.grad, "rewards": (case["beta"] * r).detach()}
    a = s["advantages"].double()
    a = a[rows] if case["per_token"] else a[seq[rows]]
    rho = torch.exp(logp[rows] - s["old"].double()[rows])
    kept = rho.clamp(1 - case["clip_low"], 1 + case["clip_high"])
    loss, kl = -torch.minimum(a * rho, a * kept), torch.zeros_like(rho)
    if s["ref"] is not None:
        e = s["ref"].double()[rows] - logp[rows]
        kl = torch.expm1(e) - e
        loss = loss + case["kl_coef"] * kl
    if case["reduction"] == "token":
        loss = loss.sum() / max(1, len(rows))
    else:
        loss = (total(loss) / n.clamp(min=1)).sum() / (n > 0).sum().clamp(min=1)
    loss.backward()
    stats = torch.stack([kl.sum(), (a * kept < a * rho).double().sum()]).detach() / max(1, len(rows))
    return {"loss": loss.detach(), "dlogp": logp.grad, "stats": stats}
