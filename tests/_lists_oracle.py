"""64-bit statements of the operators on rows of logits and lists of tokens,
written from their definitions."""
import math

import torch


def _row(z, tau):
    """The row's tokens (indices), their log-probabilities and their order."""
    z = z.double()
    at = (z > -math.inf).nonzero()[:, 0]  # not NaN either
    z = z[at]
    order = torch.sort(z, descending=True, stable=True).indices
    if bool((z == math.inf).any()):
        z = torch.where(z == math.inf, 0.0, -math.inf).double()
        logp = torch.where(z == 0, -math.log(int((z == 0).sum())), -math.inf)
    else:
        logp = torch.log_softmax((z - z.max()) / tau, 0) if len(at) else z
    return at, logp, order


def topk(logits, k, tau):
    ids = torch.full((logits.shape[0], k), -1)
    out = torch.zeros(logits.shape[0], k, dtype=torch.float64)
    for r, z in enumerate(logits.cpu()):
        at, logp, order = _row(z, tau)
        best = order[:k]
        ids[r, :len(best)], out[r, :len(best)] = at[best], logp[best]
    return out, ids


def sample(logits, u, tau, top_k, top_p, min_p):
    tokens, out = [], []
    for z, x in zip(logits.cpu(), u.cpu().double()):
        at, logp, order = _row(z, tau)
        if not len(at):
            tokens.append(-1)
            out.append(0.0)
            continue
        if top_k:
            order = order[:top_k]
        p = torch.exp(logp[order] - logp[order[0]])
        if top_p < 1:
            order = order[p.cumsum(0) - p < top_p * p.sum()]
            p = torch.exp(logp[order] - logp[order[0]])
        order = order[p >= min_p].sort().values
        # Relative to the likeliest, so that equal weights are 1 and their sums exact: half of 2000 such is reached with
        # token 1001, where 2000 times a rounded 1 / 4001, added up one by one, may pass half of their sum with token 1000.
        p = torch.exp(logp[order] - logp.max())
        cdf = p.cumsum(0)
        x = min(max(float(x), 0.0), 1 - 2.0 ** -53) if x == x else 0.0
        hit = order[int((cdf <= x * cdf[-1]).sum())]
        tokens.append(int(at[hit]))
        out.append(float(logp[hit]))
    return torch.tensor(tokens), torch.tensor(out, dtype=torch.float64)


def listed_logprob(x, w, ids, tau, dlogp=None):
    """(logp, lse) and, with dlogp, (dx, dw)."""
    T, K = ids.shape
    V = w.shape[0]
    logp = torch.zeros(T, K, dtype=torch.float64, device=x.device)
    lse = torch.zeros(T, dtype=torch.float64, device=x.device)
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    wd = w.double()
    dw = torch.zeros_like(wd)
    keep = (ids >= 0) & (ids < V)
    for part in keep.any(1).nonzero()[:, 0].split(512):
        xd = x[part].double()
        l = xd @ wd.t() / tau
        lp = torch.log_softmax(l, 1)
        lse[part] = torch.logsumexp(l, 1)
        r, k = keep[part].nonzero(as_tuple=True)
        at = ids[part][r, k]
        logp[part[r], k] = lp[r, at]
        if dlogp is not None:
            up = torch.zeros_like(l).index_put_((r, at), dlogp[part][r, k].double(), accumulate=True)
            d = (up - lp.exp() * up.sum(1, keepdim=True)) / tau
            dx[part] = d @ wd
            dw += d.t() @ xd
    return logp, lse, dx, dw


def distillation(logp, teacher, ids, kind, tail, floor=2.0 ** -20):
    """(loss, dlogp, divergence, size): by autograd, row by row; size [T] is
    what roundings are relative to, (p + q) (|log p| + |log q| + 1) summed."""
    T = logp.shape[0]
    lp = logp.double().requires_grad_()
    keep = (ids >= 0) & (teacher.double() > -math.inf)
    each, size, live = [], [], 0
    for t in range(T):
        k = keep[t].nonzero()[:, 0]
        if not len(k):
            each.append(lp[t].new_zeros(()))
            size.append(0.0)
            continue
        live += 1
        a, b = lp[t, k], teacher[t, k].double()
        if tail:
            rest = lambda v: torch.log((1 - v.exp().sum()).clamp(min=floor)).reshape(1)  # noqa: E731
            a, b = torch.cat([a, rest(a)]), torch.cat([b, rest(b)])
        else:
            a, b = torch.log_softmax(a, 0), torch.log_softmax(b, 0)
        p, q = a.exp(), b.exp()
        if kind == "forward":
            f = q * (b - a)
        elif kind == "reverse":
            f = p * (a - b)
        else:
            m = torch.log((p + q) / 2)
            f = (p * (a - m) + q * (b - m)) / 2
        each.append(f.sum())
        size.append(float(((p + q) * (a.abs() + b.abs() + 1)).sum().detach()))
    each = torch.stack(each) if T else lp.sum(1)
    loss = each.sum() / max(1, live)
    if live:
        loss.backward()
    grad = torch.zeros_like(lp) if lp.grad is None else lp.grad
    return loss.detach(), grad, each.detach(), torch.tensor(size, dtype=torch.float64)
