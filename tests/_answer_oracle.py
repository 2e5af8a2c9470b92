"""64-bit statements of the log-probability and loss operators, by autograd."""
import torch
import torch.nn.functional as F


def logprob(x, w, targets, vocab, ignore_index=-100, temperature=1.0, dlogp=None):
    """(logp, lse) and, with dlogp, (dx, dw), all fp64."""
    valid = (targets != ignore_index) & (targets >= 0) & (targets < vocab)
    rows = valid.nonzero()[:, 0]
    T = x.shape[0]
    logp = torch.zeros(T, dtype=torch.float64, device=x.device)
    lse, dx = logp.clone(), torch.zeros(T, x.shape[1], dtype=torch.float64, device=x.device)
    wd = w.double()
    dw = torch.zeros_like(wd)
    for part in rows.split(512):
        xd = x[part].double()
        l = xd @ wd.t() / temperature
        lp = F.log_softmax(l, dim=1)
        lse[part] = torch.logsumexp(l, dim=1)
        logp[part] = lp.gather(1, targets[part, None])[:, 0]
        if dlogp is not None:
            u = F.one_hot(targets[part], vocab) - lp.exp()
            u = u * (dlogp[part].double() / temperature)[:, None]
            dx[part] = u @ wd
            dw += u.t() @ xd
    return logp, lse, dx, dw


def preference(logp, ref, targets, S, beta, kind, smoothing, average, ignore_index=-100):
    lp = logp.double().requires_grad_()
    r = []
    for b in range(logp.shape[0] // S):
        at = (targets[b * S:(b + 1) * S] != ignore_index).nonzero()[:, 0] + b * S
        v = lp[at] - (ref[at].double() if ref is not None else 0.0)
        s = v.sum()
        r.append((s / max(1, len(at)) if average else s, len(at)))
    P = len(r) // 2
    losses = []
    for (c, nc), (j, nj) in zip(r[:P], r[P:]):
        if nc + nj == 0:
            continue
        m = c - j
        if kind == "sigmoid":
            losses.append(-(1 - smoothing) * F.logsigmoid(beta * m) - smoothing * F.logsigmoid(-beta * m))
        elif kind == "hinge":
            losses.append(F.relu(1 - beta * m))
        else:
            losses.append((m - 1 / (2 * beta)) ** 2)
    loss = sum(losses) / len(losses) if losses else lp[:0].sum()
    loss.backward()
    rewards = torch.stack([v for v, _ in r]).detach() * beta if r else lp.detach()[:0]
    return loss.detach(), lp.grad, rewards


def policy(logp, old, ref, adv, targets, S, lo, hi, kl_coef, reduction, ignore_index=-100):
    T = logp.shape[0]
    lp = logp.double().requires_grad_()
    at = (targets != ignore_index).nonzero()[:, 0]
    seq = at // S
    a = adv.double()[at] if adv.shape[0] == T and S != 1 else adv.double()[seq]
    rho = torch.exp(lp[at] - old[at].double())
    cut = rho.clamp(1 - lo, 1 + hi)
    l = -torch.minimum(a * rho, a * cut)
    kl = torch.zeros_like(rho)
    if ref is not None:
        e = ref[at].double() - lp[at]
        kl = torch.expm1(e) - e
        l = l + kl_coef * kl
    if reduction == "token":
        loss = l.sum() / max(1, len(at))
    else:
        n = torch.bincount(seq, minlength=T // S).clamp(min=1)
        loss = (l / n[seq]).sum() / max(1, len(seq.unique()))
    loss.backward()
    stats = torch.stack([kl.sum(), (a * cut < a * rho).double().sum()]).detach() / max(1, len(at))
    return loss.detach(), lp.grad, stats
