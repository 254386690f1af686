"""The distillation loss and its gradient from their formulas in 64 bits, entry by entry."""
import math

import torch


def oracle(x, ids, values, rest, tau, target=None, hard=0.0, ignore=-100, upstream=1.0):
    """-> loss, dx, and what their errors are relative to: (sum of the terms' magnitudes of each)."""
    x = x.detach().double().cpu()
    rows, V = x.shape
    values, ids = values.detach().double().cpu(), ids.long().cpu()
    counted = torch.ones(rows, dtype=torch.bool)
    if target is not None:
        target = target.long().cpu()
        counted = (target != ignore) & (target >= 0) & (target < V)
    n = max(1, int(counted.sum()))
    loss = size = 0.0
    dx, dsize = torch.zeros_like(x), torch.zeros_like(x)
    for r in range(rows):
        if not counted[r]:
            continue
        z = x[r] / tau
        q = torch.softmax(z, -1)
        logz = torch.logsumexp(z, -1)
        entries = [(int(j), float(t) / tau) for j, t in zip(ids[r], values[r]) if 0 <= j < V]
        members = sorted({j for j, _ in entries})
        outside = torch.ones(V, dtype=torch.bool)
        outside[members] = False
        t = [v for _, v in entries] + ([float(rest[r])] if rest is not None else [])
        t = torch.tensor(t, dtype=torch.float64)
        kl = kl_size = 0.0
        grad, grad_size = torch.zeros_like(q), torch.zeros_like(q)
        if t.numel() and t.max() > -math.inf:
            logp = torch.log_softmax(t, -1)
            p = logp.exp()
            grad, grad_size = q.clone(), q.clone()
            logq = [float(z[j] - logz) for j, _ in entries]
            if rest is not None:
                logq.append(float(torch.logsumexp(z[outside], -1) - logz) if outside.any() else -math.inf)
            for i, lq in enumerate(logq):
                if p[i] == 0:
                    continue
                kl += float(p[i]) * (float(logp[i]) - lq)
                kl_size += float(p[i]) * (abs(float(logp[i])) + abs(lq) + 1)
                if i < len(entries):
                    grad[entries[i][0]] -= p[i]
                    grad_size[entries[i][0]] += p[i]
                elif outside.any():
                    share = torch.where(outside, torch.softmax(torch.where(outside, z, -math.inf), -1), 0.0)
                    grad -= p[i] * share
                    grad_size += p[i] * share
        kl, kl_size = (1 - hard) * tau ** 2 * kl, (1 - hard) * tau ** 2 * kl_size
        grad, grad_size = (1 - hard) * tau * grad, (1 - hard) * tau * grad_size
        if hard:
            y = int(target[r])
            q1 = torch.softmax(x[r], -1)
            ce = float(torch.logsumexp(x[r], -1) - x[r, y])
            kl += hard * ce
            kl_size += hard * (float(x[r].max() - x[r, y]) + 1 + abs(ce))
            grad = grad + hard * q1
            grad_size = grad_size + hard * q1
            grad[y] -= hard
            grad_size[y] += hard
        loss += kl / n
        size += kl_size / n
        dx[r] = upstream / n * grad
        dsize[r] = abs(upstream) / n * grad_size
    return loss, dx, size, dsize
