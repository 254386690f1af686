"""Drawing from a given number as its definition says it, in extended precision, one row at a time."""
import numpy as np


def kept_and_mass(row, t, k, p, m):
    """ids that are kept, ascending, and their masses (the largest logit's is 1)."""
    x = np.asarray(row, dtype=np.float64)
    w = np.exp((x.astype(np.longdouble) - x.max()) / np.longdouble(t))
    w[x == -np.inf] = 0
    keep = np.ones(x.size, dtype=bool)
    order = np.argsort(-x, kind="stable")
    if 0 < k < x.size:
        keep &= x >= x[order[k - 1]]
    if p < 1:
        total, larger, i = w[keep].sum(), np.longdouble(0), 0
        while i < x.size and keep[order[i]]:
            j = i
            while j < x.size and x[order[j]] == x[order[i]]:
                j += 1
            if larger > max(p, 0.0) * total and i > 0:
                keep[order[i:]] = False
                break
            larger += w[order[i:j]].sum()
            i = j
    if m > 0:
        keep &= w >= min(m, 1.0)
    ids = np.nonzero(keep)[0]
    return ids, w[ids]


def oracle(row, u, t, k, p, m):
    """-> token, log-probability, distance of u from the token's borders (a share of the mass)."""
    x = np.asarray(row, dtype=np.float64)
    if not t > 0:
        w = np.exp(x.astype(np.longdouble) - x.max())
        return int(x.argmax()), float(-np.log(w.sum())), 1.0
    ids, w = kept_and_mass(row, max(t, float(np.float32(1e-8))), k, p, m)
    sums = np.cumsum(w)
    target = np.longdouble(u) * sums[-1]
    hit = np.nonzero((sums > target) & (w > 0))[0]
    i = hit[0] if hit.size else np.nonzero(w > 0)[0][-1]
    near = abs(np.concatenate([[np.longdouble(0)], sums]) - target)
    near = near[near > 0].min() if u == 0 else near.min()
    return int(ids[i]), float(np.log(w[i] / sums[-1])), float(near / sums[-1])
