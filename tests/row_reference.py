"""The vocabulary-row operators (cortex_score, cortex_score_grad,
cortex_distill) in 64 bits, one row at a time, from their definitions in
include/cortex.h; and the error a float32 evaluation of them may make."""
import numpy as np

U32 = 2.0 ** -24  # half a step of float32, relative


def order(z):
    """Ids by descending logit, equal logits by ascending id."""
    return np.lexsort((np.arange(len(z)), -z))


def logp_row(z, T):
    """log p of a row; None when it holds a NaN or +inf (no distribution)."""
    z = np.asarray(z, dtype=np.float64)
    if np.isnan(z).any() or (z == np.inf).any():
        return None
    m = z.max()
    if m == -np.inf:
        return np.full(len(z), -np.inf)
    d = (z - m) / T
    return d - np.log(np.exp(d).sum())


def score_row(z, tokens, T, k):
    V = len(z)
    lp = logp_row(z, T)
    tok = np.asarray(tokens)
    if lp is None:
        return (np.where((tok < 0) | (tok >= V), 0.0, np.nan), np.nan, np.full(k, -1), np.full(k, np.nan))
    p = np.exp(lp)
    ent = -(p[p > 0] * lp[p > 0]).sum() if (p > 0).any() else 0.0
    ids = order(np.asarray(z, dtype=np.float64))[:k]
    at = np.array([0.0 if t < 0 or t >= V else lp[t] for t in tok])
    return at, ent, ids, lp[ids]


def score_grad_row(z, tokens, g, gh, T):
    """(gradient, sum of the magnitudes of its terms)."""
    z = np.asarray(z, dtype=np.float64)
    V = len(z)
    use = [(int(t), float(x)) for t, x in zip(tokens, g) if 0 <= t < V]
    if not use and gh == 0.0:
        return np.zeros(V), np.zeros(V)
    lp = logp_row(z, T)
    if lp is None:
        return np.full(V, np.nan), np.zeros(V)
    p = np.exp(lp)
    lpf = np.where(p > 0, lp, 0.0)
    ent = -(p * lpf).sum()
    out = -p * sum(x for _, x in use) - gh * p * (lpf + ent)
    mag = p * sum(abs(x) for _, x in use) + abs(gh) * p * (np.abs(lpf) + ent + 1.0)
    for t, x in use:
        out[t] += x
        mag[t] += abs(x)
    keep = z != -np.inf
    return np.where(keep, out, 0.0) / T, np.where(keep, mag, 0.0) / T


def distill_row(z, ids, vals, label, T, a, rest):
    """(loss, gradient of the loss, sum of its terms' magnitudes, sum of the loss's terms' magnitudes)."""
    z = np.asarray(z, dtype=np.float64)
    V = len(z)
    ids = np.asarray(ids)
    ok = (ids >= 0) & (ids < V)
    y = int(label) if a > 0 and 0 <= label < V else -1
    zero = np.zeros(V)
    if not ok.any() and y < 0:
        return 0.0, zero, zero, 0.0
    lp = logp_row(z, T)
    if lp is None:
        return np.nan, np.full(V, np.nan), zero, 0.0
    p = np.exp(lp)
    idx, t = ids[ok], np.asarray(vals, dtype=np.float64)[ok]
    q = np.zeros(len(idx))
    lq = np.full(len(idx), -np.inf)
    fin = t > -np.inf
    if fin.any():
        lq[fin] = t[fin] if rest else t[fin] / T - np.log(np.exp((t[fin] - t.max()) / T).sum()) - t.max() / T
        q[fin] = np.exp(lq[fin])
    pos = q > 0
    kl = (q[pos] * (lq[pos] - lp[idx[pos]])).sum()
    lmag = (q[pos] * (np.abs(lq[pos]) + np.abs(lp[idx[pos]]))).sum()
    target = np.zeros(V)
    np.add.at(target, idx, q)
    unlisted = np.ones(V, dtype=bool)
    unlisted[idx] = False
    back = np.zeros(V)
    if rest and len(idx):
        u = p[unlisted].sum()
        r = max(0.0, 1.0 - q.sum())
        if u > 0 and r > 0:
            kl += r * (np.log(r) - np.log(u))
            lmag += r * (abs(np.log(r)) + abs(np.log(u)))
            back[unlisted] = r * p[unlisted] / u
    mass = target.sum() + back.sum()
    c = (1.0 - a) * T
    grad = c * (mass * p - target - back)
    mag = c * (mass * p + target + back)
    loss = c * T * kl if a < 1.0 else 0.0
    lmag = c * T * lmag if a < 1.0 else 0.0
    if y >= 0:
        l1 = logp_row(z, 1.0)
        loss -= a * l1[y]
        lmag += a * abs(l1[y])
        grad = grad + a * np.exp(l1)
        mag = mag + a * np.exp(l1)
        grad[y] -= a
        mag[y] += a
    keep = z != -np.inf
    return loss, np.where(keep, grad, 0.0), np.where(keep, mag, 0.0), lmag


def rel_err_bound(z, T):
    """Relative error of exp(d_i) / S in float32, d = (z - max) / T: d carries
    three roundings (the difference, 1 / T, the product), the exponential and
    its argument in base 2 four more units, and S is a sum of nonnegative
    terms over at most 512 sequential and 16 pairwise additions of each
    term's own error.  log S and a row's other sums stay within it too."""
    z = np.asarray(z, dtype=np.float64)
    f = z[np.isfinite(z)]
    dmax = min((f.max() - f.min()) / T, 110.0) if f.size else 0.0  # exp is 0 below
    return U32 * (8.0 * dmax + 8.0 + 528.0)
