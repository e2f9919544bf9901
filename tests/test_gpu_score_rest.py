"""Distillation with the rest as one outcome, where the student's unlisted
probability is far below the listed one's or the other way round: the outcome
is left out only when every unlisted id is masked, by -inf or a finite value
that leaves it no probability in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from row_reference import rel_err_bound  # noqa: E402
from snai_b200 import distill_device  # noqa: E402
from test_gpu_score import DEV, DT, LOWEST, check_grad, in_f32, on_gpu  # noqa: E402


def log_sum(x):
    m = x.max() if x.size else -np.inf
    return m if m == -np.inf else m + np.log(np.exp(x - m).sum())


def rest_row(z, ids, vals, label, T, a):
    """(loss, gradient, magnitudes of the gradient's and the loss's terms) in
    64 bits, the unlisted mass by its logarithm.  Ids are distinct."""
    V = len(z)
    on = np.zeros(V, dtype=bool)
    on[ids] = True
    # logits go first less their maximum: the lowest values of a type keep their differences
    top = z.max()
    d = (z - top) / T
    lp = d - log_sum(d)
    mu = z[~on].max() if (~on).any() else -np.inf
    q = np.exp(vals.astype(np.float64))
    with np.errstate(invalid="ignore"):
        loss = np.where(q > 0, q * (vals - lp[ids]), 0.0).sum()
        lmag = np.where(q > 0, q * (np.abs(vals) + np.abs(lp[ids])), 0.0).sum()
    target = np.zeros(V)
    target[ids] = q
    back, r = np.zeros(V), 0.0
    if mu > -np.inf:
        du = np.where(on, -np.inf, (z - mu) / T)
        su = np.exp(du).sum()
        log_u = (mu - top) / T + np.log(su) - log_sum(d)
        r = max(0.0, 1.0 - q.sum()) if log_u > -745.0 else 0.0
        back = r * np.exp(du) / su
        if r > 0:
            loss += r * (np.log(r) - log_u)
            lmag += r * (abs(np.log(r)) + abs(log_u))
    p = np.exp(lp)
    c = (1.0 - a) * T
    mass = q.sum() + r
    grad, mag = c * (mass * p - target - back), c * (mass * p + target + back)
    loss, lmag = c * T * loss, c * T * lmag
    if a > 0 and 0 <= label < V:
        l1 = (z - top) - log_sum(z - top)
        loss -= a * l1[label]
        lmag += a * abs(l1[label])
        grad, mag = grad + a * np.exp(l1), mag + a * np.exp(l1)
        grad[label] -= a
        mag[label] += a
    keep = z != -np.inf
    return loss, np.where(keep, grad, 0.0), np.where(keep, mag, 0.0), lmag, r


# by how many temperatures the best listed logit is above the best unlisted one; e^-87.3 is fp32's least normal number
GAPS = [0, 3, 24, 60, 80, 85, 86, 87, 87.5, 88, 90, 95, 100, 103, 104, 110, 200, 500, 700, 800, 1000, 5000, -3, -60, -86, -88, -100,
        -300]


def rows_with_gaps(rng, V, k, dtype, T, masked, few):
    R = len(GAPS)
    z = rng.normal(0, 1, (R, V)) * min(T, 1.0)
    ids = np.stack([rng.choice(V, k, replace=False) for _ in range(R)])
    for r, gap in enumerate(GAPS):
        on = np.zeros(V, dtype=bool)
        on[ids[r]] = True
        if few:  # a few unlisted ids are left, the others masked
            off = np.flatnonzero(~on)
            z[r, rng.permutation(off)[few:]] = -np.inf
        elif masked:
            z[r, ~on & (rng.random(V) < masked)] = -np.inf
        z[r, on] += z[r, ~on].max() + gap * T - z[r, on].max()
    z = torch.from_numpy(z.astype(np.float32)).to(DT[dtype]).double().numpy()
    q = rng.random((R, k))
    q *= rng.uniform(0.5, 0.95, (R, 1)) / q.sum(1, keepdims=True)
    return z, ids.astype(np.int32), np.log(q).astype(np.float32)


def compare(z, dtype, ids, vals, y, T, a, rg, pad=0, shift=0):
    R = len(z)
    it, vt, rt = (torch.from_numpy(x).to(DEV) for x in (ids, vals, rg))
    yt = None if y is None else torch.from_numpy(y).to(DEV)
    t = on_gpu(z, dtype, pad, shift)
    loss, grad = distill_device(t, it, vt, yt, T, a, True, rt)
    alone, _ = distill_device(t, it, vt, yt, T, a, True, want_grad=False)
    want = [rest_row(z[r], ids[r], vals[r], -1 if y is None else y[r], T, a) for r in range(R)]
    for got in (loss, alone):
        g = got.double().cpu().numpy()
        for r in range(R):
            w, lmag = float(in_f32(want[r][0])), want[r][3]
            if not np.isfinite(w):
                assert w == g[r], (r, w, g[r])
                continue
            # as in test_gpu_score.test_distill: every log is off by the sums' relative error, and with T's half a
            # step by that of the difference of logits in it, which lmag counts
            tol = rel_err_bound(z[r], min(T, 1.0))
            assert abs(g[r] - w) <= tol * (2 * max(T * T, 1.0) + lmag), (r, g[r], w, tol)
            if a == 0.0 and want[r][4] > 0:  # a divergence is not negative
                assert g[r] >= -tol * (2 * max(T * T, 1.0) + lmag)
    s = np.abs(rg.astype(np.float64))[:, None]
    check_grad(grad, np.stack([w[1] for w in want]) * rg[:, None].astype(np.float64),
               np.stack([w[2] for w in want]) * s, z, min(T, 1.0), dtype)


@pytest.mark.parametrize("V,k,dtype,T,a,masked,few", [
    (1000, 8, "fp32", 1.0, 0.0, 0.0, 0),
    (1000, 8, "fp32", 1.0, 0.5, 0.3, 0),
    (1000, 64, "fp32", 0.3, 0.0, 0.3, 0),
    (1000, 64, "fp32", 0.3, 0.5, 0.0, 0),
    (1001, 33, "fp32", 2.0, 0.5, 0.5, 0),
    (1001, 33, "fp32", 4.0, 0.5, 0.0, 0),
    (1000, 16, "fp32", 1.0, 0.0, 0.0, 1),
    (1000, 16, "fp32", 0.5, 0.5, 0.0, 3),
    (700, 300, "fp32", 3.0, 0.25, 0.0, 2),
    (4099, 20, "bf16", 1.0, 0.5, 0.1, 0),
    (4099, 512, "fp16", 2.0, 0.0, 0.0, 5),
    (16384, 128, "fp32", 0.3, 0.5, 0.0, 0),
    (50001, 64, "bf16", 0.7, 0.0, 0.9, 0),
    (131072, 20, "fp32", 1.5, 0.5, 0.0, 2),
], ids=str)
def test_rest_across_gaps(built, V, k, dtype, T, a, masked, few):
    rng = np.random.default_rng(V * 3 + k)
    z, ids, vals = rows_with_gaps(rng, V, k, dtype, T, masked, few)
    R = len(z)
    y = None
    if a:
        y = ids[:, 0].copy()  # on the list, off it, none
        for r in range(1, R, 3):
            on = np.isfinite(z[r])
            on[ids[r]] = False
            y[r] = rng.choice(np.flatnonzero(on))
        y[2::6] = -1
    compare(z, dtype, ids, vals, y, T, a, rng.normal(0, 1, R).astype(np.float32), pad=3 if V % 2 else 0, shift=V % 2)


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T", [0.3, 1.0, 2.0])
def test_rest_of_finite_masks(built, dtype, T):
    """Masks of a type's lowest value, of -1e4 or of -200 on all unlisted ids, on all but one, and on all listed ones."""
    V, k = 3001, 12
    rng = np.random.default_rng(7)
    rows, ids = [], []
    for low in (LOWEST[dtype], -1e4, -200.0):
        for which in range(3):
            i = rng.choice(V, k, replace=False)
            on = np.zeros(V, dtype=bool)
            on[i] = True
            x = rng.normal(0, 1, V)
            x[on if which == 2 else ~on] = low
            if which == 1:
                x[np.flatnonzero(~on)[5]] = 0.25
            rows.append(x)
            ids.append(i)
    z = torch.from_numpy(np.stack(rows).astype(np.float32)).to(DT[dtype]).double().numpy()
    vals = np.log(np.full((len(z), k), 0.9 / k)).astype(np.float32)
    compare(z, dtype, np.stack(ids).astype(np.int32), vals, None, T, 0.0, np.ones(len(z), dtype=np.float32))
    y = np.array([i[3] for i in ids], dtype=np.int32)
    compare(z, dtype, np.stack(ids).astype(np.int32), vals, y, T, 0.5, np.ones(len(z), dtype=np.float32))


def test_rest_with_every_unlisted_id_masked(built):
    """The outcome is left out; masked logits take no gradient."""
    V, k = 1000, 16
    rng = np.random.default_rng(9)
    z, ids, vals = rows_with_gaps(rng, V, k, "fp32", 1.0, 0.0, 1)
    for r in range(len(z)):
        on = np.zeros(V, dtype=bool)
        on[ids[r]] = True
        z[r, ~on] = -np.inf
    compare(z, "fp32", ids, vals, None, 1.0, 0.0, np.ones(len(z), dtype=np.float32))


@pytest.mark.parametrize("left", [1e-6, 1e-8, 1e-9])
def test_rest_that_a_list_nearly_fills(built, left):
    """What the list leaves of 1 is a difference of 64-bit numbers, and so are
    the gradients of the few unlisted ids: -r p_i / u for the greater part."""
    V, k, R = 320, 300, 6
    rng = np.random.default_rng(int(-np.log10(left)))
    z = rng.normal(0, 1, (R, V)).astype(np.float32).astype(np.float64)
    ids = np.stack([rng.choice(V, k, replace=False) for _ in range(R)]).astype(np.int32)
    for r in range(R):  # unlisted ids of little probability: the rest's term is not lost beside their own
        on = np.zeros(V, dtype=bool)
        on[ids[r]] = True
        z[r, ~on] -= 40.0
    z = z.astype(np.float32).astype(np.float64)
    q = rng.dirichlet(np.ones(k), R)
    q[:, 0] = 0.7  # an exponential in the middle between two powers of 2, where it is hardest
    q[:, 1:] *= 0.3 / q[:, 1:].sum(1, keepdims=True)
    vals = np.log(q * (1 - left)).astype(np.float32)
    for r in range(R):  # the float32 values' own sum is off by more than `left`: some take it up
        for _ in range(60):
            s = np.exp(vals[r].astype(np.float64)).sum()
            j = int(np.argsort(-vals[r])[1 + _ % 30])
            vals[r, j] = np.log(max(np.exp(float(vals[r, j])) + (1 - left - s), 1e-12))
    rest = np.array([1 - np.exp(v.astype(np.float64)).sum() for v in vals])
    keep = rest > left / 4
    assert keep.sum() >= 2, rest
    z, ids, vals, rest = z[keep], ids[keep], vals[keep], rest[keep]
    _, grad = distill_device(on_gpu(z, "fp32"), torch.from_numpy(ids).to(DEV), torch.from_numpy(vals).to(DEV), rest=True)
    got = grad.double().cpu().numpy()
    for r in range(len(z)):
        want = rest_row(z[r], ids[r], vals[r], -1, 1.0, 0.0)[1]
        off = np.ones(V, dtype=bool)
        off[ids[r]] = False
        # r: 64-bit values, each to 1e-11 of itself, that make 1 in all; its share p_i / u: rel_err_bound
        tol = (1e-11 / rest[r] + 2 * rel_err_bound(z[r], 1.0)) * np.abs(want[off])
        assert (np.abs(got[r][off] - want[off]) <= tol).all(), (r, rest[r], got[r][off][:4], want[off][:4])
