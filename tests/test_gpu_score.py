"""The vocabulary-row operators on the GPU (cortex_score, cortex_score_grad,
cortex_distill) against their definitions in 64 bits (row_reference.py), at
the sizes, alignments and masks where they can go wrong; then streams, graphs
and what lies around the arrays."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from row_reference import distill_row, order, rel_err_bound, score_grad_row, score_row  # noqa: E402
from snai_b200 import CortexError, distill_device, score_device, score_grad_device  # noqa: E402

DEV = torch.device("cuda")
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LOWEST = {"fp32": np.finfo(np.float32).min, "bf16": -3.3895313892515355e38, "fp16": -65504.0}
TINY = {"fp32": 2.0 ** -126, "bf16": 2.0 ** -126, "fp16": 2.0 ** -25}  # below: flushed or half a subnormal step


def rows_of(rng, R, V, dtype, mask="none", spread=3.0):
    """Logits as stored in dtype, as float64 [R, V]."""
    z = rng.normal(0, spread, (R, V))
    z[np.arange(R), rng.integers(0, V, R)] += 10.0
    low = LOWEST[dtype]
    for r in range(R):
        m = mask if mask != "mixed" else ["none", "tenth", "one", "empty", "lowest", "equal", "nan", "inf", "far",
                                          "halflow", "zeros"][r % 11]
        if m == "tenth":
            z[r, rng.random(V) < 0.1] = -np.inf
        elif m == "one":
            keep = rng.integers(0, V)
            z[r, np.arange(V) != keep] = -np.inf
        elif m == "empty":
            z[r] = -np.inf
        elif m == "lowest":
            z[r] = low
        elif m == "halflow":
            z[r, rng.random(V) < 0.5] = low
        elif m == "equal":
            z[r] = 1.25
        elif m == "nan":
            z[r, V // 2] = np.nan
        elif m == "inf":
            z[r, V // 3] = np.inf
        elif m == "far":
            z[r] *= 500.0
        elif m == "zeros":
            z[r] = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    t = torch.from_numpy(z.astype(np.float32)).to(DT[dtype])
    return t.double().numpy()


def on_gpu(z, dtype, pad=0, shift=0):
    """z in rows of V + pad elements, starting `shift` elements into its allocation."""
    R, V = z.shape
    flat = torch.full((shift + R * (V + pad) + 64,), 7.0, dtype=DT[dtype], device=DEV)
    t = flat[shift:shift + R * (V + pad)].view(R, V + pad)[:, :V]
    t.copy_(torch.from_numpy(z).to(DT[dtype]))
    return t


def in_f32(w):
    """Values past float32's range (log p of the lowest logits at T < 1) are infinite in it."""
    return np.where(np.abs(w) > np.finfo(np.float32).max, np.copysign(np.inf, w), w)


def check_score(z, dtype, tok, T, k, got):
    R, V = z.shape
    lp, ent = got.logprob.double().cpu().numpy().reshape(R, -1), got.entropy.double().cpu().numpy()
    ids = got.top_ids.cpu().numpy() if k else None
    top = got.top_logprob.double().cpu().numpy() if k else None
    for r in range(R):
        wl, we, wi, wt = score_row(z[r], tok[r], T, k)
        tol = rel_err_bound(z[r], T)
        # log p = d - log S: d's own relative error, and S's
        for w, g in ((wl, lp[r]),) + (((wt, top[r]),) if k else ()):
            w = in_f32(w)
            fin = np.isfinite(w)
            assert np.array_equal(np.isnan(w), np.isnan(g)) and np.array_equal(w == -np.inf, g == -np.inf), (r, w, g)
            assert (np.abs(g[fin] - w[fin]) <= tol + 8 * 2.0 ** -24 * np.abs(w[fin])).all(), (
                r, np.abs(g[fin] - w[fin]).max(), tol)
        if np.isnan(we):
            assert np.isnan(ent[r])
        else:  # sum p |log p| <= log V, each p off by tol
            assert abs(ent[r] - we) <= 2 * tol * (1.0 + np.log(V)), (r, ent[r], we)
        if k:
            assert np.array_equal(ids[r], wi), (r, ids[r][:8], wi[:8])


SIZES = [  # rows, vocab, dtype, pad, shift, temperature, top_k, tokens a row
    (1, 1, "fp32", 0, 0, 1.0, 1, 1),
    (3, 2, "bf16", 0, 0, 1.0, 2, 1),
    (4, 7, "fp32", 3, 1, 0.7, 7, 3),
    (1, 16384, "fp32", 0, 0, 1.0, 20, 1),
    (22, 1001, "fp32", 0, 0, 2.0, 64, 2),
    (22, 1001, "bf16", 1, 3, 1.0, 512, 1),
    (11, 4099, "fp16", 5, 1, 0.5, 33, 5),
    (11, 16384, "fp32", 8, 4, 1.0, 512, 512),
    (13, 16383, "bf16", 0, 0, 1.0, 17, 1),
    (12, 32000, "fp16", 0, 8, 1.3, 128, 1),
    (11, 50001, "fp32", 0, 0, 1.0, 1, 1),
    (11, 131072, "bf16", 0, 0, 1.0, 64, 1),
    (11, 131072, "fp32", 0, 0, 0.7, 20, 64),
    (2, 300001, "fp32", 2, 1, 1.0, 512, 1),
    (2, 524288, "fp32", 0, 0, 1.0, 40, 1),
    (2, 524287, "fp16", 1, 0, 1.0, 40, 1),
    (700, 300, "fp32", 0, 0, 1.0, 5, 1),
    (650, 2048, "bf16", 0, 0, 1.0, 0, 1),
    (330, 16384, "fp32", 0, 0, 1.0, 20, 1),
]


@pytest.mark.parametrize("R,V,dtype,pad,shift,T,k,n", SIZES, ids=str)
def test_score(built, R, V, dtype, pad, shift, T, k, n):
    rng = np.random.default_rng(R * 31 + V)
    z = rows_of(rng, R, V, dtype, "mixed")
    tok = rng.integers(0, V, (R, n)).astype(np.int32)
    tok[::3, 0] = np.nanargmax(np.where(np.isfinite(z[::3]), z[::3], -1e300), axis=1)
    tok[1::4, -1] = -1
    tok[2::4, 0] = V
    t = on_gpu(z, dtype, pad, shift)
    tt = torch.from_numpy(tok).to(DEV)
    got = score_device(t, tt, T, k)
    check_score(z, dtype, tok, T, k, got)
    again = score_device(t, tt[:, 0].contiguous(), T, 0, want_entropy=False)  # without the entropy and alternatives
    assert again.entropy is None and again.top_ids is None
    a, b = again.logprob, got.logprob[:, 0]
    assert torch.allclose(a, b, rtol=1e-6, atol=1e-5, equal_nan=True)
    one = score_device(t, tt, T, k)
    for x, y in zip(got, one):  # the same bits again
        assert x is None or torch.equal(x.view(torch.int32), y.view(torch.int32))


@pytest.mark.parametrize("V,dtype,k", [(16384, "bf16", 512), (16384, "fp32", 20), (2048, "fp32", 512),
                                       (131072, "fp16", 100), (40000, "fp32", 300)])
def test_alternatives_of_ties_and_sorted_rows(built, V, dtype, k):
    """Rows that defeat a selection by sampled maxima: few distinct values,
    all equal but a few, ascending, descending, everything masked but fewer
    than k, the top ones adjacent."""
    rng = np.random.default_rng(V + k)
    z = np.empty((9, V))
    z[0] = rng.integers(0, 3, V)
    z[1] = 0.0
    z[1, rng.integers(0, V, k // 2)] = 1.0
    z[2] = np.arange(V) / V * 8
    z[3] = -np.arange(V) / V * 8
    z[4] = -np.inf
    z[4, rng.integers(0, V, k // 3 + 1)] = rng.normal(0, 1, k // 3 + 1)
    z[5] = rng.normal(0, 0.01, V)
    z[5, V // 2:V // 2 + 2 * k] += 5.0
    z[6] = -1.0
    z[7] = rng.choice([-0.0, 0.0], V)
    z[8] = np.where(np.arange(V) % 2 == 0, 1.0, 2.0)
    t = torch.from_numpy(z.astype(np.float32)).to(DT[dtype])
    z = t.double().numpy()
    got = score_device(t.to(DEV), None, 1.0, k)
    ids = got.top_ids.cpu().numpy()
    for r in range(len(z)):
        assert np.array_equal(ids[r], order(z[r])[:k]), r


def check_grad(got, want, mag, z, T, dtype, factor=1.0):
    """Every term is off by at most its relative error, and the sum is rounded once to dtype."""
    got = got.double().cpu().numpy()
    eps = torch.finfo(DT[dtype]).eps / 2
    for r in range(len(z)):
        nan = np.isnan(want[r])
        assert np.array_equal(nan, np.isnan(got[r])), r
        tol = factor * rel_err_bound(z[r], T) * mag[r] + eps * np.abs(want[r]) * (1 + 1e-3) + TINY[dtype]
        # exponentials below 2^-126 (d < -87.33) are flushed to 0, and with them a term of at most
        # mag <= 2^-126 (|log p| + H + 1) times the gradients: below 1e-35 here
        f = np.where(np.isfinite(z[r]), z[r], -np.inf)
        if np.isfinite(f.max()):
            tol = tol + np.where((f - f.max()) / T < -87.3, np.minimum(mag[r], 1e-35), 0.0)
        bad = ~nan & (np.abs(got[r] - want[r]) > tol)
        assert not bad.any(), (r, np.flatnonzero(bad)[:5], got[r][bad][:5], want[r][bad][:5], tol[bad][:5])
        if not nan.any():
            assert (got[r][z[r] == -np.inf] == 0).all()


@pytest.mark.parametrize("R,V,dtype,pad,shift,T,k,n", SIZES, ids=str)
def test_score_grad(built, R, V, dtype, pad, shift, T, k, n):
    rng = np.random.default_rng(R * 37 + V)
    z = rows_of(rng, R, V, dtype, "mixed")
    tok = rng.integers(0, V, (R, n)).astype(np.int32)
    tok[1::4, -1] = -1
    tok[2::4, 0] = V + 5
    if n > 2:
        tok[:, 1] = tok[:, 2]  # the same id twice
    g = rng.normal(0, 1, (R, n)).astype(np.float32)
    gh = rng.normal(0, 0.3, R).astype(np.float32)
    gh[1::4] = 0.0  # with n 1: rows of padding, whatever they hold
    t = on_gpu(z, dtype, pad, shift)
    tt, gt, ht = (torch.from_numpy(a).to(DEV) for a in (tok, g, gh))
    for entropy in (True, False):
        pairs = [score_grad_row(z[r], tok[r], g[r], gh[r] if entropy else 0.0, T) for r in range(R)]
        want, mag = np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs])
        got = score_grad_device(t, tt, gt, ht if entropy else None, T)
        # p (log p + H): p and log p off by the bound, H by 2 (1 + log V) of it
        check_grad(got, want, mag, z, T, dtype, 4 + 2 * np.log(V) if entropy else 1.0)
    only = score_grad_device(t, None, None, ht, T)
    pairs = [score_grad_row(z[r], [], [], gh[r], T) for r in range(R)]
    check_grad(only, np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]), z, T, dtype,
               4 + 2 * np.log(V))


def teacher_lists(rng, z, k, rest, T):
    """Lists as a teacher gives them, then what can go wrong in them."""
    R, V = z.shape
    ids = np.empty((R, k), dtype=np.int32)
    vals = np.empty((R, k), dtype=np.float32)
    for r in range(R):
        zr = np.where(np.isfinite(z[r]), np.clip(z[r], -50, 50), -60.0) + rng.normal(0, 0.5, V)
        ids[r] = order(zr)[:k] if k <= V else np.resize(order(zr), k)
        v = zr[ids[r]]
        if rest:
            v = v / T - np.log(np.exp(zr / T - zr.max() / T).sum()) - zr.max() / T
        vals[r] = v
    if k > 3:
        ids[1::5, k // 2:] = -1       # a short list
        ids[2::5, 1] = ids[2::5, 0]   # an id twice
        vals[3::5, 0] = -np.inf       # an entry without mass
    ids[4::7] = -1                    # no list
    if rest:  # twice the same id may take the sum past 1: halve those rows' probabilities
        vals[2::5] -= np.float32(np.log(2.0))
    return ids, vals


DISTILL = [  # rows, vocab, dtype, pad, shift, temperature, entries, label weight
    (1, 1, "fp32", 0, 0, 1.0, 1, 0.5),
    (5, 2, "fp32", 0, 0, 1.0, 2, 0.0),
    (11, 9, "fp32", 3, 1, 2.0, 12, 0.3),
    (1, 16384, "fp32", 0, 0, 1.0, 20, 0.5),
    (22, 1001, "fp32", 0, 0, 2.0, 64, 0.5),
    (22, 1001, "bf16", 1, 3, 1.0, 512, 0.0),
    (11, 4099, "fp16", 5, 1, 0.5, 33, 1.0),
    (11, 16384, "fp32", 4, 0, 2.0, 512, 0.25),
    (13, 16383, "bf16", 0, 0, 1.0, 17, 0.5),
    (12, 32000, "bf16", 0, 8, 1.3, 128, 0.0),
    (11, 131072, "fp32", 0, 0, 1.5, 20, 0.5),
    (11, 131072, "fp16", 0, 0, 1.0, 64, 0.0),
    (2, 524288, "fp32", 0, 0, 1.0, 40, 0.5),
    (700, 300, "fp32", 0, 0, 1.0, 5, 0.5),
    (330, 16384, "fp32", 0, 0, 2.0, 64, 0.5),
]


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("R,V,dtype,pad,shift,T,k,a", DISTILL, ids=str)
def test_distill(built, R, V, dtype, pad, shift, T, k, a, rest):
    rng = np.random.default_rng(R * 41 + V + k)
    z = rows_of(rng, R, V, dtype, "mixed", spread=2.0)
    ids, vals = teacher_lists(rng, z, k, rest, T)
    y = rng.integers(0, V, R).astype(np.int32)
    y[4::7] = -1   # with an empty list: rows of padding
    y[5::7] = V
    rg = rng.normal(0, 1, R).astype(np.float32)
    t = on_gpu(z, dtype, pad, shift)
    it, vt, yt, rt = (torch.from_numpy(x).to(DEV) for x in (ids, vals, y, rg))
    loss, grad = distill_device(t, it, vt, yt if a > 0 else None, T, a, rest, rt)
    alone, none = distill_device(t, it, vt, yt if a > 0 else None, T, a, rest, want_grad=False)
    assert none is None
    want = [distill_row(z[r], ids[r], vals[r], y[r], T, a, rest) for r in range(R)]
    for got in (loss, alone):
        g = got.double().cpu().numpy()
        for r in range(R):
            w, lmag = float(in_f32(want[r][0])), want[r][3]
            tol = rel_err_bound(z[r], min(T, 1.0))
            if not np.isfinite(w):
                assert np.array_equal(w, g[r], equal_nan=True), (r, w, g[r])
            else:  # every log is off by the sums' relative error, weighted by at most 1 in all; one rounding at the end
                assert abs(g[r] - w) <= tol * (2 * max(T * T, 1.0) + lmag), (r, g[r], w, tol)
    wg = np.stack([x[1] * s for x, s in zip(want, rg)])
    mag = np.stack([x[2] * abs(float(s)) for x, s in zip(want, rg)])
    check_grad(grad, wg, mag, z, min(T, 1.0), dtype)
    # the gradient in the logits' place, and next to them in rows of the same stride
    wide = torch.full((R, 2 * V + 5), 3.0, dtype=DT[dtype], device=DEV)
    left, right = wide[:, :V], wide[:, V + 2:2 * V + 2]
    left.copy_(t)
    same = lambda p, q: torch.equal(torch.nan_to_num(p.float(), 9.0), torch.nan_to_num(q.float(), 9.0))  # noqa: E731
    _, g2 = distill_device(left, it, vt, yt if a > 0 else None, T, a, rest, rt, grad_dev=right)
    assert torch.allclose(g2.float(), grad.float(), rtol=1e-2 if dtype != "fp32" else 1e-5, atol=1e-6, equal_nan=True)
    assert same(left, t) and (wide[:, V:V + 2] == 3).all() and (wide[:, 2 * V + 2:] == 3).all()
    _, g3 = distill_device(left, it, vt, yt if a > 0 else None, T, a, rest, rt, grad_dev=left)
    assert g3.data_ptr() == left.data_ptr() and same(left, right)
    assert (wide[:, V:V + 2] == 3).all() and (wide[:, 2 * V + 2:] == 3).all()


def test_confident_student_rest(built):
    """The unlisted mass far below the listed: 1 - sum would lose it."""
    V, k = 16384, 8
    rng = np.random.default_rng(5)
    z = rng.normal(-14, 1, (6, V)).astype(np.float32).astype(np.float64)
    ids = np.stack([rng.choice(V, k, replace=False) for _ in range(6)]).astype(np.int32)
    for r in range(6):
        z[r, ids[r]] = np.float32(rng.normal(10, 1, k))
    vals = np.log(np.full((6, k), (1 - 2.0 ** -12) / k)).astype(np.float32)
    loss, grad = distill_device(on_gpu(z, "fp32"), torch.from_numpy(ids).to(DEV), torch.from_numpy(vals).to(DEV),
                                rest=True)
    want = [distill_row(z[r], ids[r], vals[r], -1, 1.0, 0.0, True) for r in range(6)]
    for r in range(6):
        assert abs(float(loss[r]) - want[r][0]) <= rel_err_bound(z[r], 1.0) * (2 + want[r][3])
    check_grad(grad, np.stack([w[1] for w in want]), np.stack([w[2] for w in want]), z, 1.0, "fp32")


def small(rng, R=40, V=3001, k=16):
    z = torch.from_numpy(rng.normal(0, 3, (R, V)).astype(np.float32)).to(DEV)
    tok = torch.from_numpy(rng.integers(0, V, R).astype(np.int32)).to(DEV)
    val, ids = torch.topk(z + 0.3, k)
    return z, tok, ids.int(), val


def test_rows_do_not_depend_on_one_another(built):
    rng = np.random.default_rng(11)
    z, tok, ids, val = small(rng, 640, 2050)
    all_ = score_device(z, tok, 1.0, 10)
    loss, grad = distill_device(z, ids, val, tok, 2.0, 0.5)
    for lo, hi in ((0, 1), (5, 9), (100, 400)):
        part = score_device(z[lo:hi].contiguous(), tok[lo:hi].contiguous(), 1.0, 10)
        l, g = distill_device(z[lo:hi].contiguous(), ids[lo:hi].contiguous(), val[lo:hi].contiguous(),
                              tok[lo:hi].contiguous(), 2.0, 0.5)
        assert torch.equal(part.top_ids, all_.top_ids[lo:hi])
        # a call of few rows may spread a row over more of the GPU: another order of the sums
        for a, b in ((part.logprob, all_.logprob[lo:hi]), (part.entropy, all_.entropy[lo:hi]), (l, loss[lo:hi]),
                     (g, grad[lo:hi])):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)


def test_side_stream_and_order(built):
    """Queued on the stream it is given, after that stream's earlier work."""
    rng = np.random.default_rng(12)
    z, tok, ids, val = small(rng)
    ref = score_device(z, tok, 1.0, 8)
    rl, rg = distill_device(z, ids, val)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        z2 = torch.zeros_like(z)
        torch.cuda._sleep(20_000_000)
        z2.copy_(z)
        a = score_device(z2, tok, 1.0, 8)          # torch's current stream
        l, g = distill_device(z2, ids, val, stream=s.cuda_stream)
    s.synchronize()
    for x, y in zip(a, ref):
        assert torch.equal(x, y)
    assert torch.equal(l, rl) and torch.equal(g, rg)


def test_two_streams_at_once(built):
    rng = np.random.default_rng(13)
    z, tok, ids, val = small(rng, 600, 16384, 64)
    ref = score_device(z, tok, 1.0, 64)
    rl, rg = distill_device(z, ids, val, rest=False)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            for _ in range(3):
                got.append((score_device(z, tok, 1.0, 64), distill_device(z, ids, val)))
    torch.cuda.synchronize()
    for a, (l, g) in got:
        assert all(torch.equal(x, y) for x, y in zip(a, ref)) and torch.equal(l, rl) and torch.equal(g, rg)


def test_captured_graphs(built):
    """Two captured graphs, replayed on new inputs, one after and beside the other."""
    rng = np.random.default_rng(14)
    z, tok, ids, val = small(rng, 64, 16384, 20)
    gl = torch.ones(64, device=DEV)
    graphs, outs = [], []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            o = (score_device(z, tok, 1.0, 20), distill_device(z, ids, val, tok, 2.0, 0.5),
                 score_grad_device(z, tok, gl))
        graphs.append(gr)
        outs.append(o)
    for rep in range(3):
        z.copy_(torch.randn(64, 16384, device=DEV) * 3)
        want = (score_device(z, tok, 1.0, 20), distill_device(z, ids, val, tok, 2.0, 0.5),
                score_grad_device(z, tok, gl))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(x, y) for x, y in zip(o[0], want[0]))
            assert all(torch.equal(x, y) for x, y in zip(o[1], want[1])) and torch.equal(o[2], want[2])


def test_rows_beyond_32_bit_offsets(built):
    """A row stride past 2^31 elements."""
    V, ld = 5003, (1 << 31) + 8
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    rng = np.random.default_rng(15)
    z = rows_of(rng, 2, V, "bf16")
    flat = torch.empty(ld + V, dtype=torch.bfloat16, device=DEV)
    t = torch.as_strided(flat, (2, V), (ld, 1))
    t.copy_(torch.from_numpy(z).to(torch.bfloat16))
    tok = np.array([[3], [V - 1]], dtype=np.int32)
    check_score(z, "bf16", tok, 1.0, 9, score_device(t, torch.from_numpy(tok).to(DEV), 1.0, 9))
    want = [score_grad_row(z[r], tok[r], [1.0], 0.0, 1.0) for r in range(2)]
    g = score_grad_device(t, torch.from_numpy(tok).to(DEV), torch.ones(2, 1, device=DEV), grad_dev=t)
    check_grad(g, np.stack([w[0] for w in want]), np.stack([w[1] for w in want]), z, 1.0, "bf16")


def test_refusals_on_the_gpu(built):
    z = torch.zeros(4, 100, device=DEV)
    tok = torch.zeros(4, dtype=torch.int32, device=DEV)
    ids, val = torch.zeros(4, 3, dtype=torch.int32, device=DEV), torch.zeros(4, 3, device=DEV)
    bad = [lambda: score_device(z, tok.long()), lambda: score_device(z, tok.cpu()), lambda: score_device(z, tok[:3]),
           lambda: score_device(z.double(), tok), lambda: score_device(z.t(), tok), lambda: score_device(z, tok, 0.0),
           lambda: score_device(z, tok, 1.0, 101), lambda: score_device(z[0], tok),
           lambda: score_device(z[:1].expand(4, 100), tok),  # rows on top of one another
           lambda: score_device(z, None, want_entropy=False),
           lambda: score_grad_device(z, tok, None), lambda: score_grad_device(z, tok, torch.ones(3, device=DEV)),
           lambda: score_grad_device(z, tok, torch.ones(4, device=DEV), grad_dev=z.half()),
           lambda: distill_device(z, ids.long(), val), lambda: distill_device(z, ids, val[:, :2]),
           lambda: distill_device(z, ids, val, label_weight=0.5), lambda: distill_device(z, ids[:, :0], val[:, :0]),
           lambda: distill_device(z, ids, val, tok, 1.0, 1.5)]
    for f in bad:
        with pytest.raises(CortexError):
            f()
    lib_err = None
    host = torch.zeros(4, 100)
    from snai_b200 import last_error, load
    rc = load().cortex_score(host.data_ptr(), 0, 4, 100, 100, tok.data_ptr(), 1, 1.0, 0, val.data_ptr(), None, None,
                             None, None)
    lib_err = last_error()
    assert rc < 0 and "device memory" in lib_err
    torch.cuda.synchronize()  # nothing was launched that could fail


def test_empty_batch(built):
    z = torch.zeros(0, 100, device=DEV)
    s = score_device(z, torch.zeros(0, dtype=torch.int32, device=DEV), 1.0, 5)
    assert s.logprob.shape == (0,) and s.top_ids.shape == (0, 5)
    loss, grad = distill_device(z, torch.zeros(0, 3, dtype=torch.int32, device=DEV), torch.zeros(0, 3, device=DEV))
    assert loss.shape == (0,) and grad.shape == (0, 100)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one(built):
    rng = np.random.default_rng(16)
    z, tok, ids, val = small(rng)
    ref = score_device(z, tok, 1.0, 8)
    other = torch.device("cuda", 1)
    with torch.cuda.device(0):
        got = score_device(z.to(other), tok.to(other), 1.0, 8)
    for x, y in zip(got, ref):
        assert torch.equal(x.cpu(), y.cpu())
