"""The vocabulary-row operators over ranges: drawn shapes, types, alignments,
masks and lists against 64 bits, calls of very many short rows, long lists on
short rows, what padding entries may hold, and what lies around the outputs."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from row_reference import distill_row, rel_err_bound, score_grad_row, score_row  # noqa: E402
from snai_b200 import distill_device, score_device, score_grad_device  # noqa: E402
from test_gpu_score import (DEV, DT, check_grad, check_score, in_f32, on_gpu, rows_of, small,  # noqa: E402
                            teacher_lists)


def dev(*arrays):
    return [torch.from_numpy(np.ascontiguousarray(a)).to(DEV) for a in arrays]


def check_distill(z, dtype, ids, vals, y, T, a, rest, rg, loss, grad):
    """As test_gpu_score.test_distill bounds them."""
    want = [distill_row(z[r], ids[r], vals[r], y[r], T, a, rest) for r in range(len(z))]
    got = loss.double().cpu().numpy()
    for r in range(len(z)):
        w, tol = float(in_f32(want[r][0])), rel_err_bound(z[r], min(T, 1.0))
        if not np.isfinite(w):
            assert np.array_equal(w, got[r], equal_nan=True), (r, w, got[r])
        else:
            assert abs(got[r] - w) <= tol * (2 * max(T * T, 1.0) + want[r][3]), (r, got[r], w, tol)
    if grad is not None:
        check_grad(grad, np.stack([x[1] * s for x, s in zip(want, rg)]),
                   np.stack([x[2] * abs(float(s)) for x, s in zip(want, rg)]), z, min(T, 1.0), dtype)


def drawn(seed):
    rng = np.random.default_rng(seed)
    V = int(2 ** rng.uniform(0, 17))
    R = int(min(2 ** rng.uniform(0, 9), max(1, 600_000 // V)))
    k = int(min(512, V, 2 ** rng.uniform(0, 9.2)))
    return rng, R, V, ["fp32", "bf16", "fp16"][rng.integers(3)], int(rng.integers(0, 9)), int(rng.integers(0, 9)), \
        float(rng.choice([0.5, 0.8, 1.0, 1.0, 2.0, 3.0, 4.0])), k


@pytest.mark.parametrize("seed", range(40))
def test_drawn_scores(built, seed):
    rng, R, V, dtype, pad, shift, T, k = drawn(seed)
    n = int(2 ** rng.uniform(0, 5))
    z = rows_of(rng, R, V, dtype, "mixed")
    tok = rng.integers(-1, V + 1, (R, n)).astype(np.int32)
    g, gh = rng.normal(0, 1, (R, n)).astype(np.float32), rng.normal(0, 0.3, R).astype(np.float32)
    t, (tt, gt, ht) = on_gpu(z, dtype, pad, shift), dev(tok, g, gh)
    check_score(z, dtype, tok, T, k, score_device(t, tt, T, k))
    pairs = [score_grad_row(z[r], tok[r], g[r], gh[r], T) for r in range(R)]
    check_grad(score_grad_device(t, tt, gt, ht, T), np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]),
               z, T, dtype, 4 + 2 * np.log(V))


@pytest.mark.parametrize("seed", range(40))
def test_drawn_distillations(built, seed):
    rng, R, V, dtype, pad, shift, T, k = drawn(100 + seed)
    rest, a = bool(rng.integers(2)), float(rng.choice([0.0, 0.3, 1.0]))
    z = rows_of(rng, R, V, dtype, "mixed", spread=2.0)
    ids, vals = teacher_lists(rng, z, k, rest, T)
    y = rng.integers(-1, V + 1, R).astype(np.int32)
    y[::5] = ids[::5, 0]  # a label that the list holds
    rg = rng.normal(0, 1, R).astype(np.float32)
    it, vt, yt, rt = dev(ids, vals, y, rg)
    t = on_gpu(z, dtype, pad, shift)
    loss, grad = distill_device(t, it, vt, yt if a else None, T, a, rest, rt)
    check_distill(z, dtype, ids, vals, y, T, a, rest, rg, loss, grad)


@pytest.mark.parametrize("V,dtype,k", [(1, "fp32", 1), (5, "bf16", 5), (33, "fp32", 33), (130, "fp16", 100),
                                       (520, "bf16", 512)])
def test_many_short_rows(built, V, dtype, k):
    """More rows than the GPU holds at once, each shorter than a CTA's words."""
    R = 5003
    rng = np.random.default_rng(V)
    z = rows_of(rng, R, V, dtype, "mixed", spread=2.0)
    tok = rng.integers(-1, V + 1, (R, 1)).astype(np.int32)
    ids, vals = teacher_lists(rng, z, k, True, 2.0)
    rg = np.ones(R, dtype=np.float32)
    t, (tt, it, vt, rt) = on_gpu(z, dtype, 1, 1), dev(tok, ids, vals, rg)
    s = score_device(t, tt, 1.0, k)
    loss, grad = distill_device(t, it, vt, tt[:, 0].contiguous(), 2.0, 0.5, True, rt)
    pick = np.concatenate([np.arange(40), rng.choice(R, 200, replace=False), np.arange(R - 40, R)])
    dp = torch.from_numpy(pick).to(DEV)
    check_score(z[pick], dtype, tok[pick], 1.0, k, type(s)(*(x[dp] for x in s)))
    check_distill(z[pick], dtype, ids[pick], vals[pick], tok[pick, 0], 2.0, 0.5, True, rg[pick], loss[dp], grad[dp])


@pytest.mark.parametrize("V,dtype", [(1001, "fp32"), (1001, "bf16"), (40000, "fp32"), (131072, "bf16")])
def test_padding_entries_may_hold_anything(built, V, dtype):
    """NaN and infinities beside ids outside [0, vocab), and a row's columns past it."""
    R, k = 14, 9
    rng = np.random.default_rng(V)
    z = rows_of(rng, R, V, dtype, spread=2.0)
    ids, vals = teacher_lists(rng, z, k, False, 1.0)
    tok = rng.integers(0, V, (R, 3)).astype(np.int32)
    g = rng.normal(0, 1, (R, 3)).astype(np.float32)
    tok[::2, 1], tok[1::2, 2], tok[5] = -1, V, -7
    ids[::2, 3], ids[1::2, 5], ids[6] = V, np.iinfo(np.int32).min, -1
    ids[0, 0], tok[0, 0] = np.iinfo(np.int32).max, np.iinfo(np.int32).max
    y = np.where(np.arange(R) % 3 == 0, -5, tok[:, 0]).astype(np.int32)
    out = (ids < 0) | (ids >= V)
    vals[out] = rng.choice([np.nan, np.inf, -np.inf], out.sum())
    gout = (tok < 0) | (tok >= V)
    g[gout] = rng.choice([np.nan, np.inf], gout.sum())
    wide = torch.full((R, V + 40), float("nan"), dtype=DT[dtype], device=DEV)
    t = wide[:, 3:3 + V]
    t.copy_(torch.from_numpy(z).to(DT[dtype]))
    it, vt, yt, tt, gt = dev(ids, vals, y, tok, g)
    for rest in (False, True):
        loss, grad = distill_device(t, it, vt, yt, 1.0, 0.5, rest)
        check_distill(z, dtype, ids, np.where(out, 0, vals), y, 1.0, 0.5, rest, np.ones(R), loss, grad)
    check_score(z, dtype, tok, 1.0, 5, score_device(t, tt, 1.0, 5))
    pairs = [score_grad_row(z[r], tok[r], np.where(gout, 0, g)[r], 0.0, 1.0) for r in range(R)]
    check_grad(score_grad_device(t, tt, gt, None, 1.0), np.stack([p[0] for p in pairs]),
               np.stack([p[1] for p in pairs]), z, 1.0, dtype)


@pytest.mark.parametrize("V", [200, 16384, 100000])
def test_lists_of_one_id(built, V):
    """512 times the same id, once with the label on it, once on a masked one."""
    R, k = 8, 512
    rng = np.random.default_rng(V)
    z = rows_of(rng, R, V, "fp32", spread=2.0)
    at = rng.integers(0, V, R)
    z[3, at[3]] = z[4, at[4]] = -np.inf
    ids = np.repeat(at[:, None], k, 1).astype(np.int32)
    vals = rng.normal(0, 1, (R, k)).astype(np.float32)
    y = at.astype(np.int32)
    y[1] = (y[1] + 1) % V
    t, (it, vt, yt, ones) = on_gpu(z, "fp32"), dev(ids, vals, y, np.ones((R, k), np.float32))
    loss, grad = distill_device(t, it, vt, yt, 1.0, 0.5)
    check_distill(z, "fp32", ids, vals, y, 1.0, 0.5, False, np.ones(R), loss, grad)
    lv = np.full((R, k), np.log(0.9 / k), np.float32)
    loss, grad = distill_device(t, it, dev(lv)[0], yt, 4.0, 0.5, True)
    check_distill(z, "fp32", ids, lv, y, 4.0, 0.5, True, np.ones(R), loss, grad)
    pairs = [score_grad_row(z[r], ids[r], np.ones(k), 0.0, 1.0) for r in range(R)]
    # the id's own sum of 512 ones is exact; p times it carries p's error
    check_grad(score_grad_device(t, it, ones), np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]), z,
               1.0, "fp32")


@pytest.mark.parametrize("R,V,dtype", [(3, 7, "bf16"), (40, 1003, "fp32"), (500, 2049, "fp16"), (9, 70001, "bf16")])
def test_outputs_end_where_they_end(built, R, V, dtype):
    """Guards before and behind every output, the gradient in rows of its own stride."""
    from snai_b200 import DistillParams, load

    rng = np.random.default_rng(R + V)
    k, n, gld = 5, 3, V + 6
    z = rows_of(rng, R, V, dtype, "mixed")
    t = on_gpu(z, dtype, 2, 1)
    tok = rng.integers(0, V, (R, n)).astype(np.int32)
    ids, vals = teacher_lists(rng, z, k, False, 1.0)
    tt, it, vt, gt = dev(tok, ids, vals, rng.normal(0, 1, (R, n)).astype(np.float32))
    f = {x: torch.full((c + 64,), 77, dtype=d, device=DEV) for x, c, d in
         (("lp", R * n, torch.float32), ("ent", R, torch.float32), ("ids", R * k, torch.int32),
          ("top", R * k, torch.float32), ("loss", R, torch.float32), ("g1", R * gld, DT[dtype]),
          ("g2", R * gld, DT[dtype]))}
    p = {x: b.data_ptr() + 32 * b.element_size() for x, b in f.items()}
    lib, st, code = load(), torch.cuda.current_stream().cuda_stream, {"fp32": 0, "bf16": 1, "fp16": 2}[dtype]
    prm = DistillParams(1.0, 0.0, 0)
    assert lib.cortex_score(t.data_ptr(), code, R, V, V + 2, tt.data_ptr(), n, 1.0, k, p["lp"], p["ent"], p["ids"],
                            p["top"], st) == 0
    assert lib.cortex_score_grad(t.data_ptr(), code, R, V, V + 2, tt.data_ptr(), n, 1.0, gt.data_ptr(), None, p["g1"],
                                 gld, st) == 0
    assert lib.cortex_distill(t.data_ptr(), code, R, V, V + 2, it.data_ptr(), vt.data_ptr(), k, None, None,
                              ctypes.byref(prm), p["loss"], p["g2"], gld, st) == 0
    torch.cuda.synchronize()
    for x, b in f.items():
        assert (b[:32] == 77).all() and (b[-32:] == 77).all(), x
    ref = score_device(t, tt, 1.0, k)
    assert torch.equal(f["lp"][32:-32].view(R, n).nan_to_num(9), ref.logprob.nan_to_num(9))
    assert torch.equal(f["ids"][32:-32].view(R, k), ref.top_ids)
    for x, want in (("g1", score_grad_device(t, tt, gt)), ("g2", distill_device(t, it, vt)[1])):
        rows = f[x][32:-32].view(R, gld)
        assert (rows[:, V:] == 77).all(), x
        # another alignment of the gradient's rows may take another path: a rounding of its own
        assert torch.allclose(rows[:, :V].float(), want.float(), rtol=1e-5 if dtype == "fp32" else 1e-2, atol=1e-6,
                              equal_nan=True), x


@pytest.mark.parametrize("V,dtype", [(1001, "fp32"), (16384, "bf16"), (16383, "fp16"), (131072, "fp32")])
def test_score_gradient_in_place(built, V, dtype):
    R = 30
    rng = np.random.default_rng(V)
    z = rows_of(rng, R, V, dtype, "mixed")
    tok = rng.integers(0, V, (R, 4)).astype(np.int32)
    g, gh = rng.normal(0, 1, (R, 4)).astype(np.float32), rng.normal(0, 0.3, R).astype(np.float32)
    t, (tt, gt, ht) = on_gpu(z, dtype, 3, 2), dev(tok, g, gh)
    got = score_grad_device(t, tt, gt, ht, 1.0, grad_dev=t)
    assert got is t
    pairs = [score_grad_row(z[r], tok[r], g[r], gh[r], 1.0) for r in range(R)]
    check_grad(t, np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]), z, 1.0, dtype, 4 + 2 * np.log(V))


@pytest.mark.parametrize("V,dtype", [(16384, "fp32"), (100001, "fp32"), (32000, "bf16")])
def test_gradients_are_the_differences(built, V, dtype):
    """grad . u against (f(z + h u) - f(z - h u)) / 2h of the kernel's own sums, h u exact in the type."""
    R, k, h = 6, 8, 2.0 ** -4
    rng = np.random.default_rng(V)
    # logits on a grid of 1/16 under 8, exact in bf16 with h u of 0 or +-1/16
    z = np.round(np.clip(rng.normal(0, 2, (R, V)), -7, 7) * 16) / 16
    if dtype == "bf16":
        z = np.round(np.clip(z, -4, 4) * 2) / 2  # 8 bits: up to 4 in steps of 1/32 and h u
        z = np.clip(z, -3.5, 3.5)
    u = rng.choice([-1.0, 0.0, 1.0], (R, V))
    tok = rng.integers(0, V, (R, 1)).astype(np.int32)
    ids, vals = teacher_lists(rng, z, k, False, 2.0)
    rg = rng.uniform(0.5, 1.5, R).astype(np.float32)
    tt, it, vt, rt = dev(tok, ids, vals, rg)
    y = tt[:, 0].contiguous()
    at = lambda s: on_gpu(z + s * h * u, dtype)  # noqa: E731
    ud = torch.from_numpy(u).to(DEV)
    f32 = torch.float32

    def values(t):
        s = score_device(t, tt, 2.0)
        loss, _ = distill_device(t, it, vt, y, 2.0, 0.5, want_grad=False)
        return ((s.logprob[:, 0].double() * rt + 0.5 * s.entropy.double()), loss.double() * rt)

    plus, minus = values(at(1)), values(at(-1))
    gs = score_grad_device(at(0), tt, rt.view(R, 1), torch.full((R,), 0.5, dtype=f32, device=DEV), 2.0)
    _, gd = distill_device(at(0), it, vt, y, 2.0, 0.5, False, rt)
    for p, m, g in zip(plus, minus, (gs, gd)):
        diff, dot = (p - m) / (2 * h), (g.double() * ud).sum(1)
        # central differences: h^2 / 6 times the third derivative along u (|u| <= 1: third cumulants of p, below
        # 8 in all with the weights and T here, entropy's times its log V); the values' float32 error (16 units of
        # values below 40, twice, over 2h); the gradient's own rounding (relative to the sum of |g|, below 16)
        eps = torch.finfo(DT[dtype]).eps
        tol = h * h / 6 * 8 * (1 + np.log(V)) / 2 + 16 * 2.0 ** -24 * 40 / h + eps * 16
        assert ((diff - dot).abs() <= tol).all(), (diff, dot, tol)


def test_first_call_of_a_shape_in_a_capture(built):
    """Nothing is set up on a first call that a capture would not take."""
    rng = np.random.default_rng(21)
    z, tok, ids, val = small(rng, 37, 9973, 41)
    gl = torch.ones(37, device=DEV)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        a = score_device(z, tok, 1.5, 41)
        b = distill_device(z, ids, val, tok, 3.0, 0.25, True)
        c = score_grad_device(z, tok, gl, gl)
    gr.replay()
    torch.cuda.synchronize()
    want = (score_device(z, tok, 1.5, 41), distill_device(z, ids, val, tok, 3.0, 0.25, True),
            score_grad_device(z, tok, gl, gl))
    assert all(torch.equal(x, y) for x, y in zip(a, want[0])) and all(torch.equal(x, y) for x, y in zip(b, want[1]))
    assert torch.equal(c, want[2])


def test_a_run_of_them(built):
    """As they are used: a teacher's rows are scored for alternatives, the
    student learns from them."""
    R, V, k, T = 64, 5003, 32, 2.0
    gen = torch.Generator(device=DEV).manual_seed(3)
    teacher = torch.randn(R, V, device=DEV, generator=gen) * 3
    student = torch.randn(R, V, device=DEV, generator=gen)
    s = score_device(teacher, None, T, k)
    y = s.top_ids[:, 0].contiguous()
    zt, zs = teacher.double().cpu().numpy(), student.double().cpu().numpy()
    loss, grad = distill_device(student, s.top_ids, s.top_logprob, y, T, 0.5, True)
    vals = np.stack([score_row(zt[r], [], T, k)[3] for r in range(R)])
    got = loss.double().cpu().numpy()
    for r in range(R):
        w = distill_row(zs[r], s.top_ids[r].cpu().numpy(), vals[r], int(y[r]), T, 0.5, True)
        # the teacher's own log probabilities are off by its bound
        tol = (rel_err_bound(zs[r], 1.0) + rel_err_bound(zt[r], 1.0)) * (2 * T * T + w[3]) * 2
        assert abs(got[r] - w[0]) <= tol
    want = [distill_row(zs[r], s.top_ids[r].cpu().numpy(), vals[r], int(y[r]), T, 0.5, True) for r in range(R)]
    # q's relative error is its log's absolute one, the teacher's bound: at most twice the student's own
    assert all(rel_err_bound(zt[r], T) <= 2 * rel_err_bound(zs[r], 1.0) for r in range(R))
    check_grad(grad, np.stack([w[1] for w in want]), np.stack([w[2] for w in want]), zs, 1.0, "fp32", 3.0)


@pytest.mark.parametrize("V,k,dtype", [(4, 4, "fp16"), (700, 512, "bf16"), (20000, 20, "fp32"), (70000, 512, "bf16"),
                                       (300000, 64, "fp32")])
def test_fewer_numbers_than_alternatives(built, V, k, dtype):
    """NaNs in all but a few places, beside rows of few values."""
    rng = np.random.default_rng(V)
    z = np.full((6, V), np.nan)
    z[0, rng.permutation(V)[:k - 1]] = 1.0
    z[1, V // 2:] = -np.inf
    z[2] = -np.inf
    z[2, -1] = np.nan
    z[3] = 0.0
    z[3, 0] = np.nan
    z[4] = np.inf
    z[5] = 0.5
    t = on_gpu(z, dtype, 1, 1)
    got = score_device(t, torch.zeros(6, 1, dtype=torch.int32, device=DEV), 1.0, k)
    check_score(z, dtype, np.zeros((6, 1), np.int32), 1.0, k, got)
