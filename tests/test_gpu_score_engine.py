"""Scoring and distillation on a state: cortex_score_batch against
cortex_forward_batch's logits, cortex_distill_grads against the training
step's gradients and against differences, and the two together: a teacher
scores a text, a student learns from its top logits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

import oracle as O  # noqa: E402
from conftest import make_model, rel_err  # noqa: E402
from row_reference import order, rel_err_bound, score_row  # noqa: E402
from snai_b200 import PREC_BF16, PREC_FP32, PREC_TF32, Cortex, CortexError, VARIANT_B, sample_params  # noqa: E402


def every_logits(eng, tokens, slots=None):
    """[B, n, V] logits of every position, one token at a time."""
    return np.stack([eng.forward(tokens[:, i:i + 1], slots) for i in range(tokens.shape[1])], 1)


# logits of one pass of many rows against passes of few: FP32 engines sum in
# another order (the logits test's 2e-5); the tensor-core ones give a row the
# same bits whatever the pass, except through attention's split form
LOGIT_TOL = {PREC_FP32: 2e-5, PREC_TF32: 4e-3, PREC_BF16: 3e-2}


@pytest.mark.parametrize("precision", [PREC_FP32, PREC_TF32, PREC_BF16])
def test_score_batch_scores_every_position(model_dir, built, precision):
    V, k, T = 1000, 7, 0.8
    p = make_model(model_dir, "score_a.snai", V, 128, 96, 2, seed=5, std=0.06)
    rng = np.random.default_rng(1)
    tokens = rng.integers(0, V, (5, 20)).astype(np.int32)
    targets = rng.integers(0, V, (5, 20)).astype(np.int32)
    targets[1, 3], targets[2, 0] = -1, V
    ref, eng = (Cortex(p, num_heads=2, max_seqs=6, precision=precision) for _ in range(2))
    slots = [4, 0, 2, 5, 1]
    ref.reset()
    lg = every_logits(ref, tokens, slots).astype(np.float64)
    got = eng.score(tokens, targets, T, k, slots)
    tol = LOGIT_TOL[precision] * np.abs(lg).max() / T
    for b in range(5):
        for i in range(20):
            lp, ent, ids, top = score_row(lg[b, i], targets[b, i:i + 1], T, k)
            # a logit off by tol moves log p by at most 2 tol, the entropy by 2 tol times sum p |log p + H| <= 2 log V
            assert abs(got.logprob[b, i] - lp[0]) <= 2 * tol + rel_err_bound(lg[b, i], T) * 2
            assert abs(got.entropy[b, i] - ent) <= 4 * np.log(V) * tol + 1e-3
            assert np.abs(got.top_logprob[b, i] - top).max() <= 2 * tol + rel_err_bound(lg[b, i], T) * 2
            assert len(set(got.top_ids[b, i])) == k
    # the state goes on as after forward: positions, logits, history
    assert [eng.pos(s) for s in slots] == [20] * 5 and eng.pos(3) == 0
    a, b = eng.logits(slots), ref.logits(slots)
    assert rel_err(a, b) <= LOGIT_TOL[precision]
    # the last position's alternatives are those of the logits kept in the slot
    for r in range(5):
        assert np.array_equal(got.top_ids[r, -1], order(a[r].astype(np.float64))[:k])
    prm = sample_params(VARIANT_B, 0.7, 1.1, 10, 0.9)
    u = rng.random((3, 5)).astype(np.float32)
    ids = eng.decode_steps(u, prm, slots)
    assert ids.shape == (3, 5) and ((ids >= 0) & (ids < V)).all()
    eng.close()
    ref.close()


def test_score_batch_many_positions_and_ctx(model_dir, built):
    """More positions than are scored at a time, slots that meet ctx, and what is left alone."""
    V, ctx = 2048, 64
    p = make_model(model_dir, "score_b.snai", V, 128, ctx, 1, seed=6, std=0.06)
    rng = np.random.default_rng(2)
    B, n = 40, 50
    tokens = rng.integers(0, V, (B, n)).astype(np.int32)
    eng, ref = (Cortex(p, num_heads=2, max_seqs=B, precision=PREC_BF16) for _ in range(2))
    for e in (eng, ref):
        e.forward(tokens[:3, :30], slots=[0, 7, 39])  # these meet ctx after 34 more
    got = eng.score(tokens, tokens, 1.0, 3)  # 2000 - 48 positions
    lg = ref.forward(tokens)
    cut = np.array([34 if b in (0, 7, 39) else n for b in range(B)])
    for b in range(B):
        assert eng.pos(b) == ref.pos(b) == (ctx if b in (0, 7, 39) else n)
        assert (got.top_ids[b, cut[b]:] == -1).all() and (got.logprob[b, cut[b]:] == 0).all()
        assert (got.top_ids[b, :cut[b]] >= 0).all() and (got.logprob[b, :cut[b]] < 0).all()
        if cut[b] == n:
            want = score_row(lg[b].astype(np.float64), tokens[b, -1:], 1.0, 3)
            assert np.array_equal(got.top_ids[b, -1], want[2])
            assert abs(got.logprob[b, -1] - want[0][0]) <= rel_err_bound(lg[b], 1.0) * 2
    keep = [b for b in range(B) if cut[b] == n]
    assert np.array_equal(eng.logits(keep), ref.logits(keep))
    eng.close()
    ref.close()


def test_score_batch_device_pointers(model_dir, built):
    import ctypes

    from snai_b200 import _lib, load
    V = 1000
    p = make_model(model_dir, "score_a.snai", V, 128, 96, 2, seed=5, std=0.06)
    rng = np.random.default_rng(3)
    tokens = rng.integers(0, V, (4, 9)).astype(np.int32)
    eng, ref = (Cortex(p, num_heads=2, max_seqs=4) for _ in range(2))
    want = ref.score(tokens, tokens, 1.0, 5)
    dev = torch.device("cuda")
    t = torch.from_numpy(tokens).to(dev)
    lp, ent = torch.zeros(4, 9, device=dev), torch.zeros(4, 9, device=dev)
    ids, top = torch.zeros(4, 9, 5, dtype=torch.int32, device=dev), torch.zeros(4, 9, 5, device=dev)
    torch.cuda.synchronize()
    P = lambda x: ctypes.c_void_p(x.data_ptr())  # noqa: E731
    rc = load().cortex_score_batch(eng.h, P(t), 4, 9, None, P(t), 1.0, 5, P(lp), P(ent), P(ids), P(top),
                                   _lib.DEVICE_PTRS)
    assert rc == 0
    eng.synchronize()
    assert np.array_equal(lp.cpu().numpy(), want.logprob) and np.array_equal(ent.cpu().numpy(), want.entropy)
    assert np.array_equal(ids.cpu().numpy(), want.top_ids) and np.array_equal(top.cpu().numpy(), want.top_logprob)
    eng.profile(True)
    eng.score(tokens, None, 1.0, 2)
    assert eng.profile_read()["score"][0] == 1
    eng.close()
    ref.close()


def test_score_batch_refuses_before_feeding(model_dir, built):
    p = make_model(model_dir, "score_a.snai", 1000, 128, 96, 2, seed=5, std=0.06)
    eng = Cortex(p, num_heads=2, max_seqs=2)
    t = np.ones((2, 3), dtype=np.int32)
    for bad in (dict(temperature=0.0), dict(top_k=513), dict(slots=[0, 0]), dict(slots=[0, 2]), dict(slots=[0]),
                dict(targets=np.ones((2, 2)))):
        with pytest.raises(CortexError):
            eng.score(t, **bad)
    assert eng.pos(0) == 0 and eng.pos(1) == 0
    for bad in (dict(temperature=0.0), dict(label_weight=0.5), dict(label_weight=-1.0)):
        with pytest.raises(CortexError):
            eng.distill_grads([1, 2], np.zeros((2, 1)), np.zeros((2, 1)), **bad)
    with pytest.raises(CortexError):
        eng.distill_grads([1, 2], np.zeros((3, 1)), np.zeros((3, 1)))
    eng.close()


def test_score_batch_lengths_beyond_the_context(model_dir, built):
    """Token counts far past ctx: the positions that fit are scored; counts that no array could hold are refused."""
    p = make_model(model_dir, "score_a.snai", 1000, 128, 96, 2, seed=5, std=0.06)
    ref, eng = (Cortex(p, num_heads=2, max_seqs=2) for _ in range(2))
    ctx = 96
    t = (np.arange(ctx, dtype=np.int32) * 7 % 1000).reshape(1, ctx)
    want = ref.score(t, t)
    lp, ent = np.zeros(ctx, np.float32), np.zeros(ctx, np.float32)
    args = (t.ctypes.data, t.ctypes.data, lp.ctypes.data, ent.ctypes.data)

    def call(batch, n):
        return eng.lib.cortex_score_batch(eng.h, args[0], batch, n, None, args[1], 1.0, 0, args[2], args[3], None,
                                          None, 0)
    assert call(2, 2 ** 31 - 1) < 0 and eng.pos(0) == 0
    # of 2^31 - 1 tokens only the first ctx are read; the scores of a slot at its end are left alone
    assert call(1, 2 ** 31 - 1) == 0 and eng.pos(0) == ctx
    assert np.array_equal(lp, want.logprob[0]) and np.array_equal(ent, want.entropy[0])
    lp[:] = 7.0
    assert call(1, 5) == 0 and (lp == 7.0).all()
    eng.close()
    ref.close()


GRAD_TOL = {PREC_FP32: 2e-5, PREC_TF32: 1e-2}
KEYS = [(-1, 0), (-1, 1), (-1, 2)] + [(l, t) for l in range(2) for t in (10, 11, 12, 13, 14, 15, 16, 17)]


@pytest.mark.parametrize("precision", [PREC_FP32, PREC_TF32])
def test_distill_gradients_are_a_mix_of_the_oracles(model_dir, built, precision):
    """At temperature 1 the gradient is linear in the teacher's probabilities:
    the same list of weights at every position gives that mix of the
    cross-entropy gradients of the listed ids (of the oracle's step)."""
    V, n = 1001, 61
    p = make_model(model_dir, "tr_a.snai", V, 128, 140, 2, seed=21, std=0.08)
    rng = np.random.default_rng(4)
    x = rng.integers(0, V, n).astype(np.int32)
    ids = np.stack([rng.choice(V, 3, replace=False) for _ in range(n)]).astype(np.int32)
    y = rng.integers(0, V, n).astype(np.int32)
    q, a = np.array([0.5, 0.3, 0.2]), 0.25
    e, o = Cortex(p, num_heads=2, precision=precision), O.Oracle(p, num_heads=2)
    pad = np.concatenate([ids, np.full((n, 2), -1, dtype=np.int32)], 1)
    vals = np.broadcast_to(np.concatenate([np.log(q) + 1.7, [50.0, np.nan]]), pad.shape)  # padding holds anything
    loss = e.distill_grads(x, pad, vals, y, 1.0, a)
    want = {k: 0.0 for k in KEYS}
    lw = (1 - a) * (q * np.log(q)).sum()
    scorer = Cortex(p, num_heads=2, precision=precision)
    for w, t in [((1 - a) * q[j], ids[:, j]) for j in range(3)] + [(a, y)]:
        lw += w * o.train_grads(x, np.ascontiguousarray(t))
        # the oracle's loss is -log(p + 1e-7) (core/cortex.nim:616): 1e-7 / p below -log p
        scorer.reset()
        lw += w * 1e-7 * np.exp(-scorer.score(x[None], np.ascontiguousarray(t)[None]).logprob.astype(np.float64)).mean()
        for k in KEYS:
            want[k] = want[k] + w * o.tensor(k[0], k[1], "grad").astype(np.float64)
    assert abs(loss - lw) <= (2e-5 if precision == PREC_FP32 else 2e-3) * abs(lw)
    for k in KEYS:
        assert rel_err(e.tensor(k[0], k[1], "grad"), want[k]) < GRAD_TOL[precision], k
    scorer.close()
    e.close()
    o.close()


def test_distill_gradient_is_the_difference(model_dir, built):
    """rest, a temperature and labels: the loss's change along a direction of a weight."""
    V, n, k = 1001, 40, 12
    p = make_model(model_dir, "tr_a.snai", V, 128, 140, 2, seed=21, std=0.08)
    rng = np.random.default_rng(5)
    x = rng.integers(0, V, n).astype(np.int32)
    teacher = Cortex(make_model(model_dir, "tr_t.snai", V, 128, 140, 2, seed=22, std=0.08), num_heads=2)
    s = teacher.score(x[None], None, 2.0, k)
    e = Cortex(p, num_heads=2)
    args = (x, s.top_ids[0], s.top_logprob[0], x, 2.0, 0.3, True)
    e.distill_grads(*args)
    for key in ((-1, 1), (1, 16), (0, 12)):
        g = e.tensor(key[0], key[1], "grad").astype(np.float64)
        w = e.tensor(*key)
        d = g / np.linalg.norm(g)
        slope = (g * d).sum() / n  # of the mean loss
        # fp32 losses near 5 carry about 1e-6; a change of 2 h slope = 0.02 leaves 1e-4 of it, the third
        # derivative's h^2 the rest of the percent
        h = 0.01 / slope
        vals = []
        for sign in (1, -1):
            e.set_tensor(key[0], key[1], (w + sign * h * d).astype(np.float32))
            vals.append(e.distill_grads(*args))
        e.set_tensor(key[0], key[1], w)
        assert abs((vals[0] - vals[1]) / (2 * h) - slope) < 0.02 * slope, (key, vals, slope)
    teacher.close()
    e.close()


@pytest.mark.parametrize("precision", [PREC_FP32, PREC_BF16])
def test_teacher_scores_student_learns(model_dir, built, precision):
    """The pieces as they are used: a teacher's scores of a text train a
    student, step by step; equal steps give equal students, the padded tail of
    a batch changes nothing, and longer lists reuse the student's buffers."""
    V, n = 1001, 50
    rng = np.random.default_rng(6)
    text = rng.integers(0, V, n + 1).astype(np.int32)
    teacher = Cortex(make_model(model_dir, "tr_t.snai", V, 128, 140, 2, seed=22, std=0.08), num_heads=2,
                     precision=precision)
    path = make_model(model_dir, "tr_a.snai", V, 128, 140, 2, seed=21, std=0.08)
    students = [Cortex(path, num_heads=2, precision=precision) for _ in range(2)]
    losses = [[], []]
    for step, k in enumerate((4, 16, 4)):
        teacher.reset()
        s = teacher.score(text[None, :n], text[None, 1:], 2.0, k)
        ids, vals = s.top_ids[0], s.top_logprob[0]
        for i, st in enumerate(students):
            losses[i].append(st.distill_step(text[:n], ids, vals, 1e-3, text[1:], 2.0, 0.5, rest=True))
    assert losses[0] == losses[1] and np.isfinite(losses[0]).all()
    for k in KEYS:
        assert np.array_equal(students[0].tensor(*k), students[1].tensor(*k))
    assert students[0].train_info()["adam_steps"] == 3
    before = students[0].score(text[None, :n], text[None, 1:], 1.0, 0)
    assert np.isfinite(before.logprob).all()
    # rows of padding alone: no gradient anywhere
    loss = students[0].distill_grads(text[:n], np.full((n, 4), -1), np.zeros((n, 4)), np.full(n, -1), 1.0, 0.5)
    assert loss == 0.0
    for k in KEYS:
        assert not students[0].tensor(k[0], k[1], "grad").any()
    assert students[0].distill_grads([], np.zeros((0, 2)), np.zeros((0, 2))) == 0.0
    teacher.close()
    for st in students:
        st.close()
