"""CPU tests of the vocabulary-row operators: the 64-bit reference's
gradients against differences of its own values, and every refusal of the
entry points (arguments are checked before the GPU is touched)."""
import ctypes

import numpy as np
import pytest

from row_reference import distill_row, logp_row, score_grad_row, score_row


def differences(f, z, h=1e-5):
    out = np.zeros(len(z))
    for i in range(len(z)):
        a, b = z.copy(), z.copy()
        a[i] += h
        b[i] -= h
        out[i] = (f(a) - f(b)) / (2 * h)
    return out


# central differences of a smooth function with values of order 1: h^2 for
# the third derivative (bounded by a few hundred here: 1 / T^3) and the
# value's rounding over h
DIFF_TOL = 500 * 1e-10 + 100 * 2.0 ** -52 / 1e-5


@pytest.mark.parametrize("T", [1.0, 0.5, 2.0])
def test_reference_score_gradient_is_the_difference(T):
    rng = np.random.default_rng(1)
    z = rng.normal(0, 2, 23)
    tok, g, gh = np.array([3, 7, 3, -1, 30]), rng.normal(0, 1, 5), 0.7

    def f(x):
        lp, ent, _, _ = score_row(x, tok, T, 0)
        return float((np.where((tok >= 0) & (tok < 23), g, 0.0) * lp).sum() + gh * ent)

    got, _ = score_grad_row(z, tok, g, gh, T)
    assert np.abs(got - differences(f, z)).max() < DIFF_TOL * 10


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("T,a", [(1.0, 0.0), (2.0, 0.5), (0.5, 1.0), (1.0, 0.25)])
def test_reference_distill_gradient_is_the_difference(rest, T, a):
    rng = np.random.default_rng(2)
    z = rng.normal(0, 2, 19)
    ids = np.array([4, 9, -1, 4, 0])
    t = rng.normal(0, 2, 5)
    if rest:
        t = t - np.log(np.exp(t[[0, 1, 3, 4]]).sum()) - 0.4
    f = lambda x: distill_row(x, ids, t, 6, T, a, rest)[0]  # noqa: E731
    got = distill_row(z, ids, t, 6, T, a, rest)[1]
    assert np.abs(got - differences(f, z)).max() < DIFF_TOL * 10


def test_reference_edges():
    z = np.full(5, -np.inf)
    lp, ent, ids, top = score_row(z, [2, -1], 1.0, 2)
    assert lp.tolist() == [-np.inf, 0.0] and ent == 0.0 and ids.tolist() == [0, 1] and np.all(top == -np.inf)
    assert logp_row([1.0, np.nan], 1.0) is None and logp_row([1.0, np.inf], 1.0) is None
    assert distill_row(np.array([np.nan, 1.0]), [-1], [0.0], -1, 1.0, 0.5, False)[0] == 0.0


P = ctypes.c_void_p(1 << 20)  # never read: the refusals below come first


def score(lib, logits=P, dtype=0, rows=2, vocab=100, ld=100, tokens=P, n_tok=1, T=1.0, k=3, lp=P, ent=P, ids=P, top=P):
    return lib.cortex_score(logits, dtype, rows, vocab, ld, tokens, n_tok, T, k, lp, ent, ids, top, None)


def score_grad(lib, logits=P, dtype=0, rows=2, vocab=100, ld=100, tokens=P, n_tok=1, T=1.0, gl=P, gh=P,
               grad=ctypes.c_void_p(1 << 24), gld=100):
    return lib.cortex_score_grad(logits, dtype, rows, vocab, ld, tokens, n_tok, T, gl, gh, grad, gld, None)


def distill(lib, logits=P, dtype=0, rows=2, vocab=100, ld=100, ids=P, vals=P, k=3, labels=None, rg=None, T=1.0,
            a=0.0, rest=0, loss=P, grad=ctypes.c_void_p(1 << 24), gld=100, params=True):
    from snai_b200 import DistillParams
    prm = DistillParams(T, a, rest)
    return lib.cortex_distill(logits, dtype, rows, vocab, ld, ids, vals, k, labels, rg,
                              ctypes.byref(prm) if params else None, loss, grad, gld, None)


COMMON = [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 19) + 1, ld=1 << 20),
          dict(ld=99), dict(ld=-100), dict(T=0.0), dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")),
          dict(T=1e-4), dict(logits=None), dict(logits=ctypes.c_void_p((1 << 20) + 2)),
          dict(rows=(1 << 30) + 1), dict(rows=2 ** 31 - 1),  # rows past 2^30
          dict(rows=1 << 30, ld=1 << 20), dict(ld=(1 << 47) + 1), dict(rows=1, ld=2 ** 63 - 1)]  # offsets past any memory


@pytest.mark.parametrize("bad", COMMON + [
    dict(n_tok=-1), dict(n_tok=513), dict(k=-1), dict(k=513, vocab=600, ld=600), dict(k=101), dict(tokens=None),
    dict(lp=None), dict(ids=None), dict(top=None), dict(n_tok=0, k=0, ent=None)], ids=str)
def test_score_refuses(built, bad):
    from snai_b200 import last_error, load
    assert score(load(), **bad) < 0
    assert "cortex_score" in last_error()


@pytest.mark.parametrize("bad", COMMON + [
    dict(n_tok=-1), dict(n_tok=513), dict(tokens=None), dict(gl=None), dict(grad=None), dict(gld=99),
    dict(n_tok=0, gh=None), dict(grad=ctypes.c_void_p((1 << 24) + 2)),
    dict(grad=ctypes.c_void_p((1 << 20) + 4)),              # one element on: overlaps
    dict(grad=ctypes.c_void_p((1 << 20) + 400)),            # one row on
    dict(gld=1 << 60),
    dict(grad=P, gld=101)], ids=str)                        # same memory, other stride
def test_score_grad_refuses(built, bad):
    from snai_b200 import last_error, load
    assert score_grad(load(), **bad) < 0
    assert "cortex_score_grad" in last_error()


@pytest.mark.parametrize("bad", COMMON + [
    dict(k=0), dict(k=513), dict(ids=None), dict(vals=None), dict(loss=None), dict(a=-0.1), dict(a=1.1),
    dict(a=float("nan")), dict(a=0.5), dict(rest=2), dict(gld=99), dict(params=False),
    dict(grad=ctypes.c_void_p((1 << 20) + 4)), dict(grad=P, gld=128)], ids=str)
def test_distill_refuses(built, bad):
    from snai_b200 import last_error, load
    assert distill(load(), **bad) < 0
    assert "cortex_distill" in last_error()


def test_no_rows_is_nothing(built):
    from snai_b200 import load
    lib = load()
    assert score(lib, rows=0) == 0 and score_grad(lib, rows=0) == 0 and distill(lib, rows=0) == 0


def test_state_calls_refuse_null(built):
    from snai_b200 import DistillParams, load
    lib = load()
    assert lib.cortex_score_batch(None, None, 1, 1, None, None, 1.0, 0, None, None, None, None, 0) < 0
    loss = ctypes.c_float(0.0)
    prm = DistillParams(1.0, 0.0, 0)
    assert lib.cortex_distill_grads(None, None, None, None, 1, None, 1, ctypes.byref(prm), ctypes.byref(loss)) < 0


def test_host_tensors_are_refused(built):
    torch = pytest.importorskip("torch")
    from snai_b200 import CortexError, score_device
    with pytest.raises(CortexError):
        score_device(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32))
