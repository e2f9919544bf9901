"""More refusals of the vocabulary-row operators, the Python binding's own first:
sizes that an int of the C interface would take modulo 2^32, and lists,
labels and inputs of a distillation step that do not go together; then
addresses that the GPU cannot read."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from snai_b200 import Cortex, CortexError, distill_device, score_device, score_grad_device  # noqa: E402
from test_score_cpu import distill, score, score_grad  # noqa: E402


class Rows:
    """Stands for CUDA logits of a shape that no test can hold; nothing of it is read before it is refused."""

    is_cuda, dtype, device = True, torch.bfloat16, torch.device("cuda", 0)

    def __init__(self, *shape):
        self.shape = torch.Size(shape)

    def dim(self):
        return 2

    def stride(self):
        return self.shape[1], 1

    def __getattr__(self, name):
        raise AssertionError(f"{name} was read")


@pytest.mark.parametrize("shape", [(2 ** 32 + 5, 1), (2 ** 31, 4), (1, 2 ** 32 + 100)], ids=str)
def test_sizes_past_an_int_are_refused(shape):
    z, ids = Rows(*shape), Rows(shape[0], 3)
    for call in (lambda: score_device(z, None), lambda: score_grad_device(z, None, None, z),
                 lambda: distill_device(z, ids, ids)):
        with pytest.raises(CortexError, match="does not fit"):
            call()


@pytest.mark.parametrize("k", [2 ** 32 + 5, -(2 ** 32) + 1, 2 ** 31])
def test_alternatives_past_an_int_are_refused(k):
    with pytest.raises(CortexError, match="top_k"):
        score_device(Rows(4, 100), None, 1.0, k)
    state = object.__new__(Cortex)  # refused before the state is used
    state.lib = state.h = None
    with pytest.raises(CortexError, match="top_k"):
        state.score(np.ones((1, 3), dtype=np.int32), None, 1.0, k)


@pytest.mark.parametrize("inputs,ids,vals,labels", [
    ((5,), (5, 3), (5, 3), (5, 2)),  # two labels a position
    ((5,), (5, 3), (5, 3), (4,)),
    ((5, 2), (5, 3), (5, 3), None),  # two inputs a position
    ((1, 5), (5, 3), (5, 3), None),
    ((5,), (5,), (5,), None),
    ((5,), (5, 3), (5, 2), None),
    ((5,), (4, 3), (4, 3), None),
], ids=str)
def test_distillation_arrays_go_together(inputs, ids, vals, labels):
    state = object.__new__(Cortex)
    state.lib = state.h = None
    with pytest.raises(CortexError, match="do not match"):
        state.distill_grads(np.ones(inputs, dtype=np.int32), np.ones(ids, dtype=np.int32),
                            np.zeros(vals, dtype=np.float32), None if labels is None else np.ones(labels, dtype=np.int32),
                            1.0, 0.0 if labels is None else 0.5)


ODD = ctypes.c_void_p((1 << 21) + 2)


@pytest.mark.parametrize("call,name,kw", [
    (score, "tokens", dict(tokens=ODD)), (score, "logprob", dict(lp=ODD)), (score, "entropy", dict(ent=ODD)),
    (score, "top_ids", dict(ids=ODD)), (score, "top_logprob", dict(top=ODD)),
    (score_grad, "tokens", dict(tokens=ODD)), (score_grad, "g_logprob", dict(gl=ODD)),
    (score_grad, "g_entropy", dict(gh=ODD)),
    (distill, "teacher_ids", dict(ids=ODD)), (distill, "teacher_logits", dict(vals=ODD)),
    (distill, "labels", dict(labels=ODD, a=0.5)), (distill, "row_grad", dict(rg=ODD)), (distill, "loss", dict(loss=ODD)),
], ids=str)
def test_odd_addresses_are_refused(built, call, name, kw):
    """They would fault the GPU."""
    from snai_b200 import last_error, load
    assert call(load(), **kw) == -2
    assert name in last_error() and "aligned" in last_error()
