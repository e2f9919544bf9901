"""What the Python binding of the vocabulary-row operators refuses by itself:
sizes that an int of the C interface would take modulo 2^32, and lists,
labels and inputs of a distillation step that do not go together."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from snai_b200 import Cortex, CortexError, distill_device, score_device, score_grad_device  # noqa: E402


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
