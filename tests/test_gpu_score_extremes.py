"""Rows that hold both ends of a type's range: differences of two logits that
float32 cannot hold, log probabilities that it can."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from row_reference import distill_row, order, score_grad_row  # noqa: E402
from snai_b200 import distill_device, score_device, score_grad_device  # noqa: E402
from test_gpu_score import DEV, DT, LOWEST, check_grad, check_score, in_f32, on_gpu  # noqa: E402


def both_ends(rng, V, dtype):
    low = LOWEST[dtype]
    z = rng.normal(0, 2, (8, V))
    z[0, [1, V - 1]] = -low, low
    z[1], z[1, V // 2] = low, -low
    z[2], z[2, V // 3] = -low, low
    z[3, 0], z[3, 1], z[3, 2] = 0.9 * -low, 0.9 * low, -np.inf
    z[4, 2], z[4, 5] = 0.3 * -low, 0.3 * low
    z[5] = np.where(np.arange(V) % 2 == 0, low, -low)
    z[6], z[6, 3], z[6, 4] = -np.inf, -low, low
    z[7, 0] = low
    return torch.from_numpy(z.astype(np.float32)).to(DT[dtype]).double().numpy()


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T", [0.7, 1.0, 1.3, 2.0, 4.0, 1000.0])
@pytest.mark.parametrize("V", [40, 5003, 70001])
def test_both_ends_of_the_range(built, V, T, dtype):
    rng = np.random.default_rng(V)
    z = both_ends(rng, V, dtype)
    R, k = len(z), 7
    tok = np.stack([np.concatenate([order(z[r])[[0, 1, -1, -2]], [0, 1, 2, 3, 4, 5, V // 2, V // 3, V - 1]])
                    for r in range(R)]).astype(np.int32)
    t, tt = on_gpu(z, dtype, 1, 1), torch.from_numpy(tok).to(DEV)
    got = score_device(t, tt, T, k)
    check_score(z, dtype, tok, T, k, got)
    # without alternatives, and without the entropy too: other instances of the kernel
    ent = score_device(t, tt, T, 0)
    alone = score_device(t, tt, T, 0, want_entropy=False)
    for s in (ent, alone):
        check_score(z, dtype, tok, T, 0, s._replace(entropy=got.entropy))
    g, gh = rng.normal(0, 1, tok.shape).astype(np.float32), rng.normal(0, 0.3, R).astype(np.float32)
    gt, ht = torch.from_numpy(g).to(DEV), torch.from_numpy(gh).to(DEV)
    pairs = [score_grad_row(z[r], tok[r], g[r], gh[r], T) for r in range(R)]
    check_grad(score_grad_device(t, tt, gt, ht, T), np.stack([p[0] for p in pairs]), np.stack([p[1] for p in pairs]), z,
               T, dtype, 4 + 2 * np.log(V))
    # the teacher lists the two greatest and the least
    ids = tok[:, [0, 1, 3]]
    vals = np.log(np.broadcast_to([0.5, 0.3, 0.2], ids.shape)).astype(np.float32)
    rows = [distill_row(z[r], ids[r], vals[r], -1, T, 0.0, False) for r in range(R)]
    loss, grad = distill_device(t, *(torch.from_numpy(np.ascontiguousarray(x)).to(DEV) for x in (ids, vals)),
                                temperature=T)
    got = loss.double().cpu().numpy()
    for r in range(R):
        w = float(in_f32(rows[r][0]))
        # logits' differences in 64 bits, T's half step on them, and one rounding
        assert got[r] == w or abs(got[r] - w) <= 2.0 ** -22 * abs(w) + 1e-4 * max(T * T, 1.0), (r, got[r], w)
    check_grad(grad, np.stack([x[1] for x in rows]), np.stack([x[2] for x in rows]), z, min(T, 1.0), dtype)
