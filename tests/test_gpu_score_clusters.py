"""Scores of rows that are spread over clusters of CTAs, several rows to a
cluster one after the other: rows of ties, whose candidates pass what the
leading CTA holds and are cut down by all of the cluster together, between
rows that need no such thing and rows without a distribution."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from row_reference import order, rel_err_bound, score_row  # noqa: E402
from snai_b200 import score_device  # noqa: E402

DEV = torch.device("cuda")


# A row goes to as many CTAs as keep all of them at twice (more than 32
# alternatives) or 5.5 times the SMs' number; clusters of 8 of 256 threads do
# not pack that densely, so the last rows of 37 are some clusters' second.
@pytest.mark.parametrize("R,V,k", [(37, 65536, 300), (37, 131072, 512), (74, 65536, 300), (148, 16384, 200),
                                   (101, 65536, 32), (100, 32768, 20), (3, 262144, 512)])
def test_ties_over_clusters_row_after_row(built, R, V, k):
    rng = np.random.default_rng(R + V + k)
    z = np.empty((R, V), dtype=np.float32)
    for r in range(R):
        kind = (r * 5 + r // 7) % 6
        if kind == 0:
            z[r] = 0.5
        elif kind == 1:
            z[r] = rng.integers(0, 2, V)
        elif kind == 2:
            z[r] = rng.normal(0, 3, V)
        elif kind == 3:
            z[r] = -np.inf
            z[r, rng.integers(0, V, 5)] = 1.0
        elif kind == 4:
            z[r] = 0.0
            z[r, rng.integers(0, V)] = np.nan
        else:
            z[r] = np.where(np.arange(V) % 16 < 8, 2.0, rng.normal(0, 1, V))
    t = torch.from_numpy(z).to(DEV)
    first = score_device(t, None, 1.0, k)
    ids = first.top_ids.cpu().numpy()
    top, ent = first.top_logprob.double().cpu().numpy(), first.entropy.double().cpu().numpy()
    for r in range(R):
        if np.isnan(z[r]).any():
            assert (ids[r] == -1).all() and np.isnan(top[r]).all() and np.isnan(ent[r])
            continue
        zd = z[r].astype(np.float64)
        assert np.array_equal(ids[r], order(zd)[:k]), r
        _, we, _, wt = score_row(zd, [], 1.0, k)
        tol = rel_err_bound(zd, 1.0)
        fin = np.isfinite(wt)
        assert np.array_equal(top[r] == -np.inf, ~fin)
        assert (np.abs(top[r][fin] - wt[fin]) <= tol + 8 * 2.0 ** -24 * np.abs(wt[fin])).all()
        assert abs(ent[r] - we) <= 2 * tol * (1.0 + np.log(V))
    for _ in range(20):
        again = score_device(t, None, 1.0, k)
        assert torch.equal(again.top_ids, first.top_ids)
        assert torch.equal(again.top_logprob.view(torch.int32), first.top_logprob.view(torch.int32))
