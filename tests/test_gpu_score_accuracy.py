"""How near the sums' results come, in the mean over many rows: errors that
every row has alike (a temperature's rounding, the hardware's 2^x) show there
far below a single row's roundings.  64-bit definitions on the GPU."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA GPU", allow_module_level=True)

from snai_b200 import distill_device, score_device, score_grad_device  # noqa: E402

DEV = torch.device("cuda")
U32 = 2.0 ** -24


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# float32's log2(e) / T is off by -5.0e-8, 4.9e-8, 4.8e-8 of itself at these, 1 / T by 0.8e-8, 1.5e-8, 3.7e-8
@pytest.mark.parametrize("T", [0.69, 1.25, 2.69])
def test_log_probabilities_carry_the_temperature(built, T):
    """Logits about 9 T below the top one have nearly all of the mass.  A
    temperature off by 5e-8 would move every log p by 5e-8 * 8, one of 1 / T
    off by 3.7e-8 those of the bulk by 3.7e-8 * 9: both above 3e-7.  Left are
    the mean error of 2^x (5.2e-8), of the sums' and results' roundings none
    in the mean: their 4.8e-7 a value at most is below 1e-8 over 16384."""
    R, V, n = 1024, 65536, 16
    g = generator(3)
    z = (torch.rand(R, V, generator=g, device=DEV) - 0.5) * T
    z[:, 17] += 9.0 * T
    tok = torch.randint(18, V, (R, n), generator=g, device=DEV, dtype=torch.int32)
    got = score_device(z, tok, T)
    lp = torch.log_softmax(z.double() / T, 1)
    err = got.logprob.double() - lp.gather(1, tok.long())
    assert abs(err.mean().item()) < 1.5e-7, err.mean().item()
    # a value: its own rounding and its parts' (12 at most), the terms' roundings within log S
    assert err.abs().max().item() < 24 * U32 + 2e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [0.7, 1.0, 1.25])
def test_small_losses_are_not_the_difference_of_rounded_ones(built, T, dtype):
    """A student near its teacher, the rest as one outcome: a loss of some 1e-3
    between terms of several units.  2^x is low by 5e-8 in the mean in the
    terms below a part's greatest; log2(e) / T is rounded.  Left as they are,
    the first moves the mean loss by 2e-8 and the second by up to 2e-8 (at 1.25, whose
    rounding is the largest, by more).  With both taken care of there remain
    2^x's 2e-9 between its arguments' ranges and the losses' own roundings,
    some 5e-8 a row: 2e-9 in the mean over 1024, and four times that."""
    R, V, k = 1024, 16384, 64
    g = generator(1)
    z = (torch.randn(R, V, generator=g, device=DEV) * 3).to(dtype)
    teacher = z.double() + torch.randn(R, V, generator=g, device=DEV, dtype=torch.float64) * 0.05
    val, ids = torch.topk(teacher, k, 1)
    lv = torch.log_softmax(teacher / T, 1).gather(1, ids).float()
    p = torch.softmax(z.double() / T, 1)
    lq, lp = lv.double(), torch.log_softmax(z.double() / T, 1).gather(1, ids)
    q = lq.exp()
    r, u = 1 - q.sum(1), p.scatter(1, ids, 0.0).sum(1)
    want = (q * (lq - lp)).sum(1) + r * (r / u).log()
    got, _ = distill_device(z, ids.int(), lv, temperature=T, rest=True)
    err = got.double() / (T * T) - want
    assert abs(err.mean().item()) < 1.0e-8, err.mean().item()
    # a row: half a step of S at most 16 times over (log S and the unlisted sum's take most of each other's)
    assert err.abs().max().item() < 16 * U32, err.abs().max().item()


@pytest.mark.parametrize("R,V,dtype", [(600, 524288, torch.float32), (700, 131072, torch.float32),
                                       (600, 300001, torch.bfloat16), (2, 524288, torch.float32)])
def test_sums_over_long_rows(built, R, V, dtype):
    """A row in one CTA of 128 threads adds V / 256 terms one after the other
    in each of a pair's halves, then 2 + 5 + 2 partial sums: as many half steps
    relative to S at most, with 2^x's 2^-22 and its argument's rounding (a
    logit here is at most 40 below the top: 3 * 40 half steps)."""
    g = generator(V)
    z = (torch.randn(R, V, generator=g, device=DEV) * 2).to(dtype)
    tok = torch.randint(0, V, (R, 2), generator=g, device=DEV, dtype=torch.int32)
    got = score_device(z, tok, 1.0, 8)
    grad = score_grad_device(z, tok, torch.ones(R, 2, device=DEV), torch.ones(R, device=DEV))
    tol = U32 * (V / 256 + 9 + 4 + 3 * 40)
    eps = torch.finfo(dtype).eps / 2
    for lo in range(0, R, 50):
        zd = z[lo:lo + 50].double()
        lp = torch.log_softmax(zd, 1)
        p = lp.exp()
        t = tok[lo:lo + 50].long()
        want = lp.gather(1, t)
        # log S, and the value's rounding with its parts'
        assert ((got.logprob[lo:lo + 50].double() - want).abs() <= tol + 2 * U32 * want.abs()).all()
        ent = -(p * lp).sum(1)
        # W / S: each sum's terms of one sign, W = sum e |x| <= 40 S at most, here its own H + log S
        assert ((got.entropy[lo:lo + 50].double() - ent).abs() <= tol * (2 + 2 * (ent + math.log(V)))).all()
        ids = zd.topk(8, 1).values
        assert torch.equal(zd.gather(1, got.top_ids[lo:lo + 50].long()), ids)
        d = torch.zeros_like(p).scatter_add_(1, t, torch.ones_like(want)) - 2 * p - p * (lp + ent[:, None])
        # p's and (log p + H)'s relative errors, one rounding
        mag = 2 * p + p * (lp.abs() + ent[:, None] + 1)
        mag.scatter_add_(1, t, torch.ones_like(want))
        bound = mag * tol * (4 + 2 * math.log(V)) + eps * d.abs() * 1.001 + 1e-35
        assert ((grad[lo:lo + 50].double() - d).abs() <= bound).all()
