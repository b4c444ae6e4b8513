"""What linear_cross_entropy's sums may lose, where a plain bound on sums of
products would not see it: targets that are all but certain, long sums of one
sign, operands with the low bits set."""
import pytest
import torch

from silarray_b200 import gpu
from tests.test_gpu_cross_entropy import U

pytestmark = pytest.mark.gpu


# ------------------------------------------------- targets that are all but certain
def certain(rows, V, D, score, seed):
    """Every row's target is entry 0 with a score of about `score`; the others' are 0."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    H = (torch.rand(rows, D, generator=g, device="cuda") + 0.5).bfloat16()
    W = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16)
    W[0] = ((torch.rand(D, generator=g, device="cuda") + 0.5) * (score / D)).bfloat16()
    return H, W, torch.zeros(rows, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("rows,V,D,score", [(40, 300, 16384, 12), (140, 300, 131072, 12), (2048, 8192, 4096, 18),
                                            (300, 300, 1000, 12)])
def test_both_passes_see_the_same_scores(cuda, rows, V, D, score):
    """ds of a target with p near 1 is -(1 - p): exp(-loss) - 1 of the forward's loss, if the
    backward's score is the forward's.  lse - score is exact there, so what is left is
    p's error, lse 2^-24 from the exponent's rounding and 2^-22 of the exponential, and
    the roundings of ds and dH to bf16, 2^-8 each.  At D = 131072 the scores themselves
    are held against fp64: 128 chunks of 64 additions, truncated by 2^-22 of the chunk's sum so
    far (half of it on average), joined by additions that round by 2^-24 of theirs."""
    H, W, y = certain(rows, V, D, score, 1)
    loss, lse = gpu.linear_cross_entropy(H, W, y, reduction="none")
    dH, _ = gpu.linear_cross_entropy_backward(H, W, y, lse, reduction="sum", need_dW=False)
    w = W[0].double()
    ds = dH.double() @ w / (w @ w)  # dH = ds_0 W_0, the others being 0
    want = torch.expm1(-loss.double())
    tol = U * lse.double() + 2.0 ** -22 + 2.0 ** -7 * want.abs()
    err = (ds - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    if D >= 131072:
        s = H.double() @ w
        ref = -1.0 / (1.0 + torch.exp(s) / (V - 1))
        one = s * (D / 1024 / 2 * U + 32.5 * 2.0 ** -22)  # of a score, in each pass
        assert bool(((ds - ref).abs() <= 2 * one + tol).all()), float((ds - ref).abs().max())
