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


@pytest.mark.parametrize("rows,V,D,score", [(40, 300, 4096, 12), (300, 300, 4096, 12), (2048, 4096, 1024, 14)])
def test_both_passes_see_the_same_fp32_scores(cuda, rows, V, D, score):
    """The same in fp32, whose ds and dH keep 2^-19 and 2^-24 of themselves."""
    H, W, y = certain(rows, V, D, score, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    H = H.float() + torch.rand(H.shape, generator=g, device="cuda") * 2.0 ** -9  # low bits set
    W = W.float()
    W[0] *= 1.0 + torch.rand(D, generator=g, device="cuda") * 2.0 ** -9
    loss, lse = gpu.linear_cross_entropy(H, W, y, reduction="none")
    dH, _ = gpu.linear_cross_entropy_backward(H, W, y, lse, reduction="sum", need_dW=False)
    w = W[0].double()
    ds, want = dH.double() @ w / (w @ w), torch.expm1(-loss.double())
    tol = U * lse.double() + 2.0 ** -22 + 2.0 ** -18 * want.abs()
    assert bool(((ds - want).abs() <= tol).all()), float(((ds - want).abs() / tol).max())


# ------------------------------------------------------- long sums of one sign
# All scores are 0 here, so p is 1 / V everywhere.  The target's term comes last in its sum and
# takes away what the others add up to, as bf16 holds it: what is left is rounded to bf16
# so finely that the error of the sum itself shows.
def tiles_of_every_pair():
    """As many tiles of 256 columns as there are pairs of SMs: no reason to split a sum for them."""
    return torch.cuda.get_device_properties(0).multi_processor_count // 2


def positive(rows, cols, seed):
    """bf16 values of [0.5, 1.5)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
    for i in range(0, rows, 8192):
        part = out[i:i + 8192]
        part.copy_(torch.rand(part.shape, generator=g, device="cuda").add_(0.5))
    return out


def ds_of(V):
    """p and p - 1 as ds holds them.  p has bits enough for products that fill the sums' last
    ones, and lies where an error of 2^-20 does not round it another way."""
    p = float(torch.tensor(1.0 / V, dtype=torch.float64).bfloat16())
    assert abs(1.0 / V - p) * V < 2.0 ** -11 and not p.hex().startswith("0x1.0")
    return p, float(torch.tensor(1.0 / V - 1.0, dtype=torch.float64).bfloat16())


def check_sum(got, others, target):
    """Against `others` + `target` (fp64): 1024 additions (16384 k) truncated by 2^-22 of the chunk's
    sum so far, half of it on average, then a few rounded joins, and the result's rounding."""
    ref = others + target
    tol = (512 * 2.0 ** -22 + 40 * U) * others + 2.0 ** -8 * ref.abs()
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


@pytest.mark.parametrize("rows", [128, 256])
def test_long_sums_over_the_vocabulary(cuda, rows):
    V, D = 211000, 256 * tiles_of_every_pair()
    p, p1 = ds_of(V)
    W = positive(V, D, 1)
    others = p * W[:-1].sum(0, dtype=torch.float64)
    W[-1] = (-others / p1).bfloat16()
    H = torch.zeros(rows, D, device="cuda", dtype=torch.bfloat16)
    y = torch.full((rows,), V - 1, device="cuda", dtype=torch.int32)
    _, lse = gpu.linear_cross_entropy(H, W, y)
    dH, _ = gpu.linear_cross_entropy_backward(H, W, y, lse, reduction="sum", need_dW=False)
    check_sum(dH, others, p1 * W[-1].double())


def test_long_sums_over_the_rows(cuda):
    rows, V, D = 262144, 217, 256 * tiles_of_every_pair()
    p, p1 = ds_of(V)
    H = positive(rows, D, 2)
    others = p * H[:-1].sum(0, dtype=torch.float64)
    H[-1] = (-others / p1).bfloat16()
    W = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16)
    y = torch.full((rows,), 1, device="cuda", dtype=torch.int32)
    y[-1] = 0
    _, lse = gpu.linear_cross_entropy(H, W, y)
    _, dW = gpu.linear_cross_entropy_backward(H, W, y, lse, reduction="sum", need_dH=False)
    check_sum(dW[0], others, p1 * H[-1].double())


# ------------------------------------------------ operands with the low bits set
@pytest.mark.parametrize("rows", [8, 200])  # W as it lies in memory, W with a copy of its remainders
@pytest.mark.parametrize("h,w", [(1.0, 1.0 + 2.0 ** -10 - 2.0 ** -23), (1.0 + 2.0 ** -10 - 2.0 ** -20,) * 2])
def test_fp32_operands_keep_their_low_bits(cuda, rows, h, w):
    """One product per score, 64 h w, so lse is the score.  x = hi + lo, and lo rounds to tf32: 13 bits
    to 11, off by 2^-22 of w at most.  What lo lo would add is below 2^-21 of the product where one
    factor is cut to hi (lo < 2^-10) and the other rounded (2^-11); where both are cut and
    have their low bits set it would be 2^-20.  Here h rounds to 2^-20 of itself: lo lo is 2^-30.
    The sum of the three terms may lose its last bit, 2^-23."""
    V, D = 300, 64
    H, W = torch.zeros(rows, D, device="cuda"), torch.zeros(V, D, device="cuda")
    H[:, 0] = h
    W[:, 0] = -64.0
    W[5, 0] = 64.0 * w
    _, lse = gpu.linear_cross_entropy(H, W, torch.full((rows,), 5, device="cuda", dtype=torch.int32))
    err = (lse.double() / (64.0 * H[:, 0].double() * (W[5, 0].double() / 64.0)) - 1.0).abs()
    assert float(err.max()) <= (2.0 ** -22 if h == 1.0 else 2.0 ** -30 + 2.0 ** -23) + 2.0 ** -28
