"""linear_cross_entropy on the GPU against its formulas in fp64.

Tolerances, from the arithmetic.  u = 2^-24.  A score is a sum of D products:
  bf16  products are exact; the tensor core adds 16 of them at a time into an
        fp32 sum that it truncates (at most 2^-22 of the terms' absolute sum
        each time): (D / 16 + 1) 2^-22
  f32   x = hi + lo: lo enters as tf32 (2^-10 of itself), and lo lo is dropped.
        |lo| is at most 2^-11 |x|, or 2^-10 |x| for a W that is cut instead of rounded:
        2^-21 + 2^-20 + 2^-21 = 2^-19; and 3 * 16 truncated additions per 128 k,
        then D / 128 rounded ones: 48 * 2^-22 + D / 128 u
of sum |h w| each; call the row's largest such error e.  lse is off by e, the
exponentials' 2^-20 (their arguments' roundings, up to 30 in size) and its own
rounding; p = exp(s - lse) by the relative sum of both; ds takes a rounding to
bf16 (half_step) there.  The gradients are sums over V or rows with the same
bounds on their products."""
import numpy as np
import pytest
import torch

from silarray_b200 import gpu
from tests.test_training_cpu import cross_entropy_ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def half_step(t):
    return torch.finfo(t).eps / 2


def product_error(n, dtype):
    """Error of a sum of n products, relative to the sum of their absolute values."""
    if dtype == torch.bfloat16:
        return (n / 16 + 1) * 2.0 ** -22
    return 2.0 ** -19 + 48 * 2.0 ** -22 + (n / 128 + 8) * U


def inside(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst "
                           f"{float((err / tol).nan_to_num(9e9).max()):.3g} x")


def make(rows, V, D, dtype, seed, left_out=0.2, std=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    H = torch.randn(rows, D, generator=g, device="cuda").to(dtype)
    W = (torch.randn(V, D, generator=g, device="cuda") * (std / D ** 0.5)).to(dtype)
    y = torch.randint(0, V, (rows,), generator=g, device="cuda", dtype=torch.int32)
    drop = torch.rand(rows, generator=g, device="cuda") < left_out
    y[drop] = torch.where(torch.arange(int(drop.sum()), device="cuda") % 2 == 0, -100, V).int()
    return H, W, y


def check(H, W, y, loss, lse, dH=None, dW=None, reduction="mean", dloss=None):
    dt = H.dtype
    rows, V = H.shape[0], W.shape[0]
    used = (y >= 0) & (y < V)
    h = torch.where(used[:, None], H.double(), torch.zeros_like(H.double())) if dH is not None else H.double()
    w = W.double()
    r = cross_entropy_ref(H.double(), w, y.long(), reduction, None if dloss is None else dloss.double())
    size = h.abs() @ w.abs().T  # sum |h w| of every score
    e = product_error(H.shape[1], dt) * size
    del size
    worst = e.amax(1)
    dlse = worst + 2.0 ** -20 + 2 * U * r["lse"].abs()
    if reduction == "none" or dH is None:
        inside(lse[used], r["lse"][used], dlse[used] * 1.01, "lse")
    loss_tol = torch.where(used, worst + dlse + 2 * U * r["row_loss"].abs(), torch.zeros_like(worst))
    if reduction == "none":
        inside(loss, r["loss"], loss_tol * 1.01, "loss")
        assert bool((loss[~used] == 0).all())
    else:
        n = max(1, int(used.sum())) if reduction == "mean" else 1
        inside(loss, r["loss"], loss_tol.sum() / n * 1.01 + 2 * U * r["loss"].abs() + 1e-30, "loss")
    if dH is None:
        return
    # ds: p relative, then its rounding to the products' operand type
    g = r["scale"].abs()[:, None]
    rel = e + (dlse + 2.0 ** -20)[:, None]
    op = half_step(torch.bfloat16) if dt == torch.bfloat16 else 2 * U
    ads = r["ds"].abs()
    dds = g * r["p"] * rel * 1.05 + ads * (op + 2 * U)
    del rel, e
    hs, os_ = dds + ads * product_error(V, dt), half_step(dt)
    inside(dH, r["dH"], hs @ w.abs() + os_ * r["dH"].abs() + 1e-30, "dH")
    hs = dds + ads * product_error(rows, dt)
    inside(dW, r["dW"], hs.T @ h.abs() + os_ * r["dW"].abs() + 1e-30, "dW")
    assert bool((dH[~used] == 0).all())
    # independent roundings of ds and of the result: together 2^-8 of the norm at most in bf16
    lim = 2.0 ** -8 if dt == torch.bfloat16 else 1e-5
    for got, ref in ((dH, r["dH"]), (dW, r["dW"])):
        n = float(ref.norm())
        assert float((got.double() - ref).norm()) <= lim * n + 1e-30


def run(H, W, y, reduction="mean", dloss=None):
    loss, lse = gpu.linear_cross_entropy(H, W, y, reduction=reduction)
    dH, dW = gpu.linear_cross_entropy_backward(H, W, y, lse, dloss=dloss, reduction=reduction)
    gpu.device_status()
    return loss, lse, dH, dW


SHAPES = [(1, 1, 1), (8, 3000, 1024), (512, 1500, 160), (513, 1500, 160), (97, 5000, 516), (3, 7, 5), (1, 1000, 64), (17, 300, 33), (128, 256, 64), (129, 257, 72), (200, 513, 100),
          (300, 2048, 8), (2, 130, 4096), (64, 5000, 768), (333, 1003, 771), (1000, 4099, 256), (700, 40, 520)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,V,D", SHAPES)
def test_loss_and_gradients(cuda, rows, V, D, dtype):
    H, W, y = make(rows, V, D, dtype, rows + V + D)
    loss, lse, dH, dW = run(H, W, y)
    check(H, W, y, loss, lse, dH, dW)
    again = run(H, W, y)
    for p, q in zip((loss, lse, dH, dW), again):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_reductions(cuda, reduction, dtype):
    H, W, y = make(150, 999, 96, dtype, 3)
    dloss = torch.randn(150, device="cuda") if reduction == "none" else torch.tensor(-1.75, device="cuda")
    if reduction == "none":
        dloss[7] = 0.0
    loss, lse, dH, dW = run(H, W, y, reduction, dloss)
    check(H, W, y, loss, lse, dH, dW, reduction, dloss)
    loss, lse = gpu.linear_cross_entropy(H, W, y, reduction=reduction)
    check(H, W, y, loss, lse, reduction=reduction)
    for need in ((True, False), (False, True)):
        got = gpu.linear_cross_entropy_backward(H, W, y, lse, dloss=dloss, reduction=reduction, need_dH=need[0],
                                                need_dW=need[1])
        for g, full, n in zip(got, (dH, dW), need):
            assert (g is None) if not n else torch.equal(g, full)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,V,D,piece", [(300, 1500, 200, 256), (130, 1025, 64, 512), (40, 5000, 65, 1024),
                                            (600, 900, 520, 256), (100, 3000, 64, 512), (1, 2000, 160, 256)])
def test_vocabulary_pieces(cuda, monkeypatch, rows, V, D, piece, dtype):
    """The same result from several pieces, a short last one among them."""
    H, W, y = make(rows, V, D, dtype, V)
    monkeypatch.setenv("SILCU_LOSS_PIECE", str(piece))
    check(H, W, y, *run(H, W, y))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,V,D", [(31, 1200, 100), (128, 600, 264), (129, 600, 264)])
def test_one_gradient_alone(cuda, rows, V, D, dtype):
    """dH or dW by itself is what both together give, and nothing past its rows or columns is written."""
    H, W, y = make(rows, V, D, dtype, 8)
    _, lse, dH, dW = run(H, W, y)
    for i, full in enumerate((dH, dW)):
        wide = torch.full((full.shape[0] + 2, D + 24), 7.0, device="cuda", dtype=dtype)
        out = wide[1:-1, 8:-16]
        kw = {"need_dW": False, "dH": out} if i == 0 else {"need_dH": False, "dW": out}
        got = gpu.linear_cross_entropy_backward(H, W, y, lse, **kw)
        assert got[1 - i] is None and torch.equal(out, full)
        out.fill_(7.0)
        assert bool((wide == 7.0).all())


@pytest.mark.parametrize("dtype,rows,V,D", [(torch.bfloat16, 8192, 70001, 64), (torch.float32, 8192, 20011, 64)])
def test_many_rows(cuda, dtype, rows, V, D):
    """Sizes that need several pieces and the split of a product's long axis by themselves."""
    H, W, y = make(rows, V, D, dtype, 11)
    check(H, W, y, *run(H, W, y))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_strided_operands_and_outputs(cuda, dtype, shift):
    """Operands and gradients as column ranges of wider matrices, aligned and
    not; nothing around the gradients changes."""
    rows, V, D = 140, 700, 104
    H0, W0, y = make(rows, V, D, dtype, 21)
    HB, WB = torch.randn(rows, 128, device="cuda").to(dtype), torch.randn(V, 136, device="cuda").to(dtype)
    H, W = HB[:, shift:shift + D], WB[:, shift:shift + D]
    H.copy_(H0), W.copy_(W0)
    loss, lse = gpu.linear_cross_entropy(H, W, y)
    gh, gw = torch.full((rows + 3, 128), 5.0, device="cuda", dtype=dtype), torch.full((V + 3, 136), 5.0, device="cuda",
                                                                                       dtype=dtype)
    dH, dW = gh[:rows, shift:shift + D], gw[:V, shift:shift + D]
    gpu.linear_cross_entropy_backward(H, W, y, lse, dH=dH, dW=dW)
    check(H, W, y, loss, lse, dH, dW)
    for full, n in ((gh, rows), (gw, V)):
        assert bool((full[n:] == 5).all()) and bool((full[:, :shift] == 5).all()) and bool((full[:, shift + D:] == 5).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_rows_left_out(cuda, dtype):
    """Left-out rows may hold anything: NaN and infinities there reach neither
    the loss nor a gradient.  With no row left in, the loss and all gradients are zero."""
    H, W, y = make(200, 600, 72, dtype, 5, left_out=0.5)
    clean = run(H, W, y)
    used = (y >= 0) & (y < 600)
    bad = H.clone()
    bad[~used] = float("nan")
    bad[int((~used).nonzero()[0]), 3] = float("inf")
    dirty = run(bad, W, y)
    assert torch.equal(dirty[0], clean[0]) and torch.equal(dirty[1][used], clean[1][used])
    assert torch.equal(dirty[2], clean[2]) and torch.equal(dirty[3], clean[3])
    loss, lse, dH, dW = run(bad, W, torch.full_like(y, -1))
    assert float(loss) == 0 and bool((dH == 0).all()) and bool((dW == 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [40, 300])
def test_every_left_out_target_alike(cuda, rows, dtype):
    """The vocabulary's size, the smallest and the largest int32 leave a row out just as -1 does."""
    H, W, y = make(rows, 600, 72, dtype, 6, left_out=0.5)
    out = ~((y >= 0) & (y < 600))
    y[out] = -1
    want = run(H, W, y)
    for t in (600, -2 ** 31, 2 ** 31 - 1, -100):
        y[out] = t
        for p, q in zip(run(H, W, y), want):
            assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_bad_values_in_rows_that_count(cuda, dtype):
    H, W, y = make(130, 600, 72, dtype, 6, left_out=0.0)
    H[4, 5] = float("nan")
    loss, lse = gpu.linear_cross_entropy(H, W, y, reduction="none")
    keep = torch.arange(130, device="cuda") != 4
    assert torch.isnan(loss[4]) and torch.isnan(lse[4]) and bool(torch.isfinite(loss[keep]).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_saturated_softmax(cuda, dtype):
    """Scores thousands apart: one exponential is 1, the others vanish, the
    running maximum moves in every part."""
    rows, V, D = 40, 1000, 64
    H, W, y = make(rows, V, D, dtype, 8, left_out=0.0)
    H = (H * 300).to(dtype)
    loss, lse = gpu.linear_cross_entropy(H, W, y, reduction="none")
    check(H, W, y, loss, lse, reduction="none")
    W[:, 0], H[:, 0] = torch.arange(V, device="cuda") * 0.5, 1.0  # maxima that rise along the vocabulary
    W = W.to(dtype)
    loss, lse = gpu.linear_cross_entropy(H, W, y, reduction="none")
    check(H, W, y, loss, lse, reduction="none")


def test_no_rows(cuda):
    H, W = torch.empty(0, 16, device="cuda"), torch.randn(50, 16, device="cuda")
    y = torch.empty(0, dtype=torch.int32, device="cuda")
    loss, lse = gpu.linear_cross_entropy(H, W, y)
    dH, dW = gpu.linear_cross_entropy_backward(H, W, y, lse)
    assert float(loss) == 0 and lse.numel() == 0 and dH.shape == (0, 16) and bool((dW == 0).all())


def test_gradient_against_differences(cuda):
    """<dH, v> and <dW, v> equal the central difference of the fp64 loss along v."""
    H, W, y = make(9, 77, 24, torch.float32, 31)
    _, _, dH, dW = run(H, W, y)
    g = torch.Generator(device="cuda").manual_seed(1)
    t = 1e-5
    for which, grad in (("H", dH), ("W", dW)):
        v = torch.randn(grad.shape, generator=g, device="cuda", dtype=torch.float64)

        def f(s):
            h, w = H.double(), W.double()
            h, w = (h + s * v, w) if which == "H" else (h, w + s * v)
            return cross_entropy_ref(h, w, y.long(), "mean", None)["loss"]
        slope = float((f(t) - f(-t)) / (2 * t))
        terms = float((grad.double() * v).abs().sum())
        # the gradient's own bound (product_error is ~1.3e-5 of its terms' sizes, which cancel
        # up to ten times here); the difference is good to t^2 and 1e-15 / t
        assert abs(float((grad.double() * v).sum()) - slope) <= 2e-4 * terms + 1e-9


def test_python_refusals(cuda):
    H, W, y = make(8, 40, 16, torch.float32, 1)
    _, lse = gpu.linear_cross_entropy(H, W, y)
    with pytest.raises(TypeError):
        gpu.linear_cross_entropy(H, W.bfloat16(), y)
    with pytest.raises(TypeError):
        gpu.linear_cross_entropy(H, W, y.long())
    with pytest.raises(TypeError):
        gpu.linear_cross_entropy(H.half(), W.half(), y)
    with pytest.raises(ValueError):
        gpu.linear_cross_entropy(H, W[:, :8], y)
    with pytest.raises(ValueError):
        gpu.linear_cross_entropy(H.T.contiguous().T, W, y)
    with pytest.raises(ValueError):
        gpu.linear_cross_entropy(H, W, y[:4])
    with pytest.raises(ValueError):
        gpu.linear_cross_entropy(H, W, y, reduction="median")
    with pytest.raises(ValueError):
        gpu.linear_cross_entropy_backward(H, W, y, lse[:3])
    with pytest.raises(ValueError):
        gpu.linear_cross_entropy_backward(H, W, y, lse, dloss=torch.ones(8, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_two_graphs_at_once(cuda, dtype):
    """Two captured steps replayed together on two streams equal eager calls."""
    sets = [make(300, 2000, 128, dtype, s) for s in (1, 2)]
    refs = [[t.clone() for t in run(*s)] for s in sets]
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                loss, lse = gpu.linear_cross_entropy(*s)
                outs.append([loss, lse, *gpu.linear_cross_entropy_backward(*s, lse)])
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    gpu.device_status()
    for got, ref in zip(outs, refs):
        for p, q in zip(got, ref):
            assert torch.equal(p, q)
