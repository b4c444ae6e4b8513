"""layer_norm's training pair and the gradient norm on the GPU, against the
formulas in fp64 on the same inputs.

Tolerances count roundings.  u = 2^-24 is half a step of fp32; a sum of n
terms along a chain of d additions is off by at most d u sum|terms|.  A
result stored as type T is off by finfo(T).eps / 2 of itself more."""
import numpy as np
import pytest
import torch

from silarray_b200 import gpu
from tests.test_training_cpu import ln_backward_ref, ln_forward_ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16]


def half_step(t):
    return torch.finfo(t).eps / 2


def ln_depth(cols):
    """Additions on the way of one element into a row's sum: at most 32 in a
    thread (cols / 512 beyond 16384 columns), 5 in its warp, 16 over warps."""
    return 53 + (cols // 512 if cols > 16384 else 0)


def check(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float((err / tol).nan_to_num(9e9).max()):.3g} x"


def make_ln(rows, cols, dtype, seed, shift=0):
    """x, dy, residual gradient, gamma, beta; `shift` elements off a 16-byte boundary."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def n(std, mean=0.0, t=dtype, size=rows * cols):
        buf = torch.randn(size + shift, generator=g, device="cuda").mul_(std).add_(mean).to(t)
        return buf[shift:]
    x, dy, dr = (n(2.0, 0.5).view(rows, cols), n(1.0).view(rows, cols), n(1.0).view(rows, cols))
    return x, dy, dr, n(0.1, 1.0, torch.float32, cols), n(0.1, 0.0, torch.float32, cols)


def check_forward(x, gamma, beta, out, mean, rstd, eps):
    cols = x.shape[1]
    d = ln_depth(cols)
    r_out, r_mean, r_rstd = ln_forward_ref(x.double(), gamma.double(), beta.double(), eps)
    ax = x.double().abs()
    dm = (d + 2) * U * ax.mean(1)  # the mean's error
    check(mean, r_mean, dm + 1e-30, "mean")
    # (x - mean)^2 carries 2 |x - mean| dm of it; the sum d u; 1 / sqrt halves; 6 more roundings
    var = (x.double() - r_mean[:, None]).square().mean(1)
    dev = (x.double() - r_mean[:, None]).abs()
    dvar = (d + 4) * U * var + 2 * (dm + U * dev.mean(1)) * dev.mean(1) + dm * dm
    dr = r_rstd * (0.5 * dvar / (var + eps) + 6 * U)
    check(rstd, r_rstd, dr * 1.01 + 1e-30, "rstd")
    xh = dev * r_rstd[:, None]
    tol = gamma.double().abs() * (xh * (dr / r_rstd + 4 * U)[:, None] + (dm * r_rstd)[:, None])
    tol = tol * 1.01 + (2 * U + half_step(out.dtype)) * r_out.abs() + 1e-30
    check(out, r_out, tol, "out")


def check_backward(x, dy, dres, gamma, mean, rstd, din, dgamma, dbeta):
    rows, cols = x.shape
    d = ln_depth(cols)
    r_dx, r_dg, r_db = ln_backward_ref(dy.double(), x.double(), mean.double(), rstd.double(), gamma.double(),
                                       None if dres is None else dres.double())
    xh = ((x.double() - mean.double()[:, None]) * rstd.double()[:, None]).abs()
    a = (dy.double() * gamma.double()).abs()
    s1, s2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    tol = rstd.double()[:, None] * U * ((d + 10) * (s1 + xh * s2) + 8 * a)
    if dres is not None:
        tol = tol + U * (r_dx.abs() + dres.double().abs())
    check(din, r_dx, tol + (2 * U + half_step(din.dtype)) * r_dx.abs() + 1e-30, "din")
    # a thread's rows (over 148 CTAs or more), 8 groups, then 32 slices of at most 12 * 148 partials
    chain = rows // 148 + 8 + 12 * 148 // 32 + 32 + 6
    check(dgamma, r_dg, chain * U * (dy.double().abs() * xh).sum(0) + 1e-30, "dgamma")
    check(dbeta, r_db, chain * U * dy.double().abs().sum(0) + 1e-30, "dbeta")


LN_SHAPES = [(1, 1), (3, 5), (1, 768), (37, 256), (9, 300), (700, 512), (6000, 768), (5, 771), (333, 1024),
             (20, 1023), (64, 2048), (31, 2047), (700, 4096), (13, 4090), (33, 8192), (7, 8191), (650, 16384),
             (5, 16383), (3, 16388), (40, 20001)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", LN_SHAPES)
def test_layer_norm_pair(cuda, rows, cols, dtype):
    x, dy, dr, gamma, beta = make_ln(rows, cols, dtype, rows * 31 + cols)
    eps = 1e-5
    out, mean, rstd = gpu.layer_norm_forward(x, gamma=gamma, beta=beta, eps=eps)
    check_forward(x, gamma, beta, out, mean, rstd, eps)
    for dres in (None, dr):
        got = gpu.layer_norm_backward(dy, x, mean, rstd, gamma, dresidual=dres)
        check_backward(x, dy, dres, gamma, mean, rstd, *got)
        again = gpu.layer_norm_backward(dy, x, mean, rstd, gamma, dresidual=dres)
        for p, q in zip(got, again):
            assert torch.equal(p, q)  # a fixed order of sums


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(50, 768), (9, 4096), (3, 8192)])
def test_layer_norm_unaligned_and_in_place(cuda, rows, cols, dtype):
    """Operands off 16-byte boundaries, outputs in the middle of a larger
    buffer whose surroundings stay as they were, and outputs over inputs."""
    x, dy, dr, gamma, beta = make_ln(rows, cols, dtype, cols, shift=1)
    n = rows * cols
    buf = torch.full((n + 77,), 7.0, device="cuda", dtype=dtype)
    out, mean, rstd = gpu.layer_norm_forward(x, buf[33:33 + n], gamma=gamma, beta=beta)
    check_forward(x, gamma, beta, out.view(rows, cols), mean, rstd, 1e-5)
    assert bool((buf[:33] == 7).all()) and bool((buf[33 + n:] == 7).all())
    same = x.clone()
    gpu.layer_norm_forward(same, same, gamma=gamma, beta=beta)
    apart, _, _ = gpu.layer_norm_forward(x.clone(), gamma=gamma, beta=beta)  # the same element-wise variant
    assert torch.equal(same, apart)
    aligned = gpu.layer_norm_forward(x.clone(), gamma=gamma.clone(), beta=beta.clone())  # the vector one
    check_forward(x, gamma, beta, *aligned, 1e-5)
    ref = gpu.layer_norm_backward(dy, x, mean, rstd, gamma, dresidual=dr)
    check_backward(x, dy, dr, gamma, mean, rstd, *ref)
    for k in range(3):
        ops = [dy.clone(), x.clone(), dr.clone()]
        plain = gpu.layer_norm_backward(*ops[:2], mean, rstd, gamma, dresidual=ops[2])
        got = gpu.layer_norm_backward(*ops[:2], mean, rstd, gamma, dresidual=ops[2], din=ops[k])
        assert got[0].data_ptr() == ops[k].data_ptr()
        for p, q in zip(got, plain):
            assert torch.equal(p.reshape(-1), q.reshape(-1))


def test_layer_norm_gradient_against_differences(cuda):
    """d/dt sum(w * layer_norm(x + t v)) by a central difference in fp64 of
    the formula equals <dx, v>, and the same for gamma and beta."""
    rows, cols = 4, 96
    x, w, _, gamma, beta = make_ln(rows, cols, torch.float32, 5)
    _, mean, rstd = gpu.layer_norm_forward(x, gamma=gamma, beta=beta)
    dx, dg, db = gpu.layer_norm_backward(w, x, mean, rstd, gamma)
    gen = torch.Generator(device="cuda").manual_seed(6)
    t = 1e-5
    X, G, B, Wd = x.double(), gamma.double(), beta.double(), w.double()
    for which, grad in (("x", dx), ("gamma", dg), ("beta", db)):
        v = torch.randn(grad.shape, generator=gen, device="cuda", dtype=torch.float64)

        def f(s):
            args = {"x": X, "gamma": G, "beta": B}
            args[which] = args[which] + s * v
            return (ln_forward_ref(args["x"], args["gamma"], args["beta"], 1e-5)[0] * Wd).sum()
        slope = float((f(t) - f(-t)) / (2 * t))
        got = float((grad.double() * v).sum())
        scale = float((grad.double() * v).abs().sum())
        # fp32 gradient: at most ~100 u of its terms; the difference is good to t^2 and 1e-16 / t
        assert abs(got - slope) <= (100 * U + 1e-8) * scale


def test_layer_norm_bad_rows_stay_alone(cuda):
    """A row of NaN or infinities spoils that row and the weights' gradients
    only; a row of zeros (variance 0) is fine."""
    x, dy, _, gamma, beta = make_ln(24, 512, torch.float32, 9)
    x[3] = float("nan")
    x[5, 7] = float("inf")
    x[6] = 0.0
    out, mean, rstd = gpu.layer_norm_forward(x, gamma=gamma, beta=beta)
    keep = torch.ones(24, dtype=torch.bool)
    keep[[3, 5]] = False
    assert torch.isnan(out[3]).all() and torch.isnan(out[5]).all() and torch.isfinite(out[keep]).all()
    check_forward(x[keep], gamma, beta, out[keep], mean[keep], rstd[keep], 1e-5)
    dx, dg, _ = gpu.layer_norm_backward(dy, x, mean, rstd, gamma)
    assert torch.isfinite(dx[keep]).all() and torch.isnan(dx[3]).all() and torch.isnan(dg).all()


def test_layer_norm_no_rows(cuda):
    gamma = torch.ones(16, device="cuda")
    e = torch.empty(0, 16, device="cuda")
    out, mean, rstd = gpu.layer_norm_forward(e, gamma=gamma, beta=gamma, rows=0, cols=16)
    assert out.numel() == mean.numel() == rstd.numel() == 0
    dg = torch.full((16,), 5.0, device="cuda")
    _, dg, db = gpu.layer_norm_backward(e, e, mean, rstd, gamma, rows=0, cols=16, dgamma=dg)
    assert bool((dg == 0).all()) and bool((db == 0).all())


# ---------------------------------------------------------- norm and clipping
def make_list(sizes, dtypes, seed, std=1.0, shift=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        t = dtypes[i % len(dtypes)]
        out.append(torch.randn(n + shift, generator=g, device="cuda").mul_(std).to(t)[shift:])
    return out


def norm64(ts):
    return float(sum(float(t.double().square().sum()) for t in ts) ** 0.5)


LISTS = [[1], [3, 0, 5], [255, 256, 257], [768 * 768, 768, 768, 3 * 768], [1] * 70, [17] * 1500,
         [4097] * 65, [1 << 22, 1, 1 << 20, 12345], [3000001, 7, 7, 999]]


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("kinds", [DTYPES[:1], DTYPES[1:], DTYPES], ids=["f32", "bf16", "mixed"])
@pytest.mark.parametrize("sizes", LISTS, ids=[f"{len(s)}x{max(s)}" for s in LISTS])
def test_norm_and_clip(cuda, sizes, kinds, shift):
    ts = make_list(sizes, kinds, len(sizes) + shift, 0.3, shift)
    ref = norm64(ts)
    norm = float(gpu.grad_norm(ts))
    # at most 8 squares of a vector and 3 of its neighbours add in fp32: 10 u of a sum of positive
    # terms, halved by the root; stored in fp32
    assert abs(norm - ref) <= 6 * U * ref
    for max_norm in (0.37 * ref, 10 * ref):
        c = min(1.0, max_norm / (ref + 1e-6))
        outs = [torch.full_like(t, 9.0) for t in ts]
        n2 = gpu.clip_grad_norm(ts, max_norm, OUT=outs)
        # copies at the same offset from a 16-byte boundary, so that sums group alike
        inplace = [torch.empty(t.numel() + shift, device="cuda", dtype=t.dtype)[shift:].copy_(t) for t in ts]
        n3 = gpu.clip_grad_norm(gpu.TensorList(inplace), max_norm)
        assert float(n2) == norm == float(n3)
        for t, o, i in zip(ts, outs, inplace):
            want = t.double() * c
            # the factor: the norm's 6 u and its own rounding; then the product's
            tol = want.abs() * (8 * U + half_step(t.dtype)) + 1e-40
            check(o, want, tol, "clipped")
            assert torch.equal(o, i)
            if c == 1.0:
                assert torch.equal(o, t)


def test_clip_leaves_the_surroundings(cuda):
    """Tensors that share one buffer with gaps: the gaps stay as they were."""
    buf = torch.full((5000,), 3.0, device="cuda", dtype=torch.bfloat16)
    cuts = [(1, 700), (703, 704), (1000, 3001), (3005, 4990)]
    keep = torch.ones(5000, dtype=torch.bool, device="cuda")
    for a, b in cuts:
        keep[a:b] = False
    gpu.clip_grad_norm([buf[a:b] for a, b in cuts], 1.0)
    assert bool((buf[keep] == 3).all()) and bool((buf[~keep] < 1).all())


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e19, 1e25, 3e38])
def test_norm_keeps_its_range(cuda, scale):
    """Elements whose squares overflow or vanish in fp32."""
    ts = [torch.full((n,), scale, device="cuda") for n in (5, 4096, 33333)]
    ts[1][::2] = 1.0 if scale > 1 else 0.0
    ref = norm64(ts)
    got = float(gpu.grad_norm(ts))
    assert abs(got - ref) <= 6 * U * ref if ref < 3.4e38 else got == float("inf")


def test_norm_of_bad_values(cuda):
    ts = make_list([1000, 70000], DTYPES[:1], 3)
    ts[1][777] = float("inf")
    outs = [torch.empty_like(t) for t in ts]
    assert float(gpu.clip_grad_norm(ts, 1.0, OUT=outs)) == float("inf")
    assert bool((outs[0] == 0).all()) and torch.isnan(outs[1][777]) and int(torch.isnan(outs[1]).sum()) == 1
    ts[0][1] = float("nan")
    assert np.isnan(float(gpu.grad_norm(ts)))
    gpu.clip_grad_norm(ts, 1.0, OUT=outs)
    assert all(bool(torch.isnan(o).all()) for o in outs)
    zero = [torch.zeros(100, device="cuda")]
    assert float(gpu.clip_grad_norm(zero, 1.0)) == 0 and bool((zero[0] == 0).all())
    assert float(gpu.clip_grad_norm([torch.ones(4, device="cuda")], 0.0)) == 2.0
    gpu.clip_grad_norm(zero, 0.0, eps=0.0)
    assert bool((zero[0] == 0).all())


def test_overlapping_lists(cuda):
    """The norm counts a tensor as often as it is listed; clipping refuses
    tensors, or outputs, that overlap."""
    buf = torch.ones(1000, device="cuda")
    a, b = buf[:600], buf[500:]
    assert abs(float(gpu.grad_norm([a, a])) - 1200 ** 0.5) <= 6 * U * 1200 ** 0.5
    c, d = torch.ones(600, device="cuda"), torch.ones(500, device="cuda")
    for tensors, out in (([a, b], None), ([a, a], None), ([a, d], [b[:0].new_empty(600), a[:500]]), ([c, d], [a, b]),
                         ([c, c.clone()], [c.clone(), c])):
        with pytest.raises(ValueError):
            gpu.clip_grad_norm(tensors, 1.0, OUT=out)
    tl = gpu.TensorList([c, d])
    gpu.clip_grad_norm(tl, 1.0, OUT=[c, torch.empty_like(d)])  # an output that is its own input is fine
    assert bool((buf == 1).all()) and bool((d == 1).all()) and bool((c < 1).all())


def test_tensor_list_follows_its_tensors(cuda):
    """A tensor given new storage is seen at the next call."""
    a, b = torch.ones(100, device="cuda"), torch.ones(300, device="cuda")
    tl = gpu.TensorList([a, b])
    assert float(gpu.grad_norm(tl)) == 20.0
    b.data = torch.full((300,), 3.0, device="cuda")
    assert abs(float(gpu.grad_norm(tl)) - (100 + 2700) ** 0.5) < 1e-4


def test_tensor_list_sees_other_views(cuda):
    """The same storage read as another type, or with gaps, is checked again."""
    a = torch.full((100,), 2.0, device="cuda")
    tl = gpu.TensorList([a])
    assert float(gpu.grad_norm(tl)) == 20.0
    whole = a.data
    a.data = whole.view(torch.int32)
    with pytest.raises(TypeError):
        gpu.grad_norm(tl)
    a.data = torch.empty_strided((100,), (2,), device="cuda")
    with pytest.raises((TypeError, ValueError)):
        gpu.grad_norm(tl)
    a.data = whole
    assert float(gpu.grad_norm(tl)) == 20.0


def test_streams_and_graphs(cuda):
    """Calls on a side stream, and two captured graphs replayed at the same
    time on two streams, give what eager calls give."""
    x, dy, dr, gamma, beta = make_ln(2000, 768, torch.float32, 1)
    y, dz, _, _, _ = make_ln(1500, 768, torch.float32, 2)
    ts = make_list([100000, 5, 4096], DTYPES, 4)

    def work(x, dy):
        out, mean, rstd = gpu.layer_norm_forward(x, gamma=gamma, beta=beta)
        g = gpu.layer_norm_backward(dy, x, mean, rstd, gamma)
        return [out, *g, gpu.grad_norm(ts)]
    refs = [[t.clone() for t in work(x, dy)], [t.clone() for t in work(y, dz)]]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for (a, b), s in zip(((x, dy), (y, dz)), streams):
        with torch.cuda.stream(s):
            work(a, b)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(work(a, b))
            graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for got, ref in zip(outs, refs):
        for p, q in zip(got, ref):
            assert torch.equal(p, q)
