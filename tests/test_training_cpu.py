"""The training operators without a GPU: their formulas (the references of the
GPU tests) against torch's autograd in fp64, and what the C entry points and the
Python mirror refuse before they touch a device."""
import ctypes as C

import pytest
import torch

from silarray_b200 import _build, _lib


# ----------------------------------------------------------------- references
def ln_forward_ref(x, gamma, beta, eps):
    mean = x.mean(1)
    var = (x - mean[:, None]).square().mean(1)
    rstd = 1.0 / (var + eps).sqrt()
    return (x - mean[:, None]) * rstd[:, None] * gamma + beta, mean, rstd


def ln_backward_ref(dy, x, mean, rstd, gamma, dres=None):
    xh = (x - mean[:, None]) * rstd[:, None]
    a = dy * gamma
    dx = rstd[:, None] * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    return dx if dres is None else dx + dres, (dy * xh).sum(0), dy.sum(0)


def cross_entropy_ref(H, W, y, reduction, dloss):
    V = W.shape[0]
    used = (y >= 0) & (y < V)
    H = torch.where(used[:, None], H, H.nan_to_num(0.0, 0.0, 0.0))
    s = H @ W.T
    lse = torch.logsumexp(s, 1)
    at = torch.where(used, y, torch.zeros_like(y))
    row = torch.where(used, lse - s.gather(1, at[:, None])[:, 0], torch.zeros_like(lse))
    n = max(1, int(used.sum()))
    loss = {"none": row, "sum": row.sum(), "mean": row.sum() / n}[reduction]
    d = torch.ones((), dtype=H.dtype, device=H.device) if dloss is None else dloss
    scale = torch.where(used, (d / n if reduction == "mean" else d).expand_as(row), torch.zeros_like(row))
    p = torch.exp(s - lse[:, None])
    ds = p.clone()
    ds[torch.arange(len(y), device=H.device), at] -= 1.0
    ds = ds * scale[:, None]
    hz = torch.where(used[:, None], H, torch.zeros_like(H))
    return {"loss": loss, "lse": lse, "row_loss": row, "scale": scale, "p": p, "ds": ds, "dH": ds @ W, "dW": ds.T @ hz}


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_cross_entropy_reference_is_the_gradient(reduction):
    g = torch.Generator().manual_seed(0)
    H, W = (torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((6, 9), (13, 9)))
    y = torch.tensor([0, 12, -100, 13, 5, 5])
    dloss = torch.randn(6 if reduction == "none" else (), generator=g, dtype=torch.float64)
    target = torch.where(y < 13, y, torch.full_like(y, -100))
    loss = torch.nn.functional.cross_entropy(H @ W.T, target, ignore_index=-100, reduction=reduction)
    r = cross_entropy_ref(H.detach(), W.detach(), y, reduction, dloss)
    assert torch.allclose(r["loss"], loss.detach())
    for p, q in zip((r["dH"], r["dW"]), torch.autograd.grad((loss * dloss).sum(), (H, W))):
        assert torch.allclose(p, q, rtol=1e-10, atol=1e-12)


def test_layer_norm_reference_is_the_gradient():
    g = torch.Generator().manual_seed(0)
    x, gamma, beta = (torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True) for s in ((5, 33), 33, 33))
    dy = torch.randn(5, 33, generator=g, dtype=torch.float64)
    out, mean, rstd = ln_forward_ref(x, gamma, beta, 1e-5)
    grads = torch.autograd.grad((out * dy).sum(), (x, gamma, beta))
    for p, q in zip(ln_backward_ref(dy, x, mean, rstd, gamma), grads):
        assert torch.allclose(p, q, rtol=1e-10, atol=1e-12)


# ------------------------------------------------------------------- refusals
@pytest.fixture(scope="module")
def lib():
    _build.build()
    return _lib.lib()


P = C.c_void_p(1 << 20)  # never dereferenced: every call below fails its checks first


def test_layer_norm_refusals(lib):
    f, b = lib.silcu_layer_norm_forward, lib.silcu_layer_norm_backward
    assert f(None, None, None, None, None, None, 0, 5, 1e-5, 0, None) == 0  # no rows: nothing to do
    assert f(P, P, None, None, P, None, 4, 8, 1e-5, 0, None) == 1  # no beta
    assert f(P, P, None, None, P, P, 4, 0, 1e-5, 0, None) == 1  # no columns
    assert f(P, P, None, None, P, P, 4, 8, 1e-5, 2, None) == 1 and b"dtype" in lib.silcu_last_error()
    assert f(P, P, None, None, P, P, 4, (1 << 24) + 1, 1e-5, 0, None) == 5
    assert f(P, P, None, None, P, P, 1 << 31, 8, 1e-5, 0, None) == 5
    need = lib.silcu_layer_norm_backward_workspace_bytes(100, 768, 0)
    assert need >= 2 * 768 * 4
    args = (P, P, P, P, P, None, P, P, P, 100, 768, 0)
    assert b(*args, P, need - 1, None) == 4
    assert b(*args, None, need, None) == 4
    assert b(*args, C.c_void_p((1 << 20) + 2), need, None) == 1
    assert b(P, P, None, P, P, None, P, P, P, 100, 768, 0, P, need, None) == 1
    assert b(P, P, P, P, P, None, P, None, P, 100, 768, 0, P, need, None) == 1
    odd, half = C.c_void_p((1 << 20) + 1), C.c_void_p((1 << 20) + 2)
    assert f(half, P, None, None, P, P, 4, 8, 1e-5, 0, None) == 1 and f(P, odd, None, None, P, P, 4, 8, 1e-5, 1, None) == 1
    assert f(P, P, half, None, P, P, 4, 8, 1e-5, 1, None) == 1
    assert b(P, P, P, P, P, half, P, P, P, 100, 768, 0, P, need, None) == 1
    assert b(P, P, P, P, P, None, P, half, P, 100, 768, 1, P, need, None) == 1
    assert lib.silcu_layer_norm_backward_workspace_bytes(0, 768, 0) == 0


def test_gradient_list_refusals(lib):
    norm, clip = lib.silcu_grad_norm, lib.silcu_clip_grad_norm
    two = (_lib.Tensor * 2)(_lib.Tensor(1 << 20, 100, 0), _lib.Tensor(1 << 21, 50, 1))
    need = lib.silcu_grad_norm_workspace_bytes(two, 2)
    assert need >= 8
    assert norm(two, 2, None, P, need, None) == 1
    assert norm(two, 2, P, P, need - 1, None) == 4
    assert norm(None, 2, P, P, 64, None) == 1
    assert norm(two, 2, P, C.c_void_p((1 << 20) + 4), need, None) == 1
    for bad in (_lib.Tensor(1 << 20, 100, 7), _lib.Tensor(0, 100, 0), _lib.Tensor((1 << 20) + 2, 100, 0),
                _lib.Tensor((1 << 20) + 1, 100, 1)):
        lst = (_lib.Tensor * 2)(two[0], bad)
        assert norm(lst, 2, P, P, 1 << 20, None) == 1 and b"tensor 1" in lib.silcu_last_error()
    assert norm((_lib.Tensor * 1)(_lib.Tensor(1 << 20, 1 << 48, 0)), 1, P, P, 1 << 20, None) == 5
    assert clip(two, None, 2, -1.0, 1e-6, P, P, need, None) == 1
    assert clip(two, None, 2, float("nan"), 1e-6, P, P, need, None) == 1
    assert clip(two, None, 2, 1.0, -1.0, P, P, need, None) == 1
    outs = (C.c_void_p * 2)(1 << 20, 0)
    assert clip(two, outs, 2, 1.0, 1e-6, P, P, need, None) == 1 and b"output 1" in lib.silcu_last_error()


def _loss_args(**kw):
    a = _lib.CrossEntropyArgs()
    for i, k in enumerate(("dH", "W", "targets", "loss", "lse", "H", "dW")):
        setattr(a, k, (1 << 20) + (i << 16))
    a.rows, a.V, a.D, a.ldh, a.ldw, a.lddh, a.lddw = 10, 100, 64, 64, 64, 64, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_cross_entropy_refusals(lib):
    size, fwd, bwd = (lib.silcu_linear_cross_entropy_workspace_bytes, lib.silcu_linear_cross_entropy,
                      lib.silcu_linear_cross_entropy_backward)
    big = 1 << 30
    for status, kw in [(1, dict(dtype=2)), (1, dict(reduction=3)), (1, dict(rows=-1)), (1, dict(V=0)), (1, dict(D=0)),
                       (1, dict(ldh=63)), (1, dict(ldw=10)), (5, dict(rows=(1 << 20) + 1)), (5, dict(V=(1 << 24) + 1)),
                       (5, dict(ldh=(1 << 32) + 1)), (1, dict(H=0)), (1, dict(W=0)), (1, dict(targets=0)),
                       (1, dict(lse=0)), (1, dict(H=(1 << 20) + 2)), (1, dict(W=(1 << 20) + 1, dtype=1))]:
        a = _loss_args(**kw)
        assert fwd(C.byref(a), P, big, None) == status, kw
        assert bwd(C.byref(a), P, big, None) == status, kw
    assert fwd(None, P, big, None) == 1 and bwd(None, P, big, None) == 1
    a = _loss_args(loss=0)
    assert fwd(C.byref(a), P, big, None) == 1
    for kw in (dict(lddh=63), dict(lddw=1), dict(dH=(1 << 20) + 1), dict(dloss=(1 << 20) + 2), dict(targets=(1 << 20) + 2),
               dict(dW=(1 << 20) + (1 << 16)), dict(dH=(1 << 20) + (5 << 16))):
        a = _loss_args(**kw)
        assert bwd(C.byref(a), P, big, None) == 1, kw
    for dtype in (0, 1):
        a = _loss_args(dtype=dtype)
        need = size(C.byref(a), 1)
        assert need >= size(C.byref(a), 0) > 0
        assert bwd(C.byref(a), P, need - 1, None) == 4 and bwd(C.byref(a), None, need, None) == 4
        assert fwd(C.byref(a), P, 10, None) == 4
    a = _loss_args(dH=0, dW=0)
    assert bwd(C.byref(a), None, 0, None) == 0  # nothing wanted
    a = _loss_args(rows=0, reduction=2, loss=0)
    assert fwd(C.byref(a), None, 0, None) == 0 and size(C.byref(a), 1) == 0


def test_cross_entropy_workspace_stays_in_pieces(lib):
    """The workspace of a large vocabulary does not grow with it: a piece of the
    score gradients, not the logits."""
    a = _loss_args(rows=8192, V=1 << 17, D=2048, ldh=2048, ldw=2048, lddh=2048, lddw=2048, dtype=1)
    logits = 2 * 8192 * (1 << 17)
    assert lib.silcu_linear_cross_entropy_workspace_bytes(C.byref(a), 1) < logits / 4


def test_workspace_of_many_tensors(lib):
    """One fp64 partial per CTA, whatever the list's length; empty tensors ask for none."""
    many = (_lib.Tensor * 3000)(*[_lib.Tensor(1 << 20, 10, 0)] * 3000)
    assert 8 <= lib.silcu_grad_norm_workspace_bytes(many, 3000) <= 8 * 3 * 148 * 8
    none = (_lib.Tensor * 2)(_lib.Tensor(0, 0, 0), _lib.Tensor(0, 0, 1))
    assert lib.silcu_grad_norm_workspace_bytes(none, 2) == 0


def test_python_refuses_cpu_tensors():
    from silarray_b200 import gpu
    x = torch.ones(4, 8)
    with pytest.raises(TypeError):
        gpu.layer_norm_forward(x, gamma=x[0], beta=x[0])
    with pytest.raises(TypeError):
        gpu.grad_norm([x])
    with pytest.raises(ValueError):
        gpu.TensorList([])


def test_overlapping_operands_are_refused(lib):
    """Results that share memory with an operand or with one another; an
    operand written in place and column ranges of one matrix are another matter."""
    at = lambda *offsets: [C.c_void_p((1 << 20) + o) for o in offsets]  # noqa: E731
    f, b = lib.silcu_layer_norm_forward, lib.silcu_layer_norm_backward
    n, far = 100 * 768 * 4, 1 << 22
    x, near, out, mean, rstd, g, be = at(0, 768 * 4, far, 2 * far, 3 * far, 4 * far, 5 * far)
    for args in [(x, near, mean, rstd, g, be), (x, out, mean, mean, g, be), (x, out, x, rstd, g, be), (x, out, mean, rstd, out, be)]:
        assert f(*args, 100, 768, 1e-5, 0, None) == 1 and b"overlap" in lib.silcu_last_error()
    ws = C.c_void_p(1 << 30)
    dy, dg, db = at(6 * far, 7 * far, 8 * far)
    for args in [(dy, x, mean, rstd, g, None, near, dg, db), (dy, x, mean, rstd, g, near, x, dg, db),
                 (dy, x, mean, rstd, g, None, out, dg, dg), (dy, x, mean, rstd, g, None, out, mean, db),
                 (dy, x, mean, rstd, g, None, out, out, db)]:
        assert b(*args, 100, 768, 0, ws, n * 8, None) == 1 and b"overlap" in lib.silcu_last_error()

    fwd, bwd = lib.silcu_linear_cross_entropy, lib.silcu_linear_cross_entropy_backward
    base = _loss_args()
    for kw in (dict(loss=base.H + 8), dict(loss=base.lse + 4), dict(lse=base.W), dict(lse=base.targets + 36)):
        a = _loss_args(**kw)
        assert fwd(C.byref(a), ws, far, None) == 1 and b"overlap" in lib.silcu_last_error(), kw
    for kw in (dict(dH=base.H + 256), dict(dH=base.W - 4), dict(dW=base.W + 256), dict(dW=base.dH + 2304), dict(dH=base.lse),
               dict(dloss=base.dW + 25596), dict(dH=base.H + 252, ldh=128, lddh=128), dict(dH=base.H + 256, ldh=128, lddh=130)):
        a = _loss_args(**kw)
        assert bwd(C.byref(a), ws, far, None) == 1 and b"overlap" in lib.silcu_last_error(), kw
