"""clip_grad_norm where the limit or the norm is infinite."""
import pytest
import torch

from silarray_b200 import gpu

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_infinite_limits_and_norms(cuda, dtype):
    """An infinite limit leaves gradients of a finite norm as they are; an infinite norm makes finite
    elements 0 for a finite limit, and inf / inf = NaN of every element for an infinite one."""
    g = torch.Generator(device="cuda").manual_seed(1)
    grads = [torch.randn(n, generator=g, device="cuda").to(dtype) for n in (1000, 7)]
    want = [t.clone() for t in grads]
    norm = gpu.clip_grad_norm(grads, INF)
    assert all(torch.equal(a, b) for a, b in zip(grads, want)) and bool(torch.isfinite(norm))
    grads[1][3] = INF
    finite = [torch.isfinite(t) for t in grads]
    for limit, check in ((1.0, lambda t: t == 0), (INF, torch.isnan)):
        out = [torch.ones_like(t) for t in grads]
        assert float(gpu.clip_grad_norm(grads, limit, OUT=out)) == INF
        assert all(bool(check(t)[f].all()) for t, f in zip(out, finite)) and bool(torch.isnan(out[1][3]))
