"""linear_cross_entropy_backward with a gradient of the loss that is not finite, as an
overflowed loss scale gives it: rows that are left out keep their zeros."""
import pytest
import torch

from silarray_b200 import gpu
from tests.test_gpu_cross_entropy import DTYPES, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("rows,piece", [(40, None), (40, 256), (300, None), (300, 256)])
def test_left_out_rows_stay_zero(cuda, monkeypatch, rows, piece, bad, reduction, dtype):
    if piece:
        monkeypatch.setenv("SILCU_LOSS_PIECE", str(piece))
    V = 600
    H, W, y = make(rows, V, 72, dtype, 7, left_out=0.5)
    used = (y >= 0) & (y < V)
    shape = (rows,) if reduction == "none" else ()
    dloss = torch.full(shape, bad, device="cuda")
    _, lse = gpu.linear_cross_entropy(H, W, y, reduction=reduction)
    dH, dW = gpu.linear_cross_entropy_backward(H, W, y, lse, dloss=dloss, reduction=reduction)
    assert bool((dH[~used] == 0).all())
    assert not bool(torch.isfinite(dH[used]).any()) and not bool(torch.isfinite(dW).any())
    dH, dW = gpu.linear_cross_entropy_backward(H, W, torch.full_like(y, -1), lse, dloss=dloss, reduction=reduction)
    assert bool((dH == 0).all()) and bool((dW == 0).all())
    # one row that counts: its own gradient alone is touched
    if reduction == "none":
        one = torch.where(torch.arange(rows, device="cuda") == int(used.nonzero()[0]), dloss, torch.ones_like(dloss))
        dH, _ = gpu.linear_cross_entropy_backward(H, W, y, lse, dloss=one, reduction=reduction)
        assert bool(torch.isfinite(dH[1 + int(used.nonzero()[0]):]).all()) and bool((dH[~used] == 0).all())
    gpu.device_status()
