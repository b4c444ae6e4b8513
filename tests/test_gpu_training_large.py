"""The training operators where element offsets pass 2^31: rows far apart,
matrices and tensors of more than 2^31 elements."""
import pytest
import torch

from silarray_b200 import gpu
from tests.test_gpu_cross_entropy import check as check_loss
from tests.test_gpu_cross_entropy import make
from tests.test_gpu_training import check as check_values
from tests.test_gpu_training import check_forward, half_step
from tests.test_training_cpu import ln_backward_ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(autouse=True)
def free_memory(cuda):
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def far_apart(t, ld, shift):
    """t's rows ld elements apart in a new buffer, `shift` elements off its start."""
    buf = torch.empty((t.shape[0] - 1) * ld + t.shape[1] + shift, dtype=t.dtype, device=t.device)
    return buf[shift:].as_strided(t.shape, (ld, 1)).copy_(t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows,shift", [(5, 0), (5, 1), (150, 0), (150, 1)])
def test_weights_far_apart(cuda, rows, shift, dtype):
    """W and dW of 40 rows over 2.7 G elements, read in place (shift 0) and copied."""
    H, W, y = make(rows, 40, 64, dtype, 21)
    ld = 2 ** 26 + 8
    far, grad = far_apart(W, ld, shift), far_apart(torch.zeros_like(W), ld, shift)
    loss, lse = gpu.linear_cross_entropy(H, far, y)
    dH, dW = gpu.linear_cross_entropy_backward(H, far, y, lse, dW=grad)
    assert dW is grad
    check_loss(H, W, y, loss, lse, dH, dW.contiguous())
    gpu.device_status()


def test_layer_norm_past_2_31_elements(cuda):
    rows, cols = 262400, 8192
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(3))
    gamma, beta = torch.linspace(0.5, 1.5, cols, device="cuda"), torch.linspace(-1, 1, cols, device="cuda")
    out, mean, rstd = gpu.layer_norm_forward(x, gamma=gamma, beta=beta)
    some = torch.tensor([0, 262143, 262144, rows - 1], device="cuda")
    check_forward(x[some], gamma, beta, out[some], mean[some], rstd[some], 1e-5)
    del out
    din, _, dbeta = gpu.layer_norm_backward(x, x, mean, rstd, gamma)
    ref, _, _ = ln_backward_ref(x[some].double(), x[some].double(), mean[some].double(), rstd[some].double(), gamma.double())
    # 8192 columns: 53 additions on the way into a row's sums of terms below 6 on average
    check_values(din[some], ref, 80 * U * 12.0 + (2 * U + half_step(din.dtype)) * ref.abs(), "din")
    # sums of `rows` values of which all are exact in fp64
    total = sum(x[i:i + 8200].double().sum(0) for i in range(0, rows, 8200))
    size = sum(x[i:i + 8200].double().abs().sum(0) for i in range(0, rows, 8200))
    check_values(dbeta, total, (rows // 148 + 200) * U * size, "dbeta")


def test_norm_past_2_31_elements(cuda):
    n = 2 ** 31 + 1001
    t = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    t[-1] = 1024.0
    want = float(n - 1 + 1024 ** 2) ** 0.5
    norm = gpu.clip_grad_norm([t], want / 4, eps=0.0)
    # fp32 sums of up to 32 ones are exact; the root is rounded once, the factor 1/4 and the elements not at all or by one step
    assert abs(float(norm) - want) <= 2 * U * want
    assert abs(float(t[-1]) - 256.0) <= 1.0 and abs(float(t[0]) - 0.25) <= 2.0 ** -10
    assert bool((t[:-1] == t[0]).all())
