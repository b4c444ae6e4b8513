"""The training operators on tensors of another GPU than the current one: the
workspace's size is asked for, and the launch made, with the tensors' GPU current."""
import contextlib

import pytest
import torch

from silarray_b200 import _lib, gpu


class OnGpu1(torch.Tensor):
    """A CPU tensor that says it lies on cuda:1."""
    is_cuda = property(lambda t: True)

    def get_device(self):
        return 1


def tensor(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnGpu1)


@pytest.fixture
def calls(monkeypatch):
    """[(entry point, current GPU)] of a library that does nothing, while cuda:0 is current."""
    current, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    class Library:
        def __getattr__(self, name):
            def fn(*args):
                seen.append((name, current[0]))
                return 64 if name.endswith("_bytes") else 0
            return fn
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0])
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index)
    monkeypatch.setattr(torch.cuda, "device", device)
    library = Library()
    monkeypatch.setattr(gpu, "lib", lambda: library)
    monkeypatch.setattr(_lib, "lib", lambda: library)
    # what is made for a call: CPU memory here
    monkeypatch.setattr(gpu, "_scratch", lambda nbytes, device: (None, None))
    return seen


def test_sizes_and_launches_on_the_tensors_gpu(calls):
    x, g = tensor(4, 8), tensor(8)
    gpu.layer_norm_forward(x, gamma=g, beta=g.clone())
    gpu.layer_norm_backward(x, x.clone(), tensor(4), tensor(4), g, din=tensor(4, 8), dgamma=tensor(8), dbeta=tensor(8))
    y = tensor(4, dtype=torch.int32)
    loss, lse = gpu.linear_cross_entropy(x, tensor(9, 8), y, loss=tensor(), lse=tensor(4))
    gpu.linear_cross_entropy_backward(x, tensor(9, 8), y, lse, dH=tensor(4, 8), dW=tensor(9, 8))
    gpu.grad_norm([x, g])
    gpu.clip_grad_norm([x.clone(), g.clone()], 1.0)
    assert len(calls) == 11 and all(index == 1 for _, index in calls), calls
