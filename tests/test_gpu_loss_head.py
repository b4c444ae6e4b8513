"""The training operators together, as transformer.LossHead calls them after a
block: loss and gradients against torch's autograd in fp64 on the block's
output, clipping, and a whole step as a CUDA graph."""
import numpy as np
import pytest
import torch

from silarray_b200 import gpu, transformer

pytestmark = pytest.mark.gpu

CFG = transformer.Config(batch=3, seq=40, d_model=128, heads=2, d_ff=256)
VOCAB = 517


def block_output(seed):
    block = transformer.Block(CFG, transformer.init_params(CFG, seed=1), device="cuda:0", graphs=False)
    return block.forward(torch.from_numpy(transformer.init_input(CFG, seed=seed)).cuda())


def make_targets(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    y = torch.randint(0, VOCAB, (CFG.tokens,), generator=g, device="cuda", dtype=torch.int32)
    y[::7] = -100
    return y


def autograd64(head, x, y, dres=None):
    leaves = [t.double().requires_grad_() for t in (x, head.gamma, head.beta, head.w)]
    xd, g, b, w = leaves
    h = torch.nn.functional.layer_norm(xd, (xd.shape[1],), g, b, head.eps)
    loss = torch.nn.functional.cross_entropy(h @ w.T, y.long(), ignore_index=-100)
    return loss.detach(), torch.autograd.grad(loss + (0.0 if dres is None else (xd * dres.double()).sum()), leaves)


def relative(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


# Per output, in half steps of its type: bf16 rounds h, ds, dh and the result, each of
# them at random within 2^-8, so the norm of the sum stays below 2 * 2^-8 by far (rms of one
# rounding: 2^-8 / 2.3).  fp32 carries the products' 2^-16 of sum |h w| at most, whose
# share of the norm is below 1e-5.
TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -7}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_step_against_autograd(cuda, dtype):
    x = block_output(2).to(dtype)
    y = make_targets(3)
    head = transformer.LossHead(transformer.init_head(VOCAB, CFG.d_model, seed=4), dtype=dtype)
    dres = torch.randn(x.shape, device="cuda").mul_(1e-3).to(dtype)
    with pytest.raises(RuntimeError):
        head.backward()
    loss = head.forward(x, y)
    dx = head.backward(dresidual=dres)
    ref_loss, ref = autograd64(head, x, y, dres)
    assert abs(float(loss) - float(ref_loss)) <= TOL[dtype] * float(ref_loss)
    for name, got, r in zip(("dx", "dgamma", "dbeta", "dw"), (dx, *head.grads.values()), ref):
        assert relative(got, r) <= TOL[dtype], name
    before = [g.clone() for g in head.grads.values()]
    norm = float(head.clip(1e-3))
    ref_norm = float(sum(b.double().square().sum() for b in before).sqrt())
    assert abs(norm - ref_norm) <= 6 * 2.0 ** -24 * ref_norm and norm > 1e-3
    for b, g in zip(before, head.grads.values()):
        assert relative(g, b.double() * (1e-3 / (ref_norm + 1e-6))) <= torch.finfo(g.dtype).eps
    gpu.device_status()


def test_step_as_a_graph(cuda):
    """Captured once, replayed on new activations and targets in the same buffers."""
    head = transformer.LossHead(transformer.init_head(VOCAB, CFG.d_model, seed=4))
    x, y = block_output(5), make_targets(6)
    xs, ys = x.clone(), y.clone()

    def step():
        loss = head.forward(xs, ys)
        dx = head.backward()
        return loss, dx, head.clip(1e-2), *head.grads.values()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (5, 8):
        xs.copy_(block_output(seed))
        ys.copy_(make_targets(seed + 1))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for p, q in zip(got, step()):
            assert torch.equal(p, q)
    gpu.device_status()


def test_three_steps_move_the_weights_like_autograd(cuda):
    """Three plain gradient steps on W give the weights that fp64 autograd gives."""
    params = transformer.init_head(VOCAB, CFG.d_model, seed=9)
    head = transformer.LossHead(params)
    x, y = block_output(10), make_targets(11)
    w64 = head.w.double()
    start = w64.clone()
    for _ in range(3):
        head.forward(x, y)
        head.backward()
        head.w.sub_(head.grads["w"], alpha=2.0)
        w = w64.clone().requires_grad_()
        h = torch.nn.functional.layer_norm(x.double(), (CFG.d_model,), head.gamma.double(), head.beta.double(), head.eps)
        torch.nn.functional.cross_entropy(h @ w.T, y.long(), ignore_index=-100).backward()
        w64 = w64 - 2.0 * w.grad
    moved = float((w64 - start).norm())
    # three gradients of 1e-5 and three roundings of W
    assert float((head.w.double() - w64).norm()) <= 1e-5 * 3 * moved + 3 * 2.0 ** -24 * float(w64.norm())
    assert np.isfinite(moved) and moved > 0


def test_clip_takes_the_gradients_that_are_there(cuda):
    """A gradient replaced by another tensor is the one that is written and clipped."""
    head = transformer.LossHead(transformer.init_head(VOCAB, CFG.d_model, seed=4))
    x, y = block_output(2), make_targets(3)
    head.forward(x, y)
    head.backward()
    norm = head.clip(1e9)
    first, head.grads["w"] = head.grads["w"], torch.empty_like(head.w)
    head.backward()
    kept = first.clone()
    assert torch.equal(head.grads["w"], first)
    assert torch.equal(head.clip(1e-3), norm)
    assert torch.equal(first, kept) and float(head.grads["w"].norm()) <= 1e-3
