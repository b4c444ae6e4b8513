"""The operators of a training step's tail, as cases to measure: layer_norm with its backward pass, the
vocabulary projection with its softmax cross entropy and gradients, and the global norm of a list of
gradients with its clipping.  `run` computes them in plain torch operations, or (own = True) through
silarray_b200.gpu."""
import math

import torch

own = False

EPS = 1e-5
CLIP_EPS = 1e-6
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # the final layer_norm of the transformer block's own batch (32 sequences of 512 tokens)
        {"name": "ln_forward_block_f32", "op": "ln_forward", "dtype": "f32", "rows": 16384, "cols": 768},
        # a wide model's layer_norm over one micro-batch
        {"name": "ln_forward_wide_bf16", "op": "ln_forward", "dtype": "bf16", "rows": 4096, "cols": 8192},
        # one 512-token sequence: the call is short, its latency counts
        {"name": "ln_backward_seq_f32", "op": "ln_backward", "dtype": "f32", "rows": 512, "cols": 768,
         "residual": False},
        # the same batch as the first case, with the residual branch's gradient added
        {"name": "ln_backward_block_f32", "op": "ln_backward", "dtype": "f32", "rows": 16384, "cols": 768,
         "residual": True},
        # a wide model, a ragged number of tokens
        {"name": "ln_backward_wide_bf16", "op": "ln_backward", "dtype": "bf16", "rows": 8190, "cols": 4096,
         "residual": True},
        # scoring eight tokens: reading the vocabulary matrix is all there is
        {"name": "loss_score_bf16", "op": "loss", "dtype": "bf16", "rows": 8, "vocab": 32768, "dim": 4096,
         "left_out": 0.0},
        # evaluation of a batch over a vocabulary of odd size, prompt tokens left out
        {"name": "loss_eval_bf16", "op": "loss", "dtype": "bf16", "rows": 2048, "vocab": 50021, "dim": 768,
         "left_out": 0.25},
        # a short ragged micro-batch in full precision, padding left out
        {"name": "loss_train_ragged_f32", "op": "loss_train", "dtype": "f32", "rows": 333, "vocab": 10007,
         "dim": 768, "left_out": 0.1},
        # the block's own batch trained in full precision
        {"name": "loss_train_block_f32", "op": "loss_train", "dtype": "f32", "rows": 16384, "vocab": 32768,
         "dim": 768, "left_out": 0.0},
        # a large vocabulary in mixed precision: the largest step
        {"name": "loss_train_large_bf16", "op": "loss_train", "dtype": "bf16", "rows": 8192, "vocab": 131072,
         "dim": 2048, "left_out": 0.05},
        # the norm of one block's gradients, to be logged each step
        {"name": "grad_norm_block_f32", "op": "grad_norm", "dtype": "f32", "tensors": 16, "elements": 7087872,
         "packed": False},
        # clipping a model's gradients that lie in one bucket, at offsets that are not aligned
        {"name": "clip_packed_bf16", "op": "clip", "dtype": "bf16", "tensors": 195, "elements": 350000003,
         "packed": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln_forward", "ln_backward", "loss", "loss_train", "loss_train", "grad_norm", "clip"])
    dtype = rng.choice(["f32", "bf16"])
    if op.startswith("ln_"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.7:
            cols = max(64, cols // 8 * 8)
        rows = _log(rng, 1, min(65536, (1 << 26) // cols))
        case = {"op": op, "dtype": dtype, "rows": rows, "cols": cols}
        if op == "ln_backward":
            case["residual"] = rng.random() < 0.5
        return case
    if op.startswith("loss"):
        dim = _log(rng, 64, 4096)
        if rng.random() < 0.75:
            dim = max(64, dim // 8 * 8)
        vocab = _log(rng, 1000, 131072)
        top = (1 << 41) if dtype == "bf16" else (1 << 38)
        rows = _log(rng, 1 if op == "loss" else 16, max(17, min(16384, top // (dim * vocab))))
        return {"op": op, "dtype": dtype, "rows": rows, "vocab": vocab, "dim": dim,
                "left_out": rng.choice([0.0, 0.1, 0.5])}
    return {"op": op, "dtype": dtype, "tensors": _log(rng, 1, 400), "elements": _log(rng, 5000, 1 << 28),
            "packed": rng.random() < 0.5}


def _sizes(case):
    """Tensor sizes as a model has them: matrices, and vectors a few hundred times smaller."""
    n, total = case["tensors"], case["elements"]
    small = max(1, total // (400 * n))
    vectors = n // 2
    matrices = n - vectors
    each = (total - vectors * small) // matrices
    sizes = []
    for i in range(n):
        sizes.append(small if i % 2 else each)
    sizes[0] += total - sum(sizes)
    return sizes


# ------------------------------------------------------------------ the inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=t):
        return torch.randn(shape, generator=gen, device="cuda").mul_(std).add_(mean).to(dtype)

    op = case["op"]
    state = {"op": op, "case": case}
    if op.startswith("ln_"):
        rows, cols = case["rows"], case["cols"]
        state["x"] = normal(rows, cols, std=2.0, mean=0.3)
        state["gamma"] = normal(cols, std=0.1, mean=1.0, dtype=torch.float32)
        state["beta"] = normal(cols, std=0.1, dtype=torch.float32)
        if op == "ln_backward":
            state["dy"] = normal(rows, cols)
            state["dresidual"] = normal(rows, cols) if case["residual"] else None
            x = state["x"].float()
            state["mean"] = x.mean(1)
            state["rstd"] = (x.var(1, correction=0) + EPS).rsqrt()
    elif op.startswith("loss"):
        rows, vocab, dim = case["rows"], case["vocab"], case["dim"]
        state["H"] = normal(rows, dim)
        state["W"] = normal(vocab, dim, std=2.0 / math.sqrt(dim))  # logits of a few units, as a trained head's
        y = torch.randint(0, vocab, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        out = torch.rand(rows, generator=gen, device="cuda") < case["left_out"]
        out[0] = False
        state["targets"] = torch.where(out, torch.full_like(y, -1), y)
    else:
        sizes = _sizes(case)
        starts, at = [], 0
        for n in sizes:
            starts.append(at)
            at += n if case["packed"] else (n + 7) // 8 * 8
        flat = normal(at, std=2e-2)
        state["grads"] = [flat[s:s + n] for s, n in zip(starts, sizes)]
        if op == "clip":
            state["flat_out"] = torch.zeros_like(flat)
            state["outs"] = [state["flat_out"][s:s + n] for s, n in zip(starts, sizes)]
        if own:
            from silarray_b200 import gpu
            state["list"] = gpu.TensorList(state["grads"])
            state["out_list"] = gpu.TensorList(state["outs"]) if op == "clip" else None
    return state


# --------------------------------------------------------------- the operators
def run(state):
    if own:
        return _run_own(state)
    return {"ln_forward": _ln_forward, "ln_backward": _ln_backward, "loss": _loss, "loss_train": _loss_train,
            "grad_norm": _grad_norm, "clip": _clip}[state["op"]](state)


def _run_own(state):
    from silarray_b200 import gpu
    op = state["op"]
    if op == "ln_forward":
        out, mean, rstd = gpu.layer_norm_forward(state["x"], gamma=state["gamma"], beta=state["beta"], eps=EPS)
        return {"out": out, "mean": mean, "rstd": rstd}
    if op == "ln_backward":
        dx, dgamma, dbeta = gpu.layer_norm_backward(state["dy"], state["x"], state["mean"], state["rstd"],
                                                    state["gamma"], dresidual=state["dresidual"])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if op == "loss":
        loss, lse = gpu.linear_cross_entropy(state["H"], state["W"], state["targets"], reduction="none")
        return {"loss": loss, "lse": lse}
    if op == "loss_train":
        loss, lse = gpu.linear_cross_entropy(state["H"], state["W"], state["targets"], reduction="mean")
        dH, dW = gpu.linear_cross_entropy_backward(state["H"], state["W"], state["targets"], lse, reduction="mean")
        return {"loss": loss, "lse": lse, "dH": dH, "dW": dW}
    if op == "grad_norm":
        return {"norm": gpu.grad_norm(state["list"])}
    return {"norm": gpu.clip_grad_norm(state["list"], 1.0, OUT=state["out_list"], eps=CLIP_EPS),
            "grads": state["flat_out"]}


def _ln_forward(state):
    x = state["x"].float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1.0 / torch.sqrt((c * c).mean(1, keepdim=True) + EPS)
    out = (c * rstd * state["gamma"] + state["beta"]).to(state["x"].dtype)
    return {"out": out, "mean": mean[:, 0], "rstd": rstd[:, 0]}


def _ln_backward(state):
    dy = state["dy"].float()
    rstd = state["rstd"][:, None]
    xh = (state["x"].float() - state["mean"][:, None]) * rstd
    a = dy * state["gamma"]
    dx = rstd * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    if state["dresidual"] is not None:
        dx = dx + state["dresidual"].float()
    return {"dx": dx.to(state["x"].dtype), "dgamma": (dy * xh).sum(0), "dbeta": dy.sum(0)}


def _scores(state):
    H, W, y = state["H"].float(), state["W"].float(), state["targets"].long()
    s = H @ W.T
    m = s.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(s - m).sum(1, keepdim=True))
    used = (y >= 0) & (y < W.shape[0])
    at = torch.where(used, y, torch.zeros_like(y))
    loss = torch.where(used, (lse - s.gather(1, at[:, None]))[:, 0], torch.zeros_like(lse[:, 0]))
    return H, W, s, lse, used, at, loss


def _loss(state):
    _, _, _, lse, _, _, loss = _scores(state)
    return {"loss": loss, "lse": lse[:, 0]}


def _loss_train(state):
    H, W, s, lse, used, at, loss = _scores(state)
    count = used.sum().clamp(min=1).float()
    ds = torch.exp(s - lse)
    ds[torch.arange(ds.shape[0], device=ds.device), at] -= 1.0
    ds *= (used.float() / count)[:, None]
    t = state["H"].dtype
    return {"loss": loss.sum() / count, "lse": lse[:, 0], "dH": (ds @ W).to(t), "dW": (ds.T @ H).to(t)}


def _grad_norm(state):
    return {"norm": _norm64(state["grads"]).float()}


def _norm64(grads):
    return torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()


def _clip(state):
    norm = _norm64(state["grads"])
    c = torch.clamp(1.0 / (norm + CLIP_EPS), max=1.0).float()
    [o.copy_(g.float() * c) for g, o in zip(state["grads"], state["outs"])]
    return {"norm": norm.float(), "grads": state["flat_out"]}


# ------------------------------------------------------------ what it has to do
def work(case):
    e = SIZE[case["dtype"]]
    op = case["op"]
    if op.startswith("ln_"):
        n = case["rows"] * case["cols"]
        if op == "ln_forward":
            return {"bytes": 2 * n * e + 8 * case["rows"] + 8 * case["cols"], "flops": 8 * n}
        streams = 4 if case["residual"] else 3
        return {"bytes": streams * n * e + 8 * case["rows"] + 12 * case["cols"], "flops": 14 * n}
    if op.startswith("loss"):
        rows, vocab, dim = case["rows"], case["vocab"], case["dim"]
        io = (rows + vocab) * dim * e
        if op == "loss":
            return {"bytes": io + 12 * rows, "flops": 2 * rows * vocab * dim + 4 * rows * vocab}
        return {"bytes": 2 * io + 8 * rows + 4, "flops": 6 * rows * vocab * dim + 6 * rows * vocab}
    n = case["elements"]
    if op == "grad_norm":
        return {"bytes": n * e + 4, "flops": 2 * n}
    return {"bytes": 2 * n * e + 4, "flops": 3 * n}


# ----------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    d = torch.float64
    if op == "ln_forward":
        x = state["x"].to(d)
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + EPS).rsqrt()
        out = torch.addcmul(state["beta"].to(d), (x - mean[:, None]) * rstd[:, None], state["gamma"].to(d))
        return {"out": out, "mean": mean, "rstd": rstd}
    if op == "ln_backward":
        n = case["cols"]
        dx, dgamma, dbeta = [], 0.0, 0.0
        for r in range(0, case["rows"], 2048):
            cut = slice(r, r + 2048)
            x, dy, rstd = state["x"][cut].to(d), state["dy"][cut].to(d), state["rstd"][cut].to(d)[:, None]
            z = (x - state["mean"][cut].to(d)[:, None]) * rstd
            g = dy * state["gamma"].to(d)
            v = (n * g - g.sum(1, keepdim=True) - z * torch.einsum("ij,ij->i", g, z)[:, None]) * (rstd / n)
            dx.append(v if state["dresidual"] is None else v + state["dresidual"][cut].to(d))
            dgamma = dgamma + torch.einsum("ij,ij->j", dy, z)
            dbeta = dbeta + torch.einsum("ij->j", dy)
        return {"dx": torch.cat(dx), "dgamma": dgamma, "dbeta": dbeta}
    if op.startswith("loss"):
        W, y = state["W"].to(d), state["targets"].long()
        valid = (y >= 0) & (y < case["vocab"])
        count = max(1, int(valid.sum()))
        losses, lses, dH, dW = [], [], [], torch.zeros_like(W) if op == "loss_train" else None
        for r in range(0, case["rows"], 1024):
            h, t, ok = state["H"][r:r + 1024].to(d), y[r:r + 1024], valid[r:r + 1024]
            logits = torch.einsum("td,vd->tv", h, W)
            lse = torch.logsumexp(logits, 1)
            one = torch.zeros_like(logits)
            one[ok, t[ok]] = 1.0
            losses.append(torch.where(ok, lse - (logits * one).sum(1), torch.zeros_like(lse)))
            lses.append(lse)
            if dW is not None:
                p = torch.softmax(logits, 1).sub_(one)
                p[~ok] = 0.0
                p /= count
                dH.append(torch.einsum("tv,vd->td", p, W))
                dW += torch.einsum("tv,td->vd", p, h)
        if op == "loss":
            return {"loss": torch.cat(losses), "lse": torch.cat(lses)}
        return {"loss": torch.cat(losses).sum() / count, "lse": torch.cat(lses), "dH": torch.cat(dH), "dW": dW}
    norm = torch.linalg.vector_norm(torch.cat([torch.linalg.vector_norm(g.to(d)).reshape(1) for g in state["grads"]]))
    if op == "grad_norm":
        return {"norm": norm}
    c = min(1.0, 1.0 / (float(norm) + CLIP_EPS))
    out = torch.zeros(state["flat_out"].shape, dtype=d, device="cuda")
    base = state["flat_out"].storage_offset()
    for g, o in zip(state["grads"], state["outs"]):
        start = o.storage_offset() - base
        out[start:start + o.numel()] = g.to(d) * c
    return {"norm": norm, "grads": out}
