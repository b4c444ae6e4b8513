"""Pre-norm transformer block forward on the B200 backend.

The block is the graph of the reference's bench/composite/bench_transformer.cpp:56-67
(layer_norm -> Q/K/V linear -> Q.K^T * scale -> softmax -> .V -> linear(Wo)
-> residual -> layer_norm -> linear(W1).relu() -> linear(W2) -> residual),
generalised to a batch of sequences and multi-head attention (scale
1/sqrt(head_dim), attention per (sequence, head)).

Each reference node maps onto one launch of include/silcu.h, with the
reference's elementwise nodes folded into GEMM epilogues where they follow a
dot (bias add, the `* scale` affine node, relu, the residual add); the
rounding sequence per element is the reference's (dot, then + bias, then
act, then + residual).  Q, K and V come from one GEMM against [Wq|Wk|Wv]
(columns are independent, so the values equal three separate GEMMs).

Launches per forward: layer_norm, QKV gemm, fused attention (scores,
softmax and the context product in one tcgen05 kernel, per sequence x head,
Q, K and V read in place through strided views), Wo gemm (+bias +residual),
layer_norm, W1 gemm (+bias, relu), W2 gemm (+bias +residual); a GEMM whose
tiles fill its last wave poorly adds one finishing pass for its split-K
tiles.  Every product is 3xTF32 on tcgen05.  After the first forward over a
given set of buffers, the launches replay as one CUDA graph.
"""
import os
from dataclasses import dataclass

import numpy as np
import torch

from . import gpu


@dataclass
class Config:
    batch: int = 32
    seq: int = 512
    d_model: int = 768
    heads: int = 12
    d_ff: int = 3072
    eps: float = 1e-5

    @property
    def head_dim(self):
        return self.d_model // self.heads

    @property
    def tokens(self):
        return self.batch * self.seq

    def gemm_flops(self):
        """Algorithmic FLOPs of one forward (2*M*N*K summed over the GEMMs)."""
        T, d, f, S, h = self.tokens, self.d_model, self.d_ff, self.seq, self.head_dim
        qkv = 2 * T * d * 3 * d
        attn = 2 * (2 * self.batch * self.heads * S * S * h)
        wo = 2 * T * d * d
        ffn = 2 * (2 * T * d * f)
        return qkv + attn + wo + ffn


PARAM_NAMES = ("g1", "be1", "wq", "bq", "wk", "bk", "wv", "bv", "wo", "bo",
               "g2", "be2", "w1", "b1", "w2", "b2")


def _normal(rng, shape, std):
    return (rng.standard_normal(shape, dtype=np.float32) * np.float32(std)).astype(np.float32)


def init_params(cfg, seed=0):
    """Weights ~ N(0, 0.02^2), biases 0, gamma 1, beta 0 (the benchmark config)."""
    rng = np.random.default_rng(seed)
    d, f = cfg.d_model, cfg.d_ff
    p = {
        "g1": np.ones(d, np.float32), "be1": np.zeros(d, np.float32),
        "g2": np.ones(d, np.float32), "be2": np.zeros(d, np.float32),
        "bq": np.zeros(d, np.float32), "bk": np.zeros(d, np.float32), "bv": np.zeros(d, np.float32),
        "bo": np.zeros(d, np.float32), "b1": np.zeros(f, np.float32), "b2": np.zeros(d, np.float32),
    }
    for k in ("wq", "wk", "wv", "wo"):
        p[k] = _normal(rng, (d, d), 0.02)
    p["w1"] = _normal(rng, (d, f), 0.02)
    p["w2"] = _normal(rng, (f, d), 0.02)
    return p


def init_input(cfg, seed=1):
    """Activations ~ N(0, 1), [batch*seq, d_model]."""
    rng = np.random.default_rng(seed)
    return rng.standard_normal((cfg.tokens, cfg.d_model), dtype=np.float32)


class Block:
    """Device-resident weights plus preallocated activations for one config.

    Operands of the tensor-core GEMMs travel as exact tf32 splits (hi, lo):
    the weights are split (and transposed to K-major) once here; in the
    forward, layer_norm, attention and the GEMM epilogues write their results
    already split, so no kernel re-reads an operand just to split it;
    attention reads Q, K and V in place from the QKV output (V as the MN-major
    operand of its P.V product)."""

    MAX_GRAPHS = 8  # captured buffer sets kept (the oldest is dropped beyond this)
    # k values per TMEM accumulation chunk of the block's GEMMs: with weights
    # of ~0.02 the tensor core's truncating accumulation stays far inside the
    # dot tolerance over 384 k (measured |g - r| / bound <= 0.1 on the block's
    # distributions, 0.04 at the library default of 128), and the epilogue
    # stalls the MMAs a third as often (the forward 1.43 -> ~1.27 ms).
    ACC_CHUNK_K = 384

    def __init__(self, cfg, params, device="cuda", graphs=None):
        self.cfg = cfg
        self.dev = torch.device(device)
        # Each distinct (input, output, sequence range) runs eagerly once, is
        # then captured as a CUDA graph of its launches and replayed from then
        # on (SILCU_GRAPHS=0 or graphs=False: always eager).
        self.graphs = (os.environ.get("SILCU_GRAPHS", "1") != "0") if graphs is None else bool(graphs)
        self._graph_cache = {}
        self.replayed_launches = 0  # kernels launched by graph replays (the library counts the rest)
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(self.dev)  # noqa: E731
        d, f = cfg.d_model, cfg.d_ff
        self.g1, self.be1, self.g2, self.be2 = t(params["g1"]), t(params["be1"]), t(params["g2"]), t(params["be2"])
        wqkv = t(np.concatenate([params["wq"], params["wk"], params["wv"]], axis=1))  # [d, 3d]
        self.bqkv = t(np.concatenate([params["bq"], params["bk"], params["bv"]]))
        self.bo, self.b1, self.b2 = t(params["bo"]), t(params["b1"]), t(params["b2"])
        # K-major splits of the constant weights: W[K,N] -> (hi, lo) of W^T [N,K]
        self.wqkv_t = gpu.split(wqkv, d, 3 * d, transpose=True)
        self.wo_t = gpu.split(t(params["wo"]), d, d, transpose=True)
        self.w1_t = gpu.split(t(params["w1"]), d, f, transpose=True)
        self.w2_t = gpu.split(t(params["w2"]), f, d, transpose=True)
        T, S, H = cfg.tokens, cfg.seq, cfg.heads
        e = lambda *s: torch.empty(*s, dtype=torch.float32, device=self.dev)  # noqa: E731
        pair = lambda n: (e(n), e(n))  # noqa: E731
        self.h = pair(T * d)
        self.qkv = pair(T * 3 * d)
        self.ctx = pair(T * d)
        self.r1 = e(T * d)
        self.ff = pair(T * f)
        self.scale = float(np.float32(1.0) / np.sqrt(np.float32(cfg.head_dim)))
        self._x_dev = None  # device staging of forward_host, made on first use

    def forward(self, x, out=None):
        """One block forward of all cfg.batch sequences; x and out are device
        tensors of cfg.tokens x d_model."""
        cfg = self.cfg
        x = x.reshape(-1)
        out = torch.empty(cfg.tokens * cfg.d_model, dtype=torch.float32, device=self.dev) if out is None else out
        self._run(x, out.reshape(-1), 0, cfg.batch)
        return out.reshape(cfg.tokens, cfg.d_model)

    def forward_host(self, x_host, out_host, chunks=2):
        """The forward from host memory to host memory: the batch runs in
        `chunks` groups of sequences, and the copy of group c + 1 to the device
        and of group c - 1 back to the host overlap the compute of group c
        (three streams: copy in, compute = the current stream, copy out; pinned
        host buffers of cfg.tokens x d_model floats).  Ordered on the current
        stream: when it completes, out_host holds the result.  Two groups is
        the measured optimum at the bench shape: more groups hide more of the
        copies but shrink the GEMMs' M until their last wave runs mostly empty."""
        cfg = self.cfg
        S, d, B = cfg.seq, cfg.d_model, cfg.batch
        if not (x_host.is_pinned() and out_host.is_pinned()):
            raise ValueError("forward_host needs pinned host buffers")
        if x_host.numel() != cfg.tokens * d or out_host.numel() != cfg.tokens * d:
            raise ValueError("forward_host: buffers must hold cfg.tokens x d_model floats")
        chunks = max(1, min(int(chunks), B))
        if self._x_dev is None:
            self._x_dev = torch.empty(cfg.tokens * d, dtype=torch.float32, device=self.dev)
            self._o_dev = torch.empty(cfg.tokens * d, dtype=torch.float32, device=self.dev)
            self._s_in = torch.cuda.Stream(device=self.dev)
            self._s_out = torch.cuda.Stream(device=self.dev)
        xh, oh = x_host.reshape(-1), out_host.reshape(-1)
        comp = torch.cuda.current_stream(self.dev)
        bounds = [B * c // chunks for c in range(chunks + 1)]
        self._s_in.wait_stream(comp)
        self._s_out.wait_stream(comp)
        ready = []
        for c in range(chunks):
            r0, r1 = bounds[c] * S * d, bounds[c + 1] * S * d
            with torch.cuda.stream(self._s_in):
                self._x_dev[r0:r1].copy_(xh[r0:r1], non_blocking=True)
                ev = torch.cuda.Event()
                ev.record(self._s_in)
            ready.append(ev)
        for c in range(chunks):
            r0, r1 = bounds[c] * S * d, bounds[c + 1] * S * d
            comp.wait_event(ready[c])
            self._run(self._x_dev, self._o_dev, bounds[c], bounds[c + 1] - bounds[c])
            done = torch.cuda.Event()
            done.record(comp)
            self._s_out.wait_event(done)
            with torch.cuda.stream(self._s_out):
                oh[r0:r1].copy_(self._o_dev[r0:r1], non_blocking=True)
        comp.wait_stream(self._s_out)
        comp.wait_stream(self._s_in)
        return out_host

    def forward_host_stream(self, x_hosts, out_hosts):
        """Forwards of consecutive batches from host to host, overlapped
        across batches: while batch k computes, batch k + 1 is copied in and
        batch k - 1 is copied out (three streams, two device buffers each for
        input and output); the first and the last batch run as two
        half-batches, so their unoverlapped copies shrink by half.  x_hosts /
        out_hosts are sequences of pinned host buffers of cfg.tokens x d_model
        floats (an output buffer may be listed
        again two or more batches later: the copies into it stay in order).
        Ordered on the current stream: when it completes, every out_hosts[k]
        holds the forward of x_hosts[k]."""
        cfg = self.cfg
        n = cfg.tokens * cfg.d_model
        if len(x_hosts) != len(out_hosts):
            raise ValueError("forward_host_stream: as many outputs as inputs")
        for t in list(x_hosts) + list(out_hosts):
            if not t.is_pinned() or t.numel() != n:
                raise ValueError("forward_host_stream needs pinned host buffers of cfg.tokens x d_model floats")
        if getattr(self, "_stream_bufs", None) is None:
            e = lambda: torch.empty(n, dtype=torch.float32, device=self.dev)  # noqa: E731
            self._stream_bufs = ([e(), e()], [e(), e()])
            self._s_in2 = torch.cuda.Stream(device=self.dev)
            self._s_out2 = torch.cuda.Stream(device=self.dev)
        din, dout = self._stream_bufs
        comp = torch.cuda.current_stream(self.dev)
        self._s_in2.wait_stream(comp)
        self._s_out2.wait_stream(comp)
        computed = [None, None]  # per device buffer: the compute that last read din / wrote dout
        copied_out = [None, None]  # per device buffer: the copy that last read dout
        nbat = len(x_hosts)
        S, d, B = cfg.seq, cfg.d_model, cfg.batch
        for k in range(nbat):
            i = k & 1
            # The first and the last batch run as two half-batches, so that
            # the copy that nothing else can overlap (the first in, the last
            # out) overlaps the other half's compute.
            halves = [(0, B // 2), (B // 2, B - B // 2)] if (k == 0 or k == nbat - 1) and B >= 2 else [(0, B)]
            with torch.cuda.stream(self._s_in2):
                if computed[i] is not None:
                    self._s_in2.wait_event(computed[i])  # din[i] free once batch k - 2 computed
                ready = []
                for b0, nb in halves:
                    r0, r1 = b0 * S * d, (b0 + nb) * S * d
                    din[i][r0:r1].copy_(x_hosts[k].reshape(-1)[r0:r1], non_blocking=True)
                    ev = torch.cuda.Event()
                    ev.record(self._s_in2)
                    ready.append(ev)
            if copied_out[i] is not None:
                comp.wait_event(copied_out[i])  # dout[i] read out for batch k - 2
            done = []
            for (b0, nb), ev in zip(halves, ready):
                comp.wait_event(ev)
                self._run(din[i], dout[i], b0, nb)
                dn = torch.cuda.Event()
                dn.record(comp)
                done.append(dn)
            computed[i] = done[-1]
            with torch.cuda.stream(self._s_out2):
                for (b0, nb), dn in zip(halves, done):
                    r0, r1 = b0 * S * d, (b0 + nb) * S * d
                    self._s_out2.wait_event(dn)
                    out_hosts[k].reshape(-1)[r0:r1].copy_(dout[i][r0:r1], non_blocking=True)
                c = torch.cuda.Event()
                c.record(self._s_out2)
            copied_out[i] = c
        comp.wait_stream(self._s_out2)
        comp.wait_stream(self._s_in2)
        return out_hosts

    def _run(self, x, out, b0, nb):
        """_forward_seqs on the current stream, through a CUDA graph per
        (x, out, b0, nb) once that combination has run eagerly: the replay
        launches the same kernels with the same arguments, without the
        per-launch host work.  The graph keeps the shared workspace it was
        captured with alive (a later, larger request replaces the cached
        buffer but not this one)."""
        need = (b0 + nb) * self.cfg.seq * self.cfg.d_model
        on_dev = lambda t: t.device.type == self.dev.type and self.dev.index in (None, t.device.index)  # noqa: E731
        if x.numel() < need or out.numel() < need or not on_dev(x) or not on_dev(out):
            raise ValueError("Block: input / output must be device tensors of cfg.tokens x d_model floats")
        if not self.graphs:
            self._forward_seqs(x, out, b0, nb)
            return
        key = (x.data_ptr(), out.data_ptr(), b0, nb)
        g = self._graph_cache.get(key)
        if g is None:
            self._forward_seqs(x, out, b0, nb)  # sizes the workspace, sets kernel attributes, computes out
            graph = torch.cuda.CUDAGraph()
            n0 = gpu.lib().silcu_kernel_launches()
            with torch.cuda.graph(graph):
                self._forward_seqs(x, out, b0, nb)
            n = gpu.lib().silcu_kernel_launches() - n0
            if len(self._graph_cache) >= self.MAX_GRAPHS:  # bounded: drop the oldest capture
                old = self._graph_cache.pop(next(iter(self._graph_cache)))
                # the dropped graph's workspace may be its last reference: a replay of it
                # may still run on this stream, so free it only after the stream's work
                if old[2] is not None:
                    old[2].record_stream(torch.cuda.current_stream(self.dev))
            self._graph_cache[key] = (graph, n, gpu.workspace(0, self.dev))
            return
        g[0].replay()
        self.replayed_launches += g[1]

    def _forward_seqs(self, x, out, b0, nb):
        """Sequences [b0, b0 + nb) of the batch: every operand and activation
        is the view of those rows, so the groups of a chunked forward share
        nothing."""
        cfg = self.cfg
        d, f, S, H, hd = cfg.d_model, cfg.d_ff, cfg.seq, cfg.heads, cfg.head_dim
        T = nb * S
        t0 = b0 * S
        rows = lambda pair, w: (pair[0][t0 * w:(t0 + T) * w], pair[1][t0 * w:(t0 + T) * w])  # noqa: E731
        xs, outs = x[t0 * d:(t0 + T) * d], out[t0 * d:(t0 + T) * d]
        h, qkv, ctx, ff = rows(self.h, d), rows(self.qkv, 3 * d), rows(self.ctx, d), rows(self.ff, f)
        r1 = self.r1[t0 * d:(t0 + T) * d]
        qh, ql = qkv
        gpu.layer_norm_split(xs, self.g1, self.be1, T, d, cfg.eps, *h)
        ck = self.ACC_CHUNK_K
        gpu.gemm(h, self.wqkv_t, M=T, N=3 * d, K=d, trans_b=True, bias=self.bqkv, no_c=True, C_split=qkv,
                 acc_chunk_k=ck)
        # ctx[b*S + s, h*hd + j] = softmax(Q_bh . K_bh^T * scale) . V_bh, fused; Q_bh rows are
        # qkv[b*S + s, h*hd : h*hd + hd], K_bh the same at +d, V_bh at +2d: all read in place.
        gpu.attention((qh, ql), (qh[d:], ql[d:]), None, V=(qh[2 * d:], ql[2 * d:]), Sq=S, Sk=S, batch=nb,
                      heads=H, ldq=3 * d, sq_b=S * 3 * d, sq_h=hd, ldk=3 * d, sk_b=S * 3 * d, sk_h=hd,
                      ldv=3 * d, sv_b=S * 3 * d, sv_h=hd, scale=self.scale,
                      O_split=ctx, ldo=d, so_b=S * d, so_h=hd)
        gpu.gemm(ctx, self.wo_t, r1, M=T, N=d, K=d, trans_b=True, bias=self.bo, residual=xs, acc_chunk_k=ck)
        gpu.layer_norm_split(r1, self.g2, self.be2, T, d, cfg.eps, *h)
        gpu.gemm(h, self.w1_t, M=T, N=f, K=d, trans_b=True, bias=self.b1, act="relu", no_c=True, C_split=ff,
                 acc_chunk_k=ck)
        gpu.gemm(ff, self.w2_t, outs, M=T, N=d, K=f, trans_b=True, bias=self.b2, residual=r1, acc_chunk_k=ck)


def init_head(vocab, d_model, seed=0):
    """A loss head's parameters: gamma 1, beta 0, W [vocab, d_model] ~ N(0, 0.02^2)."""
    rng = np.random.default_rng(seed)
    return {"g": np.ones(d_model, np.float32), "be": np.zeros(d_model, np.float32),
            "w": _normal(rng, (vocab, d_model), 0.02)}


class LossHead:
    """What follows the last block in training: the final layer_norm, the
    vocabulary projection with its mean cross entropy, their gradients, and
    the clipping of the parameters' gradients.

        loss = head.forward(block.forward(x), targets)   # 0-d device tensor
        dx = head.backward()                              # gradient of the block's output
        norm = head.clip(1.0)                             # head.grads, in place

    Activations and W are fp32, or bf16 with dtype=torch.bfloat16 (gamma, beta
    and their gradients stay fp32).  Targets are int32; one outside
    [0, vocab) leaves its row out.  A whole step can be captured in a CUDA graph.

    forward keeps x and targets themselves for backward, not copies: their buffers (a block's
    output may be written again by its next forward) stay as they are until then.  backward
    writes self.grads, it does not add to them."""

    def __init__(self, params, device="cuda", dtype=torch.float32, eps=1e-5):
        t = lambda a, dt: torch.from_numpy(np.ascontiguousarray(a)).to(device, dt)  # noqa: E731
        self.gamma, self.beta = t(params["g"], torch.float32), t(params["be"], torch.float32)
        self.w = t(params["w"], dtype)
        self.eps = eps
        self.grads = {"g": torch.empty_like(self.gamma), "be": torch.empty_like(self.beta),
                      "w": torch.empty_like(self.w)}
        self._grad_list = gpu.TensorList(self.grads.values())
        self._saved = None

    def forward(self, x, targets):
        """Mean loss of x [rows, d_model] against targets [rows]."""
        h, mean, rstd = gpu.layer_norm_forward(x, gamma=self.gamma, beta=self.beta, eps=self.eps)
        loss, lse = gpu.linear_cross_entropy(h, self.w, targets)
        self._saved = (x, targets, h, mean, rstd, lse)
        return loss

    def backward(self, dloss=None, dresidual=None):
        """Gradient of the last forward's x (dresidual is added to it); the
        parameters' gradients are written to self.grads.  dloss: 0-d, None = 1."""
        if self._saved is None:
            raise RuntimeError("LossHead: backward without a forward")
        x, targets, h, mean, rstd, lse = self._saved
        dh, _ = gpu.linear_cross_entropy_backward(h, self.w, targets, lse, dloss=dloss, dW=self.grads["w"])
        dx, _, _ = gpu.layer_norm_backward(dh, x, mean, rstd, self.gamma, dresidual=dresidual, din=dh,
                                           dgamma=self.grads["g"], dbeta=self.grads["be"])
        return dx

    def clip(self, max_norm):
        """Clips self.grads by their common norm; returns it (0-d)."""
        self._grad_list.tensors = list(self.grads.values())  # whatever tensors are there now
        return gpu.clip_grad_norm(self._grad_list, max_norm)
