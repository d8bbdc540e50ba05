"""One training step of a gated graph layer, every operator a call into the library.

    x -> A x -> layer norm -> act(n Wg^T) * (n Wu^T) -> dropout -> + x

A is the graph (rows normalised by degree) as a plan for the sparse product, whose fp32 output the layer
norm turns into the 16-bit operand of the projections; the backward pass ends in the 16-bit operand of
the transposed product. The loss is the mean squared distance to a target; the weights take one step of
gradient descent, and the loss before and after is printed.

    python examples/gated_graph_layer.py [--nodes-log2 14] [--steps 5] [--dtype fp16|bf16]
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import xspmm_b200 as xs  # noqa: E402
from xspmm_b200 import synth  # noqa: E402


def transpose_csr(rows, row_ptr, col, val):
    """The transposed matrix of a square CSR matrix (host arrays)."""
    src = np.repeat(np.arange(rows), np.diff(row_ptr))
    order = np.argsort(col, kind="stable")
    ptr = np.zeros(rows + 1, dtype=np.int64)
    np.cumsum(np.bincount(col, minlength=rows), out=ptr[1:])
    return ptr, src[order], val[order]


class GatedGraphLayer:
    """Keeps the plans of the graph and of its transpose, the parameters and the buffers of a step."""

    def __init__(self, ex, rows, row_ptr, col, val, width, dtype, p=0.1, eps=1e-5, seed=0):
        self.ex, self.rows, self.width, self.p, self.eps = ex, rows, width, p, eps
        v = torch.as_tensor(np.asarray(val, np.float32)).to(dtype)
        self.graph = xs.SpMMPlan(ex, xs.CSRMatrix.from_host(ex, rows, rows, row_ptr, col, v))
        tp, tc, tv = transpose_csr(rows, row_ptr, col, v.float().numpy())
        self.graph_t = xs.SpMMPlan(ex, xs.CSRMatrix.from_host(ex, rows, rows, tp, tc,
                                                              torch.as_tensor(tv).to(dtype)))
        d, g = ex.device, torch.Generator(device=ex.device)
        g.manual_seed(seed)
        self.norm_w, self.norm_b = torch.ones(width, device=d), torch.zeros(width, device=d)
        self.wg, self.wu = (torch.randn(width, width, generator=g, device=d).mul_(width ** -0.5).to(dtype)
                            for _ in range(2))
        self.seed, self.offset = seed, 0

        def buf(t=dtype):
            return torch.empty(rows, width, dtype=t, device=d)

        self.agg, self.n, self.gate, self.up, self.h, self.y = buf(torch.float32), buf(), buf(), buf(), buf(), buf()
        self.mean, self.rstd = torch.empty(rows, device=d), torch.empty(rows, device=d)
        self.dh, self.dn, self.dagg, self.dx = buf(), buf(), buf(), buf(torch.float32)
        self.dwg, self.dwu = torch.empty_like(self.wg), torch.empty_like(self.wu)
        self.dnw, self.dnb = torch.empty_like(self.norm_w), torch.empty_like(self.norm_b)

    def forward(self, x):
        ex = self.ex
        self.graph.execute(x, self.agg, self.width)
        xs.layer_norm(ex, self.agg, self.norm_w, self.norm_b, self.eps, self.n, self.mean, self.rstd)
        xs.gated_ffn(ex, self.n, self.wg, self.wu, self.h, "silu", self.gate, self.up)
        xs.dropout(ex, self.h, self.p, self.seed, self.offset, self.y, residual=x)
        return self.y

    def backward(self, dy):
        """Gradients of the parameters, and of x in fp32 (without the residual's own, which is dy)."""
        ex = self.ex
        xs.dropout_backward(ex, dy, self.p, self.seed, self.offset, self.dh)
        self.offset += -(-dy.numel() // 4)  # the next step draws a new mask
        xs.gated_ffn_backward(ex, self.dh, self.n, self.wg, self.wu, self.gate, self.up, self.dn,
                              self.dwg, self.dwu)
        xs.layer_norm_backward(ex, self.dn, self.agg, self.norm_w, self.mean, self.rstd, self.dagg,
                               self.dnw, self.dnb)
        self.graph_t.execute(self.dagg, self.dx, self.width)
        return self.dx

    def step(self, lr):
        for w, d in ((self.wg, self.dwg), (self.wu, self.dwu), (self.norm_w, self.dnw), (self.norm_b, self.dnb)):
            w.sub_(d, alpha=lr)


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--nodes-log2", type=int, default=14)
    ap.add_argument("--width", type=int, default=128)
    ap.add_argument("--steps", type=int, default=5)
    ap.add_argument("--dtype", choices=("fp16", "bf16"), default="bf16")
    a = ap.parse_args(argv)
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}[a.dtype]
    ex = xs.CudaExecutor(0)
    P = synth.cfg5_rmat(seed=3, scale=a.nodes_log2, N=a.width)
    layer = GatedGraphLayer(ex, P.M, P.row_ptr, P.col_ind, P.values, a.width, dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn(P.M, a.width, generator=g, device="cuda").to(dtype)
    target = torch.randn(P.M, a.width, generator=g, device="cuda")
    losses = []
    for _ in range(a.steps):
        diff = layer.forward(x).float() - target
        losses.append(diff.square().mean().item())
        # the mean's gradient, scaled up by `scale` so that it does not vanish in fp16
        scale = 1024.0 * a.width
        layer.backward((diff * (2.0 / diff.numel() * scale)).to(dtype))
        layer.step(lr=0.05 * a.width / scale)
    print(f"nodes={P.M} nnz={P.nnz} width={a.width} loss " + " ".join(f"{v:.6f}" for v in losses))
    return losses


if __name__ == "__main__":
    main()
