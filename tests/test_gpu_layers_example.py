"""The layer operators together, as a graph layer uses them (examples/gated_graph_layer.py): the loss falls,
one step's forward and backward pass equal a 64-bit restatement with the same dropout mask, and the calls
can be captured in a CUDA graph."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import xspmm_b200 as xs
from xspmm_b200 import synth

pytestmark = pytest.mark.gpu

_PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                     "gated_graph_layer.py")
_spec = importlib.util.spec_from_file_location("gated_graph_layer", _PATH)
example = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(example)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_the_loss_falls(dtype):
    losses = example.main(["--nodes-log2", "11", "--steps", "4", "--dtype", dtype])
    assert all(np.isfinite(losses)) and losses[-1] < losses[0]


def _layer(executor, width=96, dtype=torch.bfloat16):
    P = synth.cfg5_rmat(seed=5, scale=9, N=width)
    layer = example.GatedGraphLayer(executor, P.M, P.row_ptr, P.col_ind, P.values, width, dtype, p=0.25)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    layer.norm_w.normal_(1.0, 0.2, generator=g)
    layer.norm_b.normal_(0.0, 0.2, generator=g)
    x = torch.randn(P.M, width, generator=g, device="cuda").to(dtype)
    dy = torch.randn(P.M, width, generator=g, device="cuda").to(dtype)
    dense = torch.zeros(P.M, P.M, dtype=torch.float64)
    v = torch.as_tensor(np.asarray(P.values, np.float32)).to(dtype).double()
    for r in range(P.M):  # a later duplicate of a column replaces an earlier one, as in the conversion
        for j in range(P.row_ptr[r], P.row_ptr[r + 1]):
            dense[r, P.col_ind[j]] = v[j]
    return layer, x, dy, dense.cuda()


def test_one_step_against_64_bits(executor):
    """Relative Frobenius error of every result. bf16 rounds at most eight times along the longest chain
    (n, gate, up, dh, dg or du, dn, dagg, the result), each by at most 2^-8 of a value and 2^-8 / sqrt(3) of
    its norm at random; 8 * 2^-8 bounds their sum."""
    layer, x, dy, A = _layer(executor)
    y = layer.forward(x).clone()
    ones = torch.ones_like(x)
    mask = torch.empty_like(x)
    xs.dropout(executor, ones, layer.p, layer.seed, layer.offset, mask)
    mask = (mask != 0).double() / (1 - layer.p)
    dx = layer.backward(dy)
    leaves = [t.double().requires_grad_() for t in (x, layer.wg, layer.wu, layer.norm_w, layer.norm_b)]
    x64, wg, wu, nw, nb = leaves
    agg = A @ x64
    c = agg - agg.mean(1, keepdim=True)
    n = c / torch.sqrt((c * c).mean(1, keepdim=True) + layer.eps) * nw + nb
    g = n @ wg.t()
    ref = x64 + mask * (g * torch.sigmoid(g) * (n @ wu.t()))
    grads = torch.autograd.grad((ref * dy.double()).sum(), leaves)
    got = (y, dx + dy.float(), layer.dwg, layer.dwu, layer.dnw, layer.dnb)
    for a, b, name in zip(got, (ref.detach(), *grads), ("y", "dx", "dwg", "dwu", "dnw", "dnb")):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel <= 8 * 2.0 ** -8, (name, rel)


def test_capture_in_a_graph(executor):
    """A captured pass, replayed on new inputs in the same buffers, gives the bits of a direct one."""
    layer, x, dy, _ = _layer(executor, dtype=torch.float16)
    x2 = x.flip(0).contiguous()
    layer.forward(x2)
    want = [t.clone() for t in (layer.forward(x2), layer.gate)]
    layer.backward(dy)
    want += [t.clone() for t in (layer.dwg, layer.dnw, layer.dn)]
    layer.offset = 0
    buf = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.forward(buf)
        layer.backward(dy)
    torch.cuda.current_stream().wait_stream(side)
    layer.offset = 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.forward(buf)
        layer.backward(dy)
    buf.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip((layer.y, layer.gate, layer.dwg, layer.dnw, layer.dn), want):
        assert torch.equal(a, b)
