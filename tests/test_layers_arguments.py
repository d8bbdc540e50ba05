"""CPU tests of the argument checks of the group norm, the 8-bit rows and their product, and the orthogonalised
update: what is refused is refused with a message before anything runs."""
import os
import subprocess

import pytest
import torch

import xspmm_b200 as xs
from xspmm_b200 import _lib

f16, bf16, f32, f64 = torch.float16, torch.bfloat16, torch.float32, torch.float64


class Reached(Exception):
    """Raised where a call would have gone to the library."""


class HostExecutor:
    """Stands in for an executor: its tensors live on the host and no call gets past the checks."""
    device = torch.device("cpu")

    @property
    def handle(self):
        raise Reached


EX = HostExecutor()


def t(*shape, dtype=f16):
    return torch.zeros(*shape, dtype=dtype)


def refused(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(EX, *args, **kw)


def reached(fn, *args, **kw):
    with pytest.raises(Reached):
        fn(EX, *args, **kw)


def test_group_norm():
    x, w, off, m = t(6, 8), t(8, dtype=f32), torch.tensor([0, 2, 6]), t(2, 4, dtype=f32)
    reached(xs.group_norm, x, 4, w, w, 1e-5, x, offsets=off, activation="silu", mean=m, rstd=m)
    reached(xs.group_norm, t(6, 30)[:, 3:11], 1, None, None, 0.0, x)
    reached(xs.group_norm, t(0, 8), 8, None, None, 0.0, t(0, 8))
    reached(xs.group_norm, x.float(), 4, w, w, 1e-5, x.bfloat16())
    refused("takes", xs.group_norm, x, 4, w, w, 1e-5, x.float())
    refused("takes", xs.group_norm, x.double(), 4, w, w, 1e-5, x.double())
    refused("groups must", xs.group_norm, x, 3, w, w, 1e-5, x)
    refused("groups must", xs.group_norm, x, 0, w, w, 1e-5, x)
    refused("groups must", xs.group_norm, x, 2.0, w, w, 1e-5, x)
    refused("at most 16384", xs.group_norm, t(1, 16385), 1, None, None, 1e-5, t(1, 16385))
    refused("at least one column", xs.group_norm, t(6, 0), 1, None, None, 1e-5, t(6, 0))
    refused("eps must", xs.group_norm, x, 4, w, w, float("nan"), x)
    refused("eps must", xs.group_norm, x, 4, w, w, -1e-5, x)
    refused("activation must", xs.group_norm, x, 4, w, w, 1e-5, x, activation="tanh")
    refused("y must be 6 x 8", xs.group_norm, x, 4, w, w, 1e-5, t(6, 7))
    refused("weight must be", xs.group_norm, x, 4, t(8), w, 1e-5, x)
    refused("bias must be", xs.group_norm, x, 4, w, t(7, dtype=f32), 1e-5, x)
    refused("offsets must be torch.int64", xs.group_norm, x, 4, w, w, 1e-5, x, offsets=off.int())
    refused("one more value", xs.group_norm, x, 4, w, w, 1e-5, x, offsets=off[:0])
    refused("one more value", xs.group_norm, x, 4, w, w, 1e-5, x, offsets=off[None])
    refused("offsets must be contiguous", xs.group_norm, x, 4, w, w, 1e-5, x, offsets=torch.zeros(6, dtype=torch.int64)[::2])
    refused("executor on", xs.group_norm, x, 4, w, w, 1e-5, x, offsets=off.to("meta"))
    refused("mean must be", xs.group_norm, x, 4, w, w, 1e-5, x, mean=m)  # one sample without offsets
    refused("rstd must be", xs.group_norm, x, 4, w, w, 1e-5, x, offsets=off, rstd=t(2, 3, dtype=f32))
    refused("contiguous rows", xs.group_norm, t(8, 6).t(), 4, w, w, 1e-5, x)


def test_group_norm_backward():
    x, w, off, m = t(6, 8), t(8, dtype=f32), torch.tensor([0, 2, 6]), t(2, 4, dtype=f32)
    reached(xs.group_norm_backward, x, x, 4, w, w, m, m, x, w, w, offsets=off, activation="gelu")
    reached(xs.group_norm_backward, x.bfloat16(), x.float(), 4, None, None, m, m, offsets=off)
    refused("dy must be 6 x 8", xs.group_norm_backward, t(5, 8), x, 4, w, w, m, m, offsets=off)
    refused("takes", xs.group_norm_backward, x.float(), x, 4, w, w, m, m, offsets=off)
    refused("dx must be torch.float16", xs.group_norm_backward, x, x, 4, w, w, m, m, x.float(), offsets=off)
    refused("mean is needed", xs.group_norm_backward, x, x, 4, w, w, None, m, offsets=off)
    refused("rstd is needed", xs.group_norm_backward, x, x, 4, w, w, m, None, offsets=off)
    refused("mean must be", xs.group_norm_backward, x, x, 4, w, w, m, m)
    refused("dweight must be", xs.group_norm_backward, x, x, 4, w, w, m, m, x, x, offsets=off)
    refused("dbias must be", xs.group_norm_backward, x, x, 4, w, w, m, m, x, w, w[:7], offsets=off)


def test_quantize_rows():
    x, q, s = t(4, 8), t(4, 8, dtype=torch.int8), t(4, dtype=f32)
    reached(xs.quantize_rows, x, q, s)
    reached(xs.quantize_rows, t(4, 20)[:, 1:9], t(4, 11, dtype=torch.int8)[:, :8], s)
    refused("takes no", xs.quantize_rows, x.double(), q, s)
    refused("q must be torch.int8", xs.quantize_rows, x, x, s)
    refused("q must be 4 x 8", xs.quantize_rows, x, q[:3], s)
    refused("scale is needed", xs.quantize_rows, x, q, None)
    refused("scale must be", xs.quantize_rows, x, q, s[:3])
    refused("scale must be torch.float32", xs.quantize_rows, x, q, s.half())
    refused("executor on", xs.quantize_rows, x.to("meta"), q, s)


def test_linear_int8():
    x, w, a, b, y = t(4, 8, dtype=torch.int8), t(6, 8, dtype=torch.int8), t(4, dtype=f32), t(6, dtype=f32), t(4, 6)
    reached(xs.linear_int8, x, a, w, b, y)
    reached(xs.linear_int8, x, a, w, b, y.float(), bias=b)
    refused("x must be torch.int8", xs.linear_int8, x.half(), a, w, b, y)
    refused("w must be torch.int8", xs.linear_int8, x, a, w.to(torch.uint8), b, y)
    refused("w must be rows x 8", xs.linear_int8, x, a, w[:, :7], b, y)
    refused("x_scale is needed", xs.linear_int8, x, None, w, b, y)
    refused("w_scale is needed", xs.linear_int8, x, a, w, None, y)
    refused("x_scale must be", xs.linear_int8, x, b, w, b, y)
    refused("w_scale must be", xs.linear_int8, x, a, w, a, y)
    refused("bias must be", xs.linear_int8, x, a, w, b, y, bias=a)
    refused("y must be 4 x 6", xs.linear_int8, x, a, w, b, y[:, :5])
    refused("gives no", xs.linear_int8, x, a, w, b, y.double())
    refused("at most 131071", xs.linear_int8, t(1, 131072, dtype=torch.int8), a[:1], t(6, 131072, dtype=torch.int8), b, y[:1])
    refused("contiguous rows", xs.linear_int8, x, a, t(8, 6, dtype=torch.int8).t(), b, y)


def test_orthogonalize():
    g, y = t(4, 8, dtype=f32), t(4, 8)
    reached(xs.orthogonalize, g, y)
    reached(xs.orthogonalize, y, y, steps=0, eps=0)
    refused("takes", xs.orthogonalize, g, g)
    refused("takes", xs.orthogonalize, y, y.bfloat16())
    refused("takes", xs.orthogonalize, g.double(), y)
    refused("y must be 4 x 8", xs.orthogonalize, g, t(8, 4))
    refused("steps must", xs.orthogonalize, g, y, steps=-1)
    refused("steps must", xs.orthogonalize, g, y, steps=101)
    refused("steps must", xs.orthogonalize, g, y, steps=2.0)
    refused("eps must", xs.orthogonalize, g, y, eps=float("inf"))
    refused("eps must", xs.orthogonalize, g, y, eps=-1.0)
    refused("g must be rows x cols", xs.orthogonalize, g[None], y)
    refused("overlap", xs.orthogonalize, g[:1].expand(4, 8), y)


def test_eps_past_fp32():
    """eps becomes float32 on its way: what is infinite there is refused like an infinity."""
    x, g, w = t(6, 8), t(4, 8, dtype=f32), t(8, dtype=f32)
    for eps in (1e39, 1e308, float("inf"), float("nan"), -1e-300):
        refused("eps must", xs.layer_norm, x, w, w, eps, x)
        refused("eps must", xs.group_norm, x, 4, w, w, eps, x)
        refused("eps must", xs.orthogonalize, g, t(4, 8), eps=eps)
    for eps in (0, 1, 1e-300, 3.4e38):
        reached(xs.layer_norm, x, w, w, eps, x)
        reached(xs.group_norm, x, 4, w, w, eps, x)
        reached(xs.orthogonalize, g, t(4, 8), eps=eps)


def test_c_entries_reject_a_null_handle():
    L = _lib.lib()
    for suf in ("f16f16", "bf16bf16", "f32f32", "f32f16", "f32bf16"):
        assert getattr(L, "xspmm_group_norm_" + suf)(None, 1, 8, 1, 1, None, None, 8, None, None, 1e-5, -1, None, 8, None, None) == 1
        assert getattr(L, "xspmm_group_norm_backward_" + suf)(
            None, 1, 8, 1, 1, None, None, 8, None, 8, None, None, None, None, -1, None, 8, None, None) == 1
    for suf in ("f16", "bf16", "f32"):
        assert getattr(L, "xspmm_quantize_rows_" + suf)(None, 1, 8, None, 8, None, 8, None) == 1
        assert getattr(L, "xspmm_linear_int8_" + suf)(None, 1, 8, 8, None, 8, None, None, 8, None, None, None, 8) == 1
    for suf in ("f16f16", "bf16bf16", "f32f16", "f32bf16"):
        assert getattr(L, "xspmm_orthogonalize_" + suf)(None, 1, 8, None, 8, 5, 1e-7, None, 8) == 1
    assert b"null handle" in L.xspmm_last_error()


_CPP = r"""
#include "xspmm/layers.hpp"
using E = std::shared_ptr<const xspmm::Executor>;
template <typename X, typename Y> void group(E e, X* x, Y* y, float* f, const int64_t* o) {
    xspmm::group_norm<X, Y>(e, 4, 8, 2, {}, {x, 8}, f, f, 1e-5f, xspmm::Activation::None, {y, 8});
    xspmm::group_norm_backward<X, Y>(e, 4, 8, 2, {3, o}, {y, 8}, {x, 8}, f, f, f, f, xspmm::Activation::Silu, {y, 8}, f, f);
}
template <typename T> void narrow(E e, T* x, int8_t* q, float* s) {
    xspmm::quantize_rows<T>(e, 4, 8, {x, 8}, {q, 8}, s);
    xspmm::linear_int8<T>(e, 4, 8, 6, {q, 8}, s, {q, 8}, s, {x, 6}, s);
}
template <typename X, typename Y> void update(E e, X* x, Y* y) { xspmm::orthogonalize<X, Y>(e, 4, 8, {x, 8}, {y, 8}); }
template void group(E, __half*, __half*, float*, const int64_t*);
template void group(E, __nv_bfloat16*, __nv_bfloat16*, float*, const int64_t*);
template void group(E, float*, float*, float*, const int64_t*);
template void group(E, float*, __half*, float*, const int64_t*);
template void group(E, float*, __nv_bfloat16*, float*, const int64_t*);
template void narrow(E, __half*, int8_t*, float*);
template void narrow(E, __nv_bfloat16*, int8_t*, float*);
template void narrow(E, float*, int8_t*, float*);
template void update(E, __half*, __half*);
template void update(E, __nv_bfloat16*, __nv_bfloat16*);
template void update(E, float*, __half*);
template void update(E, float*, __nv_bfloat16*);
"""


def test_cpp_header_instantiates_every_type(tmp_path):
    src = tmp_path / "layers.cpp"
    src.write_text(_CPP)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run(["g++", "-std=c++20", "-fsyntax-only", "-I" + os.path.join(root, "include"),
                        "-I/usr/local/cuda/include", str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
