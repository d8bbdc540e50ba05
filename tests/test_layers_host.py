"""CPU tests of the layer operators' argument checks (xspmm_b200/layers.py and the C entries behind
it): what is refused is refused with a message before anything runs. No kernel is launched."""
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


def refused(fn, match):
    with pytest.raises(ValueError, match=match):
        fn()


def test_layer_norm_refusals():
    w = t(8, dtype=f32)
    ok = dict(mean=t(4, dtype=f32), rstd=t(4, dtype=f32))
    with pytest.raises(Reached):
        xs.layer_norm(EX, t(4, 8), w, w, 1e-5, t(4, 8), **ok)
    with pytest.raises(Reached):  # a slice of columns keeps its row stride
        xs.layer_norm(EX, t(4, 20)[:, 3:11], None, None, 1e-5, t(4, 8))
    refused(lambda: xs.layer_norm(EX, t(4, 8), w, w, 1e-5, t(4, 8, dtype=f32)), "takes")
    refused(lambda: xs.layer_norm(EX, t(4, 8, dtype=f64), w, w, 1e-5, t(4, 8)), "takes")
    refused(lambda: xs.layer_norm(EX, t(4, 8), w, w, 1e-5, t(4, 7)), "y must be 4 x 8")
    refused(lambda: xs.layer_norm(EX, t(8), w, w, 1e-5, t(8)), "x must be rows x cols")
    refused(lambda: xs.layer_norm(EX, t(8, 4).t(), w, w, 1e-5, t(4, 8)), "contiguous rows")
    refused(lambda: xs.layer_norm(EX, t(1, 8).expand(4, 8), w, w, 1e-5, t(4, 8)), "overlap")
    refused(lambda: xs.layer_norm(EX, t(4, 8), t(8), w, 1e-5, t(4, 8)), "weight must be torch.float32")
    refused(lambda: xs.layer_norm(EX, t(4, 8), t(7, dtype=f32), w, 1e-5, t(4, 8)), "weight must be")
    refused(lambda: xs.layer_norm(EX, t(4, 8), w, w, 1e-5, t(4, 8), mean=t(3, dtype=f32)), "mean")
    refused(lambda: xs.layer_norm_backward(EX, t(4, 8), t(4, 7), w, *ok.values()), "x must be 4 x 8")
    refused(lambda: xs.layer_norm_backward(EX, t(4, 8), t(4, 8), w, *ok.values(),
                                           dx=t(4, 8, dtype=f32)), "dx must be torch.float16")
    refused(lambda: xs.layer_norm_backward(EX, t(4, 8, dtype=bf16), t(4, 8), w, *ok.values()), "takes")


def test_dropout_refusals():
    x = t(4, 8)
    with pytest.raises(Reached):
        xs.dropout(EX, x, 0.5, 2 ** 64 - 1, 0, x, residual=x)
    refused(lambda: xs.dropout(EX, x, 1.5, 0, 0, x), "p must lie")
    refused(lambda: xs.dropout(EX, x, float("nan"), 0, 0, x), "p must lie")
    refused(lambda: xs.dropout(EX, x, 0.5, -1, 0, x), "unsigned")
    refused(lambda: xs.dropout(EX, x, 0.5, 0, 2 ** 64, x), "unsigned")
    refused(lambda: xs.dropout(EX, t(4, 8, dtype=f64), 0.5, 0, 0, x), "takes no")
    refused(lambda: xs.dropout(EX, x, 0.5, 0, 0, t(4, 8, dtype=f32)), "y must be")
    refused(lambda: xs.dropout(EX, x, 0.5, 0, 0, t(8, 4)), "y must be")
    refused(lambda: xs.dropout(EX, t(4, 16)[:, :8], 0.5, 0, 0, x), "x must be contiguous")
    refused(lambda: xs.dropout(EX, x, 0.5, 0, 0, x, residual=t(4, 7)), "residual must be")
    refused(lambda: xs.dropout_backward(EX, x, -0.1, 0, 0, x), "p must lie")


def test_gated_ffn_refusals():
    x, w, y = t(4, 8), t(6, 8), t(4, 6)
    with pytest.raises(Reached):
        xs.gated_ffn(EX, x, w, w, y, "gelu", y, y)
    refused(lambda: xs.gated_ffn(EX, x, w, w, y, activation="tanh"), "activation must be")
    refused(lambda: xs.gated_ffn(EX, x.float(), w.float(), w.float(), y.float()), "16-bit types")
    refused(lambda: xs.gated_ffn(EX, x, w, t(5, 8), y), "w_up must be 6 x 8")
    refused(lambda: xs.gated_ffn(EX, x, w.bfloat16(), w, y), "w_gate must be torch.float16")
    refused(lambda: xs.gated_ffn(EX, x, w, w, t(4, 5)), "y must be 4 x 6")
    refused(lambda: xs.gated_ffn(EX, x, t(8, 6).t(), w, y), "w_gate must have contiguous rows")
    refused(lambda: xs.gated_ffn(EX, x, w, w, y, gate=t(4, 12)[:, :6]), "gate must be contiguous")
    refused(lambda: xs.gated_ffn_backward(EX, t(3, 6), x, w, w, y, y), "dy must be 4 x 6")
    refused(lambda: xs.gated_ffn_backward(EX, y, x, w, w, y, y, dw_gate=t(8, 6)), "dw_gate must be")


def test_tensors_of_another_device_are_refused():
    refused(lambda: xs.gated_ffn(EX, t(4, 8).to("meta"), t(6, 8), t(6, 8), t(4, 6)), "executor on")
    refused(lambda: xs.dropout(EX, t(4, 8).to("meta"), 0.5, 0, 0, t(4, 8)), "executor on")


def test_c_entries_reject_a_null_handle():
    L = _lib.lib()
    assert L.xspmm_layer_norm_f32f16(None, 1, 8, None, 8, None, None, 1e-5, None, 8, None, None) == 1
    assert L.xspmm_layer_norm_backward_bf16bf16(None, 1, 8, None, 8, None, 8, None, None, None, None,
                                                8, None, None) == 1
    assert L.xspmm_dropout_f32(None, 4, None, None, 0.5, 1, 2, None) == 1
    assert L.xspmm_gated_ffn_f16(None, 1, 8, 8, 0, None, 8, None, 8, None, 8, None, 8, None, None) == 1
    assert L.xspmm_gated_ffn_backward_bf16(None, 1, 8, 8, 0, None, 8, None, 8, None, 8, None, 8, None,
                                           None, None, 8, None, None) == 1
    assert b"null handle" in L.xspmm_last_error()


_CPP = r"""
#include "xspmm/layers.hpp"
using E = std::shared_ptr<const xspmm::Executor>;
template <typename X, typename Y> void norm(E e, X* x, Y* y, float* f) {
    xspmm::layer_norm<X, Y>(e, 4, 8, {x, 8}, f, f, 1e-5f, {y, 8}, f, f);
    xspmm::layer_norm_backward<X, Y>(e, 4, 8, {y, 8}, {x, 8}, f, f, f, {y, 8}, f, f);
}
template <typename T> void drop(E e, T* x) { xspmm::dropout<T>(e, 8, x, nullptr, 0.5, 1u, 2u, x); }
template <typename T> void gated(E e, T* t) {
    xspmm::gated_ffn<T>(e, 4, 8, 6, xspmm::Activation::Gelu, {t, 8}, {t, 8}, {t, 8}, {t, 6}, t, t);
    xspmm::gated_ffn_backward<T>(e, 4, 8, 6, xspmm::Activation::Silu, {t, 6}, {t, 8}, {t, 8}, {t, 8}, t, t,
                                 {t, 8}, t, t);
}
template void norm(E, __half*, __half*, float*);
template void norm(E, __nv_bfloat16*, __nv_bfloat16*, float*);
template void norm(E, float*, float*, float*);
template void norm(E, float*, __half*, float*);
template void norm(E, float*, __nv_bfloat16*, float*);
template void drop(E, __half*);
template void drop(E, __nv_bfloat16*);
template void drop(E, float*);
template void gated(E, __half*);
template void gated(E, __nv_bfloat16*);
"""


def test_cpp_header_instantiates_every_type(tmp_path):
    src = tmp_path / "layers.cpp"
    src.write_text(_CPP)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run(["g++", "-std=c++20", "-fsyntax-only", "-I" + os.path.join(root, "include"),
                        "-I/usr/local/cuda/include", str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
