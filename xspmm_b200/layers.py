"""The operators of the layer around the sparse product, over the C ABI: layer norm, dropout and the
gated feed-forward block, each with its gradient.

Rows are nodes or tokens and features are contiguous, as in B and C of `spmm`. Matrices are 2-D
device tensors whose last dimension has stride 1; their row stride is free (a slice of columns of
a wider tensor is taken as it is), except where a function says contiguous. Outputs are the
caller's tensors and are overwritten. Work is enqueued on torch's current stream; nothing
synchronizes. Wrong shapes, types, strides, devices or values and missing inputs raise ValueError
before anything runs.
"""
from __future__ import annotations

import math

import torch

from ._lib import check, lib
from .api import _VAL, CudaExecutor

_ACT = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
_NORM_TYPES = ("f16f16", "bf16bf16", "f32f32", "f32f16", "f32bf16")


def _matrix(exec: CudaExecutor, t: torch.Tensor, name: str, rows=None, cols=None, dtype=None):
    """Checks a matrix argument; returns its address and row stride."""
    shape = t.shape
    if len(shape) != 2 or (rows is not None and shape[0] != rows) or (
            cols is not None and shape[1] != cols):
        want = ("rows" if rows is None else rows, "cols" if cols is None else cols)
        raise ValueError(f"{name} must be {want[0]} x {want[1]}, got {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != exec.device:
        raise ValueError(f"{name} on {t.device}, executor on {exec.device}")
    rows, cols = shape
    if rows == 0 or cols == 0:
        return None, cols
    ld, unit = t.stride()
    if unit != 1 and cols > 1:
        raise ValueError(f"{name} must have contiguous rows")
    if rows == 1:
        return t.data_ptr(), cols
    if ld < cols:
        raise ValueError(f"the rows of {name} must not overlap")
    return t.data_ptr(), ld


def _dense(exec: CudaExecutor, t, name: str, shape, dtype):
    """Checks a contiguous argument (or None); returns its address."""
    if t is None:
        return None
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != exec.device:
        raise ValueError(f"{name} on {t.device}, executor on {exec.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr() or None


def _needed(exec: CudaExecutor, t, name: str, shape, dtype):
    """Checks a contiguous argument that may not be None; returns its address."""
    if t is None:
        raise ValueError(f"{name} is needed")
    return _dense(exec, t, name, shape, dtype)


def _norm_rows(exec: CudaExecutor, t: torch.Tensor, name: str):
    """Checks the first matrix of a layer norm, which has to have features; returns _matrix's."""
    found = _matrix(exec, t, name)
    if t.shape[1] == 0:
        raise ValueError(f"{name} must have at least one column")
    return found


def _norm_suffix(x: torch.Tensor, y: torch.Tensor) -> str:
    suffix = _VAL.get(x.dtype, "?") + _VAL.get(y.dtype, "?")
    if suffix not in _NORM_TYPES:
        raise ValueError(f"layer norm takes {x.dtype} to no {y.dtype}")
    return suffix


def layer_norm(exec: CudaExecutor, x: torch.Tensor, weight, bias, eps: float, y: torch.Tensor,
               mean=None, rstd=None) -> None:
    """y = (x - mean) * rstd * weight + bias over each row; x and y of one type, or x float32 and
    y 16 bits. weight and bias: float32 (cols) or None. mean, rstd: float32 (rows), written where
    given. y may be x."""
    suffix = _norm_suffix(x, y)
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and non-negative")
    px, ldx = _norm_rows(exec, x, "x")
    rows, cols = x.shape
    py, ldy = _matrix(exec, y, "y", rows, cols)
    f32 = torch.float32
    pw, pb = _dense(exec, weight, "weight", (cols,), f32), _dense(exec, bias, "bias", (cols,), f32)
    pm, pr = _dense(exec, mean, "mean", (rows,), f32), _dense(exec, rstd, "rstd", (rows,), f32)
    check(getattr(lib(), "xspmm_layer_norm_" + suffix)(
        exec.handle, rows, cols, px, ldx, pw, pb, eps, py, ldy, pm, pr))


def layer_norm_backward(exec: CudaExecutor, dy: torch.Tensor, x: torch.Tensor, weight,
                        mean: torch.Tensor, rstd: torch.Tensor, dx=None, dweight=None,
                        dbias=None) -> None:
    """Gradients of layer_norm from the forward pass's mean and rstd. dy and dx have the type of y;
    dweight and dbias are float32 (cols). Outputs that are None are not computed. dx may be dy."""
    suffix = _norm_suffix(x, dy)
    pdy, lddy = _norm_rows(exec, dy, "dy")
    rows, cols = dy.shape
    px, ldx = _matrix(exec, x, "x", rows, cols)
    pdx, lddx = (None, cols) if dx is None else _matrix(exec, dx, "dx", rows, cols, dy.dtype)
    f32 = torch.float32
    pw = _dense(exec, weight, "weight", (cols,), f32)
    pm, pr = _needed(exec, mean, "mean", (rows,), f32), _needed(exec, rstd, "rstd", (rows,), f32)
    pdw = _dense(exec, dweight, "dweight", (cols,), f32)
    pdb = _dense(exec, dbias, "dbias", (cols,), f32)
    check(getattr(lib(), "xspmm_layer_norm_backward_" + suffix)(
        exec.handle, rows, cols, pdy, lddy, px, ldx, pw, pm, pr, pdx, lddx, pdw, pdb))


def dropout(exec: CudaExecutor, x: torch.Tensor, p: float, seed: int, offset: int,
            y: torch.Tensor, residual=None) -> None:
    """y = residual + keep * x / (1 - p), elementwise over contiguous tensors of one type and shape
    (residual None: 0). The mask is a function of (seed, offset, element index) and is not stored;
    a call uses ceil(numel / 4) counters from offset on. y may be x or residual."""
    if x.dtype not in _VAL:
        raise ValueError(f"dropout takes no {x.dtype}")
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must lie in [0, 1]")
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError("seed and offset are unsigned 64-bit numbers")
    px = _dense(exec, x, "x", x.shape, x.dtype)
    py = _dense(exec, y, "y", x.shape, x.dtype)
    pr = _dense(exec, residual, "residual", x.shape, x.dtype)
    check(getattr(lib(), "xspmm_dropout_" + _VAL[x.dtype])(
        exec.handle, x.numel(), px, pr, p, seed, offset, py))


def dropout_backward(exec: CudaExecutor, dy: torch.Tensor, p: float, seed: int, offset: int,
                     dx: torch.Tensor) -> None:
    """dx = keep * dy / (1 - p) with the mask of the forward call of the same p, seed and offset
    (the residual's gradient is dy itself). dx may be dy."""
    dropout(exec, dy, p, seed, offset, dx)


def _gated(exec, x, w_gate, w_up, activation):
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"the gated feed-forward block takes 16-bit types, not {x.dtype}")
    if activation not in _ACT:
        raise ValueError(f"activation must be one of {', '.join(_ACT)}, not {activation!r}")
    px, ldx = _matrix(exec, x, "x")
    rows, K = x.shape
    pg, ldg = _matrix(exec, w_gate, "w_gate", None, K, x.dtype)
    F = w_gate.shape[0]
    pu, ldu = _matrix(exec, w_up, "w_up", F, K, x.dtype)
    return rows, K, F, (px, ldx, pg, ldg, pu, ldu)


def gated_ffn(exec: CudaExecutor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
              y: torch.Tensor, activation: str = "silu", gate=None, up=None) -> None:
    """y = act(x @ w_gate.T) * (x @ w_up.T), x (rows x K), weights (F x K), y (rows x F), all of one
    16-bit type, sums in float32. activation: silu, gelu (erf), relu or sigmoid. gate, up (rows x F,
    contiguous) receive the two projections where given: the gradient needs them."""
    rows, K, F, operands = _gated(exec, x, w_gate, w_up, activation)
    py, ldy = _matrix(exec, y, "y", rows, F, x.dtype)
    pg = _dense(exec, gate, "gate", (rows, F), x.dtype)
    pu = _dense(exec, up, "up", (rows, F), x.dtype)
    check(getattr(lib(), "xspmm_gated_ffn_" + _VAL[x.dtype])(
        exec.handle, rows, K, F, _ACT[activation], *operands, py, ldy, pg, pu))


def gated_ffn_backward(exec: CudaExecutor, dy: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor,
                       w_up: torch.Tensor, gate: torch.Tensor, up: torch.Tensor, dx=None,
                       dw_gate=None, dw_up=None, activation: str = "silu") -> None:
    """Gradients of gated_ffn from dy and the projections it kept. dx (rows x K) may be None; dw_gate
    and dw_up (F x K, contiguous) are both given or both None. All of x's type."""
    rows, K, F, operands = _gated(exec, x, w_gate, w_up, activation)
    pdy, lddy = _matrix(exec, dy, "dy", rows, F, x.dtype)
    pg = _needed(exec, gate, "gate", (rows, F), x.dtype)
    pu = _needed(exec, up, "up", (rows, F), x.dtype)
    pdx, lddx = (None, K) if dx is None else _matrix(exec, dx, "dx", rows, K, x.dtype)
    pdg = _dense(exec, dw_gate, "dw_gate", (F, K), x.dtype)
    pdu = _dense(exec, dw_up, "dw_up", (F, K), x.dtype)
    if (dw_gate is None) != (dw_up is None):
        raise ValueError("dw_gate and dw_up are given both or neither")
    check(getattr(lib(), "xspmm_gated_ffn_backward_" + _VAL[x.dtype])(
        exec.handle, rows, K, F, _ACT[activation], pdy, lddy, *operands, pg, pu, pdx, lddx, pdg,
        pdu))
