"""The operators of the layer around the sparse product, over the C ABI: layer norm, group norm with an
activation, dropout and the gated feed-forward block, each with its gradient; rows in 8-bit integers and
their product, for serving; the orthogonalised update of a weight matrix, for training.

Rows are nodes or tokens and features are contiguous, as in B and C of `spmm`. Matrices are 2-D
device tensors whose last dimension has stride 1; their row stride is free (a slice of columns of
a wider tensor is taken as it is), except where a function says contiguous. Outputs are the
caller's tensors and are overwritten. Work is enqueued on torch's current stream; nothing
synchronizes. Wrong shapes, types, strides, devices or values and missing inputs raise ValueError
before anything runs.
"""
from __future__ import annotations

import torch

from ._lib import check, lib
from .api import _VAL, CudaExecutor

_ACT = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
_GROUP_ACT = {None: -1, **_ACT}
_MAX_GROUP, _MAX_INT8_K = 16384, 131071
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


def _check_eps(eps):
    """eps is passed on in float32."""
    if not 0.0 <= eps <= torch.finfo(torch.float32).max:
        raise ValueError("eps must be finite and non-negative")


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
    _check_eps(eps)
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


def _group_norm(exec, x, y, y_name, groups, weight, bias, offsets, activation):
    """Checks what group_norm and its gradient have in common; returns the C arguments before and
    after x's address and stride, and the shape of the statistics."""
    suffix = _VAL.get(x.dtype, "?") + _VAL.get(y.dtype, "?")
    if suffix not in _NORM_TYPES:
        raise ValueError(f"group norm takes {x.dtype} to no {y.dtype}")
    if activation not in _GROUP_ACT:
        raise ValueError(f"activation must be None or one of {', '.join(_ACT)}, not {activation!r}")
    found = _norm_rows(exec, x, "x")
    rows, cols = x.shape
    if not (isinstance(groups, int) and groups >= 1 and cols % groups == 0):
        raise ValueError(f"groups must be a whole number that divides {cols}, not {groups!r}")
    if cols // groups > _MAX_GROUP:
        raise ValueError(f"a group has at most {_MAX_GROUP} channels, not {cols // groups}")
    samples = 1
    if offsets is not None:
        if offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("offsets must hold one more value than there are samples")
        samples = offsets.numel() - 1
    po = _dense(exec, offsets, "offsets", (samples + 1,), torch.int64)
    out = _matrix(exec, y, y_name, rows, cols)
    pw = _dense(exec, weight, "weight", (cols,), torch.float32)
    pb = _dense(exec, bias, "bias", (cols,), torch.float32)
    return suffix, (rows, cols, groups, samples, po), found, out, (pw, pb), (samples, groups)


def group_norm(exec: CudaExecutor, x: torch.Tensor, groups: int, weight, bias, eps: float,
               y: torch.Tensor, offsets=None, activation=None, mean=None, rstd=None) -> None:
    """y = act((x - mean) * rstd * weight + bias) with the statistics of each sample's rows and each of
    `groups` groups of neighbouring channels. offsets (int64, samples + 1): sample i is rows
    [offsets[i], offsets[i + 1]); rows outside all of them are left as they were in y, and a sample may be
    empty. None: all rows are one sample. activation: None, silu, gelu (erf), relu or sigmoid. x and y of
    one type, or x float32 and y 16 bits. weight and bias: float32 (cols) or None. mean, rstd: float32
    (samples, groups), written where given. y may be x. The offsets' values are not checked: see the C
    header for what those out of order mean."""
    suffix, sizes, (px, ldx), (py, ldy), wb, shape = _group_norm(
        exec, x, y, "y", groups, weight, bias, offsets, activation)
    _check_eps(eps)
    pm = _dense(exec, mean, "mean", shape, torch.float32)
    pr = _dense(exec, rstd, "rstd", shape, torch.float32)
    check(getattr(lib(), "xspmm_group_norm_" + suffix)(
        exec.handle, *sizes, px, ldx, *wb, eps, _GROUP_ACT[activation], py, ldy, pm, pr))


def group_norm_backward(exec: CudaExecutor, dy: torch.Tensor, x: torch.Tensor, groups: int, weight,
                        bias, mean: torch.Tensor, rstd: torch.Tensor, dx=None, dweight=None,
                        dbias=None, offsets=None, activation=None) -> None:
    """Gradients of group_norm from the forward pass's mean and rstd, with its weight, bias, offsets and
    activation. dy and dx have the type of y; dweight and dbias are float32 (cols). Outputs that are None
    are not computed. dx may be dy."""
    suffix, sizes, (px, ldx), (pdy, lddy), wb, shape = _group_norm(
        exec, x, dy, "dy", groups, weight, bias, offsets, activation)
    rows, cols = x.shape
    pdx, lddx = (None, cols) if dx is None else _matrix(exec, dx, "dx", rows, cols, dy.dtype)
    f32 = torch.float32
    pm, pr = _needed(exec, mean, "mean", shape, f32), _needed(exec, rstd, "rstd", shape, f32)
    pdw = _dense(exec, dweight, "dweight", (cols,), f32)
    pdb = _dense(exec, dbias, "dbias", (cols,), f32)
    check(getattr(lib(), "xspmm_group_norm_backward_" + suffix)(
        exec.handle, *sizes, pdy, lddy, px, ldx, *wb, pm, pr, _GROUP_ACT[activation], pdx, lddx, pdw,
        pdb))


def quantize_rows(exec: CudaExecutor, x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor) -> None:
    """Rows of x in 8-bit integers: scale = max|x| / 127 of each row (float32), q = 127 x / max|x| rounded to
    the nearest (int8, of x's shape). A row of zeros has scale 0, one with an infinity or NaN scale NaN."""
    if x.dtype not in _VAL:
        raise ValueError(f"quantize_rows takes no {x.dtype}")
    px, ldx = _matrix(exec, x, "x")
    rows, cols = x.shape
    pq, ldq = _matrix(exec, q, "q", rows, cols, torch.int8)
    ps = _needed(exec, scale, "scale", (rows,), torch.float32)
    check(getattr(lib(), "xspmm_quantize_rows_" + _VAL[x.dtype])(
        exec.handle, rows, cols, px, ldx, pq, ldq, ps))


def linear_int8(exec: CudaExecutor, x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor,
                w_scale: torch.Tensor, y: torch.Tensor, bias=None) -> None:
    """y = (x @ w.T) * x_scale[:, None] * w_scale + bias: x (rows x K) and w (F x K) int8, as
    quantize_rows makes them of activations and of a weight; the sum is exact. Operands whose rows start on
    16 bytes (the first row and the stride) are read in place, others of more than 16 rows of x are copied
    in every call: a weight with K no multiple of 16 is best kept as a slice of padded rows. y (rows x F)
    float16, bfloat16 or float32; x_scale (rows), w_scale (F) and bias (F, or None) float32."""
    if y.dtype not in _VAL:
        raise ValueError(f"linear_int8 gives no {y.dtype}")
    px, ldx = _matrix(exec, x, "x", None, None, torch.int8)
    rows, K = x.shape
    if K > _MAX_INT8_K:
        raise ValueError(f"x has at most {_MAX_INT8_K} columns, not {K}")
    pw, ldw = _matrix(exec, w, "w", None, K, torch.int8)
    F = w.shape[0]
    f32 = torch.float32
    pxs = _needed(exec, x_scale, "x_scale", (rows,), f32)
    pws = _needed(exec, w_scale, "w_scale", (F,), f32)
    pb = _dense(exec, bias, "bias", (F,), f32)
    py, ldy = _matrix(exec, y, "y", rows, F)
    check(getattr(lib(), "xspmm_linear_int8_" + _VAL[y.dtype])(
        exec.handle, rows, K, F, px, ldx, pxs, pw, ldw, pws, pb, py, ldy))


def orthogonalize(exec: CudaExecutor, g: torch.Tensor, y: torch.Tensor, steps: int = 5,
                  eps: float = 1e-7) -> None:
    """The update of a weight matrix from its gradient or momentum g with every singular value driven to
    about 1, by Newton-Schulz steps X <- a X + (b A + c A A) X, A = X X^T, from X = g / (|g| + eps),
    (a, b, c) = (3.4445, -4.7750, 2.0315). g float16, bfloat16 or float32; y float16 or bfloat16, g's
    type where that is 16 bits. y may be g."""
    suffix = _VAL.get(g.dtype, "?") + _VAL.get(y.dtype, "?")
    if suffix not in ("f16f16", "bf16bf16", "f32f16", "f32bf16"):
        raise ValueError(f"orthogonalize takes {g.dtype} to no {y.dtype}")
    if not (isinstance(steps, int) and 0 <= steps <= 100):
        raise ValueError("steps must be a whole number in [0, 100]")
    _check_eps(eps)
    pg, ldg = _matrix(exec, g, "g")
    rows, cols = g.shape
    py, ldy = _matrix(exec, y, "y", rows, cols)
    check(getattr(lib(), "xspmm_orthogonalize_" + suffix)(
        exec.handle, rows, cols, pg, ldg, steps, eps, py, ldy))
