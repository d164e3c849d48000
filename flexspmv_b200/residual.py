"""Operators of a residual stream around a routed expert layer: layer norm with the sum and the dropout in front of it, and dropout.

    n = layer_norm(z, weight, bias, residual=x, p=0.1, seed=seed)        # n.sum = x + dropout(z), n.y = its rows normalised
    g = layer_norm_backward(dy, n.sum, weight, n.mean, n.rstd, dsum=dsum, p=0.1, seed=seed)
    out = dropout(z, 0.1, seed, residual=x)                              # the backward pass is dropout(dout, 0.1, seed)

``seed`` is an int64 CUDA tensor of two values, a seed and an offset, read by the kernels when they run: the loop that uses them raises the offset
(``seed[1] += 1``, in a captured graph too) and every call with the same two values drops the same places, whatever the type, the strides or the
launch.  Nothing of the mask is stored.  The generator is Philox4x32-10, the rule is in ``include/flexspmv.h``.

Rows are float32, bfloat16 or float16 of any width, their values contiguous; statistics and sums are in 32 bits, results rounded once.  Checks,
streams, errors and ``experts.bind`` are those of ``experts``.  (The reference has no operator of the kind: its reduces are sums over a row's edges,
include/merged_spmv.cuh:149-182.)
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch

from .binding import FlexSpmvError, _pointers
from .experts import _BYTES, _PLAIN, _TYPE, _WITH_WORKSPACE, BoundCall, _check, _function, _operator, _out, _rows_of, _tensor, _whole

MAX_WIDTH = 1 << 24                          # FLEXSPMV_MAX_WIDTH


class Desc(ctypes.Structure):
    """flexspmv_rows_desc (include/flexspmv.h)."""
    _fields_ = [("rows", ctypes.c_int64), ("width", ctypes.c_int64), ("stride", ctypes.c_int64 * 3), ("type", ctypes.c_int32), ("param_type", ctypes.c_int32),
                ("eps", ctypes.c_float), ("reserved", ctypes.c_int32), ("p", ctypes.c_double)]


class Normed(NamedTuple):
    y: torch.Tensor
    sum: Optional[torch.Tensor]              # what was normalised, rounded to its type; None: x itself
    mean: torch.Tensor                       # (rows) float32
    rstd: torch.Tensor


class NormGradients(NamedTuple):
    dx: torch.Tensor                         # of what went through the dropout; without one, dresidual itself
    dresidual: torch.Tensor                  # of the sum
    dweight: Optional[torch.Tensor]
    dbias: Optional[torch.Tensor]


_ANY, _WIDE, _SEED = tuple(_TYPE), {t: (torch.float32, t) for t in _TYPE}, (torch.int64,)


def _stride(t, name: str, rows: int, width: int) -> int:
    """Row stride of a checked matrix, whose rows must be contiguous."""
    if t.is_contiguous():
        return width
    return _rows_of(t, name, aligned=False)


def _first(x, name: str):
    """Checks the matrix that says the type, shape and device of a call's others; returns device, rows, width and row stride."""
    dev = _tensor(x, name, _ANY, 2)
    rows, width = x.shape
    if not 1 <= width <= MAX_WIDTH:
        raise FlexSpmvError(f"{name} must have 1 to {MAX_WIDTH} columns, not {width}")
    return dev, rows, width, _stride(x, name, rows, width)


def _matrix(t, name: str, like, dev: int, rows: int, width: int) -> int:
    """Checks another matrix of the call; returns its row stride.  None: 0."""
    if t is None:
        return 0
    _tensor(t, name, (like.dtype,), 2, dev)
    if t.shape != like.shape:
        raise FlexSpmvError(f"{name} must have the shape {tuple(like.shape)}, not {tuple(t.shape)}")
    return _stride(t, name, rows, width)


def _vector(t, name: str, dtypes, n: int, dev: int, of: str):
    _tensor(t, name, dtypes, 1, dev)
    if t.shape[0] != n:
        raise FlexSpmvError(f"{name} must have {n} values, one for each {of}, not {t.shape[0]}")
    _whole(t, name)


def _params(weight, bias, x, width: int, dev: int) -> int:
    """Checks weight and bias; returns their type."""
    kinds = _WIDE[x.dtype]
    if weight is not None:
        _vector(weight, "weight", kinds, width, dev, "column")
        kinds = (weight.dtype,)
    if bias is not None:
        _vector(bias, "bias", kinds, width, dev, "column")
        kinds = (bias.dtype,)
    return _TYPE[kinds[0]]


def _drops(p, seed, dev: int) -> float:
    p = float(p)
    if not 0.0 <= p < 1.0:
        raise FlexSpmvError(f"p must be at least 0 and below 1, not {p}")
    if p > 0.0:
        if seed is None:
            raise FlexSpmvError("p > 0 takes a seed")
        _vector(seed, "seed", _SEED, 2, dev, "of seed and offset")
    return p


def _at(*tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() if t is not None else 0 for t in tensors])


@_operator
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None, p: float = 0.0, seed: Optional[torch.Tensor] = None) -> Normed:
    """``y = (s - mean) * rstd * weight + bias`` over the rows of ``s = residual + dropout(x)``, with ``rstd = 1 / sqrt(variance + eps)``.

    ``x`` and ``residual`` (rows, width) of one type; ``weight`` and ``bias`` (width) of that type or float32.  ``s`` is normalised before it is
    rounded; it is returned, rounded, where it is not ``x`` itself."""
    dev, rows, width, xs = _first(x, "x")
    rs = _matrix(residual, "residual", x, dev, rows, width)
    kind, p, eps = _params(weight, bias, x, width, dev), _drops(p, seed, dev), float(eps)
    if not eps >= 0.0:
        raise FlexSpmvError(f"eps must not be negative or NaN: {eps}")
    y = x.new_empty((rows, width))
    total = torch.empty_like(y) if residual is not None or p > 0.0 else None
    mean = x.new_empty(rows, dtype=torch.float32)
    out = Normed(y, total, mean, torch.empty_like(mean))
    d = Desc(rows, width, (xs, rs, 0), _TYPE[x.dtype], kind, eps, 0, p)
    ins, outs = _at(x, residual, weight, bias, seed if p > 0.0 else None), _at(y, total, out.mean, out.rstd)
    return BoundCall(_function("layer_norm", _PLAIN), (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs)), dev,
                     (d, ins, outs, x, residual, weight, bias, seed, out), out)


@functools.lru_cache(maxsize=256)
def _backward_bytes(rows: int, width: int, device: int) -> int:
    need = ctypes.c_size_t()
    d = Desc(rows, width)
    with torch.cuda.device(device):
        _check(_function("layer_norm_backward_bytes", _BYTES)(ctypes.addressof(d), ctypes.addressof(need)), "layer_norm_backward")
    return need.value


@_operator
def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor, rstd: torch.Tensor,
                        dsum: Optional[torch.Tensor] = None, p: float = 0.0, seed: Optional[torch.Tensor] = None,
                        bias: Optional[torch.Tensor] = None) -> NormGradients:
    """Gradients of ``layer_norm``.  ``x`` is what was normalised (``Normed.sum`` where there is one), ``dsum`` a gradient that reaches it directly;
    ``dx`` is what passes the dropout of ``p`` and ``seed``.  ``dweight`` and ``dbias`` are of the weight's type; without a weight there is ``dbias`` alone, of
    the type of ``bias`` (whose values are not read), or none."""
    dev, rows, width, ys = _first(dy, "dy")
    if x is None:
        raise FlexSpmvError("x is what was normalised")
    xs, ds = _matrix(x, "x", dy, dev, rows, width), _matrix(dsum, "dsum", dy, dev, rows, width)
    kind, p = _params(weight, bias, dy, width, dev), _drops(p, seed, dev)
    _vector(mean, "mean", (torch.float32,), rows, dev, "row")
    _vector(rstd, "rstd", (torch.float32,), rows, dev, "row")
    dresidual = dy.new_empty((rows, width))
    dx = torch.empty_like(dresidual) if p > 0.0 else dresidual
    dweight = dbias = ws = None
    need = 0
    of = weight if weight is not None else bias
    if of is not None:
        dweight, dbias = torch.empty_like(of), torch.empty_like(of)
        need = _backward_bytes(rows, width, dev)
        ws = dy.new_empty(need, dtype=torch.uint8)
    out = NormGradients(dx, dresidual, dweight if weight is not None else None, dbias)
    d = Desc(rows, width, (ys, xs, ds), _TYPE[dy.dtype], kind, 0.0, 0, p)
    ins, outs = _at(dy, x, weight, mean, rstd, dsum, seed if p > 0.0 else None), _at(dx if p > 0.0 else None, dresidual, dweight, dbias)
    return BoundCall(_function("layer_norm_backward", _WITH_WORKSPACE),
                     (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs), ws.data_ptr() if ws is not None else None, need), dev,
                     (d, ins, outs, dy, x, weight, mean, rstd, dsum, seed, ws, dweight, out), out)


@_operator
def dropout(x: torch.Tensor, p: float, seed: torch.Tensor, residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + x * keep / (1 - p)`` (no residual: 0), where ``keep`` is 1 with the probability ``1 - p``.  Its gradient with respect to ``x`` is
    ``dropout(dout, p, seed)``."""
    dev, rows, width, xs = _first(x, "x")
    rs = _matrix(residual, "residual", x, dev, rows, width)
    p = _drops(p, seed, dev)
    if p == 0.0:
        _drops(0.5, seed, dev)               # the seed is not used, but is one
    if out is None:
        out = x.new_empty((rows, width))
    else:
        out = _out(out, (rows, width), x.dtype, x.device, x=x, residual=residual, seed=seed)
    d = Desc(rows, width, (xs, rs, 0), _TYPE[x.dtype], 0, 0.0, 0, p)
    ins, outs = _at(x, residual, seed), _pointers((out,))
    return BoundCall(_function("dropout", _PLAIN), (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs)), dev,
                     (d, ins, outs, x, residual, seed, out), out)
