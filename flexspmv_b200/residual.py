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
from .experts import _BYTES, _PLAIN, _TYPE, _WITH_WORKSPACE, BoundCall, _check, _function, _need, _operator, _out, _rows_of, _tensor, _whole

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


def _matrix(t, name: str, like=None) -> int:
    """Checks a matrix argument, of the type, shape and device of ``like``; returns its row stride."""
    _tensor(t, name, tuple(_TYPE) if like is None else (like.dtype,), 2, None if like is None else like.get_device())
    if like is not None and t.shape != like.shape:
        raise FlexSpmvError(f"{name} must have the shape {tuple(like.shape)}, not {tuple(t.shape)}")
    _need(1 <= t.shape[1] <= MAX_WIDTH, f"{name} must have 1 to {MAX_WIDTH} columns")
    return _rows_of(t, name, aligned=False)


def _params(weight, bias, x) -> int:
    """Checks weight and bias; returns their type."""
    kind = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _tensor(t, name, (torch.float32, x.dtype) if kind is None else (kind,), 1, x.get_device())
            _whole(t, name)
            _need(t.shape[0] == x.shape[1], f"{name} must have a value for each column")
            kind = t.dtype
    return _TYPE[kind or torch.float32]


def _drops(p, seed, x) -> float:
    p = float(p)
    _need(0.0 <= p < 1.0, f"p must be at least 0 and below 1, not {p}")
    if p > 0.0:
        _need(seed is not None, "p > 0 takes a seed")
        _tensor(seed, "seed", (torch.int64,), 1, x.get_device())
        _whole(seed, "seed")
        _need(seed.shape[0] == 2, "seed must have two values, a seed and an offset")
    return p


def _at(*tensors):
    return (ctypes.c_void_p * len(tensors))(*[t.data_ptr() if t is not None else 0 for t in tensors])


@_operator
def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None, p: float = 0.0, seed: Optional[torch.Tensor] = None) -> Normed:
    """``y = (s - mean) * rstd * weight + bias`` over the rows of ``s = residual + dropout(x)``, with ``rstd = 1 / sqrt(variance + eps)``.

    ``x`` and ``residual`` (rows, width) of one type; ``weight`` and ``bias`` (width) of that type or float32.  ``s`` is normalised before it is
    rounded; it is returned, rounded, where it is not ``x`` itself."""
    dev = _tensor(x, "x", tuple(_TYPE), 2)
    xs = _matrix(x, "x")
    rs = _matrix(residual, "residual", x) if residual is not None else 0
    kind, p = _params(weight, bias, x), _drops(p, seed, x)
    eps = float(eps)
    _need(eps >= 0.0, f"eps must not be negative or NaN: {eps}")
    rows, width = x.shape
    y = torch.empty((rows, width), dtype=x.dtype, device=x.device)
    total = torch.empty_like(y) if residual is not None or p > 0.0 else None
    stats = torch.empty((2, rows), dtype=torch.float32, device=x.device)
    out = Normed(y, total, stats[0], stats[1])
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
                        dsum: Optional[torch.Tensor] = None, p: float = 0.0, seed: Optional[torch.Tensor] = None) -> NormGradients:
    """Gradients of ``layer_norm``.  ``x`` is what was normalised (``Normed.sum`` where there is one), ``dsum`` a gradient that reaches it directly;
    ``dx`` is what passes the dropout of ``p`` and ``seed``.  ``dweight`` and ``dbias`` are of the weight's type; without a weight there are none."""
    dev = _tensor(dy, "dy", tuple(_TYPE), 2)
    ys, xs = _matrix(dy, "dy"), _matrix(x, "x", dy)
    ds = _matrix(dsum, "dsum", dy) if dsum is not None else 0
    kind, p = _params(weight, None, dy), _drops(p, seed, dy)
    rows, width = dy.shape
    for name, t in (("mean", mean), ("rstd", rstd)):
        _tensor(t, name, (torch.float32,), 1, dev)
        _whole(t, name)
        _need(t.shape[0] == rows, f"{name} must have a value for each row")
    dresidual = torch.empty((rows, width), dtype=dy.dtype, device=dy.device)
    dx = torch.empty_like(dresidual) if p > 0.0 else dresidual
    dweight = dbias = ws = None
    need = 0
    if weight is not None:
        dweight, dbias = torch.empty_like(weight), torch.empty_like(weight)
        need = _backward_bytes(rows, width, dev)
        ws = torch.empty(need, dtype=torch.uint8, device=dy.device)
    out = NormGradients(dx, dresidual, dweight, dbias)
    d = Desc(rows, width, (ys, xs, ds), _TYPE[dy.dtype], kind, 0.0, 0, p)
    ins, outs = _at(dy, x, weight, mean, rstd, dsum, seed if p > 0.0 else None), _at(dx if p > 0.0 else None, dresidual, dweight, dbias)
    return BoundCall(_function("layer_norm_backward", _WITH_WORKSPACE),
                     (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs), ws.data_ptr() if ws is not None else None, need), dev,
                     (d, ins, outs, dy, x, weight, mean, rstd, dsum, seed, ws, out), out)


@_operator
def dropout(x: torch.Tensor, p: float, seed: torch.Tensor, residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``residual + x * keep / (1 - p)`` (no residual: 0), where ``keep`` is 1 with the probability ``1 - p``.  Its gradient with respect to ``x`` is
    ``dropout(dout, p, seed)``."""
    dev = _tensor(x, "x", tuple(_TYPE), 2)
    xs = _matrix(x, "x")
    rs = _matrix(residual, "residual", x) if residual is not None else 0
    _need(seed is not None, "dropout takes a seed")
    p = _drops(p, seed, x)
    if p == 0.0:
        _drops(0.5, seed, x)                 # the seed is not used, but is one
    out = _out(out, tuple(x.shape), x.dtype, x.device, x=x, residual=residual, seed=seed)
    d = Desc(x.shape[0], x.shape[1], (xs, rs, 0), _TYPE[x.dtype], 0, 0.0, 0, p)
    ins, outs = _at(x, residual, seed), _pointers((out,))
    return BoundCall(_function("dropout", _PLAIN), (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs)), dev,
                     (d, ins, outs, x, residual, seed, out), out)
