"""Low-rank adapters of many requests beside a projection that they share.

    plan = adapters.plan(ids, num_adapters)                       # once for a batch: ids[t] is token t's adapter, -1 none
    y = adapters.project(x, weight, a, b, plan, scale=scale)      # y[t] = weight x[t] + scale[i] b[i] (a[i] x[t]), i = ids[t]

It is the grouped product's gather -> map by type -> reduce with two maps an edge: the matrix that all tokens share and the product of two thin ones
that the token's request names.  Tokens stay in their order; one token or a prompt, all with one adapter or each with its own, go through the same
two launches.  The second begins while the first runs: only its stores wait for the adapters' part, which is added before y's only rounding.

Checks, streams, errors and ``experts.bind`` are those of ``experts``; results carry no gradient (an adapter is trained as ``experts.grouped_matmul``
twice, with its gradients).  Ids that are no adapter are noticed on the device and count as none; so is a bound plan that a projection reads before its
first launch: the next call of a projection on the device, or ``experts.check()``, raises.  (The reference has no operator of the kind.)
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple, Optional

import torch

from .binding import FlexSpmvError
from .experts import _HALF, _P, _TYPE, BoundCall, _check, _flag, _function, _need, _operator, _out, _rows_of, _tensor, _whole

MAX_ADAPTERS, MAX_RANK = 1024, 512           # FLEXSPMV_MAX_ADAPTERS, FLEXSPMV_MAX_RANK

_BYTES = ctypes.CFUNCTYPE(ctypes.c_int, _P, _P)
_PLAN = ctypes.CFUNCTYPE(ctypes.c_int, _P, _P, _P, ctypes.c_size_t, _P, _P)
_PROJECT = ctypes.CFUNCTYPE(ctypes.c_int, _P, _P, _P, _P, ctypes.c_size_t, _P, _P)


class Desc(ctypes.Structure):
    """flexspmv_adapter_desc (include/flexspmv.h)."""
    _fields_ = [("tokens", ctypes.c_int64), ("x_stride", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("adapters", "rank", "n", "k", "type", "reserved")]


class Plan(NamedTuple):
    """What ``plan`` returns, for all projections of a batch."""
    data: torch.Tensor
    tokens: int
    adapters: int


def _bytes(name: str, d: Desc) -> int:
    need = ctypes.c_size_t()
    _check(_function(name, _BYTES)(ctypes.addressof(d), ctypes.addressof(need)), name)
    return need.value


@functools.lru_cache(maxsize=256)
def _project_bytes(tokens: int, rank: int, kind: int) -> int:
    return _bytes("adapted_project_bytes", Desc(tokens, 8, 1, rank, 8, 8, kind))


@functools.lru_cache(maxsize=256)
def _plan_bytes(tokens: int, adapters: int) -> int:
    return _bytes("adapter_plan_bytes", Desc(tokens, 0, adapters))


@_operator
def plan(ids: torch.Tensor, num_adapters: int) -> Plan:
    """The tokens by adapter.  ``ids`` (tokens) int32, -1: a token without one.  Bound, a launch takes what ``ids`` then holds."""
    dev = _tensor(ids, "ids", (torch.int32,), 1)
    _whole(ids, "ids")
    if not (1 <= num_adapters <= MAX_ADAPTERS):
        raise FlexSpmvError(f"1 to {MAX_ADAPTERS} adapters, not {num_adapters}")
    d = Desc(ids.numel(), 0, num_adapters)
    need = _plan_bytes(d.tokens, num_adapters)
    data = torch.empty(need // 4, dtype=torch.int32, device=ids.device)
    flag = _flag(dev)
    return BoundCall(_function("adapter_plan", _PLAN), (ctypes.addressof(d), ids.data_ptr(), data.data_ptr(), need, flag.tensor.data_ptr()), dev,
                     (d, ids, data, flag), Plan(data, ids.numel(), num_adapters), flag.view)


@_operator
def project(x: torch.Tensor, weight: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: Plan, scale: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[t] = weight @ x[t] + scale[i] * b[i] @ (a[i] @ x[t])`` with the adapter ``i`` of token ``t``, or none.

    ``x`` (tokens, k), ``weight`` (n, k), ``a`` (adapters, rank, k) and ``b`` (adapters, n, rank) of one 16-bit type, ``scale`` (adapters) float32; n, k and the
    rank are multiples of 8, x's rows may be apart.  Adapters of different ranks: rows of zeros in ``a``.  What an adapter holds reaches the tokens that name
    it, and no others."""
    dev = _tensor(x, "x", _HALF, 2)
    _tensor(weight, "weight", (x.dtype,), 2, dev)
    _tensor(a, "a", (x.dtype,), 3, dev)
    _tensor(b, "b", (x.dtype,), 3, dev)
    at = [x.data_ptr(), weight.data_ptr(), a.data_ptr(), b.data_ptr(), 0, 0]
    for name, t, first in (("weight", weight, at[1]), ("a", a, at[2]), ("b", b, at[3])):
        _whole(t, name)
        if first % 16:
            raise FlexSpmvError(f"{name}: the first value must be on 16 bytes")
    (tokens, width), (n, k), (adapters, rank, k_a) = x.shape, weight.shape, a.shape
    if width != k or k_a != k:
        raise FlexSpmvError(f"x's rows and a's must have {k} values, as weight's, not {width} and {k_a}")
    if b.shape != (adapters, n, rank):
        raise FlexSpmvError(f"b must have the shape {(adapters, n, rank)}, not {tuple(b.shape)}")
    if not (n >= 8 and k >= 8 and rank >= 8 and n % 8 == 0 and k % 8 == 0 and rank % 8 == 0):
        raise FlexSpmvError(f"both sides of weight and the rank must be multiples of 8, not {n} x {k} and {rank}")
    if not (rank <= MAX_RANK and n <= 0x7fffffff and k <= 0x7fffffff):
        raise FlexSpmvError(f"a rank of at most {MAX_RANK} and sides of 31 bits, not {rank} and {n} x {k}")
    if not (isinstance(plan, Plan) and plan.data.get_device() == dev):
        raise FlexSpmvError("plan must be one of this module, on x's device")
    if plan.tokens != tokens or plan.adapters != adapters:
        raise FlexSpmvError(f"the plan is of {plan.tokens} tokens and {plan.adapters} adapters, not of {tokens} and {adapters}")
    if scale is not None:
        _tensor(scale, "scale", (torch.float32,), 1, dev)
        _whole(scale, "scale")
        _need(scale.numel() == adapters, "scale must have a value for each adapter")
        at[4] = scale.data_ptr()
    at[5] = plan.data.data_ptr()
    stride = _rows_of(x, "x")
    if out is None:
        out = x.new_empty((tokens, n))
    else:
        out = _out(out, (tokens, n), x.dtype, x.device, x=x, weight=weight, a=a, b=b, scale=scale, plan=plan.data)
    d = Desc(tokens, stride, adapters, rank, n, k, _TYPE[x.dtype])
    need = _project_bytes(tokens, rank, d.type)
    ws = x.new_empty(need, dtype=torch.uint8)
    ins = (_P * 6)(*at)
    outs = (_P * 1)(out.data_ptr())
    flag = _flag(dev)
    return BoundCall(_function("adapted_project", _PROJECT),
                     (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs), ws.data_ptr(), need, flag.tensor.data_ptr()), dev,
                     (d, ins, outs, x, weight, a, b, scale, plan, out, ws, flag), out, flag.view)
