"""Operators of a routed expert layer: ``y[t] = sum_j w[t, j] * W[e[t, j]] x[t]``.

It is this library's gather -> per-edge map -> segmented reduce with (token, choice) pairs as the edges, the expert that a router chose
as an edge's type, and that expert's matrix as the map.  (The reference has no operator of the kind: its maps work on records of a few
values, data_struct_shared.cuh:80-659.)

    plan = route(logits, k)                                     # weights, experts, and the plan: offsets, rows, slots
    h = grouped_matmul(x, w1, plan.offsets, rows=plan.rows)     # h[i] = w1[e] x[rows[i]], places in expert order
    z = grouped_matmul(act(h), w2, plan.offsets)
    y = combine(z, plan.slots, plan.weights)                    # y[t] = sum_j weights[t, j] z[slots[t, j]]

with the gradients ``route_backward``, ``grouped_matmul_dx``, ``grouped_matmul_dw`` and ``combine_backward``, ``balance_loss`` with its gradient,
which keeps a router from using few of its experts, and ``grad_norm`` and ``clip_grad_norm`` over the many tensors that such a layer's training has.  ``expert_layer.RoutedExperts`` runs them together.

Results carry no gradient: while gradients are recorded, tensors that require one are refused (``expert_layer`` has the functions that do carry
them); only the norm of the last two, as usual, is a plain number.

The operators take CUDA tensors, enqueue on torch's current stream of the tensors' device and never synchronise; the plan stays on the
device.  Arguments that do not fit, an ``out`` that shares memory with an input among them, raise ``FlexSpmvError``; there is no CPU path.  ``bind(op, *args)`` checks and allocates once and returns
an object whose ``launch()`` is one foreign call on the same tensors, as ``GraphExtension.prepare`` does for graphs: for loops over fixed
buffers and for capture in a CUDA graph.  Index arrays that do not fit their arrays (offsets that descend, rows out of range) are
noticed on the device, where nothing is read or written out of range: the next call of a grouped product on the device, or ``check()``, raises.
"""
from __future__ import annotations

import array
import ctypes
import functools
import operator
from typing import Dict, NamedTuple, Optional, Sequence

import torch

from .binding import FlexSpmvError, _current_device, _pointers, _raw_stream, check as _check_status, load_library

MAX_EXPERTS, MAX_CHOICES = 1024, 32          # FLEXSPMV_MAX_EXPERTS, FLEXSPMV_MAX_CHOICES
_TYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HALF = (torch.bfloat16, torch.float16)
_RENORMALIZE = 1


class Desc(ctypes.Structure):
    """flexspmv_expert_desc (include/flexspmv.h)."""
    _fields_ = [("tokens", ctypes.c_int64), ("slots", ctypes.c_int64)] + \
               [(n, ctypes.c_int32) for n in ("experts", "choices", "n", "k", "type", "out_type", "flags", "reserved")] + \
               [("in_stride", ctypes.c_int64), ("in2_stride", ctypes.c_int64)]


class Plan(NamedTuple):
    """What ``route`` returns.  A *place* is a pair's position in the order by expert, then token."""
    weights: torch.Tensor        # (tokens, k) float32, largest first; 0 where there is no expert
    experts: torch.Tensor        # (tokens, k) int32, -1: none
    offsets: torch.Tensor        # (experts + 1) int32: places offsets[e] .. offsets[e + 1] are expert e's
    rows: torch.Tensor           # (tokens * k) int32: the token of a place, -1 from offsets[-1] on
    slots: torch.Tensor          # (tokens, k) int32: a pair's place, -1: none
    renormalize: bool


class BoundCall:
    """One operator bound to its tensors: ``launch()`` enqueues it on the current stream of their device and returns the outputs, the
    same tensors every time.  Launches of one object must be ordered with one another: they share outputs and workspace.  It holds its
    tensors; like them it must outlive what it has enqueued on streams other than theirs."""
    __slots__ = ("_fn", "_args", "_device", "_keep", "_flag", "outputs")

    def __init__(self, fn, args, device, keep, outputs, flag=None):
        self._fn, self._args, self._device, self._keep, self.outputs, self._flag = fn, args, device, keep, outputs, flag

    def launch(self):
        if self._flag is not None and self._flag[0]:
            _raise_flag(self._device)
        if _current_device() != self._device:
            with torch.cuda.device(self._device):
                st = self._fn(*self._args, _raw_stream(self._device))
        else:
            st = self._fn(*self._args, _raw_stream(self._device))
        if st != 0:
            _check(st, "launch")
        return self.outputs

    __call__ = launch


class PlannedCall(BoundCall):
    """A bound call whose workspace was planned on the stream that was current when it was bound; a first launch on another one waits for that."""
    __slots__ = ("_planned", "_ordered")

    def __init__(self, *args):
        super().__init__(*args)
        self._planned, self._ordered = None, None

    def bound(self):
        self._planned = torch.cuda.Event()
        stream = torch.cuda.current_stream(self._device)
        self._planned.record(stream)
        self._ordered = {stream.cuda_stream}

    def launch(self):
        if self._ordered is not None:
            stream = _raw_stream(self._device)
            if stream not in self._ordered:
                if torch.cuda.is_current_stream_capturing():
                    raise FlexSpmvError("first launch of a bound call on a stream that is being captured: launch it once on that stream before the "
                                        "capture begins")
                torch.cuda.current_stream(self._device).wait_event(self._planned)
                self._ordered.add(stream)
        return super().launch()

    __call__ = launch


_P, _I, _N = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
_WITH_WORKSPACE = ctypes.CFUNCTYPE(_I, _P, _P, _P, _P, _N, _P)
_GROUPED, _GROUPED_DW = ctypes.CFUNCTYPE(_I, _P, _P, _P, _P, _P), ctypes.CFUNCTYPE(_I, _P, _P, _P, _P, _N, _P, _P)
_PLAIN = ctypes.CFUNCTYPE(_I, _P, _P, _P, _P)
_CLIP = ctypes.CFUNCTYPE(_I, ctypes.c_int32, ctypes.c_int32, ctypes.c_float, _P, _P, _N, _P)
_CLIP_BYTES = ctypes.CFUNCTYPE(_I, ctypes.c_int32, _P, _P, _P)
_CLIP_PLAN = ctypes.CFUNCTYPE(_I, ctypes.c_int32, _P, _P, _P, _P, _P, _P, _N, _P)
_BYTES = ctypes.CFUNCTYPE(_I, _P, _P)
_FIVE = _P * 5
_functions: Dict[str, object] = {}


def _function(name: str, proto):
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = proto((f"flexspmv_{name}", load_library()))
    return f


def _check(status: int, what: str):
    if status != 0:
        _check_status(load_library(), status, what)


class _Flag:
    __slots__ = ("tensor", "view")

    def __init__(self):
        self.tensor = torch.zeros(1, dtype=torch.int32).pin_memory()
        self.view = self.tensor.numpy()


_flags: Dict[int, _Flag] = {}


def _flag(device: int) -> _Flag:
    """The page-locked int in which the kernels of a device leave an error."""
    if device not in _flags:
        _flags[device] = _Flag()
    return _flags[device]


def _raise_flag(device: int):
    st = int(_flag(device).view[0])
    _flag(device).view[0] = 0
    text = "offsets, rows or ids that do not fit their arrays" if st == -5 else load_library().flexspmv_error_string(st).decode()
    raise FlexSpmvError(f"an earlier grouped product on cuda:{device} failed: {text} (status {st}); its outputs are undefined", st)


def check(device=None) -> None:
    """Waits for the device and raises where a grouped product on it has found an error."""
    index = torch.device(device).index if device is not None else None
    index = _current_device() if index is None else index
    torch.cuda.synchronize(index)
    if index in _flags and _flags[index].view[0]:
        _raise_flag(index)


def _need(ok: bool, what: str):
    if not ok:
        raise FlexSpmvError(what)


def _tensor(t, name: str, dtypes, dim: int, device=None) -> int:
    """Checks a tensor argument; returns its device's index."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise FlexSpmvError(f"{name} must be a CUDA tensor")
    if t.dtype not in dtypes or t.dim() != dim:
        raise FlexSpmvError(f"{name} must have {dim} dimension(s) and one of the types {', '.join(str(d) for d in dtypes)}, "
                            f"not {tuple(t.shape)} {t.dtype}")
    if device is not None and t.get_device() != device:
        raise FlexSpmvError(f"{name} is on cuda:{t.device.index}, not cuda:{device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise FlexSpmvError(f"{name} requires a gradient, which the result would not carry: call expert_layer's functions, or this one under torch.no_grad() "
                            "or on detached tensors")
    return t.get_device()


def _rows_of(t: torch.Tensor, name: str, aligned: bool = True) -> int:
    """Row stride of a matrix whose rows are contiguous."""
    n, stride = t.shape[1], t.stride(0) if t.shape[0] > 1 else t.shape[1]
    if not ((n <= 1 or t.stride(1) == 1) and stride >= n):
        raise FlexSpmvError(f"{name}: rows must be contiguous and must not overlap")
    if aligned:
        if not (n % 8 == 0 and stride % 8 == 0 and t.data_ptr() % 16 == 0):
            raise FlexSpmvError(f"{name}: rows must be multiples of 8 values, apart by multiples of 8, the first on 16 bytes")
    return stride


def _whole(t: torch.Tensor, name: str):
    if not t.is_contiguous():
        raise FlexSpmvError(f"{name} must be contiguous")


def _meets(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether the contiguous ``out`` shares memory with ``t``, whose rows are contiguous; between the rows it may lie."""
    if out.numel() == 0 or t.numel() == 0:
        return False
    size, at = t.element_size(), out.data_ptr() - t.data_ptr()
    rows, row, stride = (1, t.numel() * size, 1) if t.is_contiguous() else (t.shape[0], t.shape[1] * size, t.stride(0) * size)
    first = 0 if at < row else (at - row) // stride + 1
    return first < rows and first * stride < at + out.numel() * out.element_size()


def _out(out, shape, dtype, device, **inputs):
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    _tensor(out, "out", (dtype,), len(shape), device.index)
    if not (tuple(out.shape) == tuple(shape)):
        raise FlexSpmvError(f"out must have the shape {tuple(shape)}, not {tuple(out.shape)}")
    _whole(out, "out")
    end = out.data_ptr() + out.nbytes
    for name, t in inputs.items():
        if t is not None and t.data_ptr() < end and _meets(out, t):
            raise FlexSpmvError(f"out and {name} share memory")
    return out


# ---- the operators -----------------------------------------------------------------------------------------------

_BINDERS = {}


def _operator(binder):
    """The public function of a binder: the call bound and launched once."""
    def op(*args, **kwargs):
        return binder(*args, **kwargs).launch()
    op.__name__, op.__doc__, op.__wrapped__ = binder.__name__, binder.__doc__, binder
    op.__qualname__ = binder.__name__
    op.__module__ = binder.__module__
    _BINDERS[op] = binder
    return op


def bind(op, *args, **kwargs) -> BoundCall:
    """Checks the arguments of an operator of this module (or of ``residual``, ``adapters``) and allocates its outputs and workspace once; the
    ``BoundCall``'s ``launch()`` runs it on them as often as wanted."""
    _need(op in _BINDERS, "bind takes an operator of this module, of residual or of adapters")
    # the plan would run with the graph's replays only, and a launch before the first would take whatever the workspace holds for one
    if op in (grad_norm, clip_grad_norm) and torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
        raise FlexSpmvError(f"{op.__name__} is bound while a stream is captured: bind it before, or call it unbound")
    call = _BINDERS[op](*args, **kwargs)
    if isinstance(call, PlannedCall):
        call.bound()
    return call


@functools.lru_cache(maxsize=256)
def _route_bytes(tokens: int, experts: int) -> int:
    need = ctypes.c_size_t()
    d = Desc(tokens, 0, experts)
    _check(_function("expert_route_bytes", _BYTES)(ctypes.addressof(d), ctypes.addressof(need)), "route")
    return need.value


@_operator
def route(logits: torch.Tensor, k: int, renormalize: bool = False) -> Plan:
    """Softmax over each row of ``logits`` (tokens, experts; float32, bfloat16 or float16), its k largest values and the plan.

    Equal logits: the lowest expert first.  A logit of -infinity forbids an expert; a row with fewer than k others has experts of -1 and
    weights of 0 for the rest, a row without any takes no place.  ``renormalize`` divides a row's weights by their sum."""
    dev = _tensor(logits, "logits", tuple(_TYPE), 2)
    tokens, experts = logits.shape
    if not (1 <= k <= experts):
        raise FlexSpmvError(f"k must be 1 to the number of experts, not {k}")
    if not (experts <= MAX_EXPERTS and k <= MAX_CHOICES):
        raise FlexSpmvError(f"at most {MAX_EXPERTS} experts and {MAX_CHOICES} choices")
    stride = _rows_of(logits, "logits", aligned=False)
    d = Desc(tokens, tokens * k, experts, k, 0, 0, _TYPE[logits.dtype], 0, _RENORMALIZE if renormalize else 0, 0, stride)
    need = _route_bytes(tokens, experts)
    # one allocation: the plan's arrays behind one another, then the workspace, on 16 bytes
    pairs = tokens * k
    used = 4 * pairs + experts + 1
    at = -(-used // 4) * 4
    buf = torch.empty(at + need // 4, dtype=torch.int32, device=logits.device)
    weights, ids, slots, rows, offsets, _ = buf.split_with_sizes((pairs, pairs, pairs, pairs, experts + 1, at + need // 4 - used))
    plan = Plan(weights.view(torch.float32).view(tokens, k), ids.view(tokens, k), offsets, rows, slots.view(tokens, k), bool(renormalize))
    base = buf.data_ptr()
    outs = _FIVE(base, base + 4 * pairs, base + 16 * pairs, base + 12 * pairs, base + 8 * pairs)
    ins = (ctypes.c_void_p * 1)(logits.data_ptr())
    return BoundCall(_function("expert_route", _WITH_WORKSPACE),
                     (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs), base + 4 * at, need), dev,
                     (d, ins, outs, logits, buf), plan)


@_operator
def route_backward(dweights: torch.Tensor, logits: torch.Tensor, plan: Plan, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``route``'s weights with respect to ``logits``, of their type; the choice itself has none."""
    dev = _tensor(logits, "logits", tuple(_TYPE), 2)
    tokens, experts = logits.shape
    stride = _rows_of(logits, "logits", aligned=False)
    _tensor(dweights, "dweights", (torch.float32,), 2, dev)
    for name, t, dt in (("weights", plan.weights, torch.float32), ("experts", plan.experts, torch.int32)):
        _tensor(t, f"plan.{name}", (dt,), 2, dev)
        _whole(t, f"plan.{name}")
    k = plan.weights.shape[1]
    _need(plan.weights.shape[0] == tokens and plan.experts.shape == plan.weights.shape and dweights.shape == plan.weights.shape,
          "dweights and the plan must be of the logits' rows")
    _need(plan.offsets.numel() == experts + 1, "the plan must be of the logits' experts")
    _whole(dweights, "dweights")
    out = _out(out, (tokens, experts), logits.dtype, logits.device, dweights=dweights, logits=logits, weights=plan.weights, experts=plan.experts)
    d = Desc(tokens, tokens * k, experts, k, 0, 0, _TYPE[logits.dtype], 0, _RENORMALIZE if plan.renormalize else 0, 0, stride)
    ins, outs = _pointers((dweights, logits, plan.weights, plan.experts)), _pointers((out,))
    return BoundCall(_function("expert_route_backward", _PLAIN), (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs)), dev,
                     (d, ins, outs, dweights, logits, plan, out), out)


class Balance(NamedTuple):
    """What ``balance_loss`` returns."""
    loss: torch.Tensor           # () float32
    counts: torch.Tensor         # (experts) int32: the pairs of an expert
    mean: torch.Tensor           # (experts) float32: its mean probability
    tokens: torch.Tensor         # () int32: rows of the logits that are not all -infinity


@functools.lru_cache(maxsize=256)
def _balance_bytes(tokens: int, experts: int, device: int) -> int:
    need = ctypes.c_size_t()
    d = Desc(tokens, 0, experts)
    with torch.cuda.device(device):
        _check(_function("balance_loss_bytes", _BYTES)(ctypes.addressof(d), ctypes.addressof(need)), "balance_loss")
    return need.value


@_operator
def balance_loss(logits: torch.Tensor, plan: Plan) -> Balance:
    """How unevenly ``plan`` uses the experts: ``experts / pairs * sum_e counts[e] * mean[e]`` with the softmax's mean over the tokens, 1 where all are
    used alike.  Rows of -infinity alone count for nothing.  Over several devices add up ``counts`` and ``tokens`` before the backward pass."""
    dev = _tensor(logits, "logits", tuple(_TYPE), 2)
    tokens, experts = logits.shape
    if not (1 <= experts <= MAX_EXPERTS):
        raise FlexSpmvError(f"1 to {MAX_EXPERTS} experts, not {experts}")
    _tensor(plan.offsets, "plan.offsets", (torch.int32,), 1, dev)
    _whole(plan.offsets, "plan.offsets")
    _need(plan.offsets.numel() == experts + 1 and plan.experts.shape[0] == tokens, "the plan must be of these logits")
    stride = _rows_of(logits, "logits", aligned=False)
    d = Desc(tokens, 0, experts, 0, 0, 0, _TYPE[logits.dtype], 0, 0, 0, stride)
    need = _balance_bytes(tokens, experts, dev)
    # no views: a training step may add to its loss, and no result keeps the workspace
    empty, device = torch.empty, logits.device
    out = Balance(empty((), dtype=torch.float32, device=device), empty(experts, dtype=torch.int32, device=device),
                  empty(experts, dtype=torch.float32, device=device), empty((), dtype=torch.int32, device=device))
    ws = empty(need, dtype=torch.uint8, device=device)
    ins, outs = (_P * 2)(logits.data_ptr(), plan.offsets.data_ptr()), (_P * 4)(*[t.data_ptr() for t in out])
    return BoundCall(_function("balance_loss", _WITH_WORKSPACE), (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs), ws.data_ptr(), need), dev,
                     (d, ins, outs, logits, plan, ws, out), out)


@_operator
def balance_loss_backward(dloss: torch.Tensor, logits: torch.Tensor, balance: Balance, plan: Optional[Plan] = None, dweights: Optional[torch.Tensor] = None,
                          out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``balance_loss`` with respect to ``logits``, the counts being constants; ``dloss`` () float32.  With ``plan`` and ``dweights`` the
    router's gradient (``route_backward``) is added, in one pass over the logits and with one rounding."""
    dev = _tensor(logits, "logits", tuple(_TYPE), 2)
    tokens, experts = logits.shape
    if not (1 <= experts <= MAX_EXPERTS):
        raise FlexSpmvError(f"1 to {MAX_EXPERTS} experts, not {experts}")
    stride = _rows_of(logits, "logits", aligned=False)
    _tensor(dloss, "dloss", (torch.float32,), 0, dev)
    _tensor(balance.counts, "balance.counts", (torch.int32,), 1, dev)
    _whole(balance.counts, "balance.counts")
    _need(balance.counts.numel() == experts, "balance must be of the logits' experts")
    _tensor(balance.tokens, "balance.tokens", (torch.int32,), 0, dev)
    _need((plan is None) == (dweights is None), "the router's gradient takes both plan and dweights")
    k, renormalize, weights, ids = 0, False, None, None
    if plan is not None:
        weights, ids, renormalize = plan.weights, plan.experts, plan.renormalize
        _tensor(dweights, "dweights", (torch.float32,), 2, dev)
        for name, t, dt in (("plan.weights", weights, torch.float32), ("plan.experts", ids, torch.int32)):
            _tensor(t, name, (dt,), 2, dev)
            _whole(t, name)
        _whole(dweights, "dweights")
        k = weights.shape[1]
        _need(weights.shape[0] == tokens and ids.shape == weights.shape and dweights.shape == weights.shape, "dweights and the plan must be of the logits' rows")
        _need(plan.offsets.numel() == experts + 1, "the plan must be of the logits' experts")
    out = _out(out, (tokens, experts), logits.dtype, logits.device, dloss=dloss, logits=logits, counts=balance.counts, tokens=balance.tokens, dweights=dweights,
               weights=weights, experts=ids)
    d = Desc(tokens, tokens * k, experts, k, 0, 0, _TYPE[logits.dtype], 0, _RENORMALIZE if renormalize else 0, 0, stride)
    ins = (_P * 7)(*[t.data_ptr() if t is not None else 0 for t in (dloss, logits, balance.counts, balance.tokens, dweights, weights, ids)])
    outs = _pointers((out,))
    return BoundCall(_function("balance_loss_backward", _PLAIN), (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs)), dev,
                     (d, ins, outs, dloss, logits, balance, plan, dweights, out), out)


def _grouped(name: str, d: Desc, ins, out, dev: int, ws=None) -> BoundCall:
    flag = _flag(dev)
    pin, pout = (_P * len(ins))(*[t.data_ptr() if t is not None else 0 for t in ins]), _pointers((out,))
    args = (ctypes.addressof(d), ctypes.addressof(pin), ctypes.addressof(pout))
    if ws is not None:
        args += (ws.data_ptr(), ws.numel())
    return BoundCall(_function(name, _GROUPED if ws is None else _GROUPED_DW), args + (flag.tensor.data_ptr(),), dev,
                     (d, pin, pout, ins, out, flag, ws), out, flag.view)


def _plan_arrays(offsets, rows, experts: int, dev: int):
    _tensor(offsets, "offsets", (torch.int32,), 1, dev)
    if not (offsets.numel() == experts + 1):
        raise FlexSpmvError(f"offsets must have {experts + 1} entries, not {offsets.numel()}")
    _whole(offsets, "offsets")
    if rows is not None:
        _tensor(rows, "rows", (torch.int32,), 1, dev)
        _whole(rows, "rows")


def _weights_of(weight, dtype, dev: int):
    _tensor(weight, "weight", (dtype,), 3, dev)
    _whole(weight, "weight")
    e, n, k = weight.shape
    if not (1 <= e <= MAX_EXPERTS):
        raise FlexSpmvError(f"1 to {MAX_EXPERTS} experts, not {e}")
    if not (n >= 8 and k >= 8 and n % 8 == 0 and k % 8 == 0 and weight.data_ptr() % 16 == 0):
        raise FlexSpmvError(f"weight: both sides of a matrix must be multiples of 8 and the first value on 16 bytes, not {n} x {k}")
    return e, n, k


@_operator
def grouped_matmul(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, rows: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[i] = weight[e] @ x[rows[i]]`` for the places ``offsets[e] <= i < offsets[e + 1]`` (``rows`` None: ``x[i]``).

    ``x`` (tokens, k) and ``weight`` (experts, n, k) of one 16-bit type; n and k multiples of 8; x's rows may be apart.  ``y`` is (places, n), the
    places being ``rows.numel()`` or x's rows; sums are in 32 bits, rounded once.  Rows of no expert are zeros."""
    dev = _tensor(x, "x", _HALF, 2)
    e, n, k = _weights_of(weight, x.dtype, dev)
    if not (x.shape[1] == k):
        raise FlexSpmvError(f"x's rows must have {k} values, not {x.shape[1]}")
    _plan_arrays(offsets, rows, e, dev)
    slots = rows.numel() if rows is not None else x.shape[0]
    _need(slots == 0 or x.shape[0] > 0, "x has no rows to take")
    stride = _rows_of(x, "x")
    out = _out(out, (slots, n), x.dtype, x.device, x=x, weight=weight, offsets=offsets, rows=rows)
    d = Desc(x.shape[0], slots, e, 0, n, k, _TYPE[x.dtype], _TYPE[x.dtype], 0, 0, stride)
    return _grouped("grouped_matmul", d, (x, weight, offsets, rows), out, dev)


@_operator
def grouped_matmul_dx(dy: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dx[i] = weight[e].T @ dy[i]``: the gradient of ``grouped_matmul`` with respect to the rows it took, one for each place (``combine(dx,
    slots)`` adds a token's).  ``dy`` (places, n), its rows may be apart."""
    dev = _tensor(dy, "dy", _HALF, 2)
    e, n, k = _weights_of(weight, dy.dtype, dev)
    if not (dy.shape[1] == n):
        raise FlexSpmvError(f"dy's rows must have {n} values, not {dy.shape[1]}")
    _plan_arrays(offsets, None, e, dev)
    slots, stride = dy.shape[0], _rows_of(dy, "dy")
    out = _out(out, (slots, k), dy.dtype, dy.device, dy=dy, weight=weight, offsets=offsets)
    d = Desc(slots, slots, e, 0, n, k, _TYPE[dy.dtype], _TYPE[dy.dtype], 0, 0, stride)
    return _grouped("grouped_matmul_dx", d, (dy, weight, offsets), out, dev)


@_operator
def grouped_matmul_dw(dy: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, rows: Optional[torch.Tensor] = None,
                      dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dw[e] = sum over e's places i of outer(dy[i], x[rows[i]])``: (experts, n, k) of ``dtype`` (the inputs', or float32); experts without
    places have zeros."""
    dev = _tensor(dy, "dy", _HALF, 2)
    _tensor(x, "x", (dy.dtype,), 2, dev)
    _need(isinstance(offsets, torch.Tensor) and offsets.dim() == 1 and offsets.numel() >= 2, "offsets must have an entry for each expert and one more")
    e = offsets.numel() - 1
    if not (e <= MAX_EXPERTS):
        raise FlexSpmvError(f"at most {MAX_EXPERTS} experts")
    _plan_arrays(offsets, rows, e, dev)
    slots, n, k = dy.shape[0], dy.shape[1], x.shape[1]
    _need(n >= 8 and k >= 8, "dy and x must have rows of at least 8 values")
    _need((rows.numel() if rows is not None else x.shape[0]) == slots, "dy must have a row for each place")
    _need(slots == 0 or x.shape[0] > 0, "x has no rows to take")
    dtype = dtype or (out.dtype if out is not None else dy.dtype)
    if not (dtype in (torch.float32, dy.dtype)):
        raise FlexSpmvError(f"dw is {dy.dtype} or torch.float32, not {dtype}")
    dy_stride, x_stride = _rows_of(dy, "dy"), _rows_of(x, "x")
    out = _out(out, (e, n, k), dtype, dy.device, dy=dy, x=x, offsets=offsets, rows=rows)
    d = Desc(x.shape[0], slots, e, 0, n, k, _TYPE[dy.dtype], _TYPE[dtype], 0, 0, dy_stride, x_stride)
    ws = torch.empty(2 * slots * k if rows is not None else 0, dtype=torch.uint8, device=dy.device)          # a copy of x's rows
    return _grouped("grouped_matmul_dw", d, (dy, x, offsets, rows), out, dev, ws)


def _combine_arrays(slots, weights, dev: int):
    _tensor(slots, "slots", (torch.int32,), 2, dev)
    _whole(slots, "slots")
    if not (1 <= slots.shape[1] <= MAX_CHOICES):
        raise FlexSpmvError(f"1 to {MAX_CHOICES} choices, not {slots.shape[1]}")
    if weights is not None:
        _tensor(weights, "weights", (torch.float32,), 2, dev)
        _whole(weights, "weights")
        _need(weights.shape == slots.shape, "weights must have the shape of slots")


@_operator
def combine(z: torch.Tensor, slots: torch.Tensor, weights: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * z[slots[t, j]]`` (no weights: ones), sums in 32 bits in the order of j, rounded once; slots of -1 add nothing."""
    dev = _tensor(z, "z", _HALF, 2)
    _combine_arrays(slots, weights, dev)
    _need(z.shape[1] >= 1, "z must have columns")
    stride = _rows_of(z, "z", aligned=False)
    out = _out(out, (slots.shape[0], z.shape[1]), z.dtype, z.device, z=z, slots=slots, weights=weights)
    d = Desc(slots.shape[0], z.shape[0], 0, slots.shape[1], z.shape[1], 0, _TYPE[z.dtype], 0, 0, 0, stride)
    ins = (ctypes.c_void_p * 3)(z.data_ptr(), slots.data_ptr(), weights.data_ptr() if weights is not None else 0)
    outs = _pointers((out,))
    return BoundCall(_function("expert_combine", _PLAIN), (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs)), dev,
                     (d, ins, outs, z, slots, weights, out), out)


@_operator
def combine_backward(dout: torch.Tensor, z: torch.Tensor, slots: torch.Tensor, weights: Optional[torch.Tensor], offsets: torch.Tensor):
    """Gradients of ``combine``: ``dz`` (z's shape; rows from ``offsets[-1]`` on are zeros) and ``dweights`` (float32).  ``slots`` names each of
    the other rows once, as ``route``'s does."""
    dev = _tensor(z, "z", _HALF, 2)
    _tensor(dout, "dout", (z.dtype,), 2, dev)
    _combine_arrays(slots, weights, dev)
    _tensor(offsets, "offsets", (torch.int32,), 1, dev)
    _whole(offsets, "offsets")
    _need(offsets.numel() >= 2, "offsets must have an entry for each expert and one more")
    _need(z.shape[1] >= 1 and tuple(dout.shape) == (slots.shape[0], z.shape[1]), "dout must have combine's result's shape")
    dz, dweights = torch.empty(z.shape, dtype=z.dtype, device=z.device), torch.empty(slots.shape, dtype=torch.float32, device=z.device)
    d = Desc(slots.shape[0], z.shape[0], offsets.numel() - 1, slots.shape[1], z.shape[1], 0, _TYPE[z.dtype], 0, 0, 0,
             _rows_of(dout, "dout", aligned=False), _rows_of(z, "z", aligned=False))
    ins = (ctypes.c_void_p * 5)(dout.data_ptr(), z.data_ptr(), slots.data_ptr(), weights.data_ptr() if weights is not None else 0, offsets.data_ptr())
    outs = _pointers((dz, dweights))
    return BoundCall(_function("expert_combine_backward", _PLAIN), (ctypes.addressof(d), ctypes.addressof(ins), ctypes.addressof(outs)), dev,
                     (d, ins, outs, dout, z, slots, weights, offsets, dz, dweights), (dz, dweights))


_get_device, _numel, _is_contiguous, _data_ptr = torch.Tensor.get_device, torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.data_ptr
_dtype_of = operator.attrgetter("dtype")


def _at(values: array.array) -> int:
    return values.buffer_info()[0]


def _list_of(tensors, name: str):
    """Checks a list of tensors; returns their device, types, lengths and addresses.  Several hundred of them are usual, so each question is one
    loop inside the interpreter."""
    try:
        devices, types = set(map(_get_device, tensors)), list(map(_TYPE.get, map(_dtype_of, tensors)))
        good = len(devices) == 1 and None not in types and all(map(_is_contiguous, tensors))
    except (TypeError, AttributeError):
        good, devices = False, ()
    dev = next(iter(devices), -1)
    if not good or dev < 0:
        raise FlexSpmvError(f"{name} must be contiguous CUDA tensors of float32, bfloat16 or float16 on one device")
    return dev, types, list(map(_numel, tensors)), list(map(_data_ptr, tensors))


def _clip(tensors: list, max_norm: float, outs) -> BoundCall:
    _need(len(tensors) > 0, "there must be a tensor")
    n = len(tensors)
    dev, type_list, length_list, addresses = _list_of(tensors, "the tensors")
    lengths, types, pin = array.array("q", length_list), array.array("i", type_list), array.array("Q", addresses)
    pout, out_types = None, None
    if outs is tensors:
        pout, out_types = pin, types
    elif outs is not None:
        outs = list(outs)
        if len(outs) != n:
            raise FlexSpmvError(f"out must have {n} tensors, not {len(outs)}")
        out_dev, out_type_list, out_lengths, out_addresses = _list_of(outs, "out")
        if out_dev != dev or out_lengths != length_list:
            raise FlexSpmvError("out must be on the tensors' device and have as many values, each as its tensor")
        pout, out_types = array.array("Q", out_addresses), array.array("i", out_type_list)
    need, pieces = ctypes.c_size_t(), ctypes.c_int32()
    _check(_function("clip_gradients_bytes", _CLIP_BYTES)(n, _at(lengths), ctypes.addressof(need), ctypes.addressof(pieces)), "clip_gradients")
    ws = torch.empty(need.value // 8, dtype=torch.float64, device=tensors[0].device)
    norm = torch.empty((), dtype=torch.float32, device=tensors[0].device)
    plan = (n, _at(pin), _at(types), _at(lengths), _at(pout) if pout is not None else None, _at(out_types) if out_types is not None else None,
            ws.data_ptr(), need.value, _raw_stream(dev))
    if _current_device() == dev:
        st = _function("clip_gradients_plan", _CLIP_PLAN)(*plan)
    else:
        with torch.cuda.device(dev):
            st = _function("clip_gradients_plan", _CLIP_PLAN)(*plan)
    if st == -1:
        raise FlexSpmvError("tensors that are written must not share memory with others", st)
    _check(st, "clip_gradients_plan")
    args = (pieces.value, outs is not None, float(max_norm), norm.data_ptr(), ws.data_ptr(), need.value)
    return PlannedCall(_function("clip_gradients", _CLIP), args, dev, (ws, tensors, outs), norm)


@_operator
def grad_norm(tensors: Sequence[torch.Tensor]) -> torch.Tensor:
    """``sqrt(sum of all squares)`` over contiguous tensors of any of the three types: one float32 on the device, the same bits every time."""
    return _clip(list(tensors), 0.0, None)


@_operator
def clip_grad_norm(tensors: Sequence[torch.Tensor], max_norm: float, out: Optional[Sequence[torch.Tensor]] = None) -> torch.Tensor:
    """Scales the tensors by ``min(1, max_norm / (norm + 1e-6))``, in place or into ``out`` (tensors of the same lengths, of any of the three
    types), and returns the norm before it.  No two of them may share memory, but a tensor and its own result."""
    tensors = list(tensors)
    if not (max_norm >= 0):
        raise FlexSpmvError(f"max_norm must not be negative or NaN: {max_norm}")
    return _clip(tensors, max_norm, tensors if out is None else out)
