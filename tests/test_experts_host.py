"""What the expert operators answer without a GPU: the C entries' checks of their arguments, which come before any device work, and the
Python layer's refusal of host tensors."""
import ctypes

import pytest
import torch

from flexspmv_b200 import experts
from flexspmv_b200.binding import FlexSpmvError, load_library
from flexspmv_b200.experts import Desc

BAD_ARG, ALIGN, WORKSPACE, TOO_LARGE = -1, -2, -3, -4


@pytest.fixture(scope="module")
def lib():
    return load_library()


def desc(**kw):
    base = dict(tokens=16, slots=32, experts=4, choices=2, n=64, k=128, type=1, out_type=1, in_stride=128, in2_stride=128)
    base.update(kw)
    return Desc(**base)


def ptrs(*values):
    return (ctypes.c_void_p * len(values))(*values)


def test_descriptor_has_the_headers_size():
    assert ctypes.sizeof(Desc) == 64


@pytest.mark.parametrize("change,status", [
    (dict(tokens=-1), BAD_ARG), (dict(experts=0), BAD_ARG), (dict(choices=0), BAD_ARG), (dict(choices=5), BAD_ARG), (dict(in_stride=3), BAD_ARG),
    (dict(type=3), BAD_ARG), (dict(experts=1025, in_stride=1025), TOO_LARGE), (dict(experts=64, choices=33), TOO_LARGE), (dict(tokens=1 << 31), TOO_LARGE),
])
def test_route_refusals(lib, change, status):
    d = desc(**change)
    some = ptrs(*[4096] * 5)
    for call in (lambda: lib.flexspmv_expert_route(ctypes.byref(d), some, some, ctypes.c_void_p(4096), ctypes.c_size_t(1 << 40), None),
                 lambda: lib.flexspmv_expert_route_backward(ctypes.byref(d), some, some, None)):
        assert call() == status


def test_route_workspace_and_pointers(lib):
    n = ctypes.c_size_t()
    d = desc()
    assert lib.flexspmv_expert_route_bytes(ctypes.byref(d), ctypes.byref(n)) == 0 and n.value >= 16
    assert lib.flexspmv_expert_route_bytes(None, ctypes.byref(n)) == BAD_ARG
    some = ptrs(*[4096] * 5)
    assert lib.flexspmv_expert_route(ctypes.byref(d), some, some, None, ctypes.c_size_t(0), None) == WORKSPACE
    assert lib.flexspmv_expert_route(ctypes.byref(d), some, some, ctypes.c_void_p(4104), n, None) == ALIGN
    assert lib.flexspmv_expert_route(ctypes.byref(d), ptrs(0), some, ctypes.c_void_p(4096), n, None) == BAD_ARG
    assert lib.flexspmv_expert_route(ctypes.byref(d), some, ptrs(4096, 4096, 0, 4096, 4096), ctypes.c_void_p(4096), n, None) == BAD_ARG


def grouped(lib, which, d, ins, outs):
    if which == "dw":
        return lib.flexspmv_grouped_matmul_dw(ctypes.byref(d), ins, outs, None, ctypes.c_size_t(0), None, None)
    return getattr(lib, "flexspmv_grouped_matmul" + ("_dx" if which == "dx" else ""))(ctypes.byref(d), ins, outs, None, None)


@pytest.mark.parametrize("which", ["forward", "dx", "dw"])
@pytest.mark.parametrize("change,status", [
    (dict(slots=-1), BAD_ARG), (dict(experts=0), BAD_ARG), (dict(n=0), BAD_ARG), (dict(k=0), BAD_ARG), (dict(type=0), BAD_ARG), (dict(type=7), BAD_ARG),
    (dict(in_stride=56), BAD_ARG), (dict(n=60), ALIGN), (dict(k=124), ALIGN), (dict(in_stride=132), ALIGN), (dict(experts=1025), TOO_LARGE),
    (dict(slots=1 << 31), TOO_LARGE), (dict(slots=1 << 30, n=1 << 20, in_stride=1 << 20), TOO_LARGE),
])
def test_grouped_refusals(lib, which, change, status):
    assert grouped(lib, which, desc(**change), ptrs(*[4096] * 4), ptrs(4096)) == status


def test_grouped_pointers(lib):
    good, out = ptrs(*[4096] * 4), ptrs(4096)
    for which in ("forward", "dx", "dw"):
        for i in range(3):
            broken = ptrs(*[0 if j == i else 4096 for j in range(4)])
            assert grouped(lib, which, desc(), broken, out) == BAD_ARG
        assert grouped(lib, which, desc(), good, ptrs(0)) == BAD_ARG and grouped(lib, which, desc(), None, out) == BAD_ARG
        for i in range(2):
            assert grouped(lib, which, desc(), ptrs(*[4104 if j == i else 4096 for j in range(4)]), out) == ALIGN
        assert grouped(lib, which, desc(), good, ptrs(4104)) == ALIGN
    assert grouped(lib, "dw", desc(out_type=2), good, out) == BAD_ARG            # bfloat16 in, float16 out
    assert grouped(lib, "dw", desc(), good, out) == WORKSPACE                    # a list of rows, no workspace
    assert grouped(lib, "forward", desc(tokens=0), good, out) == BAD_ARG         # rows of nothing
    assert grouped(lib, "forward", desc(slots=17), ptrs(4096, 4096, 4096, 0), out) == BAD_ARG      # more places than rows, no list
    assert grouped(lib, "forward", desc(slots=0), good, out) == 0
    n = ctypes.c_size_t()
    assert lib.flexspmv_grouped_matmul_dw_bytes(ctypes.byref(desc()), ctypes.byref(n)) == 0 and n.value == 32 * 128 * 2


def test_combine_refusals(lib):
    some = ptrs(*[4096] * 5)
    for change, status in ((dict(n=0), BAD_ARG), (dict(choices=0), BAD_ARG), (dict(type=0), BAD_ARG), (dict(in_stride=63), BAD_ARG),
                           (dict(choices=33), TOO_LARGE), (dict(slots=1 << 31), TOO_LARGE)):
        assert lib.flexspmv_expert_combine(ctypes.byref(desc(**change)), some, some, None) == status
        assert lib.flexspmv_expert_combine_backward(ctypes.byref(desc(**change)), some, some, None) == status
    assert lib.flexspmv_expert_combine(ctypes.byref(desc()), ptrs(4096, 0, 0), some, None) == BAD_ARG
    assert lib.flexspmv_expert_combine(ctypes.byref(desc(tokens=0)), ptrs(0, 0, 0), ptrs(0), None) == 0
    assert lib.flexspmv_expert_combine_backward(ctypes.byref(desc(in2_stride=8)), some, some, None) == BAD_ARG
    assert lib.flexspmv_expert_combine_backward(ctypes.byref(desc()), ptrs(4096, 4096, 4096, 0, 0), some, None) == BAD_ARG


def test_clip_refusals(lib):
    n, pieces = ctypes.c_size_t(), ctypes.c_int32()
    lengths = (ctypes.c_int64 * 3)(10, 0, 100_000)
    types = (ctypes.c_int32 * 3)(0, 1, 2)
    assert lib.flexspmv_clip_gradients_bytes(3, lengths, ctypes.byref(n), ctypes.byref(pieces)) == 0
    assert pieces.value == 1 + 25 and n.value > 24 * 26
    assert lib.flexspmv_clip_gradients_bytes(1, (ctypes.c_int64 * 1)(-1), ctypes.byref(n), ctypes.byref(pieces)) == BAD_ARG
    lib.flexspmv_clip_gradients_bytes(3, lengths, ctypes.byref(n), ctypes.byref(pieces))

    def plan(grads=(4096, 0, 8192), t=types, outs=None, out_types=None, ws=4096, size=n):
        return lib.flexspmv_clip_gradients_plan(3, ptrs(*grads), t, lengths, ptrs(*outs) if outs else None, out_types, ctypes.c_void_p(ws), size, None)
    assert plan(grads=(0, 0, 8192)) == BAD_ARG and plan(t=(ctypes.c_int32 * 3)(0, 1, 3)) == BAD_ARG
    assert plan(grads=(4098, 0, 8192)) == ALIGN and plan(outs=(4096, 0, 8192)) == BAD_ARG            # no types for the outputs
    assert plan(outs=(4096, 0, 8192), out_types=(ctypes.c_int32 * 3)(0, 1, 0)) == BAD_ARG            # in place, another type
    assert plan(ws=0) == WORKSPACE and plan(size=ctypes.c_size_t(8)) == WORKSPACE and plan(ws=4104) == ALIGN
    run = lib.flexspmv_clip_gradients
    assert run(pieces, 0, ctypes.c_float(1), None, ctypes.c_void_p(4096), n, None) == BAD_ARG
    assert run(pieces, 0, ctypes.c_float(1), ctypes.c_void_p(4096), None, n, None) == WORKSPACE


def test_host_tensors_are_refused():
    x, w, off = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((2, 64, 64), dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    slots = torch.zeros((4, 1), dtype=torch.int32)
    for call in (lambda: experts.route(torch.zeros((4, 8)), 2), lambda: experts.grouped_matmul(x, w, off), lambda: experts.grouped_matmul_dx(x, w, off),
                 lambda: experts.grouped_matmul_dw(x, x, off), lambda: experts.combine(x, slots), lambda: experts.combine_backward(x, x, slots, None, off),
                 lambda: experts.grad_norm([x]), lambda: experts.clip_grad_norm([x], 1.0), lambda: experts.bind(experts.combine, x, slots)):
        with pytest.raises(FlexSpmvError, match="CUDA"):
            call()
