"""What the residual stream's and the adapters' operators answer without a GPU: the C entries' checks of their arguments, which come before any device work,
the Python layer's refusal of host tensors, and the tests' generator against the published known answers."""
import ctypes

import numpy as np
import pytest
import torch

from flexspmv_b200 import adapters, experts, residual
from flexspmv_b200.binding import FlexSpmvError, load_library
from tests.philox import keep_mask, philox

BAD_ARG, ALIGN, WORKSPACE, TOO_LARGE = -1, -2, -3, -4


@pytest.fixture(scope="module")
def lib():
    return load_library()


def ptrs(*values):
    return (ctypes.c_void_p * len(values))(*values)


def spread(n, but=(), value=0):
    """n addresses far from one another, those of `but` replaced."""
    return ptrs(*[value if i in but else (i + 1) << 32 for i in range(n)])


def rows(**kw):
    base = dict(rows=16, width=64, type=1, param_type=0, eps=1e-5, p=0.1)
    base.update(kw)
    stride = base.pop("stride", (0, 0, 0))
    d = residual.Desc(**base)
    d.stride[:] = stride
    return d


OUT = 1 << 40          # far from all inputs


def outs(n, but=(), value=0):
    return ptrs(*[value if i in but else OUT + (i << 32) for i in range(n)])


def call(lib, name, d, ins, out, ws=1 << 50, size=1 << 40):
    if name == "layer_norm_backward":
        return lib.flexspmv_layer_norm_backward(ctypes.byref(d), ins, out, ctypes.c_void_p(ws), ctypes.c_size_t(size), None)
    return getattr(lib, f"flexspmv_{name}")(ctypes.byref(d), ins, out, None)


def test_descriptors_have_the_headers_sizes():
    assert ctypes.sizeof(residual.Desc) == 64 and ctypes.sizeof(adapters.Desc) == 40


def test_generator_has_the_published_answers():
    assert [int(v) for v in philox([0] * 4, [0] * 2)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert [int(v) for v in philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2)] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert [int(v) for v in philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0])] == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    keep = keep_mask(300, 501, 0.3, -5, 1 << 40)
    assert abs(keep.mean() - 0.7) < 5 * (0.21 / keep.size) ** 0.5 and not np.array_equal(keep, keep_mask(300, 501, 0.3, -5, (1 << 40) + 1))


@pytest.mark.parametrize("name,ins,out", [("layer_norm", 5, 4), ("layer_norm_backward", 7, 4), ("dropout", 3, 1)])
def test_rows_refusals(lib, name, ins, out):
    for change, status in ((dict(rows=-1), BAD_ARG), (dict(width=0), BAD_ARG), (dict(type=3), BAD_ARG), (dict(type=-1), BAD_ARG), (dict(p=-0.1), BAD_ARG),
                           (dict(p=1.0), BAD_ARG), (dict(p=float("nan")), BAD_ARG), (dict(stride=(63, 0, 0)), BAD_ARG), (dict(stride=(0, 63, 0)), BAD_ARG),
                           (dict(rows=1 << 31), TOO_LARGE), (dict(width=(1 << 24) + 1), TOO_LARGE)):
        assert call(lib, name, rows(**change), spread(ins), outs(out)) == status, change
    assert call(lib, name, rows(), None, outs(out)) == BAD_ARG and call(lib, name, rows(), spread(ins), None) == BAD_ARG
    if name != "dropout":
        for change in (dict(param_type=2), dict(eps=-1.0), dict(eps=float("nan"))):
            assert call(lib, name, rows(**change), spread(ins), outs(out)) == BAD_ARG


def test_rows_pointers(lib):
    for but, status in (((0,), BAD_ARG), ((4,), BAD_ARG)):
        assert call(lib, "layer_norm", rows(), spread(5, but), outs(4)) == status
    for but in (0, 2, 3):
        assert call(lib, "layer_norm", rows(), spread(5), outs(4, (but,))) == BAD_ARG
    assert call(lib, "layer_norm", rows(), spread(5, (0,), 4097), outs(4)) == ALIGN and call(lib, "layer_norm", rows(), spread(5, (4,), 4100), outs(4)) == ALIGN
    assert call(lib, "layer_norm", rows(rows=0), spread(5, range(5)), outs(4, range(4))) == 0
    for but in (0, 1, 3, 4, 6):
        assert call(lib, "layer_norm_backward", rows(), spread(7, (but,)), outs(4)) == BAD_ARG
    for but in (0, 1, 2, 3):             # one of dweight and dbias alone, too
        assert call(lib, "layer_norm_backward", rows(), spread(7), outs(4, (but,))) == BAD_ARG
    assert call(lib, "layer_norm_backward", rows(), spread(7), outs(4), ws=0) == WORKSPACE
    assert call(lib, "layer_norm_backward", rows(), spread(7), outs(4), size=8) == WORKSPACE
    assert call(lib, "layer_norm_backward", rows(), spread(7), outs(4), ws=(1 << 50) + 4) == ALIGN
    for but in (0, 2):
        assert call(lib, "dropout", rows(), spread(3, (but,)), outs(1)) == BAD_ARG
    assert call(lib, "dropout", rows(), spread(3), outs(1, (0,))) == BAD_ARG and call(lib, "dropout", rows(), spread(3), outs(1, (0,), OUT + 1)) == ALIGN
    n = ctypes.c_size_t()
    assert lib.flexspmv_layer_norm_backward_bytes(ctypes.byref(rows()), ctypes.byref(n)) == 0 and n.value >= 2 * 64 * 4
    assert lib.flexspmv_layer_norm_backward_bytes(ctypes.byref(rows(width=0)), ctypes.byref(n)) == BAD_ARG


def test_results_that_share_memory_are_refused(lib):
    at = 1 << 32                         # x: 16 rows of 64 values of 16 bits
    size = 16 * 64 * 2
    for inside in (at, at + size - 2, at - size + 2):
        assert call(lib, "dropout", rows(), spread(3), ptrs(inside)) == BAD_ARG
        assert call(lib, "layer_norm", rows(), spread(5), outs(4, (1,), inside)) == BAD_ARG
    assert call(lib, "layer_norm", rows(), spread(5), ptrs(OUT, OUT + 2, OUT + (2 << 32), OUT + (3 << 32))) == BAD_ARG          # y and the sum
    assert call(lib, "layer_norm_backward", rows(), spread(7), outs(4, (1,), at)) == BAD_ARG
    assert call(lib, "layer_norm_backward", rows(), spread(7), outs(4), ws=OUT + (1 << 32)) == BAD_ARG


def expert(**kw):
    base = dict(tokens=16, slots=32, experts=8, choices=2, type=1, in_stride=8)
    base.update(kw)
    return experts.Desc(**base)


def balance(lib, d, ins=None, out=None, ws=1 << 50, size=1 << 30):
    return lib.flexspmv_balance_loss(ctypes.byref(d), ins or spread(2), out or outs(4), ctypes.c_void_p(ws), ctypes.c_size_t(size), None)


def balance_backward(lib, d, ins=None, out=None):
    return lib.flexspmv_balance_loss_backward(ctypes.byref(d), ins or spread(7), out or outs(1), None)


def test_balance_refusals(lib):
    for change, status in ((dict(tokens=-1), BAD_ARG), (dict(experts=0), BAD_ARG), (dict(in_stride=7), BAD_ARG), (dict(type=3), BAD_ARG),
                           (dict(experts=1025, in_stride=1025), TOO_LARGE), (dict(tokens=1 << 31), TOO_LARGE)):
        assert balance(lib, expert(**change)) == status and balance_backward(lib, expert(**change)) == status
    for but in range(2):
        assert balance(lib, expert(), ins=spread(2, (but,))) == BAD_ARG
    for but in range(4):
        assert balance(lib, expert(), out=outs(4, (but,))) == BAD_ARG
    assert balance(lib, expert(), ws=0) == WORKSPACE and balance(lib, expert(), size=4) == WORKSPACE and balance(lib, expert(), ws=4104) == ALIGN
    assert balance(lib, expert(), out=outs(4, (2,), 1 << 32)) == BAD_ARG                      # shares memory with the logits
    for but in (0, 1, 2, 3, 5, 6):
        assert balance_backward(lib, expert(), ins=spread(7, (but,))) == BAD_ARG
    assert balance_backward(lib, expert(choices=9)) == BAD_ARG and balance_backward(lib, expert(experts=64, in_stride=64, choices=33)) == TOO_LARGE
    assert balance_backward(lib, expert(), out=ptrs(1 << 33)) == BAD_ARG and balance_backward(lib, expert(), out=ptrs(OUT + 1)) == ALIGN
    n = ctypes.c_size_t()
    assert lib.flexspmv_balance_loss_bytes(ctypes.byref(expert()), ctypes.byref(n)) == 0 and n.value >= 36


def adapter(**kw):
    base = dict(tokens=16, x_stride=64, adapters=4, rank=16, n=128, k=64, type=1)
    base.update(kw)
    return adapters.Desc(**base)


def project(lib, d, ins=None, out=None, ws=1 << 50, size=1 << 40):
    return lib.flexspmv_adapted_project(ctypes.byref(d), ins or spread(6), out or outs(1), ctypes.c_void_p(ws), ctypes.c_size_t(size), None, None)


def test_adapter_refusals(lib):
    for change, status in ((dict(tokens=-1), BAD_ARG), (dict(adapters=0), BAD_ARG), (dict(rank=0), BAD_ARG), (dict(n=0), BAD_ARG), (dict(k=0), BAD_ARG),
                           (dict(type=0), BAD_ARG), (dict(x_stride=56), BAD_ARG), (dict(rank=12), ALIGN), (dict(n=124), ALIGN), (dict(k=60), ALIGN),
                           (dict(x_stride=66), ALIGN), (dict(adapters=1025), TOO_LARGE), (dict(rank=520), TOO_LARGE), (dict(tokens=1 << 31), TOO_LARGE)):
        assert project(lib, adapter(**change)) == status, change
    for but in (0, 1, 2, 3, 5):
        assert project(lib, adapter(), ins=spread(6, (but,))) == BAD_ARG
        assert project(lib, adapter(), ins=spread(6, (but,), 4104)) == ALIGN
    assert project(lib, adapter(), ins=spread(6, (4,), 4098)) == ALIGN
    assert project(lib, adapter(), out=ptrs(0)) == BAD_ARG and project(lib, adapter(), out=ptrs(OUT + 8)) == ALIGN
    assert project(lib, adapter(), ws=0) == WORKSPACE and project(lib, adapter(), size=100) == WORKSPACE and project(lib, adapter(), ws=4104) == ALIGN
    for i in (0, 1, 2, 3, 5):
        assert project(lib, adapter(), out=ptrs((i + 1) << 32)) == BAD_ARG                    # shares memory with an input
        assert project(lib, adapter(), ws=(i + 1) << 32) == BAD_ARG
    assert project(lib, adapter(tokens=0)) == 0
    n = ctypes.c_size_t()
    assert lib.flexspmv_adapted_project_bytes(ctypes.byref(adapter()), ctypes.byref(n)) == 0 and n.value == 16 * 64 * 2
    assert lib.flexspmv_adapter_plan_bytes(ctypes.byref(adapter(rank=0)), ctypes.byref(n)) == 0          # a plan is of tokens and adapters alone

    def plan(ids=4096, to=1 << 40, size=n, d=adapter()):
        return lib.flexspmv_adapter_plan(ctypes.byref(d), ctypes.c_void_p(ids), ctypes.c_void_p(to), size, None, None)
    assert plan(ids=0) == BAD_ARG and plan(to=0) == WORKSPACE and plan(size=ctypes.c_size_t(n.value - 1)) == WORKSPACE and plan(to=4104) == ALIGN
    assert plan(ids=4098) == ALIGN and plan(ids=(1 << 40) + 16) == BAD_ARG and plan(d=adapter(adapters=1025)) == TOO_LARGE


def test_host_tensors_are_refused():
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros(64)
    stats, seed = torch.zeros(4), torch.zeros(2, dtype=torch.int64)
    logits = torch.zeros((4, 8))
    plan = experts.Plan(torch.zeros(4, 2), torch.zeros((4, 2), dtype=torch.int32), torch.zeros(9, dtype=torch.int32), None, None, False)
    matrix = torch.zeros((64, 64), dtype=torch.bfloat16)
    a, b = torch.zeros((2, 8, 64), dtype=torch.bfloat16), torch.zeros((2, 64, 8), dtype=torch.bfloat16)
    made = adapters.Plan(torch.zeros(64, dtype=torch.int32), 4, 2)
    for run in (lambda: residual.layer_norm(x, w, w), lambda: residual.layer_norm_backward(x, x, w, stats, stats), lambda: residual.dropout(x, 0.1, seed),
                lambda: experts.balance_loss(logits, plan), lambda: experts.bind(residual.dropout, x, 0.1, seed),
                lambda: experts.balance_loss_backward(torch.zeros(()), logits, experts.Balance(stats, stats, stats, stats)),
                lambda: adapters.plan(torch.zeros(4, dtype=torch.int32), 2), lambda: adapters.project(x, matrix, a, b, made)):
        with pytest.raises(FlexSpmvError, match="CUDA"):
            run()
