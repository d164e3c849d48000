"""The expert operators' refusal of results that share memory with what a call reads: checked before anything is enqueued, so that
addresses which nothing reads will do."""
import ctypes
import random

import pytest
import torch

from flexspmv_b200 import experts
from flexspmv_b200.binding import FlexSpmvError, load_library
from flexspmv_b200.experts import Desc, _meets

BAD_ARG, FAR = -1, 1 << 32
SIZES = dict(tokens=16, slots=32, experts=4, choices=2, n=64, k=128, type=1, out_type=1, in_stride=128, in2_stride=136)
PAIRS, OFFSETS, MATRICES = 16 * 2 * 4, 5 * 4, 4 * 64 * 128 * 2


def rows(count, n, stride, size=2):
    """Bytes from the first row's beginning to the last one's end."""
    return ((count - 1) * stride + n) * size


# of each call: the inputs' and results' lengths in bytes, the workspace last
CALLS = {
    "expert_route": ([rows(16, 4, 128)], [PAIRS, PAIRS, OFFSETS, PAIRS, PAIRS, 16]),
    "expert_route_backward": ([PAIRS, rows(16, 4, 128), PAIRS, PAIRS], [16 * 4 * 2]),
    "grouped_matmul": ([rows(16, 128, 128), MATRICES, OFFSETS, 32 * 4], [32 * 64 * 2]),
    "grouped_matmul_dx": ([rows(32, 64, 128), MATRICES, OFFSETS], [32 * 128 * 2]),
    "grouped_matmul_dw": ([rows(32, 64, 128), rows(16, 128, 136), OFFSETS, 32 * 4], [MATRICES, 32 * 128 * 2]),
    "expert_combine": ([rows(32, 64, 128), PAIRS, PAIRS], [16 * 64 * 2]),
    "expert_combine_backward": ([rows(16, 64, 128), rows(32, 64, 136), PAIRS, PAIRS, OFFSETS], [32 * 64 * 2, PAIRS]),
}


def status(name, ins, outs):
    d = Desc(**SIZES)
    pointers = lambda p: (ctypes.c_void_p * len(p))(*p)
    args = [ctypes.byref(d), pointers(ins), pointers(outs)]
    if name in ("expert_route", "grouped_matmul_dw"):
        args += [ctypes.c_void_p(outs[-1]), ctypes.c_size_t(1 << 30)]
    if name.startswith("grouped"):
        args.append(None)
    return getattr(load_library(), f"flexspmv_{name}")(*args, None)


@pytest.mark.parametrize("name", CALLS)
def test_results_that_meet_what_is_read_or_written(name):
    in_bytes, out_bytes = CALLS[name]
    ins = [FAR * (1 + i) for i in range(len(in_bytes))]
    outs = [FAR * (20 + i) for i in range(len(out_bytes))]
    step = 16                                        # addresses stay on 16 bytes, so that no other check comes first
    for o, length in enumerate(out_bytes):
        others = list(zip(ins, in_bytes)) + [(a, n) for i, (a, n) in enumerate(zip(outs, out_bytes)) if i != o]
        for at, n in others:
            for place in {at, at + (n - 1) // step * step, at - (length - 1) // step * step}:
                moved = outs[:o] + [place] + outs[o + 1:]
                assert status(name, ins, moved) == BAD_ARG, (name, o, at, place)


def test_rows_apart():
    """Against the bytes themselves: what lies between the rows of a strided tensor, and beside it, is free."""
    r, base = random.Random(0), torch.zeros(4096, dtype=torch.uint8)
    for _ in range(5000):
        count, n, start, at, length = r.randint(1, 6), r.randint(1, 9), r.randint(0, 40), r.randint(0, 110), r.randint(1, 30)
        stride = n + r.randint(0, 5)
        t, out = base[start:].as_strided((count, n), (stride, 1)), base[at:at + length]
        held = {start + i * stride + j for i in range(count) for j in range(n)}
        assert _meets(out, t) == (not held.isdisjoint(range(at, at + length)))
    assert not _meets(base[:0], base) and not _meets(base, base[:0].view(0, 8))


def test_clip_of_tensors_that_meet():
    """The same tensor twice in place, results that meet one another, another tensor, a part of their own one, or the workspace."""
    lib, n = load_library(), 3
    lengths = (ctypes.c_int64 * n)(1000, 0, 500)
    types, wide = (ctypes.c_int32 * n)(1, 1, 1), (ctypes.c_int32 * n)(0, 0, 0)
    need, pieces = ctypes.c_size_t(), ctypes.c_int32()
    assert lib.flexspmv_clip_gradients_bytes(n, lengths, ctypes.byref(need), ctypes.byref(pieces)) == 0
    ws = FAR * 9

    def plan(grads, outs=None, out_types=types):
        return lib.flexspmv_clip_gradients_plan(n, (ctypes.c_void_p * n)(*grads), types, lengths, (ctypes.c_void_p * n)(*outs) if outs else None,
                                                out_types if outs else None, ctypes.c_void_p(ws), need, None)
    a, b, c = FAR, FAR * 2, FAR * 3
    for grads, outs, out_types in (
        ((a, 0, a), (a, 0, a), types), ((a, 0, a + 1998), (a, 0, a + 1998), types), ((a, 0, a - 998), (a, 0, a - 998), types),
        ((a, 0, b), (c, 0, c), types), ((a, 0, b), (c, 0, c + 1998), types), ((a, 0, b), (c, 0, c + 3996), wide), ((a, 0, b), (b, 0, c), types),
        ((a, 0, b), (c, 0, a), types), ((a, 0, b), (a + 2, 0, c), types), ((a, 0, b), (a - 2, 0, c), types),
    ):
        assert plan(grads, outs, out_types) == BAD_ARG, (grads, outs)
    assert plan((ws + need.value - 16, 0, b)) == BAD_ARG and plan((a, 0, b), (ws - 1984, 0, c)) == BAD_ARG and plan((a, 0, ws)) == BAD_ARG


ALIGN = -2
# bytes of a value, in the order of CALLS: bfloat16 in and out, 32-bit weights and indices; the products' matrices begin on 16 bytes
VALUES = {
    "expert_route": ([2], [4] * 5 + [16]), "expert_route_backward": ([4, 2, 4, 4], [2]), "grouped_matmul": ([16, 16, 4, 4], [16]),
    "grouped_matmul_dx": ([16, 16, 4], [16]), "grouped_matmul_dw": ([16, 16, 4, 4], [16, 16]), "expert_combine": ([2, 4, 4], [2]),
    "expert_combine_backward": ([2, 2, 4, 4, 4], [2, 4]),
}


@pytest.mark.parametrize("name", CALLS)
def test_arrays_that_begin_inside_a_value(name):
    in_bytes, out_bytes = CALLS[name]
    base = [FAR * (1 + i) for i in range(len(in_bytes) + len(out_bytes))]
    for i, value in enumerate(VALUES[name][0] + VALUES[name][1]):
        for off in {1, value // 2, value - 1}:
            at = list(base)
            at[i] += off
            assert status(name, at[:len(in_bytes)], at[len(in_bytes):]) == ALIGN, (name, i, off)


def test_clip_of_a_workspace_that_begins_inside_a_record():
    run = load_library().flexspmv_clip_gradients
    for norm, ws in ((FAR, FAR * 2 + 8), (FAR, FAR * 2 + 4), (FAR + 2, FAR * 2)):
        assert run(1, 0, ctypes.c_float(1), ctypes.c_void_p(norm), ctypes.c_void_p(ws), ctypes.c_size_t(1 << 30), None) == ALIGN


def test_host_tensors_of_a_bound_clip():
    for call in (lambda: experts.bind(experts.grad_norm, [torch.zeros(3)]), lambda: experts.bind(experts.clip_grad_norm, [torch.zeros(3)], 1.0)):
        with pytest.raises(FlexSpmvError, match="CUDA"):
            call()
