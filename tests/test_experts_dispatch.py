"""Which kernel the experts' linears take (no GPU): the shapes that the GPU
tests use for each of them still reach it on 256 CUs, whatever the output."""
import ctypes
import itertools

import pytest

import bonsai_b1
from tests.experts_ref import KERNELS


def plan(routes, experts, in_dim, out_dim, kind):
    waves, units = ctypes.c_int(-1), ctypes.c_int(-1)
    rows = bonsai_b1.load().b1_experts_plan(routes, experts, in_dim, out_dim, kind, 256, ctypes.byref(waves),
                                            ctypes.byref(units))
    return rows, waves.value, units.value


@pytest.mark.parametrize("shape", KERNELS)
def test_shapes_reach_their_kernel(shape):
    tokens, experts, k, in_dim, out_dim = shape
    for kind in (0, 1, 2, 3):
        assert plan(tokens * k, experts, in_dim, out_dim, kind) == KERNELS[shape], kind


def test_every_kernel_is_among_them():
    assert {(v if v[0] == 0 else (v[0],)) for v in KERNELS.values()} == {
        (0, 3, 1), (0, 4, 1), (0, 3, 2), (0, 4, 2), (0, 8, 2), (0, 8, 4), (32,), (64,), (128,)}


@pytest.mark.parametrize("experts", [1, 2, 7, 64, 300, 1024])
def test_a_plan_holds_for_every_size(experts):
    """It ends, and few rows are never chosen where their inputs' widest is passed."""
    for routes, in_dim, out_dim, kind in itertools.product([1, 2, 15, 100, 5000, (1 << 24) - 1],
                                                           [64, 320, 2048, 8192, 8256, 65536],
                                                           [1, 64, 1408, 1 << 17], [0, 3]):
        if kind == 3 and out_dim % 64:
            continue
        rows, waves, units = plan(routes, experts, in_dim, out_dim, kind)
        if rows == 0:
            assert in_dim <= 8192 and waves * units * 256 >= in_dim
        else:
            assert rows in (32, 64, 128)
