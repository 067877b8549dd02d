"""The dense operators' descriptors and plans without a GPU."""

import ctypes
import math
import random

import pytest
import torch

from qkan_b200 import Linear, _abi
from qkan_b200 import functional as F


def _lib():
    from qkan_b200 import build

    build.build()
    return _abi.load()


def _linear(M, K, N, dtype=_abi.QK_BF16, act=_abi.QK_ACT_NONE, flags=0):
    return _abi.desc_pointer(_abi.QkLinearDesc(M, K, N, dtype, act, flags))


def test_flags_of_the_linear_map():
    lib = _lib()
    for flags in (1, 4, 3, 1 << 31):
        assert lib.qk_linear_backward_workspace_bytes(_linear(64, 64, 64, flags=flags)) == 0
        assert b"flag" in lib.qk_last_error()
    sizes = {}
    for flags in (0, _abi.QK_LINEAR_ROUND_GRADS):
        sizes[flags] = lib.qk_linear_backward_workspace_bytes(_linear(8192, 256, 256, act=_abi.QK_ACT_SILU, flags=flags))
        assert lib.qk_linear_forward_workspace_bytes(_linear(8192, 256, 256, flags=flags)) >= 1
    # the second part of gz, 8192 x 256 bfloat16
    assert sizes[0] - sizes[_abi.QK_LINEAR_ROUND_GRADS] >= 8192 * 256 * 2
    one = lib.qk_linear_backward_workspace_bytes
    for dtype, act in ((_abi.QK_F32, _abi.QK_ACT_SILU), (_abi.QK_BF16, _abi.QK_ACT_NONE)):
        assert one(_linear(8192, 256, 256, dtype, act)) == one(_linear(8192, 256, 256, dtype, act, _abi.QK_LINEAR_ROUND_GRADS))


def test_rounding_of_the_gradients_is_off_unless_asked_for():
    assert Linear(4, 3).round_grads is False and Linear(4, 3, round_grads=True).round_grads is True


def _plan(product, M, K, N, dtype=_abi.QK_BF16, act=_abi.QK_ACT_NONE, flags=0):
    plan = _abi.QkLinearPlan()
    assert _lib().qk_linear_plan(_linear(M, K, N, dtype, act, flags), product, ctypes.byref(plan)) == _abi.QK_OK
    return plan


def test_plans_that_are_refused():
    lib, plan = _lib(), _abi.QkLinearPlan()
    for product in (-1, 3):
        assert lib.qk_linear_plan(_linear(64, 64, 64), product, ctypes.byref(plan)) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_linear_plan(_linear(64, 64, 64), 0, None) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_linear_plan(None, 0, ctypes.byref(plan)) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_linear_plan(_linear(-1, 64, 64), 0, ctypes.byref(plan)) == _abi.QK_ERR_BAD_ARGUMENT
    for size in ((0, 8, 8), (8, 0, 8), (8, 8, 0)):
        for product in range(3):
            assert _plan(product, *size).path == _abi.QK_LINEAR_NOTHING


def _cut(plan):
    return plan.tile_cols, plan.slices, plan.blocks


def test_gradients_run_one_by_one_take_the_plans_that_are_best_alone():
    """grad_x over the whole GPU has the sizes of a forward product; it is not left with the plan of a share of the SMs."""
    rng = random.Random(5)
    sizes = [(73, 3648, 648), (1816, 480, 888)]
    for _ in range(600):
        sizes.append([max(8, int(math.exp(rng.uniform(math.log(8), math.log(4096)))) // 8 * 8) for _ in range(3)])
    alone = 0
    for M, K, N in sizes:
        weight, x = (_plan(p, M, K, N) for p in (1, 2))
        assert weight.paired == x.paired and weight.sums_bias == (weight.tile_cols <= 128)
        if x.paired:
            assert weight.units + x.units <= 148 and weight.tile_cols == x.tile_cols, (M, K, N)
            continue
        alone += 1
        assert _cut(x) == _cut(_plan(0, M, N, K)), (M, K, N)
        if weight.tile_cols > 128:
            assert _cut(weight) == _cut(_plan(0, N, M, K)), (M, K, N)
    assert alone > 20
    # a pair is not given up for narrower tiles where it is the cheaper of the two
    assert _plan(2, 1816, 480, 888).paired


def test_eps_beyond_float32_is_refused():
    """Where eps is infinite every row would come out as the bias."""
    for eps in (1e39, 1e300, float("inf"), float("nan"), -1e-5):
        with pytest.raises(ValueError, match="eps"):
            F.layer_norm(torch.zeros(2, 4), eps=eps)
    lib, one = _lib(), ctypes.c_void_p(256)
    desc = _abi.desc_pointer(_abi.QkNormDesc(4, 4, 0, 0, float("inf"), 0))
    assert lib.qk_layer_norm_forward(desc, one, None, None, one, None, None) == _abi.QK_ERR_BAD_ARGUMENT
    assert b"eps" in lib.qk_last_error()
    with pytest.raises(RuntimeError, match="no CPU fallback"):  # the last of the checks
        F.layer_norm(torch.zeros(2, 4), eps=3e38)


def test_plans_of_the_largest_sizes():
    most = 0x7fffff00
    for dtype in (_abi.QK_F32, _abi.QK_BF16):
        for size in ((most, 64, most), (most, most, 64), (64, most, most), (most, most, most)):
            for product in range(3):
                plan = _plan(product, *size, dtype=dtype)
                assert plan.path == _abi.QK_LINEAR_TENSOR and plan.units >= 1 and plan.slices >= 1 and plan.blocks >= 1
    assert _plan(0, most, 64, most).units == 2 ** 31 - 1
