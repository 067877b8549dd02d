"""The dense operators' descriptors and plans without a GPU."""

from qkan_b200 import Linear, _abi


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
