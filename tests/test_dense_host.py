"""The dense operators without a GPU: refusals at the C entry points and in Python, modules, descriptors."""
import ctypes

import pytest
import torch
from torch import nn

import qkan_b200
from qkan_b200 import QKAN, HQKANBlock, LayerNorm, Linear, _abi
from qkan_b200 import functional as F


def _lib():
    from qkan_b200 import build

    build.build()
    return _abi.load()


def test_descriptors_have_the_header_layout():
    assert ctypes.sizeof(_abi.QkLinearDesc) == 24 and ctypes.sizeof(_abi.QkNormDesc) == 24


@pytest.mark.parametrize("fields,text", [
    ((-1, 4, 4, 0, 0, 0), b"negative"), ((4, -1, 4, 0, 0, 0), b"negative"), ((4, 4, -1, 0, 0, 0), b"negative"),
    ((4, 4, 4, 2, 0, 0), b"io_dtype"), ((4, 4, 4, 0, 7, 0), b"activation"), ((4, 4, 4, 0, -1, 0), b"activation"),
    ((4, 4, 4, 0, 0, 1), b"flag")])
def test_linear_descriptors_that_are_refused(fields, text):
    lib = _lib()
    dp = _abi.desc_pointer(_abi.QkLinearDesc(*fields))
    assert lib.qk_linear_forward_workspace_bytes(dp) == 0 and text in lib.qk_last_error()
    assert lib.qk_linear_backward_workspace_bytes(dp) == 0
    one = ctypes.c_void_p(256)
    assert lib.qk_linear_forward(dp, one, one, None, None, one, None, one, 1 << 30, None) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_linear_backward(dp, one, one, one, one, one, one, one, one, 1 << 30, None) == _abi.QK_ERR_BAD_ARGUMENT


def test_dimensions_beyond_the_index_range_are_refused():
    lib = _lib()
    for fields in ((2 ** 31 - 1, 1, 1), (1, 2 ** 31 - 1, 1), (1, 1, 2 ** 31 - 1)):
        dp = _abi.desc_pointer(_abi.QkLinearDesc(*fields, 0, 0, 0))
        one = ctypes.c_void_p(256)
        assert lib.qk_linear_forward_workspace_bytes(dp) == 0 and b"exceeds" in lib.qk_last_error()
        assert lib.qk_linear_forward(dp, one, one, None, None, one, None, one, 1 << 30, None) == _abi.QK_ERR_UNSUPPORTED
        assert lib.qk_linear_backward(dp, one, one, one, one, one, one, one, one, 1 << 30, None) == _abi.QK_ERR_UNSUPPORTED


def test_linear_pointers_and_workspaces_that_are_refused():
    lib = _lib()
    dp = _abi.desc_pointer(_abi.QkLinearDesc(640, 640, 640, _abi.QK_F32, _abi.QK_ACT_SILU, 0))
    one = ctypes.c_void_p(256)
    big = 1 << 40
    for x, w, y in ((None, one, one), (one, None, one), (one, one, None)):
        assert lib.qk_linear_forward(dp, x, w, None, None, y, None, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_linear_forward(dp, one, one, None, None, one, None, None, big, None) == _abi.QK_ERR_WORKSPACE
    assert lib.qk_linear_forward(dp, one, one, None, None, one, None, one, 0, None) == _abi.QK_ERR_WORKSPACE
    assert lib.qk_linear_forward(dp, one, one, None, None, one, None, ctypes.c_void_p(264), big, None) == _abi.QK_ERR_WORKSPACE
    # (x, weight, tape, gy): each is needed by what is asked for
    for x, w, t, g in ((None, one, one, one), (one, None, one, one), (one, one, None, one), (one, one, one, None)):
        assert lib.qk_linear_backward(dp, x, w, t, g, one, one, one, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_linear_backward(dp, one, one, one, one, one, one, one, one, 0, None) == _abi.QK_ERR_WORKSPACE
    # nothing asked for, nothing to do
    assert lib.qk_linear_backward(dp, None, None, None, None, None, None, None, None, 0, None) == _abi.QK_OK
    assert lib.qk_linear_forward(None, one, one, None, None, one, None, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT


def test_misaligned_rows_are_refused_where_they_are_read_in_place():
    lib = _lib()
    one, odd, big = ctypes.c_void_p(256), ctypes.c_void_p(258), 1 << 40
    dp = _abi.desc_pointer(_abi.QkLinearDesc(64, 64, 64, _abi.QK_BF16, 0, 0))
    for x, w in ((odd, one), (one, odd)):
        assert lib.qk_linear_forward(dp, x, w, None, None, one, None, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT
        assert b"aligned" in lib.qk_last_error()
        assert lib.qk_linear_backward(dp, x, w, None, one, one, one, one, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_linear_backward(dp, one, one, None, odd, one, one, one, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT


@pytest.mark.parametrize("fields,text", [
    ((-1, 4, 0, 0, 1e-5, 0), b"rows"), ((4, 0, 0, 0, 1e-5, 0), b"dim"), ((4, 4, 5, 0, 1e-5, 0), b"io_dtype"),
    ((4, 4, 0, 5, 1e-5, 0), b"param_dtype"), ((4, 4, 0, 0, -1.0, 0), b"eps"), ((4, 4, 0, 0, float("nan"), 0), b"eps"),
    ((4, 4, 0, 0, 1e-5, 2), b"flag")])
def test_norm_descriptors_that_are_refused(fields, text):
    lib = _lib()
    dp = _abi.desc_pointer(_abi.QkNormDesc(*fields))
    one = ctypes.c_void_p(256)
    assert lib.qk_layer_norm_backward_workspace_bytes(dp) == 0 and text in lib.qk_last_error()
    assert lib.qk_layer_norm_forward(dp, one, None, None, one, None, None) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_layer_norm_backward(dp, one, None, one, one, one, one, one, one, 1 << 30, None) == _abi.QK_ERR_BAD_ARGUMENT


def test_norm_pointers_and_workspaces_that_are_refused():
    lib = _lib()
    dp = _abi.desc_pointer(_abi.QkNormDesc(64, 64, _abi.QK_F32, _abi.QK_F32, 1e-5, 0))
    one = ctypes.c_void_p(256)
    assert lib.qk_layer_norm_forward(dp, None, None, None, one, None, None) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_layer_norm_forward(dp, one, None, None, None, None, None) == _abi.QK_ERR_BAD_ARGUMENT
    for x, s, g in ((None, one, one), (one, None, one), (one, one, None)):
        assert lib.qk_layer_norm_backward(dp, x, None, s, g, one, one, one, one, 1 << 30, None) == _abi.QK_ERR_BAD_ARGUMENT
    assert lib.qk_layer_norm_backward(dp, one, None, one, one, one, one, one, one, 0, None) == _abi.QK_ERR_WORKSPACE
    assert lib.qk_layer_norm_backward(dp, None, None, None, None, None, None, None, None, 0, None) == _abi.QK_OK


def test_pointers_off_their_elements_boundary_are_refused():
    lib = _lib()
    one, big = ctypes.c_void_p(256), 1 << 40
    for dtype, off in ((_abi.QK_F32, 258), (_abi.QK_BF16, 257)):
        odd = ctypes.c_void_p(off)
        dp = _abi.desc_pointer(_abi.QkLinearDesc(64, 65, 63, dtype, _abi.QK_ACT_SILU, 0))
        for k in range(6):  # x, weight, bias, residual, y, tape
            p = [odd if i == k else one for i in range(6)]
            assert lib.qk_linear_forward(dp, *p, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT
        for k in range(7):  # x, weight, tape, gy and the gradients
            p = [odd if i == k else one for i in range(7)]
            assert lib.qk_linear_backward(dp, *p, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT
        dp = _abi.desc_pointer(_abi.QkNormDesc(64, 65, dtype, dtype, 1e-5, 0))
        for k in range(5):  # x, weight, bias, y, stats
            p = [odd if i == k else one for i in range(5)]
            assert lib.qk_layer_norm_forward(dp, *p, None) == _abi.QK_ERR_BAD_ARGUMENT
        for k in range(7):  # x, weight, stats, gy and the gradients
            p = [odd if i == k else one for i in range(7)]
            assert lib.qk_layer_norm_backward(dp, *p, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT
        # a row's two statistics are read at once
        stats = ctypes.c_void_p(260)
        assert lib.qk_layer_norm_forward(dp, one, one, one, one, stats, None) == _abi.QK_ERR_BAD_ARGUMENT
        assert lib.qk_layer_norm_backward(dp, one, one, stats, one, one, one, one, one, big, None) == _abi.QK_ERR_BAD_ARGUMENT
        assert b"stats must be 8-byte aligned" in lib.qk_last_error()


def test_norm_rows_beyond_the_index_range_are_refused():
    # the loops over a row step past its end in 32 bits
    lib, one = _lib(), ctypes.c_void_p(256)
    for dim in (2 ** 31 - 1, 2 ** 31 - 255):
        dp = _abi.desc_pointer(_abi.QkNormDesc(1, dim, _abi.QK_BF16, _abi.QK_BF16, 1e-5, 0))
        assert lib.qk_layer_norm_backward_workspace_bytes(dp) == 0
        assert lib.qk_layer_norm_forward(dp, one, None, None, one, None, None) == _abi.QK_ERR_UNSUPPORTED
        assert lib.qk_layer_norm_backward(dp, one, None, one, one, one, one, one, one, 1 << 40, None) == _abi.QK_ERR_UNSUPPORTED


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    for call in (lambda: F.fused_linear(x, w), lambda: F.linear_backward(x, w, torch.zeros(2, 3)),
                 lambda: F.layer_norm(x), lambda: F.layer_norm_backward(x, None, torch.zeros(2, 2), x),
                 lambda: Linear(4, 3)(x), lambda: LayerNorm(4)(x)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_linear_arguments_that_are_refused():
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    gy = torch.zeros(2, 3)
    bad = [
        lambda: F.fused_linear(x, torch.zeros(3, 5)), lambda: F.fused_linear(x, torch.zeros(4)),
        lambda: F.fused_linear(torch.zeros(()), w), lambda: F.fused_linear(x, w.to(torch.bfloat16)),
        lambda: F.fused_linear(x, w, torch.zeros(4)), lambda: F.fused_linear(x, w, torch.zeros(3, dtype=torch.float64)),
        lambda: F.fused_linear(x, w, residual=torch.zeros(3)),  # no broadcasting
        lambda: F.fused_linear(x, w, residual=torch.zeros(2, 3, dtype=torch.bfloat16)),
        lambda: F.fused_linear(x, w, activation="selu"), lambda: F.fused_linear(x, w, activation=3),
        lambda: F.linear_backward(x, w, torch.zeros(2, 4)), lambda: F.linear_backward(x, w, gy, want=("y",)),
        lambda: F.linear_backward(x, w, gy, activation="silu"),
        lambda: F.linear_backward(x, w, gy, activation="silu", tape=gy.half()),
        lambda: F.linear_backward(x, w, gy.to(torch.bfloat16)),
        lambda: F.fused_linear(torch.empty(1, device="meta").expand(1 << 31, 1), torch.empty(2, 1, device="meta")),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was not refused")
    for dt in (torch.float64, torch.float16, torch.int32):
        with pytest.raises(TypeError):
            F.fused_linear(x.to(dt), w.to(dt))


def test_norm_arguments_that_are_refused():
    x = torch.zeros(2, 4)
    s = torch.zeros(2, 2)
    bad = [
        lambda: F.layer_norm(torch.zeros(2, 0)), lambda: F.layer_norm(torch.zeros(())),
        lambda: F.layer_norm(x, torch.zeros(3)), lambda: F.layer_norm(x, torch.zeros(1, 4)),
        lambda: F.layer_norm(x, torch.zeros(4), torch.zeros(4, dtype=torch.bfloat16)),
        lambda: F.layer_norm(x, eps=-1.0), lambda: F.layer_norm(x, eps=float("nan")),
        lambda: F.layer_norm(x, eps=float("inf")),
        lambda: F.layer_norm_backward(x, None, s, torch.zeros(2, 3)),
        lambda: F.layer_norm_backward(x, None, torch.zeros(2), x), lambda: F.layer_norm_backward(x, None, s.double(), x),
        lambda: F.layer_norm_backward(x, None, s, x, want=("gamma",)),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k} was not refused")
    with pytest.raises(TypeError):
        F.layer_norm(x.half())
    with pytest.raises(TypeError):
        F.layer_norm(x, torch.zeros(4).half())
    with pytest.raises(TypeError):
        F.layer_norm_backward(x, None, s, x, param_dtype=torch.float16)


def test_modules_keep_torchs_parameters_and_initialisation():
    for ours, theirs in ((Linear, nn.Linear), ):
        torch.manual_seed(3)
        a = ours(5, 7)
        torch.manual_seed(3)
        b = theirs(5, 7)
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
        assert list(a.state_dict()) == list(b.state_dict())
    assert list(LayerNorm(6).state_dict()) == list(nn.LayerNorm(6).state_dict())
    assert LayerNorm(6, bias=False).bias is None and LayerNorm(6, elementwise_affine=False).weight is None
    with pytest.raises(NotImplementedError):
        LayerNorm((3, 4))
    with pytest.raises(ValueError):
        Linear(3, 4, activation="nope")
    assert "activation=silu" in repr(Linear(3, 4, activation="silu"))


def test_block_and_head_keep_the_names_of_what_they_replace():
    block = HQKANBlock(24, 6, device="cpu")
    fused = qkan_b200.FusedHQKAN(24, 6, device="cpu")
    missing = block.load_state_dict(fused.state_dict(), strict=False)
    assert sorted(missing.missing_keys) == ["norm.bias", "norm.weight"] and not missing.unexpected_keys
    kw = dict(width=[4, 3, 6, 2], reps=1, seed=11, is_map=True, hidden=6)
    plain, head = QKAN(**kw), QKAN(**kw, fused_head=True)
    a, b = plain.state_dict(), head.state_dict()
    assert list(a) == list(b) and all(torch.equal(a[k], b[k]) for k in a)
    assert isinstance(head.layers[2], Linear) and head.layers[2].activation == "silu"
    bigger = head.refine(2)
    assert bigger.fused_head and torch.equal(bigger.layers[2].weight, head.layers[2].weight)
