"""What the dense operators' float64 comparisons with element bounds cannot see: values that are not finite, roundings that
show in the mean square only, and which kernel a problem takes."""
import pytest
import torch

from qkan_b200 import functional as F
from tests.dense_util import act64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    F.dense_status()


def _randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * sum((k + 1) * n for k, n in enumerate(shape)))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def _same_non_finite(got, want, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), f"{what}: other infinities"


# ---------------------------------------------------------------- gz = gy act'(z) of a bfloat16 backward
def _tape_problem(M, K, N, seed=0):
    """No zero in x, W or gy, so that none meets an infinity by accident."""
    x, w, gy = (_randn(*s, seed=seed + k, dtype=torch.bfloat16) for k, s in enumerate(((M, K), (N, K), (M, N))))
    tape = _randn(M, N, seed=seed + 3).half()
    for t in (x, w, gy):
        t[t == 0] = 1
    return x, w, gy, tape


def _gradients64(x, w, gy, tape, act):
    gz = gy.double() * act64(tape.double(), act)[1]
    return {"x": gz @ w.double(), "weight": gz.t() @ x.double(), "bias": gz.sum(0)}


@pytest.mark.parametrize("act", ["silu", "tanh", "sigmoid"])
@pytest.mark.parametrize("size", [(64, 72, 56), (40, 33, 51), (800, 72, 400), (3, 72, 56)], ids=lambda s: "x".join(map(str, s)))
def test_infinities_reach_the_gradients_as_infinities(size, act):
    """One infinity in x or W against gz, whose own parts must neither cancel it nor miss it."""
    M, K, N = size
    x, w, gy, tape = _tape_problem(*size)
    gy[:, :8] = gy[:, :8].sign() * 0.5  # with a slope of 1/4 (sigmoid) or 1/2 (silu) at 0: gz is a bfloat16 as it is
    tape[:, :8] = 0
    x[M // 2, 5], x[0, 7] = float("inf"), float("-inf")
    w[3, 9], w[N - 1, 0] = float("-inf"), float("inf")
    got = F.linear_backward(x, w, gy, tape=tape, activation=act)
    for k, v in _gradients64(x, w, gy, tape, act).items():
        _same_non_finite(got[k], v, f"grad {k}")


@pytest.mark.parametrize("size", [(64, 72, 56), (800, 72, 400), (3, 72, 56)], ids=lambda s: "x".join(map(str, s)))
def test_infinite_and_nan_gradients_stay_in_their_rows(size):
    M, K, N = size
    x, w, gy, tape = _tape_problem(*size, seed=20)
    gy[1, 4], gy[2, 6] = float("inf"), float("nan")
    x[1, 3], w[4, 2] = float("inf"), float("-inf")  # and where they meet an infinity
    got = F.linear_backward(x, w, gy, tape=tape, activation="silu")
    for k, v in _gradients64(x, w, gy, tape, "silu").items():
        _same_non_finite(got[k], v, f"grad {k}")
