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


def _rounding_ratio(got, want):
    """Root mean square error over that of rounding the exact values to bfloat16, which no kernel can be without."""
    unit = (want.bfloat16().double() - want).square().mean().sqrt()
    return float((got.double() - want).square().mean().sqrt() / unit)


# few rows, up to and above 2^18 values of gz, odd widths, a long batch, more units of work than SMs
@pytest.mark.parametrize("size", [(4, 512, 600), (64, 72, 56), (520, 264, 512), (800, 72, 400), (1501, 517, 333), (20000, 40, 24),
                                  (2100, 1032, 2056)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
def test_bfloat16_gradients_carry_one_rounding(size, act):
    """gz in 15 bits or more and a tape in half: the first is off by 2^-15 at most, the second moves gz by 2^-11 |z| times
    the second derivative, some 2^-12 of gy in the mean. Beside the gradient's own rounding, 2^-9 and 2^-10 in the mean
    square, they add a few hundredths; gz rounded to bfloat16 would make it 1.41."""
    x, w, gy, _ = _tape_problem(*size, seed=40)
    _, tape = F.linear_forward(x, w, activation=act, return_tape=True)
    tape = torch.randn_like(tape)  # arguments of order one, where the slope is no constant
    want = _gradients64(x, w, gy, tape, act)
    got = F.linear_backward(x, w, gy, tape=tape, activation=act)
    for k, v in want.items():
        assert _rounding_ratio(got[k], v) <= 1.05, k
    # rounded once on request, by each entry point
    fast = F.linear_backward(x, w, gy, tape=tape, activation=act, round_grads=True)
    assert torch.equal(fast["bias"], got["bias"])
    for k in ("x", "weight"):
        assert _rounding_ratio(fast[k], want[k]) <= 1.5, k
    if size[0] > 4:  # few rows have gz in float32 whatever is asked for
        assert not torch.equal(fast["x"], got["x"]) and not torch.equal(fast["weight"], got["weight"])


def test_rounding_of_the_gradients_is_the_callers_choice():
    from qkan_b200 import Linear

    x, w, gy, _ = _tape_problem(200, 96, 136, seed=60)
    grads = {}
    for round_grads in (False, True):
        lin = Linear(96, 136, bias=False, device="cuda", dtype=torch.bfloat16, activation="silu", round_grads=round_grads)
        with torch.no_grad():
            lin.weight.copy_(w)
        lin(x).backward(gy)
        _, tape = F.linear_forward(x, w, activation="silu", return_tape=True)
        grads[round_grads] = lin.weight.grad
        want = F.linear_backward(x, w, gy, tape=tape, activation="silu", round_grads=round_grads)["weight"]
        assert torch.equal(lin.weight.grad, want)
    assert not torch.equal(grads[False], grads[True])
    # no activation: gz is grad_y itself, float32: nothing is rounded
    for dtype, act in ((torch.bfloat16, "none"), (torch.float32, "silu")):
        a, b, g = x.to(dtype), w.to(dtype), gy.to(dtype)
        _, tape = F.linear_forward(a, b, activation=act, return_tape=True)
        plain, fast = (F.linear_backward(a, b, g, tape=tape, activation=act, round_grads=r) for r in (False, True))
        assert all(torch.equal(plain[k], fast[k]) for k in plain)
