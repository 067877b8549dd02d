"""What the dense operators' float64 comparisons with element bounds cannot see: values that are not finite, roundings that
show in the mean square only, and which kernel a problem takes."""
import math

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
    """gz in 16 bits or more and a tape in half: the first is off by 2^-16 at most, the second moves gz by 2^-11 |z| times
    the second derivative, some 2^-12 of gy in the mean. Beside the gradient's own rounding, 2^-9 and 2^-10 in the mean
    square, they add a few hundredths; gz rounded to bfloat16 would make it 1.41."""
    x, w, gy, _ = _tape_problem(*size, seed=40)
    w = (w * size[1] ** -0.5).bfloat16()  # arguments of order one, where the slope is no constant
    _, tape = F.linear_forward(x, w, activation=act, return_tape=True)
    want = _gradients64(x, w, gy, x.double() @ w.double().t(), act)
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


# ---------------------------------------------------------------- layer norm of rows far from zero
DTYPES = [torch.float32, torch.bfloat16]
STEP = 2.0 ** -24
HALF = 2.0 ** -8  # of a bfloat16 result


def _norm_gradients64(xh, rstd, w, gy):
    """Gradients and the sizes of what they are made of, from the exact normalised rows."""
    gw = gy if w is None else gy * w
    m1, m2 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
    size = rstd * (gw.abs() + gw.abs().mean(-1, keepdim=True) + xh.abs() * (gw * xh).abs().mean(-1, keepdim=True))
    return rstd * (gw - m1 - xh * m2), size


def _close(got, want, bound, what):
    d = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all() and float(d.max()) <= 0, f"{what}: {float(d.max()):.3e} beyond its bound"


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [2, 96, 768, 1000, 1024, 2052, 5000, 8191, 9000])
@pytest.mark.parametrize("value", [3.0, -1000.0, 3300.0, 1e4, 2.0 ** 120])
def test_layer_norm_of_constant_rows_is_its_bias(value, D, dtype):
    """The sum of a constant row is exact here (few bits), so its mean is the constant, and nothing is left of x - mean."""
    if value > 1e30 and D > 128:
        pytest.skip("the sum is beyond float32")
    M = 6
    x = torch.full((M, D), value, dtype=dtype, device="cuda")
    w, b, gy = (_randn(*s, seed=k, dtype=dtype) for k, s in enumerate(((D,), (D,), (M, D))))
    y, stats = F.layer_norm_forward(x, w, b)
    assert torch.equal(y, b.expand(M, D))
    assert torch.equal(stats[:, 0], x[:, 0].float())
    g = F.layer_norm_backward(x, w, stats, gy)
    assert not g["weight"].any()
    want, size = _norm_gradients64(torch.zeros(M, D, device="cuda").double(), 1e-5 ** -0.5, w.double(), gy.double())
    # sums of up to 64 additions in a row, a few operations around them
    _close(g["x"], want, 72 * STEP * size + (HALF * want.abs() if dtype == torch.bfloat16 else 0), "grad x")


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [2, 96, 768, 1000, 1024, 2052, 5000, 8190, 9000])
def test_layer_norm_far_from_zero_is_as_exact_as_near(D, dtype):
    """Whole numbers on both sides of a mean that is one: sums, mean and variance's sum are exact, so that what is left
    are the roundings of rstd (4 steps) and of two products. A variance as E[x^2] - mean^2, or x * rstd - mean * rstd, would be off
    by the mean's square or the mean itself instead."""
    M = 40
    mean = 192 if dtype == torch.bfloat16 else 1500  # bfloat16 holds whole numbers up to 256
    g = torch.Generator().manual_seed(D)
    k = torch.randint(1, 8, (M, D // 2), generator=g)
    x = torch.stack((mean + k, mean - k), -1).view(M, D).to(dtype).cuda()
    w, b, gy = (_randn(*s, seed=j, dtype=dtype) for j, s in enumerate(((D,), (D,), (M, D))))
    dev = x.double() - mean
    rstd = 1 / torch.sqrt((dev * dev).mean(-1, keepdim=True) + 1e-5)
    xh = dev * rstd
    half = dtype == torch.bfloat16
    y, stats = F.layer_norm_forward(x, w, b)
    want = xh * w.double() + b.double()
    _close(y, want, 8 * STEP * (xh * w.double()).abs() + 2 * STEP * want.abs() + (HALF * want.abs() if half else 0), "y")
    assert bool((stats[:, 0] == mean).all())
    got = F.layer_norm_backward(x, w, stats, gy)
    want, size = _norm_gradients64(xh, rstd, w.double(), gy.double())
    _close(got["x"], want, 80 * STEP * size + (HALF * want.abs() if half else 0), "grad x")
    want = (gy.double() * xh).sum(0)
    _close(got["weight"], want, (M + 8) * STEP * (gy.double() * xh).abs().sum(0) + (HALF * want.abs() if half else 0), "grad weight")


def test_bounds_of_the_far_rows_tell_a_naive_variance_and_zeros():
    """The rows above, computed the ways that they are to tell apart, in float32 by torch."""
    mean, D = 1500.0, 768
    k = torch.randint(1, 8, (40, D // 2), generator=torch.Generator().manual_seed(D))
    x = torch.stack((mean + k, mean - k), -1).view(40, D).float().cuda()
    dev = x.double() - mean
    rstd = 1 / torch.sqrt((dev * dev).mean(-1, keepdim=True) + 1e-5)
    xh = dev * rstd
    bound = 10 * STEP * xh.abs()
    naive = (x - mean) * torch.rsqrt((x * x).mean(-1, keepdim=True) - mean * mean + 1e-5)
    spread = x * rstd.float() - mean * rstd.float()
    for wrong in (naive, spread, torch.zeros_like(x)):
        assert float(((wrong.double() - xh).abs() - bound).max()) > 0
    _close((x - mean) * rstd.float(), xh, bound, "as the kernels take it")


def test_status_of_a_device_and_in_training():
    from qkan_b200 import QKAN

    for device in (None, "cuda", "cuda:0", torch.device("cuda"), 0):
        F.dense_status(device)
    model = QKAN([6, 5, 3], is_map=True, hidden=8, fused_head=True, seed=1).to("cuda")
    data = {k: _randn(40, 6 if k.endswith("input") else 3, seed=j) for j, k in
            enumerate(("train_input", "train_label", "test_input", "test_label"))}
    out = model.train_(data, steps=3, log=2, verbose=False)
    assert len(out["train_loss"]) == 3


@pytest.mark.parametrize("M,D", [(600, 100), (600, 768), (600, 1037), (600, 4096), (600, 9000), (8192, 9000), (70000, 8192), (1 << 20, 100)])
def test_layer_norm_parameter_gradients_are_added_without_further_rounding(M, D):
    """Some 300 partial sums of a few rows each. Added in order, K numbers carry sqrt(K / 6) steps of the root of their
    squares' sum: eight rows or groups at most make 1.2 (64 rows, as in a long batch, 3.3), the last rounding 0.3, and for
    the weight the roundings in xhat 1.5 at most; adding 300 of them in float32, 32 by 32, would bring 2.5 more, and 443 rows
    of a long batch 8.6. Above 8192 columns a thread adds rows / 64, in double."""
    x, w, gy = _randn(M, D), _randn(D, seed=1), _randn(M, D, seed=2)
    _, stats = F.layer_norm_forward(x, w)
    got = F.layer_norm_backward(x, w, stats, gy)
    xd, gyd = x.double(), gy.double()
    xc = xd - xd.mean(-1, keepdim=True)
    xh = xc / torch.sqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    long = 2.1 if M > 10000 else 0.0
    for name, terms, steps in (("bias", gyd, 1.3 + long), ("weight", gyd * xh, 2.4 + long)):
        off = (got[name].double() - terms.sum(0)) / terms.square().sum(0).sqrt()
        assert float(off.square().mean().sqrt()) <= steps * STEP, (name, float(off.square().mean().sqrt()) / STEP)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
def test_captures_that_fork_and_join(dtype):
    """The operators on two streams of one capture, whose kernels each wait for what is before them on their own stream, and
    for the other stream where it was told to."""
    sizes = ((1, 64, 72), (8, 100, 30), (300, 256, 256), (700, 264, 520), (2100, 1032, 2056))
    problems = [(_randn(M, K, dtype=dtype), _randn(N, K, dtype=dtype, scale=K ** -0.5), _randn(K, dtype=dtype)) for M, K, N in sizes]
    side = torch.cuda.Stream()

    def step(fork):
        out = []
        for x, w, n in problems:
            here = torch.cuda.current_stream()
            other = side if fork else here
            other.wait_stream(here)
            with torch.cuda.stream(other):
                a, stats = F.layer_norm_forward(x, n)
                g = F.layer_norm_backward(x, n, stats, x)["x"]
            z, tape = F.linear_forward(x, w, activation="silu", return_tape=True)
            here.wait_stream(other)
            y = F.linear_forward(a, w, residual=z)
            out += [y, *F.linear_backward(g, w, y, tape=tape, activation="silu").values()]
        return out

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = step(True)
    for seed in (1, 2):
        for x, *_ in problems:
            x.copy_(_randn(*x.shape, seed=seed, dtype=dtype))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(replayed, step(False)):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


@pytest.mark.parametrize("size", [(5, 64, 512), (16, 264, 4096), (40, 72, 520), (1000, 264, 16), (1000, 264, 520), (20000, 24, 16),
                                  (20000, 24, 1001), (200000, 16, 16)], ids=lambda s: "x".join(map(str, s)))
def test_float32_grad_bias_adds_few_numbers_in_order(size):
    """A thread adds rows / (592 slabs x the threads beside it) values in float32, 16 in flight at most; all sums of those are in
    double, each rounded once: sqrt(K / 6) steps for K of them, and 0.5."""
    M, K, N = size
    x, w, gy = _randn(M, K), _randn(N, K), _randn(M, N)
    got = F.linear_backward(x, w, gy, want=("bias",))["bias"]
    assert torch.equal(F.linear_backward(x, w, gy)["bias"], got)
    groups = max(N, 64) / 8
    beside = 256 / min(32, 2 ** math.ceil(math.log2(groups)))
    rows = M / beside / max(1, min(592 / math.ceil(groups / 32), M / (4 * beside)))
    off = (got.double() - gy.double().sum(0)) / gy.double().square().sum(0).sqrt()
    steps = math.sqrt(max(rows, 4) / 6) + 0.5
    assert float(off.square().mean().sqrt()) <= steps * STEP, (float(off.square().mean().sqrt()) / STEP, steps)
