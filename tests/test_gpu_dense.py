"""The dense operators on the GPU: layer norm, the linear map with its epilogue, and the blocks that use them."""
import pytest
import torch

from qkan_b200 import QKAN, HQKANBlock, LayerNorm, Linear
from qkan_b200 import functional as F
from tests.dense_util import ACTS, linear64, linear64_grads, norm64, norm64_grads, within

pytestmark = pytest.mark.gpu

@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    F.dense_status()


DTYPES = [torch.float32, torch.bfloat16]


def _randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * sum((k + 1) * n for k, n in enumerate(shape)))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def _problem(M, K, N, dtype, seed=0):
    return (_randn(M, K, seed=seed, dtype=dtype), _randn(N, K, seed=seed + 1, dtype=dtype, scale=max(K, 1) ** -0.5),
            _randn(N, seed=seed + 2, dtype=dtype), _randn(M, N, seed=seed + 3, dtype=dtype),
            _randn(M, N, seed=seed + 4, dtype=dtype))


# (rows, in, out): single elements, single tokens, few tokens, odd everything, widths that break 16-byte rows, the
# hybrid block's narrow projections, more than one tile each way, long sums that are cut into slices
SIZES = [(1, 1, 1), (1, 768, 10), (1, 10, 768), (1, 515, 1030), (2, 2048, 64), (3, 17, 5), (4, 4096, 33), (7, 264, 520),
         (8, 1000, 40), (9, 64, 128), (16, 130, 257), (17, 8, 8), (33, 64, 300), (48, 512, 256), (64, 784, 128),
         (100, 65, 127), (130, 10, 768), (129, 768, 10), (257, 100, 129), (300, 256, 256), (512, 520, 1000),
         (1025, 24, 72), (2000, 72, 40), (4100, 40, 24), (5000, 16, 16), (260, 1032, 136), (700, 333, 260),
         # partial sums whose float32 rows are whole 16-byte words and whose bfloat16 rows are not
         (300, 1000, 700)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_linear_forward_and_backward(size, dtype):
    M, K, N = size
    act = ACTS[(M + K + N) % len(ACTS)]
    x, w, b, r, gy = _problem(M, K, N, dtype)
    y, tape = F.linear_forward(x, w, b, activation=act, residual=r, return_tape=True)
    want, bound, z, zb = linear64(x, w, b, r, act)
    within(y, want, bound, f"y {act}")
    if tape is not None:
        within(tape, z, zb + (2.0 ** -11 * (z.abs() + zb) + 2.0 ** -24 if dtype == torch.bfloat16 else 0), "tape")
    g = F.linear_backward(x, w, gy, tape=tape, activation=act)
    for k, (v, e) in linear64_grads(x, w, b, gy, act).items():
        if act == "relu":  # where z is within its own error of the kink, either side is right
            continue
        within(g[k], v, e, f"grad {k} {act}")
    # without an epilogue
    within(F.linear_forward(x, w), *linear64(x, w)[:2], "plain product")
    g = F.linear_backward(x, w, gy)
    for k, (v, e) in linear64_grads(x, w, None, gy).items():
        within(g[k], v, e, f"plain grad {k}")


# one to four rows per thread, 16 and 32 columns, a depth that ends inside a chunk, cut or not, rows of whole words and others
@pytest.mark.parametrize("size", [(17, 1, 1), (24, 100, 32), (100, 3445, 10), (400, 4100, 17), (2000, 768, 31), (5000, 1030, 20),
                                  (700, 5, 3), (40000, 36, 32), (20001, 33, 16), (513, 32, 16), (129, 4096, 32),
                                  # little of everything
                                  (19, 184, 186), (64, 64, 64), (100, 1000, 33), (24, 600, 1001), (512, 64, 512)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_few_outputs_in_float32(size, act):
    M, K, N = size
    x, w, b, r, _ = _problem(M, K, N, torch.float32, seed=40)
    want, bound, z, zb = linear64(x, w, b, r, act)
    y, tape = F.linear_forward(x, w, b, activation=act, residual=r, return_tape=True)
    within(y, want, bound, "y")
    if tape is not None:
        within(tape, z, zb, "tape")
    # rows that do not start on a 16-byte boundary, and the same bits again
    odd = torch.empty(M * K + 1, device="cuda")[1:].view(M, K).copy_(x)
    within(F.linear_forward(odd, w), *linear64(x, w)[:2], "odd start")
    assert torch.equal(F.linear_forward(x, w, b, activation=act, residual=r), y)
    # what is not finite stays in its row and column
    x[M // 2, K // 2], w[N // 2, K // 3] = float("inf"), float("nan")
    got = F.linear_forward(x, w)
    there = torch.zeros(M, N, dtype=torch.bool, device="cuda")
    there[M // 2], there[:, N // 2] = True, True
    assert torch.equal(~torch.isfinite(got), there)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows", [1, 6, 150])
def test_linear_every_activation(act, dtype, rows):
    x, w, b, r, gy = _problem(rows, 96, 200, dtype, seed=5)
    w = w * 4
    if act == "relu":  # whole numbers: z is exact, and so is its sign
        x, w, b = x.round(), (4 * w).round(), b.round()
    for res in (None, r):
        y, tape = F.linear_forward(x, w, b, activation=act, residual=res, return_tape=True)
        within(y, *linear64(x, w, b, res, act)[:2], f"y {act}")
    g = F.linear_backward(x, w, gy, tape=tape, activation=act)
    for k, (v, e) in linear64_grads(x, w, b, gy, act).items():
        within(g[k], v, e, f"grad {k} {act}")


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows", [2, 140])
def test_linear_each_gradient_alone(dtype, rows):
    x, w, b, _, gy = _problem(rows, 72, 56, dtype, seed=9)
    _, tape = F.linear_forward(x, w, b, activation="silu", return_tape=True)
    every = F.linear_backward(x, w, gy, tape=tape, activation="silu")
    for k in ("x", "weight", "bias"):
        alone = F.linear_backward(x, w, gy, tape=tape, activation="silu", want=(k,))
        assert list(alone) == [k]
        assert torch.equal(alone[k], every[k]), k
    assert F.linear_backward(x, w, gy, want=()) == {}


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
def test_linear_empty_axes(dtype):
    for M, K, N in ((0, 8, 5), (6, 0, 5), (6, 8, 0), (0, 0, 0), (200, 0, 300)):
        x, w, b, r, gy = _problem(M, K, N, dtype)
        y, tape = F.linear_forward(x, w, b, activation="silu", residual=r, return_tape=True)
        within(y, *linear64(x, w, b, r, "silu")[:2], f"y {M, K, N}")
        g = F.linear_backward(x, w, gy, tape=tape, activation="silu")
        for k, (v, e) in linear64_grads(x, w, b, gy, "silu").items():
            within(g[k], v, e + 1e-30, f"{k} {M, K, N}")


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_linear_non_finite_values_stay_in_their_rows(dtype, rows):
    """An infinity or a NaN in one row of x reaches that row of y alone, and as float32 arithmetic would have it."""
    x, w, b, _, _ = _problem(rows, 200, 136, dtype, seed=3)
    x[0, 5] = float("inf")
    if rows > 2:
        x[1, 7] = float("nan")
        x[2, 3], x[2, 4] = float("inf"), float("-inf")
    y = F.linear_forward(x, w, b)
    want, bound, _, _ = linear64(x, w, b)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(y[inf].double(), want[inf])
    within(y[3:], want[3:], bound[3:], "other rows")


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows", [4, 200])
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e18])
def test_linear_values_of_any_scale(dtype, rows, scale):
    x, w, b, _, gy = _problem(rows, 120, 144, dtype, seed=4)
    x, b = x * scale, b * scale
    within(F.linear_forward(x, w, b), *linear64(x, w, b)[:2], "y")
    g = F.linear_backward(x, w, gy * scale)
    for k, (v, e) in linear64_grads(x, w, b, gy * scale).items():
        within(g[k], v, e + 1e-44, k)  # 1e-44: products below float32's smallest number


def test_float32_extremes_survive_the_split():
    """Values next to float32's largest, whose upper part must not round to infinity, and subnormal ones."""
    big = torch.finfo(torch.float32).max
    for rows in (2, 160):
        x = torch.zeros(rows, 64, device="cuda")
        x[:, 0], x[:, 1] = big, 1e-41
        w = torch.zeros(128, 64, device="cuda")
        w[:, 0], w[::2, 1] = 0.5, 1.0
        y = F.linear_forward(x, w)
        want = x.double() @ w.double().t()
        within(y, want, 2.0 ** -22 * want.abs(), "y")
        tiny = F.linear_forward(x[:, 1:], w[:, 1:].contiguous())
        within(tiny, x[:, 1:].double() @ w[:, 1:].double().t(), torch.full_like(want, 1e-40), "subnormal")


def test_far_arguments_of_the_activation():
    """What half precision cannot hold: relu's tape keeps the sign of tiny values, and beyond the range every derivative
    has its limit. A NaN stays one (relu's derivative asks for z > 0, as torch's does, and is 0 there)."""
    z = torch.tensor([[1e-30], [-1e-30], [3e38], [-3e38], [0.0], [float("inf")], [float("-inf")], [float("nan")]],
                     dtype=torch.bfloat16, device="cuda")
    w = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda")
    limits = {"relu": (1, 0), "silu": (1, 0), "gelu": (1, 0), "gelu_tanh": (1, 0), "tanh": (0, 0), "sigmoid": (0, 0)}
    for x in (z[:2], z, z.repeat(40, 1), z.float(), z.float().repeat(40, 1)):
        for act, (up, down) in limits.items():
            _, tape = F.linear_forward(x, w.to(x.dtype), activation=act, return_tape=True)
            g = F.linear_backward(x, w.to(x.dtype), torch.ones_like(x), tape=tape, activation=act, want=("x",))["x"]
            g = g[:8, 0].tolist()
            if act == "relu":
                assert g[:2] == [1, 0], (act, g)
            if len(g) > 2:
                assert g[2:4] == [up, down] and g[5:7] == [up, down], (act, g)
                assert g[7] == 0 if act == "relu" else g[7] != g[7], (act, g)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
def test_linear_is_bitwise_repeatable_and_independent_of_its_surroundings(dtype):
    x, w, b, r, gy = _problem(515, 300, 200, dtype)
    y, tape = F.linear_forward(x, w, b, activation="gelu", residual=r, return_tape=True)
    g = F.linear_backward(x, w, gy, tape=tape, activation="gelu")
    for _ in range(3):
        junk = torch.full((1 << 20,), float("nan"), device="cuda")  # what freed scratch may hold
        del junk
        y2, tape2 = F.linear_forward(x, w, b, activation="gelu", residual=r, return_tape=True)
        g2 = F.linear_backward(x, w, gy, tape=tape2, activation="gelu")
        assert torch.equal(y, y2) and torch.equal(tape, tape2) and all(torch.equal(g[k], g2[k]) for k in g)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows", [3, 150])
def test_linear_views_offsets_and_transposes(dtype, rows):
    """Non-contiguous and misaligned inputs: every tensor starts one element into its storage, or is a transpose."""
    M, K, N = rows, 64, 80
    x, w, b, r, gy = _problem(M, K, N, dtype, seed=2)

    def shifted(t):
        s = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape)
        return s.copy_(t)

    want, bound, _, _ = linear64(x, w, b, r)
    for f in (shifted, lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        within(F.linear_forward(f(x), f(w), f(b), residual=f(r)), want, bound, "y")
        g = F.linear_backward(f(x), f(w), f(gy))
        for k, (v, e) in linear64_grads(x, w, b, gy).items():
            within(g[k], v, e, k)
    # leading axes, and a gradient that is an expanded scalar
    x3 = x.view(1, M, K).requires_grad_(True)
    F.fused_linear(x3, w, b).sum().backward()
    ones = torch.ones_like(gy)
    v, e = linear64_grads(x, w, b, ones)["x"]
    within(x3.grad[0], v, e, "grad of a sum")


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("act", ["none", "silu", "gelu"])
def test_fused_linear_autograd(dtype, act):
    x, w, b, r, gy = _problem(70, 96, 136, dtype, seed=6)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    y = F.fused_linear(*leaves[:3], activation=act, residual=leaves[3])
    assert y.requires_grad
    y.backward(gy)
    direct = linear64_grads(x, w, b, gy, act)
    for leaf, k in zip(leaves, ("x", "weight", "bias")):
        within(leaf.grad, *direct[k], k)
    assert torch.equal(leaves[3].grad, gy)
    # frozen inputs, no bias, no residual
    wl = w.clone().requires_grad_(True)
    F.fused_linear(x, wl, activation=act).backward(gy)
    within(wl.grad, *linear64_grads(x, w, None, gy, act)["weight"], "weight alone")
    rl = r.clone().requires_grad_(True)
    F.fused_linear(x, w, b, activation=act, residual=rl).backward(gy)
    assert torch.equal(rl.grad, gy)
    with torch.no_grad():
        assert not F.fused_linear(*leaves[:3], activation=act).requires_grad


def _difference(f, t, d, h=1e-6):
    """d/dh of f along d, by a central difference of float64 values (off by about h^2 and 1e-16 / h)."""
    t, d = t.double(), d.double()
    return float((f(t + h * d) - f(t - h * d)) / (2 * h))


def test_gradients_against_differences():
    x, w, b, r, gy = _problem(40, 48, 56, torch.float32, seed=8)
    for act in ACTS:
        if act == "relu":
            continue
        _, tape = F.linear_forward(x, w, b, activation=act, return_tape=True)
        g = F.linear_backward(x, w, gy, tape=tape, activation=act)
        loss = lambda x_, w_, b_: (linear64(x_, w_, b_, None, act)[0] * gy.double()).sum()  # noqa: E731
        for k, t, f in (("x", x, lambda t: loss(t, w, b)), ("weight", w, lambda t: loss(x, t, b)),
                        ("bias", b, lambda t: loss(x, w, t))):
            d = _randn(*t.shape, seed=77)
            slack = float((linear64_grads(x, w, b, gy, act)[k][1] * d.abs().double()).sum())
            assert abs(float((g[k].double() * d.double()).sum()) - _difference(f, t, d)) <= slack + 1e-6, (act, k)
    x, wn, bn, gy = _randn(30, 72, seed=1), _randn(72, seed=2), _randn(72, seed=3), _randn(30, 72, seed=4)
    _, stats = F.layer_norm_forward(x, wn, bn)
    g = F.layer_norm_backward(x, wn, stats, gy)
    loss = lambda x_, w_, b_: (norm64(x_, w_, b_)[0] * gy.double()).sum()  # noqa: E731
    for k, t, f in (("x", x, lambda t: loss(t, wn, bn)), ("weight", wn, lambda t: loss(x, t, bn)),
                    ("bias", bn, lambda t: loss(x, wn, t))):
        d = _randn(*t.shape, seed=78)
        slack = float((norm64_grads(x, wn, gy)[k][1] * d.abs().double()).sum())
        assert abs(float((g[k].double() * d.double()).sum()) - _difference(f, t, d)) <= slack + 1e-6, k


# ---------------------------------------------------------------- layer norm
# every number of threads per row, with and without 16-byte rows, and rows too wide for registers
NORM_SIZES = [(1, 1), (1, 768), (3, 5), (7, 31), (5, 512), (300, 512), (9, 513), (4, 768), (2000, 768), (33, 1037),
              (64, 1024), (6, 2048), (5, 2052), (3, 4096), (400, 4096), (2, 4100), (3, 8192), (2, 8184), (150, 8191),
              (2, 8200), (70, 10000), (1, 33333)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", NORM_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_forward_and_backward(size, dtype):
    M, D = size
    pdt = torch.float32 if (M + D) % 2 else dtype
    x = _randn(M, D, dtype=torch.float32) * (0.3 + _randn(M, 1, seed=5).abs()) + 2 * _randn(M, 1, seed=6)
    x, gy = x.to(dtype), _randn(M, D, seed=9, dtype=dtype)
    w, b = (1 + 0.3 * _randn(D, seed=7)).to(pdt), _randn(D, seed=8, dtype=pdt)
    for ww, bb in ((w, b), (w, None), (None, b), (None, None)):
        y, stats = F.layer_norm_forward(x, ww, bb)
        within(y, *norm64(x, ww, bb)[:2], "y")
        g = F.layer_norm_backward(x, ww, stats, gy, param_dtype=pdt)
        for k, (v, e) in norm64_grads(x, ww, gy, half_params=pdt == torch.bfloat16).items():
            within(g[k], v, e, f"grad {k}")


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [96, 768, 1000, 9000])
def test_layer_norm_hard_rows(dtype, D):
    """A constant row, a row far from zero, rows with infinity and NaN: each keeps to itself."""
    x = _randn(6, D, dtype=torch.float32)
    x[1] = 3.0
    x[2] = x[2] + 1e4
    x[3, 0] = float("inf")
    x[4, 1] = float("nan")
    x = x.to(dtype)
    w, b = _randn(D, seed=1, dtype=dtype), _randn(D, seed=2, dtype=dtype)
    y, stats = F.layer_norm_forward(x, w, b)
    want, bound, *_ = norm64(x, w, b)
    fine = [0, 1, 2, 5]
    # eps bounds the constant row: its deviations are rounding errors of the mean, times 1/sqrt(eps)
    within(y[fine], want[fine], bound[fine], "y")
    assert torch.isnan(y[4]).all() and torch.isnan(y[3]).all()
    gy = _randn(6, D, seed=3, dtype=dtype)
    g = F.layer_norm_backward(x, w, stats, gy, want=("x",))["x"]
    v, e = norm64_grads(x, w, gy)["x"]
    within(g[fine], v[fine], e[fine], "grad x")


def test_layer_norm_empty_batch_and_each_gradient_alone():
    for dtype in DTYPES:
        x = torch.empty(0, 40, dtype=dtype, device="cuda")
        w = torch.ones(40, dtype=dtype, device="cuda")
        y, stats = F.layer_norm_forward(x, w, w)
        g = F.layer_norm_backward(x, w, stats, y)
        assert y.shape == (0, 40) and g["x"].shape == (0, 40) and not g["weight"].any() and not g["bias"].any()
        for D in (40, 9001):
            x, w, gy = _randn(20, D, dtype=dtype), _randn(D, seed=1, dtype=dtype), _randn(20, D, seed=2, dtype=dtype)
            _, stats = F.layer_norm_forward(x, w, None)
            every = F.layer_norm_backward(x, w, stats, gy)
            for k in ("x", "weight", "bias"):
                assert torch.equal(F.layer_norm_backward(x, w, stats, gy, want=(k,))[k], every[k])
            again = F.layer_norm_backward(x, w, stats, gy)
            assert all(torch.equal(again[k], every[k]) for k in every)


@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
def test_layer_norm_autograd_views_and_offsets(dtype):
    x, w, b = _randn(12, 64, dtype=dtype), _randn(64, seed=1, dtype=dtype), _randn(64, seed=2, dtype=dtype)
    gy = _randn(12, 64, seed=3, dtype=dtype)
    leaves = [x.view(3, 4, 64).clone().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
    y = F.layer_norm(*leaves)
    y.backward(gy.view(3, 4, 64))
    within(y.view(12, 64), *norm64(x, w, b)[:2], "y")
    want = norm64_grads(x, w, gy, half_params=dtype == torch.bfloat16)
    for leaf, k in zip(leaves, ("x", "weight", "bias")):
        within(leaf.grad.view_as(want[k][0]), *want[k], k)
    s = torch.empty(12 * 64 + 1, dtype=dtype, device="cuda")[1:].view(12, 64).copy_(x)
    within(F.layer_norm(s, w, b), *norm64(x, w, b)[:2], "offset")
    within(F.layer_norm(x.t().contiguous().t(), w, b), *norm64(x, w, b)[:2], "transposed")
    bl = b.float().requires_grad_(True)  # a bias alone, of another type than x
    F.layer_norm(x, None, bl).backward(gy)
    assert bl.grad.dtype == torch.float32
    within(bl.grad, *norm64_grads(x, None, gy)["bias"], "bias alone")


# ---------------------------------------------------------------- far offsets
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16"])
@pytest.mark.parametrize("M,D", [(5, 100), (3, 9001)])
def test_layer_norm_statistics_of_any_view(dtype, M, D):
    # the statistics of a row lie on a 4-byte boundary here, or apart
    x, gy = _randn(M, D, seed=31, dtype=dtype), _randn(M, D, seed=32, dtype=dtype)
    w = _randn(D, seed=33, dtype=dtype)
    _, stats = F.layer_norm_forward(x, w)
    want = F.layer_norm_backward(x, w, stats, gy)
    shifted = torch.empty(2 * M + 1, device="cuda")[1:].view(M, 2).copy_(stats)
    apart = torch.empty(2, M, device="cuda").t().copy_(stats)
    assert shifted.data_ptr() % 8 == 4 and not apart.is_contiguous()
    for view in (shifted, apart):
        got = F.layer_norm_backward(x, w, view, gy)
        for name in want:
            assert torch.equal(got[name], want[name])


@pytest.mark.parametrize("rows", [1, 40])
def test_views_whose_sign_is_still_to_be_turned(rows):
    x = torch.view_as_complex(_randn(rows, 24, 2, seed=34)).conj().imag
    w = torch.view_as_complex(_randn(16, 24, 2, seed=35)).conj().imag
    assert x.is_neg() and w.is_neg()
    plain_x, plain_w = x.resolve_neg().contiguous(), w.resolve_neg().contiguous()
    assert torch.equal(F.fused_linear(x, w), F.fused_linear(plain_x, plain_w))
    assert torch.equal(F.layer_norm(x), F.layer_norm(plain_x))


def test_rows_beyond_32_bit_offsets():
    """More than 2^31 elements: rows at both ends of the tensors are as the same rows by themselves."""
    M, D = (1 << 18) + 24, 8192 + 8
    assert M * D > 1 << 31
    x = torch.empty(M, D, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    some = torch.tensor([0, 1, M // 2, M - 2, M - 1], device="cuda")
    w = _randn(D, seed=2)
    y, stats = F.layer_norm_forward(x, w)
    ys, ss = F.layer_norm_forward(x[some], w)
    assert torch.equal(y[some], ys) and torch.equal(stats[some], ss)
    g = F.layer_norm_backward(x, w, stats, y, want=("x",))["x"]
    assert torch.equal(g[some], F.layer_norm_backward(x[some], w, ss, ys, want=("x",))["x"])
    del g, y
    # a narrow input and a wide output, an odd output, and the gradients of the former
    for N in (D, D + 1):
        xs, wn = x[:, :16].contiguous(), _randn(N, 16, seed=3, dtype=torch.bfloat16)
        y = F.linear_forward(xs, wn)
        within(y[some], *linear64(xs[some], wn)[:2], f"y {N}")
        if N == D:
            gx = F.linear_backward(xs, wn, x, want=("x",))["x"]
            v, e = linear64_grads(xs[some], wn, None, x[some])["x"]
            within(gx[some], v, e, "grad x")
        del y


# ---------------------------------------------------------------- streams, graphs, modules
def test_operators_on_another_stream_and_two_streams_at_once():
    x, w, b, r, gy = _problem(600, 320, 264, torch.bfloat16)
    want = F.linear_forward(x, w, b, residual=r)
    ref = F.linear_backward(x, w, gy)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append((F.linear_forward(x, w, b, residual=r), F.linear_backward(x, w, gy)))
    torch.cuda.synchronize()
    for y, g in outs:
        assert torch.equal(y, want) and all(torch.equal(g[k], ref[k]) for k in ref)


@pytest.mark.parametrize("rows", [1, 5, 300])
def test_operators_in_a_captured_graph(rows):
    """Two graphs of the same step, replayed side by side on two streams as well: each has scratch of its own."""
    x, w, b, r, gy = _problem(rows, 264, 520, torch.bfloat16)
    nw = _randn(264, seed=11, dtype=torch.bfloat16)

    def step():
        n, stats = F.layer_norm_forward(x, nw, None)
        y, tape = F.linear_forward(n, w, b, activation="silu", residual=r, return_tape=True)
        g = F.linear_backward(n, w, gy, tape=tape, activation="silu")
        return [y, *g.values(), *F.layer_norm_backward(x, nw, stats, g["x"]).values()]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, each with scratch of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in (1, 2):
        x.copy_(_randn(rows, 264, seed=seed, dtype=torch.bfloat16))
        torch.cuda.synchronize()
        for graph, _ in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_block_matches_its_parts_and_trains_captured():
    from qkan_b200.graph import make_graphed_inference, make_graphed_train_step

    torch.manual_seed(0)
    for p_dtype, c_dtype in ((torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)):
        block = HQKANBlock(48, 10, p_dtype=p_dtype, c_dtype=c_dtype)
        x = _randn(4, 16, 48, dtype=p_dtype)
        y = block(x)
        n = torch.nn.functional.layer_norm(x.float(), (48,), block.norm.weight.float(), block.norm.bias.float(), 1e-5).to(p_dtype)
        h = torch.nn.functional.linear(n.float(), block.down.weight.float(), block.down.bias.float()).to(p_dtype)
        h = block.qkan(h.view(-1, 10)).view(4, 16, 10)
        want = x.float() + torch.nn.functional.linear(h.float(), block.up.weight.float(), block.up.bias.float())
        tol = 2e-2 if p_dtype == torch.bfloat16 else 1e-5  # the composed block's bounds, as in tests/util.py
        assert float((y.float() - want).abs().max()) <= tol * float(want.abs().max())
        target = _randn(4, 16, 48, seed=1, dtype=p_dtype)
        loss_fn = lambda o, t: (o.float() - t.float()).square().mean()  # noqa: E731
        loss = loss_fn(block(x), target)
        loss.backward()
        eager = {k: p.grad.clone() for k, p in block.named_parameters() if p.grad is not None}
        assert {"norm.weight", "norm.bias", "down.weight", "up.weight", "up.bias", "qkan.layers.0.theta"} <= set(eager)
        step = make_graphed_train_step(block, x, target, loss_fn, torch.optim.SGD(block.parameters(), lr=0.0))
        step(x, target)
        torch.cuda.synchronize()
        for k, p in block.named_parameters():
            if k in eager:
                assert torch.equal(p.grad, eager[k]), k
        infer = make_graphed_inference(block, x[:1, :1])
        one = infer(x[2:3, 3:4])
        with torch.no_grad():
            assert torch.equal(one, block(x[2:3, 3:4]))


def test_head_on_the_package_kernels_matches_the_library_head():
    kw = dict(width=[6, 5, 12, 3], reps=2, seed=4, is_map=True, hidden=12, preact_trainable=True)
    a, b = QKAN(**kw).to("cuda"), QKAN(**kw, fused_head=True).to("cuda")
    x = torch.rand(50, 6, device="cuda") * 2 - 1
    ya, yb = a(x), b(x)
    assert float((ya - yb).abs().max()) <= 1e-5 * float(ya.abs().max())
    ya.square().mean().backward()
    yb.square().mean().backward()
    for (k, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        if p.grad is not None:
            assert float((p.grad - q.grad).abs().max()) <= 1e-5 * float(p.grad.abs().max()) + 1e-7, k


def test_modules_in_eval_and_training():
    lin, norm = Linear(64, 40, activation="gelu", device="cuda"), LayerNorm(64, device="cuda")
    x = _randn(5, 64)
    y = lin(norm(x))
    y.sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in [*lin.parameters(), *norm.parameters()])
    with torch.no_grad():
        assert torch.equal(lin(norm(x)), y)
    with pytest.raises(ValueError):
        norm(_randn(5, 63))


def test_captured_backward_while_an_eager_graph_of_the_same_leaves_lives():
    """make_graphed_train_step differentiates aliases of the parameters, so an eager graph that is still alive does not
    tie the capture to its stream."""
    from qkan_b200.graph import make_graphed_train_step

    torch.manual_seed(0)
    model = torch.nn.Sequential(LayerNorm(40, device="cuda"), Linear(40, 72, activation="silu", device="cuda"),
                                Linear(72, 24, device="cuda"))
    x, target = _randn(150, 40), _randn(150, 24, seed=1)
    loss_fn = torch.nn.functional.mse_loss
    alive = loss_fn(model(x), target)
    alive.backward(retain_graph=True)
    eager = [p.grad.clone() for p in model.parameters()]
    step = make_graphed_train_step(model, x, target, loss_fn, torch.optim.SGD(model.parameters(), lr=0.0))
    step(x, target)
    torch.cuda.synchronize()
    assert all(torch.equal(p.grad, g) for p, g in zip(model.parameters(), eager))
    assert alive.requires_grad


def test_operators_from_two_threads():
    """Plans and error texts are kept per thread; calls from several at once do not meet."""
    import threading

    cases = [_problem(30 + 7 * k, 40 + 8 * k, 24 + 5 * k, DTYPES[k % 2], seed=k) for k in range(6)]
    failures = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    x, w, b, r, gy = cases[k]
                    y = F.linear_forward(x, w, b, residual=r)
                    g = F.linear_backward(x, w, gy)
                within(y, *linear64(x, w, b, r)[:2], "y")
                for n, (v, e) in linear64_grads(x, w, b, gy).items():
                    within(g[n], v, e, n)
        except Exception as exc:  # seen in the main thread
            failures.append(exc)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


def test_operators_on_a_second_device():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    x, w, b, r, gy = (t.to("cuda:1") for t in _problem(300, 72, 80, torch.float32))
    assert torch.cuda.current_device() == 0
    within(F.linear_forward(x, w, b, residual=r), *linear64(x, w, b, r)[:2], "y")
    with pytest.raises(ValueError):
        F.linear_forward(x, w.to("cuda:0"))
