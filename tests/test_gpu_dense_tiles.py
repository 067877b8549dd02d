"""Every tile shape of the linear map's tensor-core products, with CTAs that walk several units of work, and the float32
split with values of every kind. Each test says which plan its sizes take, so that another choice of plans cannot empty it."""
import ctypes
import math

import pytest
import torch

from qkan_b200 import _abi
from qkan_b200 import functional as F
from tests.dense_util import ACTS, linear64, linear64_grads, norm64, norm64_grads, within

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
SMS = 148
STEP = 2.0 ** -24


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    F.dense_status()


def _randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed + 7919 * sum((k + 1) * n for k, n in enumerate(shape)))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _problem(M, K, N, dtype, seed=0):
    return (_randn(M, K, seed=seed, dtype=dtype), _randn(N, K, seed=seed + 1, dtype=dtype, scale=K ** -0.5),
            _randn(N, seed=seed + 2, dtype=dtype), _randn(M, N, seed=seed + 3, dtype=dtype),
            _randn(M, N, seed=seed + 4, dtype=dtype))


def plan_of(product, M, K, N, dtype, act="none", tensor=True):
    """The plan of product 0 (y), 1 (grad_weight) or 2 (grad_x); `tensor`: which has to be one of the tensor cores."""
    desc = _abi.QkLinearDesc(M, K, N, _abi.QK_BF16 if dtype == BF16 else _abi.QK_F32, _abi.ACTIVATION_CODES[act], 0)
    plan = _abi.QkLinearPlan()
    assert _abi.load().qk_linear_plan(_abi.desc_pointer(desc), product, ctypes.byref(plan)) == _abi.QK_OK
    assert not tensor or plan.path == _abi.QK_LINEAR_TENSOR, (product, M, K, N)
    return plan


def kind_of(product, plan, act):
    """The kernel's kind: with activation and tape, with the sums of gz, or plain."""
    if product == 1 and plan.sums_bias:
        return "sums"
    return "full" if product == 0 and act != "none" and plan.slices == 1 else "plain"


def rms_bound(x, w):
    """What float32 products of x (.., K) and w (N, K) may be off in the mean square, per element. A sum of K products taken in
    order carries sqrt(K / 6) steps of its own size sqrt(sum x^2 w^2) on average; the tensor core cuts off where it adds 16
    products at a time, eight times between two drains, which is 4 steps at most, as are the three-part products' dropped and
    small terms."""
    return STEP * (math.sqrt(x.shape[-1] / 6) + 8) * torch.sqrt((x.double() ** 2) @ (w.double() ** 2).t())


def within_rms(got, want, bound, what):
    ratio = ((got.double() - want) / bound.clamp(min=1e-300)).square().mean().sqrt()
    assert float(ratio) <= 1, f"{what}: root mean square {float(ratio):.2f} times its bound"


# (dtype, activation, size): {product: (columns of a tile, kind, units at least)}. More units than SMs: CTAs walk from one to
# the next; more than twice as many: both accumulators and every barrier's second phase are used again.
CASES = [
    (F32, "silu", (20000, 136, 40), {0: (64, "full", 2)}),
    (F32, "gelu", (2100, 24, 2056), {0: (128, "full", SMS + 1)}),
    (F32, "tanh", (20000, 264, 136), {0: (64, "full", 2 * SMS + 1), 2: (128, "plain", 2 * SMS + 1)}),
    (F32, "none", (20000, 264, 24), {1: (64, "plain", 2 * SMS + 1)}),
    (F32, "none", (40000, 40, 200), {2: (64, "plain", 2 * SMS + 1), 0: (128, "plain", 2 * SMS + 1)}),
    (F32, "none", (600, 2056, 264), {0: (64, "plain", SMS + 1)}),
    (F32, "none", (20000, 1032, 72), {0: (128, "plain", 2 * SMS + 1)}),
    (F32, "none", (9000, 136, 520), {1: (128, "plain", SMS + 1)}),
    (F32, "silu", (2100, 1031, 2055), {0: (128, "full", SMS + 1), 1: (64, "plain", SMS + 1), 2: (64, "plain", SMS + 1)}),
    (BF16, "silu", (40000, 136, 24), {0: (64, "full", 2 * SMS + 1)}),
    (BF16, "gelu", (40000, 136, 72), {0: (128, "full", 2 * SMS + 1), 2: (256, "plain", 2 * SMS + 1)}),
    (BF16, "sigmoid", (2100, 24, 2056), {0: (128, "full", SMS + 1)}),
    (BF16, "silu", (40000, 264, 136), {0: (256, "full", 2 * SMS + 1), 2: (128, "plain", 2 * SMS + 1)}),
    (BF16, "relu", (40000, 264, 136), {0: (256, "full", 2 * SMS + 1)}),
    (BF16, "gelu_tanh", (2100, 1032, 2056), {0: (128, "full", SMS + 1), 1: (256, "plain", SMS + 1), 2: (256, "plain", SMS + 1)}),
    (BF16, "silu", (2100, 1031, 2055), {0: (128, "full", SMS + 1), 1: (256, "plain", SMS + 1)}),
    (BF16, "none", (40000, 24, 24), {0: (64, "plain", 2 * SMS + 1), 2: (64, "plain", 2 * SMS + 1)}),
    (BF16, "none", (20000, 24, 2056), {0: (256, "plain", 2 * SMS + 1)}),
    (BF16, "none", (150, 1032, 2056), {1: (64, "sums", SMS + 1)}),
    (BF16, "none", (150, 2056, 2056), {1: (128, "sums", SMS + 1)}),
    (BF16, "none", (9000, 264, 2056), {1: (128, "sums", 2 * SMS + 1)}),
    (BF16, "none", (8192, 768, 768), {1: (128, "sums", 2)}),
    (BF16, "none", (48, 2048, 2048), {1: (128, "sums", 2)}),
    (BF16, "none", (2100, 1032, 4104), {2: (256, "plain", SMS + 1)}),
]


@pytest.mark.parametrize("dtype,act,size,plans", CASES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else
                         v if isinstance(v, str) else "" if isinstance(v, dict) else str(v)[6:])
def test_every_tile_against_float64(dtype, act, size, plans):
    M, K, N = size
    for product, (cols, kind, units) in plans.items():
        plan = plan_of(product, M, K, N, dtype, act)
        assert (plan.tile_cols, kind_of(product, plan, act)) == (cols, kind) and plan.units >= units, (product, plan.units)
    x, w, b, r, gy = _problem(M, K, N, dtype)
    if act == "relu":  # whole numbers: z is exact, and so is its sign
        x, w, b = x.round(), (4 * w * K ** 0.5).round(), b.round()
    y, tape = F.linear_forward(x, w, b, activation=act, residual=r, return_tape=True)
    want, bound, z, zb = linear64(x, w, b, r, act)
    within(y, want, bound, f"y {act}")
    if tape is not None:
        within(tape, z, zb + (2.0 ** -11 * (z.abs() + zb) + 2.0 ** -24 if dtype == BF16 else 0), "tape")
    del want, bound, z, zb
    assert torch.equal(F.linear_forward(x, w, b, activation=act, residual=r), y)
    got = F.linear_backward(x, w, gy, tape=tape, activation=act)
    for k, (v, e) in linear64_grads(x, w, b, gy, act).items():
        within(got[k], v, e, f"grad {k} {act}")
    again = F.linear_backward(x, w, gy, tape=tape, activation=act)
    assert all(torch.equal(got[k], again[k]) for k in got)
    if dtype == F32:
        within_rms(F.linear_forward(x, w), x.double() @ w.double().t(), rms_bound(x, w), "plain product")
        got = F.linear_backward(x, w, gy)
        within_rms(got["x"], gy.double() @ w.double(), rms_bound(gy, w.t()), "plain grad x")
        within_rms(got["weight"], gy.double().t() @ x.double(), rms_bound(gy.t(), x.t()), "plain grad weight")
        assert torch.equal(got["bias"], F.linear_backward(x, w, gy, want=("bias",))["bias"])
    elif act != "none":
        fast = F.linear_backward(x, w, gy, tape=tape, activation=act, round_grads=True)
        for k, (v, e) in linear64_grads(x, w, b, gy, act).items():  # these bounds allow gz its rounding
            within(fast[k], v, e, f"grad {k} {act}, rounded")


def test_cases_reach_every_kernel():
    """All instances of the product kernel that the launcher names, with more units than SMs."""
    reached = set()
    for dtype, act, size, _ in CASES:
        for product in range(3):
            plan = plan_of(product, *size, dtype, act, tensor=False)
            if plan.units > SMS:
                reached.add((dtype, plan.tile_cols, kind_of(product, plan, act)))
    want = {(F32, bn, kind) for bn in (64, 128) for kind in ("plain", "full")}
    want |= {(BF16, bn, kind) for bn in (64, 128, 256) for kind in ("plain", "full")}
    want |= {(BF16, bn, "sums") for bn in (64, 128)}
    assert reached == want, (want - reached, reached - want)


def test_rms_bound_tells_a_missing_third_part():
    """Operands cut to the 16 bits of two parts, in float64: inside the element bounds, and far outside this one."""
    x, w, *_ = _problem(300, 264, 520, F32)

    def two_parts(t):
        h = (t.view(torch.int32) & -65536).view(F32)
        return h.double() + (t - h).bfloat16().double()

    want = x.double() @ w.double().t()
    got = two_parts(x) @ two_parts(w).t()
    assert float(((got - want) / rms_bound(x, w)).square().mean().sqrt()) > 4
    within_rms((x.double() @ w.double().t()).float(), want, rms_bound(x, w), "rounded once")


# ---------------------------------------------------------------- float32 in three parts
# one slice of the depth and several, a short depth, aligned rows and odd ones; all of them products on the tensor cores
SPLIT_SIZES = [(700, 264, 520), (260, 1032, 136), (9000, 24, 72), (1001, 333, 301)]


def _split(size, act="none"):
    for product in range(3):
        plan_of(product, *size, F32, act)
    return size


def test_split_sizes_cut_the_depth_and_do_not():
    slices = [plan_of(p, *s, F32).slices for s in SPLIT_SIZES for p in range(3)]
    assert min(slices) == 1 and max(slices) > 2


def _same_non_finite(got, want, what):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    inf = torch.isinf(want)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], want[inf]), f"{what}: other infinities"


@pytest.mark.parametrize("size", SPLIT_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_split_keeps_what_is_not_finite_where_it_is(size):
    M, K, N = _split(size)
    x, w, b, _, gy = _problem(M, K, N, F32, seed=3)
    clean = (x.clone(), w.clone(), gy.clone())
    inf, nan = float("inf"), float("nan")
    x[0, 5], x[1, 7], x[2, 3], x[2, 4], x[M - 1, K - 1] = inf, nan, inf, -inf, -inf
    w[3, 9], w[N - 1, 0] = -inf, inf
    y = F.linear_forward(x, w, b)
    want, bound, _, _ = linear64(x, w, b)
    _same_non_finite(y, want, "y")
    fine = torch.isfinite(want)
    within(y[fine], want[fine], bound[fine], "finite y")
    # each factor of the gradients
    for k in range(3):
        a, v, g = (t.clone() for t in clean)
        if k == 0:
            a[4, 6], a[M - 1, 0] = inf, nan
        elif k == 1:
            v[2, 8], v[N - 1, K - 1] = -inf, nan
        else:
            g[5, 1], g[M - 1, 2], g[7, N - 1] = inf, nan, -inf
        got = F.linear_backward(a, v, g)
        for name, (value, e) in linear64_grads(a, v, None, g).items():
            _same_non_finite(got[name], value, name)
            fine = torch.isfinite(value)
            within(got[name][fine], value[fine], e[fine], name)


@pytest.mark.parametrize("size", SPLIT_SIZES, ids=lambda s: "x".join(map(str, s)))
def test_split_of_float32s_largest_and_smallest(size):
    """The upper part of a value next to float32's largest must not round to infinity, and sums beyond it are infinite.
    Of a value below 2^-110 the third part falls below bfloat16's smallest number, 2^-133, and of smaller ones all of them do."""
    M, K, N = _split(size)
    big = torch.finfo(F32).max
    x, w, gy = torch.zeros(M, K, device="cuda"), torch.zeros(N, K, device="cuda"), torch.zeros(M, N, device="cuda")
    x[:, 0], x[::2, 1], x[1::3, K - 1] = big, -big, 1e-41
    w[:, 0], w[::2, 1], w[1::3, K - 1] = 0.5, 0.25, 1.0
    gy[:, 0], gy[::2, 1] = 0.5, -0.25
    lost = 2.0 ** -133
    y = F.linear_forward(x, w)
    want = x.double() @ w.double().t()
    within(y, want, 2.0 ** -22 * (x.abs().double() @ w.abs().double().t()) + lost, "y")
    got = F.linear_backward(x, w, gy)
    gx, gw = gy.double() @ w.double(), gy.double().t() @ x.double()
    within(got["x"], gx, 2.0 ** -22 * (gy.abs().double() @ w.abs().double()) + lost, "grad x")
    # sums of M values of this size are beyond float32: infinities of the same signs, and zeros
    over = gw.abs() > 2 * big
    assert bool(over.any()) and torch.equal(torch.isinf(got["weight"]), over)
    assert torch.equal(got["weight"][over].sign().double(), gw[over].sign())
    within(got["weight"][~over], gw[~over], torch.full_like(gw[~over], lost * M), "grad weight")
    # largest values as the gradient
    gy.zero_()[:, 2], w = big, torch.full_like(w, 0.5)
    within(F.linear_backward(x, w, gy, want=("x",))["x"], gy.double() @ w.double(), torch.full((M, K), 2.0 ** -22 * big, device="cuda").double(), "grad x of the largest")


@pytest.mark.parametrize("size", SPLIT_SIZES[:2], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e12, 1e17])
def test_split_values_of_any_scale(size, scale):
    M, K, N = _split(size)
    x, w, b, _, gy = _problem(M, K, N, F32, seed=4)
    x, b, gy = x * scale, b * scale, gy * scale
    within(F.linear_forward(x, w, b), *linear64(x, w, b)[:2], "y")
    within_rms(F.linear_forward(x, w), x.double() @ w.double().t(), rms_bound(x, w), "y")
    g = F.linear_backward(x, w, gy)
    for k, (v, e) in linear64_grads(x, w, b, gy).items():
        within(g[k], v, e + 1e-44, k)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("size", [(700, 264, 520), (1001, 333, 301)], ids=lambda s: "x".join(map(str, s)))
def test_split_every_activation(size, act):
    M, K, N = _split(size, act)
    x, w, b, r, gy = _problem(M, K, N, F32, seed=5)
    w = w * 4
    if act == "relu":
        x, w, b = x.round(), w.round(), b.round()
    for res in (None, r):
        y, tape = F.linear_forward(x, w, b, activation=act, residual=res, return_tape=True)
        within(y, *linear64(x, w, b, res, act)[:2], f"y {act}")
    g = F.linear_backward(x, w, gy, tape=tape, activation=act)
    for k, (v, e) in linear64_grads(x, w, b, gy, act).items():
        within(g[k], v, e, f"grad {k} {act}")
        assert torch.equal(F.linear_backward(x, w, gy, tape=tape, activation=act, want=(k,))[k], g[k])


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [(700, 264, 520), (2100, 136, 520)], ids=lambda s: "x".join(map(str, s)))
def test_products_of_views_and_under_autograd(size, dtype):
    M, K, N = size
    for product in range(3):
        plan_of(product, M, K, N, dtype)
    x, w, b, r, gy = _problem(M, K, N, dtype, seed=2)

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)

    want, bound, _, _ = linear64(x, w, b, r)
    grads = linear64_grads(x, w, b, gy)
    for f in (shifted, lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        within(F.linear_forward(f(x), f(w), f(b), residual=f(r)), want, bound, "y")
        g = F.linear_backward(f(x), f(w), f(gy))
        for k, (v, e) in grads.items():
            within(g[k], v, e, k)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    F.fused_linear(*leaves[:3], residual=leaves[3]).backward(gy)
    for leaf, k in zip(leaves, ("x", "weight", "bias")):
        within(leaf.grad, *grads[k], k)
    assert torch.equal(leaves[3].grad, gy)


# ---------------------------------------------------------------- layer norm, by the depth of the kernels' own sums
def _norm_bound(x, xh, rstd):
    """xhat's error. A thread adds 12 pairs at most and the two halves, five shuffles and 15 more warps follow: 33 additions;
    above 8192 columns dim / 256, five and seven. The mean is off by that many steps of mean |x| (and two), the deviation by one
    of its own, rstd by half of the squares' additions and 4."""
    D = x.shape[-1]
    depth = 33 if D <= 8192 else D / 256 + 12
    return STEP * ((depth + 2) * x.double().abs().mean(-1, keepdim=True) * rstd + (depth / 2 + 6) * xh.abs())


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("size", [(40, 96), (33, 768), (20, 1037), (9, 4096), (5, 8191), (4, 9000), (3, 33333)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("offset", [0.0, 30.0, 1e4])
def test_layer_norm_by_the_depth_of_its_sums(size, offset, dtype):
    M, D = size
    x = (_randn(M, D) + offset).to(dtype)
    w, b, gy = _randn(D, seed=1, dtype=dtype), _randn(D, seed=2, dtype=dtype), _randn(M, D, seed=3, dtype=dtype)
    half = dtype == BF16
    _, _, xh, rstd, _ = norm64(x, w, b)
    off = _norm_bound(x, xh, rstd)
    wd, gyd = w.double(), gy.double()
    y, stats = F.layer_norm_forward(x, w, b)
    want = xh * wd + b.double()
    e = off * wd.abs() + 2 * STEP * ((xh * wd).abs() + want.abs())
    within(y, want, e + (2.0 ** -8 * (want.abs() + e) if half else 0), "y")
    g = F.layer_norm_backward(x, w, stats, gy)
    depth = 33 if D <= 8192 else D / 256 + 12
    gw = gyd * wd
    m1, m2 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
    e1 = depth * STEP * gw.abs().mean(-1, keepdim=True)
    e2 = (gw.abs() * off).mean(-1, keepdim=True) + depth * STEP * (gw * xh).abs().mean(-1, keepdim=True)
    rest = (depth / 2 + 10) * STEP * (gw.abs() + m1.abs() + (xh * m2).abs())
    e = rstd * (e1 + xh.abs() * e2 + off * m2.abs() + rest)
    want = rstd * (gw - m1 - xh * m2)
    within(g["x"], want, e + (2.0 ** -8 * (want.abs() + e) if half else 0), "grad x")
    for name, (v, _) in norm64_grads(x, w, gy).items():
        if name == "x":
            continue
        e = (M + 2) * STEP * gyd.abs().sum(0) if name == "bias" else (gyd.abs() * off).sum(0) + (M + 2) * STEP * (gyd * xh).abs().sum(0)
        within(g[name], v, e + (2.0 ** -8 * (v.abs() + e) if half else 0), f"grad {name}")


@pytest.mark.parametrize("size", [(7, 31), (33, 768), (20, 1036), (20, 1037), (9, 4096), (4, 9000)], ids=lambda s: "x".join(map(str, s)))
def test_layer_norm_of_float32_rows_with_bfloat16_parameters(size):
    M, D = size
    x, gy = _randn(M, D), _randn(M, D, seed=3)
    w, b = _randn(D, seed=1, dtype=BF16), _randn(D, seed=2, dtype=BF16)
    y, stats = F.layer_norm_forward(x, w, b)
    within(y, *norm64(x, w, b)[:2], "y")
    g = F.layer_norm_backward(x, w, stats, gy)
    assert g["weight"].dtype == g["bias"].dtype == BF16 and g["x"].dtype == F32
    for k, (v, e) in norm64_grads(x, w, gy, half_params=True).items():
        within(g[k], v, e, k)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 200])
def test_a_vocabulary_projection(rows, dtype):
    """An odd number of outputs, far more of them than anything else."""
    x, w, b, _, gy = _problem(rows, 768, 50257, dtype, seed=12)
    within(F.linear_forward(x, w, b), *linear64(x, w, b)[:2], "y")
    g = F.linear_backward(x, w, gy)
    for k, (v, e) in linear64_grads(x, w, b, gy).items():
        within(g[k], v, e, k)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
def test_gradients_of_more_than_32_bits_of_values(dtype):
    """gz of 2^31 values and more, behind an activation: the gradients of rows at both ends as those rows by themselves."""
    M, N, K = (1 << 18) + 24, 8192 + 8, 16
    if dtype == F32:
        M, N = (1 << 17) + 24, 16384 + 8
    assert M * N > 1 << 31
    x, w = _randn(M, K, dtype=dtype), _randn(N, K, seed=1, dtype=dtype)
    gy = torch.empty(M, N, dtype=dtype, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(2))
    _, tape = F.linear_forward(x, w, activation="silu", return_tape=True)
    some = torch.tensor([0, 1, M // 2, M - 2, M - 1], device="cuda")
    got = F.linear_backward(x, w, gy, tape=tape, activation="silu", want=("x", "bias"))
    v, e = linear64_grads(x[some], w, None, gy[some], "silu")["x"]
    within(got["x"][some], v, e, "grad x")
    gy[:-2] = 0
    got = F.linear_backward(x, w, gy, tape=tape, activation="silu", want=("weight", "bias"))
    for k, (v, e) in linear64_grads(x[-2:], w, None, gy[-2:], "silu").items():
        if k != "x":  # zeros add nothing to a sum, but the slices are cut otherwise
            within(got[k], v, e * 4, k)
