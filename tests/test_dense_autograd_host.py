"""What the dense operators' public functions tell autograd, on the CPU: the compiled binding is replaced by plain products."""
import pytest
import torch
from torch.autograd import forward_ad

from qkan_b200 import LayerNorm, Linear, _abi
from qkan_b200 import functional as F


class PlainBinding:
    """Results without a history, as the binding's are."""

    def linear_forward(self, x, w, b, r, act, want_tape):
        return (x.detach() @ w.detach().t()), None

    def linear_backward(self, x, w, gy, tape, act, want, round_grads):
        return gy.detach() @ w.detach() if want & 1 else None, None, None

    def norm_backward(self, x, w, stats, gy, want, param_dtype):
        return gy.detach() * 2, *[gy.detach().sum(0) if want & bit else None for bit in (2, 4)]

    def norm_forward(self, x, w, b, eps, want_stats):
        return x.detach() * 2, (torch.zeros(*x.shape[:-1], 2) if want_stats else None)


@pytest.fixture(autouse=True)
def plain(monkeypatch):
    monkeypatch.setattr(_abi, "dense", PlainBinding)


x, w, b = torch.randn(3, 4), torch.randn(5, 4), torch.randn(5)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", range(4))
def test_forward_mode_tangents_are_refused_and_not_dropped(which, grad):
    args = [x, w, b, torch.randn(3, 5)]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError, match="forward mode AD|jvp"):
            F.fused_linear(*args[:3], residual=args[3])
        if which == 0:
            for call in (lambda: F.layer_norm(args[0]), lambda: LayerNorm(4).requires_grad_(False)(args[0]),
                         lambda: Linear(4, 5).requires_grad_(False)(args[0])):
                with pytest.raises(RuntimeError, match="forward mode AD|jvp"):
                    call()


@pytest.mark.parametrize("which", range(2))
def test_forward_mode_tangents_of_a_layer_norms_parameters_are_refused(which):
    params = [torch.ones(4), torch.zeros(4)]
    with forward_ad.dual_level():
        params[which] = forward_ad.make_dual(params[which], torch.ones(4))
        with pytest.raises(RuntimeError, match="forward mode AD|jvp"):
            F.layer_norm(x, *params)


def test_a_dual_level_without_tangents_changes_nothing():
    want = x @ w.t()
    with forward_ad.dual_level():
        assert torch.equal(F.fused_linear(x, w), want) and torch.equal(F.layer_norm(x), x * 2)
        assert not F._wants_grad(x, w, None, None)
    assert F._wants_grad(x, w.clone().requires_grad_(True))
    with torch.no_grad():
        assert not F._wants_grad(x, w.clone().requires_grad_(True))


@pytest.mark.parametrize("f", [lambda t: F.fused_linear(t, w), F.layer_norm])
def test_a_tangent_of_the_outputs_gradient_is_refused(f):
    leaf = x.clone().requires_grad_(True)
    y = f(leaf)
    with forward_ad.dual_level():
        gy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
        with pytest.raises(RuntimeError, match="forward-mode AD"):
            torch.autograd.grad(y, leaf, gy, retain_graph=True)
        assert torch.autograd.grad(y, leaf, torch.ones_like(y))[0].shape == x.shape


@pytest.mark.parametrize("want", [(), ("x",), ("weight", "x"), ("x", "weight", "bias")])
def test_gradients_asked_for_by_any_iterable(want):
    gy, stats = torch.randn(3, 4), torch.zeros(3, 2)
    for form in (tuple, list, iter, lambda names: (name for name in names), dict.fromkeys):
        assert list(F.layer_norm_backward(x, None, stats, gy, want=form(want))) == list(want)
        assert list(F.linear_backward(x, w, torch.randn(3, 5), want=form(want))) == list(want)


@pytest.mark.parametrize("f", [lambda t: F.fused_linear(t, w), F.layer_norm])
def test_second_derivatives_are_refused_and_not_zero(f):
    """With create_graph=True, also where the output's gradient is a constant."""
    leaf = x.clone().requires_grad_(True)
    plain, = torch.autograd.grad(f(leaf).sum(), leaf)
    assert not plain.requires_grad
    for loss in (f(leaf).sum(), f(leaf).square().sum()):
        g, = torch.autograd.grad(loss, leaf, create_graph=True)
        assert g.requires_grad and torch.isfinite(g).all()
        with pytest.raises(RuntimeError, match="no second derivatives"):
            (g.square().sum() + leaf.sum()).backward()
    g, = torch.autograd.grad(f(leaf).sum(), leaf, create_graph=True)
    assert torch.equal(g, plain)
    leaf.grad = None
    f(leaf).sum().backward(create_graph=True)  # asked for and not used
    assert torch.equal(leaf.grad.detach(), plain)
    with pytest.raises(RuntimeError, match="no second derivatives"):
        torch.autograd.functional.hessian(lambda t: f(t).sum(), x)


def test_the_residuals_gradient_is_differentiable_as_it_is():
    leaf, r = x.clone().requires_grad_(True), torch.randn(3, 5, requires_grad=True)
    y = F.fused_linear(leaf, w, residual=r) + r
    gr, = torch.autograd.grad((y * r.detach().clone().requires_grad_(True)).sum(), r, create_graph=True)
    assert gr.requires_grad
    again, = torch.autograd.grad(y.square().sum(), r, create_graph=True)
    assert torch.autograd.grad(again.sum(), r)[0].shape == r.shape
