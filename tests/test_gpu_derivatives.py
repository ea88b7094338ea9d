"""Derivatives that the routing and int8 classes have and those that they refuse, on both call paths."""
import pytest
import torch
from torch.autograd import forward_ad as fwd

import inference_rs_b200 as pkg
from inference_rs_b200 import kernel_library as kl

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"], autouse=True)
def call_path(request, monkeypatch):
    """Both call paths of the torch front end."""
    if request.param == "python":
        monkeypatch.setattr(kl, "_host", kl.NoNativePath())


def int8_weight(*shape):
    g = torch.Generator(device="cuda").manual_seed(len(shape))
    return pkg.Int8Tensor(torch.randint(-128, 128, shape, device="cuda", generator=g, dtype=torch.int8), torch.full(shape[:-1], 1e-3, device="cuda"))


@pytest.fixture
def state():
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(-1, 4, (9, 2), device="cuda", generator=g)
    x, rows, w = torch.randn(9, 64, device="cuda", generator=g), torch.randn(18, 64, device="cuda", generator=g), torch.rand(9, 2, device="cuda", generator=g)
    layer = pkg.Int8Experts(int8_weight(4, 32, 64), int8_weight(4, 32, 64), int8_weight(4, 64, 32))
    return pkg.TokenRouting(ids, 4), ids, x, rows, w, pkg.Int8MatMul(int8_weight(24, 64)), layer


def test_tangents_are_refused(state):
    r, ids, x, rows, w, linear, layer = state
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for call in (lambda: r.dispatch(dual(x)), lambda: r.combine(dual(rows), w), lambda: r.combine(rows, dual(w)), lambda: r.dispatch(dual(x)[:, :16])):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward mode"):
                    call()
        for call in (lambda: linear(dual(x)), lambda: layer(dual(x), ids, w), lambda: layer(x, ids, dual(w))):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(ValueError, match="forward mode"):
                    call()
        plain = r.dispatch(x), r.combine(rows, w), linear(x), layer(x, ids, w)
        with torch.inference_mode():  # forward mode is off in it
            same = r.dispatch(dual(x)), r.combine(dual(rows), w), linear(dual(x)), layer(dual(x), ids, w)
        assert all(torch.equal(a, b) for a, b in zip(plain, same))


def test_tangents_of_gradients_are_refused(state):
    r, _, x, rows, w, _, _ = state
    for t in (x, rows, w):
        t.requires_grad_()
    for out, inputs in ((r.dispatch(x), (x,)), (r.combine(rows, w), (rows, w))):
        with fwd.dual_level():
            grad = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward mode"):
                torch.autograd.grad(out, inputs, grad)


def test_function_transforms_are_refused(state):
    """Their tensors are wrappers without memory of their own: an error, never a result without its derivative."""
    r, ids, x, rows, w, linear, layer = state
    for call in (r.dispatch, linear, lambda t: layer(t, ids, w)):
        for transform in (lambda f: torch.vmap(f)(torch.stack([x, x])), lambda f: torch.func.grad(lambda t: f(t).sum())(x), lambda f: torch.func.jvp(f, (x,), (x,))):
            with pytest.raises((RuntimeError, ValueError)):
                transform(call)
    for call in (lambda t: r.combine(t, w), lambda t: r.combine(t.detach() * 0 + rows, w * t.sum())):
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.grad(lambda t: call(t).sum())(rows)
        with pytest.raises((RuntimeError, ValueError)):
            torch.func.jvp(call, (rows,), (rows,))


def test_first_gradients_under_create_graph_and_no_second_ones(state):
    r, _, x, rows, w, _, _ = state
    for t in (x, rows, w):
        t.requires_grad_()
    for fn, inputs in ((lambda: r.dispatch(x), (x,)), (lambda: r.combine(rows, w), (rows, w)), (lambda: r.combine(rows.unsqueeze(1)[:, 0], w), (rows, w))):
        loss = lambda: (fn() ** 2).sum()
        plain, first = torch.autograd.grad(loss(), inputs), torch.autograd.grad(loss(), inputs, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(plain, first)) and all(g.requires_grad for g in first)
        for g in first:
            with pytest.raises(RuntimeError, match="differentiated again"):
                g.sum().backward(retain_graph=True)
    # the output's own gradient is a constant here, but those of rows and weights depend on each other
    first = torch.autograd.grad(r.combine(rows, w).sum(), (rows, w), create_graph=True)
    for g in first:
        with pytest.raises(RuntimeError, match="differentiated again"):
            g.sum().backward(retain_graph=True)
    # and that of dispatch on nothing
    assert not torch.autograd.grad(r.dispatch(x).sum(), x, create_graph=True)[0].requires_grad
    only, = torch.autograd.grad(r.combine(rows, w.detach()).sum(), rows, create_graph=True)
    assert not only.requires_grad
    # inside a larger graph
    v = torch.ones(64, device="cuda", requires_grad=True)
    out = (r.combine(r.dispatch(x), w) * v).sum() + (v ** 3).sum()
    gx, _ = torch.autograd.grad(out, (x, v), create_graph=True)
    assert torch.equal(gx, torch.autograd.grad((r.combine(r.dispatch(x), w) * v).sum(), x)[0])
