"""What the routing and int8 classes refuse of derivatives, on the Python call path: no GPU needed."""
import pytest
import torch
from torch.autograd import forward_ad as fwd

import inference_rs_b200 as pkg
from inference_rs_b200 import kernel_library as kl
from inference_rs_b200 import ops


@pytest.fixture(autouse=True)
def python_path(monkeypatch):
    monkeypatch.setattr(kl, "_host", kl.NoNativePath())


def routing(tokens=3, topk=2):
    """A routing of every slot to its own row, without the kernel that sorts."""
    r = pkg.TokenRouting.__new__(pkg.TokenRouting)
    r.position = torch.arange(tokens * topk, dtype=torch.int32).view(tokens, topk)
    r.order, r.offsets, r.experts = r.position.flatten(), torch.tensor([0, tokens * topk], dtype=torch.int32), 1
    return r


@pytest.fixture
def stubbed(monkeypatch):
    """The routing's kernels as torch operations."""
    def dispatch(x, position, offsets):
        return x.detach().repeat_interleave(position.shape[1], 0)

    def combine(rows, position, weights, out_dtype):
        t, k = position.shape
        w = torch.ones(t, k) if weights is None else weights
        return (rows.detach().view(t, k, -1) * w.detach()[..., None]).sum(1).to(out_dtype)

    def combine_grad(grad, rows, position, offsets, weights, need_rows=True, need_weights=True):
        t, k = position.shape
        g, r, w = grad.detach(), rows.detach().view(t, k, -1), weights.detach()
        return ((g[:, None] * w[..., None]).flatten(0, 1) if need_rows else None), ((g[:, None] * r).sum(2) if need_weights else None)

    for name, fn in (("route_dispatch", dispatch), ("route_combine", combine), ("route_combine_grad", combine_grad)):
        monkeypatch.setattr(ops, name, fn)


def test_tangents_are_refused(stubbed):
    r = routing()
    x, rows, w = torch.randn(3, 4), torch.randn(6, 4), torch.rand(3, 2)
    linear = pkg.Int8MatMul(pkg.Int8Tensor(torch.zeros(8, 16, dtype=torch.int8), torch.ones(8)))
    int8 = lambda *shape: pkg.Int8Tensor(torch.zeros(shape, dtype=torch.int8), torch.ones(shape[:-1]))
    layer = pkg.Int8Experts(int8(2, 8, 16), int8(2, 8, 16), int8(2, 16, 8))
    ids = torch.zeros(3, 2, dtype=torch.int32)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))
        for call in (lambda: r.dispatch(dual(x)), lambda: r.combine(dual(rows), w), lambda: r.combine(rows, dual(w)), lambda: r.dispatch(dual(x)[:, :2]),
                     lambda: r.combine(rows, dual(w.double()))):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(NotImplementedError, match="forward mode"):
                    call()
        for call in (lambda: linear(dual(torch.randn(3, 16))), lambda: layer(dual(torch.randn(3, 16)), ids, w), lambda: layer(torch.randn(3, 16), ids, dual(w))):
            for mode in (torch.enable_grad, torch.no_grad):
                with mode(), pytest.raises(ValueError, match="forward mode"):
                    call()
        # without one, and where forward mode is off, nothing is refused
        assert torch.equal(r.dispatch(x), x.repeat_interleave(2, 0))
        with torch.inference_mode():
            assert torch.equal(r.dispatch(dual(x)), x.repeat_interleave(2, 0))


def test_tangents_of_gradients_are_refused(stubbed):
    r = routing()
    x, rows, w = torch.randn(3, 4, requires_grad=True), torch.randn(6, 4, requires_grad=True), torch.rand(3, 2, requires_grad=True)
    for out, inputs in ((r.dispatch(x), (x,)), (r.combine(rows, w), (rows, w))):
        with fwd.dual_level():
            grad = fwd.make_dual(torch.ones_like(out), torch.ones_like(out))
            with pytest.raises(NotImplementedError, match="forward mode"):
                torch.autograd.grad(out, inputs, grad)


def test_first_gradients_under_create_graph_and_no_second_ones(stubbed):
    r = routing()
    x, rows, w = torch.randn(3, 4, requires_grad=True), torch.randn(6, 4, requires_grad=True), torch.rand(3, 2, requires_grad=True)
    for fn, inputs in ((lambda: r.dispatch(x), (x,)), (lambda: r.combine(rows, w), (rows, w))):
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
