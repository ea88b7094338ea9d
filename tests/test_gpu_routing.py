"""Tokens sorted by expert and back, and the gradients, against the definition in 64 bits.

combine: a sum of `slots` products in f32 by fused multiply-adds: at most slots * 2^-24 of the sum of their magnitudes, then one rounding
to the output's type (eps / 2). A gradient towards a weight is a sum of h products in some order: h * 2^-24 of the sum of magnitudes.
"""
import math

import pytest
import torch

import inference_rs_b200 as pkg
from inference_rs_b200 import kernel_library as kl
from inference_rs_b200 import ops
from gpu_util import assert_device_ok

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


@pytest.fixture(params=["native", "python"], autouse=True)
def call_path(request, monkeypatch):
    """Both call paths of the torch front end."""
    if request.param == "python":
        monkeypatch.setattr(kl, "_host", kl.NoNativePath())
SHAPES = [(1, 1, 1, 1), (1, 8, 2, 64), (7, 128, 8, 100), (33, 60, 4, 1037), (300, 2, 1, 512), (513, 1024, 3, 24), (1000, 5, 6, 130), (64, 16, 16, 2048),
          (3, 4, 2, 5637), (16, 5, 3, 7168), (130, 6, 2, 2100)]  # the last three: several CTAs to a row


def choose(tokens, experts, topk, dropped, dtype=torch.int64, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, experts, (tokens, topk), generator=g, dtype=dtype)  # the same expert twice at times
    ids[torch.rand(ids.shape, generator=g) < dropped] = -1
    return ids.cuda()


def sort_reference(ids, experts):
    flat = ids.flatten().tolist()
    order = sorted((i for i, e in enumerate(flat) if 0 <= e < experts), key=lambda i: flat[i])
    position = [-1] * len(flat)
    for r, i in enumerate(order):
        position[i] = r
    offsets = [sum(1 for e in flat if 0 <= e < b) for b in range(experts + 1)]
    return order + [-1] * (len(flat) - len(order)), offsets, position


def values(m, h, dtype, seed):
    return torch.randn(m, h, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def close(got, want, magnitude, roundings):
    eps = torch.finfo(got.dtype).eps
    tol = roundings * U * magnitude + (eps / 2) * (want.abs() + roundings * U * magnitude) + torch.finfo(got.dtype).smallest_normal * eps / 2
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off: {got[bad][0]} for {want[bad][0]}"


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,experts,topk,h", [*SHAPES, (5000, 37, 7, 1), (1, 1, 0, 1), (0, 4, 2, 1)])
@pytest.mark.parametrize("dropped", [0.0, 0.4, 1.0])
def test_sort(tokens, experts, topk, h, dropped, dtype):
    ids = choose(tokens, experts, topk, dropped, dtype)
    if ids.numel() > 3 and dropped:
        ids.view(-1)[:3] = torch.tensor([experts, torch.iinfo(dtype).max, torch.iinfo(dtype).min], dtype=dtype)
    if topk == 0:
        with pytest.raises(ValueError, match="no slots"):
            pkg.TokenRouting(ids, experts)
        return
    r = pkg.TokenRouting(ids, experts)
    order, offsets, position = sort_reference(ids, experts)
    assert r.order.tolist() == order and r.offsets.tolist() == offsets and r.position.flatten().tolist() == position
    assert r.position.shape == ids.shape and r.order.dtype == r.offsets.dtype == r.position.dtype == torch.int32
    assert_device_ok()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,experts,topk,h", SHAPES)
@pytest.mark.parametrize("dropped", [0.0, 0.3, 1.0])
def test_dispatch_and_combine_with_gradients(tokens, experts, topk, h, dropped, dtype):
    ids = choose(tokens, experts, topk, dropped)
    r = pkg.TokenRouting(ids, experts)
    order, _, _ = sort_reference(ids, experts)
    slots, used = tokens * topk, sum(i >= 0 for i in order)
    slot_of = torch.tensor(order[:used], dtype=torch.int64, device="cuda")
    token_of = slot_of // topk
    x, y, weights = values(tokens, h, dtype, 1), values(slots, h, dtype, 2), torch.rand(tokens, topk, device="cuda")
    y[used:] = math.nan  # rows of no slot are not read
    grad_rows, grad_out = values(slots, h, dtype, 3), values(tokens, h, dtype, 4)
    grad_rows[used:] = math.nan
    weights[r.position < 0] = math.nan  # nor are the weights of slots without a row
    for t in (x, y, weights):
        t.requires_grad_()
    rows, out = r.dispatch(x), r.combine(y, weights)
    assert rows.dtype == out.dtype == dtype and rows.requires_grad and out.requires_grad
    assert torch.equal(rows[:used], x[token_of]) and not rows[used:].any()
    w64, y64 = weights.detach().double().flatten()[slot_of][:, None], y.detach().double()[:used]
    zero = torch.zeros(tokens, h, dtype=torch.float64, device="cuda")
    close(out.detach(), zero.index_add(0, token_of, w64 * y64), zero.index_add(0, token_of, (w64 * y64).abs()), topk)
    gx, gy, gw = torch.autograd.grad([rows, out], [x, y, weights], [grad_rows, grad_out])
    g64 = grad_rows.double()[:used]
    close(gx, zero.index_add(0, token_of, g64), zero.index_add(0, token_of, g64.abs()), topk)
    o64 = grad_out.double()[token_of]
    close(gy[:used], w64 * o64, (w64 * o64).abs(), 1)
    assert not gy[used:].any()
    want = torch.zeros(slots, dtype=torch.float64, device="cuda")
    size = want.clone()
    want[slot_of], size[slot_of] = (o64 * y64).sum(1), (o64 * y64).abs().sum(1)
    close(gw.flatten(), want, size, h)
    assert_device_ok()


def test_gradients_against_differences():
    """Both steps are linear in each input, so a difference quotient is the derivative but for rounding: f32 outputs of about 30 terms of
    size 1 and a step of 1/2 leave 30 * 2^-24 * 2 * h."""
    ids = choose(6, 4, 3, 0.2)
    r = pkg.TokenRouting(ids, 4)
    x, w = values(6, 40, torch.float32, 1).requires_grad_(), torch.rand(6, 3, device="cuda").requires_grad_()
    loss_weights = values(6, 40, torch.float32, 9)
    loss = lambda x, w: (r.combine(torch.tanh(r.dispatch(x)), w) * loss_weights).double().sum()
    loss(x, w).backward()
    tanh_rows = torch.tanh(r.dispatch(x.detach()))
    for t, j in ((0, 0), (3, 2), (5, 1)):
        step = torch.zeros_like(w)
        step[t, j] = 0.5
        diff = loss(x.detach(), w.detach() + step) - loss(x.detach(), w.detach() - step)
        assert abs(float(diff) - float(w.grad[t, j])) <= 40 * 30 * U * 4
    # towards x: d/dx of tanh is 1 - tanh^2, the rest is linear
    want = torch.zeros(6, 40, dtype=torch.float64, device="cuda")
    for t in range(6):
        for j in range(3):
            p = int(r.position[t, j])
            if p >= 0:
                want[t] += float(w.detach()[t, j]) * loss_weights[t].double() * (1 - tanh_rows[p].double() ** 2)
    assert torch.allclose(x.grad.double(), want, rtol=0, atol=30 * U * float(want.abs().max() + 1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_other_types_strides_and_shapes(dtype):
    ids = choose(30, 5, 3, 0.2).view(5, 6, 3)
    r = pkg.TokenRouting(ids, 5)
    x = values(30, 400, dtype, 1)
    for v in (x[:, :128], x[:, 1:130], x[:, ::2], x[:1].expand(30, 400)):
        assert torch.equal(r.dispatch(v.unflatten(0, (5, 6))), r.dispatch(v.contiguous().view(5, 6, -1)))
    y, w = values(90, 400, dtype, 2), torch.rand(5, 6, 3, device="cuda")
    for out in DTYPES:
        full = r.combine(y.float(), w, out)
        assert full.shape == (5, 6, 400) and full.dtype == out
        assert torch.equal(r.combine(y, w, out), full)
        assert torch.equal(r.combine(y[:, 8:200], w, out), full[..., 8:200]) and torch.equal(r.combine(y[:, 1:200], w, out), full[..., 1:200])
    # a gradient that is one value everywhere (the sum's) and weights in another type
    y.requires_grad_()
    w16 = w.to(torch.bfloat16).requires_grad_()
    r.combine(y, w16).sum().backward()
    live = (r.position >= 0).flatten()
    assert torch.equal(y.grad[r.position.flatten()[live].long()], w16.detach().float().flatten()[live][:, None].to(dtype).expand(-1, 400))
    assert w16.grad.dtype == torch.bfloat16 and not w16.grad[r.position < 0].any()


def test_only_the_gradients_asked_for():
    ids = choose(9, 4, 2, 0.0)
    r = pkg.TokenRouting(ids, 4)
    y, w = values(18, 64, torch.float32, 1), torch.rand(9, 2, device="cuda")
    both = torch.autograd.grad(r.combine(y.requires_grad_(), w.requires_grad_()).sum(), [y, w])
    assert torch.equal(torch.autograd.grad(r.combine(y, w.detach()).sum(), y)[0], both[0])
    assert torch.equal(torch.autograd.grad(r.combine(y.detach(), w).sum(), w)[0], both[1])
    with torch.no_grad():
        assert not r.combine(y, w).requires_grad and not r.dispatch(values(9, 8, torch.float32, 1).requires_grad_()).requires_grad


def test_no_second_derivatives():
    r = pkg.TokenRouting(choose(9, 4, 2, 0.0), 4)
    y, w = values(18, 64, torch.float32, 1).requires_grad_(), torch.rand(9, 2, device="cuda").requires_grad_()
    x = values(9, 64, torch.float32, 2).requires_grad_()
    for out, inputs in ((r.combine(y, w), (y, w)), (r.dispatch(x), (x,))):
        with pytest.raises(RuntimeError, match="differentiat"):
            first = torch.autograd.grad((out ** 2).sum(), inputs, create_graph=True)
            sum((g ** 2).sum() for g in first).backward()


def test_in_graphs_and_on_other_streams():
    ids = choose(40, 6, 2, 0.0)
    x, w = values(40, 72, torch.bfloat16, 1), torch.rand(40, 2, device="cuda")

    def step():
        r = pkg.TokenRouting(ids, 6)
        rows = r.dispatch(x)
        g = ops.route_combine_grad(x, rows, r.position, r.offsets, w)
        return r.order, r.offsets, r.position, rows, r.combine(rows, w), *g

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    side = torch.cuda.Stream()
    for seed in (1, 2):
        ids.copy_(choose(40, 6, 2, 0.3, seed=seed))
        x.copy_(values(40, 72, torch.bfloat16, seed + 10))
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_a_captured_backward_pass():
    ids, w = choose(40, 6, 3, 0.2), torch.rand(40, 3, device="cuda")
    x, go, gr = values(40, 72, torch.bfloat16, 1), values(40, 72, torch.bfloat16, 2), values(120, 72, torch.bfloat16, 3)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w)]
        r = pkg.TokenRouting(ids, 6)
        rows = r.dispatch(leaves[0])
        return torch.autograd.grad([rows, r.combine(rows, leaves[1])], leaves, [gr, go])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for seed in (4, 5):
        ids.copy_(choose(40, 6, 3, 0.3, seed=seed))
        x.copy_(values(40, 72, torch.bfloat16, seed))
        w.copy_(torch.rand(40, 3, device="cuda"))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(grads, step()))


def test_no_tokens_and_narrow_rows():
    r = pkg.TokenRouting(torch.zeros(0, 3, dtype=torch.int32, device="cuda"), 4)
    assert r.dispatch(torch.zeros(0, 8, device="cuda")).shape == (0, 8) and r.offsets.tolist() == [0] * 5
    assert r.combine(torch.zeros(0, 8, device="cuda"), torch.zeros(0, 3, device="cuda")).shape == (0, 8)
    r = pkg.TokenRouting(choose(5, 4, 2, 0.0), 4)
    x, w = torch.zeros(5, 0, device="cuda", requires_grad=True), torch.ones(5, 2, device="cuda", requires_grad=True)
    rows = r.dispatch(x)
    out = r.combine(rows, w)
    assert rows.shape == (10, 0) and out.shape == (5, 0)
    gx, gw = torch.autograd.grad([out], [x, w], [torch.zeros(5, 0, device="cuda")])
    assert gx.shape == (5, 0) and not gw.any()


def test_beyond_32_bit_offsets():
    tokens, topk, h = 300000, 2, 4096  # 2.46e9 values in the rows
    ids = torch.randint(0, 7, (tokens, topk), device="cuda")
    r = pkg.TokenRouting(ids, 7)
    x = torch.zeros(tokens, h, dtype=torch.float16, device="cuda")
    x[:, 0] = torch.arange(tokens, device="cuda") % 2048
    rows = r.dispatch(x)
    assert torch.equal(rows[-5000:, 0], x[(r.order[-5000:] // topk).long(), 0]) and not rows[-5000:, 1:].any()
    out = r.combine(rows, torch.ones(tokens, topk, device="cuda"))
    assert torch.equal(out[:, 0], 2 * x[:, 0]) and not out[-5000:, 1:].any()


def test_refusals():
    ids = choose(4, 3, 2, 0.0)
    r = pkg.TokenRouting(ids, 3)
    with pytest.raises(ValueError, match="tokens"):
        r.dispatch(values(5, 8, torch.float32, 0))
    with pytest.raises(TypeError, match="f32, f16 or bf16"):
        r.dispatch(torch.zeros(4, 8, dtype=torch.float64, device="cuda"))
    with pytest.raises(ValueError, match="rows for"):
        r.combine(values(7, 8, torch.float32, 0), torch.ones(4, 2, device="cuda"))
    with pytest.raises(ValueError, match="weights"):
        r.combine(values(8, 8, torch.float32, 0), torch.ones(4, 3, device="cuda"))
    with pytest.raises(pkg.KernelLibraryError, match="1024 experts"):
        pkg.TokenRouting(ids, 1025)
    with pytest.raises(pkg.KernelLibraryError, match="1024 experts"):
        pkg.TokenRouting(ids, 0)
