"""Int8 rows, their products and the layer of experts on them, against the definition in 64 bits.

Integers and scales have one right value each. A product is the exact integer sum a, then three roundings to f32 (a itself, a * x_scale,
that * w_scale; 2^-24 each, relative) and one to the output's type (half a step: eps / 2): |y - exact| <= (4 * 2^-24 + eps / 2) |exact|,
the fourth 2^-24 for the products of the small terms, and half of the type's smallest step where the value is below its normal range.
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


def rows64(x):
    """Integers and scales of rows, from the definition."""
    x = x.double()
    amax = x.abs().amax(1) if x.shape[1] else x.new_zeros(x.shape[0])
    s = (amax / 127).float()
    s = torch.where(torch.isfinite(x).all(1), s, torch.nan)
    q = torch.round(x / s.double()[:, None]).clamp(-127, 127)  # (a scale among the smallest floats may be rounded by half of itself)
    q = torch.where((s == 0)[:, None], 0.0, q)
    return torch.where(torch.isfinite(q), q, 0.0), s


def close(got, want, extra=0.0):
    """Within the module's bound of `want`, plus `extra`."""
    eps = torch.finfo(got.dtype).eps
    tol = (4 * U + eps / 2) * want.abs() + extra + torch.finfo(got.dtype).smallest_normal * eps / 2
    bad = ~((got.double() - want).abs() <= tol) & ~(got.isnan() & want.isnan())
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first {bad.nonzero()[0].tolist()}: {got[bad][0]} for {want[bad][0]}"


def int8_weight(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    data = torch.randint(-128, 128, shape, device="cuda", generator=g, dtype=torch.int8)
    return pkg.Int8Tensor(data, torch.rand(shape[:-1], device="cuda", generator=g) * 1e-3 + 1e-4)


def acts(m, k, dtype, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(m, k, device="cuda", generator=g).to(dtype)


# ---- rows -----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (1, 4096), (600, 1024), (5, 1001), (2, 8200), (513, 4104), (2, 32768), (1, 40000), (2, 40001)])
def test_quantize_is_the_definition(m, k, dtype):
    x = acts(m, k, dtype)
    x[0] *= 3e4 if dtype == torch.float16 else 1e30
    if m > 1:
        x[1] *= 1e-6 if dtype == torch.float16 else 1e-42
    if m > 2:
        x[2] = 0
    if m > 4:
        x[4] = x[4].sign() * (torch.arange(k, device="cuda") % 128).to(dtype)  # quotients that are integers and halves
        x[3] = (torch.arange(k, device="cuda") % 254 - 127).to(dtype) / 2
        x[3, -1] = 127
    want_q, want_s = rows64(x)
    t = pkg.Int8Tensor.quantize(x)
    same = lambda a, b: torch.allclose(a, b, rtol=0, atol=0, equal_nan=True)  # (f16 rows whose values have overflowed are NaN)
    assert same(t.scales, want_s)
    assert torch.equal(t.data[:, :k].double(), want_q) and not t.data[:, k:].any()
    for out in DTYPES:
        assert same(t.dequantize(out), (want_q.float() * want_s[:, None]).to(out))
    assert_device_ok()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_the_smallest_numbers(dtype):
    g = torch.Generator(device="cuda").manual_seed(4)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # the step of the subnormals
    x = (torch.randint(-130, 131, (6, 300), device="cuda", generator=g).double() * tiny).to(dtype)
    x[1] *= 0
    x[2, 1:] = 0
    x[3] *= 100
    want_q, want_s = rows64(x)
    t = pkg.Int8Tensor.quantize(x)
    assert torch.equal(t.scales, want_s) and torch.equal(t.data[:, :300].double(), want_q)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quotients_on_a_half(dtype):
    """Scales of few bits, m 2^e, have values whose quotients are halves exactly: all that the type holds, among their neighbours."""
    rows = []
    for m in range(1, 17):
        for e in (-12, -5, 0, 4):
            s = m * 2.0 ** e
            half = ((torch.arange(-127, 127).double() + 0.5) * s).to(dtype)
            inf = torch.tensor(math.inf, dtype=dtype)
            row = torch.cat([half, torch.nextafter(half, inf), torch.nextafter(half, -inf)]).clamp(-127 * s, 127 * s)
            row[0] = 127 * s
            rows.append(row)
    x = torch.stack(rows).cuda()
    for x in (x, x.repeat(20, 2)):
        want_q, want_s = rows64(x)
        q, s = ops.int8_quantize(x)
        assert torch.equal(s, want_s) and torch.equal(q[:, :x.shape[1]].double(), want_q)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1025, 1032, 1408, 1409, 1529, 1536, 1537, 1544])
def test_quantize_of_many_rows_of_middling_length(k, dtype):
    x = acts(1100, k + 3, dtype)[:, 3 * (k % 2):][:, :k]
    want_q, want_s = rows64(x)
    q, s = ops.int8_quantize(x)
    assert torch.equal(q[:, :k].double(), want_q) and torch.equal(s, want_s) and not q[:, k:].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_of_strided_and_unaligned_rows(dtype):
    big, wide, many = acts(9, 300, dtype), acts(6, 9000, dtype), acts(700, 1100, dtype)
    parts = [big[:, i:i + n] for i in range(9) for n in (1, 7, 8, 9, 15, 16, 17, 250)]
    parts += [wide[:, i:i + n] for i in (0, 1, 5) for n in (2049, 4095, 8193)] + [many[:, i:i + n] for i in (0, 3, 8) for n in (900, 1007, 1024, 1025, 1099 - i)]
    for x in (*parts, big[:, :256], big[:, 1:257], big[::2, 3:40], big.t(), big[:, :1], big[4:5, 8:264], acts(3, 32751, dtype), acts(2, 32761, dtype)):
        want_q, want_s = rows64(x)
        q, s = ops.int8_quantize(x)
        assert torch.equal(q[:, :x.shape[1]].double(), want_q) and torch.equal(s, want_s) and not q[:, x.shape[1]:].any(), tuple(x.shape)


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_value_that_is_not_finite_spoils_its_row_alone(dtype, value):
    w = int8_weight(40, 72)
    x = acts(4, 72, dtype)
    x[2, 70] = value
    q, s = ops.int8_quantize(x)
    assert s.isnan().tolist() == [False, False, True, False] and not q[2].any()
    y = pkg.Int8MatMul(w)(x)
    assert y.isnan().all(1).tolist() == [False, False, True, False] and y[[0, 1, 3]].isfinite().all()


def test_quantize_brings_host_weights_over():
    w = torch.randn(3, 5, 24)
    t = pkg.Int8Tensor.quantize(w)
    assert t.shape == (3, 5, 24) and t.data.is_cuda and torch.equal(t.data, pkg.Int8Tensor.quantize(w.cuda()).data)


def test_from_qtensor():
    g = torch.Generator(device="cuda").manual_seed(3)
    qs = [pkg.QTensor.quantize(torch.randn(48, 512, device="cuda", generator=g) * 0.02, t) for t in (pkg.GgmlDType.Q8_0, pkg.GgmlDType.Q4K)]
    for got, srcs in ((pkg.Int8Tensor.from_qtensor(qs[0]), qs[:1]), (pkg.Int8Tensor.from_qtensor(*qs), qs)):
        want_q, want_s = rows64(torch.cat([q.dequantize() for q in srcs]))
        assert got.shape == ((48, 512) if len(srcs) == 1 else (2, 48, 512))
        assert torch.equal(got.data.reshape(want_q.shape).double(), want_q) and torch.equal(got.scales.flatten(), want_s)
    x = acts(5, 512, torch.bfloat16)
    xq, xs = rows64(x)
    w = pkg.Int8Tensor.from_qtensor(qs[1])
    close(pkg.Int8MatMul.from_qtensor(qs[1])(x), (xq @ w.data.double().T) * xs.double()[:, None] * w.scales.double())


# ---- products -------------------------------------------------------------------------------------------------------------

ROWS = [1, 2, 5, 8, 9, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 129, 200, 255, 257, 333, 513, 1000]


def check_product(m, n, k, dtype, seed=0):
    w = int8_weight(n, k, seed=seed)
    x = acts(m, k, dtype, seed + 1)
    xq, xs = rows64(x)
    want = (xq @ w.data[:, :k].double().T) * xs.double()[:, None] * w.scales.double()
    got = pkg.Int8MatMul(w)(x)
    assert got.shape == (m, n) and got.dtype == dtype
    close(got, want)
    return got


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", [(1, 1), (72, 100), (1000, 1040), (513, 4096), (9001, 70), (25000, 200)])
def test_products(m, n, k):
    for dtype in DTYPES if n < 9000 else DTYPES[m % 3:m % 3 + 1]:
        check_product(m, n, k, dtype)
    assert_device_ok()


@pytest.mark.parametrize("m,n,k", [(1, 1024, 4096), (4, 64, 20000), (16, 4096, 14336), (40, 6144, 130), (333, 6144, 4096), (1500, 2000, 3008), (2, 16, 131071),
                                   (300, 16, 131071)])
def test_larger_products(m, n, k):
    check_product(m, n, k, torch.bfloat16)
    assert_device_ok()


@pytest.mark.parametrize("m", [33, 64, 65, 96, 130, 161, 200, 225, 256, 300, 512])
@pytest.mark.parametrize("n,k", [(2048, 2048), (4096, 2500), (4000, 14336), (8000, 2100), (9300, 4096)])
def test_few_tiles_and_long_sums(m, n, k):
    """Shapes whose tiles are few for the chip: k is divided."""
    check_product(m, n, k, DTYPES[m % 3])
    assert_device_ok()


def test_the_largest_sums_are_exact():
    """131071 products of -128 and -128: 2^31 - 16384."""
    k = 131071
    w = pkg.Int8Tensor(torch.full((40, k), -128, dtype=torch.int8, device="cuda"), torch.ones(40, device="cuda"))
    for m in (1, 30, 130, 600):
        x = pkg.Int8Tensor(torch.full((m, k), -128, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda"))
        y = ops.int8_gemm(x.data, x.scales, w.data, w.scales, k, torch.float32)
        assert (y.double() == 2.0 ** 31 - 2 ** 14).all()  # (17 bits)


def test_rows_of_a_batch_are_independent_and_strides_do_not_matter():
    w = int8_weight(200, 512)
    x = acts(300, 1024, torch.bfloat16)
    y = ops.int8_matmul(x[:, 256:768], w.data, w.scales)
    assert torch.equal(y, ops.int8_matmul(x[:, 256:768].contiguous(), w.data, w.scales))
    for m in (1, 3, 12, 40, 130):
        assert torch.equal(ops.int8_matmul(x[:m, 256:768], w.data, w.scales), y[:m])
    assert torch.equal(pkg.Int8MatMul(w)(x[:, 256:768].contiguous().view(3, 100, 512)), y.view(3, 100, 200))


def test_bias_and_empty_batches():
    w, x = int8_weight(24, 64), acts(3, 64, torch.float32)
    b = torch.randn(24, device="cuda")
    assert torch.equal(pkg.Int8MatMul(w, b)(x), pkg.Int8MatMul(w)(x) + b)
    assert pkg.Int8MatMul(w)(x[:0]).shape == (0, 24)
    assert pkg.Int8MatMul(int8_weight(0, 64))(x).shape == (3, 0)


def test_outputs_and_weights_beyond_32_bit_offsets():
    n, k = 40000, 16
    w, x = int8_weight(n, k), acts(60000, k, torch.float16)
    y = pkg.Int8MatMul(w)(x)  # 2.4e9 outputs
    xq, xs = rows64(x[-70:])
    close(y[-70:], (xq @ w.data.double().T) * xs.double()[:, None] * w.scales.double())
    del y
    n, k = 18000, 131056  # 2.36e9 bytes of weights
    data = torch.zeros(n, k, dtype=torch.int8, device="cuda")
    data[-100:] = torch.randint(-128, 128, (100, k), dtype=torch.int8, device="cuda")
    w = pkg.Int8Tensor(data, torch.ones(n, device="cuda"))
    for m in (1, 20, 140):
        x = acts(m, k, torch.bfloat16)
        xq, xs = rows64(x)
        y = pkg.Int8MatMul(w)(x)
        close(y[:, -100:], (xq @ data[-100:].double().T) * xs.double()[:, None])
        assert not y[:, :-100].any()
    assert_device_ok()


@pytest.mark.parametrize("m", [1, 20, 300])
def test_other_streams_and_graphs(m):
    w = int8_weight(320, 640)
    x = [acts(m, 640, torch.bfloat16, s) for s in (1, 2, 3)]
    lin = pkg.Int8MatMul(w)
    want = [lin(v) for v in x]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [lin(v) for v in x]
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    both = []
    for i in range(12):  # two streams at once, on the same weights
        with torch.cuda.stream(side if i % 2 else other):
            both.append(lin(x[i % 3]))
    side.synchronize()
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(y, want[i % 3]) for i, y in enumerate(both))
    # two graphs, replayed in turn: each has a workspace of its own
    buf = [x[0].clone(), x[1].clone()]
    graphs, outs = [], []
    for b in buf:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(lin(b))
        graphs.append(g)
    for a, b in ((0, 1), (2, 0), (1, 2)):
        buf[0].copy_(x[a])
        buf[1].copy_(x[b])
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[a]) and torch.equal(outs[1], want[b])


# ---- several matrices -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("counts", [[0, 0, 0], [1], [0, 1, 0, 2, 0], [5, 0, 300, 17], [33, 64, 1, 0, 129], [700, 3], [1] * 130, [9] * 40])
@pytest.mark.parametrize("n,k", [(40, 100), (520, 1024)])
def test_rows_meet_their_experts_matrix(counts, n, k):
    e, used, spare = len(counts), sum(counts), 11
    w = int8_weight(e, n, k)
    x = acts(used + spare, k, torch.float32)
    xq, xs = ops.int8_quantize(x)
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    for dtype in DTYPES:
        out = torch.full((used + spare, n), 7.0, dtype=dtype, device="cuda")
        got = ops.int8_gemm(xq, xs, w.data, w.scales, k, dtype, offsets, out)
        assert got is out and (out[used:] == 7).all()  # rows of no expert stay as they were
        at = 0
        for i, c in enumerate(counts):
            want = (xq[at:at + c, :k].double() @ w.data[i, :, :k].double().T) * xs[at:at + c].double()[:, None] * w.scales[i].double()
            close(got[at:at + c], want)
            at += c
    assert_device_ok()


@pytest.mark.parametrize("rows,n,k", [(9, 40, 100), (60, 520, 1024), (700, 300, 512)])
@pytest.mark.parametrize("experts", [1, 2])
def test_rows_before_the_first_offset_belong_to_none(experts, rows, n, k):
    w, x = int8_weight(experts, n, k), acts(rows, k, torch.float32)
    xq, xs = ops.int8_quantize(x)
    for first, last in ((4, rows - 2), (rows - 1, rows), (3, 3), (5, 2), (rows + 5, rows + 9)):
        offsets = torch.tensor([first, *[last] * experts], dtype=torch.int32, device="cuda")
        out = torch.full((rows, n), 7.0, device="cuda")
        ops.int8_gemm(xq, xs, w.data, w.scales, k, torch.float32, offsets, out)
        want = (xq[:, :k].double() @ w.data[0, :, :k].double().T) * xs.double()[:, None] * w.scales[0].double()
        close(out[first:last], want[first:last])
        assert (out[:first] == 7).all() and (out[max(first, last):] == 7).all()
    assert_device_ok()


def check_experts(counts, n, k, dtype):
    w, x = int8_weight(len(counts), n, k), acts(sum(counts), k, torch.float32)
    xq, xs = ops.int8_quantize(x)
    offsets = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    got = ops.int8_gemm(xq, xs, w.data, w.scales, k, dtype, offsets)
    at = 0
    for i, c in enumerate(counts):
        want = (xq[at:at + c, :k].double() @ w.data[i, :, :k].double().T) * xs[at:at + c].double()[:, None] * w.scales[i].double()
        close(got[at:at + c], want)
        at += c
    assert_device_ok()


def test_tiles_of_every_height():
    check_experts([252, 31, 220, 60, 190, 90, 157, 125, 256, 513, 255, 1], 300, 272, torch.float32)


def test_a_thousand_experts():
    g = torch.Generator().manual_seed(2)
    check_experts(torch.randint(0, 40, (1024,), generator=g).tolist(), 272, 100, torch.bfloat16)
    check_experts((torch.rand(1024, generator=g) < 0.2).int().tolist(), 272, 100, torch.bfloat16)


def test_offsets_that_lead_nowhere_are_harmless():
    """Rows are taken from inside the buffers only, whatever the offsets say."""
    w, x = int8_weight(4, 40, 64), acts(30, 64, torch.float32)
    xq, xs = ops.int8_quantize(x)
    for bad in ([5, 3, 90, -7, 2], [0, 10, 4, 2 ** 31 - 1, 2 ** 31 - 1], [-(2 ** 31)] * 5):
        out = torch.full((32, 40), 7.0, device="cuda")
        ops.int8_gemm(xq, xs, w.data, w.scales, 64, torch.float32, torch.tensor(bad, dtype=torch.int32, device="cuda"), out[:30])
        assert (out[30:] == 7).all()
    assert_device_ok()


def test_product_refusals():
    w, x = int8_weight(2, 16, 32), acts(4, 32, torch.float32)
    xq, xs = ops.int8_quantize(x)
    with pytest.raises(ValueError, match="offsets"):
        ops.int8_gemm(xq, xs, w.data, w.scales, 32, torch.float32)
    with pytest.raises(TypeError, match="int32"):
        ops.int8_gemm(xq, xs, w.data, w.scales, 32, torch.float32, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="16-byte"):
        ops.int8_gemm(xq[:, :31], xs, w.data[0], w.scales[0], 31, torch.float32)
    with pytest.raises(ValueError, match="token scales"):
        ops.int8_gemm(xq, xs[:3], w.data[0], w.scales[0], 32, torch.float32)
    with pytest.raises(TypeError, match="f32, f16 or bf16"):
        ops.int8_gemm(xq, xs, w.data[0], w.scales[0], 32, torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.int8_matmul(x, w.data[0].cpu(), w.scales[0])
    with pytest.raises(pkg.KernelLibraryError, match="131071"):
        ops.int8_quantize(torch.zeros(1, 131072, device="cuda"))


# ---- the layer of experts -------------------------------------------------------------------------------------------------

def activation64(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)))
    if name == "relu":
        return g.clamp(min=0)
    if name == "gelu_erf":
        return 0.5 * g * (1 + torch.erf(g / math.sqrt(2)))
    return torch.sigmoid(g)


def experts64(x, ids, weights, gate, up, down, act):
    """The layer in 64 bits with its two roundings (hidden values to x's type, then to integers), and how far a kernel may be from it.

    Its hidden values in f32 are off by some roundings (products 4 U each, the activation's exp, division and polynomial 2^-19 of the
    value, of which most is the cancellation inside tanh's and erf's small arguments: 2^-19 of |up * gate| covers it). Where that can
    carry a value over a border of its type's rounding, it may be one step of the type off; where that, or the same in the row's largest
    value and so in its scale, can carry it over a border between integers, one integer. Each of these is charged in full: |down| * scale
    for an integer, and for the scale its relative change times the row's absolute sum.
    """
    eps = torch.finfo(x.dtype).eps
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    tol = torch.zeros_like(out)
    xq, xs = rows64(x)
    for e in range(gate.shape[0]):
        t, j = torch.where(ids == e)
        if t.numel() == 0:
            continue
        part = lambda w: (xq[t] @ w.data[e, :, :w.shape[2]].double().T) * xs[t].double()[:, None] * w.scales[e].double()
        g, u = part(gate), part(up)
        h = activation64(act, g) * u
        off = 2.0 ** -19 * (g * u).abs() + 2.0 ** -19 * h.abs()
        lo, hi, mid = (h - off).to(x.dtype), (h + off).to(x.dtype), h.to(x.dtype)
        lo, hi, mid = lo.double(), hi.double(), mid.double()
        q, s = rows64(mid.to(x.dtype))
        s = s.double()
        worst = torch.maximum(lo.abs(), hi.abs()).amax(1)
        least = torch.where((lo.sign() == hi.sign()), torch.minimum(lo.abs(), hi.abs()), 0.0).amax(1)
        slack = (worst - least) / least.clamp(min=1e-300) + 2 * U  # relative, of the scale
        top, bottom = hi / s[:, None], lo / s[:, None]
        reach = slack[:, None] * top.abs().maximum(bottom.abs()) + 1e-12
        moved = (torch.round(top + reach) - torch.round(bottom - reach)).clamp(min=0)
        d = down.data[e, :, :down.shape[2]].double() * down.scales[e].double()[:, None]
        y = (q @ d.T) * s[:, None]
        w = weights[t, j].double()[:, None]
        ytol = (moved @ d.abs().T) * s[:, None] * (1 + slack[:, None]) + slack[:, None] * (q.abs() @ d.abs().T) * s[:, None] + 4 * U * y.abs()
        out.index_add_(0, t, y * w)
        tol.index_add_(0, t, (ytol + ids.shape[1] * U * y.abs()) * w.abs())
    return out, tol * (1 + eps)


def router(tokens, experts, topk, dropped, seed=5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    top, ids = torch.randn(tokens, experts, device="cuda", generator=g).topk(topk, dim=1)
    if dropped:
        ids[torch.rand(ids.shape, device="cuda", generator=g) < dropped] = -1
    return ids, top.softmax(1)


@pytest.mark.parametrize("tokens,experts,topk,hidden,ffn,dropped", [
    (1, 8, 2, 256, 512, 0.0), (1, 1, 1, 16, 8, 0.0), (7, 16, 4, 100, 37, 0.3), (48, 64, 6, 512, 352, 0.0), (130, 4, 2, 256, 1000, 0.0),
    (300, 3, 3, 136, 264, 0.5), (700, 2, 1, 520, 129, 0.0), (5, 130, 8, 64, 40, 0.9)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_experts(tokens, experts, topk, hidden, ffn, dropped, dtype):
    gate, up, down = int8_weight(experts, ffn, hidden, seed=1), int8_weight(experts, ffn, hidden, seed=2), int8_weight(experts, hidden, ffn, seed=3)
    ids, weights = router(tokens, experts, topk, dropped)
    x = acts(tokens, hidden, dtype)
    for act in ("silu", "gelu", "relu", "gelu_erf", "sigmoid") if tokens == 7 else ("silu",):
        got = pkg.Int8Experts(gate, up, down, act)(x, ids, weights)
        want, tol = experts64(x, ids, weights, gate, up, down, act)
        assert got.dtype == dtype
        close(got, want, tol)
    assert torch.equal(got, pkg.Int8Experts(gate, up, down, act)(x, ids.int(), weights))
    assert_device_ok()


@pytest.mark.parametrize("tokens,experts,topk", [(1, 8, 2), (40, 16, 4), (300, 16, 2), (1500, 3, 2)])
def test_layers_one_after_the_other_see_their_own_routing(tokens, experts, topk):
    """Calls follow each other in the same memory, their launches overlapping: none may see what the call before left."""
    layer = pkg.Int8Experts(*(int8_weight(experts, *s, seed=i) for i, s in enumerate([(352, 512), (352, 512), (512, 352)])))
    x = acts(tokens, 512, torch.bfloat16)
    routes = [router(tokens, experts, topk, dropped, seed) for seed, dropped in ((1, 0.0), (2, 0.5), (3, 1.0), (4, 0.0))]
    want = []
    for ids, weights in routes:
        want.append(layer(x, ids, weights).clone())
        torch.cuda.synchronize()
    off = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(200):
        off += (layer(x, *routes[i % 4]) != want[i % 4]).sum()
    assert off.item() == 0 and (want[2] == 0).all()
    assert_device_ok()


def test_experts_are_the_operators_one_after_the_other():
    """Routing, rows, products and combination, called one by one, give the layer's bits (ReLU: nothing of its arithmetic differs
    between this library and torch)."""
    gate, up, down = int8_weight(6, 72, 128, seed=1), int8_weight(6, 72, 128, seed=2), int8_weight(6, 128, 72, seed=3)
    layer = pkg.Int8Experts(gate, up, down, "relu")
    ids, weights = router(50, 6, 3, 0.2)
    x = acts(50, 128, torch.bfloat16)
    routing = pkg.TokenRouting(ids, 6)
    rows, scales = ops.int8_quantize(routing.dispatch(x))
    used = int(routing.offsets[-1])
    g, u = (ops.int8_gemm(rows, scales, w.data, w.scales, 128, torch.float32, routing.offsets) for w in (gate, up))
    hidden = torch.zeros(150, 72, dtype=torch.bfloat16, device="cuda")
    hidden[:used] = (g.clamp(min=0) * u)[:used].to(torch.bfloat16)
    hq, hs = ops.int8_quantize(hidden)
    y = ops.int8_gemm(hq, hs, down.data, down.scales, 72, torch.float32, routing.offsets)
    assert torch.equal(layer(x, ids, weights), routing.combine(y, weights, torch.bfloat16))


def test_slots_of_no_expert_count_for_nothing():
    gate, up, down = int8_weight(4, 16, 32, seed=1), int8_weight(4, 16, 32, seed=2), int8_weight(4, 32, 16, seed=3)
    layer = pkg.Int8Experts(gate, up, down)
    ids = torch.tensor([[0, -1], [4, 2 ** 31], [3, 3], [-7, 1]], device="cuda")
    weights = torch.tensor([[0.5, math.nan], [math.inf, math.nan], [0.25, 0.5], [math.nan, 1.0]], device="cuda")
    x = acts(4, 32, torch.bfloat16)
    got = layer(x, ids, weights)
    assert got.isfinite().all() and not got[1].any()
    assert torch.equal(got[0:1], layer(x[:1], ids[:1, :1], weights[:1, :1])) and torch.equal(got[3:], layer(x[3:], ids[3:, 1:], weights[3:, 1:]))
    want, tol = experts64(x[2:3], ids[2:3], weights[2:3], gate, up, down, "silu")
    close(got[2:3], want, tol)
    assert layer(x[:0], ids[:0], weights[:0]).shape == (0, 32)
    assert torch.equal(layer(x.view(2, 2, 32), ids.view(2, 2, 2), weights.view(2, 2, 2)), got.view(2, 2, 32))


def test_experts_in_graphs():
    gate, up, down = int8_weight(8, 64, 96, seed=1), int8_weight(8, 64, 96, seed=2), int8_weight(8, 96, 64, seed=3)
    layer = pkg.Int8Experts(gate, up, down)
    for tokens in (2, 90):
        x, (ids, weights) = acts(tokens, 96, torch.bfloat16), router(tokens, 8, 2, 0.0)
        layer(x, ids, weights)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x, ids, weights)
        for seed in (7, 8):
            x.copy_(acts(tokens, 96, torch.bfloat16, seed))
            new_ids, new_weights = router(tokens, 8, 2, 0.4, seed)
            ids.copy_(new_ids)
            weights.copy_(new_weights)
            graph.replay()
            assert torch.equal(out, layer(x, ids, weights))
    assert_device_ok()
