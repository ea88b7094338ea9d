"""Int8 products and layers of experts as several threads call them, and layers of other shapes than the usual: wide ones on the tensor
cores, more slots a token than the quantizer routes, tokens that are a part of a wider tensor."""
import threading

import pytest
import torch

import inference_rs_b200 as pkg
from inference_rs_b200 import kernel_library as kl
from gpu_util import assert_device_ok
from test_gpu_int8 import acts, close, experts64, int8_weight, router

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"], autouse=True)
def call_path(request, monkeypatch):
    """Both call paths of the torch front end."""
    if request.param == "python":
        monkeypatch.setattr(kl, "_host", kl.NoNativePath())


def test_threads_on_streams_of_their_own():
    w = int8_weight(2048, 4096)
    layer = pkg.Int8Experts(*(int8_weight(4, *s, seed=i) for i, s in enumerate([(352, 512), (352, 512), (512, 352)])))
    lin = pkg.Int8MatMul(w)
    rows = (1, 20, 64, 130, 300)
    x = [acts(m, 4096, torch.bfloat16) for m in rows]
    xe, (ids, weights) = acts(90, 512, torch.bfloat16), router(90, 4, 2, 0.2)
    torch.cuda.synchronize()
    results, errors = {}, []
    start = threading.Barrier(4)

    def work(i):
        try:
            start.wait()
            with torch.cuda.stream(torch.cuda.Stream()):
                for turn in range(20):
                    results[i, turn] = [lin(a) for a in x] + [layer(xe, ids, weights)]
                torch.cuda.current_stream().synchronize()
        except Exception as exc:  # noqa: BLE001 - shown below
            errors.append(exc)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    want = [lin(a) for a in x] + [layer(xe, ids, weights)]
    for got in results.values():
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert_device_ok()


@pytest.mark.parametrize("tokens,experts,topk,hidden,ffn", [(200, 2, 2, 2056, 1500), (600, 4, 1, 1040, 2100), (40, 2, 1, 4096, 1030), (33, 16, 12, 136, 264), (300, 20, 9, 264, 72)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_wide_layers_and_many_slots(tokens, experts, topk, hidden, ffn, dtype):
    gate, up, down = int8_weight(experts, ffn, hidden, seed=1), int8_weight(experts, ffn, hidden, seed=2), int8_weight(experts, hidden, ffn, seed=3)
    # hidden values that f16 holds
    gate.scales.mul_(0.1)
    up.scales.mul_(0.1)
    ids, weights = router(tokens, experts, topk, 0.1)
    x = acts(tokens, hidden, dtype)
    for act in ("silu", "gelu"):
        got = pkg.Int8Experts(gate, up, down, act)(x, ids, weights)
        want, tol = experts64(x, ids, weights, gate, up, down, act)
        assert got.dtype == dtype and got.isfinite().all()
        close(got, want, tol)
    assert_device_ok()


@pytest.mark.parametrize("tokens", [1, 5, 300])
def test_tokens_that_are_part_of_a_wider_tensor(tokens):
    layer = pkg.Int8Experts(*(int8_weight(4, *s, seed=i) for i, s in enumerate([(96, 128), (96, 128), (128, 96)])))
    ids, weights = router(tokens, 4, 2, 0.1)
    wide = acts(2 * tokens, 300, torch.bfloat16)
    for x in (wide[:tokens, 8:136], wide[:tokens, 3:131], wide[::2, 100:228], wide[:tokens, :256:2], wide[:tokens].t()[:128].t(), wide[:1, :128].expand(tokens, 128)):
        assert torch.equal(layer(x, ids, weights), layer(x.contiguous(), ids, weights))
    # ids and weights that are parts of wider ones, too
    ids3, weights3 = torch.cat([ids, ids], 1), torch.cat([weights, weights], 1)
    assert torch.equal(layer(wide[:tokens, :128], ids3[:, :2], weights3[:, 2:]), layer(wide[:tokens, :128].contiguous(), ids, weights))
    assert_device_ok()
