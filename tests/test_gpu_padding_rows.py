"""Rows behind the last sequence may hold anything, NaN too: a call with such rows gives NaN in them, leaves the others as they are and
takes about as long as without (results that are summed again stop at the first NaN; running each to its end took 60 to 200 times)."""
import pytest
import torch

from test_gpu_router_grad import router_inputs
from test_gpu_w4 import make_store, to, weights

pytestmark = pytest.mark.gpu


def milliseconds(call):
    call()
    best = float("inf")
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(3):
            out = call()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) / 3)
    return best, out


def compare(call, rows, padded):
    """call(rows) and call(padded), equal but for NaN rows: results of the NaN rows, the others' bits, the times."""
    t0, want = milliseconds(lambda: call(rows))
    t1, got = milliseconds(lambda: call(padded))
    odd = padded.isnan().any(1)
    assert got[odd].isnan().all() and torch.equal(got[~odd], want[~odd])
    assert t1 <= 15 * max(t0, 0.05), f"{t1} ms with rows of NaN, {t0} without"


@pytest.mark.parametrize("M", [16, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_rows_of_nan(dev, M, dtype):
    from mi355moe import w4
    g = torch.Generator().manual_seed(M)
    W = w4.W4Matrix(*to(dev, weights(g, 4096, 4096, 128, True)))
    x = torch.randn((M, 4096), generator=g).to(dtype).to(dev)
    y = x.clone()
    y[M // 2:] = float("nan")
    compare(lambda v: w4.linear(v, W), x, y)


def test_experts_rows_of_nan(dev):
    from mi355moe import moe
    g = torch.Generator().manual_seed(1)
    store, _, _ = make_store(g, 16, 2048, 1024, 128, False, dev)
    x = torch.randn((200, 2048), generator=g).bfloat16().to(dev)
    ids = torch.stack([torch.randperm(16, generator=g)[:4] for _ in range(200)]).to(dev)
    w = (torch.rand((200, 4), generator=g) + 0.1).to(dev)
    y = x.clone()
    y[100:] = float("nan")
    compare(lambda v: moe.moe_forward(store, v, ids, w), x, y)


def test_router_backward_rows_of_nan(dev):
    from mi355moe import router
    x, gate, ids, w, _, dl = router_inputs(2000, 2048, 384, 8, 1, dev)
    y = dl.clone()
    y[1000:] = float("nan")
    compare(lambda d: router.topk_backward(x, gate, ids, w, None, d, need_gate=False)[0], dl, y)
