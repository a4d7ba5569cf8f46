"""4-bit products at the library's shapes, on both sides of their switches, and invalid picks in calls of many routes."""
import pytest
import torch

from test_gpu_w4 import check_experts, check_linear, dense64, make_store, roundings, to, weights, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,k,E", [(4200, 5, 24), (5000, 4, 40)])
@pytest.mark.parametrize("shared", [None, 2])
def test_experts_invalid_picks_of_many_routes(dev, T, k, E, shared):
    """More than 16,384 routes: their order comes from the permutation, which keeps picks outside the experts apart."""
    from mi355moe import moe
    g = torch.Generator().manual_seed(T + k)
    store, a, b = make_store(g, E, 64, 32, 32, True, dev)
    x = torch.randn((T, 64), generator=g).bfloat16()
    ids = torch.randint(-3, E + 5, (T, k), generator=g)
    ids[0], ids[1], ids[-1] = -1, E, 2 ** 40
    ids[5:900, 1] = 7
    w = torch.rand((T, k), generator=g)
    w[0] = float("nan")                                       # weights of no expert are not used
    out = moe.moe_forward(store, x.to(dev), ids.to(dev), w.to(dev), shared_expert=shared)
    w[0] = 0.0
    check_experts(out, a, b, x, ids, w, shared, 10.0)
    if shared is None:
        assert (out[[0, 1, T - 1]] == 0).all()


@pytest.mark.parametrize("T,E,H,I,k,group,dtype,zeros,shared", [
    (1, 12, 4096, 2048, 8, 128, torch.bfloat16, False, 11),
    (4, 12, 4096, 2048, 8, 128, torch.float32, False, 11),
    (9, 6, 5120, 2304, 6, 128, torch.float16, True, None),
    (24, 8, 5120, 2304, 6, 128, torch.float16, True, None),
    (40, 4, 4096, 2048, 2, 64, torch.bfloat16, True, None)])
def test_experts_of_the_library_shapes(dev, T, E, H, I, k, group, dtype, zeros, shared):
    from mi355moe import moe
    g = torch.Generator().manual_seed(T + H)
    store, a, b = make_store(g, E, H, I, group, zeros, dev)
    x = torch.randn((T, H), generator=g).to(dtype)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    w = torch.softmax(torch.randn((T, k), generator=g), 1)
    out = moe.moe_forward(store, x.to(dev), ids.to(dev), w.to(dev), shared_expert=shared)
    check_experts(out, a, b, x, ids, w, shared, 10.0)


@pytest.mark.parametrize("group,dtype,zeros", [(128, torch.bfloat16, False), (64, torch.float16, True), (32, torch.float32, True),
                                               (128, torch.float32, False)])
def test_linear_rows_agree_whatever_form_a_call_takes(dev, group, dtype, zeros):
    """A row multiplied alone, with few, with a hundred and with thousands of others: every form the number of rows chooses, at sizes on
    both sides of each switch. Each is held to the 64-bit product, and to the others within both bounds."""
    from mi355moe import w4
    g = torch.Generator().manual_seed(group)
    K, N = 1024 + group, 1000
    q, s, z = weights(g, N, K, group, zeros)
    W = w4.W4Matrix(*to(dev, (q, s, z)))
    x = torch.randn((6000, K), generator=g).to(dtype)
    w, m = dense64(q, s, z)
    first = x[:5].double()
    tol = roundings(K, group) * 2.0 ** -23 * (first.abs() @ m.t()) + 2.0 ** -24 * (first @ w.t()).abs()
    xd = x.to(dev)
    one = None
    for M in (5, 6, 10, 11, 16, 17, 32, 33, 64, 65, 80, 81, 300, 700, 2100, 6000):
        y = w4.linear(xd[:M], W, out_dtype=torch.float32)
        within(y[:5], first @ w.t(), tol)
        one = y[:5].cpu().double() if one is None else one
        within(y[:5], one, 2 * tol)
        if M <= 300:
            check_linear(y, x[:M], q, s, z)
        assert torch.equal(w4.linear(xd[:M], W, out_dtype=torch.float32), y)
