"""The load-balance loss with its counts and gradient and the router's backward pass, against the definitions in float64.

Tolerances: a score p comes from expf (2 ulp) and fp32 sums of at most 16 values per lane and 6 wave stages, so its relative
error is below 32 x 2^-23; sums of positive scores in at most 64 sequential steps keep that (load, loss: twice it). The
gradient g p (c - sum c p) is off by that share of g p (c + sum c p), and by half a step of its type. The router's products
accumulate N fp32 terms: N 2^-23 of the sum of their magnitudes at most; dx also leaves out 2^-15 of that and is rounded to
bf16 (2^-8)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

P_TOL = 64 * 2.0 ** -23
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24}


def close(got, ref, tol):
    """|got - ref| <= tol everywhere, NaN exactly where ref has one."""
    got, ref = got.detach().cpu().double(), ref.double()
    nan = ref.isnan()
    bad = (got.isnan() != nan) | (~nan & ((got - ref).abs() > tol))
    if bad.any():
        at = bad.nonzero()[:4].tolist()
        tol = torch.as_tensor(tol).expand_as(ref)
        pytest.fail(f"{int(bad.sum())} of {bad.numel()} off, first at {at}: {got[bad][:4].tolist()} for {ref[bad][:4].tolist()}, "
                    f"tolerance {tol[bad][:4].tolist()}")


def scores64(x, score):
    """[.., E] float64 scores of logits; rows of -inf only have none."""
    x = x.double()
    none = (x == -torch.inf).all(-1, keepdim=True)
    x = torch.where(none, torch.zeros_like(x), x)
    if score == "softmax":
        p, one = torch.softmax(x, -1), torch.ones_like(x)
    else:
        sg = torch.sigmoid(x)
        ls = torch.nn.functional.logsigmoid(x)                # ratios of sigmoids far below zero
        p, one = torch.softmax(ls, -1), 1 - sg
    return torch.where(none, torch.zeros_like(p), p), one


def balance64(logits, ids, mask, score, dloss):
    """(loss, counts, tokens, load, dlogits, gradient magnitude) per sequence, float64 on the CPU."""
    logits, ids, dloss = logits.cpu(), ids.cpu(), dloss.cpu().double()
    B, T, E = logits.shape
    k = ids.shape[2]
    live = torch.ones((B, T), dtype=torch.bool) if mask is None else mask.cpu().bool()
    loss, counts = torch.zeros(B, dtype=torch.float64), torch.zeros((B, E), dtype=torch.int64)
    load, d, mag = torch.zeros((B, E), dtype=torch.float64), torch.zeros((B, T, E), dtype=torch.float64), torch.zeros((B, T, E), dtype=torch.float64)
    for b in range(B):
        rows = live[b].nonzero()[:, 0]
        n = rows.numel()
        if n == 0:
            continue
        p, one = scores64(logits[b, rows], score)
        e = ids[b, rows].reshape(-1)
        counts[b] = torch.bincount(e[(e >= 0) & (e < E)], minlength=E)
        c = counts[b].double()
        load[b] = p.sum(0)
        fac = E / (k * n * n)
        loss[b] = fac * (c * load[b]).sum()
        dot = (p @ c)[:, None]
        d[b, rows] = dloss[b] * fac * p * (c - dot) * one
        mag[b, rows] = (dloss[b] * fac).abs() * p * (c + dot)
    return loss, counts, live.sum(1), load, d, mag


def make(B, T, E, k, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((B, T, E), generator=g) * scale).to(dtype)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(B * T)]).view(B, T, k) if B * T else torch.zeros((B, T, k), dtype=torch.int64)
    dloss = torch.randn((B,), generator=g)
    return logits, ids, dloss, g


def run_and_compare(dev, logits, ids, mask, score, dloss):
    from mi355moe import router
    k = ids.shape[2]
    lg, idd, dl = logits.to(dev), ids.to(dev), dloss.to(dev)
    md = None if mask is None else mask.to(dev)
    loss, counts, tokens, load = router.balance_loss_forward(lg, idd, md, score)
    d = router.balance_loss_backward(dl, lg, counts, tokens, k, md, score)
    torch.cuda.synchronize()
    r_loss, r_counts, r_tokens, r_load, r_d, mag = balance64(logits, ids, mask, score, dloss)
    assert torch.equal(counts.cpu().long(), r_counts)
    assert torch.equal(tokens.cpu().long(), r_tokens.long())
    close(load, r_load, P_TOL * r_load + 1e-37)
    close(loss, r_loss, 2 * P_TOL * r_loss.abs() + 1e-37)
    assert d.dtype == logits.dtype and d.shape == logits.shape
    close(d, r_d, P_TOL * mag + HALF[d.dtype] * r_d.abs() + TINY[d.dtype])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("B,T,E,k,dtype", [
    (1, 1, 8, 1, torch.float32), (1, 64, 384, 8, torch.float32), (1, 65, 384, 8, torch.bfloat16),
    (3, 129, 1, 1, torch.float32), (2, 200, 129, 6, torch.float16), (1, 1000, 511, 8, torch.float32),
    (5, 77, 1024, 32, torch.float32), (1, 17000, 64, 4, torch.bfloat16), (2, 333, 257, 3, torch.bfloat16)])
def test_balance(dev, B, T, E, k, dtype, score):
    logits, ids, dloss, _ = make(B, T, E, k, dtype, 100 + T + E)
    run_and_compare(dev, logits, ids, None, score, dloss)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [40, 300])
def test_balance_masks_and_odd_values(dev, T, score):
    """Padded tokens with NaN and infinite logits, a sequence with no token, picks outside the experts, an expert picked
    twice, experts masked by -inf and by the type's lowest value, rows of -inf only, logits far below and above zero."""
    B, E, k = 4, 100, 4
    logits, ids, dloss, g = make(B, T, E, k, torch.float32, 7)
    mask = torch.rand((B, T), generator=g) < 0.7
    mask[1] = False
    logits[~mask] = float("nan")
    logits[2][~mask[2]] = float("inf")
    logits[0, :, 10:20] = -torch.inf
    logits[2, :, 50:] = torch.finfo(torch.float32).min
    logits[3, 3] = -torch.inf
    logits[3, 5] = torch.finfo(torch.float32).min
    logits[3, 7] -= 150.0
    logits[3, 9] += 150.0
    mask[3, 3:10] = True
    logits[3, 4], logits[3, 6], logits[3, 8] = 0.5, -0.5, 1.0
    ids[0, ::3, 1] = -1
    ids[0, 1::3, 2] = E
    ids[2, :, 1] = ids[2, :, 0]
    run_and_compare(dev, logits, ids, mask, score, dloss)
    run_and_compare(dev, logits, ids, mask.to(torch.uint8), score, dloss)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [40, 300])
def test_balance_rows_of_odd_values(dev, T, score):
    """Live tokens among masked NaN ones: a row of -inf only, one of the type's lowest value, logits far from zero, one expert
    left."""
    logits, ids, dloss, g = make(2, T, 70, 3, torch.float32, 8)
    mask = torch.rand((2, T), generator=g) < 0.8
    for r in (3, 5, 7, 9, 11):
        mask[0, r] = True
    logits[~mask] = float("nan")
    logits[0, 3] = -torch.inf
    logits[0, 5] = torch.finfo(torch.float32).min
    logits[0, 7] = torch.randn(70, generator=g) - 150.0
    logits[0, 9] = torch.randn(70, generator=g) + 150.0
    logits[0, 11] = -torch.inf
    logits[0, 11, 4] = -300.0
    run_and_compare(dev, logits, ids, mask, score, dloss)


def test_balance_nan_reaches_its_row_only(dev):
    from mi355moe import router
    logits, ids, dloss, _ = make(1, 70, 50, 2, torch.float32, 9)
    logits[0, 5, 3] = float("nan")
    lg, idd = logits.to(dev), ids.to(dev)
    loss, counts, tokens, _ = router.balance_loss_forward(lg, idd)
    d = router.balance_loss_backward(dloss.to(dev), lg, counts, tokens, 2).cpu()
    assert loss.isnan().all() and d[0, 5].isnan().all()
    keep = torch.arange(70) != 5
    assert d[0, keep].isfinite().all()


def test_balance_unbatched_empty_and_autograd(dev):
    from mi355moe import router
    logits, ids, _, _ = make(1, 90, 33, 3, torch.float32, 11)
    x = logits[0].to(dev).requires_grad_()
    loss, counts = router.balance_loss(x, ids[0].to(dev))
    assert loss.shape == () and counts.shape == (33,)
    g, = torch.autograd.grad(loss * 3.0, x)
    ref = balance64(logits, ids, None, "softmax", torch.tensor([3.0]))
    close(g, ref[4][0], P_TOL * ref[5][0] + 2.0 ** -24 * ref[4][0].abs())
    for shape in ((0, 5), (2, 0, 5)):
        lg = torch.zeros(shape, device=dev, requires_grad=True)
        idd = torch.zeros(shape[:-1] + (2,), dtype=torch.int64, device=dev)
        loss, counts = router.balance_loss(lg, idd)
        assert (loss == 0).all() and (counts == 0).all()
        g, = torch.autograd.grad(loss.sum(), lg)
        assert g.shape == lg.shape


def test_balance_views_and_repeatability(dev):
    """Inputs that are views in another order, and twice the same result bit for bit."""
    from mi355moe import router
    logits, ids, dloss, _ = make(3, 500, 96, 4, torch.float32, 13)
    lg = logits.to(dev).transpose(0, 1).contiguous().transpose(0, 1)
    idd = torch.cat([ids, ids], 2).to(dev)[:, :, :4]
    assert not lg.is_contiguous() and not idd.is_contiguous()
    a = router.balance_loss_forward(lg, idd)
    b = router.balance_loss_forward(logits.to(dev), ids.to(dev))
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    da = router.balance_loss_backward(dloss.to(dev), lg, a[1], a[2], 4)
    db = router.balance_loss_backward(dloss.to(dev), logits.to(dev), b[1], b[2], 4)
    assert torch.equal(da, db)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_balance_gradient_against_differences(dev, score):
    """<gradient, v> against the central difference of the float64 loss along v (counts fixed)."""
    from mi355moe import router
    logits, ids, dloss, g = make(2, 60, 40, 3, torch.float32, 17)
    lg = logits.to(dev)
    _, counts, tokens, _ = router.balance_loss_forward(lg, ids.to(dev), score=score)
    d = router.balance_loss_backward(dloss.to(dev), lg, counts, tokens, 3, score=score).cpu().double()
    v = torch.randn(logits.shape, generator=g, dtype=torch.float64)
    h = 1e-5
    up = balance64(logits.double() + h * v, ids, None, score, dloss)[0]
    dn = balance64(logits.double() - h * v, ids, None, score, dloss)[0]
    want = ((up - dn) / (2 * h) * dloss.double()).sum()
    mag = balance64(logits, ids, None, score, dloss)[5]
    # differences: h^2 of the third derivative (below 1e-8 of the magnitudes) and 2^-52 / h of the loss
    tol = ((P_TOL + 1e-8) * (mag * v.abs()).sum() + 2.0 ** -52 / h * 4 * up.abs().sum())
    assert (d * v).sum() == pytest.approx(float(want), abs=float(tol))


# ------------------------------------------------------------------------------------------ router backward

def router64(x, gate, ids, w, dw, dlogits):
    """(dx, dgate, their sums of magnitudes, the error that D itself may have carried through) in float64."""
    x, gate, ids = x.cpu().double(), gate.cpu().double(), ids.cpu()
    T, E = x.shape[0], gate.shape[0]
    k = ids.shape[1]
    D = torch.zeros((T, E), dtype=torch.float64)
    err = torch.zeros((T, E), dtype=torch.float64)
    if dlogits is not None:
        D += dlogits.cpu().double()
    if dw is not None:
        w, dw = w.cpu().double(), dw.cpu().double()
        d = w * (dw - (w * dw).sum(1, keepdim=True))
        m = w.abs() * (dw.abs() + (w * dw).abs().sum(1, keepdim=True))
        ok = (ids >= 0) & (ids < E)
        at = torch.where(ok, ids, torch.zeros_like(ids))
        D.scatter_add_(1, at, torch.where(ok, d, torch.zeros_like(d)))
        err.scatter_add_(1, at, torch.where(ok, m, torch.zeros_like(m)))
    err = (k + 4) * 2.0 ** -24 * (err + D.abs())
    a = D.abs()
    return D @ gate, D.t() @ x, a @ gate.abs(), a.t() @ x.abs(), err @ gate.abs(), err.t() @ x.abs()


def check_router(x, gate, ids, w, dw, dlogits, dx, dgate):
    T, E = x.shape[0], gate.shape[0]
    rx, rg, mx, mg, ex, eg = router64(x, gate, ids, w, dw, dlogits)
    if dx is not None:
        assert dx.dtype == torch.bfloat16
        tol = 2.0 ** -8 * rx.abs() + (2.0 ** -15 + 3 * E * 2.0 ** -23) * mx + ex + 1e-37
        close(dx, rx, tol)
    if dgate is not None:
        tol = (3 * T + 64) * 2.0 ** -23 * mg + eg + 1e-37
        close(dgate, rg, tol)
        # as a random walk, the accumulation error is about sqrt(3 T) 2^-24 of the result's own size; eight times that
        if rg.norm() > 0:
            assert (dgate.cpu().double() - rg).norm() <= 8 * (3 * T + 64) ** 0.5 * 2.0 ** -24 * rg.norm() + eg.norm()


def router_inputs(T, H, E, k, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((T, H), generator=g).bfloat16()
    gate = torch.randn((E, H), generator=g) / H ** 0.5
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]) if T else torch.zeros((0, k), dtype=torch.int64)
    w = torch.softmax(torch.randn((T, k), generator=g), 1)
    dw, dl = torch.randn((T, k), generator=g), torch.randn((T, E), generator=g) * 0.1
    return [t.to(dev) for t in (x, gate, ids, w, dw, dl)]


@pytest.mark.parametrize("T,H,E,k", [(1, 256, 8, 2), (3, 16, 5, 1), (31, 2080, 40, 8), (33, 1024, 384, 8), (129, 4096, 200, 6),
                                     (300, 272, 1024, 32), (700, 512, 129, 4), (257, 128, 1, 1), (2100, 64, 33, 3)])
def test_router_backward(dev, T, H, E, k):
    from mi355moe import router
    x, gate, ids, w, dw, dl = router_inputs(T, H, E, k, T + H, dev)
    for a, b in ((dw, dl), (dw, None), (None, dl)):
        dx, dgate = router.topk_backward(x, gate, ids, w, a, b)
        check_router(x, gate, ids, w, a, b, dx, dgate)
    dx, none = router.topk_backward(x, gate, ids, w, dw, dl, need_gate=False)
    assert none is None
    only, dg = router.topk_backward(x, gate, ids, w, dw, dl, need_x=False)
    assert only is None
    both = router.topk_backward(x, gate, ids, w, dw, dl)
    assert torch.equal(both[0], dx) and torch.equal(both[1], dg)


def test_router_backward_odd_picks_and_no_tokens(dev):
    """Picks outside the experts, an expert picked twice, views and misaligned inputs, no tokens at all."""
    from mi355moe import router
    x, gate, ids, w, dw, dl = router_inputs(50, 96, 20, 4, 3, dev)
    ids[::4, 1] = -1
    ids[1::4, 2] = 20
    ids[2::4, 3] = ids[2::4, 0]
    dx, dgate = router.topk_backward(x, gate, ids, w, dw, dl)
    check_router(x, gate, ids, w, dw, dl, dx, dgate)
    xo = torch.empty(50 * 96 + 1, dtype=torch.bfloat16, device=dev)[1:].view(50, 96).copy_(x)
    go = gate.t().contiguous().t()
    dlo = torch.cat([dl, dl], 1)[:, :20]
    dx2, dgate2 = router.topk_backward(xo, go, ids, w, dw, dlo)
    assert torch.equal(dx, dx2) and torch.equal(dgate, dgate2)
    e = [t[:0] for t in (x, ids, w, dw, dl)]
    dx, dgate = router.topk_backward(e[0], gate, e[1], e[2], e[3], e[4])
    assert dx.shape == (0, 96) and dgate.shape == (20, 96) and (dgate == 0).all()


def test_router_backward_large_and_infinite_gradients(dev):
    """Gradients near the type's largest value keep their size; an infinite one stays infinite in its own row and columns."""
    from mi355moe import router
    x, gate, ids, w, dw, dl = router_inputs(40, 64, 16, 2, 5, dev)
    dl[7] = 0.0
    dl[7, 3] = 3.4e38
    gate[3] = 2.0 ** -4
    dx, _ = router.topk_backward(x, gate, ids, w, None, dl, need_gate=False)
    rx = router64(x, gate, ids, w, None, dl)[0]
    close(dx[7], rx[7], (2.0 ** -8 + 2.0 ** -15) * rx[7].abs())
    dl[7, 3] = torch.inf
    dx, _ = router.topk_backward(x, gate, ids, w, None, dl, need_gate=False)
    assert (dx[7] == torch.inf).all()
    keep = torch.arange(40) != 7
    assert dx.cpu()[keep].isfinite().all()


def loss_of(x, gate, ids, dw, coef, score):
    """sum dw * w + coef * balance, float64, as a function of x and gate at fixed picks."""
    logits = x @ gate.t()
    w = torch.softmax(logits.gather(1, ids), 1)
    E, (T, k) = gate.shape[0], ids.shape
    c = torch.bincount(ids.reshape(-1), minlength=E).double()
    p = torch.softmax(logits, 1) if score == "softmax" else torch.sigmoid(logits) / torch.sigmoid(logits).sum(1, keepdim=True)
    return (dw * w).sum() + coef * E / (k * T * T) * (c * p.sum(0)).sum()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_router_training_step_through_autograd(dev, score):
    """Top-k, balance loss and the sum of both losses through autograd, against float64 autograd at the same picks and against
    differences of the float64 loss."""
    from mi355moe import router
    T, H, E, k = 96, 256, 48, 4
    x, gate, _, _, dw, _ = router_inputs(T, H, E, k, 21, dev)
    x.requires_grad_()
    gate.requires_grad_()
    ids, w, logits = router.topk(x, gate, k)
    loss, counts = router.balance_loss(logits, ids, score=score)
    assert int(counts.sum()) == T * k
    gx, gg = torch.autograd.grad((dw * w).sum() + 10.0 * loss, (x, gate))
    x64, g64 = x.detach().cpu().double().requires_grad_(), gate.detach().cpu().double().requires_grad_()
    ic, dc = ids.cpu(), dw.cpu().double()
    total = loss_of(x64, g64, ic, dc, 10.0, score)
    rx, rg = torch.autograd.grad(total, (x64, g64))
    # logits (sums of H products) carry H 2^-23 into w and p, whose gradients' magnitudes are bounded by those of dw and 10 E / T
    D = dc.abs().max() * 2 + 10.0 * 2 * E / T
    tol = (H + 3 * max(T, E) + 64) * 2.0 ** -23
    mx, mg = D * g64.detach().abs().sum(0), D * x64.detach().abs().sum(0)
    close(gx, rx, 2.0 ** -8 * rx.abs() + (tol + 2.0 ** -15) * mx)
    close(gg, rg, tol * mg)
    v = torch.randn((E, H), generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    h = 1e-5
    with torch.no_grad():
        diff = (loss_of(x64, g64 + h * v, ic, dc, 10.0, score) - loss_of(x64, g64 - h * v, ic, dc, 10.0, score)) / (2 * h)
    assert (gg.cpu().double() * v).sum() == pytest.approx(float(diff), abs=float((tol * mg * v.abs()).sum() + 1e-4 * diff.abs()))


def test_router_step_in_a_graph_and_on_another_stream(dev):
    """Forward, loss and both backward passes captured (no eager autograd graph involved) and replayed with new inputs, with eager work in
    between; and the same on a side stream."""
    from mi355moe import router
    T, H, E, k = 200, 512, 64, 4

    def step(x, gate, dw, dl):
        ids, w, logits = router.topk_forward(x, gate, k)
        loss, counts, tokens, _ = router.balance_loss_forward(logits, ids)
        d = router.balance_loss_backward(dl, logits, counts, tokens, k)
        dx, dg = router.topk_backward(x, gate, ids, w, dw, d)
        return ids, loss, counts, d, dx, dg

    def inputs(seed):
        x, gate, _, _, dw, _ = router_inputs(T, H, E, k, seed, dev)
        return x, gate, dw, torch.tensor(0.5 + seed, device=dev)

    held = inputs(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*held)
    for seed in (2, 3, 4, 5):
        new = inputs(seed)
        for a, b in zip(held, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step(*new)
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
    new = inputs(6)
    torch.cuda.synchronize()
    ids, w, logits = router.topk_forward(new[0], new[1], k, stream=side)
    loss, counts, tokens, _ = router.balance_loss_forward(logits, ids, stream=side)
    d = router.balance_loss_backward(new[3], logits, counts, tokens, k, stream=side)
    dx, dg = router.topk_backward(new[0], new[1], ids, w, new[2], d, stream=side)
    side.synchronize()
    want = step(*new)
    for a, b in zip((ids, loss, counts, d, dx, dg), want):
        assert torch.equal(a, b)


def test_router_step_captured_through_autograd(dev):
    """topk and balance_loss with their backward passes captured (no eager graph of the leaves alive), replayed with new inputs."""
    from mi355moe import router
    T, H, E, k = 120, 256, 32, 4
    x, gate, _, _, dw, _ = router_inputs(T, H, E, k, 7, dev)
    x, gate = x.clone().requires_grad_(), gate.clone().requires_grad_()

    def step():
        ids, w, logits = router.topk(x, gate, k)
        loss, _ = router.balance_loss(logits, ids)
        return torch.autograd.grad([w, loss], [x, gate], [dw, torch.ones_like(loss)])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (8, 9, 10):
        nx, ng, _, _, nd, _ = router_inputs(T, H, E, k, seed, dev)
        with torch.no_grad():
            x.copy_(nx)
            gate.copy_(ng)
            dw.copy_(nd)
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
