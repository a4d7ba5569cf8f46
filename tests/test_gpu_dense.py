"""The layer on 16-bit experts (dense.moe, moe.moe_forward) with its gradients, alone and behind the router, against float64 autograd of
the definition; the grouped operators in captured graphs, on streams, and their gradients against differences.

Tolerances of the layer: between its kernels the gate and up rows, the weighted activation and the gradients are rounded to 16 bits. Each
such rounding is off by at most half a step (2^-8 for bf16, 2^-11 for fp16) of its value, and every result depends on a handful of them in
a row: as independent errors their relative sizes add as squares in the 2-norm, to less than sqrt(6) half steps for six roundings in a row
(x is exact; forward: 2 and the result's; weights' gradients: 5 and the result's, of which the activation's derivative may raise one by its
condition, below 4 here). The 2-norm of the error over a result is held to 8 half steps of its norm."""
import pytest
import torch

from test_gpu_grouped import BF, HALF, HF, picks, saved64, within

pytestmark = pytest.mark.gpu


def layer64(x, w, w13, w2, ids, limit, hold=None):
    """The layer in float64; `hold` maps the gate and up rows to what the backward pass sees of them (values only)."""
    E, _, I, H = w13.shape
    lim = limit or float("inf")
    flat = ids.reshape(-1)
    out = torch.zeros(x.shape, dtype=torch.float64)
    for e in range(E):
        r = (flat == e).nonzero()[:, 0]
        if not len(r):
            continue
        t = r // ids.shape[1]
        g, u = x[t] @ w13[e, 0].t(), x[t] @ w13[e, 1].t()
        if hold is not None:
            v = hold(torch.cat([g, u], 1))
            g, u = g + (v[:, :I] - g).detach(), u + (v[:, I:] - u).detach()
        h = (g * torch.sigmoid(g)).clamp(max=lim) * u.clamp(-lim, lim)
        out = out.index_add(0, t, (h * w.reshape(-1)[r][:, None]) @ w2[e].t())
    return out


def close(got, ref, half, steps=8):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape and got.isfinite().all()
    assert (got - ref).norm() <= steps * half * ref.norm() + 1e-30, ((got - ref).norm() / ref.norm() / half).item()


def tensors(g, T, k, E, H, I, dtype):
    x = torch.randn((T, H), generator=g).to(dtype)
    w13 = (torch.randn((E, 2, I, H), generator=g) / H ** 0.5).to(dtype)
    w2 = (torch.randn((E, H, I), generator=g) / I ** 0.5).to(dtype)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    ids[torch.rand((T, k), generator=g) < 0.1] = -1
    return x, w13, w2, ids, torch.rand((T, k), generator=g)


@pytest.mark.parametrize("T,k,E,H,I,dtype,limit,save8,shared", [
    (1, 2, 4, 64, 32, BF, 10.0, False, None), (37, 3, 7, 200, 72, HF, 10.0, False, 2), (150, 2, 4, 128, 96, BF, 1.0, True, None),
    (60, 4, 5, 256, 64, HF, 0.0, True, 4), (300, 1, 2, 72, 160, BF, 0.5, False, None)])
def test_layer_and_its_gradients(dev, T, k, E, H, I, dtype, limit, save8, shared):
    from mi355moe import dense, moe
    g = torch.Generator().manual_seed(T + H)
    x, w13, w2, ids, w = tensors(g, T, k, E, H, I, dtype)
    dout = torch.randn((T, H), generator=g).to(dtype).float()
    leaves = [t.to(dev).requires_grad_() for t in (x, w, w13, w2)]
    store = dense.DenseStore(leaves[2], leaves[3], limit=limit, save8=save8)
    out = moe.moe_forward(store, leaves[0], ids.to(dev), leaves[1], shared_expert=shared)
    assert out.dtype == torch.float32
    got = torch.autograd.grad(out, leaves, dout.to(dev))
    ref = [t.double().requires_grad_() for t in (x, w, w13, w2)]
    all_ids, all_w = ids, ref[1]
    if shared is not None:
        all_ids = torch.cat([ids, torch.full((T, 1), shared)], 1)
        all_w = torch.cat([ref[1], torch.ones((T, 1)).double()], 1)
    half = HALF[dtype]
    ref_out = layer64(ref[0], all_w, ref[2], ref[3], all_ids, limit)
    close(out, ref_out.detach(), half)
    # The gradients are those of the held rows (in 16 bits, or 8 of those): a row's value whose rounding takes it across a clamp has another
    # derivative, not one near by. (At limit 0.5, 4 phi(0.5) 0.5 2^-8 = 0.3 % of N(0, 1) values lie that near to it, and with 38 % of the values
    # inside the clamp they are up to sqrt(0.007) = 22 half steps of the gradient's norm.)
    hold = lambda gu: saved64(gu.detach().to(dtype)) if save8 else gu.detach().to(dtype).double()      # noqa: E731
    for name, a, b in zip(("x", "w", "w13", "w2"), got, torch.autograd.grad(layer64(ref[0], all_w, ref[2], ref[3], all_ids, limit, hold), ref, dout.double())):
        print(f"layer T {T} gradient of {name}", flush=True)
        assert a.dtype == (torch.float32 if name == "w" else dtype)
        # (a value whose code differs by one, or that lies next to a clamp, moves whole steps of 2^-7: few of them)
        close(a, b, half, 8 if not save8 else 24)
    with torch.no_grad():
        assert torch.equal(dense.moe(store, leaves[0], ids.to(dev), leaves[1], shared_expert=shared), out)
    frozen = moe.moe_forward(dense.DenseStore(leaves[2].detach(), leaves[3].detach(), limit=limit, save8=save8), leaves[0].detach(), ids.to(dev),
                             leaves[1], shared_expert=shared)
    assert torch.equal(torch.autograd.grad(frozen, leaves[1], dout.to(dev))[0], got[1])


def test_training_step_through_the_router(dev):
    """Router, load-balance loss and experts in one graph: every gradient against float64 autograd with the router's own picks."""
    from mi355moe import dense, moe, router
    g = torch.Generator().manual_seed(11)
    T, H, I, E, k = 90, 128, 64, 6, 2
    x, w13, w2, _, _ = tensors(g, T, k, E, H, I, BF)
    gate = torch.randn((E, H), generator=g) / H ** 0.5
    target = torch.randn((T, H), generator=g)
    leaves = [t.to(dev).requires_grad_() for t in (x, gate, w13, w2)]
    ids, w, logits = router.topk(leaves[0], leaves[1], k)
    balance, counts = router.balance_loss(logits, ids)
    out = moe.moe_forward(dense.DenseStore(leaves[2], leaves[3]), leaves[0], ids, w)
    loss = (out * target.to(dev)).sum() + 3.0 * balance
    loss.backward()
    assert int(counts.sum()) == T * k
    ref = [t.double().requires_grad_() for t in (x, gate, w13, w2)]
    ids = ids.cpu()
    lg = ref[0] @ ref[1].t()
    picked = torch.softmax(lg.gather(1, ids), 1)
    f = torch.bincount(ids.reshape(-1), minlength=E).double()
    ref_loss = (layer64(ref[0], picked, ref[2], ref[3], ids, 10.0) * target.double()).sum() + 3.0 * E / (k * T * T) * (torch.softmax(lg, 1).sum(0) * f).sum()
    ref_loss.backward()
    for name, a, b in zip(("x", "gate", "w13", "w2"), leaves, ref):
        print(f"router step, gradient of {name}", flush=True)
        close(a.grad, b.grad, HALF[BF])


def test_products_gradients_are_differences(dev):
    """On small whole numbers every product and sum is exact: the change of <dy, y> with x and with w is the gradient's, to the bit."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(12)
    ids = picks(g, [3, 0, 17, 70], 2, 3)
    for gather, reduce in ((False, False), (True, False), (False, True)):
        T, k = ids.shape
        def whole(*shape):
            return torch.randint(-3, 4, shape, generator=g).float()
        x, dy, w = whole(T if gather else T * k, 40), whole(T if reduce else T * k, 24), whole(4, 24, 40)
        ex, ew = whole(*x.shape), whole(*w.shape)
        plan = grouped.Plan(ids.to(dev), 4)
        b = lambda t: t.to(BF).to(dev)           # noqa: E731
        y = lambda x, w: grouped.linear_forward(b(x), b(w), plan, gather, reduce, torch.float32).cpu().double()      # noqa: E731
        dx, dw = grouped.linear_backward(b(dy), b(x), b(w), plan, gather, reduce, dw_dtype=torch.float32)
        # of a linear form, the difference over w + e and w - e is twice its value at e
        lhs = (dy.double() * (y(x, w + ew) - y(x, w - ew))).sum()
        assert lhs == 2 * (dw.cpu().double() * ew.double()).sum()
        # dx is rounded to bf16 (8 bits): whole numbers up to 256 are exact, and multiples of 2 up to 512
        d = (dy.double() * (y(x + ex, w) - y(x - ex, w))).sum() - 2 * (dx.cpu().double() * ex.double()).sum()
        slack = 2 * ((dx.cpu().double().abs() > 256) * dx.cpu().double().abs() * 2.0 ** -8 * ex.abs().double()).sum()
        assert d.abs() <= slack


def test_activation_gradients_are_differences(dev):
    """Against central differences of the definition in float64 (error of the differences: h^2 / 6 of the third derivative, below 1e-8)."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(13)
    gu, dh, wt = torch.randn((5, 64), generator=g).to(BF), torch.randn((5, 32), generator=g).to(BF), torch.rand(5, generator=g)
    dgu, dwt, _ = grouped.swiglu_backward(dh.to(dev), gu.to(dev), weights=wt.to(dev), limit=1.5)

    def value(gu, wt):
        a, u = gu.chunk(2, 1)
        return (wt[:, None] * (a * torch.sigmoid(a)).clamp(max=1.5) * u.clamp(-1.5, 1.5) * dh.double()).sum(1)

    base, h = gu.double(), 1e-4
    ref = torch.empty_like(base)
    for c in range(64):
        e = torch.zeros(64).double()
        e[c] = h
        ref[:, c] = (value(base + e, wt.double()) - value(base - e, wt.double())) / (2 * h)
    a, u = base.chunk(2, 1)
    near = torch.cat([(a * torch.sigmoid(a) - 1.5).abs() < 1e-3, (u.abs() - 1.5).abs() < 1e-3], 1)
    within(torch.where(near.to(dev), 0.0, dgu.double()), torch.where(near, 0.0, ref), 2.0 ** -8 * ref.abs() + 2.0 ** -19 + 1e-6)
    within(dwt, value(base, torch.ones(5).double()), 1e-5 * dh.double().abs().sum(1))


def test_captured_and_replayed(dev):
    """Plan, products, activation and their gradients in one graph, replayed on other inputs between eager calls; no replay differs
    from the eager result in a bit. Two graphs captured from the same operators stay apart."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(14)
    T, k, E, H, I = 50, 2, 5, 128, 64
    x, w13, w2, ids, w = (t.to(dev) for t in tensors(g, T, k, E, H, I, BF))
    dout = torch.randn((T, H), generator=g).to(BF).to(dev)

    def step():
        plan = grouped.Plan(ids, E)
        gu = grouped.linear_forward(x, w13.flatten(1, 2), plan, gather=True)
        h, kept = grouped.swiglu_forward(gu, plan, w, save8=True)
        y = grouped.linear_forward(h, w2, plan, reduce=True)
        dh, d2 = grouped.linear_backward(dout, h, w2, plan, reduce=True)
        dgu, dw, again = grouped.swiglu_backward(dh, kept, plan, w, need_h=True)
        dx, d13 = grouped.linear_backward(dgu, x, w13.flatten(1, 2), plan, gather=True)
        return y, d2, dgu, dw, again, dx, d13

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for i in range(3):
        x.copy_(torch.randn(x.shape, generator=g))
        ids.copy_(torch.randint(-1, E, ids.shape, generator=g))
        dout.copy_(torch.randn(dout.shape, generator=g))
        want = [t.clone() for t in step()]
        for graph, outs in graphs:
            print(f"replay {i}", flush=True)
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_captured_training_step(dev):
    """The layer with autograd inside a capture; the same leaves with an eager graph alive are refused."""
    from mi355moe import dense
    g = torch.Generator().manual_seed(15)
    x, w13, w2, ids, w = (t.to(dev) for t in tensors(g, 40, 2, 4, 64, 32, BF))
    store = dense.DenseStore(w13.requires_grad_(), w2.requires_grad_())
    x.requires_grad_()

    def step():
        return torch.autograd.grad(dense.moe(store, x, ids, w).sum(), (x, w13, w2))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g))
        print(f"replay {i}", flush=True)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_captured_step_with_a_shared_expert(dev):
    """The routing weights as a leaf in 64 bits, beside a shared expert, inside a capture: their gradient has their type and shape."""
    from mi355moe import dense
    g = torch.Generator().manual_seed(17)
    x, w13, w2, ids, w = (t.to(dev) for t in tensors(g, 30, 2, 4, 64, 32, HF))
    store = dense.DenseStore(w13.requires_grad_(), w2)
    w = w.double().requires_grad_()

    def step():
        return torch.autograd.grad(dense.moe(store, x, ids, w, shared_expert=3).sum(), (w, w13))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    assert outs[0].dtype == torch.float64 and outs[0].shape == w.shape
    for i in range(3):
        x.copy_(torch.randn(x.shape, generator=g))
        print(f"replay {i}", flush=True)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_two_streams_at_once(dev):
    """Calls of one plan on two streams do not touch each other's workspaces."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(16)
    ids = picks(g, [200, 300, 0, 100], 4)
    T, k = ids.shape
    x, w = torch.randn((T * k, 256), generator=g).to(BF).to(dev), torch.randn((4, 512, 256), generator=g).to(BF).to(dev)
    dy = torch.randn((T, 512), generator=g).to(BF).to(dev)
    plan = grouped.Plan(ids.to(dev), 4)

    def calls():
        return [grouped.linear_forward(x, w, plan, reduce=True), *grouped.linear_backward(dy, x, w, plan, reduce=True)]

    want = calls()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(calls())
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)
