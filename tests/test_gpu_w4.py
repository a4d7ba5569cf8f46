"""Products with 4-bit weights, dense and as the routed experts of a layer, against float64.

Tolerances: every product is exact, a sum of K terms x (16 + q) s and x (16 + z) s passes through G + K / G + 16 fp32
roundings (within a group, over groups, over waves), each at most 2^-23 of the sum of the terms' magnitudes; results are
rounded once to their type (half a step). As a random walk the same roundings come to sqrt(G + K / G + 16) 2^-23 of the root of the sum
of squares, which the 2-norm of the error over all outputs is held to (twice)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def within(got, ref, tol):
    got = got.cpu().double()
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        tol = torch.as_tensor(tol).expand_as(ref)
        pytest.fail(f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[:4].tolist()}: {got[bad][:4].tolist()} for "
                    f"{ref[bad][:4].tolist()}, tolerance {tol[bad][:4].tolist()}")


def weights(g, N, K, group, zeros, sdtype=torch.float16, lead=()):
    """(q, scales, zeros) on the CPU."""
    q = torch.randint(-2 ** 31, 2 ** 31, lead + (N, K // 8), generator=g, dtype=torch.int64).to(torch.int32)
    s = ((0.5 + torch.rand(lead + (N, K // group), generator=g)) / (4.6 * K ** 0.5)).to(sdtype)
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


def dense64(q, s, z):
    """(w, the magnitudes 16 + q and 16 + z take part with) float64 [N, K]."""
    K = q.shape[-1] * 8
    v = ((q.long()[..., None] >> torch.arange(0, 32, 4)) & 15).flatten(-2).double()
    G = K // s.shape[-1]
    zz = (torch.full_like(s, 8.0).double() if z is None else z.double()).repeat_interleave(G, -1)
    ss = s.double().repeat_interleave(G, -1)
    return (v - zz) * ss, (32 + v + zz) * ss.abs()


def roundings(K, G):
    return G + K // G + 16


def to(dev, ts):
    return tuple(None if t is None else t.to(dev) for t in ts)


def check_linear(y, x, q, s, z):
    w, m = dense64(q, s, z)
    x = x.double()
    G = q.shape[-1] * 8 // s.shape[-1]
    ref, mag = x @ w.t(), x.abs() @ m.t()
    n = roundings(w.shape[1], G)
    half = HALF[y.dtype]
    d = (y.cpu().double() - ref).abs()
    within(y, ref, n * 2.0 ** -23 * mag + half * ref.abs() + (2.0 ** -25 if y.dtype == torch.float16 else 1e-37))
    rms = ((x ** 2) @ (m ** 2).t()).sum().sqrt()
    assert d.norm() <= 2 * n ** 0.5 * 2.0 ** -23 * rms + half * ref.norm() + 1e-6 * (y.dtype == torch.float16) * ref.numel() ** 0.5


@pytest.mark.parametrize("M,K,N,group,dtype,zeros,sdtype", [
    (1, 4096, 4096, 128, torch.bfloat16, False, torch.float16),
    (1, 128, 1, 128, torch.float32, True, torch.bfloat16),
    (3, 32, 17, 32, torch.float32, True, torch.float16),
    (5, 96, 100, 32, torch.bfloat16, True, torch.bfloat16),
    (16, 192, 48, 64, torch.float16, True, torch.float16),
    (17, 2080, 1000, 32, torch.float32, False, torch.float16),
    (32, 1088, 130, 64, torch.float32, True, torch.float16),
    (33, 1024, 512, 128, torch.float16, False, torch.bfloat16),
    (64, 640, 2304, 128, torch.float32, True, torch.float16),
    (65, 1344, 77, 64, torch.bfloat16, True, torch.float16),
    (130, 2304, 300, 32, torch.float32, True, torch.float16),
    (300, 512, 264, 128, torch.bfloat16, False, torch.float16)])
def test_linear(dev, M, K, N, group, dtype, zeros, sdtype):
    from mi355moe import w4
    g = torch.Generator().manual_seed(M + K + N)
    q, s, z = weights(g, N, K, group, zeros, sdtype)
    x = torch.randn((M, K), generator=g).to(dtype)
    W = w4.W4Matrix(*to(dev, (q, s, z)))
    check_linear(w4.linear(x.to(dev), W), x, q, s, z)
    check_linear(w4.linear(x.to(dev), W, out_dtype=torch.float32), x, q, s, z)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,K,N,group,dtype", [
    (100, 128, 300, 128, torch.bfloat16), (60, 160, 140, 32, torch.float16), (40, 384, 200, 64, torch.float32),
    (33, 640, 129, 128, torch.bfloat16), (64, 1216, 64, 64, torch.float16),
    (20000, 128, 100, 128, torch.bfloat16), (20000, 96, 70, 32, torch.float16), (6500, 448, 100, 64, torch.float32),
    (40000, 96, 64, 32, torch.bfloat16), (13000, 256, 50, 64, torch.float32)])
def test_linear_of_many_rows(dev, M, K, N, group, dtype, zeros):
    """Every split of the waves (by rows and columns), with fewer blocks of inputs than groups of waves, and K's last block cut."""
    from mi355moe import w4
    g = torch.Generator().manual_seed(M + K + N)
    q, s, z = weights(g, N, K, group, zeros, torch.bfloat16)
    x = torch.randn((M, K), generator=g).to(dtype)
    check_linear(w4.linear(x.to(dev), w4.W4Matrix(*to(dev, (q, s, z)))), x, q, s, z)


@pytest.mark.parametrize("group", [32, 64, 128])
def test_linear_every_weight_value_in_every_place(dev, group):
    """x = unit vectors picks single weights: 256 columns of every nibble value at every k, exact in fp32."""
    from mi355moe import w4
    g = torch.Generator().manual_seed(4)
    K, N = 256, 64
    q, s, z = weights(g, N, K, group, True)
    W = w4.W4Matrix(*to(dev, (q, s, z)))
    y = w4.linear(torch.eye(K).to(dev), W, out_dtype=torch.float32)
    w, _ = dense64(q, s, z)
    # (16 + q) - (16 + z) is exact, times one scale: one rounding
    within(y, w.t(), 2.0 ** -24 * w.t().abs())


def test_linear_views_ranks_and_empty(dev):
    from mi355moe import w4
    g = torch.Generator().manual_seed(5)
    q, s, z = weights(g, 200, 256, 64, True)
    W = w4.W4Matrix(*to(dev, (q, s, z)))
    x = torch.randn((6, 256), generator=g).bfloat16().to(dev)
    y = w4.linear(x, W)
    off = torch.empty(6 * 256 + 1, dtype=torch.bfloat16, device=dev)[1:].view(6, 256).copy_(x)
    wide = torch.cat([x, x], 1)[:, :256]
    assert torch.equal(w4.linear(off, W), y) and torch.equal(w4.linear(wide, W), y)
    assert torch.equal(w4.linear(x.view(2, 3, 256), W), y.view(2, 3, 200))
    assert torch.equal(w4.linear(x[2], W), w4.linear(x[2:3], W)[0])
    assert w4.linear(x[:0], W).shape == (0, 200)


def test_linear_infinities_and_nan_stay_in_their_rows_and_columns(dev):
    from mi355moe import w4
    g = torch.Generator().manual_seed(6)
    q, s, z = weights(g, 70, 256, 64, True)
    s[5, 2] = torch.inf
    s[9, 0] = float("nan")
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn((20, 256), generator=g).to(dtype)
        x[3, 100] = float("nan")
        y = w4.linear(x.to(dev), w4.W4Matrix(*to(dev, (q, s, z))), out_dtype=torch.float32).cpu()
        assert not y[:, 5].isfinite().any() and y[:, 9].isnan().all() and y[3].isnan().all()
        rows = [i for i in range(20) if i != 3]
        cols = [j for j in range(70) if j not in (5, 9)]
        w, _ = dense64(q, s, z)
        assert y[rows][:, cols].isfinite().all()


def test_linear_large_and_small_fp32_inputs(dev):
    """fp32 inputs are used to their last bit: magnitudes from 1e-20 to 1e20 and a value whose bits fill all three parts."""
    from mi355moe import w4
    g = torch.Generator().manual_seed(8)
    q, s, z = weights(g, 33, 128, 32, False)
    x = torch.randn((4, 128), generator=g) * torch.tensor([1e-20, 1.0, 1e20, 1.0])[:, None]
    x[3] = 1.0 + 2.0 ** -23
    check_linear(w4.linear(x.to(dev), w4.W4Matrix(*to(dev, (q, s, z)))), x, q, s, z)


# ------------------------------------------------------------------------------------------ routed experts

def make_store(g, E, H, I, group, zeros, dev, limit=10.0, sdtype=torch.float16):
    from mi355moe import w4
    a = weights(g, I, H, group, zeros, sdtype, (E, 2))
    b = weights(g, H, I, group, zeros, sdtype, (E,))
    return w4.W4Store(*to(dev, a), *to(dev, b), limit=limit), a, b


def experts64(a, b, x, ids, w, shared, limit):
    """(out, error bound) float64: sum_j w expert(x), the roundings of gate and up carried through the activation."""
    E, H = b[0].shape[:2]
    I = a[0].shape[2]
    T = x.shape[0]
    ids, w = ids.clone(), w.double()
    if shared is not None:
        ids = torch.cat([ids, torch.full((T, 1), shared)], 1)
        w = torch.cat([w, torch.ones((T, 1), dtype=torch.float64)], 1)
    x = x.double()
    out, err = torch.zeros((T, H), dtype=torch.float64), torch.zeros((T, H), dtype=torch.float64)
    G = H // a[1].shape[-1]
    n13, n2 = roundings(H, G) * 2.0 ** -23, roundings(I, G) * 2.0 ** -23
    for e in torch.unique(ids).tolist():
        if not 0 <= e < E:
            continue
        t, j = (ids == e).nonzero(as_tuple=True)
        W = [dense64(a[0][e, i], a[1][e, i], None if a[2] is None else a[2][e, i]) for i in (0, 1)]
        g, u = x[t] @ W[0][0].t(), x[t] @ W[1][0].t()
        eg, eu = n13 * (x[t].abs() @ W[0][1].t()), n13 * (x[t].abs() @ W[1][1].t())
        act, uc = g * torch.sigmoid(g), u
        if limit:
            act, uc = act.clamp(max=limit), u.clamp(-limit, limit)
        h = act * uc
        # |silu'| <= 1.1; expf, the quotient and the product: 8 roundings
        eh = 1.1 * eg * (uc.abs() + eu) + act.abs() * eu + 8 * 2.0 ** -24 * h.abs()
        w2, m2 = dense64(b[0][e], b[1][e], None if b[2] is None else b[2][e])
        y = h @ w2.t()
        ey = eh @ w2.abs().t() + n2 * ((h.abs() + eh) @ m2.t())
        for row, (tt, jj) in enumerate(zip(t.tolist(), j.tolist())):
            out[tt] += w[tt, jj] * y[row]
            err[tt] += w[tt, jj].abs() * (ey[row] + (ids.shape[1] + 1) * 2.0 ** -24 * y[row].abs())
    return out, err


def check_experts(out, a, b, x, ids, w, shared, limit):
    ref, err = experts64(a, b, x.cpu(), ids.cpu(), w.cpu(), shared, limit)
    d = (out.cpu().double() - ref).abs()
    assert out.dtype == torch.float32
    within(out, ref, err + 1e-37)
    # the bound is the worst case of some 300 roundings; as a random walk they stay far below 2e-5 of the layer's output
    assert d.norm() <= 2e-5 * ref.norm() + 1e-30


@pytest.mark.parametrize("T,k,E,H,I,group,dtype,zeros,shared", [
    (1, 1, 1, 128, 128, 128, torch.bfloat16, False, None),
    (1, 8, 16, 512, 256, 128, torch.bfloat16, False, 15),
    (4, 8, 24, 256, 384, 64, torch.float32, True, 3),
    (7, 6, 12, 320, 96, 32, torch.float16, True, None),
    (8, 8, 8, 256, 128, 64, torch.bfloat16, True, None),
    (32, 2, 3, 256, 160, 32, torch.float32, False, None),
    (40, 1, 2, 128, 128, 128, torch.float16, True, 0),
    (64, 1, 4, 128, 64, 64, torch.bfloat16, False, None),
    (65, 1, 40, 128, 96, 32, torch.float32, True, None),
    (130, 4, 20, 192, 128, 64, torch.bfloat16, True, 19),
    (200, 3, 5, 256, 128, 128, torch.float16, False, None),
    (300, 8, 9, 128, 256, 128, torch.float32, True, 2),
    (900, 6, 300, 64, 64, 32, torch.bfloat16, False, None),
    (2400, 7, 30, 64, 64, 64, torch.float32, True, 4),
    (8300, 2, 12, 64, 32, 32, torch.bfloat16, False, 0)])
def test_experts(dev, T, k, E, H, I, group, dtype, zeros, shared):
    from mi355moe import moe
    g = torch.Generator().manual_seed(T + E + H)
    store, a, b = make_store(g, E, H, I, group, zeros, dev, sdtype=torch.bfloat16 if E == 20 else torch.float16)
    x = torch.randn((T, H), generator=g).to(dtype)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    w = torch.softmax(torch.randn((T, k), generator=g), 1)
    out = moe.moe_forward(store, x.to(dev), ids.to(dev), w.to(dev), shared_expert=shared)
    check_experts(out, a, b, x, ids, w, shared, 10.0)
    again = moe.moe_forward(store, x.to(dev), ids.to(dev), w.to(dev), shared_expert=shared)
    assert torch.equal(out, again)


@pytest.mark.parametrize("T", [6, 64, 150])
@pytest.mark.parametrize("shared", [None, 2])
def test_experts_invalid_and_repeated_picks(dev, T, shared):
    """Picks outside the experts add nothing (tokens with none left give zeros), an expert picked twice by a token counts
    twice, all tokens on one expert, and no clamp."""
    from mi355moe import moe
    g = torch.Generator().manual_seed(31 + T)
    store, a, b = make_store(g, 6, 256, 128, 64, True, dev, limit=0.0)
    x = torch.randn((T, 256), generator=g).bfloat16()
    ids = torch.randint(-2, 9, (T, 5), generator=g)
    ids[0] = -1
    ids[1] = 4
    ids[2] = 6
    ids[3:, 2] = 1
    w = torch.rand((T, 5), generator=g)
    w[0] = float("nan")                                       # weights of no expert are not used
    out = moe.moe_forward(store, x.to(dev), ids.to(dev), w.to(dev), shared_expert=shared)
    w[0] = 0.0
    check_experts(out, a, b, x, ids, w, shared, 0.0)
    if shared is None:
        assert (out[0] == 0).all() and (out[2] == 0).all()


def test_experts_types_strides_and_empty(dev):
    from mi355moe import moe
    g = torch.Generator().manual_seed(33)
    store, a, b = make_store(g, 6, 256, 128, 128, False, dev)
    x = torch.randn((5, 256), generator=g).half().to(dev)
    ids = torch.randint(0, 6, (5, 3), generator=g).to(dev)
    w = torch.rand((5, 3), generator=g).to(dev)
    out = moe.moe_forward(store, x, ids, w)
    off = torch.empty(5 * 256 + 1, dtype=torch.float16, device=dev)[1:].view(5, 256).copy_(x)
    assert torch.equal(moe.moe_forward(store, off, ids.int(), w.t().contiguous().t()), out)
    assert moe.moe_forward(store, x[:0], ids[:0], w[:0]).shape == (0, 256)
    with pytest.raises(ValueError, match="shared expert"):
        moe.moe_forward(store, x, ids, w, shared_expert=6)
    with pytest.raises(ValueError, match="expected"):
        moe.moe_forward(store, x[:, :128], ids, w)
    with pytest.raises(TypeError):
        moe.moe_forward(store, x.double(), ids, w)
    with pytest.raises(ValueError, match="is on cpu"):
        moe.moe_forward(store, x, ids.cpu(), w)


def test_router_and_experts_in_a_graph(dev):
    """Router top-k into the 4-bit experts and a dense 4-bit product, captured and replayed with new inputs; two calls of other
    sizes and a side stream in between."""
    from mi355moe import moe, router, w4
    g = torch.Generator().manual_seed(41)
    H, I, E, k = 512, 256, 16, 4
    store, a, b = make_store(g, E, H, I, 128, True, dev)
    W = w4.W4Matrix(*to(dev, weights(g, 96, H, 128, False)))
    gate = (torch.randn((E, H), generator=g) / H ** 0.5).to(dev)

    def step(x):
        ids, w, _ = router.topk_forward(x, gate, k)
        out = moe.moe_forward(store, x, ids, w, shared_expert=1)
        return ids, w, out, w4.linear(out, W)

    for T in (3, 40):
        x = torch.randn((T, H), generator=g).bfloat16().to(dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(x)
        for i in range(4):
            new = torch.randn((T, H), generator=g).bfloat16().to(dev)
            x.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            want = step(new)
            torch.cuda.synchronize()
            for p, q in zip(outs, want):
                assert torch.equal(p, q)
            check_experts(outs[2], a, b, new, outs[0], outs[1], 1, 10.0)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            moe.moe_forward(store, new, want[0], want[1], shared_expert=1)
        y = moe.moe_forward(store, new, want[0], want[1], shared_expert=1, stream=side)
        side.synchronize()
        assert torch.equal(y, want[2])


# ------------------------------------------------------------------------------------------ odd values, equal rows

def alike(got, ref, tol):
    """Same infinities and NaN, the rest within tol."""
    got = got.cpu().double()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got == torch.inf, ref == torch.inf)
    assert torch.equal(got == -torch.inf, ref == -torch.inf)
    ok = ref.isfinite()
    within(got[ok], ref[ok], tol[ok])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M", [1, 20, 70])
def test_linear_an_infinite_or_largest_input_gives_what_the_formula_gives(dev, M, dtype):
    """One infinite input: +-inf by the weight's sign, NaN where the weight is zero; one input of fp32's largest: finite. Outputs summed
    again have K roundings of 2^-24 of sum |x w|, less than the tolerance of the others (|q - z| <= 15, against 32 + q + z)."""
    from mi355moe import w4
    g = torch.Generator().manual_seed(M)
    q, s, z = weights(g, 150, 256, 64, True)
    x = torch.randn((M, 256), generator=g).to(dtype)
    x[0, 77] = -torch.inf
    if M > 1:
        x[M - 1, 200] = torch.finfo(dtype).max
    y = w4.linear(x.to(dev), w4.W4Matrix(*to(dev, (q, s, z))), out_dtype=torch.float32)
    w, m = dense64(q, s, z)
    ref = torch.stack([(x[i].double() * w).sum(1) for i in range(M)])
    alike(y, ref, 84 * 2.0 ** -23 * (x.double().abs() @ m.t()) + HALF[torch.float32] * ref.abs())


@pytest.mark.parametrize("T,k,E", [(3, 2, 6), (40, 2, 6), (90, 3, 6)])
def test_experts_odd_tokens_stay_alone(dev, T, k, E):
    """A token with NaN gives NaN (no clamp hides it); the others are as without it."""
    from mi355moe import moe
    g = torch.Generator().manual_seed(T)
    store, a, b = make_store(g, E, 128, 64, 64, True, dev, limit=2.0)
    x = torch.randn((T, 128), generator=g).bfloat16()
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    w = torch.rand((T, k), generator=g) + 0.1
    plain = moe.moe_forward(store, x.to(dev), ids.to(dev), w.to(dev))
    y = x.clone()
    y[0, 5] = float("nan")
    out = moe.moe_forward(store, y.to(dev), ids.to(dev), w.to(dev))
    assert out[0].isnan().all() and torch.equal(out[1:], plain[1:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,E,most", [(80, 16, 17), (80, 16, 33), (130, 20, 65), (200, 20, 40), (190, 20, 65), (700, 20, 130)])
def test_experts_equal_tokens_get_equal_results(dev, T, E, most, group, dtype):
    """Tokens that are equal and go to one expert get the same bits, in whichever row and record they come: the order of an expert's
    routes is not fixed, the results are."""
    from mi355moe import moe
    g = torch.Generator().manual_seed(T + most)
    store, a, b = make_store(g, E, 256, 128, group, True, dev)
    x = torch.randn((T, 256), generator=g).to(dtype)
    x[:most] = x[0]
    ids = torch.randint(1, E, (T, 1), generator=g)
    ids[:most] = 0
    w = torch.ones((T, 1))
    out = moe.moe_forward(store, x.to(dev), ids.to(dev), w.to(dev))
    assert torch.equal(out[:most], out[:1].expand(most, -1))
    check_experts(out, a, b, x, ids, w, None, 10.0)


def test_experts_picks_and_weights_must_match(dev):
    from mi355moe import w4
    g = torch.Generator().manual_seed(3)
    store, _, _ = make_store(g, 4, 128, 64, 64, False, dev)
    x, ids, w = torch.randn((2, 128)).to(dev), torch.zeros((2, 3), dtype=torch.int64, device=dev), torch.zeros((2, 3), device=dev)
    for bad in ((ids, w.t()), (ids, w[:, :2]), (ids[:, :0], w[:, :0]), (ids[:1, :1], w[:1, :1])):
        with pytest.raises(ValueError, match="ids and w"):
            w4.moe(store, x, *bad)
