"""Products grouped by expert, the gated activation between them with its 8-bit form, and the layer they make, against float64.

Tolerances: products of 16-bit values are exact in fp32. A sum of K terms passes through at most K fp32 roundings, each at most 2^-23 of the
sum of the terms' magnitudes, whatever the order (matrix cores may truncate: a whole unit instead of a half); as a random walk the same
roundings come to sqrt(K) 2^-23 of the root of the sum of squares, which the 2-norm of the error over all outputs is held to (twice).
Results are rounded once to their type (half a step, and half the smallest subnormal). Rows that are summed per token into bf16 are kept in between
in 11 bits under a power of two per 32 columns: off by at most 2^-11 of themselves (half a step of fp16), and by half of fp16's smallest subnormal where
the largest of the 32 is at least 2^14 times it: 2^-25 / 2^14 of that largest."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
BF, HF = torch.bfloat16, torch.float16


def within(got, ref, tol):
    got = got.cpu().double()
    bad = ~((got - ref).abs() <= tol)
    if bad.any():
        tol = torch.as_tensor(tol).expand_as(ref)
        pytest.fail(f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[:4].tolist()}: {got[bad][:4].tolist()} for "
                    f"{ref[bad][:4].tolist()}, tolerance {tol[bad][:4].tolist()}")


def picks(g, counts, k=1, none=0):
    """ids [T, k] with counts[e] picks of expert e and `none` of none, in random places (a token may pick an expert twice)."""
    flat = torch.cat([torch.full((c,), e) for e, c in enumerate(counts)] + [torch.tensor([-1, len(counts), -7, 10 ** 9] * none)[:none]]).long()
    flat = torch.cat([flat, torch.full((-len(flat) % k,), -1)])
    return flat[torch.randperm(len(flat), generator=g)].view(-1, k)


def order_of(ids, E):
    """(flat routes in the plan's order, expert of each of its rows) by the definition."""
    flat = ids.reshape(-1)
    e = torch.where((flat >= 0) & (flat < E), flat, E)
    order = torch.argsort(e, stable=True)
    return order, e[order]


def products(x, dy, w, ids, gather, reduce):
    """{forward, inputs, weights: (result, sum of magnitudes, root of the sum of squares, terms)} in float64."""
    E, N, K = w.shape
    T, k = ids.shape
    order, expert = order_of(ids, E)
    token = order // k
    x, dy, w = x.double(), dy.double(), w.double()
    xr, dr = x[token] if gather else x, dy[token] if reduce else dy

    def all_(x, dy, w):
        y, dx, dw = torch.zeros((T * k, N)).double(), torch.zeros((T * k, K)).double(), torch.zeros((E, N, K)).double()
        for e in range(E):
            r = (expert == e).nonzero()[:, 0]
            y[r], dx[r], dw[e] = x[r] @ w[e].t(), dy[r] @ w[e], dy[r].t() @ x[r]
        sums = lambda v: torch.zeros((T, v.shape[1])).double().index_add_(0, token, v)       # noqa: E731
        return sums(y) if reduce else y, sums(dx) if gather else dx, dw
    live = (expert < E)[:, None]
    xr, dr = torch.where(live, xr, 0.0), torch.where(live, dr, 0.0)
    res, mag = all_(xr, dr, w), all_(xr.abs(), dr.abs(), w.abs())
    sq = [v.sqrt() for v in all_(xr ** 2, dr ** 2, w ** 2)]
    most = int(torch.bincount(expert[expert < E], minlength=E).max()) if E else 0
    terms = (K + k, N + k, max(most, 1))
    # what the rows that are summed per token may be off by as they are kept
    rows = [None, None, None]
    if (reduce or gather) and w.dtype == torch.float64 and T * k > 16:
        each = torch.zeros((T * k, N if reduce else K)).double()
        for e in range(E):
            r = (expert == e).nonzero()[:, 0]
            each[r] = xr[r] @ w[e].t() if reduce else dr[r] @ w[e]
        rows[0 if reduce else 1] = torch.zeros((T, each.shape[1])).double().index_add_(0, token, 2.0 ** -11 * each.abs() + 2.0 ** -39 * each.abs().amax(1, keepdim=True))
    return dict(zip(("forward", "inputs", "weights"), zip(res, mag, sq, terms, rows)))


def check(got, want):
    ref, mag, sq, terms, rows = want
    half, tiny = HALF[got.dtype], TINY[got.dtype]
    kept = rows if rows is not None and got.dtype == BF else torch.zeros(1).double()
    assert got.shape == ref.shape
    within(got, ref, terms * 2.0 ** -23 * mag + half * (ref.abs() + kept) + kept + tiny)
    err = (got.cpu().double() - ref).norm()
    assert err <= 2 * terms ** 0.5 * 2.0 ** -23 * sq.norm() + half * (ref.norm() + kept.norm()) + kept.norm() + tiny * ref.numel() ** 0.5


def inputs(g, ids, E, K, N, dtype, gather, reduce):
    T, k = ids.shape
    x = torch.randn((T if gather else T * k, K), generator=g).to(dtype)
    dy = torch.randn((T if reduce else T * k, N), generator=g).to(dtype)
    w = (torch.randn((E, N, K), generator=g) / K ** 0.5).to(dtype)
    return x, dy, w


def run_all(dev, x, dy, w, ids, gather, reduce, out_dtype=None, stream=None):
    from mi355moe import grouped
    xd, dyd, wd = x.to(dev), dy.to(dev), w.to(dev)
    plan = grouped.Plan(ids.to(dev), w.shape[0])
    y = grouped.linear_forward(xd, wd, plan, gather, reduce, out_dtype)
    dx, dw = grouped.linear_backward(dyd, xd, wd, plan, gather, reduce, dw_dtype=out_dtype)
    return {"forward": y, "inputs": dx, "weights": dw}


COUNTS = {"edges": [0, 1, 15, 16, 17, 0, 31, 32, 33, 63, 64, 65, 2], "tiles": [127, 128, 129, 0, 255, 256, 257], "long": [5, 800, 0, 301],
          "sizes": [90, 97, 128, 129, 150, 161, 180, 193, 210, 225, 256, 257, 5, 300, 20, 700, 40], "few": [1, 0, 0, 2, 1], "one": [0, 0, 1], "none": [0, 0]}


@pytest.mark.parametrize("rows,k,none,K,N,dtype,gather,reduce", [
    ("edges", 1, 0, 64, 256, BF, False, False),
    ("edges", 2, 5, 200, 264, HF, True, False),
    ("edges", 3, 4, 72, 520, BF, False, True),
    ("tiles", 1, 9, 136, 248, HF, False, False),
    ("tiles", 4, 0, 320, 24, BF, True, False),
    ("tiles", 8, 3, 8, 512, HF, False, True),
    ("long", 2, 300, 264, 136, BF, True, False),
    ("long", 5, 1, 1032, 8, HF, False, True),
    # enough large tiles for every form of them: of columns forward, of inputs backward
    ("sizes", 1, 5, 72, 4096, BF, False, False),
    ("sizes", 2, 300, 4096, 72, HF, True, False),
    ("sizes", 3, 4, 200, 3848, HF, False, True),
    ("sizes", 4, 1, 3848, 136, BF, False, True),
    ("few", 1, 0, 1024, 512, BF, True, False),
    ("few", 2, 1, 512, 1024, HF, False, True),
    ("one", 1, 0, 8, 8, BF, False, False),
    ("none", 2, 6, 64, 64, BF, True, False),
    ("none", 2, 6, 64, 64, HF, False, True)])
def test_products(dev, rows, k, none, K, N, dtype, gather, reduce):
    g = torch.Generator().manual_seed(K + N + k)
    counts = COUNTS[rows]
    ids = picks(g, counts, k, none)
    x, dy, w = inputs(g, ids, len(counts), K, N, dtype, gather, reduce)
    want = products(x, dy, w, ids, gather, reduce)
    for out in (None, torch.float32):
        print(f"products {rows} K {K} N {N} out {out}", flush=True)
        for name, got in run_all(dev, x, dy, w, ids, gather, reduce, out).items():
            check(got, want[name])


@pytest.mark.parametrize("T,k,E,K,N", [(1, 1, 1, 64, 64), (1, 8, 384, 512, 256), (3, 2, 1024, 64, 72), (700, 6, 64, 128, 320), (5000, 2, 9, 64, 64),
                                         (1024, 4, 384, 64, 64), (1025, 4, 1024, 8, 16), (4096, 1, 1, 8, 8), (4097, 1, 1, 8, 8), (127, 9, 1023, 16, 8), (65, 1, 512, 8, 8),
                                         (40000, 8, 1024, 8, 8), (131073, 1, 3, 8, 8), (16384, 8, 384, 8, 16)])
def test_plan(dev, T, k, E, K, N):
    """The order by its definition, for one kernel's calls and for many; picks of none last."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(T + E)
    ids = torch.randint(-1, E + 1, (T, k), generator=g)
    plan = grouped.Plan(ids.to(dev), E)
    order, expert = order_of(ids, E)
    assert torch.equal(plan.order.cpu().long(), order) and torch.equal(plan.token.cpu().long(), order // k)
    assert torch.equal(plan.inv.cpu().long()[order], torch.arange(T * k))
    counts = torch.bincount(expert, minlength=E + 1)[:E]
    assert torch.equal(plan.counts.cpu().long(), counts)
    assert torch.equal(plan.offsets.cpu().long(), torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]))
    x, dy, w = inputs(g, ids, E, K, N, BF, True, False)
    want = products(x, dy, w, ids, True, False)
    for name, got in run_all(dev, x, dy, w, ids, True, False).items():
        check(got, want[name])


def test_what_belongs_to_no_expert_takes_no_part(dev):
    """NaN in rows of no expert, in the weights of experts without rows, and in tokens without picks reaches nothing."""
    g = torch.Generator().manual_seed(3)
    counts = [3, 0, 40, 300]
    for gather, reduce in ((False, False), (True, False), (False, True)):
        ids = picks(g, counts, 1, 30)
        x, dy, w = inputs(g, ids, 4, 200, 264, BF, gather, reduce)
        clean = run_all(dev, x, dy, w, ids, gather, reduce)
        order, expert = order_of(ids, 4)
        dead = (expert == 4).nonzero()[:, 0]
        x[order[dead] if gather else dead] = float("nan")
        dy[order[dead] if reduce else dead] = float("nan")
        w[1] = float("nan")
        for name, got in run_all(dev, x, dy, w, ids, gather, reduce).items():
            assert torch.equal(got, clean[name]), (name, gather, reduce)


def test_infinite_and_nan_rows_stay_their_own(dev):
    from mi355moe import grouped
    g = torch.Generator().manual_seed(4)
    ids = picks(g, [20, 100])
    x, _, w = inputs(g, ids, 2, 72, 64, HF, False, False)
    plan, wd = grouped.Plan(ids.to(dev), 2), w.to(dev)
    clean = grouped.linear_forward(x.to(dev), wd, plan)
    x[5, 3], x[50, 71], x[119, 0] = float("inf"), float("nan"), -float("inf")
    got = grouped.linear_forward(x.to(dev), wd, plan)
    rows = torch.tensor([r for r in range(120) if r not in (5, 50, 119)])
    assert torch.equal(got[rows.to(dev)], clean[rows.to(dev)])
    ref = torch.sign(w[0][:, 3].float()) * float("inf")
    assert torch.equal(got[5].cpu().float(), ref) and got[50].isnan().all() and got[119].isinf().all()


def test_summed_rows_of_all_sizes(dev):
    """Rows kept between product and sum: columns 2^60 apart, rows of zeros, values at bf16's ends, an infinity beside large finite values."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(5)
    ids = picks(g, [30, 50], 2)
    T = ids.shape[0]
    x, w = torch.randn((2 * T, 64), generator=g).to(BF), torch.randn((2, 200, 64), generator=g)
    w *= 2.0 ** torch.randint(-30, 31, (2, 200, 1), generator=g)
    w[:, 40:80] = 0
    x[:8] *= 2.0 ** -90
    x[8:12] *= 2.0 ** 90
    w = w.to(BF)
    plan = grouped.Plan(ids.to(dev), 2)
    y = grouped.linear_forward(x.to(dev), w.to(dev), plan, reduce=True)
    dy = torch.zeros((T, 200)).to(BF)
    check(y, products(x, dy, w, ids, False, True)["forward"])
    w[0, 3, 5] = float("inf")
    y = grouped.linear_forward(x.to(dev), w.to(dev), plan, reduce=True).cpu()
    rows = grouped.linear_forward(x.to(dev), w.to(dev), plan, out_dtype=torch.float32).cpu()
    want = torch.zeros((T, 200)).index_add_(0, order_of(ids, 2)[0] // 2, rows)
    assert torch.equal(y.isfinite(), want.to(BF).isfinite()) and torch.equal(y.isnan(), want.isnan())


def test_products_repeat_and_take_views(dev):
    """Same bits on every call, from strided and misaligned rows too, and on another stream than the tensors'."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(6)
    ids = picks(g, [70, 3, 200], 3, 2)
    x, dy, w = (t.to(dev) for t in inputs(g, ids, 3, 136, 72, BF, True, False))
    plan = grouped.Plan(ids.to(dev), 3)
    first = grouped.linear_forward(x, w, plan, gather=True), *grouped.linear_backward(dy, x, w, plan, gather=True)
    wide = torch.zeros((x.shape[0], 2 * 136 + 1), dtype=BF, device=dev)
    wide[:, 1:137] = x
    odd = torch.zeros(dy.numel() + 1, dtype=BF, device=dev)
    odd[1:] = dy.reshape(-1)
    xs, dys = wide[:, 1:137], odd[1:].view_as(dy)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    again = grouped.linear_forward(xs, w, plan, gather=True, stream=s), *grouped.linear_backward(dys, xs, w, plan, gather=True, stream=s)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_no_tokens(dev):
    from mi355moe import dense, grouped
    plan = grouped.Plan(torch.zeros((0, 3), dtype=torch.int64, device=dev), 4)
    w = torch.ones((4, 16, 8), dtype=BF, device=dev)
    x, dy = torch.ones((0, 8), dtype=BF, device=dev), torch.ones((0, 16), dtype=BF, device=dev)
    assert grouped.linear_forward(x, w, plan).shape == (0, 16) and plan.offsets.tolist() == [0] * 5
    dx, dw = grouped.linear_backward(dy, x, w, plan)
    assert dx.shape == (0, 8) and not dw.any() and dw.shape == w.shape
    h, _ = grouped.swiglu_forward(dy, plan)
    assert h.shape == (0, 8)
    st = dense.DenseStore(torch.ones((4, 2, 16, 8), dtype=BF, device=dev), torch.ones((4, 8, 16), dtype=BF, device=dev))
    assert dense.moe(st, x, torch.zeros((0, 2), dtype=torch.int64, device=dev), torch.zeros((0, 2), device=dev)).shape == (0, 8)


# ------------------------------------------------------------------------------------------ activation

LIMIT = 10.0


def act64(gu, limit):
    g, u = gu.double().chunk(2, 1)
    s, lim = torch.sigmoid(g), limit or float("inf")
    return g, u, s, (g * s).clamp(max=lim), u.clamp(-lim, lim), lim


def saved64(gu):
    """gu as 8 bits hold it, by the definition: the exponent found by trying."""
    x = gu.double().unflatten(1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(top, -126.0)
    for _ in range(300):
        e = torch.where(top > 127 * 2.0 ** e, e + 1, e)
    return (torch.round(x / 2.0 ** e) * 2.0 ** e).flatten(1)


def gated64(gu, dh, w, live, limit, kept=None):
    """(h, dgu, dweights per row, h again) in float64 with the magnitudes their tolerances count."""
    g, u, s, a, c, lim = act64(gu, limit)
    h = w * a * c
    g, u, s, a, c, lim = act64(gu if kept is None else kept, limit)
    d = w * dh.double()
    dg = torch.where(g * s <= lim, d * c * (s * (1 + g * (1 - s))), 0.0)
    du = torch.where(u.abs() <= lim, d * a, 0.0)
    # silu' = s (1 + g (1 - s)) cancels near its zero: its magnitude without the cancellation
    mag = torch.cat([(d * c * s).abs() * (1 + g.abs() * (1 - s)), (d * a).abs()], 1)
    return h, torch.cat([dg, du], 1), torch.where(live, dh.double() * a * c, 0.0), mag, w * a * c


# a sigmoid by v_exp_f32 and v_rcp_f32: |g| 2^-24 of the exponent's rounding (log2(e) g and its product), 2^-23 each of the two
# instructions, and the adds and products after it: within (|g| + 8) 2^-23
def act_error(gu):
    g = gu.double().chunk(2, 1)[0].abs()
    return (g + 8) * 2.0 ** -23


GATED = [(1, 1, 1, 8, BF, LIMIT, False, 0), (1, 8, 384, 2048, BF, LIMIT, True, 0), (40, 3, 5, 520, HF, LIMIT, True, 17), (70, 2, 9, 64, BF, 0.0, True, 3),
         (9, 4, 4, 2304, HF, 1.5, False, 5), (300, 1, 2, 32, BF, 0.25, True, 300), (5, 2, 3, 4128, BF, 7.0, True, 0)]


@pytest.mark.parametrize("T,k,E,I,dtype,limit,weighted,none,save8", [c + (s,) for s in (False, True) for c in GATED if not s or c[3] % 32 == 0])
def test_gated(dev, T, k, E, I, dtype, limit, weighted, none, save8):
    from mi355moe import grouped
    g = torch.Generator().manual_seed(T + I)
    n = T * k
    ids = torch.randint(0, E, (n,), generator=g)
    ids[torch.randperm(n, generator=g)[:none]] = -1
    ids = ids.view(T, k)
    gu = (3 * torch.randn((n, 2 * I), generator=g)).to(dtype)
    dh = torch.randn((n, I), generator=g).to(dtype)
    weights = torch.rand((T, k), generator=g) if weighted else None
    order, expert = order_of(ids, E)
    live = (expert < E)[:, None]
    w = (weights.reshape(-1, 1)[order].double() if weighted else torch.ones((n, 1)).double()) * live
    kept64 = saved64(gu) if save8 else None
    h64, dgu64, terms, mag, again64 = gated64(gu, dh, w, live, limit, kept64)
    plan = grouped.Plan(ids.to(dev), E)
    wd = None if weights is None else weights.to(dev)
    h, kept = grouped.swiglu_forward(gu.to(dev), plan, wd, limit, save8)
    half, tiny = HALF[dtype], TINY[dtype]
    within(h, h64, (half + act_error(gu) + 2.0 ** -22) * h64.abs() + tiny)
    if save8:
        values = kept.codes.cpu().double() * 2.0 ** kept.exps.cpu().double().repeat_interleave(32, 1)
        live2 = live.expand_as(values)
        assert torch.equal(values[live2], kept64[live2])
    dgu, dweights, again = grouped.swiglu_backward(dh.to(dev), kept, plan, wd, limit, need_h=True)
    src = gu if kept64 is None else kept64
    err = act_error(src)
    # a value within its error of a clamp may lie on the other side of it
    _, u, s, a, c, lim = act64(src, limit)
    gs = src.double().chunk(2, 1)[0] * s
    near = torch.cat([((gs - lim).abs() <= err * gs.abs()) & bool(limit), torch.zeros_like(gs, dtype=torch.bool)], 1)
    tol = half * dgu64.abs() + torch.cat([err, err], 1) * mag + 2.0 ** -22 * mag + tiny
    within(torch.where(near.to(dev), 0.0, dgu.double()), torch.where(near, 0.0, dgu64), tol)
    within(again, again64, (half + err + 2.0 ** -22) * again64.abs() + tiny)
    if weighted:
        dw64 = torch.zeros(n).double()
        dw64[order] = terms.sum(1)
        tol = torch.zeros(n).double()
        tol[order] = ((err + (I + 8) * 2.0 ** -24) * terms.abs()).sum(1)
        within(dweights.reshape(-1), dw64, tol + 2.0 ** -100)
    else:
        assert dweights is None
    alone, no = grouped.swiglu_backward(dh.to(dev), kept, plan, wd, limit, need_weights=False)[:2]
    assert no is None and torch.equal(alone, dgu)


def test_gated_without_a_plan(dev):
    from mi355moe import grouped
    g = torch.Generator().manual_seed(8)
    gu, weights = torch.randn((37, 64), generator=g).to(BF), torch.rand(37, generator=g)
    h, _ = grouped.swiglu_forward(gu.to(dev), weights=weights.to(dev), limit=0.0)
    h64 = gated64(gu, torch.zeros((37, 32)), weights.double()[:, None], torch.ones((37, 1), dtype=torch.bool), 0.0)[0]
    within(h, h64, (HALF[BF] + act_error(gu) + 2.0 ** -22) * h64.abs() + TINY[BF])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_8_bits_hold_what_they_say(dev, dtype):
    """Every exponent's edge: groups of zeros, of one value, next to 127 2^e, of the type's smallest and largest values, and
    groups with an infinity or NaN, which come back as NaN alone."""
    from mi355moe import grouped
    info = torch.finfo(dtype)
    tops = [0.0, 1.0, 127.0, 127.5, 128.0, 126.0, 2.0 ** -9, info.smallest_normal, info.smallest_normal * info.eps, info.max, 3.0, 63.5, 64.0]
    x = torch.zeros((len(tops) + 2, 64), dtype=torch.float64)
    for i, t in enumerate(tops):
        x[i, :32] = t * torch.linspace(-1, 1, 32).double()
        x[i, 32:] = t
    x[-2, 5], x[-1, 40] = float("inf"), float("nan")
    x = x.to(dtype)
    _, kept = grouped.swiglu_forward(x.to(dev), save8=True)
    codes, exps = kept.codes.cpu().double(), kept.exps.cpu().double().repeat_interleave(32, 1)
    values = torch.where(exps == 127, float("nan"), codes * 2.0 ** exps)
    fine = torch.ones_like(x, dtype=torch.bool)
    fine[-2, :32] = fine[-1, 32:] = False
    assert torch.equal(values[fine], saved64(torch.nan_to_num(x, 0.0, 0.0, 0.0))[fine]) and values[~fine].isnan().all()
    top = x.double().unflatten(1, (-1, 32)).abs().amax(-1, keepdim=True).expand(-1, -1, 32).flatten(1)
    assert ((values - x.double()).abs()[fine] <= (top / 127).clamp(min=2.0 ** -127)[fine]).all()
    dgu, _, _ = grouped.swiglu_backward(torch.ones((len(tops) + 2, 32), dtype=dtype, device=dev), kept)
    # a gate of NaN passes into du, an up of NaN into dg; their own derivatives are cut
    assert dgu[:-2].isfinite().all() and dgu[-2, 32:].isnan().all() and dgu[-1, :32].isnan().all()


def test_clamps_keep_nan_and_cut_gradients(dev):
    from mi355moe import grouped
    g = [12.0, -3.0, float("nan"), 2.0, 2.0, 10.0, 2.0, 2.0]
    u = [1.0, 11.0, 1.0, -11.0, float("nan"), 10.0, -10.0, 10.0]
    gu = torch.tensor([g + u]).to(BF).to(dev)
    h, kept = grouped.swiglu_forward(gu, limit=10.0)
    dgu, _, _ = grouped.swiglu_backward(torch.ones((1, 8), dtype=BF, device=dev), kept, limit=10.0)
    h, dg, du = h[0].cpu(), dgu[0, :8].cpu(), dgu[0, 8:].cpu()
    assert h[2].isnan() and h[4].isnan() and h[[0, 1, 3, 5, 6, 7]].isfinite().all() and h[0] == 10.0
    assert dg[0] == 0 and du[1] == 0 and du[3] == 0 and dg[1] != 0 and (du[[5, 6, 7]] != 0).all()
