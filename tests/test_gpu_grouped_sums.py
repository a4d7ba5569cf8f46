"""Rows of grouped products that are summed per token: fp32 rows, fp32 sums, one rounding, whatever the results' type, the number of
routes and the workspace.

Tolerances: products of 16-bit values are exact in fp32, and a result passes through at most K + k fp32 roundings (K terms of a row, k rows),
each at most 2^-23 of the terms' magnitudes (a whole unit: matrix cores may truncate), and one rounding to its type, half a step of it and half its
smallest subnormal. Nothing counts rows of fewer bits. Beside that a result is compared, bit for bit, with the fp32 result of the same call rounded
to its type: sums that are rounded once give no other value."""
import pytest
import torch

from test_gpu_grouped import BF, COUNTS, HALF, HF, TINY, inputs, order_of, picks, within

pytestmark = pytest.mark.gpu

ROWS = {**COUNTS, "16": [9, 7], "17": [9, 8], "even": [64, 64, 64, 64]}


def summed64(rows, w, ids, turn):
    """(sums per token, sums of magnitudes) of rows [n, K] times w[e] [N, K] transposed, with `turn` rows [n, N] times w[e], in float64."""
    E, (T, k) = w.shape[0], ids.shape
    order, expert = order_of(ids, E)
    rows, w = rows.double(), w.double()
    out = [torch.zeros((T * k, w.shape[2 if turn else 1])).double() for _ in range(2)]
    for e in range(E):
        r = (expert == e).nonzero()[:, 0]
        m = w[e] if turn else w[e].t()
        out[0][r], out[1][r] = rows[r] @ m, rows[r].abs() @ m.abs()
    return [torch.zeros((T, v.shape[1])).double().index_add_(0, order // k, v) for v in out]


def rounded_once(got, ref, mag, terms):
    half = HALF[got.dtype]
    within(got, ref, (1 + half) * terms * 2.0 ** -23 * mag + half * ref.abs() + TINY[got.dtype])


def call_c(name, plan, rows, w, out_dtype, ws_bytes):
    """The C entry point on a workspace of so many bytes, with what lies behind it looked at."""
    from mi355moe import _lib
    E, N, K = w.shape
    codes = {HF: _lib.DTYPE_F16, BF: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
    forward = name == "mm_group_linear"
    guard = 4096
    ws = torch.full((ws_bytes + guard,), 0xA5, dtype=torch.uint8, device=w.device)
    out = torch.full((plan.T + 1, N if forward else K), 7.0, dtype=out_dtype, device=w.device)
    _lib.call(name, plan._ref, rows.data_ptr(), w.data_ptr(), codes[w.dtype], K, N, 0 if forward else 1, 1 if forward else 0, out.data_ptr(),
              codes[out_dtype], ws.data_ptr(), ws_bytes, _lib.raw_stream(w.device))
    assert (ws[ws_bytes:] == 0xA5).all() and (out[plan.T] == 7.0).all()
    return out[:plan.T]


# columns of the sums: fewer than a tile's, no multiple of one, several of them; the last ones with every large tile
CASES = [("16", 2, 0, 64, 72), ("17", 1, 0, 64, 72), ("edges", 3, 4, 72, 520), ("few", 2, 20, 136, 1032), ("long", 5, 300, 200, 264), ("even", 4, 0, 128, 2048),
         ("tiles", 2, 9, 136, 24), ("edges", 2, 1, 64, 8), ("none", 2, 30, 64, 40), ("sizes", 3, 4, 200, 3848), ("sizes", 2, 300, 72, 4096)]


@pytest.mark.parametrize("rows,k,none,terms,cols", CASES)
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_sums_are_rounded_once(dev, rows, k, none, terms, cols, turn, dtype):
    """Forward and gradient of the inputs, through the package and through the C ABI on the least workspace and on one of all rows in fp32."""
    from mi355moe import _lib, grouped
    g = torch.Generator().manual_seed(terms + cols + k)
    counts = ROWS[rows]
    ids = picks(g, counts, k, none)
    K, N = (cols, terms) if turn else (terms, cols)
    _, _, w = inputs(g, ids, len(counts), K, N, dtype, turn, not turn)
    r = torch.randn((ids.numel(), terms), generator=g).to(dtype)
    ref, mag = summed64(r, w, ids, turn)
    plan, rd, wd = grouped.Plan(ids.to(dev), len(counts)), r.to(dev), w.to(dev)
    print(f"sums {rows} {cols} columns turn {turn}", flush=True)
    name = "mm_group_linear_inputs" if turn else "mm_group_linear"
    full = 4 * ids.numel() * cols
    exact = call_c(name, plan, rd, wd, torch.float32, full)
    rounded_once(exact, ref, mag, terms + k)
    if turn:
        got = grouped.linear_backward(rd, None, wd, plan, gather=True, need_w=False)[0]
    else:
        got = grouped.linear_forward(rd, wd, plan, reduce=True)
        assert torch.equal(grouped.linear_forward(rd, wd, plan, reduce=True, out_dtype=torch.float32), exact)
    rounded_once(got, ref, mag, terms + k)
    assert torch.equal(got, exact.to(dtype))
    least = _lib.load().mm_group_linear_workspace(plan.T, plan.k, cols, 1, {HF: _lib.DTYPE_F16, BF: _lib.DTYPE_BF16}[dtype])
    assert least <= full
    for size in (least, full):
        assert torch.equal(call_c(name, plan, rd, wd, dtype, size), got)


@pytest.mark.parametrize("T", [8, 9, 700])
@pytest.mark.parametrize("turn", [False, True])
def test_rows_that_cancel(dev, T, turn):
    """Two picks of each token give rows that differ by a hundredth: their sum has the error of fp32 sums, not of rows of fewer bits."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(T)
    terms, cols = 64, 328
    ids = torch.tensor([[0, 1]]).repeat(T, 1)
    r = torch.randn((T, 2, terms), generator=g)
    r[:, 1] = r[:, 0]
    r[:, 1, :4] *= 1 + 2.0 ** -6
    order, _ = order_of(ids, 2)
    r = r.view(2 * T, terms)[order].to(BF)
    w = torch.randn((1, terms, cols) if turn else (1, cols, terms), generator=g) / 8
    w = torch.cat([w, -w]).to(BF)
    ref, mag = summed64(r, w, ids, turn)
    assert 0 < ref.abs().mean() < 0.01 * mag.mean()
    plan, rd, wd = grouped.Plan(ids.to(dev), 2), r.to(dev), w.to(dev)
    got = grouped.linear_backward(rd, None, wd, plan, gather=True, need_w=False)[0] if turn else grouped.linear_forward(rd, wd, plan, reduce=True)
    rounded_once(got, ref, mag, terms + 2)


def test_columns_of_all_sizes(dev):
    """Neighbouring runs of 32 columns 2^50 apart, and a last run of 8: each is as exact as it is alone."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(5)
    ids = picks(g, [30, 50, 70], 2)
    terms, cols = 64, 200
    r, w = torch.randn((ids.numel(), terms), generator=g).to(BF), torch.randn((3, cols, terms), generator=g)
    w *= 2.0 ** (25 * (1 - 2 * ((torch.arange(cols) // 32) % 2)))[:, None].float()
    w = w.to(BF)
    plan = grouped.Plan(ids.to(dev), 3)
    ref, mag = summed64(r, w, ids, False)
    rounded_once(grouped.linear_forward(r.to(dev), w.to(dev), plan, reduce=True), ref, mag, terms + 2)
    w = w.transpose(1, 2).contiguous()
    rounded_once(grouped.linear_backward(r.to(dev), None, w.to(dev), plan, gather=True, need_w=False)[0], ref, mag, terms + 2)


@pytest.mark.parametrize("turn", [False, True])
def test_long_sums_take_no_more_than_half_the_rows(dev, turn):
    """320,000 rows of 4,096 columns are 5.2 GB in fp32: a bf16 result asks for less than 3, and has the same bits."""
    from mi355moe import grouped
    g = torch.Generator(device=dev).manual_seed(9)
    T, k, E, terms, cols = 40000, 8, 8, 64, 4096
    ids = torch.randint(-1, E, (T, k), generator=g, device=dev)
    r = torch.randn((T * k, terms), generator=g, device=dev).to(BF)
    w = torch.randn((E, terms, cols) if turn else (E, cols, terms), generator=g, device=dev).to(BF)
    plan = grouped.Plan(ids, E)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = grouped.linear_backward(r, None, w, plan, gather=True, need_w=False)[0] if turn else grouped.linear_forward(r, w, plan, reduce=True)
    torch.cuda.synchronize()
    out = 2 * T * cols
    assert torch.cuda.max_memory_allocated() - before - out < 3e9
    exact = call_c("mm_group_linear_inputs" if turn else "mm_group_linear", plan, r, w, torch.float32, 4 * T * k * cols)
    assert torch.equal(got, exact.to(BF))
