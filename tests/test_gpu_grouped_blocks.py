"""Grouped products over many blocks of terms and many tiles: the row products past the places that their blocks have in LDS, in every large
tile and in both directions, and the weights' gradient where a workgroup takes several tiles, so that a tile's loads run ahead of the last one's stores.

Tolerances: products of 16-bit values are exact in fp32; a sum of K terms passes through at most K fp32 roundings, each at most 2^-23 of the terms'
magnitudes (a whole unit: matrix cores may truncate), and one rounding to its type. As a random walk the same roundings come to sqrt(K) 2^-23 of the
root of the sum of squares, to which the 2-norm of the error over all results is held (twice); a block lost or read early is far outside."""
import pytest
import torch

from test_gpu_grouped import BF, HALF, HF, TINY, order_of, picks

pytestmark = pytest.mark.gpu

# rows of an expert by the largest tile they make: 16, 32, 64, 96, 128, 160, 192, 224 and 256 rows in one tile, and in several 160, 224 and 256
ROWS = [5, 20, 40, 90, 97, 128, 129, 150, 161, 180, 193, 210, 225, 256, 257, 300, 400, 700, 0]


def close(got, ref, mag, sq, terms):
    half, tiny, got = HALF[got.dtype], TINY[got.dtype], got.double()
    assert got.shape == ref.shape
    bad = ~((got - ref).abs() <= (1 + half) * terms * 2.0 ** -23 * mag + half * ref.abs() + tiny)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[:4].tolist()}"
    err = (got - ref).norm()
    assert err <= 2 * (1 + half) * terms ** 0.5 * 2.0 ** -23 * sq.norm() + half * ref.norm() + tiny * ref.numel() ** 0.5


def sums64(a, b):
    """a @ b, its magnitudes and the root of its squares, in float64."""
    a, b = a.double(), b.double()
    return a @ b, a.abs() @ b.abs(), ((a ** 2) @ (b ** 2)).sqrt()


@pytest.mark.parametrize("terms,cols", [(1032, 3848), (584, 4096), (1032, 136)])
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("per_token", [False, True])
def test_rows_of_many_blocks(dev, terms, cols, turn, dtype, per_token):
    """17 and 10 blocks, the last of 8 terms, in large tiles, and 17 in small ones."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(terms + turn)
    ids = picks(g, ROWS, 3, 40)
    T, k, E = *ids.shape, len(ROWS)
    order, expert = order_of(ids, E)
    rows = torch.randn((T if per_token else T * k, terms), generator=g).to(dtype).to(dev)
    gd = torch.Generator(device=dev).manual_seed(7)
    w = (torch.randn((E, terms, cols) if turn else (E, cols, terms), generator=gd, device=dev) / terms ** 0.5).to(dtype)
    plan = grouped.Plan(ids.to(dev), E)
    print(f"rows of {terms} terms, {cols} columns, turn {turn}, per token {per_token}", flush=True)
    if turn:
        got = grouped.linear_backward(rows, None, w, plan, reduce=per_token, need_w=False)[0]
    else:
        got = grouped.linear_forward(rows, w, plan, gather=per_token)
    rows = rows[(order // k).to(dev)] if per_token else rows
    want = [torch.zeros((T * k, cols), dtype=torch.float64, device=dev) for _ in range(3)]
    for e in range(E):
        r = (expert == e).nonzero()[:, 0].to(dev)
        if len(r):
            for t, v in zip(want, sums64(rows[r], w[e] if turn else w[e].t().contiguous())):
                t[r] = v
    close(got, *want, terms)


# experts of 0 to 14 blocks of 32 rows, around the five that have places
TURNS = [0, 1, 33, 65, 97, 129, 161, 400]


@pytest.mark.parametrize("side", ["gather", "reduce", "neither"])
@pytest.mark.parametrize("dtype,out", [(BF, None), (HF, None), (BF, torch.float32)])
@pytest.mark.parametrize("N,K", [(776, 768), (512, 1032)])
def test_weights_of_many_tiles(dev, side, dtype, out, N, K):
    """72 experts of 12 and 10 tiles: full ones, whose stores the next tile's loads are counted with, beside those at the edges."""
    from mi355moe import grouped
    g = torch.Generator().manual_seed(N + K)
    counts = TURNS * 9
    k = 1 if side == "neither" else 2
    ids = picks(g, counts, k, 6)
    T, E = ids.shape[0], len(counts)
    order, expert = order_of(ids, E)
    token = (order // k).to(dev)
    gather, reduce = side == "gather", side == "reduce"
    x = torch.randn((T if gather else T * k, K), generator=g).to(dtype).to(dev)
    dy = torch.randn((T if reduce else T * k, N), generator=g).to(dtype).to(dev)
    w = torch.zeros((E, N, K), dtype=dtype, device=dev)
    print(f"weights {side} {dtype} {out} {N} x {K}", flush=True)
    got = grouped.linear_backward(dy, x, w, grouped.Plan(ids.to(dev), E), gather, reduce, need_x=False, dw_dtype=out)[1]
    xr, dr = x[token] if gather else x, dy[token] if reduce else dy
    for e in range(E):
        r = (expert == e).nonzero()[:, 0].to(dev)
        assert len(r) == counts[e]
        if not len(r):
            assert not got[e].any()
            continue
        close(got[e], *sums64(dr[r].t().contiguous(), xr[r]), len(r))
