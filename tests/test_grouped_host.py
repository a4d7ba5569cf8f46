"""Argument checks of the products grouped by expert, of the gated activation and of the layer on 16-bit experts: refused before any device
work."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

BF = torch.bfloat16


def plan(T=4, k=2, E=3):
    return SimpleNamespace(T=T, k=k, E=E, n=T * k, device=torch.device("cpu"), _ref=None)


def test_plan_refusals():
    from mi355moe import grouped
    ids = torch.zeros((4, 2), dtype=torch.int64)
    for exc, match, args in [(ValueError, "int64", (ids.int(), 3)), (ValueError, r"\[T, k\]", (ids.reshape(-1), 3)),
                             (ValueError, r"\[T, k\]", (ids[:, :0], 3)), (ValueError, "1024", (ids, 1025)), (ValueError, "1024", (ids, 0)),
                             (ValueError, "routes", (ids.new_zeros((1, 1)).expand(1 << 28, 8), 3)), (ValueError, "GPU", (ids, 3))]:
        with pytest.raises(exc, match=match):
            grouped.Plan(*args)


def test_linear_refusals():
    from mi355moe import grouped
    p, x, w, dy = plan(), torch.zeros((8, 16), dtype=BF), torch.zeros((3, 24, 16), dtype=BF), torch.zeros((8, 24), dtype=BF)
    odd = torch.zeros(3 * 24 * 16 + 1, dtype=BF)[1:].view(3, 24, 16)
    for exc, match, args, kw in [
            (TypeError, "fp16 or bf16", (x.float(), w.float()), {}), (TypeError, "w's type", (x.half(), w), {}),
            (ValueError, r"w \[3, N, K\]", (x, w[:2]), {}), (ValueError, r"w \[3, N, K\]", (x, w[0]), {}),
            (ValueError, "multiples of 8", (x[:, :12], w[:, :, :12].contiguous()), {}), (ValueError, "multiples of 8", (x, w[:, :20].contiguous()), {}),
            (ValueError, "contiguous", (x, w.transpose(1, 2).contiguous().transpose(1, 2)), {}), (ValueError, "16-byte", (x, odd), {}),
            (ValueError, r"x must be \[8, 16\]", (x[:4], w), {}), (ValueError, r"x must be \[4, 16\]", (x, w), {"gather": True}),
            (ValueError, "different products", (x, w), {"gather": True, "reduce": True}),
            (TypeError, "results", (x, w), {"out_dtype": torch.float16}), (ValueError, "GPU", (x, w), {})]:
        for call in (grouped.linear_forward, grouped.linear):
            with pytest.raises(exc, match=match):
                call(*args, p, **kw)
    for exc, match, args, kw in [
            (TypeError, "w's type", (dy.float(), x, w), {}), (ValueError, r"dy must be \[8, 24\]", (dy[:, :16], x, w), {}),
            (ValueError, r"dy must be \[4, 24\]", (dy, x, w), {"reduce": True}), (ValueError, "dw needs x", (dy, None, w), {}),
            (ValueError, r"x must be \[4, 16\]", (dy, x, w), {"gather": True}), (TypeError, "results", (dy, x, w), {"dw_dtype": torch.float64}),
            (ValueError, "GPU", (dy, x, w), {}), (ValueError, "GPU", (dy, None, w), {"need_w": False})]:
        with pytest.raises(exc, match=match):
            grouped.linear_backward(*args, p, **kw)


def test_swiglu_refusals():
    from mi355moe import grouped
    p, gu, wt, dh = plan(), torch.zeros((8, 64), dtype=BF), torch.zeros((4, 2)), torch.zeros((8, 32), dtype=BF)
    for exc, match, args, kw in [
            (TypeError, "fp16 or bf16", (gu.float(), p), {}), (ValueError, r"\[n, 2 I\]", (gu[0], p), {}), (ValueError, r"\[n, 2 I\]", (gu[:, :63], p), {}),
            (ValueError, "multiple of 8", (gu[:, :40], p), {}), (ValueError, "8 rows", (gu[:4], p), {}), (ValueError, "limit", (gu, p), {"limit": -1.0}),
            (ValueError, "limit", (gu, p), {"limit": float("nan")}), (ValueError, r"weights must be fp32 \[4, 2\]", (gu, p, wt.reshape(-1)), {}),
            (ValueError, "weights must be fp32", (gu, p, wt.half()), {}), (ValueError, r"weights must be fp32 \[8\]", (gu, None, wt), {}),
            (ValueError, "multiple of 32", (gu[:, :48], p), {"save8": True}), (ValueError, "GPU", (gu, p, wt), {}), (ValueError, "GPU", (gu,), {})]:
        with pytest.raises(exc, match=match):
            grouped.swiglu_forward(*args, **kw)
    saved = grouped.Saved8(torch.zeros((8, 64), dtype=torch.int8), torch.zeros((8, 2), dtype=torch.int8), BF)
    for bad in (grouped.Saved8(saved.codes, saved.exps[:, :1], BF), grouped.Saved8(saved.codes.float(), saved.exps, BF),
                grouped.Saved8(saved.codes, saved.exps[:4], BF), grouped.Saved8(saved.codes.t().contiguous().t(), saved.exps, BF)):
        with pytest.raises(ValueError, match="must be contiguous int8"):
            grouped.swiglu_backward(dh, bad, p)
    for kept in (gu, saved):
        for exc, match, args in [(ValueError, "dh must be", (dh.half(), kept, p)), (ValueError, "dh must be", (dh[:, :16], kept, p)),
                                 (ValueError, "6 rows", (dh, kept, plan(3))), (ValueError, "GPU", (dh, kept, p))]:
            with pytest.raises(exc, match=match):
                grouped.swiglu_backward(*args)


def test_dense_store_and_layer_refusals():
    from mi355moe import dense, moe
    w13, w2 = torch.zeros((3, 2, 32, 16), dtype=BF), torch.zeros((3, 16, 32), dtype=BF)
    for exc, match, args, kw in [
            (ValueError, "expected", (w13[:, 0], w2), {}), (ValueError, "expected", (w13[:, :1], w2), {}), (ValueError, "w2 must be", (w13, w2[:2]), {}),
            (TypeError, "fp16 or both bf16", (w13.float(), w2.float()), {}), (TypeError, "fp16 or both bf16", (w13, w2.half()), {}),
            (ValueError, "H a multiple of 8", (w13[..., :12].contiguous(), w2[:, :12].contiguous()), {}),
            (ValueError, "I of 32", (w13[:, :, :24].contiguous(), w2[..., :24].contiguous()), {"save8": True}),
            (ValueError, "contiguous", (w13.transpose(1, 2).contiguous().transpose(1, 2), w2), {}), (ValueError, "limit", (w13, w2), {"limit": -2.0}),
            (ValueError, "GPU", (w13, w2), {})]:
        with pytest.raises(exc, match=match):
            dense.DenseStore(*args, **kw)
    store = object.__new__(dense.DenseStore)
    store.E, store.H, store.I, store.w13, store.w2, store.limit, store.save8 = 3, 16, 32, w13, w2, 10.0, False
    x, ids, w = torch.zeros((4, 16), dtype=BF), torch.zeros((4, 2), dtype=torch.int64), torch.zeros((4, 2))
    for exc, match, args, kw in [
            (TypeError, "weights' type", (x.float(), ids, w), {}), (ValueError, r"x \[T, 16\]", (x[:, :8], ids, w), {}),
            (ValueError, "ids and w", (x, ids.t(), w.t()), {}), (ValueError, "ids and w", (x, ids, w[:, :1]), {}), (ValueError, "ids and w", (x, ids[:, :0], w[:, :0]), {}),
            (ValueError, "shared expert 3", (x, ids, w), {"shared_expert": 3}), (ValueError, "GPU", (x, ids, w), {})]:
        for call in (dense.moe, moe.moe_forward):
            with pytest.raises(exc, match=match):
                call(store, *args, **kw)
    for call in (lambda: moe.decode_routes(store, x, ids, w, 2), lambda: moe.moe_prefill(store, x, ids, w), lambda: moe.fused_moe(store, x, ids, w, 32)):
        with pytest.raises(TypeError, match="DenseStore.*moe.moe_forward"):
            call()


def test_c_argument_errors():
    """The C ABI's own checks, with addresses that are never touched."""
    from mi355moe import _lib
    L = _lib.load()

    def err(rc, text):
        assert rc == -1 and text in L.mm_last_error(), L.mm_last_error()

    def p(T=4, k=2, E=3, **kw):
        f = dict(offsets=256, order=256, token=256, inv=256, tiles=256, ntiles=256, T=T, topk=k, E=E) | kw
        return ctypes.byref(_lib.MMGroupPlan(*f.values()))

    assert L.mm_group_tiles(8, 3) > 0 and L.mm_group_tiles(0, 3) == 0 and L.mm_group_linear_workspace(4, 2, 24, 1, 1) == 4 * 2 * 24 * 4
    assert L.mm_group_linear_workspace(4, 2, 24, 0, 1) == 0 and L.mm_group_linear_workspace(9, 2, 72, 1, 2) == 18 * 72 * 4
    assert L.mm_group_linear_workspace(9, 2, 72, 1, 0) == 18 * 72 * 4 and L.mm_group_linear_workspace(9, 2, 72, 1, 1) == 18 * (72 * 2 + 3)
    err(L.mm_group_plan(256, p(order=None), 256, None, 0, None), b"null")
    err(L.mm_group_plan(None, p(), 256, None, 0, None), b"null")
    err(L.mm_group_plan(256, p(T=0), 256, None, 0, None), b"need tokens")
    err(L.mm_group_plan(256, p(E=1025), 256, None, 0, None), b"E <= 1024")
    err(L.mm_group_plan(256, p(T=1 << 28, k=8), 256, None, 0, None), b"2^30")
    err(L.mm_group_plan(256, p(tiles=264), 256, None, 0, None), b"misaligned")
    err(L.mm_group_plan(256, p(T=1 << 16), 256, None, 0, None), b"workspace")
    row = [256, 256, 1, 16, 24, 0, 0, 256, 1, None, 0, None]
    for fn, name in ((L.mm_group_linear, b"mm_group_linear:"), (L.mm_group_linear_inputs, b"mm_group_linear_inputs:")):
        for at, value, text in [(0, None, b"null"), (1, None, b"null"), (2, 2, b"fp16 or bf16"), (3, 20, b"multiples of 8"), (4, 0, b"multiples of 8"),
                                (3, (1 << 20) + 8, b"2^20"), (7, 264, b"misaligned"), (0, 264, b"misaligned"), (8, 0, b"weights' type")]:
            a = list(row)
            a[at] = value
            err(fn(p(), *a), text)
            assert name in L.mm_last_error()
        err(fn(p(token=None), *row), b"incomplete plan")
        err(fn(p(k=0), *row), b"bad plan")
        err(fn(None, *row), b"incomplete plan")
        big = list(row)
        big[3] = big[4] = 1 << 16
        err(fn(p(), *big), b"K N below 2^31")
    sums = list(row)
    sums[6] = 1
    err(L.mm_group_linear(p(), *sums), b"workspace too small (0 < 768)")
    sums[5], sums[6] = 1, 0
    err(L.mm_group_linear_inputs(p(), *sums), b"workspace too small (0 < 512)")
    far = list(row)
    far[3], far[5] = 1 << 12, 1
    err(L.mm_group_linear(p(T=1 << 20, k=1), *far), b"4 GiB")
    wts = [256, 256, 1, 16, 24, 0, 0, 256, 1, None]
    for at, value, text in [(0, None, b"null"), (1, None, b"null"), (7, None, b"null"), (2, 2, b"fp16 or bf16"), (8, 0, b"weights' type"), (1, 264, b"misaligned")]:
        a = list(wts)
        a[at] = value
        err(L.mm_group_linear_weights(p(), *a), text)
    both = list(wts)
    both[5] = both[6] = 1
    err(L.mm_group_linear_weights(p(), *both), b"one of x and dy")
    g = [256, 1, 8, 32, None, 10.0, 256, None, None, None]
    for at, value, text in [(0, None, b"null"), (6, None, b"null"), (1, 2, b"fp16 or bf16"), (2, 9, b"other rows"), (3, 36, b"multiple of 8"), (5, -1.0, b"limit"),
                            (7, 256, b"go together"), (0, 264, b"misaligned")]:
        a = list(g)
        a[at] = value
        err(L.mm_gated(p(), *a), text)
    err(L.mm_gated(p(), 256, 1, 8, 40, None, 10.0, 256, 256, 256, None), b"multiple of 32")
    err(L.mm_gated(None, 256, 1, 0, 32, None, 10.0, 256, None, None, None), b"2^30 rows")
    b = [256, 256, None, None, 1, 8, 32, None, 10.0, 256, None, None, None]
    for at, value, text in [(0, None, b"null"), (1, None, b"null"), (9, None, b"null"), (4, 3, b"fp16 or bf16"), (11, 264, b"misaligned"), (2, 256, b"go together")]:
        a = list(b)
        a[at] = value
        err(L.mm_gated_backward(p(), *a), text)
    err(L.mm_gated_backward(p(), 256, 256, 256, 256, *b[4:]), b"both forms")


def test_a_captured_layer_names_what_to_capture_instead(monkeypatch):
    from mi355moe import router

    class Double(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return 2 * t

        @staticmethod
        def backward(ctx, d):
            return 2 * d

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    t = torch.ones(3, requires_grad=True)
    eager = t.sum()
    with pytest.raises(RuntimeError, match="dense.moe: .* or capture the others"):
        router._captured_apply("dense.moe", Double, (t,), t, instead="the others")
    del eager


@pytest.mark.parametrize("dtype,shared", [(torch.float32, None), (torch.float32, 1), (torch.bfloat16, None), (torch.float64, 0)])
def test_a_layer_names_the_callers_own_tensors_as_leaves(monkeypatch, dtype, shared):
    """Under capture the leaves are looked at for older graphs: the routing weights as the caller has them, not a copy with another type or
    the shared expert's column."""
    import contextlib
    from mi355moe import _lib, dense
    monkeypatch.setattr(_lib, "check_tensors", lambda *a, **k: None)
    monkeypatch.setattr(_lib, "on", lambda *a: contextlib.nullcontext())
    seen = []
    monkeypatch.setattr(dense, "_captured_apply", lambda what, fn, leaves, *args, **k: seen.append(leaves))
    store = dense.DenseStore(torch.zeros(2, 2, 8, 8, dtype=torch.bfloat16), torch.zeros(2, 8, 8, dtype=torch.bfloat16))
    x, w = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(3, 1, dtype=dtype, requires_grad=True)
    dense.moe(store, x, torch.zeros(3, 1, dtype=torch.int64), w, shared_expert=shared)
    assert [id(t) for t in seen[0]] == [id(t) for t in (x, w, store.w13, store.w2)]
