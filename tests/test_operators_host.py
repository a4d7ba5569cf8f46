"""Argument checks of the router's gradient operators and of the 4-bit products: refused before any device work."""
import ctypes

import pytest
import torch


def test_balance_refusals():
    from mi355moe import router
    lg, ids = torch.zeros((4, 8)), torch.zeros((4, 2), dtype=torch.int64)
    bad = [
        (ValueError, "logits", (torch.zeros(8), ids)),
        (TypeError, "logits must be", (lg.double(), ids)),
        (ValueError, "ids must be", (lg, ids[:3])),
        (ValueError, "ids must be", (lg[None], ids)),
        (TypeError, "int64", (lg, ids.int())),
        (ValueError, "score", (lg, ids, None, "tanh")),
        (ValueError, "mask must be", (lg, ids, torch.ones(3, dtype=torch.bool))),
        (TypeError, "bool or uint8", (lg, ids, torch.ones(4))),
        (ValueError, "k", (lg, torch.zeros((4, 33), dtype=torch.int64))),
        (ValueError, "k", (lg, torch.zeros((4, 0), dtype=torch.int64))),
        (ValueError, "GPU", (lg, ids)),
    ]
    for exc, match, args in bad:
        with pytest.raises(exc, match=match):
            router.balance_loss_forward(*args)
    one, c, n = torch.tensor(1.0), torch.zeros(8, dtype=torch.int32), torch.tensor(4, dtype=torch.int32)
    for exc, match, args in [(ValueError, "dloss", (one[None], lg, c, n, 2)), (ValueError, "counts", (one, lg, c.float(), n, 2)),
                             (ValueError, "tokens", (one, lg, c, n[None], 2)), (ValueError, "k", (one, lg, c, n, 0)),
                             (ValueError, "GPU", (one, lg, c, n, 2))]:
        with pytest.raises(exc, match=match):
            router.balance_loss_backward(*args)


def test_router_refusals():
    from mi355moe import router
    x, gate = torch.zeros((4, 32), dtype=torch.bfloat16), torch.zeros((8, 32))
    ids, w = torch.zeros((4, 2), dtype=torch.int64), torch.zeros((4, 2))
    for exc, match, args in [
            (ValueError, "neither", (x, gate, ids, w)), (ValueError, "expected", (x[:, :16], gate, ids, w, w)),
            (TypeError, "bf16", (x.half(), gate, ids, w, w)), (TypeError, "fp32", (x, gate.half(), ids, w, w)),
            (ValueError, "ids and w", (x, gate, ids[:2], w, w)), (ValueError, "ids and w", (x, gate, ids[:, :0], w[:, :0], w)),
            (ValueError, "dw must", (x, gate, ids, w, w[:, :1])), (ValueError, "dlogits must", (x, gate, ids, w, None, w)),
            (TypeError, "int64", (x, gate, ids.int(), w, w)), (ValueError, "GPU", (x, gate, ids, w, w))]:
        with pytest.raises(exc, match=match):
            router.topk_backward(*args)
    with pytest.raises(ValueError, match="GPU"):
        router.topk(x, gate, 2)


def test_w4_refusals():
    from mi355moe import w4
    q, s = torch.zeros((16, 16), dtype=torch.int32), torch.zeros((16, 1), dtype=torch.float16)
    z = torch.zeros((16, 1), dtype=torch.uint8)
    for exc, match, args in [
            (TypeError, "int32", (q.long(), s)), (TypeError, "fp16 or bf16", (q, s.float())), (ValueError, "match", (q, s[:8])),
            (ValueError, "group", (q, torch.zeros((16, 8), dtype=torch.float16))),
            (ValueError, "group", (q, torch.zeros((16, 3), dtype=torch.float16))),
            (ValueError, "zeros", (q, s, z.int())), (ValueError, "zeros", (q, s, z[:4])),
            (ValueError, "contiguous", (q.t().contiguous().t(), s)), (ValueError, "match", (q[:0], s[:0])),
            (ValueError, "16-byte", (torch.zeros(257, dtype=torch.int32)[1:].view(16, 16), s)),
            (ValueError, "GPU", (q, s, z))]:
        with pytest.raises(exc, match=match):
            w4.W4Matrix(*args)
    q13, s13 = torch.zeros((3, 2, 32, 8), dtype=torch.int32), torch.zeros((3, 2, 32, 2), dtype=torch.float16)
    q2, s2 = torch.zeros((3, 64, 4), dtype=torch.int32), torch.zeros((3, 64, 1), dtype=torch.float16)
    for match, args in [("expected", (q13[:, 0].contiguous(), s13[:, 0].contiguous(), None, q2, s2, None)),
                        ("q2 must", (q13, s13, None, q2[:2], s2[:2], None)),
                        ("share", (q13, s13, None, q2, s2.bfloat16(), None)),
                        ("share", (q13, s13[..., :1].contiguous(), None, q2, s2, None)),
                        ("GPU", (q13, s13, None, q2, s2, None))]:
        with pytest.raises(ValueError, match=match):
            w4.W4Store(*args)


def test_c_argument_errors():
    """The C ABI's own checks, with addresses that are never touched."""
    from mi355moe import _lib
    L = _lib.load()

    def err(rc, text):
        assert rc == -1 and text in L.mm_last_error(), L.mm_last_error()

    err(L.mm_balance_loss(256, 5, 256, None, 1, 4, 8, 2, 0, 256, 256, 256, 256, None, 0, None), b"logits type")
    err(L.mm_balance_loss(256, 2, 256, None, 1, 4, 2000, 2, 0, 256, 256, 256, 256, None, 0, None), b"E <= 1024")
    err(L.mm_balance_loss(256, 2, 256, None, 1, 4, 8, 2, 2, 256, 256, 256, 256, None, 0, None), b"score")
    err(L.mm_balance_loss(None, 2, 256, None, 1, 4, 8, 2, 0, 256, 256, 256, 256, None, 0, None), b"null")
    err(L.mm_balance_loss(256, 2, 256, None, 1, 1 << 27, 8, 32, 0, 256, 256, 256, 256, None, 0, None), b"too many picks")
    assert L.mm_balance_workspace(1, 16384, 384) > 0 and L.mm_balance_workspace(1, 1, 384) == 0
    err(L.mm_balance_loss(256, 2, 256, None, 1, 16384, 384, 8, 0, 256, 256, 256, 256, 256,
                          L.mm_balance_workspace(1, 16384, 384) - 1, None), b"workspace too small")
    err(L.mm_balance_loss_backward(None, 256, 2, None, 256, 256, 1, 4, 8, 2, 0, 256, None), b"null")
    need = L.mm_router_backward_workspace(100, 256, 8)
    ok = [256, 100, 256, 256, 8, 2, 256, 256, 256, 256, 256, 256, 256, need, None]
    for at, value, text in [(2, 250, b"H % 16"), (4, 1025, b"E <= 1024"), (5, 33, b"k <= 32"), (1, (1 << 21) + 1, b"2^21"),
                            (0, 264, b"aligned"), (6, None, b"needs ids"), (3, None, b"gate"), (13, need - 1, b"workspace")]:
        a = list(ok)
        a[at] = value
        err(L.mm_router_backward(*a), text)
    a = list(ok)
    a[8] = a[9] = None
    err(L.mm_router_backward(*a), b"neither")
    W = _lib.MMW4(256, 256, None)
    lin = [256, 1, 4, 256, 16, ctypes.byref(W), 64, 0, 256, 1, None, 0, None]
    for at, value, text in [(3, 250, b"multiple of the group"), (6, 16, b"group must"), (7, 2, b"scales must"), (0, 264, b"misaligned"),
                            (1, 3, b"element type"), (9, -1, b"element type"), (1, 2, b"workspace"), (8, None, b"null")]:
        a = list(lin)
        a[at] = value
        err(L.mm_w4_linear(*a), text)
    lay = _lib.MMW4Layer(W, W, 8, 256, 128, 64, 0, 10.0)
    need = L.mm_w4_moe_workspace(1, 5, 2, -1, 8, 256, 128)
    mo = [ctypes.byref(lay), 256, 1, 5, 2, 256, 256, -1, 256, 256, need, None]
    for at, value, text in [(7, 8, b"shared expert"), (4, 0, b"routes"), (1, 264, b"misaligned"), (2, 7, b"input type"),
                            (10, need - 1, b"workspace"), (5, None, b"null")]:
        a = list(mo)
        a[at] = value
        err(L.mm_w4_moe(*a), text)
    for bad in (_lib.MMW4Layer(W, W, 8, 256, 100, 64, 0, 10.0), _lib.MMW4Layer(W, W, 1025, 256, 128, 64, 0, 10.0)):
        err(L.mm_w4_moe(ctypes.byref(bad), *mo[1:]), b"multiples of the group")


def test_a_capture_beside_an_eager_autograd_graph_is_refused(monkeypatch):
    """As seen under stream capture: a leaf that an earlier autograd graph holds is refused, one that only calls of this capture hold is
    not."""
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
    with pytest.raises(RuntimeError, match="capture topk_forward and topk_backward"):
        router._captured_apply("topk", Double, (t,), t)
    del eager
    a = router._captured_apply("topk", Double, (t,), t)
    b = router._captured_apply("topk", Double, (t,), t)
    (a + b).sum().backward()
    assert torch.equal(t.grad, torch.full((3,), 4.0))
    with torch.no_grad():
        assert not router._captured_apply("topk", Double, (t,), t).requires_grad


def test_a_stream_of_another_device_is_refused():
    from mi355moe import _lib

    class Stream:
        device = torch.device("cuda", 1)

    with pytest.raises(ValueError, match="stream of cuda:1"):
        _lib.on(torch.device("cuda", 0), Stream())


def test_a_later_capture_is_held_to_its_own_stream(monkeypatch):
    """A gradient node that a call of an earlier capture made, kept alive by an eager graph, passes in a capture of that stream only."""
    from mi355moe import router

    class Double(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return 2 * t

        @staticmethod
        def backward(ctx, d):
            return 2 * d

    capturing, stream = True, 1
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing)
    monkeypatch.setattr(router, "_capture_stream", lambda device: stream, raising=False)

    def call():
        return router._captured_apply("topk", Double, (t,), t)

    t = torch.ones(3, requires_grad=True)
    first = call()
    capturing = False
    eager = t.sum()
    del first
    capturing, stream = True, 2
    with pytest.raises(RuntimeError, match="from before the stream capture"):
        call()
    stream = 1                                                # the node's own: refusing the other one left its mark in place
    assert call().requires_grad
    stream = 2
    del eager
    a, b = call(), call()                                     # nothing holds the old node: a new one of this capture
    assert a.requires_grad and b.requires_grad
    stream = 1
    with pytest.raises(RuntimeError, match="from before the stream capture"):
        call()


def test_linear_refuses_more_columns_than_a_launch_has():
    from mi355moe import _lib
    L = _lib.load()
    W = _lib.MMW4(256, 256, None)
    for N in ((1 << 26) + 1, 1 << 27, 1 << 30):
        assert L.mm_w4_linear(256, 1, 4, 256, N, ctypes.byref(W), 64, 0, 256, 1, None, 0, None) == -1
        assert b"N at most 2^26" in L.mm_last_error()


def test_balance_refuses_more_than_2_30_tokens():
    from mi355moe import _lib
    L = _lib.load()
    T = (1 << 30) + 1
    assert L.mm_balance_loss(256, 2, 256, None, 1, T, 8, 1, 0, 256, 256, 256, 256, 256, 1 << 40, None) == -1
    assert b"2^30" in L.mm_last_error()
    assert L.mm_balance_loss_backward(256, 256, 2, None, 256, 256, 1, T, 8, 1, 0, 256, None) == -1
    assert b"2^30" in L.mm_last_error()


def test_inputs_that_want_a_gradient_are_not_silently_cut_off():
    """The 4-bit products refuse them; the layer on EXL3 experts, which took them before the router had gradients, warns."""
    from types import SimpleNamespace

    from mi355moe import moe, w4
    W = SimpleNamespace(K=64, N=16, _device=torch.device("cpu"))
    x = torch.zeros((2, 64), requires_grad=True)
    with pytest.raises(RuntimeError, match="x requires a gradient"):
        w4.linear(x, W)
    store = object.__new__(w4.W4Store)
    store.E, store.H, store.I, store.q13 = 4, 64, 32, torch.zeros(1)
    ids, w = torch.zeros((2, 1), dtype=torch.int64), torch.ones((2, 1), requires_grad=True)
    for args, name in (((x, ids, w.detach()), "x"), ((x.detach(), ids, w), "w")):
        with pytest.raises(RuntimeError, match=f"{name} requires a gradient"):
            moe.moe_forward(store, *args)
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            moe.moe_forward(store, *args)
    with pytest.raises(ValueError, match="GPU"):
        moe.moe_forward(store, x.detach(), ids, w.detach())

    class Store:
        E, H, I = 4, 64, 32

        def mm_layer(self):
            raise LookupError("reached the layer")

    for T in (2, 40):
        wt = torch.ones((T, 1), requires_grad=True)
        a = (torch.zeros((T, 64)).half(), torch.zeros((T, 1), dtype=torch.int64))
        with pytest.warns(UserWarning, match="no gradient"), pytest.raises(LookupError):
            moe.moe_forward(Store(), *a, wt)


def test_experts_take_picks_as_tokens_by_k_only():
    """[k, T] has as many elements as [T, k], and would be read as other tokens' picks."""
    from mi355moe import w4
    store = object.__new__(w4.W4Store)
    store.E, store.H, store.I, store.q13 = 4, 64, 32, torch.zeros(1)
    x, ids = torch.zeros((6, 64)), torch.zeros((6, 2), dtype=torch.int64)
    for bad in (ids.t(), ids.reshape(-1), ids.reshape(3, 4), ids.reshape(6, 2, 1), ids[:, 0]):
        with pytest.raises(ValueError, match=r"ids and w must be \[6, k\]"):
            w4.moe(store, x, bad, bad.float())
    with pytest.raises(ValueError, match="GPU"):
        w4.moe(store, x, ids, ids.float())
    with pytest.raises(ValueError, match="GPU"):
        w4.moe(store, x[:0], ids[:0], ids[:0].float())


def test_exl3_paths_refuse_a_store_of_4_bit_experts():
    from mi355moe import moe, w4
    store = object.__new__(w4.W4Store)
    store.E, store.H, store.I = 4, 64, 32
    x, ids, w = torch.zeros((2, 64)).half(), torch.zeros((2, 1), dtype=torch.int64), torch.ones((2, 1))
    for call in (lambda: moe.decode_routes(store, x, ids, w, 2), lambda: moe.moe_prefill(store, x, ids, w),
                 lambda: moe.fused_moe(store, x, ids, w, 32), lambda: moe.expert_gemv(store, x, ids, 2, 2, 1, 2),
                 lambda: moe.grouped_gemm(store, x, ids)):
        with pytest.raises(TypeError, match="W4Store.*moe.moe_forward"):
            call()


def test_balance_refuses_a_misaligned_workspace():
    """Its slices are counted with 32-bit atomics, which fault at odd addresses."""
    from mi355moe import _lib
    L = _lib.load()
    need = L.mm_balance_workspace(1, 16384, 384)
    for ws in (257, 258, 264):
        assert L.mm_balance_loss(256, 2, 256, None, 1, 16384, 384, 8, 0, 256, 256, 256, 256, ws, need, None) == -1
        assert b"misaligned" in L.mm_last_error()
