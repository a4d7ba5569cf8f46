"""Products grouped by expert over ragged rows, and the gated activation between them: what an expert layer in 16-bit weights is made
of, forward and backward (dense.moe is the layer itself).

A Plan sorts the routes of a call by expert; its n = T k rows are the rows of every product. linear() and swiglu() record themselves
in autograd; the *_forward / *_backward functions are the same kernels without it. Every computation runs in libmi355moe.so on
the current stream (or `stream`); no call synchronises the host.
"""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .router import _captured_apply

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_OUT = {**_DTYPES, torch.float32: _lib.DTYPE_F32}
SAVE_GROUP = 32            # values that share an exponent in a Saved8

_p = _lib.ptr


class Plan:
    """Order of the routes ids int64 [T, k] over E experts (mm_group_plan): by expert, then by route; picks outside [0, E) come last
    and belong to none. offsets int32 [E + 1]: rows offsets[e] .. offsets[e + 1] - 1 are expert e's; counts int32 [E]; order, token int32
    [n]: flat route and token of each row; inv int32 [n]: row of each route. Made for the ids as they are now, on the current stream."""

    def __init__(self, ids, E, stream=None):
        if ids.dim() != 2 or ids.dtype != torch.int64 or ids.shape[1] == 0:
            raise ValueError(f"Plan: ids must be int64 [T, k] (got {ids.dtype} {tuple(ids.shape)})")
        if not 1 <= E <= 1024:
            raise ValueError(f"Plan: need 1 <= E <= 1024 (got {E})")
        (self.T, self.k), self.E, dev = ids.shape, int(E), ids.device
        n = self.n = self.T * self.k
        if n > 2 ** 30:
            raise ValueError(f"Plan: {n} routes, at most 2^30 expected")
        _lib.check_tensors("Plan", dev)
        with _lib.on(dev, stream):
            lib = _lib.load()
            tiles = lib.mm_group_tiles(n, E)
            # one buffer: tiles, offsets [E + 2], counts [E + 1], ntiles, order, token, inv [n]
            at = [tiles // 4]
            for size in (E + 2, E + 1, 2, n, n, n):
                at.append(at[-1] + size)
            make = torch.empty if n else torch.zeros
            self._buf = buf = make(at[-1], dtype=torch.int32, device=dev)
            self.offsets, self.counts = buf[at[0]:at[1] - 1], buf[at[1]:at[2] - 1]
            self.order, self.token, self.inv = (buf[at[i]:at[i + 1]] for i in (3, 4, 5))
            a = buf.data_ptr()
            self._c = _lib.MMGroupPlan(a + 4 * at[0], a + 4 * at[3], a + 4 * at[4], a + 4 * at[5], a, a + 4 * at[2], self.T, self.k, self.E)
            self._ref, self.device = ctypes.byref(self._c), dev
            if n:
                ids = ids.contiguous()
                wsb = lib.mm_group_plan_workspace(n, E)
                ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
                _lib.call("mm_group_plan", ids.data_ptr(), self._ref, a + 4 * at[1], _p(ws), wsb, _lib.raw_stream(dev))


def _check_linear(what, w, plan, gather, reduce):
    """(N, K, type code) of w [E, N, K]."""
    code = _DTYPES.get(w.dtype)
    if code is None:
        raise TypeError(f"{what}: w must be fp16 or bf16 (got {w.dtype})")
    if w.dim() != 3 or w.shape[0] != plan.E:
        raise ValueError(f"{what}: w [{plan.E}, N, K] expected (got {tuple(w.shape)})")
    _, N, K = w.shape
    if K % 8 or N % 8 or not K or not N:
        raise ValueError(f"{what}: K and N must be multiples of 8 (got w {tuple(w.shape)})")
    if not w.is_contiguous() or w.data_ptr() % 16:
        raise ValueError(f"{what}: w must be contiguous and start at a 16-byte boundary")
    if gather and reduce:
        raise ValueError(f"{what}: gather and reduce are of different products")
    return N, K, code


def _check_rows(what, name, t, rows, width, dtype):
    if t.dtype != dtype:
        raise TypeError(f"{what}: {name} must have w's type {dtype} (got {t.dtype})")
    if t.shape != (rows, width):
        raise ValueError(f"{what}: {name} must be {[rows, width]} (got {tuple(t.shape)})")


def _check_out(what, dtype, w):
    if dtype not in (w.dtype, torch.float32):
        raise TypeError(f"{what}: results must have w's type or be fp32 (got {dtype})")
    return _OUT[dtype]


ROWS_AT_ONCE = 1 << 32     # bytes


def _rows_workspace(plan, cols, code):
    """Bytes for the rows to be summed: fp32 rows of all columns, which takes the fewest launches, up to ROWS_AT_ONCE; beyond it the least, which for
    bf16 results is about half, in bands of columns (of 2 GB of rows the bands take between 4 % less time and 3 % more)."""
    size = _lib.load().mm_group_linear_workspace
    full = size(plan.T, plan.k, cols, 1, _lib.DTYPE_F32)
    return full if full <= ROWS_AT_ONCE else size(plan.T, plan.k, cols, 1, code)


def linear_forward(x, w, plan, gather=False, reduce=False, out_dtype=None, stream=None):
    """Row p of expert e times w[e] transposed (mm_group_linear): x [n, K] in the plan's order, or with `gather` [T, K], one row per
    token; w [E, N, K] (fp16 or bf16, as x). Returns [n, N], zero in rows of no expert, or with `reduce` [T, N], each token's rows summed
    in the order of its picks; in w's type or fp32 (`out_dtype`). Rows and sums are fp32, results are rounded once."""
    N, K, code = _check_linear("linear", w, plan, gather, reduce)
    _check_rows("linear", "x", x, plan.T if gather else plan.n, K, w.dtype)
    out_dtype = w.dtype if out_dtype is None else out_dtype
    out_code, dev = _check_out("linear", out_dtype, w), plan.device
    _lib.check_tensors("linear", dev, x=x, w=w)
    with _lib.on(dev, stream):
        y = torch.empty((plan.T if reduce else plan.n, N), dtype=out_dtype, device=dev)
        if plan.n:
            x = _lib.aligned(x)
            wsb = _rows_workspace(plan, N, out_code) if reduce else 0
            ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
            _lib.call("mm_group_linear", plan._ref, x.data_ptr(), w.data_ptr(), code, K, N, int(gather), int(reduce), y.data_ptr(), out_code,
                      _p(ws), wsb, _lib.raw_stream(dev))
    return y


def linear_backward(dy, x, w, plan, gather=False, reduce=False, need_x=True, need_w=True, dw_dtype=None, stream=None):
    """(dx, dw) of linear_forward from dy [n, N] (with `reduce` [T, N]), in w's type; dw also in fp32 (`dw_dtype`). None for one that is
    not needed; x may be None without dw. With `gather` dx is [T, K], rows summed per token as by linear_forward. Experts without rows have a
    dw of zeros (mm_group_linear_inputs, mm_group_linear_weights)."""
    N, K, code = _check_linear("linear_backward", w, plan, gather, reduce)
    _check_rows("linear_backward", "dy", dy, plan.T if reduce else plan.n, N, w.dtype)
    dw_dtype = w.dtype if dw_dtype is None else dw_dtype
    dw_code, dev = _check_out("linear_backward", dw_dtype, w), plan.device
    if need_w:
        if x is None:
            raise ValueError("linear_backward: dw needs x")
        _check_rows("linear_backward", "x", x, plan.T if gather else plan.n, K, w.dtype)
    _lib.check_tensors("linear_backward", dev, dy=dy, w=w, x=x)
    dx = dw = None
    with _lib.on(dev, stream):
        dy = _lib.aligned(dy)
        if need_x:
            dx = torch.empty((plan.T if gather else plan.n, K), dtype=w.dtype, device=dev)
            if plan.n:
                wsb = _rows_workspace(plan, K, code) if gather else 0
                ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
                _lib.call("mm_group_linear_inputs", plan._ref, dy.data_ptr(), w.data_ptr(), code, K, N, int(gather), int(reduce), dx.data_ptr(),
                          code, _p(ws), wsb, _lib.raw_stream(dev))
        if need_w:
            if not plan.n:
                return dx, torch.zeros(w.shape, dtype=dw_dtype, device=dev)
            x = _lib.aligned(x)
            dw = torch.empty(w.shape, dtype=dw_dtype, device=dev)
            _lib.call("mm_group_linear_weights", plan._ref, dy.data_ptr(), x.data_ptr(), code, K, N, int(gather), int(reduce), dw.data_ptr(),
                      dw_code, _lib.raw_stream(dev))
    return dx, dw


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, plan, gather, reduce, out_dtype):
        y = linear_forward(x, w, plan, gather, reduce, out_dtype)
        ctx.save_for_backward(x, w)
        ctx.plan, ctx.rows = plan, (gather, reduce)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        dx, dw = linear_backward(dy.to(w.dtype), x, w, ctx.plan, *ctx.rows, need_x=ctx.needs_input_grad[0], need_w=ctx.needs_input_grad[1])
        return dx, dw, None, None, None, None


def linear(x, w, plan, gather=False, reduce=False, out_dtype=None):
    """linear_forward on the current stream, with gradients into x and w (an fp32 gradient is rounded to w's type first: the
    products take 16-bit operands). Under stream capture a leaf must not have an autograd graph from before the capture (refused), nor may an
    input that is not a leaf come from one (not seen here)."""
    return _captured_apply("grouped.linear", _Linear, (x, w), x, w, plan, gather, reduce, out_dtype)


# ------------------------------------------------------------------------------------------ activation

class Saved8:
    """Rows [n, 2 I] in 8 bits: codes int8 [n, 2 I] and exps int8 [n, 2 I / 32], value = code 2^exp (exp 127: NaN)."""

    def __init__(self, codes, exps, dtype):
        self.codes, self.exps, self.dtype = codes, exps, dtype


def _check_swiglu(what, rows, dtype, width, plan, weights, limit):
    if dtype not in _DTYPES:
        raise TypeError(f"{what}: rows must be fp16 or bf16 (got {dtype})")
    if width % 8 or not width:
        raise ValueError(f"{what}: I must be a multiple of 8 (got {width})")
    if plan is not None and rows != plan.n:
        raise ValueError(f"{what}: {plan.n} rows expected (got {rows})")
    if not limit >= 0:
        raise ValueError(f"{what}: limit must not be negative (got {limit})")
    if weights is not None:
        shape = (rows,) if plan is None else (plan.T, plan.k)
        if weights.dtype != torch.float32 or weights.shape != shape:
            raise ValueError(f"{what}: weights must be fp32 {list(shape)} (got {weights.dtype} {tuple(weights.shape)})")


def swiglu_forward(gu, plan=None, weights=None, limit=10.0, save8=False, stream=None):
    """(h, kept) of rows gu [n, 2 I] = [g | u]: h [n, I] = w min(silu(g), limit) clamp(u, -limit, limit) (limit 0: no clamp), with the
    routing weights fp32 [T, k] of the plan's routes (without a plan [n]; None: 1); rows of no expert are zero (mm_gated). kept is what
    swiglu_backward takes: gu, or with `save8` a Saved8 of it, in the same pass (I a multiple of 32)."""
    # (a decode step's call takes as long as its launch: little is done twice here)
    shape, dev, dtype = gu.shape, gu.device, gu.dtype
    if len(shape) != 2 or shape[1] % 2:
        raise ValueError(f"swiglu: gu [n, 2 I] expected (got {tuple(shape)})")
    n, I = shape[0], shape[1] // 2
    _check_swiglu("swiglu", n, dtype, I, plan, weights, limit)
    if save8 and I % SAVE_GROUP:
        raise ValueError(f"swiglu: save8 needs I a multiple of {SAVE_GROUP} (got {I})")
    _lib.check_tensors("swiglu", dev if plan is None else plan.device, gu=gu, weights=weights)
    with _lib.on(dev, stream):
        h = torch.empty((n, I), dtype=dtype, device=dev)
        kept = gu
        if save8:
            kept = Saved8(torch.empty((n, 2 * I), dtype=torch.int8, device=dev),
                          torch.empty((n, 2 * I // SAVE_GROUP), dtype=torch.int8, device=dev), dtype)
        if n:
            gu = _lib.aligned(gu)
            weights = None if weights is None else weights.contiguous()
            _lib.call("mm_gated", None if plan is None else plan._ref, gu.data_ptr(), _DTYPES[dtype], n, I, _p(weights), float(limit), h.data_ptr(),
                      kept.codes.data_ptr() if save8 else None, kept.exps.data_ptr() if save8 else None, _lib.raw_stream(dev))
    return h, kept


def swiglu_backward(dh, kept, plan=None, weights=None, limit=10.0, need_weights=True, need_h=False, stream=None):
    """(dgu [n, 2 I], dweights fp32 like weights, h [n, I]) from dh [n, I] and what swiglu_forward kept (mm_gated_backward). dweights is
    None without weights or need_weights; h, computed once more for the product that follows, only with need_h."""
    saved = isinstance(kept, Saved8)
    if not saved and (kept.dim() != 2 or kept.shape[1] % 2):
        raise ValueError(f"swiglu_backward: gu [n, 2 I] expected (got {tuple(kept.shape)})")
    n, I = (kept.codes if saved else kept).shape[0], (kept.codes if saved else kept).shape[1] // 2
    _check_swiglu("swiglu_backward", n, kept.dtype, I, plan, weights, limit)
    if saved:
        for name, t, shape in (("codes", kept.codes, (n, 2 * I)), ("exps", kept.exps, (n, 2 * I // SAVE_GROUP))):
            if t.dtype != torch.int8 or tuple(t.shape) != shape or not t.is_contiguous() or I % SAVE_GROUP:
                raise ValueError(f"swiglu_backward: {name} must be contiguous int8 {list(shape)}, I a multiple of {SAVE_GROUP} (got {t.dtype} {tuple(t.shape)})")
    if dh.dtype != kept.dtype or tuple(dh.shape) != (n, I):
        raise ValueError(f"swiglu_backward: dh must be {kept.dtype} {[n, I]} (got {dh.dtype} {tuple(dh.shape)})")
    dev = dh.device
    _lib.check_tensors("swiglu_backward", dev if plan is None else plan.device, dh=dh, weights=weights,
                       **({"codes": kept.codes, "exps": kept.exps} if saved else {"gu": kept}))
    with _lib.on(dev, stream):
        dgu = torch.empty((n, 2 * I), dtype=dh.dtype, device=dev)
        h = torch.empty((n, I), dtype=dh.dtype, device=dev) if need_h else None
        dweights = torch.empty(weights.shape, dtype=torch.float32, device=dev) if weights is not None and need_weights else None
        if n:
            dh = _lib.aligned(dh)
            gu = None if saved else _lib.aligned(kept)
            weights = None if weights is None else weights.contiguous()
            _lib.call("mm_gated_backward", None if plan is None else plan._ref, dh.data_ptr(), _p(gu), kept.codes.data_ptr() if saved else None,
                      kept.exps.data_ptr() if saved else None, _DTYPES[dh.dtype], n, I, _p(weights), float(limit), dgu.data_ptr(), _p(dweights),
                      _p(h), _lib.raw_stream(dev))
    return dgu, dweights, h


class _Swiglu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gu, weights, plan, limit, save8):
        h, kept = swiglu_forward(gu, plan, weights, limit, save8)
        ctx.save_for_backward(weights, *((kept.codes, kept.exps) if save8 else (gu,)))
        ctx.plan, ctx.limit, ctx.save8, ctx.dtype = plan, limit, save8, gu.dtype
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        weights, *kept = ctx.saved_tensors
        kept = Saved8(*kept, ctx.dtype) if ctx.save8 else kept[0]
        dgu, dweights, _ = swiglu_backward(dh, kept, ctx.plan, weights, ctx.limit, need_weights=ctx.needs_input_grad[1])
        return dgu, dweights, None, None, None


def swiglu(gu, plan=None, weights=None, limit=10.0, save8=False):
    """h of swiglu_forward on the current stream, with gradients into gu and the routing weights; `save8` holds gu in 8 bits between the
    passes (the gradient is that of the held values). Under stream capture as linear."""
    return _captured_apply("grouped.swiglu", _Swiglu, (gu,) if weights is None else (gu, weights), gu, weights, plan, limit, save8)
