"""The routed experts of a layer in 16-bit weights, trainable: a DenseStore of the weights, and the layer moe() with its gradients
(moe.moe_forward takes a DenseStore as it takes an ExpertStore).

Forward: the plan of the picks, gate and up rows (grouped.linear, one row of x per token), the gated activation with the routing
weights, and the down product summed per token. Between the passes a call keeps x, the plan and the gate and up rows (4 I bytes a
route, with save8 2 I); the activation's output is computed again in the backward pass.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib, grouped
from .router import _captured_apply


class DenseStore:
    """The experts of one layer: w13 [E, 2, I, H] (gate rows, then up rows) and w2 [E, H, I], both fp16 or both bf16, contiguous.
    Keeps the tensors it names and reads them on every call; the ones that require gradients get them. limit: SwiGLU clamp (0 =
    off). save8: the gate and up rows of a training step are held in 8 bits (grouped.Saved8)."""

    def __init__(self, w13, w2, limit=10.0, save8=False):
        if w13.dim() != 4 or w13.shape[1] != 2 or w2.dim() != 3 or 0 in w13.shape:
            raise ValueError(f"DenseStore: w13 [E, 2, I, H] and w2 [E, H, I] expected (got {tuple(w13.shape)} and {tuple(w2.shape)})")
        self.E, _, self.I, self.H = w13.shape
        if tuple(w2.shape) != (self.E, self.H, self.I):
            raise ValueError(f"DenseStore: w2 must be {[self.E, self.H, self.I]} (got {tuple(w2.shape)})")
        if w13.dtype not in (torch.float16, torch.bfloat16) or w2.dtype != w13.dtype:
            raise TypeError(f"DenseStore: w13 and w2 must both be fp16 or both bf16 (got {w13.dtype} and {w2.dtype})")
        step = grouped.SAVE_GROUP if save8 else 8
        if self.E > 1024 or self.H % 8 or self.I % step:
            raise ValueError(f"DenseStore: need E <= 1024, H a multiple of 8 and I of {step} (got {tuple(w13.shape)})")
        for name, t in (("w13", w13), ("w2", w2)):
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"DenseStore: {name} must be contiguous and start at a 16-byte boundary")
        if not limit >= 0:
            raise ValueError(f"DenseStore: limit must not be negative (got {limit})")
        _lib.check_tensors("DenseStore", w13.device, w2=w2)
        self.w13, self.w2, self.limit, self.save8 = w13, w2, float(limit), bool(save8)

    def mm_layer(self):
        """The EXL3 paths ask their store for its layer here: this one has none."""
        raise TypeError("a DenseStore holds no EXL3 layer: it runs on moe.moe_forward or dense.moe")


class _Moe(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, w13, w2, ids, shared, limit, save8, keep):
        ctx.w = w.dtype, w.shape[1]
        ids, w = ids.long(), w.float()
        if shared >= 0:
            one = (x.shape[0], 1)
            ids = torch.cat([ids, torch.full(one, shared, dtype=torch.long, device=x.device)], 1)
            w = torch.cat([w, torch.ones(one, dtype=torch.float32, device=x.device)], 1)
        plan = grouped.Plan(ids, w13.shape[0])
        gu = grouped.linear_forward(x, w13.flatten(1, 2), plan, gather=True)
        h, kept = grouped.swiglu_forward(gu, plan, w, limit, save8 and keep)
        out = grouped.linear_forward(h, w2, plan, reduce=True, out_dtype=torch.float32)
        if keep:
            save8 = isinstance(kept, grouped.Saved8)
            ctx.save_for_backward(x, w, w13, w2, *((kept.codes, kept.exps) if save8 else (kept,)))
            ctx.plan, ctx.limit, ctx.save8 = plan, limit, save8
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, w, w13, w2, *kept = ctx.saved_tensors
        need_x, need_w, need_13, need_2 = ctx.needs_input_grad[:4]
        plan, up = ctx.plan, w13.flatten(1, 2)
        kept = grouped.Saved8(*kept, x.dtype) if ctx.save8 else kept[0]
        dout = _lib.aligned(dout.to(x.dtype))        # the products take 16-bit operands
        dx = dw = d13 = d2 = None
        dh, _ = grouped.linear_backward(dout, None, w2, plan, reduce=True, need_w=False)
        dgu, dw, h = grouped.swiglu_backward(dh, kept, plan, w, ctx.limit, need_weights=need_w, need_h=need_2)
        if need_2:
            _, d2 = grouped.linear_backward(dout, h, w2, plan, reduce=True, need_x=False)
        if need_x or need_13:
            dx, d13 = grouped.linear_backward(dgu, x, up, plan, gather=True, need_x=need_x, need_w=need_13)
        if dw is not None:
            dtype, k = ctx.w
            dw = dw[:, :k].to(dtype)
        return dx, dw, None if d13 is None else d13.view_as(w13), d2, None, None, None, None, None


def moe(store, x, ids, w, shared_expert=None, stream=None):
    """out fp32 [T, H] = sum_j w[t, j] * expert_{ids[t, j]}(x_t) (+ expert `shared_expert` with weight 1), expert(x) = W2 (min(silu(Wg x),
    limit) clamp(Wu x)), with gradients into x, w and the store's weights. x [T, H] in the weights' type, ids int64 and w [T, k]; ids
    outside [0, E) contribute nothing and get no gradient. Gate and up rows, the weighted activation and, backward, the gradients between the
    products are rounded to the weights' type (the products' operands); sums are fp32. Under stream capture as router.topk."""
    if x.dtype != store.w13.dtype:
        raise TypeError(f"dense.moe: x must have the weights' type {store.w13.dtype} (got {x.dtype})")
    if x.dim() != 2 or x.shape[1] != store.H:
        raise ValueError(f"dense.moe: x [T, {store.H}] expected (got {tuple(x.shape)})")
    T = x.shape[0]
    if ids.dim() != 2 or ids.shape != w.shape or ids.shape[0] != T or ids.shape[1] == 0:
        raise ValueError(f"dense.moe: ids and w must be [{T}, k] (got {tuple(ids.shape)} and {tuple(w.shape)})")
    shared = -1 if shared_expert is None else int(shared_expert)
    if shared_expert is not None and not 0 <= shared < store.E:
        raise ValueError(f"dense.moe: shared expert {shared} of {store.E}")
    dev = store.w13.device
    _lib.check_tensors("dense.moe", dev, x=x, ids=ids, w=w)
    with _lib.on(dev, stream):
        leaves = (x, w, store.w13, store.w2)
        keep = torch.is_grad_enabled() and any(t.requires_grad for t in leaves)
        return _captured_apply("dense.moe", _Moe, leaves, *leaves, ids, shared, store.limit, store.save8, keep,
                               instead="the *_forward and *_backward functions of grouped")
