"""The router with gradients: top-k routing and its backward pass, and the load-balance loss with per-expert counts.

For calibrating or training a router over a layer's experts: topk() and balance_loss() record themselves in autograd; the
*_forward / *_backward functions are the same kernels without it. Every computation runs in libmi355moe.so on the current
stream (or `stream`); no call synchronises the host.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_SCORES = {"softmax": 0, "sigmoid": 1}        # MM_SCORE_*

_p = _lib.ptr


def _capture_stream(device):
    """Address of the device's current stream, on which a capture runs."""
    return _lib.raw_stream(device) if device.type == "cuda" else None


def _captured_apply(what, fn, leaves, *args, instead=None):
    """fn.apply(*args), for `what`, whose kernels without autograd are `instead`. Under stream capture, a leaf among its inputs may not
    have its gradient node in an autograd graph from before the capture: the captured backward would go to that node's stream, which
    invalidates the capture and ends the process. (A node that a captured call made belongs to that capture's stream, and passes in
    captures of that stream only.)"""
    leaves = [t for t in leaves if t.requires_grad and t.is_leaf]
    if not (leaves and torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing()):
        return fn.apply(*args)

    def notes(t):
        return torch.autograd.graph.get_gradient_edge(t).node.metadata

    for t in leaves:
        if notes(t).get("mi355moe captured") == (t.device, _capture_stream(t.device)):
            continue
        notes(t)["mi355moe seen"] = True                      # gone with the node if no graph holds it
        if notes(t).pop("mi355moe seen", None):
            raise RuntimeError(f"{what}: an input has an autograd graph from before the stream capture; drop it first, or capture "
                               f"{instead or f'{what}_forward and {what}_backward'}")
    out = fn.apply(*args)
    for t in leaves:
        notes(t)["mi355moe captured"] = (t.device, _capture_stream(t.device))
    return out


# ------------------------------------------------------------------------------------------ router top-k

def _check_router(what, x, gate):
    if x.dim() != 2 or gate.dim() != 2 or x.shape[1] != gate.shape[1]:
        raise ValueError(f"{what}: x [T, H] and gate [E, H] expected (got {tuple(x.shape)} and {tuple(gate.shape)})")
    if x.dtype != torch.bfloat16 or gate.dtype != torch.float32:
        raise TypeError(f"{what}: x must be bf16 and gate fp32 (got {x.dtype} and {gate.dtype})")


def topk_forward(x, gate, k, stream=None):
    """(ids int64 [T, k], w fp32 [T, k], logits fp32 [T, E]) of x bf16 [T, H] and gate fp32 [E, H]: the k largest logits of
    each token (ties to the lower expert) and the softmax over them (mm_router_topk)."""
    _check_router("topk", x, gate)
    (T, H), E = x.shape, gate.shape[0]
    _lib.check_tensors("topk", x.device, gate=gate)
    with _lib.on(x.device, stream):
        x, gate = _lib.aligned(x), _lib.aligned(gate)
        ids = torch.empty((T, k), dtype=torch.int64, device=x.device)
        w = torch.empty((T, k), dtype=torch.float32, device=x.device)
        logits = torch.empty((T, E), dtype=torch.float32, device=x.device)
        if T:
            _lib.call("mm_router_topk", _p(x), T, H, _p(gate), E, int(k), _p(logits), _p(ids), _p(w), _lib.raw_stream(x.device))
    return ids, w, logits


def topk_backward(x, gate, ids, w, dw=None, dlogits=None, need_x=True, need_gate=True, stream=None):
    """(dx bf16 [T, H], dgate fp32 [E, H]) from the gradients dw [T, k] and dlogits [T, E] (fp32, either may be None) of
    topk_forward's outputs (mm_router_backward); None for one that is not needed."""
    _check_router("topk_backward", x, gate)
    (T, H), E = x.shape, gate.shape[0]
    if dw is None and dlogits is None:
        raise ValueError("topk_backward: neither dw nor dlogits given")
    k = ids.shape[1] if ids.dim() == 2 else 0
    if tuple(ids.shape) != (T, k) or k < 1 or tuple(w.shape) != (T, k):
        raise ValueError(f"topk_backward: ids and w must be [{T}, k] (got {tuple(ids.shape)} and {tuple(w.shape)})")
    for name, t, shape in (("dw", dw, (T, k)), ("dlogits", dlogits, (T, E))):
        if t is not None and (tuple(t.shape) != shape or t.dtype != torch.float32):
            raise ValueError(f"topk_backward: {name} must be fp32 {list(shape)} (got {t.dtype} {tuple(t.shape)})")
    if ids.dtype != torch.int64 or w.dtype != torch.float32:
        raise TypeError(f"topk_backward: ids must be int64 and w fp32 (got {ids.dtype} and {w.dtype})")
    _lib.check_tensors("topk_backward", x.device, gate=gate, ids=ids, w=w, dw=dw, dlogits=dlogits)
    if not (need_x or need_gate):
        return None, None
    with _lib.on(x.device, stream):
        x, gate, ids, w = _lib.aligned(x), gate.contiguous(), ids.contiguous(), w.contiguous()
        dw = None if dw is None else dw.contiguous()
        dlogits = None if dlogits is None else dlogits.contiguous()
        dx = torch.empty((T, H), dtype=x.dtype, device=x.device) if need_x else None
        dgate = torch.empty((E, H), dtype=torch.float32, device=x.device) if need_gate else None
        wsb = _lib.load().mm_router_backward_workspace(T, H, E)
        ws = torch.empty(max(wsb, 1), dtype=torch.uint8, device=x.device)
        _lib.call("mm_router_backward", _p(x), T, H, _p(gate), E, k, _p(ids), _p(w), _p(dw), _p(dlogits), _p(dx), _p(dgate),
                  _p(ws), wsb, _lib.raw_stream(x.device))
    return dx, dgate


class _TopK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, k):
        ids, w, logits = topk_forward(x, gate, k)
        ctx.save_for_backward(x, gate, ids, w)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return ids, w, logits

    @staticmethod
    @once_differentiable
    def backward(ctx, _dids, dw, dlogits):
        if dw is None and dlogits is None:
            return None, None, None
        x, gate, ids, w = ctx.saved_tensors
        dx, dgate = topk_backward(x, gate, ids, w, dw, dlogits, ctx.needs_input_grad[0], ctx.needs_input_grad[1])
        return dx, dgate, None


def topk(x, gate, k):
    """topk_forward on the current stream, with gradients of w and logits into x and gate. Under stream capture a leaf must not
    have an autograd graph from before the capture (refused), nor may an input that is not a leaf come from one (not seen here)."""
    return _captured_apply("topk", _TopK, (x, gate), x, gate, k)


# ------------------------------------------------------------------------------------------ load balance

def _check_balance(what, logits, k, mask, score):
    """(B, T, E) of logits [T, E] or [B, T, E]."""
    if logits.dim() not in (2, 3):
        raise ValueError(f"{what}: logits [T, E] or [B, T, E] expected (got {tuple(logits.shape)})")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"{what}: logits must be fp16, bf16 or fp32 (got {logits.dtype})")
    if score not in _SCORES:
        raise ValueError(f"{what}: score must be one of {sorted(_SCORES)} (got {score!r})")
    if mask is not None:
        if mask.shape != logits.shape[:-1]:
            raise ValueError(f"{what}: mask must be {list(logits.shape[:-1])} (got {tuple(mask.shape)})")
        if mask.dtype not in (torch.bool, torch.uint8):
            raise TypeError(f"{what}: mask must be bool or uint8 (got {mask.dtype})")
    if not 1 <= k <= 32:
        raise ValueError(f"{what}: need 1 <= k <= 32 (got {k})")
    return (1,) * (3 - logits.dim()) + tuple(logits.shape)


def balance_loss_forward(logits, ids, mask=None, score="softmax", stream=None):
    """(loss fp32, counts int32, tokens int32, load fp32) of the load-balance loss
    E / (k n^2) sum_e counts[e] sum_t p[t][e] (mm_balance_loss): logits [T, E] and ids int64 [T, k] of one loss (loss and
    tokens 0-d, counts and load [E]), or [B, T, E] and [B, T, k] with a loss per sequence ([B] and [B, E]). p are the
    softmax of the logits or their normalised sigmoids; tokens with mask False take no part."""
    k = ids.shape[-1] if ids.dim() else 0
    B, T, E = _check_balance("balance_loss", logits, k, mask, score)
    if ids.shape[:-1] != logits.shape[:-1] or ids.dim() != logits.dim():
        raise ValueError(f"balance_loss: ids must be {list(logits.shape[:-1])} + [k] (got {tuple(ids.shape)})")
    if ids.dtype != torch.int64:
        raise TypeError(f"balance_loss: ids must be int64 (got {ids.dtype})")
    _lib.check_tensors("balance_loss", logits.device, ids=ids, mask=mask)
    lead, dev = logits.shape[:-2], logits.device
    with _lib.on(dev, stream):
        logits, ids = logits.contiguous(), ids.contiguous()
        mask = None if mask is None else mask.contiguous()
        loss = torch.empty(lead, dtype=torch.float32, device=dev)
        load = torch.empty(lead + (E,), dtype=torch.float32, device=dev)
        tokens, counts = torch.empty_like(loss, dtype=torch.int32), torch.empty_like(load, dtype=torch.int32)
        wsb = _lib.load().mm_balance_workspace(B, T, E)
        ws = torch.empty(wsb, dtype=torch.uint8, device=dev) if wsb else None
        _lib.call("mm_balance_loss", _p(logits), _DTYPES[logits.dtype], _p(ids), _p(mask), B, T, E, k, _SCORES[score],
                  _p(loss), _p(counts), _p(tokens), _p(load), _p(ws), wsb, _lib.raw_stream(dev))
    return loss, counts, tokens, load


def balance_loss_backward(dloss, logits, counts, tokens, k, mask=None, score="softmax", stream=None):
    """Gradient of balance_loss_forward's loss into the logits (their type and shape) from dloss (fp32, the loss's shape) and
    the forward's counts and tokens (mm_balance_loss_backward). Counts and tokens summed over data-parallel ranks give the
    gradient of the loss over all ranks' tokens."""
    B, T, E = _check_balance("balance_loss_backward", logits, k, mask, score)
    lead, dev = logits.shape[:-2], logits.device
    if dloss.shape != lead or dloss.dtype != torch.float32:
        raise ValueError(f"balance_loss_backward: dloss must be fp32 {list(lead)} (got {dloss.dtype} {tuple(dloss.shape)})")
    if counts.shape != lead + (E,) or counts.dtype != torch.int32:
        raise ValueError(f"balance_loss_backward: counts must be int32 {list(lead + (E,))} (got {counts.dtype} {tuple(counts.shape)})")
    if tokens.shape != lead or tokens.dtype != torch.int32:
        raise ValueError(f"balance_loss_backward: tokens must be int32 {list(lead)} (got {tokens.dtype} {tuple(tokens.shape)})")
    _lib.check_tensors("balance_loss_backward", dev, dloss=dloss, counts=counts, tokens=tokens, mask=mask)
    with _lib.on(dev, stream):
        logits, dloss, counts, tokens = logits.contiguous(), dloss.contiguous(), counts.contiguous(), tokens.contiguous()
        mask = None if mask is None else mask.contiguous()
        dlogits = torch.empty_like(logits)
        _lib.call("mm_balance_loss_backward", _p(dloss), _p(logits), _DTYPES[logits.dtype], _p(mask), _p(counts), _p(tokens), B, T,
                  E, int(k), _SCORES[score], _p(dlogits), _lib.raw_stream(dev))
    return dlogits


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask, score):
        loss, counts, tokens, _ = balance_loss_forward(logits, ids, mask, score)
        ctx.save_for_backward(logits, mask, counts, tokens)
        ctx.k, ctx.score = ids.shape[-1], score
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        return loss, counts

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _dcounts):
        if dloss is None:
            return None, None, None, None
        logits, mask, counts, tokens = ctx.saved_tensors
        return balance_loss_backward(dloss, logits, counts, tokens, ctx.k, mask, ctx.score), None, None, None


def balance_loss(logits, ids, mask=None, score="softmax"):
    """(loss, counts) of balance_loss_forward on the current stream, with the gradient of the loss into the logits (the counts
    are constants of it); under stream capture as topk."""
    return _captured_apply("balance_loss", _BalanceLoss, (logits,), logits, ids, mask, score)
