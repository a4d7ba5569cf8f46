"""4-bit weights with group scales: dense products (W4Matrix, linear) and the routed experts of a layer (W4Store, moe).

Tensors are read in place, in this layout (checkpoints that order the weights otherwise, or pack their zero points into
words, are to be repacked first):
  q       int32 [N, K / 8]        weight k = 8 j + i of a row in bits 4 i .. 4 i + 3 of its word j
  scales  fp16 or bf16 [N, K / G] G = 32, 64 or 128 inputs per group
  zeros   uint8 [N, K / G], 0 to 16, or None (8): weight = (q - zero) * scale
Products are exact, sums fp32 (of x (16 + q) and x (16 + z), with the roundings of those). For serving: nothing here records itself in autograd, and inputs that
require a gradient are refused. moe.moe_forward takes a W4Store as it takes
an ExpertStore.
"""
import ctypes

import torch

from . import _lib

_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_OUT = {v: k for k, v in _DTYPES.items()}
_p = _lib.ptr


def _group(what, q, scales, zeros):
    """Group size of one weight tensor [..., N, K / 8], after checking its parts against each other."""
    if q.dtype != torch.int32 or scales.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"{what}: q must be int32 and scales fp16 or bf16 (got {q.dtype} and {scales.dtype})")
    if q.dim() < 2 or scales.dim() != q.dim() or scales.shape[:-1] != q.shape[:-1] or 0 in q.shape or 0 in scales.shape:
        raise ValueError(f"{what}: q [..., K / 8] and scales [..., K / group] do not match ({tuple(q.shape)}, "
                         f"{tuple(scales.shape)})")
    K, ng = q.shape[-1] * 8, scales.shape[-1]
    if K % ng or K // ng not in (32, 64, 128):
        raise ValueError(f"{what}: group must be 32, 64 or 128 (K = {K}, {ng} groups)")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError(f"{what}: zeros must be uint8 {list(scales.shape)} (got {zeros.dtype} {tuple(zeros.shape)})")
    for name, t in (("q", q), ("scales", scales), ("zeros", zeros)):
        if t is not None and not t.is_contiguous():
            raise ValueError(f"{what}: {name} must be contiguous")
    if q.data_ptr() % 16:
        raise ValueError(f"{what}: q must start at a 16-byte boundary")
    return K // ng


class W4Matrix:
    """One matrix [N, K]. Keeps the tensors it names and reads them on every product."""

    def __init__(self, q, scales, zeros=None):
        self.group = _group("W4Matrix", q, scales, zeros)
        if q.dim() != 2:
            raise ValueError(f"W4Matrix: q must be [N, K / 8] (got {tuple(q.shape)})")
        _lib.check_tensors("W4Matrix", q.device, scales=scales, zeros=zeros)
        self.q, self.scales, self.zeros = q, scales, zeros
        self.N, self.K = q.shape[0], q.shape[1] * 8
        self._c = _lib.MMW4(_p(q), _p(scales), _p(zeros))
        self._ref, self._device, self._scale_code = ctypes.byref(self._c), q.device, _DTYPES[scales.dtype]


def linear(x, W, out_dtype=None, stream=None):
    """x [..., K] times W [N, K] transposed: [..., N] in x's type or `out_dtype` (fp16, bf16 or fp32). Built for few rows."""
    # (a decode step's call takes as long as its launch: little is done twice here)
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"w4.linear: x must be fp16, bf16 or fp32 (got {x.dtype})")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    out_code = _DTYPES.get(out_dtype)
    if out_code is None:
        raise TypeError(f"w4.linear: out_dtype must be fp16, bf16 or fp32 (got {out_dtype})")
    shape, dev = x.shape, W._device
    if not shape or shape[-1] != W.K:
        raise ValueError(f"w4.linear: x [..., {W.K}] expected (got {tuple(shape)})")
    if x.requires_grad:
        _lib.no_gradient("w4.linear", x=x)
    _lib.check_tensors("w4.linear", dev, x=x)
    M = x.numel() // W.K
    with _lib.on(dev, stream):
        y = torch.empty(shape[:-1] + (W.N,), dtype=out_dtype, device=dev)
        if M == 0:
            return y
        x = _lib.aligned(x)
        ws, wsb = None, 0
        if code == _lib.DTYPE_F32:
            wsb = _lib.load().mm_w4_linear_workspace(code, M, W.K)
            ws = torch.empty(wsb, dtype=torch.uint8, device=dev)
        _lib.call("mm_w4_linear", x.data_ptr(), code, M, W.K, W.N, W._ref, W.group, W._scale_code, y.data_ptr(), out_code, _p(ws), wsb,
                  _lib.raw_stream(dev))
    return y


class W4Store:
    """The experts of one layer: gate and up rows q13 [E, 2, I, H / 8] (gate first), down rows q2 [E, H, I / 8], with their
    scales and zero points; both matrices share the group and the scales' type. limit: SwiGLU clamp (0 = off)."""

    def __init__(self, q13, scales13, zeros13, q2, scales2, zeros2, limit=10.0):
        self.group = _group("W4Store w13", q13, scales13, zeros13)
        if q13.dim() != 4 or q13.shape[1] != 2 or q2.dim() != 3:
            raise ValueError(f"W4Store: q13 [E, 2, I, H / 8] and q2 [E, H, I / 8] expected (got {tuple(q13.shape)} and "
                             f"{tuple(q2.shape)})")
        self.E, self.I, self.H = q13.shape[0], q13.shape[2], q13.shape[3] * 8
        if tuple(q2.shape) != (self.E, self.H, self.I // 8) or self.I % 8:
            raise ValueError(f"W4Store: q2 must be {[self.E, self.H, self.I // 8]} (got {tuple(q2.shape)})")
        if _group("W4Store w2", q2, scales2, zeros2) != self.group or scales2.dtype != scales13.dtype:
            raise ValueError("W4Store: w13 and w2 must share the group and the scales' type")
        _lib.check_tensors("W4Store", q13.device, scales13=scales13, zeros13=zeros13, q2=q2, scales2=scales2, zeros2=zeros2)
        self.q13, self.scales13, self.zeros13 = q13, scales13, zeros13
        self.q2, self.scales2, self.zeros2 = q2, scales2, zeros2
        self.limit = float(limit)
        self._c = _lib.MMW4Layer(_lib.MMW4(_p(q13), _p(scales13), _p(zeros13)), _lib.MMW4(_p(q2), _p(scales2), _p(zeros2)),
                                 self.E, self.H, self.I, self.group, _DTYPES[scales13.dtype], self.limit)

    def mm_layer(self):
        """The EXL3 paths ask their store for its layer here: this one has none."""
        raise TypeError("a W4Store holds no EXL3 layer: it runs on moe.moe_forward or w4.moe")


def moe(store, x, ids, w, shared_expert=None, stream=None):
    """out fp32 [T, H] = sum_j w[t, j] * expert_{ids[t, j]}(x_t) (+ expert `shared_expert` with weight 1) on 4-bit experts
    (mm_w4_moe). ids outside [0, E) contribute nothing."""
    if x.dtype not in _DTYPES:
        raise TypeError(f"w4.moe: x must be fp16, bf16 or fp32 (got {x.dtype})")
    if x.dim() != 2 or x.shape[1] != store.H:
        raise ValueError(f"w4.moe: x [T, {store.H}] expected (got {tuple(x.shape)})")
    T = x.shape[0]
    if ids.dim() != 2 or ids.shape != w.shape or ids.shape[0] != T or T and ids.shape[1] == 0:
        raise ValueError(f"w4.moe: ids and w must be [{T}, k] (got {tuple(ids.shape)} and {tuple(w.shape)})")
    shared = -1 if shared_expert is None else int(shared_expert)
    if shared_expert is not None and not 0 <= shared < store.E:
        raise ValueError(f"w4.moe: shared expert {shared} of {store.E}")
    dev = store.q13.device
    if x.requires_grad or w.requires_grad:
        _lib.no_gradient("w4.moe", x=x, w=w)
    _lib.check_tensors("w4.moe", dev, x=x, ids=ids, w=w)
    with _lib.on(dev, stream):
        out = torch.empty((T, store.H), dtype=torch.float32, device=dev)
        if T == 0:
            return out
        k = ids.shape[1]
        x, ids, w = _lib.aligned(x), ids.long().contiguous(), w.float().contiguous()
        code = _DTYPES[x.dtype]
        wsb = _lib.load().mm_w4_moe_workspace(code, T, k, shared, store.E, store.H, store.I)
        ws = torch.empty(max(wsb, 1), dtype=torch.uint8, device=dev)
        _lib.call("mm_w4_moe", ctypes.byref(store._c), _p(x), code, T, k, _p(ids), _p(w), shared, _p(out), _p(ws), wsb,
                  _lib.raw_stream(dev))
    return out
