"""Operators around the expert layer as timed and checked cases: the load-balance loss of a router with its gradient, the
router's backward pass, and products with 4-bit group-scaled weights, dense and as the routed experts of a layer.

A case names the operator (`kind`), its sizes and its types:

  balance   router.balance_loss_forward over the logits and picks of B sequences; with `grad` also
            router.balance_loss_backward
  router    router.topk_backward: gradients of the routing weights and of the logits into the hidden states and the gate
  linear    w4.linear: y = x W^T with W in 4 bits, one scale (and zero point) per group of `group` inputs
  experts   moe.moe_forward over a w4.W4Store: gate/up, SwiGLU, down and the weighted sum of a layer's routed experts

Expert shapes are the library's own (H 4096 / I 2048, H 5120 / I 2304) and the small one of its tests (H 1024 / I 512).
`own` False computes the definitions with elementary torch operations in fp32.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
LIMIT = 10.0                                                # SwiGLU clamp of the expert layers


def _package():
    path = os.path.join(_ROOT, "dsv41-flash-offload_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from mi355moe import moe, router, w4
    return moe, router, w4


def _balance(name, B, T, E, k, dtype="f32", score="softmax", mask=False, grad=True):
    return {"name": name, "kind": "balance", "B": B, "T": T, "E": E, "k": k, "dtype": dtype, "score": score, "mask": mask,
            "grad": grad}


def _router(name, T, H, E, k, dense=True):
    return {"name": name, "kind": "router", "T": T, "H": H, "E": E, "k": k, "dense": dense}


def _linear(name, M, K, N, group, dtype="bf16", zeros=False):
    return {"name": name, "kind": "linear", "M": M, "K": K, "N": N, "group": group, "dtype": dtype, "zeros": zeros}


def _experts(name, T, E, H, I, k, group, dtype="bf16", zeros=False, shared=False):
    return {"name": name, "kind": "experts", "T": T, "E": E, "H": H, "I": I, "k": k, "group": group, "dtype": dtype,
            "zeros": zeros, "shared": shared}


def listed():
    return [
        # load statistics of one small step: the smallest call
        _balance("balance 64 tokens", 1, 64, 384, 8, grad=False),
        # a micro-batch of padded sequences, each with its own loss, bf16 logits and sigmoid scores
        _balance("balance 8 sequences", 8, 1500, 160, 6, dtype="bf16", score="sigmoid", mask=True),
        # a whole training batch, loss and gradient
        _balance("balance 16384 tokens", 1, 16384, 384, 8),
        # router calibration on a short batch of odd length
        _router("router backward 700", 700, 4096, 384, 8),
        # ... and on a whole batch
        _router("router backward 16384", 16384, 4096, 384, 8),
        # one token through a square projection: latency counts
        _linear("linear 1 row", 1, 4096, 4096, 128),
        # a speculative step of five tokens through a shared expert's gate/up, zero points
        _linear("linear 5 rows", 5, 5120, 4608, 64, dtype="f16", zeros=True),
        # a short prompt
        _linear("linear 300 rows", 300, 4096, 8192, 128),
        # one request decoding through 384 routed experts and the shared one
        _experts("experts 1 token", 1, 384, 4096, 2048, 8, 128, shared=True),
        # the batch the decode benchmark is quoted on, fp32 hidden states as the previous layer leaves them
        _experts("experts 4 tokens", 4, 384, 4096, 2048, 8, 128, dtype="f32", shared=True),
        # two dozen requests on the larger experts of a smaller layer, zero points
        _experts("experts 24 tokens", 24, 64, 5120, 2304, 6, 128, dtype="f16", zeros=True),
        # a full batch through small experts with fine groups: some twenty rows each
        _experts("experts 200 tokens", 200, 32, 1024, 512, 4, 32),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(["balance", "router", "linear", "experts"], [0.25, 0.2, 0.3, 0.25])[0]
    if kind == "balance":
        B = rng.choice([1, 1, 2, 5, 8])
        E = _log_int(rng, 8, 512)
        return {"kind": kind, "B": B, "T": _log_int(rng, 1, 16384 // B), "E": E, "k": rng.randint(1, 8),
                "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "score": rng.choice(["softmax", "sigmoid"]),
                "mask": rng.random() < 0.5, "grad": rng.random() < 0.75}
    if kind == "router":
        E = _log_int(rng, 8, 384)
        return {"kind": kind, "T": _log_int(rng, 1, 16384), "H": 16 * _log_int(rng, 16, 256), "E": E, "k": rng.randint(1, 8),
                "dense": rng.random() < 0.7}
    group = rng.choice([32, 64, 128])
    if kind == "linear":
        return {"kind": kind, "M": _log_int(rng, 1, 300), "K": group * _log_int(rng, 256 // group, 4096 // group),
                "N": _log_int(rng, 64, 8192), "group": group, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "zeros": rng.random() < 0.5}
    H, I, E, most = rng.choice([(4096, 2048, 384, 8), (4096, 2048, 48, 24), (5120, 2304, 64, 20), (1024, 512, 32, 200)])
    return {"kind": kind, "T": _log_int(rng, 1, most), "E": E, "H": H, "I": I, "k": rng.randint(1, 8 if E > 32 else 4),
            "group": group, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]), "zeros": rng.random() < 0.5,
            "shared": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _picks(g, T, E, k):
    """k distinct experts per token with a skewed popularity, int64 [T, k]."""
    pop = -1.1 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    pop = pop[torch.randperm(E, generator=g, device="cuda")]
    u = torch.rand((T, E), generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
    return torch.topk(pop - torch.log(-torch.log(u)), k, dim=1).indices.contiguous()


def _weights(g, group, zeros, *shape):
    """4-bit weights [..., N, K]: packed int32 [..., N, K / 8] (k = 8 j + i in bits 4 i .. 4 i + 3), fp16 scales and uint8
    zero points (or None) [..., N, K / group], scaled so that a product with N(0, 1) inputs is N(0, 1)."""
    K = shape[-1]
    q = torch.empty(shape[:-1] + (K // 8,), dtype=torch.int32, device="cuda").random_(-2 ** 31, 2 ** 31, generator=g)
    gs = shape[:-1] + (K // group,)
    s = ((0.5 + torch.rand(gs, generator=g, device="cuda")) / (4.6 * math.sqrt(K))).half()
    z = torch.randint(5, 12, gs, generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return q, s, z


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["kind"] == "balance":
        B, T, E, k = (case[n] for n in ("B", "T", "E", "k"))
        s["logits"] = _rand(g, B, T, E).to(DTYPES[case["dtype"]])
        s["ids"] = _picks(g, B * T, E, k).view(B, T, k)
        s["mask"] = None
        if case["mask"]:                                     # right-padded sequences
            lens = torch.randint(T // 2, T + 1, (B,), generator=g, device="cuda")
            s["mask"] = torch.arange(T, device="cuda")[None, :] < lens[:, None]
        s["dloss"] = 0.5 + torch.rand((B,), generator=g, device="cuda")
    elif case["kind"] == "router":
        T, H, E, k = (case[n] for n in ("T", "H", "E", "k"))
        s["x"] = _rand(g, T, H).bfloat16()
        s["gate"] = _rand(g, E, H) / math.sqrt(H)
        s["ids"] = _picks(g, T, E, k)
        s["w"] = torch.softmax(_rand(g, T, k), 1)
        s["dw"] = _rand(g, T, k)
        s["dlogits"] = _rand(g, T, E) * 0.05 if case["dense"] else None
    elif case["kind"] == "linear":
        s["x"] = _rand(g, case["M"], case["K"]).to(DTYPES[case["dtype"]])
        s["w"] = _weights(g, case["group"], case["zeros"], case["N"], case["K"])
    else:
        T, E, H, I, k = (case[n] for n in ("T", "E", "H", "I", "k"))
        n = E + 1 if case["shared"] else E                   # the shared expert is the last one
        s["x"] = _rand(g, T, H).to(DTYPES[case["dtype"]])
        s["w13"] = _weights(g, case["group"], case["zeros"], n, 2, I, H)
        s["w2"] = _weights(g, case["group"], case["zeros"], n, H, I)
        s["ids"] = _picks(g, T, E, k)
        s["w"] = torch.softmax(_rand(g, T, k), 1)
        s["shared"] = E if case["shared"] else None
    if own:
        moe, router, w4 = _package()
        s["moe"], s["router"], s["w4"] = moe, router, w4
        if case["kind"] == "linear":                         # the handles name the tensors above, nothing is laid out anew
            s["handle"] = w4.W4Matrix(*s["w"])
        elif case["kind"] == "experts":
            s["handle"] = w4.W4Store(*s["w13"], *s["w2"], limit=LIMIT)
    return s


# ------------------------------------------------------------------------------------------------- plain forms

def _plain_probs(logits, score):
    x = logits.float()
    if score == "softmax":
        p = torch.exp(x - x.amax(-1, keepdim=True))
        return p / p.sum(-1, keepdim=True), None
    sg = 1.0 / (1.0 + torch.exp(-x))
    return sg / sg.sum(-1, keepdim=True), sg


def _plain_balance(s):
    c = s["case"]
    B, T, E, k = (c[n] for n in ("B", "T", "E", "k"))
    p, sg = _plain_probs(s["logits"], c["score"])
    live = torch.ones((B, T), dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    counts = torch.zeros((B, E), dtype=torch.int32, device="cuda")
    counts.scatter_add_(1, s["ids"].reshape(B, T * k), live[:, :, None].expand(B, T, k).reshape(B, T * k).int())
    n = live.sum(1)
    load = torch.where(live[:, :, None], p, 0.0).sum(1)
    fac = E / (k * (n.float() ** 2).clamp_min(1.0))
    loss = fac * (counts.float() * load).sum(1)
    if not c["grad"]:
        return loss, counts
    f = counts.float()[:, None, :]
    d = p * (f - (f * p).sum(-1, keepdim=True))
    if sg is not None:
        d = d * (1.0 - sg)
    d = torch.where(live[:, :, None], d * (s["dloss"] * fac)[:, None, None], 0.0)
    return loss, counts, d.to(s["logits"].dtype)


def _plain_router(s):
    T, E = s["case"]["T"], s["case"]["E"]
    w, dw = s["w"], s["dw"]
    d = torch.zeros((T, E), device="cuda") if s["dlogits"] is None else s["dlogits"].clone()
    d.scatter_add_(1, s["ids"], w * (dw - (w * dw).sum(1, keepdim=True)))
    return (d @ s["gate"]).to(s["x"].dtype), d.t() @ s["x"].float()


def _plain_dense(q, sc, z):
    """fp32 weights [..., N, K] of packed ones."""
    sh = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    v = ((q[..., None] >> sh) & 15).float().flatten(-2)
    v = v.unflatten(-1, (sc.shape[-1], -1))
    v -= 8.0 if z is None else z[..., None].float()
    v *= sc[..., None].float()
    return v.flatten(-2)


def _plain_linear(s):
    return (s["x"].float() @ _plain_dense(*s["w"]).t()).to(s["x"].dtype)


def _plain_experts(s):
    T, k = s["ids"].shape
    ids, w = s["ids"], s["w"]
    if s["shared"] is not None:
        ids = torch.cat([ids, torch.full((T, 1), s["shared"], dtype=ids.dtype, device="cuda")], 1)
        w = torch.cat([w, torch.ones((T, 1), device="cuda")], 1)
        k += 1
    r = ids.reshape(-1)
    x = s["x"].float().repeat_interleave(k, 0)[:, :, None]

    def pick(t):
        return None if t is None else t[r]

    q, sc, z = s["w13"]
    gu = torch.matmul(_plain_dense(q[r], sc[r], pick(z)).flatten(1, 2), x)[:, :, 0]
    g, u = gu.chunk(2, 1)
    h = (g / (1.0 + torch.exp(-g))).clamp(max=LIMIT) * u.clamp(-LIMIT, LIMIT)
    q, sc, z = s["w2"]
    y = torch.matmul(_plain_dense(q[r], sc[r], pick(z)), h[:, :, None])[:, :, 0]
    return (y.view(T, k, -1) * w[:, :, None]).sum(1)


# ------------------------------------------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    if not own:
        return {"balance": _plain_balance, "router": _plain_router, "linear": _plain_linear,
                "experts": _plain_experts}[c["kind"]](s)
    if c["kind"] == "balance":
        loss, counts, tokens, _ = s["router"].balance_loss_forward(s["logits"], s["ids"], mask=s["mask"], score=c["score"])
        if not c["grad"]:
            return loss, counts
        return loss, counts, s["router"].balance_loss_backward(s["dloss"], s["logits"], counts, tokens, c["k"], mask=s["mask"],
                                                               score=c["score"])
    if c["kind"] == "router":
        return s["router"].topk_backward(s["x"], s["gate"], s["ids"], s["w"], dw=s["dw"], dlogits=s["dlogits"])
    if c["kind"] == "linear":
        return s["w4"].linear(s["x"], s["handle"])
    return s["moe"].moe_forward(s["handle"], s["x"], s["ids"], s["w"], shared_expert=s["shared"])


def work(case):
    """Bytes and FLOPs of one pass: inputs read once, outputs written once, the products of the definition."""
    size = {"f16": 2, "bf16": 2, "f32": 4}
    if case["kind"] == "balance":
        B, T, E, k = (case[n] for n in ("B", "T", "E", "k"))
        el = B * T * E
        passes = 3 if case["grad"] else 1                    # read forward, read backward, gradient written
        return {"bytes": passes * el * size[case["dtype"]] + B * T * (8 * k + (1 if case["mask"] else 0)) + 4 * B * (E + 1),
                "flops": el * (12 if case["grad"] else 5)}
    if case["kind"] == "router":
        T, H, E, k = (case[n] for n in ("T", "H", "E", "k"))
        return {"bytes": 4 * T * H + 8 * E * H + T * (16 * k + (4 * E if case["dense"] else 0)), "flops": 4 * T * H * E}
    per = 0.5 + (3 if case["zeros"] else 2) / case["group"]  # bytes of a weight with its share of scale and zero point
    if case["kind"] == "linear":
        M, K, N = (case[n] for n in ("M", "K", "N"))
        return {"bytes": int(K * N * per) + M * (K + N) * size[case["dtype"]], "flops": 2 * M * K * N}
    T, E, H, I, k = (case[n] for n in ("T", "E", "H", "I", "k"))
    # distinct experts of T k picks at the popularity of _picks, as successive independent draws meet them
    p = np.arange(1, E + 1, dtype=np.float64) ** -1.1
    used = float((1 - (1 - np.minimum(1.0, k * p / p.sum())) ** T).sum())
    used = min(max(used, float(k)), float(E)) + (1 if case["shared"] else 0)
    routes = T * (k + (1 if case["shared"] else 0))
    return {"bytes": int(used * 3 * H * I * per) + T * H * (size[case["dtype"]] + 4) + 12 * routes,
            "flops": 6 * routes * H * I}


# ------------------------------------------------------------------------------------------------- 64-bit results

def _exact_weights(q, sc, z):
    """float64 weights [N, K] from the packed words of one matrix, nibble by nibble of the bytes."""
    b = q.contiguous().view(torch.uint8).to(torch.int16)
    v = torch.stack([b % 16, b // 16], -1).reshape(q.shape[0], -1).double()
    group = v.shape[1] // sc.shape[1]
    zero = torch.full_like(sc, 8.0, dtype=torch.float64) if z is None else z.double()
    return (v - zero.repeat_interleave(group, 1)) * sc.double().repeat_interleave(group, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "balance":
        B, T, E, k = (case[n] for n in ("B", "T", "E", "k"))
        losses, grads = [], []
        for b in range(B):
            rows = torch.arange(T, device="cuda") if s["mask"] is None else s["mask"][b].nonzero()[:, 0]
            x, n = s["logits"][b, rows].double(), rows.numel()
            sg = torch.sigmoid(x)
            p = torch.softmax(x, 1) if case["score"] == "softmax" else sg / sg.sum(1, keepdim=True)
            f = torch.bincount(s["ids"][b, rows].reshape(-1), minlength=E).double()
            fac = E / (k * n * n) if n else 0.0
            losses.append(fac * (p @ f).sum())
            if case["grad"]:
                dp = f[None, :] - (p @ f)[:, None]           # dL/dp up to a constant per row, times the row's Jacobian
                d = p * dp if case["score"] == "softmax" else p * (1 - sg) * dp
                full = torch.zeros((T, E), dtype=torch.float64, device="cuda")
                full[rows] = d * (fac * s["dloss"][b].double())
                grads.append(full)
        loss = torch.stack(losses)
        return (loss, None, torch.stack(grads)) if case["grad"] else (loss, None)
    if case["kind"] == "router":
        T, E = case["T"], case["E"]
        w, dw = s["w"].double(), s["dw"].double()
        d = w * dw - w * (w * dw).sum(1, keepdim=True)
        full = torch.zeros((T, E), dtype=torch.float64, device="cuda")
        full[torch.arange(T, device="cuda")[:, None], s["ids"]] = d
        if s["dlogits"] is not None:
            full += s["dlogits"].double()
        return full @ s["gate"].double(), full.t().contiguous() @ s["x"].double()
    if case["kind"] == "linear":
        return s["x"].double() @ _exact_weights(*s["w"]).t().contiguous()
    T, k = s["ids"].shape
    out = torch.zeros((T, case["H"]), dtype=torch.float64, device="cuda")
    x = s["x"].double()

    def part(t, *at):
        return None if t is None else t[at]

    def expert(e, rows):
        g, u = (x[rows] @ _exact_weights(s["w13"][0][e, j], s["w13"][1][e, j], part(s["w13"][2], e, j)).t() for j in (0, 1))
        h = torch.clamp(g * torch.sigmoid(g), max=LIMIT) * torch.clamp(u, -LIMIT, LIMIT)
        return h @ _exact_weights(s["w2"][0][e], s["w2"][1][e], part(s["w2"][2], e)).t()

    for e in torch.unique(s["ids"]).tolist():
        t, j = (s["ids"] == e).nonzero(as_tuple=True)
        out.index_add_(0, t, expert(e, t) * s["w"][t, j].double()[:, None])
    if s["shared"] is not None:
        out += expert(s["shared"], torch.arange(T, device="cuda"))
    return out
