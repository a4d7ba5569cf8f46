"""Trainable experts as timed and checked cases: products grouped by expert over ragged rows, in each direction, and the gated
activation between them with its 8-bit checkpoint.

A case names the operator (`kind`), its sizes and its types. T tokens pick k of E experts each; the n = T k routes, sorted by
expert, are the rows of the products.

  product  y[p] = x[p] W[e]^T over the rows p of each expert e, W [E, N, K]. `pass` is the direction: "forward"
           (grouped.linear_forward, with the plan made from the picks in the pass), "inputs" or "weights" (grouped.linear_backward
           for one of the two gradients, with the forward's plan). `side` is the layer's product: "up" reads one row of x per token
           (gather), "down" reads one row per route and sums the rows of a token (reduce).
  gated    grouped.swiglu_forward over the rows [g | u] and, with `grad`, grouped.swiglu_backward; with `save8` what the forward
           keeps for the backward is held in 8 bits, and the backward gives h again.

Expert shapes are the library's own (H 4096 / I 2048, H 5120 / I 2304) and the small one of its tests (H 1024 / I 512).
`own` False computes the definitions with elementary torch operations in fp32.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = 10.0                                                # SwiGLU clamp of the expert layers
GROUP = 32                                                  # values that share a scale in the 8-bit checkpoint


def _package():
    path = os.path.join(_ROOT, "dsv41-flash-offload_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from mi355moe import grouped
    return grouped


def _product(name, way, side, T, E, k, H, I, dtype="bf16", skew=0.5, drop=0.0):
    return {"name": name, "kind": "product", "pass": way, "side": side, "T": T, "E": E, "k": k, "H": H, "I": I, "dtype": dtype,
            "skew": skew, "drop": drop}


def _gated(name, T, E, k, I, dtype="bf16", weighted=True, save8=False, grad=False, drop=0.0):
    return {"name": name, "kind": "gated", "T": T, "E": E, "k": k, "I": I, "dtype": dtype, "weighted": weighted, "save8": save8,
            "grad": grad, "skew": 0.5, "drop": drop}


def listed():
    return [
        # one request decoding through a trained layer: eight experts of one row each
        _product("up 1 token", "forward", "up", 1, 384, 8, 4096, 2048),
        # two dozen requests on the larger experts of a smaller layer, summed per token
        _product("down 24 tokens", "forward", "down", 24, 64, 6, 5120, 2304, dtype="f16"),
        # a prompt of odd length through small experts, some picks dropped
        _product("up 701 tokens", "forward", "up", 701, 32, 4, 1024, 512, drop=0.1),
        # a training batch through all experts of a layer: some 340 ragged rows each
        _product("up 16384 tokens", "forward", "up", 16384, 384, 8, 4096, 2048),
        # gradient into the tokens of a short sequence
        _product("up inputs 700 tokens", "inputs", "up", 700, 64, 6, 5120, 2304),
        # ... and into the activations of a whole batch
        _product("down inputs 16384 tokens", "inputs", "down", 16384, 64, 8, 4096, 2048),
        # gradient of small experts' weights, fp16
        _product("down weights 701 tokens", "weights", "down", 701, 32, 4, 1024, 512, dtype="f16", drop=0.1),
        # ... and of a large layer's gate and up over a whole batch
        _product("up weights 16384 tokens", "weights", "up", 16384, 64, 8, 4096, 2048),
        # the activation of one decoded token
        _gated("gated 1 token", 1, 384, 8, 2048),
        # a short sequence: forward, and backward from the values as they were
        _gated("gated 700 tokens", 700, 64, 6, 2304, dtype="f16", grad=True),
        # a whole batch: forward, and backward from the 8-bit checkpoint
        _gated("gated 16384 tokens", 16384, 384, 8, 2048, save8=True, grad=True, drop=0.02),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    H, I = rng.choice([(4096, 2048), (5120, 2304), (1024, 512)])
    dtype, drop = rng.choice(["bf16", "bf16", "f16"]), rng.choice([0.0, 0.0, 0.05, 0.3])
    if rng.random() < 0.7:
        way = rng.choice(["forward", "forward", "inputs", "weights"])
        E = _log_int(rng, 4, 64) if way == "weights" or H > 4096 else _log_int(rng, 4, 384)
        c = _product(None, way, rng.choice(["up", "down"]), _log_int(rng, 1, 11000), E, rng.randint(1, min(8, E)), H, I, dtype,
                     rng.choice([0.0, 0.5, 1.1]), drop)
    else:
        E = _log_int(rng, 8, 384)
        c = _gated(None, _log_int(rng, 1, 11000), E, rng.randint(1, 8), I, dtype, rng.random() < 0.7, rng.random() < 0.5,
                   rng.random() < 0.7, drop)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _rand(g, dtype, *shape):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)


def _picks(g, case):
    """k distinct experts per token, popularity spread by `skew`, int64 [T, k]; a share `drop` of the picks is -1 (none)."""
    T, E, k = (case[n] for n in ("T", "E", "k"))
    pop = -case["skew"] * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    pop = pop[torch.randperm(E, generator=g, device="cuda")]
    u = torch.rand((T, E), generator=g, device="cuda").clamp_(1e-7, 1 - 1e-7)
    ids = torch.topk(pop - torch.log(-torch.log(u)), k, dim=1).indices.contiguous()
    if case["drop"]:
        ids[torch.rand((T, k), generator=g, device="cuda") < case["drop"]] = -1
    return ids


def _shape(case):
    """(K, N) of a product."""
    return (case["H"], 2 * case["I"]) if case["side"] == "up" else (case["I"], case["H"])


def prepare(case, seed):
    g = _gen(seed)
    T, E, k, dt = case["T"], case["E"], case["k"], DTYPES[case["dtype"]]
    s = {"case": case, "ids": _picks(g, case)}
    if case["kind"] == "product":
        K, N = _shape(case)
        up = case["side"] == "up"
        s["w"] = _rand(g, dt, E, N, K).mul_(1 / math.sqrt(K))
        if case["pass"] != "inputs":
            s["x"] = _rand(g, dt, T if up else T * k, K)
        if case["pass"] != "forward":                        # the gradient that comes in: per route, or per token where rows are summed
            s["dy"] = _rand(g, dt, T * k if up else T, N)
    else:
        I = case["I"]
        s["gu"] = _rand(g, dt, T * k, 2 * I).mul_(2.0)       # a few values pass the clamp
        s["weights"] = torch.softmax(torch.randn((T, k), generator=g, device="cuda"), 1) if case["weighted"] else None
        s["dh"] = _rand(g, dt, T * k, I) if case["grad"] else None
    if own:
        s["grouped"] = _package()
        if case["kind"] == "gated" or case["pass"] != "forward":
            s["plan"] = s["grouped"].Plan(s["ids"], E)       # the product before made it
    return s


# ------------------------------------------------------------------------------------------------- plain forms

def _sorted(ids, E):
    """(order int64 [n], offsets int64 [E + 1]): the flat routes by expert, then by number, and where each expert's begin; picks of
    none come last."""
    e = ids.reshape(-1)
    e = torch.where((e >= 0) & (e < E), e, E)
    e, order = torch.sort(e, stable=True)
    return order, torch.searchsorted(e, torch.arange(E + 1, device="cuda"))


def _per_token(rows, order, T, k, live):
    """Sum of each token's rows (fp32, rows in the plan's order)."""
    flat = torch.zeros_like(rows)
    flat[order[:live]] = rows[:live]
    return flat.view(T, k, -1).sum(1)


def _plain_product(s):
    c = s["case"]
    T, E, k, w = c["T"], c["E"], c["k"], s["w"]
    K, N = _shape(c)
    up, way = c["side"] == "up", c["pass"]
    order, offsets = _sorted(s["ids"], E)
    n = T * k
    if way == "weights":
        out = torch.zeros((E, N, K), device="cuda")
    else:
        out = torch.zeros((n, N if way == "forward" else K), device="cuda")
    token = order // k
    if way == "forward" and n <= 64:                         # few rows: every route with its own copy of its expert's weights
        live = (s["ids"].reshape(-1)[order] >= 0)[:, None]
        x = s["x"][token] if up else s["x"]
        y = torch.matmul(w[s["ids"].reshape(-1)[order].clamp(min=0)].float(), x.float()[:, :, None])[:, :, 0]
        out = torch.where(live, y, 0.0)
        return (out if up else _per_token(out, order, T, k, n)).to(w.dtype)
    # one product per expert (padding all experts to the longest would multiply the work)
    ends = offsets.tolist()
    for e in range(E):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        if way != "inputs":
            x = (s["x"][token[a:b]] if up else s["x"][a:b]).float()
        if way != "forward":
            dy = (s["dy"][a:b] if up else s["dy"][token[a:b]]).float()
        if way == "forward":
            torch.mm(x, w[e].float().t(), out=out[a:b])
        elif way == "inputs":
            torch.mm(dy, w[e].float(), out=out[a:b])
        else:
            torch.mm(dy.t(), x, out=out[e])
    if way == ("inputs" if up else "forward"):               # one row per token
        out = _per_token(out, order, T, k, ends[E])
    return out.to(w.dtype)


def _plain_saved8(gu):
    """gu as its 8-bit checkpoint holds it: groups of 32 values, whole multiples up to 127 of the smallest power of two that allows it."""
    x = gu.float().unflatten(1, (-1, GROUP))
    m, e = torch.frexp(x.abs().amax(-1, keepdim=True))
    step = ((e + (120 + (m > 127 / 128).int())) << 23).view(torch.float32)      # 2^(e - 7), or twice that
    return (torch.round(x / step) * step).flatten(1)


def _plain_gated(s):
    c = s["case"]
    T, E, k = c["T"], c["E"], c["k"]
    order, offsets = _sorted(s["ids"], E)
    live = (torch.arange(T * k, device="cuda") < offsets[E])[:, None]
    w = torch.ones((T * k, 1), device="cuda") if s["weights"] is None else s["weights"].reshape(-1, 1)[order]
    w = torch.where(live, w, 0.0)

    def parts(gu):
        g, u = gu.float().chunk(2, 1)
        sg = 1.0 / (1.0 + torch.exp(-g))
        return g, u, sg, (g * sg).clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)

    *_, a, u = parts(s["gu"])
    h = (w * a * u).to(s["gu"].dtype)
    if not c["grad"]:
        return h
    kept = _plain_saved8(s["gu"]) if c["save8"] else s["gu"]
    g, u, sg, a, uc = parts(kept)
    dh = s["dh"].float()
    d = w * dh
    dg = torch.where(g * sg <= LIMIT, d * uc * sg * (1.0 + g * (1.0 - sg)), 0.0)
    du = torch.where(u.abs() <= LIMIT, d * a, 0.0)
    out = [h, torch.cat([dg, du], 1).to(h.dtype)]
    if s["weights"] is not None:
        dw = torch.zeros(T * k, device="cuda")
        dw[order] = torch.where(live, dh * a * uc, 0.0).sum(1)
        out.append(dw.view(T, k))
    if c["save8"]:
        out.append((w * a * uc).to(h.dtype))
    return tuple(out)


# ------------------------------------------------------------------------------------------------- one pass

def run(s):
    c = s["case"]
    if not own:
        return _plain_product(s) if c["kind"] == "product" else _plain_gated(s)
    grouped = s["grouped"]
    if c["kind"] == "product":
        rows = {"gather": c["side"] == "up", "reduce": c["side"] == "down"}
        if c["pass"] == "forward":
            return grouped.linear_forward(s["x"], s["w"], grouped.Plan(s["ids"], c["E"]), **rows)
        want_x = c["pass"] == "inputs"
        dx, dw = grouped.linear_backward(s["dy"], s.get("x"), s["w"], s["plan"], need_x=want_x, need_w=not want_x, **rows)
        return dx if want_x else dw
    h, kept = grouped.swiglu_forward(s["gu"], s["plan"], weights=s["weights"], limit=LIMIT, save8=c["save8"])
    if not c["grad"]:
        return h
    dgu, dw, again = grouped.swiglu_backward(s["dh"], kept, s["plan"], weights=s["weights"], limit=LIMIT, need_h=c["save8"])
    return tuple(t for t in (h, dgu, dw, again) if t is not None)


def work(case):
    """Bytes and FLOPs of one pass: inputs read once (weights of the experts that are met), outputs written once."""
    T, E, k = case["T"], case["E"], case["k"]
    n = T * k * (1 - case["drop"])
    if case["kind"] == "product":
        K, N = _shape(case)
        up, way = case["side"] == "up", case["pass"]
        p = [i ** -case["skew"] for i in range(1, E + 1)]
        met = sum(1 - (1 - min(1.0, k * q / sum(p))) ** T for q in p)
        met = min(max(met, min(k, E)), E)
        x, y = (T if up else n) * K, (n if up else T) * N
        return {"bytes": int(2 * (x + y) + 2 * (E if way == "weights" else met) * K * N + 8 * T * k), "flops": int(2 * n * K * N)}
    I, e = case["I"], T * k * case["I"]
    bytes_, flops = 6 * e, 8 * e                             # gu in, h out
    if case["save8"] and case["grad"]:
        bytes_ += 2 * e + 2 * e // GROUP                     # written
    if case["grad"]:
        bytes_ += (2 * e + 2 * e // GROUP + 2 * e if case["save8"] else 4 * e) + 6 * e     # gu again, dh in, dgu out, h again
        flops += 20 * e
    return {"bytes": bytes_ + 12 * T * k, "flops": flops}


# ------------------------------------------------------------------------------------------------- 64-bit results

def exact(case, seed):
    s = prepare(case, seed)
    T, E, k = case["T"], case["E"], case["k"]
    flat = s["ids"].reshape(-1)
    # the plan's order from the definition: by expert, then by route; none last
    key = torch.where((flat >= 0) & (flat < E), flat, E) * (T * k) + torch.arange(T * k, device="cuda")
    order = torch.argsort(key)
    if case["kind"] == "product":
        K, N = _shape(case)
        up, way = case["side"] == "up", case["pass"]
        shape = {"forward": (T * k if up else T, N), "inputs": (T if up else T * k, K), "weights": (E, N, K)}[way]
        out = torch.zeros(shape, dtype=torch.float64, device="cuda")
        place = torch.empty_like(order)
        place[order] = torch.arange(T * k, device="cuda")
        for e in range(E):
            routes = (flat == e).nonzero()[:, 0]
            if not routes.numel():
                continue
            rows, tokens = place[routes], torch.div(routes, k, rounding_mode="floor")
            x_at, y_at = (tokens, rows) if up else (rows, tokens)
            if way == "forward":
                out.index_add_(0, y_at, s["x"][x_at].double() @ s["w"][e].double().t().contiguous())
            elif way == "inputs":
                out.index_add_(0, x_at, s["dy"][y_at].double() @ s["w"][e].double())
            else:
                out[e] = s["dy"][y_at].double().t().contiguous() @ s["x"][x_at].double()
        return out
    I = case["I"]
    live = (flat[order] >= 0).double()[:, None]
    w = live if s["weights"] is None else live * s["weights"].double().reshape(-1, 1)[order]

    def act(t):
        g, u = t[:, :I], t[:, I:]
        return torch.minimum(g * torch.sigmoid(g), torch.tensor(LIMIT, dtype=t.dtype, device="cuda")), torch.clamp(u, -LIMIT, LIMIT)

    a, u = act(s["gu"].double())
    h = w * a * u
    if not case["grad"]:
        return h
    gu = s["gu"].double()
    if case["save8"]:
        x = gu.reshape(T * k, -1, GROUP)
        top = x.abs().amax(-1, keepdim=True)
        step = torch.exp2(torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -126) / 127)))
        step = torch.where(top > 127 * step, 2 * step, step)              # a logarithm next to a whole number
        step = torch.where(top <= 127 * step / 2, step / 2, step)
        gu = (torch.round(x / step) * step).reshape(T * k, -1)
    a, uc = act(gu)
    g, u = gu[:, :I], gu[:, I:]
    sg, d = torch.sigmoid(g), w * s["dh"].double()
    dg = d * uc * (sg + g * sg * (1 - sg)) * (g * sg <= LIMIT)
    du = d * a * (u.abs() <= LIMIT)
    out = [h, torch.cat([dg, du], 1)]
    if s["weights"] is not None:
        dw = torch.zeros(T * k, dtype=torch.float64, device="cuda")
        dw[order] = (live * s["dh"].double() * a * uc).sum(1)
        out.append(dw.view(T, k))
    if case["save8"]:
        out.append(w * a * uc)
    return tuple(out)
