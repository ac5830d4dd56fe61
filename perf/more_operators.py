"""What is timed of the operators of block-scaled fp8 checkpoints: a linear layer whose weight has one scale per 128 × 128
block, the router of a mixture of experts, and the experts of such a layer on the tokens that the router sends them.

Every case is one of five kinds:

  linear   rows of activations through one fp8 weight: quantized on the way, multiplied
  codes    the same in two calls: codes and scales that several weights of a layer can share, then the product
  route    scores of every expert to the top_k experts of each token and their weights
  experts  tokens with their experts and weights to the weighted sum of the experts' gated MLPs
  layer    router logits and tokens: routed, then through the experts, nothing of it on the host

Activations are e4m3 codes with one f32 scale per row and 128 values: s = max(amax / 448, 1e-12) and codes that are x / s,
an f32 number like s, rounded to nearest even (ties are common: a few bits of x over a few bits of amax). Products of a
block of 128 are scaled by its two scales and summed in f32. An expert's silu(gate) · up rows are quantized the same way in
front of its down product.
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 128
TOP = 448.0  # the largest e4m3 value
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one generated token through the q|k|v projection of a 30B-A3B layer: latency
        dict(name="linear_token", kind="linear", m=1, n=5120, k=2048, x="bf16", c="bf16"),
        # a decode step of 48 sequences through its output projection
        dict(name="linear_batch", kind="linear", m=48, n=2048, k=4096, x="f16", c="f16"),
        # the widest matrix of a vision layer of 2394 patches: rows and columns that fill no tile
        dict(name="linear_vision", kind="linear", m=2394, n=4304, k=1152, x="f16", c="f16"),
        # prompts of 16000 tokens through a square projection of 4096
        dict(name="linear_prompts", kind="linear", m=16000, n=4096, k=4096, x="bf16", c="bf16"),
        # a padded batch of passages, K that ends inside a block, f32 both sides
        dict(name="codes_odd", kind="codes", m=333, n=1000, k=1104, x="f32", c="f32"),
        # 3633 tokens of passages through the narrow side of an embedding model's MLP
        dict(name="codes_passages", kind="codes", m=3633, n=1024, k=2560, x="f16", c="f16"),
        # the router of a decode step: softmax over 128 experts
        dict(name="route_step", kind="route", m=8, e=128, top=8, score="softmax", groups=1, top_groups=1, bias=False, norm=True, scale=1.0, x="f32"),
        # the router of long prompts: sigmoid scores with a bias for balance, 4 of 8 groups of 32 experts
        dict(name="route_prompts", kind="route", m=16384, e=256, top=8, score="sigmoid", groups=8, top_groups=4, bias=True, norm=True, scale=2.5, x="f32"),
        # one sequence that generates, its 8 experts of a 30B-A3B layer: the weights' bytes
        dict(name="experts_token", kind="experts", m=1, e=128, top=8, h=2048, i=768, x="bf16"),
        # a step of a busy server: most experts have a few rows
        dict(name="experts_batch", kind="experts", m=64, e=128, top=8, h=2048, i=768, x="f16"),
        # a prompt of 1024 tokens, router and experts
        dict(name="layer_prompt", kind="layer", m=1024, e=128, top=8, h=2048, i=768, x="bf16", score="softmax", groups=1, top_groups=1, bias=False, norm=True, scale=1.0),
        # prompts of 8192 tokens with grouped sigmoid routing
        dict(name="layer_prompts", kind="layer", m=8192, e=64, top=6, h=2048, i=1408, x="bf16", score="sigmoid", groups=8, top_groups=4, bias=True, norm=True, scale=2.5),
    ]


def _log(rng, lo, hi):
    """Whole numbers of [lo, hi], even over their logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# the most that a listed case asks for: operations, bytes, and bytes of an expert stack
FLOPS, BYTES, STACK = 8.5e11, 8.0e8, 6.1e8


def _draw_router(rng, c):
    c["score"] = rng.choice(["softmax", "sigmoid"])
    c["groups"] = rng.choice([1, 1, 4, 8]) if c["e"] % 8 == 0 else 1
    c["top_groups"] = rng.randint(1, c["groups"])
    c["top"] = min(c["top"], c["e"] // c["groups"] * c["top_groups"])
    c.update(bias=rng.random() < 0.5, norm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]))


def draw(rng):
    while True:
        kind = rng.choice(["linear", "codes", "route", "experts", "layer"])
        c = dict(kind=kind)
        if kind in ("linear", "codes"):
            c.update(m=_log(rng, 1, 16000), n=_log(rng, 96, 8192), k=16 * _log(rng, 8, 512), x=rng.choice(["f16", "bf16", "bf16", "f32"]))
            c["c"] = rng.choice([c["x"], "f16", "bf16"])
        elif kind == "route":
            c.update(m=_log(rng, 1, 16384), e=rng.choice([8, 60, 64, 128, 160, 256, 384]), x=rng.choice(["f32", "f32", "f16", "bf16"]))
            c["top"] = rng.randint(1, 8)
            _draw_router(rng, c)
        else:
            c.update(m=_log(rng, 1, 8192), e=rng.choice([8, 16, 60, 64, 128]), h=16 * _log(rng, 32, 256), i=16 * _log(rng, 8, 96), x=rng.choice(["f16", "bf16"]))
            c["top"] = rng.randint(1, 8)
            if kind == "layer":
                _draw_router(rng, c)
        w = work(c)
        if w["flops"] <= FLOPS and w["bytes"] <= BYTES and c.get("e", 0) * 3 * c.get("h", 0) * c.get("i", 0) <= STACK:
            return c


def _blocks(n):
    return -(-n // BLOCK)


SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def work(case):
    c = case
    m, xb = c["m"], SIZES[c["x"]]
    route = {"bytes": m * c["e"] * xb + m * c["top"] * 8, "flops": 8 * m * c["e"]} if c["kind"] in ("route", "layer") else {"bytes": 0, "flops": 0}
    if c["kind"] == "route":
        return route
    if c["kind"] in ("linear", "codes"):
        n, k = c["n"], c["k"]
        codes = m * k + 4 * m * _blocks(k) if c["kind"] == "codes" else 0  # handed to the caller
        return {"bytes": m * k * xb + n * k + 4 * _blocks(n) * _blocks(k) + m * n * SIZES[c["c"]] + codes, "flops": 2 * m * n * k}
    h, i = c["h"], c["i"]
    seen = c["e"] * (1 - (1 - c["top"] / c["e"]) ** m)  # experts that some token goes to, as expected
    return {"bytes": route["bytes"] + int(seen * 3 * h * i) + 2 * m * h * xb + m * c["top"] * 8, "flops": route["flops"] + 6 * m * c["top"] * h * i}


# ------------------------------------------------------------------ inputs ----
def _weight(g, *shape, std=0.02):
    """e4m3 codes of normally distributed weights and their scales: a block's largest of 16384 values, near four
    standard deviations, is near the top of the type."""
    codes = (torch.randn(*shape, generator=g, device="cuda") * 105.0).clamp_(-TOP, TOP).to(torch.float8_e4m3fn)
    rows, cols = _blocks(shape[-2]), _blocks(shape[-1])
    return codes, std / 105.0 * (0.8 + 0.4 * torch.rand(*shape[:-2], rows, cols, generator=g, device="cuda"))


def _inputs(c, seed):
    """The case's tensors, the same for prepare() and exact()."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, m, t = DTYPES[c["x"]], c["m"], {}
    if c["kind"] in ("linear", "codes"):
        t["w"], t["ws"] = _weight(g, c["n"], c["k"])
        t["x"] = _activations(g, m, c["k"]).to(dt)
        return t
    if c["kind"] != "route":
        e, h, i = c["e"], c["h"], c["i"]
        t["x"] = _activations(g, m, h).to(dt)
        t["gate"], t["gate_s"] = _weight(g, e, i, h)
        t["up"], t["up_s"] = _weight(g, e, i, h)
        t["down"], t["down_s"] = _weight(g, e, h, i)
    logits = torch.randn(m, c["e"], generator=g, device="cuda") * 1.5
    if c["kind"] == "experts":
        top = torch.topk(logits, c["top"], dim=1)
        t["ids"] = top.indices.to(torch.int32).contiguous()
        t["wts"] = torch.softmax(top.values, 1).contiguous()
        return t
    t["logits"] = logits.to(torch.float32 if c["kind"] == "layer" else dt)
    t["bias"] = 0.1 * torch.randn(c["e"], generator=g, device="cuda") if c["bias"] else None
    return t


def _activations(g, m, k):
    """Rows behind a norm: a few channels are much larger than the others."""
    x = torch.randn(m, k, generator=g, device="cuda")
    return x * (1.0 + 12.0 * (torch.rand(k, generator=g, device="cuda") < 0.01))


def prepare(case, seed):
    c, t = case, _inputs(case, seed)
    s = dict(c=c, t=t)
    m = c["m"]
    if c["kind"] in ("linear", "codes"):
        s["out"] = torch.empty(m, c["n"], dtype=DTYPES[c["c"]], device="cuda")
        if c["kind"] == "codes":
            s["q"] = torch.empty(m, c["k"], dtype=torch.float8_e4m3fn, device="cuda")
            s["scale"] = torch.empty(m, _blocks(c["k"]), dtype=torch.float32, device="cuda")
    else:
        if c["kind"] != "experts":
            s["ids"] = torch.empty(m, c["top"], dtype=torch.int32, device="cuda")
            s["wts"] = torch.empty(m, c["top"], dtype=torch.float32, device="cuda")
        if c["kind"] != "route":
            s["y"] = torch.empty(m, c["h"], dtype=DTYPES[c["x"]], device="cuda")
    if own:
        rk = s["rk"] = _rk()
        rk.init(0)
        host = lambda name: t[name].view(torch.uint8).cpu().numpy() if t[name].element_size() == 1 else t[name].cpu().numpy()  # noqa: E731
        if c["kind"] in ("linear", "codes"):
            s["id"] = rk.pack_fp8(host("w"), host("ws"))
        elif c["kind"] != "route":
            s["id"] = rk.pack_moe_fp8(*(host(p + q) for p in ("gate", "up", "down") for q in ("", "_s")))
            s["plan"] = rk.routed_plan(s["id"], m, c["top"])
        torch.cuda.synchronize()  # the inputs come from torch's stream, the calls run on the library's
    return s


def _rk():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "burn-rocket_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import burn_rocket
    return burn_rocket


# --------------------------------------------------------------------- run ----
def run(state):
    s, kind = state, state["c"]["kind"]
    if own:
        _own(s)
    else:
        _plain(s)
    if kind == "linear":
        return s["out"]
    if kind == "codes":
        return {"q": s["q"], "scale": s["scale"], "out": s["out"]}
    if kind == "route":
        return {"ids": s["ids"], "wts": s["wts"]}
    if kind == "experts":
        return s["y"]
    return {"ids": s["ids"], "wts": s["wts"], "y": s["y"]}


def _own(s):
    c, t, rk = s["c"], s["t"], s["rk"]
    lib, m = rk.lib(), c["m"]
    types, p = {"f32": rk.DTYPE_F32, "f16": rk.DTYPE_F16, "bf16": rk.DTYPE_BF16}, torch.Tensor.data_ptr
    rcs = []
    if c["kind"] == "linear":
        rcs.append(lib.rk_matmul_fp8_dev(s["id"], p(t["x"]), types[c["x"]], m, c["k"], p(s["out"]), types[c["c"]], None))
    elif c["kind"] == "codes":
        rcs.append(lib.rk_quantize_fp8_dev(p(t["x"]), types[c["x"]], m, c["k"], p(s["q"]), p(s["scale"]), None))
        rcs.append(lib.rk_matmul_fp8_codes_dev(s["id"], p(s["q"]), p(s["scale"]), m, c["k"], p(s["out"]), types[c["c"]], None))
    else:
        ids, wts = (t["ids"], t["wts"]) if c["kind"] == "experts" else (s["ids"], s["wts"])
        if c["kind"] != "experts":
            score = {"softmax": rk.ROUTE_SOFTMAX, "sigmoid": rk.ROUTE_SIGMOID}[c["score"]]
            bias = p(t["bias"]) if c["bias"] else None
            dt = types[c["x"]] if c["kind"] == "route" else rk.DTYPE_F32
            rcs.append(lib.rk_moe_route_dev(p(t["logits"]), dt, m, c["e"], c["top"], score, bias, c["groups"], c["top_groups"], int(c["norm"]),
                                            c["scale"], p(ids), p(wts), None))
        if c["kind"] != "route":
            rcs.append(lib.rk_moe_plan_route_dev(s["plan"].ptr, m, p(ids), p(wts), None))
            rcs.append(lib.rk_moe_experts_fp8_dev(s["id"], s["plan"].ptr, p(t["x"]), p(s["y"]), types[c["x"]], 0, None))
    if any(rcs):
        raise RuntimeError(lib.rk_last_error().decode())


def _quantize(x):
    """Codes, as values, and scales of rows: [m, k] and [m, blocks of k]."""
    m, k = x.shape
    b = torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k)).view(m, -1, BLOCK)
    scale = (b.abs().amax(-1).double() / TOP).float().clamp(min=1e-12)  # (a quotient of 32-bit tensors may be a step off)
    q = (b.double() / scale[..., None].double()).float().to(torch.float8_e4m3fn)
    return q.view(m, -1)[:, :k], scale


def _spread(scale, rows, cols):
    """A scale per block to one per value."""
    return scale.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]


def _values(q, scale):
    """Quantized rows as the f32 values they stand for."""
    return q.float() * scale.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _plain(s):
    c, t = s["c"], s["t"]
    if c["kind"] in ("linear", "codes"):
        q, scale = _quantize(t["x"].float())
        if c["kind"] == "codes":
            s["q"].copy_(q)
            s["scale"].copy_(scale)
        w = t["w"].float() * _spread(t["ws"], c["n"], c["k"])
        s["out"].copy_(_values(q, scale) @ w.t())
        return
    ids, wts = (t["ids"], t["wts"]) if c["kind"] == "experts" else (s["ids"], s["wts"])
    if c["kind"] != "experts":
        _plain_route(c, t["logits"], t["bias"], ids, wts)
    if c["kind"] != "route":
        _plain_experts(c, t, ids.long(), wts, s["y"])


def _plain_route(c, logits, bias, ids, wts):
    """In 64 bits: which of two experts with all but equal scores is taken decides what the token computes. Without a
    bias the order of the scores is that of the logits."""
    m, e = logits.shape
    x = logits.double()
    if c["score"] == "softmax":
        p = (x - x.amax(1, keepdim=True)).exp()
        p = p / p.sum(1, keepdim=True)
    else:
        p = 1 / (1 + (-x).exp())
    by = x if bias is None else p + bias.double()
    if c["groups"] > 1:
        per = by.view(m, c["groups"], -1)
        best = per.amax(2) if bias is None else per.sort(dim=2, descending=True).values[..., :2].sum(2)
        at = best.sort(dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        open_ = torch.zeros(m, c["groups"], dtype=torch.bool, device=x.device).scatter_(1, at, True)
        by = per.masked_fill(~open_[..., None], -math.inf).view(m, e)
    at = by.sort(dim=1, descending=True, stable=True).indices[:, :c["top"]]
    w = p.gather(1, at)
    if c["norm"]:
        w = w / w.sum(1, keepdim=True)
    ids.copy_(at)
    wts.copy_(w * c["scale"])


def _plain_experts(c, t, ids, wts, y):
    """Every expert's rows padded to the longest list, batched products, the rows back to their tokens."""
    e, h, i, k = c["e"], c["h"], c["i"], c["top"]
    flat = ids.reshape(-1)
    order = flat.sort(stable=True).indices
    expert, count = flat[order], flat.bincount(minlength=e)
    at = torch.arange(flat.numel(), device=flat.device) - (count.cumsum(0) - count)[expert]
    rows = torch.zeros(e, int(count.max()), h, device=flat.device)
    rows[expert, at] = _values(*_quantize(t["x"].float()))[order // k]

    def product(a, name, n, kk):
        w = t[name].float() * _spread(t[name + "_s"], n, kk)
        return torch.matmul(a, w.transpose(1, 2).contiguous())

    g, u = product(rows, "gate", i, h), product(rows, "up", i, h)
    act = _values(*_quantize((g / (1 + (-g).exp()) * u).view(-1, i))).view(e, -1, i)
    back = torch.empty(flat.numel(), h, device=flat.device)
    back[order] = product(act, "down", h, i)[expert, at]
    y.copy_((back.view(-1, k, h) * wts[..., None]).sum(1))


# ------------------------------------------------------------------- exact ----
def _e4m3(v):
    """The nearest e4m3 values of 64-bit ones within its range, ties to even: three bits behind the leading one, whose
    place is at least 2^-6."""
    place = torch.frexp(v).exponent.clamp(min=-5).double() - 4
    return torch.round(v / 2.0 ** place) * 2.0 ** place


def _exact_rows(x):
    """(codes as values, scales, values) of rows in 64 bits. Scale and quotient are f32 numbers by their definition."""
    m, k = x.shape
    q, scales = torch.zeros_like(x), []
    for b in range(0, k, BLOCK):
        part = x[:, b:b + BLOCK]
        scale = (part.abs().max(1, keepdim=True).values / TOP).float().double().clamp(min=float(torch.tensor(1e-12)))
        q[:, b:b + BLOCK] = _e4m3((part / scale).float().double())
        scales.append(scale)
    scales = torch.cat(scales, 1)
    return q, scales, q * torch.cat([scales[:, b:b + 1].expand(m, min(BLOCK, k - b * BLOCK)) for b in range(scales.shape[1])], 1)


def _exact_weight(codes, scales):
    w = codes.double()
    for a in range(scales.shape[0]):
        for b in range(scales.shape[1]):
            w[a * BLOCK:(a + 1) * BLOCK, b * BLOCK:(b + 1) * BLOCK] *= scales[a, b].double()
    return w


def _exact_route(c, logits, bias):
    """One choice at a time, the largest that is left."""
    x = logits.double()
    p = torch.softmax(x, 1) if c["score"] == "softmax" else torch.sigmoid(x)
    by = x.clone() if bias is None else p + bias.double()
    m, size = x.shape[0], x.shape[1] // c["groups"]
    if c["groups"] > 1:
        score = torch.stack([torch.topk(by[:, a * size:(a + 1) * size], min(size, 1 if bias is None else 2), 1).values.sum(1) for a in range(c["groups"])], 1)
        keep = torch.zeros_like(by, dtype=torch.bool)
        for _ in range(c["top_groups"]):
            best = score.argmax(1)
            score[torch.arange(m), best] = -math.inf
            keep |= (torch.arange(x.shape[1], device=x.device)[None] // size) == best[:, None]
        by[~keep] = -math.inf
    ids = []
    for _ in range(c["top"]):
        best = by.argmax(1)
        by[torch.arange(m), best] = -math.inf
        ids.append(best)
    ids = torch.stack(ids, 1)
    w = torch.gather(p, 1, ids)
    return ids, (w / w.sum(1, keepdim=True) if c["norm"] else w) * c["scale"]


def exact(case, seed):
    """The definitions in 64 bits, an expert at a time."""
    c, t = case, _inputs(case, seed)
    if c["kind"] in ("linear", "codes"):
        q, scale, x = _exact_rows(t["x"].double())
        out = x @ _exact_weight(t["w"], t["ws"]).T
        return out if c["kind"] == "linear" else {"q": q, "scale": scale, "out": out}
    if c["kind"] == "experts":
        ids, wts = t["ids"].long(), t["wts"].double()
    else:
        ids, wts = _exact_route(c, t["logits"], t["bias"])
        if c["kind"] == "route":
            return {"ids": None, "wts": wts}
    x = _exact_rows(t["x"].double())[2]
    y = torch.zeros_like(x)
    for e in range(c["e"]):
        tok, slot = torch.nonzero(ids == e, as_tuple=True)
        if tok.numel() == 0:
            continue
        gate, up, down = (_exact_weight(t[n][e], t[n + "_s"][e]) for n in ("gate", "up", "down"))
        a = x[tok] @ gate.T
        a = _exact_rows(a * torch.sigmoid(a) * (x[tok] @ up.T))[2]
        y.index_add_(0, tok, wts[tok, slot][:, None] * (a @ down.T))
    return y if c["kind"] == "experts" else {"ids": None, "wts": wts, "y": y}
