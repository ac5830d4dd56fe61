"""What is timed of the operators on batches of sequences: a paged KV cache that is appended to, attention over it, and
attention over packed sequences.

Every case is one of three kinds:

  packed   attention over whole sequences of different lengths that lie one behind the other (an embedding server's batch,
           prompts that need no cache)
  append   the new tokens' q|k|v rows: RMSNorm and rotate-half RoPE of q and k, K and V into the pages of their sequences
  paged    attention of the new tokens (one a sequence, a chunk, or both kinds in one step) over the paged cache

A case names its lengths by a range and a number that they are drawn from, so that `work` knows them. Page tables are
shuffled, as an allocator that has run for a while leaves them.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

EPS = 1e-6
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # search queries that arrived together, through a 0.6B embedding model's attention: launches and latency
        dict(name="packed_queries", kind="packed", n=24, lens=1, q_lo=4, q_hi=40, h=16, kv=8, d=128, mode="causal", window=-1, dtype="f16"),
        # a batch of passages to be embedded
        dict(name="packed_passages", kind="packed", n=64, lens=2, q_lo=100, q_hi=512, h=16, kv=8, d=128, mode="causal", window=-1, dtype="f16"),
        # texts through the sliding-window layer of a text encoder with one kv head of 256
        dict(name="packed_window", kind="packed", n=6, lens=3, q_lo=300, q_hi=2587, h=3, kv=1, d=256, mode="window", window=512, dtype="bf16"),
        # two long prompts through a layer of 32 heads
        dict(name="packed_documents", kind="packed", n=2, lens=4, q_lo=6000, q_hi=8191, h=32, kv=4, d=128, mode="causal", window=-1, dtype="bf16"),
        # one step of sequences that generate: 48 rows
        dict(name="append_decode", kind="append", n=48, lens=5, q_lo=1, q_hi=1, kv_lo=20, kv_hi=1200, page=16, h=16, kv=8, d=128, norm=True, tables="f16", dtype="f16"),
        # chunks of prompts, heads of 64 without norms
        dict(name="append_chunks", kind="append", n=9, lens=6, q_lo=5, q_hi=300, kv_lo=300, kv_hi=2000, page=32, h=16, kv=4, d=64, norm=False, tables="f32", dtype="f16"),
        # prompts of a large layer
        dict(name="append_prompts", kind="append", n=6, lens=7, q_lo=900, q_hi=2400, kv_lo=2400, kv_hi=4000, page=64, h=32, kv=4, d=128, norm=True, tables="f32", dtype="bf16"),
        # one generated token against the keys so far
        dict(name="decode_one", kind="paged", n=1, lens=8, q_lo=1, q_hi=1, kv_lo=4097, kv_hi=4097, page=16, h=32, kv=4, d=128, mode="causal", window=-1, dtype="f16"),
        # one step of a busy server
        dict(name="decode_batch", kind="paged", n=64, lens=9, q_lo=1, q_hi=1, kv_lo=100, kv_hi=8000, page=16, h=16, kv=8, d=128, mode="causal", window=-1, dtype="f16"),
        # a few sequences far into long contexts
        dict(name="decode_far", kind="paged", n=3, lens=10, q_lo=1, q_hi=1, kv_lo=60000, kv_hi=131072, page=64, h=32, kv=4, d=128, mode="causal", window=-1, dtype="bf16"),
        # a chunk of a long prompt against what is cached of it
        dict(name="chunk_extend", kind="paged", n=1, lens=11, q_lo=512, q_hi=512, kv_lo=16901, kv_hi=16901, page=64, h=32, kv=4, d=128, mode="causal", window=-1, dtype="f16"),
        # a step that carries prompt chunks and generating sequences, a sliding-window layer
        dict(name="mixed_step", kind="paged", n=32, lens=12, q_lo=1, q_hi=700, kv_lo=700, kv_hi=6000, page=32, h=16, kv=4, d=64, mode="causal_window", window=1024, dtype="f16", chunks=3),
    ]


def _log(rng, lo, hi):
    """Whole numbers of [lo, hi], even over their logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lengths(c):
    """(new tokens, keys with them) of each sequence. `chunks`: the first so many take the range, the others one token."""
    rng = random.Random(c["lens"])
    q = [rng.randint(c["q_lo"], c["q_hi"]) for _ in range(c["n"])]
    if c.get("chunks"):
        q = [x if i < c["chunks"] else 1 for i, x in enumerate(q)]
    if c["kind"] == "packed":
        return q, list(q)
    return q, [max(x, rng.randint(c["kv_lo"], c["kv_hi"])) for x in q]


# the most score elements that a plain form lays out, and the most operations and bytes that a listed case asks for
SCORES, FLOPS, BYTES = 4.3e9, 1.0e12, 6.0e8


def draw(rng):
    while True:
        kind = rng.choice(["packed", "append", "paged"])
        h, kv, d = rng.choice([(16, 8, 128), (32, 4, 128), (16, 4, 64), (3, 1, 256), (12, 12, 64), (8, 8, 96), (14, 2, 80)])
        c = dict(kind=kind, n=_log(rng, 1, 64), lens=rng.randrange(1 << 30), h=h, kv=kv, d=d, dtype=rng.choice(["f16", "bf16"]))
        if kind == "packed":
            c["q_hi"] = _log(rng, 3, 8191)
            c["q_lo"] = max(1, int(c["q_hi"] * rng.uniform(0.05, 1.0)))
        else:
            c["kv_hi"] = _log(rng, 5, 131072 if kind == "paged" else 4000)
            c["kv_lo"] = max(1, int(c["kv_hi"] * rng.uniform(0.02, 1.0)))
            c["q_hi"] = rng.choice([1, _log(rng, 1, min(c["kv_lo"], 1024 if kind == "paged" else 2400))])
            c["q_lo"] = max(1, int(c["q_hi"] * rng.uniform(0.1, 1.0)))
            c["page"] = rng.choice([16, 32, 64, 128, 256])
        if kind == "append":
            c.update(norm=rng.random() < 0.6, tables=rng.choice(["f32", c["dtype"]]))
        else:
            c["mode"] = rng.choice(["causal", "causal", "causal", "none", "window", "causal_window"])
            c["window"] = rng.choice([100, 512, 1024]) if "window" in c["mode"] else -1
        if kind == "paged" and rng.random() < 0.3:
            c["chunks"] = rng.randint(1, 3)
        w = work(c)
        q, k = _lengths(c)
        if w["flops"] <= FLOPS and w["bytes"] <= BYTES and (kind == "append" or c["n"] * h * max(q) * max(k) <= SCORES):
            return c


def _pairs(q, k, mode, window):
    """(visible (query, key) pairs, keys that some query sees) of one sequence."""
    t = np.arange(k - q, k, dtype=np.int64)
    lo, hi = _interval(t, mode, window)
    lo, hi = np.maximum(lo, 0), np.minimum(hi, k - 1)
    return int(np.maximum(hi - lo + 1, 0).sum()), int(hi.max() - lo.min() + 1)


def _interval(t, mode, window):
    """The first and the last key that the query at position t sees."""
    far = 1 << 40
    if mode == "causal":
        return t - far, t
    if mode == "window":
        return t - window, t + window
    if mode == "causal_window":
        return t - window + 1, t
    return t - far, t + far


def work(case):
    c = case
    q, k = _lengths(c)
    t, h, kv, d = sum(q), c["h"], c["kv"], c["d"]
    if c["kind"] == "append":
        tab = t * d * (4 if c["tables"] == "f32" else 2)
        return {"bytes": 2 * t * (h + 2 * kv) * d * 2 + tab, "flops": t * (h + kv) * d * (8 if c["norm"] else 4)}
    pairs = [_pairs(a, b, c["mode"], c["window"]) for a, b in zip(q, k)]
    return {"bytes": 2 * t * h * d * 2 + 2 * sum(p[1] for p in pairs) * kv * d * 2, "flops": 4 * d * h * sum(p[0] for p in pairs)}


# ------------------------------------------------------------------ inputs ----
def _inputs(c, seed):
    """The case's tensors, the same for prepare() and exact()."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[c["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    q, k = _lengths(c)
    h, kv, d, n, toks = c["h"], c["kv"], c["d"], c["n"], sum(q)
    t = dict(q_lens=np.array(q, np.int32), kv_lens=np.array(k, np.int32))
    if c["kind"] == "packed":
        t["q"], t["k"], t["v"] = randn(toks, h * d), randn(toks, kv * d), randn(toks, kv * d)
        return t
    need = [-(-x // c["page"]) for x in k]
    n_pages = sum(need) + 3
    ids = np.random.default_rng(int(seed)).permutation(n_pages).astype(np.int32)
    table, at = np.full((n, max(need)), -1, np.int32), 0
    for i, m in enumerate(need):
        table[i, :m] = ids[at:at + m]
        at += m
    t.update(table=table, n_pages=n_pages)
    shape = (n_pages, kv, c["page"], d)
    t["k_cache"], t["v_cache"] = randn(*shape), randn(*shape)
    if c["kind"] == "paged":
        t["q"] = randn(toks, h * d)
        return t
    t["qkv"] = randn(toks, (h + 2 * kv) * d, std=1.5)
    if c["norm"]:
        t["qw"], t["kw"] = (1 + 0.1 * torch.randn(2, d, generator=g, device="cuda")).to(dt)
    ang = torch.arange(max(k), device="cuda", dtype=torch.float64)[:, None] * (
        1e6 ** (-torch.arange(d // 2, device="cuda", dtype=torch.float64) / (d // 2)))[None, :]
    tab = torch.float32 if c["tables"] == "f32" else dt
    t["cos"], t["sin"] = ang.cos().to(tab).contiguous(), ang.sin().to(tab).contiguous()
    return t


def prepare(case, seed):
    c, t = case, _inputs(case, seed)
    s = dict(c=c, t=t)
    toks = int(t["q_lens"].sum())
    name = "q_out" if c["kind"] == "append" else "out"
    s[name] = torch.zeros(toks, c["h"] * c["d"], dtype=DTYPES[c["dtype"]], device="cuda")
    # the batch on the device, as a program that schedules sequences holds it
    ql, kl = (torch.from_numpy(t[x].astype(np.int64)).cuda() for x in ("q_lens", "kv_lens"))
    s["seq"] = torch.repeat_interleave(torch.arange(c["n"], device="cuda"), ql)
    s["first"] = torch.cumsum(ql, 0) - ql
    s["at"] = torch.arange(toks, device="cuda") - s["first"][s["seq"]]  # a token's place among its sequence's new ones
    s["pos"] = s["at"] + (kl - ql)[s["seq"]]
    s["ql"], s["kl"] = ql, kl
    if "table" in t:
        s["table"] = torch.from_numpy(t["table"].astype(np.int64)).cuda()
    if own:
        rk = s["rk"] = _rk()
        rk.init(0)
        modes = {"none": rk.MASK_NONE, "causal": rk.MASK_CAUSAL, "window": rk.MASK_WINDOW, "causal_window": rk.MASK_CAUSAL_WINDOW}
        heads = (c["h"], c["kv"], c["d"], modes[c.get("mode", "causal")], c.get("window", -1))
        if c["kind"] == "packed":
            s["plan"] = rk.packed_plan(t["q_lens"], *heads)
        else:
            s["plan"] = rk.paged_plan(t["q_lens"], t["kv_lens"], t["table"], t["n_pages"], c["page"], *heads)
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
    kind = state["c"]["kind"]
    if own:
        _own(state)
    elif kind == "append":
        _plain_append(state)
    else:
        _plain_attention(state)
    if kind == "append":
        return {"q": state["q_out"], "k_cache": state["t"]["k_cache"], "v_cache": state["t"]["v_cache"]}
    return state["out"]


def _own(s):
    c, t, rk = s["c"], s["t"], s["rk"]
    lib, h, kv, d = rk.lib(), c["h"], c["kv"], c["d"]
    types = {"f32": rk.DTYPE_F32, "f16": rk.DTYPE_F16, "bf16": rk.DTYPE_BF16}
    dt, plan, p = types[c["dtype"]], s["plan"].ptr, torch.Tensor.data_ptr
    if c["kind"] == "packed":
        rc = lib.rk_attention_packed_dev(plan, p(t["q"]), h * d, p(t["k"]), kv * d, p(t["v"]), kv * d, d ** -0.5, 0.0, p(s["out"]), h * d, dt, None)
    elif c["kind"] == "paged":
        rc = lib.rk_attention_paged_dev(plan, p(t["q"]), h * d, p(t["k_cache"]), p(t["v_cache"]), d ** -0.5, 0.0, p(s["out"]), h * d, dt, None)
    else:
        qw, kw = (p(t["qw"]), p(t["kw"])) if c["norm"] else (None, None)
        rc = lib.rk_paged_append_dev(plan, p(t["qkv"]), (h + 2 * kv) * d, qw, kw, EPS, p(t["cos"]), p(t["sin"]), types[c["tables"]],
                                     t["cos"].shape[0], p(s["q_out"]), h * d, p(t["k_cache"]), p(t["v_cache"]), dt, None)
    if rc != 0:
        raise RuntimeError(lib.rk_last_error().decode())


def _plain_append(s):
    c, t = s["c"], s["t"]
    h, kv, d = c["h"], c["kv"], c["d"]
    x = t["qkv"].view(-1, h + 2 * kv, d).float()
    qk, v = x[:, :h + kv], x[:, h + kv:]
    if c["norm"]:
        w = torch.cat([t["qw"].float().expand(h, d), t["kw"].float().expand(kv, d)])
        qk = qk * (qk.square().mean(-1, keepdim=True) + EPS).rsqrt() * w
    cos, sin = t["cos"].float()[s["pos"]][:, None], t["sin"].float()[s["pos"]][:, None]
    a, b = qk[..., :d // 2], qk[..., d // 2:]
    qk = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(t["qkv"].dtype)
    s["q_out"].copy_(qk[:, :h].reshape(-1, h * d))
    page = s["table"][s["seq"], s["pos"] // c["page"]]
    t["k_cache"][page, :, s["pos"] % c["page"]] = qk[:, h:]
    t["v_cache"][page, :, s["pos"] % c["page"]] = v.to(t["qkv"].dtype)


def _plain_attention(s):
    """Every sequence padded to the longest: scores of all of them, masked, exponentials over their sum, times V."""
    c, t = s["c"], s["t"]
    n, h, kv, d = c["n"], c["h"], c["kv"], c["d"]
    lq, lk = int(t["q_lens"].max()), int(t["kv_lens"].max())
    i, j = torch.arange(lq, device="cuda"), torch.arange(lk, device="cuda")
    if c["kind"] == "packed":
        rows = (s["first"][:, None] + j).clamp_(max=t["k"].shape[0] - 1)
        k, v = (x[rows].view(n, lk, kv, d).transpose(1, 2).float() for x in (t["k"], t["v"]))
    else:
        page = s["table"].clamp(min=0)[:, j // c["page"]]
        k, v = (x[page, :, j % c["page"]].transpose(1, 2).float() for x in (t["k_cache"], t["v_cache"]))
    q = t["q"][(s["first"][:, None] + i).clamp_(max=t["q"].shape[0] - 1)].float()
    q = q.view(n, lq, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, h // kv * lq, d)
    p = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(d ** -0.5).view(n, kv, h // kv, lq, lk)
    lo, hi = _interval((s["kl"] - s["ql"])[:, None] + i, c["mode"], c["window"])
    seen = (j >= lo[..., None]) & (j <= hi[..., None]) & (j < s["kl"][:, None, None])
    p.masked_fill_(~seen[:, None, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, kv, h // kv * lq, lk), v).view(n, kv, h // kv, lq, d) / total
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n, lq, h * d)[s["seq"], s["at"]])


# ------------------------------------------------------------------- exact ----
def exact(case, seed):
    """The definitions, a sequence at a time, in 64 bits."""
    c, t = case, _inputs(case, seed)
    h, kv, d, page = c["h"], c["kv"], c["d"], c.get("page")
    out, at = [], 0
    kc, vc = (t[x].double() for x in ("k_cache", "v_cache")) if c["kind"] == "append" else (None, None)
    for b in range(c["n"]):
        lq, lk = int(t["q_lens"][b]), int(t["kv_lens"][b])
        pos = torch.arange(lk - lq, lk, device="cuda")
        if c["kind"] != "packed":
            keys = torch.arange(lk, device="cuda")
            ids = torch.from_numpy(t["table"][b].astype(np.int64)).cuda()
        if c["kind"] == "append":
            x = t["qkv"][at:at + lq].double().view(lq, h + 2 * kv, d)
            parts = []
            for part, w in ((x[:, :h], "qw"), (x[:, h:h + kv], "kw")):
                if c["norm"]:
                    part = part / torch.sqrt((part ** 2).sum(-1, keepdim=True) / d + EPS) * t[w].double()
                z = torch.complex(part[..., :d // 2].contiguous(), part[..., d // 2:].contiguous())
                z = z * torch.complex(t["cos"][pos].double(), t["sin"][pos].double())[:, None]
                parts.append(torch.cat([z.real, z.imag], -1))
            out.append(parts[0].reshape(lq, h * d))
            kc[ids[pos // page], :, pos % page] = parts[1]
            vc[ids[pos // page], :, pos % page] = x[:, h + kv:]
        else:
            q = t["q"][at:at + lq].view(lq, h, d)
            if c["kind"] == "packed":
                k, v = (t[x][at:at + lq].view(lq, kv, d) for x in ("k", "v"))
            else:
                k, v = (t[x][ids[keys // page], :, keys % page] for x in ("k_cache", "v_cache"))
            lo, hi = _interval(pos[:, None], c["mode"], c["window"])
            j = torch.arange(lk, device="cuda")[None]
            hidden = (j < lo) | (j > hi)
            o = []
            for e in range(h):
                w = q[:, e].double() @ k[:, e // (h // kv)].double().T / math.sqrt(d)
                w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                o.append(w @ v[:, e // (h // kv)].double())
            out.append(torch.cat(o, -1))
        at += lq
    if c["kind"] == "append":
        return {"q": torch.cat(out), "k_cache": kc, "v_cache": vc}
    return torch.cat(out)
