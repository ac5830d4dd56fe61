"""Plain 64-bit forms of the operators on batches of sequences, and the error bounds that their tests use."""
import numpy as np

HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of the type, relative


def encode(x, dtype):
    """Bits of x in dtype, rounded to nearest even."""
    x = np.asarray(x, np.float32)
    if dtype == "f16":
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def decode(b, dtype):
    b = np.asarray(b, np.uint16)
    if dtype == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def hidden(pos, n_kv, mode, window):
    """[queries, keys]: whether the mask hides the key. Rows that see nothing see every key alike (None)."""
    t, j = np.asarray(pos)[:, None], np.arange(n_kv)[None]
    if mode == 2 and window < 0:
        mode = 0
    if mode == 3 and window < 0:
        mode = 1
    h = np.zeros((len(t), n_kv), bool)
    if mode in (1, 3):
        h |= j > t
    if mode == 2:
        h |= np.abs(t - j) > window
    if mode == 3:
        h |= j <= t - window
    return h


def attention(q, k, v, pos, scale, softcap, mode, window, half):
    """One sequence: q [n, H, D], k and v [m, KV, D] (f64) -> (out, bound), both [n, H, D].

    The bound, with A = softmax·|v|: the result is rounded once (half·|out|), every probability once (half·A; its
    subnormals by at most 2^-25 of the largest); f32 scores are off by at most (D + 4)·2^-24·scale·|q|·|k|, which
    moves a probability and the row sum by twice that together, and exp2 and the sums over the keys add
    (n + 16)·2^-23."""
    n, H, D = q.shape
    m, KV = k.shape[0], k.shape[1]
    hide = hidden(pos, m, mode, window)
    empty = hide.all(1)
    out, bound = np.empty(q.shape), np.empty(q.shape)
    for h in range(H):
        kh, vh = k[:, h // (H // KV)], v[:, h // (H // KV)]
        s = scale * (q[:, h] @ kh.T)
        ds = (D + 4) * 2.0 ** -24 * scale * (np.abs(q[:, h]) @ np.abs(kh).T)
        if softcap:
            s = softcap * np.tanh(s / softcap)
            ds = ds + 2.0 ** -21 * softcap
        s = np.where(hide, -np.inf, s)
        s[empty] = 0.0
        ds = np.where(hide, 0.0, ds).max(1, keepdims=True)
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h] = p @ vh
        A = p @ np.abs(vh)
        bound[:, h] = half * np.abs(out[:, h]) * 1.01 + A * (half + 2 * ds + (m + 16) * 2.0 ** -23) + \
            m * 2.0 ** -25 * np.abs(vh).max(initial=0.0) + 2.0 ** -25
    return out, bound


def prologue(x, w, cos, sin, eps, half):
    """x [n, heads, D] at positions with cos, sin [n, D/2] -> (rotated, bound). One rounding (half), and f32
    arithmetic: the norm's factor and the two products of a rotation are off by a few steps of 2^-24 of the pair."""
    D = x.shape[-1]
    y = x
    if w is not None:
        y = x / np.sqrt((x ** 2).sum(-1, keepdims=True) / D + eps) * w
    a, b = y[..., :D // 2], y[..., D // 2:]
    c, s = cos[:, None], sin[:, None]
    out = np.concatenate([a * c - b * s, b * c + a * s], -1)
    size = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)], -1)
    return out, half * np.abs(out) * 1.01 + size * (D + 16) * 2.0 ** -24 + 2.0 ** -25


def close(got, want, bound, what=""):
    assert np.isfinite(got).all(), what
    over = np.abs(got - want) / bound
    assert over.max(initial=0.0) <= 1.0, f"{what}: {over.max():.3f} of the bound at {np.unravel_index(over.argmax(), over.shape)}"


class Pages:
    """A page table for sequences of kv_lens keys, pages in shuffled order with some to spare."""

    def __init__(self, rng, kv_lens, ps, spare=3):
        need = [-(-int(x) // ps) for x in kv_lens]
        self.n_pages, self.ps = sum(need) + spare, ps
        ids = rng.permutation(self.n_pages).astype(np.int32)
        self.table, at = np.full((len(need), max(need + [1])), -1, np.int32), 0
        for i, n in enumerate(need):
            self.table[i, :n] = ids[at:at + n]
            at += n

    def put(self, cache, i, keys):
        """Keys [n, KV, D] of sequence i into cache [n_pages, KV, ps, D]."""
        j = np.arange(len(keys))
        cache[self.table[i, j // self.ps], :, j % self.ps] = keys
