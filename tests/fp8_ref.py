"""Block-scaled fp8 restated on the CPU: e4m3 by a table of its values, products in 64 bits."""
import numpy as np

BLOCK = 128
_c = np.arange(128)
VALUES = np.where(_c >> 3 == 0, (_c & 7) / 8.0 * 2.0**-6, (1 + (_c & 7) / 8.0) * 2.0 ** ((_c >> 3) - 7.0))
VALUES[127] = np.nan
_MID = (VALUES[:126] + VALUES[1:127]) / 2


def blocks(n):
    return -(-n // BLOCK)


def decode(codes):
    codes = np.asarray(codes, np.uint8)
    v = VALUES[codes & 127]
    return np.where(codes & 128, -v, v)


def encode(v):
    """Nearest codes of values within ±448, ties to the even code; NaN to a NaN code (127)."""
    v = np.asarray(v, np.float64)
    a = np.abs(v)
    at = np.searchsorted(_MID, a, side="left")  # the midpoint itself: the lower of the two
    tie = (at < 126) & (_MID[np.minimum(at, 125)] == a)
    at = np.where(tie & (at % 2 == 1), at + 1, at)
    at = np.where(np.isnan(v), 127, at)
    return (at | (np.signbit(v).astype(np.int64) << 7)).astype(np.uint8)


def quantize(x):
    """(codes, scales) of rows: scales max(amax / 448, 1e-12) and quotients are f32 numbers."""
    x = np.asarray(x, np.float32)
    m, k = x.shape
    q, s = np.zeros((m, k), np.uint8), np.zeros((m, blocks(k)), np.float32)
    with np.errstate(all="ignore"):
        for b in range(blocks(k)):
            p = x[:, b * BLOCK:(b + 1) * BLOCK]
            amax = np.fmax.reduce(np.abs(p), axis=1, initial=0)  # (a NaN is left out)
            s[:, b] = np.maximum((amax.astype(np.float64) / 448).astype(np.float32), np.float32(1e-12))
            q[:, b * BLOCK:(b + 1) * BLOCK] = encode((p.astype(np.float64) / s[:, b:b + 1].astype(np.float64)).astype(np.float32))
    return q, s


def quantize_weight(w):
    """(codes, scales [ceil(N/128), ceil(K/128)]) of an f32 weight."""
    n, k = w.shape
    q, s = np.zeros((n, k), np.uint8), np.zeros((blocks(n), blocks(k)), np.float32)
    for a in range(blocks(n)):
        for b in range(blocks(k)):
            at = np.s_[a * BLOCK:(a + 1) * BLOCK, b * BLOCK:(b + 1) * BLOCK]
            s[a, b] = max(np.float32(np.abs(w[at]).max() / 448.0), np.float32(1e-12))
            q[at] = encode((w[at].astype(np.float64) / np.float64(s[a, b])).astype(np.float32))
    return q, s


def values(q, s):
    """Rows as the values they stand for, in 64 bits."""
    return decode(q) * np.repeat(s.astype(np.float64), BLOCK, 1)[:, :q.shape[1]]


def weight_values(q, s):
    n, k = q.shape
    return decode(q) * np.repeat(np.repeat(s.astype(np.float64), BLOCK, 0)[:n], BLOCK, 1)[:, :k]


def random_weight(r, n, k):
    codes = encode(np.clip(r.standard_normal((n, k)) * 105, -448, 448))
    return codes, (2e-4 * (0.8 + 0.4 * r.random((blocks(n), blocks(k))))).astype(np.float32)


def random_stack(r, e, n, k):
    parts = [random_weight(r, n, k) for _ in range(e)]
    return np.stack([p[0] for p in parts]), np.stack([p[1] for p in parts])


def to_bf16(x):
    """bf16 bits of f32 values, to nearest even."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    out = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), out)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


def cast(x, dtype):
    """f32 values as an array of the named type (bf16 as its bits), and the values that it holds."""
    x = np.asarray(x, np.float32)
    if dtype == "bf16":
        b = to_bf16(x)
        return b, from_bf16(b)
    a = x.astype(np.float16 if dtype == "f16" else np.float32)
    return a, a.astype(np.float32)


def widen(a, dtype):
    return (from_bf16(a) if dtype == "bf16" else a).astype(np.float64)


# Half a step of each type, relative.
HALF = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def sum_error(k, dtype):
    """How far the f32 sums of a product may be off, as a share of the sum of its terms' magnitudes. f32 results: at most
    one rounding (2^-24) for each of the 128 terms of a block, for each block, and four for the scales. fp16 and bf16
    results: the fp8 instructions cut terms 2^-13 below the largest at worst; on normally distributed codes 2^-15 of the sum
    of magnitudes covers what they lose twice."""
    return (128 + blocks(k) + 4) * 2.0**-24 + (0 if dtype == "f32" else 2.0**-14)
