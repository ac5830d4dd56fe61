"""The schedules of batches of sequences, without a device: which rows and keys the items cover, and what they depend
on. The planner is compiled for the host from its own source."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CUS = 256
FIELDS = ["tok0", "pos0", "rows", "row0", "kv_len", "k_begin", "k_end", "k_lo", "table", "n_parts", "sp", "part0"]


class Geom(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in ("paged", "n_head", "n_kv_heads", "head_dim", "mask_mode", "page_size")] + \
        [("window", ctypes.c_int64), ("n_pages", ctypes.c_int64)]


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("plan") / "seq_plan_host.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(HERE, "seq_plan_host.cpp"), "-o", so], check=True)
    lib = ctypes.CDLL(so)
    assert lib.item_words() == len(FIELDS)
    return lib


def geom(h=8, kv=2, d=64, mode=1, window=-1, ps=0, n_pages=1 << 20):
    return Geom(ps > 0, h, kv, d, mode, ps, window, n_pages)


def plan(host, g, q, kv=None, cus=CUS):
    """Row items and tile items (a dict of columns each), and the counts."""
    q = np.array(q, np.int32)
    kvl = np.array(q if kv is None else kv, np.int32)
    stride = int(max([1, *(-(-int(m) // g.page_size) for m in kvl)])) if g.paged else 0
    table = np.arange(max(1, len(q) * stride), dtype=np.int32) % g.n_pages
    counts, items = (ctypes.c_int64 * 8)(), np.zeros((1 << 16, len(FIELDS)), np.int32)
    rc = host.plan(ctypes.byref(g), ctypes.c_void_p(q.ctypes.data), ctypes.c_void_p(kvl.ctypes.data if g.paged else None),
                   ctypes.c_void_p(table.ctypes.data if g.paged else None), ctypes.c_int64(stride), ctypes.c_int64(len(q)), cus, counts,
                   ctypes.c_void_p(items.ctypes.data), ctypes.c_int64(len(items)))
    assert rc == 0
    n, m = counts[0], counts[1]
    cols = lambda a: {f: a[:, i].astype(np.int64) for i, f in enumerate(FIELDS)}  # noqa: E731
    return cols(items[:n]), cols(items[n:n + m]), list(counts)


@pytest.mark.parametrize("h,kv,d", [(16, 4, 64), (8, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("mode,window", [(3, 512), (2, 200)])
def test_a_longer_hidden_prefix_changes_no_kernel(host, h, kv, d, mode, window):
    """What a window hides costs nothing: the same new tokens behind a longer prefix are cut alike."""
    for q in ([64], [1], [200], [64, 1, 1], [16] * 16):
        shapes = set()
        for prefix in (4096, 16384, 65536, 1 << 20):
            r, t, counts = plan(host, geom(h, kv, d, mode, window, 64), q, [prefix + x for x in q])
            shapes.add((tuple(counts[:4]), counts[6], *((tuple(i["k_end"] - i["k_begin"]), tuple(i["n_parts"])) for i in (r, t))))
        assert len(shapes) == 1, f"{q}: {[s[0] for s in shapes]}"


def test_parts_of_a_tile_follow_its_keys(host):
    """16 states are merged in one pass, which pays up to a length that depends on the kind of items."""
    def parts(kv, n, q=1, g=8, d=128):
        r, t, _ = plan(host, geom(kv * g, kv, d, ps=64), [q], [n])
        return [int(i["n_parts"].max(initial=0)) for i in (r, t)]

    for kv in (1, 4):
        assert parts(kv, 8000)[0] == 16 and parts(kv, 12000)[0] == 16
        assert parts(kv, 16000)[0] == 32 and parts(kv, 30000)[0] == 32 and parts(kv, 60000)[0] == (64 if kv == 1 else 32)
    assert parts(8, 16000)[0] == 16 and parts(8, 20000)[0] == 32  # (every CU has work with 16)
    # tiles, of batches that are too large for the kernel of few rows
    assert parts(1, 12000, 256)[1] == 16 and parts(1, 24000, 128)[1] == 32 and parts(4, 24000, 32)[1] == 32
    assert parts(1, 20000, 256, d=64)[1] == 16


def random_batch(rng, max_seqs=40):
    """A geometry and the lengths of a batch: few or many sequences, single tokens, chunks or both."""
    kv = int(rng.choice([1, 2, 3, 4, 8, 48]))
    g = int(rng.choice([1, 2, 3, 4, 7, 8, 17]))
    mode = int(rng.integers(0, 4))
    window = int(rng.choice([-1, 0, 1, 15, 100, 1024])) if mode >= 2 else -1
    paged = bool(rng.integers(0, 2))
    n = int(rng.integers(0, max_seqs))
    top = int(rng.choice([1, 3, 40, 300, 2000]))
    q = [int(x) for x in rng.integers(0, top + 1, n)]
    if rng.integers(0, 2):
        q = [x if i < 2 else min(x, 1) for i, x in enumerate(q)]
    k = [x + int(rng.integers(0, rng.choice([1, 50, 9000]))) if paged else x for x in q]
    return geom(kv * g, kv, int(rng.choice([32, 64, 128, 256])), mode, window, 32 if paged else 0), q, k


def visible(g, t, kv_len):
    lo, hi = 0, kv_len - 1
    if g.mask_mode == 3 and g.window == 0:
        return lo, hi
    if g.mask_mode in (1, 3):
        hi = min(hi, t)
    if g.window >= 0 and g.mask_mode == 2:
        lo, hi = max(0, t - g.window), min(hi, t + g.window)
    if g.window >= 0 and g.mask_mode == 3:
        lo = max(0, t - g.window + 1)
    return lo, hi


@pytest.mark.parametrize("seed", range(6))
def test_items_cover_every_row_and_visible_key_once(host, seed):
    rng = np.random.default_rng(seed)
    for _ in range(60):
        g, q, k = random_batch(rng)
        G = g.n_head // g.n_kv_heads
        cus = int(rng.choice([256, 256, 32]))
        r, t, counts = plan(host, g, q, k, cus)
        first = np.cumsum([0, *q])
        seqs = {int(first[i]): i for i in range(len(q)) if q[i]}
        tiles = {}
        for kind, (items, rows_of, step) in enumerate(((r, 16, 32), (t, 128 if g.head_dim <= 128 else 64, 64))):
            slots = []
            length = items["k_end"] - items["k_begin"]
            steps = -(-length // step)
            assert (steps[:-1] >= steps[1:]).all()  # the longest first
            for x in zip(*(items[f] for f in FIELDS)):
                x = dict(zip(FIELDS, map(int, x)))
                i = seqs[x["tok0"]]
                assert (x["rows"], x["kv_len"], x["pos0"]) == (q[i] * G, k[i], k[i] - q[i])
                assert x["row0"] % rows_of == 0 and x["row0"] < x["rows"] and x["k_begin"] % step == 0
                tiles.setdefault((i, x["row0"], rows_of), []).append(x)
            for (i, row0, w), parts in ((a, b) for a, b in tiles.items() if a[2] == rows_of):
                parts.sort(key=lambda p: p["sp"])
                n = parts[0]["n_parts"]
                assert [p["sp"] for p in parts] == list(range(n)) and len({(p["part0"], p["n_parts"]) for p in parts}) == 1
                slots += [*range(parts[0]["part0"], parts[0]["part0"] + n)] if n > 1 else []
                last = min(row0 + w, q[i] * G) - 1
                lo, hi = visible(g, k[i] - q[i] + row0 // G, k[i])[0], visible(g, k[i] - q[i] + last // G, k[i])[1]
                assert parts[0]["k_lo"] == lo and parts[0]["k_begin"] == lo // step * step and parts[-1]["k_end"] == hi + 1
                assert all(a["k_end"] == b["k_begin"] and a["k_begin"] < a["k_end"] and a["k_end"] % step == 0 for a, b in zip(parts, parts[1:]))
            assert sorted(slots) == list(range(counts[2 + kind]))  # no two states share a slot
        want = {i: set() for i in seqs.values()}
        for i, row0, w in tiles:
            rows = set(range(row0, min(row0 + w, q[i] * G)))
            assert not rows & want[i]
            want[i] |= rows
        assert all(len(want[i]) == q[i] * G for i in want)


@pytest.mark.parametrize("seed", range(4))
def test_a_reservation_holds_every_smaller_batch(host, seed):
    rng = np.random.default_rng(100 + seed)
    for _ in range(60):
        g, q, k = random_batch(rng)
        n_seqs, toks, max_q, cus = len(q), sum(q), max([*q, int(rng.integers(1, 500))]), int(rng.choice([256, 32]))
        top = (ctypes.c_int64 * 4)()
        host.bound(ctypes.byref(g), ctypes.c_int64(n_seqs), ctypes.c_int64(toks), ctypes.c_int64(max_q), cus, top)
        for _ in range(8):
            left, ql = toks, []
            for _ in range(int(rng.integers(0, n_seqs + 1))):
                x = int(min(left, max_q, rng.choice([0, 1, max_q, int(rng.integers(0, max_q + 1))])))
                ql.append(x)
                left -= x
            kl = [x + int(rng.integers(0, 20000)) if g.paged else x for x in ql]
            _, _, c = plan(host, g, ql, kl, cus)
            assert c[0] <= top[0] and c[2] <= top[1] and c[1] <= top[2] and c[3] <= top[3], (ql, kl, c, list(top))
