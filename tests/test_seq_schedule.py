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
