"""Block-scaled fp8: the quantizer, the resident weights and the products against 64-bit restatements."""
import ctypes
import sys

import numpy as np
import pytest

import fp8_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": 0, "f16": 1, "bf16": 2}


def note(msg):
    print(f"[case] {msg}", file=sys.stderr, flush=True)


def rows(r, m, k):
    """Activations with a few large channels."""
    return r.standard_normal((m, k)) * (1 + 12 * (r.random(k) < 0.02))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k", [(1, 16), (3, 128), (5, 144), (2, 1104), (67, 2048)])
def test_quantizer_equals_the_definition(rk, m, k, dtype):
    note(f"fp8 quantize m={m} k={k} {dtype}")
    r = np.random.default_rng(m * k)
    x, v = ref.cast(rows(r, m, k), dtype)
    q, s = rk.quantize_fp8(x, bf16=dtype == "bf16")
    want_q, want_s = ref.quantize(v)
    assert (s == want_s).all()
    assert (q == want_q).all()


def test_quantizer_at_the_edges_of_its_types(rk):
    note("fp8 quantize edges")
    r = np.random.default_rng(0)
    x = np.zeros((10, 256), np.float32)
    x[1, 3] = 1e-30                      # below what the least scale resolves
    x[2] = r.standard_normal(256) * 1e-11
    x[3] = 3.0e38 * r.uniform(-1, 1, 256)
    x[4] = r.standard_normal(256)
    x[4, 130] = np.inf                   # an infinite scale for its block alone
    x[5] = r.standard_normal(256)
    x[5, 7] = np.nan                     # the NaN code, a scale without it
    x[6, :128] = np.float32(1e-42) * np.arange(128)  # subnormal
    x[7, ::2] = -0.0
    x[8] = np.float32(448) * (1 + np.arange(256) % 16 / 16) / 2  # exact ties
    x[8, 0] = x[8, 128] = 448
    x[9] = -np.inf
    q, s = rk.quantize_fp8(x)
    want_q, want_s = ref.quantize(x)
    assert (s == want_s).all()
    nan = (want_q & 127) == 127
    assert (((q & 127) == 127) == nan).all()
    assert (q[~nan] == want_q[~nan]).all()


def product(rk, x, dtype, wid, n, c_dtype, codes):
    """c [m, n] by either form, with a row behind it that must stay as it was."""
    lib, (m, k) = rk.lib(), x.shape
    width = 4 if c_dtype == "f32" else 2
    dx = rk.DeviceBuffer.from_array(x)
    dc = rk.DeviceBuffer.from_array(np.full((m + 1) * n * width, 0x5A, np.uint8))
    if codes:
        q, s = rk.DeviceBuffer(m * k), rk.DeviceBuffer(m * ref.blocks(k) * 4)
        assert lib.rk_quantize_fp8_dev(dx.ptr, TYPES[dtype], m, k, q.ptr, s.ptr, None) == 0
        rc = lib.rk_matmul_fp8_codes_dev(int(wid), q.ptr, s.ptr, m, k, dc.ptr, TYPES[c_dtype], None)
    else:
        rc = lib.rk_matmul_fp8_dev(int(wid), dx.ptr, TYPES[dtype], m, k, dc.ptr, TYPES[c_dtype], None)
    assert rc == 0, lib.rk_last_error()
    rk.synchronize()
    raw = dc.download(((m + 1) * n * width,), np.uint8)
    assert (raw[m * n * width:] == 0x5A).all(), "a value behind the last row was written"
    return raw[:m * n * width].view({"f32": np.float32, "f16": np.float16, "bf16": np.uint16}[c_dtype]).reshape(m, n)


def check(got, c_dtype, x_codes, w_codes, k, what):
    x, w = ref.values(*x_codes), ref.weight_values(*w_codes)
    want, size = x @ w.T, np.abs(x) @ np.abs(w).T
    off = np.abs(ref.widen(got, c_dtype) - want)
    most = ref.sum_error(k, c_dtype) * size
    most = most + (np.abs(want) + most) * ref.HALF[c_dtype] + (2.0**-25 if c_dtype == "f16" else 0)
    assert (off <= most).all(), f"{what}: {np.max(off / most):.3g} times what it may be off"


SHAPES = [(1, 5, 16), (1, 1000, 2048), (2, 32, 128), (31, 33, 144), (32, 96, 1104), (33, 260, 512), (48, 64, 4096), (64, 129, 256),
          (65, 128, 256), (100, 100, 400), (128, 31, 640), (129, 130, 272), (200, 1, 128), (257, 300, 1152), (513, 513, 528)]


@pytest.mark.parametrize("dtype,c_dtype", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products(rk, m, n, k, dtype, c_dtype):
    note(f"fp8 product m={m} n={n} k={k} {dtype}->{c_dtype}")
    r = np.random.default_rng(m * 7 + n * 3 + k)
    codes, scales = ref.random_weight(r, n, k)
    x, v = ref.cast(rows(r, m, k), dtype)
    wid = rk.pack_fp8(codes, scales)
    assert rk.weight_info(wid)[1:3] == (n, k)
    for by_codes in (True, False):
        got = product(rk, x, dtype, wid, n, c_dtype, by_codes)
        check(got, c_dtype, ref.quantize(v), (codes, scales), k, f"codes={by_codes}")


@pytest.mark.parametrize("m,n,k", [(2900, 4100, 384), (16384, 257, 128), (300, 16400, 256)])
def test_large_grids(rk, m, n, k):
    """Tiles of 256, whole and ragged, and every output block of a wide weight."""
    note(f"fp8 large m={m} n={n} k={k}")
    r = np.random.default_rng(n)
    codes, scales = ref.random_weight(r, n, k)
    x, v = ref.cast(rows(r, m, k), "bf16")
    wid = rk.pack_fp8(codes, scales)
    got = product(rk, x, "bf16", wid, n, "bf16", False)
    q, s = ref.quantize(v)
    some = np.unique(np.concatenate([r.integers(0, m, 60), [0, m - 1]]))
    check(got[some], "bf16", (q[some], s[some]), (codes, scales), k, "rows")
    for at in (np.s_[:, :40], np.s_[:, -40:]):
        x64, w64 = ref.values(q, s), ref.weight_values(codes, scales)[at[1]]
        want, size = x64 @ w64.T, np.abs(x64) @ np.abs(w64).T
        off = np.abs(ref.widen(got[at], "bf16") - want)
        assert (off <= ref.sum_error(k, "bf16") * size * 1.01 + np.abs(want) * 2.0**-8).all()


def test_weights_from_f32(rk):
    note("fp8 pack f32")
    r = np.random.default_rng(4)
    for n, k in [(1, 16), (130, 144), (256, 384)]:
        w = (r.standard_normal((n, k)) * 0.03).astype(np.float32)
        x = rows(r, 9, k).astype(np.float32)
        wid = rk.pack_fp8_f32(w)
        check(rk.matmul_fp8(x, wid), "f32", ref.quantize(x), ref.quantize_weight(w), k, f"{n}x{k}")
        # rk_matmul on host rows, through its chunks
        check(rk.matmul(x, wid), "f32", ref.quantize(x), ref.quantize_weight(w), k, f"host {n}x{k}")


@pytest.mark.parametrize("m", [5, 40, 300])
def test_non_finite_values_stay_in_their_rows(rk, m):
    note(f"fp8 non-finite m={m}")
    r = np.random.default_rng(m)
    n, k = 70, 272
    codes, scales = ref.random_weight(r, n, k)
    codes[3, 200] = 127  # a NaN in the weight: output 3 of every row
    x = rows(r, m, k).astype(np.float32)
    clean = x.copy()
    x[1, 20], x[m - 1, 270] = np.inf, np.nan
    wid = rk.pack_fp8(codes, scales)
    for c_dtype in ("f32", "bf16"):
        got = ref.widen(product(rk, x, "f32", wid, n, c_dtype, True), c_dtype)
        assert np.isnan(got[[1, m - 1]]).all() and np.isnan(got[:, 3]).all()
        keep = [i for i in range(m) if i not in (1, m - 1)]
        cols = [j for j in range(n) if j != 3]
        want = ref.widen(product(rk, clean, "f32", wid, n, c_dtype, True), c_dtype)
        assert (got[np.ix_(keep, cols)] == want[np.ix_(keep, cols)]).all()


def test_refusals(rk):
    note("fp8 refusals")
    lib, r = rk.lib(), np.random.default_rng(1)
    codes, scales = ref.random_weight(r, 64, 256)
    wid, f16 = int(rk.pack_fp8(codes, scales)), int(rk.pack(r.standard_normal((64, 256)).astype(np.float32)))
    b = rk.DeviceBuffer(1 << 16)
    out = ctypes.c_uint64()
    h = codes.ctypes.data
    assert lib.rk_pack_fp8(h, scales.ctypes.data, 64, 250, ctypes.byref(out)) == rk.RK_E_SHAPE
    assert lib.rk_pack_fp8(h, scales.ctypes.data, 0, 256, ctypes.byref(out)) == rk.RK_E_SHAPE
    assert lib.rk_pack_fp8(h, None, 64, 256, ctypes.byref(out)) == rk.RK_E_SHAPE
    assert lib.rk_pack_fp8_f32(None, 64, 256, ctypes.byref(out)) == rk.RK_E_SHAPE
    q = lambda x, dt, m, k, o, s: lib.rk_quantize_fp8_dev(x, dt, m, k, o, s, None)  # noqa: E731
    assert q(b.ptr, 3, 2, 256, b.ptr, b.ptr) == rk.RK_E_SHAPE
    assert q(b.ptr, 0, 2, 8, b.ptr, b.ptr) == rk.RK_E_SHAPE
    assert q(b.ptr, 0, -1, 256, b.ptr, b.ptr) == rk.RK_E_SHAPE
    assert q(b.ptr + 4, 0, 2, 256, b.ptr, b.ptr) == rk.RK_E_SHAPE
    assert q(b.ptr, 0, 2, 256, None, b.ptr) == rk.RK_E_SHAPE
    assert q(b.ptr, 0, 2, 256, b.ptr, None) == rk.RK_E_SHAPE
    assert q(None, 0, 0, 256, None, None) == 0
    for f in (lambda i, x, m, k, c, dt: lib.rk_matmul_fp8_dev(i, x, 0, m, k, c, dt, None),
              lambda i, x, m, k, c, dt: lib.rk_matmul_fp8_codes_dev(i, x, b.ptr, m, k, c, dt, None)):
        assert f(wid, b.ptr, 2, 240, b.ptr, 0) == rk.RK_E_SHAPE
        assert f(wid, b.ptr, -1, 256, b.ptr, 0) == rk.RK_E_SHAPE
        assert f(wid, b.ptr, 2, 256, b.ptr, 5) == rk.RK_E_SHAPE
        assert f(wid, b.ptr + 8, 2, 256, b.ptr, 0) == rk.RK_E_SHAPE
        assert f(wid, b.ptr, 2, 256, b.ptr + 8, 0) == rk.RK_E_SHAPE
        assert f(wid, None, 2, 256, b.ptr, 0) == rk.RK_E_SHAPE
        assert f(wid, b.ptr, 2, 256, None, 0) == rk.RK_E_SHAPE
        assert f(f16, b.ptr, 2, 256, b.ptr, 0) == rk.RK_E_UNSUPPORTED
        assert f(123456789, b.ptr, 2, 256, b.ptr, 0) == rk.RK_E_SHAPE
        assert f(wid, None, 0, 256, None, 0) == 0
    # other products do not take an fp8 weight
    assert lib.rk_matmul_f16_dev(wid, b.ptr, 2, 256, b.ptr, None) == rk.RK_E_UNSUPPORTED
    assert lib.rk_matmul_w8a8_dev(wid, b.ptr, b.ptr, 256, 2, 256, b.ptr, None) == rk.RK_E_UNSUPPORTED
    assert lib.rk_matmul_i8_raw_dev(wid, b.ptr, 2, 256, b.ptr, None) == rk.RK_E_UNSUPPORTED


@pytest.mark.parametrize("k", [16, 144, 272, 400, 528, 1104])
@pytest.mark.parametrize("m,n,c_dtype", [(260, 2100, "bf16"), (500, 2100, "f32"), (1100, 4100, "bf16"), (1100, 4100, "f32"), (2900, 4100, "f16")])
def test_products_of_tiles(rk, m, n, k, c_dtype):
    """Grids that are too large for the kernel of few rows, at one to nine blocks of K: 64 x 128 tiles in 16 and in 32 bits,
    128 x 128 in both, 256 x 256."""
    note(f"fp8 tiles m={m} n={n} k={k} {c_dtype}")
    r = np.random.default_rng(m + n + k)
    codes, scales = ref.random_weight(r, n, k)
    x = rows(r, m, k).astype(np.float32)
    got = product(rk, x, "f32", rk.pack_fp8(codes, scales), n, c_dtype, True)
    q, s = ref.quantize(x)
    some = np.unique(np.concatenate([r.integers(0, m, 150), [0, 63, 64, 127, 128, 255, 256, m - 1]]))
    check(got[some], c_dtype, (q[some], s[some]), (codes, scales), k, "rows")
    x64, w64 = ref.values(q, s), ref.weight_values(codes, scales)[-140:]
    want, size = x64 @ w64.T, np.abs(x64) @ np.abs(w64).T
    most = ref.sum_error(k, c_dtype) * size
    most = most + (np.abs(want) + most) * ref.HALF[c_dtype] + (2.0**-25 if c_dtype == "f16" else 0)
    assert (np.abs(ref.widen(got[:, -140:], c_dtype) - want) <= most).all(), "columns"


def test_captured_calls(rk):
    """Quantizer and product in a graph; small calls by one entry, one of them larger than it takes in one launch outside a
    capture. Replayed on new rows, with calls of other sizes in between."""
    note("fp8 captured")
    from test_gpu_sequences import Graph
    lib, r = rk.lib(), np.random.default_rng(31)
    n, k = 200, 1040
    codes, scales = ref.random_weight(r, n, k)
    wid, st = int(rk.pack_fp8(codes, scales)), rk.new_stream()
    sizes = (3, 32, 40, 700)
    x = {m: rk.DeviceBuffer(m * k * 2) for m in sizes}
    c = {m: rk.DeviceBuffer(m * n * 2) for m in sizes}
    q, s = rk.DeviceBuffer(700 * k), rk.DeviceBuffer(700 * ref.blocks(k) * 4)
    for m in sizes:
        x[m].zero()

    def step():
        for m in (3, 32):
            assert lib.rk_matmul_fp8_dev(wid, x[m].ptr, TYPES["bf16"], m, k, c[m].ptr, TYPES["bf16"], st) == 0
        assert lib.rk_matmul_fp8_dev(wid, x[40].ptr, TYPES["bf16"], 40, k, c[40].ptr, TYPES["bf16"], st) == rk.RK_E_UNSUPPORTED
        for m in (40, 700):
            assert lib.rk_quantize_fp8_dev(x[m].ptr, TYPES["bf16"], m, k, q.ptr, s.ptr, st) == 0
            assert lib.rk_matmul_fp8_codes_dev(wid, q.ptr, s.ptr, m, k, c[m].ptr, TYPES["bf16"], st) == 0
    g = Graph(st, step)
    for _ in range(4):
        host = {}
        for m in sizes:
            host[m], v = ref.cast(rows(r, m, k), "bf16")
            x[m].upload(host[m])
            host[m] = (host[m], v)
        g.replay()
        rk.synchronize(st)
        for m in sizes:
            got = c[m].download((m, n), np.uint16)
            check(got, "bf16", ref.quantize(host[m][1]), (codes, scales), k, f"captured m={m}")
            if m != 32:
                assert (got == product(rk, host[m][0], "bf16", wid, n, "bf16", m > 3)).all()
    g.destroy()
    rk.destroy_stream(st)


def test_two_streams_share_the_codes_memory(rk):
    """Calls in turn on two streams, larger ones after smaller ones: each waits for the codes of the last."""
    note("fp8 two streams")
    lib, r = rk.lib(), np.random.default_rng(32)
    n, k = 300, 528
    codes, scales = ref.random_weight(r, n, k)
    wid, sts = int(rk.pack_fp8(codes, scales)), [rk.new_stream(), rk.new_stream()]
    work = []
    for i, m in enumerate((40, 700, 64, 1500, 33, 2000, 900, 50)):
        x, v = ref.cast(rows(r, m, k), "f16")
        work.append((v, rk.DeviceBuffer.from_array(x), rk.DeviceBuffer(m * n * 4)))
    rk.synchronize()
    for i, (v, x, c) in enumerate(work):
        assert lib.rk_matmul_fp8_dev(wid, x.ptr, TYPES["f16"], len(v), k, c.ptr, TYPES["f32"], sts[i % 2]) == 0
    for st in sts:
        rk.synchronize(st)
    for v, _, c in work:
        check(c.download((len(v), n), np.float32), "f32", ref.quantize(v), (codes, scales), k, f"m={len(v)}")
    for st in sts:
        rk.destroy_stream(st)


@pytest.mark.parametrize("m,k", [(32, 2048), (1, 65536), (2, 32768), (3, 21840), (31, 2112), (5, 13104)])
def test_captured_calls_up_to_64_kb_of_codes(rk, m, k):
    """The largest calls that may be captured by one entry, K of whole blocks and not."""
    note(f"fp8 captured m={m} k={k}")
    from test_gpu_sequences import Graph
    assert m * k <= 65536
    lib, r = rk.lib(), np.random.default_rng(k)
    n = 40
    codes, scales = ref.random_weight(r, n, k)
    wid, st = int(rk.pack_fp8(codes, scales)), rk.new_stream()
    x, c = rk.DeviceBuffer(m * k * 2), rk.DeviceBuffer(m * n * 2)
    x.zero()
    rcs = []
    g = Graph(st, lambda: rcs.append(lib.rk_matmul_fp8_dev(wid, x.ptr, TYPES["bf16"], m, k, c.ptr, TYPES["bf16"], st)))
    assert rcs == [0], lib.rk_last_error()
    for _ in range(3):
        host, v = ref.cast(rows(r, m, k), "bf16")
        x.upload(host)
        g.replay()
        rk.synchronize(st)
        check(c.download((m, n), np.uint16), "bf16", ref.quantize(v), (codes, scales), k, f"captured m={m}")
        product(rk, host, "bf16", wid, n, "bf16", False)  # and the call outside of one, in between
    g.destroy()
    rk.destroy_stream(st)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_rows_behind_2_31_bytes(rk, dtype):
    """A million rows, whose codes and results each pass 2^31 bytes: the same rows over and over, the last of them as the first."""
    note(f"fp8 past 2^31 bytes {dtype}")
    lib, r = rk.lib(), np.random.default_rng(41)
    m, n, k, part = (1 << 20) + 37, 1040, 2064, 8192 + 64
    codes, scales = ref.random_weight(r, n, k)
    wid = int(rk.pack_fp8(codes, scales))
    x, v = ref.cast(rows(r, part, k), dtype)
    width = x.itemsize
    dx, dc = rk.DeviceBuffer(m * k * width), rk.DeviceBuffer(m * n * width)
    dx.upload(x)
    done = part
    while done < m:
        more = min(done, m - done)  # whole parts: rows of the same index modulo the part
        assert lib.rk_memcpy_dtod(dx.ptr + done * k * width, dx.ptr, more * k * width, None) == 0
        done += more
    assert lib.rk_matmul_fp8_dev(wid, dx.ptr, TYPES[dtype], m, k, dc.ptr, TYPES[dtype], None) == 0, lib.rk_last_error()
    rk.synchronize()
    got = []
    for at in (0, m - 500):
        dst = rk.DeviceBuffer(500 * n * width)
        assert lib.rk_memcpy_dtod(dst.ptr, dc.ptr + at * n * width, 500 * n * width, None) == 0
        rk.synchronize()
        got.append(dst.download((500, n), x.dtype))
        of = np.arange(at, at + 500) % part
        q, s = ref.quantize(v[of])
        check(got[-1], dtype, (q, s), (codes, scales), k, f"rows from {at}")
