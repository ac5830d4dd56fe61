"""GPU parity of the operators on batches of sequences (packed attention, attention over a paged KV cache, the
append in front of it) against plain 64-bit forms, with bounds that follow from the types."""
import ctypes
import sys

import numpy as np
import pytest

import seqs_ref as ref

pytestmark = pytest.mark.gpu
DIMS = [32, 48, 64, 72, 80, 96, 112, 128, 256]


def note(msg):
    print(f"[case] {msg}", file=sys.stderr, flush=True)


def dt(rk, dtype):
    return {"f16": rk.DTYPE_F16, "bf16": rk.DTYPE_BF16}[dtype]


def rows(rng, dtype, *shape, scale=1.0):
    return ref.encode(rng.standard_normal(shape) * scale, dtype)


def upload(rk, *arrays):
    return [rk.DeviceBuffer.from_array(a) for a in arrays]


def ok(rk, rc):
    assert rc == 0, rk.lib().rk_last_error()


FILL = 0x1234  # what lies in output rows beforehand


def packed(rk, q, k, v, lens, h, kv, d, dtype, scale, softcap=0.0, mode=1, window=-1, extra=0, plan=None, stream=None):
    """Bits [tokens + extra, h*d] of one call."""
    plan = plan or rk.packed_plan(lens, h, kv, d, mode, window)
    b = upload(rk, q, k, v, np.full((len(q) + extra, h * d), FILL, np.uint16))
    ok(rk, rk.lib().rk_attention_packed_dev(plan.ptr, b[0].ptr, h * d, b[1].ptr, kv * d, b[2].ptr, kv * d, scale, softcap,
                                            b[3].ptr, h * d, dt(rk, dtype), stream))
    rk.synchronize(stream)
    return b[3].download((len(q) + extra, h * d), np.uint16)


def check_packed(got, q, k, v, lens, h, kv, d, dtype, scale, softcap=0.0, mode=1, window=-1):
    at = 0
    for i, n in enumerate(lens):
        if n:
            qs, ks, vs = (ref.decode(t[at:at + n], dtype).reshape(n, -1, d) for t in (q, k, v))
            want, bound = ref.attention(qs, ks, vs, np.arange(n), scale, softcap, mode, window, ref.HALF[dtype])
            ref.close(ref.decode(got[at:at + n], dtype).reshape(n, h, d), want, bound, f"sequence {i} of {n}")
        at += n


def crowd(h, kv):
    """Sequences of one token that make a batch of these heads one with many tiles: its longer sequences go to the
    kernel of many rows, not to that of few as in a small batch."""
    return 1024 // (kv * -(-(h // kv) // 16)) + 1


def packed_case(rk, seed, lens, h, kv, d, dtype, **kw):
    one_packed_case(rk, seed, lens, h, kv, d, dtype, **kw)
    if max(lens) * (h // kv) > 16:
        one_packed_case(rk, seed, [*lens, *[1] * crowd(h, kv)], h, kv, d, dtype, **kw)


def one_packed_case(rk, seed, lens, h, kv, d, dtype, **kw):
    rng, toks = np.random.default_rng(seed), sum(lens)
    q, k, v = (rows(rng, dtype, toks, n * d) for n in (h, kv, kv))
    got = packed(rk, q, k, v, lens, h, kv, d, dtype, d ** -0.5, extra=3, **kw)
    assert (got[toks:] == FILL).all()  # rows behind the last sequence
    check_packed(got[:toks], q, k, v, lens, h, kv, d, dtype, d ** -0.5, **kw)
    again = packed(rk, q, k, v, lens, h, kv, d, dtype, d ** -0.5, extra=3, **kw)
    assert (again == got).all()  # the sums have one order


# Every head dim and type: lengths of none, one, around the 16-, 64- and 128-row edges, several groups.
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("lens,h,kv", [([0, 1, 15, 16, 17, 0, 64, 65], 4, 2), ([129, 5, 200], 2, 2), ([43, 1], 21, 3)])
def test_packed_head_dims(rk, d, dtype, lens, h, kv):
    note(f"packed d={d} {dtype} {lens} {h}/{kv}")
    packed_case(rk, d + len(lens), lens, h, kv, d, dtype)


@pytest.mark.parametrize("mode,window,softcap", [(0, -1, 0.0), (1, -1, 20.0), (2, 0, 0.0), (2, 33, 0.0), (2, 500, 0.0),
                                                 (2, -1, 0.0), (3, 1, 0.0), (3, 70, 15.0), (3, 0, 0.0), (3, 0, 5.0),
                                                 (3, 4000, 0.0), (3, -1, 0.0), (2, 1 << 50, 0.0)])
@pytest.mark.parametrize("h,kv,d", [(6, 2, 64), (3, 1, 256)])
def test_packed_masks(rk, mode, window, softcap, h, kv, d):
    note(f"packed masks mode={mode} window={window} softcap={softcap} d={d}")
    packed_case(rk, window % 97 + mode, [150, 1, 333, 64], h, kv, d, "f16", mode=mode, window=window, softcap=softcap)


@pytest.mark.parametrize("lens,h,kv,d,dtype", [([1500, 700], 16, 8, 128, "f16"), ([2100], 8, 1, 64, "bf16"),
                                               ([1030, 3, 600], 4, 1, 256, "f16"), ([999], 64, 1, 32, "f16"),
                                               ([1300], 2, 2, 72, "f16")])
@pytest.mark.parametrize("mode", [0, 1])
def test_packed_long(rk, lens, h, kv, d, dtype, mode):
    note(f"packed long {lens} {h}/{kv} d={d} {dtype} mode={mode}")
    packed_case(rk, sum(lens), lens, h, kv, d, dtype, mode=mode)


@pytest.mark.parametrize("lens,h,kv,d", [([1, 40, 300], 128, 1, 32), ([130, 1], 256, 2, 48), ([90, 3, 17], 300, 300, 32),
                                         ([20, 1], 600, 600, 64)])
def test_packed_widest_groups_and_many_kv_heads(rk, lens, h, kv, d):
    note(f"packed {lens} {h}/{kv} d={d}")
    packed_case(rk, h, lens, h, kv, d, "f16")


def test_empty_batches(rk):
    note("empty batches")
    for plan in (rk.packed_plan([], 4, 2, 64), rk.paged_plan([], [], np.zeros((0, 0), np.int32), 1, 16, 4, 2, 64),
                 rk.paged_plan([0, 0], [0, 9], np.full((2, 1), -1), 1, 16, 4, 2, 64)):
        assert plan.n_tokens == 0
        plan.reserve()
        plan.destroy()


def test_packed_many_short_sequences(rk):
    note("packed, 700 sequences")
    packed_case(rk, 3, [1 + i % 7 for i in range(700)], 4, 2, 64, "f16")


def test_packed_reads_a_fused_projection_where_it_lies(rk):
    """q, k and v as column ranges of wider rows, out wider than its heads, bytes between them untouched."""
    note("packed, strided")
    rng, lens, h, kv, d = np.random.default_rng(5), [40, 130, 7], 6, 2, 80
    toks, w = sum(lens), (h + 2 * kv) * d + 16
    qkv = rows(rng, "bf16", toks, w)
    plan = rk.packed_plan(lens, h, kv, d)
    b, o = upload(rk, qkv, np.full((toks, h * d + 24), FILL, np.uint16))
    ok(rk, rk.lib().rk_attention_packed_dev(plan.ptr, b.ptr, w, b.ptr + 2 * h * d, w, b.ptr + 2 * (h + kv) * d, w, 0.1, 0.0,
                                            o.ptr, h * d + 24, rk.DTYPE_BF16, None))
    rk.synchronize()
    got = o.download((toks, h * d + 24), np.uint16)
    assert (got[:, h * d:] == FILL).all()
    q, k, v = qkv[:, :h * d], qkv[:, h * d:(h + kv) * d], qkv[:, (h + kv) * d:(h + 2 * kv) * d]
    check_packed(got[:, :h * d], q, k, v, lens, h, kv, d, "bf16", 0.1)


@pytest.mark.parametrize("lens,h,kv,d", [([1500], 8, 1, 64), ([5, 1, 700, *[1] * 300], 16, 4, 128), ([900, 40], 3, 1, 256),
                                         ([20, 300], 4, 4, 72)])
def test_packed_onto_the_queries(rk, lens, h, kv, d):
    """out on q itself: the split tiles too read all of their queries before a row is stored."""
    note(f"packed in place {h}/{kv} d={d}")
    rng, toks = np.random.default_rng(d), sum(lens)
    q, k, v = (rows(rng, "f16", toks, n * d) for n in (h, kv, kv))
    want = packed(rk, q, k, v, lens, h, kv, d, "f16", 0.1)
    plan, b = rk.packed_plan(lens, h, kv, d), upload(rk, q, k, v)
    ok(rk, rk.lib().rk_attention_packed_dev(plan.ptr, b[0].ptr, h * d, b[1].ptr, kv * d, b[2].ptr, kv * d, 0.1, 0.0, b[0].ptr, h * d,
                                            rk.DTYPE_F16, None))
    rk.synchronize()
    assert (b[0].download(want.shape, np.uint16) == want).all()


def test_packed_large_and_rising_scores(rk):
    """Scores in the hundreds that rise along the keys, and one key that outweighs the others."""
    note("packed, rising scores")
    rng, n, h, kv, d = np.random.default_rng(7), 1900, 4, 1, 128
    q, v = rows(rng, "f16", n, h * d), rows(rng, "f16", n, kv * d)
    k = ref.encode(rng.standard_normal((n, kv * d)) * np.linspace(0.1, 6, n)[:, None], "f16")
    for lens in ([n - more, *[1] * more] for more in (0, crowd(h, kv))):
        for mode in (0, 1):
            check_packed(packed(rk, q, k, v, lens, h, kv, d, "f16", 1.0, mode=mode), q, k, v, lens, h, kv, d, "f16", 1.0, mode=mode)


@pytest.mark.parametrize("many", [False, True])
def test_packed_hidden_keys_that_are_not_finite(rk, many):
    """NaN and infinities in keys that a row does not see leave its scores alone; a value that no row of the
    sequence's other tiles sees does not reach them."""
    note("packed, NaN in hidden keys")
    rng, n, h, kv, d = np.random.default_rng(8), 300, 2, 1, 64
    lens = [n, *[1] * crowd(h, kv) * many]
    q, k, v = (rows(rng, "f16", sum(lens), m * d) for m in (h, kv, kv))
    bad = k.copy()
    bad[290] = 0x7E00  # NaN
    bad[295] = 0x7C00  # infinity
    got = packed(rk, q, bad, v, lens, h, kv, d, "f16", d ** -0.5)
    want = packed(rk, q, k, v, lens, h, kv, d, "f16", d ** -0.5)
    assert (got[:290] == want[:290]).all() and (got[n:] == want[n:]).all()
    # a NaN value beyond the window of every row of the first tiles
    badv = v.copy()
    badv[299] = 0x7E00
    got = packed(rk, q, k, badv, lens, h, kv, d, "f16", d ** -0.5, mode=2, window=20)
    want = packed(rk, q, k, v, lens, h, kv, d, "f16", d ** -0.5, mode=2, window=20)
    assert (got[:128] == want[:128]).all() and (got[n:] == want[n:]).all()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("scale,softcap", [(0.0, 0.0), (-0.2, 0.0), (-0.2, 8.0), (0.0, 8.0)])
def test_packed_scales_of_zero_and_below(rk, scale, softcap, many):
    note(f"packed, scale {scale} softcap {softcap}")
    rng, h, kv, d = np.random.default_rng(9), 4, 2, 96
    lens = [170, 20, *[1] * crowd(h, kv) * many]
    q, k, v = (rows(rng, "bf16", sum(lens), m * d) for m in (h, kv, kv))
    got = packed(rk, q, k, v, lens, h, kv, d, "bf16", scale, softcap)
    check_packed(got, q, k, v, lens, h, kv, d, "bf16", scale, softcap)


# ------------------------------------------------------------------- paged ----
def paged_inputs(seed, kv_lens, ps, h, kv, d, dtype, q_lens, fill=None):
    rng = np.random.default_rng(seed)
    pg = ref.Pages(rng, kv_lens, ps)
    shape = (pg.n_pages, kv, ps, d)
    caches = []
    keys = []
    for _ in range(2):
        c = np.full(shape, 0x7E00 if dtype == "f16" else 0x7FC0, np.uint16)  # every unused slot holds NaN
        ks = [rows(rng, dtype, n, kv, d) for n in kv_lens]
        for i, x in enumerate(ks):
            pg.put(c, i, x)
        caches.append(c)
        keys.append(ks)
    return pg, caches, keys, rows(rng, dtype, sum(q_lens), h * d)


def paged(rk, pg, caches, q, q_lens, kv_lens, h, kv, d, dtype, scale, softcap=0.0, mode=1, window=-1, plan=None, stream=None):
    plan = plan or rk.paged_plan(q_lens, kv_lens, pg.table, pg.n_pages, pg.ps, h, kv, d, mode, window)
    b = upload(rk, q, *caches, np.full((len(q) + 2, h * d), FILL, np.uint16))
    ok(rk, rk.lib().rk_attention_paged_dev(plan.ptr, b[0].ptr, h * d, b[1].ptr, b[2].ptr, scale, softcap, b[3].ptr, h * d,
                                           dt(rk, dtype), stream))
    rk.synchronize(stream)
    got = b[3].download((len(q) + 2, h * d), np.uint16)
    assert (got[len(q):] == FILL).all()
    return got[:len(q)]


def check_paged(got, keys, q, q_lens, kv_lens, h, kv, d, dtype, scale, softcap=0.0, mode=1, window=-1):
    at = 0
    for i, (n, m) in enumerate(zip(q_lens, kv_lens)):
        if n:
            qs = ref.decode(q[at:at + n], dtype).reshape(n, h, d)
            ks, vs = (ref.decode(t[i], dtype) for t in keys)
            want, bound = ref.attention(qs, ks, vs, np.arange(m - n, m), scale, softcap, mode, window, ref.HALF[dtype])
            ref.close(ref.decode(got[at:at + n], dtype).reshape(n, h, d), want, bound, f"sequence {i}: {n} of {m}")
        at += n


def paged_case(rk, seed, q_lens, kv_lens, ps, h, kv, d, dtype, **kw):
    one_paged_case(rk, seed, q_lens, kv_lens, ps, h, kv, d, dtype, 0, **kw)
    if max(q_lens) * (h // kv) > 16:
        one_paged_case(rk, seed, q_lens, kv_lens, ps, h, kv, d, dtype, crowd(h, kv), **kw)


def one_paged_case(rk, seed, q_lens, kv_lens, ps, h, kv, d, dtype, more, **kw):
    """`more` sequences of one token with two keys, all in one page that they share."""
    q_lens, kv_lens = [*q_lens, *[1] * more], [*kv_lens, *[2] * min(more, 1)]
    pg, caches, keys, q = paged_inputs(seed, kv_lens, ps, h, kv, d, dtype, q_lens)
    if more:
        kv_lens += [2] * (more - 1)
        pg.table = np.concatenate([pg.table, np.repeat(pg.table[-1:], more - 1, axis=0)])
        for t in keys:
            t += t[-1:] * (more - 1)
    got = paged(rk, pg, caches, q, q_lens, kv_lens, h, kv, d, dtype, d ** -0.5, **kw)
    check_paged(got, keys, q, q_lens, kv_lens, h, kv, d, dtype, d ** -0.5, **kw)
    assert (paged(rk, pg, caches, q, q_lens, kv_lens, h, kv, d, dtype, d ** -0.5, **kw) == got).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("q_lens,kv_lens,ps,h,kv", [([1, 0, 1, 1], [1, 40, 16, 129], 16, 4, 2),
                                                    ([1, 37, 5], [700, 300, 5], 64, 8, 1),
                                                    ([3], [2050], 32, 6, 2)])
def test_paged_head_dims(rk, d, dtype, q_lens, kv_lens, ps, h, kv):
    note(f"paged d={d} {dtype} {q_lens} of {kv_lens} pages of {ps} {h}/{kv}")
    paged_case(rk, d + ps, q_lens, kv_lens, ps, h, kv, d, dtype)


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("h,kv,d", [(8, 2, 128), (2, 2, 80), (71, 1, 64)])
def test_paged_page_sizes_and_edges(rk, ps, h, kv, d):
    """Keys that end before, at and behind the ends of pages and of the kernels' steps; one token and chunks."""
    note(f"paged pages of {ps} {h}/{kv} d={d}")
    kv_lens = [1, ps - 1, ps, ps + 1, 63, 64, 65, 255, 256, 257, 3 * ps + 7]
    q_lens = [1] * len(kv_lens)
    paged_case(rk, ps, q_lens, kv_lens, ps, h, kv, d, "f16")
    paged_case(rk, ps + 1, [min(n, 1 + 13 * i) for i, n in enumerate(kv_lens)], kv_lens, ps, h, kv, d, "f16")


@pytest.mark.parametrize("mode,window,softcap", [(0, -1, 0.0), (1, -1, 30.0), (2, 40, 0.0), (2, 300, 10.0), (3, 1, 0.0),
                                                 (3, 100, 0.0), (3, 257, 20.0), (3, 0, 0.0)])
@pytest.mark.parametrize("h,kv,d", [(6, 2, 64), (16, 2, 128), (3, 1, 256)])
def test_paged_masks(rk, mode, window, softcap, h, kv, d):
    note(f"paged masks mode={mode} window={window} softcap={softcap} {h}/{kv} d={d}")
    paged_case(rk, mode + window + 1, [1, 70, 2, 150], [900, 600, 2, 150], 32, h, kv, d, "f16", mode=mode, window=window,
               softcap=softcap)


@pytest.mark.parametrize("q_lens,kv_lens,ps,h,kv,d,dtype", [
    ([1], [9001], 16, 32, 4, 128, "f16"), ([1], [20011], 64, 8, 8, 64, "bf16"), ([1, 1, 1], [6000, 33, 12345], 128, 4, 1, 256, "f16"),
    ([1], [40003], 64, 4, 1, 64, "f16"), ([64], [5000], 64, 8, 2, 128, "f16"), ([300], [3000], 16, 4, 4, 96, "f16"), ([200, 1, 1, 1], [2500, 2000, 70, 4100], 32, 16, 4, 64, "bf16")])
def test_paged_long(rk, q_lens, kv_lens, ps, h, kv, d, dtype):
    note(f"paged long {q_lens} of {kv_lens}")
    paged_case(rk, sum(kv_lens), q_lens, kv_lens, ps, h, kv, d, dtype)


def test_paged_many_sequences(rk):
    note("paged, 300 sequences of one token")
    kv_lens = [1 + (37 * i) % 500 for i in range(300)]
    paged_case(rk, 9, [1] * 300, kv_lens, 16, 4, 2, 64, "f16")


def test_paged_pages_behind_the_window_need_not_exist(rk):
    note("paged, dropped pages")
    h, kv, d, ps, w = 4, 2, 64, 16, 50
    q_lens, kv_lens = [1, 20], [400, 333]
    pg, caches, keys, q = paged_inputs(2, kv_lens, ps, h, kv, d, "f16", q_lens)
    for i, (n, m) in enumerate(zip(q_lens, kv_lens)):
        gone = (m - n - w + 1) // ps  # pages that end before the first token's window
        for c in caches:
            c[pg.table[i, :gone]] = 0x7E00
        pg.table[i, :gone] = -12345
    got = paged(rk, pg, caches, q, q_lens, kv_lens, h, kv, d, "f16", 0.125, mode=3, window=w)
    check_paged(got, keys, q, q_lens, kv_lens, h, kv, d, "f16", 0.125, mode=3, window=w)


def test_paged_sequences_share_a_prefix(rk):
    note("paged, shared pages")
    h, kv, d, ps = 8, 2, 128, 16
    pg, caches, keys, q = paged_inputs(4, [160, 16], ps, h, kv, d, "f16", [1, 1])
    table = np.concatenate([pg.table[:1, :10], pg.table[:1, :10]])
    table[1, 9] = pg.table[1, 0]
    pg.table = table
    for t in keys:
        t[1] = np.concatenate([t[0][:144], t[1]])
    got = paged(rk, pg, caches, q, [1, 1], [160, 160], h, kv, d, "f16", 0.1)
    check_paged(got, keys, q, [1, 1], [160, 160], h, kv, d, "f16", 0.1)


def test_paged_cache_past_32_bit_offsets(rk):
    """Pages that lie more than 4 GiB into the cache."""
    note("paged, 5 GiB caches")
    h, kv, d, ps, n_pages = 8, 8, 128, 16, 160000
    q_lens, kv_lens = [1, 40], [300, 90]
    pg, caches, keys, q = paged_inputs(6, kv_lens, ps, h, kv, d, "f16", q_lens)
    page = kv * ps * d * 2
    big = [rk.DeviceBuffer(n_pages * page) for _ in range(2)]
    far = pg.table + (n_pages - pg.n_pages)
    lib = rk.lib()
    for b, c in zip(big, caches):
        c = np.ascontiguousarray(c)
        ok(rk, lib.rk_memcpy_htod(ctypes.c_void_p(b.ptr + (n_pages - pg.n_pages) * page), c.ctypes.data, c.nbytes))
    plan = rk.paged_plan(q_lens, kv_lens, np.where(pg.table < 0, -1, far), n_pages, ps, h, kv, d)
    dq, o = upload(rk, q, np.zeros((len(q), h * d), np.uint16))
    ok(rk, lib.rk_attention_paged_dev(plan.ptr, dq.ptr, h * d, big[0].ptr, big[1].ptr, 0.1, 0.0, o.ptr, h * d, rk.DTYPE_F16, None))
    rk.synchronize()
    check_paged(o.download((len(q), h * d), np.uint16), keys, q, q_lens, kv_lens, h, kv, d, "f16", 0.1)
    # the append writes there too
    rng = np.random.default_rng(1)
    x = rows(rng, "f16", len(q), (h + 2 * kv) * d)
    cs = [np.ones((400, d // 2), np.float32), np.zeros((400, d // 2), np.float32)]
    bx, bc, bs = upload(rk, x, *cs)
    ok(rk, lib.rk_paged_append_dev(plan.ptr, bx.ptr, (h + 2 * kv) * d, None, None, 1e-6, bc.ptr, bs.ptr, rk.DTYPE_F32, 400, o.ptr,
                                   h * d, big[0].ptr, big[1].ptr, rk.DTYPE_F16, None))
    rk.synchronize()
    back = np.empty(caches[0].shape, np.uint16)
    for b, c, part in zip(big, caches, (x[:, h * d:(h + kv) * d], x[:, (h + kv) * d:])):
        ok(rk, lib.rk_memcpy_dtoh(back.ctypes.data, ctypes.c_void_p(b.ptr + (n_pages - pg.n_pages) * page), back.nbytes))
        want, at = c.copy(), 0
        for i, (n, m) in enumerate(zip(q_lens, kv_lens)):
            for t in range(m - n, m):
                want[pg.table[i, t // ps], :, t % ps] = part[at].reshape(kv, d)
                at += 1
        assert (back == want).all()


# ------------------------------------------------------------------ append ----
def append_case(rk, seed, q_lens, kv_lens, ps, h, kv, d, dtype, norm, tables, in_place=False, pad=0):
    rng = np.random.default_rng(seed)
    pg = ref.Pages(rng, kv_lens, ps)
    toks, w, n_pos = sum(q_lens), (h + 2 * kv) * d + pad, max(kv_lens) + 2
    x = rows(rng, dtype, toks + 2, w, scale=1.5)
    shape = (pg.n_pages, kv, ps, d)
    caches = [rows(rng, dtype, *shape) for _ in range(2)]
    norms = [rows(rng, dtype, d) for _ in range(2)] if norm else []
    ang = rng.uniform(-np.pi, np.pi, (n_pos, d // 2))
    cs = [np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)]
    if tables != "f32":
        cs = [ref.encode(c, tables) for c in cs]
    plan = rk.paged_plan(q_lens, kv_lens, pg.table, pg.n_pages, ps, h, kv, d)
    bx, bk, bv, bc, bs, bo = upload(rk, x, *caches, *cs, np.full((toks + 2, h * d), FILL, np.uint16))
    bw = upload(rk, *norms)
    out, stride = (bx.ptr, w) if in_place else (bo.ptr, h * d)
    types = {"f32": rk.DTYPE_F32, "f16": rk.DTYPE_F16, "bf16": rk.DTYPE_BF16}
    ok(rk, rk.lib().rk_paged_append_dev(plan.ptr, bx.ptr, w, *([b.ptr for b in bw] or [None, None]), 1e-5, bc.ptr, bs.ptr,
                                        types[tables], n_pos, out, stride, bk.ptr, bv.ptr, types[dtype], None))
    rk.synchronize()
    after = bx.download(x.shape, np.uint16)
    got_q = after if in_place else bo.download((toks + 2, h * d), np.uint16)
    if in_place:
        assert (after[:, h * d:] == x[:, h * d:]).all() and (after[toks:] == x[toks:]).all()
    else:
        assert (after == x).all() and (got_q[toks:] == FILL).all()
    got_q = got_q[:toks, :h * d]
    got = [b.download(shape, np.uint16) for b in (bk, bv)]
    pos = np.concatenate([np.arange(m - n, m) for n, m in zip(q_lens, kv_lens)]).astype(int)
    seq = np.repeat(np.arange(len(q_lens)), q_lens)
    c64, s64 = ((t.astype(np.float64) if tables == "f32" else ref.decode(t, tables))[pos] for t in cs)
    x64 = ref.decode(x[:toks, :(h + 2 * kv) * d], dtype).reshape(toks, h + 2 * kv, d)
    nw = [ref.decode(n, dtype) for n in norms] or [None, None]
    want, bound = ref.prologue(x64[:, :h], nw[0], c64, s64, 1e-5, ref.HALF[dtype])
    ref.close(ref.decode(got_q, dtype).reshape(toks, h, d), want, bound, "q")
    want, bound = ref.prologue(x64[:, h:h + kv], nw[1], c64, s64, 1e-5, ref.HALF[dtype])
    page, off = pg.table[seq, pos // ps], pos % ps
    ref.close(ref.decode(got[0][page, :, off], dtype), want, bound, "k")
    assert (got[1][page, :, off] == x[:toks].reshape(toks, -1)[:, (h + kv) * d:(h + 2 * kv) * d].reshape(toks, kv, d)).all()
    for g, c in zip(got, caches):  # every other slot is as it was
        c = c.copy()
        c[page, :, off] = g[page, :, off]
        assert (g == c).all()


@pytest.mark.parametrize("d", DIMS)
@pytest.mark.parametrize("dtype,norm,tables", [("f16", True, "f16"), ("f16", False, "f32"), ("bf16", True, "f32"),
                                               ("bf16", False, "bf16")])
def test_append(rk, d, dtype, norm, tables):
    note(f"append d={d} {dtype} norm={norm} tables {tables}")
    append_case(rk, d, [1, 0, 33, 5, 1], [1, 20, 50, 5, 300], 16, 4, 2, d, dtype, norm, tables)


@pytest.mark.parametrize("ps", [16, 64, 256])
def test_append_in_place_and_strided(rk, ps):
    note(f"append in place, pages of {ps}")
    append_case(rk, ps, [700, 1, 90], [1000, 257, 90], ps, 16, 8, 128, "f16", True, "f32", in_place=True, pad=24)
    append_case(rk, ps, [3, 3], [ps + 1, 2 * ps], ps, 3, 1, 256, "bf16", True, "f32", pad=8)
    append_case(rk, ps, [1] * 65, list(range(1, 66)), ps, 7, 1, 72, "f16", True, "f16", in_place=True)


# ---------------------------------------------------------------- together ----
def test_a_prompt_in_chunks_then_tokens_equals_the_packed_prompt(rk):
    """Two prompts in chunks of different sizes, then a few tokens each, through append and paged attention: every
    row's result is that of attention over the whole sequences, packed."""
    note("append + paged attention against packed")
    rng, h, kv, d, ps = np.random.default_rng(11), 8, 2, 64, 32
    total = [207, 90]
    steps = [(100, 40), (64, 0), (40, 47), (1, 1), (1, 1), (1, 1)]
    assert [sum(s[i] for s in steps) for i in (0, 1)] == total
    ang = np.arange(256)[:, None] * 10000.0 ** (-np.arange(d // 2) / (d // 2))
    cos, sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
    qkv = [rows(rng, "f16", n, (h + 2 * kv) * d) for n in total]
    qw, kw = (rows(rng, "f16", d) for _ in range(2))
    f16 = lambda a: a.view(np.float16)  # noqa: E731
    pg = ref.Pages(rng, total, ps)
    cache = rk.PagedCache(pg.n_pages, ps, kv, d)
    done, outs, qs = [0, 0], [[], []], [[], []]
    for step in steps:
        lens = [a + b for a, b in zip(done, step)]
        plan = cache.plan(step, lens, pg.table, h)
        x = np.concatenate([qkv[i][done[i]:lens[i]] for i in (0, 1)])
        q = cache.append(plan, f16(x), cos, sin, f16(qw), f16(kw))
        o = cache.attention(plan, q, d ** -0.5)
        for i, (a, b) in enumerate(((0, step[0]), (step[0], step[0] + step[1]))):
            outs[i].append(o[a:b].view(np.uint16))
            qs[i].append(q[a:b].view(np.uint16))
        done = lens
    k, v = (b.download((pg.n_pages, kv, ps, d), np.uint16) for b in (cache.k, cache.v))
    keys = [[c[pg.table[i, np.arange(n) // ps], :, np.arange(n) % ps].reshape(n, kv * d) for i, n in enumerate(total)] for c in (k, v)]
    q, k, v = np.concatenate([np.concatenate(x) for x in qs]), np.concatenate(keys[0]), np.concatenate(keys[1])
    whole = rk.attention_packed(f16(q), f16(k), f16(v), total, h, kv, d, d ** -0.5)
    check_packed(np.concatenate([np.concatenate(x) for x in outs]), q, k, v, total, h, kv, d, "f16", d ** -0.5)
    check_packed(whole.view(np.uint16), q, k, v, total, h, kv, d, "f16", d ** -0.5)


def test_one_sequence_agrees_with_the_single_sequence_attention(rk):
    note("packed against rk_attention_dev")
    rng, n, h, kv, d = np.random.default_rng(12), 700, 8, 2, 128
    q, k, v = (rows(rng, "f16", n, m * d) for m in (h, kv, kv))
    b = upload(rk, q, k, v, np.zeros((n, h * d), np.uint16))
    ok(rk, rk.lib().rk_attention_dev(b[0].ptr, b[1].ptr, b[2].ptr, n, n, h, kv, d, 0.1, 0.0, 3, 0, 0, 0, b[3].ptr, None))
    rk.synchronize()
    want = b[3].download((n, h * d), np.uint16)
    got = packed(rk, q, k, v, [n], h, kv, d, "f16", 0.1, mode=3, window=0)  # no key visible: the mean of V
    a, w = ref.decode(got, "f16"), ref.decode(want, "f16")
    assert np.abs(a - w).max() <= 2 * (2.0 ** -11 * np.abs(w).max() + 2.0 ** -11 * np.abs(ref.decode(v, "f16")).mean() * 4)


# --------------------------------------------------------- plans and streams ----
def test_plan_update_serves_the_next_step(rk):
    note("plan update")
    h, kv, d, ps = 4, 2, 64, 16
    pg, caches, keys, q = paged_inputs(20, [600, 41, 500], ps, h, kv, d, "f16", [1, 1, 1])
    plan = rk.paged_plan([1, 1], [5, 41], pg.table[:2], pg.n_pages, ps, h, kv, d)
    for q_lens, kv_lens in (([1, 1, 1], [600, 41, 500]), ([2, 0, 1], [17, 3, 200]), ([1], [600]), ([], []), ([3, 0, 0], [599, 0, 1])):
        n = len(q_lens)
        if n:
            plan.update(q_lens, kv_lens, pg.table[:n])
        else:
            plan.update([], [], np.zeros((0, 1), np.int32))
        qn = q[:sum(q_lens)]
        if sum(q_lens) == 0:
            continue
        got = paged(rk, pg, caches, qn, q_lens, kv_lens, h, kv, d, "f16", 0.1, plan=plan)
        check_paged(got, [[t[i][:m] for i, m in enumerate(kv_lens)] for t in keys], qn, q_lens, kv_lens, h, kv, d, "f16", 0.1)
    with pytest.raises(rk.RocketError) as e:  # a bad batch leaves the plan as it was
        plan.update([1], [600], np.full((1, 50), 10**6))
    assert e.value.rc == rk.RK_E_SHAPE
    got = paged(rk, pg, caches, q, [3, 0, 0], [599, 0, 1], h, kv, d, "f16", 0.1, plan=plan)
    check_paged(got, [[t[i][:m] for i, m in enumerate([599, 0, 1])] for t in keys], q, [3, 0, 0], [599, 0, 1], h, kv, d, "f16", 0.1)


def test_one_plan_on_two_streams(rk):
    """Calls and updates from two streams take turns; each sees its own batch."""
    note("two streams")
    h, kv, d, ps = 8, 1, 128, 16
    kv_lens = [5000, 4000]
    pg, caches, keys, q = paged_inputs(21, kv_lens, ps, h, kv, d, "f16", [1, 1])
    plan = rk.paged_plan([1, 1], kv_lens, pg.table, pg.n_pages, ps, h, kv, d)
    want = paged(rk, pg, caches, q, [1, 1], kv_lens, h, kv, d, "f16", 0.1, plan=plan)
    check_paged(want, keys, q, [1, 1], kv_lens, h, kv, d, "f16", 0.1)
    bufs = upload(rk, q, *caches)
    outs = [rk.DeviceBuffer(q.nbytes) for _ in range(6)]
    sts = [rk.new_stream(), rk.new_stream()]
    for i, o in enumerate(outs):
        st = sts[i % 2]
        plan.update([1, 1], kv_lens, pg.table, stream=st)
        ok(rk, rk.lib().rk_attention_paged_dev(plan.ptr, bufs[0].ptr, h * d, bufs[1].ptr, bufs[2].ptr, 0.1, 0.0, o.ptr, h * d,
                                               rk.DTYPE_F16, st))
    for st in sts:
        rk.synchronize(st)
        rk.destroy_stream(st)
    for o in outs:
        assert (o.download(q.shape, np.uint16) == want).all()
    plan.destroy()


def test_refusals_on_the_device_side(rk):
    note("refusals")
    lib, h, kv, d = rk.lib(), 4, 2, 64
    a, p = rk.packed_plan([4, 5], h, kv, d), rk.paged_plan([1], [20], np.array([[1, 2]]), 4, 16, h, kv, d)
    b = rk.DeviceBuffer(1 << 16)
    x = b.ptr

    def pk(plan=a.ptr, q=x, qs=256, k=x, ks=128, v=x, vs=128, o=x, os_=256, dtype=1):
        return lib.rk_attention_packed_dev(plan, q, qs, k, ks, v, vs, 0.1, 0.0, o, os_, dtype, None)

    def pa(plan=p.ptr, q=x, qs=256, k=x, v=x, o=x, os_=256, dtype=1):
        return lib.rk_attention_paged_dev(plan, q, qs, k, v, 0.1, 0.0, o, os_, dtype, None)

    def ap(plan=p.ptr, qkv=x, rs=512, qw=None, kw=None, c=x, s=x, ct=0, n=20, o=x + 8192, os_=256, k=x, v=x, dtype=1):
        return lib.rk_paged_append_dev(plan, qkv, rs, qw, kw, 1e-6, c, s, ct, n, o, os_, k, v, dtype, None)

    for rc in (pk(plan=None), pk(plan=x), pk(plan=p.ptr), pa(plan=a.ptr), ap(plan=a.ptr), pk(q=None), pk(qs=255), pk(qs=248), pk(qs=260),
               pk(ks=120), pk(vs=0), pk(o=None), pk(o=x + 8), pk(k=x + 2), pa(q=None), pa(k=None), pa(v=x + 4), pa(os_=128),
               ap(qkv=None), ap(rs=504), ap(rs=516), ap(qw=x), ap(kw=x), ap(c=None), ap(s=x + 4), ap(n=19), ap(o=None), ap(os_=248),
               ap(o=x, os_=256), ap(k=None), ap(v=x + 2), ap(qw=x + 2, kw=x)):
        assert rc == rk.RK_E_SHAPE, lib.rk_last_error()
    for rc in (pk(dtype=0), pa(dtype=7), ap(dtype=0), ap(ct=2)):
        assert rc == rk.RK_E_UNSUPPORTED
    # two sequences whose new tokens share a slot may be read, not appended
    two = rk.paged_plan([2, 1], [18, 17], np.array([[1, 2], [3, 2]]), 4, 16, h, kv, d)
    assert ap(plan=two.ptr) == rk.RK_E_SHAPE and b"slot" in lib.rk_last_error()
    dead = two.ptr
    two.destroy()
    assert pa(plan=dead) == rk.RK_E_SHAPE and lib.rk_seq_plan_destroy(dead) == rk.RK_E_SHAPE
    # batches without a token: nothing to do, whatever the buffers
    none = rk.packed_plan([0, 0], h, kv, d)
    assert pk(plan=none.ptr, q=None) == 0 and lib.rk_seq_plan_destroy(None) == 0


class Graph:
    """A captured step on a stream, through the HIP runtime that the library is linked with."""

    def __init__(self, st, step):
        with open("/proc/self/maps") as f:
            self.hip = ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))
        self.graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        self.st = ctypes.c_void_p(st)
        assert self.hip.hipStreamBeginCapture(self.st, 2) == 0  # relaxed: only this stream is looked at
        try:
            step()
        finally:
            rc = self.hip.hipStreamEndCapture(self.st, ctypes.byref(self.graph))
        assert rc == 0
        assert self.hip.hipGraphInstantiate(ctypes.byref(self.exec), self.graph, None, None, ctypes.c_size_t(0)) == 0

    def replay(self):
        assert self.hip.hipGraphLaunch(self.exec, self.st) == 0

    def destroy(self):
        assert self.hip.hipGraphExecDestroy(self.exec) == 0 and self.hip.hipGraphDestroy(self.graph) == 0


def test_captured_step_replays_with_updates(rk):
    """Append and attention in one graph, replayed on later steps of a batch that shrinks and grows again."""
    note("graph capture")
    h, kv, d, ps, n_pos = 16, 2, 64, 16, 4096
    rng = np.random.default_rng(30)
    pg = ref.Pages(rng, [3000, 900, 64], ps)
    shape, xs = (pg.n_pages, kv, ps, d), (4, (h + 2 * kv) * d)
    now = [rows(rng, "f16", *shape) for _ in range(2)]  # what the caches hold
    ang = rng.uniform(-3, 3, (n_pos, d // 2))
    cos, sin = upload(rk, *(f(ang).astype(np.float32) for f in (np.cos, np.sin)))
    filled = np.full((4, h * d), FILL, np.uint16)
    mine, other = ([*upload(rk, *now, np.zeros(xs, np.uint16), filled, filled)] for _ in range(2))
    lib, st = rk.lib(), rk.new_stream()

    def step(plan, k, v, x, q, o):
        ok(rk, lib.rk_paged_append_dev(plan.ptr, x.ptr, xs[1], None, None, 1e-6, cos.ptr, sin.ptr, rk.DTYPE_F32, n_pos, q.ptr, h * d,
                                       k.ptr, v.ptr, rk.DTYPE_F16, st))
        ok(rk, lib.rk_attention_paged_dev(plan.ptr, q.ptr, h * d, k.ptr, v.ptr, 0.1, 0.0, o.ptr, h * d, rk.DTYPE_F16, st))

    plan = rk.paged_plan([2, 1, 1], [3000, 900, 64], pg.table, pg.n_pages, ps, h, kv, d)
    refused = []
    Graph(st, lambda: refused.append(lib.rk_attention_paged_dev(plan.ptr, mine[3].ptr, h * d, mine[0].ptr, mine[1].ptr, 0.1, 0.0,
                                                                mine[4].ptr, h * d, rk.DTYPE_F16, st))).destroy()
    assert refused == [rk.RK_E_UNSUPPORTED]  # nothing is reserved yet
    plan.reserve(4)
    g = Graph(st, lambda: step(plan, *mine))
    batches = [([2, 1, 1], [3000, 900, 64]), ([1], [1234]), ([1, 1, 1], [2048, 16, 60]), ([2, 2], [500, 899]), ([4], [3000]),
               ([1, 0, 1], [2999, 5, 1])]
    for i, (q_lens, kv_lens) in enumerate(batches):
        n, x = sum(q_lens), rows(rng, "f16", *xs)
        table = pg.table[:len(q_lens)]
        # eager, on buffers and with a plan of their own
        for b, a in zip(other, (*now, x, filled, filled)):
            b.upload(a)
        eager = rk.paged_plan(q_lens, kv_lens, table, pg.n_pages, ps, h, kv, d)
        step(eager, *other)
        rk.synchronize(st)
        want = [b.download(a.shape, np.uint16) for b, a in zip(other, (*now, x, filled, filled))]
        keys = [[c[table[s, np.arange(m) // ps], :, np.arange(m) % ps] for s, m in enumerate(kv_lens)] for c in want[:2]]
        outs = [want.pop()]
        for _ in range(3):
            for b, a in zip(mine, (*now, x, filled, filled)):
                b.upload(a)
            plan.update(q_lens, kv_lens, table, stream=st)
            g.replay()
            rk.synchronize(st)
            for b, w in zip(mine, want):
                assert (b.download(w.shape, np.uint16) == w).all(), f"batch {i}"
            outs.append(mine[4].download(filled.shape, np.uint16))
        for o in outs:
            assert (o[n:] == FILL).all()
            check_paged(o[:n], keys, want[3][:n], q_lens, kv_lens, h, kv, d, "f16", 0.1)
        assert all((o == outs[1]).all() for o in outs[2:]), f"batch {i}"
        now = want[:2]
    with pytest.raises(rk.RocketError):  # five tokens: more than the graph has room for
        plan.update([2, 2, 1], [10, 10, 10], pg.table, stream=st)
    with pytest.raises(rk.RocketError):  # a longer chunk than was reserved for
        plan.update([5], [10], pg.table[:1], stream=st)
    with pytest.raises(rk.RocketError):  # past the tables that the graph reads
        plan.update([1], [4097], np.zeros((1, 300), np.int32), stream=st)
    g.destroy()
    plan.destroy()
    rk.destroy_stream(st)


@pytest.mark.parametrize("d", [128, 256])
def test_captured_packed_batches_of_both_kinds(rk, d):
    """One graph, replayed on batches that are small, that have long sequences among many short ones, and empty."""
    note(f"graph capture, packed, d={d}")
    h, kv, n = 8, 2, 1200
    rng, lib, st = np.random.default_rng(31), rk.lib(), rk.new_stream()
    q, k, v = (rows(rng, "bf16", n, m * d) for m in (h, kv, kv))
    filled = np.full((n, h * d), FILL, np.uint16)
    b = upload(rk, q, k, v, filled)
    plan = rk.packed_plan([2] * 600, h, kv, d)
    plan.reserve(500)
    g = Graph(st, lambda: ok(rk, lib.rk_attention_packed_dev(plan.ptr, b[0].ptr, h * d, b[1].ptr, kv * d, b[2].ptr, kv * d, 0.1, 0.0,
                                                             b[3].ptr, h * d, rk.DTYPE_BF16, st)))
    for lens in ([2] * 600, [500, 3, 77], [400, *[1] * 520], [0, 0], [500, 200, *[1] * 500], [1]):
        plan.update(lens, stream=st)
        seen = []
        for _ in range(3):
            b[3].upload(filled)
            g.replay()
            rk.synchronize(st)
            seen.append(b[3].download(filled.shape, np.uint16))
        t = sum(lens)
        assert all((o == seen[0]).all() for o in seen) and (seen[0][t:] == FILL).all()
        check_packed(seen[0][:t], q, k, v, lens, h, kv, d, "bf16", 0.1)
    g.destroy()
    plan.destroy()
    rk.destroy_stream(st)


@pytest.mark.parametrize("h,kv,d,max_q", [(8, 2, 128, 1), (8, 2, 64, 40), (4, 4, 256, 400), (64, 1, 32, 64), (48, 48, 80, 7)])
def test_a_reserved_plan_has_room_for_every_smaller_batch(rk, h, kv, d, max_q):
    """A plan that a graph holds takes any batch of no more sequences, tokens and pages, short or long, few or many."""
    note(f"reserve {h}/{kv} d={d} q_len {max_q}")
    rng, ps, n_seqs, toks, n_pages = np.random.default_rng(d), 64, 40, 900, 4000
    q = [max_q] * (toks // max_q) if max_q > 22 else [max_q] * n_seqs
    q += [0] * (n_seqs - len(q))
    toks = sum(q)
    table = np.arange(n_seqs * 100, dtype=np.int32).reshape(n_seqs, 100)
    plan, st = rk.paged_plan(q, [6400 if x else 0 for x in q], table, n_pages, ps, h, kv, d), rk.new_stream()
    pages = 100 * sum(x > 0 for x in q)
    plan.reserve(max_q)
    (buf,) = upload(rk, np.zeros(64, np.uint16))  # (the graph is not launched)
    g = Graph(st, lambda: ok(rk, rk.lib().rk_attention_paged_dev(plan.ptr, buf.ptr, h * d, buf.ptr, buf.ptr, 0.1, 0.0, buf.ptr, h * d,
                                                                 rk.DTYPE_F16, st)))
    for i in range(150):
        n = int(rng.integers(1, n_seqs + 1))
        left, held, ql, kl = toks, pages, [], []
        for _ in range(n):
            x = int(min(left, max_q, rng.choice([1, max_q, int(rng.integers(0, max_q + 1))])))
            m = int(min(6400, held * ps, max(x, rng.choice([x, 100, 6400, int(rng.integers(1, 6401))])))) if x else 0
            x = min(x, m)
            left, held, ql, kl = left - x, held - -(-m // ps), [*ql, x], [*kl, m]
        plan.update(ql, kl, table[:n], stream=st)
    rk.synchronize(st)
    g.destroy()
    plan.destroy()
    rk.destroy_stream(st)


def test_an_update_inside_a_capture_is_refused(rk):
    note("update in a capture")
    plan, st, seen = rk.packed_plan([4], 4, 2, 64), rk.new_stream(), []

    def step():
        with pytest.raises(rk.RocketError) as e:
            plan.update([3], stream=st)
        seen.append(e.value.rc)

    Graph(st, step).destroy()
    assert seen == [rk.RK_E_UNSUPPORTED]
    rk.destroy_stream(st)


def test_numpy_helpers(rk):
    note("numpy helpers")
    rng, h, kv, d = np.random.default_rng(40), 4, 2, 64
    q, k, v = (rows(rng, "bf16", 9, n * d) for n in (h, kv, kv))
    got = rk.attention_packed(q, k, v, [4, 5], h, kv, d, 0.125, bf16=True)
    check_packed(got, q, k, v, [4, 5], h, kv, d, "bf16", 0.125)
    assert rk.attention_packed(q[:0], k[:0], v[:0], [0], h, kv, d, 0.125, bf16=True).shape == (0, h * d)
    cache = rk.PagedCache(4, 16, kv, d)
    plan = cache.plan([1], [3], np.array([[1]]), h)
    with pytest.raises(rk.RocketError):
        cache.attention(plan, np.zeros((2, h * d), np.float16), 0.1)
    other = rk.paged_plan([1], [3], np.array([[1]]), 4, 32, h, kv, d)
    with pytest.raises(rk.RocketError):
        cache.attention(other, np.zeros((1, h * d), np.float16), 0.1)


def test_a_captured_call_s_buffers_bound_later_batches(rk):
    """A graph's buffers have room for the tokens at its capture. Room that a plan has beyond that (for splits, or from
    a larger batch before) admits no more."""
    note("tokens of a captured call")
    lib, st, h, kv, d, ps = rk.lib(), rk.new_stream(), 8, 2, 64, 16
    rng = np.random.default_rng(50)
    q, k, v = (rows(rng, "f16", 10, n * d) for n in (h, kv, kv))
    filled = np.full((12, h * d), FILL, np.uint16)
    b = upload(rk, q, k, v, filled)
    plan = rk.packed_plan([4], h, kv, d)
    plan.reserve(1000)  # longer sequences, not more tokens
    g = Graph(st, lambda: ok(rk, lib.rk_attention_packed_dev(plan.ptr, b[0].ptr, h * d, b[1].ptr, kv * d, b[2].ptr, kv * d, 0.1, 0.0,
                                                             b[3].ptr, h * d, rk.DTYPE_F16, st)))
    for lens in ([5], [1000], [2, 3], [1] * 5, [0, 4, 1]):
        with pytest.raises(rk.RocketError) as e:
            plan.update(lens, stream=st)
        assert e.value.rc == rk.RK_E_SHAPE and "tokens" in str(e.value)
    for lens in ([4], [1, 3], [2], [0, 0]):
        plan.update(lens, stream=st)
        b[3].upload(filled)
        g.replay()
        rk.synchronize(st)
        got, t = b[3].download(filled.shape, np.uint16), sum(lens)
        assert (got[t:] == FILL).all()
        check_packed(got[:t], q, k, v, lens, h, kv, d, "f16", 0.1)
    g.destroy()
    plan.destroy()
    # paged: the plan had a larger batch before; the append's tokens count as well
    pg, caches, keys, q = paged_inputs(51, [64, 64], ps, h, kv, d, "f16", [6, 4])
    x = rows(rng, "f16", 10, (h + 2 * kv) * d)
    b = upload(rk, q, *caches, filled, x, np.ones((64, d // 2), np.float32))
    for call in (lambda p: lib.rk_attention_paged_dev(p, b[0].ptr, h * d, b[1].ptr, b[2].ptr, 0.1, 0.0, b[3].ptr, h * d, rk.DTYPE_F16, st),
                 lambda p: lib.rk_paged_append_dev(p, b[4].ptr, (h + 2 * kv) * d, None, None, 1e-6, b[5].ptr, b[5].ptr, rk.DTYPE_F32, 64,
                                                   b[3].ptr, h * d, b[1].ptr, b[2].ptr, rk.DTYPE_F16, st)):
        plan = rk.paged_plan([50, 50], [64, 64], pg.table, pg.n_pages, ps, h, kv, d)
        plan.update([6, 4], [64, 64], pg.table, stream=st)
        plan.reserve(50)
        g = Graph(st, lambda: ok(rk, call(plan.ptr)))
        for lens in ([6, 5], [50, 50], [11, 0]):
            with pytest.raises(rk.RocketError) as e:
                plan.update(lens, [64, 64], pg.table, stream=st)
            assert e.value.rc == rk.RK_E_SHAPE
        plan.update([10, 0], [64, 64], pg.table, stream=st)
        rk.synchronize(st)
        g.destroy()
        plan.destroy()
    rk.destroy_stream(st)


def test_out_on_the_queries_with_another_stride_is_refused(rk):
    note("out on q, another stride")
    lib, b = rk.lib(), rk.DeviceBuffer(1 << 16)
    x, a, p = b.ptr, rk.packed_plan([4, 5], 4, 2, 64), rk.paged_plan([1], [20], np.array([[1, 2]]), 4, 16, 4, 2, 64)
    for qs, os_ in ((256, 264), (512, 256)):
        assert lib.rk_attention_packed_dev(a.ptr, x, qs, x + 16384, 128, x + 16384, 128, 0.1, 0.0, x, os_, rk.DTYPE_F16, None) == rk.RK_E_SHAPE
        assert b"stride" in lib.rk_last_error()
        assert lib.rk_attention_paged_dev(p.ptr, x, qs, x + 16384, x + 16384, 0.1, 0.0, x, os_, rk.DTYPE_F16, None) == rk.RK_E_SHAPE
    assert lib.rk_attention_packed_dev(a.ptr, x, 264, x + 16384, 128, x + 16384, 128, 0.1, 0.0, x, 264, rk.DTYPE_F16, None) == 0
    rk.synchronize()


def tokens_of_a_tile(small, g, d):
    """New tokens of the rows that are computed together."""
    return (16 if small else 128 if d <= 128 else 64) // g


@pytest.mark.parametrize("n,many", [(300, False), (300, True), (2000, True)])
@pytest.mark.parametrize("h,kv,d", [(8, 1, 64), (1, 1, 128), (4, 2, 80), (8, 1, 256)])
def test_values_that_no_row_of_a_tile_sees_do_not_reach_it(rk, n, many, h, kv, d):
    """A NaN or infinity in V just behind the last key that any row of a tile sees, or just before the first one,
    leaves the tile's results as they are, bit for bit."""
    note(f"hidden values, n={n} many={many} {h}/{kv} d={d}")
    rng, tile = np.random.default_rng(60), tokens_of_a_tile(not many, h // kv, d)
    lens = [n, *[1] * crowd(h, kv) * many]
    q, k, v = (rows(rng, "f16", sum(lens), m * d) for m in (h, kv, kv))
    tok = np.arange(n)
    first, last = tok // tile * tile, np.minimum(tok // tile * tile + tile, n) - 1  # of each token's tile
    for mode, window in ((1, -1), (3, 50), (2, 37), (3, 130)):
        want = packed(rk, q, k, v, lens, h, kv, d, "f16", 0.1, mode=mode, window=window)
        lo = first - {1: n, 2: window, 3: window - 1}[mode]
        hi, hidden = last + (window if mode == 2 else 0), 0
        for at, bits in ((tile, 0x7E00), (tile + 1, 0x7C00), (2 * tile + 4, 0xFC00), (100, 0x7E00), (n // 2 + 1, 0x7E00), (n - 2, 0x7E00)):
            bad = v.copy()
            bad[at] = bits
            got = packed(rk, q, k, bad, lens, h, kv, d, "f16", 0.1, mode=mode, window=window)
            clean = (at < lo) | (at > hi)
            hidden += clean.sum()  # (none of a key in a causal prompt's first tile)
            wrong = np.flatnonzero((got[:n] != want[:n]).any(1) & clean)
            assert wrong.size == 0, f"mode {mode} window {window}: key {at} reached tokens {wrong[:4]}"
            assert (got[n:] == want[n:]).all()
        assert hidden > 0


@pytest.mark.parametrize("h,kv,d", [(8, 2, 64), (32, 4, 128), (3, 1, 256)])
@pytest.mark.parametrize("n,m", [(1, 400), (1, 7000), (5, 333), (40, 6000)])
def test_paged_values_beside_the_window_do_not_reach_the_tokens(rk, h, kv, d, n, m):
    """The keys on either side of what the new tokens see: of a page that the sequence still holds, or of later slots."""
    note(f"paged, hidden values, {n} of {m} {h}/{kv} d={d}")
    ps = 32
    pg, caches, keys, q = paged_inputs(61, [m], ps, h, kv, d, "f16", [n])
    for window in (50, 64, 333):
        want = paged(rk, pg, caches, q, [n], [m], h, kv, d, "f16", 0.1, mode=3, window=window)
        assert np.isfinite(ref.decode(want, "f16")).all()
        first = m - n - window + 1
        if first <= 0:
            continue
        bad = [caches[0], caches[1].copy()]
        for at in range(max(0, first - 40), first):
            bad[1][pg.table[0, at // ps], :, at % ps] = 0x7E00
        assert (paged(rk, pg, bad, q, [n], [m], h, kv, d, "f16", 0.1, mode=3, window=window) == want).all(), f"window {window}"


# ----------------------------------------------------------- probabilities ----
# A probability is held as two values of the type: what the second leaves is 2^-16 of it at most (bf16: 2^-7 of it is
# the second one's range, 2^-9 of that its rounding; fp16: 2^-10 and 2^-10).
P_LEFT = 2.0 ** -16


def close_once_rounded(got, q, k, v, pos, scale, softcap, mode, window, dtype, what):
    """`got` is the exact result but for its own rounding and f32 arithmetic."""
    want, rest = ref.attention(q, k, v, pos, scale, softcap, mode, window, P_LEFT)
    ref.close(got, want, rest + 1.01 * ref.HALF[dtype] * np.abs(want), what)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("h,kv,d,mode,window,softcap", [(4, 2, 64, 1, -1, 0.0), (16, 8, 128, 1, -1, 0.0), (2, 2, 72, 0, -1, 0.0),
                                                        (3, 1, 256, 2, 40, 0.0), (8, 1, 32, 1, -1, 20.0), (4, 4, 96, 3, 70, 30.0)])
def test_packed_rounds_the_result_alone(rk, dtype, many, h, kv, d, mode, window, softcap):
    note(f"packed, once rounded, {dtype} many={many} {h}/{kv} d={d}")
    rng = np.random.default_rng(70)
    lens = [150, 7, *[1] * crowd(h, kv) * many]
    q, k, v = (rows(rng, dtype, sum(lens), m * d) for m in (h, kv, kv))
    got = packed(rk, q, k, v, lens, h, kv, d, dtype, d ** -0.5, softcap, mode, window)
    for at, n in ((0, 150), (150, 7)):
        a = [ref.decode(t[at:at + n], dtype).reshape(n, -1, d) for t in (got, q, k, v)]
        close_once_rounded(*a, np.arange(n), d ** -0.5, softcap, mode, window, dtype, f"sequence of {n}")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("q_lens,kv_lens,h,kv,d", [([1, 1], [4097, 33], 32, 4, 128), ([40, 1], [900, 700], 16, 4, 64), ([200], [1500], 8, 1, 128),
                                                   ([1], [3000], 4, 1, 256)])
def test_paged_rounds_the_result_alone(rk, dtype, q_lens, kv_lens, h, kv, d):
    note(f"paged, once rounded, {dtype} {q_lens} of {kv_lens} {h}/{kv} d={d}")
    pg, caches, keys, q = paged_inputs(71, kv_lens, 32, h, kv, d, dtype, q_lens)
    got, at = paged(rk, pg, caches, q, q_lens, kv_lens, h, kv, d, dtype, d ** -0.5), 0
    for i, (n, m) in enumerate(zip(q_lens, kv_lens)):
        a = [ref.decode(t[at:at + n], dtype).reshape(n, h, d) for t in (got, q)]
        close_once_rounded(*a, *(ref.decode(t[i], dtype) for t in keys), np.arange(m - n, m), d ** -0.5, 0.0, 1, -1, dtype, f"{n} of {m}")
        at += n


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,h,kv,d,mode", [(1024, 16, 8, 128, 1), (2116, 16, 16, 72, 0), (24, 16, 8, 128, 1)])
def test_packed_meets_the_gate_of_the_single_sequence_attention(rk, orc, dtype, n, h, kv, d, mode):
    """Cosine 0.9999 and max-rel 1e-2, which rk_attention_dev is held to, at its sizes."""
    note(f"packed, parity gate, {dtype} n={n} {h}/{kv} d={d}")
    rng = np.random.default_rng(72)
    x = [rng.standard_normal((n, m * d)) for m in (h, kv, kv)]
    x = [ref.encode(np.where(np.abs(a) < 2.0 ** -6, 0.0, a), dtype) for a in x]  # (bf16 values of this range are fp16 values)
    got = ref.decode(packed(rk, *x, [n], h, kv, d, dtype, d ** -0.5, mode=mode), dtype)
    want = orc.attention_ref(*(ref.decode(a, dtype).astype(np.float16) for a in x), h, kv, d, d ** -0.5, 0.0, mode)
    assert orc.cosine(got, want) >= 0.9999 and orc.max_rel(got, want) <= 1e-2, (orc.cosine(got, want), orc.max_rel(got, want))


def test_mem_stats_count_live_plans(rk):
    note("mem_stats of plans")
    h, kv, d = 8, 1, 128
    before = rk.mem_stats()
    plan = rk.paged_plan([1], [30000], np.arange(2000, dtype=np.int32)[None], 2000, 16, h, kv, d)
    made = rk.mem_stats()
    held = made.scratch_bytes - before.scratch_bytes
    # page ids, and a state of 16 rows for each part of a tile that is split
    assert held >= 4 * 1875 + 16 * 16 * d * 4 and made.attention_bytes - before.attention_bytes == held
    assert made.host_bytes == before.host_bytes and made.n_scratch == before.n_scratch
    plan.update([1], [29999], np.arange(2000, dtype=np.int32)[None])
    now = rk.mem_stats()
    assert now.host_bytes - before.host_bytes >= 4 * 1875 and now.scratch_bytes - before.scratch_bytes == held
    plan.reserve(300)
    assert rk.mem_stats().scratch_bytes > now.scratch_bytes
    plan.destroy()
    after = rk.mem_stats()
    assert (after.scratch_bytes, after.attention_bytes, after.host_bytes) == (before.scratch_bytes, before.attention_bytes, before.host_bytes)


def test_updates_of_a_captured_plan_allocate_nothing(rk):
    """All that they need is there with the reserve: none can fail for want of memory and leave a graph with lists that
    the plan no longer knows."""
    note("updates of a captured plan")
    h, kv, d, n = 8, 2, 64, 40
    st, b = rk.new_stream(), rk.DeviceBuffer(n * (h + 2 * kv) * d * 2)
    plan, before = rk.packed_plan([1] * n, h, kv, d), rk.mem_stats()
    plan.reserve(n)
    held = rk.mem_stats()
    assert held.host_bytes > before.host_bytes
    g = Graph(st, lambda: ok(rk, rk.lib().rk_attention_packed_dev(plan.ptr, b.ptr, h * d, b.ptr, kv * d, b.ptr, kv * d, 0.1, 0.0, b.ptr,
                                                                  h * d, rk.DTYPE_F16, st)))
    for lens in ([n], [1], [n // 2] * 2, [], [1] * n):
        plan.update(lens, stream=st)
        now = rk.mem_stats()
        assert (now.host_bytes, now.scratch_bytes) == (held.host_bytes, held.scratch_bytes)
    rk.synchronize(st)
    g.destroy()
    plan.destroy()
    rk.destroy_stream(st)


@pytest.mark.parametrize("q,kv_len", [(64, 2000), (64, 20000), (200, 60000)])
@pytest.mark.parametrize("mode,window", [(3, 512), (2, 100)])
def test_windowed_chunks_behind_long_prefixes(rk, q, kv_len, mode, window):
    note(f"paged, chunk of {q} of {kv_len}, mode {mode} window {window}")
    paged_case(rk, q + window, [q, 1], [kv_len, 90], 64, 16, 4, 64, "bf16", mode=mode, window=window)


class CallerStream:
    """A stream that the library did not make."""

    def __init__(self):
        with open("/proc/self/maps") as f:
            self.hip = ctypes.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))
        s = ctypes.c_void_p()
        assert self.hip.hipStreamCreateWithFlags(ctypes.byref(s), 1) == 0  # non-blocking
        self.ptr = s.value

    def destroy(self):
        assert self.hip.hipStreamDestroy(ctypes.c_void_p(self.ptr)) == 0


def two_streams(rk, own):
    made = [None if own else CallerStream() for _ in range(2)]
    sts = [rk.new_stream() if own else m.ptr for m in made]

    def done():
        for st, m in zip(sts, made):
            rk.synchronize(st)
            rk.destroy_stream(st) if own else m.destroy()

    return sts, done


@pytest.mark.parametrize("own", [True, False])
def test_a_plan_s_batches_on_two_streams_each_see_their_own(rk, own):
    """Updates alternate between two batches, each on its own stream, with nothing waited for between them: neither's
    lists reach the other's call."""
    note(f"two batches on two streams, the library's own: {own}")
    h, kv, d, ps = 32, 4, 128, 16
    pg, caches, keys, q = paged_inputs(80, [60000, 3000], ps, h, kv, d, "f16", [1, 1])
    other = pg.table.copy()
    other[[0, 1]] = other[[1, 0]]
    batches = [([1, 1], [60000, 2900], pg.table), ([1, 1], [70, 41000], other)]
    want = []
    for ql, kl, table in batches:
        plan = rk.paged_plan(ql, kl, table, pg.n_pages, ps, h, kv, d)
        want.append(paged(rk, pg, caches, q, ql, kl, h, kv, d, "f16", 0.1, plan=plan))
    check_paged(want[0], [[t[0], t[1][:2900]] for t in keys], q, [1, 1], batches[0][1], h, kv, d, "f16", 0.1)
    check_paged(want[1], [[t[1][:70], t[0][:41000]] for t in keys], q, [1, 1], batches[1][1], h, kv, d, "f16", 0.1)
    assert (want[0] != want[1]).any(1).all()
    b = upload(rk, q, *caches)
    outs = [rk.DeviceBuffer(q.nbytes) for _ in range(12)]
    plan = rk.paged_plan(*batches[0], pg.n_pages, ps, h, kv, d)
    plan.update(*batches[1])  # (room for both: no later update waits to allocate)
    sts, done = two_streams(rk, own)
    for i, o in enumerate(outs):
        plan.update(*batches[i % 2], stream=sts[i % 2])
        for _ in range(3):
            ok(rk, rk.lib().rk_attention_paged_dev(plan.ptr, b[0].ptr, h * d, b[1].ptr, b[2].ptr, 0.1, 0.0, o.ptr, h * d, rk.DTYPE_F16,
                                                   sts[i % 2]))
    done()
    for i, o in enumerate(outs):
        assert (o.download(q.shape, np.uint16) == want[i % 2]).all(), f"call {i}"
    plan.destroy()


@pytest.mark.parametrize("own", [True, False])
def test_an_update_that_grows_a_plan_in_use_waits_for_it(rk, own):
    """The lists and states of a call that still runs on another stream are not given back under it."""
    note(f"growth in use, the library's own streams: {own}")
    rng, h, kv, d = np.random.default_rng(81), 8, 1, 128
    small, large = [3000], [2500, *[3] * 500]
    toks = sum(large)
    q, k, v = (rows(rng, "bf16", toks, n * d) for n in (h, kv, kv))
    want = [packed(rk, *(a[:sum(lens)] for a in (q, k, v)), lens, h, kv, d, "bf16", 0.1) for lens in (small, large)]
    b = upload(rk, q, k, v)
    sts, done = two_streams(rk, own)
    for i in range(4):
        plan, outs = rk.packed_plan(small, h, kv, d), [rk.DeviceBuffer(q.nbytes) for _ in range(2)]

        def call(o, st):
            ok(rk, rk.lib().rk_attention_packed_dev(plan.ptr, b[0].ptr, h * d, b[1].ptr, kv * d, b[2].ptr, kv * d, 0.1, 0.0, o.ptr, h * d,
                                                    rk.DTYPE_BF16, st))

        for _ in range(5):
            call(outs[0], sts[0])
        plan.update(large, stream=sts[1])
        call(outs[1], sts[1])
        for st in sts:
            rk.synchronize(st)
        for o, w in zip(outs, want):
            assert (o.download(w.shape, np.uint16) == w).all()
        plan.destroy()
    done()


@pytest.mark.parametrize("mode,window", [(1, -1), (3, 200), (0, -1)])
@pytest.mark.parametrize("h,kv,d", [(8, 2, 64), (16, 2, 128), (3, 1, 256), (4, 4, 72)])
def test_paged_softcap_in_bf16(rk, mode, window, h, kv, d):
    note(f"paged, bf16, softcap, mode {mode} {h}/{kv} d={d}")
    paged_case(rk, 82, [1, 150, 20], [700, 600, 20], 32, h, kv, d, "bf16", mode=mode, window=window, softcap=20.0)


def test_other_streams_are_refused_while_the_last_call_s_stream_is_captured(rk):
    """A plan's last call ran on a stream that is then captured: a call elsewhere, which has to wait for it, does not
    become part of the capture, and works afterwards."""
    note("another stream beside a capture")
    rng, lib, h, kv, d, lens = np.random.default_rng(83), rk.lib(), 8, 2, 64, [40, 1, 9]
    q, k, v = (rows(rng, "f16", 50, n * d) for n in (h, kv, kv))
    b, outs = upload(rk, q, k, v), [rk.DeviceBuffer(q.nbytes) for _ in range(2)]
    plan, sts, seen = rk.packed_plan(lens, h, kv, d), [rk.new_stream(), rk.new_stream()], []
    plan.reserve(50)

    def call(i):
        return lib.rk_attention_packed_dev(plan.ptr, b[0].ptr, h * d, b[1].ptr, kv * d, b[2].ptr, kv * d, 0.1, 0.0, outs[i].ptr, h * d,
                                           rk.DTYPE_F16, sts[i])

    ok(rk, call(0))  # a warm-up, as programs make before they capture

    def step():
        ok(rk, call(0))
        seen.append(call(1))
        for change in (lambda: plan.update([50], stream=sts[1]), lambda: plan.destroy()):
            with pytest.raises(rk.RocketError) as e:
                change()
            seen.append(e.value.rc)

    g = Graph(sts[0], step)
    assert seen == [rk.RK_E_UNSUPPORTED] * 3
    ok(rk, call(1))
    for _ in range(3):
        rk.synchronize(sts[1])  # (the order of replays and other calls is the caller's)
        outs[0].upload(np.full(q.shape, FILL, np.uint16))
        g.replay()
        rk.synchronize(sts[0])
        ok(rk, call(1))
        rk.synchronize(sts[1])
        for o in outs:
            check_packed(o.download(q.shape, np.uint16), q, k, v, lens, h, kv, d, "f16", 0.1)
    g.destroy()
    plan.destroy()
    for st in sts:
        rk.destroy_stream(st)
