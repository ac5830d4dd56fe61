"""Routed fp8 layers at the edges of their ranges: stacks whose rows fill LDS, and what the calls on them refuse."""
import ctypes

import numpy as np
import pytest

import fp8_ref as ref
from test_gpu_moe_routed import choices, experts, note, run_host, run_routed

pytestmark = pytest.mark.gpu


def random_layer(rk, r, e, h, i):
    stack = [ref.random_stack(r, e, n, k) for n, k in ((i, h), (i, h), (h, i))]
    return stack, rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2])


@pytest.mark.parametrize("s,how", [(1, "any"), (2, "one"), (7, "any"), (11, "one"), (12, "twice")])
@pytest.mark.parametrize("h,i", [(36000, 48), (48, 36000), (18000, 64)])
def test_tiles_of_two_and_four_rows(rk, h, i, s, how):
    """Stacks so wide that a workgroup has LDS for two rows (four), in tiles that are whole and that are not: bit for bit the
    results of the host's lists."""
    note(f"fp8 experts, very wide h={h} i={i} s={s} {how}")
    r = np.random.default_rng(h + s)
    e, k = 3, 2
    stack, wid = random_layer(rk, r, e, h, i)
    x = r.standard_normal((s, h)).astype(np.float32)
    ids, wts = choices(r, s, e, k, how)
    plan = rk.routed_plan(wid, 12, k)
    got = run_routed(rk, wid, plan, x, ids, wts)
    assert (got == run_host(rk, wid, x, ids, wts)).all()
    want, most = experts(x, ids, wts, stack, "f32")
    assert (np.abs(got - want) <= most + np.abs(want) * 2.0**-23).all()
    plan.destroy()


def run_fp8(rk, wid, x, ids, wts, dtype):
    """rk_moe_experts_fp8_dev on rows of a 16-bit or 32-bit type."""
    lib, s = rk.lib(), len(x)
    plan = rk.routed_plan(wid, s, ids.shape[1])
    bufs = [rk.DeviceBuffer.from_array(a) for a in (x, ids, wts, x)]
    plan.route(s, bufs[1].ptr, bufs[2].ptr)
    assert lib.rk_moe_experts_fp8_dev(int(wid), plan.ptr, bufs[0].ptr, bufs[3].ptr, {"f32": 0, "f16": 1, "bf16": 2}[dtype], 0, None) == 0
    rk.synchronize()
    got = ref.widen(bufs[3].download(x.shape, x.dtype), dtype)
    plan.destroy()
    return got


def positive_weight(r, e, n, k):
    """Codes of 1 to 2 in steps of a quarter: with rows of such values every product of codes is a multiple of 2^-10 of the
    largest, which no instruction cuts."""
    codes = ref.encode(1 + r.integers(0, 5, (e, n, k)) / 4)
    return codes, (0.02 * (0.8 + 0.4 * r.random((e, ref.blocks(n), ref.blocks(k))))).astype(np.float32)


def rows_error(ids, wts, stack, x, dtype):
    """What bf16 layers on tiles of many rows may lose besides: each expert's weighted row as an fp16 number."""
    if dtype != "bf16":
        return 0
    return 2.0**-11 * sum(np.abs(experts(x, ids[:, j:j + 1], wts[:, j:j + 1], stack, dtype)[0]) for j in range(ids.shape[1]))


@pytest.mark.parametrize("rows", [128, 256])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_experts_that_nearly_cancel(rk, monkeypatch, rows, dtype):
    """Two equal experts under weights of nearly the same size and opposite signs: what a token's rows lose before they are
    summed is as large as the result."""
    note(f"fp8 experts that cancel rows={rows} {dtype}")
    monkeypatch.setenv("RK_MOE_FP8_ROWS", str(rows))
    r = np.random.default_rng(rows)
    s, h, i = 40, 256, 272
    stack = [positive_weight(r, 1, n, k) for n, k in ((i, h), (i, h), (h, i))]
    stack = [(np.repeat(c, 2, 0), np.repeat(sc, 2, 0)) for c, sc in stack]
    wid = rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2])
    x, v = ref.cast(1 + r.random((s, h)), dtype)
    ids = np.ascontiguousarray(np.tile([[0, 1]], (s, 1)), np.uint32)
    w = r.uniform(0.5, 1, (s, 1))
    wts = np.ascontiguousarray(np.concatenate([w, -w * (1 + 2.0**-9 * r.random((s, 1)))], 1), np.float32)
    want, most = experts(v, ids, wts, stack, dtype)
    most = most + rows_error(ids, wts, stack, v, dtype)
    off = np.abs(run_fp8(rk, wid, x, ids, wts, dtype) - want)
    bound = most + (np.abs(want) + most) * ref.HALF[dtype] + 2.0**-24 * np.abs(want)
    assert (off <= bound).all(), f"{np.max(off / bound):.3g} times what it may be off"


@pytest.mark.parametrize("rows", [128, 256])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_an_infinite_result_leaves_its_neighbours(rk, monkeypatch, rows, dtype):
    """One output of a token beyond the largest f32; the others of its group are large but finite, and stay that."""
    note(f"fp8 experts, an infinite result, rows={rows} {dtype}")
    monkeypatch.setenv("RK_MOE_FP8_ROWS", str(rows))
    r = np.random.default_rng(rows)
    s, h, i, at = 40, 256, 272, 5
    stack = [positive_weight(r, 2, n, k) for n, k in ((i, h), (i, h), (h, i))]
    codes, scales = stack[2]
    codes[:] = 1            # 2^-9
    codes[:, at] = 126      # 448
    scales[:] = np.float32(2.0**108)
    wid = rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2])
    x, v = ref.cast(1 + r.random((s, h)), dtype)
    ids, wts = choices(r, s, 2, 2, "any")
    want, most = experts(v, ids, wts, stack, dtype)
    most = most + rows_error(ids, wts, stack, v, dtype)
    got = run_fp8(rk, wid, x, ids, wts, dtype)
    rest = np.arange(h) != at
    assert (want[:, at] > 2.0**128).all() and (want[:, rest] < 2.0**127).all()
    assert (got[:, at] == np.inf).all()
    off, bound = np.abs(got - want)[:, rest], (most + (np.abs(want) + most) * ref.HALF[dtype] + 2.0**-24 * np.abs(want))[:, rest]
    assert (off <= bound).all(), f"{np.max(off / bound):.3g} times what it may be off"


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_batches_whose_rows_pass_2_31_bytes(rk, dtype):
    """33000 tokens of 8 experts: bucket rows of 2048 f32 values end behind 2^31 bytes, those of fp16 behind 2^30."""
    note(f"fp8 experts, many tokens {dtype}")
    r = np.random.default_rng(3)
    s, e, k, h, i = 33000, 16, 8, 2048, 144
    stack, wid = random_layer(rk, r, e, h, i)
    x, v = ref.cast(r.standard_normal((s, h), dtype=np.float32), dtype)
    ids = np.ascontiguousarray(r.random((s, e)).argsort(1)[:, :k], np.uint32)
    wts = np.ascontiguousarray(r.uniform(0.1, 1, (s, k)), np.float32)
    got = run_fp8(rk, wid, x, ids, wts, dtype)
    some = np.unique(np.concatenate([[0, 1, s - 2, s - 1], r.integers(0, s, 60)]))
    want, most = experts(v[some], ids[some], wts[some], stack, dtype)
    most = most + rows_error(ids[some], wts[some], stack, v[some], dtype)
    off, bound = np.abs(got[some] - want), most + (np.abs(want) + most) * ref.HALF[dtype] + 2.0**-24 * np.abs(want) + (2.0**-25 if dtype == "f16" else 0)
    assert (off <= bound).all(), f"{np.max(off / bound):.3g} times what it may be off"
    assert np.isfinite(got).all()


def test_batches_that_are_too_large(rk):
    note("fp8 experts, too large")
    lib, r = rk.lib(), np.random.default_rng(4)
    out = ctypes.c_void_p()
    make = lambda w, s, top: lib.rk_moe_routed_plan_create(int(w), s, top, ctypes.byref(out))  # noqa: E731
    _, wid = random_layer(rk, r, 2, 16, 65536)
    assert make(wid, 1 << 16, 2) == rk.RK_E_SHAPE       # s·top_k·inter
    _, wid = random_layer(rk, r, 2, 2048, 16)
    assert make(wid, 1 << 20, 1) == rk.RK_E_SHAPE       # s·hidden
    assert make(wid, 1 << 60, 1) == rk.RK_E_SHAPE
    q8 = rk.pack_moe_f32(*[np.zeros(n, np.float32) for n in ((2, 32, 2048), (2, 32, 2048), (2, 2048, 32))])
    assert make(q8, 1 << 18, 1) == rk.RK_E_SHAPE        # its rows are addressed in 32 bits


def test_null_buffers_and_empty_batches(rk):
    """Null buffers are refused before anything reads them; a batch without tokens needs none."""
    note("moe null buffers")
    lib, r = rk.lib(), np.random.default_rng(5)
    q8 = int(rk.pack_moe_f32(*[r.standard_normal(n).astype(np.float32) for n in ((4, 32, 64), (4, 32, 64), (4, 64, 32))]))
    ids, wts, out = np.zeros((3, 2), np.uint32), np.ones((3, 2), np.float32), ctypes.c_void_p()
    make = lambda i, w, o: lib.rk_moe_plan_create(q8, 3, 2, i, w, o)  # noqa: E731
    assert make(None, wts.ctypes.data, ctypes.byref(out)) == rk.RK_E_SHAPE
    assert make(ids.ctypes.data, None, ctypes.byref(out)) == rk.RK_E_SHAPE
    assert make(ids.ctypes.data, wts.ctypes.data, None) == rk.RK_E_SHAPE
    plan = rk.routed_plan(q8, 3, 2)
    b = rk.DeviceBuffer(1 << 14)
    b.zero()
    plan.route(3, b.ptr, b.ptr)
    assert lib.rk_moe_gate_up_dev(q8, plan.ptr, None, b.ptr, None) == rk.RK_E_SHAPE
    assert lib.rk_moe_gate_up_dev(q8, plan.ptr, b.ptr, None, None) == rk.RK_E_SHAPE
    plan.route(0, None, None)
    assert lib.rk_moe_gate_up_dev(q8, plan.ptr, None, None, None) == 0
    plan.destroy()
    _, wid = random_layer(rk, r, 8, 64, 48)
    ids, wts = rk.route_experts(np.zeros((0, 8), np.float32), 2)
    assert ids.shape == wts.shape == (0, 2)
    assert rk.moe_layer(np.zeros((0, 64), np.float16), np.zeros((0, 8), np.float32), wid, 2).shape == (0, 64)


@pytest.mark.parametrize("kind", ["q8", "fp8"])
def test_host_ids_are_refused_in_a_capture_that_goes_on(rk, kind):
    """rk_moe_experts_dev waits for its stream; in a capture it is refused, and the capture holds what else was recorded."""
    note(f"moe host ids, captured, {kind}")
    from test_gpu_sequences import Graph
    lib, r = rk.lib(), np.random.default_rng(6)
    s, e, k, h, i = 5, 4, 2, 64, 64
    wid = int(random_layer(rk, r, e, h, i)[1] if kind == "fp8" else
              rk.pack_moe_f32(*[r.standard_normal(n).astype(np.float32) for n in ((e, i, h), (e, i, h), (e, h, i))]))
    ids, wts = choices(r, s, e, k, "any")
    st = rk.new_stream()
    x, y = rk.DeviceBuffer.from_array(r.standard_normal((s, h)).astype(np.float32)), rk.DeviceBuffer(s * h * 4)
    q, sc = rk.DeviceBuffer(s * h), rk.DeviceBuffer(s * 4)
    call = lambda f: f(wid, x.ptr, s, k, ids.ctypes.data, wts.ctypes.data, y.ptr, st)  # noqa: E731
    rcs = []

    def step():
        assert lib.rk_quantize_fp8_dev(x.ptr, 0, s, h, q.ptr, sc.ptr, st) == 0
        rcs.extend(call(f) for f in (lib.rk_moe_experts_dev, lib.rk_moe_experts_acc_dev))
    g = Graph(st, step)
    assert rcs == [rk.RK_E_UNSUPPORTED] * 2
    for _ in range(2):
        q.zero()
        g.replay()
        rk.synchronize(st)
        assert (q.download((s, h), np.uint8) == ref.quantize(x.download((s, h), np.float32))[0]).all()
        assert call(lib.rk_moe_experts_dev) == 0
    g.destroy()
    rk.destroy_stream(st)


def test_an_error_is_reported_once(rk):
    """A call that the device has no memory for fails; the next one knows nothing of it."""
    note("an error is reported once")
    lib, r = rk.lib(), np.random.default_rng(7)
    x = r.standard_normal((3, 64)).astype(np.float32)
    b, q, sc = rk.DeviceBuffer.from_array(x), rk.DeviceBuffer(3 * 64), rk.DeviceBuffer(12)
    out = ctypes.c_void_p()
    assert lib.rk_device_alloc(1 << 50, ctypes.byref(out)) == rk.RK_E_NOMEM
    assert lib.rk_quantize_fp8_dev(b.ptr, 0, 3, 64, q.ptr, sc.ptr, None) == 0, lib.rk_last_error()
    rk.synchronize()
    assert (q.download((3, 64), np.uint8) == ref.quantize(x)[0]).all()


def test_plans_come_and_go_during_a_capture(rk):
    """A plan made, and one whose graph is gone destroyed, while another stream is captured: the capture goes on."""
    note("routed plans during a capture")
    from test_gpu_sequences import Graph
    lib, r = rk.lib(), np.random.default_rng(8)
    s, e, k, h, i = 40, 4, 2, 256, 128
    _, wid = random_layer(rk, r, e, h, i)
    x = r.standard_normal((s, h)).astype(np.float32)
    ids, wts = choices(r, s, e, k, "any")
    b = [rk.DeviceBuffer.from_array(a) for a in (x, ids, wts, x)]
    sts = [rk.new_stream(), rk.new_stream()]

    def layer(plan, st):
        plan.route(s, b[1].ptr, b[2].ptr, st)
        assert lib.rk_moe_experts_planned_dev(int(wid), plan.ptr, b[0].ptr, b[3].ptr, st) == 0
    old, now, made = rk.routed_plan(wid, s, k), rk.routed_plan(wid, s, k), []
    g = Graph(sts[0], lambda: layer(old, sts[0]))
    for _ in range(20):
        g.replay()  # still running when the graph goes
    g.destroy()

    def step():
        layer(now, sts[1])
        made.append(rk.routed_plan(wid, s, k))
        old.destroy()
    g = Graph(sts[1], step)
    rk.synchronize(sts[0])
    want = run_host(rk, wid, x, ids, wts)
    for _ in range(3):
        b[3].upload(np.zeros_like(x))
        g.replay()
        rk.synchronize(sts[1])
        assert (b[3].download(x.shape, np.float32) == want).all()
    assert (run_routed(rk, wid, made[0], x, ids, wts) == want).all()
    g.destroy()
    for p in (now, made[0]):
        p.destroy()
    # on the library's own stream it is refused, and the capture goes on too
    rcs, out = [], ctypes.c_void_p()

    def own():
        assert lib.rk_quantize_fp8_dev(b[0].ptr, 0, s, h, b[3].ptr, b[3].ptr + s * h, None) == 0
        rcs.append(lib.rk_moe_routed_plan_create(int(wid), s, k, ctypes.byref(out)))
    g = Graph(rk.stream(), own)
    assert rcs == [rk.RK_E_UNSUPPORTED]
    g.replay()
    rk.synchronize()
    assert (b[3].download((s, h), np.uint8) == ref.quantize(x)[0]).all()
    g.destroy()
    for st in sts:
        rk.destroy_stream(st)
