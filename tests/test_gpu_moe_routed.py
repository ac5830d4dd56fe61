"""MoE layers routed on the GPU: the router, the lists built from its choices, fp8 experts, and the three as a layer."""
import ctypes
import sys

import numpy as np
import pytest

import fp8_ref as ref

pytestmark = pytest.mark.gpu
TYPES = {"f32": 0, "f16": 1, "bf16": 2}


def note(msg):
    print(f"[case] {msg}", file=sys.stderr, flush=True)


def ok(rk, rc):
    assert rc == 0, rk.lib().rk_last_error()


@pytest.fixture(params=["by size", "128", "256"])
def tiles(request, monkeypatch):
    """fp8 experts on the tiles that the library picks for a batch, and on those of many rows."""
    if request.param != "by size":
        monkeypatch.setenv("RK_MOE_FP8_ROWS", request.param)


# ------------------------------------------------------------------ router ----
def route(logits, top_k, score="softmax", bias=None, groups=1, top_groups=1, norm=True, scale=1.0):
    """The definition in 64 bits, a token at a time."""
    x = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        if score == "softmax":
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
        else:
            p = 1 / (1 + np.exp(-x))
        by = x.copy() if bias is None else p + bias.astype(np.float64)
    by[np.isnan(by)] = -np.inf
    s, e = x.shape
    ids, wts = np.zeros((s, top_k), np.uint32), np.zeros((s, top_k))
    for t in range(s):
        mine, size = list(range(e)), e // groups
        if groups > 1:
            def of(i):
                best = sorted(by[t, i * size:(i + 1) * size], reverse=True)
                return best[0] if bias is None else sum(best[:2])
            keep = sorted(range(groups), key=lambda i: (-of(i), i))[:top_groups]
            mine = [i for i in mine if i // size in keep]
        ids[t] = sorted(mine, key=lambda i: (-by[t, i], i))[:top_k]
        w = p[t, ids[t]]
        wts[t] = (w / (w.sum() + 1e-20) if norm else w) * scale
    return ids, wts


ROUTERS = [(1, 1, 1, {}), (8, 2, 5, {}), (60, 4, 33, dict(norm=False)), (64, 8, 64, {}), (65, 6, 7, dict(score="sigmoid")),
           (128, 8, 100, dict(scale=2.5)), (160, 6, 50, dict(groups=8, top_groups=3)), (256, 8, 70, dict(score="sigmoid", bias=True, groups=8, top_groups=4, scale=2.5)),
           (256, 8, 40, dict(bias=True)), (384, 8, 20, dict(score="sigmoid", groups=4, top_groups=2)), (1024, 64, 9, dict(score="sigmoid", bias=True, groups=64, top_groups=5)),
           (8, 8, 6, dict(groups=8, top_groups=8, bias=True)), (32, 3, 6, dict(groups=32, top_groups=3, bias=True, score="sigmoid"))]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("e,k,s,how", ROUTERS)
def test_router(rk, e, k, s, how, dtype):
    note(f"route e={e} k={k} s={s} {how} {dtype}")
    r = np.random.default_rng(e + k)
    how = dict(how)
    if how.pop("bias", False):
        how["bias"] = (0.1 * r.standard_normal(e)).astype(np.float32)
    logits, v = ref.cast(r.standard_normal((s, e)) * 1.5, dtype)
    mine = dict(how, score=rk.ROUTE_SIGMOID if how.get("score") == "sigmoid" else rk.ROUTE_SOFTMAX, norm_topk=how.get("norm", True),
                n_groups=how.get("groups", 1), top_groups=how.get("top_groups", 1))
    for name in ("norm", "groups"):
        mine.pop(name, None)
    ids, wts = rk.route_experts(logits, k, bf16=dtype == "bf16", **mine)
    want_ids, want = route(v, k, **how)
    assert (ids == want_ids).all()
    # f32 throughout: exp and a division to two steps each, the sums of up to 1024 positive terms in a tree of at most 20,
    # three more operations
    assert (np.abs(wts - want) <= 30 * 2.0**-24 * want + 1e-37).all()


def test_router_at_ties_and_non_finite_logits(rk):
    note("route ties")
    x = np.zeros((6, 128), np.float32)          # all equal: the first ids
    x[1, 70] = x[1, 90] = 5                     # two equal ones across lanes' registers
    x[2] = -np.inf
    x[2, 3] = 0
    x[3, 5], x[3, 6] = np.nan, 1
    x[4] = np.arange(128)[::-1] * np.float32(2.0**-149)  # the least differences
    x[5] = 1
    x[5, 100] = np.nextafter(np.float32(1), np.float32(2))
    for score in (rk.ROUTE_SOFTMAX, rk.ROUTE_SIGMOID):
        ids, wts = rk.route_experts(x, 4, score=score)
        assert list(ids[0]) == [0, 1, 2, 3] and list(ids[1]) == [70, 90, 0, 1]
        assert list(ids[2]) == [3, 0, 1, 2] and list(ids[3]) == [6, 0, 1, 2]
        assert list(ids[4]) == [0, 1, 2, 3] and list(ids[5]) == [100, 0, 1, 2]
        assert np.allclose(wts[0], 0.25, rtol=1e-6) and np.allclose(wts[2], [1, 0, 0, 0])
    # every score below the least f32: weights of 0, not of 0 / 0
    ids, wts = rk.route_experts(np.full((1, 8), -200, np.float32), 2, score=rk.ROUTE_SIGMOID)
    assert list(ids[0]) == [0, 1] and (wts == 0).all()
    # a bias of the least value closes an expert until nothing else is left; infinite biases tie
    b = np.zeros(8, np.float32)
    b[0], b[6], b[7] = np.finfo(np.float32).min, np.inf, np.inf
    ids, _ = rk.route_experts(np.zeros((1, 8), np.float32), 8, bias=b)
    assert list(ids[0]) == [6, 7, 1, 2, 3, 4, 5, 0]
    b[:] = -np.inf
    ids, _ = rk.route_experts(np.zeros((1, 8), np.float32), 3, bias=b, n_groups=4, top_groups=2)
    assert list(ids[0]) == [0, 1, 2]


def test_router_choices_a_rounding_apart(rk):
    """Scores that f32 cannot tell apart, with a bias: the order is that of f64."""
    note("route near ties")
    r = np.random.default_rng(5)
    x = (r.standard_normal((400, 1)) + r.standard_normal((400, 64)) * 1e-6).astype(np.float32)
    bias = np.zeros(64, np.float32)
    for score, name in ((rk.ROUTE_SIGMOID, "sigmoid"), (rk.ROUTE_SOFTMAX, "softmax")):
        for b in (None, bias):
            ids, _ = rk.route_experts(x, 8, score=score, bias=b)
            assert (ids == route(x, 8, name, b)[0]).all()


def test_router_agrees_with_the_host_router(rk):
    note("route host")
    x = np.random.default_rng(6).standard_normal((300, 128)).astype(np.float32)
    for norm in (True, False):
        ids, wts = rk.route_experts(x, 8, norm_topk=norm)
        hids, hwts = rk.moe_route(x, 8, norm)
        assert (ids == hids).all() and np.allclose(wts, hwts, rtol=4e-6, atol=0)


# ------------------------------------------------------------------- lists ----
def q8_stack(rk, r, e, h, i):
    return rk.pack_moe_f32(*[(r.standard_normal(s) * 0.05).astype(np.float32) for s in ((e, i, h), (e, i, h), (e, h, i))])


def run_routed(rk, wid, plan, x, ids, wts, y0=None, acc=False, stream=None):
    """The planned call of f32 rows on a routed plan, with a row behind the last that must stay."""
    lib, s = rk.lib(), len(x)
    y = np.full((s + 1, x.shape[1]), 7.5, np.float32)
    if y0 is not None:
        y[:s] = y0
    bufs = [rk.DeviceBuffer.from_array(a) for a in (x, ids, wts, y)]
    plan.route(s, bufs[1].ptr, bufs[2].ptr, stream)
    call = lib.rk_moe_experts_planned_acc_dev if acc else lib.rk_moe_experts_planned_dev
    ok(rk, call(int(wid), plan.ptr, bufs[0].ptr, bufs[3].ptr, stream))
    rk.synchronize(stream)
    got = bufs[3].download(y.shape, np.float32)
    assert (got[s] == 7.5).all()
    return got[:s]


def run_host(rk, wid, x, ids, wts, y0=None, acc=False):
    lib, s = rk.lib(), len(x)
    dx, dy = rk.DeviceBuffer.from_array(x), rk.DeviceBuffer.from_array(np.zeros_like(x) if y0 is None else y0)
    call = lib.rk_moe_experts_acc_dev if acc else lib.rk_moe_experts_dev
    ok(rk, call(int(wid), dx.ptr, s, ids.shape[1], ids.ctypes.data, wts.ctypes.data, dy.ptr, None))
    rk.synchronize()
    return dy.download(x.shape, np.float32)


def choices(r, s, e, k, how):
    if how == "one":  # every token to the same expert first
        ids = np.stack([np.concatenate([[e - 1], r.permutation(e - 1)[:k - 1]]) for _ in range(s)])
    elif how == "twice":  # an expert named more than once
        ids = r.integers(0, min(e, 3), (s, k))
    else:
        ids = np.stack([r.permutation(e)[:k] for _ in range(s)])
    return np.ascontiguousarray(ids, np.uint32), np.ascontiguousarray(r.uniform(0.1, 1, (s, k)), np.float32)


@pytest.mark.parametrize("kind", ["q8", "fp8"])
@pytest.mark.parametrize("how", ["any", "one", "twice"])
@pytest.mark.parametrize("s", [1, 7, 8, 9, 16, 17, 33, 255, 256, 257, 700, 1100, 2900])
def test_lists_equal_those_of_the_host(rk, s, how, kind):
    """Bit for bit the results of the host's lists: one block of pairs, several, tiles of every size, one plan for
    batches of changing size."""
    note(f"routed lists s={s} {how} {kind}")
    r = np.random.default_rng(s)
    e, k, h, i = 16, 4, 128, 64
    if kind == "q8":
        wid = q8_stack(rk, r, e, h, i)
    else:
        wid = rk.pack_moe_fp8(*ref.random_stack(r, e, i, h), *ref.random_stack(r, e, i, h), *ref.random_stack(r, e, h, i))
    plan = rk.routed_plan(wid, s + 5, k)
    x = r.standard_normal((s, h)).astype(np.float32)
    for n in (s, (s + 1) // 2, s):
        ids, wts = choices(r, n, e, k, how)
        assert (run_routed(rk, wid, plan, x[:n], ids, wts) == run_host(rk, wid, x[:n], ids, wts)).all()
    y0 = r.standard_normal((s, h)).astype(np.float32)
    assert (run_routed(rk, wid, plan, x, ids, wts, y0, True) == run_host(rk, wid, x, ids, wts, y0, True)).all()
    plan.destroy()


@pytest.mark.parametrize("kind", ["q8", "fp8"])
@pytest.mark.parametrize("e,s", [(1, 40), (2, 3000), (130, 90), (1024, 300)])
def test_lists_of_few_and_many_experts(rk, e, s, kind):
    note(f"routed lists e={e} s={s} {kind}")
    r = np.random.default_rng(e)
    k, h, i = min(e, 3), 32, 32
    if kind == "q8":
        wid = q8_stack(rk, r, e, h, i)
    else:
        wid = rk.pack_moe_fp8(*ref.random_stack(r, e, i, h), *ref.random_stack(r, e, i, h), *ref.random_stack(r, e, h, i))
    plan = rk.routed_plan(wid, s, k)
    x = r.standard_normal((s, h)).astype(np.float32)
    ids, wts = choices(r, s, e, k, "any")
    assert (run_routed(rk, wid, plan, x, ids, wts) == run_host(rk, wid, x, ids, wts)).all()


@pytest.mark.parametrize("kind", ["q8", "fp8"])
@pytest.mark.parametrize("s", [3, 40, 400])
def test_ids_of_no_expert_add_nothing(rk, tiles, s, kind):
    note(f"routed no expert s={s} {kind}")
    r = np.random.default_rng(s)
    e, k, h, i = 6, 4, 96, 64
    if kind == "q8":
        wid = q8_stack(rk, r, e, h, i)
    else:
        wid = rk.pack_moe_fp8(*ref.random_stack(r, e, i, h), *ref.random_stack(r, e, i, h), *ref.random_stack(r, e, h, i))
    x = r.standard_normal((s, h)).astype(np.float32)
    ids, wts = choices(r, s, e, k, "any")
    gone = r.random((s, k)) < 0.4
    gone[0] = False
    gone[1] = True  # a token without experts
    plan = rk.routed_plan(wid, s, k)
    for bad in (np.uint32(e), np.uint32(0xFFFFFFFF)):
        mine, weights = np.where(gone, bad, ids).astype(np.uint32), np.where(gone, np.float32(np.nan), wts).astype(np.float32)
        # the host's form: the same expert, with a weight of zero
        zero = np.where(gone, np.float32(0), wts).astype(np.float32)
        got = run_routed(rk, wid, plan, x, mine, weights)
        assert (got == run_host(rk, wid, x, ids, zero)).all() and (got[1] == 0).all()
        y0 = r.standard_normal((s, h)).astype(np.float32)
        got = run_routed(rk, wid, plan, x, mine, weights, y0, True)
        assert (got == run_host(rk, wid, x, ids, zero, y0, True)).all() and (got[1] == y0[1]).all()
    # every pair without an expert
    got = run_routed(rk, wid, plan, x, np.full((s, k), e, np.uint32), wts)
    assert (got == 0).all()


def test_empty_batches_and_refusals(rk):
    note("routed refusals")
    lib, r = rk.lib(), np.random.default_rng(0)
    e, k, h, i = 4, 2, 64, 64
    q8 = int(q8_stack(rk, r, e, h, i))
    fp8 = int(rk.pack_moe_fp8(*ref.random_stack(r, e, i, h), *ref.random_stack(r, e, i, h), *ref.random_stack(r, e, h, i)))
    out = ctypes.c_void_p()
    make = lambda w, s, top, o=ctypes.byref(out): lib.rk_moe_routed_plan_create(w, s, top, o)  # noqa: E731
    assert make(fp8, 0, k) == rk.RK_E_SHAPE and make(fp8, 5, 5) == rk.RK_E_SHAPE and make(fp8, 5, 0) == rk.RK_E_SHAPE
    assert make(1 << 40, 5, 2) == rk.RK_E_SHAPE and make(fp8, 1 << 20, 2) == rk.RK_E_SHAPE and make(fp8, 5, 2, None) == rk.RK_E_SHAPE
    plan = rk.routed_plan(fp8, 8, k)
    b = rk.DeviceBuffer(1 << 14)
    b.zero()
    run = lambda w, p, x, y, dt=0: lib.rk_moe_experts_fp8_dev(w, p, x, y, dt, 0, None)  # noqa: E731
    assert run(fp8, plan.ptr, b.ptr, b.ptr) == rk.RK_E_SHAPE  # no batch yet
    assert lib.rk_moe_experts_planned_dev(fp8, plan.ptr, b.ptr, b.ptr, None) == rk.RK_E_SHAPE
    assert lib.rk_moe_plan_route_dev(plan.ptr, 9, b.ptr, b.ptr, None) == rk.RK_E_SHAPE
    assert lib.rk_moe_plan_route_dev(plan.ptr, -1, b.ptr, b.ptr, None) == rk.RK_E_SHAPE
    assert lib.rk_moe_plan_route_dev(plan.ptr, 4, None, b.ptr, None) == rk.RK_E_SHAPE
    assert lib.rk_moe_plan_route_dev(None, 4, b.ptr, b.ptr, None) == rk.RK_E_SHAPE
    ok(rk, lib.rk_moe_plan_route_dev(plan.ptr, 0, None, None, None))
    ok(rk, run(fp8, plan.ptr, None, None))
    ok(rk, lib.rk_moe_experts_planned_dev(fp8, plan.ptr, None, None, None))
    plan.route(4, b.ptr, b.ptr)
    assert run(fp8, None, b.ptr, b.ptr) == rk.RK_E_SHAPE and run(fp8, plan.ptr, None, b.ptr) == rk.RK_E_SHAPE
    assert run(fp8, plan.ptr, b.ptr, b.ptr + 4) == rk.RK_E_SHAPE and run(fp8, plan.ptr, b.ptr, b.ptr, 4) == rk.RK_E_SHAPE
    assert run(q8, plan.ptr, b.ptr, b.ptr) == rk.RK_E_SHAPE  # another stack's plan
    assert lib.rk_moe_experts_planned_dev(fp8, plan.ptr, b.ptr + 8, b.ptr, None) == rk.RK_E_SHAPE
    assert lib.rk_moe_gate_up_dev(fp8, plan.ptr, b.ptr, b.ptr, None) == rk.RK_E_UNSUPPORTED
    qplan = rk.routed_plan(q8, 8, k)
    qplan.route(4, b.ptr, b.ptr)
    assert run(q8, qplan.ptr, b.ptr, b.ptr) == rk.RK_E_UNSUPPORTED
    rk.synchronize()
    # a plan of host lists is none that is routed here
    ids, wts = np.zeros((4, k), np.uint32), np.ones((4, k), np.float32)
    ok(rk, lib.rk_moe_plan_create(fp8, 4, k, ids.ctypes.data, wts.ctypes.data, ctypes.byref(out)))
    assert lib.rk_moe_plan_route_dev(out, 4, b.ptr, b.ptr, None) == rk.RK_E_SHAPE
    ok(rk, lib.rk_moe_plan_destroy(out))
    before = rk.mem_stats().scratch_bytes
    plan.destroy()
    assert rk.mem_stats().scratch_bytes < before
    # the router's
    go = lambda e, k, score=0, g=1, tg=1, dt=0, s=2: lib.rk_moe_route_dev(b.ptr, dt, s, e, k, score, None, g, tg, 1, 1.0, b.ptr, b.ptr, None)  # noqa: E731
    assert go(8, 0) == rk.RK_E_SHAPE and go(8, 9) == rk.RK_E_SHAPE and go(0, 1) == rk.RK_E_SHAPE and go(8, 2, 2) == rk.RK_E_SHAPE
    assert go(8, 2, 0, 3, 1) == rk.RK_E_SHAPE and go(8, 2, 0, 4, 5) == rk.RK_E_SHAPE and go(8, 3, 0, 4, 1) == rk.RK_E_SHAPE
    assert go(8, 2, 0, 4, 0) == rk.RK_E_SHAPE and go(8, 2, dt=3) == rk.RK_E_SHAPE and go(8, 2, s=-1) == rk.RK_E_SHAPE
    assert go(1025, 2) == rk.RK_E_UNSUPPORTED and go(128, 65) == rk.RK_E_UNSUPPORTED and go(128, 2, 0, 128, 2) == rk.RK_E_UNSUPPORTED
    assert lib.rk_moe_route_dev(None, 0, 2, 8, 2, 0, None, 1, 1, 1, 1.0, b.ptr, b.ptr, None) == rk.RK_E_SHAPE
    assert lib.rk_moe_route_dev(None, 0, 0, 8, 2, 0, None, 1, 1, 1, 1.0, None, None, None) == 0


# ------------------------------------------------------------- fp8 experts ----
def silu(g):
    return g / (1 + np.exp(-g))


def experts(x, ids, wts, stack, dtype):
    """(y, how far it may be off) in 64 bits. A code of an expert's first product is exact unless the value lies so near a
    border between two codes that the product's own error may carry it across: those may be a step off."""
    (gq, gs), (uq, us), (dq, ds) = stack
    e, i, h = gq.shape
    q, s = ref.quantize(x)
    a = ref.values(q, s)
    y, most = np.zeros((len(x), h)), np.zeros((len(x), h))
    # the first product has f32 sums unless the rows are bf16, the second one where they are f32
    first, second = ref.sum_error(h, "bf16" if dtype == "bf16" else "f32"), ref.sum_error(i, dtype)
    for n in range(e):
        tok, slot = np.nonzero(ids == n)
        if not len(tok):
            continue
        wg, wu, wd = ref.weight_values(gq[n], gs[n]), ref.weight_values(uq[n], us[n]), ref.weight_values(dq[n], ds[n])
        g, u = a[tok] @ wg.T, a[tok] @ wu.T
        eg, eu = first * (np.abs(a[tok]) @ np.abs(wg).T), first * (np.abs(a[tok]) @ np.abs(wu).T)
        act = silu(g) * u
        # |silu'| <= 1.1; exp to two steps, a division, two products
        off = 1.1 * eg * (np.abs(u) + eu) + np.abs(silu(g)) * eu + 8 * 2.0**-24 * np.abs(act)
        scale = np.repeat(np.maximum(np.stack([np.abs(act[:, b:b + 128]).max(1) for b in range(0, i, 128)], 1) / 448, 1e-12), 128, 1)[:, :i]
        soff = np.repeat(np.stack([off[:, b:b + 128].max(1) for b in range(0, i, 128)], 1) / 448, 128, 1)[:, :i]
        v = act / scale
        voff = off / scale + np.abs(v) * (soff / scale + 3 * 2.0**-24)
        lo, hi = ref.decode(ref.encode(np.clip(v - voff, -448, 448))), ref.decode(ref.encode(np.clip(v + voff, -448, 448)))
        mid = ref.decode(ref.encode(np.clip(v, -448, 448)))
        val, voff = mid * scale, np.maximum(hi - mid, mid - lo) * scale + np.abs(mid) * soff * 2
        out, err = val @ wd.T, voff @ np.abs(wd).T + second * (np.abs(val) + voff) @ np.abs(wd).T
        w = wts[tok, slot].astype(np.float64)[:, None]
        np.add.at(y, tok, w * out)
        np.add.at(most, tok, np.abs(w) * (err + 2 * 2.0**-24 * np.abs(out)) + len(wts[0]) * 2.0**-24 * np.abs(w * out))
    return y, most


EXPERTS = [(1, 5, 3, 144, 80), (2, 4, 1, 16, 16), (33, 4, 2, 256, 272), (70, 8, 3, 400, 128), (40, 3, 3, 640, 400), (300, 4, 2, 272, 144)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("s,e,k,h,i", EXPERTS)
def test_fp8_experts(rk, tiles, s, e, k, h, i, dtype):
    note(f"fp8 experts s={s} e={e} k={k} h={h} i={i} {dtype}")
    lib, r = rk.lib(), np.random.default_rng(s + h)
    stack = [ref.random_stack(r, e, n, kk) for n, kk in ((i, h), (i, h), (h, i))]
    wid = rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2])
    x, v = ref.cast(r.standard_normal((s, h)) * 3, dtype)
    ids, wts = choices(r, s, e, k, "any")
    want, most = experts(v, ids, wts, stack, dtype)
    plan = rk.routed_plan(wid, s, k)
    bufs = [rk.DeviceBuffer.from_array(a) for a in (x, ids, wts, x)]
    plan.route(s, bufs[1].ptr, bufs[2].ptr)
    for acc in (0, 1):  # (y starts as x where it is added to)
        ok(rk, lib.rk_moe_experts_fp8_dev(int(wid), plan.ptr, bufs[0].ptr, bufs[3].ptr, TYPES[dtype], acc, None))
        rk.synchronize()
        got = ref.widen(bufs[3].download(x.shape, x.dtype), dtype)
        goal = want + (v if acc else 0)
        bound = most + (np.abs(goal) + most) * ref.HALF[dtype] + 2.0**-24 * np.abs(goal) + (2.0**-25 if dtype == "f16" else 0)
        off = np.abs(got - goal)
        assert (off <= bound).all(), f"accumulate={acc}: {np.max(off / bound):.3g} times what it may be off"
        bufs[3].upload(x)
    # x and y on one buffer
    ok(rk, lib.rk_moe_experts_fp8_dev(int(wid), plan.ptr, bufs[3].ptr, bufs[3].ptr, TYPES[dtype], 1, None))
    rk.synchronize()
    assert (ref.widen(bufs[3].download(x.shape, x.dtype), dtype) == got).all()


@pytest.mark.parametrize("dtype,by", [("f32", 1.01), ("bf16", 1.5)])
def test_bounds_of_the_expert_tests_are_tight(dtype, by):
    """They would show a wrong scale of one block of one expert's gate: by a hundredth with f32 rows, by half with bf16
    ones, whose own rounding of a result hides a hundredth of a quarter of its terms."""
    note("fp8 experts, planted mistake in the oracle")
    r = np.random.default_rng(8)
    e, h, i, s = 3, 256, 256, 20
    stack = [ref.random_stack(r, e, n, kk) for n, kk in ((i, h), (i, h), (h, i))]
    x = (r.standard_normal((s, h)) * 3).astype(np.float32)
    ids, wts = choices(r, s, e, 2, "any")
    want, most = experts(x, ids, wts, stack, dtype)
    stack[0][1][1, 1, 0] *= by
    other, _ = experts(x, ids, wts, stack, dtype)
    assert (np.abs(other - want) > most + np.abs(want) * ref.HALF[dtype]).any()


@pytest.mark.parametrize("router", [dict(), dict(score=1, bias=True, n_groups=4, top_groups=2, scale=2.5)])
@pytest.mark.parametrize("s", [1, 50])
def test_a_routed_layer(rk, tiles, s, router):
    """Logits to the layer's output: router, lists and experts one behind the other."""
    note(f"routed layer s={s} {router}")
    r = np.random.default_rng(s)
    e, k, h, i = 16, 4, 256, 144
    stack = [ref.random_stack(r, e, n, kk) for n, kk in ((i, h), (i, h), (h, i))]
    wid = rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2])
    x, v = ref.cast(r.standard_normal((s, h)) * 3, "bf16")
    logits = r.standard_normal((s, e)).astype(np.float32)
    router = dict(router)
    bias = (0.1 * r.standard_normal(e)).astype(np.float32) if router.pop("bias", False) else None
    ids, wts = route(logits, k, "sigmoid" if router.get("score") else "softmax", bias, router.get("n_groups", 1), router.get("top_groups", 1),
                     scale=router.get("scale", 1.0))
    want, most = experts(v, ids, wts.astype(np.float32), stack, "bf16")
    got = ref.widen(rk.moe_layer(x, logits, wid, k, bf16=True, bias=bias, **router), "bf16")
    assert (np.abs(got - want) <= most * 1.001 + np.abs(want) * (ref.HALF["bf16"] * 1.001 + 40 * 2.0**-24)).all()


def test_a_captured_layer_replays_on_new_inputs(rk, tiles):
    """Router, lists and experts in one graph, replayed on new logits and rows with eager work on the plan in between."""
    note("routed layer, captured")
    from test_gpu_sequences import Graph
    lib, r = rk.lib(), np.random.default_rng(11)
    e, k, h, i, s = 8, 3, 128, 160, 40
    stack = [ref.random_stack(r, e, n, kk) for n, kk in ((i, h), (i, h), (h, i))]
    for kind in ("fp8", "q8"):
        wid = int(rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2]) if kind == "fp8" else q8_stack(rk, r, e, h, i))
        plan, other, st = rk.routed_plan(wid, s, k), rk.routed_plan(wid, s, k), rk.new_stream()
        b = [rk.DeviceBuffer.from_array(a) for a in (np.zeros((s, h), np.float32), np.zeros((s, e), np.float32), np.zeros((s, k), np.uint32),
                                                     np.zeros((s, k), np.float32), np.zeros((s, h), np.float32))]
        def layer(p, out, stream):
            ok(rk, lib.rk_moe_route_dev(b[1].ptr, 0, s, e, k, 0, None, 1, 1, 1, 1.0, b[2].ptr, b[3].ptr, stream))
            ok(rk, lib.rk_moe_plan_route_dev(p.ptr, s, b[2].ptr, b[3].ptr, stream))
            ok(rk, lib.rk_moe_experts_planned_dev(wid, p.ptr, b[0].ptr, out.ptr, stream))
        g = Graph(st, lambda: layer(plan, b[4], st))
        assert lib.rk_moe_experts_planned_dev(wid, plan.ptr, b[0].ptr, b[4].ptr, st) == rk.RK_E_UNSUPPORTED  # its lists are the graph's
        assert lib.rk_moe_plan_route_dev(plan.ptr, s - 1, b[2].ptr, b[3].ptr, st) == rk.RK_E_SHAPE  # a captured size
        y2 = rk.DeviceBuffer(s * h * 4)
        for n in range(4):
            x, logits = r.standard_normal((s, h)).astype(np.float32), r.standard_normal((s, e)).astype(np.float32)
            b[0].upload(x)
            b[1].upload(logits)
            g.replay()
            rk.synchronize(st)
            got = b[4].download((s, h), np.float32)
            layer(other, y2, None)
            rk.synchronize()
            assert np.isfinite(got).all() and (got == y2.download((s, h), np.float32)).all(), f"replay {n} {kind}"
            if n == 1:  # eager work on the captured plan
                layer(plan, y2, st)
                rk.synchronize(st)
                assert (y2.download((s, h), np.float32) == got).all()
        g.destroy()
        plan.destroy()
        other.destroy()
        rk.destroy_stream(st)


def test_two_streams_on_one_plan(rk):
    """Batches in turn on two streams: each call waits for the plan's last one."""
    note("routed plan, two streams")
    r = np.random.default_rng(12)
    e, k, h, i, s = 8, 2, 256, 128, 200
    stack = [ref.random_stack(r, e, n, kk) for n, kk in ((i, h), (i, h), (h, i))]
    wid = rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2])
    lib, plan, sts = rk.lib(), rk.routed_plan(wid, s, k), [rk.new_stream(), rk.new_stream()]
    sets = []
    for n in range(6):
        x = r.standard_normal((s, h)).astype(np.float32)
        ids, wts = choices(r, s, e, k, "any")
        sets.append((x, ids, wts, [rk.DeviceBuffer.from_array(a) for a in (x, ids, wts, x)]))
    for n, (x, ids, wts, b) in enumerate(sets):
        st = sts[n % 2]
        plan.route(s, b[1].ptr, b[2].ptr, st)
        ok(rk, lib.rk_moe_experts_planned_dev(int(wid), plan.ptr, b[0].ptr, b[3].ptr, sts[n // 2 % 2]))
    for st in sts:
        rk.synchronize(st)
    for x, ids, wts, b in sets:
        assert (b[3].download(x.shape, np.float32) == run_host(rk, wid, x, ids, wts)).all()
    for st in sts:
        rk.destroy_stream(st)
    plan.destroy()


def test_wide_experts(rk):
    """Rows that only tiles of fewer than 32 have LDS for."""
    note("fp8 experts, wide")
    r = np.random.default_rng(13)
    e, k, h, i, s = 2, 1, 9040, 48, 60
    stack = [ref.random_stack(r, e, n, kk) for n, kk in ((i, h), (i, h), (h, i))]
    wid = rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2])
    x = r.standard_normal((s, h)).astype(np.float32)
    ids, wts = choices(r, s, e, k, "any")
    want, most = experts(x, ids, wts, stack, "f32")
    for got in (run_routed(rk, wid, rk.routed_plan(wid, s, k), x, ids, wts), run_host(rk, wid, x, ids, wts)):
        assert (np.abs(got - want) <= most + np.abs(want) * 2.0**-23).all()


# ------------------------------------------- few tokens: each pair by itself ----
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("s,e,k,h,i", [(1, 64, 8, 144, 80), (4, 64, 8, 272, 256), (3, 128, 16, 160, 144), (1, 70, 32, 64, 400),
                                       (1, 70, 33, 48, 64), (8, 16, 1, 48, 1040), (1, 4, 2, 1040, 16), (1, 16, 8, 32, 8208)])
def test_fp8_experts_of_few_tokens(rk, s, e, k, h, i, dtype):
    """At most half as many pairs as experts; a top_k and an inter that are too large for that among them."""
    test_fp8_experts(rk, None, s, e, k, h, i, dtype)


@pytest.mark.parametrize("how", ["any", "one", "twice"])
def test_few_tokens_without_some_experts(rk, how):
    """A token's result is its own: that of the same token among many, up to the order of sums, and bit for bit that of
    the host's lists. Ids that name no expert add nothing, whatever their weight."""
    note(f"few tokens, no expert, {how}")
    r = np.random.default_rng(21)
    s, e, k, h, i = 5, 64, 6, 176, 144
    stack = [ref.random_stack(r, e, n, kk) for n, kk in ((i, h), (i, h), (h, i))]
    wid = rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2])
    x = r.standard_normal((s, h)).astype(np.float32)
    ids, wts = choices(r, s, e, k, how)
    plan = rk.routed_plan(wid, 40, k)
    gone = r.random((s, k)) < 0.4
    gone[0], gone[1] = False, True
    for bad in (np.uint32(e), np.uint32(0xFFFFFFFF)):
        mine, weights = np.where(gone, bad, ids).astype(np.uint32), np.where(gone, np.float32(np.nan), wts).astype(np.float32)
        zero = np.where(gone, np.float32(0), wts).astype(np.float32)
        got = run_routed(rk, wid, plan, x, mine, weights)
        assert (got == run_host(rk, wid, x, ids, zero)).all() and (got[1] == 0).all()
        y0 = r.standard_normal((s, h)).astype(np.float32)
        got = run_routed(rk, wid, plan, x, mine, weights, y0, True)
        assert (got == run_host(rk, wid, x, ids, zero, y0, True)).all() and (got[1] == y0[1]).all()
    # the plan between small batches and large ones
    many = np.repeat(x, 8, 0)
    large = run_routed(rk, wid, plan, many, np.repeat(ids, 8, 0), np.repeat(wts, 8, 0))
    want, most = experts(x, ids, wts, stack, "f32")
    for n in range(s):
        assert (run_routed(rk, wid, plan, x[n:n + 1], ids[n:n + 1], wts[n:n + 1]) == run_routed(rk, wid, plan, x, ids, wts)[n]).all()
        assert (np.abs(large[8 * n] - want[n]) <= most[n] + np.abs(want[n]) * 2.0**-23).all()
    plan.destroy()


def test_few_tokens_with_non_finite_rows(rk):
    """What is not finite in a token's rows or in an expert's weights stays with the tokens that it reaches."""
    note("few tokens, not finite")
    r = np.random.default_rng(22)
    s, e, k, h, i = 4, 32, 3, 160, 144
    stack = [ref.random_stack(r, e, n, kk) for n, kk in ((i, h), (i, h), (h, i))]
    stack[2][0][5, 7, 9] = 127  # NaN in expert 5's second matrix
    wid = rk.pack_moe_fp8(*stack[0], *stack[1], *stack[2])
    x = r.standard_normal((s, h)).astype(np.float32)
    x[1, 3], x[2, 130] = np.inf, np.nan
    ids = np.array([[5, 1, 2], [6, 7, 8], [9, 10, 11], [12, 13, 14]], np.uint32)
    wts = np.ones((s, k), np.float32)
    got = run_routed(rk, wid, rk.routed_plan(wid, s, k), x, ids, wts)
    clean, most = experts(np.where(np.isfinite(x), x, 0), ids, wts, [(np.where(c == 127, 0, c).astype(np.uint8), sc) for c, sc in stack], "f32")
    assert np.isnan(got[0, 7]) and not np.isfinite(got[1]).any() and np.isnan(got[2]).all()
    for n, cols in ((0, np.arange(h) != 7), (3, np.full(h, True))):
        assert (np.abs(got[n] - clean[n])[cols] <= (most[n] + np.abs(clean[n]) * 2.0**-23)[cols]).all()


def test_few_tokens_captured(rk):
    note("few tokens, captured")
    from test_gpu_sequences import Graph
    lib, r = rk.lib(), np.random.default_rng(23)
    e, k, h, i, s = 32, 4, 256, 160, 3
    wid = int(rk.pack_moe_fp8(*ref.random_stack(r, e, i, h), *ref.random_stack(r, e, i, h), *ref.random_stack(r, e, h, i)))
    plan, st = rk.routed_plan(wid, s, k), rk.new_stream()
    b = [rk.DeviceBuffer.from_array(a) for a in (np.zeros((s, h), np.float32), np.zeros((s, k), np.uint32), np.zeros((s, k), np.float32), np.zeros((s, h), np.float32))]

    def layer():
        ok(rk, lib.rk_moe_plan_route_dev(plan.ptr, s, b[1].ptr, b[2].ptr, st))
        ok(rk, lib.rk_moe_experts_planned_dev(wid, plan.ptr, b[0].ptr, b[3].ptr, st))
    g = Graph(st, layer)
    for n in range(4):
        x = r.standard_normal((s, h)).astype(np.float32)
        ids, wts = choices(r, s, e, k, "any")
        for buf, a in zip(b, (x, ids, wts)):
            buf.upload(a)
        g.replay()
        rk.synchronize(st)
        assert (b[3].download((s, h), np.float32) == run_host(rk, wid, x, ids, wts)).all(), f"replay {n}"
    g.destroy()
    plan.destroy()
    rk.destroy_stream(st)


def test_host_lists_of_fp8_experts_are_refused_in_a_capture(rk):
    note("fp8 host lists, captured")
    from test_gpu_sequences import Graph
    lib, r = rk.lib(), np.random.default_rng(24)
    e, k, h, i, s = 4, 2, 64, 64, 8
    wid = int(rk.pack_moe_fp8(*ref.random_stack(r, e, i, h), *ref.random_stack(r, e, i, h), *ref.random_stack(r, e, h, i)))
    ids, wts = choices(r, s, e, k, "any")
    plan, st = ctypes.c_void_p(), rk.new_stream()
    ok(rk, lib.rk_moe_plan_create(wid, s, k, ids.ctypes.data, wts.ctypes.data, ctypes.byref(plan)))
    x = rk.DeviceBuffer.from_array(r.standard_normal((s, h)).astype(np.float32))
    y = rk.DeviceBuffer(s * h * 4)
    y.zero()
    for call in (lambda: lib.rk_moe_experts_fp8_dev(wid, plan, x.ptr, y.ptr, 0, 0, st),
                 lambda: lib.rk_moe_experts_planned_dev(wid, plan, x.ptr, y.ptr, st)):
        rcs = []

        def step():
            ok(rk, lib.rk_quantize_fp8_dev(x.ptr, 0, s, h, y.ptr, y.ptr + s * h, st))  # (a graph has to hold something)
            rcs.append(call())
        g = Graph(st, step)
        assert rcs == [rk.RK_E_UNSUPPORTED]
        g.destroy()
        ok(rk, call())  # and outside of one
        rk.synchronize(st)
    assert (y.download((s, h), np.float32) == run_host(rk, wid, x.download((s, h), np.float32), ids, wts)).all()
    ok(rk, lib.rk_moe_plan_destroy(plan))
    rk.destroy_stream(st)
