"""Plans of batches of sequences without a device: what is refused, before anything touches the GPU (a valid
request passes to the device stage, which answers RK_E_DEVICE here)."""
import ctypes

import numpy as np
import pytest


@pytest.fixture(scope="module")
def lib():
    import burn_rocket
    lib = burn_rocket.load_library()
    s = burn_rocket.Stats()
    if lib.rk_stats(ctypes.byref(s)) == 0:
        pytest.skip("engine already initialised in this process")
    return lib


def i32(*a):
    return np.array(a, dtype=np.int32)


def ptr(a):
    return None if a is None else a.ctypes.data


def packed(lib, q, n=None, h=8, kv=2, d=64, mode=1, window=-1):
    out = ctypes.c_void_p()
    rc = lib.rk_packed_plan_create(ptr(q), len(q) if n is None else n, h, kv, d, mode, window, ctypes.byref(out))
    assert out.value is None
    return rc, lib.rk_last_error().decode()


def paged(lib, q, kv, table, n_pages=10, ps=16, h=8, hkv=2, d=64, mode=1, window=-1, n=None, stride=None):
    out = ctypes.c_void_p()
    rc = lib.rk_paged_plan_create(ptr(q), ptr(kv), ptr(table), table.shape[1] if stride is None else stride,
                                  len(q) if n is None else n, n_pages, ps, h, hkv, d, mode, window, ctypes.byref(out))
    assert out.value is None
    return rc, lib.rk_last_error().decode()


def test_valid_batches_reach_the_device_stage(lib):
    from burn_rocket import RK_E_DEVICE
    t = np.array([[3, 1], [9, 0]], np.int32)
    for rc, msg in (packed(lib, i32(5, 0, 1)), packed(lib, i32()), packed(lib, None, n=0), packed(lib, i32(4), d=256),
                    packed(lib, i32(4), mode=3, window=0), packed(lib, i32(4), mode=2, window=1 << 60),
                    paged(lib, i32(1, 2), i32(32, 17), t), paged(lib, i32(0, 2), i32(500, 17), t),
                    paged(lib, i32(1), i32(20), np.array([[-7, 2]], np.int32), mode=3, window=4),
                    paged(lib, i32(1), i32(17), np.array([[2, 2, 88]], np.int32))):
        assert rc == RK_E_DEVICE and "rk_init" in msg, msg


@pytest.mark.parametrize("over,rc,word", [
    (dict(h=7), -1, "multiple"), (dict(h=0), -1, "multiple"), (dict(kv=0), -1, "multiple"), (dict(h=-8, kv=-2), -1, "multiple"),
    (dict(h=258, kv=2), -1, "group"), (dict(d=65), -5, "head_dim"), (dict(d=192), -5, "head_dim"), (dict(d=0), -5, "head_dim"),
    (dict(mode=4), -1, "mask"), (dict(mode=-1), -1, "mask"), (dict(n=-1), -1, "n_seqs"), (dict(n=1 << 40), -1, "n_seqs")])
def test_bad_geometry_is_refused(lib, over, rc, word):
    got, msg = packed(lib, i32(4, 5), **over)
    assert got == rc and word in msg, msg


def test_bad_lengths_and_pages_are_refused(lib):
    t = np.array([[3, 1], [9, 0]], np.int32)
    cases = [packed(lib, i32(4, -1)), packed(lib, None, n=2), packed(lib, i32(*[2**30] * 3)), packed(lib, i32(2**30 + 1)),
             packed(lib, i32(2**29), h=64, kv=2),
             paged(lib, i32(3, 1), i32(2, 20), t),                       # fewer keys than new tokens
             paged(lib, i32(1, 1), i32(33, 20), t),                      # more pages than the row holds
             paged(lib, i32(1, 1), i32(20, 20), np.array([[3, 10], [9, 0]], np.int32)),
             paged(lib, i32(1, 1), i32(20, 20), np.array([[3, 1], [-1, 0]], np.int32)),
             paged(lib, i32(1), i32(20), np.array([[-7, 2]], np.int32), mode=3, window=5),  # key 15 is seen
             paged(lib, i32(2), i32(20), np.array([[-7, 2]], np.int32), mode=3, window=4),  # by the first of two
             paged(lib, i32(1), i32(20), np.array([[-7, 2]], np.int32), mode=3, window=0),  # the mean of all keys
             paged(lib, i32(1, 1), None, t), paged(lib, i32(1, 1), i32(1, -5), t),
             paged(lib, i32(1, 1), i32(20, 20), t, n_pages=0), paged(lib, i32(1, 1), i32(20, 20), t, stride=1),
             paged(lib, i32(1, 1), i32(20, 20), t, stride=-1)]
    cases += [paged(lib, i32(1, 1), i32(20, 20), t, ps=ps) for ps in (0, 1, 8, 24, 512, -16)]
    for rc, msg in cases:
        assert rc == -1 and msg, msg
    assert "page 1 has id 10 of 10" in paged(lib, i32(1, 1), i32(20, 20), np.array([[3, 10], [9, 0]], np.int32))[1]


def test_null_output_and_calls_without_an_engine(lib):
    from burn_rocket import RK_E_DEVICE, RK_E_SHAPE
    assert lib.rk_packed_plan_create(ptr(i32(4)), 1, 8, 2, 64, 1, -1, None) == RK_E_SHAPE
    assert lib.rk_seq_plan_destroy(None) == RK_E_DEVICE
    assert lib.rk_attention_packed_dev(None, None, 0, None, 0, None, 0, 1.0, 0.0, None, 0, 1, None) == RK_E_DEVICE


def test_binding_refuses_lengths_that_do_not_fit(lib):
    import burn_rocket as rk
    for bad in ([2**31], [1.5], [-2**40]):
        with pytest.raises(rk.RocketError) as e:
            rk.packed_plan(bad, 8, 2, 64)
        assert e.value.rc == rk.RK_E_SHAPE
    with pytest.raises(rk.RocketError):
        rk.paged_plan([1, 1], [1], np.zeros((2, 1)), 4, 16, 8, 2, 64)


class FakeCache:
    """A PagedCache's shape without its device memory."""

    def __new__(cls, n_pages, ps, kv, d, bf16=False):
        import burn_rocket as rk
        c = rk.PagedCache.__new__(rk.PagedCache)
        c.shape, c.bf16, c.dtype = (n_pages, kv, ps, d), bf16, rk.DTYPE_BF16 if bf16 else rk.DTYPE_F16
        return c


def test_a_cache_refuses_plans_that_name_pages_it_lacks():
    import burn_rocket as rk
    plan = rk.SeqPlan(None, 1, (4, 2, 64), 16, 9)
    q, x, cs = np.zeros((1, 256), np.float16), np.zeros((1, 512), np.float16), np.zeros((9, 32), np.float32)
    for cache in (FakeCache(8, 16, 2, 64), FakeCache(9, 32, 2, 64), FakeCache(9, 16, 4, 64), FakeCache(9, 16, 2, 32)):
        for call in (lambda: cache.attention(plan, q, 0.1), lambda: cache.append(plan, x, cs, cs)):
            with pytest.raises(rk.RocketError) as e:
                call()
            assert e.value.rc == rk.RK_E_SHAPE and "pages" in str(e.value)


def test_append_refuses_one_norm_weight_alone():
    import burn_rocket as rk
    plan, cache = rk.SeqPlan(None, 1, (4, 2, 64), 16, 8), FakeCache(8, 16, 2, 64)
    x, cs, w = np.zeros((1, 512), np.float16), np.zeros((9, 32), np.float32), np.ones(64, np.float16)
    for norms in ((w, None), (None, w)):
        with pytest.raises(rk.RocketError) as e:
            cache.append(plan, x, cs, cs, *norms)
        assert e.value.rc == rk.RK_E_SHAPE and "both" in str(e.value)


def test_an_update_of_packed_sequences_refuses_cached_keys():
    import burn_rocket as rk
    plan = rk.SeqPlan(None, 1, (4, 2, 64))
    for extra in (dict(kv_lens=[5]), dict(page_table=[[0]]), dict(kv_lens=[5], page_table=[[0]])):
        with pytest.raises(rk.RocketError) as e:
            plan.update([1], **extra)
        assert e.value.rc == rk.RK_E_SHAPE and "packed" in str(e.value)


@pytest.mark.parametrize("rc,left", [(-1, 3), (-5, 3), (-3, 0), (-4, 0)])
def test_a_plan_whose_change_failed_has_no_tokens(monkeypatch, rc, left):
    """Calls on such a plan write nothing: the binding expects no rows of them then."""
    import burn_rocket as rk

    class Failing:
        rk_packed_plan_update = rk_paged_plan_update = rk_seq_plan_reserve = staticmethod(lambda *a: rc)
        rk_last_error = staticmethod(lambda: b"planted")

    monkeypatch.setattr(rk, "_lib", Failing)
    for plan, change in ((rk.SeqPlan(None, 3, (4, 2, 64)), lambda p: p.update([2])), (rk.SeqPlan(None, 3, (4, 2, 64)), lambda p: p.reserve(9)),
                         (rk.SeqPlan(None, 3, (4, 2, 64), 16, 8), lambda p: p.update([2], [9], [[1]]))):
        with pytest.raises(rk.RocketError) as e:
            change(plan)
        assert e.value.rc == rc and plan.n_tokens == left


def test_query_rows_stay_inside_32_bits(lib):
    """A sequence of nearly 2^31 query rows: its last tile's rows are counted past the end."""
    from burn_rocket import RK_E_DEVICE, RK_E_SHAPE
    for q, rc in (((2**31 - 129) // 127, RK_E_DEVICE), ((2**31 - 129) // 127 + 1, RK_E_SHAPE), ((2**31 - 1) // 127, RK_E_SHAPE)):
        assert packed(lib, i32(q), h=127, kv=1, d=32)[0] == rc, q
