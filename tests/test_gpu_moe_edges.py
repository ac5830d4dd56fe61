"""Routed fp8 layers at the edges of their ranges: stacks whose rows fill LDS, and what the calls on them refuse."""
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
