"""The router's choices where f32 scores cannot decide: groups and experts a rounding apart, and biases that close or force
experts, against the definition in 64 bits."""
import numpy as np
import pytest

from test_gpu_moe_routed import note, route

pytestmark = pytest.mark.gpu

# experts of one, two, four, eight and sixteen a lane; groups of whole lanes, of parts of lanes, of one expert
GROUPS = [(64, 8, 3, 4), (60, 5, 2, 6), (96, 8, 3, 6), (128, 8, 4, 8), (128, 64, 9, 9), (128, 4, 1, 5), (160, 8, 3, 6), (256, 8, 4, 8), (256, 64, 7, 8),
          (512, 8, 4, 8), (640, 64, 5, 12), (1024, 8, 4, 8), (1024, 64, 33, 20), (48, 48, 7, 7), (30, 10, 4, 5)]


def near_ties(r, s, e, score):
    """Logits whose scores, and biases that, are a few roundings apart; biases off the scores' grid, so that sums of two do not
    tie in 64 bits either."""
    x = (r.standard_normal((s, 1)) + r.standard_normal((s, e)) * 10.0 ** r.uniform(-7, -5, (s, 1))).astype(np.float32)
    return x, (1e-7 * r.standard_normal(e) / (1 if score == "sigmoid" else e)).astype(np.float32)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("e,groups,top_groups,k", GROUPS)
def test_groups_a_rounding_apart(rk, e, groups, top_groups, k, score):
    note(f"route near groups e={e} groups={groups} top={top_groups} k={k} {score}")
    r = np.random.default_rng(e + groups)
    x, bias = near_ties(r, 120, e, score)
    ids, _ = rk.route_experts(x, k, score=rk.ROUTE_SIGMOID if score == "sigmoid" else rk.ROUTE_SOFTMAX, bias=bias, n_groups=groups, top_groups=top_groups)
    assert (ids == route(x, k, score, bias, groups, top_groups)[0]).all()


@pytest.mark.parametrize("spread", [1e-6, 1.0])
@pytest.mark.parametrize("groups,top_groups,k", [(1, 1, 8), (8, 4, 8), (16, 3, 6), (64, 20, 12)])
@pytest.mark.parametrize("e", [64, 192, 256, 1024])
def test_biases_that_close_and_force_experts(rk, e, groups, top_groups, k, spread):
    """Large and infinite biases beside scores that are a rounding apart, and beside ordinary ones: what they close stays
    closed, what they force comes first, and the rest is in the order of 64 bits."""
    note(f"route masked e={e} groups={groups} top={top_groups} k={k} spread={spread}")
    r = np.random.default_rng(e + groups + k)
    s = 60
    base = (1e-7 * r.standard_normal(e)).astype(np.float32)
    x = (r.standard_normal((s, 1)) + r.standard_normal((s, e)) * spread).astype(np.float32)
    least = np.finfo(np.float32).min
    for what in (-1e9, least, -np.inf, 1e9, np.inf, "both"):
        bias = base.copy()
        if what == "both":  # sums of two of large magnitudes that cancel
            bias[0::5], bias[1::5] = 1e6, -1e6
        elif what > 0:
            bias[r.permutation(e)[:3]] = what
        else:
            bias[r.random(e) < 0.4] = what
        for score, name in ((rk.ROUTE_SIGMOID, "sigmoid"), (rk.ROUTE_SOFTMAX, "softmax")):
            ids, _ = rk.route_experts(x, k, score=score, bias=bias, n_groups=groups, top_groups=top_groups)
            assert (ids == route(x, k, name, bias, groups, top_groups)[0]).all(), f"{what} {name}"
