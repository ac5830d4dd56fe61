"""What moe_layer refuses before it touches a device."""
import numpy as np
import pytest

import burn_rocket as rk


@pytest.mark.parametrize("x,logits", [((4, 64), (3, 8)), ((3, 64), (4, 8)), ((4, 48), (4, 8)), ((4, 80), (4, 8)), ((4, 8, 8), (4, 8)),
                                      ((4,), (4, 8)), ((4, 64), (4,)), ((0, 48), (0, 8)), ((0, 64), (1, 8))])
def test_rows_that_do_not_fit_are_refused(monkeypatch, x, logits):
    monkeypatch.setattr(rk, "weight_info", lambda wid: (0, 64, 64, 128))  # a stack of hidden 64
    monkeypatch.setattr(rk, "route_experts", lambda *a, **k: pytest.fail("routed"))
    with pytest.raises(rk.RocketError) as e:
        rk.moe_layer(np.zeros(x, np.float32), np.zeros(logits, np.float32), rk.WeightId(1), 2)
    assert e.value.rc == rk.RK_E_SHAPE
