"""The order of expert tiles that the GPU's lists have, without a device: compiled for the host from its own source."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("tiles") / "moe_tiles_host.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", os.path.join(HERE, "moe_tiles_host.cpp"), "-o", so], check=True)
    return ctypes.CDLL(so)


@pytest.mark.parametrize("most", [1, 3, 5, 40, 700])
@pytest.mark.parametrize("T", [1, 2, 4, 8, 16, 32, 64, 128, 256])
def test_every_row_is_in_one_tile_and_long_tiles_come_first(host, T, most):
    r = np.random.default_rng(T * 1000 + most)
    for n_experts in (1, 2, 7, 64):
        rows = np.ascontiguousarray(r.integers(0, most + 1, n_experts), np.int32)
        want = [(e, at, min(T, n - at)) for e, n in enumerate(rows.tolist()) for at in range(0, n, T)]
        room = min(int(rows.sum()), n_experts + 1 + int(rows.sum()) // T)  # what the launches take
        assert len(want) <= room
        out = [np.zeros((max(room, 1), 3), np.int32) for _ in range(2)]
        n = host.tile_lists(ctypes.c_void_p(rows.ctypes.data), n_experts, T, room, *(ctypes.c_void_p(o.ctypes.data) for o in out))
        assert n == len(want)
        by_expert, by_length = ([tuple(t) for t in o[:n].tolist()] for o in out)
        assert by_expert == want
        # quarters of T, longest first; in expert order within one, an expert's whole tiles ahead of its last
        assert by_length == sorted(want, key=lambda t: -4 * t[2] // T)
