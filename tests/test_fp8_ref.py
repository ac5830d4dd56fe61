"""The restatement that the fp8 tests compare with, against torch's own e4m3 and by properties."""
import numpy as np
import torch

import fp8_ref as ref


def test_e4m3_equals_torch():
    all_codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(all_codes).view(torch.float8_e4m3fn).float().numpy()
    got = ref.decode(all_codes)
    assert np.array_equal(got, want, equal_nan=True)
    r = np.random.default_rng(0)
    v = np.concatenate([r.uniform(-448, 448, 5000), r.standard_normal(5000) * 0.01, ref.VALUES[:127], ref._MID, -ref._MID]).astype(np.float32)
    assert (ref.encode(v) == torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()).all()


def test_quantized_rows_are_near():
    r = np.random.default_rng(1)
    x = r.standard_normal((7, 300)).astype(np.float32)
    q, s = ref.quantize(x)
    off = np.abs(ref.values(q, s) - x)
    step = np.repeat(s, 128, 1)[:, :300]
    # half a step of e4m3, relative, or of its subnormals
    assert (off <= np.maximum(np.abs(x) * 2.0**-4, step * 2.0**-10) * (1 + 1e-6)).all()
    assert (np.abs(ref.decode(q)).reshape(7, -1).max() == 448)
    assert (ref.quantize(np.zeros((1, 128), np.float32))[1] == np.float32(1e-12)).all()


def test_bf16_is_torch():
    x = np.random.default_rng(2).standard_normal(1000).astype(np.float32)
    assert (ref.to_bf16(x) == torch.from_numpy(x).bfloat16().view(torch.int16).numpy().view(np.uint16)).all()
