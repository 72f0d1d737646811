"""The serving module's host side: frequencies, argument checks, and the test
reference's own consistency (no GPU)."""
import math

import numpy as np
import pytest
import torch

import serving_ref as R
from sili__new_b200 import serving as S


def test_frequencies():
    inv, gain = S.rotary_frequencies(128, 10000.0)
    assert gain == 1.0 and inv[0] == 1.0 and inv.shape == (64,)
    np.testing.assert_allclose(inv[1:] / inv[:-1], 10000.0 ** (-2 / 128), rtol=1e-12)
    lin, _ = S.rotary_frequencies(128, scaling={"type": "linear", "factor": 4.0})
    np.testing.assert_allclose(lin, inv / 4, rtol=1e-15)
    b, _ = S.rotary_frequencies(128, scaling={"type": "base", "factor": 8.0})
    np.testing.assert_allclose([b[0], b[-1] * 8], [inv[0], inv[-1]], rtol=1e-12)
    for kind, fast in (("yarn", 32.0), ("wavelength", 4.0)):
        s, gain = S.rotary_frequencies(128, scaling={"type": kind, "factor": 16.0, "original": 4096})
        turns = 4096 * inv / (2 * math.pi)
        np.testing.assert_allclose(s[turns > fast * 1.3], inv[turns > fast * 1.3], rtol=1e-12)
        np.testing.assert_allclose(s[turns < 0.8], inv[turns < 0.8] / 16, rtol=1e-12)
        assert (np.diff(s) < 0).all()
        assert gain == (1.0 if kind == "wavelength" else pytest.approx(0.1 * math.log(16.0) + 1))
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0),
                dict(rotary_dim=8, scaling={"type": "other"}), dict(rotary_dim=8, scaling={"type": "linear", "factor": 0}),
                dict(rotary_dim=8, scaling={"type": "yarn", "factor": 2, "original": 64, "fast": 1, "slow": 2}),
                dict(rotary_dim=2, scaling={"type": "base", "factor": 2})):
        with pytest.raises(ValueError):
            S.rotary_frequencies(**bad)


def test_reference_quantiser_keeps_its_own_values():
    rng = np.random.default_rng(0)
    x = rng.normal(0, 3, (50, 64)).astype(np.float32)
    c, b = R.quantise(x)
    v = R.values(c, b)
    amax = np.abs(x.reshape(50, 2, 32)).max(-1).repeat(32, -1).reshape(50, 64)
    # half the widest step is one scale, a scale at most 1/16 above amax / 6; or saturation by the same 1/16
    assert (np.abs(v - x) <= amax / 6 * (1 + 1 / 16) + amax / 16 + 1e-9).all()
    assert not ((c & 15) == 8).any() and not ((c >> 4) == 8).any()


def test_host_arrays_are_refused():
    x = torch.zeros(2, 2, 64)
    cos = torch.zeros(4, 16)
    pos = torch.zeros(2, dtype=torch.int32)
    codes, scales = torch.zeros(2, 2, 2, 16, 32, dtype=torch.uint8), torch.zeros(2, 2, 2, 16, 2, dtype=torch.uint8)
    slots = torch.zeros(2, dtype=torch.int64)
    table, lens = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    for call in (lambda: S.rotary(x, None, cos, cos, pos), lambda: S.cache_append(x, x, codes, scales, slots),
                 lambda: S.cache_read(codes, scales, slots), lambda: S.cache_attention(x, codes, scales, table, lens),
                 lambda: S.page_tables(lens, lens, table, torch.zeros(4, dtype=torch.int32),
                                       torch.zeros(2, dtype=torch.int64), 16, 4)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
