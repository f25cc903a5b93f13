"""The 8-bit cache's oracle against brute force and torch's e4m3."""

import numpy as np
import pytest
import torch

from oracle import kv8


def test_e4m3_levels_are_torchs():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(kv8.levels("e4m3"), codes)


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_least_scale_by_trying_them_all(code):
    halves = torch.arange(0x7C00, dtype=torch.int32).to(torch.int16).view(torch.float16).double().numpy()
    want = np.empty_like(halves)
    for i, x in enumerate(halves):
        e = -24
        while x > kv8.LARGEST[code] * 2.0 ** e:
            e += 1
        want[i] = 2.0 ** e
    assert np.array_equal(kv8.least_scale(halves, code), want)
    assert np.isnan(kv8.least_scale([np.inf, np.nan], code)).all()


def test_nearest_is_torchs_rounding():
    x = torch.arange(0x7C00, dtype=torch.int32).to(torch.int16).view(torch.float16).double()
    x = x[x <= 448]
    want = x.float().to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(kv8.nearest(x.numpy(), 1.0, "e4m3"), want)
    y = np.arange(-127, 127.25, 0.25)
    assert np.array_equal(kv8.nearest(y, 1.0, "int8"), np.rint(y))


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_values_stay_within_fp16(code):
    x = np.array([[[65504.0] * 64]] * 3)
    values, scales = np.zeros((16, 1, 64)), np.zeros((1, 1))
    kv8.append(values, scales, 0, x, code)
    d = kv8.dense(values, scales)
    assert d.max() <= kv8.MOST and d[0, 0, 0] >= 61440.0


@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_error_of_one_write(code):
    """Half a step: of the block's scale for int8, of the value (2^-4) or the least one for e4m3."""
    x = np.random.default_rng(0).standard_normal((64, 2, 64))
    values, scales = np.zeros((64, 2, 64)), np.zeros((4, 2))
    kv8.append(values, scales, 0, x, code)
    off = np.abs(kv8.dense(values, scales) - x)
    s = np.repeat(scales, 16, axis=0)[:, :, None]
    if code == "int8":
        assert (off <= s / 2).all()
    else:
        assert (off <= np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -10)).all()
