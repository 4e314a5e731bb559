"""The float64 oracle of the 8-bit cache against torch's float8 and by cases."""

import numpy as np
import pytest
import torch

from oracle import quantized as oracle


def test_e4m3_rounding_is_torchs():
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16)
    for dtype in (torch.bfloat16, torch.float16):
        x = bits.view(dtype).float()
        x = x[x.abs() <= 448]
        want = x.to(torch.float8_e4m3fn).double().numpy()
        np.testing.assert_array_equal(oracle.nearest(x.double().numpy(), "fp8"), want)


def test_int8_rounding_ties_to_even():
    np.testing.assert_array_equal(oracle.nearest([0.5, 1.5, -2.5, 126.5, -0.4], "int8"),
                                  [0, 2, -2, 126, 0])


@pytest.mark.parametrize("kind,most", [("fp8", 448.0), ("int8", 127.0)])
def test_least_scale_is_a_power_of_two_and_least(kind, most):
    assert oracle.least_scale(most, kind) == 1
    assert oracle.least_scale(np.nextafter(most, np.inf), kind) == 2
    assert oracle.least_scale(most / 2, kind) == 0.5
    assert oracle.least_scale(0.0, kind) == 2.0 ** -126
    assert oracle.least_scale(3e38, kind) * most >= 3e38


def test_a_block_grows_and_begins_anew():
    codes, scales = np.zeros((2, 4, 1, 16)), np.zeros((2, 1))
    one = np.ones((1, 1, 16))
    oracle.append(codes, scales, [4], 127 * one, "int8")
    assert scales[1, 0] == 1 and codes[1, 0, 0, 0] == 127
    oracle.append(codes, scales, [5], 200 * one, "int8")  # 127 / 2 ties to 64
    assert scales[1, 0] == 2 and codes[1, 0, 0, 0] == 64 and codes[1, 1, 0, 0] == 100
    oracle.append(codes, scales, [6], one, "int8")
    assert scales[1, 0] == 2 and codes[1, 2, 0, 0] == 0
    oracle.append(codes, scales, [4], one, "int8")
    assert scales[1, 0] == 2.0 ** -6 and codes[1, 0, 0, 0] == 64
    oracle.append(codes, scales, [5], np.full_like(one, np.inf), "int8")
    assert np.isnan(scales[1, 0])
    oracle.append(codes, scales, [6, -1, 8], np.ones((3, 1, 16)), "int8")
    assert np.isnan(scales[1, 0]) and scales[0, 0] == 0
    oracle.append(codes, scales, [4], one, "int8")
    assert scales[1, 0] == 2.0 ** -6


def test_attention_of_one_position_is_its_value():
    rng = np.random.default_rng(0)
    k, v = rng.integers(-5, 6, (2, 3, 4, 2, 16)).astype(np.float64)
    scales = np.full((3, 2), 0.5)
    q = rng.standard_normal((2, 4, 16))
    out, around, _, peak = oracle.attention(q, k, v, scales, scales, [[2, 1], [-1, 0]], [1, 4],
                                      [0, 1, 2], 0.25)
    np.testing.assert_array_equal(out[0], np.repeat(v[2, 0] * 0.5, 2, axis=0))
    assert (peak[0] == 0.5).all()
    assert not out[1].any() and not around[1].any()  # its only block is not there
