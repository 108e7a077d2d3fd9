"""The 8-bit format's oracle against torch's own e4m3 / E8M0 types, and against its definition."""
import numpy as np
import pytest
import torch

from oracle import fp8_ref


def test_codes_are_torchs():
    codes = torch.arange(256, dtype=torch.uint8)
    np.testing.assert_array_equal(fp8_ref.E4M3, codes.view(torch.float8_e4m3fn).double().numpy())


def test_scale_bytes_are_torchs():
    e = torch.arange(1, 255, dtype=torch.uint8)
    v = fp8_ref.values(np.full((254, 1, 1, 1), 0x38, np.uint8), e.numpy().reshape(254, 1, 1))  # (0x38: 1.0)
    np.testing.assert_array_equal(v.reshape(-1), e.view(torch.float8_e8m0fnu).double().numpy())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_16_bit_value_rounds_as_torch_rounds_it(dtype):
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[x.isfinite() & (x.abs() <= 448)]
    rows = torch.stack([torch.full_like(x, 448.0), x], dim=-1)  # (448: the scale is 1)
    codes, scales = fp8_ref.quantise(rows.double().numpy())
    assert (scales == 127).all()
    np.testing.assert_array_equal(codes[:, 1], x.float().to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_scale_is_the_smallest_power_of_two_that_fits():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((500, 8)) * 2.0 ** rng.integers(-120, 100, (500, 1))
    x[0], x[1, 0] = 0.0, 448.0 * 2.0 ** 5
    x[1, 1:] = 1.0
    x[2, 0], x[2, 1:] = np.nextafter(448.0, 500.0), 1.0
    _, s = fp8_ref.quantise(x)
    amax, scale = np.abs(x).max(-1), 2.0 ** (s.astype(float) - 127)
    assert (amax <= 448 * scale).all()
    assert ((amax > 224 * scale) | (s == 1)).all()
    assert s[0] == 1 and s[1] == 132 and s[2] == 128


def test_written_again_its_values_are_the_same():
    rng = np.random.default_rng(4)
    x = rng.standard_normal((64, 32)) * 2.0 ** rng.integers(-20, 20, (64, 1))
    c, s = fp8_ref.quantise(x)
    v = fp8_ref.E4M3[c] * 2.0 ** (s.astype(float) - 127)[:, None]
    c2, s2 = fp8_ref.quantise(v)  # (a maximum rounded down to 224 s fits s / 2 too: other codes, the same values)
    np.testing.assert_array_equal(fp8_ref.E4M3[c2] * 2.0 ** (s2.astype(float) - 127)[:, None], v)


def test_what_is_not_finite_is_nan_and_leaves_the_scale_alone():
    c, s = fp8_ref.quantise(np.array([[np.inf, 1.0, -np.inf, np.nan]]))
    assert s[0] == 127 - 8 and c[0, 1] == 0x78  # (1 = 2^8 * 2^-8: code of 256)
    assert np.isnan(fp8_ref.E4M3[c[0, [0, 2, 3]]]).all()
