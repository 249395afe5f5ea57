"""The 4-bit oracle against closed forms and against a plain arithmetic statement of the
rounding, and the rotation's oracle against complex products."""
import numpy as np
import pytest

from oracle import fp4, rope


def test_code_values():
    want = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    assert [fp4.e2m1_value(c) for c in range(16)] == want + [-w for w in want]


@pytest.mark.parametrize("y,want", [
    (0.25, 0), (0.75, 1), (1.25, 1), (1.75, 2), (2.5, 2), (3.5, 4), (5, 4), (0.26, 0.5),
    (0.74, 0.5), (1.76, 2), (2.49, 2), (5.01, 6), (6.9, 6), (7.9, 6)])
def test_ties_go_to_the_even_code(y, want):
    for sign in (1, -1):
        code = fp4.nearest_code(np.array([sign * y]))[0]
        assert fp4.e2m1_value(int(code)) == sign * want


@pytest.mark.parametrize("most,e", [
    (0.0, -120), (1e-38, -120), (7.0, 0), (7.0 + 2.0 ** -5, 1), (6.0, 0), (3.5, -1), (3.53125, 0),
    (1.0, -2), (7 * 2.0 ** -120, -120), (7.03125 * 2.0 ** -120, -119), (3.3895313892515355e38, 125)])
def test_scales(most, e):
    assert fp4.scale_exponent(most) == e


def test_rows_read_back_within_half_a_step():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((40, 256))
    rows = fp4.quantize_rows(x)
    assert rows.shape == (40, fp4.ROW)
    got = fp4.values(rows)
    scale = 2.0 ** (rows[:, 128:].astype(np.float64) - 127)
    # the widest step is 2 (between 4 and 6, and from 6 up to 7)
    assert (np.abs(got - x).reshape(40, 8, 32) <= scale[..., None]).all()
    again = fp4.values(fp4.quantize_rows(got))
    assert np.array_equal(again, got)  # values of the pool are kept as they are


def test_the_even_dim_is_in_the_low_half():
    x = np.zeros((1, 256))
    x[0, 0], x[0, 1], x[0, 40] = 6.0, -1.0, 3.0
    rows = fp4.quantize_rows(x)[0]
    assert rows[0] == 0x7 | 0xA << 4 and rows[20] == 7 and rows[128] == 127 and rows[129] == 126


def test_not_finite_blocks_read_back_as_nan():
    x = np.ones((1, 256))
    x[0, 5], x[0, 70] = np.inf, np.nan
    rows = fp4.quantize_rows(x)
    got = fp4.values(rows)[0]
    assert np.isnan(got[:32]).all() and np.isnan(got[64:96]).all()
    assert (got[32:64] == 1).all() and (rows[0, :16] == 0).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_is_a_complex_product(interleaved):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((5, 3, 64))
    pos = np.array([0, 1, 7, 1000, 262143])
    freq = 1e4 ** (-np.arange(0, 32, 2) / 32)
    got, _ = rope.norm_rope(x, pos, freq, rope_scale=1.5, interleaved=interleaved)
    a, b = (x[..., 0:32:2], x[..., 1:32:2]) if interleaved else (x[..., :16], x[..., 16:32])
    z = (a + 1j * b) * 1.5 * np.exp(1j * pos[:, None] * freq)[:, None]
    want = x.copy()
    if interleaved:
        want[..., 0:32:2], want[..., 1:32:2] = z.real, z.imag
    else:
        want[..., :16], want[..., 16:32] = z.real, z.imag
    assert np.allclose(got, want, rtol=0, atol=1e-9)


def test_norm_gives_unit_mean_squares():
    x = np.random.default_rng(3).standard_normal((4, 2, 128)) * 7
    got, _ = rope.norm_rope(x, np.arange(4), np.ones(8), weight=np.zeros(128), eps=0.0,
                            zero_centered=True)
    assert np.allclose((got * got).mean(-1), 1)
