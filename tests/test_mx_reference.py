"""The host definitions that the 4-bit and optimizer kernels are held to, on values worked out by hand."""
import numpy as np
import pytest

from tests import mx_reference as ref


def test_block_of_known_values():
    x = np.zeros(32)
    x[:12] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5.01, 7.9, 0.2500001, -0.1]
    want = [6, 0, 1, 1, 2, 2, 4, 4, -6, 6, 0.5, -0.0]
    assert ref.mx_values(x)[:12].tolist() == want


def test_scales_of_extreme_blocks():
    tiny, huge = 2.0 ** -149, float(np.finfo(np.float32).max)
    assert ref.mx_values([tiny])[0] == 0.0                       # 2^-149 / 2^-127 is far below half of 0.5
    assert ref.mx_values([2.0 ** -128])[0] == 2.0 ** -128        # 0.5 times the smallest scale
    assert ref.mx_values([huge])[0] == 6 * 2.0 ** 125            # saturated
    assert np.isnan(ref.mx_values([1.0, np.inf])).all() and np.isnan(ref.mx_values([np.nan, 1.0])).all()
    assert ref.mx_values(np.zeros((2, 40))).tolist() == np.zeros((2, 40)).tolist()


@pytest.mark.parametrize("roots", [False, True])
def test_codes_of_moments_are_their_own_nearest(roots):
    largest = 255 if roots else 127
    codes = np.arange(256, dtype=np.uint8)
    codes[0] = largest                                            # (a block's largest magnitude is its scale)
    if not roots:
        codes[128] = 0                                            # (minus zero is zero)
    values = ref.decode(codes, [1.0], roots)
    again, scale = ref.encode(values, roots)
    assert scale[0] == 1.0 and np.array_equal(again, codes)


def test_small_moments():
    x = np.zeros(256, np.float32)
    x[:4] = [1.0, 2.0 ** -17, 2.0 ** -18, 2.0 ** -30]
    assert ref.encode(x, False)[0][:4].tolist() == [127, 0, 0, 0]
    assert ref.encode(x, True)[0][:4].tolist() == [255, 1, 1, 1]
    x[1:5] = [1.125 * 2.0 ** -17, 1.25 * 2.0 ** -16, 0.6249 * 2.0 ** -16, 0.6251 * 2.0 ** -16]  # (code 1 is 1.25 * 2^-16)
    assert ref.encode(x, False)[0][1:5].tolist() == [0, 1, 0, 1]


def test_ties_go_to_the_even_mantissa():
    x = np.zeros(256, np.float32)
    x[:5] = [1.0, 0.5 * (1 + 1 / 16), 0.5 * (1 + 3 / 16), 0.25 * (1 + 15 / 16), -0.5 * (1 + 1 / 16)]
    assert ref.decode(*ref.encode(x, False), False)[:5].tolist() == [1.0, 0.5, 0.5 * (1 + 2 / 8), 0.5, -0.5]
    x[:3] = [1.0, 0.5 * (1 + 1 / 32), 0.5 * (1 + 3 / 32)]
    assert ref.decode(*ref.encode(np.abs(x), True), True)[:3].tolist() == [1.0, 0.5, 0.5 * (1 + 2 / 16)]
