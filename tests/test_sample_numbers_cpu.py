"""Random numbers of 64 bits on their way to f32 (CPU only)."""

import numpy as np

from tvara_amd.sampling import f32_below_one


def test_numbers_below_one_stay_below_one():
    last = np.nextafter(np.float32(1), np.float32(0))
    given = [0.0, 0.25, 1 - 2.0 ** -24, 1 - 2.0 ** -25, 1 - 2.0 ** -26, np.nextafter(1.0, 0.0)]
    got = f32_below_one(given)
    assert got.dtype == np.float32 and got.tolist() == [0.0, 0.25, last, last, last, last]
    assert f32_below_one(np.array(given, np.float32)).tolist() == [0.0, 0.25, last, 1.0, 1.0, 1.0]  # (ones as they came)


def test_numbers_out_of_range_stay_out_of_range():
    got = f32_below_one([1.0, 1.5, -0.5, np.inf, np.nan, 1 + 2.0 ** -40])
    assert got[:4].tolist() == [1.0, 1.5, -0.5, np.inf] and np.isnan(got[4]) and got[5] == 1
    assert f32_below_one([]).shape == (0,) and f32_below_one(0.5).shape == ()
