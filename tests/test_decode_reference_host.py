"""The references of the decoding step's tests against numbers worked out by hand, without a GPU."""
import math

import numpy as np
import pytest

import decode_tokens_reference as R


@pytest.mark.parametrize("interleaved,frequencies,want", [
    # two pairs, both a quarter of a turn further by position 3: (1, 0) -> 2 (0, 1), (5, 2) -> 2 (-2, 5)
    (True, [math.pi / 6, math.pi / 6], [0.0, 2.0, -4.0, 10.0, 7.0]),
    # pairs (1, 5) and (0, 2), the first a quarter of a turn, the second not turned: 2 (-5, 1), 2 (0, 2)
    (False, [math.pi / 6, 0.0], [-10.0, 0.0, 2.0, 4.0, 7.0]),
])
def test_rotation_by_hand(interleaved, frequencies, want):
    x = np.array([[[1.0, 0.0, 5.0, 2.0, 7.0]]])
    got, off = R.rotate(x, np.array([3]), frequencies, interleaved, 2.0)
    assert np.allclose(got, [[want]], rtol=0, atol=1e-14) and (off[..., 4] == 0).all()
    back, _ = R.rotate(got, np.array([3]), frequencies, interleaved, 0.5, inverse=True)
    assert np.allclose(back, x, rtol=0, atol=1e-14)
