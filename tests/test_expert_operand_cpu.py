"""The activation operand of the experts' products, without a GPU: what fp16 hi + lo of a scaled row keep."""
import numpy as np

TOP, SPREAD = 14, 9  # rows are scaled below 2^(TOP + 1); blocks within 2^SPREAD of the loudest


def _parts(v):
    hi = v.astype(np.float16)
    lo = (v - hi.astype(np.float32)).astype(np.float16)
    return hi.astype(np.float64) + lo.astype(np.float64)


def test_hi_and_lo_hold_every_value_of_the_range():
    """A block whose largest element has an exponent at most SPREAD below the row's: every value code * dx, scaled, to
    2^-23 of itself; past that range the smallest codes are worse."""
    rng = np.random.default_rng(0)
    worst = {}
    for gap in (0, 4, SPREAD, SPREAD + 5):
        # the block's largest is at least 2^(TOP - gap)
        amax = np.concatenate([[2.0 ** (TOP - gap)], 2.0 ** (TOP - gap + rng.random(4000))]).astype(np.float32)
        dx = (amax / np.float32(127)).astype(np.float32)[:, None]
        v = dx * np.arange(1, 129, dtype=np.float32)
        assert (v < 65504).all()
        worst[gap] = (np.abs(_parts(v) - v) / v).max()
    assert all(worst[g] <= 2.0 ** -23 for g in (0, 4, SPREAD))
    assert worst[SPREAD + 5] > 2.0 ** -23


def test_the_sums_of_minima_stay_in_range():
    """dx * (sum of a block's codes) * 2^-5, of the loudest block: inside fp16."""
    dx = 2.0 ** (TOP + 1) / 127
    assert dx * 32 * 128 * 2.0 ** -5 * 4 / 3 < 65504  # (a scale rounded up among fp32's subnormals: 4 / 3 at most)


def test_sums_of_a_block_are_exact():
    """The largest sums of a block's products of whole numbers stay below 2^24."""
    assert 32 * 128 * max(128 * 32, 127, 31 * 63) <= 2 ** 24
