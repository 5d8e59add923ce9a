"""Layer norm's means, which its second sum is to make better, not worse."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def chx():
    import chainer_amd
    return chainer_amd


@pytest.mark.parametrize('dtype', ['float16', 'float32', 'float64'])
@pytest.mark.parametrize('cols', [7, 100, 250, 650, 1023, 2500, 5000, 11000, 20001])
def test_means_of_rows_whose_sums_are_exact(chx, cols, dtype):
    """Values of few bits, whose sums no order rounds: what is left is a division and an addition, each within half a step, 2^-24 (2^-53) of a number no larger than the mean.  Differences from a
    mean of all its bits would be rounded, those of values of one power of two all alike.

    Multiples of 2^-10 below 2^-1 in size: sums of 20001 are multiples below 400 / 1024 * 20001 = 2^12.94, 23 bits.  Rows beside 1: differences from a mean, cut or not, are below 2^-7 in size and
    exact; their sum passes through at most 40 additions in a thread and 10 behind, each within half a step of a result no larger than the sum of its terms' sizes, so that their mean is off by less
    than 50 * 2^-7 half steps of 1."""
    rng = np.random.default_rng(cols)
    around = rng.integers(-400, 401, (40, cols)) / 1024
    beside = 1 + rng.integers(-3, 4, (40, cols)) / 1024
    half = 2.0 ** -53 if dtype == 'float64' else 2.0 ** -24
    for x in (around, beside, -beside):
        _, state = chx.layer_norm(chx.array(x.astype(dtype)))
        want = x.astype(np.longdouble).mean(1)
        off = abs(state.mean.get().astype(np.longdouble) - want)
        assert (off <= (2.5 if x is not around else 2) * half * abs(want) * (1 + 2.0 ** -9)).all(), float((off / abs(want)).max() / half)


@pytest.mark.parametrize('dtype', ['float32', 'float64'])
@pytest.mark.parametrize('cols', [7, 333, 2500, 20001])
def test_deviations_of_rows_far_from_zero(chx, cols, dtype):
    """The values spread by less than 2^-11 of their mean: a variance of differences from less than the whole mean would lose that many bits twice.

    Differences from a mean that is off by some last places are exact.  Their squares' rounding and up to 50 additions are 51 half steps of the variance; the square of their mean, which is 50 half
    steps of the values at most, below a tenth of the deviation, and its subtraction 3 more at most; the root takes half of these, and rounds, as the division does: 29, and what is of second order."""
    rng = np.random.default_rng(cols)
    u = 2.0 ** -53 if dtype == 'float64' else 2.0 ** -24
    for size, step in ((30001.0, 2.0 ** -7), (-777.7, 2.0 ** -10), (3.0e4 + 5, 2.0 ** -4)):
        x = (size + step * rng.integers(-300, 301, (20, cols))).astype(dtype)
        _, state = chx.layer_norm(chx.array(x), eps=0.0)
        wide = x.astype(np.longdouble)
        d = wide - wide.mean(1, keepdims=True)
        want = 1 / np.sqrt((d * d).mean(1))
        assert (abs(state.inv_std.get() - want) <= 30 * u * want).all()
