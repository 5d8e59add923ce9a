"""Linear attention on the device where a segment, a row or a number is an extreme one, against plain forms (block_reference.py)."""
import numpy as np
import pytest

import block_reference as ref
from test_gpu_block_layers import attend_case, check_attend, check_attend_outputs, chx, up  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('length,heads', [(1, 1), (1, 3), (2, 1), (65, 2), (129, 1), (385, 1), (385, 2), (769, 1), (769, 4), (1153, 2)])
def test_gradients_of_a_sequence_whose_last_row_is_a_segment(chx, length, heads, dtype):  # noqa: F811
    """Time is cut into segments of whole tiles, so that one may hold a last row alone, which no decay follows: what lies behind the log decays has no part in it."""
    c = attend_case((1, length, heads, 1, 64, 64), dtype, seed=length)
    check_attend(chx, c, lambda a: up(chx, a), None, True, True, '%d rows %s' % (length, dtype))
    args = [up(chx, c[k]) for k in ('q', 'k', 'v', 'gy')]
    more = dict(state=up(chx, c['state']), gnew_state=up(chx, c['gnew']))
    want = [g.get() for g in chx.linear_attention_grad(*args, up(chx, c['log_decay']), **more)]
    for behind in (np.nan, np.inf, -3.0):
        wide = np.full((1, length + 1, heads), behind, np.float32)
        wide[:, :length] = c['log_decay']
        for got, w in zip(chx.linear_attention_grad(*args, chx.array(wide)[:, :length], **more), want):
            assert np.array_equal(got.get(), w)


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_gradients_of_padded_sequences_of_one_row(chx, dtype):  # noqa: F811
    """The batch's log decays are not a number behind each sequence's only row."""
    c = attend_case((5, 70, 2, 1, 20, 30), dtype, seed=2)
    c['lengths'] = np.array([1, 70, 0, 65, 1], np.int32)
    behind = np.arange(70) >= c['lengths'][:, None]
    for k in ('q', 'k', 'v', 'gy', 'log_decay'):
        c[k][behind] = np.nan
    check_attend(chx, c, lambda a: up(chx, a), None, True, True, dtype)


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_every_width_after_the_widest(chx, dtype):  # noqa: F811
    """Each kernel has its own share of LDS raised, whatever another has had before: 256 keys first, then fewer, forms for whole and for odd widths, with gradients and without, states alone."""
    for keys, values in ((256, 256), (256, 255), (128, 128), (128, 127), (127, 30), (64, 64), (63, 64), (3, 2)):
        for length in (70, 1100):
            c = attend_case((1, length, 1, 1, keys, values), dtype, seed=keys)
            check_attend(chx, c, lambda a: up(chx, a), None, True, True, '%d rows, %d keys, %d values' % (length, keys, values))


def test_products_of_float16_inputs_keep_the_bits_of_float32(chx):  # noqa: F811
    """The state's gradient where each element is one product, scale * gy, as q's rows are unit vectors: what is multiplied on the float16 pipe in two parts has lost no more than a rounding or two.

    The product is rounded by half a step of float32, 2^-24 of it.  Its first part, rounded to eleven bits, leaves at most 2^-11 of its power of two, a multiple of the last of 24 bits; the second
    one, of eleven bits, rounds that by half of 2^-22 at most.  Both are the same multiples and their sum has 24 bits, so that no addition rounds: 2^-24 + 2^-23.  (Parts that are cut off instead of
    rounded lose up to three times 2^-23, always towards zero.)"""
    rng = np.random.default_rng(3)
    zeros = np.zeros((1, 64, 1, 64), np.float16)
    q = np.eye(64, dtype=np.float16)[rng.permutation(64)].reshape(1, 64, 1, 64)
    gy = (rng.choice([-1, 1], (1, 64, 1, 64)) * (1 + rng.integers(0, 1024, (1, 64, 1, 64)) / 1024)).astype(np.float16)
    for scale in (0.3, 0.7):
        g = chx.linear_attention_grad(up(chx, q), up(chx, zeros), up(chx, zeros), up(chx, gy), scale=scale, state=chx.zeros((1, 1, 64, 64)))
        want = q[0, :, 0].astype(np.float64).T @ gy[0, :, 0] * np.float64(np.float32(scale))
        assert (np.abs(g.state.get()[0, 0] - want) <= 1.5 * 2.0 ** -23 * np.abs(want)).all(), scale


@pytest.mark.parametrize('length', [70, 300, 1100])
@pytest.mark.parametrize('zero,large', [('k', 'v'), ('v', 'k'), ('q', 'gy'), ('gy', 'q')])
@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_rows_of_zeros_next_to_large_numbers(chx, zero, large, length, dtype):  # noqa: F811
    """Rows that a mask has made zeros on one side and left as they are on the other, some 2^25 times the others' size: no other row has fewer bits for them."""
    c = attend_case((2, length, 2, 1, 40, 72), dtype, seed=7)
    rng = np.random.default_rng(8)
    c['v'], c['gy'], c['gnew'] = (c['v'] * 1e-3).astype(dtype), (c['gy'] * 1e-2).astype(dtype), c['gnew'] * np.float32(1e-2)
    c['q'], c['k'] = (c['q'] * 0.1).astype(dtype), (c['k'] * 0.1).astype(dtype)
    c['state'] = c['state'] * np.float32(1e-3)
    masked = rng.random((2, length, 2)) < 0.2
    masked[:, 0] = masked[:, -1] = True
    c[zero][masked] = 0
    c[large][masked] = (rng.choice([-1, 1], (masked.sum(), c[large].shape[3])) * rng.integers(20000, 60000, (masked.sum(), c[large].shape[3]))).astype(dtype)
    check_attend_outputs(chx, c, None)  # (element by element: many results are subnormal numbers of float16, whose half step, 2^-25, is no part of their norm)


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('length,row', [(70, 69), (100, 41), (900, 540), (900, 899)])
def test_an_infinite_key_stays_in_its_place(chx, length, row, dtype):  # noqa: F811
    """From its row on, in its head and sequence; in the state, in its key alone: nothing finite there, and elsewhere what is without it, but for other powers of two."""
    c = attend_case((2, length, 2, 1, 40, 70), dtype)
    args = lambda c: ([up(chx, c[k]) for k in ('q', 'k', 'v')], dict(log_decay=up(chx, c['log_decay']), state=up(chx, c['state'])))  # noqa: E731
    a, more = args(c)
    plain, plain_new = (x.get() for x in chx.linear_attention(*a, **more))
    _, (off, off_new) = ref.linear_attention(c['q'], c['k'], c['v'], c['log_decay'], None, c['state'])
    for value in (np.inf, -np.inf):
        bad = dict(c, k=c['k'].copy())
        bad['k'][1, row, 0, 17] = value
        a, more = args(bad)
        y, new = (x.get() for x in chx.linear_attention(*a, **more))
        touched, touched_new = np.zeros(y.shape, bool), np.zeros(new.shape, bool)
        touched[1, row:, 0] = touched_new[1, 0, 17] = True
        assert not np.isfinite(y[touched]).any() and not np.isfinite(new[touched_new]).any()
        for got, want, at, far, half in ((y, plain, touched, off, np.finfo(dtype).eps / 2), (new, plain_new, touched_new, off_new, 0)):
            assert (np.abs(got.astype(np.float64) - want) <= 2 * far + 2 * half * np.abs(want.astype(np.float64)) + 2.0 ** -24)[~at].all()


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_rows_of_few_numbers(chx, dtype):  # noqa: F811
    """Rows that are zeros but for one element, first, last or anywhere, and rows of zeros of both signs beside them: the first are not left out."""
    for keys, values in ((40, 72), (64, 64), (256, 30), (7, 9)):
        c = attend_case((2, 200, 2, 1, keys, values), dtype, seed=keys)
        rng = np.random.default_rng(keys)
        for name in ('q', 'k', 'v', 'gy'):
            a = c[name]
            width = a.shape[3]
            kept = rng.choice([0, 1, width - 1, width // 2, -1], a.shape[:3])
            some = np.where(kept == -1, rng.integers(0, width, a.shape[:3]), kept)
            one = np.arange(width) == some[..., None]
            a[...] = np.where(rng.random(a.shape[:3])[..., None] < 0.5, a, np.where(one, a, np.asarray(0, dtype)))
            gone = rng.random(a.shape[:3]) < 0.2
            a[gone] = np.where(rng.random((gone.sum(), width)) < 0.5, 0.0, -0.0).astype(dtype)
        check_attend(chx, c, lambda a: up(chx, a), None, True, True, '%d keys, %d values %s' % (keys, values, dtype))
        c['k'][:], c['v'][:] = 0, -0.0
        check_attend(chx, c, lambda a: up(chx, a), None, True, True, 'nothing but zeros, %d keys, %d values %s' % (keys, values, dtype))
