"""Single rows of so many sequences that a thread takes two of them: the same bits as few sequences at a time, and within the bounds."""
import numpy as np
import pytest

import sequence_bounds as bounds
from test_gpu_sequence_layers import scan_case, up

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def chx():
    import chainer_amd
    return chainer_amd


def device_units():
    import torch
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('batch,states,groups', [(128, 1, None), (129, 5, 1), (128, 16, 2), (129, 16, None), (129, 64, 2), (131, 24, None)])
def test_selective_scan_of_many_single_rows(chx, batch, states, groups, dtype):
    channels = 2050
    assert batch // 2 * channels * 4 >= device_units() * 1024 > 8 * channels * 4  # two to a thread, and one where there are 16
    c, _, _ = scan_case(batch, 1, channels, states, groups, dtype, seed=states)
    for variant, (without, ragged, in_place) in enumerate((((), False, False), (('d', 'state'), True, False), (('z',), True, True), (('delta_bias',), False, True))):
        lengths = None
        if ragged:  # pairs of either kind, and two empty ones
            lengths = np.array([1, 0, 0, 1, 1, 1, 0, 0] * (batch // 8 + 1))[:batch].astype(np.int64 if variant == 1 else np.int32)
        v = {k: None if k in without else a.copy() for k, a in c.items()}
        if ragged:
            for k in ('u', 'delta', 'b', 'c', 'z'):
                if v[k] is not None:
                    v[k][lengths == 0] = np.nan
        dev = {k: up(chx, a) for k, a in v.items()}
        ends, state = up(chx, lengths), dev['state']
        if in_place:
            state = chx.array(v['state'])
        y, new = chx.selective_scan(delta_softplus=True, lengths=ends, out_state=state if in_place else None, **dict(dev, state=state))
        assert not in_place or new is state
        y, new = y.get(), new.get()
        for first in range(0, batch, 16):
            part = {k: a if a is None or k in ('a', 'd', 'delta_bias') else a[first:first + 16] for k, a in dev.items()}
            few, few_new = chx.selective_scan(delta_softplus=True, lengths=None if ends is None else ends[first:first + 16], **part)
            assert np.array_equal(few.get(), y[first:first + 16]) and np.array_equal(few_new.get(), new[first:first + 16]), first
        if ragged:
            assert not y[lengths == 0].any() and np.array_equal(new[lengths == 0], v['state'][lengths == 0] if v['state'] is not None else np.zeros_like(new[lengths == 0]))
        some = [0, 1, 2, 3, 6, batch - 2, batch - 1]  # pairs, and the last ones, whole in all channels
        few = {k: a if a is None or k in ('a', 'd', 'delta_bias') else a[some] for k, a in v.items()}
        wants = bounds.selective_scan(few, True, None if lengths is None else lengths[some])
        bounds.assert_close(y[some], *wants['y'], 'y')
        bounds.assert_close(new[some], *wants['state'], 'state')
