"""CPU tests of layer norm's rows: arrays whose rows are not equally far apart are refused, those that repeat along an inner axis among them."""
import pytest

from test_block_layers import F32, F64, NORM_GRAD_REFUSALS, described, errors, norm_arguments, refused  # noqa: F401

# (shape, strides in elements): an axis of rows that repeats lies inside one that moves on, or outside
UNEVEN = [((3, 4, 5), (5, 0, 1)), ((3, 4, 5), (0, 5, 1)), ((2, 3, 4, 5), (5, 0, 0, 1)), ((2, 3, 4, 5), (20, 5, 0, 1)), ((2, 3, 4, 5), (0, 20, 5, 1)), ((2, 1, 4, 5), (5, 7, 0, 1)),
          ((3, 4, 1), (4, 0, 1)), ((3, 4, 5), (5, 0, 0))]


@pytest.mark.parametrize('dtype,item', [(F32, 4), (F64, 8)])
@pytest.mark.parametrize('shape,strides', UNEVEN)
def test_layer_norm_refuses_rows_that_repeat_inside_others(shape, strides, dtype, item):
    dimension, view, dense = errors()[1], described(shape, dtype, [s * item for s in strides]), described(shape, dtype)
    stats, cols = described(shape[:-1], dtype), described(shape[-1:], dtype)
    refused('hipcx_layer_norm', dimension, *norm_arguments(False, x=view, y=dense, mean=stats, inv_std=stats, gamma=cols, beta=cols))
    for x, gy in ((view, dense), (dense, view)):
        refused('hipcx_layer_norm_grad', dimension, *norm_arguments(True, x=x, gy=gy, gx=dense, mean=stats, inv_std=stats, gamma=cols, ggamma=cols, gbeta=cols))
