"""CPU tests: a call that is refused asks for no workspace first, so that it ends in its own error rather than for want of memory."""
import ctypes

import pytest

from test_sequence_layers import F16, F32, described


def sizes(x, w):
    from chainer_amd import _lib
    return _lib.load().hipcx_causal_conv_grad_workspace_size(ctypes.byref(x), ctypes.byref(w))


def scan_sizes(u, a, b):
    from chainer_amd import _lib
    lib, refs = _lib.load(), [ctypes.byref(v) for v in (u, a, b)]
    return lib.hipcx_selective_scan_workspace_size(*refs[:2]), lib.hipcx_selective_scan_grad_workspace_size(*refs)


def test_arguments_that_fit_have_workspaces():
    assert sizes(described((8, 2048, 2048)), described((2048, 4))) > 0
    assert min(scan_sizes(described((1, 16384, 2048), F16), described((2048, 16)), described((1, 16384, 16), F16))) > 0


@pytest.mark.parametrize('w', [(4, 2048), (2048, 9), (2048, 0), (2047, 4), (2048,)])
def test_causal_conv_grad(w):
    assert sizes(described((8, 2048, 2048)), described(w)) == 0


def test_causal_conv_grad_of_other_types():
    assert sizes(described((8, 2048, 2048), 9), described((2048, 4), 9)) == 0


@pytest.mark.parametrize('u,a,b', [((1, 16384, 2048), (16, 2048), (1, 16384, 16)), ((1, 16384, 2048), (2048, 65), (1, 16384, 65)), ((1, 16384, 2048), (2048, 0), (1, 16384, 0)),
                                   ((1, 16384, 2048), (2047, 16), (1, 16384, 16)), ((1, 64, 1 << 24), (1 << 24, 16), (1, 64, 16)), ((1, 64, 1 << 33), (1 << 33, 16), (1, 64, 16)),
                                   ((1, 1 << 30, 64), (64, 16), (1, 1 << 30, 16)), ((16384, 2048), (2048, 16), (1, 16384, 16))])
def test_selective_scan(u, a, b):
    assert scan_sizes(described(u, F32), described(a), described(b, F32)) == (0, 0)


@pytest.mark.parametrize('b', [(1, 16384, 17), (1, 16383, 16), (2, 16384, 16), (1, 16384, 3, 16), (1, 16384, 0, 16), (16384, 16)])
def test_selective_scan_grad(b):
    assert scan_sizes(described((1, 16384, 2048)), described((2048, 16)), described(b))[1] == 0
