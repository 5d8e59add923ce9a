"""Layer norm and AdamW of arrays and distances that take more than 32 bits, and steps of the block's layers that a graph replays."""
import numpy as np
import pytest

from test_gpu_block_layers import attend_case, chx, norm_case, up  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
@pytest.mark.parametrize('cols', [5, 650, 40000])
def test_layer_norm_of_rows_far_apart(chx, cols, dtype):  # noqa: F811
    """Rows more than 2^32 elements from one another, forwards and backwards in memory."""
    x, gamma, beta, gy = norm_case(3, cols, dtype, 'float32')
    gamma, beta = up(chx, gamma), up(chx, beta)
    want, state = chx.layer_norm(up(chx, x), gamma, beta)
    grads = chx.layer_norm_grad(up(chx, x), gamma, up(chx, gy), state)
    item = np.dtype(dtype).itemsize
    pitch = ((1 << 32) + 3) * item
    buffer = chx._array.alloc_bytes(2 * pitch + (1 << 20))
    far = []
    for a, first, step in ((x, 0, pitch), (gy, 2 * pitch + (1 << 19), -pitch)):
        far.append(chx.ndarray(buffer, first, a.shape, (step, item), np.dtype(dtype)))
        chx.routines._copy_into(far[-1], up(chx, a))
    y, far_state = chx.layer_norm(far[0], gamma, beta)
    for got, w in zip([y, far_state.mean, far_state.inv_std] + list(chx.layer_norm_grad(far[0], gamma, far[1], far_state)), [want, state.mean, state.inv_std] + list(grads)):
        assert np.array_equal(got.get(), w.get())


def test_layer_norm_of_more_than_32_bits_of_elements(chx):  # noqa: F811
    """One row, repeated: 2^32 results and more, all alike."""
    rows, cols = (1 << 21) + 3, 2048
    x, gamma, beta, gy = norm_case(1, cols, 'float16', 'float32')
    gamma, beta = up(chx, gamma), up(chx, beta)
    want, state = chx.layer_norm(up(chx, x), gamma, beta)
    want_gx = chx.layer_norm_grad(up(chx, x), gamma, up(chx, gy), state)[0]
    many = up(chx, x).broadcast_to((rows, cols))
    y, states = chx.layer_norm(many, gamma, beta)
    for row in (0, rows // 2, (1 << 21) - 1, 1 << 21, rows - 1):
        assert np.array_equal(y[row:row + 1].get(), want.get())
    assert (states.mean.get() == state.mean.get()[0]).all() and (states.inv_std.get() == state.inv_std.get()[0]).all()
    del y
    gx = chx.layer_norm_grad(many, gamma, up(chx, gy).broadcast_to((rows, cols)), states)[0]
    for row in (0, rows // 2, (1 << 21) - 1, 1 << 21, rows - 1):
        assert np.array_equal(gx[row:row + 1].get(), want_gx.get())


def test_adamw_of_more_than_32_bits_of_elements(chx):  # noqa: F811
    n = (1 << 32) + 300
    p, few = chx.zeros((n,), 'float16'), chx.zeros((600,), 'float16')
    grad = chx.ones((n,), 'float16')
    states = [chx.adamw_state(p), chx.adamw_state(few)]
    chx.adamw_update([p, few], [grad, grad[:600]], states, 1, alpha=0.1)
    want = few.get()
    assert (want == want[0]).all() and want[0] != 0
    for first in (0, (1 << 31) - 300, n - 600):
        assert np.array_equal(p[first:first + 600].get(), want)
        for a, b in ((states[0].m, states[1].m), (states[0].v, states[1].v)):
            assert np.array_equal(a[first:first + 600].get(), b.get())


@pytest.mark.parametrize('dtype', ['float16', 'float32'])
def test_tokens_replay_in_a_graph(chx, dtype):  # noqa: F811
    """A server's step, the state moved forward in place: each replay takes the next token."""
    from chainer_amd import graph
    c = attend_case((3, 12, 4, 2, 40, 50), dtype)
    tokens = [[up(chx, c[k][:, t:t + 1]) for k in ('q', 'k', 'v')] + [up(chx, c['log_decay'][:, t:t + 1])] for t in range(12)]
    now = [up(chx, a.get()) for a in tokens[0]]
    state, eager = up(chx, c['state']), up(chx, c['state'])
    captured = graph.capture(lambda: chx.linear_attention(*now, state=state, out_state=state))
    chx.routines._copy_into(state, eager)  # (the passes before the capture were steps, too)
    for token in tokens:
        for a, b in zip(now, token):
            chx.routines._copy_into(a, b)
        captured.replay()
        chx.synchronize()
        y, eager = chx.linear_attention(*token, state=eager)
        assert np.array_equal(captured.result[0].get(), y.get()) and np.array_equal(state.get(), eager.get())
    captured.release()


def test_gradients_of_shared_heads_replay_in_a_graph(chx):  # noqa: F811
    """float16, time in segments, padded, one decay for a head: what adds up over heads, rows and sequences, replayed with other inputs between eager calls."""
    from chainer_amd import graph
    cases = [attend_case((2, 900, 4, 2, 64, 40), 'float16', seed=i, decay='heads') for i in range(3)]
    names = ('q', 'k', 'v', 'gy', 'log_decay', 'state', 'gnew')
    now, lengths = {k: up(chx, cases[0][k]) for k in names}, up(chx, np.array([900, 517], np.int32))
    x, gamma, beta, gy = norm_case(300, 650, 'float16', 'float32')
    x, gamma, beta, gy = (up(chx, a) for a in (x, gamma, beta, gy))

    def step(a):
        more = dict(log_decay=a['log_decay'], state=a['state'], lengths=lengths)
        y, new = chx.linear_attention(a['q'], a['k'], a['v'], **more)
        n, stats = chx.layer_norm(x, gamma, beta)
        return [y, new, n] + list(chx.linear_attention_grad(a['q'], a['k'], a['v'], a['gy'], gnew_state=a['gnew'], **more)) + list(chx.layer_norm_grad(x, gamma, gy, stats))

    captured = graph.capture(lambda: step(now))
    for i in (0, 1, 2, 1):
        for k in names:
            chx.routines._copy_into(now[k], up(chx, cases[i][k]))
        want = [a.get() for a in step({k: up(chx, cases[i][k]) for k in names})]
        captured.replay()
        chx.synchronize()
        for got, w in zip(captured.result, want):
            assert np.array_equal(got.get(), w, equal_nan=True) and np.isfinite(w).all()
    captured.release()
