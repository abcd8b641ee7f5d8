"""The plain forms of tests/pool_plain.py against what they are meant to say."""
import numpy as np

import pool_plain as P


def test_rotation():
    x = np.random.default_rng(1).standard_normal((3, 2, 8))
    f = np.array([1.0, 0.1, 0.01])
    y, mag = P.rotated(x, [0, 5, 7], f)
    assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 6:], x[..., 6:])
    z = (x[..., :3] + 1j * x[..., 3:6]) * np.exp(1j * np.array([0, 5, 7])[:, None, None] * f)
    assert np.allclose(y[..., :3], z.real) and np.allclose(y[..., 3:6], z.imag) and (mag >= np.abs(y) - 1e-12).all()
    n, _ = P.rotated(x, [0, 0, 0], None, np.ones(8), 0.0, 0.0)
    assert np.allclose((n * n).mean(-1), 1.0)


def test_attention_and_selection():
    rng = np.random.default_rng(2)
    k, v = rng.standard_normal((2, 6, 4, 1, 8))
    q = rng.standard_normal((3, 2, 8))
    table, lengths, offsets = [[3, 0, 5]], [9], [0, 3]
    out, *_ = P.attention(q, k, v, table, lengths, offsets)
    kk = np.concatenate([k[3], k[0], k[5]])[:, 0]
    vv = np.concatenate([v[3], v[0], v[5]])[:, 0]
    for r, p in enumerate((6, 7, 8)):
        w = np.exp(q[r, 1] @ kk[:p + 1].T)
        assert np.allclose(out[r, 1], w @ vv[:p + 1] / w.sum())
    lim = P.bounds(k, table, lengths, [0, 9], 9, np.zeros((6, 1, 2, 8)))
    assert np.array_equal(lim[5, 0, 0], k[5, 0, 0]) and np.array_equal(lim[0, 0, 1], k[0, :, 0].max(0))
    for g in range(2):  # a bound is one
        assert (np.maximum(q[2, g] * lim[0, 0, 0], q[2, g] * lim[0, 0, 1]).sum() >= k[0, :, 0] @ q[2, g]).all()
    got = P.select(q, lim, table, lengths, offsets, 4, 2, 0, 1)
    assert (got[:2, 0] == [0, 1]).all() and got[2, 0, 1] == 2
    some, *_ = P.attention(q, k, v, table, lengths, offsets, blocks=got)
    assert np.allclose(some[:2], out[:2])


def test_rows_without_a_place():
    assert P.cells([[0]], [3], [2, 1], 4, 1, 2) == [None, None]
    assert P.cells([[0]], [3], [1, 9], 4, 1, 3) == [None, (0, 1), (0, 2)]
    assert P.cells([[0], [0]], [1, 0], [0, 2, 3], 4, 3, 3) == [(0, -1), (0, 0), (1, -1)]
