"""The plain forms that the device operators are tested against, on cases small
enough to say what the answer is."""
import numpy as np

import kv4_plain as P


def test_blocks():
    x = np.zeros(32)
    x[3], x[9], x[10] = -4.0, 2.25, 4.0
    # the first largest is -4: d = 0.5, -4 -> code 0, 4 -> clipped to 7 * 0.5, 2.25 / 0.5 = 4.5 -> 4
    want = np.zeros(32)
    want[3], want[9], want[10] = -4.0, 2.0, 3.5
    assert np.array_equal(P.quantised(x), want)
    assert np.array_equal(P.quantised(-x)[[3, 9, 10]], [4.0, -2.0, -3.5])
    x[0] = np.inf
    assert np.isnan(P.quantised(x)).all()


def test_attention_sees_its_window_only():
    k = [np.ones((5, 1, 32))]
    v = [np.arange(5.0)[:, None, None] * np.ones((5, 1, 32))]
    out, _, _ = P.attention(np.ones((2, 1, 32)), k, v, [5], [0, 2])
    assert np.allclose(out[:, 0, 0], [1.5, 2.0])
    out, _, _ = P.attention(np.ones((7, 1, 32)), k, v, [5], [0, 7], window=2)
    assert np.allclose(out[:, 0, 0], [0, 0, 0, 0.5, 1.5, 2.5, 3.5])


def test_maps():
    got = P.step_maps(4, [3, 4, 0, 8], [2, 1, 0, 3], None, [70, 71], [[10, -1, -1], [11, -1, -1], [-1] * 3, [12, 13, -1]], 6)
    assert got["offsets"] == [0, 2, 3, 3, 3] and got["taken"] == [2] and got["new_lengths"] == [5, 5, 0, 8]
    assert got["slots"] == [43, 280, 284, -1, -1, -1] and got["positions"] == [3, 4, 4, 0, 0, 0]


def test_verify():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.1, 0.8]]))
    q = np.array([[0.25, 0.75, 0.0], [1.0, 0, 0]], np.float32)
    run = lambda d, ua, us, probs=q: [a.tolist() for a in P.verify(x, [0, 2], [d, 0], probs, [1.0], [ua, 0.9], [us])]  # noqa: E731
    assert run(0, 0.99, 0.15) == [[1], [0, 1]]    # p / q = 2: accepted whatever u is; then from p: 0.1 <= 0.15 < 0.2
    assert run(1, 0.4, 0.6) == [[0], [2, -1]]     # p / q = 1/3 < 0.4: from (0.25, 0, 0.25)
    assert run(1, 0.3, 0.6) == [[1], [1, 2]]
    assert run(2, 0.2, 0.5, None) == [[1], [2, 2]]
    assert run(2, 0.3, 0.5, None) == [[0], [0, -1]]
    assert P.verify(x, [0, 2], [0, 9], None, [0.0], [0, 0], [0])[1].tolist() == [0, 2]
