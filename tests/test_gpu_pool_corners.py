"""Corners of the operators over the fp16 page pool on the GPU, against plain float64 forms.  Tolerances are those that
test_gpu_pool_ops.py derives."""
import numpy as np
import pytest
import torch

import pool_plain as P
from rstr import hip
from test_gpu_pool_ops import TYPES, Pooled, _attend, _attn_tol, _filled, _i32, _near, _table, sess  # noqa: F401

pytestmark = pytest.mark.gpu

SHAPES = [(64, 8, 2, 12), (128, 4, 1, 16), (256, 4, 2, 16)]  # head dim, heads, kv heads, page


# ---- attention -----------------------------------------------------------------------------
@pytest.mark.parametrize("D,n_q,n_kv,page", SHAPES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("news,most", [([1, 1], 1), ([4, 3], 4), ([300, 90], 300)])
@pytest.mark.parametrize("listed", [False, True])
def test_attention_of_infinite_queries(sess, D, n_q, n_kv, page, dtype, news, most, listed):  # noqa: F811
    """An infinite element beside large finite ones: rows whose scores are all -infinity are 0, also where the keys of the finite
    elements are 0; rows with a score of +infinity are no number, and so are those with an infinity times 0."""
    print("infinite queries", D, dtype, news, listed, flush=True)
    rng = np.random.default_rng(D + most)
    dt, lengths, offsets, need = TYPES[dtype], [300, 300], np.concatenate([[0], np.cumsum(news)]), -(-300 // page)
    R, pages = int(offsets[-1]), 2 * -(-300 // page) + 1
    table = _table(rng, lengths, page, pages, need)
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        k[..., 3], k[..., 5] = -k[..., 3].abs() - 0.01, 0.0
        k[1, 2, :, 3] = float("-inf")
        x.slab(0).copy_(k)
        q = torch.tensor(rng.standard_normal((R, n_q, D)), dtype=torch.float32)
        q[:, :, 3], q[:, :, 5] = q[:, :, 3].abs() + 0.1, 3000.0
        q[0, 0, 3] = q[-1, 1, 3] = float("inf")
        q[R // 2, 2, 3], q[R // 2, 3, 5] = float("-inf"), float("inf")
        q, out, kw, blocks = q.to(dt), torch.empty(R, n_q, D, dtype=dt, device="cuda"), {}, None
        if listed:
            blocks = np.stack([[rng.permutation(need)[:need - 1] for _ in range(n_kv)] for _ in range(R)])
            kw["blocks"] = _i32(blocks)
        _attend(x, q.cuda(), table, lengths, offsets, out, n_q, max_rows=most, **kw)
        want, mag, size, seen, _ = P.attention(P.as_f64(q), P.as_f64(k), P.as_f64(v), table, lengths, offsets, 0, D ** -0.5, blocks)
        whole = P.as_f64(torch.nan_to_num(q.float(), posinf=1.0, neginf=1.0)), np.where(np.isfinite(P.as_f64(k)), P.as_f64(k), -1.0)
        size = P.attention(*whole, P.as_f64(v), table, lengths, offsets, 0, D ** -0.5, blocks)[2]  # of what is finite
        want[0, 0] = want[-1, 1] = mag[0, 0] = mag[-1, 1] = 0.0
        assert np.isnan(want[R // 2, 2:4]).all() and np.isnan(want).sum() == 2 * D
        vmax = float(v.abs().max())
        _near(out, want, _attn_tol(dt, D, want, mag, size, seen, vmax, prompt=most > 16))
        assert not out[0, 0].any() and not out[-1, 1].any()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 5, 300])
@pytest.mark.parametrize("scale", [0.0, -0.0])
def test_attention_of_scale_zero(sess, dtype, D, rows, scale):  # noqa: F811
    """All tokens alike: their mean; and no number where a score is 0 times an infinity, of either sign, of a key or a query."""
    rng = np.random.default_rng(D + rows)
    n_q, n_kv, page, n, dt = 4, 2, 16, 300, TYPES[dtype]
    with Pooled(sess, n_kv, D, page, 19) as x:
        k, v = _filled(x, rng, n_kv, D, page, 19)
        k[0, 3, 0, 7] = float("-inf")
        x.slab(0).copy_(k)
        q = torch.tensor(np.abs(rng.standard_normal((rows, n_q, D))) + 0.1, dtype=torch.float32)
        q[-1, 3, 5] = float("inf")
        q, out = q.to(dt), torch.empty(rows, n_q, D, dtype=dt, device="cuda")
        _attend(x, q.cuda(), np.arange(19)[None], [n], [0, rows], out, n_q, scale=scale)
        finite = torch.nan_to_num(q.float(), posinf=1.0)
        want, mag, size, seen, _ = P.attention(P.as_f64(finite), np.maximum(P.as_f64(k), -9.0), P.as_f64(v), [list(range(19))], [n], [0, rows], 0, 0.0)
        want[[r for r in range(rows) if n - rows + r >= 3], :2] = np.nan
        want[-1, 3] = np.nan
        _near(out, want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max()), prompt=rows > 16))
