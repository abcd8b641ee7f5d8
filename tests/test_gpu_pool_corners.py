"""Corners of the operators over the fp16 page pool on the GPU, against plain float64 forms.  Tolerances are those that
test_gpu_pool_ops.py derives."""
import weakref

import numpy as np
import pytest
import torch

import pool_plain as P
from rstr import hip
from test_gpu_pool_ops import (HEADS, TYPES, Pooled, _attend, _attn_tol, _filled, _i32, _laid, _near, _own, _rope_tol, _select, _some_rows,  # noqa: F401
                               _table, sess)

pytestmark = pytest.mark.gpu

SHAPES = [(64, 8, 2, 12), (128, 4, 1, 16), (256, 4, 2, 16)]  # head dim, heads, kv heads, page


# ---- rotated append --------------------------------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [5, 2050])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norms_of_the_largest_and_smallest_rows(sess, D, rows, dtype):  # noqa: F811
    """Rows whose norm's factor is no normal fp32 number; those of zeros (the second of five in bf16 too) are no numbers without an epsilon."""
    rng = np.random.default_rng(D)
    n_q, n_kv, page, dt = 2, 1, 16, TYPES[dtype]
    size = torch.tensor([2.0 ** 126, 2.0 ** -149 * 1000, 2.0 ** -130, 1.0, 0.0])[torch.arange(rows) % 5][:, None, None]
    q, k = ((torch.tensor(rng.standard_normal((rows, n, D)), dtype=torch.float32).clamp(-1.9, 1.9) * size).to(dt) for n in (n_q, n_kv))
    gain = torch.tensor(rng.standard_normal(D), dtype=torch.float32)
    freqs, positions = torch.tensor(1e4 ** -(np.arange(0, D, 2) / D)), rng.integers(0, 1000, rows)
    with Pooled(sess, n_kv, D, page, rows // page + 1) as x:
        out = torch.empty_like(q, device="cuda")
        x.pool.rope_append(0, k.cuda(), k.cuda(), _i32(np.arange(rows)), _i32(positions), freqs.cuda(), q=q.cuda(), q_out=out,
                           q_gain=gain.cuda(), k_gain=gain.cuda(), eps=0.0)
        for got, y in ((out, q), (x.slab(0).reshape(-1, n_kv, D)[:rows], k)):
            with np.errstate(invalid="ignore"):
                want, mag = P.rotated(P.as_f64(y), positions, freqs.numpy(), gain.numpy())
            assert np.array_equal(np.isnan(want), np.broadcast_to((P.as_f64(y) == 0).all(-1, keepdims=True), want.shape))
            _near(got, want, np.nan_to_num(_rope_tol(got.dtype, want, mag, True)))


@pytest.mark.parametrize("D,n_q,n_kv,rot,page", [(64, 5, 2, 64, 12), (128, 8, 2, 128, 16), (128, 3, 1, 48, 16), (256, 4, 1, 256, 4), (128, 2, 2, 0, 20)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("how", ["plain", "odd"])
def test_rope_append_of_many_rows(sess, D, n_q, n_kv, rot, page, dtype, norm, how):  # noqa: F811
    """Rows enough that a workgroup takes four, the last fewer: norms, parts of a head, slots that are none, any alignment."""
    print("rope_append of many rows", D, n_q, rot, dtype, norm, how, flush=True)
    rng = np.random.default_rng(D + rot + page)
    dt, rows = TYPES[dtype], 2050
    pages = -(-(rows + 9) // page)
    q, k, v = (torch.tensor(rng.standard_normal((rows, h, D)) * 3, dtype=torch.float32).to(dt) for h in (n_q, n_kv, n_kv))
    slots = rng.permutation(pages * page)[:rows].astype(np.int64)
    gone = [3, 8, 9, 20, 2049]
    slots[gone] = [-1, pages * page, 2 ** 31 - 1, -2 ** 31, -7]
    pos = rng.integers(0, 1 << 20, rows)
    freqs = None if rot == 0 else 500000.0 ** (-np.arange(0, rot, 2) / rot)
    gains = [rng.standard_normal(D).astype(np.float32) for _ in "qk"] if norm else [None, None]
    gq, gk = (None if g is None else torch.tensor(g).cuda() for g in gains)
    with Pooled(sess, n_kv, D, page, pages) as x:
        for which in (0, 1):
            x.slab(which).fill_(7.0)
        out = _laid(torch.full((rows, n_q, D), 5.0, dtype=dt), how)
        x.pool.rope_append(0, _laid(k, how), _laid(v, how), _i32(slots), None if rot == 0 else _i32(pos),
                           None if rot == 0 else torch.tensor(freqs).cuda(), q=_laid(q, how), q_out=out, q_gain=gq, k_gain=gk, eps=1e-5,
                           gain_offset=0.5)
        y, mag = P.rotated(P.as_f64(q), pos, freqs, gains[0], 1e-5, 0.5)
        _near(out, y, _rope_tol(dt, y, mag, norm))
        y, mag = P.rotated(P.as_f64(k), pos, freqs, gains[1], 1e-5, 0.5)
        keep = np.delete(np.arange(rows), gone)
        for which, want, tol in ((0, y, _rope_tol(torch.float16, y, mag, norm)), (1, P.as_f64(v), _own(torch.float16, P.as_f64(v)))):
            got = P.as_f64(x.slab(which)).reshape(-1, n_kv, D)
            _near(got[slots[keep]], want[keep], tol[keep])
            assert (got[np.setdiff1d(np.arange(pages * page), slots[keep])] == 7.0).all()


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


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("wide", [False, True])
def test_attention_of_listed_blocks_past_32_bits(sess, dtype, wide):  # noqa: F811
    """Blocks whose first token would be 2^32 or more are behind every row, also where a list as long as the table names them."""
    rng = np.random.default_rng(5)
    n_q, n_kv, D, page, pages, dt, n = 2, 1, 64, 1 << 18, 2, TYPES[dtype], (1 << 18) + 70
    width = (1 << 14) + 3
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = (torch.tensor(rng.standard_normal((pages, 128, n_kv, D))).half() for _ in "kv")
        x.slab(0)[:, :128].copy_(k)
        x.slab(1)[:, :128].copy_(v)
        x.slab(1)[:, 128:].fill_(100.0)
        table = np.zeros((1, width), np.int64)
        table[0, 1] = 1
        # rows at the last two of the sequence's tokens, and one at its block's first
        q = torch.tensor(rng.standard_normal((70, n_q, D)), dtype=torch.float32).to(dt)
        blocks = np.full((70, n_kv, width if wide else 2), -1)
        blocks[:, 0, 0], blocks[:, 0, 1] = 1 << 14, 1
        blocks[-1, 0, 1] = (1 << 14) + 2
        out = torch.full((70, n_q, D), 5.0, dtype=dt, device="cuda")
        _attend(x, q.cuda(), table, [n], [0, 70], out, n_q, blocks=_i32(blocks))
        kk, vv = P.as_f64(k), P.as_f64(v)
        short = np.ones((70, n_kv, 1), np.int64)  # the same by pages of 128 tokens: the second one alone
        want, mag, size, seen, _ = P.attention(P.as_f64(q), kk, vv, [[0, 1]], [128 + 70], [0, 70], 0, D ** -0.5, short)
        want[-1], mag[-1] = 0.0, 0.0
        _near(out, want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max())))
        assert not out[-1].any()


@pytest.mark.parametrize("n_q,n_kv,D,page", HEADS)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lengths,news", [([1, 300, 64, 131], [1, 1, 1, 1]), ([900, 33, 0, 5000], [2, 1, 1, 2]), ([20011], [3]), ([2100], [1])])
def test_attention_of_few_rows_rounds_weights_once(sess, n_q, n_kv, D, page, dtype, lengths, news):  # noqa: F811
    """Where rows do not share tiles the sum of the weights is that of the unrounded ones: 2^-11 of each weight, whole items and joined ones."""
    rng = np.random.default_rng(n_q + D + page)
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows, dt = int(offsets[-1]), TYPES[dtype]
    pages, width = sum(-(-n // page) for n in lengths), -(-max(lengths) // page)
    table = _table(rng, lengths, page, pages, width)
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        q = torch.tensor(rng.standard_normal((rows, n_q, D)), dtype=torch.float32).to(dt)
        for window in (0, 300):
            out = torch.empty(rows, n_q, D, dtype=dt, device="cuda")
            _attend(x, q.cuda(), table, lengths, offsets, out, n_q, max_rows=max(news), window=window)
            want, mag, size, seen, _ = P.attention(P.as_f64(q), P.as_f64(k), P.as_f64(v), table, lengths, offsets, window, D ** -0.5)
            _near(out, want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max())))


@pytest.mark.parametrize("n_q,n_kv,D,page", HEADS)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("window", [1, 70, 400])
def test_attention_of_listed_blocks_in_a_window(sess, n_q, n_kv, D, page, dtype, window):  # noqa: F811
    """Of the listed blocks' tokens those in the window: for tokens, drafts and a prompt's rows; rows whose list holds none of them are 0."""
    rng = np.random.default_rng(D + window)
    lengths, news, dt = [700, 1, 300, 0], [3, 1, 150, 2], TYPES[dtype]
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows, pages, width = int(offsets[-1]), sum(-(-n // page) for n in lengths) + 1, -(-700 // page)
    table = _table(rng, lengths, page, pages, width)
    blocks = np.full((rows, n_kv, 12), -1)
    for r, (b, p) in enumerate(P.cells(table, lengths, offsets, page, pages, rows)):
        for h in range(n_kv):
            have = list(rng.permutation(max(p, 0) // page + 1))[:int(rng.integers(0, 12))]
            blocks[r, h, :len(have)] = have
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        q = torch.tensor(rng.standard_normal((rows, n_q, D)), dtype=torch.float32).to(dt)
        out = torch.full((rows, n_q, D), 5.0, dtype=dt, device="cuda")
        _attend(x, q.cuda(), table, lengths, offsets, out, n_q, max_rows=max(news), window=window, blocks=_i32(blocks))
        want, mag, size, seen, _ = P.attention(P.as_f64(q), P.as_f64(k), P.as_f64(v), table, lengths, offsets, window, D ** -0.5, blocks)
        _near(out, want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max())))


# ---- selection of blocks -----------------------------------------------------------------------
def _scores(q, lim, ids):
    """[heads][blocks] of one row and kv head by the definition: q [heads][D], lim [pages][2][D], ids [blocks]."""
    ok = (ids >= 0) & (ids < len(lim))
    lo, hi = lim[np.where(ok, ids, 0)].transpose(1, 0, 2)
    with np.errstate(invalid="ignore"):
        s = np.stack([np.maximum(x * lo, x * hi).sum(-1) for x in q])
    s = np.where(np.isnan(s).any(0), np.inf, s.max(0))
    return np.where(ok, s, -np.inf)


def _lists(q, lim, table, cells, page, top, first, last, n_kv):
    """The lists of rows that all have more blocks than these hold."""
    out = np.zeros((len(cells), n_kv, top), np.int64)
    group = q.shape[1] // n_kv
    for r, (b, p) in enumerate(cells):
        cur = p // page
        for h in range(n_kv):
            s = _scores(q[r, h * group:(h + 1) * group], lim[:, h], table[b, first:cur + 1 - last])
            best = np.argsort(-s, kind="stable")[:top - first - last]
            out[r, h] = np.concatenate([np.arange(first), first + np.sort(best), np.arange(cur + 1 - last, cur + 1)])
    return out


@pytest.mark.parametrize("n_q,n_kv,D", [(8, 2, 64), (4, 4, 128), (4, 2, 128), (12, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("wide", [1.0, 1000.0, 60000.0])
def test_select_of_blocks_that_differ_where_no_query_looks(sess, n_q, n_kv, D, dtype, wide):  # noqa: F811
    """Blocks that are alike in the bounds that the queries take, however the others differ, are equal: the first of them are taken."""
    page, pages, n, dt = 4, 400, 390, TYPES[dtype]
    g = torch.Generator().manual_seed(D + n_q)
    sign = torch.where(torch.rand(n_kv, 1, D, generator=g) < 0.5, -1.0, 1.0)  # of all heads of a group
    q = (torch.randn(2, n_kv, n_q // n_kv, D, generator=g).abs() + 0.01) * sign
    q = q.reshape(2, n_q, D).to(dt)
    with Pooled(sess, n_kv, D, page, pages) as x:
        b = x.open(hip.BlockBounds, x.pool)
        lim = torch.as_tensor(b.device(0), device="cuda")
        taken = torch.randn(n_kv, D, generator=g)
        other = torch.rand(pages, n_kv, D, generator=g) * wide
        lo = torch.where(sign[:, 0] > 0, taken - other, taken)
        hi = torch.where(sign[:, 0] > 0, taken, taken + other)
        lim.copy_(torch.stack([lo, hi], 2).half())
        table = np.random.default_rng(D).permutation(pages)[None, :n]
        for top, first, last in ((9, 1, 1), (300, 0, 2)):
            got = _select(x, b, q.cuda(), table, [n * page], [0, 2], top, first, last, n_q, n_kv).cpu().numpy()
            assert np.array_equal(got, np.broadcast_to(np.concatenate([np.arange(top - last), np.arange(n - last, n)]), got.shape))


@pytest.mark.parametrize("n_q,n_kv,D,rows", [(8, 8, 64, 40), (16, 8, 128, 41), (32, 8, 128, 40), (12, 2, 256, 160), (48, 8, 64, 33)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("pages", [1000, 1024, 700])
def test_select_for_many_rows(sess, n_q, n_kv, D, rows, dtype, pages):  # noqa: F811
    """Calls whose scores fill the card, and one just below that (700): with blocks that are gone, NaN and infinite bounds
    among the last of a wave, infinite ones that no query takes, and lists that end inside a wave's blocks."""
    print("select for many rows", n_q, n_kv, D, rows, dtype, pages, flush=True)
    if pages == 700:
        rows = 4095 // (n_kv * 11)
    page, dt, top, first, last = 4, TYPES[dtype], 40, 1, 2
    rng = np.random.default_rng(pages + D)
    lim = rng.standard_normal((pages, n_kv, 2, D)).astype(np.float32)
    q = rng.standard_normal((rows, n_q, D)).astype(np.float32)
    table = np.stack([rng.permutation(pages) for _ in range(2)])
    lim[table[0, [62, 63, 64, 65]], :, 0, 5], lim[table[0, 127], :, :, 6] = np.nan, np.nan
    lim[table[0, 128], :, 1, 7], lim[table[0, pages - 6], 0, 1, 8], lim[table[0, 300], -1, 0, 9] = np.inf, np.inf, -np.inf
    q[:, :, 8], q[0, :, 9] = 0.0, np.abs(q[0, :, 9])
    table[0, [40, 200]], table[1, [1, 64]] = [-1, pages], [2 ** 31 - 1, -7]
    lengths, offsets = [pages * page, (pages - 30) * page - 3], [0, rows // 2, rows]
    cells = P.cells(table, lengths, offsets, page, pages, rows)
    with Pooled(sess, n_kv, D, page, pages) as x:
        b = x.open(hip.BlockBounds, x.pool)
        device = torch.as_tensor(b.device(0), device="cuda")
        device.copy_(torch.tensor(lim).half())
        q = torch.tensor(q).to(dt)
        got = _select(x, b, q.cuda(), table, lengths, offsets, top, first, last, n_q, n_kv).cpu().numpy()
        want = _lists(P.as_f64(q), P.as_f64(device), table, cells, page, top, first, last, n_kv)
        assert np.array_equal(got, want), np.argwhere(got != want)[:5]


# ---- memory that is lent -------------------------------------------------------------------------
def test_tensors_keep_what_they_show(sess):  # noqa: F811
    """Tensors of pages, bounds and logits outlive their handles and the session, with their values; memory goes with the last of them."""
    g = torch.Generator().manual_seed(1)
    with hip.Session(0) as s:
        x = Pooled(s, 2, 128, 16, 300, layers=2)
        b = hip.BlockBounds(x.pool)
        view = x.pool.pages_device(1, 1)
        alive = weakref.ref(view)
        made = [torch.as_tensor(view, device="cuda"), torch.as_tensor(x.pool.pages_device(0, 0), device="cuda"), torch.as_tensor(b.device(1), device="cuda")]
        del view
        assert alive() is not None  # a tensor holds its view, which holds the memory
        values = [torch.randn(t.shape, generator=g).half() for t in made]
        for t, y in zip(made, values):
            t.copy_(y)
        torch.cuda.synchronize()
        b.close()
        x.pool.close()
        x.model.close()
    other = torch.full((64 << 20,), 7.0, device="cuda")  # would land in memory that had been freed
    for t, y in zip(made, values):
        assert torch.equal(t.cpu(), y)
        t.mul_(2.0)
        assert torch.equal(t.cpu(), y * 2.0)
    del t, made
    assert alive() is None and bool((other == 7.0).all())
