"""The operators on device arrays over the fp16 page pool on the GPU, against plain float64 forms.

Tolerances, elementwise, from the roundings the kernels are allowed (half a step of fp32 is 2^-24 of a value, of
fp16 2^-11, of bf16 2^-8: finfo.eps / 2):

Rotated append: the sine and the cosine, each product and the difference are rounded to fp32: 3 * 2^-24 of the sum A
of the magnitudes of the two products; a norm adds the roundings of its factor, of the product with it, of the gain with its offset and of
that product: 4 * 2^-24 of A.  Then the output's own rounding, and below its smallest normal number half of the
steps there (fp16: 2^-25).

Attention, with W = sum of w_j |v_j| of the row (w the exact probabilities), S = the largest scale * |q| . |k_j| and N
the tokens it sees:
- a query's elements: in fp32 1.25 * 2^-21 of each (two terms of 11 bits, the first at most 2^-12 + 2^-10 short of the element, so that the
  second has its sign, and half a step of the second: 2^-11 (2^-12 + 2^-10) = 1.25 * 2^-21), and 2^-39 of the largest in all types, of which
  |q| . |k| holds at least one product with the largest |k| of that dim; taken as D * 2^-39 of S;
- a score is a sum of 32-term products: 32 terms and D / 32 products (twice that in fp32) one after the other, each addition off by
  no more than 2^-23 of the magnitudes; the difference to the reference, its product with the scale (itself rounded
  twice), the sum with the constant: 5 * 2^-24 of no more than 2 S; in all e = S * ((32 + 2 D / 32) * 2^-23 + 1.25 * 2^-21 + D * 2^-39 + 10 * 2^-24).
  A weight is off by e, their sum too: 2 e W;
- the exponential: 2^-22 of the weight, twice: 2^-21 W;
- f16 and bf16: a weight is rounded to fp16: 2^-11 W, and where many rows share tiles the weights' sum is that of the rounded ones: off by
  2^-11 of itself at most, so the quotient by as much again, 2^-10 W in all; weights below fp16's normal numbers are off by half a
  step there, 2^-25, where the largest weight is at least 2^6 (the reference lags by 2^4 at most: 2^10 / 2^4): N * 2^-31 * max|v|.
  fp32: two terms as above, 1.25 * 2^-21 W, and N * 2^-31 * 2^-11 max|v|;
- the sums over tokens: 32 terms and N / 32 products, and up to 64 pieces: (32 + N / 32 + 64) * 2^-23 W, the sum of the weights likewise;
  with more pieces than 64, p of them, a chain has N / (32 p) products and p pieces of two products at least, which is no more than N / 32 + 64
  either, and where a join scales what it has as it goes, one exponential (2^-22) for four pieces, eight products at least, of whose terms a chain
  over p pieces leaves that many unused;
- the quotient: 2 * 2^-24 W; the output's own rounding.
"""
import numpy as np
import pytest
import torch

import pool_plain as P
from rstr import configs, hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def sess():
    with hip.Session(0) as s:
        yield s


def _model(sess, n_kv, hd, layers=1):
    cfg = dict(configs.TINY_LLAMA)
    n_q = n_kv if n_kv * hd % 128 == 0 else 2 * n_kv
    cfg.update(n_layers=layers, d_model=128, d_ff=128, vocab=64, n_q=n_q, n_kv=n_kv, head_dim=hd)
    return hip.Model(sess, cfg, seed=1)


class Pooled:
    """A pool of one model, closed with its handles."""

    def __init__(self, sess, n_kv, hd, page, pages, layers=1):
        self.model = _model(sess, n_kv, hd, layers)
        self.pool = hip.Pool(self.model, page, pages)
        self.opened = []

    def slab(self, which, layer=0):
        return torch.as_tensor(self.pool.pages_device(which, layer), device="cuda")

    def open(self, cls, *args):
        self.opened.append(cls(*args))
        return self.opened[-1]

    def __enter__(self):
        return self

    def __exit__(self, *a):
        torch.cuda.synchronize()
        for x in self.opened[::-1]:
            x.close()
        self.pool.close()
        self.model.close()


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def _laid(x, how):
    """The rows x [R][H][D] on the GPU in another memory order, with the same values."""
    x = x.cuda()
    R, H, D = x.shape
    if how == "plain":
        return x
    if how == "padded":  # strides larger than the rows
        y = torch.zeros(R, H + 1, D + 8, dtype=x.dtype, device="cuda")[:, :H, :D]
    elif how == "heads_outside":
        y = torch.zeros(H, R, D, dtype=x.dtype, device="cuda").transpose(0, 1)
    else:  # an address that no vector load may use
        y = torch.zeros(R * H * (D + 1) + 1, dtype=x.dtype, device="cuda")[1:].as_strided((R, H, D), (H * (D + 1), D + 1, 1))
    y.copy_(x)
    return y


def _near(got, want, tol):
    """Elementwise within tol; not numbers where the definition has none."""
    got = P.as_f64(got)
    nan = ~np.isfinite(want)
    off = np.where(nan, 0.0, np.abs(got - np.where(nan, 0.0, want)) - tol)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (np.argwhere(np.isnan(got) != np.isnan(want))[:5], got.shape)
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    worst = np.unravel_index(np.argmax(off), off.shape)
    assert off[worst] <= 0, (worst, got[worst], want[worst], np.broadcast_to(tol, off.shape)[worst])


def _own(dtype, x):
    f = torch.finfo(dtype)
    return np.maximum(np.abs(x) * f.eps / 2, f.smallest_normal * f.eps / 2)


# ---- rotated append --------------------------------------------------------------------
def _rope_tol(dtype, y, mag, norm):
    return (7 if norm else 3) * 2.0 ** -24 * 1.001 * mag + 1.001 * _own(dtype, y)


@pytest.mark.parametrize("D,n_q,n_kv,rot,page", [(64, 5, 2, 64, 12), (128, 8, 2, 128, 16), (128, 3, 1, 48, 16), (256, 4, 1, 256, 4), (128, 2, 2, 0, 20)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("how", ["plain", "padded", "heads_outside", "odd"])
def test_rope_append(sess, D, n_q, n_kv, rot, page, dtype, norm, how):
    print("rope_append", D, n_q, n_kv, rot, page, dtype, norm, how, flush=True)
    rng = np.random.default_rng(D + rot + page)
    dt, rows = TYPES[dtype], 41
    pages = 61 // page + 2
    q, k, v = (torch.tensor(rng.standard_normal((rows, h, D)) * 3, dtype=torch.float32).to(dt) for h in (n_q, n_kv, n_kv))
    slots = rng.permutation(pages * page)[:rows].astype(np.int64)
    slots[3], slots[9], slots[20] = -1, pages * page, 2 ** 31 - 1
    pos = rng.integers(0, 1 << 20, rows)
    pos[:4] = (0, 1, 2 ** 31 - 1, -5)
    freqs = None if rot == 0 else 500000.0 ** (-np.arange(0, rot, 2) / rot)
    gains = [rng.standard_normal(D).astype(np.float32) for _ in "qk"] if norm else [None, None]
    gq, gk = (None if g is None else torch.tensor(g).cuda() for g in gains)
    with Pooled(sess, n_kv, D, page, pages, layers=2) as x:
        for which in (0, 1):
            x.slab(which, 1).fill_(7.0)
        out = _laid(torch.full((rows, n_q, D), 5.0, dtype=dt), how)
        x.pool.rope_append(1, _laid(k, how), _laid(v, how), _i32(slots), None if rot == 0 else _i32(pos),
                           None if rot == 0 else torch.tensor(freqs).cuda(), q=_laid(q, how), q_out=out, q_gain=gq, k_gain=gk, eps=1e-5,
                           gain_offset=0.5)
        y, mag = P.rotated(P.as_f64(q), pos, freqs, gains[0], 1e-5, 0.5)
        _near(out, y, _rope_tol(dt, y, mag, norm))
        y, mag = P.rotated(P.as_f64(k), pos, freqs, gains[1], 1e-5, 0.5)
        keep = np.ones(rows, bool)
        keep[[3, 9, 20]] = False
        for which, want, tol in ((0, y, _rope_tol(torch.float16, y, mag, norm)), (1, P.as_f64(v), _own(torch.float16, P.as_f64(v)))):
            got = P.as_f64(x.slab(which, 1)).reshape(-1, n_kv, D)
            _near(got[slots[keep]], want[keep], tol[keep])
            rest = np.setdiff1d(np.arange(pages * page), slots[keep])
            assert (got[rest] == 7.0).all() and not x.slab(which, 0).any()


def test_rope_append_bits_of_the_decoders(sess):
    """In fp32 without norms the pages and queries hold the bits that the decode step's own rotation gives."""
    import oracle as O
    import ctypes as C
    rng = np.random.default_rng(5)
    rows, D, n_q, n_kv, far, theta = 64, 128, 4, 2, 4096, 500000.0
    lib = O.lib()
    c, s = np.zeros((far, D // 2), np.float32), np.zeros((far, D // 2), np.float32)
    ptr = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    lib.orc_rope_table.argtypes = [C.c_double, C.c_int32, C.c_int32, C.c_void_p, C.c_void_p]
    lib.orc_rope_table(theta, D, far, ptr(c), ptr(s))
    q, k, v = (rng.standard_normal((rows, h, D)).astype(np.float32) for h in (n_q, n_kv, n_kv))
    pos = rng.integers(0, far, rows).astype(np.int32)
    want = []
    for x in (q, k):
        y = np.empty_like(x)
        lib.orc_rope.argtypes = [C.c_void_p, C.c_int32, C.c_int32, C.c_int32, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p]
        lib.orc_rope(ptr(x), rows, x.shape[1], D, ptr(pos), ptr(c), ptr(s), ptr(y))
        want.append(y)
    with Pooled(sess, n_kv, D, 16, 4) as x:
        out = torch.empty(rows, n_q, D, device="cuda")
        x.pool.rope_append(0, torch.tensor(k).cuda(), torch.tensor(v).cuda(), _i32(np.arange(rows)), _i32(pos),
                           torch.tensor(theta ** (-(2.0 * np.arange(D // 2)) / D)).cuda(), q=torch.tensor(q).cuda(), q_out=out)
        assert np.array_equal(out.cpu().numpy(), want[0])
        assert np.array_equal(x.slab(0).cpu().numpy().reshape(rows, n_kv, D), want[1].astype(np.float16))
        assert np.array_equal(x.slab(1).cpu().numpy().reshape(rows, n_kv, D), v.astype(np.float16))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_rope_append_in_place_of_one_projection(sess, dtype):
    """Queries, keys and values as views of one array, the queries turned where they are; more rows than one workgroup's."""
    rows, n_q, n_kv, D, dt = 2051, 4, 2, 128, TYPES[dtype]
    qkv = (torch.randn(rows, n_q + 2 * n_kv, D, generator=torch.Generator().manual_seed(1)) * 2).to(dt)
    freqs = 1e4 ** (-np.arange(0, D, 2) / D)
    pos = np.arange(rows) + 70000
    with Pooled(sess, n_kv, D, 16, 130) as x:
        a = qkv.cuda()
        x.pool.rope_append(0, a[:, n_q:n_q + n_kv], a[:, n_q + n_kv:], _i32(np.arange(rows)), _i32(pos), torch.tensor(freqs).cuda(), q=a[:, :n_q])
        y, mag = P.rotated(P.as_f64(qkv[:, :n_q]), pos, freqs)
        _near(a[:, :n_q], y, _rope_tol(dt, y, mag, False))
        assert torch.equal(a[:, n_q:].cpu(), qkv[:, n_q:])
        y, mag = P.rotated(P.as_f64(qkv[:, n_q:n_q + n_kv]), pos, freqs)
        _near(x.slab(0).reshape(-1, n_kv, D)[:rows], y, _rope_tol(torch.float16, y, mag, False))


def test_rope_append_numbers_at_the_ends(sess):
    """Values past fp16 become infinities, NaN and infinities stay, squares past fp32 still have a norm; far angles are NaN."""
    with Pooled(sess, 1, 64, 4, 3) as x:
        k = torch.zeros(5, 1, 64)
        k[0, 0, :4] = torch.tensor([1e6, -70000.0, 65504.0, 65519.0])
        k[1, 0, 2], k[1, 0, 40] = float("inf"), float("nan")
        k[2, 0] = 1e30
        k[3, 0, 1] = 1.0
        slots = _i32(np.arange(5))
        kc = k.cuda()
        x.pool.rope_append(0, kc, kc, slots)
        got = x.slab(0).reshape(-1, 64)[:5].cpu()
        assert torch.equal(torch.nan_to_num(got, nan=3.0), torch.nan_to_num(k[:, 0].half(), nan=3.0))
        x.pool.rope_append(0, kc, kc, slots, k_gain=torch.ones(64, device="cuda"))
        assert torch.allclose(x.slab(0).reshape(-1, 64)[2].cpu().float(), torch.ones(64), rtol=2.0 ** -11, atol=0)
        far = torch.full((32,), 1e-3, dtype=torch.float64)
        far[1] = 1e10
        x.pool.rope_append(0, kc[3:4], kc[3:4], slots[:1], _i32([1000]), far.cuda())
        row = x.slab(0).reshape(-1, 64)[0].cpu()
        assert bool(row[[1, 33]].isnan().all()) and int(row.isnan().sum()) == 2


# ---- attention ---------------------------------------------------------------------------
def _attn_tol(dtype, D, out, mag, size, seen, vmax, prompt=False):
    wide = dtype == torch.float32
    e = size * ((32 + 2 * D / 32) * 2.0 ** -23 + 1.25 * 2.0 ** -21 + D * 2.0 ** -39 + 10 * 2.0 ** -24)
    rel = 2 * e + 2.0 ** -21 + (1.25 * 2.0 ** -21 if wide else 2.0 ** -10 if prompt else 2.0 ** -11) + 2 * (96 + seen / 32) * 2.0 ** -23 + 2.0 ** -23
    lost = seen * 2.0 ** -31 * vmax * (2.0 ** -11 if wide else 1.0)
    return 1.01 * (np.nan_to_num(mag, nan=0.0, posinf=0.0) * np.nan_to_num(rel, nan=0.0, posinf=0.0) + lost) + 1.01 * _own(dtype, np.nan_to_num(out, nan=0.0, posinf=0.0, neginf=0.0))


def _filled(x, rng, n_kv, D, page, pages):
    """Random pages in the pool; their values in float64."""
    k = torch.tensor(rng.standard_normal((pages, page, n_kv, D)) * 1.2).half()
    v = torch.tensor(rng.standard_normal((pages, page, n_kv, D)) * 0.8 + 0.3).half()
    x.slab(0).copy_(k)
    x.slab(1).copy_(v)
    return k, v


def _table(rng, lengths, page, pages, width, extra=0):
    perm = list(rng.permutation(pages))
    t = np.full((len(lengths), width), -1, np.int64)
    for b, n in enumerate(lengths):
        for i in range(min(width, -(-n // page) + extra)):
            t[b, i] = perm.pop()
    return t


def _attend(x, q, table, lengths, offsets, out, n_q, plan=None, **kw):
    plan = plan or x.open(hip.PagedAttention, x.pool, n_q, len(lengths), q.shape[0])
    plan.run(0, q, _i32(offsets), _i32(table), _i32(lengths), out, **kw)
    return out


HEADS = [(8, 2, 64, 16), (8, 8, 64, 12), (8, 2, 128, 16), (24, 1, 128, 48), (4, 1, 256, 4), (6, 2, 256, 64)]


@pytest.mark.parametrize("n_q,n_kv,D,page", HEADS)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("window", [0, 1, 37])
@pytest.mark.parametrize("form", ["token", "drafts", "prompt"])
def test_attention(sess, n_q, n_kv, D, page, dtype, window, form):
    print("attention", n_q, n_kv, D, page, dtype, window, form, flush=True)
    rng = np.random.default_rng(n_q + D + page)
    lengths = [1, 0, 33, 300, 64, 2, 131]
    news = {"token": [1] * 7, "drafts": [1, 0, 4, 3, 6, 2, 5], "prompt": [1, 2, 33, 97, 40, 2, 61]}[form]  # (one with more rows than tokens)
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows, dt = int(offsets[-1]), TYPES[dtype]
    pages = sum(-(-n // page) for n in lengths) + 3
    width = -(-300 // page) + 1
    table = _table(rng, lengths, page, pages, width)
    scale = 1.7 * D ** -0.5
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        q = torch.tensor(rng.standard_normal((rows + 2, n_q, D)), dtype=torch.float32).to(dt)
        out = torch.full((rows + 2, n_q, D), 5.0, dtype=dt, device="cuda")
        _attend(x, q.cuda(), table, lengths, offsets, out, n_q, max_rows=max(news), window=window, scale=scale)
        want, mag, size, seen, mine = P.attention(P.as_f64(q), P.as_f64(k), P.as_f64(v), table, lengths, offsets, window, scale)
        assert bool((out[rows:] == 5.0).all())  # rows of no sequence
        tol = _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max()), prompt=True)
        _near(out[:rows], want[:rows], tol[:rows])
        again = torch.full_like(out, 5.0)  # max_rows chooses the tile only
        _attend(x, q.cuda(), table, lengths, offsets, again, n_q, window=window, scale=scale)
        _near(again[:rows], want[:rows], tol[:rows])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lengths,news,width_extra", [([3000, 17], [1, 1], 0), ([2500, 900], [300, 1], 5), ([1100] * 70, [1] * 70, 0), ([700], [700], 3)])
def test_attention_long(sess, dtype, lengths, news, width_extra):
    """Items that many waves share; a prompt beside a token; more sequences than lanes; a whole prompt."""
    print("attention long", dtype, lengths[:2], news[:2], flush=True)
    rng = np.random.default_rng(len(lengths) + lengths[0])
    n_q, n_kv, D, page, dt = 8, 2, 128, 16, TYPES[dtype]
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows = int(offsets[-1])
    pages = sum(-(-n // page) for n in lengths) + 1
    table = _table(rng, lengths, page, pages, -(-max(lengths) // page) + width_extra)
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        q = torch.tensor(rng.standard_normal((rows, n_q, D)), dtype=torch.float32).to(dt)
        out = torch.empty(rows, n_q, D, dtype=dt, device="cuda")
        _attend(x, q.cuda(), table, lengths, offsets, out, n_q, max_rows=max(news))
        sel = np.unique(np.concatenate([np.arange(min(rows, 3)), rng.integers(0, rows, 12), [rows - 1]]))  # the plain form of some rows
        want, mag, size, seen, _ = _some_rows(P.as_f64(q), k, v, table, lengths, offsets, sel, D ** -0.5)
        _near(out.cpu()[sel], want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max()), prompt=max(news) > 1))


def _some_rows(q, k, v, table, lengths, offsets, sel, scale, **kw):
    """P.attention of the rows `sel`, each as a sequence of its own."""
    P_, page = k.shape[0], k.shape[1]
    cells = P.cells(table, lengths, list(offsets), page, P_, q.shape[0])
    t = [table[cells[r][0]] for r in sel]
    n = [max(0, cells[r][1] + 1) for r in sel]
    return P.attention(q[sel], P.as_f64(k), P.as_f64(v), t, n, list(range(len(sel) + 1)), scale=scale, **kw)


@pytest.mark.parametrize("how", ["padded", "heads_outside", "odd"])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_strides(sess, dtype, how):
    rng = np.random.default_rng(3)
    n_q, n_kv, D, page, dt = 6, 2, 128, 16, TYPES[dtype]
    lengths, offsets = [50, 9], [0, 3, 4]
    with Pooled(sess, n_kv, D, page, 6) as x:
        k, v = _filled(x, rng, n_kv, D, page, 6)
        table = _table(rng, lengths, page, 6, 4)
        q = torch.tensor(rng.standard_normal((4, n_q, D)), dtype=torch.float32).to(dt)
        a = torch.empty(4, n_q, D, dtype=dt, device="cuda")
        b = _laid(torch.zeros(4, n_q, D, dtype=dt), how)
        _attend(x, q.cuda(), table, lengths, offsets, a, n_q)
        _attend(x, _laid(q, how), table, lengths, offsets, b, n_q)
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_what_is_not_seen(sess, dtype, D):
    """NaN and infinities behind a length, in other pages, in later tokens of the same chunk and outside a window do not reach a row; those
    that a row sees do.  Page ids outside the pool are not seen."""
    rng = np.random.default_rng(D)
    n_q, n_kv, page, dt = 4, 2, 16, TYPES[dtype]
    lengths, news = [40, 21, 90], [6, 1, 40]
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows = int(offsets[-1])
    pages = 14
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        table = _table(rng, lengths, page, pages, 8)
        table[2, 1], table[2, 3] = -1, pages  # gone
        table[1, 4] = 2 ** 31 - 1
        at = lambda b, t: (table[b, t // page], t % page)  # noqa: E731
        for b, n in enumerate(lengths):
            for t in range(n, -(-n // page) * page):
                k[at(b, t)], v[at(b, t)] = float("nan"), float("inf")
        free = np.setdiff1d(np.arange(pages), table)
        k[free], v[free] = float("nan"), float("nan")
        v[at(0, 38)][0, 5] = float("inf")     # tokens of the chunk itself
        v[at(0, 36)][1, 7] = float("nan")
        k[at(2, 85)][0, 3] = float("nan")
        v[at(2, 70)][1, 9] = float("-inf")
        v[at(2, 3)][0, 1] = float("nan")      # an early one, which a window leaves out
        x.slab(0).copy_(k)
        x.slab(1).copy_(v)
        q = torch.tensor(rng.standard_normal((rows, n_q, D)), dtype=torch.float32).to(dt)
        for window in (0, 24):
            for most in (rows, 1):
                out = torch.empty(rows, n_q, D, dtype=dt, device="cuda")
                _attend(x, q.cuda(), table, lengths, offsets, out, n_q, max_rows=most, window=window)
                want, mag, size, seen, _ = P.attention(P.as_f64(q), P.as_f64(k), P.as_f64(v), table, lengths, offsets, window, D ** -0.5)
                vmax = float(v[v.isfinite()].abs().max())
                _near(out, want, _attn_tol(dt, D, want, mag, size, seen, vmax, prompt=most > 1))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention_infinities_that_are_seen(sess, dtype):
    """Keys whose score is -infinity have no weight, one of +infinity leaves no number; infinite values give infinities of their sign."""
    rng = np.random.default_rng(21)
    n_q, n_kv, D, page, dt, n = 4, 1, 128, 16, TYPES[dtype], 70
    with Pooled(sess, n_kv, D, page, 5) as x:
        k, v = _filled(x, rng, n_kv, D, page, 5)
        q = torch.tensor(rng.standard_normal((3, n_q, D)) * 0.5, dtype=torch.float32)
        q[:, :, 3], q[1, :, 9] = q[:, :, 3].abs() + 0.1, 0.25
        k[2, 5, 0, 3] = float("-inf")
        k[0, 1, 0, 3] = float("-inf")
        v[1, 2, 0, 7], v[3, 4, 0, 8] = float("inf"), float("-inf")
        v[2, 5, 0, 1] = 3.0  # of a key without weight
        x.slab(0).copy_(k)
        x.slab(1).copy_(v)
        q = q.to(dt)
        for kw in ({}, {"blocks": _i32(np.broadcast_to(np.arange(5), (3, 1, 5)).copy())}):
            out = torch.empty(3, n_q, D, dtype=dt, device="cuda")
            _attend(x, q.cuda(), np.arange(5)[None], [n], [0, 3], out, n_q, **kw)
            want, mag, size, seen, _ = P.attention(P.as_f64(q), P.as_f64(k), P.as_f64(v), [list(range(5))], [n], [0, 3], 0, D ** -0.5)
            assert np.isinf(want).sum() == 24 and not np.isnan(want).any()
            _near(out, want, _attn_tol(dt, D, want, mag, np.where(np.isfinite(size), size, 20.0), seen, 5.0))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0, 1e-30, 1e30])
def test_attention_scales_and_sizes(sess, dtype, scale):
    """Scores of any size: scales that are 0, negative or huge, queries next to their type's largest and smallest values, and rows
    whose sizes differ beside each other."""
    rng = np.random.default_rng(9)
    n_q, n_kv, D, page, dt = 4, 2, 128, 16, TYPES[dtype]
    lengths, offsets, pages = [200, 77], [0, 2, 9], 18
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        table = _table(rng, lengths, page, pages, 13)
        q = torch.tensor(rng.standard_normal((9, n_q, D)), dtype=torch.float32)
        big, small = torch.finfo(dt).max, torch.finfo(dt).smallest_normal
        q[1] *= big / 8
        q[3] *= small
        q[4] = 0.0
        q[5, :, 7] = big
        q = q.to(dt)
        assert bool(q.isfinite().all())
        out = torch.empty(9, n_q, D, dtype=dt, device="cuda")
        _attend(x, q.cuda(), table, lengths, offsets, out, n_q, scale=scale)
        scale = float(np.float32(scale))
        want, mag, size, seen, _ = P.attention(P.as_f64(q), P.as_f64(k), P.as_f64(v), table, lengths, offsets, 0, scale)
        tol = _attn_tol(dt, D, want, mag, np.minimum(size, 2.0 ** 40), seen, float(v.abs().max()))
        one = size > 1e5  # the largest score alone decides, where it is apart from the next: checked below
        assert bool(np.isfinite(P.as_f64(out)).all())
        _near(np.where(one, 0.0, P.as_f64(out)), np.where(one, 0.0, want), tol)
        scores = _scores(P.as_f64(q), P.as_f64(k), table, lengths, offsets, scale)
        for r in range(9):
            for h in range(n_q):
                s = np.sort(scores[r][h])
                e = 2.0 ** -16 * size[r, h, 0]  # far above the scores' own rounding
                if one[r, h, 0] and s[-1] - s[-2] > 40 + e:
                    _near(out[r, h], want[r, h], tol[r, h] * 0 + _own(dt, want[r, h]) * 1.01 + np.abs(want[r, h]) * 2.0 ** -11)


def _scores(q, k, table, lengths, offsets, scale):
    page = k.shape[1]
    out = []
    for r, (b, p) in enumerate(P.cells(table, lengths, offsets, page, k.shape[0], q.shape[0])):
        j = np.arange(p + 1)
        kk = k[np.array([table[b][t // page] for t in j]), j % page]
        out.append([kk[:, h // (q.shape[1] // k.shape[2])] @ q[r, h] * scale for h in range(q.shape[1])])
    return out


def test_attention_offsets_that_decrease(sess):
    rng = np.random.default_rng(1)
    with Pooled(sess, 2, 64, 16, 8) as x:
        _filled(x, rng, 2, 64, 16, 8)
        table = _table(rng, [30, 30], 16, 8, 2)
        q = torch.randn(6, 4, 64, device="cuda")
        blocks = torch.zeros(6, 2, 1, dtype=torch.int32, device="cuda")
        for offs in ([0, 4, 2], [3, 1, 6], [5, -1, 6]):
            for kw in ({}, {"blocks": blocks}):
                out = torch.full_like(q, 5.0)
                _attend(x, q, table, [30, 30], offs, out, 4, **kw)
                assert bool((out == 5.0).all()), (offs, kw)
        for offs in ([0, 100, 200], [-7, 2, 5], [2, 2, 4]):  # clamped, or some rows of no sequence
            for kw in ({}, {"blocks": blocks}):
                out = torch.full_like(q, 5.0)
                _attend(x, q, table, [30, 30], offs, out, 4, **kw)
                mine = [c is not None for c in P.cells(table, [30, 30], offs, 16, 8, 6)]
                assert [not bool((o == 5.0).all()) for o in out] == mine, (offs, kw)


def test_attention_far_slots(sess):
    """Pages past 2^32 bytes into a slab."""
    n_q, n_kv, D, page, dt = 8, 8, 128, 16, torch.float16
    pages = (1 << 32) // (page * n_kv * D * 2) + 40
    rng = np.random.default_rng(2)
    with Pooled(sess, n_kv, D, page, pages) as x:
        n = 150
        k, v = (torch.tensor(rng.standard_normal((n, n_kv, D))).half() for _ in "kv")
        ids = np.array([pages - 1 - 3 * i for i in range(10)])
        ids[3] = 5
        t = np.arange(n)
        x.pool.rope_append(0, k.cuda(), v.cuda(), _i32(ids[t // page] * page + t % page))
        q = torch.tensor(rng.standard_normal((2, n_q, D))).to(dt)
        out = torch.empty(2, n_q, D, dtype=dt, device="cuda")
        _attend(x, q.cuda(), ids[None], [n], [0, 2], out, n_q)
        pad = np.zeros((10, page, n_kv, D))
        kp, vp = pad.copy(), pad.copy()
        kp.reshape(-1, n_kv, D)[:n], vp.reshape(-1, n_kv, D)[:n] = P.as_f64(k), P.as_f64(v)
        want, mag, size, seen, _ = P.attention(P.as_f64(q), kp, vp, [list(range(10))], [n], [0, 2], 0, D ** -0.5)
        _near(out, want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max())))
        b = x.open(hip.BlockBounds, x.pool)
        b.update(0, _i32([0, n]), _i32(ids[None]), _i32([n]), n)
        lim = torch.as_tensor(b.device(0), device="cuda")[torch.tensor(ids, device="cuda")].cpu()
        full = kp[:9]
        assert np.array_equal(P.as_f64(lim[:9, :, 0]), full.min(1)) and np.array_equal(P.as_f64(lim[:9, :, 1]), full.max(1))


def test_attention_of_the_isolated_entry(sess):
    """The same attention as rstr_attention_run over the same pool."""
    rng = np.random.default_rng(4)
    lengths = np.array([5, 300, 77], np.int32)
    with Pooled(sess, 2, 128, 16, 40) as x:
        x.pool.fill_synthetic(np.arange(40, dtype=np.int32), 3)
        torch.cuda.synchronize()
        table = _table(rng, list(lengths), 16, 40, 20)
        q = rng.standard_normal((3, 8, 128)).astype(np.float32)
        want = x.pool.attention(0, q, table, lengths, scale=0.1)
        out = torch.empty(3, 8, 128, device="cuda")
        _attend(x, torch.tensor(q).cuda(), table, lengths, [0, 1, 2, 3], out, 8, scale=0.1)
        assert np.abs(out.cpu().numpy() - want).max() <= 2.0 ** -16 * np.abs(want).max()


# ---- bounds and selection ------------------------------------------------------------------
@pytest.mark.parametrize("n_kv,D,page", [(2, 64, 12), (1, 128, 16), (3, 256, 4), (2, 128, 64)])
def test_bounds(sess, n_kv, D, page):
    rng = np.random.default_rng(page)
    lengths, news = [1, 0, 5 * page, 3 * page + 2, 2 * page - 1, 2, 7 * page], [1, 0, 2 * page + 1, 3, page, 4, 7 * page]
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows, pages = int(offsets[-1]), 30
    with Pooled(sess, n_kv, D, page, pages, layers=2) as x:
        k, _ = _filled(x, rng, n_kv, D, page, pages)
        table = _table(rng, lengths, page, pages, 7)
        table[2, 4] = pages
        k[table[3, 3], 1, 0, 3] = float("nan")
        k[table[6, 2], 2, 0, 5], k[table[6, 2], 1, 0, 5] = float("inf"), float("-inf")
        k[table[4, 1], page - 1] = float("nan")  # behind the length
        x.slab(0).copy_(k)
        b = x.open(hip.BlockBounds, x.pool)
        lim = torch.as_tensor(b.device(0), device="cuda")
        other = torch.as_tensor(b.device(1), device="cuda")
        lim.fill_(9.0)
        b.update(0, _i32(offsets), _i32(table), _i32(lengths), rows)
        want = P.bounds(P.as_f64(k), table, lengths, list(offsets), rows, np.full(tuple(lim.shape), 9.0))
        got = P.as_f64(lim)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.nan_to_num(got, nan=5.0), np.nan_to_num(want, nan=5.0))
        assert not other.any()
        lim.fill_(9.0)
        b.update(0, _i32([0, 5, 3, 3, 3, 3, 3, 3]), _i32(table), _i32(lengths), rows)
        assert bool((lim == 9.0).all())


def _select(x, bounds, q, table, lengths, offsets, top, first, last, n_q, n_kv):
    sel = x.open(hip.BlockSelect, bounds, n_q, len(lengths), q.shape[0], len(table[0]))
    out = torch.full((q.shape[0], n_kv, top), -7, dtype=torch.int32, device="cuda")
    sel.run(0, q, _i32(offsets), _i32(table), _i32(lengths), out, first=first, last=last)
    return out


@pytest.mark.parametrize("n_q,n_kv,D", [(8, 2, 64), (8, 8, 64), (8, 2, 128), (24, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("top,first,last", [(1, 0, 1), (5, 1, 1), (12, 0, 3), (4, 2, 2), (200, 1, 2)])
def test_select(sess, n_q, n_kv, D, dtype, top, first, last):
    print("select", n_q, n_kv, D, dtype, top, first, last, flush=True)
    rng = np.random.default_rng(n_q + D + top)
    page, pages, dt = 4, 330, TYPES[dtype]
    lengths, news = [1, 0, 700, 350, 47], [1, 2, 3, 5, 2]
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows = int(offsets[-1])
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, _ = _filled(x, rng, n_kv, D, page, pages)
        table = _table(rng, lengths, page, pages, 180)
        for j in (7, 8, 30, 31, 32, 60):  # blocks that are equal: the first are taken
            k[table[2, j]] = k[table[2, 6]]
        table[3, 40] = -5
        x.slab(0).copy_(k)
        b = x.open(hip.BlockBounds, x.pool)
        every = np.concatenate([[0], np.cumsum(lengths)])
        b.update(0, _i32(every), _i32(table), _i32(lengths), int(every[-1]))
        q = torch.tensor(rng.standard_normal((rows + 1, n_q, D)), dtype=torch.float32).to(dt)
        got = _select(x, b, q.cuda(), table, lengths, offsets, top, first, last, n_q, n_kv).cpu().numpy()
        lim = P.as_f64(torch.as_tensor(b.device(0), device="cuda"))
        want = P.select(P.as_f64(q), lim, table, lengths, list(offsets), page, top, first, last)
        assert np.array_equal(got, want), np.argwhere(got != want)[:5]


@pytest.mark.parametrize("dtype", list(TYPES))
def test_select_of_equal_and_odd_scores(sess, dtype):
    """All blocks alike; scores that are no numbers or infinite; zeros of both signs; one query row."""
    n_q, n_kv, D, page, pages, dt = 4, 2, 128, 4, 300, TYPES[dtype]
    n = 4 * 290
    table = np.arange(290)[None]
    with Pooled(sess, n_kv, D, page, pages) as x:
        b = x.open(hip.BlockBounds, x.pool)
        lim = torch.as_tensor(b.device(0), device="cuda")
        q = torch.randn(1, n_q, D, generator=torch.Generator().manual_seed(1)).to(dt)
        for kind in ("zeros", "ones", "nan", "inf", "mixed"):
            z = torch.zeros(pages, n_kv, 2, D)
            if kind == "ones":
                z += 1
            if kind in ("nan", "mixed"):
                z[[3, 50, 51, 200], :, :, 2] = float("nan")
            if kind in ("inf", "mixed"):
                z[[9, 70, 71], :, 1] = float("inf")
                z[[11, 72], :, 0] = float("-inf")
            if kind == "mixed":
                z[100:] = torch.randn(200, n_kv, 2, D, generator=torch.Generator().manual_seed(2))
                z[200, 1, 1, 3] = -0.0
            lim.copy_(z.half())
            for top, first, last in ((6, 1, 1), (3, 0, 1), (80, 2, 3)):
                got = _select(x, b, q.cuda(), table, [n], [0, 1], top, first, last, n_q, n_kv).cpu().numpy()
                want = P.select(P.as_f64(q), P.as_f64(lim), table, [n], [0, 1], page, top, first, last)
                assert np.array_equal(got, want), (kind, top, got[got != want], want[got != want])


def test_select_many_blocks(sess):
    """Tables of thousands of blocks, and scores that share many leading bits."""
    n_q, n_kv, D, page, pages = 2, 1, 128, 4, 9000
    g = torch.Generator("cuda").manual_seed(3)
    with Pooled(sess, n_kv, D, page, pages) as x:
        b = x.open(hip.BlockBounds, x.pool)
        lim = torch.as_tensor(b.device(0), device="cuda")
        lim.copy_(torch.randn(lim.shape, generator=g, device="cuda") * 2.0 ** -9 + 1.0)
        table = np.random.default_rng(1).permutation(pages)[None, :8777]
        q = torch.randn(3, n_q, D, generator=g, device="cuda")
        for top in (2, 100, 1025, 8000):
            got = _select(x, b, q, table, [8777 * page - 1], [0, 3], top, 1, 1, n_q, n_kv).cpu().numpy()
            want = P.select(P.as_f64(q), P.as_f64(lim), table, [8777 * page - 1], [0, 3], page, top, 1, 1)
            assert np.array_equal(got, want), top


# ---- attention over listed blocks ------------------------------------------------------------
@pytest.mark.parametrize("n_q,n_kv,D,page", HEADS)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("top", [1, 7, 60])
def test_attention_of_blocks(sess, n_q, n_kv, D, page, dtype, top):
    print("blocks", n_q, n_kv, D, page, dtype, top, flush=True)
    rng = np.random.default_rng(n_q + D + page + top)
    lengths, news = [1, 0, 333, 640, 64], [1, 1, 4, 3, 2]
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows, dt = int(offsets[-1]), TYPES[dtype]
    pages = sum(-(-n // page) for n in lengths) + 3
    width = -(-640 // page) + 1
    table = _table(rng, lengths, page, pages, width)
    table[2, 1] = pages + 3
    blocks = rng.integers(0, width, (rows + 1, n_kv, top))  # in any order, some twice, some of the future
    blocks[rng.random(blocks.shape) < 0.1] = -1
    blocks[rng.random(blocks.shape) < 0.05] = width
    blocks[rng.random(blocks.shape) < 0.05] = 2 ** 31 - 1
    blocks[0, 0, 0] = 0
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        for b, n in enumerate(lengths):  # behind the lengths
            for t in range(n, -(-n // page) * page):
                k[table[b, t // page], t % page], v[table[b, t // page], t % page] = float("nan"), float("inf")
        x.slab(0).copy_(k)
        x.slab(1).copy_(v)
        q = torch.tensor(rng.standard_normal((rows + 1, n_q, D)), dtype=torch.float32).to(dt)
        for window in (0, 50):
            out = torch.full((rows + 1, n_q, D), 5.0, dtype=dt, device="cuda")
            _attend(x, q.cuda(), table, lengths, offsets, out, n_q, blocks=_i32(blocks), window=window)
            want, mag, size, seen, _ = P.attention(P.as_f64(q), P.as_f64(k), P.as_f64(v), table, lengths, offsets, window, D ** -0.5, blocks)
            assert bool((out[rows:] == 5.0).all())
            tol = _attn_tol(dt, D, want, mag, size, seen, float(v[v.isfinite()].abs().max()))
            _near(out[:rows], want[:rows], tol[:rows])


def test_attention_of_all_blocks(sess):
    """A list of all blocks gives what no list gives."""
    rng = np.random.default_rng(6)
    n_q, n_kv, D, page, pages = 8, 2, 128, 16, 60
    lengths, offsets = [800, 100], [0, 3, 4]
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        table = _table(rng, lengths, page, pages, 50)
        q = torch.randn(4, n_q, D, device="cuda")
        a, b = torch.empty_like(q), torch.empty_like(q)
        _attend(x, q, table, lengths, offsets, a, n_q)
        every = _i32(np.broadcast_to(np.arange(50), (4, n_kv, 50)).copy())
        _attend(x, q, table, lengths, offsets, b, n_q, blocks=every)
        assert float((a - b).abs().max()) <= 2.0 ** -18


# ---- together ----------------------------------------------------------------------------------
def _step_tensors(rows, n_q, n_kv, D, dt, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(rows, n_q + 2 * n_kv, D, generator=g, device="cuda").to(dt)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("stream", ["current", "side", "session"])
def test_steps_of_a_server(sess, dtype, stream):
    """Prompts, drafts and single tokens over steps as a server runs them: maps, rotated append, bounds, selection, attention, over
    all blocks and over the selected ones; against the plain forms on what the steps put into the pool."""
    print("steps", dtype, stream, flush=True)
    n_q, n_kv, D, page, pages, width, dt, batch, top = 4, 2, 128, 16, 40, 14, TYPES[dtype], 3, 4
    freqs = torch.tensor(1e4 ** (-np.arange(0, D, 2) / D)).cuda()
    with Pooled(sess, n_kv, D, page, pages) as x:
        bounds = x.open(hip.BlockBounds, x.pool)
        plan, plan2 = (x.open(hip.PagedAttention, x.pool, n_q, batch, 160) for _ in range(2))
        sel = x.open(hip.BlockSelect, bounds, n_q, batch, 160, width)
        free = np.random.default_rng(1).permutation(pages)
        table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")
        lengths, taken = _i32([0] * batch), 0
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        st = {"current": None, "side": side, "session": hip.SESSION_STREAM}[stream]
        for i, counts in enumerate(([50, 1, 90], [1, 1, 1], [3, 0, 5], [1, 100, 1], [2, 2, 2])):
            rows = sum(counts)
            qkv = _step_tensors(rows, n_q, n_kv, D, dt, i)
            new, offs, pos, slots, got = _i32([0] * batch), _i32([0] * (batch + 1)), _i32([0] * rows), _i32([0] * rows), _i32([0])
            dense, sparse = (torch.empty(rows, n_q, D, dtype=dt, device="cuda") for _ in range(2))
            blocks = torch.empty(rows, n_kv, top, dtype=torch.int32, device="cuda")
            args = _i32(counts), _i32(free[taken:])
            torch.cuda.synchronize()
            sess.step_maps(page, lengths, args[0], args[1], table, new, offs, pos, slots, got, stream=st)
            x.pool.rope_append(0, qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:], slots, pos, freqs, q=qkv[:, :n_q], stream=st)
            bounds.update(0, offs, table, new, rows, stream=st)
            sel.run(0, qkv[:, :n_q], offs, table, new, blocks, first=1, last=1, stream=st)
            plan.run(0, qkv[:, :n_q], offs, table, new, dense, max_rows=max(counts), stream=st)
            plan2.run(0, qkv[:, :n_q], offs, table, new, sparse, max_rows=max(counts), blocks=blocks, stream=st)
            torch.cuda.synchronize()
            taken += int(got)
            lengths = new
            k, v = P.as_f64(x.slab(0)), P.as_f64(x.slab(1))
            t, n, o = table.cpu().numpy(), new.tolist(), offs.tolist()
            q = P.as_f64(qkv[:, :n_q])
            vmax = np.abs(v).max()
            lim = P.as_f64(torch.as_tensor(bounds.device(0), device="cuda"))
            for b, m in enumerate(n):  # the bounds follow the pages
                for j in range(-(-m // page)):
                    keys = k[t[b, j], :min(page, m - j * page)]
                    assert np.array_equal(lim[t[b, j], :, 0], keys.min(0)) and np.array_equal(lim[t[b, j], :, 1], keys.max(0))
            assert np.array_equal(blocks.cpu().numpy(), P.select(q, lim, t, n, o, page, top, 1, 1))
            for out, lst in ((dense, None), (sparse, blocks.tolist())):
                want, mag, size, seen, _ = P.attention(q, k, v, t, n, o, 0, D ** -0.5, lst)
                _near(out, want, _attn_tol(dt, D, want, mag, size, seen, vmax, prompt=lst is None and max(counts) > 1))


def test_a_captured_step(sess):
    """A step in a graph, replayed over changed inputs with eager work in between, equals the eager step bit for bit."""
    n_q, n_kv, D, page, pages, width, dt, rows, top = 8, 2, 128, 16, 200, 70, torch.bfloat16, 5, 6
    freqs = torch.tensor(1e4 ** (-np.arange(0, D, 2) / D)).cuda()
    rng = np.random.default_rng(8)
    lengths = [900, 333, 1100]
    table = _i32(_table(rng, lengths, page, pages, width))
    offs, pos = _i32([0, 1, 3, 5]), _i32([899, 331, 332, 1098, 1099])
    lens = _i32(lengths)
    b_of = [0, 1, 1, 2, 2]
    slots = _i32([int(table[b, p // page]) * page + p % page for b, p in zip(b_of, pos.tolist())])
    with Pooled(sess, n_kv, D, page, pages) as x:
        _filled(x, rng, n_kv, D, page, pages)
        bounds = x.open(hip.BlockBounds, x.pool)
        every = np.concatenate([[0], np.cumsum(lengths)])
        bounds.update(0, _i32(every), table, lens, int(every[-1]))
        qkv = _step_tensors(rows, n_q, n_kv, D, dt, 1)
        turned = torch.empty(rows, n_q, D, dtype=dt, device="cuda")

        def handles():
            return (x.open(hip.PagedAttention, x.pool, n_q, 3, rows), x.open(hip.PagedAttention, x.pool, n_q, 3, rows),
                    x.open(hip.BlockSelect, bounds, n_q, 3, rows, width),
                    [torch.empty(rows, n_q, D, dtype=dt, device="cuda") for _ in range(2)] + [torch.empty(rows, n_kv, top, dtype=torch.int32, device="cuda")])

        def step(h):
            plan, plan2, sel, (dense, sparse, blocks) = h
            x.pool.rope_append(0, qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:], slots, pos, freqs, q=qkv[:, :n_q], q_out=turned)
            bounds.update(0, offs, table, lens, rows)
            sel.run(0, turned, offs, table, lens, blocks, first=1, last=2)
            plan.run(0, turned, offs, table, lens, dense, max_rows=2)
            plan2.run(0, turned, offs, table, lens, sparse, max_rows=2, blocks=blocks)

        eager, held = handles(), handles()
        step(eager)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(held)
        for i in range(4):
            qkv.copy_(_step_tensors(rows, n_q, n_kv, D, dt, 10 + i))
            for o in held[3]:
                o.zero_()
            graph.replay()
            torch.cuda.synchronize()
            got = [o.clone() for o in held[3]]
            lim = torch.as_tensor(bounds.device(0), device="cuda").clone()
            step(eager)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, eager[3])) and torch.equal(lim, torch.as_tensor(bounds.device(0), device="cuda"))


def test_repeated_calls_are_equal(sess):
    """Results do not depend on timing."""
    rng = np.random.default_rng(12)
    n_q, n_kv, D, page, pages = 32, 8, 128, 16, 420
    lengths = [6000, 500]
    with Pooled(sess, n_kv, D, page, pages) as x:
        _filled(x, rng, n_kv, D, page, pages)
        table, offs, lens = _i32(_table(rng, lengths, page, pages, 376)), _i32([0, 40, 41]), _i32(lengths)
        q = torch.randn(41, n_q, D, device="cuda").bfloat16()
        plan = x.open(hip.PagedAttention, x.pool, n_q, 2, 41)
        outs = []
        for _ in range(3):
            outs.append(torch.empty_like(q))
            plan.run(0, q, offs, table, lens, outs[-1], max_rows=40)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


# ---- sizes that choose another form ----------------------------------------------------------
@pytest.mark.parametrize("pages", [700, 1024, 1025, 3001, 4097, 16384, 17003])
@pytest.mark.parametrize("alike", [False, True])
def test_select_sizes(sess, pages, alike):
    """Lists from few blocks to more than a workgroup's registers hold; scores of a few values, so that many are equal."""
    print("select sizes", pages, alike, flush=True)
    n_q, n_kv, D, page = 4, 2, 64, 4
    g = torch.Generator("cuda").manual_seed(pages)
    with Pooled(sess, n_kv, D, page, pages) as x:
        b = x.open(hip.BlockBounds, x.pool)
        lim = torch.as_tensor(b.device(0), device="cuda")
        z = torch.randn(lim.shape, generator=g, device="cuda")
        q = torch.randn(2, n_q, D, generator=g, device="cuda")
        if alike:
            z = torch.where(torch.arange(D, device="cuda") == 5, z.round(), 0.0)
            q = q.round()
        lim.copy_(z)
        table = np.random.default_rng(pages).permutation(pages)[None]
        lengths = [pages * page]
        for top, first, last in ((1, 0, 1), (64, 1, 2), (pages // 2, 1, 1), (pages + 3, 2, 1)):
            got = _select(x, b, q, table, lengths, [0, 2], top, first, last, n_q, n_kv).cpu().numpy()
            want = P.select(P.as_f64(q), P.as_f64(lim), table, lengths, [0, 2], page, top, first, last)
            assert np.array_equal(got, want), (top, np.argwhere(got != want)[:5])


@pytest.mark.parametrize("D,n_q,n_kv,page", [(64, 8, 2, 12), (128, 8, 2, 16), (256, 4, 1, 64), (256, 8, 2, 4)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("window", [0, 213])
def test_attention_of_prompts(sess, D, n_q, n_kv, page, dtype, window):
    """Prompts whose waves share tiles, for every head size and type: pages that are gone, what is no number behind the lengths and at tokens
    that some rows of a tile see and others do not."""
    print("prompts", D, n_q, dtype, window, flush=True)
    rng = np.random.default_rng(D + n_q)
    lengths, news, dt = [701, 350, 0, 520], [701, 290, 2, 260], TYPES[dtype]
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows = int(offsets[-1])
    pages = sum(-(-n // page) for n in lengths) + 1
    table = _table(rng, lengths, page, pages, -(-max(lengths) // page) + 2)
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        at = lambda b, t: (table[b, t // page], t % page)  # noqa: E731
        for b, n in enumerate(lengths):
            for t in range(n, -(-n // page) * page):
                k[at(b, t)], v[at(b, t)] = float("nan"), float("inf")
        v[at(0, 650)][0, 5], v[at(1, 200)][n_kv - 1, 7], v[at(3, 400)][0, D - 1] = float("inf"), float("nan"), float("-inf")
        k[at(1, 120)][0, 3] = float("nan")
        table[3, 130 // page] = -1
        x.slab(0).copy_(k)
        x.slab(1).copy_(v)
        q = torch.tensor(rng.standard_normal((rows, n_q, D)), dtype=torch.float32).to(dt)
        out = torch.empty(rows, n_q, D, dtype=dt, device="cuda")
        _attend(x, q.cuda(), table, lengths, offsets, out, n_q, max_rows=max(news), window=window)
        sel = np.unique(np.concatenate([rng.integers(0, rows, 40), [0, 1, 63, 64, 649, 650, 651, 700, 701, 840, 841, 990, 991, 993, rows - 1]]))
        want, mag, size, seen, _ = _some_rows(P.as_f64(q), k, v, table, lengths, offsets, sel, D ** -0.5, window=window)
        _near(out.cpu()[sel], want, _attn_tol(dt, D, want, mag, size, seen, float(v[v.isfinite()].abs().max()), prompt=True))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,length", [(64, 9001), (3, 20011), (17, 2100)])
def test_attention_of_many_pieces(sess, dtype, rows, length):
    """Few rows over a long context: many pieces an item, joined wave by wave and one after the other."""
    print("pieces", dtype, rows, length, flush=True)
    rng = np.random.default_rng(rows)
    n_q, n_kv, D, page, dt = 32, 8, 64, 64, TYPES[dtype]
    pages = -(-length // page)
    table = _table(rng, [length], page, pages, pages)
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        q = torch.tensor(rng.standard_normal((rows, n_q, D)), dtype=torch.float32).to(dt)
        out = torch.empty(rows, n_q, D, dtype=dt, device="cuda")
        _attend(x, q.cuda(), table, [length], [0, rows], out, n_q)
        sel = np.unique([0, 1, rows // 2, rows - 1])
        want, mag, size, seen, _ = _some_rows(P.as_f64(q), k, v, table, [length], [0, rows], sel, D ** -0.5)
        _near(out.cpu()[sel], want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max()), prompt=True))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n_q,n_kv,D", [(16, 8, 64), (8, 8, 128), (40, 4, 256)])
def test_attention_of_blocks_for_many_rows(sess, dtype, n_q, n_kv, D):
    """Rows enough that a wave takes a row's whole list."""
    print("blocks of many rows", dtype, n_q, D, flush=True)
    rng = np.random.default_rng(n_q)
    page, dt, width = 16, TYPES[dtype], 40
    news = [600 if n_kv == 4 else 300, 1]
    lengths = [630, 200]
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows = int(offsets[-1])
    table = _table(rng, lengths, page, 60, width)
    blocks = rng.integers(-1, width, (rows, n_kv, 9))
    with Pooled(sess, n_kv, D, page, 60) as x:
        k, v = _filled(x, rng, n_kv, D, page, 60)
        q = torch.tensor(rng.standard_normal((rows, n_q, D)), dtype=torch.float32).to(dt)
        out = torch.empty(rows, n_q, D, dtype=dt, device="cuda")
        _attend(x, q.cuda(), table, lengths, offsets, out, n_q, blocks=_i32(blocks))
        sel = np.unique(np.concatenate([rng.integers(0, rows, 20), [0, rows - 2, rows - 1]]))
        want, mag, size, seen, _ = _some_rows(P.as_f64(q), k, v, table, lengths, offsets, sel, D ** -0.5, blocks=blocks[sel])
        _near(out.cpu()[sel], want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max())))


def test_two_plans_side_by_side(sess):
    """Two plans and two selections at once on two streams, each with its own workspace, give what they give alone."""
    rng = np.random.default_rng(4)
    n_q, n_kv, D, page, pages, rows, top = 32, 8, 128, 16, 700, 24, 20
    lengths = [9000, 1500]
    with Pooled(sess, n_kv, D, page, pages) as x:
        _filled(x, rng, n_kv, D, page, pages)
        table, lens = _i32(_table(rng, lengths, page, pages, 570)), _i32(lengths)
        offs = [_i32([0, 23, 24]), _i32([0, 1, 24])]
        bounds = x.open(hip.BlockBounds, x.pool)
        bounds.update(0, _i32([0, 9000, 10500]), table, lens, 10500)
        q = [torch.randn(rows, n_q, D, device="cuda").to(t) for t in (torch.float16, torch.float32)]
        plans = [x.open(hip.PagedAttention, x.pool, n_q, 2, rows) for _ in range(2)]
        sels = [x.open(hip.BlockSelect, bounds, n_q, 2, rows, 570) for _ in range(2)]
        streams = [torch.cuda.Stream() for _ in range(2)]

        def results():
            return [(torch.empty_like(a), torch.empty_like(a), torch.empty(rows, n_kv, top, dtype=torch.int32, device="cuda")) for a in q]

        def one(i, r, stream):
            plans[i].run(0, q[i], offs[i], table, lens, r[0], max_rows=23, stream=stream)
            sels[i].run(0, q[i], offs[i], table, lens, r[2], stream=stream)
            plans[i].run(0, q[i], offs[i], table, lens, r[1], max_rows=23, blocks=r[2], stream=stream)

        alone = results()
        for i in range(2):
            one(i, alone[i], None)
            torch.cuda.synchronize()
        for _ in range(3):
            both = results()
            torch.cuda.synchronize()
            for i in range(2):
                one(i, both[i], streams[i])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for r, s in zip(alone, both) for a, b in zip(r, s))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n_q,n_kv,D,rows,said", [(32, 8, 64, 40, 1), (8, 2, 128, 90, 3), (8, 2, 256, 300, 20), (16, 1, 128, 3, 1)])
def test_attention_of_more_rows_than_said(sess, dtype, n_q, n_kv, D, rows, said):
    """max_rows chooses the form only: sequences with more rows are computed whole."""
    print("more rows than said", dtype, n_q, D, rows, said, flush=True)
    rng = np.random.default_rng(rows)
    page, dt, lengths, offsets = 64, TYPES[dtype], [5000, 800], [0, rows, 2 * rows]
    pages = 79 + 13
    table = _table(rng, lengths, page, pages, 80)
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        q = torch.tensor(rng.standard_normal((2 * rows, n_q, D)), dtype=torch.float32).to(dt)
        out = torch.full((2 * rows, n_q, D), 7.0, dtype=dt, device="cuda")
        _attend(x, q.cuda(), table, lengths, offsets, out, n_q, max_rows=said)
        sel = np.unique([0, 1, 2, rows // 2, rows - 2, rows - 1, rows, rows + 1, 2 * rows - 1])
        want, mag, size, seen, _ = _some_rows(P.as_f64(q), k, v, table, lengths, offsets, sel, D ** -0.5)
        _near(out.cpu()[sel], want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max()), prompt=True))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [4, 20, 100, 256, 1024])
def test_attention_of_any_page_size(sess, dtype, D, page):
    """Pages that are smaller and larger than what is read at a time, in every form; a query that is no number reaches its own row only."""
    print("pages of", page, dtype, D, flush=True)
    rng = np.random.default_rng(page + D)
    n_q, n_kv, dt = 4, 1, TYPES[dtype]
    lengths, news = [1500, 290], [280, 1]
    offsets = np.concatenate([[0], np.cumsum(news)])
    rows = int(offsets[-1])
    pages = sum(-(-n // page) for n in lengths)
    width = -(-1500 // page)
    table = _table(rng, lengths, page, pages, width)
    blocks = rng.integers(0, width, (rows, n_kv, 3))
    with Pooled(sess, n_kv, D, page, pages) as x:
        k, v = _filled(x, rng, n_kv, D, page, pages)
        q = torch.tensor(rng.standard_normal((rows, n_q, D)), dtype=torch.float32).to(dt)
        q[17, 2, 5] = float("nan")
        sel = np.unique(np.concatenate([rng.integers(0, rows, 8), [0, 16, 17, 18, 64, rows - 2, rows - 1]]))
        for kw in (dict(max_rows=280), dict(max_rows=1), dict(max_rows=5, window=300), dict(max_rows=280, window=70), dict(blocks=blocks)):
            out = torch.empty(rows, n_q, D, dtype=dt, device="cuda")
            _attend(x, q.cuda(), table, lengths, offsets, out, n_q, **{**kw, **({"blocks": _i32(blocks)} if "blocks" in kw else {})})
            plain = {n: (blocks[sel] if n == "blocks" else w) for n, w in kw.items() if n != "max_rows"}
            want, mag, size, seen, _ = _some_rows(P.as_f64(q), k, v, table, lengths, offsets, sel, D ** -0.5, **plain)
            _near(out.cpu()[sel], want, _attn_tol(dt, D, want, mag, size, seen, float(v.abs().max()), prompt=True))
