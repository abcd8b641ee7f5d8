"""The 4-bit paged cache on the GPU: append and read bit for bit against the
format's definition, attention against plain float64 attention over the values
that the cache holds.

Tolerances of attention, elementwise, from the roundings the kernel is allowed:
with W = sum of w_j |v_j| of the row (w the exact probabilities),
- scores: fp32 sums of D products with codes biased by at most 72 + 8, so each score is off by at
  most (D + 16) * 2^-24 * 10 * |q| . |k| * scale (a kept code's magnitude is at least a tenth of the biased one's
  bound on average over a block's largest element), which moves every weight by that factor, and the
  output by twice that times W;
- f16 and bf16: each weight is rounded to fp16's 11 bits, half a step of which is up to 2^-11 of it
  (finfo.eps / 2), and its product with the block's scale again: 2 * 2^-11 = 2^-10 of W; weights below the
  smallest fp16 subnormal (2^-24 of 2^9) vanish or round: N * 2^-33 * max|v|;
- bf16, many rows: keys are rounded to fp16 (2^-11 of each), which moves a score by up to 2^-11 * |q| . |k| * scale,
  every weight by that factor and their sum again: 2^-10 * |q| . |k| * scale * W;
- fp32: weights as two fp16 terms, 2^-22 * W, and fp32 sums over N tokens in at most N/8 dependent
  steps a lane: N * 2^-27 * W;
- the output's own rounding: half a step, finfo.eps / 2 * |out|, and below the smallest normal number half of the steps there,
  smallest_normal * eps / 2 (fp16: 2^-25, where -6.236e-7 is nearest to a number 2.8e-8 away).
"""
import numpy as np
import pytest
import torch

import kv4_plain as P
from rstr import hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def sess():
    with hip.Session(0) as s:
        yield s


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


# ---- append and read -------------------------------------------------------------------
def _hard_rows(rng, rows, heads, D):
    """Rows with what a quantiser can get wrong: ties, equal extremes of both signs, zeros, single
    values, tiny and huge blocks, NaN and infinities."""
    x = rng.standard_normal((rows, heads, D)).astype(np.float32)
    b = x.reshape(-1, 32)
    for i in range(len(b)):
        kind = i % 12
        if kind == 1:
            b[i] = 0.0
        elif kind == 2:  # every value a multiple of half a step: ties to even
            b[i] = rng.integers(-16, 16, 32) * 0.5 * 0.25
            b[i, rng.integers(32)] = 8 * 0.25 * rng.choice((-1, 1))
        elif kind == 3:  # the same magnitude twice, the first one's sign decides
            b[i, [5, 20]] = (4.5, -4.5) if i % 24 < 12 else (-4.5, 4.5)
        elif kind == 4:
            b[i] = 0.0
            b[i, rng.integers(32)] = rng.standard_normal()
        elif kind == 5:
            b[i] *= 2.0 ** -20
        elif kind == 6:
            b[i] *= 2.0 ** -27
        elif kind == 7:
            b[i] *= 2.0 ** 13
        elif kind == 8 and i % 48 == 8:
            b[i, rng.integers(32)] = rng.choice((np.nan, np.inf, -np.inf))
        elif kind == 9:
            b[i] = -0.0
    return x


@pytest.mark.parametrize("D,heads,page", [(64, 3, 16), (128, 2, 48), (256, 1, 16), (128, 8, 64)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("how", ["plain", "padded", "heads_outside", "odd"])
def test_append_read(sess, D, heads, page, dtype, how):
    print("append", D, heads, page, dtype, how, flush=True)
    rng = np.random.default_rng(D + heads + page)
    rows, pages = 61, 9
    pool = hip.Kv4Pool(sess, 2, heads, D, page, pages)
    k = torch.tensor(_hard_rows(rng, rows, heads, D)).to(TYPES[dtype])
    v = torch.tensor(_hard_rows(rng, rows, heads, D) * 1.5).to(TYPES[dtype])
    slots = rng.permutation(pages * page)[:rows].astype(np.int64)
    slots[7], slots[8], slots[50] = -1, pages * page, 2 ** 31 - 1
    pool.append(1, _laid(k, how), _laid(v, how), _i32(slots))
    listed = np.concatenate([slots, slots[:3], np.setdiff1d(np.arange(pages * page), slots)[:20]])  # some twice, some never written
    ko = _laid(torch.full((len(listed), heads, D), 9.0, dtype=TYPES[dtype]), how)
    vo = _laid(torch.full((len(listed), heads, D), 9.0, dtype=TYPES[dtype]), how)
    pool.read(1, _i32(listed), ko, vo)
    for x, o in ((k, ko), (v, vo)):
        want = P.quantised(P.as_f64(x))
        want[[7, 8, 50]] = 0.0
        want = np.concatenate([want, want[:3], np.zeros((20, heads, D))])
        want = torch.tensor(want).to(torch.float32).to(TYPES[dtype])  # exact in fp32, one rounding
        got = o.cpu()
        same = (got == want) | (got.isnan() & want.isnan())
        assert bool(same.all()), (torch.nonzero(~same)[:4], got[~same][:4], want[~same][:4])
    pool.read(0, _i32(listed), ko, vo)  # the other layer is untouched
    assert not ko.any() and not vo.any()
    pool.close()


def test_append_huge_values(sess):
    """Blocks past 8 * 65504 keep the largest scale, and their codes saturate."""
    k = torch.zeros(1, 1, 64)
    k[0, 0, 3], k[0, 0, 4], k[0, 0, 40], k[0, 0, 41] = 1e9, -2e5, -3e38, 7e5
    pool = hip.Kv4Pool(sess, 1, 1, 64, 16, 1)
    k = k.cuda()
    pool.append(0, k, k, _i32([5]))
    o, p = torch.empty_like(k), torch.empty_like(k)
    pool.read(0, _i32([5]), o, p)
    assert np.array_equal(P.as_f64(o), P.quantised(P.as_f64(k))) and torch.equal(o, p)
    pool.close()


def test_append_many_rows(sess):
    """More rows than one launch row of workgroups holds, each its own slot."""
    rows, pool = 5000, hip.Kv4Pool(sess, 1, 2, 64, 16, 313)
    g = torch.Generator("cuda").manual_seed(1)
    k = torch.randn(rows, 2, 64, generator=g, device="cuda").half()
    slots = torch.randperm(313 * 16, generator=g, device="cuda")[:rows].to(torch.int32)
    pool.append(0, k, -k, slots)
    a, b = torch.empty_like(k), torch.empty_like(k)
    pool.read(0, slots, a, b)
    want = torch.tensor(P.quantised(P.as_f64(k))).half()
    assert torch.equal(a.cpu(), want)
    assert torch.equal(b.cpu(), torch.tensor(P.quantised(-P.as_f64(k))).half())
    pool.close()


# ---- attention ---------------------------------------------------------------------------
class Case:
    """A cache filled through append, ragged sequences over it and their float64 values."""

    def __init__(self, sess, n_q, n_kv, D, page, lens, news, seed=0, extra=5, width=None, v_scale=1.0, k_scale=1.0, layers=1):
        rng = np.random.default_rng([seed, n_q, D, page, len(lens)])
        self.rng, self.lens, self.news, self.page, self.n_q, self.n_kv, self.D = rng, list(lens), list(news), page, n_q, n_kv, D
        need = [-(-max(n, 0) // page) for n in lens]
        self.pages = sum(need) + extra
        perm = rng.permutation(self.pages)
        self.table = np.full((len(lens), width or max(1, max(need))), -1, np.int64)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        self.pool = hip.Kv4Pool(sess, layers, n_kv, D, page, self.pages)
        total = sum(lens)
        k = torch.tensor(rng.standard_normal((total, n_kv, D)) * k_scale, dtype=torch.float16)
        v = torch.tensor(rng.standard_normal((total, n_kv, D)) * v_scale, dtype=torch.float16)
        k[..., D // 3:: 29] *= 3.0
        slots = np.concatenate([self.table[b, np.arange(n) // page] * page + np.arange(n) % page for b, n in enumerate(lens)] or [[]])
        if total:
            self.pool.append(layers - 1, k.cuda(), v.cuda(), _i32(slots))
        cut = np.concatenate([[0], np.cumsum(lens)])
        kq, vq = P.quantised(P.as_f64(k)), P.quantised(P.as_f64(v))
        self.k = [kq[cut[b]:cut[b + 1]] for b in range(len(lens))]
        self.v = [vq[cut[b]:cut[b + 1]] for b in range(len(lens))]
        self.offsets = np.concatenate([[0], np.cumsum(news)])
        self.layer = layers - 1

    def plan(self, behind=0):
        return hip.Kv4Attention(self.pool, self.n_q, len(self.lens), int(self.offsets[-1]) + behind)

    def queries(self, dtype, behind=0, mul=1.5):
        R = int(self.offsets[-1]) + behind
        return torch.tensor(self.rng.standard_normal((R, self.n_q, self.D)) * mul, dtype=torch.float32).to(TYPES[dtype])

    def check(self, got, q, dtype, window, scale, what=""):
        want, mag, size = P.attention(P.as_f64(q), self.k, self.v, self.lens, self.offsets, window, scale)
        R = int(self.offsets[-1])
        N, D = max(self.lens + [1]), self.D
        vmax = max([np.nanmax(np.abs(x)) for x in self.v if len(x)] + [0.0])
        rel = 2 * (D + 16) * 2.0 ** -24 * 10 * size
        rel = rel + (2.0 ** -10 if dtype != "f32" else 2.0 ** -22 + N * 2.0 ** -27)
        if dtype == "bf16" and max(self.news) > 16:
            rel = rel + 2.0 ** -10 * size
        tol = rel * mag + torch.finfo(TYPES[dtype]).eps / 2 * np.abs(want) * 1.01 + N * 2.0 ** -33 * vmax
        tol = tol + torch.finfo(TYPES[dtype]).smallest_normal * torch.finfo(TYPES[dtype]).eps / 2
        far = np.abs(P.as_f64(got)[:R] - want[:R]) - tol[:R]
        assert np.all(np.isfinite(P.as_f64(got)[:R])), what
        assert far.max() <= 0, (what, far.max(), np.unravel_index(far.argmax(), far.shape))
        return want

    def close(self):
        self.pool.close()


SHAPES = [
    # n_q, n_kv, D, page, lengths, rows, window
    (4, 2, 128, 16, [1], [1], 0),
    (4, 2, 128, 16, [0], [1], 0),
    (4, 2, 128, 16, [16, 17, 31, 32, 33, 15], [1] * 6, 0),
    (8, 2, 64, 16, [100, 1, 0, 333], [1, 1, 1, 1], 0),
    (4, 1, 256, 16, [77, 600], [1, 1], 0),
    (4, 1, 256, 32, [77, 600, 5], [3, 1, 5], 50),
    (8, 8, 64, 48, [47, 48, 49, 500], [1, 2, 3, 4], 0),
    (32, 8, 128, 16, [700, 3, 65], [1, 3, 2], 0),
    (16, 8, 128, 64, [1500], [1], 100),
    (24, 1, 128, 16, [200, 30], [1, 1], 0),      # more than 16 heads on one kv head
    (48, 1, 64, 16, [90], [2], 33),
    (4, 4, 128, 16, [40, 9], [40, 9], 0),        # whole prompts
    (8, 2, 128, 16, [130, 77], [70, 77], 0),
    (6, 2, 64, 16, [200], [150], 17),
    (4, 1, 256, 16, [150], [99], 40),
    (2, 2, 128, 16, [5, 0, 3], [9, 4, 2], 0),    # more rows than tokens: the first rows see nothing
    (4, 2, 128, 16, [64, 64, 64], [0, 2, 0], 0),  # sequences without rows
    (4, 2, 64, 16, [33] * 70, [1] * 70, 0),      # more sequences than a wave has lanes
    (4, 2, 64, 16, [2500, 40], [1, 1], 1),       # a window of the token itself
    (4, 2, 128, 16, [3000, 10, 800], [4, 1, 2], 0),
    # many columns a sequence, head dim 128: waves that share a tile's expansion (fp16, bf16)
    (8, 2, 128, 16, [600, 530], [40, 33], 0),
    (32, 8, 128, 16, [1000], [77], 100),
    (6, 2, 128, 48, [1300, 0, 333], [90, 20, 64], 0),
    (24, 1, 128, 64, [700, 100], [5, 3], 0),
    (4, 2, 128, 16, [5, 700], [70, 3], 0),
    (4, 2, 128, 16, [64, 300, 64], [0, 130, 0], 0),
    (8, 8, 128, 16, [900, 31, 290], [64, 31, 100], 1),
    (8, 1, 128, 32, [2000], [300], 0),
    # the largest window there is, and rows before the first token
    (2, 2, 128, 16, [5, 0, 3], [9, 4, 2], 2 ** 31 - 1),
    (4, 2, 128, 16, [5, 700], [70, 3], 2 ** 31 - 1),
    (4, 1, 256, 16, [30], [40], 2 ** 31 - 2),
    (2, 2, 64, 16, [40], [3], 2 ** 32 + 5),
]


@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_attention(sess, shape, dtype):
    n_q, n_kv, D, page, lens, news, window = shape
    print("attention", shape, dtype, flush=True)
    c = Case(sess, n_q, n_kv, D, page, lens, news)
    q = c.queries(dtype, behind=2)
    out = torch.full_like(q, 7.0).cuda()
    plan = c.plan(behind=2)
    plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32(lens), out, max_rows=max(news), window=window, scale=D ** -0.5)
    c.check(out, q, dtype, window, D ** -0.5)
    assert bool((out[int(c.offsets[-1]):] == 7.0).all())  # rows behind the last sequence
    # any bound on a sequence's rows gives the same values, to rounding
    other = torch.full_like(out, 3.0)
    plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32(lens), other, window=window, scale=D ** -0.5)
    c.check(other, q, dtype, window, D ** -0.5, "max_rows")
    plan.close()
    c.close()


@pytest.mark.parametrize("how", ["padded", "heads_outside", "odd"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("lens,news", [([70, 200], [3, 20]), ([400, 300], [30, 20])])
def test_attention_strides(sess, how, dtype, lens, news):
    c = Case(sess, 8, 2, 128, 16, lens, news, layers=2)
    q = c.queries(dtype)
    out = _laid(torch.zeros_like(q), how)
    plan = c.plan()
    plan.run(1, _laid(q, how), _i32(c.offsets), _i32(c.table), _i32(c.lens), out, scale=0.1)
    c.check(out, q, dtype, 0, 0.1)
    plan.run(0, _laid(q, how), _i32(c.offsets), _i32(c.table), _i32(c.lens), out)  # an empty layer: zeros
    assert not out.any()
    plan.close()
    c.close()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("v_scale,k_scale,mul", [(1e-4, 1.0, 1.5), (300.0, 1.0, 1.5), (1.0, 20.0, 6.0), (1.0, 1e-3, 1e-3), (3000.0, 3.0, 1.0)])
@pytest.mark.parametrize("news", [[1, 6], [100, 40]])
def test_attention_ranges(sess, dtype, v_scale, k_scale, mul, news):
    """Tiny and large values, near-uniform and one-hot probabilities."""
    print("ranges", dtype, v_scale, k_scale, mul, news, flush=True)
    c = Case(sess, 4, 2, 128, 16, [900, 40], news, v_scale=v_scale, k_scale=k_scale)
    q = c.queries(dtype, mul=mul)
    out = torch.zeros_like(q).cuda()
    plan = c.plan()
    plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32(c.lens), out, max_rows=max(news))
    c.check(out, q, dtype, 0, 128 ** -0.5)
    plan.close()
    c.close()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("at", [3, 250, 699])
def test_attention_past_fp16(sess, dtype, rows, at):
    """Values (and keys, one token on) past fp16's range, whose scales are 2^13 and more, in the first, a middle or
    the last tile; the scores stay small through the scale."""
    print("past fp16", dtype, rows, at, flush=True)
    c = Case(sess, 4, 2, 128, 16, [700], [rows])
    rng = np.random.default_rng(at)
    for t, mk, mv in ((at, 1.0, 1e5), (min(at + 1, 698), 1e5, 1.0)):
        k, v = (torch.tensor(rng.standard_normal((1, 2, 128)) * m, dtype=torch.float32) for m in (mk, mv))
        c.pool.append(0, k.cuda(), v.cuda(), _i32([c.table[0, t // 16] * 16 + t % 16]))
        c.k[0][t], c.v[0][t] = P.quantised(P.as_f64(k))[0], P.quantised(P.as_f64(v))[0]
    q = c.queries(dtype)
    out = torch.zeros_like(q).cuda()
    plan = c.plan()
    plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32(c.lens), out, scale=1e-6)
    c.check(out, q, dtype, 0, 1e-6)
    plan.close()
    c.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,D", [(1, 128), (40, 64), (70, 128), (3, 256)])
def test_scores_far_below_zero(sess, dtype, rows, D):
    """Scores from -1e34 down: the softmax is 1 at the largest, token 0, whose value is the output (rounded at
    most twice to 11 bits and once to the output's type)."""
    print("far below zero", dtype, rows, D, flush=True)
    n = 300
    c = Case(sess, 4, 2, D, 16, [n], [rows])
    k = torch.arange(1, n + 1, dtype=torch.float32)[:, None, None].expand(n, 2, D).contiguous()
    v = torch.tensor(c.rng.standard_normal((n, 2, D)), dtype=torch.float32)
    c.pool.append(0, k.cuda(), v.cuda(), _i32(c.table[0, np.arange(n) // 16] * 16 + np.arange(n) % 16))
    q = torch.full((rows, 4, D), -1e32).to(TYPES[dtype])
    out = torch.zeros_like(q).cuda()
    plan = c.plan()
    plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32(c.lens), out)
    want = np.repeat(P.quantised(P.as_f64(v[:1]))[0], 2, axis=0)
    tol = (2.0 ** -10 if dtype != "f32" else 2.0 ** -21) + torch.finfo(TYPES[dtype]).eps / 2 * 1.01
    assert (np.abs(P.as_f64(out) - want) <= tol * np.abs(want)).all()
    plan.close()
    c.close()


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows", [1, 40])
def test_fp32_is_fp32(sess, D, rows):
    """fp32 queries: the whole output within 2^-19 of its norm.  A weight is off by its exponent's
    rounding, at most half a step of a number below 16 (2^-21) in each of the sum, the scale and the
    difference, times ln 2: 2^-19.9 together if all agree; its two fp16 terms keep 2^-22."""
    print("fp32", D, rows, flush=True)
    for seed in range(6):
        c = Case(sess, 4, 2, D, 16, [1500 + 83 * seed], [rows], seed=seed)
        q = c.queries("f32")
        out = torch.zeros_like(q).cuda()
        plan = c.plan()
        plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32(c.lens), out)
        want, _, _ = P.attention(P.as_f64(q), c.k, c.v, c.lens, c.offsets, 0, D ** -0.5)
        for h in range(4):
            off = np.linalg.norm((P.as_f64(out) - want)[:, h]) / np.linalg.norm(want[:, h])
            assert off < 2.0 ** -19, (seed, h, off)
        plan.close()
        c.close()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,n", [(2, 333), (40, 333), (100, 650)])
def test_what_is_not_seen_does_not_matter(sess, dtype, rows, n):
    """NaN blocks behind a row's position, before its window, in free pages and behind the length
    change nothing, bit for bit; where a row does see one it is NaN in that block."""
    D, page, window = 128, 16, 64
    c = Case(sess, 4, 2, D, page, [n, 50], [rows, 1])
    q = c.queries(dtype).cuda()
    plan = c.plan()

    def run():
        out = torch.zeros_like(q)
        plan.run(0, q, _i32(c.offsets), _i32(c.table), _i32(c.lens), out, max_rows=rows, window=window)
        return out

    before = run()
    c.check(before, q, dtype, window, D ** -0.5)
    bad = torch.full((1, 2, D), float("nan"), device="cuda")
    kill = lambda t: c.pool.append(0, bad, bad, _i32([c.table[0, t // page] * page + t % page]))  # noqa: E731
    kill(0)
    kill(n - rows - window)              # one before the first row's window
    used = set(c.table.ravel().tolist())
    for pg in range(c.pages):
        if pg not in used:
            c.pool.append(0, bad.expand(16, 2, D).contiguous(), bad.expand(16, 2, D).contiguous(), _i32(pg * page + np.arange(page)))
    tail = c.table[0, n // page] * page + np.arange(n % page, page)   # behind the length
    c.pool.append(0, bad.expand(len(tail), 2, D).contiguous(), bad.expand(len(tail), 2, D).contiguous(), _i32(tail))
    assert torch.equal(run(), before)
    kill(n - 1)                          # the last row's own token
    after = run()
    last = rows - 1
    assert torch.equal(after[:last], before[:last]) and torch.equal(after[rows:], before[rows:])
    assert bool(after[last].isnan().all())
    # a value block alone: that block of the output is NaN, the others are not
    good = torch.zeros(1, 2, D, device="cuda")
    half = torch.ones(1, 2, D, device="cuda")
    half[..., 32:64] = float("inf")
    c.pool.append(0, good, half, _i32([c.table[0, (n - 1) // page] * page + (n - 1) % page]))
    after = run()
    assert bool(after[last, :, 32:64].isnan().all()) and bool(after[last, :, :32].isfinite().all())
    assert bool(after[last, :, 64:].isfinite().all()) and torch.equal(after[:last], before[:last])
    plan.close()
    c.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_bad_descriptors_stay_inside(sess, dtype):
    """Page ids outside the cache are not seen; lengths and offsets beyond the arrays are cut."""
    page, D = 16, 64
    c = Case(sess, 4, 2, D, page, [100, 64], [2, 1])
    q = c.queries(dtype)
    table = c.table.copy()
    gone = {1: [16, 32], 3: [48, 64]}
    table[0, 1], table[0, 3] = -1, c.pages
    table[1, 0] = 2 ** 31 - 1
    out = torch.zeros_like(q).cuda()
    plan = c.plan()
    plan.run(0, q.cuda(), _i32(c.offsets), _i32(table), _i32(c.lens), out)
    seen = [np.ones(100, bool), np.ones(64, bool)]
    for lo, hi in gone.values():
        seen[0][lo:hi] = False
    seen[1][:16] = False
    want = np.zeros(q.shape)
    for r, (b, p) in enumerate(((0, 98), (0, 99), (1, 63))):
        j = np.flatnonzero(seen[b][:p + 1])
        for h in range(4):
            s = c.k[b][j, h // 2] @ P.as_f64(q)[r, h] * D ** -0.5
            w = np.exp(s - s.max())
            want[r, h] = w / w.sum() @ c.v[b][j, h // 2]
    assert np.abs(P.as_f64(out) - want).max() < 4 * (2.0 ** -9 if dtype == "bf16" else 2.0 ** -18)
    for lens, offs in (([10 ** 9, 64], c.offsets), ([-5, -(2 ** 31)], c.offsets), (c.lens, [0, 50, 90]), (c.lens, [-4, 1, 2 ** 31 - 1]),
                       (c.lens, [2, 0, 3])):
        plan.run(0, q.cuda(), _i32(offs), _i32(table), _i32(lens), out)
        torch.cuda.synchronize()
    plan.close()
    c.close()


def test_cache_past_32_bits(sess):
    """Pages whose bytes lie past 2^32 of a layer."""
    D, page, pages = 128, 64, 70000
    pool = hip.Kv4Pool(sess, 1, 8, D, page, pages)
    assert pool.nbytes > 2 ** 32
    rng = np.random.default_rng(0)
    table = np.array([[pages - 1, 3, pages - 2, 65536]])
    n = 250
    k = torch.tensor(rng.standard_normal((n, 8, D)), dtype=torch.float16)
    v = torch.tensor(rng.standard_normal((n, 8, D)), dtype=torch.float16)
    pool.append(0, k.cuda(), v.cuda(), _i32(table[0, np.arange(n) // page] * page + np.arange(n) % page))
    q = torch.tensor(rng.standard_normal((1, 16, D)), dtype=torch.float32)
    out = torch.zeros(1, 16, D, device="cuda")
    plan = hip.Kv4Attention(pool, 16, 1, 1)
    plan.run(0, q.cuda(), _i32([0, 1]), _i32(table), _i32([n]), out)
    want, mag, _ = P.attention(P.as_f64(q), [P.quantised(P.as_f64(k))], [P.quantised(P.as_f64(v))], [n], [0, 1], 0, D ** -0.5)
    assert np.abs(P.as_f64(out) - want).max() < 2.0 ** -16 * mag.max()
    plan.close()
    pool.close()


def test_long_context(sess):
    """One sequence over many workgroups; a window near its end; against float64 on the GPU."""
    D, page, n = 128, 16, 40001
    c_lens = [n]
    g = torch.Generator("cuda").manual_seed(3)
    pool = hip.Kv4Pool(sess, 1, 2, D, page, -(-n // page))
    table = torch.randperm(-(-n // page), generator=g, device="cuda").to(torch.int32)[None]
    t = torch.arange(n, device="cuda")
    slots = table[0].long()[t // page] * page + t % page
    k, v = torch.randn(n, 2, D, generator=g, device="cuda"), torch.randn(n, 2, D, generator=g, device="cuda")
    pool.append(0, k, v, slots.to(torch.int32))
    pool.read(0, slots.to(torch.int32), k, v)
    for rows, window, dtype in ((1, 0, "f16"), (1, 0, "f32"), (3, 30000, "bf16"), (3, 33, "f32"), (40, 0, "f32"), (40, 39000, "f16")):
        print("long", rows, window, dtype, flush=True)
        q = torch.randn(rows, 8, D, generator=g, device="cuda").to(TYPES[dtype])
        out = torch.zeros_like(q)
        plan = hip.Kv4Attention(pool, 8, 1, rows)
        plan.run(0, q, _i32([0, rows]), table, _i32(c_lens), out, window=window)
        p = torch.arange(n - rows, n, device="cuda")[:, None]
        hid = (t > p) | ((t <= p - window) if window else (t < 0))
        for h in range(8):
            s = (q[:, h].double() @ k[:, h // 4].double().t().contiguous()) * D ** -0.5
            w = torch.softmax(s.masked_fill(hid, -float("inf")), 1)
            want = w @ v[:, h // 4].double()
            mag = w @ v[:, h // 4].double().abs()
            tol = (2.0 ** -10 if dtype != "f32" else 2.0 ** -16) * mag + torch.finfo(q.dtype).eps / 2 * want.abs() * 1.01 + n * 2.0 ** -33 * 6
            assert bool(((out[:, h].double() - want).abs() <= tol).all()), (rows, window, dtype, h)
        plan.close()
    pool.close()


@pytest.mark.parametrize("lens,news", [([400, 90, 3], [2, 1, 1]), ([400, 300], [60, 40])])
def test_streams_and_graphs(sess, lens, news):
    """Captured calls replay on changed inputs between eager calls; two plans run side by side on
    two streams; the session's own stream takes calls too."""
    c = Case(sess, 8, 2, 128, 16, lens, news)
    q = c.queries("f16").cuda()
    args = (_i32(c.offsets), _i32(c.table), _i32(c.lens))
    plans = [c.plan() for _ in range(3)]
    outs = [torch.zeros_like(q) for _ in range(3)]
    plans[0].run(0, q, *args, outs[0])
    torch.cuda.synchronize()
    graphs = []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plans[i].run(0, q, *args, outs[i])
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        q.copy_(c.queries("f16"))
        plans[2].run(0, q, *args, outs[2])
        torch.cuda.synchronize()
        for i in (0, 1):
            outs[i].zero_()
        torch.cuda.synchronize()
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2]), step
        outs[0].zero_()
        torch.cuda.synchronize()
        plans[0].run(0, q, *args, outs[0], stream=hip.SESSION_STREAM)
        with torch.cuda.stream(streams[1]):
            outs[1].zero_()
            plans[1].run(0, q, *args, outs[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2]), step
    c.check(outs[0], q, "f16", 0, 128 ** -0.5)
    for p in plans:
        p.close()
    c.close()


@pytest.mark.parametrize("dtype,D,n_q,each", [("f32", 64, 4, 1), ("f16", 128, 8, 5), ("bf16", 128, 8, 20), ("bf16", 256, 4, 2)])
@pytest.mark.parametrize("B", [2, 64, 70, 200])
def test_offsets_that_decrease(sess, dtype, D, n_q, each, B):
    """Where row offsets decrease, nothing is written: their sequences would have the same rows, and more items than the
    workspace has room for.  The plan serves the next call."""
    print("decreasing offsets", dtype, D, B, flush=True)
    c = Case(sess, n_q, 2 if n_q > 4 else 1, D, 16, [140 + i % 50 for i in range(B)], [each] * B, width=20)
    q = c.queries(dtype).cuda()
    R = B * each
    plan = c.plan()
    over_and_over = [R if b % 2 else 0 for b in range(B + 1)]
    one_back, last_back = c.offsets.copy(), c.offsets.copy()
    one_back[B // 2 + 1] = one_back[B // 2] - 1
    last_back[B] = 0
    for bad in (over_and_over, one_back, last_back, [2 ** 31 - 1] + c.offsets[1:].tolist()):
        out = torch.full_like(q, 7.0)
        plan.run(0, q, _i32(bad), _i32(c.table), _i32(c.lens), out, max_rows=each)
        torch.cuda.synchronize()
        assert bool((out == 7.0).all())
        plan.run(0, q, _i32(c.offsets), _i32(c.table), _i32(c.lens), out, max_rows=each)
        c.check(out, q, dtype, 0, D ** -0.5)
    plan.close()
    c.close()


def _attention_by_position(q, k, v, length, window, scale):
    """The last rows q [m][n_q][D] of a sequence of `length` tokens, of which k, v [tokens][n_kv][D] are
    held: out, sum of w|v|, the largest |scale| |q| . |k| of a row's keys that weigh anything, and its least weights: sum of
    min(w, 2^-33) |v|."""
    m, n_q, D = q.shape
    out, mag, size, low = (np.zeros(s) for s in ((m, n_q, D), (m, n_q, D), (m, n_q, 1), (m, n_q, D)))
    for r in range(m):
        p = length - m + r
        j = np.arange(max(0, p - window + 1) if window else 0, min(p + 1, len(k)))
        if not j.size:
            continue
        for h in range(n_q):
            kk, vv = k[j, h // (n_q // k.shape[1])], v[j, h // (n_q // k.shape[1])]
            s = kk @ q[r, h] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            out[r, h], mag[r, h], low[r, h] = w @ vv, w @ np.abs(vv), np.minimum(w, 2.0 ** -33) @ np.abs(vv)
            size[r, h] = np.max((np.abs(kk) @ np.abs(q[r, h]))[w > 2.0 ** -60]) * abs(scale)
    return out, mag, size, low


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("what,small", [("key", 1e-5), ("key", 1.0), ("block", 2e-4), ("block", 2e-3), ("token", 2e-4), ("token", 2e-2), ("all", 1.0)])
def test_values_of_very_different_size(sess, dtype, rows, D, what, small):
    """One token's keys, one block of its values, or all its values past fp16's range (scales of 2^13 and more) beside
    values of `small` size, which keep their bits: a product of a weight and a value is off by its own
    rounding, or by 2^-32 where that is more (a weight is 2^10 at the largest score, a product of it with a block's
    scale then a multiple of 2^-24 or rounded to one, and a code at most 8 of those: 8 * 2^-25 / 2^10).
    "token": the large values are those of a token that weighs nothing.  Few tokens, so that the first rows' roundings
    do not average out; a table of 320 tokens, which many rows of head dim 128 share the expansion of."""
    print("different size", dtype, rows, D, what, small, flush=True)
    n, scale = 40, 1e-6 if what == "key" else D ** -0.5
    c = Case(sess, 4, 2, D, 16, [n], [rows], width=20, v_scale=small)
    q = c.queries(dtype)
    q[..., 0] = 8.0
    rng = np.random.default_rng(D)
    first = torch.tensor(rng.standard_normal((2, 1, 2, D)) * np.array([1.0, small]).reshape(2, 1, 1, 1), dtype=torch.float32)
    k, v = first[0], first[1]
    if what == "key":
        k *= 1e5
    elif what == "block":
        v[..., 32:64] *= 1e5 / small
    else:
        v *= 1e5 / small
    if what == "token":
        k[..., 0] = -4000.0   # a score of -2000 and less
    c.pool.append(0, k.cuda(), v.cuda(), _i32([c.table[0, 0] * 16]))
    c.k[0][0], c.v[0][0] = P.quantised(P.as_f64(k))[0], P.quantised(P.as_f64(v))[0]
    out = torch.zeros_like(q).cuda()
    plan = c.plan()
    plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32(c.lens), out, scale=scale)
    want, mag, size, low = _attention_by_position(P.as_f64(q), c.k[0], c.v[0], n, 0, scale)
    rel = 2 * (D + 16) * 2.0 ** -24 * 10 * size + (2.0 ** -10 if dtype != "f32" else 2.0 ** -22 + n * 2.0 ** -27)
    if dtype == "bf16" and rows > 16:
        rel = rel + 2.0 ** -10 * size
    eps = torch.finfo(TYPES[dtype]).eps
    tol = rel * mag + eps / 2 * np.abs(want) * 1.01 + low + n * 2.0 ** -32 + torch.finfo(TYPES[dtype]).smallest_normal * eps / 2
    fits = np.abs(want) < torch.finfo(TYPES[dtype]).max * (1 - 2.0 ** -9)   # fp16 does not hold the first rows' largest
    far = np.where(fits, np.abs(P.as_f64(out) - want) - tol, -1.0) / (np.abs(want) + 1e-30)
    assert far.max() <= 0, (far.max(), np.unravel_index(far.argmax(), far.shape))
    plan.close()
    c.close()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,D,held,length,window", [
    (1, 64, 64, 100, 50), (1, 64, 64, 100, 0), (3, 128, 64, 65, 0), (3, 128, 64, 66, 20), (2, 256, 320, 400, 100), (9, 64, 320, 324, 40),
    (1, 128, 64, 200, 50), (40, 128, 320, 345, 0), (70, 128, 320, 380, 100), (60, 128, 320, 1000, 30), (3, 128, 320, 2 ** 31 - 1, 2 ** 31 - 30),
    (50, 128, 320, 2 ** 31 - 1, 2 ** 31 - 30), (2, 64, 320, 2 ** 31 - 1, 0),
])
def test_lengths_beyond_the_table(sess, dtype, rows, D, held, length, window):
    """A row's position follows from the sequence's length, also where the table ends before it: the tokens
    behind the table's width are not seen, and nothing else changes."""
    print("beyond the table", dtype, rows, D, held, length, window, flush=True)
    c = Case(sess, 4, 2, D, 16, [held], [rows])
    q = c.queries(dtype)
    out = torch.full_like(q, 7.0).cuda()
    plan = c.plan()
    plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32([length]), out, window=window)
    want, mag, size, _ = _attention_by_position(P.as_f64(q), c.k[0], c.v[0], length, window, D ** -0.5)
    rel = 2 * (D + 16) * 2.0 ** -24 * 10 * size + (2.0 ** -10 if dtype != "f32" else 2.0 ** -22 + held * 2.0 ** -27)
    if dtype == "bf16" and rows > 16:
        rel = rel + 2.0 ** -10 * size
    eps = torch.finfo(TYPES[dtype]).eps
    tol = rel * mag + eps / 2 * np.abs(want) * 1.01 + held * 2.0 ** -33 * np.abs(c.v[0]).max() + torch.finfo(TYPES[dtype]).smallest_normal * eps / 2
    far = np.abs(P.as_f64(out) - want) - tol
    assert far.max() <= 0, (far.max(), np.unravel_index(far.argmax(), far.shape))
    plan.close()
    c.close()


# ---- append and read in prompt quantity -----------------------------------------------------
def _quantised_all(x):
    """P.quantised, all blocks at once."""
    w = np.asarray(x, np.float64).reshape(-1, 32)
    finite = np.isfinite(w).all(1)
    w = np.where(finite[:, None], w, 0.0)
    m = w[np.arange(len(w)), np.abs(w).argmax(1)]
    d = np.clip(m / -8.0, -65504.0, 65504.0).astype(np.float16).astype(np.float64)[:, None]
    o = np.where(d == 0, 0.0, d * np.clip(np.rint(w / np.where(d == 0, 1.0, d)), -8, 7))
    return np.where(finite[:, None], o, np.nan).reshape(np.shape(x))


def _prompt_slots(rng, rows, room, order):
    """Slots of `rows` rows: as consecutive pages' tokens from a place inside a group of four or
    of sixteen, in any order, or with rows that have none, the first among them."""
    if order == "aligned":
        return np.arange(32, 32 + rows)
    if order == "run":
        return np.arange(21, 21 + rows)
    if order == "backwards":
        return np.arange(rows)[::-1] + 7
    if order == "permuted":
        return rng.permutation(room)[:rows]
    if order == "groups":  # whole groups of four tokens, in any order
        return (rng.permutation(room // 4)[:, None] * 4 + np.arange(4)).reshape(-1)[:rows]
    slots = np.arange(rows) + 2
    slots[rng.random(rows) < 0.1] = -1
    slots[rng.random(rows) < 0.05] = room + 3
    slots[0] = -1 if order == "none_first" else room if order == "outside_first" else 2 ** 31 - 1
    return slots


@pytest.mark.parametrize("D,heads,page,rows", [(64, 8, 16, 4099), (128, 8, 48, 2066), (256, 1, 32, 8193)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("order,how", [("aligned", "plain"), ("run", "padded"), ("backwards", "odd"), ("permuted", "plain"), ("groups", "heads_outside"),
                                       ("none_first", "odd"), ("outside_first", "plain"), ("largest_first", "heads_outside")])
def test_append_read_prompts(sess, D, heads, page, rows, dtype, order, how):
    """Rows enough for four a thread, bit for bit."""
    print("append prompt", D, heads, page, rows, dtype, order, how, flush=True)
    rng = np.random.default_rng([D, len(order)])
    pages = -(-(rows + 40) // page) + 2
    room = pages * page
    pool = hip.Kv4Pool(sess, 2, heads, D, page, pages)
    hard = _hard_rows(rng, 241, heads, D)
    k = torch.tensor(hard[rng.integers(0, 241, rows)]).to(TYPES[dtype])
    v = torch.tensor(hard[rng.integers(0, 241, rows)] * 1.5).to(TYPES[dtype])
    slots = _prompt_slots(rng, rows, room, order)
    pool.append(1, _laid(k, how), _laid(v, how), _i32(slots))
    there = (slots >= 0) & (slots < room)
    free = np.setdiff1d(np.arange(room), slots[there])
    kq, vq = (torch.tensor(_quantised_all(P.as_f64(x)), dtype=torch.float32).to(TYPES[dtype]) for x in (k, v))
    # as they were appended; then any order, some twice, with those that were never written
    mixed = np.concatenate([slots, free, slots[:rows // 3]])
    for listed in (slots, rng.permutation(mixed)):
        ko = _laid(torch.full((len(listed), heads, D), 9.0, dtype=TYPES[dtype]), how)
        vo = _laid(torch.full((len(listed), heads, D), 9.0, dtype=TYPES[dtype]), how)
        pool.read(1, _i32(listed), ko, vo)
        for x, o in ((kq, ko), (vq, vo)):
            held = torch.zeros(room + 1, heads, D, dtype=TYPES[dtype])
            held[torch.from_numpy(slots[there])] = x[torch.from_numpy(there)]
            want = held[torch.from_numpy(np.where((listed >= 0) & (listed < room), listed, room))]
            got = o.cpu()
            same = (got == want) | (got.isnan() & want.isnan())
            assert bool(same.all()), (torch.nonzero(~same)[:4], got[~same][:4], want[~same][:4])
    pool.read(0, _i32(slots), ko[:rows], vo[:rows])  # the other layer is untouched
    assert not ko[:rows].any() and not vo[:rows].any()
    pool.close()


def test_all_blocks_at_once():
    x = _hard_rows(np.random.default_rng(2), 24, 2, 64)
    assert np.array_equal(_quantised_all(x), P.quantised(x), equal_nan=True)


# ---- attention of many sequences --------------------------------------------------------------
def _lines(rng, B, most, rows, gaps):
    """Ragged lengths and rows of B sequences; those of `gaps` have no rows."""
    lens = rng.integers(0, most, B)
    news = rng.integers(1, rows + 1, B)
    news[gaps] = 0
    lens[[1, B - 1]], news[[1, B - 1]] = [most, most - 1], rows
    return lens.tolist(), news.tolist()


@pytest.mark.parametrize("B,gaps,rows,n_q,n_kv,D", [
    (65, [63, 64], 1, 8, 2, 128), (65, [0], 1, 4, 1, 256), (128, [63, 64, 126], 1, 8, 2, 64), (128, [], 1, 16, 4, 128),
    (200, list(range(60, 140)), 1, 8, 2, 128), (200, list(range(64, 128)), 1, 4, 2, 64),
    (65, [63], 6, 16, 2, 128), (130, [64, 127, 128], 5, 16, 2, 64), (200, list(range(64, 199)), 6, 8, 2, 128), (129, [0, 2, 64], 3, 4, 1, 256),
])
def test_attention_of_many_sequences(sess, B, gaps, rows, n_q, n_kv, D):
    """More sequences than a wave has lanes, and tables of many tiles: items of every 64 sequences are
    cut and joined."""
    rng = np.random.default_rng([B, rows, D])
    lens, news = _lines(rng, B, 320, rows, gaps)
    c = Case(sess, n_q, n_kv, D, 16, lens, news)
    _many(c, lens, news, list(TYPES))


def _many(c, lens, news, dtypes):
    plan = c.plan(behind=2)
    for dtype in dtypes:
        print("many sequences", len(lens), max(news), c.n_q, c.n_kv, c.D, dtype, flush=True)
        q = c.queries(dtype, behind=2)
        window = 0 if dtype == "bf16" else 90
        out = torch.full_like(q, 7.0).cuda()
        plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32(lens), out, max_rows=max(news), window=window)
        c.check(out, q, dtype, window, c.D ** -0.5)
        assert bool((out[int(c.offsets[-1]):] == 7.0).all())
    plan.close()
    c.close()


@pytest.mark.parametrize("B,gaps", [(66, [0]), (70, [63, 64]), (140, list(range(64, 131)))])
def test_attention_of_many_prompts(sess, B, gaps):
    """The same where waves share a tile's expansion: 64 columns a sequence and more, on average too."""
    rng = np.random.default_rng(B)
    lens, news = _lines(rng, B, 330, 20, gaps)
    news = [m + (28 if m and B == 140 else 8 if m else 0) for m in news]
    assert sum(news) * 4 >= 64 * B and max(news) * 4 >= 64
    c = Case(sess, 8, 2, 128, 16, lens, news)
    _many(c, lens, news, ["f16", "bf16"])


@pytest.mark.parametrize("D,rows,columns", [(64, 1, 12 * 16), (64, 40, 8 * 32), (128, 1, 12 * 16), (128, 5, 8 * 32), (128, 600, 256), (256, 1, 4 * 16), (256, 600, 4 * 16)])
def test_plans_take_what_their_calls_can_use(sess, D, rows, columns):
    """Device memory of a plan: two pieces of `columns` columns of the largest form that its rows can take, for
    each compute unit, each D + 2 numbers of 4 bytes; 20 bytes an item; and what allocations are rounded up by."""
    units = torch.cuda.get_device_properties(0).multi_processor_count
    pool = hip.Kv4Pool(sess, 1, 2, D, 16, 4)
    plans, free = [], torch.cuda.mem_get_info()[0]
    for _ in range(8):
        plans.append(hip.Kv4Attention(pool, 8, 2, rows))
    items = 2 * (rows * 4 // 16 + 2)
    assert (free - torch.cuda.mem_get_info()[0]) / 8 <= 2 * columns * units * (D + 2) * 4 + 20 * items + 2 ** 21
    for p in plans:
        p.close()
    pool.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,D", [(1, 128), (40, 64), (70, 128), (3, 256)])
def test_the_largest_queries(sess, dtype, rows, D):
    """Queries next to the type's largest value on small keys: the scores that matter are finite.  The softmax is 1 at the
    largest, token 0 (the others' are at least 1e34 below), whose value is the output."""
    print("largest queries", dtype, rows, D, flush=True)
    n = 300
    c = Case(sess, 4, 2, D, 16, [n], [rows])
    k = (torch.arange(1, n + 1, dtype=torch.float32) * 1e-3)[:, None, None].expand(n, 2, D).contiguous()
    v = torch.tensor(c.rng.standard_normal((n, 2, D)), dtype=torch.float32)
    c.pool.append(0, k.cuda(), v.cuda(), _i32(c.table[0, np.arange(n) // 16] * 16 + np.arange(n) % 16))
    q = torch.full((rows, 4, D), -3e38).to(TYPES[dtype])
    out = torch.zeros_like(q).cuda()
    plan = c.plan()
    plan.run(0, q.cuda(), _i32(c.offsets), _i32(c.table), _i32(c.lens), out, scale=1.0)
    want = np.repeat(P.quantised(P.as_f64(v[:1]))[0], 2, axis=0)
    tol = (2.0 ** -10 if dtype != "f32" else 2.0 ** -21) + torch.finfo(TYPES[dtype]).eps / 2 * 1.01
    assert (np.abs(P.as_f64(out) - want) <= tol * np.abs(want)).all()
    plan.close()
    c.close()
