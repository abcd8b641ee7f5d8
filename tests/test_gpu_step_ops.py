"""Step maps and draft verification on the GPU against their definitions: whole
numbers, so everything is equal.  (Drawn numbers come from fixed seeds; a sum
over the vocabulary in 64 bits is off by about 1e-16 of itself, so the chance
that one of them lies between two forms' borders is below 1e-9 a token.)"""
import numpy as np
import pytest
import torch

import kv4_plain as P
from rstr import configs, hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sess():
    with hip.Session(0) as s:
        yield s


def _i32(a):
    return torch.tensor(np.asarray(a, np.int64), dtype=torch.int32, device="cuda")


def _maps(sess, page, lengths, counts, free, table, rows, starts=None):
    B = len(lengths)
    t = _i32(table)
    got = dict(new_lengths=torch.full((B,), -9, dtype=torch.int32, device="cuda"), offsets=torch.full((B + 1,), -9, dtype=torch.int32, device="cuda"),
               positions=torch.full((rows,), -9, dtype=torch.int32, device="cuda"), slots=torch.full((rows,), -9, dtype=torch.int32, device="cuda"),
               taken=torch.full((1,), -9, dtype=torch.int32, device="cuda"))
    sess.step_maps(page, _i32(lengths), _i32(counts), _i32(free), t, got["new_lengths"], got["offsets"], got["positions"], got["slots"],
                   got["taken"], starts=None if starts is None else _i32(starts))
    return dict(got, table=t)


@pytest.mark.parametrize("B,hi,new,page,free,slack", [
    (1, 1, 1, 16, 9, 0), (1, 0, 40, 16, 9, 3), (5, 100, 1, 16, 9, 0), (7, 64, 33, 16, 50, 5), (64, 200, 5, 48, 12, 0),
    (513, 90, 4, 16, 40, 0), (1000, 300, 100, 16, 3000, 2), (8192, 40, 3, 16, 2000, 7), (33, 50, 9, 1, 170, 0), (20, 50, 30, 16, 0, 0),
    (30, 100, 50, 16, 1000, -200),
])
def test_step_maps(sess, B, hi, new, page, free, slack):
    print("maps", B, hi, new, page, free, slack, flush=True)
    rng = np.random.default_rng(B + hi)
    lengths, counts = rng.integers(0, hi + 1, B), rng.integers(0, new + 1, B)
    if B == 1:
        counts[0] = new
    width = -(-(hi + new) // page)
    if B > 6:
        lengths[2], counts[3], counts[5] = -1, -4, hi + new * page + 1000   # out of range: left alone
        lengths[4] = width * page + 5
    table = rng.integers(0, 10 ** 6, (B, width))
    free_pages = rng.permutation(10 ** 6)[:free]
    rows = max(0, int(np.clip(counts, 0, new).sum()) + slack)
    starts = rng.integers(0, 1000, B) if B % 2 else None
    got = _maps(sess, page, lengths, counts, free_pages, table, rows, starts)
    want = P.step_maps(page, lengths, counts, starts, free_pages, table, rows)
    for name in want:
        assert np.array_equal(got[name].cpu().numpy(), np.asarray(want[name]).reshape(got[name].shape)), name


def test_step_maps_slots_past_31_bits(sess):
    """Page ids whose slots do not fit are no slots: none wraps round to another page's."""
    page, top = 48, 2 ** 31 - 1
    table = np.array([[top, 3, 0, 0], [top // page, 0, 0, 0], [top // page + 1, 0, 0, 0], [-(2 ** 31), 0, 0, 0]])
    lengths, counts, free = np.array([40, 20, 47, 5]), np.array([20, 30, 2, 3]), np.array([top, 2, 2 ** 28])
    got = _maps(sess, page, lengths, counts, free, table, 60)
    want = P.step_maps(page, lengths, counts, None, free, table, 60)
    for name in want:
        assert np.array_equal(got[name].cpu().numpy(), np.asarray(want[name]).reshape(got[name].shape)), name
    assert -1 in want["slots"][:55] and max(want["slots"]) > 2 ** 31 - 100


def test_step_maps_graph_and_loop(sess):
    """A captured call advances the tables step after step, its lengths fed back."""
    B, page, width = 40, 16, 30
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 60, B)
    have = -(-lens // page)
    perm = rng.permutation(2000)
    table = np.full((B, width), -1)
    at = 0
    for b, n in enumerate(have):
        table[b, :n] = perm[at:at + n]
        at += n
    free = perm[at:]
    d = dict(lengths=_i32(lens), counts=_i32(np.ones(B)), free=_i32(free[:200]), table=_i32(table), new=_i32(lens * 0), offs=_i32(np.zeros(B + 1)),
             pos=_i32(np.zeros(200)), slots=_i32(np.zeros(200)), taken=_i32([0]))
    call = lambda: sess.step_maps(page, d["lengths"], d["counts"], d["free"], d["table"], d["new"], d["offs"], d["pos"], d["slots"], d["taken"])  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    d["table"].copy_(_i32(table))
    for step in range(6):
        counts = rng.integers(0, 6, B)
        d["counts"].copy_(_i32(counts))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = P.step_maps(page, lens, counts, None, free[:200], table, 200)
        for k, name in (("table", "table"), ("new", "new_lengths"), ("offs", "offsets"), ("pos", "positions"), ("slots", "slots"), ("taken", "taken")):
            assert np.array_equal(d[k].cpu().numpy(), np.asarray(want[name]).reshape(d[k].shape)), (step, name)
        table, lens = want["table"], np.asarray(want["new_lengths"])
        free = free[want["taken"][0]:]
        d["lengths"].copy_(d["new"])
        d["free"].copy_(_i32(free[:200]))


# ---- verification --------------------------------------------------------------------------
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _verify_case(rng, news, V, dtype, probs, temps, masked=True):
    R = int(sum(news))
    x = rng.standard_normal((R, V)) * 2
    x[np.arange(R), rng.integers(0, V, R)] += 6
    if masked and V > 3:
        x[rng.random((R, V)) < 0.2] = -np.inf
        x[np.arange(R), rng.integers(0, V, R)] = 1.0
    logits = torch.tensor(x).to(TYPES[dtype])
    xf = P.as_f64(logits)
    q = None
    y = np.where(np.isfinite(xf), xf, -50.0) * 0.9 + rng.standard_normal((R, V)) * 0.3
    y = np.exp(y - y.max(1, keepdims=True))
    y /= y.sum(1, keepdims=True)
    drafts = np.array([rng.choice(V, p=r) for r in y])
    if probs:
        q = y.astype(np.float32)
    return logits, xf, q, drafts, np.resize(np.asarray(temps, np.float32), len(news))


def _run_verify(sess, logits, offs, drafts, q, temps, ua, us, pad=0):
    R, V = logits.shape
    B = len(offs) - 1
    v = hip.Verifier(sess, B, R, V)
    acc = torch.full((B,), -9, dtype=torch.int32, device="cuda")
    tok = torch.full((R,), -7, dtype=torch.int32, device="cuda")
    f = lambda a: torch.tensor(np.asarray(a, np.float32), device="cuda")  # noqa: E731
    x = torch.zeros(R, V + pad, dtype=logits.dtype, device="cuda")[:, :V]
    x.copy_(logits.cuda())
    p = None
    if q is not None:
        p = torch.zeros(R, V + pad, device="cuda")[:, :V]
        p.copy_(f(q))
    v.run(x, _i32(offs), _i32(drafts), f(temps), f(ua), f(us), acc, tok, draft_probs=p)
    a, t = acc.cpu().numpy(), tok.cpu().numpy()
    v.close()
    return a, t


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("V,news,temps", [
    (1, [1, 2], [1.0]), (17, [3, 0, 1, 5], [1.0, 0.5]), (4096, [6, 2], [0.7]), (4097, [1, 1, 9], [1.3, 0.0, 1.0]),
    (1000, [4] * 40, [0.0, 1.0, -1.0, np.nan, np.inf, 1e-3, 30.0]), (131071, [5, 3], [1.0]), (50000, [2] * 9, [0.9]),
])
def test_verify(sess, dtype, probs, V, news, temps):
    print("verify", dtype, probs, V, len(news), flush=True)
    rng = np.random.default_rng([V, len(news), probs])
    logits, xf, q, drafts, T = _verify_case(rng, news, V, dtype, probs, temps)
    R = len(drafts)
    offs = np.concatenate([[0], np.cumsum(news)])
    for pad in (0, 3):
        ua, us = rng.random(R).astype(np.float32), rng.random(len(news)).astype(np.float32)
        got = _run_verify(sess, logits, offs, drafts, q, T, ua, us, pad)
        want = P.verify(xf, offs, drafts, q, T, ua, us)
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


def test_verify_edges(sess):
    """Drafts outside the vocabulary, rows without a finite maximum, ties, residuals that are empty, extreme random
    numbers, all accepted, none accepted, rows behind the last sequence."""
    V = 5000
    rng = np.random.default_rng(3)
    news = [3, 3, 2, 2, 2, 4, 1, 3]
    logits, xf, q, drafts, T = _verify_case(rng, news, V, "f32", True, [1.0], masked=False)
    offs = np.concatenate([[0], np.cumsum(news)])
    drafts[0], drafts[offs[1]], drafts[offs[1] + 1] = V, -1, 2 ** 31 - 1
    x = xf.copy()
    x[offs[2]] = -np.inf
    x[offs[3], 77] = np.nan
    x[offs[3], 4999] = np.inf
    drafts[offs[3]] = 77
    x[offs[4], :] = 1.25                          # every token ties
    drafts[offs[4]] = 0
    T[4] = 0.0
    q[offs[5]:offs[6]] = np.exp(x[offs[5]:offs[6]] - x[offs[5]:offs[6]].max(1, keepdims=True))
    q[offs[5]:offs[6]] *= 2.0                     # above p everywhere: p - q has nothing left
    x[offs[6], 10] = 1e4                          # one certain token
    x[offs[7]:offs[8], 123] = 1e4
    drafts[offs[7]:offs[8]] = 123                 # certain drafts: all accepted
    for lo in (0.0, 0.5, np.float32(1) - np.float32(2 ** -24)):
        for hi in (0.0, np.float32(1) - np.float32(2 ** -24)):
            ua, us = np.full(len(drafts), lo, np.float32), np.full(len(news), hi, np.float32)
            for probs in (q, None):
                got = _run_verify(sess, torch.tensor(x).float(), offs, drafts, probs, T, ua, us)
                want = P.verify(x.astype(np.float32).astype(np.float64), offs, drafts, probs, T, ua, us)
                assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), (lo, hi, probs is None)
    R = len(drafts)
    ua, us = rng.random(R).astype(np.float32), rng.random(8).astype(np.float32)
    short = offs[:5]                              # four sequences: the other rows are left as they are
    got = _run_verify(sess, torch.tensor(x).float(), short, drafts, q, T[:4], ua, us[:4])
    want = P.verify(x.astype(np.float32).astype(np.float64), short, drafts, q, T[:4], ua, us[:4])
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]) and (got[1][offs[4]:] == -7).all()
    for bad in ([0, 2 ** 31 - 1], [-5, 3], [9, 2, 40]):  # offsets that are none: bounded
        _run_verify(sess, torch.tensor(x).float(), bad, drafts, q, T[:len(bad) - 1], ua, us[:len(bad) - 1])
        torch.cuda.synchronize()


def test_verify_draws_as_the_target(sess):
    """Over many draws the tokens follow the target's distribution whatever drafted them: of 20000 sequences each of
    16 tokens' shares lies within five standard deviations."""
    V, B = 16, 20000
    rng = np.random.default_rng(9)
    x = np.repeat(rng.standard_normal((1, V)) * 1.5, 2 * B, 0).astype(np.float32)
    y = np.exp(rng.standard_normal(V))
    y = (y / y.sum()).astype(np.float32)
    drafts = rng.choice(V, p=y.astype(np.float64) / y.astype(np.float64).sum(), size=2 * B)
    offs = np.arange(0, 2 * B + 1, 2)
    _, tok = _run_verify(sess, torch.tensor(x), offs, drafts, np.repeat(y[None], 2 * B, 0), np.ones(B), rng.random(2 * B), rng.random(B))
    p = np.exp(x[0].astype(np.float64))
    p /= p.sum()
    share = np.bincount(tok[::2], minlength=V) / B
    assert np.all(np.abs(share - p) < 5 * np.sqrt(p * (1 - p) / B) + 1e-9)


def test_decoder_step_verified_where_it_is(sess):
    """Drafted tokens as lanes of one decode step on one route, and their verification on the
    step's resident logits: greedy, the kept tokens equal plain decoding's."""
    cfg = configs.TINY_LLAMA
    ps, pages, pps, split = 16, 12, 6, 64
    first, k = 7, 4
    m = hip.Model(sess, cfg, seed=1)

    def decoder(batch):
        p = hip.Pool(m, ps, pages)
        return p, hip.Decoder(m, p, batch, pps, 96, split)

    def step(d, at, n):
        pos = np.arange(at, at + n)
        pt = np.tile(np.arange(pps), (n, 1))
        return d.step_lanes(pos, np.arange(n + 1), pos, pt, pos + 1, np.zeros(n))

    pool1, one = decoder(1)
    one.prime_lanes([0], [first])
    plain = [int(step(one, t, 1)[0]) for t in range(k + 1)]      # each token is the next step's input
    pool2, many = decoder(k + 1)
    for wrong in (None, 0, 2):
        drafts = list(plain[:k])
        if wrong is not None:
            drafts[wrong] = (drafts[wrong] + 1) % cfg["vocab"]
        many.prime_lanes(np.arange(k + 1), [first] + drafts)
        step(many, 0, k + 1)
        logits = many.logits_device()
        v = hip.Verifier(sess, 1, k + 1, cfg["vocab"])
        acc, tok = _i32([-9]), _i32([-9] * (k + 1))
        z = torch.zeros(k + 1, device="cuda")
        v.run(logits, _i32([0, k + 1]), _i32(drafts + [0]), torch.zeros(1, device="cuda"), z, z[:1], acc, tok)
        kept = k if wrong is None else wrong
        assert acc.item() == kept and tok.tolist() == plain[:kept + 1] + [-1] * (k - kept)
        assert torch.equal(torch.as_tensor(logits, device="cuda").cpu(), torch.tensor(many.logits()))
        v.close()
    for x in (one, many, pool1, pool2, m):
        x.close()


def test_the_step_as_a_whole(sess):
    """Maps, append, attention and verification together, captured once and replayed step after step with its own
    results fed back, against the plain forms."""
    B, n_q, n_kv, D, page, width, V, most = 5, 8, 2, 64, 16, 20, 700, 4
    rng = np.random.default_rng(11)
    pages = 90
    pool = hip.Kv4Pool(sess, 1, n_kv, D, page, pages)
    rows = B * most
    plan, ver = hip.Kv4Attention(pool, n_q, B, rows), hip.Verifier(sess, B, rows, V)
    f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    d = dict(lengths=i(B), counts=i(B), free=i(60), table=torch.full((B, width), -1, dtype=torch.int32, device="cuda"), new=i(B), offs=i(B + 1),
             pos=i(rows), slots=i(rows), taken=i(1), q=f(rows, n_q, D).half(), k=f(rows, n_kv, D).half(), v=f(rows, n_kv, D).half(),
             out=f(rows, n_q, D).half(), logits=f(rows, V), probs=f(rows, V), drafts=i(rows), T=torch.ones(B, device="cuda"), ua=f(rows), us=f(B),
             acc=i(B), tok=i(rows))

    def call():
        sess.step_maps(page, d["lengths"], d["counts"], d["free"], d["table"], d["new"], d["offs"], d["pos"], d["slots"], d["taken"])
        pool.append(0, d["k"], d["v"], d["slots"])
        plan.run(0, d["q"], d["offs"], d["table"], d["new"], d["out"], max_rows=most)
        ver.run(d["logits"], d["offs"], d["drafts"], d["T"], d["ua"], d["us"], d["acc"], d["tok"], draft_probs=d["probs"])

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    torch.cuda.synchronize()
    lens, table, free = np.zeros(B, np.int64), np.full((B, width), -1), rng.permutation(pages)
    keep = [np.zeros((0, n_kv, D))] * B, [np.zeros((0, n_kv, D))] * B
    for step in range(7):
        counts = rng.integers(0 if step else 1, most + 1, B)
        R = int(counts.sum())
        logits, xf, q, drafts, _ = _verify_case(rng, [rows], V, "f32", True, [1.0], masked=False)
        new = dict(counts=counts, lengths=lens, free=free[:60], drafts=drafts)
        for n, a in new.items():
            d[n].copy_(_i32(a))
        rand = lambda *s: torch.tensor(rng.standard_normal(s)).half()  # noqa: E731
        k, v, qq = rand(rows, n_kv, D), rand(rows, n_kv, D), rand(rows, n_q, D)
        ua, us = rng.random(rows).astype(np.float32), rng.random(B).astype(np.float32)
        for n, a in dict(k=k, v=v, q=qq, logits=logits, probs=torch.tensor(q), ua=torch.tensor(ua), us=torch.tensor(us)).items():
            d[n].copy_(a)
        d["table"].copy_(_i32(table))
        d["tok"].fill_(-7)
        d["out"].fill_(5.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = P.step_maps(page, lens, counts, None, free[:60], table, rows)
        for key, name in (("table", "table"), ("new", "new_lengths"), ("offs", "offsets"), ("pos", "positions"), ("slots", "slots")):
            assert np.array_equal(d[key].cpu().numpy(), np.asarray(want[name]).reshape(d[key].shape)), (step, name)
        offs, table, free = want["offsets"], want["table"], free[want["taken"][0]:]
        kq, vq = P.quantised(P.as_f64(k)), P.quantised(P.as_f64(v))
        full = [np.concatenate([keep[0][b], kq[offs[b]:offs[b + 1]]]) for b in range(B)], [np.concatenate([keep[1][b], vq[offs[b]:offs[b + 1]]]) for b in range(B)]
        o, mag, _ = P.attention(P.as_f64(qq), full[0], full[1], want["new_lengths"], offs, 0, D ** -0.5)
        got = P.as_f64(d["out"])
        # a probability and its product with a scale are rounded to fp16: at most 2^-11 of it each, 2^-10 together
        # (2^-11 would be the sum of two quarter steps); scores in fp32: 1e-5 of a weight here; the output's own half step
        past = np.abs(got[:R] - o[:R]) - ((2.0 ** -10 + 1e-5) * mag[:R] + 2.0 ** -11 * np.abs(o[:R]) + 1e-7)
        at = np.unravel_index(past.argmax(), past.shape)
        assert past.max() <= 0, (step, at, past.max(), got[at], o[at], mag[at])
        assert bool((got[R:] == 5.0).all())
        a, t = P.verify(xf, offs, drafts, q, np.ones(B), ua, us)
        assert np.array_equal(d["acc"].cpu().numpy(), a) and np.array_equal(d["tok"].cpu().numpy(), t)
        # what was refused leaves the sequences: the next step writes over it
        lens = lens + np.where(counts > 0, a + 1, 0)
        lens = np.minimum(lens, want["new_lengths"])
        keep = [full[0][b][:lens[b]] for b in range(B)], [full[1][b][:lens[b]] for b in range(B)]
        pages_now = -(-lens // page)
        for b in range(B):
            back = [p for p in table[b, pages_now[b]:] if p >= 0]
            table[b, pages_now[b]:] = -1
            free = np.concatenate([free, back]).astype(np.int64)
    ver.close()
    plan.close()
    pool.close()


def test_step_maps_lengths_past_31_bits(sess):
    """Pages so large that a table holds more tokens than a length can say: a sequence whose new length does not fit 31 bits
    is refused, one that just fits is served."""
    page, top = 2 ** 30, 2 ** 31 - 1
    lengths, counts = np.array([top, top - 4, top - 4, 5]), np.array([1, 5, 4, top])
    table = np.array([[3, 4, 5, 6], [0, 1, 2, 3], [0, 1, 2, 3], [0, 1, 2, 3]])
    got = {k: v.cpu().tolist() for k, v in _maps(sess, page, lengths, counts, np.array([7, 8]), table, 6).items()}
    assert got["new_lengths"] == [top, top - 4, top, 5] and got["offsets"] == [0, 0, 0, 4, 4]
    assert got["positions"] == [top - 4, top - 3, top - 2, top - 1, 0, 0]
    assert got["slots"] == [top - 4, top - 3, top - 2, top - 1, -1, -1]
    assert got["taken"] == [0] and got["table"] == table.tolist()
