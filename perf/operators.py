"""The operators of a serving step that drafts tokens over a 4-bit paged cache, as cases that can be timed
and compared: the step's page tables and slot maps made on the GPU, K/V rows quantised into the cache and
read back, attention over it for one or several new tokens per sequence, and the verification of drafted
tokens against the target's logits.

``own`` false computes them in plain torch operations; ``own`` true calls the framework (``rstr.hip``) on
the same inputs.  Lengths and row counts of a case are the quantiles of its distribution, dealt to the
sequences by the seed, so every seed does the same work.  A cache block is 32 consecutive elements of a
head's row: an fp16 scale d and 32 four-bit codes, standing for d * (code - 8).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
BLOCK = 32


def listed():
    return [
        # one user who has just begun: the shortest call of attention, where only latency counts
        dict(name="attend_1lane_short", kind="attend", n_q=32, n_kv=8, hd=128, dtype="f16", lanes=1, lo=37, hi=37,
             new_lo=1, new_hi=1, window=0, page=16),
        # a full server of an 8B model: one token each for 128 users at ragged lengths
        dict(name="attend_128lane", kind="attend", n_q=32, n_kv=8, hd=128, dtype="f16", lanes=128, lo=128, hi=4608,
             new_lo=1, new_hi=1, window=0, page=16),
        # a few very long contexts, one token each: the work has to be split along them
        dict(name="attend_3lane_long", kind="attend", n_q=32, n_kv=8, hd=128, dtype="bf16", lanes=3, lo=20161, hi=131072,
             new_lo=1, new_hi=1, window=0, page=64),
        # drafted tokens: one to six new rows per sequence, fp32 queries as the decode step holds them
        dict(name="attend_drafts_f32", kind="attend", n_q=16, n_kv=8, hd=128, dtype="f32", lanes=33, lo=5, hi=8192,
             new_lo=1, new_hi=6, window=0, page=16),
        # a prompt's last tile and a short one beside it
        dict(name="attend_prompt", kind="attend", n_q=32, n_kv=8, hd=128, dtype="bf16", lanes=2, lo=77, hi=4096,
             new_lo=77, new_hi=512, window=0, page=16),
        # a small model's sliding windows, head dim 256, a few rows each
        dict(name="attend_window_f32", kind="attend", n_q=4, n_kv=1, hd=256, dtype="f32", lanes=16, lo=64, hi=2048,
             new_lo=1, new_hi=3, window=512, page=16),
        # the rows that one decode step of 128 users brings
        dict(name="append_128", kind="append", n_kv=8, hd=128, dtype="f32", rows=128, page=16),
        # the rows of a layer of a long prompt
        dict(name="append_prompt", kind="append", n_kv=8, hd=128, dtype="bf16", rows=16411, page=16),
        # tables of a step of a handful of users
        dict(name="maps_5", kind="maps", lanes=5, lo=1, hi=8192, new_lo=1, new_hi=1, page=16, table=515),
        # tables of a large batch in which some bring whole prompt tiles
        dict(name="maps_1000_tiles", kind="maps", lanes=1000, lo=1, hi=16384, new_lo=0, new_hi=128, page=16, table=1056),
        # a few users with four drafted tokens each, drafts made without probabilities
        dict(name="verify_3_lookup", kind="verify", lanes=3, vocab=151936, new_lo=5, new_hi=5, dtype="f32", probs=False,
             temperature=0.8),
        # a server's verification step: up to five drafts a user, with the drafting model's probabilities
        dict(name="verify_64", kind="verify", lanes=64, vocab=128256, new_lo=1, new_hi=6, dtype="f32", probs=True,
             temperature=1.0),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choices(("attend", "append", "maps", "verify"), (5, 2, 2, 3))[0]
    if kind == "attend":
        n_q, n_kv, hd = rng.choice(((32, 8, 128), (32, 8, 128), (16, 8, 128), (4, 1, 256), (8, 2, 64), (8, 8, 64), (24, 1, 128)))
        dtype, page = rng.choice(("f32", "f16", "bf16")), rng.choice((16, 16, 32, 48, 64))
        form = rng.choice(("token", "token", "drafts", "prompt"))
        if form == "prompt":
            new = log_int(17, 512)
            hi = new + log_int(1, 3000)
            return dict(kind=kind, n_q=n_q, n_kv=n_kv, hd=hd, dtype=dtype, lanes=rng.choice((1, 1, 2)), lo=new, hi=hi,
                        new_lo=rng.randint(1, new), new_hi=new, window=rng.choice((0, 0, 0, 257, 512)), page=page)
        lanes = log_int(1, 128)
        hi = log_int(1, min(131072, 240000 // lanes))
        new = 1 if form == "token" else rng.randint(2, 8)
        return dict(kind=kind, n_q=n_q, n_kv=n_kv, hd=hd, dtype=dtype, lanes=lanes, lo=max(1, hi // rng.choice((1, 7, 40))), hi=hi,
                    new_lo=1, new_hi=min(new, hi), window=rng.choice((0, 0, 0, 100, 512)), page=page)
    if kind == "append":
        n_kv, hd = rng.choice(((8, 128), (1, 256), (2, 64), (8, 64)))
        return dict(kind=kind, n_kv=n_kv, hd=hd, dtype=rng.choice(("f32", "f16", "bf16")), rows=log_int(1, 8000),
                    page=rng.choice((16, 32, 48)))
    if kind == "maps":
        lanes, page = log_int(1, 1000), rng.choice((16, 16, 48, 64))
        hi, new = log_int(16, 16384), rng.choice((1, 1, 5, log_int(2, 128)))
        return dict(kind=kind, lanes=lanes, lo=1, hi=hi, new_lo=rng.choice((0, 1)), new_hi=new, page=page,
                    table=-(-(hi + new) // page) + rng.choice((0, 1, 13)))
    lanes = log_int(1, 48)
    return dict(kind=kind, lanes=lanes, vocab=log_int(1000, 128256), new_lo=rng.randint(1, 3), new_hi=rng.randint(3, 6),
                dtype=rng.choice(("f32", "f16", "bf16")), probs=rng.random() < 0.6, temperature=rng.choice((0.0, 0.3, 0.7, 1.0, 1.3)))


# ---- sizes of a case ------------------------------------------------------------------------------


def _spread(n, lo, hi, log):
    p = [(i + 0.5) / n for i in range(n)]
    if log:
        return [int(min(hi, max(lo, round(math.exp(math.log(lo) + x * (math.log(hi) - math.log(lo))))))) for x in p]
    return [int(min(hi, max(lo, round(lo + x * (hi - lo))))) for x in p]


def _sequences(case):
    """[(length, new rows)] of the sequences, shortest first: every case's work follows from it."""
    n = case["lanes"]
    news = _spread(n, case["new_lo"], case["new_hi"], False)
    news = [news[i * 7 % n] if n % 7 else news[i] for i in range(n)]  # not in the lengths' order
    if case["kind"] == "verify":
        return [(0, m) for m in news]
    lens = _spread(n, case["lo"], case["hi"], case["hi"] > 10 * case["lo"] and case["hi"] > 10000)
    if n == 2:  # the long one and the short one, as their bounds say
        lens, news = [case["lo"], case["hi"]], [case["new_lo"], case["new_hi"]]
    return [(max(a, m) if case["kind"] == "attend" else a, m) for a, m in zip(lens, news)]


def _dealt(case, seed):
    """(lengths, new rows) by sequence of this seed, as int arrays."""
    pairs = _sequences(case)
    order = np.random.default_rng(seed).permutation(len(pairs))
    a = np.array([pairs[i] for i in order], np.int64).reshape(-1, 2)
    return a[:, 0], a[:, 1]


def work(case):
    kind = case["kind"]
    if kind == "attend":
        n_q, n_kv, hd, w, size = case["n_q"], case["n_kv"], case["hd"], case["window"], SIZES[case["dtype"]]
        seen = pairs = rows = 0
        for length, m in _sequences(case):
            seen += min(length, w + m - 1) if w else length
            pairs += sum(min(p + 1, w) if w else p + 1 for p in range(length - m, length))
            rows += m
        return {"bytes": seen * n_kv * hd * 2 * 9 // 16 + 2 * rows * n_q * hd * size, "flops": 4 * n_q * hd * pairs}
    if kind == "append":  # rows in, blocks written, blocks read, rows out
        elems = 2 * case["rows"] * case["n_kv"] * case["hd"]
        return {"bytes": 2 * elems * SIZES[case["dtype"]] + 2 * elems * 9 // 16 + 8 * case["rows"], "flops": 4 * elems}
    seqs = _sequences(case)
    rows = sum(m for _, m in seqs)
    if kind == "maps":
        pages = sum(-(-(a + m) // case["page"]) - -(-a // case["page"]) for a, m in seqs)
        return {"bytes": 4 * (4 * len(seqs) + 2 * rows + 2 * pages), "flops": 8 * (rows + len(seqs))}
    refused = len(seqs) if case["probs"] else 0
    return {"bytes": case["vocab"] * (rows * SIZES[case["dtype"]] + 4 * refused), "flops": 3 * case["vocab"] * rows}


# ---- inputs -----------------------------------------------------------------------------------------


def _dev(a, dtype=torch.int32):
    return torch.from_numpy(np.ascontiguousarray(a)).to("cuda", dtype)


def _hip():
    pkg = os.path.join(os.getcwd(), "pretrained-rstr_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from rstr import hip

    return hip


_session = None


def _open_session():
    """The program's session: one, as long as the process lives."""
    global _session
    if _session is None:
        _session = _hip().Session(0)
    return _session


class _Held(dict):
    """A case's inputs, with the handles that a serving program keeps; closed with the object."""

    def __del__(self):
        for name in ("plan", "pool"):
            if name in self:
                self.pop(name).close()


def _paged(seqs_pages, pages, width, rng):
    """A page table of a shuffled pool: [sequences][width], -1 behind a sequence's pages."""
    perm = rng.permutation(pages)
    table = np.full((len(seqs_pages), width), -1, np.int64)
    at = 0
    for b, n in enumerate(seqs_pages):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, perm[at:]


def _rows_kv(g, rows, case):
    """K and V rows of one layer: normal values, a few channels of larger ones, as keys have them."""
    n_kv, hd, dt = case["n_kv"], case["hd"], DTYPES[case["dtype"]]
    k = torch.randn(rows, n_kv, hd, generator=g, device="cuda")
    k[..., hd // 2:: 17] *= 4.0
    v = torch.randn(rows, n_kv, hd, generator=g, device="cuda") * 0.7
    return k.to(dt), v.to(dt)


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(int(seed))
    rng = np.random.default_rng([int(seed), 7])
    return {"attend": _prepare_attend, "append": _prepare_append, "maps": _prepare_maps,
            "verify": _prepare_verify}[case["kind"]](case, int(seed), g, rng)


def _prepare_attend(case, seed, g, rng):
    lens, news = _dealt(case, seed)
    page, n_q, hd = case["page"], case["n_q"], case["hd"]
    need = -(-lens // page)
    pages = int(need.sum()) + 3
    table, _ = _paged(need, pages, int(need.max()), rng)
    offs = np.concatenate([[0], np.cumsum(news)])
    rows = int(offs[-1])
    pos = np.concatenate([np.arange(a) for a in lens])
    slots = _dev(table[np.repeat(np.arange(len(lens)), lens), pos // page] * page + pos % page)
    s = _Held(case=case, lengths=_dev(lens), offsets=_dev(offs), table=_dev(table), longest=int(lens.max()),
              most=int(news.max()), scale=hd ** -0.5, batch=len(lens))
    kv = dict(case, dtype="f16")
    k, v = _rows_kv(g, int(lens.sum()), kv)
    q = torch.randn(rows, n_q, hd, generator=g, device="cuda") * 1.5
    s["q"] = q.to(DTYPES[case["dtype"]])
    s["out"] = torch.empty_like(s["q"])
    if own:
        hip = _hip()
        s["pool"] = hip.Kv4Pool(_open_session(), 1, case["n_kv"], hd, page, pages)
        s["plan"] = hip.Kv4Attention(s["pool"], n_q, len(lens), rows)
        s["pool"].append(0, k, v, slots)
    else:
        at = slots.long()
        for name, x in (("k", k), ("v", v)):
            d, c = _quantise(x)
            s[name + "d"] = torch.zeros(pages * page, *d.shape[1:], dtype=torch.float16, device="cuda")
            s[name + "c"] = torch.full((pages * page, *c.shape[1:]), 8, dtype=torch.uint8, device="cuda")
            s[name + "d"][at], s[name + "c"][at] = d, c
    return s


def _prepare_append(case, seed, g, rng):
    rows, page = case["rows"], case["page"]
    pages = -(-rows // page) + 5
    slots = rng.permutation(pages * page)[:rows] if rows <= 256 else (
        (rng.permutation(pages)[:, None] * page + np.arange(page)).reshape(-1)[3:3 + rows])
    k, v = _rows_kv(g, rows, case)
    s = _Held(case=case, k=k, v=v, slots=_dev(slots))
    if own:
        s["pool"] = _hip().Kv4Pool(_open_session(), 1, case["n_kv"], case["hd"], page, pages)
        s["k_out"], s["v_out"] = torch.empty_like(k), torch.empty_like(v)
    else:
        for name in "kv":
            s[name + "d"] = torch.zeros(pages * page, case["n_kv"], case["hd"] // BLOCK, dtype=torch.float16, device="cuda")
            s[name + "c"] = torch.full((pages * page, case["n_kv"], case["hd"]), 8, dtype=torch.uint8, device="cuda")
    return s


def _prepare_maps(case, seed, g, rng):
    lens, news = _dealt(case, seed)
    page = case["page"]
    have, want = -(-lens // page), -(-(lens + news) // page)
    spare = int((want - have).sum())
    free = spare + 9 if seed % 3 else max(1, spare * 9 // 10)  # now and then the pages run out
    table, left = _paged(have, int(have.sum()) + free, case["table"], rng)
    return _Held(case=case, lengths=_dev(lens), counts=_dev(news), starts=_dev(rng.integers(0, 50, len(lens))),
                 free=_dev(left[:free]), old=_dev(table), rows=int(news.sum()), table=_dev(table),
                 new_lengths=_dev(lens * 0), offsets=_dev(np.zeros(len(lens) + 1)),
                 positions=_dev(np.zeros(max(1, news.sum()))), slots=_dev(np.zeros(max(1, news.sum()))), taken=_dev(np.zeros(1)))


def _prepare_verify(case, seed, g, rng):
    _, news = _dealt(case, seed)
    V, rows = case["vocab"], int(news.sum())
    offs = np.concatenate([[0], np.cumsum(news)])
    x = torch.randn(rows, V, generator=g, device="cuda") * 2.5
    top = torch.randint(0, V, (rows, 4), generator=g, device="cuda")
    x.scatter_add_(1, top, torch.rand(rows, 4, generator=g, device="cuda") * 9.0 + 4.0)  # some likely tokens
    logits = x.to(DTYPES[case["dtype"]])
    u = torch.rand(rows + len(news), generator=g, device="cuda")
    s = _Held(case=case, logits=logits, offsets=_dev(offs), most=int(news.max()), batch=len(news),
              temperature=torch.full((len(news),), case["temperature"], device="cuda"),
              u_accept=u[:rows].clone(), u_sample=u[rows:].clone(), probs=None,
              accepted=torch.empty(len(news), dtype=torch.int32, device="cuda"),
              tokens=torch.empty(rows, dtype=torch.int32, device="cuda"))
    # what a smaller model drafted: the target's distribution, blurred
    y = x * 0.9 + torch.randn(rows, V, generator=g, device="cuda") * 0.5
    y = torch.exp(y - y.amax(1, keepdim=True))
    y /= y.sum(1, keepdim=True)
    s["drafts"] = torch.multinomial(y, 1, generator=g).reshape(-1).to(torch.int32)
    if case["probs"]:
        s["probs"] = y
    if own:
        s["plan"] = _hip().Verifier(_open_session(), len(news), rows, V)
    return s


# ---- one pass ----------------------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"attend": _own_attend, "append": _own_append, "maps": _own_maps, "verify": _own_verify}[kind](s)
    return {"attend": _attend, "append": _append, "maps": _maps, "verify": _verify}[kind](s)


def _own_attend(s):
    s["plan"].run(0, s["q"], s["offsets"], s["table"], s["lengths"], s["out"], max_rows=s["most"], window=s["case"]["window"],
                  scale=s["scale"])
    return s["out"]


def _own_append(s):
    s["pool"].append(0, s["k"], s["v"], s["slots"])
    s["pool"].read(0, s["slots"], s["k_out"], s["v_out"])
    return s["k_out"], s["v_out"]


def _own_maps(s):
    _open_session().step_maps(s["case"]["page"], s["lengths"], s["counts"], s["free"], s["table"], s["new_lengths"], s["offsets"],
                              s["positions"], s["slots"], s["taken"], starts=s["starts"])
    return {k: s[k] for k in ("table", "new_lengths", "offsets", "positions", "slots", "taken")}


def _own_verify(s):
    s["plan"].run(s["logits"], s["offsets"], s["drafts"], s["temperature"], s["u_accept"], s["u_sample"], s["accepted"], s["tokens"],
                  draft_probs=s["probs"])
    return s["accepted"], s["tokens"]


# ---- the plain forms -----------------------------------------------------------------------------------


def _quantise(x):
    """Blocks of rows [..., D]: (scales fp16 [..., D/32], codes [..., D])."""
    b = x.float().unflatten(-1, (-1, BLOCK))
    a = b.abs()
    at = torch.arange(BLOCK, device=x.device)
    first = torch.where(a == a.amax(-1, keepdim=True), at, BLOCK).amin(-1, keepdim=True)  # of the greatest magnitude
    d = (b.gather(-1, first) / -8.0).clamp(-65504.0, 65504.0).half()
    q = torch.round(b.double() / d.double())  # halves to even; 64 bits: values next to a half
    q = torch.where(d == 0, 0.0, q).clamp(-8, 7) + 8
    return d.squeeze(-1), q.to(torch.uint8).flatten(-2)


def _values(d, c):
    """What blocks stand for, in float32 (exactly)."""
    return ((c.float() - 8.0).unflatten(-1, (-1, BLOCK)) * d.float().unsqueeze(-1)).flatten(-2)


def _append(s):
    at = s["slots"].long()
    out = []
    for name in "kv":
        d, c = _quantise(s[name])
        s[name + "d"][at], s[name + "c"][at] = d, c
        out.append(_values(s[name + "d"][at], s[name + "c"][at]).to(s[name].dtype))
    return tuple(out)


def _attend(s):
    case, q = s["case"], s["q"]
    n_q, n_kv, hd, page, window = case["n_q"], case["n_kv"], case["hd"], case["page"], case["window"]
    R, B, M = q.shape[0], s["batch"], s["most"]
    group = n_q // n_kv
    offs, lens = s["offsets"].long(), s["lengths"].long()
    m = offs[1:] - offs[:-1]
    pages = s["table"].long().clamp(min=0)

    def cached(name):  # [B][n_kv][tokens][hd]
        d = s[name + "d"].view(-1, page, n_kv, hd // BLOCK)[pages].flatten(1, 2)
        c = s[name + "c"].view(-1, page, n_kv, hd)[pages].flatten(1, 2)
        return _values(d, c).transpose(1, 2).contiguous()

    r = torch.arange(M, device=q.device)
    idx = (offs[:-1, None] + r).clamp(max=R - 1)  # [B][M]
    x = q.float()[idx].view(B, M, n_kv, group, hd).transpose(1, 2).reshape(B, n_kv, M * group, hd)
    k = cached("k")
    score = torch.matmul(x, k.transpose(2, 3).contiguous()) * s["scale"]
    del k
    p = (lens - m)[:, None] + r  # [B][M]: the rows' positions
    j = torch.arange(score.shape[-1], device=q.device)
    seen = (j <= p[..., None]) & (p[..., None] < lens[:, None, None])
    if window:
        seen &= j > p[..., None] - window
    seen = seen[:, None, :, None, :].expand(B, 1, M, group, -1).reshape(B, 1, M * group, -1)
    score = torch.where(seen, score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    del score
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, cached("v")) / torch.where(total == 0, 1.0, total)
    o = o.view(B, n_kv, M, group, hd).transpose(1, 2).reshape(B, M, n_q, hd)
    row = torch.arange(R, device=q.device)
    b = torch.searchsorted(offs[1:], row, right=True)
    return o[b, row - offs[b]].to(q.dtype)


def _maps(s):
    case = s["case"]
    page, width, R, F = case["page"], case["table"], s["rows"], s["free"].numel()
    n, m = s["lengths"].long(), s["counts"].long()
    fits = (n + m) <= width * page
    m = torch.where(fits, m, 0)
    have = (n + page - 1) // page
    need = (n + m + page - 1) // page - have
    end = torch.cumsum(need, 0)
    go = fits & ((need == 0) | (end <= F))
    first = end - need
    m, need = torch.where(go, m, 0), torch.where(go, need, 0)
    taken = torch.where(go & (need > 0), end, 0).amax().reshape(1)
    offs = torch.cat([m.new_zeros(1), torch.cumsum(m, 0)])
    col = torch.arange(width, device=n.device)
    new = (col >= have[:, None]) & (col < (have + need)[:, None])
    at = (first[:, None] + col - have[:, None]).clamp(0, F - 1)
    table = torch.where(new, s["free"].long()[at], s["old"].long())
    row = torch.arange(max(1, R), device=n.device)
    b = torch.searchsorted(offs[1:], row, right=True)
    live = b < n.numel()
    b = b.clamp(max=n.numel() - 1)
    t = n[b] + row - offs[b]
    pos = torch.where(live, t + s["starts"].long()[b], 0)
    slot = torch.where(live, table[b, (t // page).clamp(0, width - 1)] * page + t % page, -1)
    return {k: v.to(torch.int32) for k, v in dict(table=table, new_lengths=n + m, offsets=offs, positions=pos, slots=slot,
                                                  taken=taken).items()}


def _verify(s):
    """In 64 bits: a drawn number may lie next to the border of a running sum over the vocabulary."""
    x, probs, B, M = s["logits"].double(), s["probs"], s["batch"], s["most"]
    R, V = x.shape
    offs, drafts = s["offsets"].long(), s["drafts"].long()
    row = torch.arange(R, device=x.device)
    b = torch.searchsorted(offs[1:], row, right=True)
    last = offs[b + 1] - 1
    best = x.amax(1, keepdim=True)
    greedy = torch.where(x == best, torch.arange(V, device=x.device), V).amin(1)
    T = s["temperature"].double()
    cold = (T <= 0)[b]
    p = torch.exp((x - best) / torch.where(T <= 0, 1.0, T)[b][:, None])
    p /= p.sum(1, keepdim=True)
    pd = p.gather(1, drafts[:, None])[:, 0]
    qd = probs.gather(1, drafts[:, None])[:, 0].double() if probs is not None else torch.ones_like(pd)
    ok = torch.where(cold, greedy == drafts, s["u_accept"].double() * qd < pd)
    r = torch.arange(M, device=x.device)
    count = offs[1:] - offs[:-1] - 1
    good = ok[(offs[:-1, None] + r).clamp(max=R - 1)] & (r < count[:, None])
    accepted = torch.cumprod(good.long(), 1).sum(1)
    at = offs[:-1] + accepted
    p, whole = p[at], accepted == count
    if probs is not None:
        less = probs[at].double()
    else:
        less = torch.zeros_like(p).scatter_(1, drafts[at][:, None], 1.0)
    rest = torch.where(whole[:, None], p, (p - less).clamp(min=0))
    rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
    run_ = torch.cumsum(rest, 1)
    token = (run_ <= s["u_sample"].double()[:, None] * run_[:, -1:]).sum(1)
    end = torch.where(rest > 0, torch.arange(V, device=x.device), -1).amax(1)
    token = torch.where((T <= 0), greedy[at], torch.minimum(token, end))
    n = accepted[b]
    i = row - offs[b]
    tokens = torch.where(i < n, drafts, torch.where(i == n, token[b], -1))
    return accepted.to(torch.int32), tokens.to(torch.int32)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False  # plain inputs
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"attend": _exact_attend, "append": _exact_append, "maps": _exact_maps, "verify": _exact_verify}[case["kind"]](s)


def _exact_block(x):
    """The values that blocks of float64 rows [..., D] are kept as."""
    w = x.reshape(*x.shape[:-1], -1, 32)
    big, small = w.amax(-1, keepdim=True), w.amin(-1, keepdim=True)
    plus, minus = (w == big).long().argmax(-1, keepdim=True), (w == small).long().argmax(-1, keepdim=True)
    sign_plus = (big > -small) | ((big == -small) & (plus < minus))
    d = torch.where(sign_plus, big, small) / -8
    d = d.clamp(-65504, 65504).half().double()
    steps = torch.where(d == 0, torch.zeros_like(w), torch.round(w / d))
    return (d * steps.clamp(-8, 7)).reshape(x.shape)


def _exact_append(s):
    return _exact_block(s["k"].double()), _exact_block(s["v"].double())


def _exact_attend(s):
    case = s["case"]
    page, window, hd, n_kv = case["page"], case["window"], case["hd"], case["n_kv"]
    offs, lens, table = (s[k].tolist() for k in ("offsets", "lengths", "table"))
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    place = torch.arange(page, device="cuda")
    for b, n in enumerate(lens):
        q = s["q"][offs[b]:offs[b + 1]].double()
        m = q.shape[0]
        if not m or not n:
            continue
        slots = (torch.tensor(table[b][:-(-n // page)], device="cuda")[:, None] * page + place).reshape(-1)[:n]
        k, v = ((s[c + "c"][slots].double() - 8).view(n, n_kv, -1, 32) * s[c + "d"][slots].double()[..., None] for c in "kv")
        k, v = k.reshape(n, n_kv, hd), v.reshape(n, n_kv, hd)
        p = torch.arange(n - m, n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")
        hidden = (j > p) | ((j <= p - window) if window else (j < 0))
        for h in range(n_kv):
            x = q.view(m, n_kv, -1, hd)[:, h]
            w = torch.matmul(x.reshape(-1, hd), k[:, h].t().contiguous()).view(m, -1, n) * s["scale"]
            w = torch.softmax(w.masked_fill(hidden[:, None], -math.inf), -1)
            out.view(-1, n_kv, x.shape[1], hd)[offs[b]:offs[b + 1], h] = torch.matmul(w.reshape(-1, n), v[:, h].contiguous()).view(
                m, -1, hd)
    return out


def _exact_maps(s):
    page, width = s["case"]["page"], s["case"]["table"]
    lens, counts, starts, free, table = (s[k].tolist() for k in ("lengths", "counts", "starts", "free", "old"))
    rows = max(1, s["rows"])
    positions, slots, offs, new, want, taken = [0] * rows, [-1] * rows, [0], [], 0, 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        if n + m > width * page:
            m = 0
        have, end = -(-n // page), -(-(n + m) // page)
        first, want = want, want + end - have
        if end > have and want > len(free):
            m = 0
        elif end > have:
            table[b][have:end] = free[first:want]
            taken = want
        for t in range(n, n + m):
            positions[offs[-1] + t - n] = starts[b] + t
            slots[offs[-1] + t - n] = table[b][t // page] * page + t % page
        offs.append(offs[-1] + m)
        new.append(n + m)
    return {k: torch.tensor(v, dtype=torch.int32) for k, v in dict(table=table, new_lengths=new, offsets=offs, positions=positions,
                                                                   slots=slots, taken=[taken]).items()}


def _exact_verify(s):
    offs, drafts, temps = s["offsets"].tolist(), s["drafts"].tolist(), s["temperature"].tolist()
    ua, us = s["u_accept"].double().tolist(), s["u_sample"].double().tolist()
    accepted, tokens = [], []
    for b, T in enumerate(temps):
        lo, hi = offs[b], offs[b + 1]
        said = []
        for i in range(lo, hi):
            x = s["logits"][i].double()
            p = torch.softmax(x / T, 0) if T > 0 else torch.zeros_like(x)
            if T <= 0:
                p[int((x == x.amax()).nonzero()[0, 0])] = 1.0
            left = p
            if i < hi - 1:
                q = s["probs"][i].double() if s["probs"] is not None else torch.zeros_like(p)
                if s["probs"] is None:
                    q[drafts[i]] = 1.0
                chance = float(p[drafts[i]])
                if (chance == 1.0) if T <= 0 else (ua[i] * float(q[drafts[i]]) < chance):
                    said.append(drafts[i])
                    continue
                left = (p - q).clamp(min=0) if T > 0 else p
                if float(left.sum()) <= 0:
                    left = p
            run_ = torch.cumsum(left, 0)
            at = torch.searchsorted(run_, run_[-1:] * us[b], right=True)
            said.append(min(int(at), int(left.nonzero()[-1, 0])))
            break
        accepted.append(max(0, len(said) - 1))
        tokens += said + [-1] * (hi - lo - len(said))
    return torch.tensor(accepted, dtype=torch.int32), torch.tensor(tokens, dtype=torch.int32)
