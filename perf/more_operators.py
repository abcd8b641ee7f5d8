"""The operators of a serving step over the fp16 page pool, with a caller's arrays on the GPU, as cases that
can be timed and compared: keys rotated to their positions on their way into the pool, attention of one or
several new tokens per sequence over it, and attention over those blocks of a long context that a cheap score
selects for each query.

``own`` false computes them in plain torch operations; ``own`` true calls the framework (``rstr.hip``) on
the same inputs.  Lengths and row counts of a case are the quantiles of its distribution, dealt to the
sequences by the seed, so every seed does the same work.  A block is a page.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a small model's single row, with norms of its heads: the shortest call, where only latency counts
        dict(name="rope_1row_norm", kind="rope", n_q=4, n_kv=1, hd=256, rot=256, dtype="f32", rows=1, page=16, norm=True,
             far=32768, theta=1e6),
        # a decode step of 128 users, rows in fp32 as the step holds them
        dict(name="rope_128", kind="rope", n_q=32, n_kv=8, hd=128, rot=128, dtype="f32", rows=128, page=16, norm=False,
             far=8192, theta=5e5),
        # a layer's rows of a long prompt
        dict(name="rope_prompt", kind="rope", n_q=32, n_kv=8, hd=128, rot=128, dtype="bf16", rows=16411, page=16, norm=False,
             far=131072, theta=5e5),
        # one user who has just begun: the shortest call of attention
        dict(name="attend_1lane_short", kind="attend", n_q=32, n_kv=8, hd=128, dtype="f16", lanes=1, lo=41, hi=41, new_lo=1,
             new_hi=1, window=0, page=16),
        # a full server of an 8B model: one token each for 128 users at ragged lengths
        dict(name="attend_128lane", kind="attend", n_q=32, n_kv=8, hd=128, dtype="f16", lanes=128, lo=128, hi=4608, new_lo=1,
             new_hi=1, window=0, page=16),
        # a few very long contexts, one token each: the work has to be split along them
        dict(name="attend_4lane_long", kind="attend", n_q=32, n_kv=8, hd=128, dtype="bf16", lanes=4, lo=9001, hi=131072,
             new_lo=1, new_hi=1, window=0, page=64),
        # drafted tokens: one to six new rows per sequence, fp32 queries
        dict(name="attend_drafts_f32", kind="attend", n_q=16, n_kv=8, hd=128, dtype="f32", lanes=33, lo=5, hi=8192, new_lo=1,
             new_hi=6, window=0, page=16),
        # a chunk of a long prompt and a whole short one beside it
        dict(name="attend_prompt", kind="attend", n_q=32, n_kv=8, hd=128, dtype="bf16", lanes=2, lo=333, hi=9000, new_lo=333,
             new_hi=1000, window=0, page=16),
        # a user whose context has fewer blocks than the budget: all of them are read
        dict(name="sparse_1lane_short", kind="sparse", n_q=32, n_kv=8, hd=128, dtype="bf16", lanes=1, lo=301, hi=301, new_lo=1,
             new_hi=1, page=16, top=64, first=1, last=2),
        # one very long context, 2048 of its tokens read for the next one
        dict(name="sparse_1lane_long", kind="sparse", n_q=32, n_kv=8, hd=128, dtype="f16", lanes=1, lo=131071, hi=131071,
             new_lo=1, new_hi=1, page=16, top=128, first=1, last=2),
        # a server's step over long contexts
        dict(name="sparse_32lane", kind="sparse", n_q=32, n_kv=8, hd=128, dtype="f16", lanes=32, lo=2048, hi=16384, new_lo=1,
             new_hi=1, page=16, top=64, first=1, last=2),
        # drafted tokens of a few users, each row with blocks of its own, fp32 queries
        dict(name="sparse_drafts_f32", kind="sparse", n_q=16, n_kv=8, hd=128, dtype="f32", lanes=9, lo=700, hi=24000, new_lo=1,
             new_hi=5, page=32, top=40, first=1, last=1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(("rope", "attend", "sparse"), (2, 5, 4))[0]
    n_q, n_kv, hd = rng.choice(((32, 8, 128), (32, 8, 128), (16, 8, 128), (4, 1, 256), (8, 2, 64), (8, 8, 64), (24, 1, 128)))
    dtype, page = rng.choice(("f32", "f16", "bf16")), rng.choice((16, 16, 32, 12, 48, 64))
    if kind == "rope":
        return dict(kind=kind, n_q=n_q, n_kv=n_kv, hd=hd, rot=hd // rng.choice((1, 1, 1, 2)), dtype=dtype, rows=_log_int(rng, 1, 8000),
                    page=page, norm=rng.random() < 0.4, far=_log_int(rng, 100, 1000000), theta=rng.choice((1e4, 5e5, 1e6)))
    if kind == "attend":
        form = rng.choice(("token", "token", "drafts", "prompt"))
        if form == "prompt":
            new = _log_int(rng, 17, 900)
            return dict(kind=kind, n_q=n_q, n_kv=n_kv, hd=hd, dtype=dtype, lanes=rng.choice((1, 1, 2)), lo=new,
                        hi=new + _log_int(rng, 1, 5000), new_lo=rng.randint(1, new), new_hi=new,
                        window=rng.choice((0, 0, 0, 257, 512)), page=page)
        lanes = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, min(131072, 200000 // lanes))
        new = 1 if form == "token" else rng.randint(2, 8)
        return dict(kind=kind, n_q=n_q, n_kv=n_kv, hd=hd, dtype=dtype, lanes=lanes, lo=max(1, hi // rng.choice((1, 7, 40))),
                    hi=hi, new_lo=1, new_hi=min(new, hi), window=rng.choice((0, 0, 0, 100, 512)), page=page)
    lanes = _log_int(rng, 1, 32)
    hi = _log_int(rng, 64, min(131072, 200000 // lanes))
    return dict(kind=kind, n_q=n_q, n_kv=n_kv, hd=hd, dtype=dtype, lanes=lanes, lo=max(8, hi // rng.choice((1, 5, 30))), hi=hi,
                new_lo=1, new_hi=rng.choice((1, 1, 3, 6)), page=page, top=_log_int(rng, 4, 128), first=rng.choice((0, 1, 2)),
                last=rng.choice((1, 1, 2)))


# ---- sizes of a case ------------------------------------------------------------------------------


def _spread(n, lo, hi, log):
    p = [(i + 0.5) / n for i in range(n)]
    if log:
        return [int(min(hi, max(lo, round(math.exp(math.log(lo) + x * (math.log(hi) - math.log(lo))))))) for x in p]
    return [int(min(hi, max(lo, round(lo + x * (hi - lo))))) for x in p]


def _sequences(case):
    """[(length, new rows)] of the sequences, shortest first: every case's work follows from it."""
    n = case["lanes"]
    if n == 2:  # the long one and the short one, as their bounds say
        return [(max(case["lo"], case["new_lo"]), case["new_lo"]), (case["hi"], case["new_hi"])]
    news = _spread(n, case["new_lo"], case["new_hi"], False)
    news = [news[i * 7 % n] if n % 7 else news[i] for i in range(n)]  # not in the lengths' order
    lens = _spread(n, case["lo"], case["hi"], case["hi"] > 10 * case["lo"] and case["hi"] > 10000)
    return [(max(a, m), m) for a, m in zip(lens, news)]


def _dealt(case, seed):
    """(lengths, new rows) by sequence of this seed, as int arrays."""
    pairs = _sequences(case)
    order = np.random.default_rng(seed).permutation(len(pairs))
    a = np.array([pairs[i] for i in order], np.int64).reshape(-1, 2)
    return a[:, 0], a[:, 1]


def work(case):
    kind, n_q, n_kv, hd, size = case["kind"], case["n_q"], case["n_kv"], case["hd"], SIZES[case["dtype"]]
    if kind == "rope":
        return {"bytes": case["rows"] * hd * (2 * n_q * size + 2 * n_kv * (size + 2)), "flops": 3 * case["rows"] * (n_q + n_kv) * hd}
    page, seen, pairs, rows, blocks, scored, touched = case["page"], 0, 0, 0, 0, 0, 0
    for length, m in _sequences(case):
        rows += m
        if kind == "attend":
            w = case["window"]
            seen += min(length, w + m - 1) if w else length
            pairs += sum(min(p + 1, w) if w else p + 1 for p in range(length - m, length))
        else:
            have = -(-length // page)
            seen += min(case["top"] * page, length)  # of one row: a sequence's rows may share their blocks
            pairs += m * min(case["top"] * page, length)
            blocks += have
            scored += m * have
            touched += have - (length - m) // page
    bytes_, flops = seen * n_kv * hd * 4 + 2 * rows * n_q * hd * size, 4 * n_q * hd * pairs
    if kind == "sparse":
        bytes_ += blocks * n_kv * hd * 4 + touched * n_kv * hd * (2 * page + 4) + 4 * rows * n_kv * case["top"]
        flops += 4 * n_q * hd * scored
    return {"bytes": bytes_, "flops": flops}


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


class _Handles(list):
    """The handles that a serving program keeps, in the order of opening; closed once neither a state nor what a pass returned
    (the pool's own pages, the bounds) needs them."""

    def __del__(self):
        while self:
            self.pop().close()


class _Lent:
    """Memory of a handle as a tensor takes it, which keeps the handles open."""

    def __init__(self, view, handles):
        self.__cuda_array_interface__, self._handles = view.__cuda_array_interface__, handles


def _lent(s, view):
    return torch.as_tensor(_Lent(view, s["handles"]), device="cuda")


def _opened(s, name, handle):
    s["handles"].append(handle)
    s[name] = handle


def _open_pool(s, case, pages):
    """The pool of one layer of a model with these heads."""
    hip = _hip()
    s["handles"] = _Handles()
    cfg = dict(n_layers=1, d_model=256, d_ff=256, n_q=case["n_kv"], n_kv=case["n_kv"], head_dim=case["hd"], vocab=256, weight_bits=4,
               gain_offset=0, qk_norm=0, sandwich=0, ffn_geglu=0, rope_dual=0, global_pattern=0, sliding_window=0,
               embed_scale_sqrt_d=0, eps=1e-6, attn_scale=case["hd"] ** -0.5, rope_global=1e4, rope_local=1e4)
    if case["n_kv"] * case["hd"] % 128:
        cfg["n_q"] *= 2
    _opened(s, "model", hip.Model(_open_session(), cfg, seed=1))
    _opened(s, "pool", hip.Pool(s["model"], case["page"], pages))


def _paged(need, pages, rng):
    """A page table of a shuffled pool: [sequences][width], -1 behind a sequence's pages."""
    perm = rng.permutation(pages)
    table = np.full((len(need), max(1, int(max(need)))), -1, np.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table


def prepare(case, seed):
    g = torch.Generator("cuda")
    g.manual_seed(int(seed))
    rng = np.random.default_rng([int(seed), 11])
    return (_prepare_rope if case["kind"] == "rope" else _prepare_attend)(case, int(seed), g, rng)


def _prepare_rope(case, seed, g, rng):
    rows, page, n_q, n_kv, hd, dt = (case[k] for k in ("rows", "page", "n_q", "n_kv", "hd", "dtype"))
    dt = DTYPES[dt]
    pages = -(-rows // page) + 5
    if rows <= 256:  # a step's rows go anywhere, a prompt's fill one page after the other
        slots, positions = rng.permutation(pages * page)[:rows], rng.integers(0, case["far"], rows)
    else:
        slots = (rng.permutation(pages)[:, None] * page + np.arange(page)).reshape(-1)[3:3 + rows]
        positions = max(0, case["far"] - rows) + np.arange(rows)
    qkv = torch.randn(rows, n_q + 2 * n_kv, hd, generator=g, device="cuda")
    qkv[:, :, hd // 2:: 17] *= 4.0  # a few channels of larger values, as queries and keys have them
    qkv = qkv.to(dt)  # as a projection of all heads leaves them
    rot = case["rot"]
    s = dict(case=case, q=qkv[:, :n_q], k=qkv[:, n_q:n_q + n_kv], v=qkv[:, n_q + n_kv:], slots=_dev(slots), positions=_dev(positions),
              frequencies=_dev(case["theta"] ** (-np.arange(0, rot, 2) / rot), torch.float64), q_gain=None, k_gain=None, eps=1e-6,
              q_out=torch.empty(rows, n_q, hd, dtype=dt, device="cuda"))
    if case["norm"]:
        s["q_gain"], s["k_gain"] = (1.0 + 0.2 * torch.randn(hd, generator=g, device="cuda") for _ in "qk")
    if own:
        _open_pool(s, case, pages)
        s["pages"] = [_lent(s, s["pool"].pages_device(slab, 0)) for slab in (0, 1)]
    else:
        s["pages"] = [torch.zeros(pages, page, n_kv, hd, dtype=torch.float16, device="cuda") for _ in "kv"]
    return s


def _prepare_attend(case, seed, g, rng):
    lens, news = _dealt(case, seed)
    page, n_q, n_kv, hd = case["page"], case["n_q"], case["n_kv"], case["hd"]
    need = -(-lens // page)
    pages = int(need.sum()) + 3
    table = _paged(need, pages, rng)
    offs = np.concatenate([[0], np.cumsum(news)])
    rows, total, batch = int(offs[-1]), int(lens.sum()), len(lens)
    pos = np.concatenate([np.arange(a) for a in lens])
    seq = np.repeat(np.arange(batch), lens)
    slots = _dev(table[seq, pos // page] * page + pos % page)
    # what a stretch of the text is about shows in its keys, and a query asks for one of these subjects
    about = torch.randn(16, n_kv, hd, generator=g, device="cuda")
    k = torch.randn(total, n_kv, hd, generator=g, device="cuda") * 0.8
    k += about[_dev(rng.integers(0, 16, total // 53 + 1)[np.arange(total) // 53], torch.int64)]
    v = torch.randn(total, n_kv, hd, generator=g, device="cuda") * 0.7
    q = torch.randn(rows, n_q, hd, generator=g, device="cuda") * 0.7
    q += 0.6 * about[_dev(rng.integers(0, 16, rows), torch.int64)].repeat_interleave(n_q // n_kv, 1)
    s = dict(case=case, lengths=_dev(lens), offsets=_dev(offs), table=_dev(table), most=int(news.max()), scale=hd ** -0.5,
              batch=batch, q=q.to(DTYPES[case["dtype"]]))
    s["out"] = torch.empty_like(s["q"])
    k, v = k.half(), v.half()
    if case["kind"] == "sparse":
        s["blocks"] = torch.empty(rows, n_kv, case["top"], dtype=torch.int32, device="cuda")
    if own:
        hip = _hip()
        _open_pool(s, case, pages)
        s["pool"].rope_append(0, k, v, slots)  # the keys as they are
        _opened(s, "plan", hip.PagedAttention(s["pool"], n_q, batch, rows))
        if case["kind"] == "sparse":
            _opened(s, "bounds", hip.BlockBounds(s["pool"]))
            _opened(s, "select", hip.BlockSelect(s["bounds"], n_q, batch, rows, table.shape[1]))
            s["bounds"].update(0, _dev(np.concatenate([[0], np.cumsum(lens)])), s["table"], s["lengths"], total)
            s["limits"] = _lent(s, s["bounds"].device(0))
    else:
        s["pages"] = [torch.zeros(pages * page, n_kv, hd, dtype=torch.float16, device="cuda") for _ in "kv"]
        for to, x in zip(s["pages"], (k, v)):
            to[slots.long()] = x
        if case["kind"] == "sparse":
            s["limits"] = torch.zeros(pages, n_kv, 2, hd, dtype=torch.float16, device="cuda")
            _bounds(s, _dev(seq, torch.int64), _dev(pos, torch.int64))
    return s


# ---- one pass ----------------------------------------------------------------------------------------


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"rope": _own_rope, "attend": _own_attend, "sparse": _own_sparse}[kind](s)
    return {"rope": _rope, "attend": _attend, "sparse": _sparse}[kind](s)


def _own_rope(s):
    s["pool"].rope_append(0, s["k"], s["v"], s["slots"], s["positions"], s["frequencies"], q=s["q"], q_out=s["q_out"],
                          q_gain=s["q_gain"], k_gain=s["k_gain"], eps=s["eps"])
    return s["q_out"], *s["pages"]


def _own_attend(s):
    s["plan"].run(0, s["q"], s["offsets"], s["table"], s["lengths"], s["out"], max_rows=s["most"], window=s["case"]["window"],
                  scale=s["scale"])
    return s["out"]


def _own_sparse(s):
    case = s["case"]
    s["bounds"].update(0, s["offsets"], s["table"], s["lengths"], s["q"].shape[0])
    s["select"].run(0, s["q"], s["offsets"], s["table"], s["lengths"], s["blocks"], first=case["first"], last=case["last"])
    s["plan"].run(0, s["q"], s["offsets"], s["table"], s["lengths"], s["out"], max_rows=s["most"], scale=s["scale"], blocks=s["blocks"])
    return s["out"], s["blocks"], s["limits"]


# ---- the plain forms -----------------------------------------------------------------------------------


def _rope(s):
    rot = s["case"]["rot"]
    angle = s["positions"].double()[:, None] * s["frequencies"]  # 64 bits: far positions turn many times
    c, d = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turned(x, gain):
        x = x.float()
        if gain is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * gain
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * c - b * d, b * c + a * d, x[..., rot:]], -1)

    at = s["slots"].long()
    for to, x in zip(s["pages"], (turned(s["k"], s["k_gain"]), s["v"])):
        to.flatten(0, 1)[at] = x.half()
    s["q_out"].copy_(turned(s["q"], s["q_gain"]))
    return s["q_out"], *s["pages"]


def _rows_of(s):
    """Of every row: its sequence, its place among the sequence's rows, its position."""
    offs, lens = s["offsets"].long(), s["lengths"].long()
    row = torch.arange(s["q"].shape[0], device=offs.device)
    b = torch.searchsorted(offs[1:], row, right=True)
    i = row - offs[b]
    return b, i, lens[b] - (offs[b + 1] - offs[b]) + i


def _attend(s):
    case, q = s["case"], s["q"]
    n_q, n_kv, hd, page, window = case["n_q"], case["n_kv"], case["hd"], case["page"], case["window"]
    R, B, M = q.shape[0], s["batch"], s["most"]
    group = n_q // n_kv
    offs, lens = s["offsets"].long(), s["lengths"].long()
    m = offs[1:] - offs[:-1]
    pages = s["table"].long().clamp(min=0)

    def cached(x):  # [B][n_kv][tokens][hd]
        return x.view(-1, page, n_kv, hd)[pages].flatten(1, 2).transpose(1, 2).float().contiguous()

    r = torch.arange(M, device=q.device)
    idx = (offs[:-1, None] + r).clamp(max=R - 1)  # [B][M]
    x = q.float()[idx].view(B, M, n_kv, group, hd).transpose(1, 2).reshape(B, n_kv, M * group, hd)
    k = cached(s["pages"][0])
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
    o = torch.matmul(e, cached(s["pages"][1])) / torch.where(total == 0, 1.0, total)
    o = o.view(B, n_kv, M, group, hd).transpose(1, 2).reshape(B, M, n_q, hd)
    b, i, _ = _rows_of(s)
    return o[b, i].to(q.dtype)


def _bounds(s, seq, pos):
    """The least and the greatest element of every channel of the keys in the blocks of these tokens."""
    page, n_kv, hd = (s["case"][k] for k in ("page", "n_kv", "hd"))
    block = pos // page
    at = torch.unique(seq * (1 << 32) + block)
    seq, block = at >> 32, at & 0xFFFFFFFF
    ids = s["table"].long()[seq, block]
    k = s["pages"][0].view(-1, page, n_kv, hd)[ids].float()
    held = (block[:, None] * page + torch.arange(page, device=k.device) < s["lengths"].long()[seq][:, None])[..., None, None]
    s["limits"][ids, :, 0] = torch.where(held, k, math.inf).amin(1).half()
    s["limits"][ids, :, 1] = torch.where(held, k, -math.inf).amax(1).half()


def _select(s):
    """In 64 bits: two blocks may lie next to each other at the end of a list."""
    case, R = s["case"], s["q"].shape[0]
    n_q, n_kv, hd, page, top = (case[k] for k in ("n_q", "n_kv", "hd", "page", "top"))
    b, i, p = _rows_of(s)
    B, M, group = s["batch"], s["most"], n_q // n_kv
    lim = s["limits"][s["table"].long().clamp(min=0)].double()  # [B][W][n_kv][2][hd]
    W = lim.shape[1]
    lim = lim.permute(0, 2, 3, 4, 1).reshape(B, n_kv, 2 * hd, W).contiguous()
    x = torch.zeros(B, M, n_q, hd, dtype=torch.float64, device=lim.device)
    x[b, i] = s["q"].double()
    x = x.view(B, M, n_kv, group, hd).transpose(1, 2).reshape(B, n_kv, M * group, hd)
    x = torch.cat([x.clamp(max=0), x.clamp(min=0)], -1)  # the largest of q lo and q hi: lo for negative q, hi for positive
    score = torch.matmul(x, lim).view(B, n_kv, M, group, W).amax(3)[b, :, i]  # [R][n_kv][W]
    j, cur = torch.arange(W, device=lim.device), (p // page)[:, None]
    score = torch.where(((j < case["first"]) | (j > cur - case["last"]))[:, None], math.inf, score)
    score = torch.where((j > cur)[:, None], -math.inf, score)
    got = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :top]
    got = torch.where(got > cur[..., None], W, got).sort(-1).values
    got = torch.where(got == W, -1, got)
    return torch.cat([got, got.new_full((R, n_kv, max(0, top - W)), -1)], -1).to(torch.int32)


def _sparse(s):
    case, q = s["case"], s["q"]
    n_q, n_kv, hd, page = case["n_q"], case["n_kv"], case["hd"], case["page"]
    R, group = q.shape[0], n_q // n_kv
    b, _, p = _rows_of(s)
    _bounds(s, b, p)
    blocks = _select(s)
    j = blocks.long()
    ids = s["table"].long()[b[:, None, None], j.clamp(min=0)]
    place = torch.arange(page, device=q.device)
    seen = ((j[..., None] * page + place <= p[:, None, None, None]) & (j[..., None] >= 0)).flatten(2)  # [R][n_kv][tokens]
    head = torch.arange(n_kv, device=q.device)[:, None]

    def listed_(x):  # [R][n_kv][tokens][hd]
        return x.view(-1, page, n_kv, hd)[ids, :, head].flatten(2, 3).float()

    score = torch.matmul(q.float().view(R, n_kv, group, hd), listed_(s["pages"][0]).transpose(2, 3).contiguous()) * s["scale"]
    score = torch.where(seen[:, :, None], score, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul(e, listed_(s["pages"][1])) / e.sum(-1, keepdim=True)
    return o.view(R, n_q, hd).to(q.dtype), blocks, s["limits"]


# ---- the definitions in 64 bits ----------------------------------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False  # plain inputs
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"rope": _exact_rope, "attend": _exact_attend, "sparse": _exact_sparse}[case["kind"]](s)


def _exact_rope(s):
    half = s["case"]["rot"] // 2
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double().outer(s["frequencies"]))

    def put(x, gain):
        x = x.double()
        if gain is not None:
            x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + s["eps"]).sqrt() * gain.double()
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn.unsqueeze(1)
        x = x.clone()
        x[..., :half], x[..., half:2 * half] = z.real, z.imag
        return x

    out = [put(s["q"], s["q_gain"])]
    for x in (put(s["k"], s["k_gain"]), s["v"].double()):
        pages = torch.zeros(s["pages"][0].shape, dtype=torch.float64, device="cuda")
        pages.view(-1, *x.shape[1:])[s["slots"].long()] = x
        out.append(pages)
    return tuple(out)


def _cached(s, b, tokens):
    """Keys and values of one sequence's tokens, in 64 bits."""
    page = s["case"]["page"]
    at = s["table"][b].long()[tokens // page] * page + tokens % page
    return s["pages"][0][at].double(), s["pages"][1][at].double()


def _softmax(q, k, v, scale, hidden):
    w = torch.matmul(q, k.t().contiguous()) * scale
    return torch.matmul(torch.softmax(w.masked_fill(hidden, -math.inf), -1), v.contiguous())


def _exact_attend(s):
    case, out = s["case"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    window, n_kv, hd = case["window"], case["n_kv"], case["hd"]
    group = case["n_q"] // n_kv
    offs, lens = s["offsets"].tolist(), s["lengths"].tolist()
    for b, n in enumerate(lens):
        r0, r1 = offs[b], offs[b + 1]
        j = torch.arange(n, device="cuda")
        k, v = _cached(s, b, j)
        p = torch.arange(n - (r1 - r0), n, device="cuda").repeat_interleave(group)[:, None]
        hidden = (j > p) | ((j <= p - window) if window else (j < 0))
        for h in range(n_kv):
            q = s["q"][r0:r1, h * group:(h + 1) * group].double().reshape(-1, hd)
            out[r0:r1, h * group:(h + 1) * group] = _softmax(q, k[:, h], v[:, h], s["scale"], hidden).view(-1, group, hd)
    return out


def _exact_sparse(s):
    case, out = s["case"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    n_kv, hd, page, top = case["n_kv"], case["hd"], case["page"], case["top"]
    group = case["n_q"] // n_kv
    offs, lens, table = s["offsets"].tolist(), s["lengths"].tolist(), s["table"].long()
    blocks = np.full((out.shape[0], n_kv, top), -1, np.int64)
    limits = torch.zeros(s["limits"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        tokens = torch.arange(n, device="cuda")
        k, v = _cached(s, b, tokens)
        have = -(-n // page)
        whole = torch.cat([k, k[-1:].expand(have * page - n, -1, -1)]).view(have, page, n_kv, hd)  # the last key again: no new bound
        lo, hi = whole.amin(1), whole.amax(1)
        limits[table[b, :have], :, 0], limits[table[b, :have], :, 1] = lo, hi
        for r in range(offs[b], offs[b + 1]):
            p = n - (offs[b + 1] - r)
            cur = p // page
            for h in range(n_kv):
                q = s["q"][r, h * group:(h + 1) * group].double()
                score = torch.stack([torch.maximum(x * lo[:cur + 1, h], x * hi[:cur + 1, h]).sum(1) for x in q]).amax(0).tolist()
                kept = [j for j in range(cur + 1) if j < case["first"] or j > cur - case["last"]]
                rest = sorted((j for j in range(cur + 1) if case["first"] <= j <= cur - case["last"]), key=lambda j: (-score[j], j))
                got = sorted((kept + rest)[:top])
                blocks[r, h, :len(got)] = got
                t = (torch.tensor(got, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)
                t = t[t <= p]
                out[r, h * group:(h + 1) * group] = _softmax(q, k[t, h], v[t, h], s["scale"], torch.zeros(1, t.numel(), dtype=torch.bool, device="cuda"))
    return out, torch.from_numpy(blocks.astype(np.int32)), limits
