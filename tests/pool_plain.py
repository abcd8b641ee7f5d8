"""Plain float64 forms of the operators over the fp16 page pool (rotated append, attention over all or listed
blocks, bounds and selection of blocks), for the tests of the HIP operators (and their own tests)."""
from __future__ import annotations

import numpy as np


def as_f64(x):
    """A torch tensor's or array's values in float64."""
    return np.asarray(x.detach().cpu().double() if hasattr(x, "detach") else x, np.float64)


def rotated(x, positions, freqs, gain=None, eps=0.0, offset=0.0):
    """Rows x [R][H][D] normalised and turned; and per element the sum of the magnitudes that it is made of."""
    x = np.asarray(x, np.float64)
    if gain is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (offset + np.asarray(gain, np.float64))
    y, mag = x.copy(), np.abs(x)
    if freqs is not None:
        half = len(freqs)
        ang = np.asarray(positions, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
        c, s, a, b = np.cos(ang), np.sin(ang), x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = a * c - b * s, b * c + a * s
        mag[..., :half], mag[..., half:2 * half] = abs(a * c) + abs(b * s), abs(b * c) + abs(a * s)
    return y, mag


def cells(table, lengths, offsets, page, pages, rows):
    """Per row of a call: (sequence, position), or None where it belongs to none (all None where offsets decrease)."""
    out = [None] * rows
    if any(a > b for a, b in zip(offsets, offsets[1:])):
        return out
    for b, n in enumerate(lengths):
        r0, r1 = max(offsets[b], 0), min(offsets[b + 1], rows)
        for r in range(r0, r1):
            out[r] = (b, max(n, 0) - (r1 - r))
    return out


def attention(q, k_pages, v_pages, table, lengths, offsets, window=0, scale=1.0, blocks=None):
    """q [R][n_q][D] over pages [P][page][n_kv][D].  Returns (out, sum of w|v|, largest scale |q|.|k|, tokens seen),
    each broadcast over the head's dims; rows of no sequence are None in `out`'s mask."""
    R, n_q, D = q.shape
    P, page, n_kv, _ = k_pages.shape
    width = len(table[0])
    out, mag, size, seen = (np.zeros((R, n_q, D)) for _ in range(4))
    mine = np.zeros(R, bool)
    for r, cell in enumerate(cells(table, lengths, offsets, page, P, R)):
        if cell is None:
            continue
        mine[r] = True
        b, p = cell
        for h in range(n_kv):
            if blocks is None:
                j = np.arange(max(0, p + 1))
            else:
                lst = [int(x) for x in blocks[r][h][:min(width, p // page + 1) if p >= 0 else 0] if 0 <= x < width]
                j = (np.array(lst, np.int64)[:, None] * page + np.arange(page)).reshape(-1)
                j = j[j <= p]
            j = j[j < width * page]
            if window:
                j = j[j > p - window]
            ids = np.array([table[b][t // page] for t in j], np.int64)
            ok = (ids >= 0) & (ids < P)
            j, ids = j[ok], ids[ok]
            if j.size == 0:
                continue
            kk, vv = k_pages[ids, j % page, h], v_pages[ids, j % page, h]
            for g in range(n_q // n_kv):
                i = h * (n_q // n_kv) + g
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk @ q[r, i] * scale
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[r, i], mag[r, i] = w @ vv, w @ np.abs(vv)
                    size[r, i], seen[r, i] = np.max(np.abs(kk) @ np.abs(q[r, i])) * abs(scale), j.size
    return out, mag, size, seen, mine


def bounds(k_pages, table, lengths, offsets, rows, limits):
    """`limits` [P][n_kv][2][D] with the bounds of the blocks of the call's rows."""
    P, page, n_kv, D = k_pages.shape
    limits = np.array(limits, np.float64)
    for cell in cells(table, lengths, offsets, page, P, rows):
        if cell is None or cell[1] < 0 or cell[1] // page >= len(table[0]):
            continue
        b, p = cell
        blk = p // page
        at = table[b][blk]
        if 0 <= at < P:
            k = k_pages[at, :min(page, lengths[b] - blk * page)]
            limits[at, :, 0], limits[at, :, 1] = k.min(0), k.max(0)
    return limits


def select(q, limits, table, lengths, offsets, page, top, first, last, untouched=-7):
    """The lists [R][n_kv][top] by the definition, in float64."""
    R, n_q, D = q.shape
    P, n_kv = limits.shape[:2]
    width = len(table[0])
    out = np.full((R, n_kv, top), untouched, np.int64)
    for r, cell in enumerate(cells(table, lengths, offsets, page, P, R)):
        if cell is None:
            continue
        b, p = cell
        for h in range(n_kv):
            if p < 0:
                out[r, h] = -1
                continue
            cur = min(p // page, width - 1)
            got = list(range(cur + 1))
            if cur + 1 > top:
                score = []
                for j in range(first, cur + 1 - last):
                    at = table[b][j]
                    if not 0 <= at < P:
                        score.append(-np.inf)
                        continue
                    lo, hi = limits[at, h]
                    with np.errstate(invalid="ignore"):
                        s = [np.maximum(x * lo, x * hi).sum() for x in q[r, h * (n_q // n_kv):(h + 1) * (n_q // n_kv)]]
                    score.append(np.inf if np.isnan(s).any() else max(s))
                best = sorted(range(len(score)), key=lambda i: (-score[i], i))[:top - first - last]
                got = sorted(list(range(first)) + [first + i for i in best] + list(range(cur + 1 - last, cur + 1)))
            out[r, h] = got + [-1] * (top - len(got))
    return out
