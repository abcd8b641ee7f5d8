"""Plain float64 forms of the 4-bit cache, its attention, step maps and draft
verification, for the tests of the HIP operators (and their own tests)."""
from __future__ import annotations

import numpy as np


def as_f64(x):
    """A torch tensor's or array's values in float64."""
    return np.asarray(x.detach().cpu().double() if hasattr(x, "detach") else x, np.float64)


def block_scale(w):
    """fp16 scale of one block of 32 float64 values, as float64."""
    if not np.all(np.isfinite(w)):
        return np.nan
    i = int(np.argmax(np.abs(w)))  # the first of equals
    d = float(np.float16(np.clip(w[i] / -8.0, -65504.0, 65504.0)))
    return d if d != 0 else 0.0


def quantised(x):
    """The values that rows [..., D] are kept as, in float64 (blocks of 32 along D)."""
    x = np.asarray(x, np.float64)
    out = np.empty_like(x)
    flat, put = x.reshape(-1, 32), out.reshape(-1, 32)
    for w, o in zip(flat, put):
        d = block_scale(w)
        if np.isnan(d):
            o[:] = np.nan
        elif d == 0.0:
            o[:] = 0.0
        else:
            o[:] = d * np.clip(np.rint(w / d), -8, 7)  # halves to even; w / d is exact enough in 64 bits
    return out


def attention(q, k, v, lengths, offsets, window=0, scale=1.0):
    """q [R][n_q][D]; k, v: per sequence [tokens][n_kv][D] (None: a token that is not there, as NaN rows
    listed in `gone`).  Returns (out [R][n_q][D], sum of w|v|, largest |scale q k|-weight of a row's keys) in float64."""
    R, n_q, D = q.shape
    out, mag, size = np.zeros((R, n_q, D)), np.zeros((R, n_q, D)), np.zeros((R, n_q, 1))
    for b, n in enumerate(lengths):
        r0, r1 = offsets[b], offsets[b + 1]
        kb, vb, there = k[b], v[b], np.asarray([x is not None for x in k[b]]) if isinstance(k[b], list) else np.ones(len(k[b]), bool)
        n_kv = kb.shape[1]
        for r in range(r0, r1):
            p = n - (r1 - r)
            j = np.arange(max(0, p - window + 1) if window else 0, p + 1)
            j = j[there[j]] if p >= 0 else j[:0]
            if j.size == 0:
                continue
            for h in range(n_q):
                kk, vv = kb[j, h // (n_q // n_kv)], vb[j, h // (n_q // n_kv)]
                s = kk @ q[r, h] * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r, h], mag[r, h] = w @ vv, w @ np.abs(vv)
                size[r, h] = np.max(np.abs(kk) @ np.abs(q[r, h])) * abs(scale)
    return out, mag, size


def step_maps(page, lengths, counts, starts, free, table, rows):
    """The tables of a step, one sequence after the other."""
    table = np.array(table, np.int64)
    width = table.shape[1]
    positions, slots, offs, new, want, taken, asked = [0] * rows, [-1] * rows, [0], [], 0, 0, 0
    for b, (n, m) in enumerate(zip(lengths, counts)):
        n, m = int(n), int(m)
        if n < 0 or m < 0 or n + m > width * page:
            m = 0
        have, end = (-(-n // page), -(-(n + m) // page)) if m else (0, 0)
        first, want = want, want + end - have
        if end > have and want > len(free):
            m = 0
        asked += m
        if m and asked > rows:
            m = 0
        if m and end > have:
            table[b, have:end] = free[first:want]
            taken = want
        for t in range(n, n + m):
            i = offs[-1] + t - n
            positions[i] = (starts[b] if starts is not None else 0) + t
            slots[i] = table[b, t // page] * page + t % page if table[b, t // page] >= 0 else -1
            slots[i] = slots[i] if slots[i] < 2 ** 31 else -1
        offs.append(offs[-1] + m)
        new.append(n + m)
    return dict(table=table, new_lengths=new, offsets=offs, positions=positions, slots=slots, taken=[taken])


def _greedy(x):
    nan = np.flatnonzero(np.isnan(x))
    return int(nan[0]) if nan.size else int(np.argmax(x))


def verify(logits, offsets, drafts, probs, temperature, u_accept, u_sample, untouched=-7):
    """(accepted, tokens) by the definition, in float64; rows of no sequence keep `untouched`."""
    V = logits.shape[1]
    tokens = np.full(len(drafts), untouched, np.int64)
    accepted = []
    for b in range(len(offsets) - 1):
        r0, r1 = offsets[b], offsets[b + 1]
        T, said = float(temperature[b]), []
        for r in range(r0, r1):
            x, d = logits[r].astype(np.float64), int(drafts[r])
            top = x[_greedy(x)]
            cold = not (T > 0 and np.isfinite(T)) or not np.isfinite(top)
            g = _greedy(x)
            if not cold:
                with np.errstate(under="ignore"):
                    p = np.exp((x - top) / T)
                p /= p.sum()
            if r < r1 - 1:
                if cold:
                    ok = d == g
                else:
                    q = probs[r].astype(np.float64) if probs is not None else np.zeros(V)
                    if probs is None and 0 <= d < V:
                        q[d] = 1.0
                    ok = 0 <= d < V and float(u_accept[r]) * q[d] < p[d]
                if ok:
                    said.append(d)
                    continue
            if cold:
                said.append(g)
                break
            left = p
            if r < r1 - 1:
                left = np.maximum(p - q, 0.0)
                if probs is None and 0 <= d < V:
                    left[d] = 0.0
                if not left.sum() > 0:
                    left = p
            run = np.cumsum(left)
            at = int(np.searchsorted(run, float(u_sample[b]) * run[-1], side="right"))
            said.append(min(at, int(np.flatnonzero(left)[-1])))
            break
        accepted.append(max(0, len(said) - 1))
        tokens[r0:r1] = said + [-1] * (r1 - r0 - len(said))
    return np.array(accepted), tokens
