"""The paged 8-bit cache, attention over it and token log probabilities, from their definitions in 64 bits (numpy)."""

from __future__ import annotations

import math

import numpy as np

HD = 128


def e4m3_values():
    """The value of each of the 256 e4m3 bytes (1 sign, 4 exponent bits of bias 7, 3 bits; 0x7f and 0xff are NaN)."""
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7.0), m / 8.0 * 2.0 ** -6)
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b & 128, -v, v)


E4M3 = e4m3_values()


def step(x):
    """The distance of neighbouring e4m3 values at x."""
    e = np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -6)))
    return 2.0 ** (e - 3)


def encode(x):
    """The bytes of the e4m3 values nearest to x (ties to even, |x| <= 448; not finite: NaN)."""
    x = np.asarray(x, np.float64)
    ok = np.isfinite(x)
    v = np.where(ok, x, 0.0)
    s = step(v)
    a = np.abs(np.round(v / s) * s)
    mags = E4M3[:127]
    code = np.searchsorted(mags, a)
    assert np.array_equal(mags[code], a), "not an e4m3 value"
    return np.where(ok, code | np.where(np.signbit(v), 128, 0), 127).astype(np.uint8)


def scale_of(amax):
    e = -100
    while amax > 448 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rotate(x, pos, theta):
    """x [..., 128] at the one position pos."""
    a = pos * theta ** (-np.arange(64) / 64.0)
    c, s = np.cos(a), np.sin(a)
    lo, hi = x[..., :64], x[..., 64:]
    return np.concatenate([lo * c - hi * s, hi * c + lo * s], axis=-1)


def append(pages, scale, table, page, start, live, new):
    """One tensor's rows new[b] [n, heads, 128] into pages [pages, heads, page, 128] (bytes) and scale, in place."""
    for b, rows in enumerate(new):
        n = len(rows)
        if n == 0 or start[b] < 0:
            continue
        for j in range(start[b] // page, (start[b] + n - 1) // page + 1):
            if j >= table.shape[1] or not 0 <= table[b, j] < len(pages):
                continue
            pg = table[b, j]
            w = np.arange(max(start[b], j * page), min(start[b] + n, (j + 1) * page))
            old = np.setdiff1d(np.arange(j * page, min(live[b], (j + 1) * page)), w) - j * page
            for h in range(pages.shape[1]):
                x = rows[w - start[b], h]
                fin = np.abs(x[np.isfinite(x)])
                s = scale_of(fin.max() if fin.size else 0.0)
                if old.size:
                    was = float(scale[pg, h])
                    if s > was:
                        pages[pg, h, old] = encode(E4M3[pages[pg, h, old]] * (was / s))
                    s = max(s, was)
                scale[pg, h] = s
                pages[pg, h, w - j * page] = encode(x / s)


def attend(q, kpages, kscale, vpages, vscale, table, page, kv_len, rows, mask_block):
    """q [total, nq, 128]; pages bytes [pages, heads, page, 128] for both; rows[b] = indices of b's rows.  Returns out (0
    for rows of no sequence), and for tolerances sum p |v| and the largest sum |q| |k| / sqrt(128) of each (row, head)."""
    nq, nkv = q.shape[1], kpages.shape[1]
    G = nq // nkv
    out, mass, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for b, idx in enumerate(rows):
        total = max(0, min(kv_len[b], table.shape[1] * page))
        keys = np.array([p for p in range(total) if 0 <= table[b, p // page] < len(kpages)], dtype=np.int64)
        pg, sl = (table[b, keys // page], keys % page) if keys.size else (keys, keys)
        for h in range(nkv):
            k = E4M3[kpages[pg, h, sl]] * kscale[pg, h][:, None]
            v = E4M3[vpages[pg, h, sl]] * vscale[pg, h][:, None]
            for i, r in enumerate(idx):
                pos = kv_len[b] - len(idx) + i
                see = keys >= 0 if mask_block == 0 else keys < (pos // mask_block + 1) * mask_block if pos >= 0 else keys < 0
                if not see.any():
                    continue
                for hq in range(h * G, (h + 1) * G):
                    s = k[see] @ q[r, hq] / math.sqrt(HD)
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[r, hq] = p @ v[see]
                    mass[r, hq] = p @ np.abs(v[see])
                    reach[r, hq] = (np.abs(k[see]) @ np.abs(q[r, hq])).max() / math.sqrt(HD)
    return out, mass, reach


def logprobs(x, ids, top):
    """x [rows, vocab] float64: (logprob, entropy, top ids, top log probabilities)."""
    rows, vocab = x.shape
    lp_ids, ent = np.zeros(rows), np.zeros(rows)
    order, best = np.zeros((rows, top), np.int64), np.zeros((rows, top))
    for r in range(rows):
        row = x[r]
        m = row.max() if not np.isnan(row).any() else np.nan
        with np.errstate(all="ignore"):
            # (the difference first: m + log loses the log where m is the type's lowest value)
            lp = (row - m) - np.log(np.exp(row - m).sum())
            p = np.exp(lp)
            ent[r] = -np.where(p > 0, p * lp, p).sum()  # (p NaN stays NaN)
        if ids is not None:
            lp_ids[r] = np.nan if ids[r] >= vocab else 0.0 if ids[r] < 0 else lp[ids[r]]
        seen = np.where(np.isnan(row), -np.inf, row)
        order[r] = np.argsort(-seen, kind="stable")[:top]
        best[r] = lp[order[r]]
    return lp_ids, ent, order, best


def rotation_bounds(x, pos, theta):
    """Rotated keys from below and above, x [n, heads, 128] at positions pos [n] of at most 2^17: a rotation in 64 bits whose
    frequencies carry a dozen roundings (an angle off by 2^17 x 2^-49) and whose sines and cosines are within 2^-33, rounded
    once to fp32 (2^-24 of its size); so is one in numpy, whose angles are off by less.  Rounding to e4m3 and scaling by a power
    of two are monotone: the bytes lie between those of the bounds."""
    pos = np.asarray(pos, np.float64)[:, None, None]
    exact = rotate(x, pos, theta)
    size = np.tile(np.abs(x[..., :64]) + np.abs(x[..., 64:]), 2)
    err = np.where(pos == 0, 0.0, 2.0 ** -24 * np.abs(exact) + 2.0 ** -30 * size)  # (position 0 turns nothing)
    return exact - err, exact + err


def outside(got, lo, hi):
    """Where bytes are not between those of two bounds (equal bounds: not that byte)."""
    return np.where(lo == hi, got != lo, ~((E4M3[lo] <= E4M3[got]) & (E4M3[got] <= E4M3[hi])))
