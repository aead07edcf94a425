"""Heads' norms and rotation, the paged 4-bit cache and attention over it, from their definitions in 64 bits (numpy)."""

from __future__ import annotations

import math

import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])
# between magnitudes i and i + 1; a value on one goes to the even code
BORDERS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])


def encode(x):
    """The codes of the e2m1 values nearest to x, ties to the even code, at most 6."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)[..., None]
    up = np.where(np.arange(7) % 2 == 0, a > BORDERS, a >= BORDERS)
    return (up.sum(axis=-1) | np.where(np.signbit(x), 8, 0)).astype(np.uint8)


def pack(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack((packed & 15, packed >> 4), axis=-1).reshape(*packed.shape[:-1], -1)


def bf16(x):
    """x rounded to bfloat16 (nearest, ties to even), from 64 bits."""
    x = np.asarray(x, np.float64)
    m, e = np.frexp(x)
    return np.ldexp(np.round(m * 256), e - 8)


def key_exponent(amax):
    """The least e, -60 <= e <= 125, with amax <= 7 x 2^e (7 = 0.875 x 2^3)."""
    m, e = np.frexp(amax)
    return np.clip(np.where(amax > 0, e - 3 + (m > 0.875), -60), -60, 125)


def keys(x):
    """Keys [..., 128] as (codes [..., 128], exponents + 127 [..., 4]); a block that is not finite: 255, its codes 0."""
    b = x.reshape(*x.shape[:-1], 4, 32)
    ok = np.isfinite(b).all(axis=-1)
    b = np.where(ok[..., None], b, 0.0)
    e = key_exponent(np.abs(b).max(axis=-1))
    codes = encode(b / np.exp2(e.astype(np.float64))[..., None])
    return codes.reshape(x.shape), np.where(ok, e + 127, 255).astype(np.uint8)


def values(x):
    """Values [..., 128] as (codes, scales [...]); a row that is not finite: NaN, its codes 0."""
    ok = np.isfinite(x).all(axis=-1)
    x = np.where(ok[..., None], x, 0.0)
    s = np.maximum(bf16(np.abs(x).max(axis=-1) / 6), 2.0 ** -60)
    return encode(x / s[..., None]), np.where(ok, s, np.nan)


def key_scales(e):
    """The value of a key's scale bytes."""
    return np.where(e == 255, np.nan, np.exp2(e.astype(np.float64) - 127))


def by_slot(k_scale):
    """Scale bytes as they lie in pages [..., page / 16, 4, 4, 4] by slot [..., page, 4], and back."""
    x = np.moveaxis(k_scale, -1, -3)
    return np.ascontiguousarray(x).reshape(*x.shape[:-4], -1, 4)


def in_pages(scales):
    x = scales.reshape(*scales.shape[:-2], -1, 4, 4, 4)
    return np.ascontiguousarray(np.moveaxis(x, -3, -1))


def frequencies(theta, dim):
    return np.array([theta ** (-2 * j / dim) for j in range(dim // 2)])


def turn(x, pos, freq, dim=128, inter=False, factor=1.0, weight=None, eps=1e-6):
    """Heads x [rows, heads, 128] of rows at positions pos [rows], normed where there is a weight, and turned."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * weight
    a = np.asarray(pos, np.float64)[:, None, None] * np.asarray(freq)[None, None]
    c, s = factor * np.cos(a), factor * np.sin(a)
    y = x.copy()
    i = np.arange(dim // 2)
    p, q = (2 * i, 2 * i + 1) if inter else (i, i + dim // 2)
    y[..., p], y[..., q] = x[..., p] * c - x[..., q] * s, x[..., q] * c + x[..., p] * s
    return y


def turn_size(x, dim=128, inter=False, factor=1.0, weight=None, eps=1e-6):
    """The sum of the sizes of what each turned dim is made of."""
    x = np.abs(np.asarray(x, np.float64))
    if weight is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * np.abs(weight)
    y = x.copy()
    i = np.arange(dim // 2)
    p, q = (2 * i, 2 * i + 1) if inter else (i, i + dim // 2)
    y[..., p] = y[..., q] = abs(factor) * (x[..., p] + x[..., q])
    return y


def attend(q, k, v, table, page, pages, kv_len, rows, mask_block):
    """q [total, nq, 128] over keys and values [pages, heads, page, 128] (their values); rows[b] = indices of b's rows.  Returns
    out (0 for rows of no sequence), and for tolerances sum p |v| and the largest sum |q| |k| / sqrt(128) of each (row, head)."""
    nq, nkv = q.shape[1], k.shape[1]
    G = nq // nkv
    out, mass, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
    for b, idx in enumerate(rows):
        total = max(0, min(kv_len[b], table.shape[1] * page))
        at = np.array([p for p in range(total) if 0 <= table[b, p // page] < pages], dtype=np.int64)
        pg, sl = (table[b, at // page], at % page) if at.size else (at, at)
        for h in range(nkv):
            kk, vv = k[pg, h, sl], v[pg, h, sl]
            for i, r in enumerate(idx):
                pos = kv_len[b] - len(idx) + i
                see = at >= 0 if mask_block == 0 else at < (pos // mask_block + 1) * mask_block if pos >= 0 else at < 0
                if not see.any():
                    continue
                for hq in range(h * G, (h + 1) * G):
                    s = kk[see] @ q[r, hq] / math.sqrt(128)
                    with np.errstate(invalid="ignore"):
                        p = np.exp(s - s.max())
                        p /= p.sum()
                    out[r, hq] = p @ vv[see]
                    mass[r, hq] = p @ np.abs(vv[see])
                    reach[r, hq] = (np.abs(kk[see]) @ np.abs(q[r, hq])).max() / math.sqrt(128)
    return out, mass, reach
