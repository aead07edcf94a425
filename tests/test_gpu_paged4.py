"""HipVM.rotate_heads, the paged 4-bit cache (HipVM.paged4_append, paged4_read) and paged_attn over it against their
definitions in 64 bits (tests/paged4_reference.py), at the sizes, masks and values where they can go wrong."""

from __future__ import annotations

import ctypes
import math
import threading

import numpy as np
import pytest
import torch

import paged4_reference as ref
from helpers import log
from test_gpu_paged import HALF, TD, THETA, dev, i32, make_vm, rounded, tables

pytestmark = pytest.mark.gpu

EPS = 1e-6  # the test models' rms_norm_eps
LEAST = {"float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}  # half of the type's least step


class Pages:
    """A cache of two layers with its codes and scales on the host, by slot: k, v [2, pages, nkv, page, 128] codes, ke
    exponents + 127 [2, pages, nkv, page, 4], vs scales [2, pages, nkv, page]."""

    def __init__(self, rng, pages, nkv, page, garbage=False):
        shape = (2, pages, nkv, page)
        self.k, self.v = (rng.integers(0, 16, (*shape, 128)).astype(np.uint8) for _ in range(2))
        if garbage:  # what other owners left: scales of all kinds, NaN among them
            self.ke = rng.integers(0, 256, (*shape, 4)).astype(np.uint8)
            self.vs = ref.bf16(rng.standard_normal(shape) * 1e30)
            self.vs[rng.random(shape) < 0.3] = np.nan
        else:
            self.ke = rng.integers(124, 128, (*shape, 4)).astype(np.uint8)
            self.vs = ref.bf16(rng.uniform(0.1, 0.4, shape))
        self.page = page
        self.upload()

    def upload(self):
        from fast_dllm_relax_amd.paged4 import Paged4KVCache

        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        self.dev = Paged4KVCache(k=t(ref.pack(self.k)), v=t(ref.pack(self.v)), k_scale=t(ref.in_pages(self.ke)),
                                 v_scale=t(self.vs.astype(np.float32)).to(torch.bfloat16))

    def download(self):
        d = self.dev
        return (ref.unpack(d.k.cpu().numpy()), ref.unpack(d.v.cpu().numpy()), ref.by_slot(d.k_scale.cpu().numpy()),
                d.v_scale.double().cpu().numpy())

    def values(self, layer):
        """Keys and values of a layer, [pages, nkv, page, 128]."""
        return (ref.E2M1[self.k[layer]] * np.repeat(ref.key_scales(self.ke[layer]), 32, axis=-1),
                ref.E2M1[self.v[layer]] * self.vs[layer][..., None])


def same(a, b):
    return all(np.array_equal(x, y, equal_nan=x.dtype.kind == "f") for x, y in zip(a, b))


def rotary_of(dim=128, inter=False, scaling=None, **kw):
    from fast_dllm_relax_amd.rotary import Rotary

    return Rotary(theta=THETA, dim=dim, interleaved=inter, scaling=scaling, **kw)


# ---- norms and rotation ------------------------------------------------------------------------------------


def check_turned(got, x, pos, r, weight, dtype):
    """The angle in turns is rounded to fp32 once (an error of 2^-23.3 radians), sine and cosine and the products and sums of the
    rotation add less than 2^-21 of the sum of their sizes, the norm's three roundings 2^-22: 2^-20 in all; the result is
    rounded once.  In 64 bits a far position's angle is off by a few 2^-53 of itself."""
    exact = ref.turn(x, pos, r.frequencies, r.dim, r.interleaved, r.factor, weight, EPS)
    size = ref.turn_size(x, r.dim, r.interleaved, r.factor, weight, EPS)
    far = 2.0 ** -51 * np.abs(np.asarray(pos, np.float64))[:, None, None]
    room = size * (2.0 ** -20 + far)
    room += HALF[dtype] * (np.abs(exact) + room) + LEAST[dtype]
    worst = float(np.max(np.abs(got - exact) / room)) if got.size else 0.0
    log(f"  largest error {worst:.3f} of its bound")
    assert np.isfinite(got).all() and worst <= 1.0


ROTATES = [
    # dtype, nq, nkv, rows, dim, inter, scaling, norm, positions (an int: from there on)
    ("bfloat16", 12, 2, 1, 128, False, None, True, 2079),
    ("float16", 12, 2, 1, 128, True, None, False, [31]),
    ("bfloat16", 4, 2, 7, 64, False, dict(type="linear", factor=2.0), True, "far"),
    ("float16", 8, 8, 8, 32, True, dict(type="ntk", factor=4.0), True, "near"),
    ("bfloat16", 16, 1, 9, 16, False, None, False, -5),
    ("bfloat16", 12, 2, 33, 112, True, None, True, "far"),
    ("float16", 12, 2, 300, 128, False, dict(type="yarn", factor=4.0, original_len=32768), True, "far"),
    ("bfloat16", 5, 5, 65, 96, False, None, True, 0),
    ("bfloat16", 12, 2, 40, 0, False, None, True, "near"),
]


@pytest.mark.parametrize("case", range(len(ROTATES)))
def test_rotate_heads(case):
    dtype, nq, nkv, rows, dim, inter, scaling, norm, where = ROTATES[case]
    log(f"case: rotate {ROTATES[case]}")
    rng = np.random.default_rng(300 + case)
    vm = make_vm(dtype, nq, nkv)
    r = rotary_of(dim, inter, scaling)
    x = rounded(rng.standard_normal((rows, nq + 2 * nkv, 128)) * np.exp(rng.standard_normal((rows, 1, 1))), dtype)
    w = [rounded(1 + 0.3 * rng.standard_normal(128), dtype) if norm else None for _ in range(2)]
    if isinstance(where, int):
        pos, arg = where + np.arange(rows), where
    else:
        pos = np.array(where) if isinstance(where, list) else rng.integers(0, 1000 if where == "near" else 1000000, rows)
        arg = i32(pos)
    fused = dev(x, dtype)
    q, k = fused[:, :nq], fused[:, nq:nq + nkv]
    kw = dict(rotary=r, q_norm=dev(w[0], dtype) if norm else None, k_norm=dev(w[1], dtype) if norm else None)
    got = vm.rotate_heads(q, k, arg, **kw)
    for g, part, weight in zip(got, (x[:, :nq], x[:, nq:nq + nkv]), w):
        check_turned(g.double().cpu().numpy(), part, pos, r, weight, dtype)
    # one of the two alone; into given rows, of another stride; where they lie
    alone = vm.rotate_heads(q, None, arg, rotary=r, q_norm=kw["q_norm"]), vm.rotate_heads(None, k, arg, rotary=r, k_norm=kw["k_norm"])
    assert torch.equal(alone[0][0], got[0]) and torch.equal(alone[1][1], got[1])
    wide = torch.full((rows, nq + nkv + 1, 128), 9.0, dtype=TD[dtype], device="cuda")
    vm.rotate_heads(q, k, arg, q_out=wide[:, :nq], k_out=wide[:, nq + 1:], **kw)
    assert torch.equal(wide[:, :nq], got[0]) and torch.equal(wide[:, nq + 1:], got[1]) and (wide[:, nq] == 9.0).all()
    place = vm.rotate_heads(q, k, arg, q_out=q, k_out=k, **kw)
    assert place[0] is q and torch.equal(q, got[0]) and torch.equal(k, got[1])
    assert np.array_equal(fused[:, nq + nkv:].double().cpu().numpy(), x[:, nq + nkv:])


def test_rotate_heads_is_the_models_own_without_a_plan():
    log("case: the model's rotation")
    rng = np.random.default_rng(310)
    vm = make_vm()
    x = dev(rng.standard_normal((50, 14, 128)), "bfloat16")
    a = vm.rotate_heads(x[:, :12], x[:, 12:], 500)
    b = vm.rotate_heads(x[:, :12], x[:, 12:], 500, rotary=rotary_of())
    c = vm.rotate_heads(x[:, :12], x[:, 12:], i32(500 + np.arange(50)))
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, q) and torch.equal(p, r)
    assert vm.rotate_heads(x[:0, :12], x[:0, 12:], 0)[0].shape == (0, 12, 128)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_norms_of_hard_rows(dtype):
    """Zeros, the type's largest and least values, and rows that are not finite, which spoil their own head alone."""
    log(f"case: norms of hard rows, {dtype}")
    rng = np.random.default_rng(311)
    vm = make_vm(dtype)
    big, least = float(torch.finfo(TD[dtype]).max), 2 * LEAST[dtype]
    x = rounded(rng.standard_normal((12, 12, 128)), dtype)
    x[0] = 0
    x[1] = big * np.sign(x[1])
    x[2] = least
    x[3, :, ::2] = big
    x[4, 3, 7], x[5, 0, 100], x[6, 11, 64] = np.nan, np.inf, -np.inf
    w = rounded(1 + 0.3 * rng.standard_normal(128), dtype)
    r = rotary_of()
    g = vm.rotate_heads(dev(x, dtype), None, 1000, rotary=r, q_norm=dev(w, dtype))[0].double().cpu().numpy()
    fine = np.isfinite(x).all(axis=-1)
    bad = ~fine
    assert np.isnan(g[4, 3]).any() and np.isnan(g[5, 0]).any() and np.isnan(g[6, 11]).any() and bad.sum() == 3
    check_turned(np.where(bad[..., None], 0, g), np.where(bad[..., None], 0, x), 1000 + np.arange(12), r, w, dtype)


# ---- append and read ---------------------------------------------------------------------------------------


def between(got, lo, hi):
    """Codes stand between those of two bounds, which are in the order of the values."""
    v, a, b = (ref.E2M1[c] for c in (got, lo, hi))
    return (a <= v) & (v <= b)


def check_keys(code, e, y, size, given):
    """Codes and exponents of rows y [.., 128]: a rotation in 64 bits whose sines are within 2^-33 and whose angles are off by
    2^-31 at most, rounded once to fp32; encoding is monotone, so the codes lie between those of the bounds, and so does the
    exponent.  Hardly any is left open by them.  Dims that nothing changes are the `given` ones, exactly."""
    err = np.where(y == given, 0.0, 2.0 ** -24 * np.abs(y) + 2.0 ** -30 * size)
    top = lambda a: ref.key_exponent(a.reshape(*a.shape[:-1], 4, 32).max(axis=-1)) + 127  # noqa: E731
    lo_e, hi_e = top(np.maximum(np.abs(y) - err, 0)), top(np.abs(y) + err)
    assert ((lo_e <= e) & (e <= hi_e)).all()
    s = np.repeat(ref.key_scales(e), 32, axis=-1)
    lo, hi = ref.encode((y - err) / s), ref.encode((y + err) / s)
    log(f"  codes left open: {int((ref.E2M1[lo] != ref.E2M1[hi]).sum())} of {lo.size}; exponents: {int((lo_e != hi_e).sum())}")
    open_, fine = float((ref.E2M1[lo] != ref.E2M1[hi]).mean()), bool(between(code, lo, hi).all())
    assert open_ < 1e-4 + 2 / lo.size and fine


APPENDS = [
    # dtype, nq, nkv, page, rows per sequence, start, pos (None: start), dim, inter, scaling, norm
    ("bfloat16", 12, 2, 32, [1], [2079], None, 128, False, None, True),
    ("bfloat16", 12, 2, 32, [1, 1, 1], [0, 31, 32], None, 128, False, None, False),
    ("float16", 12, 2, 32, [8, 8], [136, 40], None, 128, False, None, True),
    ("bfloat16", 4, 2, 16, [37, 0, 5], [11, 3, 0], [100000, 0, 31000], 64, True, dict(type="linear", factor=2.0), True),
    ("float16", 8, 8, 64, [130, 64], [1, 64], None, 32, False, dict(type="ntk", factor=4.0), False),
    ("bfloat16", 16, 1, 128, [128, 300, 1], [0, 127, 500], None, 128, True, dict(type="yarn", factor=4.0, original_len=32768), True),
    ("bfloat16", 12, 2, 32, [32, 32], [-1, 0], None, 128, False, None, True),
    ("float16", 3, 3, 16, [9, 20], [7, 15], None, 16, False, None, True),
    ("bfloat16", 6, 2, 64, [9], [60], [-3], 0, False, None, False),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(case):
    dtype, nq, nkv, page, n, start, pos, dim, inter, scaling, norm = APPENDS[case]
    log(f"case: append {APPENDS[case]}")
    rng = np.random.default_rng(400 + case)
    vm = make_vm(dtype, nq, nkv)
    nseq, width = len(n), (max(s + k for s, k in zip(start, n)) + page - 1) // page + 1
    pg = Pages(rng, nseq * width + 2, nkv, page, garbage=True)
    table = tables(rng, nseq, width, nseq * width + 2)
    r = rotary_of(dim, inter, scaling)
    uniform = len(set(n)) == 1
    rows = sum(n)
    total = rows if uniform else rows + 3
    first = np.concatenate([[0], np.cumsum(n)])
    x = rounded(rng.standard_normal((total, nq + 2 * nkv, 128)) * np.exp(rng.standard_normal((total, 1, 1))), dtype)
    w = [rounded(1 + 0.3 * rng.standard_normal(128), dtype) if norm else None for _ in range(2)]
    fused = dev(x, dtype)
    q_out = torch.full((total, nq, 128), 9.0, dtype=TD[dtype], device="cuda")
    kw = {} if uniform else dict(row_start=i32(first), max_rows=max(n))
    before = [a.copy() for a in pg.download()]
    assert same(before, (pg.k, pg.v, pg.ke, pg.vs))
    got = vm.paged4_append(fused[:, nq:nq + nkv], fused[:, nq + nkv:], pg.dev, 1, i32(table), i32(start), q=fused[:, :nq], q_out=q_out,
                           pos=None if pos is None else i32(pos), rotary=r, q_norm=dev(w[0], dtype) if norm else None,
                           k_norm=dev(w[1], dtype) if norm else None, **kw)
    assert got is q_out
    after = pg.download()
    gq = q_out.double().cpu().numpy()
    for b in range(nseq):
        sl = slice(first[b], first[b + 1])
        if start[b] < 0:
            assert (gq[sl] == 9.0).all()
            continue
        at = (start if pos is None else pos)[b] + np.arange(n[b])
        check_turned(gq[sl], x[sl, :nq], at, r, w[0], dtype)
        p = start[b] + np.arange(n[b])
        pgs, sl_ = table[b, p // page], p % page
        y = ref.turn(x[sl, nq:nq + nkv], at, r.frequencies, dim, inter, r.factor, w[1], EPS)
        size = ref.turn_size(x[sl, nq:nq + nkv], dim, inter, r.factor, w[1], EPS)
        if n[b]:
            check_keys(after[0][1, pgs, :, sl_], after[2][1, pgs, :, sl_], y, size, x[sl, nq:nq + nkv])
        code, s = ref.values(x[sl, nq + nkv:])
        assert np.array_equal(after[1][1, pgs, :, sl_], code) and np.array_equal(after[3][1, pgs, :, sl_], s)
        for old, new in zip(before, after):
            old[1, pgs, :, sl_] = new[1, pgs, :, sl_]
    assert (gq[rows:] == 9.0).all()
    assert same(before, after)  # nothing else changed
    # what is read back is what the codes stand for, rounded once; q rotated in place
    pg.k, pg.v, pg.ke, pg.vs = after
    out = [torch.full((total, nkv, 128), 9.0, dtype=TD[dtype], device="cuda") for _ in range(2)]
    vm.paged4_read(pg.dev, 1, i32(table), i32(start), total, k_out=out[0], v_out=out[1], **kw)
    for o, vals in zip(out, pg.values(1)):
        g = o.double().cpu().numpy()
        for b in range(nseq):
            if start[b] < 0:
                continue
            p = start[b] + np.arange(n[b])
            assert np.array_equal(g[first[b]:first[b + 1]], rounded(vals[table[b, p // page], :, p % page], dtype))
        assert (g[rows:] == 9.0).all()
    qc = fused[:, :nq].contiguous()
    again = vm.paged4_append(fused[:, nq:nq + nkv], fused[:, nq + nkv:], pg.dev, 1, i32(table), i32(start), q=qc, q_out=qc,
                             pos=None if pos is None else i32(pos), rotary=r, q_norm=dev(w[0], dtype) if norm else None,
                             k_norm=dev(w[1], dtype) if norm else None, **kw)
    live = np.concatenate([np.arange(first[b], first[b + 1]) for b in range(nseq) if start[b] >= 0])
    assert again is qc and torch.equal(qc[live], q_out[live]) and same(pg.download(), after)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_append_values_that_are_hard(dtype):
    """Not rotated: zeros, the type's largest and least values, values on the borders between codes, and values that are not
    finite, which make their block's or row's scale NaN and no other."""
    log(f"case: hard values, {dtype}")
    rng = np.random.default_rng(420)
    vm = make_vm(dtype)
    n, page = 64, 32
    big, least = float(torch.finfo(TD[dtype]).max), 2 * LEAST[dtype]
    x = rng.standard_normal((n, 2, 128)) * np.exp2(rng.integers(-12, 12, (n, 2, 1)))
    x[0], x[1], x[2] = 0, big * np.sign(x[1]), least
    x[3] = 0.0
    x[3, :, 5] = big
    # every border of every amax with few bits: 6 / 8 of its size and so on
    for i in range(4, 40):
        top = rng.integers(128, 256) * 2.0 ** -7
        x[i] = np.resize(np.concatenate([ref.BORDERS, ref.E2M1[:8]]) * top / 6, 128) * rng.choice([-1, 1], 128)
        x[i, :, 0] = top
    x[40, 0, 3], x[41, 1, 127], x[42, 1, 64] = np.nan, np.inf, -np.inf
    x[43] = 7 * 2.0 ** -3
    x[44, :, ::32] = 6 * 2.0 ** -3
    x = rounded(x, dtype)
    pg = Pages(rng, 3, 2, page, garbage=True)
    table = tables(rng, 1, 2, 3)
    vm.paged4_append(dev(x, dtype), dev(x, dtype), pg.dev, 0, i32(table), i32([0]), rotary=rotary_of(0))
    k, v, ke, vs = (a[0, table[0]] for a in pg.download())
    order = lambda a: a.swapaxes(1, 2).reshape(n, 2, *a.shape[3:])  # noqa: E731
    code, e = ref.keys(x)
    ok = np.repeat(e != 255, 32, axis=-1)
    assert np.array_equal(order(ke), e) and np.array_equal(order(k)[ok], code[ok]) and (e == 255).sum() == 3
    code, s = ref.values(x)
    ok = ~np.isnan(s)
    assert np.array_equal(order(vs), s, equal_nan=True) and np.array_equal(order(v)[ok], code[ok]) and (~ok).sum() == 3
    kb, vb = vm.paged4_read(pg.dev, 0, i32(table), i32([0]), n)
    assert np.isnan(kb.double().cpu().numpy()).sum() == 3 * 32 and np.isnan(vb.double().cpu().numpy()).sum() == 3 * 128


def test_append_bad_pages_and_row_starts_write_nothing():
    log("case: page numbers out of range, positions past the table, hostile row starts")
    rng = np.random.default_rng(421)
    vm = make_vm()
    page = 16
    pg = Pages(rng, 5, 2, page)
    before = pg.download()
    x = dev(rng.standard_normal((60, 12, 128)), "bfloat16")
    table = i32([[-1, 5, 2 ** 31 - 1], [-2 ** 31, 9, -7], [7, 6, 100]])
    q = vm.paged4_append(x[:, :2], x[:, :2], pg.dev, 1, table, i32([0, 30, 5]), q=x)
    assert torch.isfinite(q).all() and same(pg.download(), before)
    # positions behind the table's last, where the pages are good ones
    good = i32([[0, 1], [2, 3], [4, 0]])
    vm.paged4_append(x[:, :2], x[:, :2], pg.dev, 1, good, i32([32, 2 ** 31 - 1, 2 ** 31 - 20]), q=x)
    assert same(pg.download(), before)
    start = i32([0, 0, 0])
    for rs in ([5, 2, 1, 0], [60, 2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31], [-7, -3, -2, -1]):
        out = torch.full_like(x, 9.0)
        kv = [torch.full_like(x[:, :2], 9.0) for _ in range(2)]
        vm.paged4_append(x[:, :2], x[:, :2], pg.dev, 0, good, start, row_start=i32(rs), q=x, q_out=out)
        vm.paged4_read(pg.dev, 0, good, start, 60, row_start=i32(rs), k_out=kv[0], v_out=kv[1])
        vm.paged_attn(x, pg.dev, 0, good, i32([20, 30, 40]), row_start=i32(rs), out=out)
        assert (out == 9.0).all() and (kv[0] == 9.0).all() and (kv[1] == 9.0).all()
    assert same(pg.download(), before)


@pytest.mark.parametrize("page,most", [(16, 40), (32, 7), (64, 33), (128, 150)])
def test_appends_of_all_kinds(page, most):
    """Random appends one after another, rows of earlier ones rewritten among them, rows in front of the first sequence and
    behind the last, pages that sequences share: the cache holds each position's last row and nothing else changed."""
    log(f"case: random appends of up to {most} rows, pages of {page}")
    rng = np.random.default_rng(430 + page)
    vm = make_vm()
    nseq, width = 3, max(2, 160 // page) + most // page
    pg = Pages(rng, nseq * width + 1, 2, page, garbage=True)
    table = tables(rng, nseq, width, nseq * width + 1)
    table[1, -1] = table[2, -1] = table[0, -1]  # a page that all write, at slots of their own
    third = page // 3
    k, v, ke, vs = (a.copy() for a in pg.download())
    for step in range(25):
        n = [int(rng.integers(0, most + 1)) for _ in range(nseq)]
        start = [int(rng.integers(0, max(1, (width - 1) * page - m))) for m in n]
        if step % 5 == 4:  # into the shared page
            n = [int(rng.integers(0, min(third, most) + 1)) for _ in range(nseq)]
            start = [(width - 1) * page + b * third for b in range(nseq)]
        lead, tail = int(rng.integers(0, 3)), int(rng.integers(0, 3))
        first = lead + np.concatenate([[0], np.cumsum(n)])
        rows = lead + sum(n) + tail
        if rows == 0:
            continue
        x = rounded(rng.standard_normal((rows, 2, 128)) * 2.0 ** rng.integers(-20, 21, (rows, 2, 1)), "bfloat16")
        vm.paged4_append(dev(x, "bfloat16"), dev(x, "bfloat16"), pg.dev, 1, i32(table), i32(start), rotary=rotary_of(0),
                         row_start=i32(first), max_rows=most)
        for b in range(nseq):
            p = start[b] + np.arange(n[b])
            at = (1, table[b, p // page], slice(None), p % page)
            part = x[first[b]:first[b + 1]]
            k[at], ke[at] = ref.keys(part)
            v[at], vs[at] = ref.values(part)
    fine = same(pg.download(), (k, v, ke, vs))
    assert fine


@pytest.mark.parametrize("nseq,most", [(64, 3), (65, 9), (200, 40), (511, 2), (512, 3), (700, 12), (3, 2000)])
def test_many_sequences(nseq, most):
    """Ragged batches of more sequences than a wave has lanes, empty ones among them, padded on both sides, with few rows and many:
    every row goes to its own place and comes back from there."""
    log(f"case: {nseq} sequences of up to {most} rows")
    rng = np.random.default_rng(450 + nseq)
    vm = make_vm("bfloat16", 4, 2)
    page = 16
    n = rng.integers(0, most + 1, nseq)
    n[rng.random(nseq) < 0.2] = 0
    start = rng.integers(0, 20, nseq)
    start[nseq // 3] = -1
    width = (int((start + n).max()) + page) // page
    pg = Pages(rng, nseq * width, 2, page, garbage=True)
    table = tables(rng, nseq, width, nseq * width)
    lead, tail = 3, 5
    first = lead + np.concatenate([[0], np.cumsum(n)])
    total = int(first[-1]) + tail
    x = rounded(rng.standard_normal((total, 8, 128)), "bfloat16")
    fused = dev(x, "bfloat16")
    q_out = torch.full((total, 4, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    before = [a.copy() for a in pg.download()]
    kw = dict(row_start=i32(first), max_rows=most)
    vm.paged4_append(fused[:, 4:6], fused[:, 6:], pg.dev, 1, i32(table), i32(start), q=fused[:, :4], q_out=q_out, rotary=rotary_of(0), **kw)
    seq = np.repeat(np.arange(nseq), n)
    at = np.concatenate([np.arange(k) for k in n])
    live = start[seq] >= 0
    seq, at, row = seq[live], at[live], (lead + np.arange(len(seq)))[live]
    p = start[seq] + at
    where = (1, table[seq, p // page], slice(None), p % page)
    before[0][where], before[2][where] = ref.keys(x[row, 4:6])
    before[1][where], before[3][where] = ref.values(x[row, 6:])
    fine = same(before, pg.download())
    assert fine
    want = np.full((total, 4, 128), 9.0)
    want[row] = x[row, :4]
    assert np.array_equal(q_out.double().cpu().numpy(), want)
    out = [torch.full((total, 2, 128), 9.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    vm.paged4_read(pg.dev, 1, i32(table), i32(start), total, k_out=out[0], v_out=out[1], **kw)
    pg.k, pg.v, pg.ke, pg.vs = before
    for o, vals in zip(out, pg.values(1)):
        want = np.full((total, 2, 128), 9.0)
        want[row] = rounded(vals[table[seq, p // page], :, p % page], "bfloat16")
        got = o.double().cpu().numpy()
        skipped = np.zeros(total, bool)
        skipped[first[nseq // 3]:first[nseq // 3 + 1]] = True  # (from position -1: zeros, then what is there)
        assert np.array_equal(got[~skipped], want[~skipped])


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_read(dtype):
    """All scales there are, pages that are none, negative positions, lengths that end inside a page; into rows of a contiguous
    cache, where nothing else changes, and into new tensors."""
    log(f"case: read, {dtype}")
    rng = np.random.default_rng(440)
    vm = make_vm(dtype)
    page, n, start = 32, [70, 0, 33, 9], [5, 9, 40, -4]
    pg = Pages(rng, 12, 2, page, garbage=True)
    pg.vs[:, ::2] = ref.bf16(2.0 ** rng.uniform(-20, 12, pg.vs[:, ::2].shape))
    pg.upload()
    table = np.array([[3, 11, 0, 7], [1, 1, 1, 1], [2, -1, 5, 12], [6, 4, 10, 9]])
    first = np.concatenate([[0], np.cumsum(n)])
    rows = sum(n)
    with np.errstate(over="ignore"):
        vals = [rounded(a, dtype) for a in pg.values(0)]
    kw = dict(row_start=i32(first), max_rows=70)
    whole = torch.full((2, 1, rows + 9, 2, 128), 9.0, dtype=TD[dtype], device="cuda")
    vm.paged4_read(pg.dev, 0, i32(table), i32(start), rows + 3, k_out=whole[0, 0, 2:rows + 5], v_out=whole[1, 0, 2:rows + 5], **kw)
    new = vm.paged4_read(pg.dev, 0, i32(table), i32(start), rows + 3, row_start=i32(first))
    for i in range(2):
        g = whole[i, 0].double().cpu().numpy()
        want = np.full((rows + 9, 2, 128), 9.0)
        for b in range(4):
            for j in range(n[b]):
                p = start[b] + j
                pgn = table[b, p // page] if 0 <= p < 4 * page else -1
                want[2 + first[b] + j] = vals[i][pgn, :, p % page] if 0 <= pgn < 12 else 0.0
        assert np.array_equal(g, want, equal_nan=True)
        h = new[i].double().cpu().numpy()
        assert np.array_equal(h[:rows], want[2:rows + 2], equal_nan=True) and not h[rows:].any()


# ---- attention ---------------------------------------------------------------------------------------------


def check_attn(got, want, mass, reach, dtype, few):
    """P times V's scale is rounded once to the type, in bf16 to two parts of it where a tile has few rows; the
    result once: each off by at most half a step (fp16: at least 2^-36 of the row's largest, six times which is no more than the
    largest mass of a dim, for each of at most 2^13 keys).  The scores' fp32 sums are off by less than 2^-17 of the sum of their sizes
    (the queries' parts by 2^-21 of their block's largest value, which here is no more), and exp turns that into a relative error of p and
    of the sum that divides it."""
    u = HALF[dtype] + (HALF[dtype] if dtype == "float16" or not few else 2.0 ** -16)
    least = 2.0 ** -23 * mass.max(axis=-1, keepdims=True) if dtype == "float16" else 0.0
    room = least + mass * (u * (1 + 2.0 ** -6) + 2 * reach[..., None] * 2.0 ** -17 + 2.0 ** -16) + 2 * LEAST[dtype] + 2.0 ** -100
    worst = float(np.max(np.abs(got - want) / room)) if got.size else 0.0
    log(f"  largest error {worst:.3f} of its bound")
    assert np.isfinite(got).all() and worst <= 1.0


ATTNS = [
    # dtype, nq, nkv, page, rows per sequence, kv_len, mask_block
    ("bfloat16", 12, 2, 32, [1], [1], 0),
    ("bfloat16", 12, 2, 32, [1], [2080], 0),
    ("float16", 12, 2, 32, [32, 32, 32], [160, 33, 1055], 0),
    ("bfloat16", 4, 2, 16, [37, 0, 5, 1], [37, 9, 64, 65], 1),
    ("bfloat16", 12, 2, 64, [70, 33], [97, 300], 32),
    ("float16", 8, 8, 128, [3, 1, 2], [129, 127, 640], 1),
    ("bfloat16", 16, 1, 64, [9], [400], 0),
    ("bfloat16", 6, 2, 32, [5, 4], [0, 2], 1),      # nothing cached; more rows than positions
    ("float16", 12, 2, 16, [2, 2], [0, -5], 0),
    ("bfloat16", 12, 2, 32, [1, 1, 1, 1, 1], [64, 4000, 63, 65, 1], 1),
    ("bfloat16", 12, 2, 32, [200], [8000], 32),
    ("float16", 16, 1, 16, [1, 1], [3001, 17], 1),
    ("bfloat16", 5, 5, 64, [17], [5000], 0),
    ("float16", 12, 2, 32, [200], [1000], 1),
    ("bfloat16", 64, 1, 128, [3], [700], 1),
    ("bfloat16", 12, 2, 32, [300, 100, 1], [300, 2000, 640], 32),
]


@pytest.mark.parametrize("case", range(len(ATTNS)))
def test_attention(case):
    dtype, nq, nkv, page, n, kv_len, mask = ATTNS[case]
    log(f"case: attention {ATTNS[case]}")
    rng = np.random.default_rng(500 + case)
    vm = make_vm(dtype, nq, nkv)
    nseq, width = len(n), max(1, (max(kv_len) + page - 1) // page)
    pg = Pages(rng, nseq * width + 1, nkv, page)
    table = tables(rng, nseq, width, nseq * width + 1)
    # what lies behind the sequences' ends is NaN
    for b in range(nseq):
        for p in range(max(0, kv_len[b]), width * page):
            pg.ke[:, table[b, p // page], :, p % page] = 255
            pg.vs[:, table[b, p // page], :, p % page] = np.nan
    pg.upload()
    rows = sum(n)
    uniform = len(set(n)) == 1
    total = rows if uniform else rows + 3
    first = np.concatenate([[0], np.cumsum(n)])
    q = rounded(rng.standard_normal((total, nq, 128)) * 0.5, dtype)
    out = torch.full((total, nq, 128), 9.0, dtype=TD[dtype], device="cuda")
    kw = {} if uniform else dict(row_start=i32(first), max_rows=max(n))
    got = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32(kv_len), mask_block=mask, out=out, **kw)
    assert got is out
    idx = [np.arange(first[b], first[b + 1]) for b in range(nseq)]
    want, mass, reach = ref.attend(q, *pg.values(1), table, page, nseq * width + 1, kv_len, idx, mask)
    g = out.double().cpu().numpy()
    few = max(n) * (nq // nkv) <= 16
    assert (g[rows:] == 9.0).all()
    check_attn(g[:rows], want[:rows], mass[:rows], reach[:rows], dtype, few)
    # rows without a key are zeros
    assert (g[:rows][mass[:rows].sum(axis=-1) == 0] == 0).all()
    # the same call again, planned for a bound: the split differs, the bits of one plan do not
    again = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32(kv_len), mask_block=mask, out=torch.full_like(out, 9.0), **kw)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))
    short = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32(kv_len), mask_block=mask, max_len=1,
                          out=torch.full_like(out, 9.0), **kw)
    check_attn(short.double().cpu().numpy()[:rows], want[:rows], mass[:rows], reach[:rows], dtype, few)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("nseq,most,least,mask", [(16, 150, 145, 1), (20, 200, 1, 32), (16, 80, 30, 1), (40, 17, 17, 0), (5, 150, 150, 32)])
def test_attention_of_many_sequences(dtype, nseq, most, least, mask):
    """Batches whose workgroups are several to a compute unit or few, with two tiles of rows and with three: ragged, under a
    mask, NaN behind every sequence's end."""
    log(f"case: {nseq} sequences of {least} to {most} rows, mask {mask}, {dtype}")
    rng = np.random.default_rng(530)
    vm = make_vm(dtype, 8, 8)
    page, width = 32, 10
    n = [most, *rng.integers(least, most + 1, nseq - 1)]
    kv_len = [int(rng.integers(max(0, k - 5), 32 * width + 1)) for k in n]
    pg = Pages(rng, nseq * width, 8, page)
    table = tables(rng, nseq, width, nseq * width)
    for b in range(nseq):
        for p in range(kv_len[b], width * page):
            pg.ke[:, table[b, p // page], :, p % page] = 255
            pg.vs[:, table[b, p // page], :, p % page] = np.nan
    pg.upload()
    first = np.concatenate([[0], np.cumsum(n)])
    rows = int(first[-1])
    q = rounded(rng.standard_normal((rows + 2, 8, 128)) * 0.5, dtype)
    idx = [np.arange(first[b], first[b + 1]) for b in range(nseq)]
    want, mass, reach = ref.attend(q, *pg.values(1), table, page, nseq * width, kv_len, idx, mask)
    out = torch.full((rows + 2, 8, 128), 9.0, dtype=TD[dtype], device="cuda")
    vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32(kv_len), mask_block=mask, row_start=i32(first), max_rows=most, out=out)
    g = out.double().cpu().numpy()
    assert (g[rows:] == 9.0).all() and (g[:rows][mass[:rows].sum(axis=-1) == 0] == 0).all()
    check_attn(g[:rows], want[:rows], mass[:rows], reach[:rows], dtype, False)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("rise", [0.02, 0.3, 3.0, -0.3])
def test_attention_of_rising_scores(dtype, n, rise):
    """Scores that rise (or fall) from key to key by so much in powers of two, so that the running maximum moves at every tile,
    by less than its bound or by more."""
    log(f"case: scores that rise by {rise}, {n} rows, {dtype}")
    rng = np.random.default_rng(531)
    vm = make_vm(dtype)
    page, L = 32, 640
    width = L // page
    pg = Pages(rng, width, 2, page)
    table = tables(rng, 1, width, width)
    # dims 0 .. 4 of a key hold its position's digits in base 5, 5 .. 31 nothing (the parts of the query's first block hold its
    # five values as they are: 2^9.3 lie between them, and a value keeps its bits down to 2^-21 of the largest)
    pg.ke[:] = 125
    digits = np.array([0, 2, 4, 5, 6], np.uint8)  # the codes of 0, 1, 2, 3, 4
    at = np.empty((width, page), int)
    at[table[0]] = np.arange(L).reshape(width, page)
    for layer in range(2):
        for j in range(5):
            pg.k[layer, :, :, :, j] = digits[at // 5 ** j % 5][:, None]
        pg.ke[layer, ..., 0] = 127
        pg.k[layer, ..., 5:32] = 0
    pg.upload()
    q = rng.standard_normal((n, 12, 128)) * 0.3
    q[:, :, :5] = rise * math.log(2) * math.sqrt(128) * 5.0 ** np.arange(5)
    q = rounded(q, dtype)
    want, mass, reach = ref.attend(q, *pg.values(1), table, page, width, [L], [np.arange(n)], 0)
    for max_len in (None, 1):
        g = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32([L]), max_len=max_len).double().cpu().numpy()
        check_attn(g, want, mass, reach, dtype, n == 1)


@pytest.mark.parametrize("nq,nkv,n,L,mask", [(12, 2, 100, 230, 1), (12, 2, 100, 230, 32), (12, 2, 9, 3000, 1), (16, 1, 1, 3000, 1), (12, 2, 2, 3000, 1)])
def test_attention_nan_behind_the_mask(nq, nkv, n, L, mask):
    """Keys that a row does not attend may hold NaN: rows in front of it are as without it, rows that see it are NaN throughout
    (in the head's dims)."""
    log(f"case: NaN behind a mask of {mask}, {nq} heads, {n} rows over {L}")
    rng = np.random.default_rng(510)
    vm = make_vm("bfloat16", nq, nkv)
    page = 32
    width = (L + page - 1) // page
    pg = Pages(rng, width + 1, nkv, page)
    table = tables(rng, 1, width, width + 1)
    q = rounded(rng.standard_normal((n, nq, 128)) * 0.5, "bfloat16")
    want, mass, reach = ref.attend(q, *pg.values(1), table, page, width + 1, [L], [np.arange(n)], mask)
    at_v, at_k = L - n + n // 2, L - n + (3 * n) // 4
    pg.vs[1, table[0, at_v // page], 0, at_v % page] = np.nan
    pg.ke[1, table[0, at_k // page], nkv - 1, at_k % page, 2] = 255
    pg.upload()
    pos = np.arange(L - n, L)
    sees = lambda p: (pos // mask + 1) * mask > p  # noqa: E731
    G = nq // nkv
    bad = np.zeros(q.shape, bool)
    bad[sees(at_v), :G] = True
    bad[sees(at_k), (nkv - 1) * G:] = True
    for max_len in (None, 1):
        g = vm.paged_attn(dev(q, "bfloat16"), pg.dev, 1, i32(table), i32([L]), mask_block=mask, max_len=max_len).double().cpu().numpy()
        assert np.isnan(g[bad]).all()
        check_attn(np.where(bad, want, g), want, mass, reach, "bfloat16", n * G <= 16)


@pytest.mark.parametrize("nq,nkv,n", [(12, 2, 1), (12, 2, 8)])
def test_attention_nan_of_vanishing_probability(nq, nkv, n):
    """A NaN in V at a key that is attended, at a probability that no float holds, spoils its head whether the keys are split
    over workgroups or not."""
    log(f"case: NaN at a vanishing probability, {n} rows")
    rng = np.random.default_rng(511)
    vm = make_vm("bfloat16", nq, nkv)
    page, L = 64, 3008
    width = L // page
    pg = Pages(rng, width, nkv, page)
    table = tables(rng, 1, width, width)
    pg.ke[:] = 127
    pg.k[:] = 2 | 8
    pg.k[1, table[0, 0]] = 2  # scores of +90 in the first page, of -90 elsewhere
    q = np.full((n, nq, 128), 8.0)
    want, mass, reach = ref.attend(q, *pg.values(1), table, page, width, [L], [np.arange(n)], 0)
    pg.vs[1, table[0, (L - 100) // page], 0, (L - 100) % page] = np.nan
    pg.upload()
    bad = np.zeros(q.shape, bool)
    bad[:, :nq // nkv] = True
    for max_len in (None, 1):
        g = vm.paged_attn(dev(q, "bfloat16"), pg.dev, 1, i32(table), i32([L]), max_len=max_len).double().cpu().numpy()
        assert np.array_equal(np.isnan(g), bad)
        check_attn(np.where(bad, want, g), want, mass, reach, "bfloat16", n * nq // nkv <= 16)


def test_attention_pages_that_are_none():
    log("case: page numbers out of range inside the length, a length past the table")
    rng = np.random.default_rng(512)
    vm = make_vm()
    pg = Pages(rng, 6, 2, 32)
    table = np.array([[3, -1, 5, 6], [2 ** 31 - 1, 0, -7, 2]])
    kv_len = [120, 2 ** 31 - 1]
    for n in (1, 10):
        q = rounded(rng.standard_normal((2 * n, 12, 128)) * 0.5, "bfloat16")
        want, mass, reach = ref.attend(q, *pg.values(0), table, 32, 6, kv_len, [np.arange(n), n + np.arange(n)], 0)
        g = vm.paged_attn(dev(q, "bfloat16"), pg.dev, 0, i32(table), i32(kv_len))
        check_attn(g.double().cpu().numpy(), want, mass, reach, "bfloat16", n == 1)


@pytest.mark.parametrize("dtype,lo,hi", [("bfloat16", -60, 125), ("bfloat16", -60, -50), ("bfloat16", 110, 125), ("float16", -40, 10)])
@pytest.mark.parametrize("n,L,mask", [(40, 150, 1), (2, 1500, 1), (1, 96, 0)])
def test_attention_value_scales_of_all_sizes(dtype, lo, hi, n, L, mask):
    """V's scales from 2^lo to 2^hi beside each other: what is in range comes out, and large ones behind a mask do no harm."""
    log(f"case: V scales 2^{lo} .. 2^{hi}, {dtype}, {n} rows over {L} keys, mask {mask}")
    rng = np.random.default_rng(513)
    vm = make_vm(dtype)
    page = 32
    width = (L + page - 1) // page
    pg = Pages(rng, width + 1, 2, page)
    pg.vs = ref.bf16(np.minimum(2.0 ** rng.uniform(lo, hi, pg.vs.shape), 2.0 ** 125))
    pg.upload()
    table = tables(rng, 1, width, width + 1)
    q = rounded(rng.standard_normal((n, 12, 128)) * 0.3, dtype)
    want, mass, reach = ref.attend(q, *pg.values(1), table, page, width + 1, [L], [np.arange(n)], mask)
    assert np.abs(want).max() < torch.finfo(TD[dtype]).max * 0.95
    for max_len in (None, 1):
        g = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32([L]), mask_block=mask, max_len=max_len).double().cpu().numpy()
        check_attn(g, want, mass, reach, dtype, n * 6 <= 16)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("n", [1, 7])
def test_attention_key_scales_and_queries_of_all_sizes(dtype, n):
    """K's blocks from 2^-60 to 2^100 under queries that are small where they are large (sums of products stay ordinary), queries
    of zeros, of the type's least values, with one value far above the rest; one that is not finite is NaN, its neighbours are not."""
    log(f"case: key scales and queries, {dtype}, {n} rows")
    rng = np.random.default_rng(514)
    vm = make_vm(dtype)
    page, L = 32, 200
    width = (L + page - 1) // page
    pg = Pages(rng, width, 2, page)
    table = tables(rng, 1, width, width)
    span = 12 if dtype == "float16" else 40
    shift = np.array([span // 4, 0, -span // 4, -span])
    pg.ke = (125 + shift + rng.integers(0, 2, pg.ke.shape)).astype(np.uint8)
    pg.upload()
    q = rng.standard_normal((n, 12, 128)) * 0.4 * np.repeat(np.exp2(-shift.astype(np.float64)), 32)
    q[:, 1], q[:, 2], q[:, 3] = 0.0, 2 * LEAST[dtype], rng.standard_normal(128) * 2.0 ** -9
    q[:, 3, 77] = 1.0
    q = rounded(q, dtype)
    want, mass, reach = ref.attend(q, *pg.values(1), table, page, width, [L], [np.arange(n)], 0)
    # a part's least step: 2^-21 of the largest value of a block of 32 for each of its dims
    size = np.abs(pg.values(1)[0]).reshape(width, 2, page, 4, 32).sum(axis=-1).max(axis=(0, 1, 2))
    reach = reach + (np.abs(q).reshape(n, 12, 4, 32).max(axis=-1) @ size) * 2.0 ** -4 / np.sqrt(128)
    assert reach.max() < 2.0 ** 14
    bad = np.zeros(q.shape, bool)
    spoilt = q.copy()
    for h, x in ((4, np.nan), (7, np.inf), (11, -np.inf)):
        spoilt[n - 1, h, 9 * h] = x
        bad[n - 1, h] = True
    g = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32([L])).double().cpu().numpy()
    check_attn(g, want, mass, reach, dtype, n == 1)
    h = vm.paged_attn(dev(spoilt, dtype), pg.dev, 1, i32(table), i32([L])).double().cpu().numpy()
    assert np.array_equal(np.isnan(h), bad) and np.array_equal(h[~bad], g[~bad])


def test_attention_in_place_strided_shared_and_bounded():
    """q as a slice of a fused projection, a table whose rows lie apart, pages that sequences share, out = q, and bounds on
    the rows of a sequence: looser ones change no row, a tighter one leaves the rows beyond it."""
    log("case: strides, shared pages, in place, bounds")
    rng = np.random.default_rng(515)
    vm = make_vm()
    page, n, kv_len = 32, [5, 33, 1], [70, 100, 1400]
    pg = Pages(rng, 60, 2, page)
    wide = np.stack([rng.permutation(60) for _ in range(3)])
    wide[1, :2] = wide[2, :2] = wide[0, :2]  # a common prefix
    table = i32(wide)[:, :50]
    first = np.concatenate([[0], np.cumsum(n)])
    rows = sum(n)
    qkv = rounded(rng.standard_normal((rows, 16, 128)) * 0.5, "bfloat16")
    fused = dev(qkv, "bfloat16")
    idx = [np.arange(first[b], first[b + 1]) for b in range(3)]
    want, mass, reach = ref.attend(qkv[:, :12], *pg.values(1), wide[:, :50], page, 60, kv_len, idx, 1)
    kw = dict(mask_block=1, row_start=i32(first))
    for bound in (None, 33, 1000):
        g = vm.paged_attn(fused[:, :12], pg.dev, 1, table, i32(kv_len), max_rows=bound, **kw)
        check_attn(g.double().cpu().numpy(), want, mass, reach, "bfloat16", False)
    for max_len in (64, 100000):  # (no second launch; split)
        q = fused[:, :12].clone(memory_format=torch.contiguous_format)
        out = torch.empty_like(q)
        vm.paged_attn(q, pg.dev, 1, table, i32(kv_len), max_len=max_len, out=out, **kw)
        assert vm.paged_attn(q, pg.dev, 1, table, i32(kv_len), max_len=max_len, out=q, **kw) is q
        assert torch.equal(q, out)
    out = torch.full((rows, 12, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    vm.paged_attn(fused[:, :12], pg.dev, 1, table, i32(kv_len), max_rows=4, out=out, **kw)
    g = out.cpu()
    assert (g[[4, *range(9, 38)]] == 9.0).all() and not (g[[0, 3, 5, 8, 38]] == 9.0).any()
    with pytest.raises(ValueError):
        vm.paged_attn(fused[:, :12], pg.dev, 1, table, i32(kv_len), out=fused.flatten()[:rows * 1536].view(rows, 12, 128), **kw)


# ---- together ----------------------------------------------------------------------------------------------


def test_blocks_through_graph_replays_and_back_into_a_contiguous_cache():
    """The run as a program uses it: blocks appended with their norms and rotation, the queries attended over the pages; then the
    same calls captured once and replayed with other lengths and pages on the device, against the eager calls.  At the end one
    sequence is read back into a contiguous 16-bit cache, over which the attention callback attends heads that
    rotate_heads has turned."""
    log("case: append, attend; eager and replayed; read back")
    rng = np.random.default_rng(520)
    vm = make_vm()
    page, nseq, n, width = 32, 3, 32, 8
    pg = Pages(rng, nseq * width + 1, 2, page, garbage=True)
    table_h = tables(rng, nseq, width, nseq * width + 1)
    table, start, kv_len = i32(table_h), i32([0] * nseq), i32([0] * nseq)
    qkv = torch.zeros((nseq * n, 16, 128), dtype=torch.bfloat16, device="cuda")
    w = [dev(rounded(1 + 0.2 * rng.standard_normal(128), "bfloat16"), "bfloat16") for _ in range(2)]
    r = rotary_of(64, True, dict(type="linear", factor=2.0))
    turn = dict(rotary=r, q_norm=w[0], k_norm=w[1])
    back = [torch.zeros((nseq * n, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    def run():
        q = vm.paged4_append(qkv[:, 12:14], qkv[:, 14:], pg.dev, 1, table, start, q=qkv[:, :12], **turn)
        o = vm.paged_attn(q, pg.dev, 1, table, kv_len, mask_block=32)
        return (q, o, *vm.paged4_read(pg.dev, 1, table, start, nseq * n, k_out=back[0], v_out=back[1]),
                *vm.rotate_heads(qkv[:, :12], qkv[:, 12:14], start.repeat_interleave(n), **turn))

    hist = [5 * b for b in range(nseq)]  # (prompts of 0, 5 and 10 tokens: blocks cross pages)
    new = rounded(rng.standard_normal((nseq * 10, 16, 128)), "bfloat16")
    vm.paged4_append(dev(new, "bfloat16")[:, 12:14], dev(new, "bfloat16")[:, 14:], pg.dev, 1, table, i32([0] * nseq), rotary=r, k_norm=w[1])
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    tensors = (pg.dev.k, pg.dev.v, pg.dev.k_scale, pg.dev.v_scale)
    for step in range(6):
        new = rounded(rng.standard_normal((nseq * n, 16, 128)), "bfloat16")
        qkv.copy_(dev(new, "bfloat16"))
        start.copy_(i32(hist))
        kv_len.copy_(i32([s + n for s in hist]))
        keep = [t.clone() for t in tensors]
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in outs]
        pages_r = pg.download()
        for t, o in zip(tensors, keep):
            t.copy_(o)
        eager = run()
        torch.cuda.synchronize()
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b)
        pg.k, pg.v, pg.ke, pg.vs = pg.download()
        assert same(pages_r, (pg.k, pg.v, pg.ke, pg.vs))
        q = eager[0].double().cpu().numpy()
        idx = [np.arange(b * n, (b + 1) * n) for b in range(nseq)]
        hist = [h + n for h in hist]
        want, mass, reach = ref.attend(q, *pg.values(1), table_h, page, nseq * width + 1, hist, idx, 32)
        check_attn(eager[1].double().cpu().numpy(), want, mass, reach, "bfloat16", False)
    # sequence 1 goes on in a contiguous cache, without its last block (whose rows the callback writes)
    b, P = 1, hist[1] - n
    cap = P + n
    kc, vc = (torch.zeros((2, 1, cap, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    vm.paged4_read(pg.dev, 1, table[b:b + 1], i32([0]), P, k_out=kc[1, 0, :P], v_out=vc[1, 0, :P])
    rows = qkv[b * n:(b + 1) * n]
    q, k = vm.rotate_heads(rows[:, :12], rows[:, 12:14], P, **turn)
    assert torch.equal(q, eager[0][b * n:(b + 1) * n])
    _, _, o = vm.attn_inplace(q[None], k[None], rows[None, :, 14:].contiguous(), kc, vc, 1, P, 0, n)
    kd, vd = (t[1, 0].double().cpu().numpy() for t in (kc, vc))
    want, mass, reach = ref.attend(q.double().cpu().numpy(), kd.transpose(1, 0, 2)[None], vd.transpose(1, 0, 2)[None], np.array([[0]]), cap, 1,
                                   [cap], [np.arange(n)], 0)
    check_attn(o[0].double().cpu().numpy(), want, mass, reach, "bfloat16", False)


def test_two_streams_at_once_and_two_graphs():
    """Calls on two streams over different sequences of one cache share no workspace; nor do two graphs of the same calls,
    replayed on two streams at once and between eager calls."""
    log("case: two streams, two graphs")
    rng = np.random.default_rng(521)
    vm = make_vm()
    pg = Pages(rng, 80, 2, 32)
    q = [dev(rng.standard_normal((1, 12, 128)), "bfloat16") for _ in range(2)]
    table = [i32(t[None]) for t in rng.permutation(80).reshape(2, 40)]
    lens, at = [i32([1270]), i32([1111])], [i32([1269]), i32([1110])]
    x = [dev(rng.standard_normal((1, 4, 128)), "bfloat16") for _ in range(2)]

    def run(i):
        turned = vm.paged4_append(x[i][:, :2], x[i][:, 2:], pg.dev, 0, table[i], at[i], q=q[i])
        return turned, vm.paged_attn(turned, pg.dev, 0, table[i], lens[i])

    alone = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for rep in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = run(i)
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    def work(i):  # (a thread for each stream)
        with torch.cuda.stream(streams[i]):
            for rep in range(50):
                got[i] = run(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(i))
    for rep in range(5):
        for i in range(2):
            q[i].copy_(dev(rng.standard_normal((1, 12, 128)), "bfloat16"))
            x[i].copy_(dev(rng.standard_normal((1, 4, 128)), "bfloat16"))
        want = [run(i) for i in range(2)]
        torch.cuda.synchronize()
        for _ in range(4):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_pages_past_four_gigabytes():
    log("case: page offsets of more than 32 bits")
    from fast_dllm_relax_amd.paged4 import allocate_paged4_cache

    rng = np.random.default_rng(522)
    vm = make_vm()
    num = 2 ** 32 // (2 * 128 * 64) + 7
    cache = allocate_paged4_cache(vm.cfg, num, page_size=128)
    ids = [num - 1, 3, num - 5, num - 2]
    n = 400
    qkv = rounded(rng.standard_normal((n, 16, 128)), "bfloat16")
    x = dev(qkv, "bfloat16")
    q = vm.paged4_append(x[:, 12:14], x[:, 14:], cache, 1, i32([ids]), i32([0]), q=x[:, :12])
    out = vm.paged_attn(q, cache, 1, i32([ids]), i32([n]), mask_block=32)
    back = vm.paged4_read(cache, 1, i32([ids]), i32([0]), n)
    code, s = ref.values(qkv[:, 14:])
    at = np.arange(n)
    g = cache.v[1, ids].cpu().numpy()
    assert np.array_equal(ref.unpack(g)[at // 128, :, at % 128], code)
    assert np.array_equal(cache.v_scale[1, ids].double().cpu().numpy()[at // 128, :, at % 128], s)
    assert np.array_equal(back[1].double().cpu().numpy(), rounded(ref.E2M1[code] * s[..., None], "bfloat16"))
    k = ref.E2M1[ref.unpack(cache.k[1, ids].cpu().numpy())] * np.repeat(ref.key_scales(ref.by_slot(cache.k_scale[1, ids].cpu().numpy())), 32, axis=-1)
    assert np.array_equal(back[0].double().cpu().numpy(), rounded(k[at // 128, :, at % 128], "bfloat16"))
    v = ref.E2M1[ref.unpack(g)] * cache.v_scale[1, ids].double().cpu().numpy()[..., None]
    want, mass, reach = ref.attend(q.double().cpu().numpy(), k, v, np.arange(4)[None], 128, 4, [n], [np.arange(n)], 32)
    check_attn(out.double().cpu().numpy(), want, mass, reach, "bfloat16", False)
    # nothing went to the places that the offsets' low 32 bits name
    assert not cache.v[1, [i - 2 ** 32 // (2 * 128 * 64) for i in ids if i > 1000]].any()


def test_the_library_refuses():
    """The C entry points' own checks, one wrong argument at a time; nothing is launched."""
    log("case: refusals of the C entry points")
    from fast_dllm_relax_amd import _lib

    rng = np.random.default_rng(523)
    vm = make_vm()
    lib = vm.lib
    pg = Pages(rng, 4, 2, 32)
    before = pg.download()
    x = dev(rng.standard_normal((4, 16, 128)), "bfloat16")
    table, two = i32([[0, 1], [2, 3]]), i32([0, 0])
    out = torch.full((4, 16, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    at, to = x.data_ptr(), out.data_ptr()
    cache = dict(k=pg.dev.k.data_ptr(), v=pg.dev.v.data_ptr(), ks=pg.dev.k_scale.data_ptr(), vs=pg.dev.v_scale.data_ptr(), pages=4, page=32)

    def struct(**change):
        c = {**cache, **change}
        return ctypes.byref(_lib.FdllmPaged4Cache(c["k"], c["v"], c["ks"], c["vs"], c["pages"], c["page"]))

    freq = (ctypes.c_double * 64)(*[1.0] * 64)
    odd = (ctypes.c_double * 64)(*[float("nan")] * 64)

    def plan(freq=freq, dim=128, inter=0, factor=1.0):
        return ctypes.byref(_lib.FdllmRotary(ctypes.cast(freq, ctypes.POINTER(ctypes.c_double)) if freq else None, dim, inter, factor))

    plans = [dict(rotary=plan(**c)) for c in (dict(freq=None), dict(freq=odd), dict(dim=8), dict(dim=144), dict(dim=-16), dict(inter=2),
                                              dict(factor=float("nan")), dict(factor=1e7))]
    append = dict(q=at, ldq=2048, k=at + 2 * 1536, ldk=2048, v=at + 2 * 1792, ldv=2048, rows=4, row_start=None, nseq=2, max_rows=2,
                  cache=struct(), layer=0, table=table.data_ptr(), width=2, table_ld=2, start=two.data_ptr(), pos=None, rotary=None,
                  q_norm=None, k_norm=None, q_out=to)
    attn = dict(q=at, ldq=2048, rows=4, row_start=None, nseq=2, max_rows=2, cache=struct(), layer=0, table=table.data_ptr(), width=2,
                table_ld=2, kv_len=two.data_ptr(), max_len=0, mask_block=0, out=to, ws=None, bytes=0)
    read = dict(cache=struct(), layer=0, table=table.data_ptr(), width=2, table_ld=2, start=two.data_ptr(), rows=4, row_start=None,
                nseq=2, max_rows=2, k_out=to, ldk=2048, v_out=to + 512, ldv=2048)
    turn = dict(q=at, ldq=2048, k=at + 2 * 1536, ldk=2048, rows=4, pos=None, pos0=0, rotary=None, q_norm=None, k_norm=None, q_out=to,
                ldqo=2048, k_out=to + 2 * 1536, ldko=2048)
    caches = [dict(cache=None), dict(cache=struct(page=24)), dict(cache=struct(page=0)), dict(cache=struct(pages=0)), dict(cache=struct(k=None)),
              dict(cache=struct(vs=None)), *(dict(cache=struct(**{n: cache[n] + 8})) for n in ("k", "v", "ks", "vs")), dict(layer=-1),
              dict(layer=2), dict(table=None), dict(width=0), dict(width=2 ** 31 - 1), dict(table_ld=-1), dict(rows=-1), dict(nseq=0),
              dict(nseq=65536, rows=131072), dict(max_rows=-1), dict(max_rows=3), dict(rows=3),
              dict(rows=2 ** 30, max_rows=2 ** 30, row_start=two.data_ptr(), nseq=4)]
    queries = [dict(q=at + 2), dict(ldq=2044), dict(ldq=1528)]
    refused = lambda fn, args: fn(vm.ctx, *args.values(), None) == _lib.FDLLM_EINVAL  # noqa: E731
    for change in [*caches, *queries, *plans, dict(k=None), dict(v=None), dict(start=None), dict(q=None), dict(q_out=None), dict(k=at + 4),
                   dict(ldk=248), dict(ldv=4), dict(q_out=to + 8), dict(q_out=at), dict(q_norm=at + 2), dict(k_norm=at + 2),
                   dict(q=None, q_out=None, q_norm=at)]:
        assert refused(lib.fdllm_paged4_append, {**append, **change}), change
    for change in [*caches, dict(start=None), dict(k_out=None), dict(v_out=None), dict(k_out=to + 2), dict(ldk=4), dict(ldv=248)]:
        assert refused(lib.fdllm_paged4_read, {**read, **change}), change
    for change in [*plans, *queries, dict(q=None, k=None, q_out=None, k_out=None), dict(q=None), dict(k_out=None), dict(rows=-1), dict(ldqo=1528),
                   dict(ldko=4), dict(k=at + 2), dict(k_norm=at + 2), dict(q=None, q_out=None, q_norm=at), dict(q_out=at, ldqo=1536),
                   dict(pos0=2 ** 31 - 3), dict(pos0=-2 ** 31 - 1)]:
        assert refused(lib.fdllm_rotate_heads, {**turn, **change}), change
    need = lib.fdllm_paged4_attn_workspace(vm.ctx, 4, 2, 2, 32, 1000, 0)
    assert need > 0 and lib.fdllm_paged4_attn_workspace(vm.ctx, 4, 2, 2, 32, 2, 0) == 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    long = dict(width=1000, table_ld=0, ws=ws.data_ptr(), bytes=need)
    for change in [*caches, *queries, dict(q=None), dict(kv_len=None), dict(out=None), dict(out=to + 8), dict(out=at), dict(mask_block=-1),
                   dict(max_len=-1), {**long, "bytes": need - 1}, {**long, "ws": None}, {**long, "ws": ws.data_ptr() + 4}]:
        assert refused(lib.fdllm_paged4_attn, {**attn, **change}), change
    for sizes in ((2 ** 30, 4, 2 ** 30, 32, 1000, 0), (0, 4, 1, 32, 1000, 0), (4, 4, 1, 0, 1000, 0), (4, 4, 1, 128, 2 ** 31 - 1, 0)):
        assert lib.fdllm_paged4_attn_workspace(vm.ctx, *sizes) == 0
    torch.cuda.synchronize()
    assert (out == 9.0).all() and same(pg.download(), before)


def test_the_short_way_is_the_long_one():
    """The calls' way through the extension gives the bits and the errors of the one through the checks in Python, takes nothing
    that those refuse, and is the one that a step's arguments take."""
    log("case: the two ways to the library")
    from fast_dllm_relax_amd import vm as module
    from fast_dllm_relax_amd.paged import allocate_paged_cache

    rng = np.random.default_rng(524)
    vm = make_vm()
    assert module.fdllm_calls is not None and vm._spec is not None
    pg = Pages(rng, 9, 2, 32)
    table, start, pos = i32(np.arange(8).reshape(2, 4)), i32([3, 40]), i32([9, 7])
    x = dev(rng.standard_normal((10, 16, 128)), "bfloat16")
    w = dev(rng.standard_normal(128), "bfloat16")
    q, k, v = x[:, :12], x[:, 12:14], x[:, 14:]
    new = lambda n, rows=10: torch.zeros((rows, n, 128), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    r = rotary_of(64, True)
    at = i32(np.arange(10))
    first = i32([0, 3, 8])
    long = object.__new__(type(vm))
    long.__dict__.update(vm.__dict__, _spec=None)
    took = []

    class Counted:
        def __getattr__(self, name):
            def call(*args):
                rc = getattr(calls, name)(*args)
                took.append(rc)
                return rc
            return call

    calls, module.fdllm_calls = module.fdllm_calls, Counted()
    eight = allocate_paged_cache(vm.cfg, 9)
    lens = i32([100, 77])
    try:
        good = [
            lambda m: (m.paged_attn(q, pg.dev, 1, table, lens, mask_block=1, out=new(12)),),
            lambda m: (m.paged_attn(q, pg.dev, 0, table, lens, row_start=first, max_rows=5, max_len=100, out=new(12)),),
            lambda m: (m.paged_attn(q[:1], pg.dev, 0, i32(np.arange(4000).reshape(1, -1) % 9), i32([100000]), out=new(12, 1)),),
            lambda m: (m.paged_attn(q, eight, 1, table, lens, out=new(12)),),
            lambda m: m.rotate_heads(q, k, at, rotary=r, q_norm=w, q_out=new(12), k_out=new(2)),
            lambda m: m.rotate_heads(q[:1], k[:1], at[:1], q_out=new(12, 1), k_out=new(2, 1), k_norm=w),
            lambda m: (m.paged4_append(k, v, pg.dev, 1, table, start, q=q, q_out=new(12), rotary=r, q_norm=w, k_norm=w, pos=pos), *pg.download()),
            lambda m: (m.paged4_append(k, v, pg.dev, 0, table, start, q=q, q_out=new(12), row_start=first, max_rows=5), *pg.download()),
            lambda m: (m.paged4_append(k, v, pg.dev, 0, table, start, q=q, q_out=new(12), row_start=first), *pg.download()),
            lambda m: m.paged4_read(pg.dev, 1, table, start, 10, k_out=new(2), v_out=new(2), max_rows=5),
            lambda m: m.paged4_read(pg.dev, 0, table, start, 10, k_out=new(2), v_out=new(2), row_start=first, max_rows=99),
        ]
        for i, f in enumerate(good):
            took.clear()
            a, b = f(vm), f(long)
            assert took == [0], i
            for p, s in zip(a, b):
                assert np.array_equal(p, s, equal_nan=p.dtype.kind == "f") if isinstance(p, np.ndarray) else torch.equal(p, s)
        cpu = torch.zeros(10, dtype=torch.int32)
        ok_r = dict(q=q, k=k, pos=at, q_out=new(12), k_out=new(2))
        ok_a = dict(k=k, v=v, cache=pg.dev, layer=1, page_table=table, start=start, q=q, q_out=new(12))
        ok_d = dict(cache=pg.dev, layer=1, page_table=table, start=start, rows=10, k_out=new(2), v_out=new(2))
        before = pg.download()
        bad = [("rotate_heads", {**ok_r, **c}) for c in
               (dict(q=q[:9]), dict(k=x[:, :3]), dict(pos=at[:4]), dict(pos=cpu), dict(pos=at.long()), dict(q_norm=w[:64]), dict(q_norm=w.half()),
                dict(k_norm=w.float()), dict(q_out=new(12, 9)), dict(q_out=q.half()), dict(k_out=k.cpu()), dict(rotary=5),
                dict(q=x[:, :, ::2][:, :12]), dict(q_out=new(12).transpose(0, 1).contiguous().transpose(0, 1)),
                dict(k=x[:, 12:14].flatten(1)))]
        bad += [("paged4_append", {**ok_a, **c}) for c in
                (dict(k=k[:9]), dict(v=v[:, :1]), dict(layer=2), dict(layer=-1), dict(page_table=table.t()), dict(page_table=table.long()),
                 dict(start=start[:1]), dict(pos=at), dict(q=q[:4]), dict(q_out=new(24)[:, ::2]), dict(q_out=new(12, 20)[::2]), dict(q_norm=at),
                 dict(row_start=first[:2]), dict(max_rows=4), dict(max_rows=-1, row_start=first), dict(k=q[:, :2], v=None),
                 dict(cache=None), dict(q_out=x.flatten()[:10 * 12 * 128].view(10, 12, 128), q=q))]
        bad += [("paged4_read", {**ok_d, **c}) for c in
                (dict(rows=9), dict(rows=11), dict(rows=-10), dict(rows=2 ** 31), dict(layer=7), dict(start=at), dict(k_out=new(2, 9)), dict(v_out=new(3)),
                 dict(max_rows=3), dict(page_table=table[0]), dict(v_out=new(2).half()), dict(row_start=at, max_rows=5))]
        ok_t = dict(q=q, cache=pg.dev, layer=1, page_table=table, kv_len=lens, out=new(12))
        bad += [("paged_attn", {**ok_t, **c}) for c in
                (dict(q=x[:, :11]), dict(layer=2), dict(layer=-1), dict(kv_len=at), dict(kv_len=lens.long()), dict(mask_block=-1),
                 dict(mask_block=2 ** 31), dict(max_len=-1), dict(out=new(12, 9)), dict(out=new(24)[:, ::2]), dict(max_rows=4), dict(row_start=first[:2]),
                 dict(out=x.flatten()[:10 * 12 * 128].view(10, 12, 128)), dict(page_table=table.t()), dict(q=q.cpu()))]
        for name, kw in bad:
            took.clear()
            errors = []
            for m in (vm, long):
                with pytest.raises((ValueError, TypeError, AttributeError)) as e:
                    getattr(m, name)(**kw)
                errors.append((e.type, str(e.value)))
            assert errors[0] == errors[1] and 0 not in took, (name, errors)
        torch.cuda.synchronize()
        assert same(before, pg.download())
    finally:
        module.fdllm_calls = calls
        long.ctx = None  # (the context is vm's)
