"""The paged 8-bit cache (HipVM.paged_kv_append, HipVM.paged_attn) and HipVM.token_logprobs against their definitions
in 64 bits (tests/paged_reference.py), at the sizes, masks and values where they can go wrong."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import paged_reference as ref
from helpers import log

pytestmark = pytest.mark.gpu

TD = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
HALF = {t: torch.finfo(d).eps / 2 for t, d in TD.items()}  # a rounding's largest relative error
THETA = 1e6
_VMS = {}


def make_vm(dtype="bfloat16", nq=12, nkv=2, layers=2):
    from fast_dllm_relax_amd.config import FastDLLMConfig
    from fast_dllm_relax_amd.params import param_names, param_shapes
    from fast_dllm_relax_amd.vm import HipVM

    key = (dtype, nq, nkv, layers)
    if key not in _VMS:
        cfg = FastDLLMConfig(vocab_size=256, hidden_size=128, intermediate_size=128, num_hidden_layers=layers,
                             num_attention_heads=nq, num_key_value_heads=nkv, head_dim=128, rope_theta=THETA)
        shapes = param_shapes(cfg)
        _VMS[key] = HipVM(cfg, [torch.zeros(shapes[n], dtype=TD[dtype], device="cuda") for n in param_names(cfg)], dtype=dtype)
    return _VMS[key]


def rounded(a, dtype):
    """a as values of dtype, in 64 bits."""
    return torch.from_numpy(np.asarray(a, np.float32)).to(TD[dtype]).double().numpy()


def dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to("cuda", TD[dtype])


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


class Pages:
    """A cache of two layers, with its bytes and scales on the host: K and V both [pages, heads, page, 128]."""

    def __init__(self, rng, pages, nkv, page, fill=None):
        from fast_dllm_relax_amd.paged import PagedKVCache

        shape = (2, pages, nkv, page, 128)
        # any byte but NaN, or one byte everywhere
        make = lambda: (rng.integers(0, 126, shape) | (rng.integers(0, 2, shape) << 7)).astype(np.uint8)  # noqa: E731
        self.k, self.v = (make(), make()) if fill is None else (np.full(shape, fill, np.uint8), np.full(shape, fill, np.uint8))
        self.ks, self.vs = (2.0 ** rng.integers(-9, -6, shape[:3]) for _ in range(2))
        self.page, self.cache = page, PagedKVCache
        self.upload()

    def upload(self):
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
        fp8 = torch.float8_e4m3fn
        self.dev = self.cache(k=t(self.k).view(fp8), v=t(self.v.transpose(0, 1, 2, 4, 3)).view(fp8),
                              k_scale=t(self.ks.astype(np.float32)), v_scale=t(self.vs.astype(np.float32)))

    def download(self):
        g = lambda x: x.view(torch.uint8).cpu().numpy()  # noqa: E731
        return (g(self.dev.k), np.ascontiguousarray(g(self.dev.v).transpose(0, 1, 2, 4, 3)),
                self.dev.k_scale.cpu().numpy().astype(np.float64), self.dev.v_scale.cpu().numpy().astype(np.float64))


def tables(rng, nseq, width, pages):
    return rng.permutation(pages)[:nseq * width].reshape(nseq, width)


def same_bytes(a, b):
    """Equal bytes, any NaN like another."""
    return np.array_equal(np.where((a & 127) == 127, 127, a), np.where((b & 127) == 127, 127, b))


def near_bytes(got, want, scale, exact, err):
    """got holds the e4m3 value nearest to exact / scale, or one that an error of err in exact explains."""
    v = ref.E4M3[got] * scale
    room = ref.step(np.abs(exact / scale) + err / scale) * scale / 2 + err
    return bool(np.all((got == want) | (np.abs(v - exact) <= room)))


APPENDS = [
    # dtype, nq, nkv, page, rows per sequence, start, live (None: start), pos (None: start)
    ("bfloat16", 12, 2, 32, [1], [2079], None, None),                    # one token, the last slot of a page
    ("bfloat16", 12, 2, 32, [1, 1, 1], [0, 31, 32], None, None),         # first and last slots
    ("float16", 12, 2, 32, [8, 8], [136, 40], [160, 64], None),          # inside blocks that are live
    ("bfloat16", 4, 2, 16, [37, 0, 5], [11, 3, 0], None, [100000, 0, 31000]),  # a ragged batch with an empty sequence
    ("float16", 8, 8, 64, [130, 64], [1, 64], None, None),               # more pages than one, a page exactly
    ("bfloat16", 16, 1, 128, [128, 300, 1], [0, 127, 500], [0, 400, 501], None),
    ("bfloat16", 12, 2, 32, [32, 32], [-1, 0], None, None),              # a negative start: skipped
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append(case):
    dtype, nq, nkv, page, n, start, live, pos = APPENDS[case]
    log(f"case: append {APPENDS[case]}")
    rng = np.random.default_rng(100 + case)
    vm = make_vm(dtype, nq, nkv)
    nseq, width = len(n), (max(s + k for s, k in zip(start, n)) + page - 1) // page + 1
    pg = Pages(rng, nseq * width + 2, nkv, page)
    table = tables(rng, nseq, width, nseq * width + 2)
    rows = sum(n)
    uniform = len(set(n)) == 1
    total = rows if uniform else rows + 2
    amp = np.exp(rng.standard_normal((total, 1, 1)))
    qkv = rounded(rng.standard_normal((total, nq + 2 * nkv, 128)) * amp, dtype)
    fused = dev(qkv, dtype)
    q, k, v = fused[:, :nq], fused[:, nq:nq + nkv], fused[:, nq + nkv:]
    q_out = torch.full((total, nq, 128), 7.0, dtype=TD[dtype], device="cuda")
    first = np.concatenate([[0], np.cumsum(n)])
    got_q = vm.paged_kv_append(k, v, pg.dev, 1, i32(table), i32(start), live=None if live is None else i32(live),
                               pos=None if pos is None else i32(pos), q=q, q_out=q_out,
                               row_start=None if uniform else i32(first), max_rows=None if uniform else max(n))
    assert got_q is q_out
    gk, gv, gks, gvs = pg.download()
    live = start if live is None else live
    pos = start if pos is None else pos
    knew = [np.stack([ref.rotate(qkv[first[b] + i, nq:nq + nkv], pos[b] + i, THETA) for i in range(n[b])])
            if n[b] else np.zeros((0, nkv, 128)) for b in range(nseq)]
    vnew = [qkv[first[b]:first[b] + n[b], nq + nkv:] for b in range(nseq)]
    wk, wv, wks, wvs = pg.k.copy(), pg.v.copy(), pg.ks.copy(), pg.vs.copy()
    ref.append(wk[1], wks[1], table, page, start, live, knew)
    ref.append(wv[1], wvs[1], table, page, start, live, vnew)
    # scales are powers of two and values are exact before their one rounding: V has the definition's bytes.  K's
    # rotation is fp32: two products and a sum of values of size |x| + |y|, sine and cosine to 2^-22 (angles reduced in
    # 64 bits), so within 2^-21 (|x| + |y|) of the exact value.
    assert np.array_equal(gvs, wvs) and np.array_equal(gks, wks)
    assert np.array_equal(gv, wv)
    assert np.array_equal(gk[0], wk[0])  # the other layer
    diff = gk[1] != wk[1]
    log(f"  K bytes on the other side of a rounding: {int(diff.sum())} of {diff.size}")
    for b in range(nseq):
        for i in range(n[b]):
            if start[b] < 0:
                continue
            p = start[b] + i
            x = np.abs(qkv[first[b] + i, nq:nq + nkv])
            err = 2.0 ** -21 * np.tile(x[:, :64] + x[:, 64:], 2)
            at = table[b, p // page], slice(None), p % page
            assert near_bytes(gk[1][at], wk[1][at], wks[1][at[0]][:, None], knew[b][i], err)
            diff[at] = False
    assert not diff.any()  # rows that stay and pages of no sequence: byte for byte
    got_q = q_out.double().cpu().numpy()
    for b in range(nseq):
        for i in range(n[b]):
            r = first[b] + i
            if start[b] < 0:
                assert (got_q[r] == 7.0).all()
                continue
            want = ref.rotate(qkv[r, :nq], pos[b] + i, THETA)
            x = np.abs(qkv[r, :nq])
            assert (np.abs(got_q[r] - want) <= HALF[dtype] * np.abs(want) + 2.0 ** -21 * np.tile(x[..., :64] + x[..., 64:], 2) + 2.0 ** -25).all()
    assert (got_q[rows:] == 7.0).all()  # rows behind the last sequence


@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_append_grows_and_keeps_scales(page):
    """Tokens one by one, each larger than the last, then small ones: the page's rows are encoded again while the scale
    grows and stay when it does not; a page that is written whole starts anew."""
    log(f"case: growing scales, pages of {page}")
    rng = np.random.default_rng(7)
    vm = make_vm()
    pg = Pages(rng, 4, 2, page)
    table = np.array([[2, 0]])
    wk, wv, wks, wvs = pg.k.copy(), pg.v.copy(), pg.ks.copy(), pg.vs.copy()
    for p in range(page + 3):
        amp = 2.0 ** (p if p < 9 else 0)
        kv = rounded(rng.standard_normal((2, 1, 2, 128)) * amp, "bfloat16")
        vm.paged_kv_append(dev(kv[0], "bfloat16"), dev(kv[1], "bfloat16"), pg.dev, 0, i32(table), i32([p]), pos=i32([0]))
        for pages, scale, x in ((wk, wks, kv[0]), (wv, wvs, kv[1])):
            ref.append(pages[0], scale[0], table, page, [p], [p], [x])
    gk, gv, gks, gvs = pg.download()
    assert np.array_equal(gks, wks) and np.array_equal(gvs, wvs)
    assert np.array_equal(gv, wv) and np.array_equal(gk, wk)  # (position 0 turns nothing)


def test_append_values_that_are_not_finite_and_zeros():
    log("case: NaN, infinities, zeros and subnormals")
    rng = np.random.default_rng(8)
    vm = make_vm()
    pg = Pages(rng, 3, 2, 32)
    kv = rounded(rng.standard_normal((2, 32, 2, 128)), "bfloat16")
    kv[1, 3, 0, 5], kv[1, 4, 0, 6], kv[1, 9, 1, 7] = np.nan, np.inf, -np.inf
    kv[0, :, 1] = 0.0  # a head of zeros
    kv[1, 11, 1] = rounded(kv[1, 11, 1] * 2.0 ** -12, "bfloat16")  # under e4m3's normal range
    wk, wv, wks, wvs = pg.k.copy(), pg.v.copy(), pg.ks.copy(), pg.vs.copy()
    vm.paged_kv_append(dev(kv[0], "bfloat16"), dev(kv[1], "bfloat16"), pg.dev, 0, i32([[1]]), i32([0]), pos=i32([0]))
    table = np.array([[1]])
    ref.append(wv[0], wvs[0], table, 32, [0], [0], [kv[1]])
    gk, gv, gks, gvs = pg.download()
    assert np.array_equal(gvs, wvs) and same_bytes(gv, wv)
    assert (gk[0, 1, 1] & 127 == 0).all() and gks[0, 1, 1] == 2.0 ** -100


def test_append_bad_pages_write_nothing():
    log("case: page numbers out of range, positions past the table")
    rng = np.random.default_rng(9)
    vm = make_vm()
    pg = Pages(rng, 4, 2, 32)
    kv = dev(rng.standard_normal((2, 3 * 40, 2, 128)), "bfloat16")
    table = np.array([[-1, 4], [2 ** 30, 1], [-2 ** 31, 2 ** 31 - 1]])
    before = pg.download()
    vm.paged_kv_append(kv[0], kv[1], pg.dev, 1, i32(table), i32([0, 40, 2 ** 31 - 20]))
    after = pg.download()
    # sequence 1's rows 40 .. 63 go to page 1; 64 .. 79 lie past its table
    for x, y in zip(before, after):
        assert np.array_equal(x[0], y[0]) and np.array_equal(x[1, [0, 2, 3]], y[1, [0, 2, 3]])
    assert not np.array_equal(before[1][1, 1, :, 8:], after[1][1, 1, :, 8:])


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
]


def check_attn(got, want, mass, reach, dtype):
    """P is rounded once to the model dtype and the result once: each off by at most half a step.  The scores' fp32 sums
    of 128 products are off by less than 2^-17 of the sum of their sizes, and exp turns that into a relative error of p
    (and of the sum that divides it); fp16's least step adds 2^-25 per key."""
    u = HALF[dtype]
    room = mass * (2 * u + 2 * reach[..., None] * 2.0 ** -17 + 2.0 ** -16) + (2.0 ** -14 if dtype == "float16" else 2.0 ** -100)
    worst = float(np.max(np.abs(got - want) / room)) if got.size else 0.0
    log(f"  largest error {worst:.3f} of its bound")
    assert np.isfinite(got).all() and worst <= 1.0


@pytest.mark.parametrize("case", range(len(ATTNS)))
def test_attention(case):
    dtype, nq, nkv, page, n, kv_len, mask = ATTNS[case]
    log(f"case: attention {ATTNS[case]}")
    rng = np.random.default_rng(200 + case)
    vm = make_vm(dtype, nq, nkv)
    nseq, width = len(n), max(1, (max(kv_len) + page - 1) // page)
    pg = Pages(rng, nseq * width + 1, nkv, page)
    # scales as the append leaves them (values of size 1), and one tensor's that are no powers of two
    pg.vs *= rng.uniform(0.6, 1.9, pg.vs.shape)
    pg.ks = pg.ks.astype(np.float32).astype(np.float64)
    pg.vs = pg.vs.astype(np.float32).astype(np.float64)
    table = tables(rng, nseq, width, nseq * width + 1)
    # what lies behind the sequences' ends is NaN
    for b in range(nseq):
        for p in range(max(0, kv_len[b]), width * page):
            pg.k[:, table[b, p // page], :, p % page] = 127
            pg.v[:, table[b, p // page], :, p % page] = 255
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
    want, mass, reach = ref.attend(q, pg.k[1], pg.ks[1], pg.v[1], pg.vs[1], table, page, kv_len, idx, mask)
    g = out.double().cpu().numpy()
    assert (g[rows:] == 9.0).all()
    check_attn(g[:rows], want[:rows], mass[:rows], reach[:rows], dtype)
    # rows without a key are zeros
    assert (g[:rows][mass[:rows].sum(axis=-1) == 0] == 0).all()
    # the same call again, planned for a bound: the split differs, the bits of one plan do not
    again = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32(kv_len), mask_block=mask, out=torch.full_like(out, 9.0), **kw)
    assert torch.equal(again.view(torch.int16), out.view(torch.int16))
    short = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32(kv_len), mask_block=mask, max_len=1,
                          out=torch.full_like(out, 9.0), **kw)
    check_attn(short.double().cpu().numpy()[:rows], want[:rows], mass[:rows], reach[:rows], dtype)


@pytest.mark.parametrize("mask", [1, 32])
def test_attention_nan_behind_the_mask(mask):
    """Keys that a row does not attend may hold NaN: rows in front of it are as without it, rows that see it are NaN in
    its dims (V) or throughout (K)."""
    log(f"case: NaN behind a mask of {mask}")
    rng = np.random.default_rng(11)
    vm = make_vm()
    page, L, n = 32, 230, 100  # positions 130 .. 229
    pg = Pages(rng, 9, 2, page)
    table = tables(rng, 1, 8, 9)
    q = rounded(rng.standard_normal((n, 12, 128)) * 0.5, "bfloat16")
    idx = [np.arange(n)]
    want, mass, reach = ref.attend(q, pg.k[1], pg.ks[1], pg.v[1], pg.vs[1], table, page, [L], idx, mask)
    at_v, at_k = 200, 215
    pg.v[1, table[0, at_v // page], 0, at_v % page, 17] = 127
    pg.k[1, table[0, at_k // page], 1, at_k % page, 3] = 255
    pg.upload()
    g = vm.paged_attn(dev(q, "bfloat16"), pg.dev, 1, i32(table), i32([L]), mask_block=mask).double().cpu().numpy()
    pos = np.arange(130, 230)
    sees = lambda p: (pos // mask + 1) * mask > p  # noqa: E731
    bad = np.zeros(g.shape, bool)
    bad[sees(at_v), :6, 17] = True
    bad[sees(at_k), 6:] = True
    assert np.isnan(g[bad]).all()
    fine = np.where(bad, want, g)
    check_attn(fine, want, mass, reach, "bfloat16")


def test_attention_pages_that_are_none():
    log("case: page numbers out of range inside the length, a length past the table")
    rng = np.random.default_rng(12)
    vm = make_vm()
    page = 32
    pg = Pages(rng, 6, 2, page)
    table = np.array([[3, -1, 5, 6], [2 ** 31 - 1, 0, -7, 2]])
    q = rounded(rng.standard_normal((2, 12, 128)) * 0.5, "bfloat16")
    kv_len = [120, 2 ** 31 - 1]
    want, mass, reach = ref.attend(q, pg.k[0], pg.ks[0], pg.v[0], pg.vs[0], table, page, kv_len, [[0], [1]], 0)
    g = vm.paged_attn(dev(q, "bfloat16"), pg.dev, 0, i32(table), i32(kv_len))
    check_attn(g.double().cpu().numpy(), want, mass, reach, "bfloat16")


LOGPROBS = [
    # rows, vocab, top, dtype, extra columns (row stride), offset in elements
    (1, 1, 1, "float32", 0, 0),
    (3, 7, 7, "bfloat16", 0, 0),
    (2, 33, 32, "float16", 3, 1),
    (5, 1000, 5, "float32", 0, 0),
    (4, 4099, 20, "bfloat16", 5, 3),
    (3, 5000, 0, "float32", 1, 2),
    (64, 12345, 3, "float32", 0, 1),
    (2, 151936, 20, "float32", 0, 0),
    (9, 151643, 32, "bfloat16", 0, 0),
    (1200, 2049, 10, "float16", 0, 0),
]


def check_logprobs(got, x, ids, top):
    """Sums of up to n terms in a row, n = vocab over a wave's lanes and the waves of its splits (at least one wave takes
    1024 elements an iteration): relative error n 2^-24 and a few roundings of exp and log; the differences to the
    largest logit are exact to 2^-24 of their size."""
    lp, ent, ids_t, best = (None if t is None else t[0].double().cpu().numpy() for t in got)
    wlp, went, worder, wbest = ref.logprobs(x, ids, top)
    assert np.array_equal(ids_t, worder)
    n = x.shape[1] / 256 + 64
    rel = n * 2.0 ** -24 + 2.0 ** -20
    with np.errstate(all="ignore"):
        fin = np.isfinite(x)
        spread = np.maximum(np.where(fin, x, -np.inf).max(axis=1) - np.where(fin, x, np.inf).min(axis=1), 0)

    def near(g, w, room):
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(np.isinf(g), np.isinf(w))
        f = np.isfinite(w)
        assert (g[~f & ~np.isnan(w)] == w[~f & ~np.isnan(w)]).all()
        assert (np.abs(g[f] - w[f]) <= np.broadcast_to(room, w.shape)[f]).all(), float(np.max(np.abs(g[f] - w[f])))

    if ids is not None:
        near(lp, wlp, rel + 2.0 ** -22 * (np.abs(np.nan_to_num(wlp, posinf=0, neginf=0)) + 16))
    near(best, wbest, rel + 2.0 ** -22 * (np.abs(np.nan_to_num(wbest, posinf=0, neginf=0)) + 16))
    # entropy = log s - u / s: u is a sum of e d, |d| up to the spread where e matters (e d >= -1 / e each)
    near(ent, went, rel * (4 + 2 * np.minimum(spread, 16)) + 2.0 ** -20)


@pytest.mark.parametrize("case", range(len(LOGPROBS)))
def test_logprobs(case):
    rows, vocab, top, dtype, extra, offset = LOGPROBS[case]
    log(f"case: logprobs {LOGPROBS[case]}")
    rng = np.random.default_rng(300 + case)
    vm = make_vm()
    x = rounded(rounded(rng.standard_normal((rows, vocab)) * 3, "bfloat16"), dtype)
    x[:, rng.integers(0, vocab, vocab // 50)] = -np.inf if vocab > 50 else 0.5
    ids = rng.integers(0, vocab, rows)
    ids[1::3] = -1
    if rows > 2:
        ids[2] = vocab
    buf = torch.full((rows * (vocab + extra) + offset,), float("nan"), dtype=TD[dtype], device="cuda")
    view = buf[offset:].view(1, rows, vocab + extra)[:, :, :vocab]
    view.copy_(torch.from_numpy(x.astype(np.float32)).to(TD[dtype])[None])
    got = vm.token_logprobs(view, i32(ids)[None], top_n=top)
    check_logprobs(got, x, ids, top)
    none = vm.token_logprobs(view, top_n=0)
    assert none[0] is None and none[2].shape == (1, rows, 0)
    # (the plan may differ with the number of alternatives only in the workspace)
    check_logprobs((None, none[1], none[2], none[3]), x, None, 0)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows", [1, 700])
def test_logprobs_rows_that_are_hard(rows, dtype):
    """Rows of one value, of nothing, ascending (every element beats the best so far), descending, with the type's lowest
    value as a mask, with fewer tokens than alternatives, with NaN and infinities; in one row and in many at once."""
    log(f"case: hard rows, {rows} of {dtype}")
    vm = make_vm()
    vocab, top = 9001, 20
    low = float(torch.finfo(TD[dtype]).min)
    ramp = rounded(np.linspace(-9, 9, vocab), dtype)
    base = np.stack([np.full(vocab, 0.25), np.full(vocab, -np.inf), ramp, ramp[::-1], np.full(vocab, low), np.full(vocab, -np.inf),
                     ramp.copy(), ramp.copy(), ramp.copy(), np.full(vocab, low), np.zeros(vocab), ramp * 2000])
    base[5, [17, 4000, 8999]] = [1.0, 2.0, 1.0]
    base[6, 77] = np.nan
    base[7, 4321] = np.inf
    base[8, ::2] = -np.inf
    base[9, [5, 6000]] = [0.5, -3.0]
    base[10, ::3] = -0.0
    base = rounded(base, dtype)
    for r0 in range(0, len(base) if rows == 1 else 1, 1):
        x = base[r0:r0 + 1] if rows == 1 else np.tile(base, (rows // len(base) + 1, 1))[:rows]
        ids = np.full(len(x), 4000)
        got = vm.token_logprobs(dev(x, dtype)[None], i32(ids)[None], top_n=top)
        if rows == 1:
            check_logprobs(got, x, ids, top)
        else:
            uniq = [t[:, :len(base)] for t in got]
            check_logprobs(uniq, x[:len(base)], ids[:len(base)], top)
            # the other copies of each row: the same bits where they lie alike in their 16 bytes (rows of an odd vocabulary
            # start anywhere; what comes before the first whole 16 bytes is summed apart): 24 = lcm(12 rows, 8 places)
            for t in got:
                t = t[0].reshape(rows, -1).view(torch.int32)
                assert torch.equal(t, t[:24].repeat(rows // 24 + 1, 1)[:rows])


def test_a_block_appended_attended_and_scored_through_graph_replays():
    """The run as a program uses it: a prompt and blocks appended with their rotation, the rotated queries attended over
    the pages, and the scored rows' log probabilities; then the same calls captured once and replayed with other
    lengths and pages on the device, against the eager calls."""
    log("case: append, attend, score; eager and replayed")
    rng = np.random.default_rng(13)
    vm = make_vm()
    page, nseq, n, width = 32, 3, 32, 8
    pg = Pages(rng, nseq * width + 1, 2, page, fill=127)
    table_h = tables(rng, nseq, width, nseq * width + 1)
    table, start, kv_len = i32(table_h), i32([0] * nseq), i32([0] * nseq)
    qkv = torch.zeros((nseq * n, 16, 128), dtype=torch.bfloat16, device="cuda")
    logits = torch.zeros((1, nseq * n, 5001), dtype=torch.float32, device="cuda")
    ids = torch.zeros((1, nseq * n), dtype=torch.int32, device="cuda")

    def run():
        q = vm.paged_kv_append(qkv[:, 12:14], qkv[:, 14:], pg.dev, 1, table, start, q=qkv[:, :12])
        o = vm.paged_attn(q, pg.dev, 1, table, kv_len, mask_block=32)
        return (q, o, *vm.token_logprobs(logits, ids, top_n=4))

    hist = [[0] * (5 * b) for b in range(nseq)]  # (prompts of 0, 5 and 10 tokens: blocks cross pages)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    for step in range(6):
        new = rounded(rng.standard_normal((nseq * n, 16, 128)), "bfloat16")
        qkv.copy_(dev(new, "bfloat16"))
        lg = rounded(rng.standard_normal((nseq * n, 5001)), "bfloat16")
        logits.copy_(dev(lg, "float32")[None])
        idh = rng.integers(0, 5001, nseq * n)
        ids.copy_(i32(idh)[None])
        starts = [len(h) for h in hist]
        start.copy_(i32(starts))
        kv_len.copy_(i32([s + n for s in starts]))
        keep = [t.clone() for t in (pg.dev.k, pg.dev.v, pg.dev.k_scale, pg.dev.v_scale)]
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in outs]
        pages_r = pg.download()
        for t, o in zip((pg.dev.k, pg.dev.v, pg.dev.k_scale, pg.dev.v_scale), keep):
            t.view(torch.uint8).copy_(o.view(torch.uint8))
        eager = run()
        torch.cuda.synchronize()
        for a, b in zip(replayed, eager):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        for a, b in zip(pages_r, pg.download()):
            assert np.array_equal(a, b)
        for b in range(nseq):
            hist[b] += [0] * n
        # against the definition, from the bytes in the pages
        gk, gv, gks, gvs = pg.download()
        q = eager[0].double().cpu().numpy()
        idx = [np.arange(b * n, (b + 1) * n) for b in range(nseq)]
        want, mass, reach = ref.attend(q, gk[1], gks[1], gv[1], gvs[1], table_h, page, [len(h) for h in hist], idx, 32)
        check_attn(eager[1].double().cpu().numpy(), want, mass, reach, "bfloat16")
        check_logprobs(eager[2:], lg, idh, 4)


def test_two_streams_at_once():
    """Calls on two streams over different sequences of one cache share no workspace."""
    log("case: two streams")
    rng = np.random.default_rng(14)
    vm = make_vm()
    pg = Pages(rng, 40, 2, 32)
    q = [dev(rng.standard_normal((1, 12, 128)), "bfloat16") for _ in range(2)]
    table = [i32(rng.permutation(40)[None, :40]) for _ in range(2)]
    lens = [i32([1270]), i32([1111])]
    x = [dev(rng.standard_normal((1, 3, 60000)), "float32") for _ in range(2)]
    alone = [(vm.paged_attn(q[i], pg.dev, 0, table[i], lens[i]), *vm.token_logprobs(x[i], top_n=9)[1:]) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for rep in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i] = (vm.paged_attn(q[i], pg.dev, 0, table[i], lens[i]), *vm.token_logprobs(x[i], top_n=9)[1:])
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in zip(alone[i], got[i]):
            assert torch.equal(a, b)


def test_attention_many_keys_of_small_probability():
    """One key with e^18 times the weight of each of 131071 others, which hold the values: each of theirs is under fp16's
    least step beside 1, all together are 2^-9.5."""
    log("case: many small probabilities in fp16")
    vm = make_vm("float16")
    width = 1024
    rng = np.random.default_rng(15)
    pg = Pages(rng, width, 2, 128, fill=0)
    one, c = int(ref.encode(1.0)), int(ref.encode(1.625))
    table = tables(rng, 1, width, width)
    pg.v[1] = one
    pg.ks[1] = pg.vs[1] = 1.0
    pg.k[1, table[0, 0], :, 5], pg.v[1, table[0, 0], :, 5] = c, 0
    pg.upload()
    q = np.ones((1, 12, 128))
    want, mass, reach = ref.attend(q, pg.k[1], pg.ks[1], pg.v[1], pg.vs[1], table, 128, [width * 128], [[0]], 0)
    assert 2.0 ** -10 < want.min() <= want.max() < 2.0 ** -9
    got = vm.paged_attn(dev(q, "float16"), pg.dev, 1, i32(table), i32([width * 128])).double().cpu().numpy()
    check_attn(got, want, mass, reach, "float16")
    # (whose absolute part is for values at fp16's least step: here the relative one alone holds)
    assert (np.abs(got / want - 1) <= 2 * HALF["float16"] + 2.0 ** -12).all()


def test_attention_in_place_and_strided():
    """q as a slice of a fused projection, a table whose rows lie apart, pages that sequences share, out = q, and bounds on
    the rows of a sequence: looser ones change no row, a tighter one leaves the rows beyond it."""
    log("case: strides, shared pages, in place, bounds")
    rng = np.random.default_rng(16)
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
    want, mass, reach = ref.attend(qkv[:, :12], pg.k[1], pg.ks[1], pg.v[1], pg.vs[1], wide[:, :50], page, kv_len, idx, 1)
    kw = dict(mask_block=1, row_start=i32(first))
    for bound in (None, 33, 1000):
        g = vm.paged_attn(fused[:, :12], pg.dev, 1, table, i32(kv_len), max_rows=bound, **kw)
        check_attn(g.double().cpu().numpy(), want, mass, reach, "bfloat16")
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
    # one row whose tensor has another stride, and sequences with one row of a table
    q1 = fused[:1, :12].clone(memory_format=torch.contiguous_format).reshape(12, 1, 128).transpose(0, 1)
    want, mass, reach = ref.attend(qkv[:1, :12], pg.k[1], pg.ks[1], pg.v[1], pg.vs[1], wide[:1], page, [99], [[0]], 0)
    check_attn(vm.paged_attn(q1, pg.dev, 1, table[:1], i32([99])).double().cpu().numpy(), want, mass, reach, "bfloat16")
    same = vm.paged_attn(fused[:2, :12], pg.dev, 1, table[:1].expand(2, 50), i32([99, 99]))
    check_attn(same[:1].double().cpu().numpy(), want, mass, reach, "bfloat16")


@pytest.mark.parametrize("nq,nkv,n", [(12, 2, 9), (16, 1, 9), (12, 2, 2)])
def test_attention_nan_behind_the_mask_of_a_long_sequence(nq, nkv, n):
    """As above over key ranges that several workgroups share, with 16 rows or fewer to a tile and with more."""
    log(f"case: NaN behind the mask, split, {nq} heads, {n} rows")
    rng = np.random.default_rng(17)
    vm = make_vm("bfloat16", nq, nkv)
    page, L = 64, 3000
    at = L - n + n // 2
    pg = Pages(rng, 50, nkv, page)
    table = tables(rng, 1, 48, 50)
    q = rounded(rng.standard_normal((n, nq, 128)) * 0.5, "bfloat16")
    want, mass, reach = ref.attend(q, pg.k[1], pg.ks[1], pg.v[1], pg.vs[1], table, page, [L], [np.arange(n)], 1)
    for p, byte in ((at, 127), (3000, 127), (3005, 255)):
        pg.v[1, table[0, p // page], 0, p % page, 99] = byte
        if p >= L:
            pg.k[1, table[0, p // page], :, p % page] = byte
    pg.upload()
    g = vm.paged_attn(dev(q, "bfloat16"), pg.dev, 1, i32(table), i32([L]), mask_block=1).double().cpu().numpy()
    bad = np.zeros(g.shape, bool)
    bad[n // 2:, :nq // nkv, 99] = True
    assert np.isnan(g[bad]).all()
    check_attn(np.where(bad, want, g), want, mass, reach, "bfloat16")


@pytest.mark.parametrize("page,most", [(32, 39), (16, 32), (64, 32), (128, 32), (32, 16), (64, 16), (128, 16), (64, 39),
                                       (128, 150)])
def test_append_steps_of_all_kinds(page, most):
    """Random appends one after another (from inside or the end of what is live, blocks rewritten, sizes that differ by
    2^20, rows in front of the first sequence and behind the last): V and the scales as the definition has them, bytes of
    no sequence's as they were, q rotated in place."""
    log(f"case: random appends of up to {most} rows, pages of {page}")
    rng = np.random.default_rng(18 + page + most)
    vm = make_vm()
    nseq, width = 3, max(2, 160 // page) + most // page
    pg = Pages(rng, nseq * width + 1, 2, page)
    table_h = tables(rng, nseq, width, nseq * width + 1)
    table, length = i32(table_h), [0] * nseq
    wv, wvs = pg.v.copy(), pg.vs.copy()
    for step in range(40):
        n = [int(rng.integers(0, most + 1)) for _ in range(nseq)]
        start = [int(rng.integers(max(0, length[b] - 40), min(length[b], width * page - n[b]) + 1)) if length[b] + n[b] <= width * page
                 else int(rng.integers(0, width * page - n[b] + 1)) for b in range(nseq)]
        lead, tail = int(rng.integers(0, 3)), int(rng.integers(0, 3))
        first = lead + np.concatenate([[0], np.cumsum(n)])
        rows = lead + sum(n) + tail
        if rows == 0:
            continue
        amp = 2.0 ** rng.integers(-10, 11, (rows, 2, 1))
        kv = rounded(rng.standard_normal((rows, 2, 128)) * amp, "bfloat16")
        q = dev(rng.standard_normal((rows, 12, 128)), "bfloat16")
        turned = vm.paged_kv_append(dev(kv, "bfloat16"), dev(kv, "bfloat16"), pg.dev, 0, table, i32(start), live=i32(length),
                                    q=q, row_start=i32(first), q_out=torch.zeros_like(q), max_rows=most)
        again = q.clone()
        kv_r = vm.paged_kv_append(dev(kv, "bfloat16"), dev(kv, "bfloat16"), pg.dev, 1, table, i32(start), live=i32(length),
                                  q=again, row_start=i32(first), q_out=again, max_rows=max(max(n), 1))
        assert kv_r is again and torch.equal(again[lead:rows - tail], turned[lead:rows - tail])
        assert torch.equal(again[:lead], q[:lead]) and torch.equal(again[rows - tail:], q[rows - tail:])
        for layer in range(2):
            ref.append(wv[layer], wvs[layer], table_h, page, start, length, [kv[first[b]:first[b + 1]] for b in range(nseq)])
        length = [max(length[b], start[b] + n[b]) for b in range(nseq)]
    gk, gv, gks, gvs = pg.download()
    assert np.array_equal(gvs, wvs) and np.array_equal(gv, wv)


def test_hostile_row_starts():
    log("case: row starts that fall, lie outside or cross")
    rng = np.random.default_rng(19)
    vm = make_vm()
    pg = Pages(rng, 8, 2, 32)
    table, start = i32([[0, 1], [2, 3], [4, 5]]), i32([0, 0, 0])
    x = dev(rng.standard_normal((20, 12, 128)), "bfloat16")
    kv = x[:, :2]
    before = pg.download()
    for rs in ([5, 2, 1, 0], [20, 2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31], [-7, -3, -2, -1]):
        out = torch.full_like(x, 9.0)
        vm.paged_attn(x, pg.dev, 0, table, i32([40, 50, 60]), row_start=i32(rs), out=out)
        vm.paged_kv_append(kv, kv, pg.dev, 0, table, start, row_start=i32(rs), q=x, q_out=out)
        assert (out == 9.0).all()
    for a, b in zip(before, pg.download()):
        assert np.array_equal(a, b)


def test_pages_past_four_gigabytes():
    log("case: page offsets of more than 32 bits")
    rng = np.random.default_rng(20)
    vm = make_vm()
    from fast_dllm_relax_amd.paged import allocate_paged_cache

    num = 2 ** 32 // (2 * 128 * 128) + 7
    cache = allocate_paged_cache(vm.cfg, num, page_size=128)
    ids = [num - 1, 3, num - 5, num - 2]
    n = 400
    qkv = rounded(rng.standard_normal((n, 16, 128)), "bfloat16")
    x = dev(qkv, "bfloat16")
    q = vm.paged_kv_append(x[:, 12:14], x[:, 14:], cache, 1, i32([ids]), i32([0]), q=x[:, :12])
    out = vm.paged_attn(q, cache, 1, i32([ids]), i32([n]), mask_block=32)
    g = lambda t: t.view(torch.uint8)[1, ids].cpu().numpy()  # noqa: E731
    gk, gv = g(cache.k), np.ascontiguousarray(g(cache.v).transpose(0, 1, 3, 2))
    ks, vs = (t[1, ids].double().cpu().numpy() for t in (cache.k_scale, cache.v_scale))
    wv, wvs = np.zeros((4, 2, 128, 128), np.uint8), np.ones((4, 2))
    ref.append(wv, wvs, np.arange(4)[None], 128, [0], [0], [qkv[:, 14:]])
    assert np.array_equal(gv, wv) and np.array_equal(vs, wvs)
    want, mass, reach = ref.attend(q.double().cpu().numpy(), gk, ks, gv, vs, np.arange(4)[None], 128, [n], [np.arange(n)], 32)
    check_attn(out.double().cpu().numpy(), want, mass, reach, "bfloat16")
    # nothing went to the places that the offsets' low 32 bits name
    assert not cache.v.view(torch.uint8)[1, [i - 2 ** 32 // (2 * 128 * 128) for i in ids if i > 1000]].any()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_logprobs_of_long_rows_one_workgroup_each(dtype):
    """So many rows that none is split, each longer than the iterations whose maxima a wave keeps: rising, falling, constant,
    masked, mostly -inf and random ones, at an odd length and from an odd element."""
    log(f"case: long rows in {dtype}")
    rng = np.random.default_rng(21)
    vm = make_vm()
    vocab, rows, top = 200003, 520, 20
    low = float(torch.finfo(TD[dtype]).min)
    base = rng.standard_normal((10, vocab)) * 3
    base[1] = np.linspace(-20, 20, vocab)
    base[2] = base[1][::-1]
    base[3] = 0.75
    base[4] = low
    base[4, [0, 9, 100000, vocab - 1]] = [1, 2, 2, 1]
    base[5] = -np.inf
    base[5, rng.integers(0, vocab, 25)] = 0.5
    base[6, rng.integers(0, vocab, 1000)] = np.inf * -1
    base[7, 170000] = np.nan
    base[8] = -base[8] ** 2  # (the best lie close together)
    base[9, :30], base[9, -30:] = 50.0, 50.0
    base = rounded(base, dtype)
    x = torch.empty(rows * vocab + 1, dtype=TD[dtype], device="cuda")[1:].view(1, rows, vocab)
    ids = rng.integers(0, vocab, rows)
    b = dev(base, dtype)
    for r in range(rows):
        x[0, r] = b[r % 10]
    ids = np.tile(ids[:10], rows // 10)
    got = vm.token_logprobs(x, i32(ids)[None], top_n=top)
    for start in (0, rows - 10):
        check_logprobs([t[:, start:start + 10] for t in got], base, ids[:10], top)


def test_logprobs_past_two_billion_elements():
    log("case: logits of more than 2^31 elements")
    rng = np.random.default_rng(22)
    vm = make_vm()
    rows, vocab = 18000, 120001
    x = torch.zeros((1, rows, vocab), dtype=torch.bfloat16, device="cuda")
    last = rounded(rng.standard_normal((3, vocab)) * 4, "bfloat16")
    x[0, -3:] = dev(last, "bfloat16")
    ids = np.full(rows, 77)
    got = vm.token_logprobs(x, i32(ids)[None], top_n=3)
    check_logprobs([t[:, -3:] for t in got], last, ids[-3:], 3)
    check_logprobs([t[:, :2] for t in got], np.zeros((2, vocab)), ids[:2], 3)


def test_two_graphs_of_one_vm():
    """Two graphs captured from the same calls hold workspaces of their own: replayed on two streams at once, and between
    eager calls, each gives its own results."""
    log("case: two graphs")
    rng = np.random.default_rng(23)
    vm = make_vm()
    pg = Pages(rng, 40, 2, 32)
    table, lens = i32(rng.permutation(40)[None]), i32([1270])
    q = [dev(rng.standard_normal((1, 12, 128)), "bfloat16") for _ in range(2)]
    x = [dev(rng.standard_normal((1, 3, 60000)), "float32") for _ in range(2)]
    run = lambda i: (vm.paged_attn(q[i], pg.dev, 0, table, lens), *vm.token_logprobs(x[i], top_n=9)[1:])  # noqa: E731
    run(0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(i))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(5):
        for i in range(2):
            q[i].copy_(dev(rng.standard_normal((1, 12, 128)), "bfloat16"))
            x[i].copy_(dev(rng.standard_normal((1, 3, 60000)), "float32"))
        want = [run(i) for i in range(2)]
        torch.cuda.synchronize()
        for _ in range(4):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(outs[i], want[i]):
                assert torch.equal(a, b)


def test_the_library_refuses():
    """The C entry points' own checks, one wrong argument at a time; nothing is launched."""
    log("case: refusals of the C entry points")
    import ctypes

    from fast_dllm_relax_amd import _lib

    rng = np.random.default_rng(24)
    vm = make_vm()
    lib = vm.lib
    pg = Pages(rng, 4, 2, 32)
    before = pg.download()
    x = dev(rng.standard_normal((4, 16, 128)), "bfloat16")
    table, two = i32([[0, 1], [2, 3]]), i32([0, 0])
    out = torch.full((4, 12, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    at = x.data_ptr()
    cache = dict(k=pg.dev.k.data_ptr(), v=pg.dev.v.data_ptr(), ks=pg.dev.k_scale.data_ptr(), vs=pg.dev.v_scale.data_ptr(), pages=4, page=32)

    def struct(**change):
        c = {**cache, **change}
        return ctypes.byref(_lib.FdllmPagedCache(c["k"], c["v"], c["ks"], c["vs"], c["pages"], c["page"]))

    append = dict(q=at, ldq=2048, k=at + 2 * 1536, ldk=2048, v=at + 2 * 1792, ldv=2048, rows=4, row_start=None, nseq=2, max_rows=2,
                  cache=struct(), layer=0, table=table.data_ptr(), width=2, table_ld=2, start=two.data_ptr(), live=None, pos=None,
                  q_out=out.data_ptr())
    attn = dict(q=at, ldq=2048, rows=4, row_start=None, nseq=2, max_rows=2, cache=struct(), layer=0, table=table.data_ptr(), width=2,
                table_ld=2, kv_len=two.data_ptr(), max_len=0, mask_block=0, out=out.data_ptr(), ws=None, bytes=0)
    both = [dict(cache=None), dict(cache=struct(page=24)), dict(cache=struct(page=0)), dict(cache=struct(pages=0)), dict(cache=struct(k=None)),
            dict(cache=struct(vs=None)), dict(cache=struct(k=cache["k"] + 8)), dict(layer=-1), dict(layer=2), dict(table=None), dict(width=0),
            dict(width=2 ** 31 - 1), dict(table_ld=-1), dict(rows=-1), dict(nseq=0), dict(nseq=65536, rows=131072), dict(max_rows=-1),
            dict(max_rows=3), dict(rows=3), dict(q=at + 2), dict(ldq=2044), dict(ldq=1528),
            dict(rows=2 ** 30, max_rows=2 ** 30, row_start=two.data_ptr(), nseq=4)]
    for change in [*both, dict(k=None), dict(v=None), dict(start=None), dict(q=None), dict(q_out=None), dict(k=at + 4), dict(ldk=248),
                   dict(ldv=4), dict(q_out=out.data_ptr() + 8), dict(q_out=at)]:
        assert lib.fdllm_paged_kv_append(vm.ctx, *{**append, **change}.values(), None) == _lib.FDLLM_EINVAL, change
    need = lib.fdllm_paged_attn_workspace(vm.ctx, 4, 2, 2, 32, 1000, 0)
    assert need > 0 and lib.fdllm_paged_attn_workspace(vm.ctx, 4, 2, 2, 32, 2, 0) == 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    long = dict(width=1000, table_ld=0, ws=ws.data_ptr(), bytes=need)
    for change in [*both, dict(q=None), dict(kv_len=None), dict(out=None), dict(out=out.data_ptr() + 8), dict(mask_block=-1),
                   dict(max_len=-1), {**long, "bytes": need - 1}, {**long, "ws": None}, {**long, "ws": ws.data_ptr() + 4}]:
        assert lib.fdllm_paged_attn(vm.ctx, *{**attn, **change}.values(), None) == _lib.FDLLM_EINVAL, change
    for sizes in ((2 ** 30, 4, 2 ** 30, 32, 1000, 0), (0, 4, 1, 32, 1000, 0), (4, 4, 1, 0, 1000, 0), (4, 4, 1, 128, 2 ** 31 - 1, 0)):
        assert lib.fdllm_paged_attn_workspace(vm.ctx, *sizes) == 0
    lg, ids = torch.zeros((4, 64), device="cuda"), i32([0] * 4)
    f = torch.zeros((4, 8), device="cuda")
    lp = dict(logits=lg.data_ptr(), type=_lib.LOGITS_F32, rows=4, vocab=64, ld=64, ids=ids.data_ptr(), top=2, logprob=f.data_ptr(),
              entropy=f.data_ptr() + 32, top_ids=f.data_ptr() + 64, top_lp=f.data_ptr() + 96, ws=None, bytes=0)
    for change in [dict(type=3), dict(type=-1), dict(rows=-1), dict(rows=2 ** 24), dict(vocab=0), dict(vocab=2 ** 31 - 1, ld=2 ** 31 - 1),
                   dict(ld=63), dict(top=-1), dict(top=33), dict(vocab=1), dict(logits=None), dict(entropy=None), dict(logprob=None),
                   dict(top_ids=None), dict(top_lp=None), dict(logits=lg.data_ptr() + 2), dict(rows=1, vocab=100000, ld=100000)]:
        assert lib.fdllm_token_logprobs(vm.ctx, *{**lp, **change}.values(), None) == _lib.FDLLM_EINVAL, change
    assert lib.fdllm_token_logprobs_workspace(vm.ctx, 1, 100000, 2) > 0 and lib.fdllm_token_logprobs_workspace(vm.ctx, 2 ** 31 - 1, 100000, 2) == 0
    torch.cuda.synchronize()
    assert (out == 9.0).all() and not f.any()
    for a, b in zip(before, pg.download()):
        assert np.array_equal(a, b)


def attended_room(pg, layer, table, kv_len, n, mask, dtype):
    """What fp16's least step adds to check_attn's bound for each of n rows of one sequence: p, relative to the row's largest
    p x rest (rest: what a page's scale has beyond [2^-15, 2^7], which the conversion of its bytes takes), is rounded to
    2^-39 at least, and the result to 2^-25."""
    if dtype != "float16":
        return np.full(n, 2.0 ** -126)
    room = np.zeros(n)
    for i in range(n):
        pos = kv_len - n + i
        keys = np.arange(min(kv_len, (pos // mask + 1) * mask) if mask else kv_len)
        s = pg.vs[layer][table[0, keys // pg.page]]
        rest = s / np.exp2(np.clip(np.floor(np.log2(s)), -15, 7))
        v = np.abs(ref.E4M3[pg.v[layer][table[0, keys // pg.page], :, keys % pg.page]]).max(axis=2) * s
        room[i] = 2.0 ** -25 + len(keys) * 2.0 ** -39 * (rest.max(axis=0) * (v / rest).max(axis=0)).max()
    return room


@pytest.mark.parametrize("dtype,lo,hi", [("float16", -30, -15), ("float16", -15, 8), ("float16", 8, 11), ("float16", -30, 11),
                                         ("bfloat16", -100, -60), ("bfloat16", 60, 119), ("bfloat16", -100, 119)])
@pytest.mark.parametrize("n,L,mask", [(40, 150, 1), (40, 150, 0), (2, 1500, 1)])
def test_attention_scales_of_all_sizes(dtype, lo, hi, n, L, mask):
    """V's scales from 2^lo to below 2^hi (fp16: values to 448 x 2^10, of which the average is in range), every other one no
    power of two: no value that is converted leaves the type's range, whatever its scale."""
    log(f"case: V scales 2^{lo} .. 2^{hi}, {dtype}, {n} rows over {L} keys, mask {mask}")
    rng = np.random.default_rng(30)
    vm = make_vm(dtype)
    page = 32
    width = (L + page - 1) // page
    pg = Pages(rng, width + 1, 2, page)
    pg.vs = 2.0 ** rng.integers(lo, hi, pg.vs.shape) * np.where(rng.integers(0, 2, pg.vs.shape), rng.uniform(1, 2, pg.vs.shape), 1.0)
    if dtype == "bfloat16":
        pg.vs = np.minimum(pg.vs, 2.0 ** 118)
    pg.vs = pg.vs.astype(np.float32).astype(np.float64)
    pg.upload()
    table = tables(rng, 1, width, width + 1)
    q = rounded(rng.standard_normal((n, 12, 128)) * 0.3, dtype)
    want, mass, reach = ref.attend(q, pg.k[1], pg.ks[1], pg.v[1], pg.vs[1], table, page, [L], [np.arange(n)], mask)
    assert np.abs(want).max() < torch.finfo(TD[dtype]).max * 0.95
    room = mass * (2 * HALF[dtype] + 2 * reach[..., None] * 2.0 ** -17 + 2.0 ** -16)
    room += attended_room(pg, 1, table, L, n, mask, dtype)[:, None, None]
    for max_len in (None, 1):
        got = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32([L]), mask_block=mask, max_len=max_len).double().cpu().numpy()
        worst = float(np.max(np.abs(got - want) / room))
        log(f"  max_len {max_len}: largest error {worst:.3f} of its bound")
        assert np.isfinite(got).all() and worst <= 1.0


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,L,mask", [(64, 96, 1), (64, 96, 32), (64, 96, 0), (2, 1300, 1), (1, 96, 0)])
def test_attention_over_the_types_largest_values(dtype, n, L, mask):
    """V of the type's largest value, which e4m3 rounds up past it: rows that attend such a key get their share of it, rows
    whose mask leaves it out are as without it."""
    log(f"case: V of the largest {dtype}, {n} rows over {L} keys, mask {mask}")
    rng = np.random.default_rng(31)
    vm = make_vm(dtype)
    big = float(torch.finfo(TD[dtype]).max)
    page = 32
    width = (L + page - 1) // page
    pg = Pages(rng, width + 1, 2, page)
    table = tables(rng, 1, width, width + 1)
    kv = rng.standard_normal((2, L, 2, 128)) * np.array([0.5, big * 2.0 ** -9]).reshape(2, 1, 1, 1)
    at = L - n + n // 2
    kv[1, at, 0, 7], kv[1, 3, 0, 9], kv[1, at, 1, 100] = big, -big, -big
    kv = rounded(kv, dtype)
    vm.paged_kv_append(dev(kv[0], dtype), dev(kv[1], dtype), pg.dev, 1, i32(table), i32([0]))
    pg.k, pg.v, pg.ks, pg.vs = pg.download()
    assert ref.E4M3[pg.v[1, table[0, at // page], 0, at % page, 7]] * pg.vs[1, table[0, at // page], 0] > big
    q = rounded(rng.standard_normal((n, 12, 128)) * 0.3, dtype)
    want, mass, reach = ref.attend(q, pg.k[1], pg.ks[1], pg.v[1], pg.vs[1], table, page, [L], [np.arange(n)], mask)
    assert np.abs(want).max() < 0.9 * big
    room = mass * (2 * HALF[dtype] + 2 * reach[..., None] * 2.0 ** -17 + 2.0 ** -16)
    room += attended_room(pg, 1, table, L, n, mask, dtype)[:, None, None]
    for max_len in (None, 1):
        got = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32([L]), mask_block=mask, max_len=max_len).double().cpu().numpy()
        assert np.isfinite(got).all()
        worst = float(np.max(np.abs(got - want) / room))
        log(f"  max_len {max_len}: largest error {worst:.3f} of its bound")
        assert worst <= 1.0


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_a_token_rotated_in_place_in_its_fused_projection(dtype):
    """One row's queries as a slice of the fused projection, rotated where they lie (a single row is contiguous, whatever
    its tensor says): the bits of a new tensor, and nothing else of the row is written."""
    log(f"case: one row in place, {dtype}")
    rng = np.random.default_rng(33)
    vm = make_vm(dtype)
    fused = dev(rng.standard_normal((3, 16, 128)), dtype)
    table, start = i32([[1, 0]]), i32([37])
    for rows in (slice(0, 1), slice(2, 3)):
        x = fused[rows].clone()
        ends, outs = [], []
        for place in (False, True):
            pg = Pages(np.random.default_rng(1), 2, 2, 32)
            q = x[:, :12]
            got = vm.paged_kv_append(x[:, 12:14], x[:, 14:], pg.dev, 1, table, start, q=q,
                                     q_out=q if place else torch.zeros((1, 12, 128), dtype=TD[dtype], device="cuda"))
            outs.append(got.clone())
            ends.append(pg.download())
        assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], fused[rows][:, :12])
        assert torch.equal(x[:, 12:], fused[rows][:, 12:])
        for a, b in zip(*ends):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("nq,nkv,n", [(12, 2, 1), (12, 2, 8)])
def test_attention_nan_of_vanishing_probability(nq, nkv, n):
    """A NaN in V at a key that is attended, at a probability that no float holds (e^-180), spoils its dim whether the keys are
    split over workgroups or not; K of the far keys decides which split's statistics are the row's."""
    log(f"case: NaN at a vanishing probability, {n} rows")
    rng = np.random.default_rng(32)
    vm = make_vm("bfloat16", nq, nkv)
    page, L = 64, 3008
    width = L // page
    pg = Pages(rng, width, nkv, page)
    table = tables(rng, 1, width, width)
    pg.ks[:] = 1.0
    one = int(ref.encode(1.0))
    pg.k[:] = one | 128
    pg.k[1, table[0, 0]] = one  # scores of +90 in the first page, of -90 elsewhere: far more than 2^-150 apart
    pg.v[1, table[0, (L - 100) // page], 0, (L - 100) % page, 77] = 127
    pg.upload()
    q = np.full((n, nq, 128), 8.0)
    want, mass, reach = ref.attend(q, np.where((pg.k & 127) == 127, 0, pg.k)[1], pg.ks[1],
                                   np.where((pg.v & 127) == 127, 0, pg.v)[1], pg.vs[1], table, page, [L], [np.arange(n)], 0)
    bad = np.zeros(q.shape, bool)
    bad[:, :nq // nkv, 77] = True
    for max_len in (None, 1):
        log(f"  max_len {max_len}")
        g = vm.paged_attn(dev(q, "bfloat16"), pg.dev, 1, i32(table), i32([L]), max_len=max_len).double().cpu().numpy()
        assert np.array_equal(np.isnan(g), bad)
        check_attn(np.where(bad, want, g), want, mass, reach, "bfloat16")


def test_attention_over_strided_queries_in_place_is_refused():
    """out at q's address needs a contiguous q of two rows and more (workgroups would write rows that others still read); one row
    is contiguous whatever its stride.  Nothing is launched by a refused call."""
    log("case: attention in place, strided")
    import ctypes

    from fast_dllm_relax_amd import _lib

    rng = np.random.default_rng(34)
    vm = make_vm()
    pg = Pages(rng, 4, 2, 32)
    fused = dev(rng.standard_normal((4, 16, 128)), "bfloat16")
    before = fused.clone()
    table, lens = i32([[0, 1]]), i32([50])
    cache = ctypes.byref(_lib.FdllmPagedCache(pg.dev.k.data_ptr(), pg.dev.v.data_ptr(), pg.dev.k_scale.data_ptr(),
                                              pg.dev.v_scale.data_ptr(), 4, 32))

    def call(rows, ldq):
        return vm.lib.fdllm_paged_attn(vm.ctx, fused.data_ptr(), ldq, rows, None, 1, rows, cache, 0, table.data_ptr(), 2, 2,
                                       lens.data_ptr(), 0, 0, fused.data_ptr(), None, 0, torch.cuda.current_stream().cuda_stream)

    for rows, ldq in ((4, 2048), (2, 1544)):
        assert call(rows, ldq) == _lib.FDLLM_EINVAL
    over = fused.flatten()[:4 * 1536].view(4, 12, 128)
    with pytest.raises(ValueError):
        vm.paged_attn(fused[:, :12], pg.dev, 0, table, lens, out=over)
    torch.cuda.synchronize()
    assert torch.equal(fused, before)
    want = vm.paged_attn(before[:1, :12], pg.dev, 0, table, lens)
    assert call(1, 2048) == 0
    torch.cuda.synchronize()
    assert torch.equal(fused[:1, :12], want) and torch.equal(fused[:, 12:], before[:, 12:]) and torch.equal(fused[1:], before[1:])


def check_key_bytes(got, scales, bounds):
    (lo, s_lo), (hi, s_hi) = bounds
    assert np.array_equal(s_lo, s_hi)  # (no maximum so near a power of two that the bounds differ)
    assert np.array_equal(scales, s_lo)
    log(f"  bytes left open by the bounds: {int((lo != hi).sum())} of {lo.size}, outside: {int(ref.outside(got, lo, hi).sum())}")
    assert not ref.outside(got, lo, hi).any()


@pytest.mark.parametrize("dtype,page,rows,start,pos", [("bfloat16", 32, [8192], [0], [0]), ("bfloat16", 16, [3000, 0, 1000], [7, 0, 3], [7, 0, 120000]),
                                                       ("float16", 64, [33, 700, 1201], [63, 0, 100], [90000, 0, 31000]),
                                                       ("float16", 128, [1000, 129], [5, 127], [5, 127]),
                                                       ("bfloat16", 64, [32, 1, 31, 9] * 16, [63, 64, 20, 0] * 16, [63, 64, 20, 0] * 16),
                                                       ("bfloat16", 128, [32, 1, 31, 9] * 16, [127, 100, 97, 1] * 16, [127, 100, 97, 1] * 16)])
def test_appended_keys_are_the_definitions(dtype, page, rows, start, pos):
    """Every byte and scale of K of many rows at once is what a rotation in 64 bits, rounded once to fp32, gives."""
    log(f"case: key bytes, {dtype}, pages of {page}, {sum(rows)} rows")
    rng = np.random.default_rng(35)
    vm = make_vm(dtype)
    nseq = len(rows)
    width = (max(s + n for s, n in zip(start, rows)) + page - 1) // page
    pg = Pages(rng, nseq * width + 1, 2, page)
    table = tables(rng, nseq, width, nseq * width + 1)
    first = np.concatenate([[0], np.cumsum(rows)])
    x = rounded(rng.standard_normal((sum(rows), 2, 128)) * np.exp(0.5 * rng.standard_normal((sum(rows), 1, 1))), dtype)
    t = dev(x, dtype)
    bounds = []
    at = np.concatenate([p + np.arange(n) for p, n in zip(pos, rows)])
    for new in ref.rotation_bounds(x, at, THETA):
        k, ks = pg.k.copy(), pg.ks.copy()
        ref.append(k[1], ks[1], table, page, start, start, [new[first[b]:first[b + 1]] for b in range(nseq)])
        bounds.append((k, ks))
    vm.paged_kv_append(t, t, pg.dev, 1, i32(table), i32(start), pos=i32(pos), row_start=i32(first), max_rows=max(rows))
    gk, _, gks, _ = pg.download()
    check_key_bytes(gk, gks, bounds)


@pytest.mark.parametrize("page,most", [(16, 32), (32, 39), (64, 32), (64, 39), (128, 32), (128, 150)])
def test_keys_of_appends_of_all_kinds(page, most):
    """As test_append_steps_of_all_kinds, for K: rows encoded again with larger scales, blocks rewritten, slots that hold no row
    and pages of no sequence as they were."""
    log(f"case: keys of random appends of up to {most} rows, pages of {page}")
    rng = np.random.default_rng(36 + page + most)
    vm = make_vm()
    nseq, width = 3, max(2, 160 // page) + most // page
    pg = Pages(rng, nseq * width + 1, 2, page)
    table_h = tables(rng, nseq, width, nseq * width + 1)
    table, length = i32(table_h), [0] * nseq
    bounds = [(pg.k.copy(), pg.ks.copy()) for _ in range(2)]
    for step in range(30):
        n = [int(rng.integers(0, most + 1)) for _ in range(nseq)]
        start = [int(rng.integers(max(0, length[b] - 40), min(length[b], width * page - n[b]) + 1)) if length[b] + n[b] <= width * page
                 else int(rng.integers(0, width * page - n[b] + 1)) for b in range(nseq)]
        first = np.concatenate([[0], np.cumsum(n)])
        if first[-1] == 0:
            continue
        amp = 2.0 ** rng.integers(-10, 11, (first[-1], 2, 1))
        x = rounded(rng.standard_normal((first[-1], 2, 128)) * amp, "bfloat16")
        t = dev(x, "bfloat16")
        vm.paged_kv_append(t, t, pg.dev, 1, table, i32(start), live=i32(length), row_start=i32(first), max_rows=most)
        at = np.concatenate([s + np.arange(k) for s, k in zip(start, n)])
        for (k, ks), new in zip(bounds, ref.rotation_bounds(x, at, THETA)):
            ref.append(k[1], ks[1], table_h, page, start, length, [new[first[b]:first[b + 1]] for b in range(nseq)])
        length = [max(length[b], start[b] + n[b]) for b in range(nseq)]
    gk, _, gks, _ = pg.download()
    check_key_bytes(gk, gks, bounds)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("nq,nkv,n,L", [(12, 2, [1] * 8, 40), (12, 2, [2, 1, 2], 5), (16, 1, [1], 64), (8, 8, [16], 48), (12, 2, [1], 3000)])
def test_attention_of_few_rows_rounds_once(dtype, nq, nkv, n, L):
    """With 16 flattened rows and fewer the probabilities reach the second product in two parts, each rounded by half a step u of its
    own size (u^2 of p is left), and their sum is in fp32: the one rounding that counts is the result's.  The scores' part of
    the bound as in check_attn, fp16's least step as in attended_room (the larger part's residue ends at 2^-25 x 2^-14)."""
    log(f"case: one rounding, {dtype}, {nq} heads on {nkv}, rows {n} over {L}")
    rng = np.random.default_rng(37)
    vm = make_vm(dtype, nq, nkv)
    page, nseq = 16, len(n)
    width = (L + page - 1) // page
    pg = Pages(rng, nseq * width, nkv, page)
    table = tables(rng, nseq, width, nseq * width)
    first = np.concatenate([[0], np.cumsum(n)])
    q = rounded(rng.standard_normal((sum(n), nq, 128)) * 0.25, dtype)
    idx = [np.arange(first[b], first[b + 1]) for b in range(nseq)]
    want, mass, reach = ref.attend(q, pg.k[1], pg.ks[1], pg.v[1], pg.vs[1], table, page, [L] * nseq, idx, 0)
    u = HALF[dtype]
    room = u * np.abs(want) + mass * (2 * u * u + 2 * reach[..., None] * 2.0 ** -17 + 2.0 ** -16)
    if dtype == "float16":
        room += 2.0 ** -25 + L * 2.0 ** -39 * np.abs(ref.E4M3[pg.v[1]] * pg.vs[1][..., None, None]).max()
    got = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32([L] * nseq), row_start=i32(first), max_rows=max(n))
    worst = float(np.max(np.abs(got.double().cpu().numpy() - want) / room))
    log(f"  largest error {worst:.3f} of its bound, the scores' part of it up to {float((2 * reach * 2.0 ** -17 / u).max()):.3f} u")
    assert worst <= 1.0
