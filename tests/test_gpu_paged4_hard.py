"""Values, scales and calls at the ends of what the paged 4-bit cache and the heads' norms take, against their definitions in 64
bits (tests/paged4_reference.py)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import paged4_reference as ref
import test_gpu_paged4
from helpers import log
from test_gpu_paged import HALF, THETA, dev, i32, make_vm, rounded, tables
from test_gpu_paged4 import LEAST, Pages, check_attn, rotary_of

pytestmark = pytest.mark.gpu


# ---- V's scales --------------------------------------------------------------------------------------------

# rows, keys, mask, sequences, heads: a tile of rows with full and edge tiles of keys, two tiles, keys split over workgroups,
# three tiles (512 workgroups of them)
SHAPES = [(1, 96, 0, 1, (12, 2)), (1, 640, 0, 1, (12, 2)), (20, 150, 1, 1, (12, 2)), (2, 1500, 1, 1, (12, 2)), (1, 3000, 0, 1, (16, 1)),
          (150, 200, 32, 16, (8, 8))]
KINDS = {
    "zero": lambda rng, shape: np.where(rng.random(shape) < 0.3, rng.choice([0.0, -0.0], shape), rng.uniform(0.1, 0.4, shape)),
    "all zero": lambda rng, shape: np.zeros(shape),
    "least": lambda rng, shape: np.where(rng.random(shape) < 0.5, 2.0 ** rng.integers(-133, -60, shape), rng.uniform(0.1, 0.4, shape)),
    # (a wave's first tiles: their keys come before any of ordinary size)
    "least first": lambda rng, shape: np.where(np.arange(shape[1])[None, :, None, None] < 8, 2.0 ** -120, rng.uniform(0.1, 0.4, shape)),
    "negative": lambda rng, shape: rng.uniform(0.1, 0.4, shape) * rng.choice([-1, 1], shape),
}


def scaled_pages(rng, kind, shape, L, nseq, nkv, page=32):
    width = (L + page - 1) // page
    pg = Pages(rng, nseq * width, nkv, page)
    table = np.arange(nseq * width).reshape(nseq, width)
    pg.vs = ref.bf16(KINDS[kind](rng, pg.vs.shape)) if kind in KINDS else pg.vs
    pg.upload()
    return pg, table


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_value_scales_of_other_writers(dtype, kind, shape):
    """Scales that the append does not write: a live key whose scale is 0 keeps its weight in the sum and adds nothing, one of
    under 2^-60 adds at most 6 x 2^-60 (far below fp16's least step, which check_attn allows), a negative one turns its values round."""
    n, L, mask, nseq, (nq, nkv) = SHAPES[shape]
    log(f"case: V scales {kind}, {dtype}, {n} rows of {nseq} sequences over {L} keys, mask {mask}")
    rng = np.random.default_rng(700 + shape)
    vm = make_vm(dtype, nq, nkv)
    pg, table = scaled_pages(rng, kind, shape, L, nseq, nkv)
    q = rounded(rng.standard_normal((nseq * n, nq, 128)) * 0.3, dtype)
    idx = [np.arange(b * n, (b + 1) * n) for b in range(nseq)]
    want, mass, reach = ref.attend(q, *pg.values(1), table, 32, nseq * table.shape[1], [L] * nseq, idx, mask)
    for max_len in (None, 1):
        g = vm.paged_attn(dev(q, dtype), pg.dev, 1, i32(table), i32([L] * nseq), mask_block=mask, max_len=max_len).double().cpu().numpy()
        check_attn(g, want, mass, reach, dtype, n * (nq // nkv) <= 16)


@pytest.mark.parametrize("lo,hi", [(-60, 13), (-60, 0), (4, 13)])
@pytest.mark.parametrize("n,L,mask", [(40, 150, 1), (2, 1500, 1), (1, 96, 0)])
def test_attention_value_scales_to_the_ends_in_fp16(lo, hi, n, L, mask):
    """All sizes that an append of fp16 values writes, 2^-60 to 65504 / 6, beside each other."""
    log(f"case: fp16 V scales 2^{lo} .. 2^{hi}, {n} rows over {L} keys, mask {mask}")
    rng = np.random.default_rng(710)
    vm = make_vm("float16")
    pg, table = scaled_pages(rng, None, None, L, 1, 2)
    pg.vs = ref.bf16(2.0 ** rng.uniform(lo, hi, pg.vs.shape))
    pg.upload()
    q = rounded(rng.standard_normal((n, 12, 128)) * 0.3, "float16")
    want, mass, reach = ref.attend(q, *pg.values(1), table, 32, table.shape[1], [L], [np.arange(n)], mask)
    assert np.abs(want).max() < 65504 * 0.95
    for max_len in (None, 1):
        g = vm.paged_attn(dev(q, "float16"), pg.dev, 1, i32(table), i32([L]), mask_block=mask, max_len=max_len).double().cpu().numpy()
        check_attn(g, want, mass, reach, "float16", n * 6 <= 16)


@pytest.mark.parametrize("n,L", [(1, 200), (20, 700)])
def test_attention_value_scales_past_fp16(n, L):
    """In fp16 a scale of up to 2^31 is taken as it is (here at a probability that brings its value back into range); a larger one
    makes the rows that attend it NaN, and no others."""
    log(f"case: V scales past fp16, {n} rows")
    rng = np.random.default_rng(711)
    vm = make_vm("float16")
    pg, table = scaled_pages(rng, None, None, L, 1, 2)
    page = 32
    # queries of 2, keys of +1 and, one of them, -1: scores of +-22.6, so 2^-65 of probability for the one
    pg.ke[:] = 127
    pg.k[:] = 2
    at = table[0, 70 // page], 70 % page
    pg.k[1, at[0], :, at[1]] = 2 | 8
    for power, good in ((17, True), (31, True), (32, False), (120, False), (math.inf, False)):
        pg.vs[1, at[0], 0, at[1]] = 2.0 ** power
        pg.upload()
        q = np.full((n, 12, 128), 2.0)
        if not good:
            pg.vs[1, at[0], 0, at[1]] = 0.0
        want, mass, reach = ref.attend(q, *pg.values(1), table, page, table.shape[1], [L], [np.arange(n)], 0)
        g = vm.paged_attn(dev(q, "float16"), pg.dev, 1, i32(table), i32([L])).double().cpu().numpy()
        if not good:
            assert np.isnan(g[:, :6]).all() and np.isfinite(g[:, 6:]).all()
        check_attn(np.where(np.isnan(g), want, g), want, mass, reach, "float16", n == 1)


# ---- norms and rotation ------------------------------------------------------------------------------------


@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_norms_of_large_and_small_rows_with_small_weights(eps):
    """bf16 rows from the type's least sizes to its largest under weights far from 1: the row over its norm is of ordinary size and
    so is its product with the weight, though the norm's inverse times the weight may be beyond fp32."""
    log(f"case: norms with small weights, eps {eps}")
    rng = np.random.default_rng(720)
    vm = make_vm() if eps else small_eps_vm(eps)
    # with eps the small rows are small results, without it they are of the weights' size
    sizes = np.array([125, 120, 110, 90, 40, 0, -20, *((-60, -100, -128) if not eps else ())])
    x = rounded(rng.uniform(0.25, 1.0, (len(sizes), 12, 128)) * rng.choice([-1, 1], (len(sizes), 12, 128)) * 2.0 ** sizes[:, None, None], "bfloat16")
    for power in (-40, -60, 0, 30):
        w = rounded((1 + 0.3 * rng.standard_normal(128)) * 2.0 ** power, "bfloat16")
        r = rotary_of()
        q, k = vm.rotate_heads(dev(x, "bfloat16"), dev(x[:, :2], "bfloat16"), 100, rotary=r, q_norm=dev(w, "bfloat16"), k_norm=dev(w, "bfloat16"))
        want = ref.turn(x, 100 + np.arange(len(sizes)), r.frequencies, weight=w, eps=eps)
        room = ref.turn_size(x, weight=w, eps=eps) * 2.0 ** -20  # (as check_turned has it)
        room += HALF["bfloat16"] * (np.abs(want) + room) + LEAST["bfloat16"]
        for g, sl in ((q, slice(None)), (k, slice(2))):
            e = np.abs(g.double().cpu().numpy() - want[:, sl]) / room[:, sl]
            log(f"  weights of 2^{power}: largest error {np.max(e):.3f} of its bound")
            assert e.max() <= 1.0


def small_eps_vm(eps):
    from fast_dllm_relax_amd.config import FastDLLMConfig
    from fast_dllm_relax_amd.params import param_names, param_shapes
    from fast_dllm_relax_amd.vm import HipVM

    cfg = FastDLLMConfig(vocab_size=256, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=12,
                         num_key_value_heads=2, head_dim=128, rope_theta=THETA, rms_norm_eps=eps)
    shapes = param_shapes(cfg)
    return HipVM(cfg, [torch.zeros(shapes[n], dtype=torch.bfloat16, device="cuda") for n in param_names(cfg)])


# ---- keys next to a tie ------------------------------------------------------------------------------------

# position, pair of 8, and its two values, which turn to within 2^-25 of a border between two codes, on the other side of it than
# the even code: rounded to fp32 they lie on the border
TIES = [(261, 0, 1.7421875, 3.828125), (468, 1, 0.5078125, 2.515625), (776, 2, 0.8671875, 1.84375), (818, 2, 0.333984375, 2.234375),
        (835, 6, 1.2578125, 0.279296875), (847, 0, 0.91796875, 1.53125), (885, 5, 3.625, 0.51171875), (1007, 3, 3.375, 1.296875),
        (1119, 7, 0.263671875, 2.171875), (1150, 3, 1.3984375, 0.68359375), (1280, 2, 0.65234375, 0.39453125), (1299, 7, 0.259765625, 1.3359375)]


@pytest.mark.parametrize("inter", [False, True])
def test_append_keys_next_to_a_tie(inter):
    """Codes are the nearest to the values in 64 bits, whose sines are within 2^-33."""
    log(f"case: keys next to a tie, neighbours {inter}")
    rng = np.random.default_rng(730)
    vm = make_vm()
    r = rotary_of(16, inter)
    pg = Pages(rng, len(TIES), 2, 16)
    x = np.zeros((len(TIES), 2, 128))
    x[..., 20] = 6.0  # (not turned: the block's scale is 1)
    for i, (p, j, a, b) in enumerate(TIES):
        x[i, :, 2 * j if inter else j], x[i, :, 2 * j + 1 if inter else j + 8] = a, b
    pos = np.array([t[0] for t in TIES])
    k = dev(x, "bfloat16")
    assert np.array_equal(k.double().cpu().numpy(), x)
    vm.paged4_append(k, k, pg.dev, 1, i32(np.arange(len(TIES))[:, None]), i32([3] * len(TIES)), pos=i32(pos), rotary=r)
    code, _, ke, _ = pg.download()
    y = ref.turn(x, pos, r.frequencies, 16, inter)
    want, e = ref.keys(y)
    assert (ref.keys(y.astype(np.float32).astype(np.float64))[0] != want).any(axis=-1).all()
    assert np.array_equal(code[1, :, :, 3], want) and np.array_equal(ke[1, :, :, 3], e)


def test_append_keys_next_to_a_scales_border():
    """The largest value of a block a little more than 7 x 2^e, by less than fp32 tells: the scale is 2^(e + 1)."""
    log("case: keys next to the border between two scales")
    rng = np.random.default_rng(731)
    vm = make_vm()
    n = 12
    x = np.zeros((n, 2, 128))
    x[..., 1] = 1.75 * 2.0 ** (np.arange(n) - 6)[:, None]
    gain = 1 + 2.0 ** -26 * np.where(np.arange(2) == 0, 1, -1)
    for g in gain:  # (turned by nothing, times a factor)
        from fast_dllm_relax_amd.rotary import Rotary

        r = Rotary(dim=16, frequencies=[0.0] * 8, factor=float(g))
        pg = Pages(rng, 1, 2, 16)
        vm.paged4_append(dev(x, "bfloat16"), dev(x, "bfloat16"), pg.dev, 1, i32([[0]]), i32([0]), rotary=r)
        y = ref.turn(x, np.zeros(n), r.frequencies, 16, False, r.factor)
        want, e = ref.keys(y)
        code, _, ke, _ = pg.download()
        assert np.array_equal(ke[1, 0, :, :n].swapaxes(0, 1), e) and np.array_equal(code[1, 0, :, :n].swapaxes(0, 1), want)


# ---- the two ways from Python ------------------------------------------------------------------------------


def test_the_short_way_takes_calls_with_parts_left_out(monkeypatch):
    """Keys appended without queries, one of queries and keys rotated alone, positions from a first one: these calls take the
    short way too, and give the bits and the errors of the checks in Python."""
    log("case: the short way with parts left out")
    from fast_dllm_relax_amd import vm as module

    rng = np.random.default_rng(740)
    vm = make_vm()
    pg = Pages(rng, 9, 2, 32)
    table, start, pos, first = i32(np.arange(8).reshape(2, 4)), i32([3, 40]), i32([9, 7]), i32([0, 3, 8])
    x = dev(rng.standard_normal((10, 16, 128)), "bfloat16")
    w = dev(rng.standard_normal(128), "bfloat16")
    q, k, v = x[:, :12], x[:, 12:14], x[:, 14:]
    new = lambda n, rows=10: torch.zeros((rows, n, 128), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    r, at = rotary_of(64, True), i32(np.arange(10))
    long = object.__new__(type(vm))
    long.__dict__.update(vm.__dict__, _spec=None)
    calls, took = module.fdllm_calls, []

    class Counted:
        def __getattr__(self, name):
            def call(*args):
                took.append(getattr(calls, name)(*args))
                return took[-1]
            return call

    monkeypatch.setattr(module, "fdllm_calls", Counted())
    try:
        good = [
            lambda m: (m.paged4_append(k, v, pg.dev, 1, table, start, rotary=r, k_norm=w, pos=pos), *pg.download()),
            lambda m: (m.paged4_append(k, v, pg.dev, 0, table, start, row_start=first, max_rows=5), *pg.download()),
            lambda m: m.rotate_heads(q, None, at, rotary=r, q_norm=w, q_out=new(12)),
            lambda m: m.rotate_heads(None, k, at, k_out=new(2)),
            lambda m: m.rotate_heads(None, k[:1], at[:1], k_norm=w, k_out=new(2, 1)),
            lambda m: m.rotate_heads(q, k, 2079, q_out=new(12), k_out=new(2)),
            lambda m: m.rotate_heads(q, None, -3, rotary=r, q_out=new(12)),
            lambda m: m.rotate_heads(None, k, 2 ** 31 - 11, k_out=new(2)),
        ]
        for i, f in enumerate(good):
            took.clear()
            a, b = f(vm), f(long)
            assert took == [0], i
            for p, s in zip(a, b):
                assert p is s is None or (np.array_equal(p, s, equal_nan=p.dtype.kind == "f") if isinstance(p, np.ndarray) else torch.equal(p, s)), i
        ok_r = dict(q=q, k=k, pos=3, q_out=new(12), k_out=new(2))
        ok_a = dict(k=k, v=v, cache=pg.dev, layer=1, page_table=table, start=start)
        before = pg.download()
        bad = [("rotate_heads", {**ok_r, **c}) for c in
               (dict(q=None), dict(k=None), dict(q=None, k=None, q_out=None, k_out=None), dict(q=None, q_out=None, q_norm=w),
                dict(k=None, k_out=None, k_norm=w), dict(pos=2 ** 31 - 9), dict(pos=-2 ** 31 - 1), dict(pos=2 ** 70), dict(pos=1.0), dict(pos=None))]
        bad += [("paged4_append", {**ok_a, **c}) for c in (dict(q_out=new(12)), dict(q_norm=w), dict(k_norm=w[:64]), dict(max_rows=4), dict(k=None))]
        for name, kw in bad:
            took.clear()
            errors = []
            for m in (vm, long):
                with pytest.raises((ValueError, TypeError, AttributeError)) as e:
                    getattr(m, name)(**kw)
                errors.append((e.type, str(e.value)))
            assert errors[0] == errors[1] and 0 not in took, (name, errors)
        torch.cuda.synchronize()
        after = pg.download()
        assert all(np.array_equal(p, s, equal_nan=p.dtype.kind == "f") for p, s in zip(before, after))
        # rows of one call, none
        assert vm.rotate_heads(q[:0], None, 3)[0].shape == (0, 12, 128)
    finally:
        long.ctx = None  # (the context is vm's)


# ---- masks, NaN and pages in fp16 --------------------------------------------------------------------------


@pytest.mark.parametrize("nq,nkv,n,L,mask,nseq", [(12, 2, 100, 230, 1, 1), (12, 2, 100, 230, 32, 1), (12, 2, 9, 3000, 1, 1), (16, 1, 1, 3000, 1, 1),
                                                  (12, 2, 2, 3000, 1, 1), (8, 8, 150, 200, 1, 16)])
def test_attention_nan_behind_the_mask_in_fp16(nq, nkv, n, L, mask, nseq):
    """Keys that a row does not attend may hold NaN: rows in front of it are as without it, rows that see it are NaN throughout
    (in the head's dims).  The last case takes three tiles of rows a workgroup."""
    log(f"case: fp16, NaN behind a mask of {mask}, {nq} heads, {n} rows of {nseq} sequences over {L}")
    rng = np.random.default_rng(750)
    vm = make_vm("float16", nq, nkv)
    page = 32
    width = (L + page - 1) // page
    pg = Pages(rng, nseq * width + 1, nkv, page)
    table = tables(rng, nseq, width, nseq * width + 1)
    q = rounded(rng.standard_normal((nseq * n, nq, 128)) * 0.5, "float16")
    idx = [np.arange(b * n, (b + 1) * n) for b in range(nseq)]
    want, mass, reach = ref.attend(q, *pg.values(1), table, page, nseq * width + 1, [L] * nseq, idx, mask)
    at_v, at_k = L - n + n // 2, L - n + (3 * n) // 4
    pg.vs[1, table[:, at_v // page], 0, at_v % page] = np.nan
    pg.ke[1, table[:, at_k // page], nkv - 1, at_k % page, 2] = 255
    pg.upload()
    pos = np.tile(np.arange(L - n, L), nseq)
    sees = lambda p: (pos // mask + 1) * mask > p  # noqa: E731
    G = nq // nkv
    bad = np.zeros(q.shape, bool)
    bad[sees(at_v), :G] = True
    bad[sees(at_k), (nkv - 1) * G:] = True
    for max_len in (None, 1):
        g = vm.paged_attn(dev(q, "float16"), pg.dev, 1, i32(table), i32([L] * nseq), mask_block=mask, max_len=max_len).double().cpu().numpy()
        assert np.isnan(g[bad]).all()
        check_attn(np.where(bad, want, g), want, mass, reach, "float16", n * G <= 16)


@pytest.mark.parametrize("n", [1, 8])
def test_attention_nan_of_vanishing_probability_in_fp16(n):
    """A NaN in V at a key that is attended, at a probability that no float holds, spoils its head whether the keys are split
    over workgroups or not."""
    log(f"case: fp16, NaN at a vanishing probability, {n} rows")
    rng = np.random.default_rng(751)
    vm = make_vm("float16")
    page, L = 64, 3008
    width = L // page
    pg = Pages(rng, width, 2, page)
    table = tables(rng, 1, width, width)
    pg.ke[:] = 127
    pg.k[:] = 2 | 8
    pg.k[1, table[0, 0]] = 2  # scores of +90 in the first page, of -90 elsewhere
    q = np.full((n, 12, 128), 8.0)
    want, mass, reach = ref.attend(q, *pg.values(1), table, page, width, [L], [np.arange(n)], 0)
    pg.vs[1, table[0, (L - 100) // page], 0, (L - 100) % page] = np.nan
    pg.upload()
    bad = np.zeros(q.shape, bool)
    bad[:, :6] = True
    for max_len in (None, 1):
        g = vm.paged_attn(dev(q, "float16"), pg.dev, 1, i32(table), i32([L]), max_len=max_len).double().cpu().numpy()
        assert np.array_equal(np.isnan(g), bad)
        check_attn(np.where(bad, want, g), want, mass, reach, "float16", n == 1)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,nseq,heads", [(1, 2, (12, 2)), (10, 2, (12, 2)), (150, 16, (8, 8))])
def test_attention_pages_that_are_none_inside_the_length(dtype, n, nseq, heads):
    """Their keys are as if they were not, in workgroups of one, two and three tiles of rows, between tiles that are whole."""
    log(f"case: pages that are none, {dtype}, {n} rows of {nseq} sequences")
    rng = np.random.default_rng(752)
    nq, nkv = heads
    vm = make_vm(dtype, nq, nkv)
    page, width, L = 32, 20, 620
    pg = Pages(rng, nseq * width, nkv, page)
    table = np.arange(nseq * width).reshape(nseq, width)
    for b in range(nseq):
        table[b, rng.choice(width, 4, replace=False)] = [-1, nseq * width, 2 ** 31 - 1, -2 ** 31]
    q = rounded(rng.standard_normal((nseq * n, nq, 128)) * 0.5, dtype)
    idx = [np.arange(b * n, (b + 1) * n) for b in range(nseq)]
    want, mass, reach = ref.attend(q, *pg.values(0), table, page, nseq * width, [L] * nseq, idx, 0)
    g = vm.paged_attn(dev(q, dtype), pg.dev, 0, i32(table), i32([L] * nseq))
    check_attn(g.double().cpu().numpy(), want, mass, reach, dtype, n * (nq // nkv) <= 16)


def test_attention_in_place_strided_and_shared_in_fp16():
    """q as a slice of a fused projection, a table whose rows lie apart, pages that sequences share, out = q, a ragged batch."""
    log("case: fp16, strides, shared pages, in place")
    rng = np.random.default_rng(753)
    vm = make_vm("float16")
    page, n, kv_len = 32, [5, 33, 1], [70, 100, 1400]
    pg = Pages(rng, 60, 2, page)
    wide = np.stack([rng.permutation(60) for _ in range(3)])
    wide[1, :2] = wide[2, :2] = wide[0, :2]  # a common prefix
    table = i32(wide)[:, :50]
    first = np.concatenate([[0], np.cumsum(n)])
    rows = sum(n)
    qkv = rounded(rng.standard_normal((rows, 16, 128)) * 0.5, "float16")
    fused = dev(qkv, "float16")
    idx = [np.arange(first[b], first[b + 1]) for b in range(3)]
    want, mass, reach = ref.attend(qkv[:, :12], *pg.values(1), wide[:, :50], page, 60, kv_len, idx, 1)
    kw = dict(mask_block=1, row_start=i32(first), max_rows=33)
    for max_len in (64, 100000):  # (no second launch; split)
        q = fused[:, :12].clone(memory_format=torch.contiguous_format)
        out = vm.paged_attn(fused[:, :12], pg.dev, 1, table, i32(kv_len), max_len=max_len, **kw)
        check_attn(out.double().cpu().numpy(), want, mass, reach, "float16", False)
        assert vm.paged_attn(q, pg.dev, 1, table, i32(kv_len), max_len=max_len, out=q, **kw) is q and torch.equal(q, out)


# ---- the append's variants ---------------------------------------------------------------------------------


@pytest.mark.parametrize("case", [
    # (as test_append's) workgroups of two query heads or one kv head up to 3100 of four and two, those above; odd numbers of heads
    ("bfloat16", 5, 5, 64, [3050], [9], None, 128, False, None, True),
    ("float16", 5, 5, 64, [3100], [9], None, 64, True, None, True),
    ("bfloat16", 16, 1, 128, [2100, 2101], [0, 3], [50000, 7], 128, False, dict(type="ntk", factor=2.0), False),
    ("bfloat16", 6, 3, 32, [4200, 1], [0, 3], None, 32, True, None, True),
])
def test_append_of_many_rows_and_odd_heads(case, monkeypatch):
    monkeypatch.setattr(test_gpu_paged4, "APPENDS", [case])
    test_gpu_paged4.test_append(0)


@pytest.mark.parametrize("nseq", [126, 127, 128, 129])
def test_rows_find_their_sequences_by_counting_and_by_halving(nseq):
    test_gpu_paged4.test_many_sequences(nseq, 4)
