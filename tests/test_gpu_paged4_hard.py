"""Values, scales and calls at the ends of what the paged 4-bit cache and the heads' norms take, against their definitions in 64
bits (tests/paged4_reference.py)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import paged4_reference as ref
from helpers import log
from test_gpu_paged import TD, dev, i32, make_vm, rounded, tables
from test_gpu_paged4 import Pages, check_attn

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
        values = pg.values(1)
        if not good:
            pg.vs[1, at[0], 0, at[1]] = 0.0
            values = pg.values(1)
        want, mass, reach = ref.attend(q, *values, table, page, table.shape[1], [L], [np.arange(n)], 0)
        g = vm.paged_attn(dev(q, "float16"), pg.dev, 1, i32(table), i32([L])).double().cpu().numpy()
        if not good:
            assert np.isnan(g[:, :6]).all() and np.isfinite(g[:, 6:]).all()
        check_attn(np.where(np.isnan(g), want, g), want, mass, reach, "float16", n == 1)
