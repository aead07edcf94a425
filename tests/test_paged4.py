"""The paged 4-bit cache, the heads' norms and rotation and the rotary plans on the CPU: the checks of arguments, and the
64-bit reference against other ways to say the same."""

from __future__ import annotations

import ctypes
import math
import shutil

import numpy as np
import pytest
import torch

import paged4_reference as ref
from test_paged import _Args, heads, i32, run_check, stub

import fast_dllm_relax_amd._lib as _lib
from fast_dllm_relax_amd.config import FastDLLMConfig
from fast_dllm_relax_amd.paged import allocate_paged_cache
from fast_dllm_relax_amd.paged4 import Paged4KVCache, allocate_paged4_cache, values_of
from fast_dllm_relax_amd.rotary import Rotary


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not available")
def test_rows_find_their_sequences(tmp_path):
    run_check(tmp_path, "seq_of_row_check")


def test_reference_codes_are_the_nearest():
    """By search over the values, and on the borders by their even code."""
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(-9, 9, 4000), ref.BORDERS, -ref.BORDERS, ref.E2M1, [0.0, -0.0, 6.99, 7.0, 1e30]])
    got = ref.encode(x)
    far = np.abs(np.abs(x)[:, None] - ref.E2M1[None, :8])
    assert (far[np.arange(x.size), got & 7] == far.min(axis=1)).all()
    on = np.isin(np.abs(x), ref.BORDERS)
    assert on.sum() >= 14 and (got[on] % 2 == 0).all()
    assert np.array_equal(got >> 3, np.signbit(x).astype(int))
    assert np.array_equal(ref.unpack(ref.pack(got[:4000])), got[:4000])


def test_reference_scales():
    for amax in (0.0, 1e-45, 2.0 ** -70, 7 * 2.0 ** -60, 6.99, 7.0, 7.01, 12.0, 14.0, 3e38):
        s = 2.0 ** float(ref.key_exponent(np.float64(amax)))
        assert (amax <= 7 * s or s == 2.0 ** 125) and (s == 2.0 ** -60 or amax > 7 * s / 2)
    x = np.random.default_rng(1).standard_normal(5000) * np.exp2(np.random.default_rng(2).integers(-60, 60, 5000))
    assert np.array_equal(ref.bf16(x), torch.from_numpy(x).to(torch.bfloat16).double().numpy())
    e = np.random.default_rng(3).integers(0, 256, (2, 5, 3, 64, 4)).astype(np.uint8)
    assert np.array_equal(ref.by_slot(ref.in_pages(e)), e)
    laid = ref.in_pages(e)
    assert laid.shape == (2, 5, 3, 4, 4, 4, 4) and laid[1, 2, 0, 37 // 16, 37 % 4, 3, 37 // 4 % 4] == e[1, 2, 0, 37, 3]


def test_cache_checks_and_dense():
    cfg = stub().cfg
    cache = allocate_paged4_cache(cfg, 5, page_size=64, device="cpu")
    assert (cache.num_layers, cache.num_pages, cache.num_kv_heads, cache.page_size) == (2, 5, 2, 64)
    assert cache.fits == (-1, 2, 2, 128, 4)
    for name in ("k", "v_scale", "num_pages", "struct"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name))
    for pages, page in ((4, 24), (0, 32)):
        with pytest.raises(ValueError):
            allocate_paged4_cache(cfg, pages, page_size=page, device="cpu")
    t = dict(k=cache.k, v=cache.v, k_scale=cache.k_scale, v_scale=cache.v_scale)
    for change in (dict(v=cache.v[:1]), dict(k=cache.k[0]), dict(k=cache.k.char()), dict(k_scale=cache.k_scale.flatten(3)),
                   dict(v_scale=cache.v_scale.half()), dict(v_scale=cache.v_scale.transpose(0, 1)), dict(k_scale=cache.k_scale[:, :4])):
        with pytest.raises(ValueError):
            Paged4KVCache(**{**t, **change})
    rng = np.random.default_rng(4)
    codes = rng.integers(0, 256, (2, *cache.k.shape)).astype(np.uint8)
    e = rng.integers(60, 180, (2, 5, 2, 64, 4)).astype(np.uint8)
    e[1, 3, 0, 5, 2] = 255
    cache.k.copy_(torch.from_numpy(codes[0]))
    cache.v.copy_(torch.from_numpy(codes[1]))
    cache.k_scale.copy_(torch.from_numpy(ref.in_pages(e)))
    cache.v_scale.copy_(torch.from_numpy(rng.uniform(0.5, 2, (2, 5, 2, 64))))
    k, v = cache.dense(1, [3, 0])
    want = ref.E2M1[ref.unpack(codes[0])] * np.repeat(ref.key_scales(e), 32, axis=-1)
    assert np.array_equal(k.double().numpy(), np.concatenate([want[1, p].transpose(1, 0, 2) for p in (3, 0)]), equal_nan=True)
    want = ref.E2M1[ref.unpack(codes[1])] * cache.v_scale.double().numpy()[..., None]
    assert np.array_equal(v.double().numpy(), np.concatenate([want[1, p].transpose(1, 0, 2) for p in (3, 0)]))
    assert torch.equal(values_of(torch.tensor([0x7f], dtype=torch.uint8)), torch.tensor([-6.0, 6.0]))


def test_append_checks():
    vm = stub()
    cache = allocate_paged4_cache(vm.cfg, 4, device="cpu")
    table, start, w = torch.zeros((2, 3), dtype=torch.int32), i32(0, 5), torch.ones(128, dtype=torch.bfloat16)
    ok = dict(k=heads(6, 2), v=heads(6, 2), cache=cache, layer=0, page_table=table, start=start)
    assert vm.paged4_append(**ok) is None
    assert vm.paged4_append(**ok, q=heads(6, 4), q_norm=w, k_norm=w, rotary=Rotary(dim=64)).shape == (6, 4, 128)
    fused = torch.zeros((6, 8, 128), dtype=torch.bfloat16)
    vm.paged4_append(**{**ok, "k": fused[:, 4:6], "v": fused[:, 6:]}, q=fused[:, :4], row_start=i32(0, 2, 5), max_rows=3, pos=start)
    assert vm.lib.seen == ["fdllm_paged4_append"] * 3
    other = allocate_paged4_cache(FastDLLMConfig(**{**vm.cfg.__dict__, "num_key_value_heads": 4}), 4, device="cpu")
    for change in (dict(k=heads(6, 3)), dict(k=heads(6, 2, torch.float16)), dict(v=heads(5, 2)), dict(cache=other),
                   dict(cache=allocate_paged_cache(vm.cfg, 4, device="cpu")), dict(k=heads(2, 6).transpose(0, 1)),
                   dict(page_table=table.long()), dict(page_table=table[0]), dict(start=start.long()), dict(start=i32(0)),
                   dict(pos=i32(1)), dict(q=heads(5, 4)), dict(q_out=heads(6, 4)), dict(q=heads(6, 4), q_out=heads(6, 2)),
                   dict(q=heads(6, 4), q_out=heads(12, 4)[::2]), dict(k=heads(5, 2), v=heads(5, 2)), dict(max_rows=2),
                   dict(row_start=i32(0, 6)), dict(layer=-1), dict(layer=2), dict(k_norm=w[:64]), dict(k_norm=w.half()),
                   dict(q_norm=w), dict(q=heads(6, 4), q_norm=w[None]), dict(rotary=(64, 1.0)), dict(k_norm=torch.ones(256, dtype=torch.bfloat16)[::2])):
        with pytest.raises(ValueError):
            vm.paged4_append(**{**ok, **change})
    assert len(vm.lib.seen) == 3
    vm.paged4_append(**{**ok, "k": heads(0, 2), "v": heads(0, 2)})
    assert len(vm.lib.seen) == 3  # no rows: nothing to launch
    # the calls of the 8-bit cache do not take this one, but the attention takes either
    with pytest.raises(ValueError):
        vm.paged_kv_append(heads(6, 2), heads(6, 2), cache, 0, table, start)
    with pytest.raises(ValueError):
        vm.paged_kv_append(heads(6, 2), heads(6, 2), cache, 0, table, start, q=heads(6, 4), q_out=heads(6, 4))
    vm.lib.seen.clear()
    ok = dict(q=heads(4, 4), cache=cache, layer=1, page_table=table, kv_len=i32(3, 4))
    assert vm.paged_attn(**ok).shape == (4, 4, 128)
    assert vm.lib.seen == ["fdllm_paged4_attn_workspace", "fdllm_paged4_attn"]
    vm.paged_attn(**{**ok, "cache": allocate_paged_cache(vm.cfg, 4, device="cpu")})
    assert vm.lib.seen[2:] == ["fdllm_paged_attn_workspace", "fdllm_paged_attn"]
    for change in (dict(q=heads(4, 2)), dict(kv_len=i32(3)), dict(cache=other), dict(layer=2), dict(max_len=-1), dict(mask_block=-1),
                   dict(out=heads(3, 4))):
        with pytest.raises(ValueError):
            vm.paged_attn(**{**ok, **change})


def test_read_checks():
    vm = stub()
    cache = allocate_paged4_cache(vm.cfg, 4, device="cpu")
    ok = dict(cache=cache, layer=1, page_table=torch.zeros((2, 3), dtype=torch.int32), start=i32(0, 5), rows=6)
    k, v = vm.paged4_read(**ok)
    assert k.shape == v.shape == (6, 2, 128)
    whole = torch.zeros((2, 1, 9, 2, 128), dtype=torch.bfloat16)  # rows of a contiguous cache
    got = vm.paged4_read(**ok, k_out=whole[0, 0, 2:8], v_out=whole[1, 0, 2:8], row_start=i32(0, 2, 6), max_rows=4)
    assert got[0].data_ptr() == whole[0, 0, 2].data_ptr()
    for change in (dict(rows=5), dict(k_out=heads(5, 2)), dict(v_out=heads(6, 4)), dict(v_out=heads(6, 2, torch.float32)),
                   dict(start=i32(1)), dict(layer=2), dict(cache=allocate_paged_cache(vm.cfg, 4, device="cpu")),
                   dict(row_start=i32(0, 6)), dict(k_out=heads(2, 6).transpose(0, 1))):
        with pytest.raises(ValueError):
            vm.paged4_read(**{**ok, **change})
    assert vm.lib.seen == ["fdllm_paged4_read"] * 2


def test_rotate_checks():
    vm = stub()
    w = torch.ones(128, dtype=torch.bfloat16)
    ok = dict(q=heads(6, 4), k=heads(6, 2), pos=i32(*range(6)))
    q, k = vm.rotate_heads(**ok)
    assert q.shape == (6, 4, 128) and k.shape == (6, 2, 128)
    assert vm.rotate_heads(ok["q"], None, 7, q_norm=w, rotary=Rotary(dim=0))[1] is None
    assert vm.rotate_heads(None, ok["k"], 7, k_norm=w)[0] is None
    for change in (dict(q=None, k=None), dict(q=heads(5, 4)), dict(k=heads(6, 4)), dict(pos=i32(1)), dict(pos=torch.zeros(6)),
                   dict(q_norm=w[:2]), dict(k_norm=w.float()), dict(q=None, q_norm=w), dict(k=None, k_out=heads(6, 2)),
                   dict(q_out=heads(5, 4)), dict(k_out=heads(6, 2, torch.float16)), dict(rotary=64), dict(q=heads(6, 4, torch.float16))):
        with pytest.raises(ValueError):
            vm.rotate_heads(**{**ok, **change})
    assert vm.lib.seen == ["fdllm_rotate_heads"] * 3
    # strides as a fused projection has them, in place among them; one row has none
    vm.lib = _Args()
    fused = torch.zeros((6, 8, 128), dtype=torch.bfloat16)
    q, k = vm.rotate_heads(fused[:, :4], fused[:, 4:6], 0, q_out=fused[:, :4])
    args = vm.lib.seen[-1]
    assert (args[2], args[4], args[12], args[14]) == (1024, 1024, 1024, 256) and q.data_ptr() == fused.data_ptr()
    vm.rotate_heads(fused[:1, :4], None, 0)
    assert (vm.lib.seen[-1][2], vm.lib.seen[-1][12]) == (512, 512)


def test_entry_points_refuse_a_null_context():
    lib, n = _lib.load(), None
    assert lib.fdllm_rotate_heads(n, n, 0, n, 0, 1, n, 0, n, n, n, n, 0, n, 0, n) == _lib.FDLLM_EINVAL
    assert lib.fdllm_paged4_append(n, n, 0, n, 0, n, 0, 1, n, 1, 1, n, 0, n, 1, 1, n, n, n, n, n, n, n) == _lib.FDLLM_EINVAL
    assert lib.fdllm_paged4_read(n, n, 0, n, 1, 1, n, 1, n, 1, 1, n, 0, n, 0, n) == _lib.FDLLM_EINVAL
    assert lib.fdllm_paged4_attn(n, n, 0, 1, n, 1, 1, n, 0, n, 1, 1, n, 0, 0, n, n, 0, n) == _lib.FDLLM_EINVAL
    assert lib.fdllm_paged4_attn_workspace(n, 1, 1, 1, 32, 1, 0) == 0


@pytest.mark.parametrize("dim", [16, 32, 64, 96, 128])
def test_rotary_frequencies(dim):
    plain = Rotary(theta=1e4, dim=dim)
    assert np.allclose(plain.frequencies, ref.frequencies(1e4, dim), rtol=1e-14) and plain.factor == 1.0
    linear = Rotary(theta=1e4, dim=dim, scaling=dict(type="linear", factor=4))
    assert np.allclose(linear.frequencies, ref.frequencies(1e4, dim) / 4, rtol=1e-14)
    # the fastest pair keeps its speed, the slowest is s times slower
    ntk = Rotary(theta=1e4, dim=dim, scaling=dict(type="ntk", factor=8))
    slow = np.array(plain.frequencies) / np.array(ntk.frequencies)
    assert abs(slow[0] - 1) < 1e-12 and abs(slow[-1] - 8) < 1e-9 and (np.diff(slow) > 0).all()
    yarn = Rotary(theta=1e4, dim=dim, scaling=dict(type="yarn", factor=8, original_len=4096))
    slow = np.array(plain.frequencies) / np.array(yarn.frequencies)
    turns = 4096 * np.array(plain.frequencies) / (2 * math.pi)
    # (the mix is by whole pairs: a pair next to the borders may lie on either side)
    assert (np.diff(slow) >= -1e-12).all() and (slow >= 1 - 1e-12).all() and (slow <= 8 + 1e-9).all()
    step = 1e4 ** (2 / dim)
    assert np.allclose(slow[turns > 32 * step], 1) and np.allclose(slow[turns < 1 / step], 8)
    assert yarn.factor == pytest.approx(0.1 * math.log(8) + 1)
    assert Rotary(dim=dim, scaling=dict(type="yarn", factor=8, original_len=64, attention_factor=1.5, beta_fast=16, beta_slow=2)).factor == 1.5
    given = Rotary(dim=dim, frequencies=plain.frequencies, factor=0.5, interleaved=True)
    assert given.frequencies == plain.frequencies and (given.factor, given.interleaved) == (0.5, True)
    s = ctypes.cast(given.struct, ctypes.POINTER(_lib.FdllmRotary)).contents
    assert [s.freq[i] for i in range(dim // 2)] == list(plain.frequencies) and (s.dim, s.interleaved, s.factor) == (dim, 1, 0.5)


def test_rotary_refusals():
    assert Rotary(dim=0).frequencies == ()
    for bad in (dict(dim=8), dict(dim=144), dict(dim=-16), dict(theta=0.0), dict(theta=math.inf), dict(factor=math.nan),
                dict(scaling=dict(type="linear")), dict(scaling=dict(type="other", factor=2)), dict(scaling=dict(type="ntk", factor=0.5)),
                dict(scaling=dict(type="linear", factor=2, original_len=5)), dict(scaling=dict(type="yarn", factor=2)),
                dict(scaling=dict(type="yarn", factor=2, original_len=64, beta_fast=1)), dict(frequencies=[1.0] * 3),
                dict(frequencies=[math.nan] * 64), dict(frequencies=[2e3] * 64), dict(frequencies=[1.0] * 64, scaling=dict(type="ntk", factor=2))):
        with pytest.raises(ValueError):
            Rotary(**bad)
    with pytest.raises(AttributeError):
        Rotary().dim = 64
