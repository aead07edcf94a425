"""The paged 8-bit cache and the token log probabilities on the CPU: index arithmetic, the checks of arguments, and the
64-bit reference against torch's own e4m3."""

from __future__ import annotations

import shutil
import subprocess
import sys

import numpy as np
import pytest
import torch

import paged_reference as ref
from conftest import ROOT

import fast_dllm_relax_amd._lib as _lib
from fast_dllm_relax_amd.config import FastDLLMConfig
from fast_dllm_relax_amd.paged import PagedKVCache, allocate_paged_cache
from fast_dllm_relax_amd.vm import HipVM

CPU = torch.device("cpu")


def run_check(tmp_path, name):
    """Compiles and runs tests/<name>.cpp, which prints ok."""
    exe = tmp_path / name
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    str(ROOT / "fast-dllm-relax_amd" / "csrc"), str(ROOT / "tests" / f"{name}.cpp"), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not available")
def test_results_over_their_queries(tmp_path):
    run_check(tmp_path, "paged_place_check")


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ is not available")
def test_index_arithmetic(tmp_path):
    exe = tmp_path / "paged_index_check"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    str(ROOT / "fast-dllm-relax_amd" / "csrc"), str(ROOT / "tests" / "paged_index_check.cpp"), "-o", str(exe)],
                   check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def test_reference_e4m3_is_torchs():
    b = torch.arange(256, dtype=torch.uint8)
    v = b.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(v, ref.E4M3, equal_nan=True)
    x = np.random.default_rng(0).standard_normal(20000) * np.exp2(np.random.default_rng(1).integers(-14, 7, 20000))
    x = np.clip(x, -448, 448).astype(np.float32)
    mid = (ref.E4M3[:126] + ref.E4M3[1:127]) / 2  # ties
    x = np.concatenate([x, mid, -mid, [0.0, -0.0, 448, -448]]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(ref.encode(x), want)


def test_reference_scale_holds_its_values():
    for amax in (0.0, 1e-45, 2.0 ** -110, 448 * 2.0 ** -100, 0.4375, 0.4376, 1.0, 447.9, 448, 448.1, 3e38):
        s = ref.scale_of(amax)
        assert amax <= 448 * s and (s == 2.0 ** -100 or amax > 448 * s / 2)


class _Calls:
    """Stands for the library: records the calls that pass the checks."""

    def __init__(self):
        self.seen = []

    def __getattr__(self, name):
        def call(*args):
            self.seen.append(name)
            return 0
        return call


class _Args(_Calls):
    """... and their arguments."""

    def __getattr__(self, name):
        def call(*args):
            if not name.endswith("_workspace"):
                self.seen.append(args)
            return 0
        return call


def stub():
    vm = object.__new__(HipVM)
    vm.cfg = FastDLLMConfig(vocab_size=64, hidden_size=128, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
                            num_key_value_heads=2, head_dim=128)
    vm.dtype, vm.torch_dtype, vm.device, vm.lib, vm.ctx = "bfloat16", torch.bfloat16, CPU, _Calls(), None
    vm._index, vm._ws_bytes, vm._fits = -1, {}, (-1, 2, 2, 128)
    vm._on_stream = lambda fn, *args: fn(*args, None)
    return vm


def heads(rows, n, dtype=torch.bfloat16):
    return torch.zeros((rows, n, 128), dtype=dtype)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_cache_checks():
    cfg = stub().cfg
    cache = allocate_paged_cache(cfg, 5, page_size=64, device="cpu")
    assert (cache.num_layers, cache.num_pages, cache.num_kv_heads, cache.page_size) == (2, 5, 2, 64)
    k, v = cache.dense(1, [0, 3])
    assert k.shape == v.shape == (128, 2, 128)
    for name in ("k", "v_scale", "num_pages", "struct"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name))
    for bad in (dict(page_size=24), dict(num_pages=0)):
        with pytest.raises(ValueError):
            allocate_paged_cache(cfg, bad.get("num_pages", 4), page_size=bad.get("page_size", 32), device="cpu")
    t = dict(k=cache.k, v=cache.v, k_scale=cache.k_scale, v_scale=cache.v_scale)
    for change in (dict(v=cache.k), dict(k=cache.k[0]), dict(k=cache.k.float()), dict(k_scale=cache.k_scale.double()),
                   dict(v_scale=cache.v_scale[:1]), dict(k_scale=cache.k_scale.transpose(0, 1)),
                   dict(k=cache.k[:, :, :, ::2], v=cache.v[:, :, :, :, ::2])):
        with pytest.raises(ValueError):
            PagedKVCache(**{**t, **change})


def test_append_checks():
    vm = stub()
    cache = allocate_paged_cache(vm.cfg, 4, device="cpu")
    table, start = torch.zeros((2, 3), dtype=torch.int32), i32(0, 5)
    ok = dict(k=heads(6, 2), v=heads(6, 2), cache=cache, layer=0, page_table=table, start=start)
    assert vm.paged_kv_append(**ok) is None
    assert vm.paged_kv_append(**ok, q=heads(6, 4)).shape == (6, 4, 128)
    fused = torch.zeros((6, 8, 128), dtype=torch.bfloat16)
    vm.paged_kv_append(**{**ok, "k": fused[:, 4:6], "v": fused[:, 6:]}, q=fused[:, :4], row_start=i32(0, 2, 5), max_rows=3)
    assert vm.lib.seen == ["fdllm_paged_kv_append"] * 3
    other = allocate_paged_cache(FastDLLMConfig(**{**vm.cfg.__dict__, "num_key_value_heads": 4}), 4, device="cpu")
    for change in (dict(k=heads(6, 3)), dict(k=heads(6, 2, torch.float16)), dict(v=heads(5, 2)), dict(cache=other),
                   dict(k=heads(2, 6).transpose(0, 1)), dict(k=torch.zeros((6, 2, 256), dtype=torch.bfloat16)[:, :, ::2]),
                   dict(page_table=table.long()), dict(page_table=table[0]), dict(page_table=table.t()), dict(start=start.long()),
                   dict(start=i32(0)), dict(live=i32(1, 2, 3)), dict(pos=i32(1)), dict(q=heads(5, 4)), dict(q_out=heads(6, 4)),
                   dict(q=heads(6, 4), q_out=heads(6, 2)), dict(k=heads(5, 2), v=heads(5, 2)), dict(max_rows=2),
                   dict(row_start=i32(0, 6)), dict(row_start=i32(0, 3, 6), max_rows=-1), dict(q=heads(6, 4), q_out=heads(12, 4)[::2]),
                   dict(layer=-1), dict(layer=2), dict(layer=2 ** 32), dict(layer=2 ** 32, q=heads(6, 4), q_out=heads(6, 4))):
        with pytest.raises(ValueError):
            vm.paged_kv_append(**{**ok, **change})
        # and with all that a step passes, whose checks come first and at once
        if not {"q", "q_out"} & set(change):
            with pytest.raises(ValueError):
                vm.paged_kv_append(**{**ok, "q": heads(6, 4), "q_out": heads(6, 4), "live": start, **change})
    assert len(vm.lib.seen) == 3
    vm.paged_kv_append(**{**ok, "k": heads(0, 2), "v": heads(0, 2)})
    assert len(vm.lib.seen) == 3  # no rows: nothing to launch


def test_a_single_row_has_no_stride():
    """One row's tensor may say any stride to the next: the library gets the row's own length."""
    vm = stub()
    vm.lib = _Args()
    cache = allocate_paged_cache(vm.cfg, 4, device="cpu")
    table, zero = torch.zeros((1, 3), dtype=torch.int32), i32(0)
    turned = lambda n: torch.zeros((n, 1, 128), dtype=torch.bfloat16).transpose(0, 1)  # noqa: E731
    assert turned(4).stride() == (128, 128, 1)
    for q in (None, turned(4)):
        for q_out in (None, None if q is None else heads(1, 4)):
            vm.paged_kv_append(turned(2), turned(2), cache, 0, table, zero, q=q, q_out=q_out)
            args = vm.lib.seen[-1]
            assert (args[2], args[4], args[6]) == (0 if q is None else 512, 256, 256)
    vm.paged_attn(turned(4), cache, 0, table, zero)
    assert vm.lib.seen[-1][2] == 512


def test_attention_checks():
    vm = stub()
    cache = allocate_paged_cache(vm.cfg, 4, device="cpu")
    ok = dict(q=heads(4, 4), cache=cache, layer=1, page_table=torch.zeros((2, 3), dtype=torch.int32), kv_len=i32(3, 4))
    assert vm.paged_attn(**ok).shape == (4, 4, 128)
    vm.paged_attn(**ok, out=heads(4, 4), row_start=i32(0, 1, 4), max_rows=3)
    for change in (dict(q=heads(4, 2)), dict(q=heads(3, 4)), dict(kv_len=i32(3)), dict(kv_len=torch.zeros(2)), dict(max_len=-1),
                   dict(out=heads(3, 4)), dict(out=heads(4, 4, torch.float16)), dict(row_start=i32(0, 1)), dict(layer=2 ** 32),
                   dict(mask_block=-1), dict(mask_block=2 ** 32)):
        with pytest.raises(ValueError):
            vm.paged_attn(**{**ok, **change})


def test_logprobs_checks():
    vm = stub()
    x = torch.zeros((1, 3, 50))
    got = vm.token_logprobs(x, torch.zeros((1, 3), dtype=torch.int32), top_n=4)
    assert [tuple(t.shape) for t in got] == [(1, 3), (1, 3), (1, 3, 4), (1, 3, 4)]
    vm.token_logprobs(torch.zeros((1, 3, 60))[:, :, :50])
    for bad in (dict(logits=x[0]), dict(logits=x.double()), dict(logits=torch.zeros((2, 3, 50))), dict(logits=x.transpose(1, 2)),
                dict(logits=torch.zeros((1, 1, 50)).expand(1, 3, 50)), dict(ids=torch.zeros((1, 3))), dict(ids=torch.zeros((3,), dtype=torch.int32)),
                dict(top_n=33), dict(top_n=-1), dict(logits=torch.zeros((1, 3, 5)), top_n=6)):
        with pytest.raises(ValueError):
            vm.token_logprobs(**{"logits": x, **bad})
    assert vm.token_logprobs(torch.zeros((1, 0, 50)))[1].shape == (1, 0)


def test_entry_points_refuse_a_null_context():
    lib = _lib.load()
    assert lib.fdllm_paged_kv_append(None, None, 0, None, 0, None, 0, 1, None, 1, 1, None, 0, None, 1, 1, None, None, None, None,
                                     None) == _lib.FDLLM_EINVAL
    assert lib.fdllm_paged_attn(None, None, 0, 1, None, 1, 1, None, 0, None, 1, 1, None, 0, 0, None, None, 0, None) == _lib.FDLLM_EINVAL
    assert lib.fdllm_token_logprobs(None, None, 0, 1, 1, 1, None, 0, None, None, None, None, None, 0, None) == _lib.FDLLM_EINVAL
    assert lib.fdllm_paged_attn_workspace(None, 1, 1, 1, 32, 1, 0) == 0
    assert lib.fdllm_token_logprobs_workspace(None, 1, 1, 0) == 0


def test_a_single_row_of_a_fused_projection():
    """... also where that is a longer one, as a slice of a fused projection has, no multiple of 8, and where the queries are
    rotated where they lie."""
    vm = stub()
    vm.lib = _Args()
    cache = allocate_paged_cache(vm.cfg, 4, device="cpu")
    table, zero = torch.zeros((1, 3), dtype=torch.int32), i32(0)
    for ld in (1024, 1203):
        fused = torch.zeros(2 * ld, dtype=torch.bfloat16).as_strided((1, 8, 128), (ld, 128, 1))
        q, k, v = fused[:, :4], fused[:, 4:6], fused[:, 6:]
        assert q.stride() == (ld, 128, 1) and q.is_contiguous()
        for q_out in (None, heads(1, 4), q):
            got = vm.paged_kv_append(k, v, cache, 0, table, zero, q=q, q_out=q_out)
            args = vm.lib.seen[-1]
            assert (args[1], args[2], args[4], args[6]) == (q.data_ptr(), 512, 256, 256) and args[-2] == got.data_ptr()
            assert q_out is None or got is q_out


def test_the_module_imports_without_torchs_gpu_names():
    """A torch built for the CPU alone has none of the names that the calls' short way to device and stream uses."""
    code = ("import torch\n"
            "del torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream\n"
            "import __graft_entry__\n"
            "__graft_entry__.load_package()\n"
            "from fast_dllm_relax_amd import vm\n"
            "assert vm._current_device is torch.cuda.current_device\n"
            "torch.cuda.current_stream = lambda index: type('S', (), {'cuda_stream': 100 + index})\n"
            "assert vm._raw_stream(3) == 103\n"
            "print('ok')\n")
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=ROOT)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def test_bounds_of_key_bytes_tell_a_rotation_in_fp32():
    """The bounds leave open less than one byte in 10^5, the bytes of a 64-bit rotation lie within them, and those of
    a rotation whose products and sums are in fp32 do not all."""
    rng = np.random.default_rng(40)
    n, page = 8192, 32
    x = torch.from_numpy(rng.standard_normal((n, 2, 128)).astype(np.float32)).bfloat16().double().numpy()
    pos = np.arange(n)
    table = np.arange(n // page)[None]

    def stored(rows):
        pages, scale = np.zeros((n // page, 2, page, 128), np.uint8), np.ones((n // page, 2))
        ref.append(pages, scale, table, page, [0], [0], [rows])
        return pages, scale

    (lo, s_lo), (hi, s_hi) = (stored(b) for b in ref.rotation_bounds(x, pos, 1e6))
    assert np.array_equal(s_lo, s_hi) and (lo != hi).mean() < 1e-5
    exact = ref.rotate(x, pos[:, None, None], 1e6)
    for rows in (exact, exact.astype(np.float32).astype(np.float64)):
        assert not ref.outside(stored(rows)[0], lo, hi).any()
    a = pos[:, None, None] * 1e6 ** (-np.arange(64) / 64.0)
    c, s, y = np.cos(a).astype(np.float32), np.sin(a).astype(np.float32), x.astype(np.float32)
    single = np.concatenate([y[..., :64] * c - y[..., 64:] * s, y[..., 64:] * c + y[..., :64] * s], axis=-1)
    assert single.dtype == np.float32 and ref.outside(stored(single.astype(np.float64))[0], lo, hi).any()
