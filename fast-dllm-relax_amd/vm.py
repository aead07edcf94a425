"""The nine-entry-point function table over libfdllm.so.

``HipVM`` stands where the reference holds ``tvm.relax.VirtualMachine`` (fast_dllm_relax/runners.py:614-615):
``vm["forward_cached"](embedded, k_cache, v_cache, cache_offset, prefix_len)`` and so on for every name of
REQUIRED_FNS (export_utils.py:13-17), plus ``get_confidence_m{rows}`` (model/metal.py:505-528).
Tensors are torch device tensors (PyTorch owns the memory); the packed weights are bound once at
construction instead of being passed on every call.  Work runs on torch's current stream, the stream
the reference's attention callbacks use (runtime.py:19-27).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib, paged
from .config import FastDLLMConfig
from .params import TORCH_DTYPES, param_names

REQUIRED_FNS = (
    "embed", "forward_hidden", "get_logits", "build_prefix_cache", "forward_cached",
    "forward_block_partial_rp0", "forward_block_partial_rp8",
    "forward_block_partial_rp16", "forward_block_partial_rp24",
)


_LOGITS_TYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.LOGITS_F32}


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# the current device and a device's current stream, without the objects and checks around them in torch.cuda, where torch has
# these names (a build for the CPU alone imports this module too)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


class HipVM:
    def __init__(self, cfg: FastDLLMConfig, params: list[torch.Tensor], *, dtype: str = "bfloat16",
                 max_rows: int = 64):
        if dtype not in TORCH_DTYPES:
            raise ValueError(f"unsupported dtype {dtype!r}")
        self.cfg = cfg
        self.dtype = dtype
        self.torch_dtype = TORCH_DTYPES[dtype]
        self.lib = _lib.load()
        c = _lib.FdllmConfig(cfg.vocab_size, cfg.hidden_size, cfg.intermediate_size, cfg.num_hidden_layers,
                             cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim, cfg.rms_norm_eps,
                             cfg.rope_theta, int(cfg.tie_word_embeddings), cfg.bd_size,
                             _lib.DTYPE_BF16 if dtype == "bfloat16" else _lib.DTYPE_F16, max_rows)
        h = ctypes.c_void_p()
        _lib.check(self.lib.fdllm_create(ctypes.byref(c), ctypes.byref(h)))
        self.ctx = h
        self._index = torch.cuda.current_device()
        self.device = torch.device("cuda", self._index)
        self._fits = (self._index, cfg.num_hidden_layers, cfg.num_key_value_heads, cfg.head_dim)  # a paged cache's, to be this model's
        self._ws_bytes: dict = {}
        names = [self.lib.fdllm_param_name(h, i).decode() for i in range(self.lib.fdllm_num_params(h))]
        if names != param_names(cfg):
            raise RuntimeError("libfdllm parameter order differs from params.param_names")
        self.bind(params)

    @classmethod
    def from_artifact(cls, artifact_dir, *, max_rows: int = 64, device: str = "cuda", **config_overrides) -> "HipVM":
        """A function table over the weights of a reference artifact directory (the params npz, names,
        dtype and KV-cache manifest of scripts/export_cuda.py; runners.py:597-639 loads the same files)."""
        from .params import config_from_artifact, load_artifact

        cfg = config_from_artifact(artifact_dir, **config_overrides)
        params, dtype = load_artifact(artifact_dir, cfg, device=device)
        return cls(cfg, params, dtype=dtype, max_rows=max_rows)

    def bind(self, params: list[torch.Tensor]) -> None:
        names = param_names(self.cfg)
        if len(params) != len(names):
            raise ValueError(f"expected {len(names)} params, got {len(params)}")
        for n, p in zip(names, params):
            if not p.is_cuda or p.dtype != self.torch_dtype or not p.is_contiguous():
                raise ValueError(f"param {n} must be a contiguous {self.torch_dtype} device tensor")
        self.params = list(params)
        arr = (ctypes.c_void_p * len(params))(*[p.data_ptr() for p in params])
        _lib.check(self.lib.fdllm_bind_weights(self.ctx, arr, len(params)))

    def close(self) -> None:
        if getattr(self, "ctx", None):
            self.lib.fdllm_destroy(self.ctx)
            self.ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 -- interpreter shutdown
            pass

    # ---- function table -------------------------------------------------------------------
    def __getitem__(self, name: str):
        if name in REQUIRED_FNS:
            return getattr(self, name)
        if name.startswith("get_confidence_m"):
            return self.get_confidence
        raise KeyError(name)

    def _check_cache(self, k: torch.Tensor, v: torch.Tensor) -> int:
        c = self.cfg
        exp = (c.num_hidden_layers, 1, k.shape[2], c.num_key_value_heads, c.head_dim)
        for t in (k, v):
            if tuple(t.shape) != exp or t.dtype != self.torch_dtype or not t.is_contiguous() or not t.is_cuda:
                raise ValueError(f"KV cache must be a contiguous {self.torch_dtype} device tensor of shape {exp}")
        if v.shape != k.shape:
            raise ValueError("k_cache and v_cache shapes differ")
        return int(k.shape[2])

    def _check_rows(self, x: torch.Tensor) -> int:
        if x.dim() != 3 or x.shape[0] != 1 or x.shape[2] != self.cfg.hidden_size or x.dtype != self.torch_dtype:
            raise ValueError(f"expected [1, rows, {self.cfg.hidden_size}] {self.torch_dtype}, got "
                             f"{tuple(x.shape)} {x.dtype}")
        if not x.is_contiguous():
            raise ValueError("activation tensor must be contiguous")
        return int(x.shape[1])

    def embed(self, input_ids: torch.Tensor) -> torch.Tensor:
        """ids [seq_len] int32 -> [seq_len, hidden] (cuda.py:698-699)."""
        ids = input_ids.to(dtype=torch.int32).contiguous()
        n = ids.numel()
        if n > 0:
            lo, hi = int(ids.min()), int(ids.max())
            if lo < 0 or hi >= self.cfg.vocab_size:
                raise ValueError(f"token id out of range [0, {self.cfg.vocab_size}): {lo if lo < 0 else hi}")
        out = torch.empty((n, self.cfg.hidden_size), dtype=self.torch_dtype, device=ids.device)
        _lib.check(self.lib.fdllm_embed(self.ctx, _ptr(ids), n, _ptr(out), _stream()))
        return out

    def embed_unchecked(self, ids: torch.Tensor) -> torch.Tensor:
        """embed of ids the caller has range-checked on the host (no device readback)."""
        out = torch.empty((ids.numel(), self.cfg.hidden_size), dtype=self.torch_dtype, device=ids.device)
        _lib.check(self.lib.fdllm_embed(self.ctx, _ptr(ids), ids.numel(), _ptr(out), _stream()))
        return out

    def forward_hidden(self, input_embed: torch.Tensor, attention_bias: torch.Tensor | None) -> torch.Tensor:
        s = self._check_rows(input_embed)
        if attention_bias is not None:
            if tuple(attention_bias.shape) != (1, 1, s, s) or attention_bias.dtype != torch.float32:
                raise ValueError(f"attention_bias must be [1, 1, {s}, {s}] float32")
            attention_bias = attention_bias.contiguous()
        out = torch.empty_like(input_embed)
        _lib.check(self.lib.fdllm_forward_hidden(self.ctx, _ptr(input_embed), s, _ptr(attention_bias), _ptr(out),
                                                 _stream()))
        return out

    def get_logits(self, hidden_states: torch.Tensor) -> torch.Tensor:
        rows = self._check_rows(hidden_states)
        out = torch.empty((1, rows, self.cfg.vocab_size), dtype=torch.float32, device=hidden_states.device)
        _lib.check(self.lib.fdllm_get_logits(self.ctx, _ptr(hidden_states), rows, _ptr(out), _stream()))
        return out

    def build_prefix_cache(self, prefix_embed: torch.Tensor, prefix_bias: torch.Tensor | None,
                           k_cache: torch.Tensor, v_cache: torch.Tensor):
        p = self._check_rows(prefix_embed)
        cap = self._check_cache(k_cache, v_cache)
        if prefix_bias is not None:
            if tuple(prefix_bias.shape) != (1, 1, p, p) or prefix_bias.dtype != torch.float32:
                raise ValueError(f"prefix_bias must be [1, 1, {p}, {p}] float32")
            prefix_bias = prefix_bias.contiguous()
        _lib.check(self.lib.fdllm_build_prefix_cache(self.ctx, _ptr(prefix_embed), p, _ptr(prefix_bias),
                                                     _ptr(k_cache), _ptr(v_cache), cap, _stream()))
        return k_cache, v_cache

    def forward_cached(self, active_embed: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                       cache_offset: torch.Tensor, prefix_len: int) -> torch.Tensor:
        rows = self._check_rows(active_embed)
        cap = self._check_cache(k_cache, v_cache)
        off = self._offset(cache_offset)
        out = torch.empty_like(active_embed)
        _lib.check(self.lib.fdllm_forward_cached(self.ctx, _ptr(active_embed), rows, _ptr(k_cache), _ptr(v_cache),
                                                 cap, _ptr(off), int(prefix_len), _ptr(out), _stream()))
        return out

    def _offset(self, cache_offset: torch.Tensor) -> torch.Tensor:
        if cache_offset.numel() != 1 or cache_offset.dtype != torch.int32 or not cache_offset.is_cuda:
            raise ValueError("cache_offset must be a 0-d int32 device tensor")
        return cache_offset

    def _partial(self, rp: int, active_embed, k_cache, v_cache, cache_offset, prefix_len):
        rows = self._check_rows(active_embed)
        cap = self._check_cache(k_cache, v_cache)
        off = self._offset(cache_offset)
        out = torch.empty_like(active_embed)
        _lib.check(self.lib.fdllm_forward_block_partial(self.ctx, rp, _ptr(active_embed), rows, _ptr(k_cache),
                                                        _ptr(v_cache), cap, _ptr(off), int(prefix_len), _ptr(out),
                                                        _stream()))
        return out

    def forward_block_partial_rp0(self, active_embed, k_cache, v_cache, cache_offset, prefix_len):
        return self._partial(0, active_embed, k_cache, v_cache, cache_offset, prefix_len)

    def forward_block_partial_rp8(self, active_embed, k_cache, v_cache, cache_offset, prefix_len):
        return self._partial(8, active_embed, k_cache, v_cache, cache_offset, prefix_len)

    def forward_block_partial_rp16(self, active_embed, k_cache, v_cache, cache_offset, prefix_len):
        return self._partial(16, active_embed, k_cache, v_cache, cache_offset, prefix_len)

    def forward_block_partial_rp24(self, active_embed, k_cache, v_cache, cache_offset, prefix_len):
        return self._partial(24, active_embed, k_cache, v_cache, cache_offset, prefix_len)

    # ---- batched steps (no reference counterpart: the reference is batch 1, cuda.py:796-836) ----
    # ---- the reference's attention callbacks (runtime.py:19-80) ------------------------------
    def _check_bsnh(self, t: torch.Tensor, heads: int, name: str) -> int:
        hd = self.cfg.head_dim
        if (t.dim() != 4 or t.shape[0] != 1 or t.shape[2] != heads or t.shape[3] != hd or t.dtype != self.torch_dtype
                or not t.is_cuda or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {self.torch_dtype} device tensor [1, rows, {heads}, {hd}], "
                             f"got {tuple(t.shape)} {t.dtype}")
        return int(t.shape[1])

    def kv_write(self, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, layer: int,
                 start: int):
        """fast_dllm.kv_write (runtime.py:76-80): k / v [1, rows, nkv, hd] into cache rows [start, + rows) of
        `layer`, byte for byte; returns the caches (aliases)."""
        nkv = self.cfg.num_key_value_heads
        rows = self._check_bsnh(k, nkv, "k")
        if self._check_bsnh(v, nkv, "v") != rows:
            raise ValueError("k and v rows differ")
        cap = self._check_cache(k_cache, v_cache)
        _lib.check(self.lib.fdllm_kv_write(self.ctx, _ptr(k), _ptr(v), rows, _ptr(k_cache), _ptr(v_cache), cap,
                                           int(layer), int(start), _stream()))
        return k_cache, v_cache

    def attn_inplace(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor,
                     v_cache: torch.Tensor, layer: int, prefix_len: int, write_rel: int, attend_rel: int):
        """fast_dllm.attn_inplace (runtime.py:63-73): write k / v at cache rows [prefix_len + write_rel,
        + rows), then attend the rotated queries q [1, rows, nq, hd] over rows [0, prefix_len + attend_rel)
        with no mask.  Returns (k_cache, v_cache, out [1, rows, nq, hd])."""
        # the host's part of this call is longer than its kernels at a block's rows, so what passes every check
        # is recognised in one go (four calls of 32 rows over 2080 keys 64.3 -> 57.9 us); anything else takes the checks
        # one by one, for their errors
        c, td, ts = self.cfg, self.torch_dtype, (q, k, v, k_cache, v_cache)
        qs, ks, cs, hd, nkv = q.shape, k.shape, k_cache.shape, c.head_dim, c.num_key_value_heads
        if (len(qs) == 4 and len(cs) == 5 and qs == (1, qs[1], c.num_attention_heads, hd) and ks == (1, qs[1], nkv, hd)
                and v.shape == ks and cs == (c.num_hidden_layers, 1, cs[2], nkv, hd) and v_cache.shape == cs
                and all(t.dtype is td and t.is_cuda and t.is_contiguous() for t in ts)):
            rows, cap = qs[1], cs[2]
        else:
            rows = self._check_bsnh(q, c.num_attention_heads, "q")
            if self._check_bsnh(k, nkv, "k") != rows or self._check_bsnh(v, nkv, "v") != rows:
                raise ValueError("q, k and v rows differ")
            cap = self._check_cache(k_cache, v_cache)
        out = torch.empty_like(q)
        rc = self.lib.fdllm_attn_inplace(self.ctx, q.data_ptr(), k.data_ptr(), v.data_ptr(), rows, k_cache.data_ptr(),
                                         v_cache.data_ptr(), cap, int(layer), int(prefix_len), int(write_rel),
                                         int(attend_rel), out.data_ptr(), _stream())
        if rc:
            _lib.check(rc)
        return k_cache, v_cache, out

    # ---- the paged 8-bit cache and scoring (no reference counterpart; include/fdllm.h) --------
    def _on_stream(self, fn, *args) -> None:
        """fn(*args, stream) on the current stream of the context's device, whichever device is current."""
        index = self._index
        if _current_device() == index:
            rc = fn(*args, _raw_stream(index))
        else:
            with torch.cuda.device(index):
                rc = fn(*args, _raw_stream(index))
        if rc:
            _lib.check(rc)

    def _workspace(self, key: tuple) -> tuple[torch.Tensor | None, int]:
        """A workspace of a call's own (calls on several streams, and graphs, share none) and its bytes, which depend on the
        function and sizes in key = (function, *sizes) alone and are remembered by them."""
        need = self._ws_bytes.get(key)
        if need is None:
            if len(self._ws_bytes) > 4096:
                self._ws_bytes.clear()
            need = self._ws_bytes[key] = getattr(self.lib, key[0])(self.ctx, *key[1:])
        return (torch.empty(need, dtype=torch.uint8, device=self.device) if need else None), need

    def paged_kv_append(self, k: torch.Tensor, v: torch.Tensor, cache: paged.PagedKVCache, layer: int,
                        page_table: torch.Tensor, start: torch.Tensor, *, live: torch.Tensor | None = None,
                        pos: torch.Tensor | None = None, q: torch.Tensor | None = None, q_out: torch.Tensor | None = None,
                        row_start: torch.Tensor | None = None, max_rows: int | None = None):
        """Appends k / v [rows, nkv, hd] (any row stride) of nseq = len(page_table) sequences to `layer` of a paged 8-bit
        cache, sequence b's rows at positions start[b], start[b] + 1, ..., the keys rotated by pos[b] + i (default: their
        positions); returns the queries q [rows, nq, hd] rotated alike (q_out, or a new tensor), None without q.
        live: positions each sequence held before (default: start).  row_start int32 [nseq + 1] and max_rows describe
        sequences with different numbers of rows; max_rows, a bound on them, should be tight: without it there are workgroups
        for all rows in every sequence (24 prompts of up to 509 rows: 29.6 us instead of 15.2) (fdllm_paged_kv_append)."""
        # (one condition for what a step passes, on its own device: the host's part of this call is longer than its kernel;
        # anything else takes the checks one by one, for their errors)
        td, index, i32, hd = self.torch_dtype, self._index, torch.int32, self.cfg.head_dim
        ks, kst, vst, ts = k.shape, k.stride(), v.stride(), page_table.shape
        nq, nkv = self.cfg.num_attention_heads, self.cfg.num_key_value_heads
        rows, nseq = ks[0] if ks else 0, ts[0] if ts else 0
        if (rows and nseq and q is not None and q_out is not None and ks == (rows, nkv, hd) and v.shape == ks
                and kst[1:] == vst[1:] == (hd, 1) and k.dtype is td and v.dtype is td and cache.fits == self._fits
                and k.get_device() == v.get_device() == index and q.shape == q_out.shape == (rows, nq, hd) and q.dtype is td
                and q_out.dtype is td and q.get_device() == q_out.get_device() == index and q_out.is_contiguous()
                and len(ts) == 2 and ts[1] and page_table.dtype is i32 and page_table.get_device() == index
                and start.shape == (nseq,) and start.dtype is i32 and start.get_device() == index and start.is_contiguous()
                and (live is None or (live.shape == (nseq,) and live.dtype is i32 and live.get_device() == index
                                      and live.is_contiguous()))
                and (pos is None or paged.is_i32(pos, nseq, index)) and 0 <= layer < cache.num_layers
                and (most := rows // nseq if row_start is None and max_rows is None and rows % nseq == 0
                     else paged.most_rows(rows, nseq, row_start, max_rows, index)) >= 0):
            qst, tst = q.stride(), page_table.stride()
            if qst[1:] == (hd, 1) and tst[1] == 1:
                # (a single row has no stride, whatever its tensor says: paged.row_stride)
                ldq, ldk, ldv = (qst[0], kst[0], vst[0]) if rows > 1 else (nq * hd, nkv * hd, nkv * hd)
                self._on_stream(self.lib.fdllm_paged_kv_append, self.ctx, q.data_ptr(), ldq, k.data_ptr(), ldk, v.data_ptr(), ldv,
                                rows, None if row_start is None else row_start.data_ptr(), nseq, most, cache.struct, layer,
                                page_table.data_ptr(), ts[1], tst[0], start.data_ptr(), None if live is None else live.data_ptr(),
                                None if pos is None else pos.data_ptr(), q_out.data_ptr())
                return q_out
        rows = paged.check_heads(k, nkv, hd, td, index, "k")
        if paged.check_heads(v, nkv, hd, td, index, "v") != rows:
            raise ValueError("k and v rows differ")
        paged.check_cache(cache, layer, self._fits)
        nseq, width, table_ld = paged.check_table(page_table, index)
        max_rows = paged.sequence_rows(rows, nseq, row_start, max_rows, index)
        paged.check_i32(start, nseq, index, "start")
        if live is not None:
            paged.check_i32(live, nseq, index, "live")
        if pos is not None:
            paged.check_i32(pos, nseq, index, "pos")
        ldq = 0
        if q is not None:
            if paged.check_heads(q, nq, hd, td, index, "q") != rows:
                raise ValueError("q and k rows differ")
            if q_out is None:
                q_out = torch.empty((rows, nq, hd), dtype=td, device=self.device)
            elif paged.check_heads(q_out, nq, hd, td, index, "q_out") != rows or not q_out.is_contiguous():
                raise ValueError(f"q_out must be contiguous, of {rows} rows")
            ldq = paged.row_stride(q)
        elif q_out is not None:
            raise ValueError("q_out without q")
        if rows:
            self._on_stream(self.lib.fdllm_paged_kv_append, self.ctx, _ptr(q), ldq, k.data_ptr(), paged.row_stride(k),
                            v.data_ptr(), paged.row_stride(v), rows, _ptr(row_start), nseq, max_rows, cache.struct, layer,
                            page_table.data_ptr(), width, table_ld, start.data_ptr(), _ptr(live), _ptr(pos), _ptr(q_out))
        return q_out

    def paged_attn(self, q: torch.Tensor, cache: paged.PagedKVCache, layer: int, page_table: torch.Tensor,
                   kv_len: torch.Tensor, *, mask_block: int = 0, max_len: int | None = None,
                   row_start: torch.Tensor | None = None, max_rows: int | None = None, out: torch.Tensor | None = None):
        """Attention of the rotated queries q [rows, nq, hd] of nseq = len(page_table) sequences over positions
        [0, kv_len[b]) of `layer` of a paged 8-bit cache; returns out [rows, nq, hd].  mask_block: 0 none, 1 causal, B
        block-causal, the last row of a sequence being position kv_len[b] - 1.  max_len: a bound on kv_len (host) that the
        launches are planned for (default, and 0: what the table holds); row_start, max_rows as in paged_kv_append (without
        max_rows a call may also miss the split of long contexts over workgroups); out may be q
        where q is contiguous (fdllm_paged_attn)."""
        # (checked in one condition first, as in paged_kv_append)
        td, index, nq, hd = self.torch_dtype, self._index, self.cfg.num_attention_heads, self.cfg.head_dim
        shape, qst, ts, tst, i32 = q.shape, q.stride(), page_table.shape, page_table.stride(), torch.int32
        rows, nseq = shape[0] if shape else 0, ts[0] if ts else 0
        max_len = 0 if max_len is None else int(max_len)
        if (rows and nseq and shape == (rows, nq, hd) and qst[1:] == (hd, 1) and q.dtype is td and q.get_device() == index
                and cache.fits == self._fits and 0 <= layer < cache.num_layers and len(ts) == 2 and ts[1] and tst[1] == 1
                and page_table.dtype is i32 and page_table.get_device() == index and kv_len.shape == (nseq,) and kv_len.dtype is i32
                and kv_len.get_device() == index and kv_len.is_contiguous() and 0 <= max_len <= 2 ** 31 and 0 <= mask_block < 2 ** 31
                and (out is None or (out.shape == shape and out.dtype is td and out.get_device() == index and out.is_contiguous()))
                and (most := rows // nseq if row_start is None and max_rows is None and rows % nseq == 0
                     else paged.most_rows(rows, nseq, row_start, max_rows, index)) >= 0):
            width, table_ld, max_rows = ts[1], tst[0], most
        else:
            rows = paged.check_heads(q, nq, hd, td, index, "q")
            paged.check_cache(cache, layer, self._fits)
            nseq, width, table_ld = paged.check_table(page_table, index)
            max_rows = paged.sequence_rows(rows, nseq, row_start, max_rows, index)
            paged.check_i32(kv_len, nseq, index, "kv_len")
            if out is not None and (paged.check_heads(out, nq, hd, td, index, "out") != rows or not out.is_contiguous()):
                raise ValueError(f"out must be contiguous, of {rows} rows")
            if max_len < 0 or not 0 <= mask_block < 2 ** 31:
                raise ValueError(f"max_len and mask_block must be whole numbers of at most 31 bits, got {max_len} and {mask_block}")
            max_len = min(max_len, 2 ** 31)
        if out is None:
            out = torch.empty((rows, nq, hd), dtype=td, device=self.device)
        if rows:
            ws, need = self._workspace(("fdllm_paged_attn_workspace", rows, nseq, max_rows, cache.page_size, width, max_len))
            self._on_stream(self.lib.fdllm_paged_attn, self.ctx, q.data_ptr(), qst[0] if rows > 1 else nq * hd, rows,
                            None if row_start is None else row_start.data_ptr(), nseq, max_rows, cache.struct, layer,
                            page_table.data_ptr(), width, table_ld, kv_len.data_ptr(), max_len, mask_block, out.data_ptr(),
                            None if ws is None else ws.data_ptr(), need)
        return out

    def token_logprobs(self, logits: torch.Tensor, ids: torch.Tensor | None = None, *, top_n: int = 0):
        """Of logits [1, rows, vocab] (float32, bfloat16 or float16; any row stride): (log probabilities of ids [1, rows]
        int32, 0 where an id is negative, None without ids; entropy [1, rows]; ids [1, rows, top_n] int32 and log
        probabilities of each row's top_n most probable tokens, equal ones by index) (fdllm_token_logprobs)."""
        dev, index, shape, strides = self.device, self._index, logits.shape, logits.stride()
        kind = _LOGITS_TYPES.get(logits.dtype)
        if len(shape) != 3 or shape[0] != 1 or kind is None or logits.get_device() != index:
            raise ValueError(f"logits must be a float32, bfloat16 or float16 tensor [1, rows, vocab] on {dev}, got "
                             f"{tuple(shape)} {logits.dtype} on {logits.device}")
        _, rows, vocab = shape
        ld = strides[1] if rows > 1 else vocab
        if (vocab > 1 and strides[2] != 1) or ld < vocab:
            raise ValueError(f"a row of logits must be contiguous and apart from the next, got strides {strides}")
        if ids is not None and (ids.shape != (1, rows) or ids.dtype is not torch.int32 or ids.get_device() != index
                                or not ids.is_contiguous()):
            raise ValueError(f"ids must be a contiguous int32 tensor [1, {rows}] on {dev}, got {tuple(ids.shape)} {ids.dtype} "
                             f"on {ids.device}")
        if not 0 <= top_n <= min(32, vocab):
            raise ValueError(f"top_n {top_n} outside [0, {min(32, vocab)}]")
        entropy = torch.empty(1, rows, dtype=torch.float32, device=dev)
        logprob = torch.empty_like(entropy) if ids is not None else None
        top = torch.empty(1, rows, top_n, dtype=torch.float32, device=dev)
        top_ids = torch.empty_like(top, dtype=torch.int32)
        if rows:
            ws, need = self._workspace(("fdllm_token_logprobs_workspace", rows, vocab, top_n))
            self._on_stream(self.lib.fdllm_token_logprobs, self.ctx, logits.data_ptr(), kind, rows, vocab, ld, _ptr(ids), top_n,
                            _ptr(logprob), entropy.data_ptr(), top_ids.data_ptr(), top.data_ptr(), _ptr(ws), need)
        return logprob, entropy, top_ids, top

    def _check_batch_cache(self, k: torch.Tensor, v: torch.Tensor, nseq: int) -> int:
        c = self.cfg
        exp = (c.num_hidden_layers, nseq, k.shape[2] if k.dim() == 5 else -1, c.num_key_value_heads, c.head_dim)
        for t in (k, v):
            if tuple(t.shape) != exp or t.dtype != self.torch_dtype or not t.is_contiguous() or not t.is_cuda:
                raise ValueError(f"batched KV cache must be a contiguous {self.torch_dtype} device tensor of shape {exp}")
        return int(k.shape[2])

    def _check_batch_rows(self, x: torch.Tensor) -> tuple[int, int]:
        if x.dim() != 3 or x.shape[2] != self.cfg.hidden_size or x.dtype != self.torch_dtype or not x.is_contiguous():
            raise ValueError(f"expected a contiguous [nseq, rows, {self.cfg.hidden_size}] {self.torch_dtype} tensor, "
                             f"got {tuple(x.shape)} {x.dtype}")
        return int(x.shape[0]), int(x.shape[1])

    @staticmethod
    def _batch_offsets(cache_offset: torch.Tensor, nseq: int) -> torch.Tensor:
        if cache_offset.shape != (nseq,) or cache_offset.dtype != torch.int32 or not cache_offset.is_cuda:
            raise ValueError(f"cache_offset must be an int32 device tensor of shape ({nseq},)")
        return cache_offset.contiguous()

    @staticmethod
    def _prefix_lens(prefix_lens, nseq: int):
        lens = [int(p) for p in prefix_lens]
        if len(lens) != nseq:
            raise ValueError(f"prefix_lens has {len(lens)} entries for {nseq} sequences")
        return (ctypes.c_int64 * nseq)(*lens)

    def forward_cached_batch(self, active_embed: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                             cache_offset: torch.Tensor, prefix_lens) -> torch.Tensor:
        """forward_cached of nseq sequences at once: active_embed [nseq, rows, H], caches
        [L, nseq, cap, nkv, hd], cache_offset int32 [nseq], prefix_lens nseq host ints."""
        nseq, rows = self._check_batch_rows(active_embed)
        cap = self._check_batch_cache(k_cache, v_cache, nseq)
        off = self._batch_offsets(cache_offset, nseq)
        out = torch.empty_like(active_embed)
        _lib.check(self.lib.fdllm_forward_cached_batch(self.ctx, _ptr(active_embed), nseq, rows, _ptr(k_cache),
                                                       _ptr(v_cache), cap, _ptr(off), self._prefix_lens(prefix_lens, nseq),
                                                       _ptr(out), _stream()))
        return out

    def forward_block_partial_batch(self, replace_position: int, active_embed: torch.Tensor, k_cache: torch.Tensor,
                                    v_cache: torch.Tensor, cache_offset: torch.Tensor, prefix_lens) -> torch.Tensor:
        """forward_block_partial_rp{replace_position} of nseq sequences at once (shapes as forward_cached_batch)."""
        nseq, rows = self._check_batch_rows(active_embed)
        cap = self._check_batch_cache(k_cache, v_cache, nseq)
        off = self._batch_offsets(cache_offset, nseq)
        out = torch.empty_like(active_embed)
        _lib.check(self.lib.fdllm_forward_block_partial_batch(
            self.ctx, int(replace_position), _ptr(active_embed), nseq, rows, _ptr(k_cache), _ptr(v_cache), cap,
            _ptr(off), self._prefix_lens(prefix_lens, nseq), _ptr(out), _stream()))
        return out

    def build_prefix_cache_seq(self, prefix_embed: torch.Tensor, prefix_bias: torch.Tensor | None,
                               k_cache: torch.Tensor, v_cache: torch.Tensor, seq: int):
        """build_prefix_cache of sequence `seq` into its slice of a batched cache [L, nseq, cap, nkv, hd]."""
        p = self._check_rows(prefix_embed)
        nseq = int(k_cache.shape[1]) if k_cache.dim() == 5 else -1
        cap = self._check_batch_cache(k_cache, v_cache, nseq)
        if prefix_bias is not None:
            if tuple(prefix_bias.shape) != (1, 1, p, p) or prefix_bias.dtype != torch.float32:
                raise ValueError(f"prefix_bias must be [1, 1, {p}, {p}] float32")
            prefix_bias = prefix_bias.contiguous()
        _lib.check(self.lib.fdllm_build_prefix_cache_seq(self.ctx, _ptr(prefix_embed), p, _ptr(prefix_bias),
                                                         _ptr(k_cache), _ptr(v_cache), cap, nseq, int(seq), _stream()))
        return k_cache, v_cache

    def get_confidence(self, hidden_states: torch.Tensor, logits: torch.Tensor | None = None, out=None):
        """(ids [1, rows] int32, maxp [1, rows] fp32), unshifted (metal.py:505-528).  out: an optional
        contiguous [1, 2 rows] int32 device tensor that receives ids then maxp (bit-cast), so that one
        copy brings both back to the host."""
        rows = self._check_rows(hidden_states)
        if out is None:
            ids = torch.empty((1, rows), dtype=torch.int32, device=hidden_states.device)
            maxp = torch.empty((1, rows), dtype=torch.float32, device=hidden_states.device)
        else:
            if tuple(out.shape) != (1, 2 * rows) or out.dtype != torch.int32 or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous [1, {2 * rows}] int32 tensor")
            ids, maxp = out[:, :rows], out[:, rows:].view(torch.float32)
        if logits is not None and (tuple(logits.shape) != (1, rows, self.cfg.vocab_size)
                                   or logits.dtype != torch.float32 or not logits.is_contiguous()):
            raise ValueError("logits must be a contiguous [1, rows, vocab] float32 tensor")
        _lib.check(self.lib.fdllm_get_confidence(self.ctx, _ptr(hidden_states), rows, _ptr(ids), _ptr(maxp),
                                                 _ptr(logits), _stream()))
        return ids, maxp

    def confidence_from_logits(self, logits: torch.Tensor):
        """Device confidence of given fp32 logits [1, rows, vocab] (runtime.py:176-181 restated)."""
        if logits.dim() != 3 or logits.shape[2] != self.cfg.vocab_size or logits.dtype != torch.float32:
            raise ValueError("logits must be [1, rows, vocab] float32")
        logits = logits.contiguous()
        rows = int(logits.shape[1])
        ids = torch.empty((1, rows), dtype=torch.int32, device=logits.device)
        maxp = torch.empty((1, rows), dtype=torch.float32, device=logits.device)
        _lib.check(self.lib.fdllm_confidence_from_logits(self.ctx, _ptr(logits), rows, self.cfg.vocab_size,
                                                         self.cfg.vocab_size, _ptr(ids), _ptr(maxp), _stream()))
        return ids, maxp
