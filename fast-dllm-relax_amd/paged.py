"""A paged KV cache in 8 bits: its tensors, and the argument checks of the calls that take it.

``HipVM.paged_kv_append`` writes a cache, ``HipVM.paged_attn`` attends over it (include/fdllm.h has the definitions).
The reference has no counterpart: its caches are contiguous, in the model's dtype and of one sequence
(fast_dllm_relax/export_utils.py:21-34).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .config import FastDLLMConfig

FP8 = torch.float8_e4m3fn
PAGE_SIZES = (16, 32, 64, 128)


class PagedKVCache:
    """The pages of all layers: k [L, pages, nkv, page, 128] and v [L, pages, nkv, 128, page] float8_e4m3fn (v's slots are
    innermost), and one float32 scale for each layer, page and head, k_scale / v_scale [L, pages, nkv].  Contiguous
    tensors of one device; the object is made once and keeps them."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "num_layers", "num_pages", "num_kv_heads", "page_size", "device", "struct", "address", "fits")
    kind, attn, attn_workspace = 0, "fdllm_paged_attn", "fdllm_paged_attn_workspace"

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if k.dim() != 5 or k.shape[3] not in PAGE_SIZES or k.shape[1] < 1:
            raise ValueError(f"k must be [layers, pages, kv heads, page size of {PAGE_SIZES}, head_dim], got {tuple(k.shape)}")
        layers, pages, heads, page, hd = k.shape
        for name, t, shape, dtype in (("k", k, (layers, pages, heads, page, hd), FP8), ("v", v, (layers, pages, heads, hd, page), FP8),
                                      ("k_scale", k_scale, (layers, pages, heads), torch.float32),
                                      ("v_scale", v_scale, (layers, pages, heads), torch.float32)):
            if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous() or t.device != k.device:
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {k.device}, got "
                                 f"{tuple(t.shape)} {t.dtype} on {t.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_layers, self.num_pages, self.num_kv_heads, self.page_size = int(layers), int(pages), int(heads), int(page)
        self.device = k.device
        self.fits = (k.get_device(), self.num_layers, self.num_kv_heads, int(hd))  # what a call compares
        held = _lib.FdllmPagedCache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), int(pages), int(page))
        self.struct, self.address = ctypes.byref(held), ctypes.addressof(held)  # (the first keeps it)

    def __setattr__(self, name, value):
        if hasattr(self, name):
            raise AttributeError(f"a paged cache keeps its {name}: the calls hold its address; make a new cache")
        object.__setattr__(self, name, value)

    def dense(self, layer: int, pages) -> tuple[torch.Tensor, torch.Tensor]:
        """What the given pages of a layer hold, as float32 keys and values [len(pages) x page, nkv, head_dim]."""
        idx = torch.as_tensor(pages, dtype=torch.int64, device=self.device)
        k = self.k[layer][idx].float() * self.k_scale[layer][idx][:, :, None, None]
        v = self.v[layer][idx].float() * self.v_scale[layer][idx][:, :, None, None]
        return k.transpose(1, 2).flatten(0, 1), v.permute(0, 3, 1, 2).flatten(0, 1)


def allocate_paged_cache(cfg: FastDLLMConfig, num_pages: int, *, page_size: int = 32, device="cuda") -> PagedKVCache:
    """An empty cache for a model of cfg: num_pages pages a layer (pages of bd_size tokens hold one block each)."""
    if page_size not in PAGE_SIZES or num_pages < 1:
        raise ValueError(f"a paged cache has at least one page, of {PAGE_SIZES} tokens; got {num_pages} of {page_size}")
    head = (cfg.num_hidden_layers, int(num_pages), cfg.num_key_value_heads)
    return PagedKVCache(k=torch.zeros((*head, page_size, cfg.head_dim), dtype=FP8, device=device),
                        v=torch.zeros((*head, cfg.head_dim, page_size), dtype=FP8, device=device),
                        k_scale=torch.ones(head, dtype=torch.float32, device=device),
                        v_scale=torch.ones(head, dtype=torch.float32, device=device))


# Each check reads what passes in one condition and leaves the rest to its error.  index: the device's number
# (Tensor.get_device()).

def row_stride(t: torch.Tensor) -> int:
    """Elements from row to row of [rows, heads, hd]; a single row has none, whatever its tensor says."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def check_heads(t: torch.Tensor, heads: int, hd: int, dtype: torch.dtype, index: int, name: str) -> int:
    """[rows, heads, hd] with any row stride (a slice of a fused projection); returns the rows."""
    shape, strides = t.shape, t.stride()
    if (len(shape) == 3 and shape[1] == heads and shape[2] == hd and t.dtype is dtype and t.get_device() == index
            and (strides[1:] == (hd, 1) or (heads == 1 and strides[2] == 1) or shape[0] == 0)):
        return shape[0]
    raise ValueError(f"{name} must be a {dtype} tensor [rows, {heads}, {hd}] on device {index}, the heads of a row contiguous; got "
                     f"{tuple(shape)} {t.dtype} on {t.device} with strides {strides}")


def check_cache(cache: PagedKVCache, layer: int, fits: tuple) -> None:
    if cache.fits != fits:
        raise ValueError(f"the cache must hold (device, layers, kv heads, head_dim; 4 where of 4 bits) = {fits}, got {cache.fits}")
    if not 0 <= layer < cache.num_layers:
        raise ValueError(f"layer {layer} outside [0, {cache.num_layers})")


def is_i32(t: torch.Tensor, n: int, index: int) -> bool:
    return t.shape == (n,) and t.dtype is torch.int32 and t.get_device() == index and t.is_contiguous()


def check_i32(t: torch.Tensor, n: int, index: int, name: str) -> None:
    if not is_i32(t, n, index):
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape ({n},) on device {index}, got {tuple(t.shape)} "
                         f"{t.dtype} on {t.device}")


def check_table(table: torch.Tensor, index: int) -> tuple[int, int, int]:
    """(sequences, pages per sequence, row stride)"""
    shape, strides = table.shape, table.stride()
    if (len(shape) == 2 and shape[0] > 0 and shape[1] > 0 and table.dtype is torch.int32 and table.get_device() == index
            and (strides[1] == 1 or shape[1] == 1)):
        return shape[0], shape[1], strides[0]
    raise ValueError(f"page_table must be an int32 tensor [nseq, pages per sequence] on device {index} with contiguous rows, got "
                     f"{tuple(shape)} {table.dtype} on {table.device}")


def most_rows(rows: int, nseq: int, row_start: torch.Tensor | None, max_rows: int | None, index: int) -> int:
    """What sequence_rows gives, -1 where it raises."""
    if row_start is None:
        return rows // nseq if rows % nseq == 0 and (max_rows is None or max_rows * nseq == rows) else -1
    if not is_i32(row_start, nseq + 1, index):
        return -1
    return rows if max_rows is None else min(int(max_rows), rows)


def sequence_rows(rows: int, nseq: int, row_start: torch.Tensor | None, max_rows: int | None, index: int) -> int:
    """max_rows of a call: the rows of each sequence, or with row_start the bound that the caller gives (default: all)."""
    if row_start is None:
        if rows % nseq or (max_rows is not None and max_rows * nseq != rows):
            raise ValueError(f"{rows} rows are not the same number for each of {nseq} sequences; give row_start")
        return rows // nseq
    check_i32(row_start, nseq + 1, index, "row_start")
    if max_rows is None:
        return rows
    if max_rows < 0:
        raise ValueError(f"max_rows must not be negative, got {max_rows}")
    return min(int(max_rows), rows)
