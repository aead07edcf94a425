"""A paged KV cache in 4 bits: its tensors, for ``HipVM.paged4_append``, ``paged4_read`` and ``paged_attn`` (include/fdllm.h
has the definitions).  The reference has no counterpart: its caches are contiguous, in the model's dtype and of one sequence
(fast_dllm_relax/export_utils.py:21-34).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .config import FastDLLMConfig
from .paged import PAGE_SIZES

KEY_BLOCK = 32  # dims of a key that share a scale


class Paged4KVCache:
    """The pages of all layers.  k and v [L, pages, nkv, page, 64] uint8: two e2m1 codes a byte, the lower dim in the lower four
    bits.  k_scale [L, pages, nkv, page / 16, 4, 4, 4] uint8: of slot s and block b of 32 dims the exponent + 127 of its power
    of two (255: NaN), at [s / 16, s % 4, b, s / 4 % 4], as the matrix instructions take them.  v_scale [L, pages, nkv, page]
    bfloat16 (what paged_attn makes of scales that paged4_append does not write: fdllm_paged4_attn).  Contiguous tensors of one
    device, 16-byte aligned; the object is made once and keeps them."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "num_layers", "num_pages", "num_kv_heads", "page_size", "device", "struct", "address", "fits")
    kind, attn, attn_workspace = 1, "fdllm_paged4_attn", "fdllm_paged4_attn_workspace"

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if k.dim() != 5 or k.shape[3] not in PAGE_SIZES or k.shape[1] < 1:
            raise ValueError(f"k must be [layers, pages, kv heads, page size of {PAGE_SIZES}, head_dim / 2], got {tuple(k.shape)}")
        layers, pages, heads, page, half = k.shape
        for name, t, shape, dtype in (("k", k, (layers, pages, heads, page, half), torch.uint8),
                                      ("v", v, (layers, pages, heads, page, half), torch.uint8),
                                      ("k_scale", k_scale, (layers, pages, heads, page // 16, 4, 2 * half // KEY_BLOCK, 4), torch.uint8),
                                      ("v_scale", v_scale, (layers, pages, heads, page), torch.bfloat16)):
            if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous() or t.device != k.device:
                raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {k.device}, got "
                                 f"{tuple(t.shape)} {t.dtype} on {t.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.num_layers, self.num_pages, self.num_kv_heads, self.page_size = int(layers), int(pages), int(heads), int(page)
        self.device = k.device
        self.fits = (k.get_device(), self.num_layers, self.num_kv_heads, 2 * int(half), 4)  # what a call compares
        held = _lib.FdllmPaged4Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), int(pages), int(page))
        self.struct, self.address = ctypes.byref(held), ctypes.addressof(held)  # (the first keeps it)

    def __setattr__(self, name, value):
        if hasattr(self, name):
            raise AttributeError(f"a paged cache keeps its {name}: the calls hold its address; make a new cache")
        object.__setattr__(self, name, value)

    def dense(self, layer: int, pages) -> tuple[torch.Tensor, torch.Tensor]:
        """What the given pages of a layer hold, as float32 keys and values [len(pages) x page, nkv, head_dim]."""
        idx = torch.as_tensor(pages, dtype=torch.int64, device=self.device)
        e = self.k_scale[layer][idx].movedim(-1, -3).flatten(-4, -2)  # [pages, heads, slots, blocks]
        scale = torch.where(e == 255, torch.nan, torch.exp2(e.float() - 127)).repeat_interleave(KEY_BLOCK, dim=-1)
        k = values_of(self.k[layer][idx]) * scale
        v = values_of(self.v[layer][idx]) * self.v_scale[layer][idx].float()[..., None]
        return k.transpose(1, 2).flatten(0, 1), v.transpose(1, 2).flatten(0, 1)


def values_of(codes: torch.Tensor) -> torch.Tensor:
    """The float32 values [..., 2 n] of e2m1 codes packed in bytes [..., n]."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    size = torch.tensor((0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0), device=codes.device)[(c & 7).long()]
    return torch.where(c >= 8, -size, size)


def allocate_paged4_cache(cfg: FastDLLMConfig, num_pages: int, *, page_size: int = 32, device="cuda") -> Paged4KVCache:
    """An empty cache for a model of cfg: num_pages pages a layer (pages of bd_size tokens hold one block each)."""
    if page_size not in PAGE_SIZES or num_pages < 1:
        raise ValueError(f"a paged cache has at least one page, of {PAGE_SIZES} tokens; got {num_pages} of {page_size}")
    head = (cfg.num_hidden_layers, int(num_pages), cfg.num_key_value_heads)
    codes = lambda: torch.zeros((*head, page_size, cfg.head_dim // 2), dtype=torch.uint8, device=device)  # noqa: E731
    return Paged4KVCache(k=codes(), v=codes(),
                         k_scale=torch.full((*head, page_size // 16, 4, cfg.head_dim // KEY_BLOCK, 4), 127, dtype=torch.uint8, device=device),
                         v_scale=torch.ones((*head, page_size), dtype=torch.bfloat16, device=device))
