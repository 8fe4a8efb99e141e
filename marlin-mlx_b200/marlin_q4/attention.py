"""The attention layer's operators around a quantized, paged key/value cache (torch front end).

Between the projections of a gated-attention layer (src/model/attention.cpp:82-139) a serving program
calls, per step: ``qk_norm_rope`` on the projected queries and keys, ``kv_write`` for the new keys and
values, ``paged_attention`` for the new queries over the cache.  ``kv_read`` gives cached rows back.
Forward only.  Tensors are CUDA tensors of one device; every call launches on that device's current
stream.  Padding and lengths are data on the device (negative slots, ``kv_lens``, ``cu_q``), so a call
can be captured in a CUDA graph and replayed with new ones.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._lib import check

_OUT = {torch.bfloat16: True, torch.float32: False}
_bound = None  # the compiled front end (csrc/attention_torch.cpp), with the library's entry points


def _front():
    global _bound
    if _bound is None:
        lib = _lib.load()
        try:
            from . import _attention
        except ImportError as e:
            raise ImportError("marlin_q4/_attention.so is missing or was built for another torch: build it with "
                              "`python marlin-mlx_b200/build.py` (there is no other path)") from e
        _attention.bind(*(ctypes.cast(getattr(lib, "marlin_q4_" + f), ctypes.c_void_p).value for f in (
            "kv_unit_bytes", "qk_norm_rope", "kv_write", "kv_read", "paged_attention_workspace_size", "paged_attention")))
        _bound = _attention
    return _bound


def _unit_bytes(head_dim: int, bits: int) -> int:
    """marlin_q4_kv_unit_bytes: 16 positions' codes, scales and biases, keys and values; 0 if unsupported."""
    return 32 * (head_dim * bits // 8 + head_dim // 16) if head_dim in (64, 128, 256) and bits in (4, 8) else 0


class KVCache:
    """A paged pool of quantized keys and values: ``data`` uint8 [pages, kv_heads, page_size / 16, unit
    bytes] (marlin_q4_kv_cache); groups of 64 features, 4 or 8 bits."""

    def __init__(self, data: torch.Tensor, head_dim: int, bits: int = 4):
        unit = _unit_bytes(head_dim, bits)
        if unit == 0:
            raise ValueError(f"unsupported head_dim {head_dim} or bits {bits} (64, 128, 256; 4, 8)")
        shape = data.shape
        if data.dtype is not torch.uint8 or len(shape) != 4 or shape[3] != unit or not data.is_contiguous():
            raise ValueError(f"data must be contiguous uint8 [pages, kv_heads, page_size / 16, {unit}]")
        self.data, self.head_dim, self.bits = data, head_dim, bits
        self.pages, self.kv_heads, self.page_size = shape[0], shape[1], shape[2] * 16

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 4,
              device="cuda") -> "KVCache":
        """A pool of zeros: page_size a multiple of 16."""
        unit = _unit_bytes(head_dim, bits)
        if unit == 0 or page_size <= 0 or page_size % 16:
            raise ValueError("unsupported head_dim, bits or page_size (64, 128, 256; 4, 8; a multiple of 16)")
        return cls(torch.zeros((pages, kv_heads, page_size // 16, unit), dtype=torch.uint8, device=device), head_dim, bits)


class Rotary:
    """Rotary positions: ``inv_freq`` float32 [rot_dim / 2] on the device (scaled for long contexts as the
    caller likes), pairs (2i, 2i + 1) if ``interleaved`` else (i, i + rot_dim / 2), and for positions of
    several axes the axis of each pair."""

    def __init__(self, inv_freq: torch.Tensor, interleaved: bool = False, axes=None):
        if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be contiguous float32 [rot_dim / 2]")
        if axes is not None and len(axes) != inv_freq.numel():
            raise ValueError("axes must name one axis per pair")
        self.inv_freq, self.interleaved = inv_freq, interleaved
        self.axes = None if axes is None else bytes(axes)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 positions: torch.Tensor, rotary: Rotary, eps: float = 1e-6,
                 out_dtype: torch.dtype = torch.bfloat16) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of each query and key head (multiplier 1 + weight), then the rotation, in one pass.

    q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim], bf16 or f32, may be strided views of a
    fused projection; positions int32 [tokens] or [axes, tokens].  Returns contiguous (q, k) of out_dtype."""
    if out_dtype not in _OUT:
        raise TypeError("out_dtype must be bfloat16 or float32")
    r = (_bound or _front()).qk_norm_rope(q, k, q_weight, k_weight, positions, rotary.inv_freq, rotary.interleaved,
                                          rotary.axes, eps, _OUT[out_dtype])
    if type(r) is int:
        check(r, "marlin_q4_qk_norm_rope")
    return r


def kv_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantize k, v [tokens, kv_heads, head_dim] (bf16 or f32) into the cache rows ``slots`` (int32
    [tokens], page * page_size + row; negative: skip the token).  The slots >= 0 must differ."""
    r = (_bound or _front()).kv_write(cache.data, cache.head_dim, cache.bits, k, v, slots)
    if r:
        check(r, "marlin_q4_kv_write")


def kv_read(cache: KVCache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values of cache rows ``slots`` (int32 [tokens]; negative: zeros) as bf16 [tokens,
    kv_heads, head_dim], bf16(scale * code + bias)."""
    r = (_bound or _front()).kv_read(cache.data, cache.head_dim, cache.bits, slots)
    if type(r) is int:
        check(r, "marlin_q4_kv_read")
    return r


def paged_attention(q: torch.Tensor, cache: KVCache, block_table: torch.Tensor, kv_lens: torch.Tensor,
                    cu_q: torch.Tensor | None = None, max_q: int = 1, scale: float | None = None,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of each sequence's newest tokens over its cached positions (marlin_q4_paged_attention).

    q bf16 [tokens, heads, head_dim]; block_table int32 [batch, pages per sequence]; kv_lens int32 [batch],
    the new tokens included; cu_q int32 [batch + 1] starts of the sequences in q and max_q the most tokens of
    any, or None for one token per sequence.  scale defaults to head_dim ** -0.5.  Rows of ``out`` outside
    every sequence are left as they were.  workspace: uint8 of at least attention_workspace_size bytes; calls
    that may overlap in time (other streams, graphs) need one each.  Without it one is allocated."""
    r = (_bound or _front()).paged_attention(q, cache.data, cache.head_dim, cache.bits, block_table, kv_lens, cu_q, max_q,
                                             scale, out, workspace)
    if type(r) is int:
        check(r, "marlin_q4_paged_attention")
    return r


def attention_workspace_size(tokens: int, heads: int, kv_heads: int, head_dim: int, batch: int) -> int:
    """Bytes of workspace paged_attention needs on the current device."""
    size = _lib.load().marlin_q4_paged_attention_workspace_size(tokens, heads, kv_heads, head_dim, batch)
    if size == 0:
        raise ValueError("unsupported tokens, heads, kv_heads, head_dim or batch")
    return size
