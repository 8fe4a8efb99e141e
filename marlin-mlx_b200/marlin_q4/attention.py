"""The attention layer's operators around a quantized, paged key/value cache (torch front end).

Between the projections of a gated-attention layer (src/model/attention.cpp:82-139) a serving program
calls, per step: ``qk_norm_rope`` on the projected queries and keys, ``kv_write`` for the new keys and
values, ``paged_attention`` for the new queries over the cache.  ``kv_read`` gives cached rows back.
Forward only.  Tensors are CUDA tensors of one device; every call launches on that device's current
stream.  Padding and lengths are data on the device (negative slots, ``kv_lens``, ``cu_q``), so a call
can be captured in a CUDA graph and replayed with new ones.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib
from ._lib import BF16, F32, KvCache, check

_CODES = {torch.bfloat16: BF16, torch.float32: F32}


def _device(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """The CUDA device all of them are on."""
    d = first.get_device()
    if d < 0:
        raise ValueError("expected CUDA tensors")
    for t in others:
        if t is not None and t.get_device() != d:
            raise ValueError(f"tensors on different devices: {first.device} and {t.device}")
    return d


def _current(device: int):
    """Makes the device the current one, where it is not already."""
    return contextlib.nullcontext() if device == torch.cuda.current_device() else torch.cuda.device(device)


def _call(device: int, name: str, *args) -> None:
    """Calls the library on the device's current stream (its last argument), with the device current."""
    fn = getattr(_lib.load(), name)
    stream = torch._C._cuda_getCurrentRawStream(device)
    with _current(device):
        status = fn(*args, stream)
    if status:
        check(status, name)


def _heads(t: torch.Tensor, name: str):
    """Shape and strides of a [tokens, heads, head_dim] operand."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    if t.dtype not in _CODES:
        raise TypeError(f"{name} must be bfloat16 or float32, got {t.dtype}")
    stride = t.stride()
    if stride[2] != 1:
        raise ValueError(f"{name}'s features must be contiguous")
    return t.shape, stride


def _int32(t: torch.Tensor, name: str, *shape: int) -> None:
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {list(shape)}, got {list(t.shape)}")


class KVCache:
    """A paged pool of quantized keys and values: ``data`` uint8 [pages, kv_heads, page_size / 16, unit
    bytes] (marlin_q4_kv_cache); groups of 64 features, 4 or 8 bits."""

    def __init__(self, data: torch.Tensor, head_dim: int, bits: int = 4):
        unit = _lib.load().marlin_q4_kv_unit_bytes(head_dim, bits)
        if unit == 0:
            raise ValueError(f"unsupported head_dim {head_dim} or bits {bits} (64, 128, 256; 4, 8)")
        if data.dtype != torch.uint8 or data.dim() != 4 or data.shape[3] != unit or not data.is_contiguous():
            raise ValueError(f"data must be contiguous uint8 [pages, kv_heads, page_size / 16, {unit}]")
        self.data, self.head_dim, self.bits = data, head_dim, bits
        self.pages, self.kv_heads, self.page_size = data.shape[0], data.shape[1], data.shape[2] * 16
        self._c = KvCache(data.data_ptr(), self.pages, self.page_size, self.kv_heads, head_dim, bits)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, bits: int = 4,
              device="cuda") -> "KVCache":
        """A pool of zeros: page_size a multiple of 16."""
        unit = _lib.load().marlin_q4_kv_unit_bytes(head_dim, bits)
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
    (t, h, d), qs = _heads(q, "q")
    kshape, ks = _heads(k, "k")
    if q.dtype != k.dtype or out_dtype not in _CODES:
        raise TypeError("q and k must have one dtype, out_dtype must be bfloat16 or float32")
    kvh = kshape[1]
    if kshape[0] != t or kshape[2] != d:
        raise ValueError(f"k {tuple(k.shape)} does not match q {tuple(q.shape)}")
    axes = 1 if positions.dim() == 1 else positions.shape[0]
    _int32(positions, "positions", *((t,) if positions.dim() == 1 else (axes, t)))
    for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if w.dtype is not torch.bfloat16 or w.shape != (d,) or not w.is_contiguous():
            raise ValueError(f"{name} must be contiguous bfloat16 [{d}]")
    dev = _device(q, k, q_weight, k_weight, positions, rotary.inv_freq)
    qo = q.new_empty((t, h, d), dtype=out_dtype)
    ko = q.new_empty((t, kvh, d), dtype=out_dtype)
    _call(dev, "marlin_q4_qk_norm_rope", q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], _CODES[q.dtype], t, h, kvh, d,
          q_weight.data_ptr(), k_weight.data_ptr(), eps, positions.data_ptr(), axes, rotary.axes, rotary.inv_freq.data_ptr(),
          2 * rotary.inv_freq.shape[0], rotary.interleaved, qo.data_ptr(), ko.data_ptr(), _CODES[out_dtype])
    return qo, ko


def kv_write(cache: KVCache, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantize k, v [tokens, kv_heads, head_dim] (bf16 or f32) into the cache rows ``slots`` (int32
    [tokens], page * page_size + row; negative: skip the token).  The slots >= 0 must differ."""
    (t, h, d), ks = _heads(k, "k")
    _, vs = _heads(v, "v")
    if h != cache.kv_heads or d != cache.head_dim or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [tokens, {cache.kv_heads}, {cache.head_dim}]"
                         " of one dtype")
    _int32(slots, "slots", t)
    dev = _device(cache.data, k, v, slots)
    _call(dev, "marlin_q4_kv_write", cache._ref, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1], _CODES[k.dtype],
          slots.data_ptr(), t)


def kv_read(cache: KVCache, slots: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values of cache rows ``slots`` (int32 [tokens]; negative: zeros) as bf16 [tokens,
    kv_heads, head_dim], bf16(scale * code + bias)."""
    t = slots.numel()
    _int32(slots, "slots", t)
    dev = _device(cache.data, slots)
    k = slots.new_empty((t, cache.kv_heads, cache.head_dim), dtype=torch.bfloat16)
    v = slots.new_empty((t, cache.kv_heads, cache.head_dim), dtype=torch.bfloat16)
    _call(dev, "marlin_q4_kv_read", cache._ref, slots.data_ptr(), t, k.data_ptr(), v.data_ptr())
    return k, v


def paged_attention(q: torch.Tensor, cache: KVCache, block_table: torch.Tensor, kv_lens: torch.Tensor,
                    cu_q: torch.Tensor | None = None, max_q: int = 1, scale: float | None = None,
                    out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of each sequence's newest tokens over its cached positions (marlin_q4_paged_attention).

    q bf16 [tokens, heads, head_dim]; block_table int32 [batch, pages per sequence]; kv_lens int32 [batch],
    the new tokens included; cu_q int32 [batch + 1] starts of the sequences in q and max_q the most tokens of
    any, or None for one token per sequence.  scale defaults to head_dim ** -0.5.  Rows of ``out`` outside
    every sequence are left as they were.  workspace: uint8 of at least attention_workspace_size bytes; calls
    that may overlap in time (other streams, graphs) need one each.  Without it one is allocated."""
    (t, h, d), qs = _heads(q, "q")
    if q.dtype is not torch.bfloat16:
        raise TypeError(f"q must be bfloat16, got {q.dtype}")
    if d != cache.head_dim:
        raise ValueError(f"q's head_dim {d} is not the cache's {cache.head_dim}")
    if block_table.dtype is not torch.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be int32 [batch, pages]")
    batch, width = block_table.shape
    ts = block_table.stride()
    if ts[1] != 1 and width > 1:
        raise ValueError("block_table's rows must be contiguous")
    _int32(kv_lens, "kv_lens", batch)
    if cu_q is not None:
        _int32(cu_q, "cu_q", batch + 1)
    dev = _device(q, cache.data, block_table, kv_lens, cu_q, out, workspace)
    if out is None:
        out = q.new_empty((t, h, d))
    elif out.dtype is not torch.bfloat16 or out.shape != q.shape or not out.is_contiguous():
        raise ValueError(f"out must be contiguous bfloat16 {list(q.shape)}")
    if workspace is None:
        with _current(dev):
            size = _lib.load().marlin_q4_paged_attention_workspace_size(t, h, cache.kv_heads, d, max(batch, 1))
        workspace = q.new_empty(size, dtype=torch.uint8)
    _call(dev, "marlin_q4_paged_attention", q.data_ptr(), qs[0], qs[1], cache._ref, t, h, block_table.data_ptr(), ts[0], width,
          kv_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), batch, max_q, d ** -0.5 if scale is None else scale,
          out.data_ptr(), workspace.data_ptr(), workspace.numel())
    return out


def attention_workspace_size(tokens: int, heads: int, kv_heads: int, head_dim: int, batch: int) -> int:
    """Bytes of workspace paged_attention needs on the current device."""
    size = _lib.load().marlin_q4_paged_attention_workspace_size(tokens, heads, kv_heads, head_dim, batch)
    if size == 0:
        raise ValueError("unsupported tokens, heads, kv_heads, head_dim or batch")
    return size
