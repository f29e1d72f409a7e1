"""What lies between the QKV GEMM and the output GEMM of an attention layer: the norm and rotation
of the query and key heads, the MX key-value cache and the attention of one new token over it.

    qkv = mx.gemm(x, w_qkv)                                           # [tokens, (H + 2 Hkv) * D]
    q = mx.qk_norm_rope_cache(qkv, H, Hkv, cos, sin, cache, slots, positions=pos)
    a = mx.paged_attention(q, cache, page_table, lengths)
    o = mx.gemm(a.view(tokens, H * D), w_out)

Serving forms (the library has no gradients).  As for the GEMMs, invalid arguments raise
RuntimeError, every call runs on the current stream of the tensors' device through the C ABI in
``include/mxfp4_b200.h``, may be captured into a CUDA graph, and there is no CPU path.  Index tensors
are int32 on the device; an index out of range leaves its access out and sets the device error
word (:func:`mxfp4_b200.device_error`: 0x201 slot, 0x202 position, 0x203 page, 0x204 length).
"""

from __future__ import annotations

import ctypes
import os

import torch

from . import _lib, build
from .kernels import _check, _require_cuda

KV_FORMATS = {"mxfp8": _lib.KV_MXFP8, "mxfp4": _lib.KV_MXFP4}
_PAGE_SIZES = (16, 32, 64, 128, 256)
_BOUND = ("mxfp4_error_string", "mxfp4_qk_norm_rope", "mxfp4_qk_norm_rope_cache", "mxfp4_kv_cache_write", "mxfp4_kv_cache_read",
          "mxfp4_paged_attention_workspace_bytes", "mxfp4_paged_attention")
_native = None


def _binding():
    """The compiled binding (csrc/attention_binding.cpp: checks, allocation and the C call in one step),
    bound to the library that :mod:`mxfp4_b200._lib` loads.  As there, no fallback."""
    global _native
    if _native is None:
        if os.path.exists(build.BINDING_OUT) and not build.binding_fits():
            raise RuntimeError("_attention.so was built for another torch or Python: build it with `python -m mxfp4_b200.build`")
        try:
            from . import _attention
        except ImportError as e:
            raise RuntimeError("_attention.so is missing or does not load: build it with `python -m mxfp4_b200.build`") from e
        library = _lib.lib()
        _attention.bind(*(ctypes.cast(getattr(library, name), ctypes.c_void_p).value for name in _BOUND))
        _native = _attention
    return _native


class MXKVCache:
    """A paged key-value cache in an MX format (byte layout: ``mxfp4_kv_cache`` in the C header).

    ``k_codes`` / ``v_codes``: uint8 ``[num_pages, num_kv_heads, page_size, head_dim]`` E4M3 codes
    (``format="mxfp8"``) or ``[..., head_dim // 2]`` pairs of E2M1 codes (``"mxfp4"``, even element in
    the low nibble); ``k_scales`` / ``v_scales``: uint8 ``[..., head_dim // 32]`` E8M0 bytes.  The
    tensors are contiguous and stay the caller's: the object only refers to them, always to the same
    ones (its attributes are read-only), and each call takes their memory as it is then: a tensor
    that has been given other storage of the same form serves, another form is refused.  head_dim 64, 128 or 256; page_size 16, 32, 64, 128 or 256.
    :func:`new_kv_cache` allocates one.
    """

    __slots__ = ("k_codes", "v_codes", "k_scales", "v_scales", "format", "num_pages", "num_kv_heads", "page_size",
                 "head_dim", "device", "_struct", "_native")

    def __init__(self, k_codes, v_codes, k_scales, v_scales, format: str = "mxfp8"):
        _check(format in KV_FORMATS, "format must be 'mxfp8' or 'mxfp4'")
        for t in (k_codes, v_codes, k_scales, v_scales):
            _check(isinstance(t, torch.Tensor) and t.is_cuda and t.device == k_codes.device, "all tensors must be on one GPU")
            _check(t.dtype == torch.uint8 and t.dim() == 4 and t.is_contiguous(), "cache tensors must be contiguous 4-D uint8")
        pages, heads, size, width = k_codes.shape
        dim = width * (1 if format == "mxfp8" else 2)
        _check(v_codes.shape == k_codes.shape, "v_codes shape")
        _check(dim in (64, 128, 256), "head_dim must be 64, 128 or 256")
        _check(size in _PAGE_SIZES, "page_size must be 16, 32, 64, 128 or 256")
        _check(pages > 0 and heads > 0 and pages * size < 2**31, "num_pages * page_size must be in 1 .. 2**31 - 1")
        for t in (k_scales, v_scales):
            _check(tuple(t.shape) == (pages, heads, size, dim // 32), "scales shape")
        struct = _lib.KVCache(k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                              pages, heads, size, dim, KV_FORMATS[format])
        native = (k_codes, v_codes, k_scales, v_scales, ctypes.addressof(struct), k_codes.get_device())
        for name, value in zip(self.__slots__, (k_codes, v_codes, k_scales, v_scales, format, pages, heads, size, dim,
                                                k_codes.device, struct, native)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise RuntimeError("an MXKVCache refers to the same tensors for good: make another one")

    def nbytes(self) -> int:
        return 2 * (self.k_codes.numel() + self.k_scales.numel())


def new_kv_cache(num_pages: int, num_kv_heads: int, head_dim: int, page_size: int = 64, format: str = "mxfp8",
                 device="cuda") -> MXKVCache:
    """An :class:`MXKVCache` of zeros."""
    _require_cuda()
    _check(format in KV_FORMATS, "format must be 'mxfp8' or 'mxfp4'")
    rows = (num_pages, num_kv_heads, page_size)
    width = head_dim if format == "mxfp8" else head_dim // 2
    return MXKVCache(*(torch.zeros((*rows, n), dtype=torch.uint8, device=device)
                       for n in (width, width, head_dim // 32, head_dim // 32)), format=format)


def qk_norm_rope(qkv, num_heads: int, num_kv_heads: int, cos=None, sin=None, positions=None, q_weight=None,
                 k_weight=None, eps: float = 1e-6, interleaved: bool = False):
    """RMS norm of every query and key head and its rotation, in one pass over ``qkv``.

    ``qkv`` bf16 ``[tokens, (num_heads + 2 * num_kv_heads) * head_dim]``: query, key and value heads
    side by side, rows apart by a multiple of 8; head_dim is a multiple of 32 up to
    256.  With ``q_weight`` / ``k_weight`` (``[head_dim]``, bf16 or fp32, both or neither) a head x becomes
    ``x * weight / sqrt(mean(x * x) + eps)``.  ``cos`` / ``sin`` fp32 ``[rows, rot / 2]`` turn the first
    ``rot`` values (a multiple of 16): row ``positions[token]`` (int32), or the token's own index;
    ``interleaved`` pairs values 2i and 2i + 1, otherwise i and i + rot / 2.
    Returns new ``(q [tokens, num_heads, head_dim], k [tokens, num_kv_heads, head_dim])`` in bf16, each
    value computed in fp32 and rounded once.
    """
    return (_native or _binding()).qk_norm_rope(qkv, num_heads, num_kv_heads, cos, sin, positions, q_weight, k_weight, eps, interleaved)


def qk_norm_rope_cache(qkv, num_heads: int, num_kv_heads: int, cos, sin, cache: MXKVCache, slots, positions=None,
                       q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False):
    """:func:`qk_norm_rope` that writes the keys and values into ``cache`` instead of returning keys.

    ``slots`` int32 ``[tokens]``: token t goes to row ``slots[t] % page_size`` of page ``slots[t] //
    page_size``; a negative slot stores nothing (a batch's padding); of two tokens with one slot the
    later is stored (of those whose positions the tables have).  Keys are coded from the unrounded rotated value, values from ``qkv`` as they
    are.  ``cos`` and ``sin`` may be None (no rotation).  Returns q.
    """
    if not isinstance(cache, MXKVCache):
        raise RuntimeError("cache must be an MXKVCache")
    return (_native or _binding()).qk_norm_rope_cache(qkv, num_heads, num_kv_heads, cos, sin, positions, q_weight, k_weight, eps,
                                                      interleaved, cache._native, slots)


def kv_cache_write(cache: MXKVCache, k, v, slots) -> None:
    """Codes ``k`` and ``v`` (bf16 ``[tokens, num_kv_heads, head_dim]``, each token's heads contiguous, any
    row stride that is a multiple of 8) into the cache rows ``slots`` names, as
    :func:`qk_norm_rope_cache` does: the OCP MX rule, the counterpart of
    ``quantize_mxfp4(..., rule="ocp")`` and :func:`quantize_act_mx8`."""
    if not isinstance(cache, MXKVCache):
        raise RuntimeError("cache must be an MXKVCache")
    (_native or _binding()).kv_cache_write(cache._native, k, v, slots)


def kv_cache_read(cache: MXKVCache, slots):
    """The rows ``slots`` (int32 ``[tokens]``) names, as new bf16 ``(k, v)`` of ``[tokens, num_kv_heads,
    head_dim]``; a negative slot reads zeros, the scale byte 255 NaN."""
    if not isinstance(cache, MXKVCache):
        raise RuntimeError("cache must be an MXKVCache")
    return (_native or _binding()).kv_cache_read(cache._native, slots)


def paged_attention(q, cache: MXKVCache, page_table, lengths, scale: float | None = None, return_lse: bool = False,
                    out=None):
    """Attention of one new token per sequence over the cache.

    ``q`` bf16 ``[seqs, num_heads, head_dim]`` (each sequence's heads contiguous), num_heads a multiple of
    the cache's num_kv_heads: query head h reads kv head ``h // (num_heads // num_kv_heads)``.
    ``page_table`` int32 ``[seqs, max_pages]`` (rows apart by max_pages or more): key j of sequence s is row ``j %
    page_size`` of page ``page_table[s, j // page_size]``, j < ``lengths[s]`` (int32); entries past the last
    page a sequence needs may hold anything.  A length of zero gives a row of zeros.  ``scale`` defaults to
    ``head_dim ** -0.5``.  Returns bf16 ``[seqs, num_heads, head_dim]`` (``out`` if given), with
    ``return_lse`` also fp32 ``[seqs, num_heads]``: the natural log of the sum of exp(scale * q . k), -inf
    for an empty sequence.  ``out`` may be ``q`` itself, and is refused if it overlaps it otherwise.  The same call
    gives the same bits.
    """
    if not isinstance(cache, MXKVCache):
        raise RuntimeError("cache must be an MXKVCache")
    return (_native or _binding()).paged_attention(q, cache._native, page_table, lengths, scale, return_lse, out)
