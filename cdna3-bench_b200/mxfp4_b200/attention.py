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

import contextlib
import ctypes
import math

import torch

from . import _lib
from .kernels import _check, _require_cuda

KV_FORMATS = {"mxfp8": _lib.KV_MXFP8, "mxfp4": _lib.KV_MXFP4}
_NOTHING = contextlib.nullcontext()


def _on(device: torch.device):
    """Makes `device` the current one if it is not."""
    return _NOTHING if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream_of(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _check_index(t, n: int, device, what: str):
    _check(isinstance(t, torch.Tensor) and t.is_cuda and t.device == device, f"{what} must be on the GPU of the other tensors")
    _check(t.dtype == torch.int32, f"{what} must be int32")
    _check(t.dim() == 1 and t.shape[0] == n and (n < 2 or t.stride(0) == 1), f"{what} must be a contiguous vector of {n}")


def _check_bf16(t, device, what: str):
    _check(isinstance(t, torch.Tensor) and t.is_cuda and (device is None or t.device == device),
           f"{what} must be on the GPU of the other tensors")
    _check(t.dtype == torch.bfloat16, f"{what} must be bfloat16")


class MXKVCache:
    """A paged key-value cache in an MX format (byte layout: ``mxfp4_kv_cache`` in the C header).

    ``k_codes`` / ``v_codes``: uint8 ``[num_pages, num_kv_heads, page_size, head_dim]`` E4M3 codes
    (``format="mxfp8"``) or ``[..., head_dim // 2]`` pairs of E2M1 codes (``"mxfp4"``, even element in
    the low nibble); ``k_scales`` / ``v_scales``: uint8 ``[..., head_dim // 32]`` E8M0 bytes.  The
    tensors are contiguous and stay the caller's: the object only refers to them.  head_dim 64, 128
    or 256; page_size 16, 32, 64, 128 or 256.  :func:`new_kv_cache` allocates one.
    """

    __slots__ = ("k_codes", "v_codes", "k_scales", "v_scales", "format", "num_pages", "num_kv_heads", "page_size",
                 "head_dim", "device", "_struct", "_ref")

    def __init__(self, k_codes, v_codes, k_scales, v_scales, format: str = "mxfp8"):
        _check(format in KV_FORMATS, "format must be 'mxfp8' or 'mxfp4'")
        for t in (k_codes, v_codes, k_scales, v_scales):
            _check(isinstance(t, torch.Tensor) and t.is_cuda and t.device == k_codes.device, "all tensors must be on one GPU")
            _check(t.dtype == torch.uint8 and t.dim() == 4 and t.is_contiguous(), "cache tensors must be contiguous 4-D uint8")
        pages, heads, size, width = k_codes.shape
        dim = width * (1 if format == "mxfp8" else 2)
        _check(v_codes.shape == k_codes.shape, "v_codes shape")
        _check(dim in (64, 128, 256), "head_dim must be 64, 128 or 256")
        _check(size in (16, 32, 64, 128, 256), "page_size must be 16, 32, 64, 128 or 256")
        _check(pages > 0 and heads > 0 and pages * size < 2**31, "num_pages * page_size must be in 1 .. 2**31 - 1")
        for t in (k_scales, v_scales):
            _check(tuple(t.shape) == (pages, heads, size, dim // 32), "scales shape")
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.format, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = format, pages, heads, size, dim
        self.device = k_codes.device
        self._struct = _lib.KVCache(k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(),
                                    pages, heads, size, dim, KV_FORMATS[format])
        self._ref = ctypes.byref(self._struct)

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


def _rope_arguments(qkv, num_heads, num_kv_heads, dim, cos, sin, positions, q_weight, k_weight, eps):
    _check_bf16(qkv, None, "qkv")
    _check(qkv.dim() == 2 and qkv.stride(1) == 1, "qkv must be [tokens, width] with contiguous rows")
    T, dev = qkv.shape[0], qkv.device
    _check(num_heads > 0 and num_kv_heads > 0 and qkv.shape[1] == (num_heads + 2 * num_kv_heads) * dim,
           "qkv's width must be (num_heads + 2 * num_kv_heads) * head_dim")
    rows = rot = cp = sp = 0
    if cos is not None or sin is not None:
        for t in (cos, sin):
            _check(isinstance(t, torch.Tensor) and t.is_cuda and t.device == dev, "cos and sin must be on qkv's GPU")
            _check(t.dtype == torch.float32 and t.dim() == 2 and t.is_contiguous(), "cos and sin must be contiguous 2-D float32")
        _check(cos.shape == sin.shape, "cos and sin must have one shape")
        rows, rot = cos.shape[0], 2 * cos.shape[1]
        _check(rows > 0 and rot > 0, "cos and sin must not be empty")
        cp, sp = cos.data_ptr(), sin.data_ptr()
    if positions is not None:
        _check(rot > 0, "positions without cos and sin")
        _check_index(positions, T, dev, "positions")
    else:
        _check(rot == 0 or rows >= T, "cos and sin need a row per token when no positions are given")
    _check((q_weight is None) == (k_weight is None), "q_weight and k_weight come together")
    qw = kw = 0
    wt = _lib.DTYPE_BF16
    if q_weight is not None:
        for w in (q_weight, k_weight):
            _check(isinstance(w, torch.Tensor) and w.is_cuda and w.device == dev, "weights must be on qkv's GPU")
            _check(w.dtype in (torch.bfloat16, torch.float32) and w.dtype == q_weight.dtype, "weights must be bfloat16 or float32")
            _check(tuple(w.shape) == (dim,) and w.is_contiguous(), "weights must be vectors of head_dim")
        qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
        wt = _lib.DTYPE_F32 if q_weight.dtype == torch.float32 else _lib.DTYPE_BF16
    stride = qkv.stride(0) if T > 1 else qkv.shape[1]
    return T, dev, stride, cp, sp, rows, rot, positions.data_ptr() if positions is not None else 0, qw, kw, wt, float(eps)


def qk_norm_rope(qkv, num_heads: int, num_kv_heads: int, cos=None, sin=None, positions=None, q_weight=None,
                 k_weight=None, eps: float = 1e-6, interleaved: bool = False):
    """RMS norm of every query and key head and its rotation, in one pass over ``qkv``.

    ``qkv`` bf16 ``[tokens, (num_heads + 2 * num_kv_heads) * head_dim]``: query, key and value heads
    side by side, rows of any stride that is a multiple of 8; head_dim is a multiple of 32 up to
    256.  With ``q_weight`` / ``k_weight`` (``[head_dim]``, bf16 or fp32, both or neither) a head x becomes
    ``x * weight / sqrt(mean(x * x) + eps)``.  ``cos`` / ``sin`` fp32 ``[rows, rot / 2]`` turn the first
    ``rot`` values (a multiple of 16): row ``positions[token]`` (int32), or the token's own index;
    ``interleaved`` pairs values 2i and 2i + 1, otherwise i and i + rot / 2.
    Returns new ``(q [tokens, num_heads, head_dim], k [tokens, num_kv_heads, head_dim])`` in bf16, each
    value computed in fp32 and rounded once.
    """
    _check(isinstance(qkv, torch.Tensor) and qkv.dim() == 2 and num_heads > 0 and num_kv_heads > 0,
           "qkv must be [tokens, width] with contiguous rows")
    dim = qkv.shape[1] // (num_heads + 2 * num_kv_heads)
    T, dev, stride, cp, sp, rows, rot, pos, qw, kw, wt, eps = _rope_arguments(
        qkv, num_heads, num_kv_heads, dim, cos, sin, positions, q_weight, k_weight, eps)
    with _on(dev):
        q = torch.empty((T, num_heads, dim), dtype=torch.bfloat16, device=dev)
        k = torch.empty((T, num_kv_heads, dim), dtype=torch.bfloat16, device=dev)
        _lib.check(
            _lib.lib().mxfp4_qk_norm_rope(qkv.data_ptr(), stride, T, num_heads, num_kv_heads, dim, cp, sp, rows, rot,
                                          int(interleaved), pos, qw, kw, wt, eps, q.data_ptr(), k.data_ptr(),
                                          _stream_of(dev)),
            "mxfp4_qk_norm_rope",
        )
    return q, k


def qk_norm_rope_cache(qkv, num_heads: int, num_kv_heads: int, cos, sin, cache: MXKVCache, slots, positions=None,
                       q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False):
    """:func:`qk_norm_rope` that writes the keys and values into ``cache`` instead of returning keys.

    ``slots`` int32 ``[tokens]``: token t goes to row ``slots[t] % page_size`` of page ``slots[t] //
    page_size``; a negative slot stores nothing (a batch's padding); of two tokens with one slot the
    later is stored.  Keys are coded from the unrounded rotated value, values from ``qkv`` as they
    are.  ``cos`` and ``sin`` may be None (no rotation).  Returns q.
    """
    _check(isinstance(cache, MXKVCache), "cache must be an MXKVCache")
    _check(num_kv_heads == cache.num_kv_heads, "num_kv_heads differs from the cache's")
    T, dev, stride, cp, sp, rows, rot, pos, qw, kw, wt, eps = _rope_arguments(
        qkv, num_heads, num_kv_heads, cache.head_dim, cos, sin, positions, q_weight, k_weight, eps)
    _check(dev == cache.device, "qkv must be on the cache's GPU")
    _check_index(slots, T, dev, "slots")
    with _on(dev):
        q = torch.empty((T, num_heads, cache.head_dim), dtype=torch.bfloat16, device=dev)
        _lib.check(
            _lib.lib().mxfp4_qk_norm_rope_cache(qkv.data_ptr(), stride, T, num_heads, cp, sp, rows, rot, int(interleaved),
                                                pos, qw, kw, wt, eps, q.data_ptr(), cache._ref, slots.data_ptr(),
                                                _stream_of(dev)),
            "mxfp4_qk_norm_rope_cache",
        )
    return q


def _row_stride(t, cache, T, what):
    _check_bf16(t, cache.device, what)
    _check(tuple(t.shape) == (T, cache.num_kv_heads, cache.head_dim), f"{what} must be [tokens, num_kv_heads, head_dim]")
    _check(t.stride(2) == 1 and (cache.num_kv_heads == 1 or t.stride(1) == cache.head_dim), f"{what}: a token's heads must be contiguous")
    return t.stride(0) if T > 1 else cache.num_kv_heads * cache.head_dim


def kv_cache_write(cache: MXKVCache, k, v, slots) -> None:
    """Codes ``k`` and ``v`` (bf16 ``[tokens, num_kv_heads, head_dim]``, each token's heads contiguous, any
    row stride that is a multiple of 8) into the cache rows ``slots`` names, as
    :func:`qk_norm_rope_cache` does: the OCP MX rule, the counterpart of
    ``quantize_mxfp4(..., rule="ocp")`` and :func:`quantize_act_mx8`."""
    _check(isinstance(cache, MXKVCache), "cache must be an MXKVCache")
    _check(isinstance(k, torch.Tensor) and k.dim() == 3, "k must be [tokens, num_kv_heads, head_dim]")
    T = k.shape[0]
    ks, vs = _row_stride(k, cache, T, "k"), _row_stride(v, cache, T, "v")
    _check_index(slots, T, cache.device, "slots")
    with _on(cache.device):
        _lib.check(
            _lib.lib().mxfp4_kv_cache_write(cache._ref, k.data_ptr(), ks, v.data_ptr(), vs, slots.data_ptr(), T,
                                            _stream_of(cache.device)),
            "mxfp4_kv_cache_write",
        )


def kv_cache_read(cache: MXKVCache, slots):
    """The rows ``slots`` (int32 ``[tokens]``) names, as new bf16 ``(k, v)`` of ``[tokens, num_kv_heads,
    head_dim]``; a negative slot reads zeros, the scale byte 255 NaN."""
    _check(isinstance(cache, MXKVCache), "cache must be an MXKVCache")
    _check(isinstance(slots, torch.Tensor) and slots.dim() == 1, "slots must be a vector")
    T, dev = slots.shape[0], cache.device
    _check_index(slots, T, dev, "slots")
    with _on(dev):
        k = torch.empty((T, cache.num_kv_heads, cache.head_dim), dtype=torch.bfloat16, device=dev)
        v = torch.empty_like(k)
        _lib.check(
            _lib.lib().mxfp4_kv_cache_read(cache._ref, slots.data_ptr(), T, k.data_ptr(), v.data_ptr(), _stream_of(dev)),
            "mxfp4_kv_cache_read",
        )
    return k, v


def paged_attention(q, cache: MXKVCache, page_table, lengths, scale: float | None = None, return_lse: bool = False,
                    out=None):
    """Attention of one new token per sequence over the cache.

    ``q`` bf16 ``[seqs, num_heads, head_dim]`` (each sequence's heads contiguous), num_heads a multiple of
    the cache's num_kv_heads: query head h reads kv head ``h // (num_heads // num_kv_heads)``.
    ``page_table`` int32 ``[seqs, max_pages]`` (rows of any stride): key j of sequence s is row ``j %
    page_size`` of page ``page_table[s, j // page_size]``, j < ``lengths[s]`` (int32); entries past the last
    page a sequence needs are not read.  A length of zero gives a row of zeros.  ``scale`` defaults to
    ``head_dim ** -0.5``.  Returns bf16 ``[seqs, num_heads, head_dim]`` (``out`` if given), with
    ``return_lse`` also fp32 ``[seqs, num_heads]``: the natural log of the sum of exp(scale * q . k), -inf
    for an empty sequence.  The same call gives the same bits.
    """
    _check(isinstance(cache, MXKVCache), "cache must be an MXKVCache")
    dev, D = cache.device, cache.head_dim
    _check_bf16(q, dev, "q")
    _check(q.dim() == 3 and q.shape[2] == D and q.shape[1] > 0, "q must be [seqs, num_heads, head_dim]")
    B, H = q.shape[0], q.shape[1]
    _check(H % cache.num_kv_heads == 0, "num_heads must be a multiple of num_kv_heads")
    _check(q.stride(2) == 1 and (H == 1 or q.stride(1) == D), "q: a sequence's heads must be contiguous")
    _check(isinstance(page_table, torch.Tensor) and page_table.is_cuda and page_table.device == dev
           and page_table.dtype == torch.int32, "page_table must be int32 on the cache's GPU")
    _check(page_table.dim() == 2 and page_table.shape[0] == B and page_table.shape[1] > 0
           and (page_table.shape[1] == 1 or page_table.stride(1) == 1), "page_table must be [seqs, max_pages] with contiguous rows")
    _check_index(lengths, B, dev, "lengths")
    P = page_table.shape[1]
    scale = D ** -0.5 if scale is None else float(scale)
    _check(math.isfinite(scale), "scale must be finite")
    with _on(dev):
        if out is None:
            out = torch.empty((B, H, D), dtype=torch.bfloat16, device=dev)
        else:
            _check_bf16(out, dev, "out")
            _check(tuple(out.shape) == (B, H, D) and out.is_contiguous(), "out shape/contig")
        lse = torch.empty((B, H), dtype=torch.float32, device=dev) if return_lse else None
        L = _lib.lib()
        nws = L.mxfp4_paged_attention_workspace_bytes(cache._ref, B, H, P)
        ws = torch.empty(nws, dtype=torch.uint8, device=dev)
        _lib.check(
            L.mxfp4_paged_attention(q.data_ptr(), q.stride(0) if B > 1 else H * D, cache._ref, page_table.data_ptr(),
                                    page_table.stride(0) if B > 1 else P, P, lengths.data_ptr(), B, H, scale,
                                    out.data_ptr(), lse.data_ptr() if return_lse else 0, ws.data_ptr(), nws,
                                    _stream_of(dev)),
            "mxfp4_paged_attention",
        )
    return (out, lse) if return_lse else out
