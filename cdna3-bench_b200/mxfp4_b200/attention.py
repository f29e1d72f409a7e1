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
import math

import torch

from . import _lib
from .kernels import _check, _require_cuda

KV_FORMATS = {"mxfp8": _lib.KV_MXFP8, "mxfp4": _lib.KV_MXFP4}
_PAGE_SIZES = (16, 32, 64, 128, 256)

# A decoding step calls these with GPU work of a few microseconds, so the checks are plain conditions
# (a message is only made for a call that is refused), devices are compared by index (-1: the CPU)
# and the current stream is asked for by index.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
_device = torch.cuda.current_device
_BF16, _F32, _I32, _Tensor = torch.bfloat16, torch.float32, torch.int32, torch.Tensor


def _on_device(index: int, fn, *args) -> int:
    """fn(*args, stream) with device `index`, which is not the current one, made current."""
    with torch.cuda.device(index):
        return fn(*args, _raw_stream(index))


def _index(t, n: int, dev: int, what: str) -> int:
    """Address of an int32 vector of n on device `dev`."""
    if not (isinstance(t, _Tensor) and t.dtype is _I32 and t.get_device() == dev and t.dim() == 1 and t.shape[0] == n
            and (n < 2 or t.stride(0) == 1)):
        raise RuntimeError(f"{what} must be a contiguous int32 vector of {n} on cuda:{dev}")
    return t.data_ptr()


class MXKVCache:
    """A paged key-value cache in an MX format (byte layout: ``mxfp4_kv_cache`` in the C header).

    ``k_codes`` / ``v_codes``: uint8 ``[num_pages, num_kv_heads, page_size, head_dim]`` E4M3 codes
    (``format="mxfp8"``) or ``[..., head_dim // 2]`` pairs of E2M1 codes (``"mxfp4"``, even element in
    the low nibble); ``k_scales`` / ``v_scales``: uint8 ``[..., head_dim // 32]`` E8M0 bytes.  The
    tensors are contiguous and stay the caller's: the object only refers to them.  head_dim 64, 128
    or 256; page_size 16, 32, 64, 128 or 256.  :func:`new_kv_cache` allocates one.
    """

    __slots__ = ("k_codes", "v_codes", "k_scales", "v_scales", "format", "num_pages", "num_kv_heads", "page_size",
                 "head_dim", "device", "_index", "_struct", "_ref")

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
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.format, self.num_pages, self.num_kv_heads, self.page_size, self.head_dim = format, pages, heads, size, dim
        self.device = k_codes.device
        self._index = k_codes.get_device()
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


def _rope_arguments(qkv, heads, kv_heads, dim, cos, sin, positions, q_weight, k_weight):
    """Checks what the two norm-and-rotation calls share.  Returns tokens, the device's index, qkv's row
    stride, and the C entry's cos, sin, table_rows, rot, positions, q_weight, k_weight, weight_dtype."""
    if not (isinstance(qkv, _Tensor) and qkv.dtype is _BF16 and qkv.dim() == 2 and qkv.stride(1) == 1):
        raise RuntimeError("qkv must be bfloat16 [tokens, width] on the GPU with contiguous rows")
    tokens, width = qkv.shape
    dev = qkv.get_device()
    if dev < 0 or heads <= 0 or kv_heads <= 0 or width != (heads + 2 * kv_heads) * dim:
        raise RuntimeError("qkv must be on the GPU, its width (num_heads + 2 * num_kv_heads) * head_dim")
    rows = rot = cp = sp = pos = qw = kw = 0
    wt = _lib.DTYPE_BF16
    if cos is not None or sin is not None:
        if not (isinstance(cos, _Tensor) and isinstance(sin, _Tensor) and cos.dtype is _F32 and sin.dtype is _F32
                and cos.get_device() == dev and sin.get_device() == dev and cos.dim() == 2 and cos.shape == sin.shape
                and cos.is_contiguous() and sin.is_contiguous()):
            raise RuntimeError(f"cos and sin must be contiguous float32 [rows, rot / 2] of one shape on cuda:{dev}")
        rows, rot = cos.shape
        rot *= 2
        if rows == 0 or rot == 0:
            raise RuntimeError("cos and sin must not be empty")
        cp, sp = cos.data_ptr(), sin.data_ptr()
    if positions is not None:
        if not rot:
            raise RuntimeError("positions without cos and sin")
        pos = _index(positions, tokens, dev, "positions")
    elif rows < tokens and rot:
        raise RuntimeError("cos and sin need a row per token when no positions are given")
    if q_weight is not None or k_weight is not None:
        for w in (q_weight, k_weight):
            if not (isinstance(w, _Tensor) and w.get_device() == dev and w.dtype in (_BF16, _F32) and w.dim() == 1
                    and w.shape[0] == dim and w.is_contiguous()):
                raise RuntimeError(f"q_weight and k_weight come together, contiguous bfloat16 or float32 [head_dim] on cuda:{dev}")
        if q_weight.dtype is not k_weight.dtype:
            raise RuntimeError("q_weight and k_weight must have one type")
        qw, kw = q_weight.data_ptr(), k_weight.data_ptr()
        if q_weight.dtype is _F32:
            wt = _lib.DTYPE_F32
    return tokens, dev, qkv.stride(0) if tokens > 1 else width, cp, sp, rows, rot, pos, qw, kw, wt


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
    if not (isinstance(qkv, _Tensor) and qkv.dim() == 2 and num_heads > 0 and num_kv_heads > 0):
        raise RuntimeError("qkv must be bfloat16 [tokens, width] on the GPU with contiguous rows")
    dim = qkv.shape[1] // (num_heads + 2 * num_kv_heads)
    tokens, dev, stride, cp, sp, rows, rot, pos, qw, kw, wt = _rope_arguments(
        qkv, num_heads, num_kv_heads, dim, cos, sin, positions, q_weight, k_weight)
    q, k = qkv.new_empty((tokens, num_heads, dim)), qkv.new_empty((tokens, num_kv_heads, dim))
    fn = _lib.lib().mxfp4_qk_norm_rope
    args = (qkv.data_ptr(), stride, tokens, num_heads, num_kv_heads, dim, cp, sp, rows, rot, interleaved, pos, qw, kw, wt, eps,
            q.data_ptr(), k.data_ptr())
    code = fn(*args, _raw_stream(dev)) if dev == _device() else _on_device(dev, fn, *args)
    if code:
        _lib.check(code, "mxfp4_qk_norm_rope")
    return q, k


def qk_norm_rope_cache(qkv, num_heads: int, num_kv_heads: int, cos, sin, cache: MXKVCache, slots, positions=None,
                       q_weight=None, k_weight=None, eps: float = 1e-6, interleaved: bool = False):
    """:func:`qk_norm_rope` that writes the keys and values into ``cache`` instead of returning keys.

    ``slots`` int32 ``[tokens]``: token t goes to row ``slots[t] % page_size`` of page ``slots[t] //
    page_size``; a negative slot stores nothing (a batch's padding); of two tokens with one slot the
    later is stored.  Keys are coded from the unrounded rotated value, values from ``qkv`` as they
    are.  ``cos`` and ``sin`` may be None (no rotation).  Returns q.
    """
    if not (isinstance(cache, MXKVCache) and num_kv_heads == cache.num_kv_heads):
        raise RuntimeError("cache must be an MXKVCache of num_kv_heads heads")
    dim = cache.head_dim
    tokens, dev, stride, cp, sp, rows, rot, pos, qw, kw, wt = _rope_arguments(
        qkv, num_heads, num_kv_heads, dim, cos, sin, positions, q_weight, k_weight)
    if dev != cache._index:
        raise RuntimeError("qkv must be on the cache's GPU")
    at = _index(slots, tokens, dev, "slots")
    q = qkv.new_empty((tokens, num_heads, dim))
    fn = _lib.lib().mxfp4_qk_norm_rope_cache
    args = (qkv.data_ptr(), stride, tokens, num_heads, cp, sp, rows, rot, interleaved, pos, qw, kw, wt, eps, q.data_ptr(),
            cache._ref, at)
    code = fn(*args, _raw_stream(dev)) if dev == _device() else _on_device(dev, fn, *args)
    if code:
        _lib.check(code, "mxfp4_qk_norm_rope_cache")
    return q


def _row_stride(t, cache, tokens, what):
    heads, dim = cache.num_kv_heads, cache.head_dim
    if not (isinstance(t, _Tensor) and t.dtype is _BF16 and t.get_device() == cache._index and t.shape == (tokens, heads, dim)
            and t.stride(2) == 1 and (heads == 1 or t.stride(1) == dim)):
        raise RuntimeError(f"{what} must be bfloat16 [tokens, num_kv_heads, head_dim] on the cache's GPU, a token's heads contiguous")
    return t.stride(0) if tokens > 1 else heads * dim


def kv_cache_write(cache: MXKVCache, k, v, slots) -> None:
    """Codes ``k`` and ``v`` (bf16 ``[tokens, num_kv_heads, head_dim]``, each token's heads contiguous, any
    row stride that is a multiple of 8) into the cache rows ``slots`` names, as
    :func:`qk_norm_rope_cache` does: the OCP MX rule, the counterpart of
    ``quantize_mxfp4(..., rule="ocp")`` and :func:`quantize_act_mx8`."""
    if not (isinstance(cache, MXKVCache) and isinstance(k, _Tensor) and k.dim() == 3):
        raise RuntimeError("cache must be an MXKVCache, k [tokens, num_kv_heads, head_dim]")
    tokens, dev = k.shape[0], cache._index
    ks, vs = _row_stride(k, cache, tokens, "k"), _row_stride(v, cache, tokens, "v")
    fn = _lib.lib().mxfp4_kv_cache_write
    args = (cache._ref, k.data_ptr(), ks, v.data_ptr(), vs, _index(slots, tokens, dev, "slots"), tokens)
    code = fn(*args, _raw_stream(dev)) if dev == _device() else _on_device(dev, fn, *args)
    if code:
        _lib.check(code, "mxfp4_kv_cache_write")


def kv_cache_read(cache: MXKVCache, slots):
    """The rows ``slots`` (int32 ``[tokens]``) names, as new bf16 ``(k, v)`` of ``[tokens, num_kv_heads,
    head_dim]``; a negative slot reads zeros, the scale byte 255 NaN."""
    if not (isinstance(cache, MXKVCache) and isinstance(slots, _Tensor) and slots.dim() == 1):
        raise RuntimeError("cache must be an MXKVCache, slots a vector")
    tokens, dev = slots.shape[0], cache._index
    at = _index(slots, tokens, dev, "slots")
    shape = (tokens, cache.num_kv_heads, cache.head_dim)
    k, v = slots.new_empty(shape, dtype=_BF16), slots.new_empty(shape, dtype=_BF16)
    fn = _lib.lib().mxfp4_kv_cache_read
    args = (cache._ref, at, tokens, k.data_ptr(), v.data_ptr())
    code = fn(*args, _raw_stream(dev)) if dev == _device() else _on_device(dev, fn, *args)
    if code:
        _lib.check(code, "mxfp4_kv_cache_read")
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
    if not isinstance(cache, MXKVCache):
        raise RuntimeError("cache must be an MXKVCache")
    dev, dim = cache._index, cache.head_dim
    if not (isinstance(q, _Tensor) and q.dtype is _BF16 and q.get_device() == dev and q.dim() == 3):
        raise RuntimeError("q must be bfloat16 [seqs, num_heads, head_dim] on the cache's GPU")
    seqs, heads, width = q.shape
    row, step, one = q.stride()
    if width != dim or one != 1 or heads == 0 or heads % cache.num_kv_heads or (step != dim and heads > 1):
        raise RuntimeError("q: num_heads must be a multiple of num_kv_heads, a sequence's heads contiguous")
    if not (isinstance(page_table, _Tensor) and page_table.dtype is _I32 and page_table.get_device() == dev and page_table.dim() == 2):
        raise RuntimeError("page_table must be int32 [seqs, max_pages] on the cache's GPU")
    rows, pages = page_table.shape
    table_row, one = page_table.stride()
    if rows != seqs or pages == 0 or (one != 1 and pages > 1):
        raise RuntimeError("page_table must be [seqs, max_pages] with contiguous rows")
    lens = _index(lengths, seqs, dev, "lengths")
    if scale is None:
        scale = dim ** -0.5
    elif not math.isfinite(scale):
        raise RuntimeError("scale must be finite")
    if out is None:
        out = q.new_empty((seqs, heads, dim))
    elif not (isinstance(out, _Tensor) and out.dtype is _BF16 and out.get_device() == dev and out.shape == q.shape and out.is_contiguous()):
        raise RuntimeError("out must be contiguous bfloat16 [seqs, num_heads, head_dim] on the cache's GPU")
    lse = q.new_empty((seqs, heads), dtype=_F32) if return_lse else None
    L = _lib.lib()
    nws = L.mxfp4_paged_attention_workspace_bytes(cache._ref, seqs, heads, pages)
    ws = q.new_empty(nws // 2)
    fn = L.mxfp4_paged_attention
    args = (q.data_ptr(), row if seqs > 1 else heads * dim, cache._ref, page_table.data_ptr(), table_row if seqs > 1 else pages, pages,
            lens, seqs, heads, scale, out.data_ptr(), lse.data_ptr() if return_lse else 0, ws.data_ptr(), nws)
    code = fn(*args, _raw_stream(dev)) if dev == _device() else _on_device(dev, fn, *args)
    if code:
        _lib.check(code, "mxfp4_paged_attention")
    return (out, lse) if return_lse else out
