"""CPU tests of the attention operators' argument checks: the C ABI refuses before it touches CUDA,
and the Python entry points refuse what is not on a GPU or has another form."""

import ctypes

import pytest
import torch

BIG = 1 << 40


@pytest.fixture(scope="module")
def L():
    from mxfp4_b200 import _lib

    return _lib


P = ctypes.c_void_p
p = P(4096)  # never dereferenced: the checks come first


def cache_of(L, pages=4, heads=2, page=64, dim=128, fmt=0, ptr=4096):
    return L.KVCache(ptr, ptr, ptr, ptr, pages, heads, page, dim, fmt)


def rope(L, qkv=p, stride=1024, tokens=4, heads=4, kv=2, dim=128, cos=p, sin=p, rows=8, rot=128, pos=None, qw=None, kw=None,
         wt=1, eps=1e-6, q=p, k=p):
    return L.lib().mxfp4_qk_norm_rope(qkv, stride, tokens, heads, kv, dim, cos, sin, rows, rot, 0, pos, qw, kw, wt, eps, q, k, None)


@pytest.mark.parametrize("change,code", [
    ({"qkv": None}, 1000), ({"q": None}, 1000), ({"k": None}, 1000), ({"tokens": -1}, 1000), ({"heads": 0}, 1000), ({"kv": 0}, 1000),
    ({"cos": None}, 1000), ({"rows": 0}, 1000), ({"rows": 3}, 1000), ({"qw": p}, 1000), ({"wt": 5}, 1000), ({"eps": -1.0}, 1000),
    ({"eps": float("nan")}, 1000), ({"stride": 1016}, 1000), ({"dim": 100, "rot": 0}, 1001), ({"dim": 288, "stride": 4096}, 1001),
    ({"rot": 24}, 1001), ({"rot": 144}, 1001), ({"rot": -16}, 1000), ({"stride": 1025}, 1002), ({"qkv": P(4098)}, 1002),
    ({"cos": P(4100)}, 1002), ({"k": P(4104)}, 1002), ({"heads": 1 << 23, "stride": 1 << 31}, 1001),
    ({"kv": 1 << 30, "stride": 1 << 40}, 1001),
])
def test_norm_rope_refuses(L, change, code):
    assert rope(L, **change) == code


@pytest.mark.parametrize("change,code", [
    ({"pages": 0}, 1000), ({"heads": 0}, 1000), ({"fmt": 2}, 1000), ({"dim": 96}, 1001), ({"dim": 512}, 1001), ({"page": 48}, 1001),
    ({"page": 8}, 1001), ({"page": 512}, 1001), ({"pages": 1 << 25}, 1001), ({"heads": 1 << 23}, 1001), ({"ptr": 0}, 1000), ({"ptr": 4104}, 1002),
])
def test_every_cache_entry_refuses_a_bad_cache(L, change, code):
    lib, c = L.lib(), ctypes.byref(cache_of(L, **change))
    assert lib.mxfp4_kv_cache_write(c, p, 256, p, 256, p, 4, None) == code
    assert lib.mxfp4_kv_cache_read(c, p, 4, p, p, None) == code
    assert lib.mxfp4_paged_attention(p, 4096, c, p, 4, 4, p, 2, 4, 1.0, p, None, p, BIG, None) == code
    assert lib.mxfp4_paged_attention_workspace_bytes(c, 2, 4, 4) == 0
    assert lib.mxfp4_qk_norm_rope_cache(p, 4096, 4, 4, p, p, 8, 64, 0, None, None, None, 1, 1e-6, p, c, p, None) == code


def test_cache_entries_refuse_bad_arguments(L):
    lib, c = L.lib(), ctypes.byref(cache_of(L))
    assert lib.mxfp4_kv_cache_write(None, p, 256, p, 256, p, 4, None) == 1000
    assert lib.mxfp4_kv_cache_write(c, p, 256, p, 256, None, 4, None) == 1000
    assert lib.mxfp4_kv_cache_write(c, p, 255, p, 256, p, 4, None) == 1000  # rows overlap
    assert lib.mxfp4_kv_cache_write(c, p, 260, p, 256, p, 4, None) == 1002
    assert lib.mxfp4_kv_cache_write(c, p, 256, P(4100), 256, p, 4, None) == 1002
    assert lib.mxfp4_kv_cache_write(c, p, 256, p, 256, p, -1, None) == 1000
    assert lib.mxfp4_kv_cache_write(c, None, 256, None, 256, None, 0, None) == 0  # nothing to do
    assert lib.mxfp4_kv_cache_read(c, None, 4, p, p, None) == 1000
    assert lib.mxfp4_kv_cache_read(c, p, 4, P(4100), p, None) == 1002
    assert lib.mxfp4_kv_cache_read(c, None, 0, None, None, None) == 0
    assert lib.mxfp4_qk_norm_rope_cache(p, 1024, 4, 4, p, p, 8, 64, 0, None, None, None, 1, 1e-6, p, c, None, None) == 1000
    assert lib.mxfp4_qk_norm_rope_cache(p, 1016, 4, 4, p, p, 8, 64, 0, None, None, None, 1, 1e-6, p, c, p, None) == 1000


def attend(L, q=p, stride=1024, table=p, tstride=4, pages=4, lengths=p, seqs=2, heads=4, out=p, lse=None, ws=p, n=BIG):
    c = ctypes.byref(cache_of(L))
    return L.lib().mxfp4_paged_attention(q, stride, c, table, tstride, pages, lengths, seqs, heads, 1.0, out, lse, ws, n, None)


@pytest.mark.parametrize("change,code", [
    ({"q": None}, 1000), ({"table": None}, 1000), ({"lengths": None}, 1000), ({"out": None}, 1000), ({"heads": 0}, 1000), ({"heads": 3}, 1001),
    ({"seqs": -1}, 1000), ({"pages": 0}, 1000), ({"tstride": 3}, 1000), ({"stride": 504}, 1000), ({"stride": 1028}, 1002), ({"q": P(4100)}, 1002),
    ({"out": P(4100)}, 1002), ({"ws": P(4100)}, 1002), ({"pages": 1 << 26, "tstride": 1 << 26}, 1001), ({"seqs": 1 << 30}, 1001), ({"seqs": 1 << 28}, 1001), ({"seqs": 1 << 20, "pages": 1 << 17, "tstride": 1 << 17}, 1001),
    ({"seqs": 0}, 0), ({"heads": 1 << 23, "stride": 1 << 30}, 1001),
])
def test_attention_refuses(L, change, code):
    assert attend(L, **change) == code


def test_workspace_is_none_for_short_tables_and_bounded_for_long_ones(L):
    """Nothing where a cluster takes a head; else the resident blocks' parts and a word pair per head."""
    lib = L.lib()
    c = ctypes.byref(cache_of(L, heads=8, pages=1 << 20))
    sizes = [lib.mxfp4_paged_attention_workspace_bytes(c, b, 64, n) for b, n in ((1, 1), (16, 16), (1, 4096), (64, 4096), (4096, 4096))]
    assert sizes[0] == sizes[1] == 0 and all(s % 16 == 0 for s in sizes)
    assert 0 < sizes[2] <= sizes[3] <= sizes[4] < 64 << 20


def test_python_entry_points_refuse_what_is_not_on_a_gpu():
    import mxfp4_b200 as mx

    x = torch.zeros((2, 4 * 64), dtype=torch.bfloat16)
    u = torch.zeros((2, 1, 16, 64), dtype=torch.uint8)
    s = torch.zeros((2, 1, 16, 2), dtype=torch.uint8)
    with pytest.raises(RuntimeError):
        mx.qk_norm_rope(x, 2, 1)
    with pytest.raises(RuntimeError):
        mx.MXKVCache(u, u, s, s)
    with pytest.raises(RuntimeError):
        mx.MXKVCache(u, u, s, s, format="fp8")
    with pytest.raises(RuntimeError):
        mx.kv_cache_write(None, x, x, x)
    with pytest.raises(RuntimeError):
        mx.kv_cache_read(None, x)
    with pytest.raises(RuntimeError):
        mx.paged_attention(x, None, x, x)


@pytest.mark.gpu
def test_python_entry_points_refuse_other_forms():
    import mxfp4_b200 as mx

    def gpu(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    c = mx.new_kv_cache(4, 2, 64, 16)
    idx, qkv, cos = gpu(3, dtype=torch.int32), gpu(3, 8 * 64), gpu(8, 32, dtype=torch.float32)
    w = gpu(64)
    bad = [
        lambda: mx.qk_norm_rope(qkv.float(), 4, 2, cos, cos),
        lambda: mx.qk_norm_rope(qkv, 5, 2, cos, cos),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos, None),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos, cos[:4]),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos[:2], cos[:2]),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos.double(), cos.double()),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos, cos, positions=idx.long()),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos, cos, positions=idx[:2]),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos, cos, positions=idx.cpu()),
        lambda: mx.qk_norm_rope(qkv, 4, 2, None, None, positions=idx),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos, cos, q_weight=w),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos, cos, q_weight=w, k_weight=w.float()),
        lambda: mx.qk_norm_rope(qkv, 4, 2, cos, cos, q_weight=w[:32], k_weight=w[:32]),
        lambda: mx.qk_norm_rope(qkv.t().contiguous().t(), 4, 2, cos, cos),
        lambda: mx.qk_norm_rope_cache(qkv, 6, 1, cos, cos, c, idx),
        lambda: mx.qk_norm_rope_cache(qkv, 4, 2, cos, cos, c, idx[:2]),
        lambda: mx.kv_cache_write(c, gpu(3, 2, 64), gpu(3, 2, 32), idx),
        lambda: mx.kv_cache_write(c, gpu(3, 2, 64), gpu(2, 2, 64), idx),
        lambda: mx.kv_cache_write(c, gpu(2, 3, 64).transpose(0, 1), gpu(3, 2, 64), idx),
        lambda: mx.kv_cache_write(c, gpu(3, 2, 64), gpu(3, 2, 64), idx.long()),
        lambda: mx.kv_cache_write(c, gpu(3, 130)[:, 1:129].unflatten(1, (2, 64)), gpu(3, 2, 64), idx),
        lambda: mx.kv_cache_read(c, idx.long()),
        lambda: mx.new_kv_cache(4, 2, 96),
        lambda: mx.new_kv_cache(4, 2, 64, 48),
        lambda: mx.new_kv_cache(4, 2, 64, format="e4m3"),
        lambda: mx.MXKVCache(c.k_codes[:, :1], c.v_codes, c.k_scales, c.v_scales),
        lambda: mx.MXKVCache(c.k_codes, c.v_codes, c.k_scales, c.v_scales, format="mxfp4"),
        lambda: mx.paged_attention(gpu(3, 3, 64), c, gpu(3, 2, dtype=torch.int32), idx),
        lambda: mx.paged_attention(gpu(3, 4, 32), c, gpu(3, 2, dtype=torch.int32), idx),
        lambda: mx.paged_attention(gpu(3, 4, 64), c, gpu(2, 2, dtype=torch.int32), idx),
        lambda: mx.paged_attention(gpu(3, 4, 64), c, gpu(3, 0, dtype=torch.int32), idx),
        lambda: mx.paged_attention(gpu(3, 4, 64), c, gpu(2, 3, dtype=torch.int32).t(), idx),
        lambda: mx.paged_attention(gpu(3, 4, 64), c, gpu(3, 2, dtype=torch.int32), idx.long()),
        lambda: mx.paged_attention(gpu(3, 4, 64), c, gpu(3, 2, dtype=torch.int32), idx, scale=float("inf")),
        lambda: mx.paged_attention(gpu(3, 4, 64), c, gpu(3, 2, dtype=torch.int32), idx, scale=1e39),
        lambda: setattr(c, "k_codes", c.v_codes),
        lambda: mx.paged_attention(gpu(3, 4, 64), c, gpu(3, 2, dtype=torch.int32), idx, out=gpu(3, 4, 32)),
        lambda: mx.paged_attention(gpu(3, 4, 64).float(), c, gpu(3, 2, dtype=torch.int32), idx),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was accepted")
    torch.cuda.synchronize()
