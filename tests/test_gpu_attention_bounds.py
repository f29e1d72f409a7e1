"""Bounds and ranges of the attention operators that hold past what tests/test_gpu_attention.py asks for."""

import numpy as np
import pytest
import torch

import _attention_ref as ref
from test_gpu_attention import FORMATS, _no_device_error, bf16, f64, i32, mx, random_cache, random_table  # noqa: F401

pytestmark = pytest.mark.gpu


def rows_of(cache, pages, n):
    """k and v of the first n keys of a sequence, in 64 bits [n, kv_heads, dim]."""
    out = []
    for codes, scales in ((cache.k_codes, cache.k_scales), (cache.v_codes, cache.v_scales)):
        c, s = (t.cpu().numpy()[pages].swapaxes(1, 2) for t in (codes, scales))
        out.append(ref.values(c.reshape(-1, *c.shape[2:])[:n], s.reshape(-1, *s.shape[2:])[:n], cache.format))
    return out


def check(got, lse, q, cache, table, lengths, scale):
    """Scores are fp32 sums of exact products, off by d = 2^-15 S as in test_gpu_attention.py; a weight by 2 d +
    2^-20 of the exponential and the sum, and by 2^-16 as the sum of two bf16 values (2^-8 each); the output
    is rounded to bf16 once, by 2^-8 of itself:  |err| <= 2^-8 |o| + (2^-16 + 2 d + 2^-20) A.  What is NaN has to
    be NaN, and nothing else."""
    got, qq = f64(got), f64(q)
    for b, n in enumerate(lengths):
        k, v = rows_of(cache, table[b, : -(-n // cache.page_size)], n)
        o, l, mag, size = ref.attention(qq[b], k, v, scale)
        d = 2.0**-15 * size
        lost = 2.0**-133 + n * 2.0**-126 * np.nanmax(np.abs(v))
        nan = np.isnan(o)
        assert np.array_equal(np.isnan(got[b]), nan), (b, n)
        bad = ~nan & ~(np.abs(got[b] - o) <= 2.0**-8 * np.abs(o) + (2.0**-16 + 2 * d[:, None] + 2.0**-20) * mag + lost)
        assert not bad.any(), (b, n, int(bad.sum()), got[b][bad][:4], o[bad][:4])
        if lse is not None:
            assert (np.abs(f64(lse)[b] - l) <= d + 2.0**-20 + 2.0**-22 * np.abs(l)).all(), (b, n)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 2), (64, 24, 2), (128, 8, 1), (128, 16, 1), (256, 3, 1), (256, 20, 2)])
def test_output_is_rounded_once(mx, fmt, dim, heads, kv):
    """Values of both signs whose sum is far smaller than they are: a weight rounded to 8 bits would show."""
    rng = np.random.default_rng(dim + heads)
    lengths = [3, 40, 129, 700, 6000]
    cache = random_cache(mx, rng, 110, kv, dim, 64, fmt)
    table = random_table(rng, cache, lengths)
    q = bf16(rng, (len(lengths), heads, dim), 0.05)
    out, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), scale=0.1, return_lse=True)
    check(out, lse, q, cache, table, lengths, 0.1)


@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 2), (64, 32, 2), (128, 8, 2), (128, 24, 2), (256, 6, 2)])
@pytest.mark.parametrize("longest,seqs", [(5, 6), (700, 6), (30000, 2), (900, 130)])
def test_nan_codes_of_values_are_nan(mx, dim, heads, kv, longest, seqs):
    """The two E4M3 codes that are NaN, in single values of every sequence but the last: at the first and last key and in
    between, in all places of a word.  Their own outputs are NaN, as kv_cache_read says, and no others."""
    rng = np.random.default_rng(dim + longest)
    lengths = [longest] + [int(n) for n in rng.integers(3, longest + 1, seqs - 1)]
    cache = random_cache(mx, rng, sum(-(-n // 64) for n in lengths) + 1, kv, dim, 64, "mxfp8")
    table = random_table(rng, cache, lengths)
    q = bf16(rng, (seqs, heads, dim))
    want = mx.paged_attention(q, cache, i32(table), i32(lengths))
    codes = cache.v_codes.cpu().numpy()
    for b, n in enumerate(lengths[:-1]):
        for key in {0, n - 1, n // 2, int(rng.integers(n))}:
            codes[table[b, key // 64], rng.integers(kv), key % 64, rng.integers(dim)] = (0x7F, 0xFF)[key % 2]
    cache.v_codes.copy_(torch.from_numpy(codes))
    out, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), return_lse=True)
    assert not want.isnan().any() and torch.equal(out[-1], want[-1])
    check(out, lse, q, cache, table, lengths, dim ** -0.5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads,kv", [(64, 3, 1), (64, 12, 1), (128, 8, 1), (128, 16, 1), (256, 5, 1)])
def test_value_scales_of_the_whole_range(mx, fmt, dim, heads, kv):
    """A sequence per scale byte of V, from the smallest to the largest whose values bf16 holds: none of them is
    lost, and none counts as another."""
    rng = np.random.default_rng(dim)
    last = 245 if fmt == "mxfp8" else 251
    bytes_ = [*range(0, 66), 100, 140, *range(188, 195), 220, last - 1, last]
    n = 37
    lengths = [n] * len(bytes_)
    cache = random_cache(mx, rng, len(bytes_), kv, dim, 64, fmt)
    table = random_table(rng, cache, lengths)
    for b, byte in enumerate(bytes_):
        cache.v_scales[table[b, 0]] = byte
    q = bf16(rng, (len(bytes_), heads, dim), 0.05)
    out, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), scale=0.1, return_lse=True)
    check(out, lse, q, cache, table, lengths, 0.1)
    assert (out.float().abs().amax((1, 2)) > 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 2), (128, 12, 1), (256, 2, 1)])
@pytest.mark.parametrize("longest,seqs", [(40, 8), (700, 8), (20000, 3)])
def test_value_scales_of_all_sizes_together(mx, fmt, dim, heads, kv, longest, seqs):
    """Groups of a sequence from classes far apart, a key of tiny or huge values among ordinary ones, and keys whose
    weight decides which of them counts: in full steps and at the end of a sequence."""
    rng = np.random.default_rng(longest + dim)
    lengths = [longest] + [int(n) for n in rng.integers(1, longest + 1, seqs - 1)]
    cache = random_cache(mx, rng, sum(-(-n // 64) for n in lengths) + 1, kv, dim, 64, fmt)
    table = random_table(rng, cache, lengths)
    scales = cache.v_scales.cpu().numpy()
    for b, n in enumerate(lengths):
        pages = table[b, : -(-n // 64)]
        if b % 4 == 0:
            scales[pages] = rng.integers(0, 240, scales[pages].shape)
        elif b % 4 == 1:
            scales[pages] = rng.integers(30, 100, scales[pages].shape)
        elif b % 4 == 2:  # one key's groups
            scales[pages[-1], :, (n - 1) % 64] = 20
            scales[pages[0], :, 0, 0] = 230
        else:
            scales[pages] = rng.choice([0, 62, 63, 64, 65], scales[pages].shape)
    cache.v_scales.copy_(torch.from_numpy(scales))
    q = bf16(rng, (seqs, heads, dim))
    out, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), return_lse=True)
    check(out, lse, q, cache, table, lengths, dim ** -0.5)
    again = mx.paged_attention(q, cache, i32(table), i32(lengths))
    assert torch.equal(out, again)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads,kv", [(64, 12, 3), (128, 20, 1), (256, 4, 2)])
@pytest.mark.parametrize("longest,seqs", [(60, 150), (700, 40), (20000, 3)])
def test_sums_beside_values_of_any_size(mx, fmt, dim, heads, kv, longest, seqs):
    """lse is as exact beside huge values as elsewhere, with scores near zero and in many short sums; a NaN scale
    loses no bits of the smallest values beside it; huge values of single keys meet other parts' ordinary ones."""
    rng = np.random.default_rng(longest + dim)
    lengths = [longest] + [int(n) for n in rng.integers(1, longest + 1, seqs - 1)]
    cache = random_cache(mx, rng, sum(-(-n // 64) for n in lengths) + 1, kv, dim, 64, fmt)
    table = random_table(rng, cache, lengths)
    scales = cache.v_scales.cpu().numpy()
    for b, n in enumerate(lengths):
        pages = table[b, : -(-n // 64)]
        if b % 3 == 0:
            for key in rng.integers(0, n, 3):
                scales[pages[key // 64], :, key % 64, rng.integers(dim // 32)] = rng.integers(192, 245)
        elif b % 3 == 1:
            scales[pages] = rng.integers(0, 60, scales[pages].shape)
            scales[pages[0], :, 0, 1] = 255
        else:
            scales[pages] = rng.integers(0, 245, scales[pages].shape)
    cache.v_scales.copy_(torch.from_numpy(scales))
    q = bf16(rng, (seqs, heads, dim), 0.01)
    out, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), scale=0.01, return_lse=True)
    check(out, lse, q, cache, table, lengths, 0.01)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_groups_of_zeros_among_values(mx, fmt, dim):
    """The coder gives them scale byte 0, which is the smallest scale there is when the codes are not zeros."""
    rng = np.random.default_rng(dim)
    n = 150
    cache = mx.new_kv_cache(6, 1, dim, 64, fmt)
    k, v = bf16(rng, (2 * n, 1, dim)), bf16(rng, (2 * n, 1, dim))
    v[:, :, dim // 2:] = 0
    v[3:9, :, :32] = -0.0
    v[n + 100, :, dim // 2:] = 2.0**-119  # nearly a group of zeros, in the second sequence
    pos = np.arange(n)
    table = np.array([[0, 1, 2], [3, 4, 5]])
    slots = np.r_[pos, 192 + pos]
    mx.kv_cache_write(cache, k, v, i32(slots))
    q = bf16(rng, (2, 4, dim))
    out, lse = mx.paged_attention(q, cache, i32(table), i32([n, n]), return_lse=True)
    check(out, lse, q, cache, table, [n, n], dim ** -0.5)
    assert (out[0, :, dim // 2:] == 0).all() and (out[1, :, dim // 2:] > 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads,kv,step", [(64, 4, 2, 90), (64, 20, 2, 35), (128, 8, 1, 40), (128, 16, 1, 13), (256, 3, 1, 17), (256, 9, 1, 12)])
@pytest.mark.parametrize("longest", [30, 3000])
def test_small_query_values_count(mx, fmt, dim, heads, kv, step, longest):
    """Query values 2^step smaller from group to group against keys as much larger: every group has the same share
    of a score, so none may be rounded as a part of the largest."""
    rng = np.random.default_rng(dim + step)
    lengths = [longest, 17, longest // 2]
    cache = random_cache(mx, rng, sum(-(-n // 64) for n in lengths) + 1, kv, dim, 64, fmt)
    table = random_table(rng, cache, lengths)
    groups = np.arange(dim // 32)
    mid = (groups[-1] * step) // 2
    q = bf16(rng, (3, heads, dim)).unflatten(2, (-1, 32))
    q *= torch.from_numpy(np.exp2(mid - groups * float(step))).cuda()[:, None].bfloat16()
    cache.k_scales.add_(torch.from_numpy(((groups * step - mid) % 256).astype(np.uint8)).cuda())
    out, lse = mx.paged_attention(q.flatten(2), cache, i32(table), i32(lengths), return_lse=True)
    check(out, lse, q.flatten(2), cache, table, lengths, dim ** -0.5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads", [(64, 3), (128, 16), (256, 2)])
def test_small_query_values_beside_zeros_of_keys(mx, fmt, dim, heads):
    """Within one group: the key is zero where the query is large, so the small values alone make the score."""
    rng = np.random.default_rng(dim)
    lengths = [200, 70, 16, 16]
    cache = random_cache(mx, rng, 12, 1, dim, 64, fmt)
    table = random_table(rng, cache, lengths)
    q = bf16(rng, (4, heads, dim))
    for b, power in enumerate((30, 60, 100, 126)):
        q[b, :, ::8] *= 2.0**power
        q[b, :, 1::8] *= 2.0**-100  # and smaller ones yet
    if fmt == "mxfp8":
        cache.k_codes[..., ::8] = 0
    else:
        cache.k_codes[..., ::4] &= 0xF0
    out, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), return_lse=True)
    check(out, lse, q, cache, table, lengths, dim ** -0.5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads", [(64, 3), (128, 16), (256, 2)])
@pytest.mark.parametrize("q_power,k_power,scale_power", [(-110, 110, 0), (110, -110, 0), (0, 100, -100), (100, 20, -120), (-60, -60, 120),
                                                         (126, -117, -9), (-120, 0, 120), (60, 63, -123), (-120, 124, -4), (-100, 124, -24), (120, -118, -2)])
def test_queries_and_keys_of_every_size(mx, fmt, dim, heads, q_power, k_power, scale_power):
    """Ordinary scores from factors that no product of two of them need hold."""
    rng = np.random.default_rng(dim)
    lengths = [300, 20]
    cache = random_cache(mx, rng, 8, 1, dim, 64, fmt, spread=1)
    table = random_table(rng, cache, lengths)
    cache.k_scales.add_(k_power % 256)
    q = (bf16(rng, (2, heads, dim)).float() * 2.0**q_power).bfloat16()
    scale = dim ** -0.5 * 2.0**scale_power
    out, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), scale=scale, return_lse=True)
    check(out, lse, q, cache, table, lengths, scale)


@pytest.mark.parametrize("fmt", FORMATS)
def test_key_groups_of_zeros_and_heads_of_zeros(mx, fmt):
    """A head padded with zeros, as the coder stores it (scale byte 0), and a query of zeros beside one that is not."""
    rng = np.random.default_rng(2)
    n = 150
    cache = mx.new_kv_cache(3, 2, 128, 64, fmt)
    k, v = bf16(rng, (n, 2, 128)), bf16(rng, (n, 2, 128))
    k[:, :, 96:] = 0
    k[40:50, 0, 32:64] = -0.0
    mx.kv_cache_write(cache, k, v, i32(np.arange(n)))
    q = bf16(rng, (1, 4, 128))
    q[0, 1] = 0
    table = np.array([[0, 1, 2]])
    out, lse = mx.paged_attention(q, cache, i32(table), i32([n]), return_lse=True)
    check(out, lse, q, cache, table, [n], 128 ** -0.5)


# ------------------------------------------------------------------------------- the cache's tensors
def test_a_cache_follows_its_tensors_storage(mx):
    """Each call takes the memory that the tensors have then, and refuses tensors of another form or without storage."""
    rng = np.random.default_rng(3)
    cache = random_cache(mx, rng, 6, 2, 64, 16, "mxfp8")
    names = ("k_codes", "v_codes", "k_scales", "v_scales")
    table, lengths, slots = i32([[1, 3, 5]]), i32([40]), i32([17, 18, 90])
    q, k, qkv = bf16(rng, (1, 4, 64)), bf16(rng, (3, 2, 64)), bf16(rng, (3, 8 * 64))
    want, rows = mx.paged_attention(q, cache, table, lengths), mx.kv_cache_read(cache, slots)
    for name in names:  # moved elsewhere: the same bytes at other addresses, the old ones overwritten
        t = getattr(cache, name)
        old, moved = t.data, t.detach().clone()
        t.data = moved
        old.fill_(0)
    assert torch.equal(mx.paged_attention(q, cache, table, lengths), want)
    assert all(torch.equal(a, b) for a, b in zip(mx.kv_cache_read(cache, slots), rows))
    mx.kv_cache_write(cache, k, k, slots)
    assert (cache.k_codes[1, :, 1] != 0).any()  # slot 17

    calls = [lambda: mx.paged_attention(q, cache, table, lengths), lambda: mx.kv_cache_read(cache, slots),
             lambda: mx.kv_cache_write(cache, k, k, slots), lambda: mx.qk_norm_rope_cache(qkv, 4, 2, None, None, cache, slots)]
    for name in names:
        t = getattr(cache, name)
        good = t.data
        for other in (good.cpu(), good[:3], good[..., :1], good.to(torch.int32), good.transpose(0, 2),
                      torch.empty((0,), dtype=torch.uint8, device="cuda")):
            t.data = other
            for call in calls:
                with pytest.raises(RuntimeError, match="cache's tensors"):
                    call()
        t.data = good
        storage, n = t.untyped_storage(), t.numel()
        saved = t.clone()
        storage.resize_(n - 1)
        for call in calls:
            with pytest.raises(RuntimeError, match="cache's tensors"):
                call()
        storage.resize_(n)
        t.copy_(saved)
    mx.paged_attention(q, cache, table, lengths)


# ------------------------------------------------------------------------------------------- slots
@pytest.mark.parametrize("tokens,later", [(2, 1), (7, 3), (200, 150), (200, 199), (4096, 4095), (5000, 4500)])
@pytest.mark.parametrize("shift", [0, 1])
def test_a_token_without_a_position_does_not_take_a_slot_from_another(mx, tokens, later, shift):
    """Token 0 and a later one name a slot; the later one's position is outside the tables, so it is not stored: the
    first one's rows are, whether one launch holds both or not.  A third token, in between, wins where it is good."""
    rng = np.random.default_rng(tokens)
    kv, dim, page = 2, 64, 16
    x = bf16(rng, (tokens, 6 * dim))  # 2 heads of each kind
    angle = np.arange(8)[:, None] * 10000.0 ** (-np.arange(0, dim, 2) / dim)
    cos, sin = (torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))
    for between in {0, later // 2}:
        cache = mx.new_kv_cache(-(-tokens // page) + 1, kv, dim, page)
        want = mx.new_kv_cache(cache.num_pages, kv, dim, page)
        slots, pos = np.arange(tokens), rng.integers(0, 8, tokens)
        slots[later] = slots[between] = slots[0]
        pos[later] = 8 if tokens % 2 else -1
        pad = i32(np.r_[np.full(shift, 3), slots])[shift:]
        mx.qk_norm_rope_cache(x, 2, kv, cos, sin, cache, pad, positions=i32(pos))
        assert mx.device_error() == 0x202
        alone = slots.copy()
        alone[later] = -1
        alone[:between] = np.where(alone[:between] == slots[0], -1, alone[:between])
        mx.qk_norm_rope_cache(x, 2, kv, cos, sin, want, i32(alone), positions=i32(np.maximum(pos, 0) % 8))
        for a, b in zip((cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales), (want.k_codes, want.v_codes, want.k_scales, want.v_scales)):
            assert torch.equal(a, b)
        assert mx.device_error() == 0


# ---------------------------------------------------------------------------------------- refusals
def test_out_over_a_part_of_q_is_refused(mx):
    rng = np.random.default_rng(1)
    cache = random_cache(mx, rng, 4, 1, 64, 16, "mxfp8")
    table, lengths = i32([[0, 1], [2, 3], [1, 0]]), i32([20, 30, 7])
    buf = bf16(rng, (8, 4, 64))
    q = buf[2:5]
    values = q.clone()
    want = mx.paged_attention(values, cache, table, lengths)
    wide = torch.zeros((3, 4 * 64 * 6), dtype=torch.bfloat16, device="cuda")
    rows = wide[:, :256].unflatten(1, (4, 64))
    rows.copy_(q)
    flat = wide.view(-1)
    for query, out in ((q, buf[1:4]), (q, buf[4:7]), (rows, flat[:768].view(3, 4, 64)), (rows, flat[1536 - 760:][:768].view(3, 4, 64)),
                       (rows, flat[200:968].view(3, 4, 64)), (q, buf.view(-1)[2 * 256 + 8:][:768].view(3, 4, 64))):
        with pytest.raises(RuntimeError, match="overlaps q"):
            mx.paged_attention(query, cache, table, lengths, out=out)
    for query, out in ((q, buf[5:8]), (buf[3:6], buf[:3]), (rows, flat[256:1024].view(3, 4, 64)), (rows, flat[1536 - 768:1536].view(3, 4, 64)), (q, q)):
        query.copy_(values)
        assert torch.equal(mx.paged_attention(query, cache, table, lengths, out=out), want)
