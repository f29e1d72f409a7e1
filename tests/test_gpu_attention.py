"""The operators between the QKV GEMM and the output GEMM (mxfp4_b200.attention) against plain
64-bit forms (tests/_attention_ref.py).

Tolerances, derived:
* norm and rotation: fp32 arithmetic, rounded to bf16 once: |err| <= 2^-8 |y| + 2^-18 (the sum of
  the magnitudes y is the sum of).  The second term covers the fp32 steps (a norm over at most 256
  values, its square root's two ulps, three products and a sum: under 40 roundings of 2^-24).
* cache bytes: equal.
* attention: with A = sum_j p_j |v_j| and S = the largest sum_d scale |q_d k_jd|, scores are fp32
  sums of at most 256 exact products: off by d = 2^-15 S at most (256 roundings of 2^-24, and a few
  more for the scales); a weight is then off by 2 d + 2^-20 relative (2 d: numerator and sum) and is
  rounded to bf16 once, 2^-8; the output is rounded to bf16 once:
  |err| <= 2^-8 |o| + (2^-8 + 2 d + 2^-20) A, and |lse err| <= d + 2^-20 + 2^-22 |lse|.
  What lies below the formats' range is lost: a weight under 2^-126 (the smallest normal fp32) may
  count as nothing, n 2^-126 max |v| in all, and the smallest bf16 is 2^-133.
"""

import numpy as np
import pytest
import torch

import _attention_ref as ref
import mxfp4_ref as oracle

pytestmark = pytest.mark.gpu
FORMATS = ["mxfp8", "mxfp4"]


@pytest.fixture(scope="module")
def mx():
    import mxfp4_b200

    return mxfp4_b200


@pytest.fixture(autouse=True)
def _no_device_error(mx):
    mx.device_error(clear=True)
    yield
    torch.cuda.synchronize()
    assert mx.device_error(clear=True) == 0


def f64(t):
    return t.detach().double().cpu().numpy()


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


def bf16(rng, shape, std=1.0):
    return torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).bfloat16().cuda()


def tables(rows, rot, first=0):
    a = (np.arange(rows) + first)[:, None] * 10000.0 ** (-np.arange(0, rot, 2) / rot)
    return torch.from_numpy(np.cos(a).astype(np.float32)).cuda(), torch.from_numpy(np.sin(a).astype(np.float32)).cuda()


def close_rows(got, want, mag):
    got = f64(got)
    bad = np.abs(got - want) > 2.0**-8 * np.abs(want) + 2.0**-18 * mag
    assert not bad.any(), (int(bad.sum()), np.abs(got - want)[bad][:4], want[bad][:4])


# ------------------------------------------------------------------------- norm and rotation
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,inter,weights,positions", [
    (1, 1, 1, 32, 32, False, None, False),
    (3, 3, 1, 64, 64, True, "bf16", True),
    (130, 5, 2, 96, 48, False, "f32", True),
    (7, 64, 8, 128, 128, False, "bf16", True),
    (33, 24, 24, 128, 128, True, "bf16", False),
    (2, 2, 2, 160, 16, True, None, True),
    (5, 7, 7, 256, 256, False, "f32", False),
    (4, 3, 2, 192, 0, False, "bf16", False),
    (1000, 2, 1, 64, 32, False, None, True),
    (2, 1, 1, 224, 112, False, "bf16", False),
])
def test_norm_rope(mx, tokens, heads, kv, dim, rot, inter, weights, positions):
    rng = np.random.default_rng(tokens * 7 + dim)
    width = (heads + 2 * kv) * dim
    pad = 24  # rows of a wider buffer
    wide = bf16(rng, (tokens, width + pad))
    wide[0] *= 100
    wide[-1] *= 0.001
    qkv = wide[:, :width]
    cos, sin = tables(max(tokens, 50), rot) if rot else (None, None)
    pos = rng.integers(0, max(tokens, 50), tokens) if positions and rot else None
    qw = kw = None
    if weights:
        dt = torch.bfloat16 if weights == "bf16" else torch.float32
        qw, kw = (torch.from_numpy((1 + rng.standard_normal(dim) / 4).astype(np.float32)).cuda().to(dt) for _ in range(2))
    q, k = mx.qk_norm_rope(qkv, heads, kv, cos, sin, positions=None if pos is None else i32(pos), q_weight=qw,
                           k_weight=kw, eps=1e-5, interleaved=inter)
    x = f64(qkv).reshape(tokens, heads + 2 * kv, dim)
    at = np.arange(tokens) if pos is None else pos
    c, s = (f64(cos)[at], f64(sin)[at]) if rot else (None, None)
    assert q.shape == (tokens, heads, dim) and k.shape == (tokens, kv, dim)
    close_rows(q, *ref.norm_rope(x[:, :heads], c, s, None if qw is None else f64(qw), 1e-5, inter))
    close_rows(k, *ref.norm_rope(x[:, heads:heads + kv], c, s, None if kw is None else f64(kw), 1e-5, inter))


def test_norm_rope_of_zeros_and_special_rows(mx):
    """A row of zeros norms to zeros; a NaN or an infinity stays in its own head."""
    cos, sin = tables(4, 64)
    x = torch.ones((4, 4, 64), dtype=torch.bfloat16, device="cuda")
    x[0] = 0
    x[1, 0, 5] = float("nan")
    x[2, 1, 0] = float("inf")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q, k = mx.qk_norm_rope(x.reshape(4, 256), 2, 1, cos, sin, q_weight=w, k_weight=w)
    assert (q[0] == 0).all() and (k[0] == 0).all()
    assert q[1, 0].isnan().all() and not q[1, 1].isnan().any() and not k.isnan().any()
    assert not q[2, 0].isnan().any() and q[2, 1].isnan().any() and not q[3].isnan().any()


def test_norm_rope_nothing_and_one_head_view(mx):
    cos, sin = tables(1, 64)
    q, k = mx.qk_norm_rope(torch.empty((0, 4 * 64), dtype=torch.bfloat16, device="cuda"), 2, 1, cos, sin)
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)


def test_bad_position_gives_zero_rows_and_the_error_word(mx):
    cos, sin = tables(8, 64)
    x = torch.ones((3, 4 * 64), dtype=torch.bfloat16, device="cuda")
    q, k = mx.qk_norm_rope(x, 2, 1, cos, sin, positions=i32([1, 8, -1]))
    assert mx.device_error() == 0x202
    assert (q[0] != 0).any() and (q[1:] == 0).all() and (k[1:] == 0).all()
    cache = mx.new_kv_cache(1, 1, 64, 16)
    cache.k_codes.fill_(77)
    mx.qk_norm_rope_cache(x, 2, 1, cos, sin, cache, i32([0, 1, 2]), positions=i32([1, 8, -1]))
    assert mx.device_error() == 0x202
    assert (cache.k_codes[0, 0, 1:] == 77).all() and (cache.k_codes[0, 0, 0] != 77).any()


# ------------------------------------------------------------------------------------- cache
def hard_rows(rng, tokens, heads, dim):
    """Rows with the groups that a coder can get wrong."""
    x = (rng.standard_normal((tokens, heads, dim)) * np.exp2(rng.integers(-40, 40, (tokens, heads, 1)))).astype(np.float32)
    g = x.reshape(-1, 32)
    n = len(g)
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0, 17.0, 19.0, 1.0625, 1.1875, 448.0, 464.0, 480.0, 496.0])
    for i, row in enumerate([
        np.zeros(32), -np.zeros(32), np.full(32, 2.0**-130), np.full(32, 3.0e38), np.r_[np.inf, np.ones(31)],
        np.r_[-np.inf, -np.zeros(31)], np.r_[np.nan, np.ones(31)], np.r_[np.ones(31), np.nan], np.r_[np.inf, np.nan, np.ones(30)],
        np.r_[ties, -ties], np.r_[ties, -ties] * 2.0**-100, np.r_[ties, -ties] * 2.0**100, np.r_[1.0, np.full(31, 2.0**-12)],
        np.r_[2.0**-118, np.full(31, 2.0**-126)], np.r_[1.9921875, np.full(31, -0.0)], np.r_[256.0, np.full(31, 2.0**-9 * 1.5)],
    ]):
        if i < n:
            g[(i * 5) % n] = row
    return torch.from_numpy(x).bfloat16().cuda()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens,kv,dim,page", [(40, 3, 64, 16), (9, 8, 128, 64), (21, 1, 256, 32), (1, 2, 128, 256)])
def test_write_is_byte_exact_and_reads_back(mx, fmt, tokens, kv, dim, page):
    rng = np.random.default_rng(dim + tokens)
    pages = -(-tokens // page) + 2
    cache = mx.new_kv_cache(pages, kv, dim, page, fmt)
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        t.fill_(0xA5)  # what is not written stays as it was
    k = hard_rows(rng, tokens, kv, dim)
    wide = torch.zeros((tokens, kv * dim + 8), dtype=torch.bfloat16, device="cuda")
    v = wide[:, :kv * dim].unflatten(1, (kv, dim))
    v.copy_(hard_rows(rng, tokens, kv, dim))
    slots = rng.permutation(pages * page)[:tokens]
    mx.kv_cache_write(cache, k, v, i32(slots))
    for codes, scales, x in ((cache.k_codes, cache.k_scales, k), (cache.v_codes, cache.v_scales, v)):
        c, s = ref.code_groups(f64(x), fmt)
        want_c, want_s = np.full(codes.shape, 0xA5, np.uint8), np.full(scales.shape, 0xA5, np.uint8)
        want_c[slots // page, :, slots % page], want_s[slots // page, :, slots % page] = c, s
        np.testing.assert_array_equal(scales.cpu().numpy(), want_s)
        np.testing.assert_array_equal(codes.cpu().numpy(), want_c)
    rk, rv = mx.kv_cache_read(cache, i32(slots))
    for got, codes, scales in ((rk, cache.k_codes, cache.k_scales), (rv, cache.v_codes, cache.v_scales)):
        at = (slots // page, slice(None), slots % page)
        want = ref.values(codes.cpu().numpy()[at], scales.cpu().numpy()[at], fmt)
        assert torch.equal(torch.from_numpy(want).float().bfloat16().nan_to_num(nan=-7.0), got.cpu().nan_to_num(nan=-7.0))


@pytest.mark.parametrize("dim", [64, 128])
def test_write_matches_the_librarys_other_coders(mx, dim):
    """The same bytes as quantize_mxfp4(rule="ocp") along the head, and as the oracle's MXFP8 coder."""
    rng = np.random.default_rng(3)
    k, v = bf16(rng, (50, 2, dim)), bf16(rng, (50, 2, dim), 1e-3)
    slots = i32(np.arange(50))
    c4, c8 = mx.new_kv_cache(4, 2, dim, 16, "mxfp4"), mx.new_kv_cache(4, 2, dim, 16, "mxfp8")
    for c in (c4, c8):
        mx.kv_cache_write(c, k, v, slots)

    def rows(t):
        return t.transpose(1, 2).flatten(0, 1)[:50].flatten(0, 1)

    p, s = mx.quantize_mxfp4(k.float().flatten(0, 1), axis=1, rule="ocp")
    assert torch.equal(rows(c4.k_codes), p) and torch.equal(rows(c4.k_scales), s)
    (codes, scales), = oracle.quantize_act_mx8(v.float().flatten(0, 1).cpu().numpy())
    np.testing.assert_array_equal(rows(c8.v_codes).cpu().numpy(), codes)
    np.testing.assert_array_equal(rows(c8.v_scales).cpu().numpy(), scales)


@pytest.mark.parametrize("fmt", FORMATS)
def test_read_of_every_code_and_scale(mx, fmt):
    cache = mx.new_kv_cache(16, 1, 256 if fmt == "mxfp8" else 128, 16, fmt)
    codes = torch.arange(256, dtype=torch.uint8, device="cuda") if fmt == "mxfp8" else torch.arange(64, dtype=torch.uint8, device="cuda") * 4 + 3
    cache.k_codes.copy_(codes.expand_as(cache.k_codes))
    cache.v_codes.copy_(codes.flip(0).expand_as(cache.v_codes))
    for t in (cache.k_scales, cache.v_scales):
        t.copy_(torch.arange(256, device="cuda").reshape(16, 1, 16, 1).expand_as(t))
    slots = i32(np.r_[np.arange(256), -1, -5])
    for got, c, s in zip(mx.kv_cache_read(cache, slots), (cache.k_codes, cache.v_codes), (cache.k_scales, cache.v_scales)):
        want = ref.values(c.cpu().numpy(), s.cpu().numpy(), fmt).reshape(256, 1, -1)
        want = torch.from_numpy(want).float().bfloat16().nan_to_num(nan=-7.0)
        assert torch.equal(got[:256].cpu().nan_to_num(nan=-7.0), want)
        assert (got[256:] == 0).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("heads,kv,dim,rot,inter,norm", [(8, 2, 64, 64, False, True), (5, 5, 128, 64, True, False),
                                                         (3, 1, 256, 256, False, True), (16, 2, 128, 0, False, True)])
def test_norm_rope_cache_is_byte_exact(mx, fmt, heads, kv, dim, rot, inter, norm):
    """The stored bytes are those of the 64-bit key, whatever rounding border it lies next to."""
    rng = np.random.default_rng(dim + heads)
    tokens, page = 300, 32
    qkv = bf16(rng, (tokens, (heads + 2 * kv) * dim))
    cos, sin = tables(1000, rot, 70000) if rot else (None, None)
    pos = rng.integers(0, 1000, tokens) if rot else None
    w = [torch.from_numpy((1 + rng.standard_normal(dim) / 4).astype(np.float32)).bfloat16().cuda() for _ in range(2)] if norm else [None] * 2
    cache = mx.new_kv_cache(tokens // page + 1, kv, dim, page, fmt)
    slots = rng.permutation(cache.num_pages * page)[:tokens]
    slots[-7:] = -1  # padding
    q = mx.qk_norm_rope_cache(qkv, heads, kv, cos, sin, cache, i32(slots), positions=None if pos is None else i32(pos),
                              q_weight=w[0], k_weight=w[1], interleaved=inter)
    x = f64(qkv).reshape(tokens, -1, dim)
    c, s = (f64(cos)[pos], f64(sin)[pos]) if rot else (None, None)
    close_rows(q, *ref.norm_rope(x[:, :heads], c, s, f64(w[0]) if norm else None, 1e-6, inter))
    key, _ = ref.norm_rope(x[:, heads:heads + kv], c, s, f64(w[1]) if norm else None, 1e-6, inter)
    live = slots[:-7]
    for codes, scales, rows in ((cache.k_codes, cache.k_scales, key), (cache.v_codes, cache.v_scales, x[:, heads + kv:])):
        want_c, want_s = np.zeros(codes.shape, np.uint8), np.zeros(scales.shape, np.uint8)
        a, b = ref.code_groups(rows[:-7], fmt)
        want_c[live // page, :, live % page], want_s[live // page, :, live % page] = a, b
        np.testing.assert_array_equal(scales.cpu().numpy(), want_s)
        np.testing.assert_array_equal(codes.cpu().numpy(), want_c)


def range_rows(rng, heads, dim):
    """One token per power of two, squares of whose values fp32 can and cannot hold; heads of one and of
    mixed size, and zeros among the values."""
    powers = np.r_[np.arange(-120, 121, 8), -31, -30, -29, 29, 30, 31, 33, 34, 35]
    x = rng.standard_normal((len(powers), heads, dim))
    x = np.where(np.abs(x) < 2.0**-6, 2.0**-6, x) * np.exp2(powers.astype(float))[:, None, None]
    x[:, 1] = rng.standard_normal((len(powers), dim))
    x[:, 2, ::5] = 0
    x[0] = 0
    return torch.from_numpy(x.astype(np.float32)).bfloat16().cuda()


@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6])
@pytest.mark.parametrize("weight", [1.0, 2.0**100, 2.0**-100])
@pytest.mark.parametrize("inter", [False, True])
def test_norm_rope_over_the_whole_range(mx, eps, weight, inter):
    rng = np.random.default_rng(5)
    x = range_rows(rng, 5, 64)
    if eps == 0:
        x = x[1:]  # zeros have no norm then
    cos, sin = tables(len(x), 32)
    w = ((1 + torch.rand(64, device="cuda")) * weight).bfloat16()
    q, k = mx.qk_norm_rope(x.flatten(1), 3, 1, cos, sin, q_weight=w, k_weight=w, eps=eps, interleaved=inter)
    for got, rows in ((q, x[:, :3]), (k, x[:, 3:4])):
        want, mag = ref.norm_rope(f64(rows), f64(cos), f64(sin), f64(w), eps, inter)
        keep = (np.abs(want) > 2.0**-120) | (mag == 0)  # values that bf16 can hold to its 8 bits
        close_rows(got[torch.from_numpy(keep).cuda()], want[keep], mag[keep])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("eps,weight", [(1e-6, 1.0), (1e-30, 1.0), (1e-6, 2.0**-100), (1e-30, 2.0**100), (None, 1.0)])
@pytest.mark.parametrize("inter", [False, True])
def test_norm_rope_cache_is_byte_exact_over_the_whole_range(mx, fmt, eps, weight, inter):
    rng = np.random.default_rng(6)
    x = range_rows(rng, 7, 64)  # 1 query head, 3 of each
    n = len(x)
    x[:, 1:4] = x[:, :3].clone()
    cos, sin = tables(n, 32)
    w = None if eps is None else ((1 + torch.rand(64, device="cuda")) * weight).bfloat16()
    cache = mx.new_kv_cache(-(-n // 16), 3, 64, 16, fmt)
    mx.qk_norm_rope_cache(x.flatten(1), 1, 3, cos, sin, cache, i32(np.arange(n)), q_weight=w, k_weight=w,
                          eps=eps or 0.0, interleaved=inter)
    want, _ = ref.norm_rope(f64(x[:, 1:4]), f64(cos), f64(sin), None if w is None else f64(w), eps or 0.0, inter)
    codes, scales = ref.code_groups(want, fmt)
    got, got_s = (t.cpu().numpy().transpose(0, 2, 1, 3).reshape(-1, 3, t.shape[-1])[:n] for t in (cache.k_codes, cache.k_scales))
    wrong = np.unique(np.nonzero((got_s != scales).any(-1) | (got != codes).any(-1))[0])
    assert not len(wrong), wrong


@pytest.mark.parametrize("tokens", [2, 200, 4097, 9000])
def test_same_slot_twice_keeps_the_later_token(mx, tokens):
    """Within one launch and across the launches a long call is cut into."""
    rng = np.random.default_rng(tokens)
    cache = mx.new_kv_cache(4, 2, 64, 16)
    k, v = bf16(rng, (tokens, 2, 64)), bf16(rng, (tokens, 2, 64))
    slots = rng.integers(0, 64, tokens)
    slots[0] = slots[-1]
    for shift in (0, 1, 2):  # vectors of slots that start at any address
        pad = i32(np.r_[np.full(shift, 7), slots])
        mx.kv_cache_write(cache, k, v, pad[shift:])
        last = {int(s): t for t, s in enumerate(slots)}
        at = np.array(sorted(last))
        rk, rv = mx.kv_cache_read(cache, i32(at))
        for got, x in ((rk, k), (rv, v)):
            c, s = ref.code_groups(f64(x[[last[a] for a in at]]), "mxfp8")
            np.testing.assert_array_equal(f64(got), ref.values(c, s, "mxfp8"))


def test_bad_slots_are_left_out(mx):
    cache = mx.new_kv_cache(2, 1, 64, 16)
    k = torch.ones((4, 1, 64), dtype=torch.bfloat16, device="cuda")
    mx.kv_cache_write(cache, k, k, i32([3, 32, -1, 2**31 - 1]))
    assert mx.device_error() == 0x201
    assert (cache.k_scales != 0).nonzero()[:, 2].unique().tolist() == [3]
    rk, _ = mx.kv_cache_read(cache, i32([3, 32, -1, 2**31 - 1]))
    assert mx.device_error() == 0x201
    assert (rk[0] == 1).all() and (rk[1:] == 0).all()


# --------------------------------------------------------------------------------- attention
def random_cache(mx, rng, pages, kv, dim, page, fmt, spread=2):
    """A cache whose every byte is in use: random codes (no NaN codes), scales around one."""
    cache = mx.new_kv_cache(pages, kv, dim, page, fmt)
    for t in (cache.k_codes, cache.v_codes):
        c = rng.integers(0, 256, t.shape, dtype=np.uint8)
        if fmt == "mxfp8":
            c[(c & 127) == 127] = 3
        t.copy_(torch.from_numpy(c))
    low = 119 if fmt == "mxfp8" else 125
    for t in (cache.k_scales, cache.v_scales):
        t.copy_(torch.from_numpy(rng.integers(low - spread, low + spread, t.shape, dtype=np.uint8)))
    return cache


def random_table(rng, cache, lengths, extra=2):
    need = [-(-n // cache.page_size) for n in lengths]
    ids = rng.permutation(cache.num_pages)[:sum(need)]
    table = np.full((len(lengths), max(need) + extra), -1, np.int64)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table


def check_attention(got, lse, q, cache, table, lengths, scale):
    kc, vc, ks, vs = (t.cpu().numpy() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales))
    got, qq = f64(got), f64(q)
    for b, n in enumerate(lengths):
        ids = table[b, : -(-n // cache.page_size)]
        k, v = (ref.values(c[ids].swapaxes(1, 2).reshape(-1, *c.shape[1:2], c.shape[3])[:n],
                           s[ids].swapaxes(1, 2).reshape(-1, *s.shape[1:2], s.shape[3])[:n], cache.format)
                for c, s in ((kc, ks), (vc, vs)))
        o, l, mag, size = ref.attention(qq[b], k, v, scale)
        d = 2.0**-15 * size
        lost = 2.0**-133 + n * 2.0**-126 * (np.abs(v).max() if n else 0.0)
        bad = ~(np.abs(got[b] - o) <= 2.0**-8 * np.abs(o) + (2.0**-8 + 2 * d[:, None] + 2.0**-20) * mag + lost)
        assert not bad.any(), (b, n, int(bad.sum()), got[b][bad][:4], o[bad][:4])
        if lse is not None:
            e = f64(lse)[b]
            if n == 0:
                assert (e == -np.inf).all()
            else:
                assert (np.abs(e - l) <= d + 2.0**-20 + 2.0**-22 * np.abs(l)).all(), (b, n, e, l)


EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 513, 1025]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads,kv,page", [
    (64, 8, 8, 16), (64, 28, 4, 64), (64, 33, 3, 32), (128, 8, 1, 64), (128, 6, 2, 16), (128, 36, 3, 128),
    (128, 71, 1, 32), (256, 16, 2, 64), (256, 9, 1, 16), (128, 2, 2, 256),
])
def test_attention_over_edge_lengths(mx, fmt, dim, heads, kv, page):
    rng = np.random.default_rng(dim + heads + page)
    lengths = EDGES
    pages = sum(-(-n // page) for n in lengths) + 3
    cache = random_cache(mx, rng, pages, kv, dim, page, fmt)
    table = random_table(rng, cache, lengths)
    q = bf16(rng, (len(lengths), heads, dim))
    out, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), return_lse=True)
    check_attention(out, lse, q, cache, table, lengths, dim ** -0.5)
    again, lse2 = mx.paged_attention(q, cache, i32(table), i32(lengths), return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    # one sequence at a time: other shares of the blocks, the same answer within the bound
    for b in (1, 9, len(lengths) - 1):
        o, l = mx.paged_attention(q[b:b + 1], cache, i32(table[b:b + 1]), i32(lengths[b:b + 1]), return_lse=True)
        check_attention(o, l, q[b:b + 1], cache, table[b:b + 1], lengths[b:b + 1], dim ** -0.5)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads,kv,seqs", [(64, 4, 2, 21), (64, 24, 2, 40), (128, 3, 3, 21), (128, 12, 1, 150), (256, 10, 1, 21), (256, 2, 2, 400)])
def test_attention_with_a_wide_page_table(mx, fmt, dim, heads, kv, seqs):
    """A table that could hold far longer sequences: the pieces come from the lengths on the device, with few
    heads and with more than there are blocks; entries past a sequence's pages are never read."""
    rng = np.random.default_rng(dim + seqs)
    lengths = (EDGES * 20)[:seqs]
    lengths[seqs // 2] = 5000
    page = 32
    cache = random_cache(mx, rng, sum(-(-n // page) for n in lengths) + 1, kv, dim, page, fmt)
    table = random_table(rng, cache, lengths)
    wide = np.full((seqs, 9000), 2**30)  # 288000 keys
    wide[:, :table.shape[1]] = table
    q = bf16(rng, (seqs, heads, dim))
    out, lse = mx.paged_attention(q, cache, i32(wide), i32(lengths), return_lse=True)
    check_attention(out, lse, q, cache, table, lengths, dim ** -0.5)
    again, lse2 = mx.paged_attention(q, cache, i32(wide), i32(lengths), return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    none, lse = mx.paged_attention(q, cache, i32(wide), i32([0] * seqs), return_lse=True)
    assert (none == 0).all() and (lse == -float("inf")).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("seqs,longest,dim,heads,kv", [(1, 40000, 128, 16, 2), (3, 9000, 64, 8, 1), (300, 200, 128, 4, 4),
                                                       (2, 6000, 256, 4, 1), (40, 3000, 128, 24, 2)])
def test_attention_split_and_joined(mx, fmt, seqs, longest, dim, heads, kv):
    rng = np.random.default_rng(longest + seqs)
    page = 64
    lengths = [longest] + [int(n) for n in rng.integers(0, longest + 1, seqs - 1)]
    cache = random_cache(mx, rng, sum(-(-n // page) for n in lengths) + 1, kv, dim, page, fmt)
    table = random_table(rng, cache, lengths)
    wide = bf16(rng, (seqs, heads * dim + 16))
    q = wide[:, :heads * dim].unflatten(1, (heads, dim))  # rows of a wider buffer
    many = np.full((seqs, table.shape[1] + 5), -1)
    many[:, :table.shape[1]] = table
    out = torch.full((seqs, heads, dim), float("nan"), dtype=torch.bfloat16, device="cuda")
    got, lse = mx.paged_attention(q, cache, i32(many)[:, :table.shape[1]], i32(lengths), scale=0.07, return_lse=True, out=out)
    assert got is out
    check_attention(out, lse, q, cache, table, lengths, 0.07)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads", [(64, 4), (128, 16), (256, 4)])
def test_rows_behind_a_sequence_may_hold_anything(mx, fmt, dim, heads):
    """NaN scales, NaN codes and huge values behind the last key change nothing, and pages that no
    sequence names neither."""
    rng = np.random.default_rng(5)
    lengths, page = [1, 70, 33, 130], 64
    cache = random_cache(mx, rng, 9, 1, dim, page, fmt)
    table = random_table(rng, cache, lengths)
    q = bf16(rng, (4, heads, dim))
    want, wl = mx.paged_attention(q, cache, i32(table), i32(lengths), return_lse=True)
    used = np.zeros((9, page), bool)
    for b, n in enumerate(lengths):
        for j in range(n):
            used[table[b, j // page], j % page] = True
    mask = torch.from_numpy(~used).cuda()[:, None, :, None]
    for fill_codes, fill_scales in ((0xFF, 0xFF), (0x7F, 0xFE), (0x7E, 0x00)):
        for t, f in ((cache.k_codes, fill_codes), (cache.v_codes, fill_codes), (cache.k_scales, fill_scales), (cache.v_scales, fill_scales)):
            t.masked_fill_(mask, f)
        got, gl = mx.paged_attention(q, cache, i32(table), i32(lengths), return_lse=True)
        assert torch.equal(got, want) and torch.equal(gl, wl)


@pytest.mark.parametrize("fmt", FORMATS)
def test_nan_keys_and_values_reach_their_outputs_alone(mx, fmt):
    rng = np.random.default_rng(8)
    lengths = [100, 100, 100]
    cache = random_cache(mx, rng, 8, 2, 128, 64, fmt)
    table = random_table(rng, cache, lengths)
    q = bf16(rng, (3, 4, 128))
    want = mx.paged_attention(q, cache, i32(table), i32(lengths))
    cache.k_scales[table[0, 1], 1, 7, 2] = 255  # sequence 0, kv head 1: every output of heads 2 and 3
    cache.v_scales[table[1, 0], 0, 9, 1] = 255  # sequence 1, kv head 0: values 32..63 of heads 0 and 1
    got = mx.paged_attention(q, cache, i32(table), i32(lengths))
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[0, 2:] = True
    nan[1, :2, 32:64] = True
    assert torch.equal(got.isnan(), nan) and torch.equal(got[~nan], want[~nan])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_of_values_of_very_different_size(mx, fmt, dim):
    """One key takes all the weight and has tiny values beside huge ones of weightless keys; a key of
    zeros (scale byte 0) takes it all; groups of one row differ by 2^40; whole heads are tiny or huge."""
    rng = np.random.default_rng(dim)
    n, page = 200, 16
    cache = random_cache(mx, rng, 5 * 13, 1, dim, page, fmt)
    lengths = [n] * 5
    table = random_table(rng, cache, lengths)
    q = bf16(rng, (5, 3, dim))
    low = 119 if fmt == "mxfp8" else 125
    pages = [torch.from_numpy(t[:13]).cuda() for t in table]
    # 0: scores far apart (large k scales), value scales spread over 2^-40 .. 2^40
    cache.k_scales[pages[0]] = torch.from_numpy(rng.integers(low, low + 6, (13, 1, page, dim // 32), dtype=np.uint8)).cuda()
    for i in (0, 1):
        cache.v_scales[pages[i]] = torch.from_numpy(rng.integers(low - 40, low + 40, (13, 1, page, dim // 32), dtype=np.uint8)).cuda()
    # 2: the winning key has only zeros as values
    cache.k_codes[table[2, 3], 0, 5] = 0
    cache.k_codes[table[2, 3], 0, 5, 0] = 0x78 if fmt == "mxfp8" else 0x07
    cache.k_scales[table[2, 3], 0, 5, 0] = low + 8
    q[2, :, 0] = 8
    cache.v_codes[table[2, 3], 0, 5] = 0
    cache.v_scales[table[2, 3], 0, 5] = 0
    # 3 and 4: all values tiny / large
    cache.v_scales[pages[3]] = low - 60
    cache.v_scales[pages[4]] = low + 50
    out, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), return_lse=True)
    check_attention(out, lse, q, cache, table, lengths, dim ** -0.5)


def test_attention_of_large_and_tiny_queries(mx):
    """q keeps all its bits through the f16 operand at any magnitude bf16 has."""
    rng = np.random.default_rng(4)
    lengths = [90] * 5
    cache = random_cache(mx, rng, 12, 1, 128, 64, "mxfp8")
    table = random_table(rng, cache, lengths)
    q = bf16(rng, (5, 2, 128))
    q[1] *= 2.0**100
    q[2] *= 2.0**-60
    q[3, :, 1:] *= 2.0**-14
    q[4] = 0
    # the scale brings the scores back to where exp() is at home
    for rows, scale in (([0, 2, 3, 4], 0.1), ([1], 0.1 * 2.0**-100)):
        out, lse = mx.paged_attention(q[rows], cache, i32(table[rows]), i32([90] * len(rows)), scale=scale, return_lse=True)
        check_attention(out, lse, q[rows], cache, table[rows], [90] * len(rows), scale)


@pytest.mark.parametrize("seqs,longest,heads", [(5, 900, 16), (2, 30000, 16), (70, 3000, 48)])
def test_attention_into_its_own_query(mx, seqs, longest, heads):
    """out may be q itself: one block, clusters and joined pieces."""
    rng = np.random.default_rng(seqs)
    lengths = rng.integers(0, longest, seqs)
    cache = random_cache(mx, rng, 64, 2, 128, 64, "mxfp8")
    table = i32(rng.integers(0, 64, (seqs, -(-longest // 64))))
    q = bf16(rng, (seqs, heads, 128))
    want = mx.paged_attention(q, cache, table, i32(lengths))
    assert mx.paged_attention(q, cache, table, i32(lengths), out=q) is not None
    assert torch.equal(q, want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dim,heads,kv,longest", [(64, 40, 2, 40), (128, 64, 8, 700), (256, 16, 4, 30), (128, 8, 8, 12000)])
def test_weights_of_nearly_equal_scores(mx, fmt, dim, heads, kv, longest):
    """Scores near zero: nothing but the exponential's and the sums' own errors is left of the bounds."""
    rng = np.random.default_rng(longest)
    lengths = [longest, 10, 3, longest // 2]
    cache = random_cache(mx, rng, 250, kv, dim, 64, fmt)
    table = rng.integers(0, 250, (4, -(-longest // 64)))
    q = bf16(rng, (4, heads, dim), 0.01)
    got, lse = mx.paged_attention(q, cache, i32(table), i32(lengths), scale=0.01, return_lse=True)
    check_attention(got, lse, q, cache, table, lengths, 0.01)


def test_bad_pages_and_lengths(mx):
    """A page outside the cache loses its keys, a length past the table's row is cut; both set the error word."""
    rng = np.random.default_rng(6)
    cache = random_cache(mx, rng, 6, 2, 128, 16, "mxfp8")
    q = bf16(rng, (2, 4, 128))
    good = np.array([[0, 1, 2], [3, 4, 5]])
    out = mx.paged_attention(q, cache, i32([[0, 9, 2], [-1, -3, 2**31 - 1]]), i32([48, 40]))
    assert mx.device_error() == 0x203
    want = mx.paged_attention(q[:1], cache, i32([[0, 2]]), i32([32]))
    np.testing.assert_allclose(f64(out[0]), f64(want[0]), atol=2.0**-7 * f64(want).max())
    assert (out[1] == 0).all()
    out = mx.paged_attention(q, cache, i32(good), i32([1000, -4]))
    assert mx.device_error() == 0x204
    check_attention(out, None, q, cache, good, [48, 0], 128 ** -0.5)


def test_shared_pages_and_nothing(mx):
    rng = np.random.default_rng(7)
    cache = random_cache(mx, rng, 4, 1, 64, 64, "mxfp4")
    q = bf16(rng, (3, 2, 64))
    table = np.array([[2, 1], [2, 3], [2, 2]])  # a shared prefix, and a page twice
    out, lse = mx.paged_attention(q, cache, i32(table), i32([100, 128, 128]), return_lse=True)
    check_attention(out, lse, q, cache, table, [100, 128, 128], 0.125)
    none = mx.paged_attention(q[:0], cache, i32(table)[:0], i32([]))
    assert none.shape == (0, 2, 64)
    zero, lse = mx.paged_attention(q, cache, i32(table), i32([0, 0, 0]), return_lse=True)
    assert (zero == 0).all() and (lse == -float("inf")).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_offsets_past_32_bits(mx, fmt):
    """A cache of more than 2^32 bytes of codes per array: its last pages are written, read and attended."""
    rng = np.random.default_rng(9)
    kv, dim, page = 8, 256, 256
    row = kv * page * (dim if fmt == "mxfp8" else dim // 2)
    pages = 2**32 // row + 4
    cache = mx.new_kv_cache(pages, kv, dim, page, fmt)
    n = 2 * page
    k, v = bf16(rng, (n, kv, dim)), bf16(rng, (n, kv, dim))
    slots = i32((pages - 2) * page + np.arange(n))
    mx.kv_cache_write(cache, k, v, slots)
    rk, rv = mx.kv_cache_read(cache, slots)
    small = mx.new_kv_cache(2, kv, dim, page, fmt)
    mx.kv_cache_write(small, k, v, i32(np.arange(n)))
    sk, sv = mx.kv_cache_read(small, i32(np.arange(n)))
    assert torch.equal(rk, sk) and torch.equal(rv, sv) and (rk != 0).any()
    q = bf16(rng, (1, kv, dim))
    assert torch.equal(mx.paged_attention(q, cache, i32([[pages - 2, pages - 1]]), i32([n - 3])),
                       mx.paged_attention(q, small, i32([[0, 1]]), i32([n - 3])))


# ------------------------------------------------------------- streams, graphs, runs together
def test_graphs_replay_with_new_contents_and_streams(mx):
    """Two captured graphs of the operators, replayed in turn and beside an eager call on another stream,
    after their inputs (lengths, pages, slots) have changed in place."""
    rng = np.random.default_rng(10)
    page, kv, dim, heads = 16, 2, 128, 8
    cache = random_cache(mx, rng, 64, kv, dim, page, "mxfp8")
    graphs, state = [], []
    for i in range(2):
        q, table, lengths = bf16(rng, (3, heads, dim)), torch.zeros((3, 20), dtype=torch.int32, device="cuda"), i32([1, 1, 1])
        mx.paged_attention(q, cache, table, lengths)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, lse = mx.paged_attention(q, cache, table, lengths, return_lse=True)
        graphs.append(g)
        state.append((q, table, lengths, out, lse))
    side = torch.cuda.Stream()
    for turn in range(3):
        plans = []
        for q, table, lengths, _, _ in state:
            n = [int(x) for x in rng.integers(0, 320, 3)]
            t = random_table(rng, cache, n, 0)
            full = np.zeros((3, 20), np.int64)
            full[:, :t.shape[1]] = t
            table.copy_(i32(full)), lengths.copy_(i32(n)), q.copy_(bf16(rng, (3, heads, dim)))
            plans.append((full, n))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            q0, t0, l0 = state[0][:3]
            eager, elses = mx.paged_attention(q0, cache, t0, l0, return_lse=True)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (q, _, _, out, lse), (t, n) in zip(state, plans):
            check_attention(out, lse, q, cache, t, n, dim ** -0.5)
        assert torch.equal(eager, state[0][3]) and torch.equal(elses, state[0][4])


def test_each_call_sees_what_ran_before_it(mx):
    """The row kernels may be launched while the kernel before them still runs: a copy, a memset, another
    stream's event and each other's writes come first all the same, eager and in a graph."""
    tokens, kv, dim = 3000, 8, 128
    rng = np.random.default_rng(3)
    k, v = bf16(rng, (tokens, kv, dim)), bf16(rng, (tokens, kv, dim))
    cache = mx.new_kv_cache(-(-tokens // 64), kv, dim, 64)
    slots, held, staged = i32(rng.permutation(cache.num_pages * 64)[:tokens]), torch.zeros_like(k), torch.zeros_like(v)
    zeros, other = torch.zeros_like(slots) - 1, torch.cuda.Stream()

    def steps():
        out = []
        for i in range(4):
            here = torch.cuda.current_stream()
            held.copy_(k * (i + 1))  # a kernel and a copy
            other.wait_stream(here)
            with torch.cuda.stream(other):
                staged.copy_(v * (i + 1))
            here.wait_stream(other)
            mx.kv_cache_write(cache, held, staged, slots)
            held.zero_()
            mx.kv_cache_write(cache, held, held, zeros)  # writes nothing
            out.append(mx.kv_cache_read(cache, slots))
            cache.k_codes.zero_()  # a memset
            out.append(mx.kv_cache_read(cache, slots))
            mx.kv_cache_write(cache, held, staged, slots)
            out.append(mx.kv_cache_read(cache, slots))
        return out

    def check(out):
        for i in range(4):
            mx.kv_cache_write(cache, k * (i + 1), v * (i + 1), slots)
            rk, rv = mx.kv_cache_read(cache, slots)
            (ak, av), (bk, bv), (ck, cv) = out[3 * i:3 * i + 3]
            assert torch.equal(ak, rk) and all(torch.equal(x, rv) for x in (av, bv, cv))
            assert (bk == 0).all() and (ck == 0).all()

    check(steps())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = steps()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check(out)


@pytest.mark.parametrize("seqs,longest,heads,kv", [(1, 700, 16, 2), (16, 4000, 16, 8), (3, 40000, 16, 2), (300, 500, 4, 4), (70, 3000, 20, 2)])
def test_attention_sees_what_ran_before_it(mx, seqs, longest, heads, kv):
    """However it is launched (one block or a cluster to a head, pieces and their joining), the query, lengths
    and pages of a call are those written just before it, eager and in a graph."""
    rng = np.random.default_rng(seqs)
    cache = random_cache(mx, rng, 80, kv, 128, 64, "mxfp8")
    width = -(-longest // 64)
    calls = [(bf16(rng, (seqs, heads, 128)), i32(rng.integers(0, longest, seqs)), i32(rng.integers(0, 80, (seqs, width)))) for _ in range(3)]
    want = [mx.paged_attention(q, cache, table, lengths, return_lse=True) for q, lengths, table in calls]
    q, lengths, table = (torch.zeros_like(t) for t in calls[0])

    def steps():
        out = []
        for i in range(6):
            for to, of in zip((q, lengths, table), calls[i % 3]):
                to.copy_(of)
            out.append(mx.paged_attention(q, cache, table, lengths, return_lse=True))
            out.append(mx.paged_attention(q, cache, table, lengths, return_lse=True))
            for t in (q, lengths, table):
                t.zero_()
        return out

    def check(out):
        for i, (o, lse) in enumerate(out):
            assert torch.equal(o, want[i // 2 % 3][0]) and torch.equal(lse, want[i // 2 % 3][1]), i

    check(steps())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = steps()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check(out)


@pytest.mark.parametrize("fmt", FORMATS)
def test_decoding_through_the_gemms(mx, fmt):
    """A layer's attention as it is used: a prompt, then single tokens, each through the QKV GEMM, the norm
    and rotation into the cache, the attention and the output GEMM; the step is one captured graph.  Compared
    with 64-bit attention over the values the cache stands for."""
    rng = np.random.default_rng(11)
    heads, kv, dim, hidden, page, seqs, steps = 8, 2, 64, 256, 16, 3, 5
    prompt = [20, 1, 33]

    def weight(n, k):
        p, s = mx.quantize_mxfp4(torch.from_numpy((rng.standard_normal((k, n)) * 0.06).astype(np.float32)).cuda(), axis=0, rule="ocp")
        return mx.prepack_b200(p, s)

    w_qkv, w_out = weight((heads + 2 * kv) * dim, hidden), weight(hidden, heads * dim)
    qw, kw = (torch.from_numpy((1 + rng.standard_normal(dim) / 8).astype(np.float32)).bfloat16().cuda() for _ in range(2))
    cos, sin = tables(64, dim)
    cache = mx.new_kv_cache(12, kv, dim, page, fmt)
    table = rng.permutation(12).reshape(3, 4)
    how = {"q_weight": qw, "k_weight": kw}
    # prompts, as one ragged batch padded to a round number of rows
    rows = [(b, j) for b, n in enumerate(prompt) for j in range(n)]
    x = bf16(rng, (64, hidden))
    slots = np.full(64, -1)
    slots[:len(rows)] = [table[b, j // page] * page + j % page for b, j in rows]
    pos = np.zeros(64, np.int64)
    pos[:len(rows)] = [j for _, j in rows]
    mx.qk_norm_rope_cache(mx.gemm(x, w_qkv), heads, kv, cos, sin, cache, i32(slots), positions=i32(pos), **how)

    x1, s1, p1, n1, t1 = bf16(rng, (seqs, hidden)), i32([-1] * 3), i32([0] * 3), i32([0] * 3), i32(table)

    def step():
        qkv = mx.gemm(x1, w_qkv)
        q = mx.qk_norm_rope_cache(qkv, heads, kv, cos, sin, cache, s1, positions=p1, **how)
        a = mx.paged_attention(q, cache, t1, n1)
        return qkv, q, a, mx.gemm(a.view(seqs, heads * dim), w_out)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        qkv, q, a, y = step()
    for i in range(steps):
        n = [p + i + 1 for p in prompt]
        x1.copy_(bf16(rng, (seqs, hidden)))
        p1.copy_(i32([m - 1 for m in n])), n1.copy_(i32(n))
        s1.copy_(i32([table[b, (m - 1) // page] * page + (m - 1) % page for b, m in enumerate(n)]))
        g.replay()
        torch.cuda.synchronize()
        qk = f64(qkv).reshape(seqs, -1, dim)
        c, s = f64(cos)[[m - 1 for m in n]], f64(sin)[[m - 1 for m in n]]
        close_rows(q, *ref.norm_rope(qk[:, :heads], c, s, f64(qw), 1e-6, False))
        key, _ = ref.norm_rope(qk[:, heads:heads + kv], c, s, f64(kw), 1e-6, False)
        codes, scales = ref.code_groups(key, fmt)
        at = s1.cpu().numpy()
        np.testing.assert_array_equal(cache.k_codes.cpu().numpy()[at // page, :, at % page], codes)
        np.testing.assert_array_equal(cache.k_scales.cpu().numpy()[at // page, :, at % page], scales)
        check_attention(a, None, q, cache, table, n, dim ** -0.5)
        assert torch.equal(y, mx.gemm(a.view(seqs, heads * dim), w_out))
