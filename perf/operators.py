"""Cases of the operators between the QKV GEMM and the output GEMM of an attention layer.

Four kinds of case:

* ``rope``: ``qk_norm_rope``, the norm of every query and key head and its rotation in one pass
  over the QKV GEMM's output;
* ``store``: the same pass with the keys and values quantised into the pages of a key-value
  cache (``qk_norm_rope_cache``, or ``kv_cache_write`` for rows that are rotated already), and the
  rows just written read back (``kv_cache_read``), so that the outputs are the values the codes
  stand for;
* ``read``: ``kv_cache_read`` alone, rows gathered out of scattered pages;
* ``attend``: ``paged_attention``, one new token per sequence over such a cache.

The cache holds, per page and key-value head, ``page`` rows of ``dim`` codes (E4M3, or two E2M1
to a byte, the even element in the low nibble) and one E8M0 scale byte per 32 elements.

``own`` false computes each operator in elementary torch operations; ``own`` true calls the
package.
"""

import math
import os
import sys

import torch

own = False

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_EPS = 1e-6


def _mx():
    """The package, which lives one folder below the repository's root."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cdna3-bench_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mxfp4_b200

    return mxfp4_b200


# ------------------------------------------------------------------------------------ cases
def _rope(name, rows, heads, kv_heads, dim, rot, norm, inter, table, scattered):
    return {"name": name, "kind": "rope", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "norm": norm, "inter": inter, "table": table, "scattered": scattered}


def _store(name, rows, heads, kv_heads, dim, rot, norm, inter, fmt, page, table, padded, rotate=True):
    return {"name": name, "kind": "store", "rows": rows, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "norm": norm, "inter": inter, "fmt": fmt, "page": page, "table": table, "padded": padded, "rotate": rotate}


def _read(name, rows, kv_heads, dim, fmt, page):
    return {"name": name, "kind": "read", "rows": rows, "kv_heads": kv_heads, "dim": dim, "fmt": fmt, "page": page}


def _attend(name, seqs, longest, shortest, empty, heads, kv_heads, dim, fmt, page):
    return {"name": name, "kind": "attend", "seqs": seqs, "longest": longest, "shortest": shortest, "empty": empty,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "fmt": fmt, "page": page}


def listed():
    return [
        # the image tokens of one FLUX.1 block: 24 heads of 128 each for q, k and v, one table row per token
        _rope("rope_image_block", 4608, 24, 24, 128, 128, True, True, 4608, False),
        # one decoding step of 16 sequences at the 10240-wide QKV of the Llama-70B-sized layer, far positions
        _rope("rope_step_16", 16, 64, 8, 128, 128, False, False, 131072, True),
        # an odd number of prompt rows, small heads, half of each head rotated
        _rope("rope_partial_1531", 1531, 14, 2, 64, 32, True, False, 4096, True),
        # one decoding step of 32 sequences into the cache
        _store("store_step_32", 32, 64, 8, 128, 128, True, False, "mxfp8", 64, 131072, 0),
        # a prompt of 4096 tokens into the smaller cache
        _store("store_prompt_4096", 4096, 64, 8, 128, 128, True, False, "mxfp4", 64, 8192, 0),
        # rows rotated elsewhere, wide heads, a padded batch
        _store("store_rows_777", 777, 8, 4, 256, 0, False, False, "mxfp8", 16, 0, 40, rotate=False),
        # a long prefix handed back for a prompt's chunk
        _read("read_prefix_20000", 20000, 8, 128, "mxfp8", 64),
        # a few hundred rows of small heads
        _read("read_rows_300", 300, 4, 64, "mxfp4", 16),
        # the smallest answer: one sequence of a few hundred tokens
        _attend("attend_one_700", 1, 700, 700, 0, 64, 8, 128, "mxfp8", 64),
        # ordinary serving: ragged lengths, one slot of the batch free
        _attend("attend_ragged_16", 16, 8192, 100, 1, 64, 8, 128, "mxfp8", 64),
        # many shorter sequences over the smaller cache
        _attend("attend_many_64", 64, 4096, 33, 0, 32, 8, 128, "mxfp4", 32),
        # two very long documents
        _attend("attend_long_2", 2, 131072, 98765, 0, 64, 8, 128, "mxfp8", 64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "store", "read", "attend", "attend"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 12, 16])
    fmt = rng.choice(["mxfp8", "mxfp4"])
    page = rng.choice([16, 32, 64, 128])
    norm, inter = rng.random() < 0.5, rng.random() < 0.5
    rot = rng.choice([dim, dim, dim // 2])
    if kind == "rope":
        rows = _log_int(rng, 1, min(12000, 60_000_000 // ((heads + 2 * kv_heads) * dim)))
        table = _log_int(rng, rows, 131072)
        return {k: v for k, v in _rope("", rows, heads, kv_heads, dim, rot, norm, inter, table, rng.random() < 0.7).items() if k != "name"}
    if kind == "store":
        rows = _log_int(rng, 1, min(12000, 60_000_000 // ((heads + 2 * kv_heads) * dim)))
        rotate = rng.random() < 0.75
        c = _store("", rows, heads, kv_heads, dim, rot if rotate else 0, norm and rotate, inter and rotate, fmt, page,
                   _log_int(rng, rows, 131072) if rotate else 0, rng.randrange(0, rows // 8 + 1), rotate)
        return {k: v for k, v in c.items() if k != "name"}
    if kind == "read":
        rows = _log_int(rng, 1, 40_000_000 // (kv_heads * dim))
        return {k: v for k, v in _read("", rows, kv_heads, dim, fmt, page).items() if k != "name"}
    seqs = _log_int(rng, 1, 100)
    longest = _log_int(rng, 1, min(131072, 120_000_000 // (seqs * kv_heads * dim)))
    shortest = rng.randint(1, longest)
    empty = rng.choice([0, 0, 1]) if seqs > 1 else 0
    return {k: v for k, v in _attend("", seqs, longest, shortest, empty, heads, kv_heads, dim, fmt, page).items() if k != "name"}


# ----------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _lengths(case):
    """Lengths of an attend case, longest first: the seed only shuffles them."""
    n = case["seqs"]
    span = case["longest"] - case["shortest"]
    out = [case["longest"] - round(span * (i / (n - 1)) ** 0.5) if n > 1 else case["longest"] for i in range(n)]
    out[n - case["empty"]:] = [0] * case["empty"]
    return out


def _table(gen, rows, rot):
    """cos and sin of (position x frequency): `rows` positions, each table built in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    # positions start somewhere: another seed is another window of the same sequence
    first = torch.randint(0, 4096, (1,), generator=gen, device="cuda", dtype=torch.int64)
    angle = (torch.arange(rows, device="cuda") + first).double()[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _key_like(gen, rows, heads, dim):
    """Rows as keys come: a common offset per head, a few strong channels, gaussian else."""
    x = torch.randn((rows, heads, dim), generator=gen, device="cuda")
    gain = torch.ones((heads, dim), device="cuda")
    gain[torch.rand((heads, dim), generator=gen, device="cuda") < 0.03] = 6.0
    return (x + 0.3 * torch.randn((heads, dim), generator=gen, device="cuda")) * gain


def _fill_codes(gen, pages, kv_heads, page, dim, fmt):
    """A cache of random rows, as (codes, scales): the group rule, on fp32 values."""
    codes = torch.empty((pages, kv_heads, page, dim if fmt == "mxfp8" else dim // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((pages, kv_heads, page, dim // 32), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // (kv_heads * page * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = _key_like(gen, n * page, kv_heads, dim).bfloat16().float().view(n, page, kv_heads, dim // 32, 32).transpose(1, 2)
        _, e = torch.frexp(x.abs().amax(-1, keepdim=True))
        e = e - 1 - (8 if fmt == "mxfp8" else 2)
        x = x * _two(-e).float()
        scales[at:at + n] = (e[..., 0] + 127).to(torch.uint8)
        if fmt == "mxfp8":
            codes[at:at + n] = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
        else:
            i = _e2m1_index(x.abs()) | (x < 0).to(torch.uint8) << 3
            i = i.flatten(-2)
            codes[at:at + n] = i[..., 0::2] | i[..., 1::2] << 4
    return codes, scales


def prepare(case, seed):
    g = _gen(seed)
    kind, kvh, dim = case["kind"], case["kv_heads"], case["dim"]
    s = {"case": case}
    if kind in ("rope", "store"):
        rows, heads = case["rows"], case["heads"]
        width = (heads + 2 * kvh) * dim
        s["qkv"] = _key_like(g, rows, heads + 2 * kvh, dim).view(rows, width).bfloat16()
        if case["rot"]:
            s["cos"], s["sin"] = _table(g, case["table"], case["rot"])
        s["positions"] = None
        if kind == "store" and case["rot"] or kind == "rope" and case["scattered"]:
            s["positions"] = torch.randint(0, case["table"], (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["q_weight"] = s["k_weight"] = None
        if case["norm"]:
            s["q_weight"], s["k_weight"] = ((1 + 0.2 * torch.randn(dim, generator=g, device="cuda")).bfloat16() for _ in range(2))
    if kind in ("store", "read"):
        page = case["page"]
        pages = -(-case["rows"] // page) + 3
        free = torch.randperm(pages * page, generator=g, device="cuda")[: case["rows"]].to(torch.int32)
        if kind == "store":
            free[case["rows"] - case["padded"]:] = -1  # the rows that pad the batch
            empty = (pages, kvh, page, dim if case["fmt"] == "mxfp8" else dim // 2)
            s["cache"] = [torch.zeros(empty, dtype=torch.uint8, device="cuda") for _ in range(2)]
            s["cache"] += [torch.zeros((pages, kvh, page, dim // 32), dtype=torch.uint8, device="cuda") for _ in range(2)]
        else:
            k, v = (_fill_codes(g, pages, kvh, page, dim, case["fmt"]) for _ in range(2))
            s["cache"] = [k[0], v[0], k[1], v[1]]
            free = free.sort().values if case["rows"] > 1000 else free  # a prefix comes in its order
        s["slots"] = free
    if kind == "attend":
        page, lengths = case["page"], _lengths(case)
        most = -(-max(lengths) // page)
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 2
        k, v = (_fill_codes(g, pages, kvh, page, dim, case["fmt"]) for _ in range(2))
        s["cache"] = [k[0], v[0], k[1], v[1]]
        order = torch.randperm(len(lengths), generator=g, device="cuda")
        lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")[order]
        used = torch.arange(most, device="cuda")[None] * page < lens[:, None]
        s["table"] = torch.full((len(lengths), most), -1, dtype=torch.int32, device="cuda")
        s["table"][used] = torch.randperm(pages, generator=g, device="cuda")[: sum(need)].to(torch.int32)
        s["lengths"] = lens
        s["q"] = (1.5 * torch.randn((len(lengths), case["heads"], dim), generator=g, device="cuda")).bfloat16()
    return s


# ------------------------------------------------------------------------------ plain forms
def _e2m1_index(m):
    """Nearest E2M1 magnitude of m >= 0, a tie to the even code."""
    up = [m > 0.25, m >= 0.75, m > 1.25, m >= 1.75, m > 2.5, m >= 3.5, m > 5.0]
    return torch.stack(up).sum(0).to(torch.uint8)


def _two(n):
    """2**n in 64 bits for whole n, from the bits: a power function may be an ulp off, which would break ties."""
    return ((n.long() + 1023) << 52).view(torch.float64)


def _values(codes, scales, fmt, dtype):
    """The values a cache's rows stand for."""
    if fmt == "mxfp8":
        v = codes.view(torch.float8_e4m3fn).to(dtype)
    else:
        nib = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
        v = torch.tensor(_E2M1 + tuple(-x for x in _E2M1), dtype=dtype, device=codes.device)[nib]
    two = _two(scales.long() - 127).to(dtype)
    return (v.unflatten(-1, (-1, 32)) * two[..., None]).flatten(-2)


def _rotated(x, cos, sin, inter):
    """The rotation of the first 2 * cos.shape[-1] elements of every head of x [rows, heads, dim]."""
    h = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if inter else (x[..., :h], x[..., h:2 * h])
    out = (a * c - b * s, b * c + a * s)
    head = torch.stack(out, -1).flatten(-2) if inter else torch.cat(out, -1)
    return torch.cat((head, x[..., 2 * h:]), -1)


def _norm_rope(s, dtype_q, dtype_k):
    """q and k of the QKV rows, normed and rotated, unrounded: each in its own type."""
    c = s["case"]
    x = s["qkv"].view(c["rows"], -1, c["dim"])
    at = slice(0, c["rows"]) if s["positions"] is None else s["positions"].long()
    out = []
    for part, w, dt in ((x[:, : c["heads"]], s["q_weight"], dtype_q), (x[:, c["heads"]: c["heads"] + c["kv_heads"]], s["k_weight"], dtype_k)):
        y = part.to(dt)
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * w.to(dt)
        out.append(_rotated(y, s["cos"][at].to(dt), s["sin"][at].to(dt), c["inter"]))
    return out


def _grouped(x, fmt):
    """x [..., dim] in 64 bits -> (codes, scale bytes) by the group rule."""
    x = x.unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(amax)
    e = torch.where(amax > 0, (e - 1 - (8 if fmt == "mxfp8" else 2)).clamp(-127, 127), -127)
    y = x * _two(-e)
    if fmt == "mxfp8":
        # to the grid of E4M3 in 64 bits (steps of 2^(e-3), 2^-9 at least), then the cast is exact
        _, ye = torch.frexp(y)
        step = _two((ye - 4).clamp(min=-9))
        y = ((y / step).round() * step).clamp(-448, 448)
        codes = y.float().to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    else:
        i = (_e2m1_index(y.abs()) | (y < 0).to(torch.uint8) << 3).flatten(-2)
        codes = i[..., 0::2] | i[..., 1::2] << 4
    return codes, (e[..., 0] + 127).to(torch.uint8)


def _rows_of(cache, slots, page):
    """codes and scales of the rows that `slots` names, [rows, heads, ...]; a negative one reads zeros."""
    at = slots.long().clamp(min=0)
    live = (slots >= 0)[:, None, None]
    return [torch.where(live, t[at // page, :, at % page], torch.zeros((), dtype=t.dtype, device=t.device)) for t in cache]


def _plain_store(s):
    c = s["case"]
    page, fmt = c["page"], c["fmt"]
    x = s["qkv"].view(c["rows"], -1, c["dim"])
    v = x[:, c["heads"] + c["kv_heads"]:].double()
    q = None
    if c["rotate"]:
        q, k = _norm_rope(s, torch.float32, torch.float64)  # keys meet rounding borders: 64 bits
    else:
        k = x[:, c["heads"]: c["heads"] + c["kv_heads"]].double()
    live = s["slots"] >= 0
    at = s["slots"][live].long()
    kc, vc, ks, vs = s["cache"]
    for codes, scales, rows in ((kc, ks, k), (vc, vs, v)):
        new, two = _grouped(rows[live], fmt)
        codes[at // page, :, at % page], scales[at // page, :, at % page] = new, two
    back = _plain_read(s)
    return back if q is None else (q.bfloat16(), *back)


def _plain_read(s):
    c = s["case"]
    kc, vc, ks, vs = _rows_of(s["cache"], s["slots"], c["page"])
    return tuple(_values(a, b, c["fmt"], torch.float32).bfloat16() for a, b in ((kc, ks), (vc, vs)))


def _plain_attend(s):
    c = s["case"]
    kc, vc, ks, vs = (t[s["table"].long().clamp(min=0)] for t in s["cache"])  # [seqs, pages, heads, page, ...]
    k, v = (_values(a, b, c["fmt"], torch.float32).transpose(1, 2).flatten(2, 3) for a, b in ((kc, ks), (vc, vs)))
    q = s["q"].float().unflatten(1, (c["kv_heads"], -1))
    score = torch.matmul(q, k.transpose(-1, -2)) * c["dim"] ** -0.5
    seen = torch.arange(k.shape[2], device="cuda")[None] < s["lengths"][:, None]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.clamp(min=-1e30))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / total.clamp(min=1e-30)
    lse = (top + torch.log(total))[..., 0]
    return out.flatten(1, 2).bfloat16(), lse.flatten(1, 2)


def _own(s):
    mx = _mx()
    c, kind = s["case"], s["case"]["kind"]
    if kind in ("rope", "store") and c["rot"]:
        how = {"positions": s["positions"], "q_weight": s["q_weight"], "k_weight": s["k_weight"], "eps": _EPS, "interleaved": c["inter"]}
    if kind == "rope":
        return mx.qk_norm_rope(s["qkv"], c["heads"], c["kv_heads"], s["cos"], s["sin"], **how)
    cache = s.get("handle")
    if cache is None:
        cache = s["handle"] = mx.MXKVCache(*s["cache"], format=c["fmt"])
    if kind == "attend":
        return mx.paged_attention(s["q"], cache, s["table"], s["lengths"], return_lse=True)
    if kind == "read":
        return mx.kv_cache_read(cache, s["slots"])
    if c["rotate"]:
        q = mx.qk_norm_rope_cache(s["qkv"], c["heads"], c["kv_heads"], s["cos"], s["sin"], cache, s["slots"], **how)
        return (q, *mx.kv_cache_read(cache, s["slots"]))
    x = s["qkv"].view(c["rows"], -1, c["dim"])
    mx.kv_cache_write(cache, x[:, c["heads"]: c["heads"] + c["kv_heads"]], x[:, c["heads"] + c["kv_heads"]:], s["slots"])
    return mx.kv_cache_read(cache, s["slots"])


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "rope":
        q, k = _norm_rope(state, torch.float32, torch.float32)
        return q.bfloat16(), k.bfloat16()
    if kind == "store":
        return _plain_store(state)
    return _plain_read(state) if kind == "read" else _plain_attend(state)


# ------------------------------------------------------------------------------------- work
def work(case):
    kvh, dim = case["kv_heads"], case["dim"]
    if case["kind"] == "attend":
        keys = sum(_lengths(case))
        row = 2 * kvh * (dim // (1 if case["fmt"] == "mxfp8" else 2) + dim // 32)
        return {"bytes": keys * row + case["seqs"] * case["heads"] * (4 * dim + 4), "flops": 4 * keys * case["heads"] * dim}
    rows, value = case["rows"], 2 * kvh * dim * 2  # a row's k and v in bf16
    if case["kind"] == "rope":
        parts = (case["heads"] + kvh) * dim
        return {"bytes": rows * parts * 4 + min(rows, case["table"]) * case["rot"] * 4, "flops": rows * parts * 8}
    coded = 2 * kvh * (dim // (1 if case["fmt"] == "mxfp8" else 2) + dim // 32)
    if case["kind"] == "read":
        return {"bytes": rows * (coded + value + 4), "flops": rows * value / 2}
    q = case["heads"] * dim * 4 if case["rotate"] else 0
    tables = min(rows, case["table"]) * case["rot"] * 4
    # qkv in, q out, the codes written and read, the values out
    return {"bytes": rows * (q + value + 2 * coded + value + 8) + tables, "flops": rows * (q * 2 + value * 4)}


# -------------------------------------------------------------------- the definition, 64 bits
def _power(n):
    """2**n for whole n held in any type: looked up, so that it is the number itself."""
    table = torch.tensor([math.ldexp(1.0, i) for i in range(-300, 301)], dtype=torch.float64, device="cuda")
    return table[n.long() + 300]


def _decoded(codes, scales, fmt):
    """One row set's values in 64 bits, from the fields of each code."""
    if fmt == "mxfp8":
        b = codes.long()
        e, m = b >> 3 & 15, (b & 7).double()
        mag = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * _power(e - 10))
        x = torch.where(b > 127, -mag, mag)
    else:
        b = codes.long()[..., None] >> torch.tensor([0, 4], device=codes.device) & 15
        b = b.reshape(*codes.shape[:-1], -1)
        e, m = b >> 1 & 3, (b & 1).double()
        mag = torch.where(e == 0, m / 2, (2 + m) * _power(e - 2))
        x = torch.where(b > 7, -mag, mag)
    return x * _power(scales.long() - 127).repeat_interleave(32, -1)


def _coded_value(x, fmt):
    """What a group of 32 stands for once it is coded: x to the nearest multiple of its step."""
    top, mant, big, small = (8, 3, 448.0, -6) if fmt == "mxfp8" else (2, 1, 6.0, 0)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    peak = g.abs().max(-1, keepdim=True).values
    low = torch.floor(torch.log2(torch.where(peak > 0, peak, 1.0)))
    low = torch.where(_power(low + 1) <= peak, low + 1, torch.where(_power(low) > peak, low - 1, low))
    two = _power(torch.where(peak > 0, low - top, -127.0).clamp(-127, 127))
    y = (g / two).clamp(-big, big)
    lev = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** small)))
    lev = torch.where(_power(lev) > y.abs().clamp(min=2.0 ** small), lev - 1, lev)
    step = _power(lev - mant)
    return (torch.round(y / step) * step * two).reshape(x.shape)


def _exact_rotation(s, heads, weight):
    """One set of heads [rows, n, dim] in 64 bits: norm, then the rotation as a complex product."""
    c = s["case"]
    x = heads.double()
    if weight is not None:
        x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["dim"] + _EPS) * weight.double()
    pos = torch.arange(c["rows"], device="cuda") if s["positions"] is None else s["positions"].long()
    turn = torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
    r = c["rot"]
    if c["inter"]:
        z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * turn
        y = torch.view_as_real(z).reshape(*x.shape[:-1], r)
    else:
        z = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2: r].contiguous()) * turn
        y = torch.cat((z.real, z.imag), -1)
    return torch.cat((y, x[..., r:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    kvh = case["kv_heads"]
    if case["kind"] == "attend":
        page, out, lse = case["page"], [], []
        kc, vc, ks, vs = s["cache"]
        for b, n in enumerate(s["lengths"].tolist()):
            q = s["q"][b].double().view(kvh, -1, case["dim"])
            if n == 0:
                out.append(torch.zeros_like(q).flatten(0, 1))
                lse.append(torch.full((case["heads"],), -math.inf, dtype=torch.float64, device="cuda"))
                continue
            ids = s["table"][b, : -(-n // page)].long()
            k, v = (_decoded(a[ids].transpose(0, 1).flatten(1, 2)[:, :n], t[ids].transpose(0, 1).flatten(1, 2)[:, :n], case["fmt"])
                    for a, t in ((kc, ks), (vc, vs)))
            z = torch.einsum("hgd,hnd->hgn", q, k) / math.sqrt(case["dim"])
            out.append(torch.einsum("hgn,hnd->hgd", torch.softmax(z, -1), v).flatten(0, 1))
            lse.append(torch.logsumexp(z, -1).flatten())
        return torch.stack(out), torch.stack(lse)
    if case["kind"] == "read":
        at = s["slots"].long()
        kc, vc, ks, vs = (t.transpose(1, 2).flatten(0, 1)[at] for t in s["cache"])
        return _decoded(kc, ks, case["fmt"]), _decoded(vc, vs, case["fmt"])
    x = s["qkv"].view(case["rows"], -1, case["dim"])
    q, k, v = x[:, : case["heads"]], x[:, case["heads"]: case["heads"] + kvh], x[:, case["heads"] + kvh:]
    if case["rot"]:
        q, k = _exact_rotation(s, q, s["q_weight"]), _exact_rotation(s, k, s["k_weight"])
    if case["kind"] == "rope":
        return q, k
    live = (s["slots"] >= 0).double()[:, None, None]
    k, v = (_coded_value(t.double(), case["fmt"]) * live for t in (k, v))
    return (q, k, v) if case["rotate"] else (k, v)
