"""Performance cases of an e4m3 cache of keys and values, and of the attention that reads it.

A clip that is generated a few frames at a time, or a prompt that is read and continued, keeps the keys and values
of what is already there.  They are held in 8 bits in pages of ``page`` tokens, with a power-of-two scale for each
page and head:

* ``append``: new keys and values, the keys normed per head and rotated on the way, quantized into the pages behind
  the tokens that are there; then the written pages read back as the values they stand for;
* ``attend``: queries over the pages, a whole frame or prompt of them, a few, or one per sequence;
* ``run``: a frame's queries rotated, its keys and values appended, and its attention over the old and the new.

Where ``own`` is false, ``run`` computes each from elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
HEADS, HEAD_DIM = 24, 128
FRAME_480, TOKENS_480, TOKENS_TEXT = 30 * 52, 20280, 512
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
E_MIN, E_MAX = -32, 63  # exponents that a page's scale may take; it is held as exponent + 127


def _case(name, kind, b, h, hk, d, page, new, held, causal=False, cross=False, ragged=False, pairs=0, norm=False,
          interleaved=True, dtype="bf16"):
    """b sequences that hold up to `held` tokens and get up to `new`; cross: the queries are no part of the cache;
    ragged: each sequence has a length of its own; pairs: how many pairs of a head's channels turn."""
    c = {"kind": kind, "b": b, "h": h, "hk": hk, "d": d, "page": page, "new": new, "held": held, "causal": causal,
         "cross": cross, "ragged": ragged, "pairs": pairs, "norm": norm, "interleaved": interleaved, "dtype": dtype}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one token behind a frame: latency
        _case("append_one_token", "append", 1, HEADS, HEADS, HEAD_DIM, 64, 1, FRAME_480, pairs=64, norm=True),
        # a step of 64 sequences of lengths of their own, grouped key heads, half-split pairs
        _case("append_step", "append", 64, 32, 8, HEAD_DIM, 16, 1, 4096, ragged=True, pairs=64, interleaved=False),
        # the last frame of a 480p clip
        _case("append_frame_480p", "append", 1, HEADS, HEADS, HEAD_DIM, 64, FRAME_480, TOKENS_480 - FRAME_480, pairs=64,
              norm=True),
        # a whole 480p clip at once, into an empty cache
        _case("append_clip_480p", "append", 1, HEADS, HEADS, HEAD_DIM, 64, TOKENS_480, 0, pairs=64, norm=True),
        # one query over one frame: latency
        _case("attend_one_token", "attend", 1, HEADS, HEADS, HEAD_DIM, 64, 1, FRAME_480),
        # one query over a very long cache, grouped heads: split over the keys
        _case("attend_one_token_long", "attend", 1, 32, 8, HEAD_DIM, 64, 1, 131072 + 77),
        # a step of 64 sequences, from 129 tokens to 8192, small pages
        _case("attend_step", "attend", 64, 32, 8, HEAD_DIM, 16, 1, 8191, causal=True, ragged=True),
        # five drafted tokens of 16 sequences, narrow heads
        _case("attend_drafts", "attend", 16, 40, 8, 64, 32, 5, 3001, causal=True, ragged=True, dtype="fp16"),
        # the clip's queries over its cached text
        _case("attend_text", "attend", 1, HEADS, HEADS, HEAD_DIM, 64, TOKENS_480, TOKENS_TEXT + 1, cross=True),
        # prompts of three sequences, up to 4111 tokens, grouped narrow heads
        _case("attend_prompts", "attend", 3, 32, 8, 64, 16, 4111, 130, causal=True, ragged=True, dtype="fp16"),
        # a new frame over a clip of 13 and itself
        _case("attend_frame_480p", "attend", 1, HEADS, HEADS, HEAD_DIM, 64, FRAME_480, TOKENS_480),
        # two clips' new frames in a run: queries rotated, keys and values appended, attention over all
        _case("run_frames_480p", "run", 2, HEADS, HEADS, HEAD_DIM, 64, FRAME_480, 7 * FRAME_480, pairs=64, norm=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    kind = rng.choice(["append", "append", "attend", "attend", "attend", "run"])
    d = rng.choice([64, 128, 128])
    h, hk = rng.choice([(HEADS, HEADS), (12, 12), (32, 8), (40, 8), (16, 1), (5, 5), (7, 1), (12, 4)])
    b, page = rng.choice([1, 1, 2, 3, 8, 17, 64]), rng.choice([16, 32, 64, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"] if kind == "append" else ["bf16", "bf16", "fp16"])
    ragged, causal = b > 1 and rng.random() < 0.7, rng.random() < 0.5
    turn = {} if kind == "attend" else {
        "pairs": rng.choice([d // 2, d // 2, d // 2, 0, d // 4, 21]), "norm": rng.random() < 0.5,
        "interleaved": rng.random() < 0.5}
    cells = 400_000_000 // (b * hk * d)  # tokens that a sequence may hold
    if kind == "append":
        new = rng.choice([1, log_int(1, min(TOKENS_480, 60_000_000 // (b * hk * d)))])
        return _case(None, kind, b, h, hk, d, page, new, rng.choice([0, log_int(1, min(20000, cells))]),
                     ragged=ragged, dtype=dtype, **turn)
    new = rng.choice([1, 1, log_int(2, 16), log_int(16, min(TOKENS_480, cells))])
    rows = b * h * new
    held = log_int(1, max(1, min(131072, cells, 700_000_000 // rows) - new))
    if rows * (held + new) > 750_000_000:
        new, held = 257, 1 + 700_000_000 // (b * h * 257) // 8
    cross = kind == "attend" and rng.random() < 0.2
    return _case(None, kind, b, h, hk, d, page, new, held, causal=causal and not cross, cross=cross, ragged=ragged,
                 dtype=dtype, **turn)


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _lengths(case):
    """Tokens held and tokens new of each sequence, from the shortest to the longest."""
    b = case["b"]
    if not case["ragged"]:
        return [case["held"]] * b, [case["new"]] * b
    return [-(-case["held"] * (i + 1) // b) for i in range(b)], [-(-case["new"] * (i + 1) // b) for i in range(b)]


def _span(case):
    """Pages that a sequence's new tokens may touch."""
    return (case["new"] + case["page"] - 2) // case["page"] + 1


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, device=DEV, generator=g) * std).to(dtype)


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e, from the bits of a finite amax >= 0."""
    bits = amax.contiguous().view(torch.int32)
    return (((bits + 0x1FFFFF) >> 23) - 135).clamp(E_MIN, E_MAX)


def _power(e):
    return ((e + 127) << 23).view(torch.float32)


def _codes(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _pool(g, pages, hk, page, d):
    """Pages of keys (2% of the channels four times larger) or values, each head's of a size of its own."""
    x = torch.randn((pages, hk, page, d), device=DEV, generator=g, dtype=torch.bfloat16)
    x[..., torch.randperm(d, device=DEV, generator=g)[: d // 50]] *= 4.0
    x = x * torch.exp2(torch.randint(-2, 3, (hk, 1, 1), device=DEV, generator=g).to(torch.bfloat16))
    e = _exponent(x.abs().amax((-1, -2)).to(torch.float32))
    return _codes(x.to(torch.float32) * _power(-e)[..., None, None]).view(torch.uint8), (e + 127).to(torch.uint8)


def _inputs(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    b, h, hk, d, page, new = (case[i] for i in ("b", "h", "hk", "d", "page", "new"))
    dt = DTYPES[case["dtype"]]
    held, count = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in _lengths(case))
    order = torch.randperm(b, device=DEV, generator=g)
    held, count = held[order], count[order]
    width = (case["held"] + new) // page + 2
    # pages in any order, and none behind the last that a sequence needs
    table = torch.randperm(b * width, device=DEV, generator=g).to(torch.int32).view(b, width)
    column = torch.arange(width, device=DEV)
    table = torch.where(column < (held // page + _span(case))[:, None], table, -1)
    kc, ke = _pool(g, b * width, hk, page, d)
    vc, ve = _pool(g, b * width, hk, page, d)
    s = {"case": case, "table": table, "held": held, "count": count, "first": held // page * page,
         "k_codes": kc, "k_scale": ke, "v_codes": vc, "v_scale": ve}
    s["length"] = held if case["cross"] else held + count
    # views of one projection, [b, heads, new, d]
    qkv = _randn(g, b, new, (h + 2 * hk) * d, dtype=dt).split([h * d, hk * d, hk * d], -1)
    s["q"], s["k"], s["v"] = (t.unflatten(-1, (-1, d)).transpose(1, 2) for t in qkv)
    angle = torch.rand((new, case["pairs"]), device=DEV, generator=g) * (2 * math.pi)
    s["turns"] = torch.stack([torch.cos(angle), torch.sin(angle)], -1)
    s["q_weight"], s["k_weight"] = ((1.0 + 0.1 * _randn(g, d)).to(dt) if case["norm"] else None for _ in range(2))
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from minimaxh3_amd.kernels.kv_cache import FP8KVCache

        s["cache"] = FP8KVCache.from_tensors(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
    return s


# ---------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------

def _plain_turn(x, turns, weight, interleaved):
    """The norm of a head's channels, and the rotation of its pairs, in 32 bits."""
    y = x.to(torch.float32)
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.to(torch.float32)
    p = turns.shape[-2]
    cos, sin = turns[..., 0], turns[..., 1]
    a, b = (y[..., 0: 2 * p: 2], y[..., 1: 2 * p: 2]) if interleaved else (y[..., :p], y[..., p: 2 * p])
    u, v = a * cos - b * sin, a * sin + b * cos
    out = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([out, y[..., 2 * p:]], -1)


def _plain_write(codes, scale, pages, x, is_new, is_old):
    """New tokens x [b, n, hk, page, d] and the held ones before them in `pages` [b, n] of the pool, under the scale
    that both need: a page's scale grows with its tokens, and what it held is rounded again."""
    old = codes[pages].view(torch.float8_e4m3fn).to(torch.float32)
    e_old = scale[pages].to(torch.int32) - 127
    any_old = is_old.any(-1)[..., None]
    any_new = is_new.any(-1)[..., None]
    is_new, is_old = is_new[:, :, None, :, None], is_old[:, :, None, :, None]
    e = _exponent(torch.where(is_new, x, 0.0).abs().amax((-1, -2)))
    e = torch.where(any_old, torch.maximum(e, e_old), e)
    e = torch.where(any_new, e, e_old)
    kept = torch.where(is_old, old * _power(e_old - e)[..., None, None], old)
    codes[pages] = torch.where(is_new, _codes(x * _power(-e)[..., None, None]).view(torch.uint8),
                               _codes(kept).view(torch.uint8))
    scale[pages] = (e + 127).to(torch.uint8)


def _plain_append(s):
    case = s["case"]
    page, n, b = case["page"], _span(case), case["b"]
    index = (s["first"] // page).to(torch.int64)[:, None] + torch.arange(n, device=DEV)
    pages = s["table"].gather(1, index).to(torch.int64)
    position = index[..., None] * page + torch.arange(page, device=DEV)  # [b, n, page]
    token = position - s["held"][:, None, None]
    is_new, is_old = (token >= 0) & (token < s["count"][:, None, None]), token < 0
    at = token.clamp(0, case["new"] - 1).view(b, 1, n * page, 1)
    for x, name in ((_plain_turn(s["k"], s["turns"], s["k_weight"], case["interleaved"]), "k"),
                    (s["v"].to(torch.float32), "v")):
        x = x.gather(2, at.expand(-1, x.shape[1], -1, x.shape[3]))
        x = x.unflatten(2, (n, page)).transpose(1, 2)
        _plain_write(s[name + "_codes"], s[name + "_scale"], pages, x, is_new, is_old)
    there = (position < (s["held"] + s["count"])[:, None, None]).view(b, 1, n * page, 1)
    return [torch.where(there, _plain_values(s, name, pages), 0.0).to(torch.bfloat16) for name in "kv"]


def _plain_values(s, name, pages):
    """The values of `pages` [b, n] in 32 bits, [b, hk, n * page, d]."""
    e = s[name + "_scale"][pages].to(torch.int32) - 127
    x = s[name + "_codes"][pages].view(torch.float8_e4m3fn).to(torch.float32) * _power(e)[..., None, None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(s, q):
    case = s["case"]
    b, h, new, d = q.shape
    pages = s["table"].clamp_min(0).to(torch.int64)
    k, v = _plain_values(s, "k", pages), _plain_values(s, "v", pages)
    hk, n = k.shape[1], k.shape[2]
    x = q.to(torch.float32).reshape(b, hk, h // hk * new, d) @ k.transpose(-1, -2) / math.sqrt(d)
    x = x.view(b, hk, h // hk, new, n)
    key, row = torch.arange(n, device=DEV), torch.arange(new, device=DEV)
    count, length = s["count"][:, None, None], s["length"][:, None, None]
    seen = (key < length) & (row[:, None] < count)
    if case["causal"]:
        seen = seen & (key <= length - count + row[:, None])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True).clamp_min(-1e30)
    p = x.exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, -1, n) @ v).view(b, hk, h // hk, new, d)
    return (o / total.clamp_min(1e-30)).reshape(b, h, new, d).to(q.dtype)


def _plain(s):
    case = s["case"]
    if case["kind"] == "append":
        return _plain_append(s)
    if case["kind"] == "attend":
        return [_plain_attend(s, s["q"])]
    q = _plain_turn(s["q"], s["turns"], s["q_weight"], case["interleaved"]).to(s["q"].dtype)
    written = _plain_append(s)
    return [_plain_attend(s, q), *written]


def run(state):
    if not own:
        return _plain(state)
    from minimaxh3_amd.kernels.kv_cache import append_kv, cached_attention, read_kv
    from minimaxh3_amd.kernels.rotary import rotate_qk

    s, case = state, state["case"]
    q, out = s["q"], []
    ragged = s["count"] if case["ragged"] else None
    turns = s["turns"] if case["pairs"] else None
    if case["kind"] == "run" and (case["pairs"] or case["norm"]):
        q, _ = rotate_qk(q, None, s["turns"], q_weight=s["q_weight"], eps=EPS, interleaved=case["interleaved"])
    if case["kind"] != "attend":
        append_kv(s["cache"], s["table"], s["held"], s["k"], s["v"], counts=ragged, table=turns,
                  k_weight=s["k_weight"], eps=EPS, interleaved=case["interleaved"])
        out = list(read_kv(s["cache"], s["table"], s["first"], _span(case) * case["page"], lengths=s["held"] + s["count"]))
    if case["kind"] != "append":
        out.insert(0, cached_attention(q, s["cache"], s["table"], s["length"], causal=case["causal"], q_lengths=ragged))
    return out


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    h, hk, d, page = case["h"], case["hk"], case["d"], case["page"]
    held, count = _lengths(case)
    size, flops, new = 0, 0, sum(count)
    if case["kind"] != "attend":
        # new keys and values read and written as codes; the written pages' values
        size += 2 * new * hk * d * (es + 1) + 8 * case["new"] * case["pairs"]
        size += 2 * 2 * sum(a + n - a // page * page for a, n in zip(held, count)) * hk * d
        flops += 8 * new * hk * d
    if case["kind"] != "append":
        length = [a + (0 if case["cross"] else n) for a, n in zip(held, count)]
        size += 2 * sum(length) * hk * d + 2 * es * new * h * d
        seen = sum(n * m - (n * (n - 1) // 2 if case["causal"] else 0) for n, m in zip(count, length))
        flops += 4 * seen * h * d
    return {"bytes": size, "flops": flops}


# ---------------------------------------------------------------------------------------
# the same results in 64 bits
# ---------------------------------------------------------------------------------------

def _exact_decode(codes, scale):
    """Sign, exponent and fraction of an e4m3 code, read apart; times the page's power of two."""
    c = codes.to(torch.int64)
    e, f = c >> 3 & 15, (c & 7).to(torch.float64)
    mag = torch.where(e == 0, f * 2.0 ** -9, torch.ldexp(1.0 + f / 8.0, e - 7))
    return torch.ldexp(torch.where(c >= 128, -mag, mag), (scale.to(torch.int64) - 127)[..., None, None])


def _exact_round(x):
    """The nearest number of three fraction bits, in steps of 2^-9 below 2^-6, no larger than 448; ties to even."""
    _, e = torch.frexp(x)  # |x| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp_min(-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def _exact_turn(x, turns, weight, interleaved):
    y = x.to(torch.float64)
    if weight is not None:
        y = y / torch.sqrt(torch.mean(torch.square(y), -1, keepdim=True) + EPS) * weight.to(torch.float64)
    p = turns.shape[-2]
    at = torch.arange(p, device=DEV)
    i, j = (2 * at, 2 * at + 1) if interleaved else (at, at + p)
    z = torch.complex(y[..., i], y[..., j]) * torch.view_as_complex(turns.to(torch.float64).contiguous())
    y = y.clone()
    y[..., i], y[..., j] = z.real, z.imag
    return y


def _exact_sequence(s, i, name, x):
    """All tokens of sequence i in the cache, [hk, tokens, d]; x: its new ones, or None."""
    page, held = s["case"]["page"], int(s["held"][i])
    n = int(s["count"][i]) if x is not None else 0
    total = int(s["length"][i]) if x is None else held + n
    pages = s["table"][i, : -(-total // page)].to(torch.int64)
    v = _exact_decode(s[name + "_codes"][pages], s[name + "_scale"][pages])  # [pages, hk, page, d]
    v = v.transpose(0, 1).flatten(1, 2)
    if x is not None:
        first = held // page
        v[:, held: held + n] = x[:, :n]
        touched = v[:, first * page:].unflatten(1, (-1, page))
        size = touched.clone()
        size[:, 0, : held - first * page] = 0.0  # the scale of held tokens is held
        size.flatten(1, 2)[:, held + n - first * page:] = 0.0
        top = size.abs().amax((-1, -2))
        f, e = torch.frexp(top)
        e = torch.where(top > 0, e - 9 + (f > 0.875).to(e.dtype), torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)
        if held > first * page:
            e[:, 0] = torch.maximum(e[:, 0], s[name + "_scale"][pages[first]].to(e.dtype) - 127)
        e = e[..., None, None].to(torch.int64)
        v[:, first * page:] = torch.ldexp(_exact_round(torch.ldexp(touched, -e)), e).flatten(1, 2)
    return v[:, :total]


def exact(case, seed):
    s = _inputs(case, seed)
    b, h, hk, d, new, page = (case[i] for i in ("b", "h", "hk", "d", "new", "page"))
    written = [torch.zeros((b, hk, _span(case) * page, d), dtype=torch.float64, device=DEV) for _ in range(2)]
    out = torch.zeros((b, h, new, d), dtype=torch.float64, device=DEV)
    for i in range(b):
        k = v = None
        q = s["q"][i].to(torch.float64)
        if case["kind"] != "attend":
            k = _exact_turn(s["k"][i], s["turns"], s["k_weight"], case["interleaved"])
            v = s["v"][i].to(torch.float64)
            q = _exact_turn(s["q"][i], s["turns"], s["q_weight"], case["interleaved"]).to(s["q"].dtype).to(torch.float64)
        k, v = _exact_sequence(s, i, "k", k), _exact_sequence(s, i, "v", v)
        n, length = int(s["count"][i]), int(s["length"][i])
        if case["kind"] != "attend":
            at = int(s["first"][i])
            written[0][i, :, : k.shape[1] - at], written[1][i, :, : v.shape[1] - at] = k[:, at:], v[:, at:]
        if case["kind"] == "append":
            continue
        key, row = torch.arange(length, device=DEV), torch.arange(n, device=DEV)
        for j in range(h):
            x = torch.mm(q[j, :n], k[j * hk // h].t()) * d ** -0.5
            if case["causal"]:
                x = x + torch.where(key > length - n + row[:, None], -math.inf, 0.0)
            if length:
                out[i, j, :n] = torch.mm(torch.softmax(x, -1), v[j * hk // h])
    return written if case["kind"] == "append" else [out] if case["kind"] == "attend" else [out, *written]
