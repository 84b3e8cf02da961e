"""Performance cases of a DiT block's operators around its FP8 attention: rotary positions over several
axes, the gated residual with the norms on its two sides, and the microscaled 4-bit linear.

* ``table``: cos / sin of multi-axis (time, height, width) rotary angles, once per sequence;
* ``rotate``: per-head RMS norm and rotation of the query and key parts of a fused QKV projection;
* ``block``: r = x + gate * norm(branch), y = norm(r) * (1 + scale) + shift, in 16 bits or in the e4m3 codes
  that the next linear reads;
* ``weights``: a weight matrix to 32-value blocks of 4-bit codes and back;
* ``linear``: activations quantized to 4 bits on the fly, times a 4-bit weight, with bias and GELU-tanh; also
  fed by ``block`` without the 16-bit detour.

Where ``own`` is false, ``run`` computes each from elementary torch operations in 32 bits (angles in 64).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
HIDDEN, MLP, HEADS, HEAD_DIM = 3072, 12288, 24, 128
TOKENS_480, TOKENS_720, TOKENS_AUDIO, TOKENS_TEXT = 20280, 77648, 1024, 512
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA, EPS = 10000.0, 1e-6
GROUP = 256  # values of K per slab of block scales (8 blocks of 32)


def _table(name, batch, frames, height, width, extra, dims, fractional):
    """frames x height x width patches and `extra` tokens of a second stream (audio) that moves on the time
    axis alone; fractional: times in 25ths of a frame, far into a long clip."""
    c = {"kind": "table", "batch": batch, "frames": frames, "height": height, "width": width, "extra": extra,
         "dims": "-".join(map(str, dims)), "fractional": fractional}
    return {"name": name, **c} if name else c


def _rotate(name, b, s, hq, hk, d, pairs, norm=True, interleaved=True, per_batch=False, dtype="bf16"):
    c = {"kind": "rotate", "b": b, "s": s, "hq": hq, "hk": hk, "d": d, "pairs": pairs, "norm": norm,
         "interleaved": interleaved, "per_batch": per_batch, "dtype": dtype}
    return {"name": name, **c} if name else c


def _block(name, b, s, c, norm="layer", sandwich=False, groups=1, quantize="", dtype="bf16"):
    """sandwich: the branch has its own RMS norm; groups: spans of s / groups tokens with a modulation each."""
    d = {"kind": "block", "b": b, "s": s, "c": c, "norm": norm, "sandwich": sandwich, "groups": groups,
         "quantize": quantize, "dtype": dtype}
    return {"name": name, **d} if name else d


def _linear(name, m, k, n, gelu=False, bias=True, block=False, dtype="bf16"):
    """block: the input is the gated residual's modulated norm, quantized where it is computed."""
    c = {"kind": "linear", "m": m, "k": k, "n": n, "gelu": gelu, "bias": bias, "block": block, "dtype": dtype}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a 480p clip of 13 frames of 30 x 52 patches: once per resolution and clip length
        _table("table_480p", 1, 13, 30, 52, 0, (44, 42, 42), False),
        # joint video and audio of two items, at times of their own late in a long clip
        _table("table_joint_far", 2, 13, 30, 52, TOKENS_AUDIO, (32, 48, 48), True),
        # one token (a register or time-step token): latency
        _rotate("rotate_one_token", 1, 1, HEADS, HEADS, HEAD_DIM, 64),
        # every block of the 480p clip: query and key views of the fused QKV projection
        _rotate("rotate_480p", 1, TOKENS_480, HEADS, HEADS, HEAD_DIM, 64),
        # a joint sequence of two items with half-split pairs, grouped key heads and channels that do not rotate
        _rotate("rotate_joint_half", 2, 6113, 32, 8, 64, 24, norm=False, interleaved=False, per_batch=True,
                dtype="fp16"),
        # one token's gated residual and next norm: latency
        _block("block_one_token", 1, 1, HIDDEN),
        # every block of the 480p clip: attention output gated into the residual, then the MLP's modulated norm
        _block("block_480p", 1, TOKENS_480, HIDDEN),
        # norms on both sides of the branch, a modulation per frame, an odd width
        _block("block_sandwich", 2, 13 * 391, 2730, norm="rms", sandwich=True, groups=13, dtype="bf16"),
        # a block's MLP weight, quantized on loading and read back (merging an adapter into it)
        _linear_weights("weights_mlp", MLP, HIDDEN),
        # one token through the fused QKV projection
        _linear("linear_one_token", 1, HIDDEN, 3 * HIDDEN),
        # the text context's key / value projection, an odd number of tokens
        _linear("linear_text", TOKENS_TEXT + 1, HIDDEN, HIDDEN),
        # the MLP's up projection of the 480p clip, fed by the gated residual's modulated norm, with its GELU
        _linear("mlp_up_480p", TOKENS_480, HIDDEN, MLP, gelu=True, block=True),
    ]


def _linear_weights(name, n, k, dtype="bf16"):
    c = {"kind": "weights", "n": n, "k": k, "dtype": dtype}
    return {"name": name, **c} if name else c


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["table", "rotate", "rotate", "block", "block", "weights", "linear", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    if kind == "table":
        dims = rng.choice([(44, 42, 42), (16, 56, 56), (64,), (32, 32), (8, 20, 20, 16), (32, 48, 48), (2, 10, 12)])
        return _table(None, rng.choice([1, 1, 2]), log_int(1, 21), log_int(1, 45), log_int(1, 80),
                      rng.choice([0, log_int(1, 1024)]), dims, rng.random() < 0.5)
    if kind == "rotate":
        d, pairs = rng.choice([(128, 64), (128, 64), (64, 32), (128, 48), (96, 48), (80, 33), (72, 36), (256, 128),
                               (50, 25)])
        hq, hk = rng.choice([(HEADS, HEADS), (12, 12), (32, 8), (40, 40), (5, 1), (16, 0)])
        b = rng.choice([1, 1, 2, 3])
        return _rotate(None, b, log_int(1, min(20280, 120_000_000 // (b * (hq + hk) * d))), hq, hk, d, pairs,
                       norm=rng.random() < 0.7, interleaved=rng.random() < 0.5, per_batch=rng.random() < 0.3,
                       dtype=dtype)
    if kind == "block":
        groups, b = rng.choice([1, 1, 1, 7, 13]), rng.choice([1, 1, 2, 3])
        c = rng.choice([HIDDEN, HIDDEN, 1024, 1536, 5120, 8192, 2730, 1000, 96, 33, 12288])
        s = log_int(1, min(20280, 60_000_000 // (b * c)))
        return _block(None, b, groups * max(1, s // groups), c, norm=rng.choice(["layer", "rms"]),
                      sandwich=rng.random() < 0.4, groups=groups, quantize=rng.choice(["", "", "e4m3"]), dtype=dtype)
    k = rng.choice([HIDDEN, HIDDEN, MLP, 1024, 1056, 1536, 4640, 32, 288])
    if kind == "weights":
        return _linear_weights(None, log_int(1, min(12288, 37_000_000 // k)), k, dtype=dtype)
    n = rng.choice([HIDDEN, 3 * HIDDEN, 2048, 4624, 64, 1001])
    return _linear(None, log_int(1, min(20280, 700_000_000_000 // (k * n))), k, n, gelu=rng.random() < 0.3,
                   bias=rng.random() < 0.8, block=k <= 8192 and rng.random() < 0.3, dtype=dtype)


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, device=DEV, generator=g) * std).to(dtype)


def _activations(g, *shape, dtype):
    """1% of the channels are 20 times larger: the outliers that scales of small blocks exist for."""
    x = torch.randn(shape, device=DEV, generator=g, dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16)
    x[..., torch.randperm(shape[-1], device=DEV, generator=g)[: shape[-1] // 100]] *= 20.0
    return x.to(dtype)


def _dims(case):
    return tuple(int(d) for d in case["dims"].split("-"))


def _tokens(case):
    return case["frames"] * case["height"] * case["width"] + case["extra"]


def _positions(case, seed):
    """[batch, tokens, axes] fp32 (or [tokens, axes] int64 for one item with whole positions)."""
    g = _gen(seed)
    f, h, w, extra, axes = case["frames"], case["height"], case["width"], case["extra"], len(_dims(case))
    i = torch.arange(f * h * w, device=DEV)
    grid = torch.stack([i // (h * w), i // w % h, i % w, i % 3][:axes], 1)
    more = torch.zeros((extra, axes), dtype=torch.int64, device=DEV)
    more[:, 0] = torch.arange(extra, device=DEV) * f // max(extra, 1)
    pos = torch.cat([grid, more])
    start = torch.randint(0, 4096, (case["batch"],), device=DEV, generator=g)
    pos = pos.expand(case["batch"], *pos.shape).clone()
    if not case["fractional"]:
        pos[:, :, 0] += start[:, None]
        return pos[0] if case["batch"] == 1 else pos
    pos = pos.to(torch.float32)
    pos[:, :, 0] = pos[:, :, 0] * 1.04 + 16.0 * start[:, None]
    return pos


def _qk(case, seed):
    """q, k as [B, H, S, D] views of one projection, fp32 cos / sin pairs, and the norms' weights."""
    g = _gen(seed)
    b, s, hq, hk, d, p = (case[i] for i in ("b", "s", "hq", "hk", "d", "pairs"))
    dt = DTYPES[case["dtype"]]
    qkv = _randn(g, b, s, (hq + 2 * hk) * d, dtype=dt)
    q = qkv[..., : hq * d].unflatten(-1, (hq, d)).transpose(1, 2)
    k = qkv[..., hq * d: (hq + hk) * d].unflatten(-1, (hk, d)).transpose(1, 2) if hk else None
    angle = torch.rand((b, s, p) if case["per_batch"] else (s, p), device=DEV, generator=g) * (2 * math.pi)
    table = torch.stack([torch.cos(angle), torch.sin(angle)], -1)
    qw = kw = None
    if case["norm"]:
        qw = (1.0 + 0.1 * _randn(g, d)).to(dt)
        kw = (1.0 + 0.1 * _randn(g, d)).to(dt) if hk else None
    return q, k, table, qw, kw


def _block_inputs(g, b, s, c, groups, sandwich, weighted, dtype):
    """Residual stream, branch output, and gate / shift / scale as views of one modulation tensor."""
    x = _activations(g, b, s, c, dtype=dtype)
    branch = _randn(g, b, s, c, dtype=dtype)
    mod = _randn(g, b, groups, 3 * c, std=0.3, dtype=dtype)
    gate, shift, scale = mod[..., :c], mod[..., c: 2 * c], mod[..., 2 * c:]
    if groups == 1:
        gate, shift, scale = gate[:, 0], shift[:, 0], scale[:, 0]
    bw = (1.0 + 0.1 * _randn(g, c)).to(dtype) if sandwich else None
    w = (1.0 + 0.1 * _randn(g, c)).to(dtype) if weighted else None
    return {"x": x, "branch": branch, "gate": gate, "shift": shift, "scale": scale, "branch_weight": bw, "weight": w}


def _block_case(case, seed):
    return _block_inputs(_gen(seed), case["b"], case["s"], case["c"], case["groups"], case["sandwich"],
                         case["norm"] == "rms", DTYPES[case["dtype"]])


def _linear_case(case, seed):
    """Input (or the gated residual's operands), weight [N, K] and bias; the weight is what a checkpoint holds."""
    g = _gen(seed)
    m, k, n = case["m"], case["k"], case["n"]
    dt = DTYPES[case["dtype"]]
    w = _randn(g, n, k, std=0.02, dtype=torch.bfloat16)
    bias = _randn(g, n, std=0.01, dtype=torch.bfloat16) if case["bias"] else None
    x = _block_inputs(g, 1, m, k, 1, False, False, dt) if case["block"] else _activations(g, m, k, dtype=dt)
    return x, w, bias


def prepare(case, seed):
    if case["kind"] == "table":
        return {"case": case, "positions": _positions(case, seed)}
    if case["kind"] == "rotate":
        return {"case": case, "args": _qk(case, seed)}
    if case["kind"] == "block":
        return {"case": case, "args": _block_case(case, seed)}
    if case["kind"] == "weights":
        return {"case": case, "w": _randn(_gen(seed), case["n"], case["k"], std=0.02, dtype=DTYPES[case["dtype"]])}
    x, w, bias = _linear_case(case, seed)
    w4, ws = _quantize(w)
    state = {"case": case, "x": x, "w4": w4, "w_scale": ws, "bias": bias}
    if own:  # the module of a converted model, made once
        from minimaxh3_amd.kernels.mxfp4_linear import MXFP4Linear

        state["module"] = MXFP4Linear.from_quantized(w4, ws, bias)
        state["module"].act = 1 if case["gelu"] else 0
    return state


# ---------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------

def _plain_table(positions, dims):
    inv = torch.cat([THETA ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d) for d in dims])
    axis = torch.repeat_interleave(torch.arange(len(dims), device=DEV), torch.tensor([d // 2 for d in dims], device=DEV))
    angle = positions.to(torch.float64)[..., axis] * inv
    return torch.stack([torch.cos(angle), torch.sin(angle)], -1).to(torch.float32)


def _plain_rotate(x, table, weight, interleaved):
    if x is None:
        return None
    dt, y = x.dtype, x.to(torch.float32)
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.to(torch.float32)
    p = table.shape[-2]
    t = table[:, None] if table.dim() == 4 else table
    cos, sin = t[..., 0], t[..., 1]
    a, b = (y[..., 0: 2 * p: 2], y[..., 1: 2 * p: 2]) if interleaved else (y[..., :p], y[..., p: 2 * p])
    u, v = a * cos - b * sin, a * sin + b * cos
    rot = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([rot, y[..., 2 * p:]], -1).to(dt)


def _plain_norm(x, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)


def _plain_block(a, norm):
    b, s, c = a["x"].shape
    dt = a["x"].dtype
    f = {k: None if v is None else v.to(torch.float32) for k, v in a.items()}
    rows = {k: f[k].reshape(b, -1, 1, c) for k in ("gate", "shift", "scale")}
    br = f["branch"]
    if f["branch_weight"] is not None:
        br = _plain_norm(br, "rms") * f["branch_weight"]
    span = (b, rows["gate"].shape[1], -1, c)
    r = f["x"].view(span) + rows["gate"] * br.view(span)
    n = _plain_norm(r, norm)
    if f["weight"] is not None:
        n = n * f["weight"]
    y = n * (1.0 + rows["scale"]) + rows["shift"]
    return r.view(b, s, c).to(dt), y.view(b, s, c).to(dt)


def _quantize(x):
    """x [M, K] -> 4-bit codes [M, K / 2] (two to a byte, the even column low) and power-of-two block scales
    [ceil(K / 256), M, 8] (exponent + 127)."""
    m, k = x.shape
    v = x.to(torch.float32).view(m, k // 32, 32)
    # the exponent of the block's largest magnitude, one more where it would round past 6 (from 7 / 4 on)
    top = v.abs().amax(-1).contiguous().view(torch.int32)
    e = ((top + 0x200000) >> 23) - 129
    bad = top >= 0x7F800000
    e = e.clamp(-127, 127)
    a = v * ((127 - e) << 23).clamp_min(1 << 22).view(torch.float32).unsqueeze(-1)
    mag = a.abs()
    code = ((mag > 0.25).to(torch.uint8) + (mag >= 0.75).to(torch.uint8) + (mag > 1.25).to(torch.uint8)
            + (mag >= 1.75).to(torch.uint8) + (mag > 2.5).to(torch.uint8) + (mag >= 3.5).to(torch.uint8)
            + (mag > 5.0).to(torch.uint8))
    code = (code | (torch.signbit(a).to(torch.uint8) << 3)).view(m, k)
    slabs = -(-k // GROUP)
    scale = torch.full((m, slabs * 8), 127, dtype=torch.uint8, device=x.device)
    scale[:, : k // 32] = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale.view(m, slabs, 8).transpose(0, 1).contiguous()


def _values(codes, scale):
    """The numbers that _quantize's codes and scales stand for, in 32 bits."""
    m, k = codes.shape[0], 2 * codes.shape[1]
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat([grid, -grid])
    v = grid[torch.stack([codes & 15, codes >> 4], -1).view(m, k).to(torch.int32)]
    e = scale.transpose(0, 1).reshape(m, -1)[:, : k // 32].to(torch.int32)
    p = torch.where(e == 0, torch.full_like(e, 1 << 22), e << 23).view(torch.float32)
    p = torch.where(e == 255, torch.full_like(p, math.nan), p)
    return (v.view(m, k // 32, 32) * p.unsqueeze(-1)).view(m, k)


def _plain_gelu(z):
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))


def _plain_linear(s):
    case, x = s["case"], s["x"]
    r = None
    if case["block"]:
        r, x = _plain_block(x, "layer")
        x = x[0]
    out = _values(*_quantize(x)) @ _values(s["w4"], s["w_scale"]).t()
    if s["bias"] is not None:
        out = out + s["bias"].to(torch.float32)
    if case["gelu"]:
        out = _plain_gelu(out)
    out = out.to(torch.bfloat16)
    return out if r is None else (r, out)


def _plain_codes(y):
    """y rounded to e4m3 with one scale a row, as the values that stands for (bf16)."""
    f = y.to(torch.float32)
    s = f.abs().amax(-1, keepdim=True).clamp_min(1e-12) / 448.0
    q = (f / s).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).to(torch.float32)
    return (q * s).to(torch.bfloat16)


def _plain(s):
    case = s["case"]
    if case["kind"] == "table":
        return _plain_table(s["positions"], _dims(case))
    if case["kind"] == "rotate":
        q, k, table, qw, kw = s["args"]
        out = [_plain_rotate(x, table, w, case["interleaved"]) for x, w in ((q, qw), (k, kw))]
        return out if k is not None else out[:1]
    if case["kind"] == "block":
        r, y = _plain_block(s["args"], case["norm"])
        return r, _plain_codes(y) if case["quantize"] else y
    if case["kind"] == "weights":
        return _values(*_quantize(s["w"])).to(torch.bfloat16)
    return _plain_linear(s)


def run(state):
    if not own:
        return _plain(state)
    from minimaxh3_amd.kernels.block_norms import gated_residual_norm
    from minimaxh3_amd.kernels.mxfp4_linear import dequantize_mxfp4, quantize_mxfp4
    from minimaxh3_amd.kernels.rotary import rotary_table, rotate_qk

    case = state["case"]
    if case["kind"] == "table":
        return rotary_table(state["positions"], _dims(case), theta=THETA)
    if case["kind"] == "rotate":
        q, k, table, qw, kw = state["args"]
        q, k = rotate_qk(q, k, table, q_weight=qw, k_weight=kw, eps=EPS, interleaved=case["interleaved"])
        return [q] if k is None else [q, k]
    if case["kind"] == "block":
        a = state["args"]
        if not case["quantize"]:
            return gated_residual_norm(**a, norm=case["norm"], eps=EPS)
        r, y8, ys = gated_residual_norm(**a, norm=case["norm"], eps=EPS, quantize=case["quantize"])
        return r, (y8.to(torch.float32) * ys).to(torch.bfloat16).view(r.shape)
    if case["kind"] == "weights":
        return dequantize_mxfp4(*quantize_mxfp4(state["w"]))
    if not case["block"]:
        return state["module"](state["x"]).to(torch.bfloat16)
    r, x4, xs = gated_residual_norm(**state["x"], eps=EPS, quantize="mxfp4")
    return r, state["module"].forward_quantized(x4, xs)


def work(case):
    es = 4 if case.get("dtype") == "fp32" else 2
    if case["kind"] == "table":
        n, pairs = case["batch"] * _tokens(case), sum(_dims(case)) // 2
        return {"bytes": n * len(_dims(case)) * 4 + n * pairs * 8, "flops": 8 * n * pairs}
    if case["kind"] == "rotate":
        n = case["b"] * case["s"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * es * n + 8 * case["s"] * case["pairs"] * (case["b"] if case["per_batch"] else 1),
                "flops": 8 * n}
    if case["kind"] == "block":
        n = case["b"] * case["s"] * case["c"]
        return {"bytes": n * (3 * es + (1 if case["quantize"] else es)) + 3 * es * case["b"] * case["groups"] * case["c"],
                "flops": 12 * n}
    if case["kind"] == "weights":
        n = case["n"] * case["k"]
        # written as codes and scales, read as such again, and written as bf16
        return {"bytes": es * n + 2 * (n // 2 + n // 32) + 2 * n, "flops": 4 * n}
    m, k, n = case["m"], case["k"], case["n"]
    return {"bytes": (3 if case["block"] else 1) * es * m * k + n * k // 2 + n * k // 32 + (2 * n if case["bias"] else 0)
            + 2 * m * n, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------------------
# the same results in 64 bits
# ---------------------------------------------------------------------------------------

def _exact_rms(x):
    return x / torch.sqrt(torch.mean(torch.square(x), -1, keepdim=True) + EPS)


def _exact_layer(x):
    mu = torch.mean(x, -1, keepdim=True)
    return (x - mu) / torch.sqrt(torch.var(x, -1, correction=0, keepdim=True) + EPS)


def _exact_block(a, norm, per):
    """(r, y) [B, S, C] in 64 bits, item by item; per: tokens that share a modulation row."""
    rs, ys = [], []
    for i in range(a["x"].shape[0]):
        def rows(t):
            t = t[i].to(torch.float64)
            return (t if t.dim() == 2 else t[None]).repeat_interleave(per, 0)

        u = a["branch"][i].to(torch.float64)
        if a["branch_weight"] is not None:
            u = _exact_rms(u) * a["branch_weight"].to(torch.float64)
        r = torch.addcmul(a["x"][i].to(torch.float64), rows(a["gate"]), u)
        n = _exact_layer(r) if norm == "layer" else _exact_rms(r)
        if a["weight"] is not None:
            n = n * a["weight"].to(torch.float64)
        ys.append(torch.addcmul(rows(a["shift"]), n, 1.0 + rows(a["scale"])))
        rs.append(r)
    return torch.stack(rs), torch.stack(ys)


def _exact_mx(x):
    """x [M, K] rounded to blocks of 32 four-bit values under a power of two, in 64 bits: the nearest of
    +-{0, 1/2, 1, 3/2, 2, 3, 4, 6} times the power, ties to the even code, the power chosen so that the block's
    largest magnitude lies in [7/2, 7) of it."""
    m, k = x.shape
    v = x.to(torch.float64).view(m, k // 32, 32)
    top = v.abs().amax(-1, keepdim=True)
    frac, e = torch.frexp(top)  # top = frac 2^e, frac in [1/2, 1)
    e = torch.where(top > 0, e - 3 + (frac >= 0.875).to(e.dtype), torch.full_like(e, -127)).clamp_min(-127)
    p = ((e.to(torch.int64) + 1023) << 52).view(torch.float64)
    a = (v / p).abs()
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).to(torch.float64)
    q = (torch.round(a / step) * step).clamp_max(6.0)
    return (torch.copysign(q, v) * p).view(m, k)


def exact(case, seed):
    if case["kind"] == "table":
        parts, pos = [], _positions(case, seed).to(torch.float64)
        for i, d in enumerate(_dims(case)):
            freq = torch.exp(torch.arange(d // 2, dtype=torch.float64, device=DEV) * (-2.0 * math.log(THETA) / d))
            parts.append(torch.view_as_real(torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                                                        pos[..., i: i + 1] * freq)))
        return torch.cat(parts, -2)
    if case["kind"] == "rotate":
        q, k, table, qw, kw = _qk(case, seed)
        p, d = case["pairs"], case["d"]
        turn = torch.view_as_complex(table.to(torch.float64).contiguous())
        turn = turn if turn.dim() == 2 else turn.unsqueeze(1)
        out = []
        for x, w in ((q, qw), (k, kw)):
            if x is None:
                continue
            y = x.to(torch.float64)
            if w is not None:
                y = _exact_rms(y) * w.to(torch.float64)
            first = torch.arange(p, device=DEV) * (2 if case["interleaved"] else 1)
            second = first + (1 if case["interleaved"] else p)
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            out.append(y)
        return out
    if case["kind"] == "block":
        a = _block_case(case, seed)
        r, y = _exact_block(a, case["norm"], case["s"] // case["groups"])
        if case["quantize"]:
            y = y.to(a["x"].dtype).to(torch.float64)  # the codes are those of y as it would be stored
            s = (y.abs().amax(-1, keepdim=True).to(torch.float32).clamp_min(1e-12) / 448.0).to(torch.float64)
            y = (y / s).clamp(-448.0, 448.0).to(torch.float32).to(torch.float8_e4m3fn).to(torch.float64) * s
        return r, y
    if case["kind"] == "weights":
        return _exact_mx(_randn(_gen(seed), case["n"], case["k"], std=0.02, dtype=DTYPES[case["dtype"]]))
    x, w, bias = _linear_case(case, seed)
    r = None
    if case["block"]:
        dt = x["x"].dtype
        r, y = _exact_block(x, "layer", case["m"])
        x = y[0].to(dt)
    wt = _exact_mx(w).t().contiguous()
    out = []
    for part in x.split(4096):
        y = _exact_mx(part) @ wt
        if bias is not None:
            y = y + bias.to(torch.float64)
        if case["gelu"]:
            y = y * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
        out.append(y)
    out = torch.cat(out)
    return out if r is None else (r, out)
