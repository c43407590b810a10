"""Measured cases of the 8-bit decoder-layer operators.

Three operators, as the layers of a decoder call them one after the other:

* ``linear``: the product of 16-bit rows with 8-bit weights in whole numbers. Every row of x is quantised with a scale of its own (after its RMS
  norm, where there is one), every output channel has a scale and, in the asymmetric form, a zero point; bias, activation and residual follow.
* ``heads``: RMS norm of every query and key head and rotation by the position, without a cache (whole sequences, an encoder or a first pass).
* ``append``: the same on the fused projection of a serving step, with the key and value rows going to their slots of the paged cache.

Definitions that the forms below share. Quantisation of a row y: a = max |y|, q = round_half_even(y * (127 / a)) with the quotient and the product in
32 bits, scale = a / 127; a row without a value of at least 2^-119 is zero, one with a value that is not finite has the scale NaN. Rotation: dimension
pairs (i, i + rot / 2), or (2 i, 2 i + 1) in the interleaved form, turn by positions * inv_freq[i]; dimensions from rot on stay.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-5
BLOCK = 16                 # tokens of a KV block
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _linear(name, T, N, K, type="bf16", act="none", norm=False, zero_points=False, bias=False, residual=False, out32=False):
    return {"name": name, "kind": "linear", "T": T, "N": N, "K": K, "type": type, "act": act, "norm": norm, "zero_points": zero_points, "bias": bias,
            "residual": residual, "out32": out32}


def _heads(name, B, S, Hq, Hkv, D, rot=0, type="bf16", norm=True, interleaved=False, theta=500000.0, first=0):
    return {"name": name, "kind": "heads", "B": B, "S": S, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot or D, "type": type, "norm": norm,
            "interleaved": interleaved, "theta": theta, "first": first}


def _append(name, seqs, new, past, Hq, Hkv, D, rot=0, type="bf16", norm=True, interleaved=False, theta=500000.0):
    return {"name": name, "kind": "append", "seqs": seqs, "new": new, "past": past, "Hq": Hq, "Hkv": Hkv, "D": D, "rot": rot or D, "type": type,
            "norm": norm, "interleaved": interleaved, "theta": theta}


def listed():
    return [
        # one user, one token: the fused query / key / value projection behind its norm
        _linear("linear_1_norm", 1, 6144, 4096, norm=True),
        # a few users: the down projection with its residual
        _linear("linear_7_down", 7, 4096, 14336, residual=True),
        # a decode step of 64 requests: gate and up with the gate in the epilogue, asymmetric weights as compression tools write them
        _linear("linear_64_gate", 64, 28672, 4096, act="swiglu", zero_points=True),
        # a compiled encoder: odd token count and sizes, fp16, bias and gelu
        _linear("linear_197_encoder", 197, 1000, 1333, type="f16", act="gelu_erf", zero_points=True, bias=True),
        # a prompt of ordinary length through the output projection of a large model
        _linear("linear_999_out", 999, 8192, 8192, residual=True),
        # a full prefill step, the largest product of the layer
        _linear("linear_8192_gate", 8192, 28672, 4096, act="swiglu"),
        # one sequence of 37 tokens, head norms, 16-bit floats of the encoder type
        _heads("heads_1x37_f16", 1, 37, 12, 12, 64, type="f16"),
        # four long documents, half of every head rotated, interleaved pairs, far positions
        _heads("heads_4x2048_partial", 4, 2048, 32, 8, 128, rot=64, interleaved=True, first=100000),
        # one token of one sequence
        _append("append_1", 1, 1, 613, 32, 8, 128),
        # a decode step of 64 sequences with conversations behind them
        _append("append_64", 64, 1, 4000, 32, 8, 128),
        # three prompts of odd length, heads of 80, no head norms, the first 32 dimensions rotated
        _append("append_3x333_h80", 3, 333, 0, 16, 4, 80, rot=32, norm=False, theta=10000.0),
        # a full prefill step of a large model in chunks behind earlier tokens
        _append("append_8x1024", 8, 1024, 2048, 64, 8, 128),
    ]


def _log_range(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(("linear", "linear", "linear", "heads", "append"))
    if kind == "linear":
        act = rng.choice(("none", "none", "swiglu", "gelu_erf", "silu"))
        while True:
            T, N, K = _log_range(rng, 1, 8192), _log_range(rng, 128, 28672), _log_range(rng, 128, 14336)
            if act == "swiglu":
                N = max(128, N // 128 * 128)
            if rng.random() < 0.7:
                K = max(64, K // 64 * 64)
            if rng.random() < 0.6:
                N = max(128, N // 128 * 128)
            if T * N * K <= 8192 * 28672 * 4096:
                break
        c = _linear("", T, N, K, type=rng.choice(("bf16", "bf16", "f16")), act=act, norm=rng.random() < 0.4, zero_points=rng.random() < 0.4,
                    bias=act != "swiglu" and rng.random() < 0.4, residual=act == "none" and rng.random() < 0.5)
        c["out32"] = act == "none" and not c["residual"] and rng.random() < 0.2
    else:
        D = rng.choice((64, 64, 80, 96, 128, 128, 128, 256))
        Hkv = rng.choice((1, 2, 4, 8))
        Hq = Hkv * rng.choice((1, 2, 3, 4, 8))
        args = dict(rot=rng.choice((D, D, D // 2 // 8 * 8)), type=rng.choice(("bf16", "f16")), norm=rng.random() < 0.7, interleaved=rng.random() < 0.3,
                    theta=rng.choice((10000.0, 500000.0)))
        tokens = max(1, min(_log_range(rng, 1, 16384), 8192 * 80 * 128 // ((Hq + 2 * Hkv) * D)))
        split = rng.choice((1, 1, 2, 4, 16, tokens))
        split = min(split, tokens)
        if kind == "heads":
            c = _heads("", split, tokens // split, Hq, Hkv, D, first=_log_range(rng, 1, 120000), **args)
        else:
            c = _append("", split, tokens // split, _log_range(rng, 1, 4096), Hq, Hkv, D, **args)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, t, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(t)


def _prepare_linear(c, g):
    T, N, K, t = c["T"], c["N"], c["K"], TYPES[c["type"]]
    s = {}
    # activations of a trained layer: a few channels are far larger than the others
    x = torch.randn((T, K), generator=g, device="cuda")
    loud = torch.rand(K, generator=g, device="cuda") < 0.01
    s["x"] = torch.where(loud, x * 8, x).to(t)
    s["gamma"] = (1 + 0.1 * torch.randn(K, generator=g, device="cuda")).to(t) if c["norm"] else None
    if c["zero_points"]:
        s["w"] = torch.randint(0, 256, (N, K), generator=g, device="cuda", dtype=torch.uint8)
        s["zps"] = torch.randint(112, 145, (N,), generator=g, device="cuda", dtype=torch.uint8)
    else:
        s["w"] = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
        s["zps"] = None
    s["scales"] = ((0.5 + torch.rand(N, generator=g, device="cuda")) * (0.013 / math.sqrt(K))).half()
    s["bias"] = _normal(g, (N,), t, 0.5) if c["bias"] else None
    s["residual"] = _normal(g, (T, N), t) if c["residual"] else None
    if own:                                     # the program's weights, packed when the model is loaded
        from openvino_b200.ops import cuda as K_
        s["packed"] = K_.PackedWeight.from_ir_i8(s["w"], s["scales"], s["zps"], bias=s["bias"])
    return s


def _inv_freq(c):
    rot = c["rot"]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    return (c["theta"] ** (-2.0 * i / rot)).float()


def _prepare_heads(c, g):
    B, S, Hq, Hkv, D, t = c["B"], c["S"], c["Hq"], c["Hkv"], c["D"], TYPES[c["type"]]
    qkv = _normal(g, (B, S, (Hq + 2 * Hkv) * D), t, 2.0)
    s = {"q": qkv[..., :Hq * D].view(B, S, Hq, D), "k": qkv[..., Hq * D:(Hq + Hkv) * D].view(B, S, Hkv, D), "inv_freq": _inv_freq(c)}
    s["positions"] = (torch.randint(0, 64, (B, 1), generator=g, device="cuda") + c["first"] + torch.arange(S, device="cuda")).to(torch.int32)
    for n in ("q_norm", "k_norm"):
        s[n] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(t) if c["norm"] else None
    return s


def _prepare_append(c, g):
    seqs, new, Hq, Hkv, D, t = c["seqs"], c["new"], c["Hq"], c["Hkv"], c["D"], TYPES[c["type"]]
    T = seqs * new
    past = torch.randint(0, c["past"] + 1, (seqs, 1), generator=g, device="cuda")
    s = {"qkv": _normal(g, (T, (Hq + 2 * Hkv) * D), t, 2.0), "inv_freq": _inv_freq(c)}
    s["positions"] = (past + torch.arange(new, device="cuda")).reshape(T).to(torch.int32)
    # the blocks that the new tokens touch, in scattered order; earlier tokens of a first block stay as they are
    per_seq = (BLOCK - 1 + new + BLOCK - 1) // BLOCK
    blocks = seqs * per_seq + 1
    order = torch.randperm(blocks, generator=g, device="cuda")[:seqs * per_seq].reshape(seqs, per_seq)
    at = past % BLOCK + torch.arange(new, device="cuda")
    s["slots"] = (torch.gather(order, 1, at // BLOCK) * BLOCK + at % BLOCK).reshape(T).to(torch.int32)
    for n in ("k_cache", "v_cache"):
        s[n] = _normal(g, (blocks, Hkv, BLOCK, D), t)
    s["q_out"] = torch.empty((T, Hq * D), dtype=t, device="cuda")
    for n in ("q_norm", "k_norm"):
        s[n] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(t) if c["norm"] else None
    return s


def prepare(case, seed):
    g = _gen(seed)
    s = {"linear": _prepare_linear, "heads": _prepare_heads, "append": _prepare_append}[case["kind"]](case, g)
    s["case"] = case
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _quantise(y):
    a = y.abs().amax(1, keepdim=True)
    q = torch.round(y * (torch.full_like(a, 127.0) / a))
    scale = a / torch.full_like(a, 127.0)
    small = a < 2.0 ** -119
    q = torch.where(small, torch.zeros_like(q), q)
    return torch.nan_to_num(q, 0.0), torch.where(small, torch.zeros_like(scale), torch.where(torch.isfinite(a), scale, torch.full_like(scale, math.nan)))


def _act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu_erf":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "swiglu":                          # rows of w: 64 of the gate, then the 64 of the same channels' up projection, and so on
        T, N = v.shape
        v = v.view(T, N // 128, 2, 64)
        return (v[:, :, 0] / (1 + torch.exp(-v[:, :, 0])) * v[:, :, 1]).reshape(T, N // 2)
    return v


def _plain_linear(s):
    c, y = s["case"], s["x"].float()
    if c["norm"]:
        y = y * torch.rsqrt((y * y).mean(1, keepdim=True) + EPS) * s["gamma"].float()
    q, scale = _quantise(y)
    w = s["w"].float()
    if s["zps"] is not None:
        w = w - s["zps"].float().unsqueeze(1)
    v = (q @ w.t()) * (scale * s["scales"].float())
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _act(v, c["act"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v if c["out32"] else v.to(s["x"].dtype)


def _turn(x, angle, rot, interleaved):
    """x [..., heads, D] with one angle per position and pair, [..., rot / 2]."""
    cos, sin = torch.cos(angle).to(x.dtype).unsqueeze(-2), torch.sin(angle).to(x.dtype).unsqueeze(-2)
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _head(x, weight, angle, c):
    y = x.float()
    if weight is not None:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    return _turn(y, angle, c["rot"], c["interleaved"]).to(x.dtype)


def _plain_heads(s):
    c = s["case"]
    angle = s["positions"].double().unsqueeze(-1) * s["inv_freq"].double()      # far positions: 32 bits lose the angle
    return [_head(s["q"], s["q_norm"], angle, c), _head(s["k"], s["k_norm"], angle, c)]


def _plain_append(s):
    c, T = s["case"], s["qkv"].shape[0]
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    rows = s["qkv"].view(T, Hq + 2 * Hkv, D)
    angle = s["positions"].double().unsqueeze(-1) * s["inv_freq"].double()
    s["q_out"].copy_(_head(rows[:, :Hq], s["q_norm"], angle, c).reshape(T, Hq * D))
    block, at = s["slots"].long() // BLOCK, s["slots"].long() % BLOCK
    s["k_cache"][block, :, at] = _head(rows[:, Hq:Hq + Hkv], s["k_norm"], angle, c)
    s["v_cache"][block, :, at] = rows[:, Hq + Hkv:]
    return [s["q_out"], s["k_cache"], s["v_cache"]]


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_linear(s):
    from openvino_b200.ops import cuda as K
    c = s["case"]
    act = {"none": K.ACT_NONE, "silu": K.ACT_SILU, "gelu_erf": K.ACT_GELU_ERF, "swiglu": K.ACT_SWIGLU}[c["act"]]
    return K.gemm(s["x"], s["packed"], act=act, residual=s["residual"], out_f32=c["out32"], norm=(s["gamma"], EPS) if c["norm"] else None)


def _own_heads(s):
    from openvino_b200.ops import cuda as K
    return K.qk_norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, interleaved=s["case"]["interleaved"])


def _own_append(s):
    from openvino_b200.ops import cuda as K
    c = s["case"]
    K.qk_norm_rope_kv_write(s["qkv"], s["positions"], s["slots"], s["k_cache"], s["v_cache"], s["inv_freq"], c["Hq"], c["Hkv"], c["D"], BLOCK,
                            q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, interleaved=c["interleaved"], q_out=s["q_out"])
    return [s["q_out"], s["k_cache"], s["v_cache"]]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"linear": _own_linear, "heads": _own_heads, "append": _own_append}[kind](state)
    return {"linear": _plain_linear, "heads": _plain_heads, "append": _plain_append}[kind](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["kind"] == "linear":
        T, N, K = c["T"], c["N"], c["K"]
        cols = N // 2 if c["act"] == "swiglu" else N
        n = N * K + 2 * N + T * K * 2 + T * cols * (4 if c["out32"] else 2)
        n += (N if c["zero_points"] else 0) + (2 * N if c["bias"] else 0) + (2 * K if c["norm"] else 0) + (2 * T * N if c["residual"] else 0)
        return {"bytes": n, "flops": 2 * T * N * K}
    D, Hq, Hkv = c["D"], c["Hq"], c["Hkv"]
    if c["kind"] == "heads":
        T, moved = c["B"] * c["S"], 2 * (Hq + Hkv) * D * 2
    else:
        T, moved = c["seqs"] * c["new"], 2 * (Hq + 2 * Hkv) * D * 2 + 4
    return {"bytes": T * (moved + 4) + 2 * c["rot"] + (4 * D if c["norm"] else 0), "flops": T * (Hq + Hkv) * ((4 * D if c["norm"] else 0) + 3 * c["rot"])}


# ------------------------------------------------------------------------------------------------ 64 bits, from the definitions
def _exact_linear(c, s):
    x = s["x"].double()
    if c["norm"]:
        x = x / torch.sqrt(x.pow(2).sum(1, keepdim=True) / c["K"] + EPS) * s["gamma"].double()
    top = x.abs().max(1, keepdim=True).values
    codes = torch.round(x * 127.0 / top)                                # inputs of this file have finite rows that are not zero
    weight = s["w"].double() - (0 if s["zps"] is None else s["zps"].double()[:, None])
    v = torch.matmul(codes, weight.T)
    del weight, codes, x
    v *= top / 127.0
    v *= s["scales"].double()[None, :]
    if s["bias"] is not None:
        v += s["bias"].double()
    if c["act"] == "silu":
        v = v * torch.sigmoid(v)
    elif c["act"] == "gelu_erf":
        v = v * 0.5 * torch.erfc(-v / math.sqrt(2.0))
    elif c["act"] == "swiglu":
        tiles = v.reshape(c["T"], -1, 128)
        v = (tiles[..., :64] * torch.sigmoid(tiles[..., :64]) * tiles[..., 64:]).reshape(c["T"], -1)
    if s["residual"] is not None:
        v = v + s["residual"].double()
    return v


def _exact_heads(rows, weight, pos, freq, c):
    """rows [tokens, heads, D]: as complex numbers, one for each pair of dimensions."""
    y = rows.double()
    if weight is not None:
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / c["D"] + EPS) * weight.double()
    rot = c["rot"]
    pairs = y[..., :rot].reshape(*y.shape[:-1], rot // 2, 2) if c["interleaved"] else torch.stack([y[..., :rot // 2], y[..., rot // 2:rot]], -1)
    theta = pos.double()[:, None] * freq.double()[None, :]
    z = torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(theta), theta)[:, None, :]
    out = y.clone()
    if c["interleaved"]:
        out[..., 0:rot:2], out[..., 1:rot:2] = z.real, z.imag
    else:
        out[..., :rot // 2], out[..., rot // 2:rot] = z.real, z.imag
    return out


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "linear":
        return _exact_linear(c, s)
    D, Hq, Hkv = c["D"], c["Hq"], c["Hkv"]
    if c["kind"] == "heads":
        B, S = c["B"], c["S"]
        pos = s["positions"].reshape(-1)
        return [_exact_heads(s[n].reshape(B * S, H, D), s[n + "_norm"], pos, s["inv_freq"], c).reshape(B, S, H, D) for n, H in (("q", Hq), ("k", Hkv))]
    T = c["seqs"] * c["new"]
    q, k, v = s["qkv"].reshape(T, -1).split([Hq * D, Hkv * D, Hkv * D], 1)
    q = _exact_heads(q.reshape(T, Hq, D), s["q_norm"], s["positions"], s["inv_freq"], c)
    k = _exact_heads(k.reshape(T, Hkv, D), s["k_norm"], s["positions"], s["inv_freq"], c)
    caches = []
    for cache, new in ((s["k_cache"], k), (s["v_cache"], v.reshape(T, Hkv, D).double())):
        flat = cache.double().transpose(1, 2).reshape(-1, Hkv, D).index_copy(0, s["slots"].long(), new)
        caches.append(flat.reshape(-1, BLOCK, Hkv, D).transpose(1, 2))
    return [q.reshape(T, Hq * D)] + caches
