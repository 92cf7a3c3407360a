"""Cases of the decoder-layer operators around the attention: RMS norm with residual and 8-bit
output, matrix product with a fused epilogue, rotary positions.

``own`` chooses who computes: elementary torch operations in 32 bits, or the package's kernels.
Sizes are those of this repository's configurations (hidden 1024, qkv 4096, vocabulary 151,936;
hidden 4096 with 32 / 8 heads and an MLP of 12,288) and generic odd ones around them.
"""

import math

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
TINY = 1e-12            # floor of a row's largest magnitude before it becomes a scale
EPS = 1e-6
BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
MAX_FLOPS = 2.0 * 4096 * 4096 * 24576      # the largest listed product
MAX_ELEMS = 8192 * 12288                   # the largest listed norm / quantisation
MAX_ROT = 16384 * 40 * 128                 # the largest listed rotation


def listed():
    norm = dict(op="norm", residual=True, norm=True, fp8=False)
    lin = dict(op="linear", bias=False, act="none", gated=False, residual=False, fp8=False)
    rot = dict(op="rotary", layout="half", scaling="none", factor=1.0, base=1e6)
    return [
        # one sequence's next token through the norm before a projection: latency alone
        dict(norm, name="norm_token", rows=1, hidden=1024),
        # a prefill of 8,192 tokens, hidden 4096, feeding an 8-bit projection
        dict(norm, name="norm_fp8_prefill", rows=8192, hidden=4096, fp8=True),
        # a ragged batch with an odd width: no 16-byte alignment anywhere
        dict(norm, name="norm_fp8_odd", rows=999, hidden=1537, fp8=True),
        # the MLP's 12,288 activations to 8 bits before the down projection
        dict(norm, name="quantize_mlp", rows=8192, hidden=12288, fp8=True, norm=False, residual=False),
        # qkv projection of one decode step of 8 requests, with bias
        dict(lin, name="qkv_decode", m=8, k=1024, n=4096, bias=True),
        # MLP down projection of a 64-request decode step in 8 bits, onto the residual
        dict(lin, name="down_decode_fp8", m=64, k=12288, n=4096, residual=True, fp8=True),
        # odd and ragged: tokens, inputs and outputs that fill no tile
        dict(lin, name="linear_odd", m=333, k=1000, n=1531, bias=True, act="gelu_tanh", residual=True),
        # the vocabulary's logits for a 256-request step
        dict(lin, name="lm_head", m=256, k=1024, n=151936),
        # gated MLP of a 4,096-token prefill, both types
        dict(lin, name="gated_prefill", m=4096, k=4096, n=12288, act="silu", gated=True),
        dict(lin, name="gated_prefill_fp8", m=4096, k=4096, n=12288, act="silu", gated=True, fp8=True),
        # one decode step of 64 requests far into a long context, scaled frequencies
        dict(rot, name="rotary_decode", tokens=64, heads=32, kv_heads=8, dim=128, rotary_dim=128,
             far=131072, scaling="yarn", factor=4.0),
        # a prefill of 16,384 tokens, interleaved pairs on half of the head
        dict(rot, name="rotary_prefill", tokens=16384, heads=32, kv_heads=8, dim=128, rotary_dim=64,
             far=16384, layout="interleaved"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "linear", "linear", "rotary"])
    if op == "norm":
        hidden = _log(rng, 64, 12288)
        if rng.random() < 0.6:
            hidden = max(64, hidden // 64 * 64)
        rows = _log(rng, 1, min(8192, MAX_ELEMS // hidden))
        norm = rng.random() < 0.75
        return dict(op=op, rows=rows, hidden=hidden, norm=norm, residual=norm and rng.random() < 0.7,
                    fp8=not norm or rng.random() < 0.5)
    if op == "linear":
        fp8, gated = rng.random() < 0.4, rng.random() < 0.35
        k = _log(rng, 128, 12288)
        n = _log(rng, 64, 16384)
        if rng.random() < 0.75:
            k = k // 64 * 64
        if rng.random() < 0.6:
            n = n // 16 * 16
        m = _log(rng, 1, max(1, min(8192, int(MAX_FLOPS / (2.0 * k * n * (2 if gated else 1))))))
        return dict(op=op, m=m, k=k, n=n, bias=rng.random() < 0.4, gated=gated, fp8=fp8,
                    act=rng.choice(["silu", "gelu", "gelu_tanh"] if gated else
                                   ["none", "none", "relu", "silu", "gelu", "gelu_tanh"]),
                    residual=rng.random() < 0.4)
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    rotary_dim = dim if rng.random() < 0.5 else 2 * rng.randint(4, dim // 2)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5])
    tokens = _log(rng, 1, max(1, min(16384, MAX_ROT // ((heads + kv_heads) * dim))))
    scaling = rng.choice(["none", "linear", "yarn", "bands"])
    return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary_dim=rotary_dim,
                far=max(tokens, _log(rng, 1024, 131072)), layout=rng.choice(["half", "interleaved"]),
                scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]),
                base=rng.choice([1e4, 1e6]))


# ---------------------------------------------------------------- inputs

#: context length that scaled frequencies were trained for, and the band edges in turns over it
TRAINED, BAND_LOW, BAND_HIGH, YARN_SLOW, YARN_FAST = 32768, 1.0, 4.0, 1.0, 32.0


def _quantised(x):
    scale = x.abs().amax(-1).clamp_min(TINY) / E4M3_MAX
    return (x / scale[:, None]).to(FP8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda") * std

    s = {"case": case}
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        x = randn(rows, hidden)
        x[:, :: max(1, hidden // 7)] *= 12.0          # a few channels stand out, as in trained models
        s["x"] = x.to(BF16)
        s["residual"] = randn(rows, hidden, std=3.0).to(BF16) if case["residual"] else None
        s["weight"] = (1 + randn(hidden, std=0.2)).to(BF16)
    elif case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        wide = 2 * n if case["gated"] else n
        x, w = randn(m, k), randn(wide, k, std=k ** -0.5)
        s["x_scale"] = s["w_scale"] = None
        if case["fp8"]:
            s["x"], s["x_scale"] = _quantised(x)
            s["w"], s["w_scale"] = _quantised(w)
        else:
            s["x"], s["w"] = x.to(BF16), w.to(BF16)
        del x, w
        s["bias"] = randn(wide, std=0.5).to(BF16) if case["bias"] else None
        s["residual"] = randn(m, n).to(BF16) if case["residual"] else None
    else:
        t, far = case["tokens"], case["far"]
        s["q"] = randn(t, case["heads"], case["dim"]).to(BF16)
        s["k"] = randn(t, case["kv_heads"], case["dim"]).to(BF16)
        if t >= far // 2:                              # one long prompt from its start
            s["positions"] = torch.arange(t, device="cuda")
        else:                                          # requests anywhere in their contexts
            s["positions"] = torch.randint(0, far, (t,), generator=g, device="cuda")
        if own:
            from qwen3_engine_from_scratch_b200 import RotaryPlan
            kind = case["scaling"]
            more = {"none": {}, "linear": dict(factor=case["factor"]),
                    "yarn": dict(factor=case["factor"], original_len=TRAINED,
                                 slow_turns=YARN_SLOW, fast_turns=YARN_FAST),
                    "bands": dict(factor=case["factor"], original_len=TRAINED,
                                  slow_turns=BAND_LOW, fast_turns=BAND_HIGH)}[kind]
            s["plan"] = RotaryPlan(case["rotary_dim"], base=case["base"], layout=case["layout"],
                                   scaling=None if kind == "none" else kind, device="cuda", **more)
        else:
            s["freq"], s["gain"] = _frequencies(case)
    return s


def _frequencies(case):
    """The plain form's angle a position for each pair, in 32 bits, and the factor on cos and sin."""
    r, factor = case["rotary_dim"], case["factor"]
    i = torch.arange(0, r, 2, dtype=torch.float64, device="cuda")
    f = case["base"] ** (-i / r)
    gain, turns = 1.0, TRAINED * f / (2 * math.pi)
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "bands":
        keep = ((turns - BAND_LOW) / (BAND_HIGH - BAND_LOW)).clamp(0, 1)
        f = f * (keep + (1 - keep) / factor)
    elif case["scaling"] == "yarn":
        # the ramp runs over the pair's index, between those that turn YARN_FAST and YARN_SLOW times
        at = lambda n: r * math.log(TRAINED / (2 * math.pi * n)) / (2 * math.log(case["base"]))
        lo, hi = max(math.floor(at(YARN_FAST)), 0), min(math.ceil(at(YARN_SLOW)), r // 2 - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        gain = 0.1 * math.log(factor) + 1.0
    return f.float(), gain


# ---------------------------------------------------------------- one pass


def run(s):
    return {"norm": _norm, "linear": _linear, "rotary": _rotary}[s["case"]["op"]](s)


def _norm(s):
    c, x, r, w = s["case"], s["x"], s["residual"], s["weight"]
    if own:
        import qwen3_engine_from_scratch_b200 as qb
        if not c["norm"]:
            return qb.quantize_rows_fp8(x)
        if c["fp8"]:
            return qb.rms_norm_fp8(x, w, residual=r, eps=EPS)
        return qb.rms_norm(x, w, residual=r, eps=EPS)
    h = x.float() if r is None else x.float() + r.float()
    y = h
    if c["norm"]:
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS) * w.float()
    added = () if r is None else (h.to(BF16),)
    if not c["fp8"]:
        return (y.to(BF16), *added) if added else y.to(BF16)
    scale = y.abs().amax(-1).clamp_min(TINY) / E4M3_MAX
    return ((y / scale[:, None]).to(FP8), scale, *added)


def _activated(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _linear(s):
    c = s["case"]
    if own:
        import qwen3_engine_from_scratch_b200 as qb
        return qb.linear(s["x"], s["w"], bias=s["bias"], activation=c["act"], gated=c["gated"],
                         residual=s["residual"], x_scale=s["x_scale"], weight_scale=s["w_scale"])
    y = s["x"].float() @ s["w"].float().t()
    if c["fp8"]:
        y = y * s["x_scale"][:, None] * s["w_scale"]
    if c["bias"]:
        y = y + s["bias"].float()
    if c["gated"]:
        y = _activated(y[:, :c["n"]], c["act"]) * y[:, c["n"]:]
    else:
        y = _activated(y, c["act"])
    if c["residual"]:
        y = y + s["residual"].float()
    return y.to(BF16)


def _rotary(s):
    c = s["case"]
    if own:
        import qwen3_engine_from_scratch_b200 as qb
        return qb.rotary(s["q"], s["k"], s["positions"], s["plan"])
    angle = s["positions"].float()[:, None, None] * s["freq"]
    cos, sin = angle.cos() * s["gain"], angle.sin() * s["gain"]
    return _turned(s["q"], cos, sin, c), _turned(s["k"], cos, sin, c)


def _turned(x, cos, sin, c):
    r = c["rotary_dim"]
    out = x.float()
    if c["layout"] == "half":
        a, b = out[..., :r // 2], out[..., r // 2:r]
        a, b = a * cos - b * sin, b * cos + a * sin
        out = torch.cat((a, b, out[..., r:]), -1)
    else:
        a, b = out[..., 0:r:2], out[..., 1:r:2]
        a, b = a * cos - b * sin, b * cos + a * sin
        out = torch.cat((torch.stack((a, b), -1).flatten(-2), out[..., r:]), -1)
    return out.to(BF16)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        b = n * 2 + n * (1 if case["fp8"] else 2) + (case["rows"] * 4 if case["fp8"] else 0)
        b += n * 4 if case["residual"] else 0
        b += case["hidden"] * 2 if case["norm"] else 0
        return {"bytes": b, "flops": n * 6}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        wide, size = (2 * n if case["gated"] else n), (1 if case["fp8"] else 2)
        b = (m + wide) * k * size + m * n * 2
        b += (m + wide) * 4 if case["fp8"] else 0
        b += wide * 2 if case["bias"] else 0
        b += m * n * 2 if case["residual"] else 0
        return {"bytes": b, "flops": 2.0 * m * k * wide}
    n = case["tokens"] * (case["heads"] + case["kv_heads"])
    return {"bytes": n * case["dim"] * 4 + case["tokens"] * 8, "flops": n * case["rotary_dim"] * 3}


# ---------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        y = s["x"].double()
        h = None
        if case["residual"]:
            y = h = y + s["residual"].double()
        if case["norm"]:
            y = y / (y.pow(2).sum(-1, keepdim=True) / case["hidden"] + EPS).sqrt() * s["weight"].double()
        tail = () if h is None else (h,)
        if not case["fp8"]:
            return (y, *tail) if tail else y
        top = y.abs().max(-1).values.clamp(min=TINY)
        return (y * (E4M3_MAX / top)[:, None], top / E4M3_MAX, *tail)
    if case["op"] == "linear":
        n = case["n"]
        rows = max(1, (1 << 28) // max(1, s["w"].shape[0]))
        x, w = s["x"].double(), s["w"].double()
        if case["fp8"]:
            x, w = x * s["x_scale"].double()[:, None], w * s["w_scale"].double()[:, None]
        parts = []
        for at in range(0, case["m"], rows):
            v = torch.nn.functional.linear(x[at:at + rows], w, s["bias"].double() if case["bias"] else None)
            gate = v[:, :n]
            if case["act"] == "relu":
                gate = gate.relu()
            elif case["act"] == "silu":
                gate = gate * gate.sigmoid()
            elif case["act"] == "gelu":
                gate = gate * torch.special.ndtr(gate)
            elif case["act"] == "gelu_tanh":     # tanh(z) = 1 - 2 / (exp(2 z) + 1)
                z = (2 / math.pi) ** 0.5 * (gate + 0.044715 * gate.pow(3))
                gate = gate * (1 - 1 / (torch.exp(2 * z) + 1))
            if case["gated"]:
                gate = gate * v[:, n:]
            if case["residual"]:
                gate = gate + s["residual"][at:at + rows].double()
            parts.append(gate)
        return torch.cat(parts)
    half, factor = case["rotary_dim"] // 2, case["factor"]
    freq, gain = np.empty(half), 1.0
    for i in range(half):
        wave = 2 * np.pi * case["base"] ** (2 * i / case["rotary_dim"])      # positions a turn
        stretched = wave * factor
        if case["scaling"] == "none":
            pass
        elif case["scaling"] == "linear":
            wave = stretched
        elif case["scaling"] == "bands":
            if TRAINED / wave <= BAND_LOW:
                wave = stretched
            elif TRAINED / wave < BAND_HIGH:
                a = (TRAINED / wave - BAND_LOW) / (BAND_HIGH - BAND_LOW)
                wave = 1 / ((1 - a) / stretched + a / wave)
        else:
            edges = [case["rotary_dim"] * np.log(TRAINED / (t * 2 * np.pi)) / (2 * np.log(case["base"]))
                     for t in (YARN_FAST, YARN_SLOW)]
            first, last = max(np.floor(edges[0]), 0), min(np.ceil(edges[1]), half - 1)
            a = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
            wave = 1 / ((1 - a) / wave + a / stretched)
            gain = 1 + np.log(factor) / 10
        freq[i] = 2 * np.pi / wave
    angle = s["positions"].double()[:, None] * torch.from_numpy(freq).cuda()
    turn = torch.polar(torch.full_like(angle, gain), angle)[:, None]          # complex rotation
    outs = []
    for x in (s["q"].double(), s["k"].double()):
        part = x[..., :2 * half]
        pairs = (part.unflatten(-1, (2, half)).transpose(-1, -2) if case["layout"] == "half"
                 else part.unflatten(-1, (half, 2)))
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        pairs = pairs.transpose(-1, -2) if case["layout"] == "half" else pairs
        outs.append(torch.cat((pairs.flatten(-2), x[..., 2 * half:]), -1))
    return tuple(outs)
