"""RMS norm (bf16 and 8-bit output), matrix product with its epilogue and rotary
positions on the GPU, against their definitions in 64 bits.

Tolerances, from the number formats:
* a bf16 result: half a unit in the last place, 2^-8 of the result, and 2 % more
  for the fp32 arithmetic in front of the rounding;
* an e4m3 value times its scale: half a unit, 2^-4 of the value, or half the
  smallest subnormal, 2^-10 of the scale; the scale itself 2^-20;
* a product's accumulator: one fp32 rounding (2^-23, truncation included) of the
  running sum an instruction of 32 bytes of K and one for each partial sum, each
  at most the sum of |x w|; the activations' slopes are at most 1.13, and their
  fp32 forms are good to 2^-19 of their argument and value;
* a rotation: 2^-20 of |a| + |b| for the angle (2^-31 turns) and the fp32 sine.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn
HALF_ULP = 2.0 ** -8 * 1.02          # bf16 keeps 8 significant bits


@pytest.fixture(scope="module")
def qb(cuda, native_lib):
    import qwen3_engine_from_scratch_b200 as m
    m.clear_device_status()
    yield m
    m.check_device_status()


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _place(t, how):
    """The same values with other strides: padded rows, or a base off 16 bytes."""
    if how == "plain":
        return t
    rows, n = t.shape
    pad = {"padded": 16, "odd": 3}[how]
    store = torch.empty(rows * (n + pad) + 8, dtype=torch.uint8 if t.dtype == FP8 else t.dtype,
                        device=t.device).view(t.dtype)
    view = store[(0 if how == "padded" else 1):].as_strided((rows, n), (n + pad, 1))
    view.copy_(t)
    return view


# ---------------------------------------------------------------- norm

NORM_SIZES = [(1, 1), (1, 7), (3, 8), (5, 31), (2, 32), (300, 128), (7, 1000), (9, 1024),
              (4, 1537), (65, 2048), (3, 4096), (2, 8200), (2, 9001), (2, 12288), (2, 32776),
              # many wide rows: the streaming form, every number of CTAs an SM
              (700, 2048), (1300, 4104), (700, 5120), (640, 8192), (3001, 12288), (640, 16384)]


def _norm_exact(x, w, r, eps):
    h = x.double() if r is None else x.double() + r.double()
    y = h if w is None else h / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return y, h


def _check_bf16(got, want):
    err = (got.double() - want).abs()
    assert got.dtype == BF16 and got.shape == want.shape
    assert (err <= HALF_ULP * want.abs() + 1e-37).all(), float((err / want.abs().clamp_min(1e-30)).max())


def _check_fp8(q, scale, want):
    assert q.dtype == FP8 and scale.dtype == torch.float32 and scale.shape == want.shape[:-1]
    s = want.abs().amax(-1).clamp_min(1e-12) / 448
    assert ((scale.double() - s).abs() <= 2.0 ** -20 * s).all()
    err = (q.double() * scale.double()[..., None] - want).abs()
    assert (err <= 1.02 * (2.0 ** -4 * want.abs() + 2.0 ** -10 * s[..., None])).all()


@pytest.mark.parametrize("rows,hidden", NORM_SIZES)
@pytest.mark.parametrize("how", ["plain", "padded", "odd"])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(qb, rows, hidden, how, residual):
    g = _gen(rows * 7919 + hidden)
    x = _place(_randn(g, rows, hidden, std=2.0).to(BF16), how)
    r = _place(_randn(g, rows, hidden, std=3.0).to(BF16), how) if residual else None
    w = (1 + _randn(g, hidden, std=0.3)).to(BF16)
    want, h = _norm_exact(x, w, r, 1e-5)
    got = qb.rms_norm(x, w, residual=r, eps=1e-5)
    _check_bf16(got[0] if residual else got, want)
    q = qb.rms_norm_fp8(x, w, residual=r, eps=1e-5)
    _check_fp8(q[0], q[1], want)
    if residual:
        _check_bf16(got[1], h)
        assert torch.equal(got[1], q[2])
    else:
        _check_fp8(*qb.quantize_rows_fp8(x), x.double())


def test_norm_in_place_and_batched(qb):
    g = _gen(3)
    x, r = _randn(g, 2, 5, 264).to(BF16), _randn(g, 2, 5, 264).to(BF16)
    w = (1 + _randn(g, 264, std=0.3)).to(BF16)
    want = qb.rms_norm(x, w, residual=r)
    r2, x2 = r.clone(), x.clone()
    y, h = qb.rms_norm(x2, w, residual=r2, out=x2, residual_out=r2)
    assert y.data_ptr() == x2.data_ptr() and h.data_ptr() == r2.data_ptr()
    assert torch.equal(x2, want[0]) and torch.equal(r2, want[1])
    q, s, _ = qb.rms_norm_fp8(x, w, residual=r)
    assert q.shape == x.shape and s.shape == (2, 5)
    # wide rows that are read twice, and streamed ones, in place
    for rows, hidden in ((2, 40000), (1000, 4096)):
        x, r = _randn(g, rows, hidden).to(BF16), _randn(g, rows, hidden).to(BF16)
        w = torch.ones(hidden, dtype=BF16, device="cuda")
        want, h = _norm_exact(x, w, r, 1e-6)
        y, h2 = qb.rms_norm(x, w, residual=r, residual_out=r)
        _check_bf16(y, want)
        _check_bf16(h2, h)


def test_norm_special_rows(qb):
    """Zero rows, NaN and infinities: what the definition gives, row by row."""
    for rows, wide, size in ((6, 520, 520), (6, 520, 519), (800, 4096, 4096)):
        # vectors, single elements, streamed rows
        x = _randn(_gen(5), rows, wide).to(BF16)
        x[1] = 0
        x[2, 17] = float("nan")
        x[3, wide - 1] = float("inf")
        x[4] *= 1e-30
        w = torch.ones(wide, dtype=BF16, device="cuda")
        xs, ws = x[:, -size:], w[-size:]
        y = qb.rms_norm(xs, ws)
        want, _ = _norm_exact(xs, ws, None, 1e-6)
        for row in (0, 1, 4, 5):
            _check_bf16(y[row], want[row])
        assert y[2].isnan().all()
        assert y[3].isnan().sum() == 1 and (y[3, :-1] == 0).all()
        q, s = qb.quantize_rows_fp8(xs)
        assert s[1] == torch.tensor(1e-12, dtype=torch.float32) / 448 and (q[1].float() == 0).all()
        assert s[2].isnan() and q[2].float().isnan().all()
        assert s[3].isinf() and q[3, -1].float().isnan() and (q[3, :-1].float() == 0).all()
        for row in (0, 4, 5):
            _check_fp8(q[row], s[row], xs[row].double())


def test_norm_empty_and_refusals(qb):
    w = torch.ones(16, dtype=BF16, device="cuda")
    assert qb.rms_norm(torch.empty(0, 16, dtype=BF16, device="cuda"), w).shape == (0, 16)
    x = torch.ones(2, 16, dtype=BF16, device="cuda")
    for bad in (lambda: qb.rms_norm(x.float(), w), lambda: qb.rms_norm(x, w[:15]),
                lambda: qb.rms_norm(x, w, residual=x[:1]), lambda: qb.rms_norm(x.cpu(), w),
                lambda: qb.rms_norm(x, w, residual_out=x),
                lambda: qb.rms_norm(x, w, out=x.float()),
                lambda: qb.rms_norm(torch.ones(2, 0, dtype=BF16, device="cuda"), w[:0]),
                lambda: qb.rms_norm(x, w, out=x[:1].expand(2, 16))):
        with pytest.raises(AssertionError):
            bad()


# ---------------------------------------------------------------- product

def _act(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * 0.5 * torch.special.erfc(-v / math.sqrt(2))
    if act == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def _product(g, m, k, n, fp8=False, gated=False, bias=False, residual=False, how="plain"):
    wide = 2 * n if gated else n
    x, w = _randn(g, m, k), _randn(g, wide, k, std=k ** -0.5)
    a = dict(x_scale=None, weight_scale=None, bias=None, residual=None)
    if fp8:
        a["x_scale"] = torch.rand(m, generator=g, device="cuda") + 0.5
        a["weight_scale"] = torch.rand(wide, generator=g, device="cuda") + 0.5
        x, w = (x * 8).to(FP8), (w * 8).to(FP8)
    else:
        x, w = x.to(BF16), w.to(BF16)
    a["x"], a["weight"] = _place(x, how), _place(w, how)
    if bias:
        a["bias"] = _randn(g, wide).to(BF16)
    if residual:
        a["residual"] = _place(_randn(g, m, n).to(BF16), how)
    return a


def _check_product(got, a, act, gated):
    x, w = a["x"].double(), a["weight"].double()
    v, size = x @ w.t(), x.abs() @ w.abs().t()
    if a["x_scale"] is not None:
        s = a["x_scale"].double()[:, None] * a["weight_scale"].double()
        v, size = v * s, size * s
    if a["bias"] is not None:
        v, size = v + a["bias"].double(), size + a["bias"].double().abs()
    steps = x.shape[1] * a["x"].element_size() / 32 + 12
    err = size * steps * 2.0 ** -23
    if gated:
        n = v.shape[1] // 2
        gate, up = v[:, :n], v[:, n:]
        out = _act(gate, act) * up
        fast = 2.0 ** -19 * (gate.abs() + 1)
        err = (1.13 * err[:, :n] + fast) * up.abs() + _act(gate, act).abs() * err[:, n:] + \
            1.13 * err[:, :n] * err[:, n:]
    else:
        out = _act(v, act)
        err = 1.13 * err + (0 if act == "none" else 2.0 ** -19 * (v.abs() + 1))
    if a["residual"] is not None:
        out = out + a["residual"].double()
        err = err + 2.0 ** -23 * out.abs()
    assert got.dtype == BF16 and got.shape == out.shape
    off = (got.double() - out).abs() - (HALF_ULP * out.abs() + 1.02 * err)
    assert (off <= 0).all(), (float(off.max()), int((off > 0).sum()))


PRODUCT_SIZES = [(1, 8, 1), (1, 64, 128), (1, 1000, 257), (2, 16, 3), (5, 1024, 384), (8, 1024, 4096),
                 (31, 136, 100), (33, 200, 129), (64, 4096, 1024), (65, 512, 640), (127, 768, 96),
                 (129, 320, 130), (200, 1001, 77), (257, 264, 1000), (300, 2048, 2050), (1, 12288, 16),
                 (17, 20000, 65), (511, 65, 511),
                 # enough tiles for pairs of CTAs: an odd number of weight tiles, ragged ends
                 (257, 128, 9500), (600, 192, 6400), (1000, 72, 4999), (2049, 1024, 2048),
                 # few tokens with a long K, and more weight than the direct kernel takes
                 (8, 5001, 300), (7, 4104, 64), (13, 12288, 1024)]


@pytest.mark.parametrize("m,k,n", PRODUCT_SIZES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("gated", [False, True])
def test_product_sizes(qb, m, k, n, fp8, gated):
    g = _gen(m * 31 + k * 7 + n)
    a = _product(g, m, k, n, fp8, gated, bias=n % 2 == 1, residual=m % 2 == 1)
    act = "silu" if gated else "none"
    _check_product(qb.linear(activation=act, gated=gated, **a), a, act, gated)


@pytest.mark.parametrize("m,k,n", [(25, 6208, 80256), (49, 1216, 3456), (22, 4800, 1536), (240, 11712, 128),
                                   (3202, 896, 128), (123, 11520, 1152), (42, 23680, 1536), (7854, 8640, 128),
                                   (252, 19008, 2176), (1364, 64, 51328), (200, 22656, 4352), (1247, 20608, 256),
                                   (1627, 832, 2176), (1300, 2944, 8704)])
def test_product_cuts(qb, m, k, n):
    """A shape for every cut the cost model takes: tiles of 32 to 256 tokens, K split
    2 to 8 ways, pairs of CTAs with and without a split."""
    a = _product(_gen(m + n), m, k, n, residual=True)
    got = qb.linear(activation="silu", **a)
    at = torch.arange(0, n, max(1, n // 2500), device="cuda")        # the reference: some columns of the wide ones
    part = dict(a, weight=a["weight"][at], residual=a["residual"][:, at])
    _check_product(got[:, at], part, "silu", False)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("m,k,n", [(3, 256, 160), (150, 200, 99), (600, 128, 512)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("fp8", [False, True])
def test_product_epilogue(qb, act, m, k, n, gated, fp8):
    a = _product(_gen(m + k), m, k, n, fp8, gated, bias=True, residual=True)
    _check_product(qb.linear(activation=act, gated=gated, **a), a, act, gated)


@pytest.mark.parametrize("how", ["padded", "odd"])
@pytest.mark.parametrize("m,k,n", [(1, 96, 40), (4, 96, 41), (70, 513, 33), (140, 256, 64), (8, 4999, 129),
                                   (16, 333, 600), (9, 77, 17), (300, 1031, 257)])
@pytest.mark.parametrize("fp8", [False, True])
def test_product_strides(qb, how, m, k, n, fp8):
    a = _product(_gen(m + n), m, k, n, fp8, False, bias=True, residual=True, how=how)
    _check_product(qb.linear(**a), a, "none", False)
    out = _place(torch.zeros(m, n, dtype=BF16, device="cuda"), how)
    assert qb.linear(out=out, **a) is out
    _check_product(out, a, "none", False)


def test_product_writes_its_output_only(qb):
    """Neighbouring memory of a strided result keeps its values, and a result may be its residual."""
    for m, k, n in ((3, 64, 63), (130, 64, 130), (40, 4096, 128)):
        a = _product(_gen(m), m, k, n, residual=True)
        store = torch.full((m + 2, n + 6), 7.0, dtype=BF16, device="cuda")
        out = store[1:m + 1, 4:n + 4]
        out.copy_(a["residual"])
        want = qb.linear(**a)
        a["residual"] = out
        qb.linear(out=out, **a)
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert (store == 7.0).all()


def test_product_repeats_bit_for_bit(qb):
    """Sums in a fixed order: also where the CTAs of a cluster share a tile."""
    for m, k, n in ((4, 8192, 256), (64, 4096, 512), (300, 1024, 1024)):
        a = _product(_gen(k), m, k, n)
        first = qb.linear(**a)
        assert all(torch.equal(first, qb.linear(**a)) for _ in range(20))


def test_product_rows_do_not_mix(qb):
    """An infinity or NaN of one token or output channel stays in its row or column."""
    for m in (5, 100, 300):
        a = _product(_gen(m), m, 256, 384)
        want = qb.linear(**a)
        a["x"][2, 100] = float("nan")
        a["weight"][77, 5] = float("inf")
        got = qb.linear(**a)
        assert got[2].isnan().all() and not got[:2, 77].isfinite().any()
        keep = torch.ones_like(got, dtype=torch.bool)
        keep[2], keep[:, 77] = False, False
        assert torch.equal(got[keep], want[keep])


def test_product_leading_dimensions_streams_and_graph(qb):
    a = _product(_gen(9), 12, 128, 64, fp8=True)
    flat = qb.linear(**a)
    b = dict(a, x=a["x"].view(3, 4, 128), x_scale=a["x_scale"].view(3, 4))
    assert torch.equal(qb.linear(**b).view(12, 64), flat)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = qb.linear(**a)
    side.synchronize()
    assert torch.equal(again, flat)
    out = torch.zeros_like(flat)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qb.linear(out=out, **a)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, flat)


def test_product_waits_for_the_host_after_a_timeout(qb):
    """With a timeout on record the pipelined product starts nothing; cleared, it works."""
    a = _product(_gen(1), 100, 256, 256)
    want = qb.linear(**a)
    out = torch.full_like(want, 3.0)
    qb.ops._status[torch.cuda.current_device()].fill_(0x10)       # B200_DEV_TIMEOUT
    qb.linear(out=out, **a)
    with pytest.raises(RuntimeError, match="timed out"):
        qb.check_device_status()
    assert (out == 3.0).all()
    qb.clear_device_status()
    assert torch.equal(qb.linear(out=out, **a), want)
    qb.check_device_status()


def test_product_empty_and_refusals(qb):
    x = torch.ones(2, 32, dtype=BF16, device="cuda")
    w = torch.ones(6, 32, dtype=BF16, device="cuda")
    s2, s6 = torch.ones(2, device="cuda"), torch.ones(6, device="cuda")
    assert qb.linear(x[:0], w).shape == (0, 6)
    for bad in (lambda: qb.linear(x, w.float()), lambda: qb.linear(x.float(), w.float()),
                lambda: qb.linear(x, w[:, :31]), lambda: qb.linear(x, w[:5], gated=True),
                lambda: qb.linear(x, w, bias=w[0]), lambda: qb.linear(x, w, residual=x),
                lambda: qb.linear(x, w, activation="swish"), lambda: qb.linear(x, w, x_scale=s2),
                lambda: qb.linear(x.to(FP8), w.to(FP8)), lambda: qb.linear(x[:, :0], w[:, :0]),
                lambda: qb.linear(x.to(FP8), w.to(FP8), x_scale=s6, weight_scale=s6),
                lambda: qb.linear(x.to(FP8), w.to(FP8), x_scale=s2.half(), weight_scale=s6),
                lambda: qb.linear(x.cpu(), w), lambda: qb.linear(x, w.cpu()),
                lambda: qb.linear(x, w, out=torch.empty(2, 6, device="cuda"))):
        with pytest.raises(AssertionError):
            bad()


# ---------------------------------------------------------------- rotary

def _turned(x, positions, plan):
    """x (T, H, D) in 64 bits by the plan's float64 frequencies."""
    r = plan.rotary_dim
    f = torch.tensor(plan.freq, dtype=torch.float64, device="cuda")
    t = positions.double()[:, None, None] * f
    c, s = t.cos() * plan.gain, t.sin() * plan.gain
    x = x.double()
    out = x.clone()
    i, j = (slice(0, r // 2), slice(r // 2, r)) if plan.layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., i], x[..., j]
    out[..., i], out[..., j] = a * c - b * s, b * c + a * s
    size = torch.zeros_like(x)
    size[..., i] = size[..., j] = (a.abs() + b.abs()) * plan.gain
    return out, size


def _check_turned(got, x, positions, plan):
    want, size = _turned(x, positions, plan)
    err = (got.double() - want).abs()
    # the float64 angle itself is good to position * f * 2^-52
    assert (err <= HALF_ULP * want.abs() + 2.0 ** -20 * size).all(), float(err.max())
    r = plan.rotary_dim
    assert torch.equal(got[..., r:], x[..., r:])


SCALED = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=2.0),
          dict(scaling="bands", factor=8.0, original_len=8192, slow_turns=1.0, fast_turns=4.0),
          dict(scaling="yarn", factor=4.0, original_len=32768)]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary_dim", [(128, 128), (128, 64), (96, 96), (80, 32), (64, 6), (33, 32),
                                            (256, 256), (2, 2), (48, 16)])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 1, 1), (3, 16, 8), (70, 5, 2), (2500, 8, 1)])
def test_rotary(qb, layout, dim, rotary_dim, tokens, heads, kv_heads):
    g = _gen(tokens * dim + rotary_dim)
    more = SCALED[(tokens + dim // 16 + rotary_dim // 2) % len(SCALED)]
    if rotary_dim < 4:
        more = {}
    plan = qb.RotaryPlan(rotary_dim, base=1e6, layout=layout, **more)
    q, k = _randn(g, tokens, heads, dim).to(BF16), _randn(g, tokens, kv_heads, dim).to(BF16)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda")
    for p in (positions, positions.int()):
        q2, k2 = qb.rotary(q, k, p, plan)
        _check_turned(q2, q, positions, plan)
        _check_turned(k2, k, positions, plan)


def test_rotary_strides_in_place_and_batched(qb):
    g = _gen(11)
    plan = qb.RotaryPlan(128, base=1e6, scaling="yarn", factor=4.0, original_len=32768)
    B, S, H, Hkv, D = 3, 9, 4, 2, 128
    for skew in (0, 1):                       # views of a fused projection, aligned and not
        qkv = _randn(g, B, S, (H + 2 * Hkv) * D + skew).to(BF16)[..., skew:]
        q = qkv[..., :H * D].unflatten(-1, (H, D)).transpose(1, 2)
        k = qkv[..., H * D:(H + Hkv) * D].unflatten(-1, (Hkv, D)).transpose(1, 2)
        rest = qkv[..., (H + Hkv) * D:].clone()
        positions = torch.randint(0, 200000, (S, B), generator=g, device="cuda").t()
        want = [_turned(t.transpose(1, 2).reshape(B * S, -1, D), positions.reshape(-1), plan) for t in (q, k)]
        plain = [t.transpose(1, 2).reshape(B * S, -1, D).clone() for t in (q, k)]
        q2, k2 = qb.rotary(q, k, positions, plan)
        for got, x in ((q2, plain[0]), (k2, plain[1])):
            _check_turned(got.transpose(1, 2).reshape(B * S, -1, D), x, positions.reshape(-1), plan)
        q3, k3 = qb.rotary(q, k, positions, plan, q_out=q, k_out=k)
        assert q3 is q and torch.equal(q, q2) and torch.equal(k, k2)
        assert torch.equal(qkv[..., (H + Hkv) * D:], rest) and len(want) == 2
    only, none = qb.rotary(q2, None, positions, plan)
    assert none is None and only.shape == q2.shape


def test_rotary_far_and_negative_positions(qb):
    """Angles stay exact where a product in fp32 would be off by radians."""
    plan = qb.RotaryPlan(64, base=10000.0)
    positions = torch.tensor([0, 1, -1, 2 ** 24 + 1, 2 ** 31 - 1, -(2 ** 31)], device="cuda")
    q = _randn(_gen(1), 6, 2, 64).to(BF16)
    got, _ = qb.rotary(q, None, positions, plan)
    assert torch.equal(got[0], q[0])
    want, size = _turned(q, positions, plan)
    # float64 angles: position * 2^-53 radians
    slack = positions.double().abs()[:, None, None] * 2.0 ** -52
    assert ((got.double() - want).abs() <= HALF_ULP * want.abs() + (2.0 ** -20 + slack) * size).all()


def test_rotary_tables_feed_the_prologue(qb):
    """A plan's tables through the fused QK-norm prologue turn as ``rotary`` does."""
    g = _gen(21)
    plan = qb.RotaryPlan(128, base=1e6, scaling="linear", factor=2.0)
    positions = torch.randint(0, 40000, (2, 5), generator=g, device="cuda")
    cos, sin = qb.rotary_tables(positions, plan)
    angle = positions.double()[..., None] * torch.tensor(plan.freq * 2, dtype=torch.float64, device="cuda")
    assert (cos.double() - angle.cos()).abs().max() < 2.0 ** -20
    assert (sin.double() - angle.sin()).abs().max() < 2.0 ** -20
    q, k = _randn(g, 2, 4, 5, 128).to(BF16), _randn(g, 2, 2, 5, 128).to(BF16)
    one = torch.ones(128, dtype=BF16, device="cuda")
    q2, k2 = qb.qk_norm_rope_kv_write(q, k, None, one, one, cos, sin, return_k=True)
    for got, x in ((q2, q), (k2, k)):
        normed = qb.rms_norm(x, one)
        turned, _ = qb.rotary(normed, None, positions, plan)
        # the prologue rounds cos, sin, both products and their sum to bf16
        assert ((got.double() - turned.double()).abs() <= 2.0 ** -6 * normed.double().abs().amax()).all()
    inter = qb.RotaryPlan(6, base=100.0, layout="interleaved")
    cos, sin = qb.rotary_tables(torch.arange(4, device="cuda", dtype=torch.int32), inter)
    assert cos.shape == (4, 6) and torch.equal(cos[:, 0::2], cos[:, 1::2])


def test_rotary_empty_and_refusals(qb):
    plan = qb.RotaryPlan(16)
    q = torch.ones(3, 2, 16, dtype=BF16, device="cuda")
    p = torch.arange(3, device="cuda")
    assert qb.rotary(q[:0], q[:0], p[:0], plan)[0].shape == (0, 2, 16)
    for bad in (lambda: qb.rotary(q[..., :8], None, p, plan), lambda: qb.rotary(q.float(), None, p, plan),
                lambda: qb.rotary(q, q[:2], p, plan), lambda: qb.rotary(q, None, p.float(), plan),
                lambda: qb.rotary(q, None, p[:2], plan), lambda: qb.rotary(q.cpu(), None, p.cpu(), plan),
                lambda: qb.rotary(q, None, p, qb.RotaryPlan(16, device="cpu")),
                lambda: qb.rotary(q, None, p, plan, k_out=q),
                lambda: qb.rotary(q, None, p, plan, q_out=q[:2])):
        with pytest.raises(AssertionError):
            bad()


def test_sizes_past_31_bits_are_refused(qb):
    """Not cut to their low 32 bits, which would be 8 here."""
    x = torch.empty(1, 2**32 + 8, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError):
        qb.quantize_rows_fp8(x)
    with pytest.raises(RuntimeError):
        qb.linear(x, x)
