"""What the decoder-layer operators refuse, and what they do beside the ordinary
path, on the GPU."""

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def qb(cuda, native_lib):
    import qwen3_engine_from_scratch_b200 as m
    m.clear_device_status()
    yield m
    m.check_device_status()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def test_rotary_refuses_outputs_whose_elements_overlap(qb):
    plan = qb.RotaryPlan(16)
    q = _randn(_gen(1), 3, 4, 16).to(BF16)
    p = torch.arange(3, device="cuda")
    batch = q.unsqueeze(0)                       # (1, 3 heads, 4 tokens, 16)
    for bad in (lambda: qb.rotary(q, None, p, plan, q_out=q[:1].expand(3, 4, 16)),
                lambda: qb.rotary(q, None, p, plan, q_out=q[:, :1].expand(3, 4, 16)),
                lambda: qb.rotary(q, None, p, plan, q_out=q.as_strided((3, 4, 16), (40, 16, 1))),
                lambda: qb.rotary(q, q, p, plan, k_out=q[:, :1].expand(3, 4, 16)),
                lambda: qb.rotary(batch, None, torch.arange(4, device="cuda").unsqueeze(0), plan,
                                  q_out=batch[:, :, :1].expand(1, 3, 4, 16))):
        with pytest.raises(AssertionError, match="overlap"):
            bad()
    # read from an expanded tensor, written to views of a fused one
    wide = torch.zeros(3, 9, 16, dtype=BF16, device="cuda")
    src = q[:, :1].expand(3, 4, 16)
    want, _ = qb.rotary(src.contiguous(), None, p, plan)
    got, none = qb.rotary(src, None, p, plan, q_out=wide[:, 2:6])
    assert none is None and torch.equal(got, want)
    assert (wide[:, :2] == 0).all() and (wide[:, 6:] == 0).all()


def _timed(call):
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    begin.record()
    out = call()
    end.record()
    torch.cuda.synchronize()
    return out, begin.elapsed_time(end)


def test_streamed_norm_does_not_wait_for_copies_that_nobody_issued(qb):
    """Rows in numbers stream through shared memory.  Once its rows are done a block
    has no copy under way, and a timeout that another kernel left on record must not
    make it wait for one (0.1 s a stage)."""
    x, w = _randn(_gen(2), 1000, 4096).to(BF16), torch.ones(4096, dtype=BF16, device="cuda")
    qb.rms_norm(x, w)
    qb.ops._status[torch.cuda.current_device()].fill_(0x10)       # B200_DEV_TIMEOUT
    _, ms = _timed(lambda: qb.rms_norm(x, w))
    qb.clear_device_status()
    assert ms < 50, ms


def test_streamed_norm_without_a_status_word(qb, native_lib):
    """The C entry takes no status word too."""
    x, r = _randn(_gen(3), 1000, 4096).to(BF16), _randn(_gen(4), 1000, 4096).to(BF16)
    w = (1 + _randn(_gen(5), 4096, std=0.2)).to(BF16)
    want, h = qb.rms_norm(x, w, residual=r)
    y, h2 = torch.empty_like(x), torch.empty_like(x)
    st = native_lib.b200_rms_norm(x.data_ptr(), 4096, r.data_ptr(), 4096, w.data_ptr(), y.data_ptr(), 4096, None,
                                  h2.data_ptr(), 4096, 1000, 4096, 1e-6, None,
                                  torch.cuda.current_stream().cuda_stream)
    assert st == 0 and torch.equal(y, want) and torch.equal(h2, h)


def test_streamed_norm_waits_for_the_host_after_a_timeout(qb):
    """With a timeout on record it starts nothing, as the other pipelined kernels: no
    output is written in part.  Cleared, it works."""
    x, r = _randn(_gen(6), 3000, 4096).to(BF16), _randn(_gen(7), 3000, 4096).to(BF16)
    w = torch.ones(4096, dtype=BF16, device="cuda")
    for norm, kind in ((qb.rms_norm, BF16), (qb.rms_norm_fp8, FP8)):
        want = norm(x, w, residual=r)
        out = torch.full((3000, 4096), 3.0, device="cuda").to(kind)
        h = torch.full_like(r, 3.0)
        qb.ops._status[torch.cuda.current_device()].fill_(0x10)       # B200_DEV_TIMEOUT
        norm(x, w, residual=r, out=out, residual_out=h)
        with pytest.raises(RuntimeError, match="timed out"):
            qb.check_device_status()
        assert (out.float() == 3.0).all() and (h == 3.0).all()
        qb.clear_device_status()
        got = norm(x, w, residual=r, out=out, residual_out=h)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
        qb.check_device_status()


def test_a_cleared_status_counts_from_the_next_call_on(qb):
    """The clear is a kernel of its own, and the call behind it may be scheduled while
    that one drains."""
    x, w = _randn(_gen(8), 600, 4096).to(BF16), torch.ones(4096, dtype=BF16, device="cuda")
    weight = _randn(_gen(9), 256, 4096, std=0.02).to(BF16)
    status = qb.ops._status[torch.cuda.current_device()]
    want_y, want_p = qb.rms_norm(x, w), qb.linear(x, weight)
    for _ in range(50):
        status.fill_(0x10)                                              # B200_DEV_TIMEOUT
        status.zero_()
        y = qb.rms_norm(x, w)
        status.fill_(0x10)
        status.zero_()
        p = qb.linear(x, weight)
        assert torch.equal(y, want_y) and torch.equal(p, want_p)


def _kernels(call):
    """Names of the kernels that a call launches, from a graph of it."""
    from cuda.bindings import driver
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        kept = call()                                       # noqa: F841
    raw = driver.CUgraph(graph.raw_cuda_graph())
    _, _, n = driver.cuGraphGetNodes(raw)
    err, nodes, _ = driver.cuGraphGetNodes(raw, n)
    assert err == driver.CUresult.CUDA_SUCCESS
    names = []
    for node in nodes:
        err, kind = driver.cuGraphNodeGetType(node)
        if err == driver.CUresult.CUDA_SUCCESS and kind == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            err, p = driver.cuGraphKernelNodeGetParams(node)
            assert err == driver.CUresult.CUDA_SUCCESS
            err, name = driver.cuKernelGetName(p.kern) if int(p.func) == 0 else driver.cuFuncGetName(p.func)
            assert err == driver.CUresult.CUDA_SUCCESS
            names.append(name.decode())
    return names


@pytest.mark.parametrize("rows,hidden", [(1, 4096), (1, 4104), (8, 5120), (3, 6144), (64, 8192), (148, 8192),
                                         (2, 8200), (5, 16384)])
def test_few_wide_rows_are_read_once(qb, rows, hidden):
    """A decode step's rows stay in registers up to 16,384 elements: no second read."""
    from test_gpu_layer_ops import _check_bf16, _check_fp8, _norm_exact
    g = _gen(rows * hidden)
    x, r = _randn(g, rows, hidden, std=2.0).to(BF16), _randn(g, rows, hidden, std=3.0).to(BF16)
    w = (1 + _randn(g, hidden, std=0.3)).to(BF16)
    for res in (None, r):
        want, h = _norm_exact(x, w, res, 1e-6)
        got, q = qb.rms_norm(x, w, residual=res), qb.rms_norm_fp8(x, w, residual=res)
        _check_bf16(got if res is None else got[0], want)
        _check_fp8(q[0], q[1], want)
        if res is not None:
            _check_bf16(got[1], h)
            assert torch.equal(got[1], q[2])
    _check_fp8(*qb.quantize_rows_fp8(x), x.double())
    for call in (lambda: qb.rms_norm(x, w, residual=r), lambda: qb.rms_norm_fp8(x, w),
                 lambda: qb.quantize_rows_fp8(x)):
        names = _kernels(call)
        assert len(names) == 1 and "rms_norm_kernel" in names[0], names


def test_wider_rows_are_read_twice(qb):
    x, w = torch.ones(2, 16392, dtype=BF16, device="cuda"), torch.ones(16392, dtype=BF16, device="cuda")
    names = _kernels(lambda: qb.rms_norm(x, w))
    assert len(names) == 1 and "rms_norm_wide_kernel" in names[0], names


def test_product_refuses_its_operand_as_its_output(qb):
    """Other blocks still read x and the weight when a block writes its outputs."""
    x = _randn(_gen(10), 64, 64).to(BF16)
    w = _randn(_gen(11), 64, 64, std=0.1).to(BF16)
    for bad in (x, w):
        with pytest.raises(AssertionError, match="overlap"):
            qb.linear(x, w, out=bad)
    wide = torch.zeros(64, 128, dtype=BF16, device="cuda")          # side by side in one tensor
    wide[:, :64] = x
    qb.linear(wide[:, :64], w, out=wide[:, 64:])
    assert torch.equal(wide[:, 64:], qb.linear(x, w)) and torch.equal(wide[:, :64], x)
    assert qb.linear(x[:0], w, out=x[:0]).shape == (0, 64)


@pytest.mark.parametrize("rotary_dim,base", [(128, 1000000), (64, 10000)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_angles_at_any_position(qb, rotary_dim, base, layout):
    """An angle is off by 2^-26 turns (32 bits of a turn rounded to fp32: 2^-26, and cut
    there: 2^-32) and 2^-54 turns a position (the plan's frequencies); sine and cosine
    by 2^-22 more."""
    import math
    from decimal import Decimal, localcontext
    from test_layer_contracts import turns_a_position
    at = [0, 1, -1, 17, 131071, -4097, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 2 ** 33 + 5, -(2 ** 37) + 3, 2 ** 40 + 9]
    plan = qb.RotaryPlan(rotary_dim, base=float(base), layout=layout)
    cos, sin = (t.double().cpu() for t in qb.rotary_tables(torch.tensor(at, device="cuda"), plan))
    exact = turns_a_position(rotary_dim, base)
    for row, p in enumerate(at):
        bound = 2 * math.pi * (2.0 ** -26 + 2.0 ** -32 + abs(p) * 2.0 ** -54) + 2.0 ** -22
        for i, f in enumerate(exact):
            with localcontext() as c:
                c.prec = 60
                part = float((f * p) % 1)
            for e in ((i, i + rotary_dim // 2) if layout == "half" else (2 * i, 2 * i + 1)):
                assert abs(float(cos[row, e]) - math.cos(2 * math.pi * part)) <= bound, (p, i)
                assert abs(float(sin[row, e]) - math.sin(2 * math.pi * part)) <= bound, (p, i)
