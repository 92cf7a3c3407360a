"""The pipelined (tcgen05) product in CUDA graphs and on streams of its own, in the
chains that a decoder layer makes of it: a replay has to give, bit for bit, what the
same calls give one by one."""

import numpy as np
import pytest
import torch

from test_gpu_layer_contracts import _gen, _kernels, _randn

pytestmark = pytest.mark.gpu

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def qb(cuda, native_lib):
    import qwen3_engine_from_scratch_b200 as m
    m.clear_device_status()
    yield m
    m.check_device_status()


# tokens, hidden, inner width, e4m3, and what one of the two products is there for: tiles
# of one CTA, with K split 4 or 8 ways in the second product, pairs of CTAs, rows laid out first
CHAINS = [(200, 512, 12800, False, "split"), (64, 4096, 12288, True, "split"), (64, 1024, 4096, False, "split"),
          (1500, 512, 2048, True, "single"), (2049, 1024, 2048, False, "pair"), (2049, 2048, 4096, True, "pair"),
          (40, 333, 1000, False, "packed"), (300, 1001, 640, True, "packed")]


def _chain(qb, hidden, inner, fp8, seed):
    """norm -> gated product -> product onto the residual, as a function of x and the residual."""
    g = _gen(seed)
    ln = (1 + _randn(g, hidden, std=0.2)).to(BF16)
    up = _randn(g, 2 * inner, hidden, std=hidden ** -0.5).to(BF16)
    down = _randn(g, hidden, inner, std=inner ** -0.5).to(BF16)
    if fp8:
        (up, su), (down, sd) = qb.quantize_rows_fp8(up), qb.quantize_rows_fp8(down)

    def run(x, r):
        if fp8:
            y, s, h = qb.rms_norm_fp8(x, ln, residual=r)
            a, sa = qb.quantize_rows_fp8(qb.linear(y, up, gated=True, activation="silu", x_scale=s, weight_scale=su))
            return qb.linear(a, down, residual=h, x_scale=sa, weight_scale=sd)
        y, h = qb.rms_norm(x, ln, residual=r)
        return qb.linear(qb.linear(y, up, gated=True, activation="silu"), down, residual=h)
    return run


@pytest.mark.parametrize("tokens,hidden,inner,fp8,holds", CHAINS)
def test_chain_replayed_with_other_inputs(qb, tokens, hidden, inner, fp8, holds):
    run = _chain(qb, hidden, inner, fp8, tokens)
    g = _gen(tokens + 1)
    x, r = (torch.zeros(tokens, hidden, dtype=BF16, device="cuda") for _ in range(2))
    names = _kernels(lambda: run(x, r))
    products = [n for n in names if "linear_kernel" in n]
    assert len(products) == 2 and not any("linear_small" in n for n in names), names
    assert any("pack_rows" in n for n in names) == (holds == "packed"), names
    if holds == "pair":
        assert any("Lb1EE" in n for n in products), names
    run(x, r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x, r)
    for _ in range(4):
        x.copy_(_randn(g, tokens, hidden))
        r.copy_(_randn(g, tokens, hidden, std=2.0))
        graph.replay()
        graph.replay()                                       # back to back: one's end is the next one's start
        assert torch.equal(out, run(x, r))
    del graph


@pytest.mark.parametrize("tokens,hidden,inner,fp8,holds", CHAINS)
def test_chains_on_two_streams(qb, tokens, hidden, inner, fp8, holds):
    """Each stream has its own order; the two share nothing but the weights."""
    run = _chain(qb, hidden, inner, fp8, tokens)
    g = _gen(tokens + 2)
    data = [(_randn(g, tokens, hidden).to(BF16), _randn(g, tokens, hidden).to(BF16)) for _ in range(2)]
    want = [run(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(*data[i]))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


@pytest.mark.parametrize("layer_ops", ["bf16", "fp8"])
def test_model_decode_of_a_batch_that_takes_the_pipelined_products(cuda, native_lib, qb, layer_ops):
    from qwen3_engine_from_scratch_b200 import e2e_model
    from test_gpu_layer_model import _model
    model = _model(cuda, layer_ops=layer_ops)
    prompts = e2e_model.synthetic_prompts(20, 1, 90, 4096, seed=8)
    eager, _ = e2e_model.serve(model, prompts, 6, cuda, graph=False)
    graphed, _ = e2e_model.serve(model, prompts, 6, cuda, graph=True, buckets=(32,))
    assert torch.equal(eager, graphed) and np.unique(eager.numpy()).size > 1
