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
