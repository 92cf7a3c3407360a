"""What the decoder-layer operators and the model around them accept, refuse and
promise, as far as that needs no GPU."""

import pytest

from qwen3_engine_from_scratch_b200.rope import RotaryPlan

TINY = dict(layers=1, hidden=32, heads=1, kv_heads=1, head_dim=16, intermediate=32, vocab=64, max_pos=8)


def test_model_refuses_plans_that_its_rotation_cannot_follow():
    """The fused QK-norm prologue pairs i with i + head_dim / 2: tables of another
    layout have the same shape and would turn q and k by the wrong angles."""
    from qwen3_engine_from_scratch_b200.e2e_model import Qwen3DecodeModel
    for plan in (RotaryPlan(16, layout="interleaved", device="cpu"), RotaryPlan(8, device="cpu")):
        with pytest.raises(AssertionError, match="rope_plan"):
            Qwen3DecodeModel("cpu", rope_plan=plan, **TINY)
        assert Qwen3DecodeModel("cpu", rope_plan=plan, qk_norm=False, **TINY).plan is plan
    with pytest.raises(AssertionError, match="rope_plan"):
        Qwen3DecodeModel("cpu", rope_plan=RotaryPlan(18, device="cpu"), qk_norm=False, **TINY)
    whole = RotaryPlan(16, device="cpu")
    assert Qwen3DecodeModel("cpu", rope_plan=whole, **TINY).plan is whole
