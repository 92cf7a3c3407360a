"""The decoder layer on the package's own kernels (``layer_ops`` of the
end-to-end model) against the same model with torch's norms and products, and
its prefill against its decode.

Tolerances: the two models round to bf16 at about ten places a layer, each off
by 2^-9 / sqrt(3) of its value in the mean square; over two layers and both
models that is 0.7 % of the logits' norm, and 3 % is allowed.  An e4m3 operand is
off by 2.6 % in the mean square (uniform within half a unit of 3 mantissa bits), a
product of two by 3.7 %; eight products one after another stay below 10.5 %, and
20 % is allowed.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(device, **more):
    from qwen3_engine_from_scratch_b200 import e2e_model
    return e2e_model.Qwen3DecodeModel(device, layers=2, hidden=512, heads=16, kv_heads=8,
                                      head_dim=128, intermediate=1040, vocab=4096, seed=3,
                                      max_pos=1024, **more)


def _prefill_logits(model, prompts, device):
    from qwen3_engine_from_scratch_b200 import KVCachePool
    lens = np.array([len(p) for p in prompts])
    pool = KVCachePool(sum((n + 15) // 16 for n in lens), model.layers, 16, model.Hkv, model.D,
                       device=device, dtype=torch.bfloat16, max_seq_len=1024, max_requests=len(prompts) + 1)
    starts = np.concatenate([[0], np.cumsum((lens + 15) // 16)]) * 16
    slots = np.concatenate([s + np.arange(n) for s, n in zip(starts, lens)])
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(device)  # noqa: E731
    h = model.forward_prefill(to(np.concatenate(prompts).astype(np.int64)), to(cu), int(lens.max()),
                              to(np.concatenate([np.arange(n) for n in lens])), to(slots), pool)
    return model.logits(h).float()


@pytest.mark.parametrize("layer_ops,allowed", [("bf16", 0.03), ("fp8", 0.2)])
def test_logits_near_the_torch_layers(cuda, native_lib, layer_ops, allowed):
    from qwen3_engine_from_scratch_b200 import e2e_model
    prompts = e2e_model.synthetic_prompts(7, 1, 200, 4096, seed=11)
    want = _prefill_logits(_model(cuda), prompts, cuda)
    got = _prefill_logits(_model(cuda, layer_ops=layer_ops), prompts, cuda)
    assert got.shape == want.shape
    off = (got - want).norm(dim=-1) / want.norm(dim=-1)
    assert float(off.max()) <= allowed, off.tolist()


@pytest.mark.parametrize("more", [dict(layer_ops="bf16"), dict(layer_ops="fp8"),
                                  dict(layer_ops="bf16", qk_norm=False), dict(qk_norm=False),
                                  dict(layer_ops="fp8", scaled=True), dict(scaled=True)])
def test_decode_goes_on_where_prefill_would(cuda, native_lib, more):
    """Tokens generated from graphs equal the eager ones, and prefilling a prompt
    with its generated tokens names the same next token (where one is clear)."""
    import qwen3_engine_from_scratch_b200 as qb
    from qwen3_engine_from_scratch_b200 import e2e_model
    more = dict(more)
    if more.pop("scaled", False):
        more["rope_plan"] = qb.RotaryPlan(128, base=1e6, scaling="yarn", factor=4.0, original_len=64)
    model = _model(cuda, **more)
    prompts = e2e_model.synthetic_prompts(9, 1, 120, 4096, seed=5)
    eager, _ = e2e_model.serve(model, prompts, 6, cuda, graph=False)
    graphed, _ = e2e_model.serve(model, prompts, 6, cuda, graph=True, buckets=(4, 16))
    assert torch.equal(eager, graphed)
    longer = [np.concatenate([p, t[:5].numpy()]) for p, t in zip(prompts, eager)]
    logits = _prefill_logits(model, longer, cuda)
    top = torch.topk(logits, 2).values
    clear = ((top[:, 0] - top[:, 1]) > (0.3 if more.get("layer_ops") == "fp8" else 0.05)).cpu()
    assert torch.equal(logits.argmax(-1).cpu()[clear], eager[:, 5][clear])
    qb.check_device_status()
