"""The model's rotation against a torch forward of one decoder layer in fp32 that
turns q and k by complex numbers, from angles of its own.

Tolerance: the model rounds to bf16 at about ten places of its layer (2^-9 / sqrt(3)
of the value in the mean square each) and the prologue at four more; scores of
size 1 to 2 that are off by 2^-8 of themselves move a softmax weight by less than
1 %.  3 % of the logits' norm is allowed, as between the models of the same sizes
elsewhere; the unturned forward has to be farther off than five times that.
"""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HEADS, KV, D, HIDDEN, VOCAB = 16, 8, 128, 512, 4096


def _angles(n, rotary_dim, base, factor, trained, device):
    """(n, rotary_dim / 2) angles by the index ramp between 32 turns and 1 over `trained`."""
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    f = base ** (-2 * pair / rotary_dim)
    edge = [rotary_dim * math.log(trained / (2 * math.pi * t)) / (2 * math.log(base)) for t in (32.0, 1.0)]
    lo, hi = max(0, math.floor(edge[0])), math.ceil(edge[1])
    assert lo < hi < rotary_dim // 2            # no cut at either end in this test
    squeeze = ((pair - lo) / (hi - lo)).clamp(0, 1)
    f = f * (1 - squeeze) + f / factor * squeeze
    return torch.arange(n, dtype=torch.float64, device=device)[:, None] * f


def _forward(m, tokens, turn):
    """Last token's logits of the one-layer model `m`, in fp32."""
    rms = lambda x: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + m.eps)  # noqa: E731
    h = m.embed[tokens].float()
    qkv = rms(h) @ m.wqkv[0].float()
    q, k, v = (t.unflatten(-1, (-1, D)).transpose(0, 1) for t in
               qkv.split([HEADS * D, KV * D, KV * D], -1))
    if m.qk_norm:
        q, k = rms(q), rms(k)
    q, k = turn(q), turn(k)
    k, v = (t.repeat_interleave(HEADS // KV, 0) for t in (k, v))
    n = len(tokens)
    s = q @ k.transpose(1, 2) * D ** -0.5
    s = s.masked_fill(torch.ones(n, n, device=s.device).triu(1).bool(), float("-inf"))
    h = h + (s.softmax(-1) @ v).transpose(0, 1).flatten(1) @ m.wo[0].float()
    gate, up = (rms(h) @ m.wgu[0].float()).chunk(2, -1)
    h = h + (torch.nn.functional.silu(gate) * up) @ m.wd[0].float()
    return (rms(h[-1:]) @ m.embed.float().t())[0]


def _turn(angle, gain, layout):
    by = torch.polar(torch.full_like(angle, gain), angle)
    half = angle.shape[1]

    def turn(x):
        pairs = x[..., :2 * half].double()
        pairs = pairs.unflatten(-1, (2, half)).transpose(-1, -2) if layout == "half" else \
            pairs.unflatten(-1, (half, 2))
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        pairs = pairs.transpose(-1, -2) if layout == "half" else pairs
        return torch.cat([pairs.flatten(-2).float(), x[..., 2 * half:]], -1)
    return turn


@pytest.mark.parametrize("qk_norm,layout,rotary_dim", [(True, "half", 128), (False, "half", 128),
                                                       (False, "interleaved", 128),
                                                       (False, "interleaved", 64), (False, "half", 64)])
def test_scaled_prefill_against_torch(cuda, native_lib, qk_norm, layout, rotary_dim):
    import qwen3_engine_from_scratch_b200 as qb
    from qwen3_engine_from_scratch_b200 import e2e_model
    plan = qb.RotaryPlan(rotary_dim, base=1e4, layout=layout, scaling="yarn", factor=4.0, original_len=512)
    m = e2e_model.Qwen3DecodeModel(cuda, layers=1, hidden=HIDDEN, heads=HEADS, kv_heads=KV, head_dim=D,
                                   intermediate=1040, vocab=VOCAB, seed=4, std=0.05, max_pos=256,
                                   rope_plan=plan, qk_norm=qk_norm)
    prompts = [np.random.default_rng(n).integers(0, VOCAB, size=n) for n in (200, 37, 90)]
    lens = np.array([len(p) for p in prompts])
    pool = qb.KVCachePool(sum((n + 15) // 16 for n in lens), 1, 16, KV, D, device=cuda,
                          dtype=torch.bfloat16, max_seq_len=256, max_requests=4)
    starts = np.concatenate([[0], np.cumsum((lens + 15) // 16)]) * 16
    slots = np.concatenate([s + np.arange(n) for s, n in zip(starts, lens)])
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    to = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(cuda)  # noqa: E731
    h = m.forward_prefill(to(np.concatenate(prompts)), to(cu), int(lens.max()),
                          to(np.concatenate([np.arange(n) for n in lens])), to(slots), pool)
    got = m.logits(h).float()
    with torch.no_grad():
        for row, p in zip(got, prompts):
            angle = _angles(len(p), rotary_dim, 1e4, 4.0, 512, cuda)
            off = lambda want: float((row - want).norm() / want.norm())  # noqa: E731
            want = _forward(m, to(p), _turn(angle, 0.1 * math.log(4.0) + 1, layout))
            assert off(want) <= 0.03, off(want)
            assert off(_forward(m, to(p), lambda x: x)) > 0.15
    qb.check_device_status()
