"""Qwen3-shaped model and serving loop for the end-to-end benchmark (config 5).

Config 5 measures whole-engine decode throughput with this package's kernels
swapped in: Qwen3-0.6B (28 layers, hidden 1024, 16 query / 8 kv heads of 128,
SwiGLU 3072, vocab 151,936, bf16) with seeded N(0, 0.02) weights, 256
concurrent requests with prompts of U[32, 1024] tokens and 256 generated
tokens each, decode replayed from CUDA graphs.  The reference serves this with
its Scheduler, model.forward (prefill) and GraphRunner (decode)
(bench_batched.py:150-200, qwen3/model.py:186-251, qwen3/graph_runner.py).

By default the GEMMs, embedding, RMSNorms and the MLP are plain torch (cuBLAS):
they are outside the attention hot path.  With ``layer_ops="bf16"`` or ``"fp8"``
the whole decoder layer runs on the package's kernels: ``rms_norm`` (with the
residual's addition before the MLP), ``linear`` (the gated activation and the
second residual in its epilogue) and, in 8 bits, ``rms_norm_fp8`` and
``quantize_rows_fp8`` in front of each product.  ``rope_plan`` scales the rotary
frequencies for long contexts (with the QK norm it turns the whole head in the
half layout); ``qk_norm=False`` turns q and k by ``rotary`` and any plan.
The attention path is this package's in every case:

* prefill (packed tokens of all requests): ``qk_norm_rope_kv_write`` (QK norm
  + RoPE), ``kv_scatter_slots`` (the prompt's K/V into the paged pool) and
  ``flash_attention_prefill`` (varlen causal prefill);
* decode (``forward_decode``, the contract of qwen3/model.py:240-251 that
  ``GraphRunner`` captures): ``qk_norm_rope_kv_write`` and
  ``triton_paged_attention_decode_batch`` (KV write + split-K decode, one
  launch);
* sampling: ``sample_tokens`` (greedy here).

As in the reference's scheduler (qwen3/scheduler.py:59-89), with room for all
requests the first step prefills every prompt and every later step decodes
the whole running batch; no request finishes early (no EOS), so the batch
stays full until the last step.
"""

from __future__ import annotations

import time

import numpy as np
import torch

from . import ops
from .graph_runner import GraphRunner
from .paged_kv import KVCachePool, PagedKVCache
from .rope import RotaryPlan

QWEN3_0_6B = dict(layers=28, hidden=1024, heads=16, kv_heads=8, head_dim=128,
                  intermediate=3072, vocab=151936, rope_theta=1e6, eps=1e-6)


class Qwen3DecodeModel:
    """Random-init Qwen3 decoder (seeded N(0, std) linear and embedding weights,
    unit RMSNorm weights, tied lm_head as in Qwen3-0.6B)."""

    def __init__(self, device, layers=28, hidden=1024, heads=16, kv_heads=8, head_dim=128,
                 intermediate=3072, vocab=151936, rope_theta=1e6, eps=1e-6, max_pos=4096,
                 seed=0, std=0.02, layer_ops="torch", rope_plan=None, qk_norm=True):
        assert layer_ops in ("torch", "bf16", "fp8"), "layer_ops must be torch, bf16 or fp8"
        if rope_plan is not None and qk_norm:      # by tables, which do not tell their layout
            assert not rope_plan.interleaved and rope_plan.rotary_dim == head_dim, \
                "with qk_norm a rope_plan must turn the whole head in the half layout"
        assert rope_plan is None or rope_plan.rotary_dim <= head_dim, \
            "the rope_plan's rotary_dim exceeds head_dim"
        g = torch.Generator(device=device).manual_seed(seed)
        bf = torch.bfloat16

        def w(*shape):
            return (torch.randn(*shape, generator=g, device=device) * std).to(bf)

        self.layers, self.hidden, self.H, self.Hkv, self.D = layers, hidden, heads, kv_heads, head_dim
        self.inter, self.vocab, self.eps = intermediate, vocab, eps
        self.embed = w(vocab, hidden)                                  # tied with lm_head
        self.wqkv = [w(hidden, (heads + 2 * kv_heads) * head_dim) for _ in range(layers)]
        self.wo = [w(heads * head_dim, hidden) for _ in range(layers)]
        self.wgu = [w(hidden, 2 * intermediate) for _ in range(layers)]  # gate | up
        self.wd = [w(intermediate, hidden) for _ in range(layers)]
        ones = torch.ones(hidden, dtype=bf, device=device)
        self.ln1 = [ones] * layers
        self.ln2 = [ones] * layers
        self.ln_f = ones
        self.qn = [torch.ones(head_dim, dtype=bf, device=device)] * layers
        self.kn = [torch.ones(head_dim, dtype=bf, device=device)] * layers
        inv = 1.0 / (rope_theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32,
                                                 device=device) / head_dim))
        f = torch.outer(torch.arange(max_pos, dtype=torch.float32, device=device), inv)
        emb = torch.cat([f, f], dim=-1)
        self.cos_t, self.sin_t = emb.cos(), emb.sin()                 # fp32 rows, as the reference
        self.scale = head_dim ** -0.5
        self.layer_ops, self.qk_norm = layer_ops, qk_norm
        self.plan = rope_plan if rope_plan is not None or qk_norm else \
            RotaryPlan(head_dim, base=rope_theta, device=device)
        if layer_ops != "torch":       # (out, in) rows, as ops.linear reads them
            for ws in (self.wqkv, self.wo, self.wgu, self.wd):
                for i, w_t in enumerate(ws):
                    rows = w_t.t().contiguous()
                    ws[i] = ops.quantize_rows_fp8(rows) if layer_ops == "fp8" else (rows, None)

    def _normed(self, x, w, residual=None):
        """RMS norm as a product's operand (rows, scale or None), and x + residual."""
        if self.layer_ops == "fp8":
            q, s, *h = ops.rms_norm_fp8(x, w, residual=residual, eps=self.eps)
            return (q, s), h[0] if h else x
        y = ops.rms_norm(x, w, residual=residual, eps=self.eps)
        return ((y, None), x) if residual is None else ((y[0], None), y[1])

    def _operand(self, x):
        return ops.quantize_rows_fp8(x) if self.layer_ops == "fp8" else (x, None)

    @staticmethod
    def _product(x, w, **epilogue):
        return ops.linear(x[0], w[0], x_scale=x[1], weight_scale=w[1], **epilogue)

    def _block(self, i, h, attend):
        """One decoder layer around ``attend(qkv) -> attention output``."""
        if self.layer_ops == "torch":
            h = h + attend(self._rms(h, self.ln1[i]) @ self.wqkv[i]) @ self.wo[i]
            return self._mlp(i, h)
        y, _ = self._normed(h, self.ln1[i])
        o = attend(self._product(y, self.wqkv[i]))
        o = self._product(self._operand(o), self.wo[i])
        y, h = self._normed(o, self.ln2[i], residual=h)
        a = self._product(y, self.wgu[i], gated=True, activation="silu")
        return self._product(self._operand(a), self.wd[i], residual=h)

    def _positions(self, positions):
        """What ``_rotate`` needs of the step's (B, S) positions."""
        if self.plan is None:
            return self.cos_t[positions], self.sin_t[positions]
        return ops.rotary_tables(positions, self.plan) if self.qk_norm else positions

    def _rotate(self, i, q, k, v, at):
        if not self.qk_norm:
            return ops.rotary(q, k, at, self.plan)
        return ops.qk_norm_rope_kv_write(q, k, v, self.qn[i], self.kn[i], at[0], at[1],
                                         eps=self.eps, return_k=True)

    def _rms(self, x, w):
        xf = x.float()
        return ((xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)) * w).to(x.dtype)

    def _mlp(self, i, h):
        gu = self._rms(h, self.ln2[i]) @ self.wgu[i]
        gate, up = gu[..., :self.inter], gu[..., self.inter:]
        return h + (torch.nn.functional.silu(gate) * up) @ self.wd[i]

    def logits(self, h):
        if self.layer_ops != "torch":
            return ops.linear(ops.rms_norm(h, self.ln_f, eps=self.eps), self.embed)
        return self._rms(h, self.ln_f) @ self.embed.t()

    @torch.no_grad()
    def forward_prefill(self, tokens, cu_seqlens, max_len, positions, slots, pool):
        """All prompts as packed tokens: (T,) ids, int32 cu_seqlens, (T,) positions
        and (T,) int64 pool slots.  Writes every layer's K/V into ``pool`` and
        returns the final hidden state of each sequence's last token."""
        H, Hkv, D = self.H, self.Hkv, self.D
        T = tokens.shape[0]
        at = self._positions(positions[None])
        h = self.embed[tokens][None]               # (1, T, hidden)
        for i in range(self.layers):
            def attend(qkv):
                q = qkv[..., :H * D].view(1, T, H, D).transpose(1, 2)
                k = qkv[..., H * D:(H + Hkv) * D].view(1, T, Hkv, D).transpose(1, 2)
                v = qkv[..., (H + Hkv) * D:].view(1, T, Hkv, D).transpose(1, 2)
                q, k = self._rotate(i, q, k, v, at)
                k_t, v_t = k[0].transpose(0, 1), v[0].transpose(0, 1)   # (T, Hkv, D) views
                ops.kv_scatter_slots(k_t, v_t, pool.k_buffer, pool.v_buffer, slots, i)
                o = ops.flash_attention_prefill(q[0].transpose(0, 1), k_t, v_t, cu_seqlens,
                                                self.scale, H, Hkv, D, max_seqlen=max_len)
                return o.reshape(1, T, H * D)

            h = self._block(i, h, attend)
        return h[0, cu_seqlens[1:].long() - 1]     # (B, hidden)

    @torch.no_grad()
    def forward_decode(self, input_ids, position_ids, row_ids, caches):
        """One decode step (qwen3/model.py:240-251 contract): (B, 1) ids and
        positions, (B,) int32 rows -> (B, 1, vocab) logits.  Capture-safe."""
        B = input_ids.shape[0]
        H, Hkv, D = self.H, self.Hkv, self.D
        at = self._positions(position_ids)
        h = self.embed[input_ids]                  # (B, 1, hidden)
        for i in range(self.layers):
            def attend(qkv):
                q = qkv[..., :H * D].view(B, 1, H, D).transpose(1, 2)
                k = qkv[..., H * D:(H + Hkv) * D].view(B, 1, Hkv, D).transpose(1, 2)
                v = qkv[..., (H + Hkv) * D:].view(B, 1, Hkv, D).transpose(1, 2)
                q, k = self._rotate(i, q, k, v, at)
                return ops.triton_paged_attention_decode_batch(q, k, v, caches, i, self.scale,
                                                               row_ids)

            h = self._block(i, h, attend)
        return self.logits(h)


def synthetic_prompts(n, lo, hi, vocab, seed):
    """``n`` prompt lengths U[lo, hi] and token ids U[0, vocab) (seeded)."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(lo, hi, size=n, endpoint=True)
    return [rng.integers(0, vocab, size=int(L)) for L in lens]


def serve(model, prompts, new_tokens, device, graph=True, buckets=None, pool_blocks=None,
          timers=None):
    """Prefill every prompt, then decode ``new_tokens - 1`` steps of the whole
    batch (the prefill produces the first token).  Returns (tokens (B, new_tokens)
    int64 on the host, stats).  Greedy sampling."""
    B = len(prompts)
    lens = np.array([len(p) for p in prompts], dtype=np.int64)
    max_total = int(lens.max()) + new_tokens
    pages = int(((lens + new_tokens + 15) // 16).sum())
    buckets = tuple(buckets) if buckets is not None else (B,)
    nb = pool_blocks or pages + max(buckets) + 16
    pool = KVCachePool(nb, model.layers, 16, model.Hkv, model.D, device=device,
                       dtype=torch.bfloat16, max_seq_len=max_total,
                       max_requests=B + max(buckets) + 2)
    caches = [PagedKVCache(pool) for _ in range(B)]
    for c, L in zip(caches, lens):
        c._ensure_pages(int(L))
    slots = np.concatenate([np.asarray(c.block_table, np.int64)[np.arange(L) // 16] * 16
                            + np.arange(L) % 16 for c, L in zip(caches, lens)])
    positions = np.concatenate([np.arange(L) for L in lens])
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    tok = torch.from_numpy(np.concatenate(prompts).astype(np.int64)).to(device)
    d_slots = torch.from_numpy(slots).to(device)
    d_pos = torch.from_numpy(positions).to(device)
    d_cu = torch.from_numpy(cu).to(device)
    rows = torch.tensor([c.row_id for c in caches], dtype=torch.int32, device=device)

    runner = None
    if graph:
        holders = [PagedKVCache(pool) for _ in range(max(buckets))]
        runner = GraphRunner(model, pool, holders, buckets=buckets)
    out = torch.empty((B, new_tokens), dtype=torch.int64, device=device)

    torch.cuda.synchronize()
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
    t0 = time.perf_counter()
    ev[0].record()
    last_h = model.forward_prefill(tok, d_cu, int(lens.max()), d_pos, d_slots, pool)
    for c, L in zip(caches, lens):
        c.advance_seq_len(int(L))
    nxt = ops.sample_tokens(model.logits(last_h), 0.0)             # (B, 1) greedy
    out[:, 0] = nxt[:, 0]
    ev[1].record()
    pos = torch.from_numpy(lens).to(device)[:, None]               # position of the next token
    for step in range(1, new_tokens):
        for c in caches:
            c.reserve_next()
        if runner is not None:
            logits = runner.replay(nxt, pos, rows)[:B]
        else:
            logits = model.forward_decode(nxt, pos, rows, caches)
        for c in caches:
            c.advance_seq_len(1)
        nxt = ops.sample_tokens(logits[:, 0], 0.0)
        out[:, step] = nxt[:, 0]
        pos = pos + 1
    ev[2].record()
    torch.cuda.synchronize()
    wall = time.perf_counter() - t0
    prefill_ms = ev[0].elapsed_time(ev[1])
    decode_ms = ev[1].elapsed_time(ev[2])
    stats = {"requests": B, "prompt_tokens": int(lens.sum()), "new_tokens_per_request": new_tokens,
             "prefill_ms": prefill_ms, "decode_ms": decode_ms, "wall_s": wall,
             "decode_steps": new_tokens - 1, "pool_blocks": nb}
    if runner is not None:
        runner.free()
    del pool
    return out.cpu(), stats
