"""Scores of given decoder tokens under a decode step in fewer bits.

What does a decode step lose when its weights are held in 4 bits and its K/V cache in 8? Feed it a
text instead of its own choices (full-precision output of ``Engine.generate``, or the texts one
serves) and read off each token's log probability, the entropy and the likeliest alternatives:

    scores = LowBitScorer(hf_model, max_decoder_len=64).score(requests, targets, alternatives=5)

Per step and layer: four to six ``paged_ops.linear_int4``, one ``reshape_and_cache_int8``, two
``attention_with_kv_cache_int8`` (the decoder's own tokens and the encoder's pages), and one
``token_logprobs`` a step. The encoder runs in the model's precision, as in ``Engine``.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F

from .. import paged_ops
from .engine import Request
from .model import PagedSeq2Seq


@dataclass
class TokenScores:
    """One request's target tokens under the model; tensors on the host, one row a token."""

    logprobs: torch.Tensor  # float32 [tokens]
    entropy: torch.Tensor   # float32 [tokens]
    values: torch.Tensor    # float32 [tokens, alternatives], log probability descending
    indices: torch.Tensor   # int32 [tokens, alternatives]


class _Int4Linear:
    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, group_size: int):
        self.codes, self.scales = paged_ops.quantize_int4(weight, group_size)
        self.bias = bias

    def __call__(self, x: torch.Tensor, activation: str | None = None) -> torch.Tensor:
        return paged_ops.linear_int4(x, self.codes, self.scales, self.bias, activation)


class _Cache:
    """One layer's 8-bit pool: (k_cache, v_cache, k_scale, v_scale)."""

    def __init__(self, num_blocks: int, heads: int, block_size: int, head_dim: int, device: torch.device):
        codes = torch.zeros((2, num_blocks, heads, block_size, head_dim), dtype=torch.int8, device=device)
        scales = torch.zeros((2, num_blocks, heads), dtype=torch.float32, device=device)
        self.parts = (codes[0], codes[1], scales[0], scales[1])


class LowBitScorer:
    """A HuggingFace BART-family model on a CUDA device, its decoder's linear layers in 4 bits
    (``group_size`` weights a scale; the token embedding and the norms stay) and its caches in 8."""

    def __init__(self, hf_model, *, max_decoder_len: int, block_size: int = 16, group_size: int = 64,
                 decoder_start_token_id: int | None = None):
        m = self.model = PagedSeq2Seq(hf_model, skinny_linear=False)
        if m.device.type != "cuda":
            raise ValueError(f"vflorence_b200: LowBitScorer needs a model on a CUDA device (got {m.device})")
        paged_ops.get_isa(m.dtype, block_size, m.head_dim)
        self.max_decoder_len, self.block_size = max_decoder_len, block_size
        cfg = hf_model.config.get_text_config()
        self.start_token = cfg.decoder_start_token_id if decoder_start_token_id is None else decoder_start_token_id
        self.pad_token = cfg.pad_token_id or 0
        q = lambda w, b: _Int4Linear(w, b, group_size)  # noqa: E731
        self.layers = [{"qkv": q(L.w_qkv, L.b_qkv), "self_out": q(L.self_out.weight, L.self_out.bias),
                        "cross_q": q(L.cross_q.weight, L.cross_q.bias),
                        "cross_out": q(L.cross_out.weight, L.cross_out.bias),
                        "fc1": q(L.fc1.weight, L.fc1.bias), "fc2": q(L.fc2.weight, L.fc2.bias)} for L in m.layers]
        self.head = q(m.w_head, m.b_head)

    # ------------------------------------------------------------------------------------ encoder
    def _page_encoder(self, requests: list[Request]):
        """(a cache a layer, block table, lengths on the device and the host) of the requests'
        encoder K/V; one padded batch, so the images must share a shape."""
        m, bs, dev = self.model, self.block_size, self.model.device
        lens = torch.tensor([len(r.input_ids) for r in requests], dtype=torch.int32)
        width = int(lens.max())
        per_req = -(-width // bs)
        ids = torch.full((len(requests), width), self.pad_token, dtype=torch.long)
        for i, r in enumerate(requests):
            ids[i, : len(r.input_ids)] = torch.tensor(r.input_ids)
        pos = torch.arange(width)
        real = pos[None] < lens[:, None]
        table = torch.arange(len(requests) * per_req, dtype=torch.int32).view(-1, per_req)
        slots = torch.where(real, table[:, pos // bs].long() * bs + pos % bs, -1).view(-1).to(dev)
        pixels = None
        if requests[0].pixel_values is not None:
            pixels = torch.stack([r.pixel_values for r in requests]).to(dev)
        hidden = m.encode(ids.to(dev), pixels, None if bool(real.all()) else real.long().to(dev))
        caches = []
        for i in range(len(m.layers)):
            cache = _Cache(table.numel(), m.num_heads, bs, m.head_dim, dev)
            paged_ops.reshape_and_cache_int8(*m.cross_kv(i, hidden), *cache.parts, slots)
            caches.append(cache.parts)
        return caches, table.to(dev), lens.to(dev), lens

    # ------------------------------------------------------------------------------------ decoder
    def _attend(self, query, cache, starts, lens, table, plan):
        out = torch.empty_like(query)
        paged_ops.attention_with_kv_cache_int8(query, *cache, out, starts, lens, self.model.scale, False, table, plan)
        return out

    def _plan(self, lens: torch.Tensor) -> torch.Tensor:
        m, n = self.model, lens.numel()
        return paged_ops.get_scheduler_metadata_int8(n, m.num_heads, m.num_heads, m.head_dim, lens, m.dtype,
                                                     torch.arange(n + 1, dtype=torch.int32), False, self.block_size)

    def _step(self, tokens, position: int, own, cross):
        """Logits [n, vocab] of one decoder step at ``position``; ``own`` and ``cross`` are (caches,
        starts, lengths, table, plan), ``own`` with the step's slots as well."""
        m, n = self.model, tokens.shape[0]
        own_caches, slots, *own_args = own
        cross_caches, *cross_args = cross
        where = m.pos_weight[position + m.pos_offset].expand(n, m.d_model)
        h = m._add_norm(m.embed_tokens(tokens), where, m.ln_embed)
        shape = (n, m.num_heads, m.head_dim)
        for i, (L, W) in enumerate(zip(m.layers, self.layers)):
            q, k, v = (t.reshape(shape) for t in W["qkv"](h).chunk(3, dim=-1))
            paged_ops.reshape_and_cache_int8(k, v, *own_caches[i], slots)
            a = self._attend(q, own_caches[i], *own_args).view(n, m.d_model)
            h = m._add_norm(h, W["self_out"](a), L.ln_self)
            c = self._attend(W["cross_q"](h).view(shape), cross_caches[i], *cross_args).view(n, m.d_model)
            h = m._add_norm(h, W["cross_out"](c), L.ln_cross)
            ff = W["fc1"](h, "gelu") if m.fuse_gelu else m.act(W["fc1"](h))
            h = m._add_norm(h, W["fc2"](ff), L.ln_final)
        logits = self.head(h)[:, : m.vocab_size]
        return logits if m.final_logits_bias is None else logits + m.final_logits_bias.to(logits.dtype)

    @torch.inference_mode()
    def score(self, requests: list[Request], targets: list[list[int]], alternatives: int = 0) -> list[TokenScores]:
        """Scores of each request's target tokens, every one given those before it (the first given
        the decoder's start token). Requests may differ in prompt and target length."""
        if len(requests) != len(targets) or not requests:
            raise ValueError(f"vflorence_b200: {len(targets)} targets for {len(requests)} requests")
        if any(not 1 <= len(t) <= self.max_decoder_len for t in targets):
            raise ValueError(f"vflorence_b200: targets must have 1 to {self.max_decoder_len} tokens")
        if any(not r.input_ids for r in requests):
            raise ValueError("vflorence_b200: a request needs at least one prompt token")
        if len({None if r.pixel_values is None else r.pixel_values.shape for r in requests}) != 1:
            raise ValueError("vflorence_b200: the requests' images must share a shape")
        m, bs, dev = self.model, self.block_size, self.model.device
        # the longest target first: the rows of a step are then the first ones
        order = sorted(range(len(targets)), key=lambda i: -len(targets[i]))
        texts = [targets[i] for i in order]
        rows, steps = len(texts), len(texts[0])
        want = torch.full((rows, steps), -1, dtype=torch.int32)
        for i, t in enumerate(texts):
            want[i, : len(t)] = torch.tensor(t, dtype=torch.int32)
        if not bool(((want >= -1) & (want < m.vocab_size)).all()) or any(min(t) < 0 for t in texts):
            raise ValueError(f"vflorence_b200: target tokens must be in [0, {m.vocab_size})")
        fed = torch.cat([torch.full((rows, 1), self.start_token), want[:, :-1].clamp(min=0)], 1).t().contiguous().to(dev)
        want = want.t().contiguous().to(dev)  # [step, row]

        cross_caches, cross_table, cross_lens, cross_host = self._page_encoder([requests[i] for i in order])
        per_row = -(-steps // bs)
        table = torch.arange(rows * per_row, dtype=torch.int32, device=dev).view(rows, per_row)
        own_caches = [_Cache(table.numel(), m.num_heads, bs, m.head_dim, dev).parts for _ in m.layers]
        starts = torch.arange(rows + 1, dtype=torch.int32, device=dev)
        lens = torch.arange(1, steps + 1, dtype=torch.int32)[:, None].expand(steps, rows).contiguous()
        lens_dev = lens.to(dev)

        parts, n, cross = [], 0, None
        for t in range(steps):
            now = sum(len(x) > t for x in texts)
            if now != n:
                n = now
                cross = (cross_caches, starts[: n + 1], cross_lens[:n], cross_table, self._plan(cross_host[:n]))
            slots = table[:n, t // bs].long() * bs + t % bs
            own = (own_caches, slots, starts[: n + 1], lens_dev[t, :n], table, self._plan(lens[t, :n]))
            logits = self._step(fed[t, :n], t, own, cross)
            parts.append(paged_ops.token_logprobs(logits, want[t, :n], alternatives))
        scores = [None] * rows
        host = [[p[j].cpu() for p in parts] for j in range(4)]
        for row, i in enumerate(order):
            scores[i] = TokenScores(*(torch.stack([host[j][t][row] for t in range(len(targets[i]))]) for j in range(4)))
        return scores
