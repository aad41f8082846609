"""End-to-end decode harness: a decoder stack whose MoE layers run on the trismoe_b200 kernels,
with fp16 attention and a KV cache around them, and the generation loop of the reference's
latency benchmark (``tools/benchmark_e2e_grid.py:325-420``, ``run_exact_generation``: exactly
``output_length`` tokens, greedy argmax inside the loop, synchronisation at phase boundaries only,
``decode_tokens_per_s = batch * decode_steps / decode_time``).

By default the attention half is plain PyTorch (``scaled_dot_product_attention`` over a preallocated
cache): the fixed fp16 context the MoE path is measured in.  The decode step has static shapes - the
cache has its full length from the start and a position tensor masks the unwritten tail - so one step
is captured into a CUDA graph and replayed ``output_length - 1`` times with no host work between steps.

With ``page_size`` the decoder runs on the operators of ``decode_ops``: keys and values go to a paged
cache (fp16 or e4m3), one new token attends over the tokens that are there and no others, and the
residual is added by the norm that follows it.  ``cache_scale_tokens`` gives an e4m3 cache a scale for each block of that
many tokens, and ``linear_dtype=torch.float8_e4m3fn`` runs the projections and the logits' product in 8 bits: the
norm's output goes into them as it is.  ``run_exact_generation`` takes ``logit_controls`` (penalties, biases, grammar
masks) and ``sampling`` (temperature, top-k, top-p, min-p) either way.
"""
from __future__ import annotations

import math
import time
from dataclasses import dataclass
from typing import List, Optional

import torch
import torch.nn.functional as F

from .decode_ops import (add_rms_norm, add_rms_norm_e4m3, append_paged_kv, apply_logit_controls, paged_decode_attention, raise_on_status,
                         sample_tokens)
from .e4m3_ops import GROUP, linear_e4m3, quantize_e4m3
from .moe_block import TrisSparseMoeBlock


@dataclass
class DecoderShape:
    hidden_size: int = 2048
    num_heads: int = 16
    head_dim: int = 128
    num_kv_heads: int = 16
    vocab_size: int = 50304
    rope_theta: float = 10000.0
    rms_eps: float = 1e-5


def _rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    return F.rms_norm(x, (x.shape[-1],), weight, eps)  # one kernel; statistics in fp32


def _rope_tables(max_length: int, head_dim: int, theta: float, device):
    """cos / sin of every (position, frequency), fp32 [max_length, head_dim / 2]."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    ang = torch.arange(max_length, device=device, dtype=torch.float32)[:, None] * inv
    return ang.cos().contiguous(), ang.sin().contiguous()


def _rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [B, heads, S, D]; cos / sin [B, 1, S, D/2] (fp32, already gathered at the tokens' positions)."""
    d = x.shape[-1]
    x1, x2 = x[..., : d // 2].float(), x[..., d // 2:].float()
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], dim=-1).to(x.dtype)


class TrisDecoder(torch.nn.Module):
    """``len(moe_blocks)`` decoder layers: RMSNorm -> attention (fp16, KV cache) -> RMSNorm -> MoE.  ``page_size``: the cache is
    paged and the layers run on ``decode_ops``; ``cache_dtype`` is fp16 or ``torch.float8_e4m3fn`` (scale 1: normalised keys and
    values are a few units large; with ``cache_scale_tokens``: one scale for each block of that many tokens and head).  ``linear_dtype``:
    ``torch.float8_e4m3fn`` holds the attention's projections and the logits' matrix in 8 bits with block scales."""

    def __init__(self, moe_blocks: List[TrisSparseMoeBlock], shape: DecoderShape, max_length: int, max_batch: int,
                 device, seed: int = 0, page_size: Optional[int] = None, cache_dtype: torch.dtype = torch.float16,
                 cache_scale_tokens: Optional[int] = None, linear_dtype: torch.dtype = torch.float16):
        super().__init__()
        self.shape, self.blocks = shape, list(moe_blocks)
        self.max_length, self.max_batch = int(max_length), int(max_batch)
        dev = torch.device(device)
        g = torch.Generator(device="cpu").manual_seed(seed)
        H, hd, nh, nkv = shape.hidden_size, shape.head_dim, shape.num_heads, shape.num_kv_heads
        rnd = lambda *s, std: (torch.randn(*s, generator=g) * std).to(dev, torch.float16)
        self.embed = rnd(shape.vocab_size, H, std=1.0)
        self.lm_head = rnd(shape.vocab_size, H, std=1.0 / math.sqrt(H))
        self.final_norm = torch.ones(H, dtype=torch.float16, device=dev)
        self.rope_cos, self.rope_sin = _rope_tables(self.max_length, hd, shape.rope_theta, dev)
        self.key_index = torch.arange(self.max_length, device=dev)[None, None, None, :]
        self.layers = []
        self.page_size = page_size
        self.scale_tokens = cache_scale_tokens
        self.linear8 = linear_dtype == torch.float8_e4m3fn
        what = "trismoe_b200 decode harness: "
        if cache_scale_tokens and (cache_dtype != torch.float8_e4m3fn or not page_size or page_size % cache_scale_tokens):
            raise RuntimeError(what + "scales of blocks belong to a paged cache in 8 bits, whose pages are whole blocks")
        if linear_dtype not in (torch.float16, torch.float8_e4m3fn) or (self.linear8 and (not page_size or H % GROUP)):
            raise RuntimeError(what + f"projections are fp16, or, with a paged cache and a hidden size that is a multiple of {GROUP}, e4m3")
        if page_size:
            width = -(-self.max_length // page_size)
            # a sequence's pages one after the other: an allocator would hand them out in any order
            self.block_table = torch.arange(max_batch * width, dtype=torch.int32, device=dev).view(max_batch, width)
            self.cache_status = torch.zeros((1,), dtype=torch.int32, device=dev)
            pages = lambda: torch.zeros((max_batch * width, nkv, page_size, hd), dtype=cache_dtype, device=dev).transpose(1, 2)
        elif cache_dtype != torch.float16:
            raise RuntimeError("trismoe_b200 decode harness: a cache in 8 bits is a paged one")
        else:
            pages = lambda: torch.zeros((max_batch, nkv, max_length, hd), dtype=torch.float16, device=dev)
        for _ in self.blocks:
            self.layers.append({
                "ln1": torch.ones(H, dtype=torch.float16, device=dev), "ln2": torch.ones(H, dtype=torch.float16, device=dev),
                "wqkv": rnd((nh + 2 * nkv) * hd, H, std=1.0 / math.sqrt(H)), "wo": rnd(H, nh * hd, std=1.0 / math.sqrt(nh * hd)),
                "k": pages(), "v": pages(),
            })
            if cache_scale_tokens:
                scales = lambda: torch.zeros((max_batch * width, page_size // cache_scale_tokens, nkv), dtype=torch.float32, device=dev)
                self.layers[-1].update(k_scale=scales(), v_scale=scales())
        if self.linear8:
            quantized = lambda w: quantize_e4m3(w, group_rows=GROUP)
            self.lm_head = quantized(self.lm_head)
            for layer in self.layers:
                layer.update(wqkv=quantized(layer["wqkv"]), wo=quantized(layer["wo"]))

    def _attention(self, layer: dict, x: torch.Tensor, positions: torch.Tensor, batch: int, rope, mask) -> torch.Tensor:
        """x [B, S, H]; positions [B, S] absolute positions of these tokens.  Writes K/V at the
        positions and attends over cache entries <= the token's own position.  ``rope`` (cos, sin at the
        positions) and ``mask`` are the same for every layer of a step and are built once per step."""
        s = self.shape
        B, S, _ = x.shape
        nq, nkv = s.num_heads, s.num_kv_heads
        qkv = F.linear(x, layer["wqkv"]).view(B, S, nq + 2 * nkv, s.head_dim).transpose(1, 2)
        qk = _rope(qkv[:, : nq + nkv], *rope)  # queries and keys rotate together
        q, k, v = qk[:, :nq], qk[:, nq:], qkv[:, nq + nkv:]
        idx = positions[:, None, :, None].expand(B, nkv, S, s.head_dim)
        layer["k"][:batch].scatter_(2, idx, k)
        layer["v"][:batch].scatter_(2, idx, v)
        keys, vals = layer["k"][:batch], layer["v"][:batch]
        if nkv != nq:
            rep = nq // nkv
            keys, vals = keys.repeat_interleave(rep, dim=1), vals.repeat_interleave(rep, dim=1)
        out = F.scaled_dot_product_attention(q, keys, vals, attn_mask=mask)
        return F.linear(out.transpose(1, 2).reshape(B, S, nq * s.head_dim), layer["wo"])

    def _linear(self, x, weight, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """``x`` as the weight takes it: rows in fp16 or, in 8 bits, those or values with their scales."""
        if not self.linear8:
            return F.linear(x, weight).to(dtype)
        return linear_e4m3(*(x if isinstance(x, tuple) else quantize_e4m3(x)), *weight, dtype=dtype, status=self.cache_status)

    def _norm(self, x: torch.Tensor, h: Optional[torch.Tensor], weight: torch.Tensor):
        """The residual norm ahead of a product: its rows as ``_linear`` takes them, and the new residual."""
        if not self.linear8:
            return add_rms_norm(x, h, weight, self.shape.rms_eps)
        values, scales, h = add_rms_norm_e4m3(x, h, weight, self.shape.rms_eps, group_size=GROUP)
        return (values, scales), h

    def _paged_attention(self, layer: dict, x, positions: torch.Tensor, sequences, lengths, mask) -> torch.Tensor:
        """The same over pages.  One new token per sequence attends through the block table; several (a prompt) over the pages
        gathered to the dense form."""
        s = self.shape
        B, S = positions.shape
        nq, nkv, hd = s.num_heads, s.num_kv_heads, s.head_dim
        qkv = self._linear(x, layer["wqkv"]).view(B * S, nq + 2 * nkv, hd)
        table = self.block_table[:B]
        scales = {name: layer.get(name) for name in ("k_scale", "v_scale")}
        q = append_paged_kv(qkv[:, :nq], qkv[:, nq: nq + nkv], qkv[:, nq + nkv:], layer["k"], layer["v"], table, positions.reshape(-1), sequences,
                            cos=self.rope_cos, sin=self.rope_sin, status=self.cache_status, **scales)
        if S == 1:
            out = paged_decode_attention(q, layer["k"], layer["v"], table, lengths, status=self.cache_status, **scales)
        else:
            def dense(pages, scale):
                rows = pages[table]
                if scale is not None:
                    rows = rows.float() * scale[table].repeat_interleave(self.scale_tokens, 2)[..., None]
                return rows.reshape(B, -1, nkv, hd)[:, : self.max_length].transpose(1, 2).to(q.dtype).repeat_interleave(nq // nkv, dim=1)

            k, v = dense(layer["k"], scales["k_scale"]), dense(layer["v"], scales["v_scale"])
            out = F.scaled_dot_product_attention(q.view(B, S, nq, hd).transpose(1, 2), k, v, attn_mask=mask).transpose(1, 2)
        return self._linear(out.reshape(B, S, nq * hd), layer["wo"])

    def _paged_forward(self, token_ids: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        B, S = token_ids.shape
        eps, h = self.shape.rms_eps, F.embedding(token_ids, self.embed)
        sequences = lengths = mask = None
        if S == 1:
            lengths = positions[:, 0].to(torch.int32) + 1
        else:
            sequences = torch.arange(B, dtype=torch.int32, device=h.device).repeat_interleave(S)
            mask = self.key_index <= positions[:, None, :, None]
        x, _ = self._norm(h, None, self.layers[0]["ln1"])
        for i, (layer, blk) in enumerate(zip(self.layers, self.blocks)):
            x, h = add_rms_norm(self._paged_attention(layer, x, positions, sequences, lengths, mask), h, layer["ln2"], eps)
            y, _ = blk(x)
            x, h = self._norm(y, h, self.layers[i + 1]["ln1"] if i + 1 < len(self.layers) else self.final_norm)
        last = tuple(part[:, -1] for part in x) if self.linear8 else x[:, -1]
        return self._linear(last, self.lm_head, torch.float32)

    def raise_on_kernel_status(self) -> None:
        """Raises if a paged operator met a page, position or length that does not fit, or a product in 8 bits gave up a wait: its logits are NaN then, and a token
        drawn from them is 0 (waits for the GPU)."""
        if self.page_size:
            raise_on_status(self.cache_status)

    def forward(self, token_ids: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """token_ids, positions [B, S] -> logits of the last position [B, vocab] (fp32)."""
        if self.page_size and self.layers:
            return self._paged_forward(token_ids, positions)
        B, S = token_ids.shape
        h = F.embedding(token_ids, self.embed)
        rope = (self.rope_cos[positions][:, None], self.rope_sin[positions][:, None])  # [B, 1, S, D/2]
        mask = self.key_index <= positions[:, None, :, None]
        for layer, blk in zip(self.layers, self.blocks):
            h = h + self._attention(layer, _rms_norm(h, layer["ln1"], self.shape.rms_eps), positions, B, rope, mask)
            y, _ = blk(_rms_norm(h, layer["ln2"], self.shape.rms_eps))
            h = h + y
        last = _rms_norm(h[:, -1], self.final_norm, self.shape.rms_eps)
        return self._linear(last, self.lm_head, torch.float32)


def run_exact_generation(model: TrisDecoder, input_ids: torch.Tensor, output_length: int, use_graph: bool = True,
                         measure_latency: bool = True, logit_controls: Optional[dict] = None, sampling: Optional[dict] = None) -> dict:
    """Prefill ``input_ids`` [B, L], then generate exactly ``output_length`` tokens, greedily or drawn.  Returns the
    reference benchmark's fields (prefill_ms, decode_ms, decode_tokens_per_s, ...) and the tokens.  ``logit_controls``: arguments of
    ``apply_logit_controls`` (``repetition``, ``presence``, ``frequency``, ``bias_ids``, ``bias_values``, ``allowed``) for every step; the
    history of prompt and answer is kept here.  ``sampling``: ``random`` (fp32 [output_length, B], a row for each step) and arguments of
    ``sample_tokens`` (``temperature``, ``top_k``, ``top_p``, ``min_p``); a sequence none of whose tokens can be drawn gets token 0."""
    dev = input_ids.device
    B, L = (int(v) for v in input_ids.shape)
    if L + output_length > model.max_length or B > model.max_batch:
        raise RuntimeError("trismoe_b200 decode harness: cache too small for this prompt / output length / batch")
    decode_steps = max(output_length - 1, 0)
    sync = lambda: torch.cuda.synchronize(dev)
    positions = torch.arange(L, device=dev)[None, :].expand(B, L).contiguous()
    step_index = torch.zeros((1,), dtype=torch.long, device=dev)
    history = known = prompt = None
    if logit_controls is not None:
        history = F.pad(input_ids, (0, output_length)).to(torch.int32)
        known = torch.full((B,), L, dtype=torch.int32, device=dev)
        prompt = known.clone()

    random = None
    if sampling is not None:
        sampling = dict(sampling)
        random = sampling.pop("random", None)
        if random is None or random.shape != (output_length, B) or random.dtype is not torch.float32:
            raise RuntimeError(f"trismoe_b200 decode harness: sampling needs random numbers, fp32 [{output_length}, {B}]")

    def pick(logits):
        if random is None:
            return logits.argmax(dim=-1, keepdim=True)
        return sample_tokens(logits, random.index_select(0, step_index).view(B), **sampling).clamp_(min=0)[:, None]

    def choose(logits):
        """Token [B, 1] under the controls, noted in the history."""
        if history is None:
            return pick(logits)
        chosen = pick(apply_logit_controls(logits, tokens=history, token_lengths=known, prompt_lengths=prompt, out=logits, **logit_controls))
        history.index_copy_(1, step_index + L, chosen.to(torch.int32))
        known.add_(1)
        return chosen

    sync()
    t0 = time.perf_counter()
    with torch.no_grad():
        logits = model(input_ids, positions)
    sync()
    t1 = time.perf_counter()
    tokens = torch.empty((B, output_length), dtype=torch.long, device=dev)
    cur = choose(logits)  # [B, 1]
    pos = torch.full((B, 1), L, dtype=torch.long, device=dev)
    tokens[:, 0:1] = cur
    step_index.fill_(1)

    def step():
        with torch.no_grad():
            nxt = choose(model(cur, pos))
            cur.copy_(nxt)
            tokens.index_copy_(1, step_index, nxt)
            pos.add_(1)
            step_index.add_(1)

    graph = None
    if use_graph and decode_steps > 1:
        # warm up on a side stream with the state restored afterwards, then capture one step
        state = (cur, pos, step_index, tokens) + (() if history is None else (history, known))
        saved = tuple(t.clone() for t in state)
        side = torch.cuda.Stream(device=dev)
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream(dev).wait_stream(side)
        sync()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for dst, src in zip(state, saved):
            dst.copy_(src)
    sync()
    t2 = time.perf_counter()
    for _ in range(decode_steps):
        if graph is not None:
            graph.replay()
        else:
            step()
    sync()
    t3 = time.perf_counter()
    prefill_ms, decode_ms = (t1 - t0) * 1e3, (t3 - t2) * 1e3
    out = {"batch_size": B, "input_length": L, "output_length": output_length, "decode_steps": decode_steps, "tokens": tokens,
           "launch_mode": "cuda graph" if graph is not None else "eager"}
    if measure_latency:
        out.update({
            "prefill_ms": prefill_ms, "decode_ms": decode_ms,
            "avg_decode_step_ms": decode_ms / decode_steps if decode_steps else 0.0,
            "prefill_tokens_per_s": B * L * 1e3 / prefill_ms,
            "decode_tokens_per_s": B * decode_steps * 1e3 / decode_ms if decode_steps and decode_ms > 0 else 0.0,
        })
    return out
