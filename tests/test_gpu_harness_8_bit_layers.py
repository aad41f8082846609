"""GPU tests of the decode harness in 8 bits, layer by layer against 64 bits: what a layer's attention makes of the rows that it gets, what it leaves in the cache, and the logits of the rows
that the last norm gives.  A wrong scale - one block of a projection's, one block of the cache's - does not pass, which is shown with the oracle's.

Bounds.  A key or value in the cache: half a step of e4m3 (2^-4 of it, 2^-10 of its block's scale), ahead of it a rounding to 16 bits (2^-11) of each of the pair that rotates; in fp16
the latter alone.  Attention's result behind its projection, relative to its length: in 16 bits four roundings of rows and weights, 2^-8; in 8 bits each of the projection's
inputs is off by 2^-4 at most, so a random matrix's product is by 2^-4 of its length, and a quarter of that again for rows of 256 of them.  Products of rows in 8 bits: sums of 256 exact products
in 32 bits with two scales, 2^-18 of the sum of magnitudes."""
import math

import pytest
import torch

from test_gpu_paged_decode import _ids, _model

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _weight(w, wrong=1.0):
    """A projection's matrix in 64 bits; ``wrong``: what the scale of its last block is off by."""
    if not isinstance(w, tuple):
        return w.double()
    values, scales = w
    scales = scales.double().clone()
    scales[-1, -1] *= wrong
    return values.double() * scales.repeat_interleave(128, 0)[: values.shape[0]].repeat_interleave(128, 1)[:, : values.shape[1]]


def _rows(x):
    if not isinstance(x, tuple):
        return x.double()
    values, scales = x
    return values.double() * scales.double().repeat_interleave(128, -1)[..., : values.shape[-1]]


class Oracle:
    """Watches a decoder's attention and products; ``worst``: the largest error of each kind, as a share of its bound."""

    def __init__(self, model, wqkv=1.0, wo=1.0, k_scale=1.0, v_scale=1.0):
        self.model, self.wrong = model, dict(wqkv=wqkv, wo=wo, k_scale=k_scale, v_scale=v_scale)
        self.worst = {"cache": 0.0, "attention": 0.0, "product": 0.0}
        self.attention, self.linear = model._paged_attention, model._linear
        model._paged_attention, model._linear = self.watch_attention, self.watch_linear

    def note(self, kind, share):
        share = float(share.max())
        self.worst[kind] = max(self.worst[kind], math.inf if math.isnan(share) else share)

    def watch_linear(self, x, weight, dtype=torch.float16):
        out = self.linear(x, weight, dtype)
        if isinstance(x, tuple):
            rows, w = _rows(x), _weight(weight)
            want, size = rows @ w.T, rows.abs() @ w.abs().T
            rounding = 2.0 ** -11 if dtype is torch.float16 else 2.0 ** -24
            self.note("product", (out.double() - want).abs() / (rounding * want.abs() + 2.0 ** -18 * size + 2.0 ** -25))
        return out

    def cache(self, layer, name, batch, length):
        """[batch, length, heads, head_dim] of what a layer's pages hold, and each token's scale."""
        m = self.model
        pos = torch.arange(length, device="cuda")
        at, slot = m.block_table[:batch, pos // m.page_size].long(), pos % m.page_size
        rows = layer[name][at, slot].double()
        if name + "_scale" not in layer:
            return rows, torch.zeros_like(rows[..., :1])
        scale = layer[name + "_scale"][at, slot // m.scale_tokens].double()[..., None]
        scale[:, -1] *= self.wrong[name + "_scale"]
        return rows * scale, scale

    def watch_attention(self, layer, x, positions, sequences, lengths, mask):
        out = self.attention(layer, x, positions, sequences, lengths, mask)
        m, s, (batch, S) = self.model, self.model.shape, positions.shape
        nq, nkv, hd = s.num_heads, s.num_kv_heads, s.head_dim
        qkv = (_rows(x) @ _weight(layer["wqkv"], self.wrong["wqkv"]).T).view(batch, S, nq + 2 * nkv, hd)
        cos, sin = m.rope_cos[positions].double()[:, :, None], m.rope_sin[positions].double()[:, :, None]
        a, b = qkv[:, :, : nq + nkv, : hd // 2], qkv[:, :, : nq + nkv, hd // 2:]
        qk, pair = torch.cat([a * cos - b * sin, b * cos + a * sin], -1), (a.abs() + b.abs()).repeat(1, 1, 1, 2)
        q, v = qk[:, :, :nq], qkv[:, :, nq + nkv:]
        length, where = int(positions.max()) + 1, positions[..., None, None].expand(batch, S, nkv, hd)
        held = {name: self.cache(layer, name, batch, length) for name in "kv"}
        for name, want, mag in (("k", qk[:, :, nq:], pair[:, :, nq:]), ("v", v, v.abs())):
            rows, scale = held[name]
            step = 2.0 ** -4 * want.abs() + 2.0 ** -10 * scale.gather(1, where[..., :1]) if layer[name].dtype is E4M3 else 0.0
            self.note("cache", (rows.gather(1, where) - want).abs() / (step + 2.0 ** -10 * mag + 2.0 ** -20))
        keys, values = (held[name][0].repeat_interleave(nq // nkv, 2) for name in "kv")
        score = torch.einsum("bshd,bthd->bhst", q, keys) / math.sqrt(hd)
        score = score.masked_fill(torch.arange(length, device="cuda") > positions[:, None, :, None], -math.inf)
        rows = torch.einsum("bhst,bthd->bshd", torch.softmax(score, -1), values).reshape(batch, S, nq * hd)
        want = rows @ _weight(layer["wo"], self.wrong["wo"]).T
        self.note("attention", (out.double() - want).norm(dim=-1) / want.norm(dim=-1) / (1.25 * 2.0 ** -4 if m.linear8 else 2.0 ** -8))
        return out


def _steps(tm, oracle=None, **more):
    model, _ = _model(tm, page_size=16, cache_dtype=E4M3 if "cache_scale_tokens" in more else torch.float16, **more)
    watch = Oracle(model, **(oracle or {}))
    ids, pos = _ids(3, 19)
    with torch.no_grad():
        model(ids, pos)
        for step in range(6):
            model(torch.full((3, 1), 7 + step, device="cuda"), torch.full((3, 1), 19 + step, device="cuda"))
    model.raise_on_kernel_status()
    return watch.worst


@pytest.mark.parametrize("more", [dict(cache_scale_tokens=16), dict(cache_scale_tokens=1), dict(linear_dtype=E4M3), dict(cache_scale_tokens=8, linear_dtype=E4M3)],
                         ids=["blocks", "tokens", "linear", "both"])
def test_every_layer_against_64_bits(lib, more):
    import trismoe_b200 as tm

    worst = _steps(tm, **more)
    assert max(worst.values()) <= 1.0, worst
    assert worst["cache"] > 0 and worst["attention"] > 0 and (worst["product"] > 0) == ("linear_dtype" in more)


@pytest.mark.parametrize("wrong,kind", [(dict(wqkv=1.5), "cache"), (dict(wo=1.5), "attention"), (dict(k_scale=2.0), "cache"), (dict(v_scale=0.5), "cache")], ids=lambda v: str(v))
def test_a_wrong_scale_is_seen(lib, wrong, kind):
    """The oracle's last block of a projection, or last token's scale, is off."""
    import trismoe_b200 as tm

    worst = _steps(tm, wrong, cache_scale_tokens=8, linear_dtype=E4M3)
    assert worst[kind] > 1.5, worst
