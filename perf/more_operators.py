"""Timed workloads of a decode step in 8 bits: rows are brought to e4m3 with a scale for each group of 128, multiplied by weights
with a scale for each block of 128 x 128, new keys and values go into a cache in e4m3 with a scale for each block of tokens and
head, one new token a sequence attends over that cache, and a token is drawn from the logits.

``listed()`` names the workloads, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds
before the call, ``run`` is one pass - in elementary torch operations, or with ``own`` set through the framework's entry
points -, ``exact`` the same from the definition in 64 bits and ``work`` what a pass cannot do without.  All data is
synthetic and made on the GPU from the seed.
"""
import math

import torch

own = False

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
GROUP = 128
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4}
# query heads, key/value heads, head size and rotated dimensions of the models of the benchmark and the tests
HEADS = {"olmoe": (16, 16, 128, 128), "mixtral": (32, 8, 128, 128), "qwen35": (16, 2, 256, 64), "small": (4, 2, 64, 64)}


# ---------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------
def _linear(rows, inputs, outputs, dtype, bias=False):
    return {"kind": "linear", "rows": rows, "inputs": inputs, "outputs": outputs, "dtype": dtype, "bias": bias}


def _quantize(rows, columns, dtype, group_rows=1):
    return {"kind": "quantize", "rows": rows, "columns": columns, "dtype": dtype, "group_rows": group_rows}


def _append(model, batch, tokens, dtype, page=16, block=16, interleaved=False):
    return {"kind": "append", "model": model, "batch": batch, "tokens": tokens, "dtype": dtype, "page": page, "block": block,
            "interleaved": interleaved}


def _attend(model, batch, longest, dtype, page=16, block=16, ragged=1.0, empty=False, window=0, lse=False):
    return {"kind": "attend", "model": model, "batch": batch, "longest": longest, "dtype": dtype, "page": page, "block": block,
            "ragged": ragged, "empty": empty, "window": window, "lse": lse}


def _sample(batch, vocab, dtype, spread, top_k, top_p, min_p, greedy=False, masked=False):
    return {"kind": "sample", "batch": batch, "vocab": vocab, "dtype": dtype, "spread": spread, "top_k": top_k, "top_p": top_p,
            "min_p": min_p, "greedy": greedy, "masked": masked}


def listed():
    cases = {
        # queries, keys and values of one conversation's new token: the weights' bytes, and latency
        "linear 1 x 2048 to 6144": _linear(1, 2048, 6144, "fp16"),
        # logits of 64 sequences, in 32 bits for the choice of a token
        "linear 64 x 4096 to 32000": _linear(64, 4096, 32000, "fp32"),
        # a prompt of odd length on its way through the attention's projection, with a bias
        "linear 509 x 2048 to 6144": _linear(509, 2048, 6144, "bf16", bias=True),
        # four prompts of 2048 tokens through a wide layer: the tensor cores' rate
        "linear 8192 x 4096 to 14336": _linear(8192, 4096, 14336, "bf16"),
        # attention's results of 64 sequences on their way into the output projection
        "quantize 64 x 2048": _quantize(64, 2048, "fp16"),
        # a layer's weights, a scale for each block of 128 x 128
        "quantize 14336 x 4096 blocks": _quantize(14336, 4096, "bf16", group_rows=GROUP),
        # a decode step of 64 sequences
        "append 64": _append("mixtral", 64, 64, "bf16"),
        # four prompts of some 2000 tokens on their way into the cache
        "append 4 x 2047": _append("olmoe", 4, 8188, "fp16"),
        # one conversation behind a prompt of 512 tokens
        "attend 1 x 513": _attend("olmoe", 1, 513, "fp16"),
        # a server under load: 64 sequences of very different lengths, some slots of the batch free
        "attend 64 x 1-16384": _attend("mixtral", 64, 16384, "bf16", page=64, block=32, ragged=0.0, empty=True, lse=True),
        # one conversation with the usual controls
        "sample 1 x 50304": _sample(1, 50304, "fp32", 3.0, 50, 0.9, 0.0),
        # a large batch: long and short tails, some sequences greedy, half of the vocabulary closed by a grammar
        "sample 128 x 50304": _sample(128, 50304, "fp32", 2.0, 0, 0.95, 0.02, greedy=True, masked=True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, low, high):
    return min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "quantize", "append", "attend", "attend", "sample", "sample"])
    dtype = rng.choice(["fp16", "bf16"])
    if kind == "linear":
        inputs = rng.choice([256, 2048, 4096, 14336, 16 * _log_int(rng, 1, 512)])
        outputs = rng.choice([1024, 2048, 4096, 6144, 32000, _log_int(rng, 1, 32000)])
        most = max(1, min(8192, 8192 * 4096 * 14336 // (inputs * outputs)))
        return _linear(_log_int(rng, 1, most), inputs, outputs, rng.choice(["fp16", "bf16", "fp32"]), rng.random() < 0.25)
    if kind == "quantize":
        return _quantize(_log_int(rng, 1, 8192), rng.choice([256, 2048, 4096, _log_int(rng, 1, 7168)]), dtype, rng.choice([1, 1, GROUP]))
    if kind == "sample":
        vocab = rng.choice([512, 32000, 50304, _log_int(rng, 2, 200000)])
        return _sample(_log_int(rng, 1, min(128, max(1, 128 * 50304 // vocab))), vocab, rng.choice(["fp16", "bf16", "fp32"]),
                       rng.choice([0.5, 2.0, 3.0, 5.0]), rng.choice([0, 0, 1, 20, 50, 1000]), rng.choice([1.0, 0.5, 0.9, 0.95, 0.999]),
                       rng.choice([0.0, 0.0, 0.02, 0.1]), rng.random() < 0.25, rng.random() < 0.25)
    model = rng.choice(list(HEADS))
    page = rng.choice([1, 8, 16, 16, 16, 32, 48, 64, 128])
    block = rng.choice([b for b in (1, 8, 16, 32, 48, 64, 128) if page % b == 0])
    batch = _log_int(rng, 1, 64)
    if kind == "append":
        tokens = batch if rng.random() < 0.5 else batch * _log_int(rng, 1, 8192 // batch)
        return _append(model, batch, tokens, dtype, page, block, rng.random() < 0.25)
    most = min(131071, 64 * 8192 * 8 * 128 // (batch * HEADS[model][1] * HEADS[model][2]))
    return _attend(model, batch, _log_int(rng, 1, most), dtype, page, block, rng.choice([0.0, 0.5, 0.9, 1.0]), rng.random() < 0.25,
                   rng.choice([0, 0, 0, 1000]), rng.random() < 0.25)


def _lengths(case):
    """Cached tokens of every sequence: from ``ragged`` times the longest to the longest, spread evenly in an order of their own;
    with ``empty`` every eighth place of the batch is free."""
    low = case["ragged"] * case["longest"]
    spread = [(0.618034 * (i + 1)) % 1.0 for i in range(case["batch"])]
    lengths = [max(1, int(low + (case["longest"] - low) * f)) for f in spread]
    lengths[0] = case["longest"]
    return [0 if case["empty"] and i % 8 == 7 else n for i, n in enumerate(lengths)]


def _starts(case):
    """Where every sequence's new tokens begin: decode steps stand at different places of their contexts, prompts begin at 0."""
    new = case["tokens"] // case["batch"]
    return new, [0 if new > 1 else (997 * i + 511) % 4096 for i in range(case["batch"])]


# ---------------------------------------------------------------------------------------
# what a program holds before the call
# ---------------------------------------------------------------------------------------
def _normal(g, std, *shape):
    return torch.randn(shape, generator=g, device=g.device) * std


def _uniform(g, low, high, *shape):
    return low + (high - low) * torch.rand(shape, generator=g, device=g.device)


def _coded(g, std, *shape):
    """Numbers in e4m3, as they are in a matrix or cache whose scales leave them that large."""
    out = torch.empty(shape, dtype=FP8, device=g.device)
    for part in out.split(max(1, (1 << 26) // max(1, out[:1].numel()))):
        part.copy_(_normal(g, std, *part.shape).clamp(-FP8_MAX, FP8_MAX))
    return out


def _pages(g, case, pages):
    """One cache: [pages, tokens of a page, heads, head size], a head's tokens of a page side by side in memory, and the scales of its
    blocks, powers of two that leave numbers around 1."""
    _, kv, d, _ = HEADS[case["model"]]
    blocks = case["page"] // case["block"]
    scales = torch.exp2(torch.randint(-8, -5, (pages, blocks, kv), generator=g, device=g.device).float())
    return _coded(g, 100.0, pages, kv, case["page"], d).transpose(1, 2), scales


def _tables(g, counts, spare=3):
    """Block table of sequences with that many pages each, the pages in no order; -1 behind a sequence's last page."""
    total = sum(counts) + spare
    order = torch.randperm(total, generator=g, device=g.device).to(torch.int32)
    width = max(1, max(counts))
    count = torch.tensor(counts, device=g.device)
    first = count.cumsum(0) - count
    column = torch.arange(width, device=g.device)
    table = order[(first[:, None] + column).clamp(max=total - 1)]
    return torch.where(column < count[:, None], table, -1).contiguous(), total


def _rotation(case, positions, device):
    rot = HEADS[case["model"]][3]
    inv = 1.0 / (10000.0 ** (torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot))
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, kind, state = g.device, case["kind"], {"case": case}
    dtype = DTYPES[case["dtype"]]
    if kind == "linear":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        groups = -(-inputs // GROUP)
        state["x"], state["weight"] = _coded(g, 150.0, rows, inputs), _coded(g, 100.0, outputs, inputs)
        # a few groups of columns hold outliers, so theirs are large
        state["x_scales"] = _uniform(g, 0.5, 1.5, rows, groups) / 150.0 * torch.where(torch.rand((groups,), generator=g, device=dev) < 0.05, 10.0, 1.0)
        state["weight_scales"] = _uniform(g, 0.8, 1.2, -(-outputs // GROUP), groups) / (100.0 * math.sqrt(inputs))
        state["bias"] = _normal(g, 0.5, outputs) if case["bias"] else None
    elif kind == "quantize":
        x = _normal(g, 1.0, case["rows"], case["columns"])
        x[:, torch.randperm(case["columns"], generator=g, device=dev)[: max(1, case["columns"] // 100)]] *= 20.0
        state["x"] = x.to(dtype)
    elif kind == "append":
        hq, kv, d, _ = HEADS[case["model"]]
        new, begin = _starts(case)
        state["table"], total = _tables(g, [-(-(b + new) // case["page"]) for b in begin])
        (state["k_pages"], state["k_scale"]), (state["v_pages"], state["v_scale"]) = _pages(g, case, total), _pages(g, case, total)
        qkv = _normal(g, 1.0, case["tokens"], hq + 2 * kv, d).to(dtype)  # as one projection leaves them
        state["q"], state["k"], state["v"] = qkv[:, :hq], qkv[:, hq: hq + kv], qkv[:, hq + kv:]
        state["sequences"] = torch.arange(case["batch"], device=dev, dtype=torch.int32).repeat_interleave(new)
        state["positions"] = (torch.tensor(begin, device=dev)[:, None] + torch.arange(new, device=dev)).reshape(-1)
        state["cos"], state["sin"] = _rotation(case, max(begin) + new, dev)
    elif kind == "attend":
        hq, _, d, _ = HEADS[case["model"]]
        lengths = _lengths(case)
        state["table"], total = _tables(g, [-(-n // case["page"]) for n in lengths])
        (state["k_pages"], state["k_scale"]), (state["v_pages"], state["v_scale"]) = _pages(g, case, total), _pages(g, case, total)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        state["q"] = _normal(g, 2.0, case["batch"], hq, d).to(dtype)
    else:
        batch, vocab = case["batch"], case["vocab"]
        logits = _normal(g, case["spread"], batch, vocab)
        if case["masked"]:
            closed = torch.rand((vocab,), generator=g, device=dev) < 0.5
            closed[0] = False
            logits = logits.masked_fill(closed, -math.inf)
        state["logits"] = logits.to(dtype)
        state["random"] = torch.rand((batch,), generator=g, device=dev)
        state["temperature"] = _uniform(g, 0.6, 1.2, batch)
        if case["greedy"]:
            state["temperature"][1::8] = 0.0
        state["top_k"] = state["top_p"] = state["min_p"] = None
        if case["top_k"]:
            state["top_k"] = torch.full((batch,), case["top_k"], dtype=torch.int32, device=dev)
            state["top_k"][2::4] *= 2
        if case["top_p"] < 1.0:
            state["top_p"] = 1.0 - (1.0 - case["top_p"]) * _uniform(g, 0.5, 1.0, batch)
        if case["min_p"]:
            state["min_p"] = case["min_p"] * _uniform(g, 0.5, 1.0, batch)
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    with torch.no_grad():
        return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


def _own_linear(s):
    import trismoe_b200 as tm

    return tm.linear_e4m3(s["x"], s["x_scales"], s["weight"], s["weight_scales"], s["bias"], dtype=DTYPES[s["case"]["dtype"]])


def _own_quantize(s):
    import trismoe_b200 as tm

    return tm.quantize_e4m3(s["x"], group_rows=s["case"]["group_rows"])


def _own_append(s):
    import trismoe_b200 as tm

    q = tm.append_paged_kv(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["positions"], s["sequences"],
                           cos=s["cos"], sin=s["sin"], interleaved=s["case"]["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _own_attend(s):
    import trismoe_b200 as tm

    case = s["case"]
    return tm.paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], window=case["window"],
                                     k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=case["lse"])


def _own_sample(s):
    import trismoe_b200 as tm

    return tm.sample_tokens(s["logits"], s["random"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])


def _spread(scales, rows, columns, group_rows):
    """A scale for every element of a matrix."""
    return scales.repeat_interleave(group_rows, 0)[:rows].repeat_interleave(GROUP, 1)[:, :columns]


def _plain_linear(s):
    rows, outputs, inputs = s["x"].shape[0], *s["weight"].shape
    x = s["x"].float() * _spread(s["x_scales"], rows, inputs, 1)
    weight = s["weight"].float() * _spread(s["weight_scales"], outputs, inputs, GROUP)
    y = x @ weight.T
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(DTYPES[s["case"]["dtype"]])


def _plain_quantize(s):
    (rows, columns), tall = s["x"].shape, s["case"]["group_rows"]
    down, across = -(-rows // tall), -(-columns // GROUP)
    x = torch.zeros((down * tall, across * GROUP), device=s["x"].device)
    x[:rows, :columns] = s["x"].float()
    parts = x.view(down, tall, across, GROUP)
    scales = parts.abs().amax((1, 3), keepdim=True) / FP8_MAX
    values = (parts / scales.masked_fill(scales == 0, 1.0)).clamp(-FP8_MAX, FP8_MAX).view(x.shape)
    return values[:rows, :columns].to(FP8), scales.view(down, across)


def _rotate(x, cos, sin, interleaved):
    """x [tokens, heads, head size] in 32 bits; cos and sin [tokens, rotated dimensions / 2]."""
    half = cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    rest = x[..., 2 * half:]
    if interleaved:
        a, b = x[..., : 2 * half: 2], x[..., 1: 2 * half: 2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half: 2 * half]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, rest], dim=-1)


def _power_of_two(top):
    """The smallest power of two, from 2^-64 to 2^64, by which numbers up to ``top`` fit e4m3."""
    mantissa, exponent = torch.frexp(top / FP8_MAX)  # top / 448 = mantissa * 2^exponent, mantissa from 0.5 to below 1
    exponent = torch.where(mantissa == 0.5, exponent - 1, exponent)
    return torch.exp2(exponent.clamp(-64, 64).float().masked_fill(top == 0, -64.0))


def _plain_append(s):
    case, positions = s["case"], s["positions"]
    page_size, size = case["page"], case["block"]
    cos, sin = s["cos"][positions], s["sin"][positions]
    q = _rotate(s["q"].float(), cos, sin, case["interleaved"]).to(s["q"].dtype)
    k = _rotate(s["k"].float(), cos, sin, case["interleaved"])
    page = s["table"][s["sequences"].long(), positions // page_size].long()
    slot = positions % page_size
    blocks = page_size // size
    block = page * blocks + slot // size
    for name, new in (("k", k), ("v", s["v"].float())):
        pages, scales = s[name + "_pages"], s[name + "_scale"]
        kv = pages.shape[2]
        held = scales.view(-1, kv)
        # a block whose first token is among the new ones begins anew; another one keeps its scale, or takes a larger one
        begun = torch.zeros((held.shape[0],), dtype=torch.bool, device=held.device)
        begun[block[slot % size == 0]] = True
        touched = block.unique()
        top = torch.zeros_like(held).index_reduce_(0, block, new.abs().amax(-1), "amax")
        need = _power_of_two(top[touched])
        old = held[touched]
        scale = torch.where(begun[touched][:, None], need, torch.maximum(need, old))
        # what such a block holds already is brought to its new scale
        within = torch.arange(size, device=held.device)
        where, slots = (touched // blocks)[:, None], (touched % blocks)[:, None] * size + within
        first = torch.full((held.shape[0],), size, device=held.device).index_reduce_(0, block, slot % size, "amin")[touched]
        before = (within < first[:, None])[:, :, None, None]
        values = pages[where, slots].float()
        values = torch.where(before, values * (old / scale)[:, None, :, None], values)
        pages[where, slots] = values.clamp(-FP8_MAX, FP8_MAX).to(FP8)
        held[touched] = scale
        pages[page, slot] = (new / held[block][:, :, None]).clamp(-FP8_MAX, FP8_MAX).to(FP8)
    return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _plain_attend(s):
    case, q = s["case"], s["q"].float()
    (batch, hq, d), kv, page = q.shape, s["k_pages"].shape[2], case["page"]
    pages = s["table"].clamp(min=0).long()
    length = s["lengths"][:, None]
    place = torch.arange(pages.shape[1] * page, device=q.device)
    valid = place < length
    if case["window"]:
        valid = valid & (place >= length - case["window"])

    def dense(name):
        scales = s[name + "_scale"][pages].repeat_interleave(case["block"], 2).reshape(batch, -1, kv, 1)
        return s[name + "_pages"][pages].reshape(batch, -1, kv, d).float() * scales

    k = dense("k")
    score = torch.einsum("bhgd,bthd->bhgt", q.view(batch, kv, hq // kv, d), k) * d ** -0.5
    del k
    score = score.masked_fill(~valid[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)  # a sequence without tokens has no largest score
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    out = torch.einsum("bhgt,bthd->bhgd", weight, dense("v")) / total.masked_fill(total == 0, 1.0)
    out = out.reshape(batch, hq, d).to(s["q"].dtype)
    if not case["lse"]:
        return out
    return out, torch.where(total == 0, -math.inf, top + total.log()).reshape(batch, hq)


def _plain_sample(s):
    # sums of up to 200000 weights, and a number that falls between two of them: in 64 bits
    z, order = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True)
    temperature = s["temperature"].double()[:, None]
    greedy = temperature <= 0
    weight = torch.exp((z - z[:, :1]) / torch.where(greedy, 1.0, temperature))
    rank = torch.arange(z.shape[1], device=z.device)
    kept = torch.isfinite(z) & ~(greedy & (rank > 0))
    if s["top_k"] is not None:
        kept = kept & ((s["top_k"][:, None] <= 0) | (rank < s["top_k"][:, None]))
    weight = weight * kept
    if s["top_p"] is not None:
        sums = weight.cumsum(-1)
        p = s["top_p"].double()[:, None]
        kept = kept & ((p >= 1) | (rank == 0) | (sums - weight < p * sums[:, -1:]))
    if s["min_p"] is not None:
        kept = kept & (weight >= s["min_p"].double()[:, None].clamp(max=1.0))
    weight = torch.zeros_like(weight).scatter(1, order, weight * kept)  # in the vocabulary's order again
    sums = weight.cumsum(-1)
    return (sums > s["random"].double()[:, None] * sums[:, -1:]).to(torch.uint8).argmax(-1)


_PLAIN = {"linear": _plain_linear, "quantize": _plain_quantize, "append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}
_OWN = {"linear": _own_linear, "quantize": _own_quantize, "append": _own_append, "attend": _own_attend, "sample": _own_sample}


# ---------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s)


def _exact_linear(s):
    outputs, inputs = s["weight"].shape
    y = torch.zeros((s["x"].shape[0], outputs), dtype=torch.float64, device=s["x"].device)
    for i in range(0, inputs, GROUP):  # y[t, n] = sum over groups of a row's scale * a block's scale * the product of what is held
        x = s["x"][:, i: i + GROUP].double() * s["x_scales"][:, i // GROUP, None].double()
        for n in range(0, outputs, 8192):
            scale = s["weight_scales"][n // GROUP: -(-(n + 8192) // GROUP), i // GROUP].double().repeat_interleave(GROUP)
            w = s["weight"][n: n + 8192, i: i + GROUP].double()
            y[:, n: n + 8192].addmm_(x, (w * scale[: w.shape[0], None]).T)
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_quantize(s):
    x, tall = s["x"].double(), s["case"]["group_rows"]
    rows, columns = x.shape
    scales = torch.zeros((-(-rows // tall), -(-columns // GROUP)), dtype=torch.float64, device=x.device)
    strips = [part.abs().amax(1) for part in x.split(GROUP, 1)]
    for j, strip in enumerate(strips):
        padded = torch.nn.functional.pad(strip, (0, scales.shape[0] * tall - rows))
        scales[:, j] = padded.unflatten(0, (-1, tall)).amax(1) / FP8_MAX
    at = torch.arange(rows, device=x.device) // tall
    for j in range(scales.shape[1]):
        part, scale = x[:, j * GROUP: (j + 1) * GROUP], scales[at, j][:, None]
        part.copy_(torch.where(scale > 0, part / scale, 0.0))
    return x, scales


def _exact_append(s):
    case, positions = s["case"], s["positions"]
    size, page_size = case["block"], case["page"]
    rot = 2 * s["cos"].shape[1]
    turn = torch.complex(s["cos"][positions].double(), s["sin"][positions].double())[:, None]

    def rotated(x):
        x = x.double().clone()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    page = s["table"].long()[s["sequences"].long(), positions // page_size]
    slot = positions % page_size
    results = []
    for new, pages, scales in ((rotated(s["k"]), s["k_pages"], s["k_scale"]), (s["v"].double(), s["v_pages"], s["v_scale"])):
        held, scales = pages.double(), scales.double()
        # the tokens of a block follow one another: runs begin where the block changes
        block = page * (page_size // size) + slot // size
        begins = torch.ones_like(block, dtype=torch.bool)
        begins[1:] = block[1:] != block[:-1]
        run_of = begins.cumsum(0) - 1
        at = begins.nonzero()[:, 0]
        top = new.abs().amax(-1)
        tops = torch.stack([top[run_of == r].amax(0) for r in range(at.numel())]) if at.numel() < 1024 else \
            torch.zeros((at.numel(), top.shape[1]), dtype=top.dtype, device=top.device).scatter_reduce_(0, run_of[:, None].expand_as(top), top, "amax")
        need = 2.0 ** torch.log2(tops / FP8_MAX).ceil().clamp(-64, 64)
        b_page, b_in_page, b_first = page[at], slot[at] // size, slot[at] % size
        old = scales[b_page, b_in_page]
        now = torch.where(b_first[:, None] == 0, need, torch.maximum(need, old))
        for offset in range(size):  # what stands ahead of the new tokens
            ahead = offset < b_first
            where = b_page[ahead], b_in_page[ahead] * size + offset
            held[where] = held[where] * (old / now)[ahead][:, :, None]
        scales[b_page, b_in_page] = now
        held[page, slot] = (new / now[run_of][:, :, None]).clamp(-FP8_MAX, FP8_MAX)
        results.append((held, scales))
    return rotated(s["q"]), results[0][0], results[1][0], results[0][1], results[1][1]


def _exact_attend(s):
    case, (batch, hq, d) = s["case"], s["q"].shape
    kv, page, size = s["k_pages"].shape[2], case["page"], case["block"]
    out = torch.zeros((batch, hq, d), dtype=torch.float64, device=s["q"].device)
    lse = torch.full((batch, hq), -math.inf, dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(s["lengths"].tolist()):
        if n == 0:
            continue
        place = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device=s["q"].device)
        at, slot = s["table"][b, place // page].long(), place % page
        for h in range(kv):
            heads = slice(h * (hq // kv), (h + 1) * (hq // kv))
            k = s["k_pages"][at, slot, h].double() * s["k_scale"][at, slot // size, h, None].double()
            v = s["v_pages"][at, slot, h].double() * s["v_scale"][at, slot // size, h, None].double()
            score = s["q"][b, heads].double() @ k.T / math.sqrt(d)
            lse[b, heads] = torch.logsumexp(score, -1)
            out[b, heads] = torch.softmax(score, -1) @ v
    return (out, lse) if case["lse"] else out


def _exact_sample(s):
    chosen = torch.zeros((s["logits"].shape[0],), dtype=torch.int64, device=s["logits"].device)
    for b in range(chosen.shape[0]):
        z = s["logits"][b].double()
        temperature = float(s["temperature"][b])
        best = z.max()
        if temperature <= 0:
            chosen[b] = (z == best).nonzero()[0, 0]
            continue
        ids = torch.argsort(-z, stable=True)
        ids = ids[: int(torch.isfinite(z).sum())]
        if s["top_k"] is not None and int(s["top_k"][b]) > 0:
            ids = ids[: int(s["top_k"][b])]
        p = torch.softmax(z[ids] / temperature, 0)
        if s["top_p"] is not None and float(s["top_p"][b]) < 1:
            ahead = torch.cat([p.new_zeros(1), p.cumsum(0)[:-1]])
            ids = ids[: max(1, int((ahead < float(s["top_p"][b])).sum()))]
        if s["min_p"] is not None:
            ids = ids[(z[ids] - best) / temperature >= math.log(float(s["min_p"][b]))]
        ids = ids.sort().values
        p = torch.softmax(z[ids] / temperature, 0)
        chosen[b] = ids[min(ids.numel() - 1, int((p.cumsum(0) <= float(s["random"][b])).sum()))]
    return chosen


_EXACT = {"linear": _exact_linear, "quantize": _exact_quantize, "append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], SIZES[case["dtype"]]
    if kind == "linear":
        rows, inputs, outputs = case["rows"], case["inputs"], case["outputs"]
        groups = -(-inputs // GROUP)
        scales = 4 * groups * (rows + -(-outputs // GROUP))
        return {"bytes": float((rows + outputs) * inputs + scales + size * rows * outputs + (4 * outputs if case["bias"] else 0)),
                "flops": 2.0 * rows * inputs * outputs}
    if kind == "quantize":
        elements = case["rows"] * case["columns"]
        return {"bytes": float((size + 1) * elements + 4 * -(-case["rows"] // case["group_rows"]) * -(-case["columns"] // GROUP)), "flops": 3.0 * elements}
    if kind == "append":
        hq, kv, d, rot = HEADS[case["model"]]
        tokens, (new, begin) = case["tokens"], _starts(case)
        blocks = case["batch"] * -(-new // case["block"])
        rotation = 4 * rot * (tokens if new == 1 else new)  # the prompts share their positions
        return {"bytes": float(tokens * ((2 * hq + 2 * kv) * d * size + 2 * kv * d + 16) + 16 * blocks * kv + rotation), "flops": 3.0 * tokens * (hq + kv) * rot}
    if kind == "attend":
        hq, kv, d, _ = HEADS[case["model"]]
        lengths = [min(n, case["window"] or n) for n in _lengths(case)]
        tokens = sum(lengths)
        tables = 4 * (sum(-(-n // case["page"]) for n in lengths) + case["batch"])
        scales = 8 * kv * sum(-(-n // case["block"]) for n in lengths)
        ends = case["batch"] * hq * (2 * d * size + (4 if case["lse"] else 0))
        return {"bytes": 2.0 * tokens * kv * d + tables + scales + ends, "flops": 4.0 * tokens * hq * d}
    return {"bytes": float(case["batch"] * (case["vocab"] * size + 28)), "flops": 4.0 * case["batch"] * case["vocab"]}
