"""Timed workloads of the operators around the expert layers in a decode step: keys and values go into a paged
cache with the position rotation applied, one new token a sequence attends over that cache, the residual is
added and normalised, and the logits get their penalties, biases and grammar masks.

``listed()`` names the workloads, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes what a program holds
before the call, ``run`` is one pass - in elementary torch operations, or with ``own`` set through the framework's entry
points -, ``exact`` the same from the definition in 64 bits and ``work`` what a pass cannot do without.  All data is
synthetic and made on the GPU from the seed.
"""
import math

import torch

own = False

FP8_MAX = 448.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
SIZES = {"fp16": 2, "bf16": 2, "fp32": 4, "e4m3": 1}
# query heads, key/value heads, head size and rotated dimensions of the models of the benchmark and the tests
HEADS = {"olmoe": (16, 16, 128, 128), "mixtral": (32, 8, 128, 128), "qwen35": (16, 2, 256, 64), "small": (4, 2, 64, 64)}
HIDDEN = {"olmoe": 2048, "mixtral": 4096, "qwen35": 2048, "small": 256}


# ---------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------
def _attend(model, batch, longest, dtype, cache, page=16, ragged=1.0, empty=False, window=0, lse=False):
    return {"kind": "attend", "model": model, "batch": batch, "longest": longest, "dtype": dtype, "cache": cache, "page": page,
            "ragged": ragged, "empty": empty, "window": window, "lse": lse}


def _append(model, batch, tokens, dtype, cache, page=16, interleaved=False):
    return {"kind": "append", "model": model, "batch": batch, "tokens": tokens, "dtype": dtype, "cache": cache, "page": page,
            "interleaved": interleaved}


def _norm(tokens, hidden, dtype, group=-1):
    return {"kind": "norm", "tokens": tokens, "hidden": hidden, "dtype": dtype, "group": group}


def _logits(batch, vocab, history, dtype, biases, counted):
    return {"kind": "logits", "batch": batch, "vocab": vocab, "history": history, "dtype": dtype, "biases": biases, "counted": counted}


def listed():
    cases = {
        # one conversation behind a prompt of 512 tokens: nothing is large, latency is all
        "attend 1 x 513": _attend("olmoe", 1, 513, "fp16", "fp16"),
        # the benchmark's generation, prompt 512 and up to 256 new tokens, 32 sequences, every head with its own keys
        "attend 32 x 512-768": _attend("olmoe", 32, 768, "fp16", "fp16", ragged=0.67),
        # one sequence with a very long context: the split over its length is all the parallelism there is
        "attend 1 x 131071": _attend("mixtral", 1, 131071, "fp16", "fp16", lse=True),
        # 16 sequences of 4096 tokens, heads of 256, an 8-bit cache in pages of 64
        "attend 16 x 4096 e4m3": _attend("qwen35", 16, 4096, "bf16", "e4m3", page=64, ragged=0.95),
        # a server under load: 64 sequences of very different lengths, some slots of the batch free
        "attend 64 x 1-16384": _attend("mixtral", 64, 16384, "bf16", "bf16", ragged=0.0, empty=True),
        # the step of one conversation
        "append 1": _append("olmoe", 1, 1, "fp16", "fp16"),
        # a decode step of 64 sequences, 8-bit cache
        "append 64 e4m3": _append("mixtral", 64, 64, "bf16", "e4m3"),
        # four prompts of some 2000 tokens on their way into the cache
        "append 4 x 2047": _append("olmoe", 4, 8188, "fp16", "fp16"),
        # between attention and experts of one token
        "norm 1 x 2048": _norm(1, 2048, "fp16"),
        # a prompt on its way to a product in 8 bits, a scale for 128 columns
        "norm 2047 x 4096 e4m3": _norm(2047, 4096, "bf16", group=128),
        # one conversation with a penalty and a grammar
        "logits 1 x 50304": _logits(1, 50304, 700, "fp16", 0, False),
        # a large batch with all controls and long histories
        "logits 128 x 50304": _logits(128, 50304, 4000, "fp32", 64, True),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _log_int(rng, low, high):
    n = min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))
    return n + 1 if n == 3072 else n


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "norm", "logits"])
    model = rng.choice(list(HEADS))
    dtype = rng.choice(["fp16", "bf16"])
    cache = "e4m3" if rng.random() < 0.33 else dtype
    page = rng.choice([1, 8, 16, 16, 16, 32, 48, 64, 128])
    if kind == "attend":
        batch = _log_int(rng, 1, 64)
        most = min(131071, 1_700_000_000 // (batch * 2 * HEADS[model][1] * HEADS[model][2] * SIZES[cache]))
        return _attend(model, batch, _log_int(rng, 1, most), dtype, cache, page, rng.choice([0.0, 0.5, 0.9, 1.0]), rng.random() < 0.25,
                       rng.choice([0, 0, 0, 1000]), rng.random() < 0.25)
    if kind == "append":
        batch = _log_int(rng, 1, 64)
        tokens = batch if rng.random() < 0.5 else batch * _log_int(rng, 1, 8192 // batch)
        return _append(model, batch, tokens, dtype, cache, page, rng.random() < 0.25)
    if kind == "norm":
        hidden = rng.choice([256, 2048, 2048, 4096, 8192, _log_int(rng, 17, 8192)])
        quantized = rng.random() < 0.5
        return _norm(_log_int(rng, 1, 8192), hidden, dtype, rng.choice([0, 128] if hidden % 128 == 0 else [0]) if quantized else -1)
    return _logits(_log_int(rng, 1, 128), rng.choice([32000, 50304, _log_int(rng, 1000, 50304)]), _log_int(rng, 1, 8000),
                   rng.choice(["fp16", "bf16", "fp32"]), rng.choice([0, 0, 5, 300]), rng.random() < 0.5)


def _lengths(case):
    """Cached tokens of every sequence: from ``ragged`` times the longest to the longest, spread evenly in an order of their own;
    with ``empty`` every eighth place of the batch is free."""
    low = case["ragged"] * case["longest"]
    spread = [(0.618034 * (i + 1)) % 1.0 for i in range(case["batch"])]
    lengths = [max(1, int(low + (case["longest"] - low) * f)) for f in spread]
    lengths[0] = case["longest"]
    return [0 if case["empty"] and i % 8 == 7 else n for i, n in enumerate(lengths)]


# ---------------------------------------------------------------------------------------
# what a program holds before the call
# ---------------------------------------------------------------------------------------
def _normal(g, std, *shape):
    return torch.randn(shape, generator=g, device=g.device) * std


def _pages(g, case, pages):
    """One cache: [pages, tokens of a page, heads, head size], a head's tokens of a page side by side in memory."""
    _, kv, d, _ = HEADS[case["model"]]
    out = torch.empty((pages, kv, case["page"], d), dtype=DTYPES[case["cache"]], device=g.device)
    for part in out.split(max(1, (1 << 26) // max(1, out[0].numel()))):
        part.copy_(_normal(g, 1.0, *part.shape))
    return out.transpose(1, 2)


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


def _append_positions(case):
    """Where every sequence's new tokens begin: decode steps stand at different places of their contexts, prompts begin at 0."""
    batch = case["batch"]
    new = case["tokens"] // batch
    return new, [0 if new > 1 else (997 * i + 511) % 4096 for i in range(batch)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, kind, state = g.device, case["kind"], {"case": case}
    dtype = DTYPES[case["dtype"]]
    if kind in ("attend", "append"):
        hq, kv, d, rot = HEADS[case["model"]]
        scales = (lambda: 0.02 + 0.02 * torch.rand((kv,), generator=g, device=dev)) if case["cache"] == "e4m3" else (lambda: None)
    if kind == "attend":
        lengths = _lengths(case)
        state["table"], total = _tables(g, [-(-n // case["page"]) for n in lengths])
        state["k_pages"], state["v_pages"] = _pages(g, case, total), _pages(g, case, total)
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        # 8-bit pages hold numbers around 1, too, so their scales are put back into the queries
        state["k_scale"], state["v_scale"] = scales(), scales()
        state["q"] = _normal(g, 2.0 if state["k_scale"] is None else 60.0, case["batch"], hq, d).to(dtype)
    elif kind == "append":
        new, begin = _append_positions(case)
        state["table"], total = _tables(g, [-(-(b + new) // case["page"]) for b in begin])
        state["k_pages"], state["v_pages"] = _pages(g, case, total), _pages(g, case, total)
        state["k_scale"], state["v_scale"] = scales(), scales()
        qkv = _normal(g, 1.0, case["tokens"], hq + 2 * kv, d).to(dtype)  # as one projection leaves them
        state["q"], state["k"], state["v"] = qkv[:, :hq], qkv[:, hq: hq + kv], qkv[:, hq + kv:]
        state["sequences"] = torch.arange(case["batch"], device=dev, dtype=torch.int32).repeat_interleave(new)
        state["positions"] = (torch.tensor(begin, device=dev)[:, None] + torch.arange(new, device=dev)).reshape(-1)
        state["cos"], state["sin"] = _rotation(case, max(begin) + new, dev)
    elif kind == "norm":
        state["x"] = _normal(g, 0.5, case["tokens"], case["hidden"]).to(dtype)
        residual = _normal(g, 1.0, case["tokens"], case["hidden"])
        residual[:, torch.randperm(case["hidden"], generator=g, device=dev)[: max(1, case["hidden"] // 100)]] *= 20.0
        state["residual"] = residual.to(dtype)
        state["weight"] = (1.0 + _normal(g, 0.1, case["hidden"])).to(dtype)
    else:
        batch, vocab, history = case["batch"], case["vocab"], case["history"]
        state["logits"] = _normal(g, 3.0, batch, vocab).to(dtype)
        # words repeat: most of a history comes from a small part of the vocabulary
        common = torch.randint(0, vocab, (batch, 1 + history // 4), generator=g, device=dev)
        state["tokens"] = common.gather(1, torch.randint(0, common.shape[1], (batch, history), generator=g, device=dev)).to(torch.int32)
        lengths = torch.randint(history // 2, history + 1, (batch,), generator=g, device=dev, dtype=torch.int32)
        state["token_lengths"], state["prompt_lengths"] = lengths, (lengths // 2 if case["counted"] else None)
        uniform = lambda low, high: low + (high - low) * torch.rand((batch,), generator=g, device=dev)  # noqa: E731
        state["repetition"] = uniform(1.0, 1.5)
        state["presence"], state["frequency"] = (uniform(0.0, 1.0), uniform(0.0, 0.5)) if case["counted"] else (None, None)
        state["bias_ids"] = state["bias_values"] = None
        if case["biases"]:
            state["bias_ids"] = torch.randint(-1, vocab, (batch, case["biases"]), generator=g, device=dev, dtype=torch.int32)
            state["bias_values"] = _normal(g, 5.0, batch, case["biases"])
        words = torch.randint(-2**31, 2**31, (batch, -(-vocab // 32)), generator=g, device=dev, dtype=torch.int64)
        state["allowed"] = words.to(torch.int32)
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def run(state):
    with torch.no_grad():
        return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


def _own_attend(s):
    import trismoe_b200 as tm

    case = s["case"]
    return tm.paged_decode_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], window=case["window"],
                                     k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=case["lse"])


def _own_append(s):
    import trismoe_b200 as tm

    q = tm.append_paged_kv(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["positions"], s["sequences"],
                           cos=s["cos"], sin=s["sin"], interleaved=s["case"]["interleaved"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return q, s["k_pages"], s["v_pages"]


def _own_norm(s):
    import trismoe_b200 as tm

    group = s["case"]["group"]
    if group < 0:
        return tm.add_rms_norm(s["x"], s["residual"], s["weight"], 1e-5)
    return tm.add_rms_norm_e4m3(s["x"], s["residual"], s["weight"], 1e-5, group_size=group)


def _own_logits(s):
    import trismoe_b200 as tm

    return tm.apply_logit_controls(s["logits"], tokens=s["tokens"], token_lengths=s["token_lengths"], prompt_lengths=s["prompt_lengths"],
                                   repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"],
                                   bias_values=s["bias_values"], allowed=s["allowed"])


def _plain_attend(s):
    case, q = s["case"], s["q"].float()
    (batch, hq, d), kv, page = q.shape, s["k_pages"].shape[2], case["page"]
    pages = s["table"].clamp(min=0).long()
    length = s["lengths"][:, None]
    place = torch.arange(pages.shape[1] * page, device=q.device)
    valid = place < length
    if case["window"]:
        valid = valid & (place >= length - case["window"])
    k = s["k_pages"][pages].reshape(batch, -1, kv, d).float()
    score = torch.einsum("bhgd,bthd->bhgt", q.view(batch, kv, hq // kv, d), k) * d ** -0.5
    del k
    if s["k_scale"] is not None:
        score = score * s["k_scale"][:, None, None]
    score = score.masked_fill(~valid[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)  # a sequence without tokens has no largest score
    weight = torch.exp(score - top)
    total = weight.sum(-1, keepdim=True)
    v = s["v_pages"][pages].reshape(batch, -1, kv, d).float()
    out = torch.einsum("bhgt,bthd->bhgd", weight, v) / total.masked_fill(total == 0, 1.0)
    if s["v_scale"] is not None:
        out = out * s["v_scale"][:, None, None]
    out = out.reshape(batch, hq, d).to(s["q"].dtype)
    if not case["lse"]:
        return out
    return out, torch.where(total == 0, -math.inf, top + total.log()).reshape(batch, hq)


def _rotate(x, cos, sin, interleaved):
    """x [tokens, heads, head size] in 32 or 64 bits; cos and sin [tokens, rotated dimensions / 2]."""
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


def _stored(x, scale, dtype):
    if scale is not None:
        x = (x / scale[:, None]).clamp(-FP8_MAX, FP8_MAX)
    return x.to(dtype)


def _plain_append(s):
    case, positions = s["case"], s["positions"]
    cos, sin = s["cos"][positions], s["sin"][positions]
    q = _rotate(s["q"].float(), cos, sin, case["interleaved"]).to(s["q"].dtype)
    k = _rotate(s["k"].float(), cos, sin, case["interleaved"])
    page = s["table"][s["sequences"].long(), positions // case["page"]].long()
    slot = positions % case["page"]
    for pages, new, scale in ((s["k_pages"], k, s["k_scale"]), (s["v_pages"], s["v"].float(), s["v_scale"])):
        pages[page, slot] = _stored(new, scale, pages.dtype)
    return q, s["k_pages"], s["v_pages"]


def _plain_norm(s):
    group = s["case"]["group"]
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-5) * s["weight"].float()
    if group < 0:
        return y.to(s["x"].dtype), h.to(s["x"].dtype)
    parts = y.view(y.shape[0], -1, group or y.shape[1])
    scale = parts.abs().amax(-1, keepdim=True) / FP8_MAX
    values = (parts / scale.masked_fill(scale == 0, 1.0)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return values.view(y.shape), scale.squeeze(-1), h.to(s["x"].dtype)


def _counts(s, dtype):
    """How often every token occurs in a sequence's prompt and answer, and in its answer alone."""
    tokens, place = s["tokens"].long(), torch.arange(s["tokens"].shape[1], device=s["tokens"].device)
    known = place < s["token_lengths"][:, None]
    answer = known if s["prompt_lengths"] is None else known & (place >= s["prompt_lengths"][:, None])
    none = torch.zeros(s["logits"].shape, dtype=dtype, device=tokens.device)
    return none.scatter_add(1, tokens, known.to(dtype)), none.scatter_add(1, tokens, answer.to(dtype))


def _controlled(s, z):
    seen, answered = _counts(s, z.dtype)
    column = lambda name: s[name].to(z.dtype)[:, None]  # noqa: E731
    r = column("repetition")
    z = torch.where(seen > 0, torch.where(z > 0, z / r, z * r), z)
    if s["presence"] is not None:
        z = z - column("presence") * (answered > 0) - column("frequency") * answered
    if s["bias_ids"] is not None:
        used = s["bias_ids"] >= 0
        z = z.scatter_add(1, s["bias_ids"].clamp(min=0).long(), torch.where(used, s["bias_values"], 0.0).to(z.dtype))
    bits = (s["allowed"][:, :, None] >> torch.arange(32, device=z.device, dtype=torch.int32)) & 1
    return z.masked_fill(bits.flatten(1)[:, : z.shape[1]] == 0, -math.inf)


def _plain_logits(s):
    return _controlled(s, s["logits"].float())


_PLAIN = {"attend": _plain_attend, "append": _plain_append, "norm": _plain_norm, "logits": _plain_logits}
_OWN = {"attend": _own_attend, "append": _own_append, "norm": _own_norm, "logits": _own_logits}


# ---------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s)


def _exact_attend(s):
    case, (batch, hq, d) = s["case"], s["q"].shape
    kv, page = s["k_pages"].shape[2], case["page"]
    out = torch.zeros((batch, hq, d), dtype=torch.float64, device=s["q"].device)
    lse = torch.full((batch, hq), -math.inf, dtype=torch.float64, device=s["q"].device)
    for b, n in enumerate(s["lengths"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        place = torch.arange(first, n, device=s["q"].device)
        at, slot = s["table"][b, place // page].long(), place % page
        for h in range(kv):
            heads = slice(h * (hq // kv), (h + 1) * (hq // kv))
            k, v = s["k_pages"][at, slot, h].double(), s["v_pages"][at, slot, h].double()
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][h].double(), v * s["v_scale"][h].double()
            score = s["q"][b, heads].double() @ k.T / math.sqrt(d)
            lse[b, heads] = torch.logsumexp(score, -1)
            out[b, heads] = torch.softmax(score, -1) @ v
    return (out, lse) if case["lse"] else out


def _exact_append(s):
    positions = s["positions"]
    rot = 2 * s["cos"].shape[1]
    turn = torch.complex(s["cos"][positions].double(), s["sin"][positions].double())[:, None]

    def rotated(x):
        x = x.double().clone()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if s["case"]["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
        z = torch.complex(x[..., first], x[..., second]) * turn
        x[..., first], x[..., second] = z.real, z.imag
        return x

    caches = []
    where = positions // s["case"]["page"], positions % s["case"]["page"]
    for pages, new, scale in ((s["k_pages"], rotated(s["k"]), s["k_scale"]), (s["v_pages"], s["v"].double(), s["v_scale"])):
        held = pages.double()
        if scale is not None:
            new = (new / scale.double()[:, None]).clamp(-FP8_MAX, FP8_MAX)
        held[s["table"][s["sequences"].long(), where[0]].long(), where[1]] = new
        caches.append(held)
    return rotated(s["q"]), caches[0], caches[1]


def _exact_norm(s):
    group, h = s["case"]["group"], s["x"].double() + s["residual"].double()
    y = s["weight"].double() * h / (torch.linalg.vector_norm(h, dim=-1, keepdim=True) ** 2 / h.shape[1] + 1e-5).sqrt()
    if group < 0:
        return y, h
    parts = y.unflatten(1, (-1, group or y.shape[1]))
    scale = parts.abs().amax(-1) / FP8_MAX
    return (parts / scale[..., None]).flatten(1), scale, h


def _exact_logits(s):
    z = s["logits"].double()
    batch, vocab = z.shape
    for b in range(batch):
        n = int(s["token_lengths"][b])
        begin = 0 if s["prompt_lengths"] is None else int(s["prompt_lengths"][b])
        row, tokens = z[b], s["tokens"][b].long()
        seen = torch.bincount(tokens[:n], minlength=vocab)
        row = torch.where(seen > 0, row * s["repetition"][b].double() ** -torch.sign(row), row)
        if s["presence"] is not None:
            count = torch.bincount(tokens[begin:n], minlength=vocab).double()
            row = row - s["frequency"][b].double() * count - s["presence"][b].double() * count.clamp(max=1.0)
        if s["bias_ids"] is not None:
            ids = s["bias_ids"][b].long()
            row = row.index_add(0, ids[ids >= 0], s["bias_values"][b][ids >= 0].double())
        index = torch.arange(vocab, device=z.device)
        row[(s["allowed"][b].long()[index // 32] >> (index % 32)) % 2 == 0] = -math.inf
        z[b] = row
    return z


_EXACT = {"attend": _exact_attend, "append": _exact_append, "norm": _exact_norm, "logits": _exact_logits}


# ---------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], SIZES[case["dtype"]]
    if kind == "attend":
        hq, kv, d, _ = HEADS[case["model"]]
        lengths = [min(n, case["window"] or n) for n in _lengths(case)]
        tokens = sum(lengths)
        tables = 4 * (sum(-(-n // case["page"]) for n in lengths) + case["batch"])
        ends = case["batch"] * hq * (2 * d * size + (4 if case["lse"] else 0))
        return {"bytes": 2.0 * tokens * kv * d * SIZES[case["cache"]] + tables + ends, "flops": 4.0 * tokens * hq * d}
    if kind == "append":
        hq, kv, d, rot = HEADS[case["model"]]
        tokens = case["tokens"]
        rotation = 4 * rot * (tokens if tokens == case["batch"] else tokens // case["batch"])  # the prompts share their positions
        return {"bytes": float(tokens * ((2 * hq + 2 * kv) * d * size + 2 * kv * d * SIZES[case["cache"]] + 16) + rotation),
                "flops": 3.0 * tokens * (hq + kv) * rot}
    if kind == "norm":
        rows, hidden, group = case["tokens"], case["hidden"], case["group"]
        out = size * hidden if group < 0 else hidden + 4 * (hidden // group if group else 1)
        return {"bytes": float(rows * (3 * size * hidden + out) + size * hidden), "flops": (5.0 if group < 0 else 8.0) * rows * hidden}
    batch, vocab = case["batch"], case["vocab"]
    return {"bytes": float(batch * (vocab * (size + 4) + 4 * -(-vocab // 32) + 4 * case["history"] * 3 // 4 + 8 * case["biases"] + 24)),
            "flops": 4.0 * batch * vocab}
