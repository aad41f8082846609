"""GPU tests of the paged cache in 8 bits with a scale for each block of tokens and head: the append that keeps the scales, and decode attention over them, against
definitions in 64 bits.

Tolerances.  Stored values are the nearest e4m3 numbers of x / scale, scale a power of two, x rotated in 32 bits: half a step of e4m3 of the quotient and
2^-22 of the rotated pair's magnitude.  Tokens that a growing scale brings along are off by half a step once more at most.  Attention: a score is a sum of
up to 256 products in 32 bits times two scales, below 2^-14 of its terms' magnitude, and as many relative parts of a weight; weights are 16-bit numbers (bf16 queries: 2^-11
of each, fp16: 2^-20); sums of up to some thousand weights in 32 bits, 2^-16; the result is rounded once."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(pages, page, block, heads, dim, order="heads outside"):
    """Pages of NaN and scales of NaN: nothing that has not been written may be used."""
    nan = lambda *s: torch.full(s, math.nan, device="cuda")
    if order == "heads outside":
        k, v = (nan(pages, heads, page, dim).to(E4M3).transpose(1, 2) for _ in range(2))
    else:
        both = nan(pages, page, heads, 2, dim).to(E4M3)
        k, v = both[..., 0, :], both[..., 1, :]
    scales = lambda: nan(pages, page // block, heads)
    return k, v, scales(), scales()


def _table(g, counts, extra=1):
    total = sum(counts)
    order = torch.randperm(total + 2, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(counts), max(1, max(counts)) + extra), -3, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at: at + n]
        at += n
    return table, total + 2


def _rotation(positions, rot):
    inv = 1.0 / (10000.0 ** (torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot))
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def _rotated_64(x, cos, sin, positions, interleaved):
    x = x.double().clone()
    if cos is None:
        return x, x.abs()
    rot = 2 * cos.shape[1]
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    a, b = x[..., first].clone(), x[..., second].clone()
    mag = x.abs()
    x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    mag[..., first] = mag[..., second] = a.abs() + b.abs()
    return x, mag


def _power(top):
    """The smallest power of two s, from 2^-64 to 2^64, with top <= 448 s: the logarithm is a rounding off where top is 448 s itself, so the product decides."""
    s = torch.exp2((top / 448).clamp(min=1e-300).log2().round().clamp(-70, 70))
    s = torch.where(top <= 448 * s / 2, s / 2, torch.where(top <= 448 * s, s, 2 * s))
    return s.clamp(2.0 ** -64, 2.0 ** 64)


def _half_step(q):
    return torch.exp2(q.abs().clamp(2.0 ** -6, 448).log2().floor() - 4)


class Mirror:
    """What the cache should hold, in 64 bits: the tokens' exact rows, and the scales."""

    def __init__(self, heads, dim, block):
        self.rows, self.mags, self.scales, self.grown, self.block = {}, {}, {}, {}, block

    def append(self, seq, pos, row, mag):
        """One run's rows, all of one block: lists of positions and [tokens, heads, dim]."""
        at = (seq, pos[0] // self.block)
        finite = torch.where(row.isfinite(), row.abs(), 0.0)
        need = _power(finite.amax((0, 2)))
        if pos[0] % self.block == 0:
            scale, grown = need, torch.zeros_like(need)
        else:
            scale = torch.maximum(need, self.scales[at])
            grown = self.grown[at] + (scale > self.scales[at])
        self.scales[at], self.grown[at] = scale, grown
        for i, p in enumerate(pos):
            self.rows[seq, p], self.mags[seq, p] = row[i], mag[i]

    def check(self, pages, scales, table):
        page = pages.shape[1]
        for (seq, p), row in self.rows.items():
            at, slot = int(table[seq, p // page]), p % page
            scale = self.scales[seq, p // self.block]
            assert torch.equal(scales[at, slot // self.block].double(), scale), (seq, p)
            held = pages[at, slot].double()
            q = (row / scale[:, None]).clamp(-448, 448)
            limit = (1 + self.grown[seq, p // self.block][:, None]) * _half_step(q) + 2.0 ** -22 * self.mags[seq, p] / scale[:, None]
            good = ((held - q).abs() <= limit * (1 + 2.0 ** -10)) | (row.isnan() & held.isnan())
            assert bool(good.all()), (seq, p, float(((held - q).abs() / limit).nan_to_num().max()))


def _runs(seqs, positions, block):
    start = 0
    for i in range(1, len(seqs) + 1):
        if i == len(seqs) or seqs[i] != seqs[i - 1] or positions[i] != positions[i - 1] + 1 or positions[i] // block != positions[i - 1] // block:
            yield range(start, i)
            start = i


SHAPES = [  # page, block, heads, dim, rotated, interleaved
    (16, 16, 2, 128, 128, False), (16, 1, 3, 64, 64, False), (64, 32, 1, 256, 64, False), (48, 16, 2, 64, 32, True), (8, 8, 2, 128, 0, False), (128, 128, 1, 128, 128, False),
    (7, 7, 2, 80, 40, False), (12, 3, 1, 16, 8, True), (30, 10, 2, 32, 20, False), (16, 16, 1, 96, 36, False), (1, 1, 2, 64, 64, False), (64, 64, 2, 256, 256, True)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("page,block,heads,dim,rot,interleaved", SHAPES)
def test_appends(lib, page, block, heads, dim, rot, interleaved, dtype):
    """Prompts of odd lengths at once, then tokens one by one and a few at a time, growing and shrinking."""
    import trismoe_b200 as tm

    g = _gen(page * dim + block)
    lengths, more = [37, 0, 1, 150, 16], 9
    table, pages = _table(g, [-(-(n + 3 * more) // page) for n in lengths])
    k_pages, v_pages, k_scale, v_scale = _cache(pages, page, block, heads, dim, "heads outside" if dim % 32 else "keys and values together")
    cos, sin = _rotation(200, rot) if rot else (None, None)
    mirrors = Mirror(heads, dim, block), Mirror(heads, dim, block)
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    at = [0] * len(lengths)
    steps = [lengths] + [[1] * len(lengths)] * more + [[3, 0, 2, 5, 1]] * 2
    for step, new in enumerate(steps):
        seqs = [b for b, n in enumerate(new) for _ in range(n)]
        pos = [at[b] + i for b, n in enumerate(new) for i in range(n)]
        tokens = len(seqs)
        size = 2.0 ** (step % 5 * 3 - 6)
        qkv = (torch.randn((tokens, 2 + 2 * heads, dim), generator=g, device="cuda") * size).to(dtype)
        q, k, v = qkv[:, :2], qkv[:, 2: 2 + heads], qkv[:, 2 + heads:]
        positions = torch.tensor(pos, device="cuda", dtype=torch.int64 if step % 2 else torch.int32)
        sequences = torch.tensor(seqs, device="cuda", dtype=torch.int32)
        got_q, got_k = tm.append_paged_kv(q, k, v, k_pages, v_pages, table, positions, sequences, cos=cos, sin=sin, interleaved=interleaved, k_scale=k_scale, v_scale=v_scale,
                                          return_key=True, status=status)
        where = positions.long()
        k64, k_mag = _rotated_64(k, cos, sin, where, interleaved)
        for got, x in ((got_q, q), (got_k, k)):
            want, mag = _rotated_64(x, cos, sin, where, interleaved)
            assert bool(((got.double() - want).abs() <= U[dtype] * want.abs() + 2.0 ** -22 * mag + 2.0 ** -25).all())
        for run in _runs(seqs, pos, block):
            i = list(run)
            mirrors[0].append(seqs[i[0]], [pos[j] for j in i], k64[i], k_mag[i])
            mirrors[1].append(seqs[i[0]], [pos[j] for j in i], v[i].double(), v[i].double().abs())
        at = [a + n for a, n in zip(at, new)]
        if step in (0, 1, more, len(steps) - 1):
            mirrors[0].check(k_pages, k_scale, table)
            mirrors[1].check(v_pages, v_scale, table)
    tm.raise_on_status(status)
    # nothing but the tokens' places has been written
    written = torch.zeros((pages, page), dtype=torch.bool, device="cuda")
    for b, n in enumerate(at):
        p = torch.arange(n, device="cuda")
        written[table[b, p // page].long(), p % page] = True
    for held in (k_pages, v_pages):
        assert bool(held.float().isnan()[~written].all())


def test_many_tokens_in_one_call(lib):
    """Prompts that begin anywhere in the call, blocks that lie across what a warp looks at."""
    import trismoe_b200 as tm

    for page, block in ((16, 16), (64, 64), (128, 32)):
        g = _gen(page)
        lengths = [1000, 33, 1, 701]
        table, pages = _table(g, [-(-n // page) for n in lengths])
        k_pages, v_pages, k_scale, v_scale = _cache(pages, page, block, 4, 128)
        cos, sin = _rotation(1000, 128)
        seqs = torch.arange(4, device="cuda", dtype=torch.int32).repeat_interleave(torch.tensor(lengths, device="cuda"))
        positions = torch.cat([torch.arange(n, device="cuda") for n in lengths])
        k, v = (torch.randn((sum(lengths), 4, 128), generator=g, device="cuda").half() for _ in range(2))
        tm.append_paged_kv(None, k, v, k_pages, v_pages, table, positions, seqs, cos=cos, sin=sin, k_scale=k_scale, v_scale=v_scale)
        k64, mag = _rotated_64(k, cos, sin, positions, False)
        at, slot = table[seqs.long(), positions // page].long(), positions % page
        index = seqs.long() * 1000 + positions // block
        for rows, m, held, scales in ((k64, mag, k_pages, k_scale), (v.double(), v.double().abs(), v_pages, v_scale)):
            top = torch.zeros((4000, 4), dtype=torch.float64, device="cuda").scatter_reduce_(0, index[:, None].expand(-1, 4), rows.abs().amax(2), "amax")
            scale = _power(top)[index]
            assert torch.equal(scales[at, slot // block].double(), scale)
            q = rows / scale[..., None]
            assert bool(((held[at, slot].double() - q).abs() <= _half_step(q) * (1 + 2.0 ** -10) + 2.0 ** -22 * m / scale[..., None]).all())


def test_tokens_without_a_place(lib):
    """Padding, positions beyond the table, pages that do not exist: nothing is written, the others are, and the status word says so."""
    import trismoe_b200 as tm

    table = torch.tensor([[0, 1], [2, 99]], dtype=torch.int32, device="cuda")
    k_pages, v_pages, k_scale, v_scale = _cache(4, 16, 16, 1, 64)
    k = torch.ones((6, 1, 64), dtype=F16, device="cuda")
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    sequences = torch.tensor([0, 0, 0, 1, 1, 5], dtype=torch.int32, device="cuda")
    positions = torch.tensor([3, -1, 32, 0, 16, 0], device="cuda")
    k_scale[:] = v_scale[:] = 2.0 ** -20
    q = tm.append_paged_kv(k, k, k, k_pages, v_pages, table, positions, sequences, k_scale=k_scale, v_scale=v_scale, status=status)
    assert torch.equal(q[:, 0, 0].float(), torch.tensor([1, 0, 1, 1, 1, 1], device="cuda").float())
    assert int(status) != 0
    assert sorted(k_pages.float().isfinite().all(-1).nonzero()[:, :2].tolist()) == [[0, 3], [2, 0]]
    assert float(k_pages[0, 3, 0, 0]) * float(k_scale[0, 0, 0]) == 1.0 and float(k_scale[1, 0, 0]) == 2.0 ** -20


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_zeros_nan_infinities_and_ends_of_the_range(lib, dtype):
    import trismoe_b200 as tm

    k_pages, v_pages, k_scale, v_scale = _cache(3, 4, 4, 1, 64)
    table = torch.tensor([[1, 2]], dtype=torch.int32, device="cuda")
    k = torch.zeros((8, 1, 64), dtype=dtype, device="cuda")
    v = torch.ones((8, 1, 64), dtype=dtype, device="cuda")
    v[2, 0, 5], v[2, 0, 6], v[3, 0, 7] = math.inf, math.nan, -math.inf
    if dtype is BF16:
        v[4:] = 3.0e38
        k[4:] = 1e-38
    tm.append_paged_kv(None, k, v, k_pages, v_pages, table, torch.arange(8, device="cuda"), torch.zeros((8,), dtype=torch.int32, device="cuda"), k_scale=k_scale, v_scale=v_scale)
    assert float(k_scale[1, 0, 0]) == 2.0 ** -64 and bool((k_pages[1].float() == 0).all())
    assert float(v_scale[1, 0, 0]) == 2.0 ** -8
    row = v_pages[1, :, 0].float() * 2.0 ** -8
    assert float(row[2, 5]) == 448 * 2.0 ** -8 and math.isnan(float(row[2, 6])) and float(row[3, 7]) == -448 * 2.0 ** -8 and float(row[0, 0]) == 1.0
    if dtype is BF16:
        assert float(v_scale[2, 0, 0]) == 2.0 ** 64 and bool((v_pages[2].float() == 448).all())
        assert float(k_scale[2, 0, 0]) == 2.0 ** -64 and bool((k_pages[2].float() == 0).all())


def test_other_scales_than_powers_of_two_are_kept(lib):
    """Scales that a caller has put in hold until a larger one is needed."""
    import trismoe_b200 as tm

    k_pages, v_pages, k_scale, v_scale = _cache(1, 16, 16, 1, 64)
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    k_pages[0, :3], v_pages[0, :3] = 100.0, 100.0
    k_scale[:], v_scale[:] = 0.3, 1e-4
    x = torch.full((1, 1, 64), 0.7, dtype=F16, device="cuda")
    tm.append_paged_kv(None, x, x, k_pages, v_pages, table, torch.tensor([3], device="cuda"), k_scale=k_scale, v_scale=v_scale)
    assert float(k_scale) == torch.tensor(0.3).item() and float(k_pages[0, 0, 0, 0].float()) == 96.0  # 100 is stored as 96
    assert abs(float(k_pages[0, 3, 0, 0].float()) - 0.7 / 0.3) <= 0.125
    assert float(v_scale) == 2.0 ** -9 and abs(float(v_pages[0, 0, 0, 0].float()) * 2.0 ** -9 - 96e-4) <= 96e-4 * 2.0 ** -4


# ---------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------
def _filled(g, lengths, page, block, heads, dim, spread, order="heads outside", extra=1):
    table, pages = _table(g, [-(-n // page) for n in lengths], extra)
    k_pages, v_pages, k_scale, v_scale = _cache(pages, page, block, heads, dim, order)
    for b, n in enumerate(lengths):
        p = torch.arange(n, device="cuda")
        at = table[b, p // page].long()
        for held in (k_pages, v_pages):
            held[at, p % page] = (torch.randn((n, heads, dim), generator=g, device="cuda") * 100).clamp(-448, 448).to(E4M3)
        for scales, most in ((k_scale, 2), (v_scale, spread)):
            scales[at, p % page // block] = (torch.exp2(torch.randint(-most, most + 1, (pages, page // block, heads), generator=g, device="cuda").float() - 7)
                                             * (1 + 0.7 * torch.rand((pages, page // block, heads), generator=g, device="cuda")))[at, p % page // block]
    return k_pages, v_pages, k_scale, v_scale, table


def _check_attention(tm, q, k_pages, v_pages, k_scale, v_scale, table, lengths, window=None, softmax_scale=None):
    batch, heads, dim = q.shape
    kv, page, block = k_pages.shape[2], k_pages.shape[1], k_pages.shape[1] // k_scale.shape[1]
    length = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    out, lse = tm.paged_decode_attention(q, k_pages, v_pages, table, length, window=window, softmax_scale=softmax_scale, k_scale=k_scale, v_scale=v_scale, return_lse=True, status=status)
    tm.raise_on_status(status)
    assert torch.equal(out, tm.paged_decode_attention(q, k_pages, v_pages, table, length, window=window, softmax_scale=softmax_scale, k_scale=k_scale, v_scale=v_scale))
    weight_error = 2.0 ** -11 if q.dtype is BF16 else 2.0 ** -20
    for b, n in enumerate(lengths):
        if n == 0:
            assert bool((out[b] == 0).all()) and bool((lse[b] == -math.inf).all())
            continue
        p = torch.arange(max(0, n - window) if window else 0, n, device="cuda")
        at, slot = table[b, p // page].long(), p % page
        k = (k_pages[at, slot].double() * k_scale[at, slot // block].double()[..., None]).repeat_interleave(heads // kv, 1)
        v = (v_pages[at, slot].double() * v_scale[at, slot // block].double()[..., None]).repeat_interleave(heads // kv, 1)
        factor = dim ** -0.5 if softmax_scale is None else softmax_scale
        score = torch.einsum("hd,thd->ht", q[b].double(), k) * factor
        score_mag = torch.einsum("hd,thd->ht", q[b].double().abs(), k.abs()) * factor
        w = torch.softmax(score, 1)
        want, mag = torch.einsum("ht,thd->hd", w, v), torch.einsum("ht,thd->hd", w * (1 + 2 * score_mag * 2.0 ** -14 / 2.0 ** -11), v.abs())
        limit = (weight_error + 2.0 ** -16) * torch.einsum("ht,thd->hd", w, v.abs()) + 2.0 ** -11 * (mag - torch.einsum("ht,thd->hd", w, v.abs())) + U[q.dtype] * want.abs() + 2.0 ** -25
        error = (out[b].double() - want).abs()
        assert bool((error <= limit).all()), (b, n, float((error / limit).max()))
        assert bool(((lse[b].double() - torch.logsumexp(score, 1)).abs() <= 2.0 ** -14 * (1 + score_mag.amax(1))).all())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("page,block,heads,kv,dim", [(16, 16, 8, 8, 128), (16, 1, 4, 2, 64), (64, 32, 16, 2, 256), (48, 16, 32, 4, 64), (7, 7, 6, 3, 80), (12, 4, 20, 1, 128), (1, 1, 3, 3, 16),
                                                     (128, 128, 12, 1, 64), (8, 2, 9, 1, 256)])
def test_attention(lib, page, block, heads, kv, dim, dtype):
    import trismoe_b200 as tm

    g = _gen(page + dim)
    lengths = [0, 1, 15, 16, 17, 100, 333]
    cache = _filled(g, lengths, page, block, kv, dim, 2, "heads outside" if dim != 64 else "keys and values together")
    q = torch.randn((len(lengths), heads, dim), generator=g, device="cuda").to(dtype)
    for window in (None, 1, 40):
        _check_attention(tm, q, *cache, lengths, window=window)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("lengths,extra", [([20000], 1), ([5000, 1, 700, 0, 9000], 1), ([513], 1000), ([40] * 60, 1), ([300, 200] * 30, 1)], ids=["long", "ragged", "wide", "short", "many"])
def test_attention_of_every_way_to_share_the_work(lib, lengths, extra, dtype):
    import trismoe_b200 as tm

    g = _gen(len(lengths))
    cache = _filled(g, lengths, 16, 16, 4, 128, 3, extra=extra)
    _check_attention(tm, torch.randn((len(lengths), 8, 128), generator=g, device="cuda").to(dtype), *cache, lengths)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_values_whose_scales_lie_far_apart(lib, dtype):
    """The weights' 16 bits go to what counts in the sum, whichever block has the large scores and whichever the large values."""
    import trismoe_b200 as tm

    g = _gen(1)
    lengths = [64, 333, 48]
    k_pages, v_pages, k_scale, v_scale, table = _filled(g, lengths, 16, 16, 2, 128, 30)
    q = torch.randn((3, 4, 128), generator=g, device="cuda").to(dtype)
    if dtype is F16:
        v_scale.clamp_(max=2.0 ** 4)  # results beyond fp16
    _check_attention(tm, q, k_pages, v_pages, k_scale, v_scale, table, lengths)
    k_scale *= 8.0  # scores of up to some hundred
    _check_attention(tm, q, k_pages, v_pages, k_scale, v_scale, table, lengths)


def test_a_scale_of_zero_and_scales_beyond_the_range(lib):
    import trismoe_b200 as tm

    g = _gen(2)
    k_pages, v_pages, k_scale, v_scale, table = _filled(g, [64], 16, 16, 1, 64, 1)
    q = torch.randn((1, 1, 64), generator=g, device="cuda").half()
    length = torch.tensor([64], dtype=torch.int32, device="cuda")
    v_scale[table[0, 1].long()] = 0.0  # counts as 2^-64
    v_pages[table[0, 2].long()] = 0.0
    out = tm.paged_decode_attention(q, k_pages, v_pages, table, length, k_scale=k_scale, v_scale=v_scale)
    v_scale[table[0, 1].long()] = 2.0 ** -64
    assert torch.equal(out, tm.paged_decode_attention(q, k_pages, v_pages, table, length, k_scale=k_scale, v_scale=v_scale)) and bool(out.isfinite().all())


def test_append_and_attention_together_in_a_graph(lib):
    """A captured step of both, replayed over growing sequences, against all tokens' exact keys and values."""
    import trismoe_b200 as tm

    g = _gen(5)
    heads, kv, dim, page, start, steps = 8, 2, 64, 16, 13, 24
    k_pages, v_pages, k_scale, v_scale = _cache(9, page, page, kv, dim)
    table = torch.randperm(9, generator=g, device="cuda").to(torch.int32)[:8].view(2, 4)
    qkv = torch.randn((start + steps, 2, heads + 2 * kv, dim), generator=g, device="cuda").half()
    qkv *= torch.exp2(torch.randint(-3, 4, (start + steps, 1, 1, 1), generator=g, device="cuda").float()).half()
    prompt = qkv[:start].transpose(0, 1).reshape(2 * start, heads + 2 * kv, dim)
    tm.append_paged_kv(None, prompt[:, heads: heads + kv], prompt[:, heads + kv:], k_pages, v_pages, table, torch.arange(start, device="cuda").repeat(2),
                       torch.arange(2, device="cuda", dtype=torch.int32).repeat_interleave(start), k_scale=k_scale, v_scale=v_scale)
    now, pos = qkv[start].clone(), torch.full((2,), start, device="cuda")
    length = torch.full((2,), start + 1, dtype=torch.int32, device="cuda")

    def step():
        tm.append_paged_kv(None, now[:, heads: heads + kv], now[:, heads + kv:], k_pages, v_pages, table, pos, k_scale=k_scale, v_scale=v_scale)
        return tm.paged_decode_attention(now[:, :heads], k_pages, v_pages, table, length, k_scale=k_scale, v_scale=v_scale)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(steps):
        now.copy_(qkv[start + i])
        pos.fill_(start + i)
        length.fill_(start + i + 1)
        graph.replay()
        torch.cuda.synchronize()
        n = start + i + 1
        for b in range(2):
            k, v = (x.double().repeat_interleave(heads // kv, 1) for x in (qkv[:n, b, heads: heads + kv], qkv[:n, b, heads + kv:]))
            # keys and values are off by half a step of e4m3 of their own, once for each time their block's scale has grown, and of the block's smallest
            blocks = torch.arange(n, device="cuda") // page
            top = torch.stack([x.abs().amax(2) for x in (k, v)])
            most = torch.zeros((2, n, heads), dtype=torch.float64, device="cuda")
            for j in range(int(blocks[-1]) + 1):
                most[:, blocks == j] = top[:, blocks == j].amax(1, keepdim=True)
            slack = [x.abs() * 2.0 ** -4 + m[..., None] * 2.0 ** -15 for x, m in zip((k, v), most)]
            score = torch.einsum("hd,thd->ht", qkv[start + i, b, :heads].double(), k) / dim ** 0.5
            d = torch.einsum("hd,thd->ht", qkv[start + i, b, :heads].double().abs(), slack[0]) / dim ** 0.5
            w = torch.softmax(score, 1)
            off = torch.minimum((w * torch.expm1(2 * d.amax(1, keepdim=True))), torch.ones_like(w))
            want = torch.einsum("ht,thd->hd", w, v)
            limit = torch.einsum("ht,thd->hd", off, v.abs()) + torch.einsum("ht,thd->hd", w + off, slack[1]) + 2.0 ** -9 * want.abs() + 1e-6
            assert bool(((out[b].double() - want).abs() <= limit).all())
