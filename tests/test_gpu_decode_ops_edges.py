"""GPU tests of the decode step's operators where they could go wrong unnoticed: launches that overlap, dimensions and rows that a call must not
touch, quotients that end half way between two results, numbers that are not finite, sizes that lead to each variant.

Definitions in 64 bits and the bounds' parts (U, SUB) are those of test_gpu_decode_ops.py; further bounds are derived where they stand."""
import math

import pytest
import torch

from test_gpu_decode_ops import BF16, E4M3, F16, LAYOUTS, SUB, U, _attend_64, _check_attention, _controls_64, _filled, _gen

pytestmark = pytest.mark.gpu


# ---- launches that overlap ------------------------------------------------------------------
@pytest.fixture
def overlapping(lib):
    """Programmatic launches for the stand-alone entry points, as they were before afterwards."""
    previous = lib.tris_set_programmatic_launch(1)
    try:
        yield lib
    finally:
        torch.cuda.synchronize()
        lib.tris_set_programmatic_launch(previous)


@pytest.mark.parametrize("quantized", [False, True], ids=["16 bit", "e4m3"])
@pytest.mark.parametrize("rows,hidden", [(1, 2048), (300, 4096), (3, 1001)])
def test_norm_of_a_weight_that_the_launch_before_writes(overlapping, rows, hidden, quantized):
    """A weight in the form 1 + w, made by the kernel just ahead, or by a norm whose output it is."""
    import trismoe_b200 as tm

    g = _gen(rows + hidden)
    x, r = (torch.randn((rows, hidden), generator=g, device="cuda").half() for _ in range(2))
    norm = (lambda w: tm.add_rms_norm_e4m3(x, r, w)[0].view(torch.uint8)) if quantized else (lambda w: tm.add_rms_norm(x, r, w)[0])
    deltas = [torch.randn((hidden,), generator=g, device="cuda").half() for _ in range(20)]
    one, weight = torch.ones((hidden,), dtype=F16, device="cuda"), torch.zeros((hidden,), dtype=F16, device="cuda")
    got = []
    for d in deltas:
        torch.add(d, 1.0, out=weight)
        got.append(norm(weight))
        got.append(norm(tm.add_rms_norm(d, None, one)[0]))
    torch.cuda.synchronize()
    for i, d in enumerate(deltas):
        weight = d + 1.0
        torch.cuda.synchronize()
        first = norm(weight)
        weight = tm.add_rms_norm(d, None, one)[0]
        torch.cuda.synchronize()
        assert torch.equal(got[2 * i], first) and torch.equal(got[2 * i + 1], norm(weight))


@pytest.mark.parametrize("longest", [60, 20000], ids=["clusters", "numbered"])
def test_a_chain_of_overlapping_launches_equals_one_that_does_not(overlapping, longest):
    import trismoe_b200 as tm

    g, lengths, hidden, vocab = _gen(longest), [longest, 1, 17], 512, 4000
    k_pages, v_pages, table, _ = _filled(g, [n + 30 for n in lengths], 16, 2, 64, F16, LAYOUTS[0])
    kept = k_pages.clone(), v_pages.clone()
    cos, sin = (torch.rand((longest + 40, 32), generator=g, device="cuda") for _ in range(2))
    w, wqkv, head = ((torch.randn(s, generator=g, device="cuda") / 16).half() for s in ((hidden,), (12 * 64, hidden), (vocab, hidden)))
    start = torch.randn((3, hidden), generator=g, device="cuda").half()
    tokens = torch.randint(0, vocab, (3, 50), generator=g, device="cuda", dtype=torch.int32)
    known, penalty = torch.full((3,), 50, dtype=torch.int32, device="cuda"), torch.full((3,), 1.25, device="cuda")
    places = [torch.tensor([n + step for n in lengths], dtype=torch.int32, device="cuda") for step in range(5)]

    def chain():
        k_pages.copy_(kept[0])
        v_pages.copy_(kept[1])
        x, h, out = start, start, []
        for at in places:
            x, h = tm.add_rms_norm(x, h, w)
            qkv = torch.nn.functional.linear(x, wqkv).view(3, 12, 64)
            q = tm.append_paged_kv(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], k_pages, v_pages, table, at, cos=cos, sin=sin)
            x = tm.paged_decode_attention(q, k_pages, v_pages, table, at + 1).flatten(1)
            y, h = tm.add_rms_norm(x, h, w)
            out.append(tm.apply_logit_controls(torch.nn.functional.linear(y, head), tokens=tokens, token_lengths=known, repetition=penalty))
        return out + [x, h, k_pages.nan_to_num().clone(), v_pages.nan_to_num().clone()]

    on = chain()
    overlapping.tris_set_programmatic_launch(0)
    off = chain()
    assert all(torch.equal(a, b) for a, b in zip(on, off))


def test_inputs_that_require_a_gradient_are_refused(lib):
    """Nothing here has a gradient: a call that would drop one says so."""
    import trismoe_b200 as tm

    new = lambda *s, dtype=F16: torch.zeros(s, dtype=dtype, device="cuda")
    asks = lambda *s, dtype=F16: new(*s, dtype=dtype).requires_grad_()
    i32, f32 = torch.int32, torch.float32
    table, lens, pos, pages = new(2, 3, dtype=i32), new(2, dtype=i32), new(2, dtype=i32), new(4, 16, 2, 64)
    q, k = new(2, 4, 64), new(2, 2, 64)
    calls = [
        lambda: tm.append_paged_kv(asks(2, 4, 64), k, k, pages, pages, table, pos), lambda: tm.append_paged_kv(q, k, asks(2, 2, 64), pages, pages, table, pos),
        lambda: tm.paged_decode_attention(asks(2, 4, 64), pages, pages, table, lens), lambda: tm.paged_decode_attention(q, pages, asks(4, 16, 2, 64), table, lens),
        lambda: tm.add_rms_norm(asks(2, 64), None, new(64)), lambda: tm.add_rms_norm(new(2, 64), None, asks(64)), lambda: tm.add_rms_norm_e4m3(new(2, 64), asks(2, 64), new(64)),
        lambda: tm.apply_logit_controls(asks(2, 40, dtype=f32)),
        lambda: tm.apply_logit_controls(new(2, 40, dtype=f32), bias_ids=new(2, 1, dtype=i32), bias_values=asks(2, 1, dtype=f32)),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="gradient"):
            call()
        with torch.no_grad():
            call()


# ---- append ---------------------------------------------------------------------------------
@pytest.mark.parametrize("extra", [0, 1], ids=["wide", "element by element"])
@pytest.mark.parametrize("dim,rot", [(64, 16), (128, 120), (48, 4), (80, 0), (256, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_leaves_dimensions_that_do_not_rotate_as_they_are(lib, dim, rot, interleaved, extra):
    """Infinities, NaN and zeros of both signs beside one another, behind the rotated dimensions."""
    import trismoe_b200 as tm

    g, tokens = _gen(dim + rot), 9
    k_pages, v_pages, table, _ = _filled(g, [tokens], 16, 2, dim, F16, LAYOUTS[0])
    flat = torch.randn((tokens, 8 * dim + extra), generator=g, device="cuda").half()
    rows = flat[:, extra:].unflatten(1, (8, dim))
    odd = torch.tensor([math.inf, 1.0, -0.0, -math.inf, math.nan, 2.0, -0.0, -0.0, 3.0, math.inf], device="cuda").half()
    rows[..., rot:] = odd[(torch.arange(tokens * 8 * (dim - rot), device="cuda") % 10).view(tokens, 8, dim - rot)]
    cos = sin = None
    if rot:
        angle = torch.rand((tokens, rot // 2), generator=g, device="cuda") * 6.0
        cos, sin = angle.cos(), angle.sin()
    q, k = tm.append_paged_kv(rows[:, :4], rows[:, 4:6], rows[:, 6:], k_pages, v_pages, table, torch.arange(tokens, device="cuda"),
                              torch.zeros((tokens,), dtype=torch.int32, device="cuda"), cos=cos, sin=sin, interleaved=interleaved, return_key=True)
    bits = lambda t: torch.where(t.isnan(), torch.full_like(t, math.nan), t).contiguous().view(torch.int16)
    held = k_pages[table[0, 0].long(), :tokens]
    for got, want in ((q, rows[:, :4]), (k, rows[:, 4:6]), (held, rows[:, 4:6])):
        assert torch.equal(bits(got[..., rot:]), bits(want[..., rot:]))
        assert bool(torch.isfinite(got[..., :rot]).all())


@pytest.mark.parametrize("extra", [0, 1], ids=["wide", "element by element"])
@pytest.mark.parametrize("rows,odd", [(F16, 7), (F16, 63), (BF16, 7)], ids=["fp16 7", "fp16 63", "bf16 7"])
def test_append_to_8_bits_rounds_the_quotient(lib, rows, odd, extra):
    """Half way between two e4m3 values the result is the even one.  x / scale is exact there, x * (1 / scale) need not be."""
    import trismoe_b200 as tm

    half_way = (torch.arange(16, 32, device="cuda") / 16.0).repeat(4) * torch.tensor([1.0, -1.0, 16.0, -8.0], device="cuda").repeat_interleave(16)
    scale = torch.tensor([odd / 64.0, 1.0], device="cuda")
    flat = torch.zeros((1, 2 * 64 + extra), dtype=rows, device="cuda")
    x = flat[:, extra:].view(1, 2, 64)
    x.copy_((half_way * scale[:, None])[None])
    assert torch.equal(x[0].double() / scale.double()[:, None], half_way.double().expand(2, 64))
    pages = [torch.zeros((1, 2, 16, 64), dtype=E4M3, device="cuda").transpose(1, 2) for _ in range(2)]
    table, zero = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros((1,), dtype=torch.int32, device="cuda")
    tm.append_paged_kv(None, x, x, *pages, table, zero, k_scale=scale, v_scale=scale)
    for p in pages:
        assert torch.equal(p[0, 0].float(), half_way.to(E4M3).float().expand(2, 64))


def test_append_to_8_bits_with_a_scale_whose_reciprocal_overflows(lib):
    import trismoe_b200 as tm

    x = torch.tensor([0.0, -0.0, 1.0, -2.0 ** -24] * 16, device="cuda").half().view(1, 1, 64)
    pages = [torch.ones((1, 1, 16, 64), dtype=F16, device="cuda").to(E4M3).transpose(1, 2) for _ in range(2)]
    table, zero = torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros((1,), dtype=torch.int32, device="cuda")
    scale = torch.full((1,), 2.0 ** -140, device="cuda")
    tm.append_paged_kv(None, x, x, *pages, table, zero, k_scale=scale, v_scale=scale)
    for p in pages:
        assert torch.equal(p[0, 0, 0].float(), torch.tensor([0.0, -0.0, 448.0, -448.0] * 16, device="cuda"))


@pytest.mark.parametrize("rows", [F16, BF16], ids=["fp16", "bf16"])
def test_append_to_8_bits_divides_numbers_of_any_size(lib, rows):
    """Bit for bit the quotient in 32 bits, saturated and rounded: scales from 2^-149 to 2^127, and rows with everything that is not finite."""
    import trismoe_b200 as tm

    g = _gen(49)
    scale = torch.cat([2.0 ** torch.arange(-149.0, 128.0, 4.0, dtype=torch.float64), 2.0 ** torch.tensor([-81.0, -80.0, 80.0, 81.0]).double()]).float().cuda()
    scale = scale * (1.0 + torch.rand(scale.shape, generator=g, device="cuda")).clamp(max=1.99)
    heads, tokens, dim = scale.numel(), 64, 128
    x = torch.randn((tokens, heads, dim), generator=g, device="cuda") * 10.0
    x[1::2] *= scale.clamp(1e-6, 1e6)[:, None]
    x[::2] *= 2.0 ** torch.randint(-40, 40, (tokens // 2, heads, dim), generator=g, device="cuda").float()
    x[5, :, :6] = torch.tensor([math.inf, -math.inf, math.nan, 0.0, -0.0, 65504.0], device="cuda")
    x = x.to(rows)
    pages = [torch.zeros((4, heads, 16, dim), dtype=E4M3, device="cuda").transpose(1, 2) for _ in range(2)]
    table, zero = torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.zeros((tokens,), dtype=torch.int32, device="cuda")
    tm.append_paged_kv(None, x, x, *pages, table, torch.arange(tokens, device="cuda"), zero, k_scale=scale, v_scale=scale)
    want = (x.float() / scale[:, None]).clamp(-448.0, 448.0).to(E4M3).float()
    for p in pages:
        got = p.reshape(tokens, heads, dim).float()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_append_of_tokens_that_have_no_sequence_is_refused(lib):
    import trismoe_b200 as tm

    pages = torch.zeros((4, 16, 2, 64), dtype=F16, device="cuda")
    x = torch.zeros((3, 2, 64), dtype=F16, device="cuda")
    table, at = torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.zeros((3,), dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="sequences"):
        tm.append_paged_kv(x, x, x, pages, pages, table, at)
    tm.append_paged_kv(x[:2], x[:2], x[:2], pages, pages, table, at[:2])


# ---- attention ------------------------------------------------------------------------------
@pytest.mark.parametrize("small", [2.0 ** -14, 2.0 ** -20, 2.0 ** -26])
def test_small_elements_of_a_query_over_8_bit_pages(lib, small):
    """Keys are zero where the query is large, so the scores are made of what is small in it: no bit of it may be lost beside the large element."""
    import trismoe_b200 as tm

    g, lengths, dim = _gen(40), [1, 16, 200], 64
    k_pages, v_pages, table, kept = _filled(g, lengths, 16, 1, dim, E4M3, LAYOUTS[0])
    for b, n in enumerate(lengths):
        kept[b][0][..., 0] = 0.0
        place = torch.arange(n, device="cuda")
        k_pages[table[b, place // 16].long(), place % 16] = kept[b][0].to(E4M3)
    q = torch.randn((3, 4, dim), generator=g, device="cuda") * small
    q[..., 0] = 1.75
    _check_attention(tm, q.to(BF16), (k_pages, v_pages, table, kept), lengths, softmax_scale=0.25 / small)


@pytest.mark.parametrize("rows,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)], ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("lengths", [[3, 2, 5, 64], [700, 1000], [20000]], ids=["short", "clusters", "numbered"])
def test_attention_keeps_more_of_a_weight_than_16_bits(lib, rows, cache, lengths):
    """Values of +-1 that cancel: the result is small beside the sum of magnitudes, so a rounding of the weights would show.
    Weights have the error of their scores (at most 2^-17: sums of 64 products in 32 bits) and of two roundings to 8 bits (2^-16) at most; of one to 11 bits (2^-12) in addition
    where the result is in bf16, whose own rounding is eight times as large, and pages are in 8 bits."""
    import trismoe_b200 as tm

    g, heads, dim = _gen(41), 8, 64
    k_pages, v_pages, table, kept = _filled(g, lengths, 16, 2, dim, cache, LAYOUTS[0])
    for b, n in enumerate(lengths):
        kept[b][1].sign_()
        place = torch.arange(n, device="cuda")
        v_pages[table[b, place // 16].long(), place % 16] = kept[b][1].to(cache)
    q = torch.randn((len(lengths), heads, dim), generator=g, device="cuda").to(rows)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = tm.paged_decode_attention(q, k_pages, v_pages, table, lens)
    want, _, mag = _attend_64(q, kept, 0, dim ** -0.5, None, None)
    bound = (2.0 ** -15 + (2.0 ** -12 if rows == BF16 and cache == E4M3 else 0.0)) * mag + U[rows] * want.abs() + SUB[rows]
    assert float(((out.double() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("rows,cache", [(F16, F16), (BF16, BF16), (BF16, E4M3)], ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("lengths", [[1, 2, 64, 700], [20000]], ids=["clusters", "numbered"])
def test_an_infinite_value_gives_an_infinity_whatever_its_weight(lib, rows, cache, lengths):
    """Weights that are a power of two, or a number of 16 bits, exactly, and others; what has no infinity stands in with e4m3's largest number."""
    import trismoe_b200 as tm

    g, heads, dim, n = _gen(51), 4, 64, len(lengths)
    k_pages, v_pages, table, kept = _filled(g, lengths, 16, 1, dim, cache, LAYOUTS[0], scale=0.5)
    q = torch.randn((n, heads, dim), generator=g, device="cuda").to(rows)
    q[:, 0] = 0.0  # equal weights
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if cache == E4M3:
        v_pages.copy_(torch.full_like(v_pages, 448.0, dtype=torch.float32))
        out = tm.paged_decode_attention(q, k_pages, v_pages, table, lens)
        assert float((out.double() - 448.0).abs().max()) <= 2.0 ** -8 * 448.0
        return
    for b, length in enumerate(lengths):
        for i, sign in ((0, 1.0), (length // 2, -1.0), (length - 1, 1.0)):
            v_pages[table[b, i // 16].long(), i % 16, 0, 3 * i % 61] = sign * math.inf
    out = tm.paged_decode_attention(q, k_pages, v_pages, table, lens)
    for b, length in enumerate(lengths):
        want = torch.zeros((dim,), device="cuda", dtype=torch.float64)
        for i in (0, length // 2, length - 1):
            want[3 * i % 61] += v_pages[table[b, i // 16].long(), i % 16, 0, 3 * i % 61].double()
        odd = ~torch.isfinite(want)
        assert bool(odd.any()) and bool(torch.isfinite(out[b][:, ~odd]).all())
        for h in range(heads):
            assert torch.equal(out[b, h][odd].double().nan_to_num(nan=7.0), want[odd].nan_to_num(nan=7.0))


def test_a_negative_length_is_reported(lib):
    import trismoe_b200 as tm

    g = _gen(42)
    for longest in (40, 20000):  # by clusters and numbered
        k_pages, v_pages, table, _ = _filled(g, [longest, 20], 16, 1, 64, F16, LAYOUTS[0])
        q = torch.randn((2, 2, 64), generator=g, device="cuda").half()
        status = torch.zeros((1,), dtype=torch.int32, device="cuda")
        good = tm.paged_decode_attention(q, k_pages, v_pages, table, torch.tensor([longest, 20], dtype=torch.int32, device="cuda"), status=status)
        tm.raise_on_status(status)
        out = tm.paged_decode_attention(q, k_pages, v_pages, table, torch.tensor([longest, -1], dtype=torch.int32, device="cuda"), status=status)
        with pytest.raises(RuntimeError, match="CORRUPT"):
            tm.raise_on_status(status)
        assert torch.equal(out[0], good[0]) and bool((out[1] == 0).all())


def test_a_capture_leaves_no_scratch_behind_in_its_pool(lib):
    """What a first call inside a capture allocates goes with the graph."""
    import trismoe_b200 as tm
    from trismoe_b200 import decode_ops

    g, lengths = _gen(43), [20011]
    k_pages, v_pages, table, _ = _filled(g, lengths, 16, 1, 72, F16, LAYOUTS[0])
    q = torch.randn((1, 1, 72), generator=g, device="cuda").half()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    known = dict(decode_ops._scratch)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = tm.paged_decode_attention(q, k_pages, v_pages, table, lens)
    graph.replay()
    assert decode_ops._scratch == known
    eager = tm.paged_decode_attention(q, k_pages, v_pages, table, lens)
    assert torch.equal(out, eager) and len(decode_ops._scratch) == len(known) + 1


# ---- norm -----------------------------------------------------------------------------------
@pytest.mark.parametrize("extra", [0, 1], ids=["wide", "element by element"])
@pytest.mark.parametrize("dtype,odd", [(F16, 7), (F16, 63), (BF16, 7)], ids=["fp16 7", "fp16 63", "bf16 7"])
@pytest.mark.parametrize("group", [0, 32, 96])
def test_norm_to_8_bits_rounds_the_quotients(lib, dtype, odd, group, extra):
    """Rows of +-1 have a mean square of 1, so with eps 0 y is the weight; weights half way between two e4m3 values times the scale."""
    import trismoe_b200 as tm

    scale = odd / 64.0
    part = torch.cat([torch.tensor([448.0], device="cuda"), torch.arange(16, 32, device="cuda") / 16.0, torch.arange(17, 32, device="cuda") / 2.0])
    values = part.repeat(9)  # 288 columns, every 32 of them with the largest
    w = (values * scale).to(dtype)
    assert torch.equal(w.double(), values.double() * scale)
    sign = torch.where(torch.rand((5, 288), generator=_gen(45), device="cuda") < 0.5, -1.0, 1.0)
    x = torch.empty((5, 288 + extra), dtype=dtype, device="cuda")[:, extra:]
    x.copy_(sign)
    got, scales, _ = tm.add_rms_norm_e4m3(x, None, w, 0.0, group_size=group)
    assert bool((scales == scale).all())
    assert torch.equal(got.float(), sign * values.to(E4M3).float())


@pytest.mark.parametrize("size", [2.0 ** -130, 2.0 ** -126, 2.0 ** -100, 2.0 ** -60, 1.0, 2.0 ** 60, 2.0 ** 120])
def test_norm_to_8_bits_over_the_range_of_scales(lib, size):
    """bf16 weights of any size: values are right to a rounding to e4m3, scales to a rounding to fp32 (of a subnormal scale: to 2^-149)."""
    import trismoe_b200 as tm

    w = (torch.randn((512,), generator=_gen(46), device="cuda").double() * size).to(BF16)
    x = torch.ones((2, 512), dtype=BF16, device="cuda")
    values, scales, _ = tm.add_rms_norm_e4m3(x, None, w, 0.0, group_size=128)
    want = w.double().abs().view(4, 128).amax(1) / 448.0
    assert float(((scales.double() - want).abs() - 2.0 ** -22 * want - 2.0 ** -149).max()) <= 0
    part, back = w.double().view(4, 128), values.double().view(2, 4, 128)
    # of a scale of few bits the quotient by the scale as it is stored
    quotient = part / scales.double()[..., None]
    bound = (U[E4M3] + 2.0 ** -20) * quotient.abs().clamp(max=480.0) + SUB[E4M3]
    held = scales.double()[..., None] > 2.0 ** -140
    assert float((((back - quotient.clamp(-448.0, 448.0)).abs() - bound) * held).max()) <= 0
    assert bool(torch.isfinite(back).all())


@pytest.mark.parametrize("group", [0, 16, 48, 96])
def test_norm_to_8_bits_of_what_is_not_a_number(lib, group):
    """A NaN makes its group's scale one, wherever it comes from - a weight, an infinite weight on zero, a row of zeros without eps, a negative eps -,
    in both kernels."""
    import trismoe_b200 as tm

    g = _gen(44)
    x = torch.randn((4, 288), generator=g, device="cuda").half()
    x[1] = 0.0
    x[2, 100] = 0.0
    off = torch.empty((4, 289), dtype=F16, device="cuda")[:, 1:]  # element by element
    off.copy_(x)
    w = torch.ones((288,), dtype=F16, device="cuda")
    for place, weight, eps in ((5, math.nan, 1e-5), (100, math.inf, 1e-5), (100, -math.inf, 1e-5), (0, 1.0, 0.0), (0, 1.0, -1e3)):
        w.fill_(1.0)
        w[place] = weight
        h = x.double()
        y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        want = y.view(4, -1, group or 288).abs().amax(-1) / 448.0
        assert bool(want.isnan().any())
        for rows in (x, off):
            values, scales, _ = tm.add_rms_norm_e4m3(rows, None, w, eps, group_size=group)
            assert torch.equal(scales.isnan(), want.isnan())
            assert torch.equal(scales.isinf(), want.isinf())
            assert bool(values.float().isnan()[y.isnan()].all())


# ---- logits ---------------------------------------------------------------------------------
@pytest.mark.parametrize("rows,vocab", [(2, 4000), (40, 50304)], ids=["small slices", "large slices"])
def test_repetition_divides(lib, rows, vocab):
    """Positive logits are the quotients to the last bit."""
    import trismoe_b200 as tm

    logits = 1.0 + torch.randint(0, 2000, (rows, vocab), generator=_gen(60), device="cuda").float()
    repetition = 1.0 + torch.arange(rows, device="cuda") * 2.0 + 46.0
    tokens = torch.arange(vocab, dtype=torch.int32, device="cuda").expand(rows, vocab).contiguous()
    lengths = torch.full((rows,), vocab, dtype=torch.int32, device="cuda")
    out = tm.apply_logit_controls(logits, tokens=tokens, token_lengths=lengths, repetition=repetition)
    assert torch.equal(out, (logits.double() / repetition.double()[:, None]).float())
    out = tm.apply_logit_controls(-logits, tokens=tokens, token_lengths=lengths, repetition=repetition)
    assert torch.equal(out, -logits * repetition[:, None])


def test_repetition_whose_reciprocal_is_not_finite(lib):
    import trismoe_b200 as tm

    logits = torch.tensor([[2.0 ** -100, -1.0, 2.0 ** -140, 0.0]], device="cuda")
    tokens = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    out = tm.apply_logit_controls(logits, tokens=tokens, token_lengths=torch.full((1,), 4, dtype=torch.int32, device="cuda"),
                                  repetition=torch.full((1,), 2.0 ** -130, device="cuda"))
    assert torch.equal(out, torch.tensor([[2.0 ** 30, -(2.0 ** -130), 2.0 ** -10, 0.0]], device="cuda"))


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("rows,vocab,biases", [(2, 1000, 700), (1, 50304, 9000), (40, 50304, 600), (3, 37, 5000)])
def test_repeated_biases_add_up_in_their_order(lib, rows, vocab, biases, masked):
    """Ids that occur once, a few times and very often, in any order; sums in 32 bits, one entry after the other."""
    import trismoe_b200 as tm

    g = _gen(biases)
    ids = torch.randint(-3, vocab + 3, (rows, biases), generator=g, device="cuda", dtype=torch.int32)
    ids[:, biases // 3: biases // 2] = vocab // 2
    ids[:, : biases // 3: 2] = ids[:, biases // 2: biases // 2 + len(range(0, biases // 3, 2))]
    values = torch.randn((rows, biases), generator=g, device="cuda") * 3.0
    logits = torch.randn((rows, vocab), generator=g, device="cuda")
    c = {"bias_ids": ids, "bias_values": values}
    if masked:
        c["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    want, mag = _controls_64(logits, c)
    got = tm.apply_logit_controls(logits, **c)
    assert torch.equal(got, tm.apply_logit_controls(logits, **c))
    finite = torch.isfinite(want)
    assert torch.equal(got[~finite].double(), want[~finite])
    # as many roundings as an id has entries, each at most 2^-24 of the magnitudes
    entries = torch.zeros((rows, vocab), device="cuda", dtype=torch.float64)
    ok = (ids >= 0) & (ids < vocab)
    entries.scatter_add_(1, torch.where(ok, ids, 0).long(), ok.double())
    assert float(((got.double() - want).abs() - (2 + entries) * 2.0 ** -24 * mag)[finite].max()) <= 0


def test_a_long_list_of_biases_with_a_repeated_id_takes_time_by_its_length(lib):
    """25000 entries, one of them twice: some 60 us; milliseconds would be a search of the list for each of its entries."""
    import trismoe_b200 as tm

    ids = torch.randperm(50304, generator=_gen(52), device="cuda")[None, :25000].int()
    ids[0, -1] = ids[0, 0]
    c = {"bias_ids": ids, "bias_values": torch.randn((1, 25000), generator=_gen(53), device="cuda")}
    logits = torch.randn((1, 50304), generator=_gen(54), device="cuda")
    tm.apply_logit_controls(logits, **c)
    times = []
    for _ in range(5):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        tm.apply_logit_controls(logits, **c)
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    assert min(times) < 3.0


def test_strides_of_sizes_of_one_are_of_no_account(lib):
    """A dimension of size 1 may have any stride: one head, one page, pages of one token; one row of biases."""
    import trismoe_b200 as tm

    g = _gen(50)
    for pages, page, heads in ((5, 4, 1), (1, 40, 2), (20, 1, 2)):
        k_pages, v_pages, table, rows = _filled(g, [17], page, heads, 64, F16, LAYOUTS[1], spare=pages - -(-17 // page))
        assert k_pages.shape == (pages, page, heads, 64)
        strides = [3 if n == 1 else s for n, s in zip(k_pages.shape, k_pages.stride())]
        odd = [p.as_strided(p.shape, strides) for p in (k_pages, v_pages)]
        q = torch.randn((1, 4, 64), generator=g, device="cuda").half()
        _check_attention(tm, q, (*odd, table, rows), [17])
        new = torch.randn((1, heads, 64), generator=g, device="cuda").half()
        tm.append_paged_kv(None, new, new, *odd, table, torch.tensor([16], dtype=torch.int32, device="cuda"))
        assert torch.equal(k_pages[table[0, 16 // page].long(), 16 % page], new[0]) and torch.equal(v_pages[table[0, 16 // page].long(), 16 % page], new[0])
    ids = torch.tensor([[3, 7, -1, 3, 9]], dtype=torch.int32, device="cuda")[:, :4]
    values = torch.ones((1, 40), device="cuda")[:, 10:14]
    want = torch.zeros((1, 40), device="cuda")
    want[0, 3], want[0, 7] = 2.0, 1.0
    assert torch.equal(tm.apply_logit_controls(torch.zeros((1, 40), device="cuda"), bias_ids=ids, bias_values=values), want)


def test_a_window_of_any_size(lib):
    """A window beyond 32 bits is no window; a negative one is refused."""
    import trismoe_b200 as tm

    g, lengths = _gen(55), [300, 7]
    k_pages, v_pages, table, _ = _filled(g, lengths, 16, 2, 64, F16, LAYOUTS[0])
    q = torch.randn((2, 4, 64), generator=g, device="cuda").half()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = tm.paged_decode_attention(q, k_pages, v_pages, table, lens)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 40):
        assert torch.equal(tm.paged_decode_attention(q, k_pages, v_pages, table, lens, window=window), want)
    with pytest.raises(RuntimeError, match="window"):
        tm.paged_decode_attention(q, k_pages, v_pages, table, lens, window=-2 ** 40)


def test_an_output_whose_rows_overlap_is_refused(lib):
    import trismoe_b200 as tm

    logits = torch.randn((3, 40), generator=_gen(55), device="cuda")
    for out in (torch.empty((1, 40), device="cuda").expand(3, 40), torch.empty((200,), device="cuda").as_strided((3, 40), (39, 1))):
        with pytest.raises(RuntimeError, match="out must be"):
            tm.apply_logit_controls(logits, out=out)
    assert torch.equal(tm.apply_logit_controls(logits[:1], out=torch.empty((1, 40), device="cuda").as_strided((1, 40), (0, 1))), logits[:1])


# ---- sizes that lead to each variant --------------------------------------------------------
def test_lse_of_small_scores(lib):
    """Scores below 1 and few tokens: products are exact, sums, exponentials and logarithm a few roundings of 2^-23 each; a weight of 16 bits would be
    off by 2^-12."""
    import trismoe_b200 as tm

    g, lengths = _gen(47), [1, 2, 3, 5, 9, 40]
    for rows in (F16, BF16):
        k_pages, v_pages, table, kept = _filled(g, lengths, 16, 1, 64, rows, LAYOUTS[0])
        q = (torch.randn((6, 8, 64), generator=g, device="cuda") * 0.25).to(rows)
        _, lse = tm.paged_decode_attention(q, k_pages, v_pages, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), return_lse=True)
        _, want, _ = _attend_64(q, kept, 0, 0.125, None, None)
        assert float((lse.double() - want).abs().max()) <= 2.0 ** -18


def _workspace(lib, q, k_pages, table, window=0):
    from trismoe_b200 import decode_ops

    packed, _ = decode_ops._cache("test", k_pages, k_pages, table, None, None, None)
    return lib.tris_paged_decode_attention_workspace_bytes(packed, q.shape[1], window)


def test_attention_of_so_many_blocks_that_a_warp_has_a_long_run(lib):
    """Numbered blocks, 64 and more to a warp of the doubled grid: 148 SMs x 3 CTAs x 2 x 4 warps x 64 are 227 000 blocks."""
    import trismoe_b200 as tm

    g, lengths = _gen(48), [150000, 0, 1, 90001, 63, 70000, 16, 33333, 130000]
    k_pages, v_pages, table, kept = _filled(g, lengths, 16, 8, 16, F16, LAYOUTS[0])
    q = torch.randn((9, 8, 16), generator=g, device="cuda").half()
    assert sum(-(-n // 16) for n in lengths) * 8 > 230_000 and _workspace(lib, q, k_pages, table) > 0
    _check_attention(tm, q, (k_pages, v_pages, table, kept), lengths)


@pytest.mark.parametrize("window", [4096, 4111, 9999])
@pytest.mark.parametrize("rows,cache", [(F16, F16), (BF16, E4M3)], ids=["fp16", "e4m3"])
def test_attention_in_a_window_over_numbered_blocks(lib, rows, cache, window):
    import trismoe_b200 as tm

    g, lengths = _gen(window), [20000, 5000, 0, 17, 4096]
    filled = _filled(g, lengths, 16, 1, 128, cache, LAYOUTS[0])
    q = torch.randn((5, 4, 128), generator=g, device="cuda").to(rows)
    assert _workspace(lib, q, filled[0], filled[2], window) > 0
    _check_attention(tm, q, filled, lengths, window=window)


@pytest.mark.parametrize("width", [512, 8192])
@pytest.mark.parametrize("lengths", [[513], [1, 0, 70, 300]], ids=["one", "four"])
def test_attention_of_short_sequences_in_a_wide_table(lib, lengths, width):
    """A table with room for 8192 or 131072 tokens, as a server has."""
    import trismoe_b200 as tm

    g = _gen(width)
    k_pages, v_pages, table, kept = _filled(g, lengths, 16, 4, 128, F16, LAYOUTS[0])
    wide = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    q = torch.randn((len(lengths), 8, 128), generator=g, device="cuda").half()
    _check_attention(tm, q, (k_pages, v_pages, wide, kept), lengths)


@pytest.mark.parametrize("rows,hidden,groups", [(2047, 2048, (0, 128, 512)), (2047, 4096, (0, 128, 1024)), (1000, 8192, (0, 128, 2048)), (3, 768, (48, 384)),
                                                (1200, 768, (48, 384)), (2, 1680, (240, 560)), (700, 1680, (240,)), (2000, 256, (0, 16, 64))])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_norm_of_many_rows_and_odd_groups(lib, rows, hidden, groups, dtype):
    """Several rows to a CTA in each variant, groups wider than a warp and not of a power of two, rows off 16-byte boundaries too."""
    import trismoe_b200 as tm

    g = _gen(rows + hidden)
    x, res = (s * torch.randn((rows, hidden), generator=g, device="cuda") for s in (1.0, 3.0))
    x, res = x.to(dtype), res.to(dtype)
    w = (1.0 + 0.2 * torch.randn((hidden,), generator=g, device="cuda")).to(dtype)
    h64 = x.double() + res.double()
    want = h64 / (h64.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
    off = torch.empty((rows, hidden + 1), dtype=dtype, device="cuda")[:, 1:]
    off.copy_(x)
    for rows_ in (x, off):
        y, h = tm.add_rms_norm(rows_, res, w, 1e-5)
        assert torch.equal(h, h64.to(dtype))
        assert float(((y.double() - want).abs() - (U[dtype] + 2.0 ** -17) * want.abs() - SUB[dtype]).max()) <= 0
        for group in groups:
            values, scales, h8 = tm.add_rms_norm_e4m3(rows_, res, w, 1e-5, group_size=group)
            parts = want.view(rows, -1, group or hidden)
            want_scale = parts.abs().amax(-1) / 448.0
            assert torch.equal(h8, h) and float(((scales.double() - want_scale).abs() - 2.0 ** -16 * want_scale).max()) <= 0
            back = values.double().view(parts.shape) * scales.double()[..., None]
            assert float(((back - parts).abs() - (U[E4M3] + 2.0 ** -15) * parts.abs() - 1.01 * SUB[E4M3] * want_scale[..., None]).max()) <= 0


@pytest.mark.parametrize("rows,vocab,history", [(40, 50304, 3000), (300, 4001, 64), (90, 20000, 40000), (25, 65536, 500)])
@pytest.mark.parametrize("dtype", [F16, torch.float32], ids=["fp16", "fp32"])
def test_logit_controls_in_large_slices(lib, rows, vocab, history, dtype):
    """More than two CTAs an SM would have with slices of 4096: large slices, over which a CTA streams in several turns."""
    import trismoe_b200 as tm

    assert -(-vocab // 4096) * rows >= 2 * 148
    g = _gen(rows + vocab)
    rand = lambda *s: torch.rand(s, generator=g, device="cuda")
    ints = lambda low, high, *s: torch.randint(low, high, s, generator=g, device="cuda", dtype=torch.int32)
    logits = (torch.randn((rows, vocab + 3), generator=g, device="cuda") * 5.0).to(dtype)[:, 1: vocab + 1]
    tokens = ints(-2, vocab + 2, rows, history)
    tokens[:, : history // 2] %= vocab // 50
    ids = ints(-2, vocab + 1, rows, 37)
    ids[:, 20:] = ids[:, :17]
    c = {"tokens": tokens, "token_lengths": ints(-1, history + 5, rows), "prompt_lengths": ints(0, history + 2, rows), "repetition": 0.5 + rand(rows),
         "presence": rand(rows), "frequency": rand(rows), "bias_ids": ids, "bias_values": torch.randn((rows, 37), generator=g, device="cuda"),
         "allowed": torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)}
    c["allowed"][0] = 0
    for aligned in (False, True):
        src = logits.contiguous() if aligned else logits
        want, mag = _controls_64(src, c)
        got = tm.apply_logit_controls(src, **c)
        finite = torch.isfinite(want)
        assert torch.equal(got[~finite].double(), want[~finite])
        # each of some ten roundings is at most 2^-24 of the magnitudes added up
        assert float(((got.double() - want).abs() - 12 * 2.0 ** -24 * mag)[finite].max()) <= 0
        if dtype == torch.float32:
            same = src.clone()
            assert torch.equal(tm.apply_logit_controls(same, out=same, **c), got) and bool((got == same).all())
