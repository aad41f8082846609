"""GPU tests of the operators of a decode step against plain implementations in 64 bits.

Tolerances.  u is the largest relative error of a rounding to the type (fp16 2^-11, bf16 2^-8, e4m3 2^-4); SUB half its smallest subnormal.
Attention: weights are rounded to 16 bits before they multiply values (u of sum w |v| / sum w = A), the result once more (u of it);
scores are fp32 sums of up to 256 products of magnitude up to some 60 in all, 16 to a step: below 2^-12 in a weight.
Rotation: two products and a sum in fp32, then one rounding.  Norm: fp32 sums of up to 64 squares per thread, below 2^-17."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, E4M3: 2.0 ** -4}
SUB = {F16: 2.0 ** -25, BF16: 0.0, E4M3: 2.0 ** -10}
# [num_pages, page_size, heads, head_dim] views of three memory orders
LAYOUTS = ("heads outside", "tokens outside", "keys and values together")


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pages(layout, pages, page, heads, dim, dtype):
    new = lambda *s: torch.full(s, math.nan, dtype=torch.float32, device="cuda").to(dtype)
    if layout == "heads outside":
        return tuple(new(pages, heads, page, dim).transpose(1, 2) for _ in range(2))
    if layout == "tokens outside":
        return tuple(new(pages, page, heads, dim) for _ in range(2))
    both = new(pages, page, heads, 2, dim)
    return both[..., 0, :], both[..., 1, :]


def _filled(g, lengths, page, heads, dim, dtype, layout, scale=1.0, spare=2):
    """Pages with random keys and values where a sequence has tokens and NaN everywhere else, and a block table with
    impossible pages behind every sequence's last."""
    counts = [-(-n // page) for n in lengths]
    total = sum(counts) + spare
    k_pages, v_pages = _pages(layout, total, page, heads, dim, dtype)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(1, max(counts)) + 1), 2 ** 30, dtype=torch.int32, device="cuda")
    table[:, 1::2] = -7
    rows, at = [], 0
    for b, n in enumerate(lengths):
        table[b, : counts[b]] = order[at: at + counts[b]]
        at += counts[b]
        place = torch.arange(n, device="cuda")
        k, v = (scale * torch.randn((n, heads, dim), generator=g, device="cuda") for _ in range(2))
        page_of = table[b, place // page].long()
        k_pages[page_of, place % page] = k.to(dtype)
        v_pages[page_of, place % page] = v.to(dtype)
        rows.append((k.to(dtype).double(), v.to(dtype).double()))
    return k_pages, v_pages, table, rows


def _attend_64(q, rows, window, softmax_scale, k_scale, v_scale):
    """out, lse and the mean magnitude of the values under the weights, from the definition."""
    batch, heads, dim = q.shape
    out, mag = (torch.zeros((batch, heads, dim), dtype=torch.float64, device="cuda") for _ in range(2))
    lse = torch.full((batch, heads), -math.inf, dtype=torch.float64, device="cuda")
    for b, (k, v) in enumerate(rows):
        if window:
            k, v = k[-window:], v[-window:]
        if not k.shape[0]:
            continue
        kv = k.shape[1]
        for h in range(heads):
            j = h // (heads // kv)
            ks = 1.0 if k_scale is None else k_scale[j].double()
            vs = 1.0 if v_scale is None else v_scale[j].double()
            s = (k[:, j] @ q[b, h].double()) * ks * softmax_scale
            w = torch.softmax(s, 0)
            lse[b, h] = torch.logsumexp(s, 0)
            out[b, h], mag[b, h] = w @ (v[:, j] * vs), w @ (v[:, j] * vs).abs()
    return out, lse, mag


def _check_attention(tm, q, filled, lengths, window=0, k_scale=None, v_scale=None, softmax_scale=None):
    k_pages, v_pages, table, rows = filled
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = tm.paged_decode_attention(q, k_pages, v_pages, table, lens, window=window, k_scale=k_scale, v_scale=v_scale,
                                         softmax_scale=softmax_scale, return_lse=True, status=status)
    tm.raise_on_status(status)
    want, want_lse, mag = _attend_64(q, rows, window, q.shape[2] ** -0.5 if softmax_scale is None else softmax_scale, k_scale, v_scale)
    u = U[F16 if k_pages.dtype == E4M3 else q.dtype]
    bound = (u + 2.0 ** -12) * mag + U[q.dtype] * want.abs() + SUB[q.dtype]
    assert out.dtype == q.dtype and out.shape == q.shape
    worst = ((out.double() - want).abs() - bound).max()
    assert bool(torch.isfinite(out).all()) and float(worst) <= 0, float(worst)
    empty = lens == 0
    assert bool((out[empty] == 0).all()) and bool((lse[empty] == -math.inf).all())
    assert float((lse[~empty].double() - want_lse[~empty]).abs().max() if bool((~empty).any()) else 0.0) <= 2.0 ** -11
    again = tm.paged_decode_attention(q, k_pages, v_pages, table, lens, window=window, k_scale=k_scale, v_scale=v_scale, softmax_scale=softmax_scale)
    assert torch.equal(again, out)  # the partial results join in a fixed order
    return out


SHAPES = [  # q heads, kv heads, head_dim, rows, cache
    (16, 16, 128, F16, F16), (32, 8, 128, BF16, BF16), (16, 2, 256, BF16, E4M3), (8, 8, 128, F16, E4M3), (4, 2, 64, F16, F16),
    (5, 1, 80, BF16, BF16), (12, 1, 96, F16, F16), (6, 3, 48, BF16, E4M3), (16, 1, 256, F16, F16), (40, 1, 128, BF16, BF16),
    (2, 2, 8, F16, F16), (9, 1, 64, BF16, E4M3), (20, 1, 112, F16, E4M3), (3, 1, 192, BF16, BF16), (2, 1, 16, F16, E4M3), (17, 1, 256, BF16, E4M3),
]
# short ones are attended to by clusters, long ones by numbered blocks; the last ones keep two tiles of heads together in clusters, too
LENGTHS = [[1], [0], [16, 0, 1, 17, 15], [33, 300, 1, 0, 129, 1000, 64], [2500], [9000, 1, 0, 40], [(13 * i) % 70 for i in range(100)],
           [(29 * i) % 200 for i in range(700)]]  # more than run at a time: CTAs of two warps


@pytest.mark.parametrize("heads,kv,dim,rows,cache", SHAPES, ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda v: f"{len(v)}-" + "-".join(map(str, v[:7])))
def test_attention_over_lengths(lib, heads, kv, dim, rows, cache, lengths):
    import trismoe_b200 as tm

    g = _gen(heads * dim + len(lengths))
    scales = [None, None]
    if cache == E4M3:
        scales = [0.5 + torch.rand((kv,), generator=g, device="cuda") for _ in range(2)]
    page = {1: 16, 4: 32, 5: 8, 7: 48, 100: 16, 700: 16}[len(lengths)]
    filled = _filled(g, lengths, page, kv, dim, cache, LAYOUTS[heads % 3])
    q = (torch.randn((len(lengths), heads, dim), generator=g, device="cuda") * 2.0).to(rows)
    _check_attention(tm, q, filled, lengths, k_scale=scales[0], v_scale=scales[1])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("page", [1, 3, 16, 128])
def test_attention_over_pages_and_layouts(lib, page, layout):
    import trismoe_b200 as tm

    g, lengths = _gen(page), [257, 0, 5, 128]
    filled = _filled(g, lengths, page, 2, 64, BF16, layout)
    wide = torch.randn((4, 11, 64), generator=g, device="cuda").to(BF16)
    _check_attention(tm, wide[:, 1:9], filled, lengths)                                    # heads inside wider rows
    _check_attention(tm, wide[:, 1:9].transpose(0, 1).contiguous().transpose(0, 1), filled, lengths)  # heads outside
    flat = torch.zeros(4 * 8 * 64 + 1, dtype=BF16, device="cuda")[1:].view(4, 8, 64)
    flat.copy_(wide[:, 1:9])
    _check_attention(tm, flat, filled, lengths)                                            # rows off any 16-byte boundary


@pytest.mark.parametrize("window", [1, 16, 100, 255, 5000])
def test_attention_in_a_window(lib, window):
    import trismoe_b200 as tm

    g, lengths = _gen(window), [1, 0, 99, 100, 101, 700, 17]
    q = torch.randn((7, 8, 128), generator=g, device="cuda").half()
    _check_attention(tm, q, _filled(g, lengths, 16, 2, 128, F16, LAYOUTS[0]), lengths, window=window)


def test_attention_of_one_long_sequence_beside_short_ones(lib):
    import trismoe_b200 as tm

    g, lengths = _gen(7), [3, 70001, 0, 40]
    q = torch.randn((4, 4, 128), generator=g, device="cuda").half()
    _check_attention(tm, q * 3, _filled(g, lengths, 16, 1, 128, F16, LAYOUTS[0]), lengths, softmax_scale=0.05)


def test_attention_of_many_sequences(lib):
    import trismoe_b200 as tm

    g = _gen(8)
    lengths = [(37 * i) % 90 for i in range(300)]
    q = torch.randn((300, 2, 64), generator=g, device="cuda").to(BF16)
    _check_attention(tm, q, _filled(g, lengths, 16, 2, 64, BF16, LAYOUTS[1]), lengths)


def test_attention_where_one_score_outweighs_all(lib):
    """Scores of several hundred: the largest may come first, last or in between."""
    import trismoe_b200 as tm

    g, lengths = _gen(9), [400, 400, 400]
    k_pages, v_pages, table, rows = _filled(g, lengths, 16, 1, 64, F16, LAYOUTS[0])
    q = torch.randn((3, 8, 64), generator=g, device="cuda").half()
    for b, place in enumerate((0, 399, 200)):
        k_pages[table[b, place // 16].long(), place % 16, 0] = 40.0 * q[b, 0]
        rows[b][0][place, 0] = (40.0 * q[b, 0]).double()
    # the other heads see that key, too; scores go up to some 40 * 64 / 8, so a weight's error is that of exp: 320 * 2^-20
    out = tm.paged_decode_attention(q, k_pages, v_pages, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    want, _, mag = _attend_64(q, rows, 0, 0.125, None, None)
    assert float(((out.double() - want).abs() - (2.0 ** -11 + 2.0 ** -11) * mag - 2.0 ** -11 * want.abs()).max()) <= 0


@pytest.mark.parametrize("rows,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)], ids=lambda v: str(v).replace("torch.", ""))
def test_attention_of_small_weights_beside_a_large_one_on_nothing(lib, rows, cache):
    import trismoe_b200 as tm

    # the token that has almost all of the weight has values of zero: the result is made of weights from 2^-17 to 2^-19 of it
    g, lengths, page, dim = _gen(9), [2, 3, 40, 300], 16, 64
    k_pages, v_pages, table, kept = _filled(g, lengths, page, 2, dim, cache, LAYOUTS[0])
    for b, n in enumerate(lengths):
        k, v = kept[b]
        k[..., 0] = -torch.rand((n, 2), generator=g, device="cuda").to(cache).double()
        at = (5 * b) % n
        k[at, :, 0], v[at] = 12.0, 0.0
        place = torch.arange(n, device="cuda")
        page_of = table[b, place // page].long()
        k_pages[page_of, place % page], v_pages[page_of, place % page] = k.to(cache), v.to(cache)
    q = torch.zeros((4, 6, dim), dtype=rows, device="cuda")
    q[..., 0] = 1.0
    _check_attention(tm, q, (k_pages, v_pages, table, kept), lengths, softmax_scale=1.0)


@pytest.mark.parametrize("softmax_scale", [-0.2, 0.0, 3.0])
def test_attention_with_any_scale(lib, softmax_scale):
    import trismoe_b200 as tm

    g, lengths = _gen(14), [1, 20, 333]
    q = torch.randn((3, 4, 64), generator=g, device="cuda").half()
    filled = _filled(g, lengths, 16, 2, 64, F16, LAYOUTS[0], scale=0.5)
    _check_attention(tm, q, filled, lengths, softmax_scale=softmax_scale)


def test_attention_of_queries_of_very_different_sizes(lib):
    """8-bit pages: rows around 10^-20 and 10^20 in bf16, zeros, and elements far apart in one row."""
    import trismoe_b200 as tm

    g, lengths = _gen(15), [50, 50, 50, 50]
    filled = _filled(g, lengths, 16, 1, 128, E4M3, LAYOUTS[0])
    q = torch.randn((4, 2, 128), generator=g, device="cuda")
    for b, size in enumerate((1e-20, 1e20, 0.0)):
        q[b] *= size
    q[3, :, ::2] *= 1e-6
    for b, size in enumerate((1e20, 1e-20, 1.0, 1.0)):  # one scale for the call: a row at a time
        one = lambda t: t[b: b + 1].contiguous()
        k_pages, v_pages, table, rows = filled
        _check_attention(tm, one(q.to(BF16)), (k_pages, v_pages, one(table), rows[b: b + 1]), [50], softmax_scale=size / 11.0)


def test_calls_on_nothing(lib):
    import trismoe_b200 as tm

    new = lambda *s, dtype=F16: torch.zeros(s, dtype=dtype, device="cuda")
    pages, i32 = new(4, 16, 2, 64), torch.int32
    assert tm.paged_decode_attention(new(0, 4, 64), pages, pages, new(0, 3, dtype=i32), new(0, dtype=i32)).shape == (0, 4, 64)
    out, lse = tm.paged_decode_attention(torch.ones_like(new(2, 4, 64)), pages, pages, new(2, 0, dtype=i32), new(2, dtype=i32), return_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())
    assert tm.append_paged_kv(new(0, 4, 64), new(0, 2, 64), new(0, 2, 64), pages, pages, new(1, 4, dtype=i32), new(0, dtype=i32)).shape == (0, 4, 64)
    assert tm.apply_logit_controls(new(0, 100)).shape == (0, 100) and tm.apply_logit_controls(new(3, 0)).shape == (3, 0)
    x = torch.randn((2, 40), device="cuda")
    empty = tm.apply_logit_controls(x, tokens=new(2, 0, dtype=i32), token_lengths=new(2, dtype=i32), repetition=new(2, dtype=torch.float32) + 2.0,
                                    bias_ids=new(2, 0, dtype=i32), bias_values=new(2, 0, dtype=torch.float32))
    assert torch.equal(empty, x)


def test_arguments_that_the_python_layer_refuses(lib):
    import trismoe_b200 as tm

    new = lambda *s, dtype=F16: torch.zeros(s, dtype=dtype, device="cuda")
    pages, i32 = new(4, 16, 2, 64), torch.int32
    table, lens, pos, q, k = new(2, 3, dtype=i32), new(2, dtype=i32), new(2, dtype=i32), new(2, 4, 64), new(2, 2, 64)
    attend = lambda q=q, k=pages, v=pages, t=table, n=lens, **m: tm.paged_decode_attention(q, k, v, t, n, **m)
    append = lambda q=q, k=k, v=k, kp=pages, vp=pages, t=table, p=pos, s=None, **m: tm.append_paged_kv(q, k, v, kp, vp, t, p, s, **m)
    f32 = lambda *s: new(*s, dtype=torch.float32)
    logits = f32(2, 40)
    for call, text in [
        (lambda: attend(q=new(2, 3, 64)), "share"), (lambda: attend(q=new(2, 4, 32)), "head_dim"), (lambda: attend(q=q.float()), "fp16 or bf16"),
        (lambda: attend(q=q.bfloat16()), "queries' type"), (lambda: attend(k=pages.bfloat16()), "same type"), (lambda: attend(t=table.long()), "int32"),
        (lambda: attend(t=table[:1]), "sequences"), (lambda: attend(n=lens.long()), "lengths"), (lambda: attend(window=-1), "window"),
        (lambda: attend(k_scale=f32(2)), "e4m3"), (lambda: attend(k=pages[..., ::2], v=pages[..., ::2], q=new(2, 4, 32)), "side by side"),
        (lambda: attend(status=lens), "status"), (lambda: attend(n=lens.cpu()), "one CUDA device"),
        (lambda: append(k=new(2, 1, 64)), "num_kv_heads"), (lambda: append(q=new(3, 4, 64)), "q must be"), (lambda: append(p=pos.float()), "positions"),
        (lambda: append(s=pos.long()), "sequences"), (lambda: append(cos=f32(9, 32)), "go together"), (lambda: append(cos=f32(9, 64), sin=f32(9, 64)), "rotary_dim"),
        (lambda: append(cos=f32(9, 32), sin=f32(8, 32)), "sin"), (lambda: append(k_scale=f32(2)), "e4m3"),
        (lambda: tm.add_rms_norm(new(2, 64), new(2, 32), new(64)), "residual"), (lambda: tm.add_rms_norm(new(2, 64), None, new(32)), "weight"),
        (lambda: tm.add_rms_norm(f32(2, 64), None, f32(64)), "fp16 or bf16"), (lambda: tm.add_rms_norm_e4m3(new(2, 64), None, new(64), group_size=24), "divide"),
        (lambda: tm.add_rms_norm_e4m3(new(2, 64), None, new(64), group_size=8), "multiples of 16"),
        (lambda: tm.apply_logit_controls(logits, repetition=f32(2)), "need tokens"), (lambda: tm.apply_logit_controls(logits, tokens=new(2, 5, dtype=i32)), "token_lengths"),
        (lambda: tm.apply_logit_controls(logits, bias_ids=new(2, 5, dtype=i32)), "go together"), (lambda: tm.apply_logit_controls(logits, allowed=new(2, 1, dtype=i32)), "allowed"),
        (lambda: tm.apply_logit_controls(logits, out=new(2, 40)), "out must be"), (lambda: tm.apply_logit_controls(logits.double()), "fp16, bf16 or fp32"),
    ]:
        with pytest.raises(RuntimeError, match=text):
            call()


def test_a_refused_call_does_not_spoil_the_next(lib):
    """Long caches need scratch; what a refused call of the same sizes needed is not remembered."""
    import trismoe_b200 as tm

    g, lengths = _gen(16), [20000]
    k_pages, v_pages, table, rows = _filled(g, lengths, 16, 1, 40, F16, LAYOUTS[1])
    q = torch.randn((1, 1, 40), generator=g, device="cuda").half()
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    flat = torch.zeros((k_pages.numel() + 1,), dtype=F16, device="cuda")
    off = flat[1:].view(k_pages.shape)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="16-byte boundary"):
            tm.paged_decode_attention(q, off, off, table, lens)
    _check_attention(tm, q, (k_pages, v_pages, table, rows), lengths)


def test_attention_offsets_beyond_32_bits(lib):
    import trismoe_b200 as tm

    g, page, dim, stride = _gen(10), 16, 64, 1_100_000_000  # elements: page 2 begins behind 4 GB
    store = torch.empty((2 * stride + 2 * page * dim,), dtype=F16, device="cuda")
    k_pages = store.as_strided((3, page, 1, dim), (stride, dim, page * dim, 1))
    v_pages = store.as_strided((3, page, 1, dim), (stride, dim, page * dim, 1), page * dim)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    k, v = (torch.randn((48, 1, dim), generator=g, device="cuda").half() for _ in range(2))
    q = torch.randn((48, 2, dim), generator=g, device="cuda").half()
    tm.append_paged_kv(q, k, v, k_pages, v_pages, table, torch.arange(48, device="cuda"), torch.zeros((48,), dtype=torch.int32, device="cuda"))
    assert torch.equal(k_pages[2, :, 0], k[:16, 0]) and torch.equal(v_pages[1, :, 0], v[32:, 0])
    _check_attention(tm, q[:1], (k_pages, v_pages, table, [(k.double(), v.double())]), [48])


@pytest.mark.parametrize("dtype", [F16, E4M3], ids=["fp16", "e4m3"])
def test_attention_in_a_page_of_more_than_4_gb(lib, dtype):
    """One page a sequence, 9 (18) million tokens of 512 (256) bytes; only the window at its end is ever written or read."""
    import trismoe_b200 as tm

    g, tokens, window = _gen(17), 9_000_000 if dtype == F16 else 18_000_000, 100
    pages = [torch.empty((1, 1, tokens, 256), dtype=dtype, device="cuda").transpose(1, 2) for _ in range(2)]
    k, v = (torch.randn((window, 1, 256), generator=g, device="cuda") for _ in range(2))
    table = torch.zeros((1, 1), dtype=torch.int32, device="cuda")
    where = torch.arange(tokens - window, tokens, device="cuda")
    q = tm.append_paged_kv(torch.randn((window, 2, 256), generator=g, device="cuda").half(), k.half(), v.half(), pages[0], pages[1], table, where,
                           torch.zeros((window,), dtype=torch.int32, device="cuda"))
    held = [(p[0, where].double()) for p in pages]
    assert torch.equal(held[1], v.half().to(dtype).double())
    _check_attention(tm, q[:1].contiguous(), (pages[0], pages[1], table, [tuple(held)]), [tokens], window=window)


def test_attention_reports_what_does_not_fit(lib):
    import trismoe_b200 as tm

    g = _gen(11)
    k_pages, v_pages, table, rows = _filled(g, [40, 20], 16, 1, 64, F16, LAYOUTS[0])
    q = torch.randn((2, 2, 64), generator=g, device="cuda").half()
    lens = torch.tensor([40, 20], dtype=torch.int32, device="cuda")
    good = tm.paged_decode_attention(q, k_pages, v_pages, table, lens)
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    for page in (-1, k_pages.shape[0], 2 ** 31 - 1):
        broken = table.clone()
        broken[0, 1] = page
        status.zero_()
        out = tm.paged_decode_attention(q, k_pages, v_pages, broken, lens, status=status)
        with pytest.raises(RuntimeError, match="CORRUPT"):
            tm.raise_on_status(status)
        assert torch.equal(out[1], good[1]) and bool(torch.isfinite(out).all())
    # a length beyond the table is cut off; the table's own places are read
    full = table[:, :3].contiguous()
    full[1] = full[0]
    for length in (49, 2 ** 31 - 1):
        status.zero_()
        k_pages[full[0, 2].long(), 8:] = 0.5
        v_pages[full[0, 2].long(), 8:] = 0.5
        out = tm.paged_decode_attention(q, k_pages, v_pages, full, torch.tensor([length, 40], dtype=torch.int32, device="cuda"), status=status)
        with pytest.raises(RuntimeError, match="CORRUPT"):
            tm.raise_on_status(status)
        assert torch.equal(out[0], tm.paged_decode_attention(q, k_pages, v_pages, full, torch.tensor([48, 40], dtype=torch.int32, device="cuda"))[0])
    out = tm.paged_decode_attention(q, k_pages, v_pages, table, torch.tensor([-5, 20], dtype=torch.int32, device="cuda"))
    assert bool((out[0] == 0).all()) and torch.equal(out[1], good[1])


def test_attention_keeps_a_nan_and_an_infinity_of_its_own_tokens(lib):
    import trismoe_b200 as tm

    g = _gen(12)
    k_pages, v_pages, table, _ = _filled(g, [60, 60, 60], 16, 1, 64, F16, LAYOUTS[0])
    q = torch.randn((3, 1, 64), generator=g, device="cuda").half()
    lens = torch.tensor([60, 60, 60], dtype=torch.int32, device="cuda")
    v_pages[table[0, 3].long(), 4, 0, 3] = math.inf
    k_pages[table[1, 0].long(), 2, 0, 0] = math.nan
    out = tm.paged_decode_attention(q, k_pages, v_pages, table, lens)
    assert float(out[0, 0, 3]) == math.inf and bool(torch.isfinite(out[0, 0, 4:]).all())
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isfinite(out[2]).all())


def test_a_captured_step_follows_its_lengths_on_any_stream(lib):
    """Append and attention in a graph; positions and lengths advance between replays, and the work is cut anew each time."""
    import trismoe_b200 as tm

    g, lengths, page = _gen(13), [30, 0, 500], 16
    k_pages, v_pages, table, rows = _filled(g, [n + 40 for n in lengths], page, 2, 64, F16, LAYOUTS[0])
    cos = torch.rand((600, 32), generator=g, device="cuda")
    sin = torch.rand((600, 32), generator=g, device="cuda")
    qkv = torch.randn((3, 8, 64), generator=g, device="cuda").half()
    pos = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    lens = pos + 1

    def step():
        q = tm.append_paged_kv(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], k_pages, v_pages, table, pos, cos=cos, sin=sin)
        return tm.paged_decode_attention(q, k_pages, v_pages, table, lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    for _ in range(3):
        pos += 9
        lens += 9
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(step(), replayed)


# ---- append ---------------------------------------------------------------------------------
def _rotated_64(x, cos, sin, interleaved):
    x, rot = x.double().clone(), 2 * cos.shape[1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., : rot // 2], x[..., rot // 2: rot])
    c, s = cos.double()[:, None], sin.double()[:, None]
    out = x.clone()
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    return out


@pytest.mark.parametrize("heads,kv,dim,rot", [(16, 16, 128, 128), (16, 2, 256, 64), (4, 2, 64, 64), (5, 1, 80, 24), (3, 3, 48, 8), (0, 2, 64, 64), (8, 1, 192, 0), (2, 2, 16, 4)])
@pytest.mark.parametrize("rows,cache", [(F16, F16), (BF16, BF16), (F16, E4M3), (BF16, E4M3)], ids=lambda v: str(v).replace("torch.", ""))
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(lib, heads, kv, dim, rot, rows, cache, interleaved):
    import trismoe_b200 as tm

    g, page = _gen(dim + rot), 12
    new = [5, 0, 1, 30]                      # new tokens of four sequences, at places of their own
    begin = [0, 3, 11, 40]
    k_pages, v_pages, table, _ = _filled(g, [b + n for b, n in zip(begin, new)], page, kv, dim, cache, LAYOUTS[heads % 3])
    before = k_pages.clone(), v_pages.clone()
    seq = torch.repeat_interleave(torch.arange(4, device="cuda", dtype=torch.int32), torch.tensor(new, device="cuda"))
    pos = torch.cat([torch.arange(b, b + n, device="cuda") for b, n in zip(begin, new)])
    order = torch.randperm(len(pos), generator=g, device="cuda")
    seq, pos = seq[order], pos[order]
    pos[3] = -1                              # padding
    tokens = len(pos)
    # rows wider than they need be: 16-byte boundaries, and none
    for extra in (0, 1):
        k_pages.copy_(before[0])
        v_pages.copy_(before[1])
        width = (heads + 2 * kv) * dim
        flat = torch.randn((tokens, width + extra), generator=g, device="cuda").to(rows)
        view = flat[:, extra:].unflatten(1, (heads + 2 * kv, dim))
        q, k, v = view[:, :heads], view[:, heads: heads + kv], view[:, heads + kv:]
        cos = sin = None
        if rot:
            angle = torch.rand((80, rot // 2), generator=g, device="cuda") * 6.0
            cos, sin = angle.cos(), angle.sin()
        scales = [0.01 + 0.01 * torch.rand((kv,), generator=g, device="cuda") for _ in range(2)] if cache == E4M3 else [None, None]
        status = torch.zeros((1,), dtype=torch.int32, device="cuda")
        got_q, got_k = tm.append_paged_kv(q if heads else None, k, v, k_pages, v_pages, table, pos if extra else pos.int(), seq, cos=cos, sin=sin,
                                          interleaved=interleaved, k_scale=scales[0], v_scale=scales[1], return_key=True, status=status)
        tm.raise_on_status(status)
        real = pos >= 0
        at = pos.clamp(min=0)
        turn = (lambda x: _rotated_64(x, cos[at], sin[at], interleaved)) if rot else (lambda x: x.double())
        for got, x in ((got_q, q), (got_k, k)):
            if got is None:
                assert heads == 0
                continue
            want = turn(x)
            bound = U[rows] * want.abs() + SUB[rows] + 2.0 ** -20
            assert bool((got[~real] == 0).all())
            assert float(((got.double() - want).abs() - bound)[real].max()) <= 0
        touched = torch.zeros(k_pages.shape[:2], dtype=torch.bool, device="cuda")
        place = table[seq.long(), at // page].long(), at % page
        touched[place[0][real], place[1][real]] = True
        for pages, old, x, scale in ((k_pages, before[0], turn(k), scales[0]), (v_pages, before[1], v.double(), scales[1])):
            assert torch.equal(pages[~touched].view(torch.uint8), old[~touched].view(torch.uint8))
            held = pages[place][real].double()
            want = x[real]
            if scale is not None:
                want = (want / scale.double()[:, None]).clamp(-448.0, 448.0)
            bound = U[cache] * 1.0001 * want.abs() + SUB[cache] + (2.0 ** -20 if cache != E4M3 else 2.0 ** -13)
            assert float(((held - want).abs() - bound).max()) <= 0
        if cache != E4M3:
            assert torch.equal(v_pages[place][real], v[real])


def test_append_of_a_long_prompt_equals_its_pieces(lib):
    import trismoe_b200 as tm

    g, T = _gen(20), 5000
    cos, sin = torch.rand((T, 64), generator=g, device="cuda"), torch.rand((T, 64), generator=g, device="cuda")
    qkv = torch.randn((T, 12, 128), generator=g, device="cuda").half()
    table = torch.randperm(400, generator=g, device="cuda").to(torch.int32).view(1, 400)
    whole = [torch.zeros((400, 2, 16, 128), dtype=F16, device="cuda").transpose(1, 2) for _ in range(2)]
    parts = [torch.zeros_like(p) for p in whole]
    pos, seq = torch.arange(T, device="cuda"), torch.zeros((T,), dtype=torch.int32, device="cuda")
    call = lambda s, e, p: tm.append_paged_kv(qkv[s:e, :8], qkv[s:e, 8:10], qkv[s:e, 10:], *p, table, pos[s:e], seq[s:e], cos=cos, sin=sin)
    all_q = call(0, T, whole)
    pieces = [call(s, min(T, s + 7 + s), parts) for s in (0, 7, 21, 49, 105, 217, 441, 889, 1785, 3577)]
    assert torch.equal(torch.cat(pieces), all_q) and all(torch.equal(a, b) for a, b in zip(whole, parts))


def test_append_reports_what_does_not_fit(lib):
    import trismoe_b200 as tm

    g = _gen(21)
    k_pages, v_pages, table, _ = _filled(g, [40, 20], 16, 1, 64, F16, LAYOUTS[0])
    before = k_pages.clone()
    cos = sin = torch.ones((48, 32), device="cuda")
    x = torch.randn((1, 1, 64), generator=g, device="cuda").half()
    call = lambda pos, seq=0, t=table, **more: tm.append_paged_kv(
        x, x, x, k_pages, v_pages, t, torch.tensor([pos], device="cuda"), torch.tensor([seq], dtype=torch.int32, device="cuda"), status=status, **more)
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    bad = table.clone()
    bad[0, 0] = k_pages.shape[0]
    for args in ((2 ** 40,), (table.shape[1] * 16,), (0, 2), (0, -1), (3, 0, bad), (16 * 3, 0), (16 * 1, 1, torch.full_like(table, -1))):
        status.zero_()
        call(*args)
        with pytest.raises(RuntimeError, match="CORRUPT"):
            tm.raise_on_status(status)
    status.zero_()
    call(48, cos=cos[:20], sin=sin[:20])     # beyond the rotation's rows
    with pytest.raises(RuntimeError, match="CORRUPT"):
        tm.raise_on_status(status)
    assert torch.equal(k_pages.view(torch.int16), before.view(torch.int16))


# ---- norm -----------------------------------------------------------------------------------
@pytest.mark.parametrize("hidden", [1, 7, 16, 33, 256, 1000, 2048, 4096, 5120, 8192, 33000, 40000])
@pytest.mark.parametrize("rows", [1, 3, 300])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_norm(lib, hidden, rows, dtype):
    import trismoe_b200 as tm

    g = _gen(hidden + rows)
    x = torch.randn((rows, hidden), generator=g, device="cuda").to(dtype)
    res = (3.0 * torch.randn((rows, hidden), generator=g, device="cuda")).to(dtype)
    w = (1.0 + 0.2 * torch.randn((hidden,), generator=g, device="cuda")).to(dtype)
    for residual in (res, None):
        h64 = x.double() + (0.0 if residual is None else residual.double())
        want = h64 / (h64.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
        y, h = tm.add_rms_norm(x, residual, w, 1e-5)
        assert float(((y.double() - want).abs() - (U[dtype] + 2.0 ** -17) * want.abs() - SUB[dtype]).max()) <= 0
        if residual is None:
            assert h is None
        else:
            assert torch.equal(h, h64.to(dtype))  # a sum of two 16-bit numbers is exact in 32 bits or rounded far below
        for group in [0] + [n for n in (16, 48, 128, 200, 1024) if hidden % n == 0 and n % 16 == 0 and n < hidden]:
            values, scales, h8 = tm.add_rms_norm_e4m3(x, residual, w, 1e-5, group_size=group)
            parts = want.view(rows, -1, group or hidden)
            want_scale = parts.abs().amax(-1) / 448.0
            assert scales.shape == want_scale.shape and float(((scales.double() - want_scale).abs() - 2.0 ** -16 * want_scale).max()) <= 0
            back = values.double().view(parts.shape) * scales.double()[..., None]
            assert float(((back - parts).abs() - (U[E4M3] + 2.0 ** -15) * parts.abs() - 1.01 * SUB[E4M3] * want_scale[..., None]).max()) <= 0
            assert (h8 is None) == (residual is None) and (h8 is None or torch.equal(h8, h))


def test_norm_of_views_zeros_and_what_is_not_finite(lib):
    import trismoe_b200 as tm

    g = _gen(30)
    base = torch.randn((6, 3, 520), generator=g, device="cuda").half()
    w = torch.ones((256,), dtype=F16, device="cuda")
    plain = lambda t: tm.add_rms_norm(t.contiguous(), None, w)[0]
    assert torch.equal(tm.add_rms_norm(base[:, 1, 8:264], None, w)[0], plain(base[:, 1, 8:264]))     # rows further apart
    assert torch.equal(tm.add_rms_norm(base[:, :, 1:257], None, w)[0], plain(base[:, :, 1:257]))     # three dimensions, no alignment
    skew = base[:, 0, 1:257]
    assert float((tm.add_rms_norm(skew, skew, w)[0].float() - plain(2 * skew.contiguous()).float()).abs().max()) <= 2.0 ** -8
    x = torch.zeros((4, 256), dtype=F16, device="cuda")
    x[1, 3], x[2, 5], x[3, 7] = math.nan, math.inf, 1.0
    y, _ = tm.add_rms_norm(x, None, w)
    assert bool((y[0] == 0).all()) and bool(torch.isnan(y[1]).all()) and bool(torch.isnan(y[2, 5])) and bool((y[2, :5] == 0).all())
    values, scales, _ = tm.add_rms_norm_e4m3(x, None, w, group_size=16)
    assert bool((scales[0] == 0).all()) and bool((values[0].float() == 0).all())
    assert bool(torch.isnan(scales[1]).all()) and bool(torch.isnan(values[1].float()).all())
    assert bool(torch.isnan(scales[2, 0])) and float(values[3].float()[7]) == 448.0
    assert tm.add_rms_norm(x[:0], x[:0], w)[0].shape == (0, 256)


# ---- logits ---------------------------------------------------------------------------------
def _controls_64(logits, c):
    z, rows, vocab = logits.double(), *logits.shape
    mag = z.abs().clone()
    for b in range(rows):
        n = min(max(int(c["token_lengths"][b]), 0), c["tokens"].shape[1]) if "tokens" in c else 0
        begin = int(c["prompt_lengths"][b]) if "prompt_lengths" in c else 0
        if n:
            tok = c["tokens"][b, :n].long()
            ok = (tok >= 0) & (tok < vocab)
            place = torch.arange(n, device="cuda")
            seen = torch.zeros(vocab, dtype=torch.float64, device="cuda").index_add_(0, tok[ok], torch.ones(int(ok.sum()), dtype=torch.float64, device="cuda"))
            mine = ok & (place >= begin)
            count = torch.zeros_like(seen).index_add_(0, tok[mine], torch.ones(int(mine.sum()), dtype=torch.float64, device="cuda"))
            if "repetition" in c:
                r = c["repetition"][b].double()
                z[b] = torch.where(seen > 0, torch.where(z[b] > 0, z[b] / r, z[b] * r), z[b])
            for name, times in (("frequency", count), ("presence", (count > 0).double())):
                if name in c:
                    z[b] -= c[name][b].double() * times
                    mag[b] += c[name][b].double().abs() * times
        if "bias_ids" in c:
            ids = c["bias_ids"][b].long()
            ok = (ids >= 0) & (ids < vocab)
            z[b].index_add_(0, ids[ok], c["bias_values"][b][ok].double())
            mag[b].index_add_(0, ids[ok], c["bias_values"][b][ok].double().abs())
        if "allowed" in c:
            v = torch.arange(vocab, device="cuda")
            z[b][(c["allowed"][b].long()[v // 32] >> (v % 32)) & 1 == 0] = -math.inf
    return z, mag


@pytest.mark.parametrize("rows,vocab,history", [(1, 50304, 700), (3, 1, 5), (5, 31, 40), (2, 1000, 0), (7, 32000, 3001), (130, 513, 64), (1, 131073, 9000), (2, 4000, 40000)])
@pytest.mark.parametrize("dtype", [F16, BF16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("names", ["", "repetition", "presence frequency", "bias", "allowed", "repetition presence frequency bias allowed prompt"])
def test_logit_controls(lib, rows, vocab, history, dtype, names):
    import trismoe_b200 as tm

    g = _gen(rows + vocab)
    rand = lambda *s: torch.rand(s, generator=g, device="cuda")
    logits = (torch.randn((rows, vocab + 3), generator=g, device="cuda") * 5.0).to(dtype)[:, 1: vocab + 1]
    logits[0, 0], logits[-1, -1] = math.inf, -math.inf
    c = {}
    if any(n in names for n in ("repetition", "presence")):
        c["tokens"] = torch.randint(-2, vocab + 2, (rows, history), generator=g, device="cuda", dtype=torch.int32)
        c["tokens"][:, : history // 2] %= max(1, vocab // 50)
        c["token_lengths"] = torch.randint(-1, history + 5, (rows,), generator=g, device="cuda", dtype=torch.int32)
        if "prompt" in names:
            c["prompt_lengths"] = torch.randint(0, history + 2, (rows,), generator=g, device="cuda", dtype=torch.int32)
        for name in ("repetition", "presence", "frequency"):
            if name in names:
                c[name] = 0.5 + rand(rows)
    if "bias" in names:
        c["bias_ids"] = torch.randint(-2, vocab + 1, (rows, 37), generator=g, device="cuda", dtype=torch.int32)
        c["bias_ids"][:, 20:] = c["bias_ids"][:, :17]  # some twice
        c["bias_values"] = torch.randn((rows, 37), generator=g, device="cuda")
    if "allowed" in names:
        c["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        c["allowed"][0] = 0  # a row that nothing is left of
    for aligned in (False, True):
        src = logits.contiguous() if aligned else logits
        want, mag = _controls_64(src, c)
        got = tm.apply_logit_controls(src, **c)
        assert got.dtype == torch.float32 and got.shape == src.shape
        finite = torch.isfinite(want)
        assert torch.equal(got[~finite].double(), want[~finite])
        # each of some ten roundings is at most 2^-24 of the magnitudes added up
        assert float(((got.double() - want).abs() - 12 * 2.0 ** -24 * mag)[finite].max() if bool(finite.any()) else 0.0) <= 0
        if dtype == torch.float32:
            same = src.clone()
            assert torch.equal(tm.apply_logit_controls(same, out=same, **c), got) and bool((got == same).all())


def test_masked_logits_that_are_not_numbers(lib):
    import trismoe_b200 as tm

    logits = torch.full((2, 64), math.nan, device="cuda")
    logits[1] = torch.finfo(torch.float32).min
    allowed = torch.tensor([[0, 1 << 5], [0, -1]], dtype=torch.int32, device="cuda")
    out = tm.apply_logit_controls(logits, allowed=allowed)
    assert bool((out[0, :37] == -math.inf).all()) and bool(torch.isnan(out[0, 37])) and bool((out[0, 38:] == -math.inf).all())
    assert bool((out[1, :32] == -math.inf).all()) and bool((out[1, 32:] == torch.finfo(torch.float32).min).all())
