"""GPU tests of products in 8 bits and of the quantisation that feeds them, against definitions in 64 bits.

Tolerances.  u is half a step of the type, relative (fp16 2^-11, bf16 2^-8, fp32 2^-24, e4m3 2^-4).  Products: those of e4m3 numbers are exact in 32 bits; a group's
128 of them are added in 32 bits in an order of the hardware's, each addition off by a step (2^-23) of a partial sum at most, and the groups' sums once more with a
product by the scales: below (K + 3 groups + 2) 2^-23 of the sum of magnitudes, then u of the result.  Quantisation: scale and quotient are correctly rounded
32-bit quotients, a value is the nearest e4m3 number: half a step of it, which is u of the value or 2^-10 among the smallest, and 2^-23 of the quotient."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32, E4M3 = torch.float16, torch.bfloat16, torch.float32, torch.float8_e4m3fn
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8, F32: 2.0 ** -24}
SUB = {F16: 2.0 ** -25, BF16: 0.0, F32: 0.0}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _operands(rows, outputs, inputs, seed=0, line=None):
    """x and weight as parts of wider matrices, with NaN beside them."""
    g = _gen(seed + rows + outputs + inputs)
    line = line or (inputs + 15) // 16 * 16

    def coded(n):
        wide = torch.full((n, line), math.nan, device="cuda").to(E4M3)
        wide[:, :inputs] = (torch.randn((n, inputs), generator=g, device="cuda") * 120).clamp(-448, 448).to(E4M3)
        return wide[:, :inputs]

    groups = -(-inputs // 128)
    scales = lambda n: torch.exp2(8 * torch.rand((n, groups), generator=g, device="cuda") - 12)
    return coded(rows), scales(rows), coded(outputs), scales(-(-outputs // 128))


def _product_64(x, xs, w, ws, bias=None):
    """The product, and the sum of its terms' magnitudes."""
    inputs, outputs = x.shape[1], w.shape[0]
    a = x.double() * xs.double().repeat_interleave(128, 1)[:, :inputs]
    b = w.double() * ws.double().repeat_interleave(128, 0)[:outputs].repeat_interleave(128, 1)[:, :inputs]
    y, mag = a @ b.T, a.abs() @ b.abs().T
    return (y, mag) if bias is None else (y + bias.double(), mag + bias.double().abs())


def _close(got, want, mag, inputs):
    groups = -(-inputs // 128)
    limit = (inputs + 3 * groups + 2) * 2.0 ** -23 * mag + U[got.dtype] * want.abs() + SUB[got.dtype]
    error = (got.double() - want).abs()
    assert bool((error <= limit).all()), float((error / limit).max())


SHAPES = [(1, 1, 1), (1, 128, 128), (1, 6144, 2048), (2, 129, 127), (16, 300, 2048), (17, 257, 129), (32, 96, 400), (33, 1000, 1000), (64, 32, 4096), (65, 65, 65),
          (127, 500, 640), (128, 128, 8192), (129, 513, 384), (200, 4096, 256), (256, 255, 1), (257, 1, 300), (509, 640, 2048), (513, 2000, 144), (1000, 333, 1500)]


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=str)
@pytest.mark.parametrize("rows,outputs,inputs", SHAPES)
def test_product(lib, rows, outputs, inputs, dtype):
    import trismoe_b200 as tm

    x, xs, w, ws = _operands(rows, outputs, inputs)
    y = tm.linear_e4m3(x, xs, w, ws, dtype=dtype)
    assert y.shape == (rows, outputs) and y.dtype == dtype and y.is_contiguous()
    _close(y, *_product_64(x, xs, w, ws), inputs)


@pytest.mark.parametrize("bias", [F16, BF16, F32], ids=str)
@pytest.mark.parametrize("rows,outputs,inputs", [(1, 300, 256), (1, 6144, 2048), (40, 130, 500), (100, 264, 300), (300, 520, 256), (300, 521, 256)])
def test_bias_and_leading_dimensions(lib, rows, outputs, inputs, bias):
    import trismoe_b200 as tm

    x, xs, w, ws = _operands(rows, outputs, inputs, seed=3)
    b = (torch.randn((outputs,), generator=_gen(5), device="cuda") * 30).to(bias)
    y = tm.linear_e4m3(x.view(1, rows, inputs) if x.is_contiguous() else x[None], xs[None], w, ws, b, dtype=F32)
    assert y.shape == (1, rows, outputs)
    _close(y[0], *_product_64(x, xs, w, ws, b), inputs)


@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=str)
@pytest.mark.parametrize("rows,outputs,inputs", [(5, 40, 9000), (17, 5, 1030), (33, 140, 16384), (64, 513, 14336), (65, 130, 4096), (100, 257, 5000), (128, 1, 4224), (129, 300, 14336), (200, 129, 8300)])
def test_products_cut_among_blocks(lib, rows, outputs, inputs, dtype):
    """Few tiles and many groups: a cluster's blocks have some groups each and join a share of the columns, some of which do not exist."""
    import trismoe_b200 as tm

    x, xs, w, ws = _operands(rows, outputs, inputs, seed=21)
    b = torch.randn((outputs,), generator=_gen(22), device="cuda") * 100
    y = tm.linear_e4m3(x, xs, w, ws, b, dtype=dtype)
    _close(y, *_product_64(x, xs, w, ws, b), inputs)
    for _ in range(3):
        assert torch.equal(tm.linear_e4m3(x, xs, w, ws, b, dtype=dtype).view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("rows", [3, 90, 400])
def test_rows_and_scales_that_are_parts_of_larger_ones(lib, rows):
    """Any stride: rows 16 bytes apart from one another's ends, scales that start anywhere."""
    import trismoe_b200 as tm

    x, xs, w, ws = _operands(rows, 384, 640, seed=7, line=656)
    wide_x, wide_w = torch.full((rows, 9), math.nan, device="cuda"), torch.full((3, 11), math.nan, device="cuda")
    wide_x[:, 1:6], wide_w[:, 3:8] = xs, ws
    y = tm.linear_e4m3(x, wide_x[:, 1:6], w, wide_w[:, 3:8], dtype=F32)
    _close(y, *_product_64(x, xs, w, ws), 640)
    every = torch.arange(0, rows, 2, device="cuda")
    y2 = tm.linear_e4m3(x[::2], xs[::2], w, ws, dtype=F32)
    _close(y2, *_product_64(x[every], xs[every], w, ws), 640)


@pytest.mark.parametrize("rows", [1, 20, 64, 100, 300])
def test_one_rows_nan_is_its_own(lib, rows):
    import trismoe_b200 as tm

    x, xs, w, ws = _operands(rows, 256, 512, seed=9)
    want, mag = _product_64(x, xs, w, ws)
    x = x.clone()
    x[rows // 2, 200] = math.nan
    y = tm.linear_e4m3(x, xs, w, ws, dtype=F32)
    assert bool(y[rows // 2].isnan().all())
    keep = torch.arange(rows, device="cuda") != rows // 2
    _close(y[keep], want[keep], mag[keep], 512)


@pytest.mark.parametrize("rows", [1, 64, 128, 500])
def test_the_same_bits_on_every_run_and_stream(lib, rows):
    import trismoe_b200 as tm

    x, xs, w, ws = _operands(rows, 1000, 2000, seed=11)
    first = tm.linear_e4m3(x, xs, w, ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [tm.linear_e4m3(x, xs, w, ws) for _ in range(4)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, a) for a in again)


def test_captured_calls_follow_their_inputs(lib):
    import trismoe_b200 as tm

    a, b = (torch.randn((rows, 512), generator=_gen(rows), device="cuda").half() for rows in (5, 300))
    w, ws = tm.quantize_e4m3(torch.randn((384, 512), generator=_gen(1), device="cuda").half(), group_rows=128)
    step = lambda: [tm.linear_e4m3(*tm.quantize_e4m3(t), w, ws) for t in (a, b)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (2, 3):
        for t in (a, b):
            t.copy_(torch.randn(t.shape, generator=_gen(seed), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, step()))


def test_no_rows_and_no_features(lib):
    import trismoe_b200 as tm

    x, xs, w, ws = _operands(4, 64, 128)
    assert tm.linear_e4m3(x[:0], xs[:0], w, ws).shape == (0, 64)
    assert tm.linear_e4m3(x, xs, w[:0], ws[:0]).shape == (4, 0)
    for rows in (1, 128):
        values, scales = tm.quantize_e4m3(torch.empty((0, 300), dtype=F16, device="cuda"), group_rows=rows)
        assert values.shape == (0, 300) and scales.shape == (0, 3)


def test_no_call_gives_up_a_wait(lib):
    import trismoe_b200 as tm

    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    for rows in (1, 64, 128, 600):
        x, xs, w, ws = _operands(rows, 700, 1300)
        tm.linear_e4m3(x, xs, w, ws, status=status)
    tm.raise_on_status(status)


# ---------------------------------------------------------------------------------------
# quantisation
# ---------------------------------------------------------------------------------------
def _check_quantised(x, values, scales, group_rows):
    rows, columns = x.shape
    down, across = -(-rows // group_rows), -(-columns // 128)
    assert values.dtype == E4M3 and values.shape == x.shape and scales.dtype == F32 and scales.shape == (down, across)
    padded = torch.zeros((down * group_rows, across * 128), dtype=torch.float64, device="cuda")
    padded[:rows, :columns] = x.double()
    top = padded.view(down, group_rows, across, 128).abs().amax((1, 3))
    assert torch.equal(scales, (top / 448).float())
    each = scales.double().repeat_interleave(group_rows, 0)[:rows].repeat_interleave(128, 1)[:, :columns]
    q = torch.where(each > 0, x.double() / each.masked_fill(each == 0, 1), 0.0)
    step = torch.exp2(q.abs().clamp(min=2.0 ** -6).log2().floor() - 3)
    assert bool(((values.double() - q).abs() <= step / 2 + 2.0 ** -23 * q.abs()).all())


@pytest.mark.parametrize("group_rows", [1, 128])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 128), (3, 17), (64, 2048), (130, 1000), (257, 129), (4000, 4096)])
def test_quantisation(lib, rows, columns, dtype, group_rows):
    import trismoe_b200 as tm

    x = torch.randn((rows, columns), generator=_gen(rows + columns), device="cuda") * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=_gen(1), device="cuda").float())
    x[rows // 2] = 0.0
    x = x.to(dtype)
    values, scales = tm.quantize_e4m3(x, group_rows=group_rows)
    _check_quantised(x, values, scales, group_rows)
    assert rows == 1 or values.stride(0) % 16 == 0
    wide = torch.full((rows, columns + 5), math.nan, device="cuda").to(dtype)
    wide[:, 3: columns + 3] = x
    again = tm.quantize_e4m3(wide[:, 3: columns + 3], group_rows=group_rows)  # neither aligned nor side by side
    assert torch.equal(again[0].float(), values.float()) and torch.equal(again[1], scales)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_quantisation_of_the_smallest_and_largest_numbers(lib, dtype):
    import trismoe_b200 as tm

    info = torch.finfo(dtype)
    x = torch.zeros((4, 256), dtype=dtype, device="cuda")
    x[0, 5], x[1, 200], x[2, 7], x[3, 130] = info.max, info.tiny, -info.max, info.smallest_normal
    values, scales = tm.quantize_e4m3(x)
    for row, column, sign in ((0, 5, 1), (1, 200, 1), (2, 7, -1), (3, 130, 1)):
        assert float(values[row, column]) == sign * 448.0
    top = x.double().abs().view(4, 2, 128).amax(2)
    assert bool(((scales.double() - top / 448).abs() <= top / 448 * 2.0 ** -24 + 2.0 ** -150).all())


@pytest.mark.parametrize("group_rows", [1, 128])
def test_nan_and_infinity_concern_their_group_alone(lib, group_rows):
    import trismoe_b200 as tm

    x = torch.randn((256, 384), generator=_gen(2), device="cuda").half()
    clean = tm.quantize_e4m3(x, group_rows=group_rows)
    x[200, 300], x[3, 0] = math.nan, math.inf
    values, scales = tm.quantize_e4m3(x, group_rows=group_rows)
    down = lambda r: r // group_rows
    assert math.isnan(float(scales[down(200), 2])) and float(scales[down(3), 0]) == math.inf
    keep = torch.ones(scales.shape, dtype=torch.bool, device="cuda")
    keep[down(200), 2] = keep[down(3), 0] = False
    assert torch.equal(scales[keep], clean[1][keep])
    each = keep.repeat_interleave(group_rows, 0).repeat_interleave(128, 1)
    assert torch.equal(values.float()[each], clean[0].float()[each])


def test_norm_and_quantisation_agree_with_the_product_of_rows(lib):
    """The norm's 8-bit output and rows quantised behind a 16-bit norm are the same product but for the roundings between."""
    import trismoe_b200 as tm

    g = _gen(4)
    x, r, weight = ((torch.randn(s, generator=g, device="cuda")).half() for s in ((37, 512), (37, 512), (512,)))
    w, ws = tm.quantize_e4m3(torch.randn((384, 512), generator=g, device="cuda").half() / 16, group_rows=128)
    values, scales, h = tm.add_rms_norm_e4m3(x, r, weight, group_size=128)
    y = tm.linear_e4m3(values, scales, w, ws, dtype=F32)
    h64 = x.double() + r.double()
    exact = h64 / (h64.square().mean(1, keepdim=True) + 1e-5).sqrt() * weight.double()
    b = w.double() * ws.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    # values are within 2^-4 of themselves, or half of e4m3's smallest step of their group's scale, of the exact rows
    slack = (exact.abs() * 2.0 ** -4 + scales.double().repeat_interleave(128, 1) * 2.0 ** -9) @ b.abs().T
    assert bool(((y.double() - exact @ b.T).abs() <= slack + 2.0 ** -12 * (exact.abs() @ b.abs().T)).all())
