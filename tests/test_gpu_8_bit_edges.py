"""GPU tests of what 8-bit decoding refuses, and of its largest tensors: offsets beyond 32 bits.  Tolerances as in the operators' own files."""
import math

import pytest
import torch

from test_gpu_block_scaled_cache import _check_attention, _half_step, _power
from test_gpu_e4m3_ops import _close, _product_64
from test_gpu_sample_tokens import _drawn_64

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def test_pages_beyond_four_gigabytes(lib):
    """The last pages of a cache of 4.6 GB for keys and as much for values."""
    import trismoe_b200 as tm

    pages, page, heads, dim, length = 70000, 16, 32, 128, 83
    new = lambda: torch.empty((pages, heads, page, dim), dtype=E4M3, device="cuda").transpose(1, 2)
    k_pages, v_pages = new(), new()
    k_scale, v_scale = (torch.full((pages, 1, heads), math.nan, device="cuda") for _ in range(2))
    table = torch.arange(pages - 1, pages - 7, -1, dtype=torch.int32, device="cuda")[None]
    k, v = (torch.randn((length, heads, dim), generator=_gen(i), device="cuda").half() for i in range(2))
    at = torch.arange(length, device="cuda")
    tm.append_paged_kv(None, k, v, k_pages, v_pages, table, at, torch.zeros((length,), dtype=torch.int32, device="cuda"), k_scale=k_scale, v_scale=v_scale)
    for rows, held, scales in ((k, k_pages, k_scale), (v, v_pages, v_scale)):
        for b in range(0, length, page):
            part = rows[b: b + page].double()
            scale = _power(part.abs().amax((0, 2)))
            assert torch.equal(scales[pages - 1 - b // page, 0].double(), scale)
            q = part / scale[:, None]
            assert bool(((held[pages - 1 - b // page, : part.shape[0]].double() - q).abs() <= _half_step(q) * (1 + 2.0 ** -10)).all())
    q = torch.randn((1, 64, dim), generator=_gen(3), device="cuda").half()
    _check_attention(tm, q, k_pages, v_pages, k_scale, v_scale, table, [length])


def test_logits_beyond_two_billion(lib):
    import trismoe_b200 as tm

    rows, vocab = 17000, 131072
    logits = torch.empty((rows, vocab), dtype=torch.float16, device="cuda")
    logits[:-3] = 0.0
    logits[-3:] = torch.randn((3, vocab), generator=_gen(1), device="cuda").half() * 3
    random = torch.full((rows,), 0.5, device="cuda")
    top_p = torch.full((rows,), 0.9, device="cuda")
    got = tm.sample_tokens(logits, random, top_p=top_p)
    assert torch.equal(got[-3:], _drawn_64(logits[-3:], random[-3:], top_p=top_p[-3:]))
    assert torch.equal(got[:1], _drawn_64(logits[:1], random[:1], top_p=top_p[:1])) and bool((got[:-3] == got[0]).all())


def test_rows_beyond_four_gigabytes(lib):
    """The last rows of 4.3 GB of values, their product with few features."""
    import trismoe_b200 as tm

    rows, inputs = 530000, 8192
    x = torch.empty((rows, inputs), dtype=E4M3, device="cuda")
    x[:-200] = 0.0
    part = torch.randn((200, inputs), generator=_gen(1), device="cuda").half()
    values, scales = tm.quantize_e4m3(part)
    x[-200:] = values
    xs = torch.zeros((rows, inputs // 128), device="cuda")
    xs[-200:] = scales
    w, ws = tm.quantize_e4m3(torch.randn((260, inputs), generator=_gen(2), device="cuda").half(), group_rows=128)
    y = tm.linear_e4m3(x, xs, w, ws, dtype=torch.float32)
    _close(y[-200:], *_product_64(values, scales, w, ws), inputs)  # (fewer rows are added up in another order)
    assert bool((y[:-200] == 0).all())


def _refuses(match, call):
    with pytest.raises(RuntimeError, match=match):
        call()


def test_refusals(lib):
    import trismoe_b200 as tm

    z = lambda *s, **more: torch.zeros(s, device="cuda", **more)
    e = lambda *s: z(*s).to(E4M3)
    x, xs, w, ws = e(4, 256), z(4, 2), e(300, 256), z(3, 2)
    tm.linear_e4m3(x, xs, w, ws)
    for match, call in [
            ("float8_e4m3fn", lambda: tm.linear_e4m3(z(4, 256).half(), xs, w, ws)), ("in_features", lambda: tm.linear_e4m3(e(4, 128), xs, w, ws)),
            ("x_scales", lambda: tm.linear_e4m3(x, z(4, 3), w, ws)), ("x_scales", lambda: tm.linear_e4m3(x, xs.double(), w, ws)), ("x_scales", lambda: tm.linear_e4m3(x[None], xs, w, ws)),
            ("weight_scales", lambda: tm.linear_e4m3(x, xs, w, z(2, 2))), ("weight must have a row", lambda: tm.linear_e4m3(x, xs, e(256, 300).T, ws)),
            ("bias", lambda: tm.linear_e4m3(x, xs, w, ws, z(299))), ("outputs are", lambda: tm.linear_e4m3(x, xs, w, ws, dtype=torch.float64)),
            ("16-byte", lambda: tm.linear_e4m3(e(4, 264)[:, 4: 260], xs, w, ws)), ("overlap", lambda: tm.linear_e4m3(x[:1].expand(4, 256), xs, w, ws)),
            ("one CUDA device", lambda: tm.linear_e4m3(x, xs.cpu(), w, ws)), ("status", lambda: tm.linear_e4m3(x, xs, w, ws, status=z(2, dtype=torch.int32))),
            ("gradient", lambda: tm.linear_e4m3(x, z(4, 2, requires_grad=True), w, ws)),
            ("fp16 or bf16", lambda: tm.quantize_e4m3(z(4, 256))), ("128", lambda: tm.quantize_e4m3(z(4, 256).half(), group_rows=64)),
            ("matrix", lambda: tm.quantize_e4m3(z(2, 4, 256).half(), group_rows=128)),
            ("logits", lambda: tm.sample_tokens(z(4, 9).double(), z(4))), ("random", lambda: tm.sample_tokens(z(4, 9), z(3))), ("side by side", lambda: tm.sample_tokens(z(9, 4).T, z(4))),
            ("top_k", lambda: tm.sample_tokens(z(4, 9), z(4), top_k=z(4))), ("temperature", lambda: tm.sample_tokens(z(4, 9), z(4), temperature=z(1))),
            ("no vocabulary", lambda: tm.sample_tokens(z(4, 0), z(4)))]:
        _refuses(match, call)
    pages, table = e(3, 16, 2, 64), torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    k, at, scale = z(1, 2, 64).half(), torch.zeros((1,), dtype=torch.int64, device="cuda"), z(3, 2, 2)
    append = lambda **more: tm.append_paged_kv(None, k, k, pages, pages, table, at, **more)
    attend = lambda **more: tm.paged_decode_attention(k, pages, pages, table, torch.ones((1,), dtype=torch.int32, device="cuda"), **more)
    for call in (append, attend):
        call(k_scale=scale, v_scale=scale.clone())
        for match, more in [("go together", dict(k_scale=scale)), ("cut evenly", dict(k_scale=z(3, 3, 2), v_scale=z(3, 3, 2))), ("cut evenly", dict(k_scale=z(3, 0, 2), v_scale=z(3, 0, 2))),
                            ("k_scale", dict(k_scale=z(2, 2, 2), v_scale=z(2, 2, 2))), ("v_scale", dict(k_scale=scale, v_scale=z(3, 1, 2))), ("v_scale", dict(k_scale=z(2), v_scale=scale)),
                            ("k_scale", dict(k_scale=z(3, 2, 2, dtype=torch.float16), v_scale=scale)), ("k_scale", dict(k_scale=z(3, 2, 4)[..., ::2], v_scale=scale))]:
            _refuses(match, lambda: call(**more))
    _refuses("e4m3 pages", lambda: tm.append_paged_kv(None, k, k, pages.half(), pages.half(), table, at, k_scale=scale, v_scale=scale))
