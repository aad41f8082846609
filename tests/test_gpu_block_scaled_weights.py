"""GPU tests of the softmax's weights in decode attention over block scales: values that cancel show what a weight is rounded to, which a result's own rounding hides otherwise.

Tolerance.  A query with one element has scores without sums: a product and two scales, each rounded in 32 bits, of magnitude 16 at most, lifted by a value scale's exponent of 8 at
most: an exponent of the weight is off by 2^-19 in all, in the numerator and in the sum.  Two 16-bit numbers hold a weight to 2^-21, sums of 40 terms and 2^x add as much: 2^-17 of the
sum of weight times magnitude.  One 16-bit number alone is off by up to 2^-12 of each weight."""
import pytest
import torch

from test_gpu_block_scaled_cache import BF16, E4M3, F16, U, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("kv,group,dim", [(4, 1, 128), (2, 4, 64), (1, 16, 128), (2, 8, 256)])
@pytest.mark.parametrize("n", [2, 5, 16, 40])
def test_values_that_cancel(lib, n, kv, group, dim, dtype):
    import trismoe_b200 as tm

    g = _gen(n + dim)
    batch = 6
    rand = lambda *s: torch.rand(s, generator=g, device="cuda")
    table = torch.randperm(batch * n, generator=g, device="cuda").to(torch.int32).view(batch, n)
    k_pages, v_pages = (torch.zeros((batch * n, kv, 1, dim), device="cuda").to(E4M3).transpose(1, 2) for _ in range(2))
    at, head = table.long(), torch.arange(kv, device="cuda")
    part = torch.randint(0, dim, (kv,), generator=g, device="cuda")  # the query's one element
    q = torch.zeros((batch, kv, group, dim), device="cuda")
    q[:, head, :, part] = 1.0
    key = ((rand(batch, n, kv) * 8 - 4).to(E4M3)).float()
    k = torch.randn((batch, n, kv, dim), generator=g, device="cuda").to(E4M3).float()
    k[:, :, head, part] = key
    k_scale = 0.5 + rand(batch, n, kv)
    value = ((rand(batch, n, kv) * 400 + 40).to(E4M3)).float() * torch.where(rand(batch, n, kv) < 0.5, -1.0, 1.0)
    v_scale = (0.5 + rand(batch, n, kv)) / 256
    w = torch.softmax(key.double() * k_scale.double(), 1)
    others = (w * value.double() * v_scale.double())[:, :-1].sum(1)
    value[:, -1] = -value[:, -1].abs() * others.sign().float()
    v_scale[:, -1] = (others.abs() / (w[:, -1] * value[:, -1].double().abs())).float()
    v_scale.clamp_(min=2.0 ** -20, max=1.0)  # (where that cuts, there is no cancellation; the tolerance holds all the same)
    sign = torch.where(rand(kv, dim) < 0.5, -1.0, 1.0)
    v = value[..., None] * sign
    scales = [torch.zeros((batch * n, 1, kv), device="cuda") for _ in range(2)]
    for pages, rows in ((k_pages, k), (v_pages, v)):
        pages[at, 0] = rows.to(E4M3)
    for held, s in zip(scales, (k_scale, v_scale)):
        held[at, 0] = s
    out = tm.paged_decode_attention(q.view(batch, kv * group, dim).to(dtype), k_pages, v_pages, table, torch.full((batch,), n, dtype=torch.int32, device="cuda"), softmax_scale=1.0,
                                    k_scale=scales[0], v_scale=scales[1])
    terms = w[..., None] * v.double() * v_scale.double()[..., None]
    want, size = terms.sum(1)[:, :, None], terms.abs().sum(1)[:, :, None]
    error = (out.view(batch, kv, group, dim).double() - want).abs()
    limit = 2.0 ** -17 * size + U[dtype] * want.abs() + 2.0 ** -25
    assert bool((error <= limit).all()), float((error / limit).max())
    assert float((want.abs() / size).median()) < 2.0 ** -17  # they do cancel
