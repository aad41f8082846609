"""GPU tests of appends that go on inside partly filled blocks, with more tokens than a CTA's window: every block is brought to its new scale once, whichever CTA has its run.

Tolerances are those of test_gpu_block_scaled_cache: half a step of e4m3 for a token, half a step more for each time its block's scale has grown."""
import pytest
import torch

from test_gpu_block_scaled_cache import BF16, F16, Mirror, _cache, _gen, _rotated_64, _rotation, _runs, _table

pytestmark = pytest.mark.gpu

CALLS = {"8 x 5": [5] * 8, "60 x 3": [3] * 60, "60 x 5": [5] * 60, "tail and tokens": [17] + [1] * 47, "10, 7 and tokens": [10, 7] + [1] * 40, "odd": [5, 1, 16, 2, 15, 3, 17, 1, 31, 4] * 3}


@pytest.mark.parametrize("page,block", [(16, 16), (64, 32), (128, 128), (48, 12)])
@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_calls_that_continue_blocks(lib, call, page, block):
    import trismoe_b200 as tm

    g = _gen(page + len(call))
    heads, dim, dtype = 3, 64, BF16 if block == 32 else F16
    begin = [1 + (5 * b + 2) % (block - 1) for b in range(len(call))]  # tokens that are there already: no block's end
    table, pages = _table(g, [-(-(n + more) // page) for n, more in zip(begin, call)])
    k_pages, v_pages, k_scale, v_scale = _cache(pages, page, block, heads, dim)
    cos, sin = _rotation(2 * block + 64, dim)
    mirrors = Mirror(heads, dim, block), Mirror(heads, dim, block)

    def rows(seqs, pos, size):
        tokens = len(seqs)
        k, v = (torch.randn((tokens, heads, dim), generator=g, device="cuda") * size for _ in range(2))
        # magnitudes of their own for every token: some runs grow a scale, some do not
        k, v = (x * torch.exp2(torch.randint(-2, 5, (tokens, heads, 1), generator=g, device="cuda").float()) for x in (k, v))
        positions = torch.tensor(pos, device="cuda")
        args = k.to(dtype), v.to(dtype), k_pages, v_pages, table, positions, torch.tensor(seqs, device="cuda", dtype=torch.int32)
        k64, mag = _rotated_64(args[0], cos, sin, positions, False)
        for run in _runs(seqs, pos, block):
            i = list(run)
            mirrors[0].append(seqs[i[0]], [pos[j] for j in i], k64[i], mag[i])
            mirrors[1].append(seqs[i[0]], [pos[j] for j in i], args[1][i].double(), args[1][i].double().abs())
        return args

    append = lambda args: tm.append_paged_kv(None, *args, cos=cos, sin=sin, k_scale=k_scale, v_scale=v_scale)
    append(rows([b for b, n in enumerate(begin) for _ in range(n)], [i for n in begin for i in range(n)], 2.0 ** -6))
    held = [t.clone() for t in (k_pages, v_pages, k_scale, v_scale)]
    args = rows([b for b, n in enumerate(call) for _ in range(n)], [begin[b] + i for b, n in enumerate(call) for i in range(n)], 1.0)
    append(args)
    mirrors[0].check(k_pages, k_scale, table)
    mirrors[1].check(v_pages, v_scale, table)
    first = [t.view(torch.uint8).clone() for t in (k_pages, v_pages, k_scale, v_scale)]
    for _ in range(20):  # the same from the same cache, to the last bit
        for t, was in zip((k_pages, v_pages, k_scale, v_scale), held):
            t.copy_(was)
        append(args)
        for t, want in zip((k_pages, v_pages, k_scale, v_scale), first):
            assert torch.equal(t.view(torch.uint8), want)
