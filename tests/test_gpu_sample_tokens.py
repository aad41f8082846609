"""GPU tests of drawing tokens, against the definition in 64 bits: the same token, always.  Weights are counted in units of 2^-46 of the largest (fewer bits for
vocabularies beyond 65536); the oracle rounds its weights to the same units, so that sums of either are exact and only exp itself differs, by 2^-52 of a weight."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _drawn_64(logits, random, temperature=None, top_k=None, top_p=None, min_p=None):
    vocab = logits.shape[1]
    bits = 46
    while vocab << bits >= 1 << 62:
        bits -= 1
    chosen = []
    for b in range(logits.shape[0]):
        z = logits[b].double()
        z = torch.where(z.isnan(), -math.inf, z)
        t = 1.0 if temperature is None else float(temperature[b])
        k = 0 if top_k is None else int(top_k[b])
        p = 1.0 if top_p is None else float(top_p[b])
        m = 0.0 if min_p is None else float(min_p[b])
        best = z.max()
        if best == -math.inf:
            chosen.append(-1)
            continue
        if not t > 0 or k == 1 or p <= 0 or best == math.inf:
            chosen.append(int((z == best).nonzero()[0, 0]))
            continue
        ids = torch.argsort(-z, stable=True)[: int((z > -math.inf).sum())]
        if k > 0:
            ids = ids[:k]
        w = torch.exp((z[ids] - best) / t)
        units = (w * 2.0 ** bits).round().long()
        if p < 1:
            ahead = units.cumsum(0) - units
            ids_kept = (ahead.double() < p * float(units.sum())) | (torch.arange(ids.numel(), device="cuda") == 0)
            ids, units, w = ids[ids_kept], units[ids_kept], w[ids_kept]
        if m > 0:
            keep = units >= math.ceil(min(m, 1.0) * 2.0 ** bits)
            ids, units = ids[keep], units[keep]
        order = ids.argsort()
        ids, sums = ids[order], units[order].cumsum(0)
        whole = int(sums[-1])
        u = float(random[b])
        target = min(whole - 1, int(max(u, 0.0) * whole)) if u == u else 0
        chosen.append(int(ids[int((sums <= target).sum())]))
    return torch.tensor(chosen, device="cuda")


def _controls(g, rows, names):
    uniform = lambda low, high: low + (high - low) * torch.rand((rows,), generator=g, device="cuda")
    made = {"temperature": uniform(0.3, 1.5), "top_k": torch.randint(0, 120, (rows,), generator=g, device="cuda", dtype=torch.int32),
            "top_p": uniform(0.05, 1.1), "min_p": uniform(-0.05, 0.3)}
    return {name: made[name] for name in names}


ALL = ("temperature", "top_k", "top_p", "min_p")


@pytest.mark.parametrize("names", [(), ("temperature",), ("top_k",), ("top_p",), ("min_p",), ("top_k", "top_p"), ALL], ids=lambda n: "+".join(n) or "none")
@pytest.mark.parametrize("dtype", [F16, BF16, F32], ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 31), (40, 1000), (1, 50304), (9, 50304), (170, 513), (2, 131073)])
def test_draws(lib, rows, vocab, dtype, names):
    import trismoe_b200 as tm

    g = _gen(rows + vocab)
    logits = (torch.randn((rows, vocab + 5), generator=g, device="cuda") * 2.5).to(dtype)[:, 3: vocab + 3]
    random = torch.rand((rows,), generator=g, device="cuda")
    controls = _controls(g, rows, names)
    got = tm.sample_tokens(logits, random, **controls)
    assert got.dtype == torch.int64 and got.shape == (rows,)
    assert torch.equal(got, _drawn_64(logits, random, **controls))


@pytest.mark.parametrize("k", [2, 100, 256, 257, 1000, 20000, 49999, 50304, 60000])
def test_first_k_of_any_number(lib, k):
    import trismoe_b200 as tm

    g = _gen(k)
    logits, random = torch.randn((3, 50304), generator=g, device="cuda") * 2, torch.rand((3,), generator=g, device="cuda")
    top_k = torch.full((3,), k, dtype=torch.int32, device="cuda")
    for top_p in (None, torch.full((3,), 0.9, device="cuda")):
        assert torch.equal(tm.sample_tokens(logits, random, top_k=top_k, top_p=top_p), _drawn_64(logits, random, top_k=top_k, top_p=top_p))


@pytest.mark.parametrize("values", [[0.0], [1.0, 0.0], [3.0, 3.0, -1.0], [-0.0, 0.0, -20.0], [5.0, -math.inf]], ids=str)
@pytest.mark.parametrize("vocab", [7, 5000, 50304])
def test_equal_logits_are_kept_by_their_index(lib, vocab, values):
    """Thousands of equal numbers at the border: the first ones by index, exactly as many as the limits allow."""
    import trismoe_b200 as tm

    rows = 12
    logits = torch.tensor(values, device="cuda").repeat(-(-vocab // len(values)))[:vocab].repeat(rows, 1)
    random = torch.linspace(0, 1 - 2 ** -24, rows, device="cuda")
    for controls in ({}, {"top_k": torch.arange(2, 2 + 97 * rows, 97, dtype=torch.int32, device="cuda")}, {"top_p": torch.linspace(0.01, 0.99, rows, device="cuda")},
                     {"top_k": torch.full((rows,), vocab // 2 + 1, dtype=torch.int32, device="cuda"), "top_p": torch.full((rows,), 0.5, device="cuda")},
                     {"min_p": torch.full((rows,), 1.0, device="cuda")}):
        assert torch.equal(tm.sample_tokens(logits, random, **controls), _drawn_64(logits, random, **controls))


@pytest.mark.parametrize("low", [-math.inf, -65504.0, -3.0e38, torch.finfo(F32).min], ids=str)
def test_masked_logits(lib, low):
    """Half of the vocabulary, all but one, and all of it closed, by -inf or by a type's lowest number."""
    import trismoe_b200 as tm

    g = _gen(3)
    logits = torch.randn((6, 20000), generator=g, device="cuda") * 3
    logits[0, ::2] = low
    logits[1, torch.arange(20000, device="cuda") != 777] = low
    logits[2] = low
    logits[3, 5:] = low
    logits[4, :-1] = low
    random = torch.rand((6,), generator=g, device="cuda")
    for names in ((), ("top_k",), ("top_p",), ALL):
        controls = _controls(g, 6, names)
        got = tm.sample_tokens(logits, random, **controls)
        assert torch.equal(got, _drawn_64(logits, random, **controls))
        assert int(got[1]) == 777 and int(got[4]) == 19999 and (low != -math.inf or int(got[2]) == -1)


def test_nan_and_infinite_logits(lib):
    import trismoe_b200 as tm

    g = _gen(4)
    logits = torch.randn((5, 3000), generator=g, device="cuda")
    logits[0, ::3] = math.nan
    logits[1] = math.nan
    logits[2, 1500:1510] = math.inf
    logits[3, 0] = math.nan
    random = torch.rand((5,), generator=g, device="cuda")
    for names in ((), ("top_k",), ("top_p",), ALL):
        controls = _controls(g, 5, names)
        got = tm.sample_tokens(logits, random, **controls)
        assert torch.equal(got, _drawn_64(logits, random, **controls))
        assert int(got[1]) == -1 and int(got[2]) == 1500


@pytest.mark.parametrize("temperature", [0.0, -1.0, math.nan, 1e-38, 1e-4, 0.02, 50.0, 1e30, math.inf])
def test_temperatures(lib, temperature):
    import trismoe_b200 as tm

    g = _gen(5)
    logits, random = torch.randn((4, 9001), generator=g, device="cuda").bfloat16(), torch.rand((4,), generator=g, device="cuda")
    t = torch.full((4,), temperature, device="cuda")
    for names in ((), ("top_k",), ("top_p", "min_p")):
        controls = dict(_controls(g, 4, names), temperature=t)
        assert torch.equal(tm.sample_tokens(logits, random, **controls), _drawn_64(logits, random, **controls))


@pytest.mark.parametrize("u", [0.0, 2.0 ** -24, 1 - 2.0 ** -24, 1.0, 7.0, -3.0, math.nan])
def test_ends_of_the_random_numbers(lib, u):
    import trismoe_b200 as tm

    logits = torch.randn((3, 4000), generator=_gen(6), device="cuda") * 2
    random = torch.full((3,), u, device="cuda")
    for controls in ({}, {"top_p": torch.full((3,), 0.8, device="cuda")}, {"top_k": torch.full((3,), 9, dtype=torch.int32, device="cuda")}):
        assert torch.equal(tm.sample_tokens(logits, random, **controls), _drawn_64(logits, random, **controls))


@pytest.mark.parametrize("p", [-1.0, 0.0, 1e-20, 0.5, 1 - 2.0 ** -24, 1.0, 2.0, math.nan])
def test_ends_of_the_shares(lib, p):
    import trismoe_b200 as tm

    g = _gen(8)
    logits, random = torch.randn((4, 6000), generator=g, device="cuda"), torch.rand((4,), generator=g, device="cuda")
    share = torch.full((4,), p, device="cuda")
    assert torch.equal(tm.sample_tokens(logits, random, top_p=share), _drawn_64(logits, random, top_p=share))
    assert torch.equal(tm.sample_tokens(logits, random, min_p=share), _drawn_64(logits, random, min_p=share))


def test_draws_follow_the_weights(lib):
    """Evenly spaced numbers draw every token as often as its weight says, to one."""
    import trismoe_b200 as tm

    rows = 4000
    z = torch.tensor([1.0, 2.0, 0.0, 2.0, -1.0], device="cuda")
    random = (torch.arange(rows, device="cuda") + 0.5) / rows
    got = tm.sample_tokens(z.repeat(rows, 1), random, temperature=torch.full((rows,), 0.7, device="cuda"))
    share = torch.softmax(z.double() / 0.7, 0) * rows
    assert bool(((torch.bincount(got, minlength=5) - share).abs() <= 1).all())


def test_rows_apart_streams_and_graphs(lib):
    import trismoe_b200 as tm

    g = _gen(9)
    wide = torch.randn((60, 8000), generator=g, device="cuda")
    random = torch.rand((20,), generator=g, device="cuda")
    controls = _controls(g, 20, ALL)
    logits = wide[::3, 1: 7001]
    want = _drawn_64(logits, random, **controls)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tm.sample_tokens(logits, random, **controls)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tm.sample_tokens(logits, random, **controls)
    for seed in (1, 2):
        wide.copy_(torch.randn(wide.shape, generator=_gen(seed), device="cuda"))
        random.copy_(torch.rand((20,), generator=_gen(seed + 10), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _drawn_64(logits, random, **controls))


def test_no_rows(lib):
    import trismoe_b200 as tm

    assert tm.sample_tokens(torch.empty((0, 10), device="cuda"), torch.empty((0,), device="cuda")).shape == (0,)
