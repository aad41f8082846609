"""GPU tests of the decode harness in 8 bits: projections and the logits' product with block scales, a cache with a scale for each block of tokens and head, and tokens drawn
from the logits."""
import pytest
import torch

from test_gpu_paged_decode import VOCAB, _ids, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("more,tolerance", [(dict(cache_scale_tokens=16), 0.35), (dict(cache_scale_tokens=1), 0.35), (dict(linear_dtype=torch.float8_e4m3fn), 0.6),
                                            (dict(cache_scale_tokens=8, linear_dtype=torch.float8_e4m3fn), 0.8)], ids=["blocks", "tokens", "linear", "both"])
def test_eight_bits_all_the_way(lib, more, tolerance):
    """Tolerance: keys, values, and rows and weights of three products a layer and of the logits' are off by 2^-4 at most and 2^-5.5 on average; a logit is a sum of 256 of
    them of magnitude around its own size, of which the errors add up like their squares."""
    import trismoe_b200 as tm

    paged, dh = _model(tm, page_size=16, cache_dtype=torch.float8_e4m3fn if "cache_scale_tokens" in more else torch.float16, **more)
    dense, _ = _model(tm)
    ids, pos = _ids(3, 19)
    with torch.no_grad():
        scale = float(dense(ids, pos).abs().mean())
        assert float((paged(ids, pos) - dense(ids, pos)).abs().max()) <= tolerance * max(1.0, 5 * scale)
        for step in range(4):
            nxt = torch.full((3, 1), 7 + step, device="cuda")
            at = torch.full((3, 1), 19 + step, device="cuda")
            assert float((paged(nxt, at) - dense(nxt, at)).abs().max()) <= tolerance * max(1.0, 5 * scale)
    paged.raise_on_kernel_status()


def test_drawn_generation(lib):
    """A captured step and an eager one draw the same tokens from the same numbers; a first token alone is the greedy one; a grammar is kept."""
    import trismoe_b200 as tm

    model, dh = _model(tm, page_size=16, cache_dtype=torch.float8_e4m3fn, cache_scale_tokens=16, linear_dtype=torch.float8_e4m3fn)
    ids, _ = _ids(3, 9)
    each = lambda value, dtype=torch.float32: torch.full((3,), value, dtype=dtype, device="cuda")
    sampling = {"random": torch.rand((12, 3), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda"), "temperature": each(0.9), "top_k": each(40, torch.int32),
                "top_p": each(0.95), "min_p": each(0.01)}
    eager = dh.run_exact_generation(model, ids, 12, use_graph=False, sampling=sampling)["tokens"]
    graph = dh.run_exact_generation(model, ids, 12, use_graph=True, sampling=sampling)["tokens"]
    assert torch.equal(eager, graph)
    other = dict(sampling, random=1 - sampling["random"].clamp(min=0.01))
    assert not torch.equal(eager, dh.run_exact_generation(model, ids, 12, sampling=other)["tokens"])
    greedy = dh.run_exact_generation(model, ids, 12)["tokens"]
    assert torch.equal(greedy, dh.run_exact_generation(model, ids, 12, sampling=dict(random=sampling["random"], top_k=each(1, torch.int32)))["tokens"])
    allowed = torch.zeros((3, VOCAB // 32), dtype=torch.int32, device="cuda")
    allowed[:, 2] = 0x55  # tokens 64, 66, 68 and 70
    drawn = dh.run_exact_generation(model, ids, 12, logit_controls={"allowed": allowed}, sampling=sampling)["tokens"]
    assert set(drawn.flatten().tolist()) <= {64, 66, 68, 70}
    nothing = dh.run_exact_generation(model, ids, 4, logit_controls={"allowed": torch.zeros_like(allowed)}, sampling=dict(sampling, random=sampling["random"][:4].contiguous()))["tokens"]
    assert bool((nothing == 0).all())
    model.raise_on_kernel_status()
    with pytest.raises(RuntimeError, match="random numbers"):
        dh.run_exact_generation(model, ids, 5, sampling=sampling)
