"""GPU test of the decode harness on a paged cache: the same tokens' logits as over the dense cache and from scratch, the captured
loop gives what the eager one does, and penalties, biases and grammar masks act on every step."""
import pytest
import torch

pytestmark = pytest.mark.gpu
VOCAB = 512


def _model(tm, **more):
    from trismoe_b200 import decode_harness as dh, synth

    shape = synth.LayerShape(256, 192, 8, 2, rank=96, group_size=32)
    blocks = []
    for l in range(2):
        layer = synth.synth_layer(shape, seed=80 + l)
        for name in ("gate", "up", "down"):
            layer["shared_" + name] = (layer["shared_" + name].float() * 5.0).half()
        blk = tm.TrisSparseMoeBlock(shape.hidden_size, shape.intermediate_size, shape.num_experts, shape.top_k, True)
        blk.load_grouped_payloads(layer["gate"], layer["up"], layer["down"], layer["shared_gate"], layer["shared_up"],
                                  layer["shared_down"], layer["router_weight"], device="cuda")
        blocks.append(blk)
    dshape = dh.DecoderShape(hidden_size=256, num_heads=4, head_dim=64, num_kv_heads=2, vocab_size=VOCAB)
    return dh.TrisDecoder(blocks, dshape, max_length=50, max_batch=4, device="cuda", seed=3, **more), dh


def _ids(B, L):
    ids = torch.randint(0, VOCAB, (B, L), generator=torch.Generator().manual_seed(1)).cuda()
    return ids, torch.arange(L, device="cuda")[None, :].expand(B, L).contiguous()


@pytest.mark.parametrize("page,cache,tolerance", [(16, torch.float16, 0.02), (7, torch.float16, 0.02), (16, torch.float8_e4m3fn, 0.35)], ids=["16", "7", "e4m3"])
def test_paged_cache_gives_the_dense_caches_logits(lib, page, cache, tolerance):
    """Tolerance: two layers of fp16 activations around 1 whose attention differs by roundings (dense: 16-bit weights and sums in another order);
    keys and values in 8 bits are off by 2^-4 at most, scores and averages by less."""
    import trismoe_b200 as tm

    paged, _ = _model(tm, page_size=page, cache_dtype=cache)
    dense, _ = _model(tm)
    ids, pos = _ids(3, 19)
    with torch.no_grad():
        scale = float(dense(ids, pos).abs().mean())
        assert float((paged(ids, pos) - dense(ids, pos)).abs().max()) <= tolerance * max(1.0, 5 * scale)
        for step in range(4):  # across the end of a page
            nxt = torch.full((3, 1), 7 + step, device="cuda")
            at = torch.full((3, 1), 19 + step, device="cuda")
            assert float((paged(nxt, at) - dense(nxt, at)).abs().max()) <= tolerance * max(1.0, 5 * scale)
    paged.raise_on_kernel_status()


def test_paged_generation_in_a_graph_equals_the_eager_one(lib):
    import trismoe_b200 as tm

    model, dh = _model(tm, page_size=16)
    ids, _ = _ids(3, 14)
    eager = dh.run_exact_generation(model, ids, 9, use_graph=False)
    graph = dh.run_exact_generation(model, ids, 9, use_graph=True)
    assert graph["launch_mode"] == "cuda graph" and torch.equal(eager["tokens"], graph["tokens"])
    model.raise_on_kernel_status()


@pytest.mark.parametrize("page", [None, 16])
def test_controls_act_on_every_step(lib, page):
    import trismoe_b200 as tm

    model, dh = _model(tm, page_size=page)
    ids, _ = _ids(3, 10)
    f32 = lambda v: torch.full((3,), v, device="cuda")
    # a grammar of the tokens 64 to 95, and no token twice
    allowed = torch.zeros((3, VOCAB // 32), dtype=torch.int32, device="cuda")
    allowed[:, 2] = -1
    runs = [dh.run_exact_generation(model, ids, 8, use_graph=g, logit_controls={"allowed": allowed, "presence": f32(1e4)}) for g in (False, True)]
    assert torch.equal(runs[0]["tokens"], runs[1]["tokens"])
    for row in runs[0]["tokens"].tolist():
        assert all(64 <= t < 96 for t in row) and len(set(row)) == 8
    # a bias that outweighs everything else
    ids_ = torch.tensor([[5], [6], [7]], dtype=torch.int32, device="cuda")
    out = dh.run_exact_generation(model, ids, 3, logit_controls={"bias_ids": ids_, "bias_values": torch.full((3, 1), 1e5, device="cuda")})
    assert out["tokens"].tolist() == [[5] * 3, [6] * 3, [7] * 3]
    plain = dh.run_exact_generation(model, ids, 5)["tokens"]
    assert torch.equal(dh.run_exact_generation(model, ids, 5, logit_controls={"repetition": f32(1.0)})["tokens"], plain)


def test_a_dense_cache_in_8_bits_is_refused(lib):
    import trismoe_b200 as tm

    with pytest.raises(RuntimeError, match="paged"):
        _model(tm, cache_dtype=torch.float8_e4m3fn)
