"""CPU tests of what the decode harness hands to its operators."""
import types

import pytest
import torch


def test_products_in_8_bits_report_to_the_status_word(monkeypatch):
    """A product that gave up a wait leaves NaN, of which a draw makes token 0: nothing but the word says so."""
    from trismoe_b200 import decode_harness as dh

    calls = []
    monkeypatch.setattr(dh, "linear_e4m3", lambda *args, **more: calls.append((args, more)))
    monkeypatch.setattr(dh, "quantize_e4m3", lambda x: (x, "scales"))
    model = types.SimpleNamespace(linear8=True, cache_status=torch.zeros((1,), dtype=torch.int32))
    for x in (torch.zeros(2, 128), (torch.zeros(2, 128), "scales")):
        dh.TrisDecoder._linear(model, x, ("weight", "weight scales"), torch.float32)
    assert len(calls) == 2
    for args, more in calls:
        assert args[1:] == ("scales", "weight", "weight scales") and more["dtype"] is torch.float32 and more["status"] is model.cache_status


def test_a_decoder_without_layers_has_its_logits_in_8_bits(monkeypatch):
    """Embedding, norm and the logits' product alone."""
    from trismoe_b200 import decode_harness as dh

    monkeypatch.setattr(dh, "linear_e4m3", lambda x, xs, w, ws, dtype, status: (x.float() @ w.float().T).to(dtype))
    monkeypatch.setattr(dh, "quantize_e4m3", lambda x, group_rows=1: (x, None))
    shape = dh.DecoderShape(hidden_size=128, num_heads=2, head_dim=64, num_kv_heads=2, vocab_size=32)
    plain, eight = (dh.TrisDecoder([], shape, 8, 2, "cpu", page_size=4, linear_dtype=dtype) for dtype in (torch.float16, torch.float8_e4m3fn))
    ids, positions = torch.tensor([[1, 2], [3, 4]]), torch.arange(2)[None].expand(2, 2)
    want, got = plain(ids, positions), eight(ids, positions)
    assert got.dtype is want.dtype is torch.float32 and got.shape == (2, 32)
    assert float((got - want).abs().max()) <= 2.0 ** -10 * float(want.abs().max())  # the plain logits are rounded to 16 bits


@pytest.mark.parametrize("sampling", [{}, {"random": None}, {"random": torch.zeros(4, 3)}, {"random": torch.zeros(5, 2, dtype=torch.float64)}], ids=["none", "None", "shape", "type"])
def test_sampling_without_its_random_numbers_is_refused(sampling):
    """Before the prompt runs, in the harness's own words."""
    from trismoe_b200 import decode_harness as dh

    model = types.SimpleNamespace(max_length=20, max_batch=4)
    with pytest.raises(RuntimeError, match=r"random numbers, fp32 \[5, 2\]"):
        dh.run_exact_generation(model, torch.zeros((2, 3), dtype=torch.long), 5, sampling=sampling)
