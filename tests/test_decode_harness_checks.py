"""CPU tests of what the decode harness hands to its operators."""
import types

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
