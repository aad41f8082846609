"""CPU tests of what a status word says."""
import pytest
import torch


@pytest.mark.parametrize("word,whose,text", [(4, "paged cache", "TRIS_ERR_CORRUPT .*outside the cache"), (6, "product in 8 bits", "TRIS_ERR_TIMEOUT .*a wait ran out"), (77, "status word", "77")])
def test_a_word_says_what_has_happened(word, whose, text):
    import trismoe_b200 as tm

    status = torch.tensor([word], dtype=torch.int32)
    with pytest.raises(RuntimeError, match=f"{whose}: a kernel reported {text}"):
        tm.raise_on_status(status)
    with pytest.raises(RuntimeError, match=f"layer 3: a kernel reported {text}"):
        tm.raise_on_status(status, "layer 3")
    if word == 6:
        with pytest.raises(RuntimeError) as error:
            tm.raise_on_status(status)
        assert "position" not in str(error.value)


def test_no_word_no_error():
    import trismoe_b200 as tm

    tm.raise_on_status(torch.zeros((1,), dtype=torch.int32))
