"""CPU tests of further refusals of the decode step's entry points, before any CUDA call."""
from test_decode_ops_checks import A, _cache, _call


def test_an_append_of_tokens_that_have_no_sequence(lib):
    """Without sequences token t belongs to row t of the block table, which has two."""
    import trismoe_b200 as tm

    rows = dict(k=A, v=A, positions=A, k_token_stride=128, k_head_stride=64, v_token_stride=128, v_head_stride=64)
    status, message = _call(lib, "tris_paged_kv_append", _cache(tm), tm._native.TrisPagedAppend(num_tokens=3, **rows))
    assert status == 1 and "3 tokens without sequences" in message


def test_strides_count_where_a_size_is_more_than_one(lib):
    import trismoe_b200 as tm

    for sizes in (dict(num_pages=1), dict(page_size=1), dict(num_kv_heads=1)):
        name = {"num_pages": "page", "page_size": "token", "num_kv_heads": "head"}[next(iter(sizes))]
        odd = {f"k_{name}_stride": 3, f"v_{name}_stride": -5}
        assert _call(lib, "tris_paged_kv_append", _cache(tm, **sizes, **odd), tm._native.TrisPagedAppend(num_tokens=0))[0] == 0
        for one in odd.items():
            status, message = _call(lib, "tris_paged_kv_append", _cache(tm, **dict([one])), tm._native.TrisPagedAppend(num_tokens=0))
            assert status == 2 and "strides" in message
