"""CPU tests of what the operators of a decode step refuse, before any CUDA call: wrong sizes, types, strides and missing
parts at the C entry points, and tensors that do not live on a CUDA device at the Python ones."""
import ctypes as C

import pytest
import torch

A = 1 << 20  # an address that is never followed


def _cache(tm, **more):
    c = tm._native.TrisPagedKv(k_pages=A, v_pages=A, k_page_stride=2048, k_token_stride=64, k_head_stride=1024, v_page_stride=2048, v_token_stride=64,
                               v_head_stride=1024, block_table=A, table_stride=4, num_sequences=2, table_width=4, num_pages=8, page_size=16,
                               num_kv_heads=2, head_dim=64, dtype=0)
    for name, value in more.items():
        setattr(c, name, value)
    return c


def _call(lib, entry, *structs):
    return getattr(lib, entry)(*(None if s is None else C.byref(s) for s in structs), None), lib.tris_last_error().decode()


BAD_CACHES = [
    (dict(k_pages=None), 1, "null pages"), (dict(block_table=None), 1, "null block table"), (dict(page_size=0), 1, "sizes"), (dict(num_pages=-1), 1, "sizes"),
    (dict(dtype=2), 1, "fp16, bf16 or e4m3"), (dict(head_dim=60), 2, "16 bytes"), (dict(head_dim=264), 2, "256"), (dict(dtype=3, head_dim=72), 2, "16 bytes"),
    (dict(k_token_stride=68), 2, "multiples of 16 bytes"), (dict(v_head_stride=-8), 2, "multiples of 16 bytes"), (dict(v_pages=A + 8), 2, "16-byte boundary"),
]


@pytest.mark.parametrize("change,status,text", BAD_CACHES)
def test_caches_that_are_refused(lib, change, status, text):
    import trismoe_b200 as tm

    n = tm._native
    for entry, args in (("tris_paged_kv_append", n.TrisPagedAppend(k=A, v=A, positions=A, num_tokens=1)),
                        ("tris_paged_decode_attention", n.TrisPagedAttention(q=A, out=A, lengths=A, workspace=A, num_q_heads=2))):
        st, message = _call(lib, entry, _cache(tm, **change), args)
        assert st == status and text in message, (entry, message)
    assert lib.tris_paged_decode_attention_workspace_bytes(C.byref(_cache(tm, **change)), 2, 0) == 0


def test_appends_that_are_refused(lib):
    import trismoe_b200 as tm

    good = dict(q=A, k=A, v=A, q_out=A, positions=A, cos=A, sin=A, num_tokens=1, num_q_heads=2, rotary_dim=64, max_positions=8, q_token_stride=512,
                q_head_stride=64, k_token_stride=512, k_head_stride=64, v_token_stride=512, v_head_stride=64)
    for change, status, text in [(dict(dtype=2), 1, "fp16 or bf16"), (dict(dtype=1), 1, "rows' type or e4m3"), (dict(num_tokens=-1), 1, "negative"),
                                 (dict(q=None), 1, "q_out"), (dict(sin=None), 1, "go together"), (dict(rotary_dim=63), 1, "even"), (dict(rotary_dim=66), 1, "even"),
                                 (dict(k=None), 1, "null k"), (dict(positions=None), 1, "null k"), (dict(rotary_dim=6), 2, "multiple of 4"),
                                 (dict(num_tokens=1 << 30), 2, "too many tokens")]:
        st, message = _call(lib, "tris_paged_kv_append", _cache(tm), tm._native.TrisPagedAppend(**{**good, **change}))
        assert st == status and text in message, message
    assert _call(lib, "tris_paged_kv_append", _cache(tm), None)[0] == 1 and _call(lib, "tris_paged_kv_append", None, None)[0] == 1
    assert _call(lib, "tris_paged_kv_append", _cache(tm), tm._native.TrisPagedAppend(num_tokens=0))[0] == 0


def test_attentions_that_are_refused(lib):
    import trismoe_b200 as tm

    good = dict(q=A, out=A, lengths=A, workspace=A, num_q_heads=4)
    for change, status, text in [(dict(dtype=3), 1, "fp16 or bf16"), (dict(dtype=1), 1, "queries' type or e4m3"), (dict(num_q_heads=3), 1, "share"),
                                 (dict(num_q_heads=0), 1, "share"), (dict(window=-1), 1, "window"), (dict(q=None), 1, "null q"), (dict(out=A + 4), 1, "aligned")]:
        st, message = _call(lib, "tris_paged_decode_attention", _cache(tm), tm._native.TrisPagedAttention(**{**good, **change}))
        assert st == status and text in message, message
    assert _call(lib, "tris_paged_decode_attention", _cache(tm, num_sequences=65536), tm._native.TrisPagedAttention(**good))[0] == 2
    assert _call(lib, "tris_paged_decode_attention", _cache(tm, num_sequences=0), tm._native.TrisPagedAttention(**good))[0] == 0
    assert lib.tris_paged_decode_attention_workspace_bytes(C.byref(_cache(tm)), 3, 0) == 0


def test_norms_that_are_refused(lib):
    import trismoe_b200 as tm

    good = dict(x=A, weight=A, y=A, scales=A, rows=1, hidden_size=96, group_size=32, dtype_out=3)
    for change, text in [(dict(dtype=2), "fp16 or bf16"), (dict(dtype_out=1), "rows' type or e4m3"), (dict(hidden_size=0), "sizes"), (dict(weight=None), "null x"),
                         (dict(scales=None), "null scales"), (dict(group_size=24), "multiples of 16"), (dict(group_size=64), "multiples of 16"), (dict(group_size=0), "multiples of 16")]:
        st, message = _call(lib, "tris_add_rms_norm", tm._native.TrisAddRmsNorm(**{**good, **change}))
        assert st == 1 and text in message, message
    assert _call(lib, "tris_add_rms_norm", tm._native.TrisAddRmsNorm(**{**good, "rows": 0}))[0] == 0


def test_logit_controls_that_are_refused(lib):
    import trismoe_b200 as tm

    good = dict(logits=A, out=A, rows=2, vocab=100, tokens=A, token_lengths=A, repetition=A, max_tokens=8)
    for change, status, text in [(dict(dtype=3), 1, "fp16, bf16 or fp32"), (dict(vocab=-1), 1, "negative"), (dict(out=None), 1, "null logits"),
                                 (dict(token_lengths=None), 1, "token_lengths"), (dict(tokens=None), 1, "need tokens"), (dict(bias_ids=A), 1, "go together"),
                                 (dict(rows=65536), 2, "65535"), (dict(max_tokens=1 << 30), 2, "2^30")]:
        st, message = _call(lib, "tris_logit_controls", tm._native.TrisLogitControls(**{**good, **change}))
        assert st == status and text in message, message
    assert _call(lib, "tris_logit_controls", tm._native.TrisLogitControls(**{**good, "rows": 0}))[0] == 0


def test_struct_layouts(lib):
    """The packed bytes of the Python layer are the structs of the header."""
    import trismoe_b200 as tm
    from trismoe_b200 import decode_ops as d

    for cls, packed in ((tm._native.TrisPagedKv, d._PAGED_KV), (tm._native.TrisPagedAppend, d._APPEND), (tm._native.TrisPagedAttention, d._ATTENTION),
                        (tm._native.TrisAddRmsNorm, d._NORM), (tm._native.TrisLogitControls, d._LOGITS)):
        assert C.sizeof(cls) == packed.size
        values = [1.5 if f[1] is C.c_float else i + 1 for i, f in enumerate(cls._fields_)]
        got = cls.from_buffer_copy(packed.pack(*values))
        assert [getattr(got, f[0]) for f in cls._fields_] == values


def test_cpu_tensors_are_refused(lib):
    import trismoe_b200 as tm

    x, pages = torch.zeros((1, 2, 64), dtype=torch.float16), torch.zeros((2, 16, 2, 64), dtype=torch.float16)
    table, one = torch.zeros((1, 2), dtype=torch.int32), torch.ones((1,), dtype=torch.int32)
    for call in (lambda: tm.append_paged_kv(x, x, x, pages, pages, table, one), lambda: tm.paged_decode_attention(x, pages, pages, table, one),
                 lambda: tm.add_rms_norm(x, None, torch.ones(64, dtype=torch.float16)), lambda: tm.add_rms_norm_e4m3(x, None, torch.ones(64, dtype=torch.float16)),
                 lambda: tm.apply_logit_controls(torch.zeros((1, 8)))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
