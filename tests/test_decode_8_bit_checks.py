"""CPU tests of what products in 8 bits, block-scaled caches and the drawing of tokens refuse, before any CUDA call."""
import ctypes as C

import pytest
import torch

from test_decode_ops_checks import A, _cache, _call
from test_decode_step_sources import CSRC
from test_kernel_sources import _kernels


def test_products_that_are_refused(lib):
    import trismoe_b200 as tm

    good = dict(x=A, x_scales=A, weight=A, weight_scales=A, out=A, x_stride=256, x_scales_stride=2, weight_stride=256, weight_scales_stride=2, out_stride=64, rows=3, in_features=256,
                out_features=64)
    for change, status, text in [(dict(dtype=3), 1, "fp16, bf16 or fp32"), (dict(bias=A, bias_dtype=3), 1, "bias"), (dict(rows=-1), 1, "negative"), (dict(in_features=0), 1, "no columns"),
                                 (dict(x=None), 1, "null"), (dict(weight_scales=None), 1, "null"), (dict(out=None), 1, "null"), (dict(x=A + 8), 2, "16-byte"),
                                 (dict(x_stride=264), 2, "16-byte"), (dict(weight_stride=250), 2, "16-byte"), (dict(x_stride=240), 1, "overlap"), (dict(weight_stride=128), 1, "overlap"),
                                 (dict(out_stride=63), 1, "overlap"), (dict(rows=(1 << 30) + 1), 2, "2^30")]:
        st, message = _call(lib, "tris_e4m3_linear", tm._native.TrisE4m3Linear(**{**good, **change}))
        assert st == status and text in message, message
    for change in (dict(rows=0), dict(out_features=0)):
        assert _call(lib, "tris_e4m3_linear", tm._native.TrisE4m3Linear(**{**good, **change}))[0] == 0
    assert _call(lib, "tris_e4m3_linear", None)[0] == 1


def test_quantisations_that_are_refused(lib):
    import trismoe_b200 as tm

    good = dict(x=A, values=A, scales=A, x_stride=256, values_stride=256, scales_stride=2, rows=3, columns=256, group_rows=1)
    for change, status, text in [(dict(dtype=2), 1, "fp16 or bf16"), (dict(group_rows=2), 1, "1 or 128"), (dict(group_rows=0), 1, "1 or 128"), (dict(rows=-1), 1, "negative"),
                                 (dict(x=None), 1, "null"), (dict(values_stride=255), 1, "overlap"), (dict(scales_stride=1), 1, "overlap"), (dict(columns=(1 << 30) + 1), 2, "2^30"),
                                 (dict(rows=1 << 30, group_rows=128), 2, "too many")]:
        st, message = _call(lib, "tris_quantize_e4m3", tm._native.TrisQuantizeE4m3(**{**good, **change}))
        assert st == status and text in message, message
    for change in (dict(rows=0), dict(columns=0)):
        assert _call(lib, "tris_quantize_e4m3", tm._native.TrisQuantizeE4m3(**{**good, **change}))[0] == 0


def test_draws_that_are_refused(lib):
    import trismoe_b200 as tm

    good = dict(logits=A, random=A, out=A, logits_stride=100, rows=2, vocab=100)
    for change, status, text in [(dict(dtype=3), 1, "fp16, bf16 or fp32"), (dict(rows=-1), 1, "negative"), (dict(vocab=0), 1, "no vocabulary"), (dict(random=None), 1, "null"),
                                 (dict(out=None), 1, "null"), (dict(rows=65536), 2, "65535"), (dict(vocab=(1 << 28) + 1), 2, "2^28")]:
        st, message = _call(lib, "tris_sample_tokens", tm._native.TrisSampleTokens(**{**good, **change}))
        assert st == status and text in message, message
    assert _call(lib, "tris_sample_tokens", tm._native.TrisSampleTokens(**{**good, "rows": 0}))[0] == 0


def test_block_scaled_caches_that_are_refused(lib):
    import trismoe_b200 as tm

    n = tm._native
    base = dict(dtype=3, k_page_stride=4096, v_page_stride=4096, k_scale=A, v_scale=A, scale_tokens=4)
    calls = (("tris_paged_kv_append", n.TrisPagedAppend(k=A, v=A, positions=A, num_tokens=0)), ("tris_paged_decode_attention", n.TrisPagedAttention(q=A, out=A, lengths=A, num_q_heads=2)))
    for change, text in [(dict(scale_tokens=-1), "negative"), (dict(scale_tokens=5), "multiple"), (dict(scale_tokens=32), "multiple"), (dict(dtype=0), "e4m3"), (dict(k_scale=None), "null scales"),
                         (dict(v_scale=None), "null scales")]:
        for entry, args in calls:
            st, message = _call(lib, entry, _cache(tm, **{**base, **change}), args)
            assert st == 1 and text in message, (entry, message)
    assert _call(lib, "tris_paged_kv_append", _cache(tm, **base), calls[0][1])[0] == 0
    assert _call(lib, "tris_paged_decode_attention", _cache(tm, **{**base, "num_sequences": 0}), calls[1][1])[0] == 0
    st, message = _call(lib, "tris_paged_kv_append", _cache(tm, **base), n.TrisPagedAppend(k=A, v=A, positions=A, num_tokens=3))
    assert st == 1 and "3 tokens without sequences" in message


def test_struct_layouts(lib):
    """The packed bytes of the Python layer are the structs of the header."""
    import trismoe_b200 as tm
    from trismoe_b200 import decode_ops as d, e4m3_ops as e

    for cls, packed in ((tm._native.TrisSampleTokens, d._SAMPLE), (tm._native.TrisQuantizeE4m3, e._QUANTIZE), (tm._native.TrisE4m3Linear, e._LINEAR)):
        assert C.sizeof(cls) == packed.size
        values = list(range(1, len(cls._fields_) + 1))
        got = cls.from_buffer_copy(packed.pack(*values))
        assert [getattr(got, f[0]) for f in cls._fields_] == values
    assert tm._native.TrisPagedKv.scale_tokens.offset == 124 and C.sizeof(tm._native.TrisPagedKv) == 136


def test_cpu_tensors_are_refused(lib):
    import trismoe_b200 as tm

    x, scales = torch.zeros((2, 128)).to(torch.float8_e4m3fn), torch.zeros((2, 1))
    for call in (lambda: tm.linear_e4m3(x, scales, x, scales[:1]), lambda: tm.quantize_e4m3(torch.zeros((2, 128), dtype=torch.float16)),
                 lambda: tm.sample_tokens(torch.zeros((2, 8)), torch.zeros((2,)))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


FILES = ("e4m3_linear.cu", "paged_kv_blocks.cu", "quantize_e4m3.cu", "sample_tokens.cu")
KERNELS = [k for k in _kernels() if k[0] in FILES]


@pytest.mark.parametrize("file,name,params,body", KERNELS, ids=[k[1] for k in KERNELS])
def test_nothing_is_read_ahead_of_the_wait(file, name, params, body):
    """A launch may begin before the one ahead of it has ended, and any tensor of the call may be what that one writes."""
    import re

    ahead = body[: body.index("pdl_wait()")]
    ahead = re.sub(r"auto \w+ = \[&\][^{]*\{.*?\};", "", ahead, flags=re.S)
    assert not re.search(r"_cast<const|\ba\.\w+\[|\bs\.\w+\[|\br\.\w+\[|\bc\.\w+\[", ahead), (file, name)


def test_the_kernels_are_found():
    assert {k[1] for k in KERNELS} == {"e4m3_linear_kernel", "paged_kv_append_blocks_kernel", "quantize_rows_kernel", "quantize_blocks_kernel", "sample_tokens_kernel"}


@pytest.mark.parametrize("file", FILES)
def test_the_number_of_sms_is_the_devices(file):
    import os
    import re

    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, file)).read())
    assert not re.search(r"(?<![\w.])148(?![\w.])", text), file
