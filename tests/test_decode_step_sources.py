"""CPU tests of rules of the decode step's kernel sources.  A kernel that may be launched while its predecessor still runs reads nothing from memory
ahead of its wait: any tensor of the call - a norm's weight as 1 + w, too - may be what the predecessor writes."""
import os
import re

import pytest

from test_kernel_sources import CSRC, _kernels

FILES = ("logit_controls.cu", "paged_attention.cu", "paged_kv.cu", "rms_norm.cu")
KERNELS = [k for k in _kernels() if k[0] in FILES]


@pytest.mark.parametrize("file,name,params,body", KERNELS, ids=[k[1] for k in KERNELS])
def test_nothing_is_read_ahead_of_the_wait(file, name, params, body):
    ahead = body[: body.index("pdl_wait()")]
    # a cast to a type with elements, or an element taken, ahead of the wait outside of a lambda that is only called behind it
    ahead = re.sub(r"auto \w+ = \[&\][^{]*\{.*?\};", "", ahead, flags=re.S)
    assert not re.search(r"_cast<const|\ba\.\w+\[|\bc\.\w+\[", ahead), (file, name)


def test_the_kernels_are_found():
    assert {k[1] for k in KERNELS} >= {"add_rms_norm_kernel", "add_rms_norm_any_kernel", "paged_kv_append_kernel", "paged_attention_kernel",
                                       "paged_attention_join_kernel", "logit_controls_kernel"}


@pytest.mark.parametrize("file", FILES)
def test_the_number_of_sms_is_the_devices(file):
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, file)).read())
    assert not re.search(r"(?<![\w.])148(?![\w.])", text), file
