"""CPU tests of which CTA of the append to block-scaled pages has which run of tokens: the rule of block_runs.cuh, compiled for the host, in the kernel's walk over windows."""
import ctypes as C
import os
import random
import subprocess

import pytest

from test_decode_ops_checks import A, _cache, _call
from test_kernel_sources import CSRC

WINDOW = 16


@pytest.fixture(scope="module")
def rule(tmp_path_factory):
    """tokens_of_whole_runs of the header."""
    at = tmp_path_factory.mktemp("block_runs")
    source, library = at / "rule.cpp", at / "rule.so"
    source.write_text('#include "block_runs.cuh"\nextern "C" int rule(uint32_t starts, int own, int window) { return tris::tokens_of_whole_runs(starts, own, window); }\n')
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(source), "-o", str(library)], check=True)
    f = C.CDLL(str(library)).rule
    f.argtypes, f.restype = [C.c_uint32, C.c_int, C.c_int], C.c_int
    return f


def owners(begins, rule):
    """How often each run's first token is taken, and each token appended, by the CTAs of the whole grid."""
    n = len(begins)
    runs, tokens = [0] * n, [0] * n
    bits = lambda w: sum((1 << i) for i in range(32) if w + i >= n or begins[w + i])
    for first in range(0, n, WINDOW):
        end, w = min(first + WINDOW, n), first
        starts = bits(w)
        if not starts & ((1 << WINDOW) - 1):
            continue
        skip = (starts & -starts).bit_length() - 1
        w, starts = w + skip, starts >> skip
        while w < end:
            count = rule(starts, end - w, WINDOW)
            if not count:  # one run, longer than a window
                count = WINDOW
                while True:
                    more = bits(w + count)
                    count += (more & -more).bit_length() - 1 if more else 32
                    if more:
                        break
            else:
                assert count <= WINDOW and (w + count >= n or begins[w + count])
            for t in range(w, w + count):
                if t < n:
                    tokens[t] += 1
                    runs[t] += begins[t]
            w += count
            if w < end:
                starts = bits(w)
    return runs, tokens


def _begins(lengths):
    return [i == 0 for n in lengths for i in range(n)]


def _check(lengths, rule):
    begins = _begins(lengths)
    runs, tokens = owners(begins, rule)
    assert runs == [int(b) for b in begins] and tokens == [1] * len(begins), lengths


@pytest.mark.parametrize("lengths", [[5] * 8, [3] * 60, [10, 7] + [1] * 40, [17] + [1] * 47, [16] * 9, [15, 16] * 7, [1] * 65, [128, 1, 3, 128, 16, 40], [1], [16], [17], [33, 15, 16, 1]],
                         ids=lambda lengths: f"{len(lengths)} runs, first {lengths[0]}")
def test_every_run_has_one_owner(rule, lengths):
    _check(lengths, rule)


@pytest.mark.parametrize("seed", range(8))
def test_every_run_of_random_calls_has_one_owner(rule, seed):
    rng = random.Random(seed)
    for _ in range(400):
        longest = rng.choice([1, 2, 5, 15, 16, 17, 30, 64, 128])
        _check([rng.randint(1, longest) for _ in range(rng.randint(1, 60))], rule)


def test_the_kernel_asks_the_rule():
    """The window that the kernel looks at is the one that is tried here."""
    text = open(os.path.join(CSRC, "paged_kv_blocks.cu")).read()
    assert f"kWindow = {WINDOW};" in text and text.count("tokens_of_whole_runs(starts, end - w, R)") == 1


def test_keys_and_values_need_scales_of_their_own(lib):
    """An append writes both; attention may read the same ones."""
    import trismoe_b200 as tm

    n = tm._native
    base = dict(dtype=3, k_page_stride=4096, v_page_stride=4096, scale_tokens=4)
    args = n.TrisPagedAppend(k=A, v=A, positions=A, num_tokens=1)
    st, message = _call(lib, "tris_paged_kv_append", _cache(tm, **base, k_scale=A, v_scale=A), args)
    assert st == 1 and "the same scales" in message, message
    st, message = _call(lib, "tris_paged_kv_append", _cache(tm, **base, num_pages=0), n.TrisPagedAppend(k=A, v=A, positions=A, num_tokens=3))
    assert st == 1 and "without sequences" in message, message  # a cache without pages has none of either
