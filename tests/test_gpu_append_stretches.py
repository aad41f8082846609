"""GPU tests of appends that bring one block's tokens in two stretches: the second is refused, not run beside the first; padding elsewhere is no such thing."""
import pytest
import torch

from test_gpu_block_scaled_cache import F16, _cache, _rotation

pytestmark = pytest.mark.gpu


def _append(seqs, positions, page, block, sequences=4):
    """What a call leaves: places written, scales of keys, queries and keys out, status."""
    import trismoe_b200 as tm

    width = -(-(max(positions) + 1) // page)
    table = torch.arange(sequences * width, dtype=torch.int32, device="cuda").view(sequences, width)
    k_pages, v_pages, k_scales, v_scales = _cache(sequences * width, page, block, 2, 64)
    for scales in (k_scales, v_scales):
        scales[:] = 2.0 ** -30
    n = len(positions)
    k = torch.ones((n, 2, 64), dtype=F16, device="cuda") * torch.arange(1, n + 1, device="cuda")[:, None, None].half()
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    cos, sin = _rotation(max(positions) + 1, 64)
    q_out, k_out = tm.append_paged_kv(k, k, k, k_pages, v_pages, table, torch.tensor(positions, device="cuda"), torch.tensor(seqs, dtype=torch.int32, device="cuda"), cos=cos, sin=sin,
                                      k_scale=k_scales, v_scale=v_scales, return_key=True, status=status)
    assert torch.equal(q_out, k_out)
    held = []
    for pages in (k_pages, v_pages):
        written = pages.float().isfinite().all(-1)
        assert bool((written.all(-1) == written.any(-1)).all())
        held.append({(int(p) // width, int(p) % width * page + int(s)) for p, s in written.all(-1).nonzero()})
    assert held[0] == held[1]
    values = {(b, p): float(v_pages[b * width + p // page, p % page, 0, 0].float() * v_scales[b * width + p // page, p % page // block, 0]) for b, p in held[0]}
    return held[0], values, q_out, int(status)


def _check(seqs, positions, refused, page=16, block=16):
    written, values, q_out, status = _append(seqs, positions, page, block)
    good = [i for i, p in enumerate(positions) if p >= 0 and i not in refused]
    assert written == {(seqs[i], positions[i]) for i in good}
    for i in good:  # by its block's scale, whatever has been refused
        assert abs(values[seqs[i], positions[i]] - (i + 1)) <= 2.0 ** -4 * (i + 1)
    assert (status != 0) == bool(refused)
    for i, p in enumerate(positions):  # queries and keys go out all the same, padding as zeros
        assert bool((q_out[i] != 0).any()) == (p >= 0)


@pytest.mark.parametrize("positions,refused", [
    ([3, 4, 6, 7], [2, 3]), ([3, 4, -1, 5, 6], [3, 4]), ([5, 6, 0, 1], [2, 3]), ([3, 3], [1]), ([3] + [-1] * 70 + [4, 5], [71, 72]), ([14, 15, 17, 18], []), ([14, -1, 16, 17], []),
    ([3, 5, 7, 9], [1, 2, 3]), ([14, 15, 16, 18], [3]), ([-1, -1, 7, 8], []), ([3, 4, -1, -1], []), ([0, -1, 1], [2]), ([5, 2, 3, 40, 41], [1, 2])], ids=lambda v: ",".join(map(str, v[:8])) or "-")
def test_stretches_of_one_block(lib, positions, refused):
    _check([1] * len(positions), positions, refused)


def test_stretches_longer_than_a_window(lib):
    """Blocks of 128: runs of 40 and 50 tokens of one block with padding between them, a third that goes on into the next block."""
    positions = list(range(5, 45)) + [-1] * 33 + list(range(45, 95)) + list(range(100, 140))
    _check([2] * len(positions), positions, [i for i, p in enumerate(positions) if 45 <= p < 128], page=128, block=128)


def test_padded_batches_are_whole(lib):
    """Batches padded at either end whose sequences go on inside blocks: every row is a sequence of its own, whatever the padding's sequence is."""
    for left in (False, True):
        seqs, positions = [], []
        for b, (begin, n) in enumerate([(3, 40), (17, 1), (9, 0), (30, 25)]):
            row = list(range(begin, begin + n))
            pad = [-1] * (48 - n)
            positions += pad + row if left else row + pad
            seqs += [b] * 48
        _check(seqs, positions, [])
        _check([s if p >= 0 else 99 for s, p in zip(seqs, positions)], positions, [])


def test_free_slots_between_the_tokens_of_a_step(lib):
    """A decode step of slots, some of them free, whose tokens stand inside blocks; and the same with one sequence twice, behind free slots near and far."""
    slots = [(b, 3 + b % 9) if b % 3 else (b, -1) for b in range(80)]
    seqs, positions = [b for b, _ in slots], [p for _, p in slots]
    written, _, _, status = _append(seqs, positions, 16, 16, sequences=80)
    assert status == 0 and written == {(b, p) for b, p in slots if p >= 0}
    for at, gap in ((5, 1), (20, 7), (31, 1), (32, 1), (33, 40)):  # the slot at `at`, free slots, then its sequence once more
        again = at + gap + 1
        s, p = list(seqs), list(positions)
        p[at] = 5
        for i in range(at + 1, again):
            p[i] = -1
        s[again], p[again] = s[at], 7
        written, _, _, status = _append(s, p, 16, 16, sequences=80)
        assert written == {(s[i], p[i]) for i in range(80) if p[i] >= 0 and i != again} and status != 0, (at, gap)


def test_other_sequences_at_the_same_positions(lib):
    _check([0, 1, 2, 3], [3, 3, 3, 3], [])
    _check([0, 0, 1, 1, 1], [3, 4, 4, 5, 6], [])
    _check([0, 0, 1, 0], [3, 4, -1, 5], [3])
