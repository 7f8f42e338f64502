"""Attention however its work is cut: wavefronts alone on their block of rows or keys or two to a block, a group's heads in one workgroup or in several, a
tile's sequence found among few or many.  Each against the formulas in double precision, element by element, with the bounds of
tests/test_gpu_attention.py, whose cases these are."""
import math

import pytest
import torch

from tests import test_gpu_attention as one

pytestmark = pytest.mark.gpu
SPLITS = ("attention_forward_split", "attention_dq_split", "attention_dkv_split")


class forced:
    """All kernels with so many wavefronts to a block (1: four blocks a workgroup, 2: two), a group's heads in so many workgroups (0: choose)"""

    def __init__(self, capi, split=0, parts=0):
        self.capi, self.values = capi, {**{name: split for name in SPLITS}, "attention_group_parts": parts}

    def __enter__(self):
        for name, value in self.values.items():
            self.capi.set_tunable(name, value)

    def __exit__(self, *_):
        for name in self.values:
            self.capi.set_tunable(name, 0)


def given(case, dtype):
    D, heads, keyHeads, lengths, causal = one.CASES[case]
    return one.make(sum(a for a, _ in lengths), sum(b for _, b in lengths), heads, keyHeads, D, dtype, case) + (lengths, causal)


@pytest.mark.parametrize("dtype", one.TYPES)
@pytest.mark.parametrize("split", [1, 2])
@pytest.mark.parametrize("case", range(len(one.CASES)))
def test_blocks(capi, case, split, dtype):
    with forced(capi, split):
        one.check_all(capi, *given(case, dtype))


@pytest.mark.parametrize("dtype", one.TYPES)
@pytest.mark.parametrize("parts", [1, 2, 3, 33])
@pytest.mark.parametrize("case", [i for i, c in enumerate(one.CASES) if c[1] > c[2]])
def test_heads_of_a_group(capi, case, parts, dtype):
    for split in (1, 2):
        with forced(capi, split, parts):
            one.check_all(capi, *given(case, dtype))


@pytest.mark.parametrize("dtype", one.TYPES)
@pytest.mark.parametrize("split", [1, 2])
@pytest.mark.parametrize("n,m,sequences,causal", [(196, 196, 3, False), (300, 300, 2, True), (49, 500, 4, True), (130, 70, 1, True)])
def test_blocks_of_sequences_of_one_length(capi, n, m, sequences, causal, split, dtype):
    for D in (64, 96, 128):
        q, k, v, dy = one.make(n * sequences, m * sequences, 4, 2, D, dtype, n)
        with forced(capi, split):
            one.check_all(capi, q, k, v, dy, [(n, m)] * sequences, causal, ragged=False)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("count,longest,split,dtype", [(count, longest, split, dtype) for count, longest in ((64, 300), (65, 300), (130, 200), (700, 9))
                                                       for split in (0, 1, 2) for dtype in one.TYPES] + [(4200, 5, 0, torch.float32)])
def test_values_of_many_sequences(capi, count, longest, split, dtype, causal):
    """Up to 64 sequences, more, more than 64 x 64; empty ones, ones of several tiles and ones without queries or keys among them"""
    some = lambda i, k: (i * k * 7919 + k) % (longest + 1)
    lengths = [(some(i, 1), some(i, 1) if i % 3 else some(i, 5)) for i in range(count)]
    q, k, v, dy = one.make(sum(a for a, _ in lengths), sum(b for _, b in lengths), 2, 1, 32, dtype, count)
    with forced(capi, split):
        one.check_all(capi, q, k, v, dy, lengths, causal)


@pytest.mark.parametrize("dtype", one.TYPES)
@pytest.mark.parametrize("split", [0, 1, 2])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_is_not_seen_has_no_part(capi, bad, D, split, dtype):
    """Values, keys, queries and derivatives that are not finite, several and of single heads, around tiles' borders: rows and keys that see none of them are
    as they are without; also where some that are seen by nearly all are not finite either"""
    n, heads, keyHeads = 300, 6, 2
    q, k, v, dy = one.make(n, n, heads, keyHeads, D, dtype, 8)
    y, sums = capi.attention_forward(q, k, v, causal=True)
    w = one.Want(q, k, v, dy, [(n, n)], True)
    for at in ([1], [31, 32], [63, 200], [64, 65], [127, 255], [128, 130], [290, 299], [299]):
        with forced(capi, split):
            # values and keys of the second key head: its rows ahead of the first one
            h, free = slice(3, 6), slice(0, at[0])
            v2, k2 = v.clone(), k.clone()
            v2[at, 1, 5] = bad
            k2[at, 1, 3] = bad
            y2, _ = capi.attention_forward(q, k, v2, causal=True)
            one.near(y2[free, h], w.o[free, h], w.o_off[free, h], "o")
            one.near(y2[:, :3], w.o[:, :3], w.o_off[:, :3], "o of the other head")
            assert not bool(torch.isfinite(y2[at[0]:, h, 5]).any())
            y3, sums3 = capi.attention_forward(q, k2, v2, causal=True)
            one.near(y3[free, h], w.o[free, h], w.o_off[free, h], "o")
            dq, _, _ = capi.attention_backward(q, k2, v2, y3, sums3, dy, causal=True)
            one.near(dq[free, h], w.dq[free, h], w.dq_off[free, h], "dq")
            one.near(dq[:, :3], w.dq[:, :3], w.dq_off[:, :3], "dq of the other head")
            # queries and derivatives of one head of each group: keys behind the last one
            behind = slice(at[-1] + 1, n)
            q2, dy2 = q.clone(), dy.clone()
            q2[at, 1], dy2[at, 1, 7] = bad, bad
            q2[at[0], 5] = bad
            y4, sums4 = capi.attention_forward(q2, k, v, causal=True)
        for parts in (1, 3):
            with forced(capi, split, parts):
                _, dk, dv = capi.attention_backward(q2, k, v, y4, sums4, dy2, causal=True)
            if at[-1] + 1 < n:
                one.near(dk[behind, 0], w.dk[behind, 0], w.dk_off[behind, 0], "dk")
                one.near(dv[behind, 0], w.dv[behind, 0], w.dv_off[behind, 0], "dv")
            if at[0] + 1 < n:
                one.near(dk[at[0] + 1:, 1], w.dk[at[0] + 1:, 1], w.dk_off[at[0] + 1:, 1], "dk of the other head")
                one.near(dv[at[0] + 1:, 1], w.dv[at[0] + 1:, 1], w.dv_off[at[0] + 1:, 1], "dv of the other head")
            assert not bool(torch.isfinite(dv[:at[-1] + 1, 0, 7]).any())


@pytest.mark.parametrize("dtype", one.TYPES)
@pytest.mark.parametrize("n", [4, 40])
@pytest.mark.parametrize("bad", [math.nan, -math.inf])
def test_what_is_not_seen_of_keys_in_slices(capi, bad, n, dtype):
    """Few queries against many keys, which are cut into slices: the last keys are seen by the last queries alone"""
    m, heads, keyHeads, D = 3000, 4, 2, 128
    q, k, v, dy = one.make(n, m, heads, keyHeads, D, dtype, n)
    w = one.Want(q, k, v, dy, [(n, m)], True)
    for at in (m - 1, m - 3, m - n + 1):
        free = slice(0, at - (m - n))      # queries that do not see it
        for more in ([], [1000]):          # ... in the first key head; in the second one that all see as well
            v2, k2 = v.clone(), k.clone()
            v2[at, :, 9], k2[at, :, 9] = bad, bad
            v2[more, 1, 2] = bad
            y, sums = capi.attention_forward(q, k2, v2, causal=True)
            one.near(y[free, :2], w.o[free, :2], w.o_off[free, :2], "o")
            one.near(sums[free], w.sums[free], w.sums_off[free], "log sums")
            assert not bool(torch.isfinite(y[at - (m - n):, :, 9]).any())
            if more:
                assert not bool(torch.isfinite(y[:, 2:, 2]).any())
