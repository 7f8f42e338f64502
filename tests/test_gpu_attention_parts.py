"""Derivatives of attention one by one: what is not asked for has no part in the others, whatever the workspace holds."""
import itertools
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


class Filled:
    """A workspace whose memory holds `value` ahead of every call"""

    def __init__(self, value):
        self.value = value

    def get(self, nbytes):
        self.room = torch.full(((int(nbytes) + 3) // 4 + 4,), self.value, device="cuda")
        return self.room.data_ptr(), int(nbytes)


def make(n, heads, keyHeads, D, dtype, seed):
    r = torch.Generator(device="cuda")
    r.manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=r, device="cuda")
    return [normal(n, h, D).to(dtype) for h in (heads, keyHeads, keyHeads, heads)]


def same(a, b):
    """The same bits (of a NaN: that it is one)"""
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", [math.nan, math.inf, 3e38])
@pytest.mark.parametrize("causal", [True, False])
def test_each_alone_in_a_workspace_of_anything(capi, causal, value, dtype):
    """The bits of the call that makes all three; with a query behind the last keys that is not finite as well, which those keys do not see"""
    n = 200
    for D, heads, keyHeads, bad in ((128, 4, 2, False), (64, 2, 2, False), (128, 4, 1, True), (75, 2, 1, True)):
        q, k, v, dy = make(n, heads, keyHeads, D, dtype, D)
        if bad:
            dy[150, :, 3] = math.inf
        how = dict(causal=causal)
        y, sums = capi.attention_forward(q, k, v, **how)
        full = capi.attention_backward(q, k, v, y, sums, dy, **how)
        for want in itertools.product([True, False], repeat=3):
            got = capi.attention_backward(q, k, v, y, sums, dy, want=want, ws=Filled(value), **how)
            for name, g, f in zip(("dq", "dk", "dv"), got, full):
                assert g is None or same(g, f), (D, heads, keyHeads, bad, want, name)
        if bad and causal:
            assert bool(torch.isfinite(full[2][151:]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_keys_that_no_head_asks_for(capi, dtype):
    """No query heads: the derivatives of keys and values are zero, of the sequences' rows or with fresh outputs of all"""
    M, keyHeads, D = 50, 3, 24
    q = torch.zeros(40, 0, D, dtype=dtype, device="cuda")
    k, v = [torch.randn(M, keyHeads, D, device="cuda").to(dtype) for _ in range(2)]
    qs, ks = torch.tensor([3, 10, 30], dtype=torch.int32, device="cuda"), torch.tensor([5, 20, 41], dtype=torch.int32, device="cuda")
    for how in (dict(), dict(sequences=2), dict(q_starts=qs, k_starts=ks)):
        y, sums = capi.attention_forward(q, k, v, **how)
        assert y.shape == q.shape and sums.numel() == 0
        for out in (None, [torch.empty_like(q)] + [torch.full_like(t, 7.0) for t in (k, v)]):
            if out is None:     # (what a fresh tensor is made in holds something)
                rooms = [torch.full_like(t, 9.0) for t in (k, v)]
                del rooms
            dq, dk, dv = capi.attention_backward(q, k, v, y, sums, torch.empty_like(q), out=out, **how)
            assert dq.shape == q.shape
            for t in (dk, dv):
                inside = torch.ones(M, dtype=torch.bool, device="cuda")
                if "q_starts" in how and out is not None:
                    inside[:5] = inside[41:] = False
                assert bool((t[inside] == 0).all()) and bool((t[~inside] == 7.0).all())
        _, dk, none = capi.attention_backward(q, k, v, y, sums, torch.empty_like(q), want=(False, True, False), **how)
        assert none is None and bool((dk == 0).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_some_outputs_of_the_callers_and_some_fresh(capi, dtype):
    """Rows of no sequence: left alone in the caller's tensors, zero in fresh ones beside them"""
    q, k, v, dy = make(60, 4, 2, 32, dtype, 1)
    s = torch.tensor([7, 20, 45], dtype=torch.int32, device="cuda")
    how = dict(q_starts=s, k_starts=s, causal=True)
    y, sums = capi.attention_forward(q, k, v, **how)
    full = capi.attention_backward(q, k, v, y, sums, dy, **how)
    inside = torch.zeros(60, dtype=torch.bool, device="cuda")
    inside[7:45] = True
    for given in itertools.product([True, False], repeat=3):
        rooms = [torch.full_like(t, 9.0) for t in (q, k, v)]     # (so that the memory which fresh ones get holds something)
        del rooms
        out = [torch.full_like(t, 7.0) if w else None for w, t in zip(given, (q, k, v))]
        got = capi.attention_backward(q, k, v, y, sums, dy, out=out, **how)
        for mine, g, o, f in zip(given, got, out, full):
            assert (g is o) == mine and torch.equal(g[inside], f[inside]) and bool((g[~inside] == (7.0 if mine else 0.0)).all())
    only = capi.attention_backward(q, k, v, y, sums, dy, want=(False, True, False), out=[None, None, None], **how)
    assert only[0] is None and only[2] is None and torch.equal(only[1], full[1])
