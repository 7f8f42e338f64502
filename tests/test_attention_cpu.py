"""What the entry points for models with attention refuse, and what they ask for, without a GPU: every check stands before any launch, so addresses
that nothing reads do."""
import ctypes as C

import pytest

A = 1 << 20   # an address: nothing is read


def heads(capi, position=64, head=16, data=A):
    return C.byref(capi.Heads(data, position, head))


def hnorm(capi, **other):
    g = dict(D=16, heads=4, keyHeads=2, N=8, pairs=8, axes=2, neighbours=0, normalise=1, dataType=0, epsilon=1e-6)
    g.update(other)
    return capi.HnormGeom(*[g[n] for n, _ in capi.HnormGeom._fields_])


def attention(capi, **other):
    g = dict(D=16, heads=4, keyHeads=2, N=8, M=8, sequences=2, causal=1, clear=0, dataType=0, scale=0.0)
    g.update(other)
    return capi.AttentionGeom(*[g[n] for n, _ in capi.AttentionGeom._fields_])


def message(capi):
    return capi.lib().mcn_last_error_message().decode()


def test_heads_normalised_and_rotated(capi):
    L, bad, no = capi.lib(), capi.ILLEGAL_ARGUMENT, capi.UNSUPPORTED
    t = heads(capi)

    def forward(g, yq=t, yk=t, q=t, k=t, positions=A, frequencies=A):
        return L.mcn_hnorm_forward(None, C.byref(g), yq, yk, q, k, None, None, positions, frequencies)

    for other, code, text in [(dict(dataType=2), bad, "data type"), (dict(D=-1), bad, "negative"), (dict(D=513, pairs=0), no, "512"), (dict(pairs=9), bad, "pairs"),
                              (dict(axes=0), bad, "axes"), (dict(axes=65), no, "axes"), (dict(epsilon=-1.0), bad, "EPSILON"), (dict(epsilon=float("nan")), bad, "EPSILON"),
                              (dict(heads=65537), no, "65536")]:
        assert forward(hnorm(capi, **other)) == code and text in message(capi), (other, message(capi))
    g = hnorm(capi)
    for kw, text in [(dict(q=None), "null queries"), (dict(k=heads(capi, data=None)), "null keys"), (dict(yq=heads(capi, position=63)), "overlap"),
                     (dict(yk=heads(capi, head=0)), "overlap"), (dict(q=heads(capi, data=A + 2)), "aligned"), (dict(q=heads(capi, head=-16)), "negative stride"),
                     (dict(positions=None), "positions"), (dict(frequencies=None), "positions")]:
        assert forward(g, **kw) == bad and text in message(capi), (kw, message(capi))
    assert forward(hnorm(capi, N=0)) == 0 and forward(hnorm(capi, D=0, pairs=0)) == 0 and L.mcn_hnorm_forward(None, None, t, t, t, t, None, None, A, A) == bad

    def backward(g, dq=t, dgq=A, ws=A, n=1 << 30, dyq=t):
        return L.mcn_hnorm_backward(None, C.byref(g), dq, t, dgq, A, t, t, None, None, A, A, dyq, t, ws, n)

    need = L.mcn_hnorm_workspace_bytes(C.byref(g))
    assert need > 0 and need % (2 * 16 * 4) == 0 and L.mcn_hnorm_workspace_bytes(C.byref(hnorm(capi, normalise=0))) == 0
    for kw, text in [(dict(n=0), "too small"), (dict(ws=None), "too small"), (dict(ws=A + 8), "16-byte"), (dict(dyq=None), "null queries' derivative"),
                     (dict(dq=heads(capi, position=10)), "overlap")]:
        assert backward(g, **kw) == bad and text in message(capi), (kw, message(capi))
    assert backward(hnorm(capi, normalise=0)) == bad and "without the norm" in message(capi)


def test_attention(capi):
    L, bad, no = capi.lib(), capi.ILLEGAL_ARGUMENT, capi.UNSUPPORTED
    t, kt = heads(capi), heads(capi, position=32)

    def forward(g, o=t, q=t, k=kt, v=kt, qs=None, ks=None, ws=A, n=1 << 40):
        return L.mcn_attention_forward(None, C.byref(g), o, A, q, k, v, qs, ks, ws, n)

    for other, code, text in [(dict(dataType=7), bad, "data type"), (dict(N=-8), bad, "negative"), (dict(D=129), no, "128"), (dict(sequences=-1), bad, "sequences"),
                              (dict(keyHeads=3), bad, "key heads"), (dict(keyHeads=0), bad, "key heads"), (dict(scale=-1.0), bad, "scale"),
                              (dict(scale=float("inf")), bad, "scale"), (dict(scale=float("nan")), bad, "scale"), (dict(sequences=3), bad, "one length"),
                              (dict(N=1 << 30), no, "too many"), (dict(M=(1 << 31) - 1, sequences=1), no, "too many")]:
        assert forward(attention(capi, **other)) == code and text in message(capi), (other, message(capi))
    g = attention(capi)
    need = L.mcn_attention_workspace_bytes(C.byref(g), 0)
    for kw, text in [(dict(q=None), "null queries"), (dict(k=None), "null keys"), (dict(v=heads(capi, data=None)), "null values"), (dict(o=None), "null output"),
                     (dict(o=heads(capi, position=48)), "overlap"), (dict(o=heads(capi, head=8)), "overlap"), (dict(qs=A), "starts"), (dict(ks=A), "starts"),
                     (dict(n=need - 1), "too small"), (dict(ws=None), "too small"), (dict(ws=A + 4), "16-byte"), (dict(k=heads(capi, position=-32)), "negative stride"),
                     (dict(v=heads(capi, data=A + 1)), "aligned")]:
        assert forward(g, **kw) == bad and text in message(capi), (kw, message(capi))
    assert forward(attention(capi, N=0)) == 0 and forward(attention(capi, sequences=0)) == 0 and forward(attention(capi, heads=0, keyHeads=0)) == 0

    def backward(g, dq=t, dk=kt, o=t, sums=A, dy=t, n=1 << 40, ws=A):
        return L.mcn_attention_backward(None, C.byref(g), dq, dk, kt, o, sums, t, kt, kt, dy, None, None, ws, n)

    need = L.mcn_attention_workspace_bytes(C.byref(g), 1)
    for kw, text in [(dict(o=None), "null output"), (dict(dy=None), "output's derivative"), (dict(sums=None), "log sums"), (dict(n=need - 1), "too small"),
                     (dict(ws=A + 8), "16-byte"), (dict(dq=heads(capi, position=63)), "overlap"), (dict(dk=heads(capi, position=31)), "overlap")]:
        assert backward(g, **kw) == bad and text in message(capi), (kw, message(capi))
    # nothing asked for, nothing done
    assert L.mcn_attention_backward(None, C.byref(g), None, None, None, None, None, None, None, None, None, None, None, None, 0) == 0


def test_workspaces_grow_with_what_they_hold(capi):
    """A packed copy of every operand, statistics of every row and head, parts of cut reductions"""
    L = capi.lib()
    size = lambda back, **kw: L.mcn_attention_workspace_bytes(C.byref(attention(capi, **kw)), back)
    rows = dict(D=64, heads=8, keyHeads=2, N=4096, M=4096, sequences=1, dataType=1)
    packed = 4096 * 64 * 2
    assert size(0, **rows) >= packed * (8 + 2 + 2) and size(1, **rows) >= packed * (3 * 8 + 2 + 2) + 2 * 4096 * 8 * 4
    one = dict(D=128, heads=8, keyHeads=2, N=4, M=40000, sequences=4, dataType=1)
    assert size(0, **one) > 2 * 40000 * 2 * 128 * 2 + 2 * 4 * 8 * 129 * 4     # several slices
    assert L.mcn_attention_workspace_bytes(None, 0) == 0


def test_clipping(capi):
    L, bad = capi.lib(), capi.ILLEGAL_ARGUMENT
    n = 3
    counts, types = (C.c_size_t * n)(10, 0, 20000), (C.c_int * n)(0, 1, 1)
    ders, outs = (C.c_void_p * n)(A, None, A + 4096), (C.c_void_p * n)(A, None, A + 4096)
    need = L.mcn_clip_workspace_bytes(counts, n)
    assert need == 8 * (1 + 0 + 3) and L.mcn_clip_workspace_bytes(None, 3) == 0

    def clip(outs=outs, ders=ders, counts=counts, types=types, n=n, most=1.0, ws=A, size=1 << 20):
        return L.mcn_clip_gradients(None, outs, A, ders, counts, types, n, most, ws, size)

    for kw, text in [(dict(n=-1), "negative number"), (dict(ders=None), "null argument"), (dict(counts=None), "null argument"), (dict(types=(C.c_int * n)(0, 1, 2)), "data type"),
                     (dict(ders=(C.c_void_p * n)(None, None, A)), "tensor 0 is null"), (dict(ders=(C.c_void_p * n)(A + 2, None, A)), "not aligned"),
                     (dict(outs=None), "null argument"), (dict(outs=(C.c_void_p * n)(A, None, None)), "output 2"), (dict(outs=(C.c_void_p * n)(A, None, A + 1)), "not aligned"),
                     (dict(most=-1.0), "negative"), (dict(most=float("nan")), "negative"), (dict(size=need - 1), "too small"), (dict(ws=A + 8), "16-byte")]:
        assert clip(**kw) == bad and text in message(capi), (kw, message(capi))
    assert L.mcn_gradient_norm(None, None, ders, counts, types, n, A, 1 << 20) == bad and "null norm" in message(capi)
    assert L.mcn_clip_gradients(None, None, None, None, None, None, 0, 1.0, None, 0) == 0

    def step(value=A, most=1.0, ws=A, size=1 << 20):
        return L.mcn_sgd_momentum_clipped(None, value, A, A, 4, A, A, 0.1, 0.0, 0.9, 1.0, 0, most, None, ws, size)

    for kw, text in [(dict(value=None), "null argument"), (dict(value=A + 4), "16-byte"), (dict(most=-1.0), "negative"), (dict(size=8), "too small"), (dict(ws=None), "too small"),
                     (dict(ws=A + 4), "16-byte")]:
        assert step(**kw) == bad and text in message(capi), (kw, message(capi))


def test_lists_of_gradients_are_looked_over_without_a_device(capi):
    import torch
    with pytest.raises(ValueError):
        capi.GradientList([torch.zeros(4)])
    empty = capi.GradientList([])
    assert empty.n == 0 and empty.workspace_bytes == 0
