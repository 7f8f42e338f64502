"""Attention's limits, without a GPU: what is refused before any launch (addresses that nothing reads do)."""
import ctypes as C

import pytest

A = 1 << 20


def call(capi, backward=False, **other):
    g = dict(D=16, heads=1, keyHeads=1, N=8, M=8, sequences=2, causal=1, clear=0, dataType=0, scale=0.0)
    g.update(other)
    g = capi.AttentionGeom(*[g[n] for n, _ in capi.AttentionGeom._fields_])
    t = C.byref(capi.Heads(A, 128, 16))
    need = capi.lib().mcn_attention_workspace_bytes(C.byref(g), int(backward))
    if backward:
        rc = capi.lib().mcn_attention_backward(None, C.byref(g), t, t, t, t, A, t, t, t, t, A, A, A, need)
    else:
        rc = capi.lib().mcn_attention_forward(None, C.byref(g), t, A, t, t, t, A, A, A, need)
    return rc, capi.lib().mcn_last_error_message().decode()


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("scale", [1e-31, 1e-300, 1e31, 1e300])
def test_scale_that_single_precision_cannot_divide_by(capi, backward, scale):
    rc, text = call(capi, backward, scale=scale)
    assert rc == capi.UNSUPPORTED and "scale" in text


@pytest.mark.parametrize("backward,N,sequences", [(False, 8, 1 << 26), (False, 1 << 27, 1 << 20), (True, 8, 1 << 24), (True, 8, 1 << 28)])
def test_more_tiles_than_a_launch_has_threads(capi, backward, N, sequences):
    rc, text = call(capi, backward, N=N, M=N, sequences=sequences, heads=8, keyHeads=8)
    assert rc == capi.UNSUPPORTED and "too many tiles" in text
