"""Sizes of attention's workspaces for geometries that the calls refuse, and what they refuse, without a GPU."""
import ctypes as C

import pytest


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("heads,keyHeads", [(2, 4), (1, 1 << 20), (5, 2), (0, 4), (4, 0), (-1, 2)])
def test_heads_that_are_no_multiple_of_the_key_heads(capi, heads, keyHeads, backward):
    """No workspace, and no division by the heads of an empty group: the call behind it says what is wrong"""
    g = capi.AttentionGeom(16, heads, keyHeads, 8, 8, 1, 1, 0, 0, 0.0)
    assert capi.lib().mcn_attention_workspace_bytes(C.byref(g), backward) == 0


def test_heads_of_no_channels(capi):
    """There is no output to write; log sums, which would stay unwritten, are refused"""
    call = lambda N, heads, sums: capi.lib().mcn_attention_forward(None, C.byref(capi.AttentionGeom(0, heads, heads, N, N, 1, 0, 0, 0, 0.0)), None, sums, None, None,
                                                                  None, None, None, None, 0)
    assert call(8, 2, 1 << 20) == capi.ILLEGAL_ARGUMENT and "no channels" in capi.lib().mcn_last_error_message().decode()
    assert call(8, 2, None) == 0 and call(0, 2, 1 << 20) == 0 and call(8, 0, 1 << 20) == 0
