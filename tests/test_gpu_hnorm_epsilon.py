"""An epsilon of 0: heads that do not fill a wavefront's groups leave the multipliers' derivatives finite.  Tolerances: test_gpu_hnorm.py."""
import pytest
import torch

from test_gpu_hnorm import TYPES, check_all, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,heads,keyHeads,D,pairs", [(1, 1, 1, 64, 32), (5, 3, 1, 64, 32), (33, 5, 2, 128, 64), (7, 3, 2, 75, 24), (4, 3, 1, 512, 256), (9, 1, 1, 1, 0)])
def test_no_epsilon(capi, N, heads, keyHeads, D, pairs, dtype):
    q, k, gq, gk, dyq, dyk, positions, frequencies = make(N, heads, keyHeads, D, pairs, 1, dtype, 3)
    check_all(capi, q, k, gq, gk, dyq, dyk, positions, frequencies, eps=0.0)
