"""What vl_nnhnorm and vl_nnattention refuse, without a GPU: every check stands before any launch."""
import pytest
import torch


def z(*mshape):
    return torch.zeros(tuple(reversed(mshape)))


Q, K = z(16, 4, 5, 2), z(16, 2, 7, 2)
NO = z(0, 0)
HNORM = [
    ((Q, Q, NO), "There are less than four arguments."),
    ((NO, NO, NO, NO), "Q and K are both empty."),
    ((Q, K, NO, NO), "Q and K do not have the same channels, positions and sequences."),
    ((Q, z(8, 2, 5, 2), NO, NO), "Q and K do not have the same channels, positions and sequences."),
    ((Q, Q, z(15), NO), "GQ does not have one value per channel of Q."),
    ((Q, NO, NO, z(16)), "GK does not have one value per channel of K."),
    ((Q, NO, z(16), NO, "normalise", 0.0), "GQ is taken with NORMALISE only."),
    ((Q, Q, NO, NO, Q), "DZDQ is given without DZDK."),
    ((Q, Q, NO, NO, Q, "epsilon", 0.1), "DZDQ is given without DZDK."),
    ((Q, Q, NO, NO, z(16, 4, 4, 2), Q), "Q and DZDQ do not have the same size."),
    ((Q, Q, NO, NO, Q, NO), "K and DZDK do not have the same size."),
    ((Q, Q, NO, NO, "epsilon", [1.0, 2.0]), "EPSILON is not a plain scalar."),
    ((Q, Q, NO, NO, "axes", 2.0), "Unknown option 'axes'."),
    ((Q, Q, NO, NO), "vl_nnhnorm: Q is on the CPU; this library implements the GPU (HIP, gfx950) device only"),
]
ATTENTION = [
    ((Q, K), "There are less than three arguments."),
    ((Q, K, z(16, 2, 6, 2)), "K and V do not have the same size."),
    ((z(8, 4, 5, 2), K, K), "Q and K do not have the same channels and sequences."),
    ((z(16, 4, 5, 3), K, K), "Q and K do not have the same channels and sequences."),
    ((Q, K.double(), K.double()), "Q, K and V do not have compatible formats."),
    ((Q, K, K, z(16, 4, 4, 2)), "Q and DZDY do not have the same size."),
    ((Q, K, K, Q, "output", Q), "OUTPUT and LOGSUMS are taken together."),
    ((Q, K, K, "output", Q, "logSums", z(4, 5, 2)), "OUTPUT and LOGSUMS are taken with DZDY only."),
    ((Q, K, K, Q, "output", z(16, 4, 4, 2), "logSums", z(4, 5, 2)), "Q and OUTPUT do not have the same size."),
    ((Q, K, K, Q, "output", Q, "logSums", z(4, 4, 2)), "LOGSUMS do not have one value per head and position of Q."),
    ((Q, K, K, "causal", [1.0, 2.0]), "CAUSAL is not a plain scalar."),
    ((Q, K, K, "mask", 1.0), "Unknown option 'mask'."),
    ((Q, K, K), "vl_nnattention: Q is on the CPU; this library implements the GPU (HIP, gfx950) device only"),
]


@pytest.mark.parametrize("function,args,message", [("vl_nnhnorm", *e) for e in HNORM] + [("vl_nnattention", *e) for e in ATTENTION])
def test_refusals(function, args, message):
    from matconvnet_amd import vlapi
    with pytest.raises(vlapi.VlError) as e:
        getattr(vlapi, function)(*args)
    assert e.value.message == message
