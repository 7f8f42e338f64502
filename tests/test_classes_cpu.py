"""Refusals of the operators for classifiers with many classes: layer normalisation, the fully connected loss, orthogonalised updates,
conversion.  All of it is decided on the host, before anything is launched."""
import ctypes as C

import pytest
import torch

from matconvnet_amd import capi

P = C.c_void_p(4096)   # stands for a device pointer: nothing is launched
BIG = 1 << 50


def refused(rc, code, text):
    assert rc == code, rc
    assert text in capi.lib().mcn_last_error_message().decode()


def lnorm_forward(**k):
    a = dict(type=0, y=P, mom=None, x=P, H=1, W=1, C=8, N=4, eps=1e-5, given=0)
    a.update(k)
    return capi.lib().mcn_lnorm_forward(None, a["type"], a["y"], a["mom"], a["x"], P, P, a["H"], a["W"], a["C"], a["N"], a["eps"], a["given"])


def lnorm_backward(**k):
    a = dict(type=0, dx=P, mom=None, x=P, dy=P, H=1, W=1, C=8, N=4, eps=1e-5, given=0, ws=P, bytes=BIG)
    a.update(k)
    return capi.lib().mcn_lnorm_backward(None, a["type"], a["dx"], P, P, a["mom"], a["x"], P, a["dy"], a["H"], a["W"], a["C"], a["N"], a["eps"], a["given"], a["ws"], a["bytes"])


@pytest.mark.parametrize("call", [lnorm_forward, lnorm_backward])
def test_lnorm(call):
    ill = capi.ILLEGAL_ARGUMENT
    refused(call(type=2), ill, "unknown data type")
    refused(call(H=-1), ill, "negative tensor extent")
    refused(call(eps=-1.0), ill, "EPSILON")
    refused(call(eps=float("nan")), ill, "EPSILON")
    refused(call(x=None), ill, "null tensor")
    refused(call(given=1), ill, "null moments")
    refused(call(H=1 << 16, W=1 << 16), capi.UNSUPPORTED, "too large")
    refused(call(C=(1 << 24) + 1), capi.UNSUPPORTED, "too large")
    assert call(C=0) == 0


def test_lnorm_of_its_own():
    ill = capi.ILLEGAL_ARGUMENT
    refused(lnorm_forward(y=None), ill, "null tensor")
    assert lnorm_forward(N=0) == 0
    refused(lnorm_backward(dy=None), ill, "null tensor")
    refused(lnorm_backward(ws=None), ill, "workspace too small")
    refused(lnorm_backward(bytes=16), ill, "workspace too small")
    assert capi.lib().mcn_lnorm_workspace_bytes(1, 1, 0, 4) == 0 and capi.lib().mcn_lnorm_workspace_bytes(1, 1, 100, 4) > 0


def fc(backward, **k):
    a = dict(D=16, K=10, N=4, type=0, y=P, x=P, f=P, c=P, labels=4, w=None, nw=0, ws=P, bytes=BIG)
    a.update(k)
    g = capi.FcLossGeom(a["D"], a["K"], a["N"], 1, a["type"])
    L = capi.lib()
    if backward:
        return L.mcn_fcloss_backward(None, C.byref(g), a["y"], P, P, None, a["x"], a["f"], None, a["c"], a["labels"], a["w"], a["nw"], 1.0, a["ws"], a["bytes"])
    return L.mcn_fcloss_forward(None, C.byref(g), a["y"], None, a["x"], a["f"], None, a["c"], a["labels"], a["w"], a["nw"], a["ws"], a["bytes"])


@pytest.mark.parametrize("backward", [0, 1])
def test_fcloss(backward):
    ill = capi.ILLEGAL_ARGUMENT
    refused(fc(backward, type=7), ill, "unknown data type")
    refused(fc(backward, D=-1), ill, "negative tensor extent")
    refused(fc(backward, labels=5), ill, "one label per image")
    refused(fc(backward, w=P, nw=3), ill, "cannot be broadcast")
    refused(fc(backward, w=P, nw=0), ill, "cannot be broadcast")
    refused(fc(backward, D=0), ill, "without features or classes")
    refused(fc(backward, K=0), ill, "without features or classes")
    refused(fc(backward, D=(1 << 20) + 1), capi.UNSUPPORTED, "2^20")
    refused(fc(backward, N=(1 << 30) + 1, labels=(1 << 30) + 1), capi.UNSUPPORTED, "2^30")
    refused(fc(backward, K=(1 << 24) + 1), capi.UNSUPPORTED, "2^24")
    for name in ("x", "f", "c"):
        refused(fc(backward, **{name: None}), ill, "null tensor")
    refused(fc(backward, ws=None), ill, "workspace too small")
    refused(fc(backward, bytes=1000), ill, "workspace too small")
    L = capi.lib()
    assert L.mcn_fcloss_workspace_bytes(None, backward) == 0
    small, large = capi.FcLossGeom(16, 10, 4, 1, 0), capi.FcLossGeom(64, 100000, 512, 1, 1)
    assert 0 < L.mcn_fcloss_workspace_bytes(C.byref(small), backward) < (1 << 20)
    # (a piece of the classes, not all of them: less than the 512 x 100000 scores in single precision)
    assert L.mcn_fcloss_workspace_bytes(C.byref(large), backward) < 512 * 100000 * 4


def test_fcloss_forward_needs_its_value():
    refused(fc(0, y=None), capi.ILLEGAL_ARGUMENT, "null output")


def ortho(**k):
    a = dict(y=P, x=P, K=8, D=20, count=1, steps=5, ws=P, bytes=BIG)
    a.update(k)
    return capi.lib().mcn_orthogonalise(None, a["y"], a["x"], a["K"], a["D"], a["count"], a["steps"], a["ws"], a["bytes"])


def test_orthogonalise():
    ill = capi.ILLEGAL_ARGUMENT
    refused(ortho(K=-1), ill, "negative tensor extent")
    refused(ortho(steps=-1), ill, "number of steps")
    refused(ortho(steps=101), ill, "number of steps")
    refused(ortho(x=None), ill, "null tensor")
    refused(ortho(y=None), ill, "null tensor")
    refused(ortho(ws=None), ill, "workspace too small")
    refused(ortho(bytes=100), ill, "workspace too small")
    refused(ortho(K=1 << 16, D=1 << 16), capi.UNSUPPORTED, "too large")
    refused(ortho(count=70000), capi.UNSUPPORTED, "too large")
    assert ortho(count=0) == 0 and ortho(D=0) == 0


def test_convert():
    L = capi.lib()
    refused(L.mcn_convert(None, P, 2, P, 0, 4), capi.ILLEGAL_ARGUMENT, "unknown data type")
    refused(L.mcn_convert(None, None, 1, P, 0, 4), capi.ILLEGAL_ARGUMENT, "null tensor")
    assert L.mcn_convert(None, None, 1, None, 0, 0) == 0


def test_binding_refuses_what_the_library_cannot_see():
    """Tensors on the host, of other types, strided or of other sizes are refused in Python."""
    import torch
    x = torch.zeros((2, 4, 1, 1))
    with pytest.raises(ValueError):
        capi.lnorm_forward(x, None, None)
    with pytest.raises(TypeError):
        capi.lnorm_forward(x, torch.zeros(4, dtype=torch.float64), None)
    with pytest.raises(ValueError):
        capi.fcloss_geom(torch.zeros((2, 4)), torch.zeros((3, 5)))
    with pytest.raises(TypeError):
        capi.fcloss_geom(torch.zeros((2, 4)), torch.zeros((3, 4), dtype=torch.bfloat16))
    with pytest.raises(TypeError):
        capi.data_type(torch.zeros(2, dtype=torch.float16))
    with pytest.raises(ValueError):
        capi.orthogonalise(x)
    with pytest.raises(TypeError):
        capi.orthogonalise(x.double())


def z(*mshape):
    """CPU float tensor standing for a MATLAB array of size mshape."""
    return torch.zeros(tuple(reversed(mshape)), dtype=torch.float32)


LNORM_ERRORS = [
    ((z(2, 3, 8, 4), z(8)), "The arguments are less than three."),
    ((z(2, 3, 8, 4), z(7), z(8)), "The MULTIPLIERS size does not match the DATA depth."),
    ((z(2, 3, 8, 4), z(8), z(9)), "The BIASES size does not match the DATA depth."),
    ((z(2, 3, 8, 4), z(8), z(8), z(2, 3, 8, 3)), "DATA and DEROUTPUT do not have the same size."),
    ((z(2, 3, 8, 4), z(8), z(8), "moments", z(8, 2)), "The MOMENTS size does not match the DATA pixels."),
    ((z(2, 3, 8, 4), z(8), z(8), "epsilon", [1.0, 2.0]), "EPSILON is not a plain scalar."),
    ((z(2, 3, 8, 4), z(8), z(8), "nosuchoption"), "Unknown option 'nosuchoption'."),
    ((z(2, 3, 8, 4), z(8).double(), z(8)), "DATA and MULTIPLIERS do not have compatible formats."),
    ((z(2, 3, 8, 4), z(8), z(8), "moments", z(2, 3, 4, 2)), "vl_nnlnorm: DATA is on the CPU; this library implements the GPU (HIP, gfx950) device only"),
]
FCLOSS_ERRORS = [
    ((z(2, 3, 8, 4), z(2, 3, 8, 10), z(10)), "There are less than four arguments."),
    ((z(2, 3, 8, 4), z(3, 2, 8, 10), z(10), z(4)), "The FILTERS are not of the size of X."),
    ((z(2, 3, 8, 4), z(2, 3, 8, 10), z(9), z(4)), "The number of elements of BIASES is not the same as the number of filters."),
    ((z(2, 3, 8, 4), z(2, 3, 8, 10), z(10), z(4), "logSums", z(4)), "LOGSUMS are taken with DZDY only."),
    ((z(2, 3, 8, 4), z(2, 3, 8, 10), z(10), z(4), 1.0, "logSums", z(5)), "The LOGSUMS size does not match the number of images."),
    ((z(2, 3, 8, 4), z(2, 3, 8, 10), z(10), z(4), [1.0, 2.0]), "DZDY is not a plain scalar."),
    ((z(2, 3, 8, 4), z(2, 3, 8, 10), z(10), z(4), "normalise", [1.0, 2.0]), "NORMALISE is not a plain scalar."),
    ((z(2, 3, 8, 4), z(2, 3, 8, 10), z(10), z(4), "topK", 2.0), "Unknown option 'topK'."),
    ((z(2, 3, 8, 4), z(2, 3, 8, 10).double(), z(10), z(4)), "X and FILTERS do not have compatible formats."),
    ((z(2, 3, 8, 4), z(2, 3, 8, 10), z(), z(4)), "vl_nnfcloss: X is on the CPU; this library implements the GPU (HIP, gfx950) device only"),
]


@pytest.mark.parametrize("function,args,message", [("vl_nnlnorm", *e) for e in LNORM_ERRORS] + [("vl_nnfcloss", *e) for e in FCLOSS_ERRORS])
def test_front_end(function, args, message):
    from matconvnet_amd import vlapi
    with pytest.raises(vlapi.VlError) as e:
        getattr(vlapi, function)(*args)
    assert e.value.message == message


def test_a_tensor_of_another_device(monkeypatch):
    class Fake:
        is_cuda, dtype = True, torch.float32
        is_contiguous = staticmethod(lambda: True)
        get_device = staticmethod(lambda: 1)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="x is on device 1"):
        capi._single("b x", None, Fake())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    capi._single("b x", None, Fake())


@pytest.mark.parametrize("function", ["vl_nnlnorm", "vl_nnfcloss", "vl_nnfcloss back"])
def test_front_end_workspaces_are_of_one_call(function):
    """Calls on two streams may share no memory: what a call keeps on the device comes from its allocator, as its outputs do.  (Addresses
    that stand for device pointers; the allocator hands out the workspace and then has no more, so nothing is launched.)"""
    from matconvnet_amd import vlapi
    fc = "fcloss" in function

    def array(*mshape):
        a = vlapi.Arg(kind=0, data=4096, device=1, dtype=1, ndims=len(mshape))
        for i, d in enumerate(mshape):
            a.dims[i] = d
        return a

    one = C.c_double(1.0)
    number = vlapi.Arg(kind=0, data=C.addressof(one), device=0, dtype=2, ndims=2)
    number.dims[0] = number.dims[1] = 1
    args = [array(2, 3, 8, 4), array(2, 3, 8, 10), array(10), array(4)] if fc else [array(2, 3, 8, 4), array(8), array(8), array(2, 3, 8, 4)]
    if function.endswith("back"):
        args.append(number)
    g = capi.FcLossGeom(48, 10, 4, 1, 0)
    need = capi.lib().mcn_fcloss_workspace_bytes(C.byref(g), int(len(args) == 5)) if fc else capi.lib().mcn_lnorm_workspace_bytes(2, 3, 8, 4)
    asked = []

    def alloc(user, device, nbytes):
        asked.append((device, nbytes))
        return 8192 if len(asked) == 1 else None

    rc = vlapi.lib().vlh_call(function.split()[0].encode(), 3, (vlapi.Arg * 4)(), len(args), (vlapi.Arg * len(args))(*args), vlapi.ALLOC_FN(alloc), None, None)
    assert rc != 0 and asked[0] == (1, need) and len(asked) == 2, asked
    assert vlapi.lib().vlh_last_message().decode() == "Could not allocate an output array."


@pytest.mark.parametrize("name,value,same", [("product_slices", 64, 32), ("product_slices", 1 << 30, 32), ("product_slices", -3, 0), ("product_tile", 100, 0), ("product_tile", -64, 0)])
def test_every_product_has_a_plan(name, value, same):
    """Cuts finer than are made, and tiles that there are not, are taken as the nearest that there is: the same plan, so the same workspace."""
    L = capi.lib()
    g = capi.FcLossGeom(8192, 1000, 300, 1, 1)   # (128 stages)

    def sizes(v):
        capi.set_tunable(name, v)
        return [L.mcn_fcloss_workspace_bytes(C.byref(g), b) for b in (0, 1)] + [L.mcn_orthogonalise_workspace_bytes(500, 9000, 2)]

    try:
        assert sizes(value) == sizes(same)
    finally:
        capi.set_tunable(name, 0)


def test_workspaces_are_aligned():
    off = lambda n: C.c_void_p(4096 + n)
    for n in (1, 4, 8):
        for backward in (0, 1):
            refused(fc(backward, ws=off(n)), capi.ILLEGAL_ARGUMENT, "not 16-byte aligned")
        refused(ortho(ws=off(n)), capi.ILLEGAL_ARGUMENT, "not 16-byte aligned")
    for n in (1, 2):
        refused(lnorm_backward(ws=off(n)), capi.ILLEGAL_ARGUMENT, "not 4-byte aligned")
