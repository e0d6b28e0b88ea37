"""Argument checks of the layer operators' C entries and Python surface that are
made on the host, before anything reaches a device (no GPU needed)."""
import ctypes
import struct

import pytest
import torch

import jlust_amd as J
from jlust_amd import _lib, layers
from jlust_amd.elementwise import FN_EXP, FN_GELU
from tests import _layer_cases as C


def linear(**kw):
    f = dict(value_type=1, act=0, w_layout=0, reserved=0, out=4, inp=3, cols=2, W=64, ldw=4, X=64, ldx=3, Y=64, ldy=4,
             bias=0, R=0, ldr=0, Z=0, ldz=0, groups=0, copies=1, plan=0, w_stride=0, bias_stride=0)
    assert set(kw) <= set(f)
    f.update(kw)
    return _lib.lib().jlust_hip_linear(layers._LINEAR(*f.values()), 0)


def grad(**kw):
    f = dict(value_type=1, act=0, w_layout=0, reserved=0, out=4, inp=3, cols=2, W=64, ldw=4, X=64, ldx=3, dY=64, lddy=4, Z=0,
             ldz=0, dX=64, lddx=3, dW=0, lddw=0, dbias=0, groups=0, copies=1, plan=0, w_stride=0, dw_stride=0, dbias_stride=0)
    assert set(kw) <= set(f)
    f.update(kw)
    return _lib.lib().jlust_hip_linear_grad(layers._LINEAR_GRAD(*f.values()), 0)


def test_packed_arguments_match_the_header():
    """The packed bytes are as long as the header's structures."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "jlust_hip.h")).read()
    for name, pack in (("jlust_linear", "@4i19q"), ("jlust_linear_grad", "@4i22q")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        words = sum(len(d.split(",")) * (4 if "int32_t" in d and "*" not in d else 8) for d in body.split(";") if d.strip())
        assert words == struct.calcsize(pack)


@pytest.mark.parametrize("bad,status", [
    (dict(value_type=4), 2), (dict(value_type=-1), 2), (dict(act=FN_EXP), 1), (dict(w_layout=2), 1), (dict(out=-1), 1),
    (dict(cols=1 << 31), 1), (dict(ldw=3), 1), (dict(ldx=2), 1), (dict(ldy=3), 1), (dict(W=0), 1), (dict(X=0), 1), (dict(Y=0), 1),
    (dict(R=64, ldr=3), 1), (dict(Z=64, ldz=1), 1), (dict(groups=2), 1), (dict(groups=5000, plan=64), 1), (dict(copies=2), 1),
    (dict(groups=2, plan=64, copies=3), 1)])
def test_linear_refuses(bad, status):
    assert linear(**bad) == status
    assert _lib.last_error()


@pytest.mark.parametrize("bad,status", [
    (dict(value_type=9), 2), (dict(act=FN_GELU), 1), (dict(dY=0), 1), (dict(lddx=2), 1), (dict(dW=64, lddw=1), 1), (dict(W=0), 1),
    (dict(dW=64, lddw=4, X=0), 1), (dict(groups=1), 1)])
def test_linear_grad_refuses(bad, status):
    assert grad(**bad) == status


@pytest.mark.parametrize("only", [dict(dX=0, dW=64, W=64, ldw=64, lddw=128, dbias=64),      # W 64 x 128 beside dW's transpose
                                  dict(dX=0, dW=64, W=0, ldw=0, lddw=128),
                                  dict(dX=64, lddx=128, dW=0, ldw=128, X=64, ldx=1),
                                  dict(dX=0, dW=0, ldw=0, ldx=0, dbias=64)])
def test_linear_grad_checks_what_it_reads(only):
    """W is read for dX alone and X for dW alone; the null dY is what is refused."""
    assert grad(out=64, inp=128, w_layout=1, **{**dict(lddy=64, ldx=128), **only}, dY=0) == 1
    assert "dY is null" in _lib.last_error()


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("rows,cols,ld,stride", [(4, 6, 4, 24), (4, 6, 4, 26), (4, 6, 12, 4), (4, 6, 5, 24), (4, 6, 5, 29), (4, 6, 5, 28),
                                                 (4, 6, 11, 4), (4, 6, 12, 3), (4, 6, 4, 0), (4, 6, 4, -24), (4, 6, 4, -23),
                                                 (4, 1, 4, 4), (4, 1, 4, 3), (1, 6, 3, 1), (1, 6, 2, 1)])
def test_groups_of_a_gradient_do_not_overlap(layout, rows, cols, ld, stride):
    """dW of three groups: refused just where two of them hold the same element, the
    null dY being what is refused otherwise."""
    at = [g * stride + j * ld + i for g in range(3) for j in range(cols) for i in range(rows)]
    out, inp = (rows, cols) if layout == 0 else (cols, rows)
    st = grad(out=out, inp=inp, cols=6, w_layout=layout, dX=0, dW=1 << 20, lddw=ld, dw_stride=stride, ldx=inp, lddy=out, groups=3,
              plan=64, dY=0)
    assert st == (4 if len(set(at)) < len(at) else 1)
    assert ("overlap" if st == 4 else "dY is null") in _lib.last_error()


def test_group_plan_and_layer_norm_refuse():
    L, n = _lib.lib(), ctypes.c_int64()
    assert L.jlust_hip_group_plan_ints(10, 3, 1, ctypes.byref(n)) == 0 and n.value == 14
    assert L.jlust_hip_group_plan_ints(10, 3, 2, ctypes.byref(n)) == 0 and n.value == 24
    for bad in ((-1, 3, 1), (10, 0, 1), (10, 4096, 1), (10, 3, 3), (10, 3, 0), (1 << 31, 3, 1)):
        assert L.jlust_hip_group_plan_ints(*bad, ctypes.byref(n)) == 1, bad
    assert L.jlust_hip_group_plan_build(4, 2, 1, 2, 64, 0, 64, 0) == 5          # the origin
    assert L.jlust_hip_group_plan_build(4, 2, 1, 1, 0, 0, 64, 0) == 1
    norm = lambda vt=1, d=8, cols=2, X=64, ldx=8, eps=1e-5, Y=64, ldy=8, S=0, lds=2: L.jlust_hip_layer_norm(  # noqa: E731
        vt, d, cols, X, ldx, 0, 0, eps, Y, ldy, S, lds, 0)
    assert norm(vt=7) == 2
    for bad in (dict(d=-1), dict(X=0), dict(Y=0), dict(ldx=7), dict(ldy=1), dict(eps=-1.0), dict(eps=float("nan")),
                dict(S=64, lds=1)):
        assert norm(**bad) == 1, bad
    assert L.jlust_hip_layer_norm_grad(1, 8, 2, 64, 8, 64, 8, 0, 2, 0, 64, 8, 0, 0, 0) == 1      # no stats


def test_host_memory_is_refused():
    x = torch.zeros((4, 3)).t()
    with pytest.raises(J.DeviceMismatch):
        J.execute(J.LinearOp, torch.zeros((3, 5)).t(), x, torch.zeros((4, 5)).t())
    with pytest.raises(J.DeviceMismatch):
        J.execute(J.LayerNormOp, x, x)
    with pytest.raises(J.DeviceMismatch):
        J.prepare(J.HIPBackend(), J.GroupedLinearOp, torch.ones(4, dtype=torch.int32), n_groups=2)
    with pytest.raises(TypeError):
        J.prepare(J.HIPBackend(), J.GroupedLinearOp, torch.ones(4, dtype=torch.int32))
    with pytest.raises(J.UnsupportedFormat):
        J.execute(J.LinearOp, x, x, x, backend=object())


def test_capability_table():
    dense = J.Formats.DensedRight(2)
    assert J.supports_backend(J.HIPBackend(), J.LinearOp(dense, dense, dense))
    assert not J.supports_backend(J.HIPBackend(), J.LinearOp(J.Formats.CSR, dense, dense))


def test_planned_products():
    """The kernels that tests/_layer_cases.py says its cases reach."""
    for *args, forward, dX, dW in C.PLANNED:
        f, g = C.arguments(*args)
        assert C.info(f)[:5] == forward, args
        assert tuple(i[:5] for i in C.info(g, True)) == (dX, dW), args
    kinds = {(c[0] if c[0] == "f32" else "half", i, c[4] == ("inp" if i == 0 else "out") if i < 2 else None, c[8 + i][:3])
             for c in C.PLANNED for i in range(3)}
    for kc in (True, False):                       # every tile by copies, in each direction
        for tile in ((256, 256, 1), (256, 128, 1), (128, 128, 1)):
            assert any(k[0] == "half" and k[1] < 2 and k[2] == kc and k[3] == tile for k in kinds), (kc, tile)
        assert any(k[0] == "f32" and k[1] < 2 and k[2] == kc and k[3] == (128, 128, 1) for k in kinds)
    for want in (("half", (256, 128, 1)), ("half", (128, 128, 1)), ("half", (128, 128, 0)), ("f32", (128, 128, 1)), ("f32", (128, 128, 0))):
        assert (want[0], 2, None, want[1]) in kinds, want


@pytest.mark.parametrize("T", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["out", "inp"])
def test_a_shared_matrix_is_packed_once(T, layout):
    """tests/test_gpu_layers_edges.py's groups that share a matrix: W is packed in both
    directions, shared or not, and takes one matrix's scratch where it is."""
    size = 4 if T == "f32" else 2
    scratch = []
    for shared in (True, False):
        f, g = (bytearray(b) for b in C.arguments(T, 1000, 1024, 16384, layout, 3, 0, None))
        a, b = (1000, 1024) if layout == "out" else (1024, 1000)
        for buf in (f, g):
            struct.pack_into("@q", buf, 16 + 8 * 4, a + 1)                              # ldw
            struct.pack_into("@q", buf, len(buf) - (16 if buf is f else 24), 0 if shared else (a + 1) * b)
        (dX, _), Y = C.info(bytes(g), True), C.info(bytes(f))
        assert Y[4] == 1 and dX[4] == 5
        scratch.append((Y[5], dX[5]))
    a, b = (1000, 1024) if layout == "out" else (1024, 1000)
    ld = (a * size + 15) // 16 * 16
    extra = lambda v: (v + 255) // 256 * 256  # noqa: E731
    assert all(apart - shared == extra(3 * ld * b) - extra(ld * b) for shared, apart in zip(*scratch))


def test_a_product_that_one_launch_does_not_take():
    """2^31 - 1 columns of 64 Float32 sums are 2^25 tiles; the gradient is refused too,
    before anything of it runs.  What few columns' tiles would pass takes wider ones."""
    n = (1 << 31) - 1
    big = dict(T="f32", out=64, inp=4, cols=n, layout="out", groups=0, pad=0, act=None)
    f, _ = C.arguments(**big)
    assert _lib.lib().jlust_hip_linear_info(f, (ctypes.c_int64 * 6)()) == 1 and "one launch" in _lib.last_error()
    _, g = C.arguments(**{**big, "inp": 64, "out": 4})
    assert _lib.lib().jlust_hip_linear_grad_info(g, (ctypes.c_int64 * 12)()) == 1 and "one launch" in _lib.last_error()
    few = dict(T="bf16", out=1 << 20, inp=64, cols=4000, layout="inp", pad=0, act=None)
    assert C.info(C.arguments(**few, groups=300)[0])[:2] == (128, 16)
    assert C.info(C.arguments(**{**few, "out": 1 << 16}, groups=300)[0])[:2] == (16, 16)


def test_info_of_nothing():
    f, g = C.arguments("bf16", 0, 5, 3, "out", 0, 0, None)
    assert C.info(f) == (0,) * 6 and C.info(g, True) == ((0,) * 6,) * 2
    assert _lib.lib().jlust_hip_linear_info(f, None) == 1 and _lib.lib().jlust_hip_linear_grad_info(None, (ctypes.c_int64 * 12)()) == 1
