"""Argument checks of routing, sums of experts, dropout and the 8-bit products that
are made on the host, and the plain forms that their GPU tests go by (no GPU needed)."""
import ctypes
import os
import re
import struct

import numpy as np
import pytest
import torch

import jlust_amd as J
from jlust_amd import _lib, experts, layers
from jlust_amd.elementwise import FN_EXP
from tests import _experts as E

INF, NAN = float("inf"), float("nan")


def call(entry, pack, fields, kw):
    f = dict(fields)
    assert set(kw) <= set(f)
    f.update(kw)
    return getattr(_lib.lib(), entry)(pack(*f.values()), 0)


def route(**kw):
    return call("jlust_hip_route", experts._ROUTE, dict(
        value_type=1, score=0, renormalize=1, origin=1, experts=8, cols=3, copies=2, groups=1, keep=1, best=2, L=64, ldl=8, bias=0,
        ids=64, ldi=2, weights=64, ldw=2, scale=1.0), kw)


def route_grad(**kw):
    return call("jlust_hip_route_grad", experts._ROUTE_GRAD, dict(
        value_type=1, score=0, renormalize=1, origin=1, experts=8, cols=3, copies=2, L=64, ldl=8, ids=64, ldi=2, dweights=64, lddw=2,
        dL=64, lddl=8, scale=1.0), kw)


def int8(**kw):
    return call("jlust_hip_linear_int8", layers._LINEAR_INT8, dict(
        value_type=1, act=0, out=4, inp=3, cols=2, W=64, ldw=3, w_scale=64, X=64, ldx=3, x_scale=64, Y=64, ldy=4, bias=0, R=0, ldr=0, Z=0,
        ldz=0, groups=0, copies=1, plan=0, w_stride=0, w_scale_stride=0, bias_stride=0), kw)


def test_packed_arguments_match_the_header():
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "jlust_hip.h")).read()
    for name, pack in (("jlust_linear_int8", "@2i22q"), ("jlust_route", "@4i13qd"), ("jlust_route_grad", "@4i11qd")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
        words = sum(len(d.split(",")) * (4 if "int32_t" in d and "*" not in d else 8) for d in body.split(";") if d.strip())
        assert words == struct.calcsize(pack)


@pytest.mark.parametrize("bad,status", [
    (dict(value_type=4), 2), (dict(value_type=-1), 2), (dict(score=2), 1), (dict(origin=2), 5), (dict(experts=0), 1), (dict(experts=-1), 1),
    (dict(experts=4096, ldl=4096), 1), (dict(copies=0), 1), (dict(copies=9), 1), (dict(experts=100, ldl=100, copies=65), 1), (dict(cols=-1), 1),
    (dict(cols=1 << 31), 1), (dict(groups=3), 1), (dict(groups=0), 1), (dict(groups=4, keep=5), 1), (dict(groups=4, keep=0), 1),
    (dict(groups=8, keep=1), 1), (dict(experts=130, ldl=130, groups=65, keep=2), 1), (dict(best=3), 1), (dict(best=0), 1),
    (dict(scale=INF), 1), (dict(scale=NAN), 1), (dict(L=0), 1), (dict(ids=0), 1), (dict(weights=0), 1), (dict(ldl=7), 1), (dict(ldi=1), 1),
    (dict(ldw=1), 1)])
def test_route_refuses(bad, status):
    assert route(**bad) == status
    assert _lib.last_error()


@pytest.mark.parametrize("bad,status", [
    (dict(value_type=7), 2), (dict(score=-1), 1), (dict(origin=-1), 5), (dict(copies=9), 1), (dict(experts=4096, ldl=4096), 1), (dict(L=0), 1),
    (dict(ids=0), 1), (dict(dweights=0), 1), (dict(dL=0), 1), (dict(lddl=7), 1), (dict(scale=NAN), 1)])
def test_route_grad_refuses(bad, status):
    assert route_grad(**bad) == status


@pytest.mark.parametrize("bad,status", [
    (dict(value_type=0), 2), (dict(value_type=4), 2), (dict(act=FN_EXP), 1), (dict(out=-1), 1), (dict(cols=1 << 31), 1),
    (dict(inp=1 << 17, ldw=1 << 17, ldx=1 << 17), 1), (dict(ldw=2), 1), (dict(ldx=2), 1), (dict(ldy=3), 1), (dict(W=0), 1), (dict(X=0), 1),
    (dict(Y=0), 1), (dict(w_scale=0), 1), (dict(x_scale=0), 1), (dict(R=64, ldr=3), 1), (dict(Z=64, ldz=1), 1), (dict(groups=2), 1),
    (dict(copies=2), 1), (dict(groups=5000, plan=64), 1), (dict(groups=2, plan=64, copies=3), 1)])
def test_linear_int8_refuses(bad, status):
    assert int8(**bad) == status
    assert _lib.last_error()


def test_int8_sums_that_fit():
    """Up to 131,071 products of a sum, which is where 32 bits end."""
    n = (1 << 17) - 1
    assert 128 * 128 * n < 2 ** 31 <= 128 * 128 * (n + 1)
    info = (ctypes.c_int64 * 6)()
    args = lambda inp: layers._LINEAR_INT8(1, 0, 4, inp, 2, 64, inp, 64, 64, inp, 64, 64, 4, 0, 0, 0, 0, 0, 0, 1, 0, 0, 0, 0)  # noqa: E731
    assert _lib.lib().jlust_hip_linear_int8_info(args(n), info) == 0
    assert _lib.lib().jlust_hip_linear_int8_info(args(n + 1), info) == 1
    assert _lib.lib().jlust_hip_linear_int8_info(args(n), None) == 1 and _lib.lib().jlust_hip_linear_int8_info(None, info) == 1


def test_planned_products():
    """The kernels that tests/_experts.py says its products reach."""
    for T, out, inp, cols, groups, copies, plan in E.PLANNED8:
        info, p = (ctypes.c_int64 * 6)(), 1 << 20
        args = layers._LINEAR_INT8({"f32": 1, "f16": 2, "bf16": 3}[T], 0, out, inp, cols * copies, p, inp, p, p, inp, p, p, out, 0, 0, 0, 0,
                                   0, groups, copies, p if groups else 0, inp * out, out, out)
        assert _lib.lib().jlust_hip_linear_int8_info(args, info) == 0
        assert tuple(info[:4]) == plan, (out, inp, cols, groups, copies)
    forms = {c[6][:3] for c in E.PLANNED8}
    assert forms == {(16, 16, 0), (64, 64, 0), (128, 32, 0), (128, 128, 1), (256, 128, 1), (256, 256, 1)}


def test_packed_products():
    """What tests/_experts.py says is packed, and the scratch it takes."""
    for T, out, inp, cols, groups, copies, woff, xoff, shared, plan in E.PACKED8:
        info, p = (ctypes.c_int64 * 6)(), 1 << 20
        args = layers._LINEAR_INT8({"f32": 1, "f16": 2, "bf16": 3}[T], 0, out, inp, cols * copies, p + woff, inp, p, p + xoff, inp, p, p,
                                   out, 0, 0, 0, 0, 0, groups, copies, p if groups else 0, 0 if shared else inp * out, out, out)
        assert _lib.lib().jlust_hip_linear_int8_info(args, info) == 0
        assert (info[0], info[1], info[4]) == plan and info[2] == 1, (out, inp, cols, tuple(info))
        ld = (inp + 15) // 16 * 16
        most = (plan[2] & 1) * ld * out * (1 if shared else max(groups, 1)) + (plan[2] >> 1) * ld * cols
        assert most <= info[5] < most + 512


def test_combine_dropout_and_quantize_refuse():
    lib = _lib.lib()

    def combine(vt=1, d=4, cols=3, copies=2, X=64, ldx=4, w=64, ldw=2, R=0, ldr=0, Y=64, ldy=4):
        return lib.jlust_hip_combine(vt, d, cols, copies, X, ldx, w, ldw, R, ldr, Y, ldy, 0)

    def combine_grad(vt=1, d=4, cols=3, copies=2, X=64, ldx=4, w=64, ldw=2, dY=64, lddy=4, dX=64, lddx=4, dw=64, lddw=2):
        return lib.jlust_hip_combine_grad(vt, d, cols, copies, X, ldx, w, ldw, dY, lddy, dX, lddx, dw, lddw, 0)

    def dropout(vt=1, d=4, cols=3, X=64, ldx=4, R=0, ldr=0, Y=64, ldy=4, p=0.5):
        return lib.jlust_hip_dropout(vt, d, cols, X, ldx, R, ldr, Y, ldy, p, 1, 2, 0, 0)

    def quantize(vt=1, d=4, cols=3, X=64, ldx=4, Q=64, ldq=4, s=64):
        return lib.jlust_hip_quantize_columns(vt, d, cols, X, ldx, Q, ldq, s, 0)

    for f, bad in ((combine, (dict(d=-1), dict(cols=-1), dict(copies=0), dict(copies=1 << 31), dict(cols=1 << 30, copies=2), dict(X=0),
                              dict(w=0), dict(Y=0), dict(ldx=3), dict(ldw=1), dict(ldy=3), dict(R=64, ldr=3))),
                   (combine_grad, (dict(d=-1), dict(copies=-1), dict(X=0), dict(w=0), dict(dY=0), dict(ldx=3), dict(ldw=1), dict(lddy=3),
                                   dict(lddx=3), dict(lddw=1))),
                   (dropout, (dict(d=1 << 31), dict(cols=-1), dict(X=0), dict(Y=0), dict(ldx=3), dict(ldy=3), dict(R=64, ldr=3), dict(p=-0.1),
                              dict(p=1.1), dict(p=NAN))),
                   (quantize, (dict(d=-1), dict(cols=1 << 31), dict(X=0), dict(Q=0), dict(s=0), dict(ldx=3), dict(ldq=3)))):
        assert f(vt=5) == 2
        for kw in bad:
            assert f(**kw) == 1, (f.__name__, kw)
            assert _lib.last_error()
    assert quantize(vt=0) == 2


def test_python_refusals():
    m = lambda r, c, T=torch.float32: torch.zeros((c, r), dtype=T).t()  # noqa: E731
    HIP = J.HIPBackend()
    for bad in (lambda: J.execute(J.RouteOp, m(8, 3), m(2, 3, torch.int32), m(2, 3)),
                lambda: J.execute(J.CombineOp, m(4, 6), m(2, 3), m(4, 3)),
                lambda: J.execute(J.DropoutOp, m(4, 3), m(4, 3), seed=1),
                lambda: J.execute(J.QuantizeOp, m(4, 3), m(4, 3, torch.int8), torch.zeros(3)),
                lambda: J.execute(J.LinearOp, m(3, 4, torch.int8).t(), m(3, 2, torch.int8), m(4, 2), w_scale=torch.ones(4), x_scale=torch.ones(2))):
        with pytest.raises(J.DeviceMismatch):
            bad()
    with pytest.raises(TypeError):
        J.execute(J.DropoutOp, m(4, 3), m(4, 3))
    with pytest.raises(TypeError):
        J.execute(J.DropoutOp, m(4, 3), m(4, 3), seed=1, state=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        J.execute(J.LinearOp, m(3, 4, torch.int8).t(), m(3, 2, torch.int8), m(4, 2))
    with pytest.raises(J.UnsupportedValueType):
        J.execute(J.LinearOp, m(4, 3), m(3, 2), m(4, 2), w_scale=torch.ones(4))
    with pytest.raises(J.UnsupportedFormat):
        J.execute(J.RouteOp, m(8, 3), m(2, 3, torch.int32), m(2, 3), backend=object())
    dense = J.Formats.DensedRight(2)
    for op in (J.RouteOp, J.RouteGradOp, J.CombineOp, J.CombineGradOp, J.DropoutOp, J.QuantizeOp):
        assert J.supports_backend(HIP, op(dense, dense))
        assert not J.supports_backend(HIP, op(J.Formats.CSR, dense))


# ------------------------------------------------------------- the plain forms

def test_philox_known_answers():
    """Salmon, Moraes, Dror and Shaw's known answers of Philox4x32-10."""
    for counter, key, want in (((0,) * 4, (0,) * 2, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
                               ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
                               ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
                                "d16cfe09 94fdcceb 5001e420 24126ea1")):
        assert " ".join("%08x" % int(v) for v in E.philox(counter, key)) == want


def test_plain_route():
    """A case by hand: two groups of three, the best by the sum of two."""
    l = torch.tensor([[2.0, 0.0, 0.0, 1.5, 1.5, -1.0]]).t()
    ids, w = E.route(l, 2, score="sigmoid", groups=2, keep=1)
    s = torch.sigmoid(torch.tensor(1.5)).item()
    assert ids[:, 0].tolist() == [4, 5] and np.allclose(w[:, 0], [0.5, 0.5])
    ids, w = E.route(l, 2, score="sigmoid", groups=2, keep=1, best=1, renormalize=False, origin=0)
    assert ids[:, 0].tolist() == [0, 1] and np.allclose(w[1, 0], 0.5)
    ids, w = E.route(torch.full((4, 2), -INF), 2)
    assert (ids == 0).all() and (w == 0).all()
    assert s > 0


def test_plain_route_gradient():
    gen = torch.Generator().manual_seed(0)
    l = torch.randn((6, 3), generator=gen, dtype=torch.float64)
    dw = torch.randn((2, 3), generator=gen, dtype=torch.float64)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            ids, w = E.route(l, 2, score=score, renormalize=renormalize, scale=1.5)
            x = l.clone().requires_grad_()
            s = torch.softmax(x, 0) if score == "softmax" else torch.sigmoid(x)
            c = s.gather(0, ids.long() - 1)
            v = 1.5 * (c / c.sum(0) if renormalize else c)
            assert torch.allclose(v.detach(), w)
            (v * dw).sum().backward()
            assert torch.allclose(E.route_grad(l, ids, dw, score, renormalize, 1.5)[0], x.grad)


def test_plain_quantize():
    q, s = E.quantize(torch.tensor([[127.0, 0.5, 1.5, -2.5, 0.0], [0.0] * 5, [NAN, 1.0, 1.0, 1.0, 1.0]]).t())
    assert q[:, 0].tolist() == [127, 0, 2, -2, 0] and s[0] == 1
    assert (q[:, 1:] == 0).all() and s[1] == 0 and torch.isnan(s[2])
