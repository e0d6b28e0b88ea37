"""A layer's dense products and normalisation, next to the sparse products (no
counterpart in the reference): a column is one node of a graph, one token or
one sample, and matrices are column-major as everywhere here.

    execute(LinearOp, W, X, Y, bias=b, act=gelu_fn, residual=R, preact=Z)
        Y = act.(W*X .+ b) .+ R, and Z = W*X .+ b where it is given
    execute(LinearGradOp, W, X, dY, act=gelu_fn, preact=Z, dX=.., dW=.., dbias=..)
        with G = dY .* act'.(Z): dX = W'*G, dW = G*X', dbias = G's row sums

    h = prepare(HIPBackend(), GroupedLinearOp, ids, n_groups=G)
    execute(h, W, X, Y, ...)          # or execute(GroupedLinearOp, h, W, X, Y, ...)
    execute(GroupedLinearGradOp, h, W, X, dY, ...)
        the same with W[:, :, g] and b[:, g] of each column's group g

    execute(LayerNormOp, X, Y, weight=w, bias=b, eps=1e-5, stats=S)
    execute(LayerNormGradOp, X, dY, S, weight=w, dX=.., dweight=.., dbias=..)

Float64, Float32, Float16 and BFloat16, one type for all operands of a call;
sums and the stats are Float32 (Float64 for Float64).  The results are the
caller's buffers; execute returns the first of them.  A vector stands for one
column.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .elementwise import FN_GELU, FN_IDENTITY, FN_RELU, FN_SILU, ElementwiseFn
from .errors import (DeviceMismatch, IncompatibleExtents, NonCanonicalStorage, UnsupportedFormat,
                     UnsupportedIndexType, UnsupportedValueType)
from .ops import AbstractKernelHandle, HIPBackend
from .tensor import OneBased, USTensor

_BE = HIPBackend()
_TYPES = {torch.float64: 0, torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}
_ACTS = (FN_IDENTITY, FN_RELU, FN_GELU, FN_SILU)
_I32, _I64, _P = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p


class _Linear(ctypes.Structure):
    """jlust_linear of include/jlust_hip.h."""
    _fields_ = [("value_type", _I32), ("act", _I32), ("w_layout", _I32), ("reserved", _I32),
                ("out", _I64), ("inp", _I64), ("cols", _I64),
                ("W", _P), ("ldw", _I64), ("X", _P), ("ldx", _I64), ("Y", _P), ("ldy", _I64),
                ("bias", _P), ("R", _P), ("ldr", _I64), ("Z", _P), ("ldz", _I64),
                ("groups", _I64), ("copies", _I64), ("plan", _P), ("w_stride", _I64), ("bias_stride", _I64)]


class _LinearGrad(ctypes.Structure):
    """jlust_linear_grad of include/jlust_hip.h."""
    _fields_ = [("value_type", _I32), ("act", _I32), ("w_layout", _I32), ("reserved", _I32),
                ("out", _I64), ("inp", _I64), ("cols", _I64),
                ("W", _P), ("ldw", _I64), ("X", _P), ("ldx", _I64), ("dY", _P), ("lddy", _I64),
                ("Z", _P), ("ldz", _I64), ("dX", _P), ("lddx", _I64), ("dW", _P), ("lddw", _I64), ("dbias", _P),
                ("groups", _I64), ("copies", _I64), ("plan", _P), ("w_stride", _I64), ("dw_stride", _I64),
                ("dbias_stride", _I64)]


# --------------------------------------------------------------------- checks

def _raw(t, name):
    """The torch tensor of an operand given as one or as a dense USTensor."""
    if type(t) is torch.Tensor or isinstance(t, torch.Tensor):
        return t
    if isinstance(t, USTensor):
        if not t.format.is_dense:
            raise UnsupportedFormat(t.format, _BE, f"{name} is a dense operand")
        return t.val
    raise TypeError(f"{name}: expected a dense tensor, got {type(t).__name__}")


def _first(t, name, dev, T):
    if T not in _TYPES:
        raise UnsupportedValueType(T, _BE)
    if dev.type != "cuda":
        raise DeviceMismatch(f"HIPBackend needs GPU buffers, {name} is on {dev}")
    return _TYPES[T]


def _same(t, name, dev, T):
    if t.dtype != T:
        raise UnsupportedValueType(t.dtype, _BE, f"operands must share the value type {T}; {name} does not")
    if t.device != dev:
        raise DeviceMismatch(f"operands on several devices: {name} is on {t.device}, others on {dev}")


def _matrix(t, name, rows, cols, dev, T):
    """(address, leading dimension) of a rows x cols column-major operand, a
    vector standing for one column; None stands for no operand."""
    if t is None:
        return 0, 0
    t = _raw(t, name)
    _same(t, name, dev, T)
    if t.dim() == 1:
        r, c, s0, ld = t.shape[0], 1, t.stride(0), t.shape[0]
    elif t.dim() == 2:
        (r, c), (s0, ld) = t.shape, t.stride()
    else:
        raise IncompatibleExtents(f"{name}: {t.dim()}-D arrays are not supported")
    if r != rows or c != cols:
        raise IncompatibleExtents(f"{name} is {r}x{c}, expected {rows}x{cols}")
    if (s0 != 1 and rows > 1) or (ld < rows and cols > 1):
        raise NonCanonicalStorage(f"{name}: dense matrices are column-major (Julia layout): expected stride(0) == 1 "
                                  f"and columns apart, got strides {tuple(t.stride())}")
    return t.data_ptr(), ld if cols > 1 else rows


def _extents(t, name):
    if t.dim() == 2:
        return t.shape
    if t.dim() == 1:
        return t.shape[0], 1
    raise IncompatibleExtents(f"{name}: {t.dim()}-D arrays are not supported")


def _weights(t, name, groups, dev, T):
    """(address, layout, leading dimension, group stride, out, inp) of a weight
    matrix, or of one per group: contiguous along either side."""
    _same(t, name, dev, T)
    if t.dim() != (3 if groups else 2):
        raise IncompatibleExtents(f"{name}: expected {'out x inp x groups' if groups else 'out x inp'}, got "
                                  f"{t.dim()} dimensions")
    out, inp = t.shape[0], t.shape[1]
    if groups and t.shape[2] != groups:
        raise IncompatibleExtents(f"{name} holds {t.shape[2]} matrices, expected {groups}")
    s0, s1 = t.stride(0), t.stride(1)
    if (s0 == 1 or out <= 1) and (s1 >= out or inp <= 1) and not (out <= 1 and s1 == 1):
        layout, ld = 0, s1 if inp > 1 else max(out, 1)
    elif (s1 == 1 or inp <= 1) and (s0 >= inp or out <= 1):
        layout, ld = 1, s0 if out > 1 else max(inp, 1)
    else:
        raise NonCanonicalStorage(f"{name}: a matrix is column-major or the transpose of one, got strides "
                                  f"{tuple(t.stride())}")
    return t.data_ptr(), layout, ld, t.stride(2) if groups else 0, out, inp


def _bias(t, name, out, groups, dev, T):
    """(address, stride between groups)."""
    if t is None:
        return 0, 0
    t = _raw(t, name)
    _same(t, name, dev, T)
    if tuple(t.shape) != ((out, groups) if groups else (out,)):
        raise IncompatibleExtents(f"{name} is {tuple(t.shape)}, expected {(out, groups) if groups else (out,)}")
    if out > 1 and t.stride(0) != 1:
        raise NonCanonicalStorage(f"{name}: expected stride(0) == 1, got strides {tuple(t.stride())}")
    return t.data_ptr(), t.stride(1) if groups else 0


def _apart(stride, per, groups, name):
    """A result's groups must not share memory."""
    if groups > 1 and abs(stride) < per:
        raise NonCanonicalStorage(f"{name}: the groups' matrices overlap (stride {stride}, {per} elements each)")


def _act(act):
    if act is None:
        return FN_IDENTITY
    if not isinstance(act, ElementwiseFn) or act.kind not in _ACTS:
        raise UnsupportedFormat(act, _BE, "act is one of identity_fn, relu_fn, gelu_fn, silu_fn")
    return act.kind


# ------------------------------------------------------------------- products

class GroupPlan(AbstractKernelHandle):
    """prepare(HIPBackend(), GroupedLinearOp, ids; n_groups, origin): the columns
    sorted by group on the device (jlust_hip_group_plan_build).  ids: the group
    of every column of Y, Int32 or Int64 from `origin` (OneBased()), a vector,
    or a copies x cols matrix whose column t holds the groups of the `copies`
    columns of Y that column t of X serves.  An id that names no group (0, say)
    leaves its column out: 0 .+ residual.  Nothing is read back; update(ids)
    takes new ids of the same shape."""

    takes_raw = True

    def __init__(self, ids, n_groups=None, origin=None):
        if n_groups is None:
            raise TypeError("prepare(GroupedLinearOp, ids): n_groups is needed")
        ids = _raw(ids, "ids")
        self.shape = tuple(ids.shape)
        self.groups, self.origin = int(n_groups), (OneBased() if origin is None else origin).offset
        self.dev, self.n = ids.device, ids.numel()
        if ids.dim() == 1:
            self.copies = 1
        elif ids.dim() == 2:
            self.copies = max(1, self.shape[0])
        else:
            raise IncompatibleExtents(f"ids: {ids.dim()}-D arrays are not supported")
        self._check_ids(ids)
        ints = self.groups + 1 + self.n * (2 if self.copies > 1 else 1)
        self._plan = torch.empty(max(ints, 1), dtype=torch.int32, device=self.dev)
        self._build(ids)

    def _check_ids(self, ids):
        if ids.dtype != torch.int32 and ids.dtype != torch.int64:
            raise UnsupportedIndexType(ids.dtype, _BE)
        if ids.device.type != "cuda" or ids.device != self.dev:
            raise DeviceMismatch(f"HIPBackend needs GPU buffers, ids are on {ids.device}")
        if tuple(ids.shape) != self.shape:
            raise IncompatibleExtents(f"ids are {tuple(ids.shape)}, the plan's {self.shape}")
        if not (ids if ids.dim() == 1 else ids.t()).is_contiguous():
            raise NonCanonicalStorage(f"ids must be contiguous columns, got strides {tuple(ids.stride())}")

    def _build(self, ids):
        with _lib.on_device(self.dev):
            self._stream = _lib.stream_handle(self.dev).value
            st = _lib.lib().jlust_hip_group_plan_build(
                self.n, self.groups, self.copies, self.origin, ids.data_ptr(), int(ids.dtype == torch.int64),
                self._plan.data_ptr(), self._stream)
        _lib.check(st, "group_plan", None, _BE, ids.dtype)

    def update(self, ids):
        """New groups for the same columns."""
        ids = _raw(ids, "ids")
        self._check_ids(ids)
        self._build(ids)
        return self

    def use(self, stream):
        """The plan's address, its memory kept until `stream` is done with it."""
        if stream != self._stream:
            self._plan.record_stream(torch.cuda.current_stream(self.dev))
        return self._plan.data_ptr()

    def offsets(self) -> torch.Tensor:
        """offsets[g] .. offsets[g+1]: group g's part of order(), from 0."""
        return self._plan[: self.groups + 1]

    def order(self) -> torch.Tensor:
        """The columns in the order of their groups, from 0; those of no group
        last."""
        return self._plan[self.groups + 1: self.groups + 1 + self.n]

    def execute(self, W, X, Y, **kw):
        return _linear(self, W, X, Y, **kw)


def _columns(X, Y, h):
    """Checks the batch against the plan; returns Y's columns."""
    (_, xc), (_, yc) = _extents(X, "X"), _extents(Y, "Y")
    n = yc if h is None else h.n
    if yc != n:
        raise IncompatibleExtents(f"Y has {yc} columns, the plan {n}")
    if xc * (1 if h is None else h.copies) != n:
        raise IncompatibleExtents(f"X has {xc} columns, expected {n // (1 if h is None else h.copies)}")
    return n, xc


def _linear(h, W, X, Y, bias=None, act=None, residual=None, preact=None):
    w, x, y = _raw(W, "W"), _raw(X, "X"), _raw(Y, "Y")
    T, dev = w.dtype, w.device
    vt, groups = _first(w, "W", dev, T), 0 if h is None else h.groups
    wp, layout, ldw, ws, out, inp = _weights(w, "W", groups, dev, T)
    n, xc = _columns(x, y, h)
    xp, ldx = _matrix(x, "X", inp, xc, dev, T)
    yp, ldy = _matrix(y, "Y", out, n, dev, T)
    bp, bs = _bias(bias, "bias", out, groups, dev, T)
    rp, ldr = _matrix(residual, "residual", out, n, dev, T)
    zp, ldz = _matrix(preact, "preact", out, n, dev, T)
    if h is not None and h.dev != dev:
        raise DeviceMismatch(f"the plan is on {h.dev}, W on {dev}")
    kind = _act(act)
    with _lib.on_device(dev):
        s = _lib.stream_handle(dev).value
        op = _Linear(vt, kind, layout, 0, out, inp, n, wp, ldw, xp, ldx, yp, ldy, bp, rp, ldr, zp, ldz,
                     groups, 1 if h is None else h.copies, 0 if h is None else h.use(s), ws, bs)
        st = _lib.lib().jlust_hip_linear(ctypes.byref(op), s)
    if st:
        _lib.check(st, "linear", None, _BE, T)
    return Y


def _linear_grad(h, W, X, dY, act=None, preact=None, dX=None, dW=None, dbias=None):
    w, x, dy = _raw(W, "W"), _raw(X, "X"), _raw(dY, "dY")
    T, dev = w.dtype, w.device
    vt, groups = _first(w, "W", dev, T), 0 if h is None else h.groups
    wp, layout, ldw, ws, out, inp = _weights(w, "W", groups, dev, T)
    n, xc = _columns(x, dy, h)
    kind = _act(act)
    if kind != FN_IDENTITY and preact is None:
        raise TypeError(f"the gradient of {act!r} needs preact, the pre-activation that the forward call kept")
    xp, ldx = _matrix(x, "X", inp, xc, dev, T)
    dyp, lddy = _matrix(dy, "dY", out, n, dev, T)
    zp, ldz = _matrix(preact, "preact", out, n, dev, T) if kind != FN_IDENTITY else (0, 0)
    dxp, lddx = _matrix(dX, "dX", inp, xc, dev, T)
    dwp, wlayout, lddw, dws = 0, layout, 0, 0
    if dW is not None:
        dwp, wlayout, lddw, dws, o, i = _weights(_raw(dW, "dW"), "dW", groups, dev, T)
        if (o, i) != (out, inp):
            raise IncompatibleExtents(f"dW is {o}x{i}, expected {out}x{inp}")
        _apart(dws, out * inp, groups, "dW")
    dbp, dbs = _bias(dbias, "dbias", out, groups, dev, T)
    if dbp:
        _apart(dbs, out, groups, "dbias")
    if h is not None and h.dev != dev:
        raise DeviceMismatch(f"the plan is on {h.dev}, W on {dev}")
    copies = 1 if h is None else h.copies
    L = _lib.lib()
    with _lib.on_device(dev):
        s = _lib.stream_handle(dev).value
        plan = 0 if h is None else h.use(s)
        # dW beside dX in one call where they are laid out alike.
        calls = [(layout, dxp, dwp, dbp)] if wlayout == layout or not (dxp and dwp) else \
            [(layout, dxp, 0, dbp), (wlayout, 0, dwp, 0)]
        for lay, a, b, c in calls:
            if not a:
                lay = wlayout
            op = _LinearGrad(vt, kind, lay, 0, out, inp, n, wp, ldw, xp, ldx, dyp, lddy, zp, ldz, a, lddx, b, lddw, c,
                             groups, copies, plan, ws, dws, dbs)
            st = L.jlust_hip_linear_grad(ctypes.byref(op), s)
            if st:
                _lib.check(st, "linear_grad", None, _BE, T)
    return dX if dX is not None else dW if dW is not None else dbias


# -------------------------------------------------------------- normalisation

def _norm_vector(t, name, d, dev, T):
    if t is None:
        return 0
    t = _raw(t, name)
    _same(t, name, dev, T)
    if tuple(t.shape) != (d,):
        raise IncompatibleExtents(f"{name} is {tuple(t.shape)}, expected ({d},)")
    if d > 1 and t.stride(0) != 1:
        raise NonCanonicalStorage(f"{name}: expected stride(0) == 1, got {t.stride(0)}")
    return t.data_ptr()


def _layer_norm(X, Y, weight=None, bias=None, eps=1e-5, stats=None):
    x = _raw(X, "X")
    T, dev = x.dtype, x.device
    vt = _first(x, "X", dev, T)
    d, cols = _extents(x, "X")
    xp, ldx = _matrix(x, "X", d, cols, dev, T)
    yp, ldy = _matrix(Y, "Y", d, cols, dev, T)
    wp, bp = _norm_vector(weight, "weight", d, dev, T), _norm_vector(bias, "bias", d, dev, T)
    sp, lds = _matrix(stats, "stats", 2, cols, dev, torch.float64 if T == torch.float64 else torch.float32)
    with _lib.on_device(dev):
        st = _lib.lib().jlust_hip_layer_norm(vt, d, cols, xp, ldx, wp, bp, float(eps), yp, ldy, sp, lds,
                                             _lib.stream_handle(dev).value)
    if st:
        _lib.check(st, "layer_norm", None, _BE, T)
    return Y


def _layer_norm_grad(X, dY, stats, weight=None, dX=None, dweight=None, dbias=None):
    x = _raw(X, "X")
    T, dev = x.dtype, x.device
    vt = _first(x, "X", dev, T)
    d, cols = _extents(x, "X")
    xp, ldx = _matrix(x, "X", d, cols, dev, T)
    dyp, lddy = _matrix(dY, "dY", d, cols, dev, T)
    sp, lds = _matrix(stats, "stats", 2, cols, dev, torch.float64 if T == torch.float64 else torch.float32)
    dxp, lddx = _matrix(dX, "dX", d, cols, dev, T)
    wp = _norm_vector(weight, "weight", d, dev, T)
    dwp, dbp = _norm_vector(dweight, "dweight", d, dev, T), _norm_vector(dbias, "dbias", d, dev, T)
    with _lib.on_device(dev):
        st = _lib.lib().jlust_hip_layer_norm_grad(vt, d, cols, xp, ldx, dyp, lddy, sp, lds, wp, dxp, lddx, dwp, dbp,
                                                  _lib.stream_handle(dev).value)
    if st:
        _lib.check(st, "layer_norm_grad", None, _BE, T)
    return dX if dX is not None else dweight if dweight is not None else dbias


# ------------------------------------------------------------------- dispatch

def _plan(args, what):
    if not args or not isinstance(args[0], GroupPlan):
        raise TypeError(f"{what}: the first operand is a plan, prepare(HIPBackend(), GroupedLinearOp, ids, n_groups=G)")
    return args


_RUN = {
    "Linear": lambda args, kw: _linear(None, *args, **kw),
    "LinearGrad": lambda args, kw: _linear_grad(None, *args, **kw),
    "GroupedLinear": lambda args, kw: _linear(*_plan(args, "GroupedLinearOp"), **kw),
    "GroupedLinearGrad": lambda args, kw: _linear_grad(*_plan(args, "GroupedLinearGradOp"), **kw),
    "LayerNorm": lambda args, kw: _layer_norm(*args, **kw),
    "LayerNormGrad": lambda args, kw: _layer_norm_grad(*args, **kw),
}


def execute(optype, args, backend, kw):
    """execute(LinearOp, ...) and the others of this module (ops.execute)."""
    if backend is not None and not isinstance(backend, HIPBackend):
        raise UnsupportedFormat(optype.tag, backend, "no such backend in jlust_amd")
    return _RUN[optype.tag](args, kw)
