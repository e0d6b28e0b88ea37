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

    execute(QuantizeOp, X, Xq, xs)
        Int8 columns with a Float32 scale each: Xq = X ./ xs' to the nearest
    execute(LinearOp, Wq, Xq, Y, w_scale=ws, x_scale=xs, ...)      # and execute(h, Wq, Xq, Y, ...)
        the products of Int8 matrices, W*X being (Wq*Xq) .* ws .* xs' with a scale
        for each row of W (out values, out x groups for a plan's) and each column of
        X; Wq lies along inp (QuantizeOp of W's transpose makes it).  Y, bias,
        residual and preact are Float32, Float16 or BFloat16.  No gradient.

experts.py has the operators around a layer's experts and dropout.

Float64, Float32, Float16 and BFloat16, one type for all operands of a call;
sums and the stats are Float32 (Float64 for Float64).  The results are the
caller's buffers; execute returns the first of them.  A vector stands for one
column.
"""
from __future__ import annotations

import struct
from functools import partial

import torch

from . import _lib
from .elementwise import FN_GELU, FN_IDENTITY, FN_RELU, FN_SILU, ElementwiseFn
from .errors import (DeviceMismatch, IncompatibleExtents, NonCanonicalStorage, UnsupportedFormat,
                     UnsupportedIndexType, UnsupportedValueType)
from .ops import AbstractKernelHandle, HIPBackend, _layer_calls
from .tensor import OneBased, USTensor

_BE = HIPBackend()
_TYPES = {torch.float64: 0, torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}
_ACTS = (FN_IDENTITY, FN_RELU, FN_GELU, FN_SILU)


# jlust_linear and jlust_linear_grad of include/jlust_hip.h: four 32-bit fields,
# then 64-bit ones.  Packed bytes cost a third of a ctypes structure, which counts
# in a call of a few microseconds.
_LINEAR = struct.Struct("@4i19q").pack
_LINEAR_GRAD = struct.Struct("@4i22q").pack
_LINEAR_INT8 = struct.Struct("@2i22q").pack

_current_device, _raw_stream = _lib.current_device, _lib.raw_stream


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


def _first(t, name):
    """(value type, device index) of the call, from its first operand."""
    vt, index = _TYPES.get(t.dtype), t.get_device()
    if vt is None:
        raise UnsupportedValueType(t.dtype, _BE)
    if index < 0:
        raise DeviceMismatch(f"HIPBackend needs GPU buffers, {name} is on {t.device}")
    return vt, index


def _same(t, name, index, T):
    if t.dtype != T:
        raise UnsupportedValueType(t.dtype, _BE, f"operands must share the value type {T}; {name} does not")
    if t.get_device() != index:
        raise DeviceMismatch(f"operands on several devices: {name} is on {t.device}, others on cuda:{index}")


def _matrix(t, name, rows, cols, index, T):
    """(address, leading dimension) of a rows x cols column-major operand, a
    vector standing for one column; None stands for no operand."""
    if t is None:
        return 0, 0
    if type(t) is not torch.Tensor:
        t = _raw(t, name)
    if t.dtype is not T or t.get_device() != index:
        _same(t, name, index, T)
    shape = t.shape
    if len(shape) == 2:
        s0, ld = t.stride()
        if shape[0] == rows and shape[1] == cols and (s0 == 1 or rows <= 1):
            if cols <= 1:
                return t.data_ptr(), rows
            if ld >= rows:
                return t.data_ptr(), ld
    elif len(shape) == 1:
        if cols == 1 and shape[0] == rows and (t.stride(0) == 1 or rows <= 1):
            return t.data_ptr(), rows
    else:
        raise IncompatibleExtents(f"{name}: {t.dim()}-D arrays are not supported")
    if tuple(shape) != (rows, cols) and not (len(shape) == 1 and cols == 1 and shape[0] == rows):
        raise IncompatibleExtents(f"{name} is {'x'.join(map(str, shape))}, expected {rows}x{cols}")
    raise NonCanonicalStorage(f"{name}: dense matrices are column-major (Julia layout): expected stride(0) == 1 "
                              f"and columns apart, got strides {tuple(t.stride())}")


def _extents(t, name):
    shape = t.shape
    if len(shape) == 2:
        return shape
    if len(shape) == 1:
        return shape[0], 1
    raise IncompatibleExtents(f"{name}: {t.dim()}-D arrays are not supported")


def _weights(t, name, groups, index, T):
    """(address, layout, leading dimension, group stride, out, inp) of a weight
    matrix, or of one per group: contiguous along either side."""
    if t.dtype is not T or t.get_device() != index:
        _same(t, name, index, T)
    shape, strides = t.shape, t.stride()
    if len(shape) != (3 if groups else 2):
        raise IncompatibleExtents(f"{name}: expected {'out x inp x groups' if groups else 'out x inp'}, got "
                                  f"{t.dim()} dimensions")
    out, inp = shape[0], shape[1]
    if groups and shape[2] != groups:
        raise IncompatibleExtents(f"{name} holds {shape[2]} matrices, expected {groups}")
    s0, s1 = strides[0], strides[1]
    if (s0 == 1 or out <= 1) and (s1 >= out or inp <= 1) and not (out <= 1 and s1 == 1):
        layout, ld = 0, s1 if inp > 1 else max(out, 1)
    elif (s1 == 1 or inp <= 1) and (s0 >= inp or out <= 1):
        layout, ld = 1, s0 if out > 1 else max(inp, 1)
    else:
        raise NonCanonicalStorage(f"{name}: a matrix is column-major or the transpose of one, got strides "
                                  f"{strides}")
    return t.data_ptr(), layout, ld, strides[2] if groups else 0, out, inp


def _bias(t, name, out, groups, index, T):
    """(address, stride between groups)."""
    if t is None:
        return 0, 0
    if type(t) is not torch.Tensor:
        t = _raw(t, name)
    if t.dtype is not T or t.get_device() != index:
        _same(t, name, index, T)
    if tuple(t.shape) != ((out, groups) if groups else (out,)):
        raise IncompatibleExtents(f"{name} is {tuple(t.shape)}, expected {(out, groups) if groups else (out,)}")
    if out > 1 and t.stride(0) != 1:
        raise NonCanonicalStorage(f"{name}: expected stride(0) == 1, got strides {tuple(t.stride())}")
    return t.data_ptr(), t.stride(1) if groups else 0


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
        self.shape = ids.shape
        self.groups, self.origin = int(n_groups), (OneBased() if origin is None else origin).offset
        self.dev, self.index, self.n = ids.device, ids.get_device(), ids.numel()
        if ids.dim() == 1:
            self.copies = 1
        elif ids.dim() == 2:
            self.copies = max(1, self.shape[0])
        else:
            raise IncompatibleExtents(f"ids: {ids.dim()}-D arrays are not supported")
        self._check_ids(ids)
        ints = self.groups + 1 + self.n * (2 if self.copies > 1 else 1)
        self._plan = torch.empty(max(ints, 1), dtype=torch.int32, device=self.dev)
        self._home = _lib.raw_stream(self.index)       # the stream that its memory goes back to
        self._build(ids)

    def _check_ids(self, ids):
        if ids.dtype != torch.int32 and ids.dtype != torch.int64:
            raise UnsupportedIndexType(ids.dtype, _BE)
        if ids.get_device() != self.index or self.index < 0:
            raise DeviceMismatch(f"HIPBackend needs GPU buffers, ids are on {ids.device}")
        if ids.shape != self.shape:
            raise IncompatibleExtents(f"ids are {tuple(ids.shape)}, the plan's {tuple(self.shape)}")
        if not (ids if len(self.shape) == 1 else ids.t()).is_contiguous():
            raise NonCanonicalStorage(f"ids must be contiguous columns, got strides {tuple(ids.stride())}")

    def _build(self, ids):
        _run(_lib.lib().jlust_hip_group_plan_build, self.index, "group_plan", ids.dtype, self.n, self.groups,
             self.copies, self.origin, ids.data_ptr(), ids.dtype is torch.int64, self.use())

    def update(self, ids):
        """New groups for the same columns."""
        ids = _raw(ids, "ids")
        self._check_ids(ids)
        self._build(ids)
        return self

    def use(self):
        """The plan's address, its memory kept until the current stream is done
        with it."""
        if _lib.raw_stream(self.index) != self._home:
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


def _run(f, index, what, T, *args):
    """f(*args, stream) on the operands' device; returns the stream."""
    if _current_device() == index:
        s = _raw_stream(index)
        st = f(*args, s)
    else:
        with torch.cuda.device(index):
            s = _lib.raw_stream(index)
            st = f(*args, s)
    if st:
        _lib.check(st, what, None, _BE, T)
    return s


def _columns(X, Y, h):
    """Checks the batch against the plan; returns Y's columns."""
    (_, xc), (_, yc) = _extents(X, "X"), _extents(Y, "Y")
    n = yc if h is None else h.n
    if yc != n:
        raise IncompatibleExtents(f"Y has {yc} columns, the plan {n}")
    if xc * (1 if h is None else h.copies) != n:
        raise IncompatibleExtents(f"X has {xc} columns, expected {n // (1 if h is None else h.copies)}")
    return n, xc


def _linear(h, W, X, Y, bias=None, act=None, residual=None, preact=None, w_scale=None, x_scale=None):
    w = W if type(W) is torch.Tensor else _raw(W, "W")
    x = X if type(X) is torch.Tensor else _raw(X, "X")
    y = Y if type(Y) is torch.Tensor else _raw(Y, "Y")
    T = w.dtype
    if T is torch.int8:
        return _linear_int8(h, w, x, Y, y, bias, act, residual, preact, w_scale, x_scale)
    if w_scale is not None or x_scale is not None:
        raise UnsupportedValueType(T, _BE, f"w_scale and x_scale belong to Int8 operands, W is {T}")
    vt, index = _first(w, "W")
    groups, copies, plan = 0, 1, 0
    if h is not None:
        if h.index != index:
            raise DeviceMismatch(f"the plan is on {h.dev}, W on {w.device}")
        groups, copies, plan = h.groups, h.copies, h.use()
    wp, layout, ldw, ws, out, inp = _weights(w, "W", groups, index, T)
    n, xc = _columns(x, y, h)
    xp, ldx = _matrix(x, "X", inp, xc, index, T)
    yp, ldy = _matrix(y, "Y", out, n, index, T)
    bp, bs = _bias(bias, "bias", out, groups, index, T) if bias is not None else (0, 0)
    rp, ldr = _matrix(residual, "residual", out, n, index, T)
    zp, ldz = _matrix(preact, "preact", out, n, index, T)
    _run(_lib.lib().jlust_hip_linear, index, "linear", T,
         _LINEAR(vt, _act(act), layout, 0, out, inp, n, wp, ldw, xp, ldx, yp, ldy, bp, rp, ldr, zp, ldz, groups, copies,
                 plan, ws, bs))
    return Y


def _vector(t, name, n, index, T):
    """The address of a vector of n values."""
    if type(t) is torch.Tensor and t.dtype is T and t.get_device() == index:
        shape = t.shape
        if len(shape) == 1 and shape[0] == n and (n <= 1 or t.stride(0) == 1):
            return t.data_ptr()
    return _norm_vector(t, name, n, index, T)              # another kind of operand, or what is wrong with it


def _linear_int8(h, w, x, Y, y, bias, act, residual, preact, w_scale, x_scale):
    if w_scale is None or x_scale is None:
        raise TypeError("the product of Int8 matrices needs w_scale and x_scale")
    index, T = w.get_device(), y.dtype
    if index < 0:
        raise DeviceMismatch(f"HIPBackend needs GPU buffers, W is on {w.device}")
    vt = _TYPES.get(T)
    if not vt:
        raise UnsupportedValueType(T, _BE, f"the product of Int8 matrices is Float32, Float16 or BFloat16, Y is {T}")
    groups, copies, plan = 0, 1, 0
    if h is not None:
        if h.index != index:
            raise DeviceMismatch(f"the plan is on {h.dev}, W on {w.device}")
        groups, copies, plan = h.groups, h.copies, h.use()
    shape, strides = w.shape, w.stride()
    if len(shape) != (3 if groups else 2):
        raise IncompatibleExtents(f"W: expected {'out x inp x groups' if groups else 'out x inp'}, got {w.dim()} dimensions")
    out, inp = shape[0], shape[1]
    if groups and shape[2] != groups:
        raise IncompatibleExtents(f"W holds {shape[2]} matrices, expected {groups}")
    if (strides[1] != 1 and inp > 1) or (strides[0] < inp and out > 1):
        raise NonCanonicalStorage(f"W: an Int8 matrix lies along inp, the transpose of a column-major one, got strides {strides}")
    n, xc = _columns(x, y, h)
    xp, ldx = _matrix(x, "X", inp, xc, index, torch.int8)
    yp, ldy = _matrix(y, "Y", out, n, index, T)
    if groups:
        sp, ss = _bias(w_scale, "w_scale", out, groups, index, torch.float32)
        bp, bs = _bias(bias, "bias", out, groups, index, T)
    else:
        sp, ss, bs = _vector(w_scale, "w_scale", out, index, torch.float32), 0, 0
        bp = 0 if bias is None else _vector(bias, "bias", out, index, T)
    sx = _vector(x_scale, "x_scale", xc, index, torch.float32)
    rp, ldr = (0, 0) if residual is None else _matrix(residual, "residual", out, n, index, T)
    zp, ldz = (0, 0) if preact is None else _matrix(preact, "preact", out, n, index, T)
    _run(_lib.lib().jlust_hip_linear_int8, index, "linear_int8", T,
         _LINEAR_INT8(vt, _act(act), out, inp, n, w.data_ptr(), strides[0] if out > 1 else max(inp, 1), sp, xp, ldx, sx, yp, ldy,
                      bp, rp, ldr, zp, ldz, groups, copies, plan, strides[2] if groups else 0, ss, bs))
    return Y


def _quantize(X, Y, scales):
    x = X if type(X) is torch.Tensor else _raw(X, "X")
    T = x.dtype
    vt, index = _first(x, "X")
    if vt == 0:
        raise UnsupportedValueType(T, _BE, "QuantizeOp takes Float32, Float16 or BFloat16")
    if scales is None:
        raise TypeError("QuantizeOp needs scales")
    d, cols = _extents(x, "X")
    xp, ldx = _matrix(x, "X", d, cols, index, T)
    yp, ldy = _matrix(Y, "Y", d, cols, index, torch.int8)
    _run(_lib.lib().jlust_hip_quantize_columns, index, "quantize", T, vt, d, cols, xp, ldx, yp, ldy,
         _vector(scales, "scales", cols, index, torch.float32))
    return Y


def _linear_grad(h, W, X, dY, act=None, preact=None, dX=None, dW=None, dbias=None):
    w, x, dy = _raw(W, "W"), _raw(X, "X"), _raw(dY, "dY")
    T = w.dtype
    vt, index = _first(w, "W")
    groups, copies, plan = 0, 1, 0
    if h is not None:
        if h.index != index:
            raise DeviceMismatch(f"the plan is on {h.dev}, W on {w.device}")
        groups, copies, plan = h.groups, h.copies, h.use()
    wp, layout, ldw, ws, out, inp = _weights(w, "W", groups, index, T)
    n, xc = _columns(x, dy, h)
    kind = _act(act)
    if kind != FN_IDENTITY and preact is None:
        raise TypeError(f"the gradient of {act!r} needs preact, the pre-activation that the forward call kept")
    xp, ldx = _matrix(x, "X", inp, xc, index, T)
    dyp, lddy = _matrix(dy, "dY", out, n, index, T)
    zp, ldz = _matrix(preact, "preact", out, n, index, T) if kind != FN_IDENTITY else (0, 0)
    dxp, lddx = _matrix(dX, "dX", inp, xc, index, T)
    dwp, wlayout, lddw, dws = 0, layout, 0, 0
    if dW is not None:
        dwp, wlayout, lddw, dws, o, i = _weights(_raw(dW, "dW"), "dW", groups, index, T)
        if (o, i) != (out, inp):
            raise IncompatibleExtents(f"dW is {o}x{i}, expected {out}x{inp}")
    dbp, dbs = _bias(dbias, "dbias", out, groups, index, T)
    # dW beside dX in one call where they are laid out alike; else first what the call
    # may refuse, groups that overlap.
    calls = [(layout if dxp else wlayout, dxp, dwp, dbp)] if wlayout == layout or not (dxp and dwp) else \
        [(wlayout, 0, dwp, dbp), (layout, dxp, 0, 0)]
    for lay, a, b, c in calls:
        _run(_lib.lib().jlust_hip_linear_grad, index, "linear_grad", T,
             _LINEAR_GRAD(vt, kind, lay, 0, out, inp, n, wp, ldw, xp, ldx, dyp, lddy, zp, ldz, a, lddx, b, lddw, c, groups,
                          copies, plan, ws, dws, dbs))
    return dX if dX is not None else dW if dW is not None else dbias


# -------------------------------------------------------------- normalisation

def _norm_vector(t, name, d, index, T):
    if t is None:
        return 0
    if type(t) is not torch.Tensor:
        t = _raw(t, name)
    if t.dtype is not T or t.get_device() != index:
        _same(t, name, index, T)
    if tuple(t.shape) != (d,):
        raise IncompatibleExtents(f"{name} is {tuple(t.shape)}, expected ({d},)")
    if d > 1 and t.stride(0) != 1:
        raise NonCanonicalStorage(f"{name}: expected stride(0) == 1, got {t.stride(0)}")
    return t.data_ptr()


def _layer_norm(X, Y, weight=None, bias=None, eps=1e-5, stats=None):
    x = X if type(X) is torch.Tensor else _raw(X, "X")
    T = x.dtype
    vt, index = _first(x, "X")
    d, cols = _extents(x, "X")
    xp, ldx = _matrix(x, "X", d, cols, index, T)
    yp, ldy = _matrix(Y, "Y", d, cols, index, T)
    wp, bp = _norm_vector(weight, "weight", d, index, T), _norm_vector(bias, "bias", d, index, T)
    sp, lds = _matrix(stats, "stats", 2, cols, index, torch.float64 if vt == 0 else torch.float32)
    _run(_lib.lib().jlust_hip_layer_norm, index, "layer_norm", T, vt, d, cols, xp, ldx, wp, bp, eps, yp, ldy, sp, lds)
    return Y


def _layer_norm_grad(X, dY, stats, weight=None, dX=None, dweight=None, dbias=None):
    x = _raw(X, "X")
    T = x.dtype
    vt, index = _first(x, "X")
    d, cols = _extents(x, "X")
    xp, ldx = _matrix(x, "X", d, cols, index, T)
    dyp, lddy = _matrix(dY, "dY", d, cols, index, T)
    sp, lds = _matrix(stats, "stats", 2, cols, index, torch.float64 if vt == 0 else torch.float32)
    dxp, lddx = _matrix(dX, "dX", d, cols, index, T)
    wp = _norm_vector(weight, "weight", d, index, T)
    dwp, dbp = _norm_vector(dweight, "dweight", d, index, T), _norm_vector(dbias, "dbias", d, index, T)
    _run(_lib.lib().jlust_hip_layer_norm_grad, index, "layer_norm_grad", T, vt, d, cols, xp, ldx, dyp, lddy, sp, lds, wp, dxp,
         lddx, dwp, dbp)
    return dX if dX is not None else dweight if dweight is not None else dbias


# ------------------------------------------------------------------- dispatch

def _plan(args, what):
    if not args or not isinstance(args[0], GroupPlan):
        raise TypeError(f"{what}: the first operand is a plan, prepare(HIPBackend(), GroupedLinearOp, ids, n_groups=G)")
    return args


# execute(LinearOp, ...) and the others of this module (ops.execute).
_layer_calls.update({
    "Linear": partial(_linear, None),
    "LinearGrad": partial(_linear_grad, None),
    "GroupedLinear": lambda *args, **kw: _linear(*_plan(args, "GroupedLinearOp"), **kw),
    "GroupedLinearGrad": lambda *args, **kw: _linear_grad(*_plan(args, "GroupedLinearGradOp"), **kw),
    "LayerNorm": _layer_norm,
    "LayerNormGrad": _layer_norm_grad,
    "Quantize": _quantize,
})
