"""What stands around a layer's experts, and dropout (no counterpart in the
reference): a column is a token, a node of a graph or a sample, as in layers.py.

    execute(RouteOp, L, ids, w, bias=b, score="softmax", groups=1, keep=None, best=2,
            renormalize=True, scale=1.0, origin=OneBased())
        L: experts x cols logits.  ids (copies x cols, Int32) gets the experts of
        every column, the best key first, and w their weights.  Scores are the
        softmax or the sigmoid of the logits, an expert's key its score plus its
        bias (without one, its logit); the experts make `groups` equal groups, of
        which the `keep` best are looked at, ranked by their best key (best=1) or by
        the sum of their two best scores plus biases (best=2; of one alone where no
        second is left).  Equal keys go to the lower expert, equal groups to the first.
        At most 4,095 experts, 64 groups and 64 experts a column.  A weight is scale times the score, or with renormalize times
        its share of the chosen scores' sum.  An expert whose logit (or bias) is -Inf
        or NaN is never chosen; where none is left the id is origin - 1, which names
        no group to prepare(GroupedLinearOp, ids), and the weight 0.
    execute(RouteGradOp, L, ids, dw, dL, score=.., renormalize=.., scale=.., origin=..)
        the logits' gradient from the weights'; the bias has none.

    execute(CombineOp, X, w, Y, residual=R)
        Y[:, t] = sum over c of w[c, t] * X[:, copies*t + c] .+ R[:, t]: what
        execute(h, ...) left for the `copies` experts of column t.  A column of X
        whose weight is 0 is not read.
    execute(CombineGradOp, X, w, dY, dX=.., dweights=..)

    execute(DropoutOp, X, Y, p=0.1, seed=s, offset=o, residual=R)
        Y = X .* mask ./ (1 - p) .+ R.  The mask goes by seed, offset and the
        element's row and column: the same call on dY is the backward pass.  seed and
        offset are 64-bit numbers, a new offset a call; for a call that a graph
        replays, state=t in their place, a GPU tensor of the two (Int64) that is read
        when the call runs.  p is rounded to a multiple of 2^-16.

Float64, Float32, Float16 and BFloat16; weights and biases are Float32 (Float64
for Float64).  The results are the caller's buffers; execute returns the first.
For copies = 1 ids and weights may be vectors.
"""
from __future__ import annotations

import struct

import torch

from . import _lib
from .errors import DeviceMismatch, IncompatibleExtents, NonCanonicalStorage, UnsupportedIndexType, UnsupportedValueType
from .layers import _BE, _extents, _first, _matrix, _raw, _run, _vector
from .ops import _layer_calls

# jlust_route and jlust_route_grad of include/jlust_hip.h.
_ROUTE = struct.Struct("@4i13qd").pack
_ROUTE_GRAD = struct.Struct("@4i11qd").pack

_SCORES = {"softmax": 0, "sigmoid": 1}


def _score(score):
    kind = _SCORES.get(score)
    if kind is None:
        raise ValueError(f"score is \"softmax\" or \"sigmoid\", not {score!r}")
    return kind


def _tensor(t, name):
    return t if type(t) is torch.Tensor else _raw(t, name)


def _by_column(t, name, cols):
    """`t` with a column for each of `cols`: a vector holds one value each."""
    if type(t) is not torch.Tensor:
        t = _raw(t, name)
    if cols != 1 and len(t.shape) == 1:
        return t.unsqueeze(0)
    return t


def _logits(L, ids):
    l = L if type(L) is torch.Tensor else _raw(L, "L")
    T = l.dtype
    vt, index = _first(l, "L")
    experts, cols = _extents(l, "L")
    lp, ldl = _matrix(l, "L", experts, cols, index, T)
    i = _by_column(ids, "ids", cols)
    if i.dtype is not torch.int32:
        raise UnsupportedIndexType(i.dtype, _BE)
    copies = i.shape[0] if len(i.shape) else 0
    ip, ldi = _matrix(i, "ids", copies, cols, index, torch.int32)
    return T, vt, index, experts, cols, copies, lp, ldl, ip, ldi


def _route(L, ids, weights, bias=None, score="softmax", groups=1, keep=None, best=2, renormalize=True, scale=1.0, origin=None):
    T, vt, index, experts, cols, copies, lp, ldl, ip, ldi = _logits(L, ids)
    S = torch.float32 if vt else torch.float64
    wp, ldw = _matrix(_by_column(weights, "weights", cols), "weights", copies, cols, index, S)
    bp = 0 if bias is None else _vector(bias, "bias", experts, index, S)
    _run(_lib.lib().jlust_hip_route, index, "route", T,
         _ROUTE(vt, _score(score), bool(renormalize), 1 if origin is None else origin.offset, experts, cols, copies, groups,
                groups if keep is None else keep, best, lp, ldl, bp, ip, ldi, wp, ldw, scale))
    return ids


def _route_grad(L, ids, dweights, dL, score="softmax", renormalize=True, scale=1.0, origin=None):
    T, vt, index, experts, cols, copies, lp, ldl, ip, ldi = _logits(L, ids)
    wp, ldw = _matrix(_by_column(dweights, "dweights", cols), "dweights", copies, cols, index,
                      torch.float32 if vt else torch.float64)
    dp, ldd = _matrix(dL, "dL", experts, cols, index, T)
    _run(_lib.lib().jlust_hip_route_grad, index, "route_grad", T,
         _ROUTE_GRAD(vt, _score(score), bool(renormalize), 1 if origin is None else origin.offset, experts, cols, copies, lp, ldl,
                     ip, ldi, wp, ldw, dp, ldd, scale))
    return dL


def _combine(X, weights, Y, residual=None):
    x = X if type(X) is torch.Tensor else _raw(X, "X")
    y = Y if type(Y) is torch.Tensor else _raw(Y, "Y")
    T = x.dtype
    vt, index = _first(x, "X")
    d, cols = _extents(y, "Y")
    w = _by_column(weights, "weights", cols)
    copies = w.shape[0] if len(w.shape) else 0
    wp, ldw = _matrix(w, "weights", copies, cols, index, torch.float32 if vt else torch.float64)
    xp, ldx = _matrix(x, "X", d, copies * cols, index, T)
    yp, ldy = _matrix(y, "Y", d, cols, index, T)
    rp, ldr = _matrix(residual, "residual", d, cols, index, T) if residual is not None else (0, 0)
    _run(_lib.lib().jlust_hip_combine, index, "combine", T, vt, d, cols, copies, xp, ldx, wp, ldw, rp, ldr, yp, ldy)
    return Y


def _combine_grad(X, weights, dY, dX=None, dweights=None):
    x, dy = _tensor(X, "X"), _tensor(dY, "dY")
    T = x.dtype
    vt, index = _first(x, "X")
    S = torch.float32 if vt else torch.float64
    d, cols = _extents(dy, "dY")
    w = _by_column(weights, "weights", cols)
    copies = w.shape[0] if len(w.shape) else 0
    wp, ldw = _matrix(w, "weights", copies, cols, index, S)
    xp, ldx = _matrix(x, "X", d, copies * cols, index, T)
    dyp, lddy = _matrix(dy, "dY", d, cols, index, T)
    dxp, lddx = _matrix(dX, "dX", d, copies * cols, index, T)
    dwp, lddw = (0, 0) if dweights is None else _matrix(_by_column(dweights, "dweights", cols), "dweights", copies, cols, index, S)
    _run(_lib.lib().jlust_hip_combine_grad, index, "combine_grad", T, vt, d, cols, copies, xp, ldx, wp, ldw, dyp, lddy, dxp, lddx,
         dwp, lddw)
    return dX if dX is not None else dweights


_U64 = (1 << 64) - 1


def _state(t, index):
    t = _raw(t, "state")
    if t.dtype is not torch.int64:
        raise UnsupportedValueType(t.dtype, _BE, "state is Int64: seed and offset")
    if t.get_device() != index:
        raise DeviceMismatch(f"operands on several devices: state is on {t.device}, others on cuda:{index}")
    if tuple(t.shape) != (2,):
        raise IncompatibleExtents(f"state is {tuple(t.shape)}, expected (2,)")
    if t.stride(0) != 1:
        raise NonCanonicalStorage(f"state: expected stride(0) == 1, got {t.stride(0)}")
    return t.data_ptr()


def _dropout(X, Y, p=0.5, seed=None, offset=0, residual=None, state=None):
    if (seed is None) == (state is None):
        raise TypeError("DropoutOp takes seed and offset, or state")
    x = X if type(X) is torch.Tensor else _raw(X, "X")
    T = x.dtype
    vt, index = _first(x, "X")
    d, cols = _extents(x, "X")
    xp, ldx = _matrix(x, "X", d, cols, index, T)
    yp, ldy = _matrix(Y, "Y", d, cols, index, T)
    rp, ldr = _matrix(residual, "residual", d, cols, index, T) if residual is not None else (0, 0)
    sp = 0 if state is None else _state(state, index)
    _run(_lib.lib().jlust_hip_dropout, index, "dropout", T, vt, d, cols, xp, ldx, rp, ldr, yp, ldy, p, (seed or 0) & _U64,
         offset & _U64, sp)
    return Y


_layer_calls.update({"Route": _route, "RouteGrad": _route_grad, "Combine": _combine, "CombineGrad": _combine_grad,
                     "Dropout": _dropout})
