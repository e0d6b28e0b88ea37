"""Plain 64-bit forms of routing, sums of experts, dropout's mask and 8-bit columns,
written from their definitions, and the error bounds their kernels are held to (not
collected by pytest).  u is the sums' unit roundoff (tests/_layers.py)."""
import itertools

import numpy as np
import torch

from tests import _layers as L


def log_scores(l, score):
    """Logarithms of the scores of one column, -inf where there is none."""
    live = l > -np.inf
    with np.errstate(invalid="ignore", over="ignore"):
        if score == "sigmoid":
            return np.where(live, -np.logaddexp(0.0, -l), -np.inf)
        if not live.any():
            return np.full_like(l, -np.inf)
        top = l[live].max()
        d = np.where(live, np.where(l == top, 0.0, l - top), -np.inf)
        return d - np.log(np.exp(d).sum())


def kept_groups(rank, keep, close):
    """The sets of groups that may be kept, from their (-key, number): the best ones
    first; then every other way to fill the last places from groups whose keys are
    within `close` of the last one kept."""
    rank = sorted(rank)
    yield {g for _, g in rank[:keep]}
    if len(rank) <= keep:
        return
    edge = rank[keep - 1][0]
    sure = [g for k, g in rank[:keep] if edge - k > close]
    near = [g for k, g in rank if abs(k - edge) <= close]
    for some in itertools.combinations(near, keep - len(sure)):
        yield set(sure) | set(some)


def route(logits, copies, bias=None, score="softmax", groups=1, keep=None, best=2, renormalize=True, scale=1.0, origin=1, got=None):
    """ids and weights (copies x cols) from experts x cols logits, column by column.

    `got`: ids that were found.  Sums of two scores may be equal by their formula and
    not by their rounding (those of x and -x are 1 for every x).  A score is off by at
    most 4 u (exp 1, its sum and quotient, u = 2^-53) and a sum of two by 9 u, here and
    there: groups whose sums are within 2^-48 > 18 * 2^-53 of each other may come in either
    order, and the ids are then those of `got` if one of the orders gives them."""
    lg = L.f64(logits).numpy()
    b = None if bias is None else L.f64(bias).numpy()
    E, n = lg.shape
    keep = groups if keep is None else keep
    ids, w = np.full((copies, n), origin - 1, dtype=np.int32), np.zeros((copies, n))
    for t in range(n):
        l = np.where(np.isnan(lg[:, t]), -np.inf, lg[:, t])
        logs = log_scores(l, score)
        s = np.exp(logs)
        value = s if b is None else s + b
        key = l if b is None else value
        live = (l > -np.inf) & (True if b is None else ~np.isnan(b) & (b > -np.inf))
        size = E // groups
        rank = []
        for g in range(groups):
            at = [e for e in range(g * size, (g + 1) * size) if live[e]]
            if at:
                top = sorted(at, key=lambda e: -key[e])[:best]
                rank.append((-(key[top[0]] if best == 1 else sum(value[e] for e in top)), g))
        want = None
        for chosen in kept_groups(rank, keep, 2.0 ** -48 if best == 2 else 0.0):
            at = sorted((e for e in range(E) if live[e] and e // size in chosen), key=lambda e: (-key[e], e))[:copies]
            want = at if want is None else want
            if got is None or best == 1 or got[:len(at), t].tolist() == [e + origin for e in at]:
                break
        else:
            at = want
        if not at:
            continue
        ids[:len(at), t] = np.array(at) + origin
        if renormalize:
            q = np.exp(logs[at] - logs[at].max())
            w[:len(at), t] = scale * q / q.sum()
        else:
            w[:len(at), t] = scale * s[at]
    return torch.from_numpy(ids), torch.from_numpy(w)


def weight_bound(logits, u, score):
    """A weight's relative error: the exponentials' own (2 u each), their arguments'
    rounding (u |l - m| each, twice for a quotient), and the sums' (at most one add an
    expert)."""
    l = L.f64(logits)
    l = torch.where(torch.isfinite(l), l, 0.0).clamp(-800, 800)
    span = l.abs().max(0)[0] * 2
    return (16 + 4 * span + l.shape[0]) * u


def route_grad(logits, ids, dw, score="softmax", renormalize=True, scale=1.0, origin=1):
    """(dL, what its terms add up to without their signs)."""
    lg, at = L.f64(logits).numpy(), ids.cpu().numpy().astype(np.int64) - origin
    t = L.f64(dw).numpy() * scale
    E, n = lg.shape
    dL, size = np.zeros((E, n)), np.zeros((E, n))
    for j in range(n):
        logs = log_scores(np.where(np.isnan(lg[:, j]), -np.inf, lg[:, j]), score)
        ks = [k for k in range(at.shape[0]) if 0 <= at[k, j] < E]
        es = [at[k, j] for k in ks]
        if not ks:
            continue
        tk = t[ks, j]
        q = np.exp(logs[es])
        if renormalize:
            q = np.exp(logs[es] - logs[es].max()) if np.isfinite(logs[es]).any() else np.zeros(len(es))
            q = q / q.sum() if q.sum() > 0 else q
        if score == "softmax" and not renormalize:
            p, T = np.exp(logs), np.zeros(E)
            np.add.at(T, es, tk)
            dL[:, j] = p * (T - (q * tk).sum())
            size[:, j] = p * (np.abs(T) + (q * np.abs(tk)).sum())
            continue
        dot, mag = ((q * tk).sum(), (q * np.abs(tk)).sum()) if renormalize else (0.0, 0.0)
        g, a = q * (tk - dot), q * (np.abs(tk) + mag)
        if score == "sigmoid":
            left = np.exp(-np.logaddexp(0.0, lg[es, j]))
            g, a = g * left, a * left
        np.add.at(dL[:, j], es, g)
        np.add.at(size[:, j], es, a)
    return torch.from_numpy(dL), torch.from_numpy(size)


# -------------------------------------------------------------------- dropout

def philox(counter, key):
    """Philox4x32-10 of four 32-bit numbers (arrays) under two."""
    low = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    for i in range(10):
        k0, k1 = np.uint64((key[0] + i * 0x9E3779B9) & 0xFFFFFFFF), np.uint64((key[1] + i * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ k0, b & low, (a >> np.uint64(32)) ^ c[3] ^ k1, a & low]
    return c


def kept(d, cols, p, seed, offset):
    """The mask of a d x cols matrix."""
    i = np.arange(d)[:, None]
    words = philox((i // 8 + 0 * np.arange(cols), np.arange(cols) + 0 * i, offset & 0xFFFFFFFF, offset >> 32 & 0xFFFFFFFF),
                   (seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF))
    words = np.stack(np.broadcast_arrays(*words))
    word = np.take_along_axis(words, np.broadcast_to(i % 8 // 2, (1, d, cols)), 0)[0]
    return torch.from_numpy((word >> (16 * (i % 2)).astype(np.uint64) & np.uint64(0xFFFF)) >= np.uint64(dropped(p)))


def dropped(p):
    return int(np.floor(p * 65536 + 0.5))


# ---------------------------------------------------------------- 8-bit columns

def quantize(X):
    """(whole numbers, Float32 scales as Float64)."""
    x = L.f64(X).numpy()
    d, n = x.shape
    top = np.abs(x).max(0) if d else np.zeros(n)
    with np.errstate(invalid="ignore"):
        s = (top / 127).astype(np.float32).astype(np.float64)
    bad = ~np.isfinite(top)
    s[bad] = np.nan
    ok = ~bad & (s > 0)
    q = np.zeros((d, n))
    q[:, ok] = np.clip(np.rint(x[:, ok] / s[ok]), -127, 127)
    return torch.from_numpy(q), torch.from_numpy(s)


def linear8(W, ws, Xq, xs, T, bias, act, R, ids=None, copies=1):
    """(Y, Z, bound of Y, bound of Z) of 8-bit operands without the results' rounding:
    the sum is exact, its conversion and two products round once each and a sum with
    the bias once more."""
    W, Xq, ws, xs = W.detach().cpu().double(), Xq.detach().cpu().double(), L.f64(ws), L.f64(xs)
    groups = W.shape[2] if ids is not None else 1
    if ids is None:
        W, ws = W[:, :, None], ws[:, None]
    n, u = Xq.shape[1] * copies, 2.0 ** -24
    group = L.group_of(ids, groups, n)
    Z, E = torch.zeros((W.shape[0], n), dtype=torch.float64), torch.zeros((W.shape[0], n), dtype=torch.float64)
    for g in range(groups):
        at = torch.nonzero(group == g)[:, 0]
        z = (W[:, :, g] @ Xq[:, at // copies]) * ws[:, g][:, None] * xs[at // copies]
        b = 0 if bias is None else (L.f64(bias)[:, g] if ids is not None else L.f64(bias))[:, None]
        Z[:, at] = z + b
        E[:, at] = 4 * u * z.abs() + u * (z + b).abs()
    Y = L.act_of(Z, act)
    ey = 1.13 * E + (0 if act in (None, "relu") else L.act_u(T) * Z.abs())
    if R is not None:
        ey = ey + u * (Y.abs() + L.f64(R).abs())
        Y = Y + L.f64(R)
    return Y, Z, ey, E


# Products of 8-bit integers and what is planned for each: the type of Y, out, inp, cols,
# groups, copies; the sums a workgroup makes (rows, columns), whether its operands are
# copied to LDS, the pieces of k.
PLANNED8 = [
    ("bf16", 1029, 2064, 3, 0, 1, (16, 16, 0, 1)),
    ("f32", 1029, 2053, 3, 0, 1, (16, 16, 0, 1)),
    ("f16", 1029, 2064, 10, 3, 2, (16, 16, 0, 1)),
    ("f32", 53, 208, 40, 3, 2, (64, 64, 0, 1)),
    ("bf16", 1000, 4112, 130, 0, 1, (64, 64, 0, 4)),
    ("f32", 1000, 4112, 130, 3, 1, (64, 64, 0, 4)),
    ("f16", 53, 2064, 20, 0, 1, (64, 64, 0, 16)),
    ("bf16", 53, 4105, 40, 3, 2, (64, 64, 0, 32)),
    ("f16", 2053, 2064, 20, 0, 1, (128, 32, 0, 8)),
    ("f32", 520, 4112, 130, 3, 1, (128, 32, 0, 8)),
    ("f32", 2053, 1040, 1500, 0, 1, (128, 128, 1, 1)),
    ("bf16", 136, 208, 14600, 3, 2, (128, 128, 1, 1)),
    ("f16", 2053, 2064, 1500, 0, 1, (128, 128, 1, 1)),
    ("bf16", 2499, 400, 4100, 0, 1, (256, 128, 1, 1)),
    ("f32", 2136, 1040, 2000, 32, 2, (256, 128, 1, 1)),
    ("f16", 2378, 400, 2000, 32, 2, (256, 128, 1, 1)),
    ("bf16", 520, 2064, 14600, 0, 1, (256, 256, 1, 1)),
    ("f32", 520, 2064, 14600, 0, 1, (256, 256, 1, 1)),
    ("f16", 520, 2064, 14600, 3, 1, (256, 256, 1, 1)),
]

# Products of 8-bit integers that pack operands first: type, out, inp, cols, groups, copies,
# how far W and X lie off 16 bytes, whether the groups share W; the tile, what is packed (1:
# W, 2: X).
PACKED8 = [
    ("bf16", 2053, 1033, 2500, 0, 1, 0, 0, False, (128, 128, 3)),
    ("f32", 2053, 1040, 2500, 0, 1, 1, 0, False, (128, 128, 1)),
    ("f16", 2053, 1040, 2500, 0, 1, 0, 5, False, (128, 128, 2)),
    ("bf16", 1029, 1033, 3000, 3, 2, 0, 0, False, (128, 128, 3)),
    ("f16", 1029, 1033, 3000, 3, 2, 7, 0, True, (128, 128, 3)),
]
