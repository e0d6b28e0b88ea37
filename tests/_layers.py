"""Plain 64-bit forms of a layer's products and normalisation, and the error
bounds their kernels are held to (not collected by pytest).

Bounds, with u the unit roundoff of the value type and v that of the sums
(2^-24, Float64 2^-53): a sum of k products is off by at most (k + 8) v times the
sum of their magnitudes (8: the adds of split and lane sums and the bias); an
activation passes an error on at most 1.13-fold and adds its own, 4 v |z| or, in
16 bits, 3e-7 |z| (its error function is good to 1.5e-7, doubled for exp and
rcp); the result is rounded once, u |y|, and the smallest subnormal covers
results below the normal range."""
import numpy as np
import torch

U = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float64: 0.0, torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.bfloat16, torch.float16, torch.float32, torch.float64]


def sums_u(T):
    return U[T] if T == torch.float64 else 2.0 ** -24


def act_u(T):
    return 4 * U[T] if T in (torch.float64, torch.float32) else 3e-7


def f64(t):
    return t.detach().double().cpu()


def erf(z):
    return torch.erf(z)


def act_of(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.where(torch.isnan(z), z, torch.zeros_like(z)))
    if kind == "gelu":
        return z * 0.5 * torch.erfc(-z * np.sqrt(0.5))
    if kind == "silu":
        return z / (1 + torch.exp(-z))
    return z


def slope_of(z, kind):
    if kind == "relu":
        return (z > 0).double()
    if kind == "gelu":
        return 0.5 * torch.erfc(-z * np.sqrt(0.5)) + z * torch.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    if kind == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def group_of(ids, groups, n, origin=1):
    if ids is None:
        return torch.zeros(n, dtype=torch.long)
    g = ids.detach().cpu().t().reshape(-1).long() - origin
    return torch.where((g >= 0) & (g < groups), g, torch.full_like(g, -1))


def forward(W, X, bias, act, R, ids=None, copies=1):
    """(Y, Z, bound of Y, bound of Z) without the final rounding's share."""
    T, W, X = W.dtype, f64(W), f64(X)
    groups = W.shape[2] if ids is not None else 1
    W = W if ids is not None else W[:, :, None]
    n = X.shape[1] * copies
    group = group_of(ids, groups, n)
    Z, S = torch.zeros((W.shape[0], n), dtype=torch.float64), torch.zeros((W.shape[0], n), dtype=torch.float64)
    for g in range(groups):
        at = torch.nonzero(group == g)[:, 0]
        x = X[:, at // copies]
        b = 0 if bias is None else (f64(bias)[:, g] if ids is not None else f64(bias))[:, None]
        Z[:, at] = W[:, :, g] @ x + b
        S[:, at] = W[:, :, g].abs() @ x.abs() + (0 if bias is None else b.abs())
    ez = (X.shape[0] + 8) * sums_u(T) * S
    Y = act_of(Z, act)
    ey = 1.13 * ez + (0 if act in (None, "relu") else act_u(T) * Z.abs())
    if R is not None:
        ey = ey + sums_u(T) * (Y.abs() + f64(R).abs())
        Y = Y + f64(R)
    return Y, Z, ey, ez


def gradients(W, X, dY, Z, act, ids=None, copies=1):
    """{name: (value, bound without the final rounding)} of dX, dW, dbias."""
    T, W, X, dY = W.dtype, f64(W), f64(X), f64(dY)
    groups = W.shape[2] if ids is not None else 1
    W3 = W if ids is not None else W[:, :, None]
    n = X.shape[1] * copies
    group = group_of(ids, groups, n)
    z = None if act is None else f64(Z)
    G = dY if act is None else dY * slope_of(z, act)
    # the slope's own error, and G's rounding for the products
    eg = torch.zeros_like(G) if act is None else dY.abs() * (4 * sums_u(T) + 2 * act_u(T) * (1 + z.abs()))
    er = eg if act is None else eg + U[T] * (G.abs() + eg) + TINY[T]
    per, eper = torch.zeros((X.shape[0], n), dtype=torch.float64), torch.zeros((X.shape[0], n), dtype=torch.float64)
    dW, eW = torch.zeros_like(W3), torch.zeros_like(W3)
    db, eb = torch.zeros((W3.shape[0], groups), dtype=torch.float64), torch.zeros((W3.shape[0], groups), dtype=torch.float64)
    v = sums_u(T)
    for g in range(groups):
        at = torch.nonzero(group == g)[:, 0]
        w, x, gg = W3[:, :, g], X[:, at // copies], G[:, at]
        per[:, at] = w.t() @ gg
        eper[:, at] = w.t().abs() @ (er[:, at] + (W3.shape[0] + 8) * v * gg.abs())
        dW[:, :, g] = gg @ x.t()
        eW[:, :, g] = (er[:, at] + (at.numel() + 72) * v * gg.abs()) @ x.t().abs()
        db[:, g] = gg.sum(1)
        eb[:, g] = (eg[:, at] + (at.numel() + 72) * v * gg.abs()).sum(1)
    dX = per.view(X.shape[0], X.shape[1], copies).sum(2)
    eX = (eper + copies * v * per.abs()).view(X.shape[0], X.shape[1], copies).sum(2)
    if ids is None:
        dW, eW, db, eb = dW[:, :, 0], eW[:, :, 0], db[:, 0], eb[:, 0]
    return {"dX": (dX, eX), "dW": (dW, eW), "dbias": (db, eb)}


def close(got, ref, bound, what):
    """|got - ref| <= bound + the rounding to got's type."""
    T, g = got.dtype, f64(got)
    lim = bound + U[T] * (ref.abs() + bound) + TINY[T]
    bad = ~((g - ref).abs() <= lim)
    if bad.any():
        i = torch.nonzero(bad)[0].tolist()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: got {g[tuple(i)]}, "
                             f"expected {ref[tuple(i)]} within {lim[tuple(i)]}")


def colmajor(m, n, T, gen, scale=1.0, pad=0, skip=0):
    """A column-major m x n matrix on the GPU, its columns `pad` apart, its first
    element `skip` elements into the buffer; what surrounds it is NaN."""
    ld = m + pad
    buf = torch.full((max(n, 1) * ld + skip + 8,), float("nan"), dtype=T, device="cuda")
    t = torch.as_strided(buf, (m, n), (1, ld), skip)
    t.copy_(torch.randn((n, m), generator=gen, dtype=torch.float32).t().mul_(scale).to(T))
    return t
