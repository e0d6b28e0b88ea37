"""A layer's dense products (LinearOp, GroupedLinearOp and their gradients) and
layer norm on the GPU against plain 64-bit forms (tests/_layers.py, where the
bounds are derived), at the sizes, layouts and groups where they can go wrong."""
import numpy as np
import pytest
import torch

from tests import _layers as L

pytestmark = pytest.mark.gpu

ACTS = [None, "relu", "gelu", "silu"]


@pytest.fixture(scope="module")
def J():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import jlust_amd
    return jlust_amd


def fn(J, act):
    return {None: None, "relu": J.relu_fn, "gelu": J.gelu_fn, "silu": J.silu_fn}[act]


def weights(out, inp, groups, T, gen, layout, pad=0, skip=0):
    """out x inp (x groups), contiguous along `layout`, surrounded by NaN."""
    a, b = (out, inp) if layout == "out" else (inp, out)
    ld = a + pad
    buf = torch.full((max(groups or 1, 1) * b * ld + skip + 8,), float("nan"), dtype=T, device="cuda")
    t = torch.as_strided(buf, (a, b, groups or 1), (1, ld, ld * b), skip)
    t.copy_((torch.randn((groups or 1, b, a), generator=gen) * max(inp, 1) ** -0.5).to(T).permute(2, 1, 0))
    t = t if layout == "out" else t.transpose(0, 1)
    return t if groups else t[:, :, 0]


def case(seed, T, out, inp, cols, layout, act, bias, residual, groups=None, copies=1, pad=0, skip=0):
    gen = torch.Generator().manual_seed(seed)
    n = cols * copies
    s = dict(W=weights(out, inp, groups, T, gen, layout, pad, skip), X=L.colmajor(inp, cols, T, gen, pad=pad, skip=skip),
             Y=L.colmajor(out, n, T, gen, pad=pad, skip=skip), Z=L.colmajor(out, n, T, gen, pad=pad, skip=skip),
             R=L.colmajor(out, n, T, gen, pad=pad) if residual else None, act=act,
             b=L.colmajor(out, groups or 1, T, gen, 0.5, pad=pad) if bias else None)
    if bias and not groups:
        s["b"] = s["b"][:, 0]
    return s


def check_forward(J, s, ids=None, copies=1, h=None):
    ref, refz, ey, ez = L.forward(s["W"], s["X"], s["b"], s["act"], s["R"], ids, copies)
    args = (s["W"], s["X"], s["Y"])
    kw = dict(bias=s["b"], act=fn(J, s["act"]), residual=s["R"], preact=s["Z"])
    r = J.execute(J.LinearOp, *args, **kw) if h is None else J.execute(h, *args, **kw)
    assert r is s["Y"]
    L.close(s["Y"], ref, ey, "Y")
    L.close(s["Z"], refz, ez, "Z")


def check_grad(J, s, ids=None, copies=1, h=None, seed=0):
    gen = torch.Generator().manual_seed(seed + 7)
    T = s["W"].dtype
    dY, Z = torch.empty_like(s["Y"]), s["Z"]
    dY.copy_(torch.randn(dY.shape[::-1], generator=gen).t().to(T))
    Z.copy_(torch.randn(Z.shape[::-1], generator=gen).t().mul_(1.5).to(T))
    ref = L.gradients(s["W"], s["X"], dY, Z, s["act"], ids, copies)
    nan = float("nan")
    out = dict(dX=torch.full_like(s["X"], nan), dW=torch.full_like(s["W"], nan))
    groups = None if h is None else h.groups
    out["dbias"] = torch.full((groups or 1, s["Y"].shape[0]), nan, dtype=T, device="cuda").t()
    if groups is None:
        out["dbias"] = out["dbias"][:, 0]
    kw = dict(act=fn(J, s["act"]), preact=Z if s["act"] else None, **out)
    if h is None:
        J.execute(J.LinearGradOp, s["W"], s["X"], dY, **kw)
    else:
        J.execute(J.GroupedLinearGradOp, h, s["W"], s["X"], dY, **kw)
    for k, v in out.items():
        L.close(v, *ref[k], k)


# out, inp, cols: one of everything, tile edges, odd sizes, few and many columns,
# a long k over few tiles (split), more k than one step but not a whole one.
SIZES = [(1, 1, 1), (3, 5, 2), (17, 33, 5), (64, 128, 16), (130, 70, 33), (257, 129, 100), (128, 64, 300),
         (300, 1000, 2), (8, 4096, 1), (96, 100, 1000), (520, 72, 700), (129, 2000, 49)]


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("layout", ["out", "inp"])
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_linear(J, T, layout, i):
    out, inp, cols = SIZES[i]
    k = i + L.TYPES.index(T) + (layout == "inp")
    s = case(i, T, out, inp, cols, layout, ACTS[k % 4], k % 3 != 0, k % 2 == 0)
    check_forward(J, s)
    check_grad(J, s, seed=i)


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("layout", ["out", "inp"])
@pytest.mark.parametrize("pad,skip", [(1, 1), (3, 0), (8, 8), (7, 5)])
def test_linear_strides(J, T, layout, pad, skip):
    """Columns apart, off any alignment, NaN between them."""
    s = case(3, T, 133, 77, 50, layout, "silu", True, True, pad=pad, skip=skip)
    check_forward(J, s)
    check_grad(J, s)


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["out", "inp"])
def test_linear_large_tiles(J, T, layout):
    """Enough tiles for the largest shape, none of the edges whole."""
    s = case(5, T, 2100, 200, 9000, layout, "gelu", True, False)
    check_forward(J, s)
    check_grad(J, s)


@pytest.mark.parametrize("layout", ["out", "inp"])
@pytest.mark.parametrize("act", [None, "gelu"])
@pytest.mark.parametrize("out,inp,cols,pad,skip", [(2053, 1029, 4100, 0, 0), (1024, 1032, 4096, 8, 3), (1160, 2048, 1200, 1, 0)])
def test_linear_packed(J, layout, act, out, inp, cols, pad, skip):
    """Products large enough that rows that lie badly (odd lengths, starts or
    distances) are packed first, the gradient's dY among them."""
    s = case(out, torch.bfloat16, out, inp, cols, layout, act, True, False, pad=pad, skip=skip)
    check_forward(J, s)
    check_grad(J, s)


@pytest.mark.parametrize("T", L.TYPES)
def test_linear_gradient_against_differences(J, T):
    """The gradients of sum(Y .* D) by central differences of the 64-bit form:
    step 1e-5, so 1e-10 times the third derivative and 1e-11 of rounding, next to
    which the kernel's bounds are large except in Float64 (1e-8 covers both)."""
    s = case(11, T, 9, 7, 5, "out", "gelu", True, False)
    check_forward(J, s)
    gen = torch.Generator().manual_seed(2)
    D = torch.randn((5, 9), generator=gen).to(T).t().cuda()
    W, X, b = (L.f64(s[k]) for k in ("W", "X", "b"))
    Z = torch.empty_like(s["Z"]).copy_((W @ X + b[:, None]).to(T))
    zr = L.f64(Z) - (W @ X + b[:, None])              # the pre-activation as it was kept

    def loss(W, X, b):
        return float((L.act_of(W @ X + b[:, None] + zr, "gelu") * L.f64(D)).sum())

    out = {"dX": torch.empty_like(s["X"]), "dW": torch.empty_like(s["W"]), "dbias": torch.empty_like(s["b"])}
    J.execute(J.LinearGradOp, s["W"], s["X"], D, act=J.gelu_fn, preact=Z, **out)
    ref = L.gradients(s["W"], s["X"], D, Z, "gelu")
    for name, at in (("dX", 1), ("dW", 0), ("dbias", 2)):
        base = [W, X, b]
        num = torch.zeros_like(base[at])
        for i in np.ndindex(*num.shape):
            side = []
            for d in (1e-5, -1e-5):
                t = [v.clone() for v in base]
                t[at][i] += d
                side.append(loss(*t))
            num[i] = (side[0] - side[1]) / 2e-5
        L.close(out[name], num, ref[name][1] + 1e-8, name)


def test_linear_only_what_is_asked(J):
    """Each gradient alone equals itself among the others, and layouts of dW
    other than W's."""
    T = torch.float32
    s = case(4, T, 70, 50, 40, "out", "relu", True, False)
    check_forward(J, s)
    dY = torch.randn_like(s["Y"])
    full = {"dX": torch.empty_like(s["X"]), "dW": torch.empty_like(s["W"]), "dbias": torch.empty_like(s["b"])}
    J.execute(J.LinearGradOp, s["W"], s["X"], dY, act=J.relu_fn, preact=s["Z"], **full)
    for k, v in full.items():
        one = torch.empty_like(v)
        assert J.execute(J.LinearGradOp, s["W"], s["X"], dY, act=J.relu_fn, preact=s["Z"], **{k: one}) is one
        assert torch.equal(one, v), k
    other = torch.empty((70, 50), dtype=T, device="cuda")
    again = torch.empty_like(s["X"])
    J.execute(J.LinearGradOp, s["W"], s["X"], dY, act=J.relu_fn, preact=s["Z"], dX=again, dW=other)
    assert torch.equal(again, full["dX"])
    L.close(other, *L.gradients(s["W"], s["X"], dY, s["Z"], "relu")["dW"], "dW")


def test_linear_vectors_usts_and_aliases(J):
    s = case(6, torch.float32, 33, 20, 1, "inp", "silu", True, True)
    y = torch.empty(33, device="cuda")
    J.execute(J.LinearOp, s["W"], s["X"][:, 0], y, bias=s["b"], act=J.silu_fn, residual=s["R"][:, 0])
    check_forward(J, s)
    assert torch.equal(y, s["Y"][:, 0])
    u = J.ust(torch.empty_like(s["Y"]))
    assert J.execute(J.LinearOp, s["W"], J.ust(s["X"]), u, bias=s["b"], act=J.silu_fn, residual=s["R"]) is u
    assert torch.equal(u.val, s["Y"])
    # Y over its own residual, whole and split
    for out, inp, cols in ((33, 20, 30), (64, 5000, 3)):
        s = case(7, torch.bfloat16, out, inp, cols, "out", None, False, True)
        check_forward(J, s)
        J.execute(J.LinearOp, s["W"], s["X"], s["R"], residual=s["R"])
        assert torch.equal(s["R"], s["Y"])


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("out,inp,cols", [(0, 5, 3), (5, 0, 3), (5, 3, 0)])
def test_linear_empty(J, T, out, inp, cols):
    s = case(8, T, out, inp, cols, "out", "relu", True, True)
    check_forward(J, s)
    check_grad(J, s)


@pytest.mark.parametrize("T", L.TYPES)
def test_linear_not_finite(J, T):
    """NaN and infinities reach their own column and no other; relu keeps NaN."""
    s = case(9, T, 40, 30, 20, "inp", "relu", True, False)
    s["X"][3, 4], s["X"][5, 6] = float("nan"), float("inf")
    J.execute(J.LinearOp, s["W"], s["X"], s["Y"], bias=s["b"], act=J.relu_fn, preact=s["Z"])
    ref = L.forward(s["W"], s["X"], s["b"], "relu", None)[0]
    assert torch.isnan(s["Y"][:, 4]).all()
    assert torch.equal(L.f64(s["Y"][:, 6]), ref[:, 6])
    keep = [c for c in range(20) if c not in (4, 6)]
    assert torch.isfinite(s["Y"][:, keep]).all()


def test_linear_long_offsets(J):
    """Columns whose offset passes 2^32 bytes and 2^31 elements."""
    T, inp, out, cols = torch.bfloat16, 64, 64, 35_000_000
    X = torch.zeros((cols, inp), dtype=T, device="cuda").t()
    Y = torch.full((cols, out), float("nan"), dtype=T, device="cuda").t()
    gen = torch.Generator().manual_seed(0)
    W = weights(out, inp, None, T, gen, "out")
    at = [0, 12345, 33_554_431, 33_554_432, 33_554_433, cols - 1]
    X[:, at] = torch.randn((inp, len(at)), generator=gen).to(T).cuda()
    J.execute(J.LinearOp, W, X, Y)
    ref, _, ey, _ = L.forward(W, X[:, at].contiguous(), None, None, None)
    L.close(Y[:, at], ref, ey, "Y")
    assert not torch.isnan(Y[:, -1000:]).any() and float(Y[:, 20_000_000:20_001_000].abs().max()) == 0


# ---------------------------------------------------------------------- groups

def some_ids(n, groups, seed, drop=0.1, empty=()):
    g = np.random.default_rng(seed)
    ids = g.integers(1, groups + 1, n)
    for e in empty:
        ids[ids == e] = (e % groups) + 1
    ids[g.random(n) < drop] = g.choice([0, -1, groups + 1])
    return ids.astype(np.int32)


@pytest.mark.parametrize("n,groups", [(0, 3), (1, 1), (1, 9), (63, 2), (64, 64), (65, 65), (1000, 7), (8192, 1000),
                                      (8192, 1001), (8193, 5), (100_003, 33), (50_000, 4095)])
@pytest.mark.parametrize("wide", [False, True])
def test_group_plan(J, n, groups, wide):
    ids = some_ids(n, groups, n + groups)
    for origin in (J.OneBased(), J.ZeroBased()):
        t = torch.from_numpy(ids - (0 if origin.offset else 1)).cuda()
        h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, t.long() if wide else t, n_groups=groups, origin=origin)
        bins = np.where((ids >= 1) & (ids <= groups), ids - 1, groups)
        assert np.array_equal(h.order().cpu().numpy(), np.argsort(bins, kind="stable"))
        want = np.concatenate([[0], np.cumsum(np.bincount(bins, minlength=groups + 1))])[: groups + 1]
        assert np.array_equal(h.offsets().cpu().numpy(), want)
        again = some_ids(n, groups, 5)
        h.update(torch.from_numpy(again - (0 if origin.offset else 1)).cuda().to(t.dtype))
        bins = np.where((again >= 1) & (again <= groups), again - 1, groups)
        assert np.array_equal(h.order().cpu().numpy(), np.argsort(bins, kind="stable"))


# out, inp, columns of X, copies, groups: fewer columns than groups, one group,
# runs that end inside a tile, many columns.
GROUPED = [(5, 3, 1, 1, 1), (33, 40, 7, 1, 20), (130, 64, 50, 2, 4), (64, 136, 300, 1, 3), (100, 70, 90, 3, 9),
           (48, 500, 10, 2, 70), (260, 96, 1500, 1, 5), (128, 33, 700, 4, 2)]


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("layout", ["out", "inp"])
@pytest.mark.parametrize("i", range(len(GROUPED)))
def test_grouped(J, T, layout, i):
    out, inp, cols, copies, groups = GROUPED[i]
    k = i + L.TYPES.index(T) + (layout == "inp")
    s = case(i, T, out, inp, cols, layout, ACTS[k % 4], k % 3 != 0, k % 2 == 0, groups, copies, pad=k % 2, skip=k % 3)
    ids = torch.from_numpy(some_ids(cols * copies, groups, i, 0.15 * (k % 2), (2,) if groups > 2 else ())).cuda()
    if copies > 1:
        ids = ids.view(cols, copies).t()
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=groups)
    check_forward(J, s, ids, copies, h)
    check_grad(J, s, ids, copies, h, seed=i)


@pytest.mark.parametrize("layout", ["out", "inp"])
@pytest.mark.parametrize("act", [None, "silu"])
def test_grouped_packed(J, layout, act):
    """As test_linear_packed, with columns in no group and two copies."""
    s = case(3, torch.float16, 1531, 1029, 2050, layout, act, True, False, 3, 2, pad=1)
    ids = torch.from_numpy(some_ids(4100, 3, 9, 0.1)).cuda().view(2050, 2).t()
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=3)
    check_forward(J, s, ids, 2, h)
    check_grad(J, s, ids, 2, h)


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
def test_grouped_none_and_all(J, T):
    """Every column in one group, and every column in none: Y keeps the residual
    alone and every gradient is zero."""
    for ids in (np.full(200, 3), np.zeros(200), np.full(200, 9)):
        ids = torch.from_numpy(ids.astype(np.int32)).cuda()
        s = case(1, T, 70, 60, 200, "out", "gelu", True, True, 4)
        h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=4)
        check_forward(J, s, ids, 1, h)
        check_grad(J, s, ids, 1, h)
        if int(ids[0]) != 3:
            assert torch.equal(s["Y"], s["R"])


def test_grouped_is_linear_for_one_group(J):
    """One group in order: the same tiles, so the same bits."""
    s = case(2, torch.bfloat16, 150, 90, 333, "inp", "silu", True, True)
    check_forward(J, s)
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, torch.ones(333, dtype=torch.int32, device="cuda"), n_groups=1)
    Y = torch.empty_like(s["Y"])
    J.execute(J.GroupedLinearOp, h, s["W"][:, :, None], s["X"], Y, bias=s["b"][:, None], act=J.silu_fn, residual=s["R"])
    assert torch.equal(Y, s["Y"])


# ------------------------------------------------------------------- layer norm

def norm_ref(x, w, b, eps):
    mean = x.mean(0)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(0) + eps)
    h = (x - mean) * rstd
    y = h if w is None else h * w[:, None]
    return (y if b is None else y + b[:, None]), mean, rstd, h


# One value, less than a chunk, each lane layout and its edges, past the
# registers.
WIDTHS = [1, 2, 7, 64, 100, 129, 255, 512, 1000, 2047, 4096, 8192, 10_001, 40_000]


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_layer_norm(J, T, d):
    """With a mean of 3 and deviation 1: |x| <= 8, so a mean of d values is off by
    (d/64 + 16) v 8 at most (lane sums of d/64 terms, then a tree), h by that and
    by 1e-6-scale errors of the variance, relative to rstd."""
    cols = 1 if d == 40_000 else 37
    gen = torch.Generator().manual_seed(d)
    eps, v = 1e-5, L.sums_u(T)
    X = L.colmajor(d, cols, T, gen, pad=d % 3, skip=d % 2)
    X.copy_((X.float() + 3).to(T))
    full = d % 2 == 0
    w = (torch.randn(d, generator=gen) * 0.5 + 1).to(T).cuda() if full or d == 7 else None
    b = torch.randn(d, generator=gen).to(T).cuda() if full else None
    Y = L.colmajor(d, cols, T, gen, pad=2)
    S = torch.full((cols, 2), float("nan"), dtype=torch.float64 if T == torch.float64 else torch.float32, device="cuda").t()
    assert J.execute(J.LayerNormOp, X, Y, weight=w, bias=b, eps=eps, stats=S) is Y
    x = L.f64(X)
    ref, mean, rstd, h = norm_ref(x, None if w is None else L.f64(w), None if b is None else L.f64(b), eps)
    em = (d / 64 + 16) * v * x.abs().mean(0)
    erel = (d / 64 + 24) * v + em * rstd                 # of rstd: its sum's error, and the mean's
    eh = em * rstd + erel * h.abs() + 2 * v * h.abs()
    L.close(S[0], mean, em, "mean")
    L.close(S[1], rstd, erel * rstd, "rstd")
    wa = 1.0 if w is None else L.f64(w).abs()[:, None]
    L.close(Y, ref, eh * wa + 3 * v * (ref.abs() + (0 if b is None else L.f64(b).abs()[:, None])), "Y")

    dY = L.colmajor(d, cols, T, gen, pad=1)
    out = dict(dX=torch.full_like(X, float("nan")), dweight=torch.empty(d, dtype=T, device="cuda"),
               dbias=torch.empty(d, dtype=T, device="cuda"))
    J.execute(J.LayerNormGradOp, X, dY, S, weight=w, **out)
    mean, rstd = L.f64(S)                                # the kernel goes by the stats it is given
    h, dy = (x - mean) * rstd, L.f64(dY)
    g = dy if w is None else dy * L.f64(w)[:, None]
    m1, m2 = g.mean(0), (g * h).mean(0)
    dh = 3 * v * (x.abs() + mean.abs()) * rstd           # h's own error
    e1 = (d / 64 + 16) * v * g.abs().mean(0)
    e2 = ((d / 64 + 18) * v * g.abs() * h.abs() + g.abs() * dh).mean(0)
    ex = rstd * (e1 + h.abs() * e2 + dh * m2.abs() + 6 * v * (g.abs() + m1.abs() + (h * m2).abs()))
    L.close(out["dX"], rstd * (g - m1 - h * m2), ex, "dX")
    L.close(out["dweight"], (dy * h).sum(1), ((cols + 8) * v * dy.abs() * h.abs() + dy.abs() * dh).sum(1), "dweight")
    L.close(out["dbias"], dy.sum(1), (cols + 8) * v * dy.abs().sum(1), "dbias")
    over = dY.clone(memory_format=torch.preserve_format)  # dX over dY
    J.execute(J.LayerNormGradOp, X, over, S, weight=w, dX=over)
    assert torch.equal(over, out["dX"])


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("d,cols", [(64, 100_001), (100, 20_003), (1024, 5000)])
def test_layer_norm_many_columns(J, T, d, cols):
    """More columns than workgroups: the sums over columns."""
    gen = torch.Generator().manual_seed(1)
    X, dY = L.colmajor(d, cols, T, gen), L.colmajor(d, cols, T, gen)
    S = torch.empty((cols, 2), dtype=torch.float64 if T == torch.float64 else torch.float32, device="cuda").t()
    J.execute(J.LayerNormOp, X, torch.empty_like(X), stats=S)
    dw, db = torch.empty(d, dtype=T, device="cuda"), torch.empty(d, dtype=T, device="cuda")
    J.execute(J.LayerNormGradOp, X, dY, S, dweight=dw, dbias=db)
    v, x, dy = L.sums_u(T), L.f64(X), L.f64(dY)
    mean, rstd = L.f64(S)
    h = (x - mean) * rstd
    dh = 3 * v * (x.abs() + mean.abs()) * rstd
    terms = cols / 1024 + 72                              # a lane's columns, then trees
    L.close(dw, (dy * h).sum(1), (terms * v * dy.abs() * h.abs() + dy.abs() * dh).sum(1), "dweight")
    L.close(db, dy.sum(1), terms * v * dy.abs().sum(1), "dbias")
    again = torch.empty_like(dw)
    J.execute(J.LayerNormGradOp, X, dY, S, dweight=again)
    assert torch.equal(again, dw)                         # the same sums in the same order


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("d,cols,pad,skip", [(2047, 9001, 0, 0), (1024, 17_000, 3, 1), (4096, 4200, 0, 0)])
def test_layer_norm_large_results(J, T, d, cols, pad, skip):
    """Results past the caches' size are those of the same columns in small calls, to
    the bit, and what lies between their columns stays as it was."""
    gen = torch.Generator(device="cuda").manual_seed(2)

    def matrix(fill=None):
        t = torch.empty(cols * (d + pad) + skip, dtype=T, device="cuda")
        t.normal_(generator=gen) if fill is None else t.fill_(fill)
        return t, t[skip:].view(cols, d + pad)[:, :d].t()

    X, dY = matrix()[1], matrix()[1]
    ybuf, Y = matrix(7.0)
    dbuf, dX = matrix(7.0)
    w = torch.randn(d, generator=gen, device="cuda").to(T)
    S = torch.empty((cols, 2), dtype=torch.float64 if T == torch.float64 else torch.float32, device="cuda").t()
    J.execute(J.LayerNormOp, X, Y, weight=w, bias=w, stats=S)
    J.execute(J.LayerNormGradOp, X, dY, S, weight=w, dX=dX)
    step = 500
    for c in range(0, cols, step):
        at = slice(c, c + step)
        y, dx = torch.empty_like(Y[:, at]), torch.empty_like(Y[:, at])
        J.execute(J.LayerNormOp, X[:, at], y, weight=w, bias=w)
        J.execute(J.LayerNormGradOp, X[:, at], dY[:, at], S[:, at], weight=w, dX=dx)
        assert torch.equal(Y[:, at], y) and torch.equal(dX[:, at], dx), c
    for buf in (ybuf, dbuf):
        assert torch.all(buf[:skip] == 7) and torch.all(buf[skip:].view(cols, d + pad)[:, d:] == 7)


def test_layer_norm_gradient_against_differences(J):
    """Central differences (step 1e-5) of the 64-bit form, 1e-8 for their error."""
    T, d, cols = torch.float64, 9, 4
    gen = torch.Generator().manual_seed(3)
    X, D = L.colmajor(d, cols, T, gen), L.colmajor(d, cols, T, gen)
    w, b = torch.randn(d, generator=gen, dtype=T).cuda(), torch.randn(d, generator=gen, dtype=T).cuda()
    S, Y = torch.empty((cols, 2), dtype=T, device="cuda").t(), torch.empty_like(X)
    J.execute(J.LayerNormOp, X, Y, weight=w, bias=b, stats=S)
    out = dict(dX=torch.empty_like(X), dweight=torch.empty_like(w), dbias=torch.empty_like(b))
    J.execute(J.LayerNormGradOp, X, D, S, weight=w, **out)
    base = [L.f64(X), L.f64(w), L.f64(b)]
    for at, name in enumerate(("dX", "dweight", "dbias")):
        num = torch.zeros_like(base[at])
        for i in np.ndindex(*num.shape):
            side = []
            for step in (1e-5, -1e-5):
                t = [v.clone() for v in base]
                t[at][i] += step
                side.append(float((norm_ref(*t, 1e-5)[0] * L.f64(D)).sum()))
            num[i] = (side[0] - side[1]) / 2e-5
        L.close(out[name], num, torch.full_like(num, 1e-8), name)


def test_layer_norm_degenerate(J):
    """A constant column has h = 0 and a finite rstd; NaN and infinity stay in
    their columns; no columns make zero gradients; Y may be X."""
    X = torch.randn((6, 50), device="cuda").t()
    X[:, 1], X[4, 2], X[4, 3] = 7.0, float("nan"), float("inf")
    b = torch.randn(50, device="cuda")
    Y, S = torch.empty_like(X), torch.empty((6, 2), device="cuda").t()
    J.execute(J.LayerNormOp, X, Y, bias=b, stats=S)
    assert torch.equal(Y[:, 1], b) and torch.isfinite(S[:, 1]).all()
    assert torch.isnan(Y[:, 2]).all() and torch.isnan(Y[4, 3])
    assert torch.isfinite(Y[:, [0, 4, 5]]).all()
    J.execute(J.LayerNormOp, X, X, bias=b)
    assert torch.equal(X[:, [0, 1, 4, 5]], Y[:, [0, 1, 4, 5]])
    for d in (50, 40_000):
        none = torch.empty((0, d), device="cuda").t()
        dw = torch.full((d,), float("nan"), device="cuda")
        J.execute(J.LayerNormGradOp, none, none, torch.empty((0, 2), device="cuda").t(), dX=none, dweight=dw, dbias=None)
        assert float(dw.abs().max()) == 0


# ------------------------------------------------------- streams, graphs, refusals

def test_streams_and_graphs(J):
    """On another stream, and captured: replays with eager work between them."""
    T = torch.bfloat16
    gen = torch.Generator().manual_seed(0)
    X, Y = L.colmajor(512, 40, T, gen), L.colmajor(256, 80, T, gen)
    W = weights(256, 512, 6, T, gen, "out")
    ids = torch.from_numpy(some_ids(80, 6, 3)).cuda().view(40, 2).t()
    N, S, dX, dW = torch.empty_like(X), torch.empty((40, 2), device="cuda").t(), torch.empty_like(X), torch.empty_like(W)
    w = torch.ones(512, dtype=T, device="cuda")

    def step():
        J.execute(J.LayerNormOp, X, N, weight=w, stats=S)
        h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=6)
        J.execute(h, W, N, Y)
        J.execute(J.GroupedLinearGradOp, h, W, N, Y, dX=dX, dW=dW)
        return h

    step()
    want = [t.clone() for t in (Y, dX, dW)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
        step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, (Y, dX, dW)))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        keep = step()
    for rep in range(4):
        X.uniform_(-1, 1)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (Y, dX, dW)]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (Y, dX, dW))), rep
    del keep


def test_plan_memory_on_other_streams(J, monkeypatch):
    """A plan updated or used on a stream other than the one it was made on tells
    the allocator, also when both happen on the same other stream."""
    ids = torch.tensor([1, 2, 0, 2], dtype=torch.int32, device="cuda")
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=2)
    seen = []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "record_stream", lambda t, s: seen.append((t.data_ptr(), s)))
        h.use()
        h.update(ids)
        assert not seen
        with torch.cuda.stream(side):
            h.update(ids)
            h.use()
    assert seen == [(h.offsets().data_ptr(), side)] * 2
    torch.cuda.current_stream().wait_stream(side)
    assert h.order().tolist() == [0, 1, 3, 2]


def test_refusals(J):
    T = torch.float32
    gen = torch.Generator().manual_seed(0)
    W, X, Y = weights(8, 6, None, T, gen, "out"), L.colmajor(6, 5, T, gen), L.colmajor(8, 5, T, gen)
    run = lambda *a, **k: J.execute(J.LinearOp, *a, **k)  # noqa: E731
    with pytest.raises(J.IncompatibleExtents):
        run(W, L.colmajor(7, 5, T, gen), Y)
    with pytest.raises(J.IncompatibleExtents):
        run(W, X, L.colmajor(8, 4, T, gen))
    with pytest.raises(J.IncompatibleExtents):
        run(W, X, Y, bias=torch.zeros(7, device="cuda"))
    with pytest.raises(J.IncompatibleExtents):
        run(W, X, Y, residual=L.colmajor(8, 4, T, gen))
    with pytest.raises(J.UnsupportedValueType):
        run(W, X.double(), Y)
    with pytest.raises(J.UnsupportedValueType):
        run(W.int(), X.int(), Y.int())
    with pytest.raises(J.DeviceMismatch):
        run(W, X.cpu(), Y)
    with pytest.raises(J.DeviceMismatch):
        run(W.cpu(), X.cpu(), Y.cpu())
    with pytest.raises(J.NonCanonicalStorage):
        run(W, X.contiguous(), Y)                             # row-major
    with pytest.raises(J.NonCanonicalStorage):
        run(W, X[:, :1].expand(6, 5), Y)                      # overlapping columns
    with pytest.raises(J.NonCanonicalStorage):
        run(torch.zeros((16, 12), device="cuda")[::2, ::2], X, Y)
    with pytest.raises(J.UnsupportedFormat):
        run(W, X, Y, act=J.exp_fn)
    with pytest.raises(TypeError):
        J.execute(J.LinearGradOp, W, X, Y, act=J.gelu_fn, dX=X)
    ids = torch.ones(5, dtype=torch.int32, device="cuda")
    plan = lambda i, **k: J.prepare(J.HIPBackend(), J.GroupedLinearOp, i, **k)  # noqa: E731
    with pytest.raises(J.UnsupportedIndexType):
        plan(ids.float(), n_groups=2)
    with pytest.raises(J.IncompatibleExtents):
        plan(ids, n_groups=0)
    with pytest.raises(J.IncompatibleExtents):
        plan(ids, n_groups=4096)
    with pytest.raises(J.DeviceMismatch):
        plan(ids.cpu(), n_groups=2)
    with pytest.raises(J.NonCanonicalStorage):
        plan(torch.ones(10, dtype=torch.int32, device="cuda")[::2], n_groups=2)
    h = plan(ids, n_groups=2)
    W2 = weights(8, 6, 2, T, gen, "out")
    with pytest.raises(J.IncompatibleExtents):
        J.execute(h, W, X, Y)
    with pytest.raises(J.IncompatibleExtents):
        J.execute(h, weights(8, 6, 3, T, gen, "out"), X, Y)
    with pytest.raises(J.IncompatibleExtents):
        J.execute(h, W2, L.colmajor(6, 4, T, gen), L.colmajor(8, 4, T, gen))
    with pytest.raises(J.NonCanonicalStorage):
        J.execute(J.GroupedLinearGradOp, h, W2, X, Y, dW=W2[:, :, :1].expand(8, 6, 2))
    with pytest.raises(TypeError):
        J.execute(J.GroupedLinearOp, W2, X, Y)
    with pytest.raises(J.IncompatibleExtents):
        h.update(ids[:4])
    with pytest.raises(J.IncompatibleExtents):
        J.execute(J.LayerNormOp, X, X, weight=torch.ones(5, device="cuda"))
    with pytest.raises(J.UnsupportedValueType):
        J.execute(J.LayerNormOp, X, X, stats=torch.empty((5, 2), dtype=torch.float64, device="cuda").t())
    with pytest.raises(J.IncompatibleExtents):
        J.execute(J.LayerNormOp, X, X, eps=-1.0)
    with pytest.raises(J.NonCanonicalStorage):
        J.execute(J.LayerNormOp, X, X, stats=torch.empty((2, 5), device="cuda"))


def test_elementwise_gelu_silu(J):
    """The two activations as transforms of a vector (input_fn, output_fn); the
    tails' relative accuracy needs more than 64 bits of the plain form."""
    import mpmath
    mpmath.mp.prec = 120
    many = {"gelu": lambda z: z * mpmath.erfc(-z / mpmath.sqrt(2)) / 2, "silu": lambda z: z / (1 + mpmath.exp(-z))}
    for T in (torch.float32, torch.float64):
        v = torch.linspace(-12, 12, 1001, dtype=T, device="cuda")
        z = L.f64(v)
        for f, name in ((J.gelu_fn, "gelu"), (J.silu_fn, "silu")):
            ref = torch.tensor([float(many[name](mpmath.mpf(float(t)))) for t in z], dtype=torch.float64)
            L.close(f(v), ref, 8 * L.U[T] * L.act_of(z, name).abs() * (1 + z.abs()), name)


def test_example_graph_layer(J):
    """examples/graph_layer.py: its gradients against torch's own of the same
    network in 64 bits (each result passes through a few hundred roundings of 6e-8
    at most: 1e-4 of its norm), and the loss falls."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "graph_layer.py")
    spec = importlib.util.spec_from_file_location("graph_layer", path)
    E = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(E)
    n, d, types, classes = 600, 40, 3, 7
    g = torch.Generator().manual_seed(0)
    A = E.random_graph(n, 5)
    kind = torch.randint(1, types + 1, (n,), generator=g).to(torch.int32)
    X = torch.randn(n, d, generator=g).cuda().t()
    net = E.GraphNet(A, kind.cuda(), types, d, classes)
    dS = torch.randn(n, classes, generator=g).cuda().t()
    S = net.forward(X)
    dX = net.backward(dS)
    P = {k: v.detach().cpu().double().requires_grad_() for k, v in net.p.items()}
    x = X.cpu().double().requires_grad_()
    dense = torch.zeros((n, n), dtype=torch.float64)
    rows = torch.arange(n).repeat_interleave(5)
    dense.index_put_((rows, A.crd_buffers[1].cpu().long() - 1), A.val.cpu().double(), accumulate=True)
    h = torch.nn.functional.layer_norm(x.t(), (d,), P["w"], P["s"], 1e-5)
    m = dense @ h
    z = torch.stack([P["W"][:, :, t] @ m[i] + P["b"][:, t] for i, t in enumerate((kind - 1).tolist())])
    y = torch.nn.functional.gelu(z) + x.t()
    s = y @ P["V"].t() + P["c"]
    s.backward(dS.cpu().double().t())
    near = lambda a, b: float((a.cpu().double() - b).norm() / b.norm()) < 1e-4  # noqa: E731
    assert near(S, s.detach().t()) and near(dX, x.grad)
    for k in P:
        assert near(net.grad[k], P[k].grad), k
    assert E.main(n=2000, d=32, types=3, classes=5, steps=20) < 1.6          # log 5 = 1.609 at the start
