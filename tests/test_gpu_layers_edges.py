"""Layer operators on the GPU where they went wrong once, or where the chosen
kernel has to be named: against the plain 64-bit forms of tests/_layers.py."""
import pytest
import torch

from tests import _layer_cases as C
from tests import _layers as L
from tests.test_gpu_layers import case, check_forward, check_grad, some_ids, weights

pytestmark = pytest.mark.gpu

TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def J():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import jlust_amd
    return jlust_amd


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["out", "inp"])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_groups_that_share_a_matrix(J, T, layout, act):
    """W.expand over the groups, its rows off any alignment, in products large enough
    to pack it first: the bits of the same call on a matrix per group, and the 64-bit
    form at some columns."""
    out, inp, cols, groups = 1000, 1024, 16384, 3
    s = case(1, T, out, inp, cols, layout, act, True, False, groups, pad=0)
    one = weights(out, inp, 1, T, torch.Generator().manual_seed(9), layout, pad=1, skip=1)
    shared, apart = one.expand(out, inp, groups), weights(out, inp, groups, T, torch.Generator(), layout, pad=1, skip=1)
    assert shared.stride(2) == 0
    apart.copy_(shared)
    ids = torch.from_numpy(some_ids(cols, groups, 4, 0.1)).cuda()
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=groups)
    fn = {None: None, "gelu": J.gelu_fn}[act]
    Y = torch.empty_like(s["Y"])
    J.execute(h, apart, s["X"], Y, bias=s["b"], act=fn)
    J.execute(h, shared, s["X"], s["Y"], bias=s["b"], act=fn, preact=s["Z"])
    assert torch.equal(s["Y"], Y)
    at = list(range(0, cols, 97)) + [cols - 1]
    ref, refz, ey, ez = L.forward(apart, s["X"][:, at], s["b"], act, None, ids[at], 1)
    L.close(s["Y"][:, at], ref, ey, "Y")
    L.close(s["Z"][:, at], refz, ez, "Z")

    dY = torch.randn((cols, out), generator=torch.Generator().manual_seed(5)).to(T).cuda().t()
    got = []
    for W in (apart, shared):
        dX, dW = torch.empty_like(s["X"]), torch.empty_like(apart)
        J.execute(J.GroupedLinearGradOp, h, W, s["X"], dY, act=fn, preact=s["Z"] if act else None, dX=dX, dW=dW)
        only = torch.empty_like(dX)
        J.execute(J.GroupedLinearGradOp, h, W, s["X"], dY, act=fn, preact=s["Z"] if act else None, dX=only)
        got.append((dX, dW, only))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    ref = L.gradients(apart, s["X"][:, at], dY[:, at], s["Z"][:, at], act, ids[at], 1)["dX"]
    for i in (0, 2):
        L.close(got[1][i][:, at], *ref, "dX")


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("layout", ["out", "inp"])
@pytest.mark.parametrize("out,inp", [(40, 70), (70, 40), (1, 9), (9, 1)])
@pytest.mark.parametrize("groups", [None, 3])
def test_gradient_of_the_other_layout(J, T, layout, out, inp, groups):
    """dW contiguous along the other side than W, with dX and dbias and alone: the
    64-bit form, and dX and dbias as in the call with dW laid out as W."""
    s = case(2, T, out, inp, 50, layout, "relu", True, False, groups)
    gen = torch.Generator().manual_seed(3)
    dY, Z = (L.colmajor(out, 50, T, gen) for _ in range(2))
    ids = h = None
    if groups:
        ids = torch.from_numpy(some_ids(50, groups, 4, 0.1)).cuda()
        h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=groups)
    ref = L.gradients(s["W"], s["X"], dY, Z, "relu", ids, 1)

    def run(**out):
        for v in out.values():
            v.fill_(float("nan"))
        op = (J.LinearGradOp,) if h is None else (J.GroupedLinearGradOp, h)
        J.execute(*op, s["W"], s["X"], dY, act=J.relu_fn, preact=Z, **out)
        return out

    same = run(dX=torch.empty_like(s["X"]), dW=torch.empty_like(s["W"]), dbias=torch.empty_like(s["b"]))
    other = lambda: weights(out, inp, groups, T, gen, "inp" if layout == "out" else "out")  # noqa: E731
    full, alone = run(dX=torch.empty_like(s["X"]), dW=other(), dbias=torch.empty_like(s["b"])), run(dW=other())
    assert torch.equal(full["dX"], same["dX"]) and torch.equal(full["dbias"], same["dbias"])
    for got in (full, alone):
        L.close(got["dW"], *ref["dW"], "dW")


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cols", [60, 3000])
@pytest.mark.parametrize("other", [False, True])
def test_gradient_of_interleaved_groups(J, T, cols, other):
    """dW and dbias whose groups lie within each other's leading dimension (an inp x
    groups x out array, or its transpose's), beside W as it is usual; what overlaps
    is refused before anything is written."""
    out, inp, groups = 72, 40, 3
    s = case(6, T, out, inp, cols, "out", None, True, False, groups)
    dY = L.colmajor(out, cols, T, torch.Generator().manual_seed(1))
    ids = torch.from_numpy(some_ids(cols, groups, 4, 0.1)).cuda()
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=groups)
    ref = L.gradients(s["W"], s["X"], dY, None, None, ids, 1)
    a, b = (inp, out) if other else (out, inp)
    dW = torch.full((b, groups, a), float("nan"), dtype=T, device="cuda").permute(2, 0, 1)
    dW = dW.transpose(0, 1) if other else dW
    dX, db = torch.full_like(s["X"], float("nan")), torch.full_like(s["b"], float("nan"))
    J.execute(J.GroupedLinearGradOp, h, s["W"], s["X"], dY, dX=dX, dW=dW, dbias=db)
    for k, v in (("dX", dX), ("dW", dW), ("dbias", db)):
        L.close(v, *ref[k], k)
    buf = torch.zeros(groups * (a + 1) * b + 64, dtype=T, device="cuda")
    over = torch.as_strided(buf, (a, b, groups), (1, a + 1, a * b))
    over = over.transpose(0, 1) if other else over
    dX.fill_(5)
    for bad in (dict(dW=over, dbias=db), dict(dW=dW, dbias=db[:, :1].expand(out, groups))):
        with pytest.raises(J.NonCanonicalStorage):
            J.execute(J.GroupedLinearGradOp, h, s["W"], s["X"], dY, dX=dX, **bad)
    assert (dX == 5).all() and (buf == 0).all()


def test_more_rows_than_a_launch_has_threads_for(J):
    """134 million columns: a launch of 32 threads for each would pass 2^32 threads.
    All but a few columns are zero, so that the 64-bit form takes those alone."""
    T, inp, out, cols = torch.float16, 8, 8, (1 << 27) + 40
    gen = torch.Generator().manual_seed(0)
    at = [0, 5, (1 << 26) + 3, (1 << 27) - 1, 1 << 27, cols - 1]
    W, X, dY = (weights(out, inp, 2, T, gen, "out"), torch.zeros((cols, inp), dtype=T, device="cuda").t(),
                torch.zeros((cols, out), dtype=T, device="cuda").t())
    X[:, at], dY[:, at] = (torch.randn((8, len(at)), generator=gen).to(T).cuda() for _ in range(2))
    ids = torch.ones(cols, dtype=torch.int32, device="cuda")
    ids[at[1::2]] = 2
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=2)
    dX, dW = torch.full((cols, inp), 7.0, dtype=T, device="cuda").t(), torch.empty_like(W)
    J.execute(J.GroupedLinearGradOp, h, W, X, dY, dX=dX, dW=dW)
    ref = L.gradients(W, X[:, at], dY[:, at], None, None, ids[at], 1)
    L.close(dX[:, at], *ref["dX"], "dX")
    L.close(dW, *ref["dW"], "dW")
    assert int(torch.count_nonzero(dX)) == int(torch.count_nonzero(dX[:, at]))


def test_longest_columns_sums(J):
    """dweight and dbias of a column of 134 million values, and zeros without columns."""
    T, d = torch.float16, (1 << 27) + 40
    X = torch.empty((1, d), dtype=T, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1)).t()
    dY, S = X.flip(0).t().contiguous().t(), torch.tensor([[0.25, 2.0]], device="cuda").t()
    dw, db = torch.full((d,), 7.0, dtype=T, device="cuda"), torch.full((d,), 7.0, dtype=T, device="cuda")
    J.execute(J.LayerNormGradOp, X, dY, S, dweight=dw, dbias=db)
    assert torch.equal(db, dY[:, 0])
    assert torch.equal(dw, (dY[:, 0].float() * ((X[:, 0].float() - 0.25) * 2.0)).to(T))
    none = torch.empty((0, d), dtype=T, device="cuda").t()
    J.execute(J.LayerNormGradOp, none, none, torch.empty((0, 2), device="cuda").t(), dweight=dw, dbias=db)
    assert not dw.any() and not db.any()


def test_bias_of_the_longest_columns(J):
    """dbias of columns of 134 million values, by groups and without."""
    T, out = torch.float16, (1 << 27) + 40
    dY = torch.empty((2, out), dtype=T, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1)).t()
    W, X = torch.zeros((1, out), dtype=T, device="cuda").t(), torch.zeros((2, 1), dtype=T, device="cuda").t()
    db = torch.full((out,), 7.0, dtype=T, device="cuda")
    J.execute(J.LinearGradOp, W, X, dY, dbias=db)
    assert torch.equal(db, (dY[:, 0].float() + dY[:, 1].float()).to(T))
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, torch.tensor([2, 0], dtype=torch.int32, device="cuda"), n_groups=2)
    db = torch.full((2, out), 7.0, dtype=T, device="cuda").t()
    J.execute(J.GroupedLinearGradOp, h, W[:, :, None].expand(out, 1, 2), X, dY, dbias=db)
    assert torch.equal(db[:, 1], dY[:, 0]) and not db[:, 0].any()


@pytest.mark.parametrize("i", range(len(C.PLANNED)))
def test_planned(J, monkeypatch, i):
    """The products of tests/_layer_cases.py, in the kernels that they are there for."""
    T, out, inp, cols, layout, groups, pad, act, forward, dX, dW = C.PLANNED[i]
    s = case(i, TYPES[T], out, inp, cols, layout, act, True, i % 2 == 0, groups or None, pad=pad)
    ids = h = None
    if groups:
        ids = torch.from_numpy(some_ids(cols, groups, i, 0.1)).cuda()
        h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=groups)
    made = []
    for name in ("_LINEAR", "_LINEAR_GRAD"):
        pack = getattr(C.layers, name)
        monkeypatch.setattr(C.layers, name, lambda *a, pack=pack: made.append(pack(*a)) or made[-1])
    check_forward(J, s, ids, 1, h)
    check_grad(J, s, ids, 1, h, seed=i)
    assert C.info(made[0])[:5] == forward
    assert tuple(v[:5] for v in C.info(made[1], True)) == (dX, dW)


@pytest.mark.parametrize("n", [4095, 4096, 4097, 8191])
@pytest.mark.parametrize("groups", [999, 1000, 1001])
def test_group_plan_of_one_workgroup(J, n, groups):
    """About the most columns and groups that one workgroup sorts."""
    import numpy as np
    ids = some_ids(n, groups, n + groups)
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, torch.from_numpy(ids).cuda(), n_groups=groups)
    bins = np.where((ids >= 1) & (ids <= groups), ids - 1, groups)
    assert np.array_equal(h.order().cpu().numpy(), np.argsort(bins, kind="stable"))
    want = np.concatenate([[0], np.cumsum(np.bincount(bins, minlength=groups + 1))])[: groups + 1]
    assert np.array_equal(h.offsets().cpu().numpy(), want)
