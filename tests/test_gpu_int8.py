"""Columns in 8 bits and the products of 8-bit integers on the GPU against plain
64-bit forms (tests/_experts.py): whole numbers and scales are the same ones, products
within the rounding of their scales."""
import numpy as np
import pytest
import torch

from tests import _experts as E
from tests import _layers as L

pytestmark = pytest.mark.gpu

NAN = float("nan")
OUT = [torch.bfloat16, torch.float16, torch.float32]
ACTS = [None, "relu", "gelu", "silu"]


@pytest.fixture(scope="module")
def J():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import jlust_amd
    return jlust_amd


def fn(J, act):
    return {None: None, "relu": J.relu_fn, "gelu": J.gelu_fn, "silu": J.silu_fn}[act]


def bytes_(m, n, gen, pad=0, skip=0, lo=-127, hi=127):
    """A column-major Int8 m x n matrix, its columns `pad` apart, 99 around it."""
    ld = m + pad
    buf = torch.full((max(n, 1) * ld + skip + 8,), 99, dtype=torch.int8, device="cuda")
    t = torch.as_strided(buf, (m, n), (1, ld), skip)
    t.copy_(torch.randint(lo, hi + 1, (n, m), generator=gen).to(torch.int8).t())
    return t


def check_quantize(J, X, pad=0):
    d, cols = X.shape
    buf = torch.full((max(cols, 1) * (d + pad) + 8,), 99, dtype=torch.int8, device="cuda")
    Q, s = torch.as_strided(buf, (d, cols), (1, d + pad)), torch.full((cols,), -1.0, device="cuda")
    assert J.execute(J.QuantizeOp, X, Q, s) is Q
    ref, scale = E.quantize(X)
    assert torch.equal(Q.cpu().double(), ref), int((Q.cpu().double() != ref).sum())
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(scale))
    assert torch.equal(torch.nan_to_num(s.cpu().double(), nan=-2.0), torch.nan_to_num(scale, nan=-2.0))
    if pad and cols > 1:
        assert (torch.as_strided(buf, (pad, cols - 1), (1, d + pad), d) == 99).all()
    return Q, s


@pytest.mark.parametrize("T", OUT)
@pytest.mark.parametrize("d,cols", [(1, 1), (3, 7), (8, 5), (127, 33), (128, 1), (500, 4), (1000, 3), (2047, 5), (4100, 3), (8200, 2),
                                    (16385, 2), (40001, 2)])
@pytest.mark.parametrize("pad", [0, 5])
def test_quantize(J, T, d, cols, pad):
    gen = torch.Generator().manual_seed(d)
    check_quantize(J, L.colmajor(d, cols, T, gen, 3.0, pad=pad, skip=pad), pad=pad)


@pytest.mark.parametrize("T", OUT)
def test_quantize_halves_and_ends(J, T):
    """Values halfway between two whole numbers go to the even one, those next to it do
    not; columns of zeros, of one value, of infinities and NaN, of the type's least and
    largest values."""
    k = torch.arange(-127, 128).double()
    rows = [torch.cat((k, k[:-1] + 0.5)) * s for s in (1.0, 0.25, 2.0 ** -9)]
    rows.append(torch.zeros(509, dtype=torch.double))
    rows.append(torch.full((509,), -3.25, dtype=torch.double))
    rows.append(torch.linspace(-1, 1, 509, dtype=torch.double) * torch.finfo(T).max)
    rows.append(torch.linspace(-100, 100, 509, dtype=torch.double) * float(L.TINY[T]))
    rows.append(torch.linspace(-190, 190, 509, dtype=torch.double) * 2.0 ** -149)
    rows.append(torch.linspace(-1, 1, 509, dtype=torch.double) * 2.0 ** -121)
    host = torch.stack(rows).to(T)
    near = host[:3].clone()
    i = near.view(torch.int32 if T == torch.float32 else torch.int16)
    i += torch.where(torch.arange(509) % 2 == 0, 1, -1).to(i.dtype) * (host[:3] != 0).to(i.dtype)
    near[:, 0], near[:, 254] = host[:3, 0], host[:3, 254]
    bad = host[:2].clone()
    bad[0, 7], bad[1, 400] = NAN, -float("inf")
    check_quantize(J, torch.cat((host, near, bad)).cuda().t())


@pytest.mark.parametrize("T", OUT)
def test_quantize_many_values(J, T):
    """A million quotients at scales of every mantissa."""
    gen = torch.Generator().manual_seed(2)
    host = torch.randn((500, 2048), generator=gen, dtype=torch.float64) * torch.exp(4 * torch.randn((500, 1), generator=gen).double())
    check_quantize(J, host.to(T).cuda().t())


def test_quantize_empty(J):
    s = torch.full((4,), -1.0, device="cuda")
    J.execute(J.QuantizeOp, torch.empty((4, 0), device="cuda").t(), torch.empty((4, 0), dtype=torch.int8, device="cuda").t(), s)
    assert (s == 0).all()
    J.execute(J.QuantizeOp, torch.empty((0, 3), device="cuda").t(), torch.empty((0, 3), dtype=torch.int8, device="cuda").t(), s[:0])


def case(seed, T, out, inp, cols, bias, residual, groups=None, copies=1, pad=0, skip=0):
    gen = torch.Generator().manual_seed(seed)
    n, ld = cols * copies, inp + pad
    buf = torch.full(((groups or 1) * out * ld + skip + 16,), 99, dtype=torch.int8, device="cuda")
    W = torch.as_strided(buf, (out, inp, groups or 1), (ld, 1, ld * out), skip)
    W.copy_(torch.randint(-127, 128, (groups or 1, out, inp), generator=gen).to(torch.int8).permute(1, 2, 0))
    s = dict(W=W if groups else W[:, :, 0], Xq=bytes_(inp, cols, gen, pad, skip),
             ws=(torch.rand((groups or 1, out), generator=gen) * 0.1 / max(inp, 1) ** 0.5).cuda().t(),
             xs=(torch.rand(cols, generator=gen) * 0.02).cuda(), Y=L.colmajor(out, n, T, gen, pad=pad).fill_(NAN),
             Z=L.colmajor(out, n, T, gen, pad=pad).fill_(NAN), R=L.colmajor(out, n, T, gen, pad=pad) if residual else None,
             b=L.colmajor(out, groups or 1, T, gen, 0.5) if bias else None)
    if not groups:
        s["ws"] = s["ws"][:, 0].contiguous()
        s["b"] = None if s["b"] is None else s["b"][:, 0]
    return s


def check(J, s, T, act, ids=None, copies=1, h=None, keep=True):
    ref, refz, ey, ez = E.linear8(s["W"], s["ws"], s["Xq"], s["xs"], T, s["b"], act, s["R"], ids, copies)
    kw = dict(w_scale=s["ws"], x_scale=s["xs"], bias=s["b"], act=fn(J, act), residual=s["R"], preact=s["Z"] if keep else None)
    r = J.execute(J.LinearOp, s["W"], s["Xq"], s["Y"], **kw) if h is None else J.execute(h, s["W"], s["Xq"], s["Y"], **kw)
    assert r is s["Y"]
    L.close(s["Y"], ref, ey, "Y")
    if keep:
        L.close(s["Z"], refz, ez, "Z")


SIZES = [(1, 1, 1), (3, 5, 2), (17, 33, 5), (64, 128, 16), (130, 70, 33), (257, 129, 100), (128, 64, 300), (300, 1000, 2), (8, 4096, 1),
         (100, 96, 1000), (72, 520, 700), (2000, 129, 49), (129, 2000, 17), (1, 300, 65)]


@pytest.mark.parametrize("T", OUT)
@pytest.mark.parametrize("i", range(len(SIZES)))
@pytest.mark.parametrize("pad,skip", [(0, 0), (16, 16), (3, 1)])
def test_linear_int8(J, T, i, pad, skip):
    out, inp, cols = SIZES[i]
    k = i + OUT.index(T) + pad
    check(J, case(i, T, out, inp, cols, k % 3 != 0, k % 2 == 0, pad=pad, skip=skip), T, ACTS[k % 4], keep=k % 5 != 0)


@pytest.mark.parametrize("T,out,inp,cols,groups,copies", [c[:6] for c in E.PLANNED8])
def test_linear_int8_kernels(J, T, out, inp, cols, groups, copies):
    """Every kernel and pieces of k (tests/_experts.py says which), no edge whole."""
    T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[T]
    s = case(out + cols, T, out, inp, cols, True, cols % 3 == 0, groups or None, copies)
    act = ACTS[(out + cols) % 4]
    if not groups:
        return check(J, s, T, act)
    gen = torch.Generator().manual_seed(cols)
    ids = torch.randint(0, groups + 1, (cols, copies), generator=gen, dtype=torch.int32).cuda()
    ids = ids.t() if copies > 1 else ids[:, 0].contiguous()
    check(J, s, T, act, ids, copies, J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=groups))


@pytest.mark.parametrize("T,out,inp,cols,groups,copies,woff,xoff,shared", [c[:9] for c in E.PACKED8])
def test_linear_int8_packed(J, T, out, inp, cols, groups, copies, woff, xoff, shared):
    """Operands that lie badly for copies are packed first (tests/_experts.py says which);
    the same once more, into the scratch that holds the last ones."""
    T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[T]
    s = case(out + cols, T, out, inp, cols, True, woff > 0, 1 if shared else groups or None, copies)
    for k, off in (("W", woff), ("Xq", xoff)):
        if off:
            v = s[k]
            buf = torch.zeros(v.numel() + 16, dtype=torch.int8, device="cuda")
            s[k] = torch.as_strided(buf, v.shape, v.stride(), off)
            s[k].copy_(v)
    if shared:
        s["W"] = s["W"].expand(-1, -1, groups)
        s["ws"], s["b"] = s["ws"].expand(-1, groups).t().contiguous().t(), s["b"].expand(-1, groups).t().contiguous().t()
    ids = h = None
    if groups:
        ids = torch.randint(0, groups + 1, (cols, copies), generator=torch.Generator().manual_seed(cols), dtype=torch.int32).cuda().t()
        h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=groups)
    check(J, s, T, "silu", ids, copies, h)
    s["Xq"].neg_()
    check(J, s, T, None, ids, copies, h, keep=False)


def test_packed_int8_in_a_graph(J):
    """A product that packs its operands, captured after a call of its size and replayed."""
    s = case(1, torch.bfloat16, 2053, 1033, 2500, True, False)
    kw = dict(w_scale=s["ws"], x_scale=s["xs"], bias=s["b"], act=J.gelu_fn)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        J.execute(J.LinearOp, s["W"], s["Xq"], s["Y"], **kw)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            J.execute(J.LinearOp, s["W"], s["Xq"], s["Y"], **kw)
    torch.cuda.synchronize()
    for r in range(3):
        s["Xq"].copy_(s["Xq"].roll(1, 0))
        s["Y"].zero_()
        g.replay()
        torch.cuda.synchronize()
        got = s["Y"].clone()
        J.execute(J.LinearOp, s["W"], s["Xq"], s["Y"], **kw)
        torch.cuda.synchronize()
        assert torch.equal(got, s["Y"]), r


@pytest.mark.parametrize("cols", [1, 40, 300])
def test_sums_at_the_end_of_32_bits(J, cols):
    """131,071 products of -128 and -128 are 2^31 - 2^14."""
    inp = (1 << 17) - 1
    W, X = (torch.full((n, inp), -128, dtype=torch.int8, device="cuda") for n in (20, cols))
    W[3] = 127
    Y = torch.empty((cols, 20), device="cuda").t()
    one = torch.ones(max(20, cols), device="cuda")
    J.execute(J.LinearOp, W, X.t(), Y, w_scale=one[:20], x_scale=one[:cols])
    ref = torch.full((20, cols), 128.0 * 128 * inp, dtype=torch.float64)
    ref[3] = -127.0 * 128 * inp
    assert torch.equal(Y.cpu().double(), ref.float().double())


GROUPED = [(17, 33, 5, 2, 3), (64, 128, 40, 2, 16), (130, 70, 333, 1, 7), (128, 1024, 12, 2, 16), (257, 512, 700, 2, 3), (96, 200, 500, 4, 70),
           (300, 528, 3000, 1, 2), (40, 64, 3, 1, 100)]


@pytest.mark.parametrize("T", OUT)
@pytest.mark.parametrize("i", range(len(GROUPED)))
@pytest.mark.parametrize("pad", [0, 3])
def test_grouped_int8(J, T, i, pad):
    """Groups without columns, of one and of many; columns of no group, whose scale of
    NaN does not count; the copies' order."""
    out, inp, cols, copies, groups = GROUPED[i]
    k = i + OUT.index(T) + pad
    gen = torch.Generator().manual_seed(i)
    s = case(i, T, out, inp, cols, k % 3 != 0, k % 2 == 0, groups, copies, pad)
    ids = torch.randint(0, groups + 1, (cols, copies), generator=gen, dtype=torch.int32)
    ids[torch.rand((cols, copies), generator=gen) < 0.3] = min(2, groups)
    if cols > 3:
        ids[1] = 0
        s["xs"][1] = NAN
    ids = ids.cuda().t() if copies > 1 else ids[:, 0].contiguous().cuda()
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=groups)
    check(J, s, T, ACTS[k % 4], ids, copies, h)
    for k in ("Y", "Z"):
        assert not torch.isnan(s[k]).any()


def test_grouped_int8_shared_matrix(J):
    """One matrix for all groups, its scales each group's own."""
    s = case(4, torch.float32, 50, 80, 60, True, False, 3, 1)
    one = s["W"][:, :, :1]
    s["W"] = one.expand(-1, -1, 3)
    ids = torch.randint(0, 4, (60,), dtype=torch.int32, generator=torch.Generator().manual_seed(1)).cuda()
    check(J, s, torch.float32, "relu", ids, 1, J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=3))


def test_scales_that_are_not_numbers(J):
    """NaN and infinite scales show in their rows and columns alone."""
    s = case(2, torch.float32, 40, 64, 50, False, False)
    J.execute(J.LinearOp, s["W"], s["Xq"], s["Y"], w_scale=s["ws"], x_scale=s["xs"])
    good = s["Y"].clone()
    s["ws"][7], s["xs"][20] = NAN, NAN
    J.execute(J.LinearOp, s["W"], s["Xq"], s["Y"], w_scale=s["ws"], x_scale=s["xs"])
    mask = torch.zeros((40, 50), dtype=torch.bool, device="cuda")
    mask[7], mask[:, 20] = True, True
    assert torch.equal(torch.isnan(s["Y"]), mask) and torch.equal(s["Y"][~mask], good[~mask])


@pytest.mark.parametrize("T,out,inp,cols,groups,copies", [c[:6] for c in E.PLANNED8])
def test_scales_far_from_one(J, T, out, inp, cols, groups, copies):
    """Scales over all of Float32, negative ones too, by every kernel: a result is right where it is within
    its type's range, though the product of its scales may not be; a sum of 0 gives the bias."""
    T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[T]
    s = case(out + cols, T, out, inp, cols, True, False, groups or None, copies)
    gen = torch.Generator().manual_seed(inp)

    def far(n):
        x = torch.exp2(torch.rand(n, generator=gen, dtype=torch.float64) * 276 - 149) * torch.where(torch.rand(n, generator=gen) < 0.5, -1.0, 1.0)
        return x.float()

    s["ws"].copy_(far(s["ws"].shape))
    s["xs"].copy_(far(s["xs"].shape))
    s["W"][3], s["Xq"][:, cols // 2] = 0, 0
    ids = h = None
    if groups:
        ids = torch.randint(0, groups + 1, (cols, copies), generator=gen, dtype=torch.int32).cuda()
        ids = ids.t() if copies > 1 else ids[:, 0].contiguous()
        h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=groups)
    J.execute(J.LinearOp if h is None else h, s["W"], s["Xq"], s["Y"], w_scale=s["ws"], x_scale=s["xs"], bias=s["b"])
    ref, _, bound, _ = E.linear8(s["W"], s["ws"], s["Xq"], s["xs"], T, s["b"], None, None, ids, copies)
    got, most = L.f64(s["Y"]), torch.finfo(T).max
    lim = bound + L.U[T] * ref.abs() + 2.0 ** -149
    past, within = ref.abs() - lim > most, ref.abs() + lim <= most
    assert past.any() and within.any()
    assert torch.equal(got[past], torch.sign(ref[past]) * float("inf"))
    zero = torch.zeros_like(ref)
    L.close(torch.where(within, got, zero).to(T), torch.where(within, ref, zero), torch.where(within, bound, zero), "Y")


def test_in_place_residual_and_empty(J):
    s = case(3, torch.bfloat16, 70, 96, 20, True, True)
    kw = dict(w_scale=s["ws"], x_scale=s["xs"], bias=s["b"])
    J.execute(J.LinearOp, s["W"], s["Xq"], s["Y"], residual=s["R"], **kw)
    J.execute(J.LinearOp, s["W"], s["Xq"], s["R"], residual=s["R"], **kw)
    assert torch.equal(s["Y"], s["R"])
    for out, inp, cols in ((0, 5, 3), (5, 0, 3), (5, 4, 0)):
        e = case(1, torch.float32, out, inp, cols, True, False)
        J.execute(J.LinearOp, e["W"], e["Xq"], e["Y"], w_scale=e["ws"], x_scale=e["xs"], bias=e["b"])
        if inp == 0:
            assert torch.equal(e["Y"], e["b"][:, None].expand(5, 3))


@pytest.mark.parametrize("cols", [1, 64, 700])
def test_quantized_layer(J, cols):
    """A layer's product as it is served, weights and columns quantised by the
    framework: within their rounding of the product itself.  Each value is off by at
    most half its scale, so a sum by (|W| xs + |X| ws)/2 + xs ws/4 summed over inp."""
    gen = torch.Generator().manual_seed(cols)
    inp, out = 1024, 520
    W = (torch.randn((out, inp), generator=gen) * inp ** -0.5).cuda()
    X = torch.randn((cols, inp), generator=gen).cuda().t()
    Wq, ws = torch.empty((out, inp), dtype=torch.int8, device="cuda"), torch.empty(out, device="cuda")
    Xq, xs = torch.empty((cols, inp), dtype=torch.int8, device="cuda").t(), torch.empty(cols, device="cuda")
    J.execute(J.QuantizeOp, W.t(), Wq.t(), ws)
    J.execute(J.QuantizeOp, X, Xq, xs)
    Y = torch.empty((cols, out), device="cuda").t()
    J.execute(J.LinearOp, Wq, Xq, Y, w_scale=ws, x_scale=xs)
    w, x, a, b = L.f64(W), L.f64(X), L.f64(ws)[:, None], L.f64(xs)[None, :]
    lim = w.abs().sum(1)[:, None] * b / 2 + a * x.abs().sum(0)[None, :] / 2 + inp * a * b / 4
    assert ((L.f64(Y) - w @ x).abs() <= 1.0001 * lim).all()


def test_int8_in_a_graph(J):
    """Quantise, plan and grouped product, captured and replayed with new columns."""
    T = torch.bfloat16
    s = case(6, T, 200, 256, 90, True, False, 5, 2)
    X = torch.randn((90, 256), device="cuda").to(T).t()
    ids = torch.randint(0, 6, (90, 2), dtype=torch.int32, device="cuda").t()
    h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, ids, n_groups=5)

    def go():
        J.execute(J.QuantizeOp, X, s["Xq"], s["xs"])
        J.execute(h.update(ids), s["W"], s["Xq"], s["Y"], w_scale=s["ws"], x_scale=s["xs"], bias=s["b"], act=J.silu_fn)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        go()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            go()
    torch.cuda.synchronize()
    gen = torch.Generator().manual_seed(1)
    for r in range(4):
        X.copy_(torch.randn((90, 256), generator=gen).to(T).t())
        ids.copy_(torch.randint(0, 6, (90, 2), generator=gen, dtype=torch.int32).t())
        s["Y"].zero_()
        g.replay()
        torch.cuda.synchronize()
        got = s["Y"].clone()
        s["Y"].zero_()
        go()
        torch.cuda.synchronize()
        assert torch.equal(got, s["Y"]), r
