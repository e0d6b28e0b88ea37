"""Routing to experts, the weighted sum of their results and dropout on the GPU
against plain 64-bit forms (tests/_experts.py, where the bounds are derived)."""
import numpy as np
import pytest
import torch

from tests import _experts as E
from tests import _layers as L

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def J():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import jlust_amd
    return jlust_amd


def sums(T):
    return torch.float64 if T == torch.float64 else torch.float32


def ints(copies, cols, pad=0):
    buf = torch.full((cols, copies + pad), -7, dtype=torch.int32, device="cuda")
    return buf, buf.t()[:copies]


def check_route(J, logits, copies, pad=0, **kw):
    """The call on `logits` (experts x cols on the GPU) against the definition."""
    T, (experts, cols) = logits.dtype, logits.shape
    ibuf, ids = ints(copies, cols, pad)
    wbuf = torch.full((cols, copies + pad), -3.0, dtype=sums(T), device="cuda")
    w = wbuf.t()[:copies]
    origin = kw.get("origin", 1)
    call = {**kw, "origin": J.ZeroBased() if origin == 0 else J.OneBased()}
    assert J.execute(J.RouteOp, logits, ids, w, **call) is ids
    ref_ids, ref_w = E.route(logits, copies, **kw, got=ids.cpu())
    assert torch.equal(ids.cpu(), ref_ids), (kw, int((ids.cpu() != ref_ids).sum()))
    u = L.sums_u(T)
    lim = E.weight_bound(logits, u, kw.get("score", "softmax"))[None, :] * ref_w.abs() + L.TINY[sums(T)]
    assert ((L.f64(w) - ref_w).abs() <= lim).all(), kw
    if pad:                                        # what lies between the columns is left alone
        assert (ibuf[:, copies:] == -7).all() and (wbuf[:, copies:] == -3.0).all()
    return ids, w


# experts, copies, groups, keep, best
SHAPES = [(1, 1, 1, 1, 1), (3, 3, 1, 1, 2), (8, 2, 1, 1, 1), (16, 1, 4, 1, 2), (60, 6, 1, 1, 1), (64, 8, 8, 3, 1), (90, 6, 3, 2, 2),
          (130, 5, 13, 5, 2), (160, 6, 8, 3, 1), (256, 8, 8, 4, 2), (257, 9, 1, 1, 1), (64, 10, 64, 17, 2), (300, 17, 20, 7, 2),
          (512, 64, 2, 1, 1), (1000, 40, 1, 1, 1), (4095, 7, 5, 3, 2)]


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_route(J, T, i):
    experts, copies, groups, keep, best = SHAPES[i]
    gen = torch.Generator().manual_seed(i)
    k = i + L.TYPES.index(T)
    for j, cols in enumerate((1, 37) if experts < 1000 else (3,)):
        logits = L.colmajor(experts, cols, T, gen, 2.0, pad=(k + j) % 3)
        bias = (torch.randn(experts, generator=gen, dtype=torch.float64) * 0.2).to(sums(T)).cuda() if (k + j) % 2 else None
        check_route(J, logits, copies, pad=j, score=("softmax", "sigmoid")[(k // 2 + j) % 2], groups=groups, keep=keep, best=best,
                    bias=bias, renormalize=(k + j) % 3 != 0, scale=(1.0, 2.5)[j], origin=(k // 2) % 2)


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("i", range(9))
def test_route_many_columns(J, T, i):
    """Enough columns for several of them a wave, a wave's last ones not all there;
    keys of a few values among them, columns without experts too."""
    experts, copies, groups, keep, best = [(5, 2, 1, 1, 1), (16, 4, 8, 3, 2), (24, 16, 2, 2, 1), (31, 3, 1, 1, 1), (64, 6, 16, 5, 2),
                                           (96, 5, 3, 2, 2), (128, 8, 4, 2, 1), (200, 20, 8, 5, 2), (256, 8, 8, 4, 2)][i]
    gen = torch.Generator().manual_seed(i)
    k = i + L.TYPES.index(T)
    cols = 4099 if i < 6 else 4097 + 64 * i
    logits = L.colmajor(experts, cols, T, gen, 2.0, pad=k % 2)
    logits[:, 5:9] = -INF
    logits[:, 100:300] = logits[:, 100:300].round()
    logits[experts // 3, 1000:2000] = NAN
    bias = (torch.randn(experts, generator=gen, dtype=torch.float64) * 0.2).to(sums(T)).cuda() if k % 2 else None
    check_route(J, logits, copies, pad=k % 3, score=("softmax", "sigmoid")[k // 2 % 2], groups=groups, keep=keep, best=best, bias=bias,
                renormalize=k % 3 != 0)


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_ties(J, T, score):
    """Equal keys go to the lower expert and the lower group: equal logits, few
    distinct ones, and biases of few distinct values on them."""
    gen = torch.Generator().manual_seed(5)
    same = torch.zeros((20, 96), dtype=T, device="cuda").t()
    few = torch.randint(-1, 2, (40, 96), generator=gen).to(T).cuda().t()
    bias = (torch.randint(0, 3, (96,), generator=gen) * 0.25).to(sums(T)).cuda()
    zero = torch.zeros(96, dtype=sums(T), device="cuda")
    for logits in (same, few):
        for b in (None, zero, bias):
            for groups, keep, best in ((1, 1, 1), (8, 3, 1), (8, 3, 2), (3, 2, 2)):
                check_route(J, logits, 7, score=score, bias=b, groups=groups, keep=keep, best=best)


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_masks(J, T, score, renormalize):
    """Columns that leave no expert, fewer than asked for, one; the type's lowest
    value, infinities and NaN among the logits, in the biases too."""
    gen = torch.Generator().manual_seed(9)
    low = torch.finfo(T).min
    host = (torch.randn((12, 24), generator=gen) * 2).to(T)
    host[0] = -INF
    host[1] = NAN
    host[2, 3:] = -INF
    host[3, 1:] = low
    host[4] = low
    host[5, ::2] = NAN
    host[6, 5] = INF
    host[7, [2, 11, 12]] = INF
    host[8, :20] = -INF
    host[9] = torch.finfo(T).max
    bias = (torch.randn(24, generator=gen) * 0.1).to(sums(T))
    bias[3], bias[4], bias[5] = -INF, NAN, INF
    logits = host.cuda().t()
    for b in (None, bias.cuda()):
        for groups, keep, best in ((1, 1, 1), (4, 2, 1), (4, 2, 2), (24, 5, 2)):
            check_route(J, logits, 5, score=score, bias=b, groups=groups, keep=keep, best=best, renormalize=renormalize)


def test_route_far_scores_keep_their_shares(J):
    """Renormalised sigmoids far below the type's range."""
    logits = torch.tensor([[-100.0, -101.0, -300.0, -99.5], [-2000.0, -2001.0, -2000.5, -2010.0], [88.0, 200.0, -3.0, 1e30]],
                          device="cuda").t()
    ids, w = check_route(J, logits, 3, score="sigmoid")
    assert torch.allclose(w.sum(0).cpu(), torch.ones(3), rtol=1e-5)


@pytest.mark.parametrize("T", L.TYPES)
def test_route_neighbours(J, T):
    """Keys whose Float32 values are equal or nearly: the order is that of the scores in
    64 bits.  Logits next to each other, the bias taking all but 1e-9 of what they
    differ by back."""
    gen = torch.Generator().manual_seed(3)
    l = (torch.randn((64, 1), generator=gen) + torch.arange(32) * 2.0 ** -7).to(T)
    s = torch.sigmoid(l.double())
    host = l.cuda().t()
    if T == torch.float64:
        bias = -s[0] + torch.randperm(32, generator=gen) * 1e-13
    else:
        bias = (-s[0] + torch.randperm(32, generator=gen) * 1e-9).float()
    check_route(J, host, 8, score="sigmoid", bias=bias.cuda())
    check_route(J, host, 4, score="sigmoid", bias=bias.cuda(), groups=8, keep=3)


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("cols", [70, 4100])
def test_route_near_keys(J, T, score, cols):
    """Columns most of whose keys lie as near to each other as Float32 has it, or are
    equal: more of them than are looked at one by one, in the last places kept, in the
    last groups kept, and where a column's neighbours have none such."""
    gen = torch.Generator().manual_seed(11)
    E_ = 96
    host = (torch.randn((cols, E_), generator=gen) * 2).to(T)
    host[::3] = host[::3, :1]
    host[1::7, 10:60] = host[1::7].amax(1, keepdim=True)
    host[2::11, 40:] = -INF
    for bias in (torch.zeros(E_), torch.randperm(E_, generator=gen) * 1e-9, torch.randint(0, 4, (E_,), generator=gen) * 2.0 ** -24):
        for groups, keep, best, copies in ((1, 1, 1, 6), (8, 3, 2, 9), (8, 3, 1, 36), (4, 1, 2, 24), (1, 1, 1, 64)):
            check_route(J, host.cuda().t(), copies, score=score, bias=bias.float().cuda(), groups=groups, keep=keep, best=best)


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("cols", [300, 4100])
def test_route_sums_of_two_signs(J, T, score, cols):
    """Groups ranked by sums of two keys near 1e5 of both signs, which leave the scores'
    differences: Float32 keys are off by up to 4e-3 there, the sums in 64 bits by 3e-11."""
    gen = torch.Generator().manual_seed(12)
    host = torch.randn((cols, 32), generator=gen).to(T)
    big = 1e5 * (1 + torch.rand((8, 1), generator=gen))
    bias = torch.cat([big, -big, -8 * big, -9 * big], 1).reshape(-1).float()
    bias[1::4] = -bias[0::4]
    for keep, copies in ((1, 2), (3, 5), (7, 8)):
        check_route(J, host.cuda().t(), copies, score=score, bias=bias.cuda(), groups=8, keep=keep, best=2)


def test_route_long_sums(J):
    """A softmax whose sum adds 123 terms of 0.9 u to 1 in turn (u = 2^-24, a group of 124
    experts): the first score is 1 - 110 u, and with its bias behind another group's -80 u."""
    u = 2.0 ** -24
    host = torch.full((2, 33, 124), -40.0)
    host[:, 0, 1:] = float(np.log(0.9 * u))
    host[:, 0, 0] = 0
    bias = torch.full((33, 124), -5.0)
    bias[0, 0], bias[2, 7] = -1, -80 * u
    ids, _ = check_route(J, host.view(2, -1).cuda().t(), 1, bias=bias.view(-1).cuda(), groups=33, keep=1, best=1)
    assert (ids == 2 * 124 + 7 + 1).all()


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("cols", [50, 4100])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_near_logits(J, T, cols, score):
    """Without a bias: logits whose last bits alone differ, equal ones, more of them than
    are looked at one by one, zeros of both signs."""
    gen = torch.Generator().manual_seed(13)
    host = (torch.randn((cols, 120), generator=gen) * 2).to(T)
    bits = {2: torch.int16, 4: torch.int32, 8: torch.int64}[host.element_size()]
    some = host[::2].view(bits)
    some[:, 30:50] = some[:, :1] + torch.randint(-9, 9, (some.shape[0], 20), generator=gen).to(bits)
    host[4::5, 60:110] = host[4::5].amax(1, keepdim=True)
    host[3::7] = (torch.randint(-1, 2, (len(host[3::7]), 120), generator=gen) * 0.0).to(T)
    for groups, keep, best, copies in ((1, 1, 1, 6), (8, 3, 2, 9), (8, 3, 1, 36), (1, 1, 1, 64)):
        check_route(J, host.cuda().t(), copies, score=score, groups=groups, keep=keep, best=best, renormalize=groups > 1)


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_far_biases(J, T, score):
    """Biases at the ends of their type, as masks have them: a group whose two best keys
    add up to less than the type holds is as good as any that is left, and of several such
    the order is that of the sums in 64 bits (Float64's own are equal where they pass it).
    The same columns 200 times over are routed by another number of lanes."""
    gen = torch.Generator().manual_seed(14)
    low = torch.finfo(sums(T)).min
    host = torch.randn((13, 16), generator=gen).to(T)
    logits, many = host.cuda().t(), host.repeat(200, 1).cuda().t()
    part = torch.tensor([0.59, 0.88, 1.0, 0.51], dtype=torch.float64).repeat_interleave(4)
    edge = torch.tensor([[0.5, 0.5], [0.25, 0.75], [0.5 + 2e-7, 0.5], [0.5, 0.5 - 2e-7]], dtype=torch.float64).repeat(1, 2).reshape(-1)
    masks = {"groups": torch.tensor([0.0] * 4 + [1.0] * 12), "all": torch.ones(16), "parts": part, "large": -part, "edge": edge,
             "one": torch.tensor([0.0, 1.0, 1.0, 1.0] * 4), "signs": torch.tensor([1.0, -1.0, 1.0, 0.0] * 4)}
    for m in masks.values():
        for alone in (False, True):                # a group of one key before one of two
            bias = (m.double() * low).to(sums(T))
            if alone:
                bias[1:4] = -INF
            for groups, keep, best, copies in ((4, 2, 2, 5), (4, 3, 2, 9), (4, 3, 1, 9), (8, 5, 2, 7), (16, 9, 2, 6), (2, 1, 2, 8)):
                kw = dict(score=score, bias=bias.cuda(), groups=groups, keep=keep, best=best)
                ids, w = check_route(J, logits, copies, **kw)
                ids2, w2 = ints(copies, 2600)[1], torch.empty((2600, copies), dtype=sums(T), device="cuda").t()
                J.execute(J.RouteOp, many, ids2, w2, **kw)
                assert torch.equal(ids2, ids.repeat(1, 200)), (groups, keep, best)
                lim = 2 * E.weight_bound(logits, L.sums_u(T), score).cuda() * w.double() + 2 * L.TINY[sums(T)]
                assert ((w2.double() - w.repeat(1, 200)).abs() <= lim.repeat(1, 200)).all()


def test_route_past_one_launch(J):
    """More columns than 2^21 workgroups take: two experts, so that the choice is a comparison
    and the weight a logistic, and the gradient p (1 - p) (dw) with p the chosen one's share."""
    cols = (1 << 25) + 37
    logits = torch.randn((cols, 2), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).t()
    ids, w = torch.empty(cols, dtype=torch.int32, device="cuda"), torch.empty(cols, device="cuda")
    J.execute(J.RouteOp, logits, ids, w, renormalize=False)
    assert torch.equal(ids, (logits[1] > logits[0]).int() + 1)
    p = torch.sigmoid((logits[0].double() - logits[1]).abs())
    u = (16 + 4 * 14 + 2) * 2.0 ** -24             # E.weight_bound of logits within 7
    assert ((w - p).abs() <= u * p).all()
    dL = torch.empty_like(logits)
    J.execute(J.RouteGradOp, logits, ids, torch.ones_like(w), dL, renormalize=False)
    g = torch.where(ids == 1, p * (1 - p), -p * (1 - p))
    assert ((dL[0] - g).abs() <= 4 * u * p).all() and ((dL[1] + g).abs() <= 4 * u * p).all()     # terms of p and p * p, twice as in test_route_grad


GRADS = [(1, 1), (5, 2), (64, 8), (160, 6), (255, 3), (513, 64), (4095, 9)]


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("experts,copies", GRADS)
def test_route_grad(J, T, score, renormalize, experts, copies):
    cols = 33 if experts < 500 else 3
    gen = torch.Generator().manual_seed(experts)
    logits = L.colmajor(experts, cols, T, gen, 2.0, pad=experts % 3)
    logits[experts // 2, 1] = -INF
    logits[:, 2] = -INF
    ids, w = ints(copies, cols, 1)[1], torch.empty((cols, copies), dtype=sums(T), device="cuda").t()
    J.execute(J.RouteOp, logits, ids, w, score=score, renormalize=renormalize, scale=1.5)
    dw = torch.randn((cols, copies + 2), generator=gen).to(sums(T)).cuda().t()[:copies]
    dL = L.colmajor(experts, cols, T, gen, pad=1).fill_(NAN)
    assert J.execute(J.RouteGradOp, logits, ids, dw, dL, score=score, renormalize=renormalize, scale=1.5) is dL
    ref, size = E.route_grad(logits, ids, dw, score, renormalize, 1.5)
    bound = 2 * E.weight_bound(logits, L.sums_u(T), score)[None, :] * size
    L.close(dL, ref, bound, "dL")


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("experts,copies", [(96, 17), (96, 40), (64, 64)])
def test_route_grad_of_many_copies(J, T, score, renormalize, experts, copies):
    """More of a column's experts than it has lanes; the last workgroup's columns not all there."""
    cols, gen = 45, torch.Generator().manual_seed(copies)
    logits = L.colmajor(experts, cols, T, gen, 2.0, pad=1)
    logits[5:50, 1] = -INF
    logits[:, 2] = -INF
    ids, w = ints(copies, cols)[1], torch.empty((cols, copies), dtype=sums(T), device="cuda").t()
    J.execute(J.RouteOp, logits, ids, w, score=score, renormalize=renormalize, scale=1.5)
    dw = torch.randn((cols, copies), generator=gen).to(sums(T)).cuda().t()
    dL = L.colmajor(experts, cols, T, gen).fill_(NAN)
    J.execute(J.RouteGradOp, logits, ids, dw, dL, score=score, renormalize=renormalize, scale=1.5)
    ref, size = E.route_grad(logits, ids, dw, score, renormalize, 1.5)
    L.close(dL, ref, 2 * E.weight_bound(logits, L.sums_u(T), score)[None, :] * size, "dL")


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("scale", [1e45, 1e-55])
def test_route_scales_past_float32(J, T, score, renormalize, scale):
    """A scale that Float32 does not hold, and weights and gradients that it does: far scores
    times a large one, large gradients times a small one; a share of 0 is 0 by any."""
    host = torch.tensor([[0.0, -30.0, -45.0, -55.0], [1.0, 0.5, -0.5, -200.0]])
    host = (host - 20 if score == "sigmoid" else host).to(T)
    logits = host.cuda().t()
    ids, w = ints(4, 2)[1], torch.empty((2, 4), dtype=sums(T), device="cuda").t()
    kw = dict(score=score, renormalize=renormalize, scale=scale)
    J.execute(J.RouteOp, logits, ids, w, **kw)
    ref_ids, ref = E.route(logits, 4, **kw)
    assert torch.equal(ids.cpu(), ref_ids)
    most, u = torch.finfo(sums(T)).max, L.sums_u(T)
    lim = E.weight_bound(logits, u, score)[None, :] * ref.abs() + L.TINY[sums(T)] * max(1.0, scale)      # a share is off by as much itself
    past = ref - lim > most
    got = L.f64(w)
    assert torch.equal(torch.isinf(got), past) and ((got - ref).abs() <= lim)[~past].all()
    dw = torch.full((2, 4), 1e30 if scale < 1 else 1e-30, dtype=sums(T), device="cuda").t()
    dw[1] *= -0.5
    dL = torch.full((2, 4), NAN, dtype=T, device="cuda").t()
    J.execute(J.RouteGradOp, logits, ids, dw, dL, **kw)
    ref, size = E.route_grad(logits, ids, dw, score, renormalize, scale)
    bound = 2 * E.weight_bound(logits, u, score)[None, :] * size
    if T != torch.float16 or scale < 1:            # Float16 does not hold the large ones
        L.close(dL, ref, bound, "dL")


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_grad_of_logits_that_are_no_numbers(J, T, score, renormalize):
    """An id whose logit is NaN has the score 0, as one of -infinity has: both have the same
    gradients."""
    gen = torch.Generator().manual_seed(6)
    a = L.colmajor(10, 5, T, gen)
    b = a.clone()
    a[3], b[3] = NAN, -INF
    ids = torch.tensor([[4, 1, 9]] * 5, dtype=torch.int32, device="cuda").t()
    dw = torch.randn((5, 3), generator=gen).to(sums(T)).cuda().t()
    got = []
    for l in (a, b):
        dL = torch.full((5, 10), NAN, dtype=T, device="cuda").t()
        J.execute(J.RouteGradOp, l, ids, dw, dL, score=score, renormalize=renormalize)
        got.append(dL)
    assert torch.equal(got[0], got[1])
    ref, size = E.route_grad(b, ids, dw, score, renormalize)
    L.close(got[0], ref, 2 * E.weight_bound(b, L.sums_u(T), score)[None, :] * size, "dL")


@pytest.mark.parametrize("score,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_grad_against_differences(J, score, renormalize):
    """sum(dw .* w) by central differences with the chosen experts kept: step 1e-5,
    1e-10 of its third derivative and 1e-11 of rounding."""
    gen = torch.Generator().manual_seed(1)
    logits = L.colmajor(12, 4, torch.float64, gen, 1.5)
    ids, w = ints(3, 4)[1], torch.empty((4, 3), dtype=torch.float64, device="cuda").t()
    J.execute(J.RouteOp, logits, ids, w, score=score, renormalize=renormalize, scale=2.0)
    dw = torch.randn((4, 3), generator=gen, dtype=torch.float64).t()
    dL = torch.empty((4, 12), dtype=torch.float64, device="cuda").t()
    J.execute(J.RouteGradOp, logits, ids, dw.cuda(), dL, score=score, renormalize=renormalize, scale=2.0)
    at = ids.cpu().long() - 1

    def loss(l):
        s = torch.softmax(l, 0) if score == "softmax" else torch.sigmoid(l)
        c = s.gather(0, at)
        return float((dw * 2.0 * (c / c.sum(0) if renormalize else c)).sum())

    base = L.f64(logits)
    for i in np.ndindex(12, 4):
        side = []
        for d in (1e-5, -1e-5):
            l = base.clone()
            l[i] += d
            side.append(loss(l))
        assert abs(float(dL[i]) - (side[0] - side[1]) / 2e-5) < 1e-8, i


def test_route_grad_of_other_ids(J):
    """Ids that name no expert count for nothing, one named twice for both."""
    gen = torch.Generator().manual_seed(4)
    logits = L.colmajor(10, 3, torch.float32, gen)
    ids = torch.tensor([[0, 4, 11], [-5, 2, 2], [2 ** 31 - 1, -2 ** 31, 1]], dtype=torch.int32, device="cuda").t()
    dw = torch.randn((3, 3), generator=gen).cuda().t()
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            dL = torch.full((3, 10), NAN, device="cuda").t()
            J.execute(J.RouteGradOp, logits, ids, dw, dL, score=score, renormalize=renormalize)
            ref, size = E.route_grad(logits, ids, dw, score, renormalize)
            L.close(dL, ref, 2 * E.weight_bound(logits, 2.0 ** -24, score)[None, :] * size, (score, renormalize))


# -------------------------------------------------------------------- combine

COMBINE = [(1, 1, 1), (7, 3, 2), (8, 1, 8), (100, 130, 2), (64, 300, 1), (333, 50, 3), (2047, 9, 5), (4100, 2, 8), (40000, 1, 4), (16, 7, 64)]


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("d,cols,copies", COMBINE)
@pytest.mark.parametrize("pad", [0, 3])
def test_combine(J, T, d, cols, copies, pad):
    gen = torch.Generator().manual_seed(d + pad)
    X = L.colmajor(d, cols * copies, T, gen, pad=pad, skip=pad)
    R = L.colmajor(d, cols, T, gen, pad=2 * pad) if (d + pad) % 2 else None
    w = torch.randn((cols, copies + pad), generator=gen).to(sums(T)).cuda().t()[:copies]
    Y = L.colmajor(d, cols, T, gen, pad=pad).fill_(NAN)
    assert J.execute(J.CombineOp, X, w, Y, residual=R) is Y
    u, x, ww = L.sums_u(T), L.f64(X).view(d, cols, copies), L.f64(w).t()
    ref, size = (x * ww).sum(2), (x * ww).abs().sum(2)
    if R is not None:
        ref, size = ref + L.f64(R), size + L.f64(R).abs()
    L.close(Y, ref, (copies + 2) * u * size, "Y")
    dY = L.colmajor(d, cols, T, gen, pad=pad)
    dX, dw = L.colmajor(d, cols * copies, T, gen, pad=pad).fill_(NAN), torch.full_like(w, NAN)
    assert J.execute(J.CombineGradOp, X, w, dY, dX=dX, dweights=dw) is dX
    g = L.f64(dY)[:, :, None]
    L.close(dX, (ww * g).reshape(d, -1), u * (ww * g).abs().reshape(d, -1), "dX")
    L.close(dw, (x * g).sum(0).t(), (d + 8) * u * (x * g).abs().sum(0).t(), "dweights")
    one, two = torch.full_like(dX, NAN), torch.full_like(w, NAN)
    J.execute(J.CombineGradOp, X, w, dY, dX=one)
    assert J.execute(J.CombineGradOp, X, w, dY, dweights=two) is two
    assert torch.equal(one, dX) and torch.equal(two, dw)


@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("d,cols,copies", [(100, 33, 1), (100, 130, 2), (250, 40, 5), (700, 9, 8), (2047, 65, 3), (2047, 1100, 1), (8, 1, 64)])
def test_combine_grad_reads_what_it_needs(J, T, d, cols, copies):
    """By the C entry: dweights without weights and dX without X, null and with no leading
    dimension, are those of the call that has both (every number of lanes a column)."""
    from jlust_amd import _lib
    gen = torch.Generator().manual_seed(d)
    X, dY = L.colmajor(d, cols * copies, T, gen), L.colmajor(d, cols, T, gen)
    w = torch.randn((cols, copies), generator=gen).to(sums(T)).cuda().t()
    dX, dw = torch.full_like(X, NAN), torch.full_like(w, NAN)
    J.execute(J.CombineGradOp, X, w, dY, dX=dX, dweights=dw)
    one, two = torch.full_like(X, NAN), torch.full_like(w, NAN)
    vt, s = {torch.float64: 0, torch.float32: 1, torch.float16: 2, torch.bfloat16: 3}[T], torch.cuda.current_stream().cuda_stream
    f = _lib.lib().jlust_hip_combine_grad
    assert f(vt, d, cols, copies, X.data_ptr(), d, 0, 0, dY.data_ptr(), d, 0, 0, two.data_ptr(), copies, s) == 0
    assert f(vt, d, cols, copies, 0, 0, w.data_ptr(), copies, dY.data_ptr(), d, one.data_ptr(), d, 0, 0, s) == 0
    torch.cuda.synchronize()
    assert torch.equal(one, dX) and torch.equal(two, dw)


@pytest.mark.parametrize("T", L.TYPES)
def test_combine_skips_weights_of_zero(J, T):
    """A column whose weight is 0 may hold anything; a NaN weight shows."""
    gen = torch.Generator().manual_seed(0)
    X = L.colmajor(50, 12, T, gen)
    w = torch.rand((4, 3), generator=gen).to(sums(T)).cuda().t()
    w[1, 0] = w[0, 2] = w[2, 2] = 0
    w[:, 3] = 0
    ref = (torch.where(L.f64(w).t()[None] != 0, L.f64(X).view(50, 4, 3), 0.0) * L.f64(w).t()).sum(2)
    for at in (1, 6, 8, 9, 10, 11):
        X[:, at] = NAN if at % 2 else INF
    Y = torch.full((4, 50), NAN, dtype=T, device="cuda").t()
    J.execute(J.CombineOp, X, w, Y)
    L.close(Y, ref, 5 * L.sums_u(T) * (ref.abs() + 10), "Y")
    assert (Y[:, 3] == 0).all()
    w[0, 0] = NAN
    J.execute(J.CombineOp, X, w, Y)
    assert torch.isnan(Y[:, 0]).all() and not torch.isnan(Y[:, 1:]).any()


def test_combine_in_place_and_empty(J):
    gen = torch.Generator().manual_seed(0)
    X, w = L.colmajor(33, 10, torch.float32, gen), torch.rand((5, 2), generator=gen).cuda().t()
    R = L.colmajor(33, 5, torch.float32, gen)
    Y = torch.empty((5, 33), device="cuda").t()
    J.execute(J.CombineOp, X, w, Y, residual=R)
    J.execute(J.CombineOp, X, w, R, residual=R)
    assert torch.equal(Y, R)
    for d, cols in ((0, 5), (33, 0)):
        z = torch.empty((cols, d), device="cuda").t()
        z2 = torch.empty((2 * cols, d), device="cuda").t()
        ww, dw = torch.ones((cols, 2), device="cuda").t(), torch.full((cols, 2), NAN, device="cuda").t()
        J.execute(J.CombineOp, z2, ww, z)
        J.execute(J.CombineGradOp, z2, ww, z, dX=z2, dweights=dw)
        assert (dw == 0).all()


def test_vectors_for_one_copy(J):
    gen = torch.Generator().manual_seed(0)
    logits = L.colmajor(9, 6, torch.float32, gen)
    ids, w = torch.empty(6, dtype=torch.int32, device="cuda"), torch.empty(6, device="cuda")
    J.execute(J.RouteOp, logits, ids, w, score="sigmoid", renormalize=False)
    ref_ids, ref_w = E.route(logits, 1, score="sigmoid", renormalize=False)
    assert torch.equal(ids.cpu(), ref_ids[0])
    X, Y = L.colmajor(5, 6, torch.float32, gen), torch.empty((6, 5), device="cuda").t()
    J.execute(J.CombineOp, X, w, Y)
    L.close(Y, L.f64(X) * L.f64(w), 3 * 2.0 ** -24 * (L.f64(X) * L.f64(w)).abs(), "Y")
    one, i1, w1 = logits[:, 0], torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, device="cuda")
    J.execute(J.RouteOp, one, i1, w1)
    assert torch.equal(i1.cpu(), E.route(logits[:, :1], 3)[0][:, 0])


# -------------------------------------------------------------------- dropout

@pytest.mark.parametrize("T", L.TYPES)
@pytest.mark.parametrize("d,cols,pad", [(1, 1, 0), (5, 3, 0), (8, 40, 0), (100, 33, 0), (1003, 7, 5), (64, 500, 8), (4099, 3, 1), (1, 700, 0)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_dropout(J, T, d, cols, pad, p):
    gen = torch.Generator().manual_seed(d)
    seed, offset = 0x123456789ABCDEF0 + d, (1 << 40) + cols
    X, R = L.colmajor(d, cols, T, gen, pad=pad, skip=pad), L.colmajor(d, cols, T, gen, pad=2 * pad) if d % 2 else None
    Y = L.colmajor(d, cols, T, gen, pad=pad).fill_(NAN)
    assert J.execute(J.DropoutOp, X, Y, p=p, seed=seed, offset=offset, residual=R) is Y
    keep, scale = E.kept(d, cols, p, seed, offset), 65536 / (65536 - E.dropped(p))
    ref = L.f64(X) * keep * scale
    bound = 2 * L.sums_u(T) * ref.abs()
    if R is not None:
        ref = ref + L.f64(R)
        bound = bound + L.sums_u(T) * ref.abs()
    L.close(Y, ref, bound, "Y")
    if R is None:
        assert ((L.f64(Y) == 0) == (~keep | (L.f64(X) == 0))).all()
    dY, dX = L.colmajor(d, cols, T, gen), torch.empty_like(X)
    J.execute(J.DropoutOp, dY, dX, p=p, seed=seed, offset=offset)
    ref = L.f64(dY) * keep * scale
    L.close(dX, ref, 2 * L.sums_u(T) * ref.abs(), "dX")
    state = torch.tensor([seed, offset], device="cuda")
    Z = torch.full_like(Y, NAN)
    J.execute(J.DropoutOp, X, Z, p=p, residual=R, state=state)
    assert torch.equal(Y, Z)


@pytest.mark.parametrize("T", L.TYPES)
def test_dropout_ends(J, T):
    """p = 0 keeps everything as it is, p = 1 nothing, NaN and infinity included; a
    dropped one is 0; results in place."""
    gen = torch.Generator().manual_seed(0)
    X, R = L.colmajor(77, 9, T, gen), L.colmajor(77, 9, T, gen)
    Y = torch.empty_like(X)
    J.execute(J.DropoutOp, X, Y, p=0.0, seed=1)
    assert torch.equal(Y, X)
    X[::3] = NAN
    X[1::3] = INF
    J.execute(J.DropoutOp, X, Y, p=1.0, seed=1)
    assert (Y == 0).all()
    J.execute(J.DropoutOp, X, Y, p=1, seed=1, residual=R)
    assert torch.equal(Y, R)
    J.execute(J.DropoutOp, X, Y, p=0.5, seed=-3, offset=(1 << 63) - 1)
    keep = E.kept(77, 9, 0.5, -3 & (1 << 64) - 1, (1 << 63) - 1)
    assert (Y.cpu()[~keep] == 0).all() and torch.isnan(Y.cpu()[::3][keep[::3]]).all()
    Z = X.clone()
    J.execute(J.DropoutOp, Z, Z, p=0.5, seed=-3, offset=(1 << 63) - 1)
    assert torch.equal(torch.nan_to_num(Z), torch.nan_to_num(Y))
    e = torch.empty((0, 4), dtype=T, device="cuda").t()
    J.execute(J.DropoutOp, e, e, p=0.5, seed=0)


def test_dropout_share(J):
    """Of 2^24 elements a tenth is dropped (7 standard deviations are 0.00052), other
    offsets and seeds drop others, independently."""
    X = torch.ones((4096, 4096), device="cuda").t()
    masks = []
    for seed, offset in ((1, 0), (1, 1), (2, 0)):
        Y = torch.empty_like(X)
        J.execute(J.DropoutOp, X, Y, p=0.1, seed=seed, offset=offset)
        masks.append(Y == 0)
        assert abs(float(masks[-1].double().mean()) - E.dropped(0.1) / 65536) < 0.00052
    for a, b in ((0, 1), (0, 2), (1, 2)):       # both dropped: 1 %, 7 deviations are 0.00017
        assert abs(float((masks[a] & masks[b]).double().mean()) - (E.dropped(0.1) / 65536) ** 2) < 0.00017


# ------------------------------------------------------------- together, streams

def block(J, T, gen, d, hidden, experts, copies, cols):
    dev = dict(dtype=T, device="cuda")
    f32 = dict(dtype=sums(T), device="cuda")
    n = copies * cols
    s = dict(X=L.colmajor(d, cols, T, gen), Wr=L.colmajor(experts, d, T, gen, d ** -0.5),
             W1=(torch.randn((experts, d, hidden), generator=gen) * d ** -0.5).to(T).cuda().permute(2, 1, 0),
             W2=(torch.randn((experts, hidden, d), generator=gen) * hidden ** -0.5).to(T).cuda().permute(2, 1, 0),
             bias=(torch.randn(experts, generator=gen) * 0.1).to(sums(T)).cuda(), dY=L.colmajor(d, cols, T, gen))
    for name, shape in dict(logits=(cols, experts), H=(n, hidden), Z=(n, hidden), O=(n, d), S=(cols, d), Y=(cols, d), dS=(cols, d), dO=(n, d),
                            dH=(n, hidden), dX=(cols, d), dXr=(cols, d), dL=(cols, experts)).items():
        s[name] = torch.full(shape, NAN, **dev).t()
    s.update(ids=torch.empty((cols, copies), dtype=torch.int32, device="cuda").t(), w=torch.empty((cols, copies), **f32).t(),
             dw=torch.empty((cols, copies), **f32).t(), dW1=torch.empty_like(s["W1"]), dW2=torch.empty_like(s["W2"]),
             dWr=torch.empty_like(s["Wr"]), state=torch.tensor([7, 1], device="cuda"))
    J.execute(J.LinearOp, s["Wr"], s["X"], s["logits"])
    J.execute(J.RouteOp, s["logits"], s["ids"], s["w"], bias=s["bias"], score="sigmoid", scale=1.5)
    s["plan"] = J.prepare(J.HIPBackend(), J.GroupedLinearOp, s["ids"], n_groups=experts)
    return s


def run_block(J, s, p):
    """A layer of experts, forward and backward, by the framework's calls."""
    J.execute(J.LinearOp, s["Wr"], s["X"], s["logits"])
    J.execute(J.RouteOp, s["logits"], s["ids"], s["w"], bias=s["bias"], score="sigmoid", scale=1.5)
    h = s["plan"].update(s["ids"])
    J.execute(h, s["W1"], s["X"], s["H"], act=J.gelu_fn, preact=s["Z"])
    h2 = s["plan2"].update(s["ids"].t().reshape(-1))
    J.execute(h2, s["W2"], s["H"], s["O"])
    J.execute(J.CombineOp, s["O"], s["w"], s["S"])
    J.execute(J.DropoutOp, s["S"], s["Y"], p=p, state=s["state"], residual=s["X"])
    J.execute(J.DropoutOp, s["dY"], s["dS"], p=p, state=s["state"])
    J.execute(J.CombineGradOp, s["O"], s["w"], s["dS"], dX=s["dO"], dweights=s["dw"])
    J.execute(J.GroupedLinearGradOp, h2, s["W2"], s["H"], s["dO"], dX=s["dH"], dW=s["dW2"])
    J.execute(J.GroupedLinearGradOp, h, s["W1"], s["X"], s["dH"], act=J.gelu_fn, preact=s["Z"], dX=s["dX"], dW=s["dW1"])
    J.execute(J.RouteGradOp, s["logits"], s["ids"], s["dw"], s["dL"], score="sigmoid", scale=1.5)
    J.execute(J.LinearGradOp, s["Wr"], s["X"], s["dL"], dX=s["dXr"], dW=s["dWr"])


def make_block(J, T, *shape):
    s = block(J, T, torch.Generator().manual_seed(3), *shape)
    s["plan2"] = J.prepare(J.HIPBackend(), J.GroupedLinearOp, s["ids"].t().reshape(-1), n_groups=shape[2])
    return s


def test_offsets_past_32_bits(J):
    """Columns 2^20 values apart, the last of them past 2^32: the same as side by side."""
    T, far, n = torch.bfloat16, 1 << 20, 4100
    gen = torch.Generator().manual_seed(2)

    def apart(t, fill=0):
        buf = torch.empty(far * (t.shape[1] - 1) + t.shape[0], dtype=t.dtype, device="cuda")
        v = torch.as_strided(buf, t.shape, (1, far))
        v.copy_(t) if fill is not None else None
        return v

    X, w = L.colmajor(40, n, T, gen), torch.rand((n // 2, 2), generator=gen).cuda().t()
    logits = L.colmajor(16, n, T, gen)
    far_x, far_l = apart(X), apart(logits)

    def calls(x, l, like):
        ids, lw = like(torch.empty((n, 3), dtype=torch.int32, device="cuda").t()), like(torch.empty((n, 3), device="cuda").t())
        y, s, dx = like(torch.empty_like(X)), like(torch.empty((n // 2, 40), dtype=T, device="cuda").t()), like(torch.empty_like(X))
        q, qs, dl = like(torch.empty((n, 40), dtype=torch.int8, device="cuda").t()), torch.empty(n, device="cuda"), like(torch.empty_like(logits))
        dw = torch.empty((n // 2, 2), device="cuda").t()
        J.execute(J.RouteOp, l, ids, lw)
        J.execute(J.RouteGradOp, l, ids, lw, dl)
        J.execute(J.CombineOp, x, w, s)
        J.execute(J.CombineGradOp, x, w, s, dX=dx, dweights=dw)
        J.execute(J.DropoutOp, x, y, p=0.25, seed=5, offset=6)
        J.execute(J.QuantizeOp, x, q, qs)
        Y = like(torch.empty((n, 40), dtype=T, device="cuda").t())
        J.execute(J.LinearOp, q[:, :40].t().contiguous(), q, Y, w_scale=qs[:40], x_scale=qs)
        return ids, lw, dl, s, dx, dw, y, q, qs, Y

    for near, away in zip(calls(X, logits, lambda t: t), calls(far_x, far_l, lambda t: apart(t, None))):
        assert torch.equal(near, away)


def test_layer_of_experts(J):
    """Route, experts, sum, dropout and residual, and back, in Float64 against autograd
    of the formulas (both off by some 1e-13 of values near 1: 1e-10 is far from both)."""
    T, d, hidden, experts, copies, cols, p = torch.float64, 24, 40, 10, 3, 50, 0.25
    s = make_block(J, T, d, hidden, experts, copies, cols)
    run_block(J, s, p)
    X, Wr, W1, W2 = (L.f64(s[k]).requires_grad_() for k in ("X", "Wr", "W1", "W2"))
    logits = Wr @ X
    ids, _ = E.route(logits, copies, bias=s["bias"], score="sigmoid", scale=1.5)
    assert torch.equal(ids, s["ids"].cpu())
    q = torch.sigmoid(logits).gather(0, ids.long() - 1)
    w = 1.5 * q / q.sum(0)
    cols_out = []
    for t in range(cols):
        out = 0
        for c in range(copies):
            e = int(ids[c, t]) - 1
            z = W1[:, :, e] @ X[:, t]
            out = out + w[c, t] * (W2[:, :, e] @ (0.5 * z * torch.erfc(-z * 0.5 ** 0.5)))
        cols_out.append(out)
    keep = E.kept(d, cols, p, 7, 1).double() * (65536 / (65536 - E.dropped(p)))
    Y = torch.stack(cols_out, 1) * keep + X
    (Y * L.f64(s["dY"])).sum().backward()
    for got, ref in ((s["Y"], Y.detach()), (s["dW1"], W1.grad), (s["dW2"], W2.grad), (s["dWr"], Wr.grad),
                     (s["dX"].double() + s["dXr"] + s["dY"], X.grad)):
        assert (L.f64(got) - ref).abs().max() < 1e-10


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
def test_layer_of_experts_in_a_graph(J, T):
    """Captured once and replayed with new inputs and dropout states, every replay the
    same bits as the calls themselves, with eager work between."""
    shape = (64, 96, 12, 2, 200)
    s = make_block(J, T, *shape)
    names = ("ids", "w", "Y", "dw", "dL", "dX", "dXr", "dW1", "dW2", "dWr")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_block(J, s, 0.1)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            run_block(J, s, 0.1)
    torch.cuda.synchronize()
    gen = torch.Generator().manual_seed(8)
    for r in range(4):
        s["X"].copy_(torch.randn((shape[4], shape[0]), generator=gen).to(T).t())
        s["state"].copy_(torch.tensor([7, 100 + r]))
        for k in names:
            s[k].zero_()
        g.replay()
        torch.cuda.synchronize()
        got = {k: s[k].clone() for k in names}
        for k in names:
            s[k].zero_()
        run_block(J, s, 0.1)
        torch.cuda.synchronize()
        for k in names:
            assert torch.equal(got[k], s[k]), (r, k)


def test_two_streams_at_once(J):
    """Calls on two streams, each with its own operands, and twice on one."""
    a, b = make_block(J, torch.float32, 64, 96, 12, 2, 300), make_block(J, torch.float32, 64, 96, 12, 2, 300)
    b["state"].copy_(torch.tensor([9, 9]))
    b["X"].mul_(0.5)
    names = ("ids", "w", "Y", "dL", "dX", "dXr", "dW1", "dW2", "dWr")
    run_block(J, a, 0.2)
    run_block(J, b, 0.2)
    torch.cuda.synchronize()
    want = [{k: s[k].clone() for k in names} for s in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in (a, b):
        for k in names:
            s[k].zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for st, s in zip(streams, (a, b)):
            with torch.cuda.stream(st):
                run_block(J, s, 0.2)
    torch.cuda.synchronize()
    for s, ref in zip((a, b), want):
        for k in names:
            assert torch.equal(s[k], ref[k]), k
