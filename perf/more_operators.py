"""What stands around a layer's experts, and its products in 8 bits, as a program
calls them: what they are measured by.

Every case names an `op`:

  route     the experts of every column of logits and their weights, or with
            `grad` the logits' gradient
  combine   Y[:, t] = sum over c of weights[c, t] * X[:, (c, t)] (+ R), the
            `copies` columns of X that belong to t being consecutive; or with
            `grad` the gradients of X and the weights
  dropout   Y = X .* mask / (1 - p) (+ R) with the mask of a counter-based
            generator; the backward pass is the same call on dY
  linear8   X's columns quantised to 8 bits with a scale each, then
            Y = act.(W*X .+ b) .+ R by products of 8-bit integers, W having a
            scale a row; with `groups` a W per group of columns, as for experts

A column is one token, one node of a graph or one sample; dense matrices are
column-major.  Expert and group ids count from 1, 0 stands for none.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------- the cases

def listed():
    return [
        # One new token is routed: nothing but latency.
        dict(name="route_token", op="route", grad=False, dtype="f32", cols=1, experts=256, copies=8, score="sigmoid",
             groups=8, keep=4, best=2, bias=True, renormalize=True, scale=2.5, pad=0.0, off=0),
        # The router of a training batch: many small experts in groups, scores
        # balanced by a bias; a few columns are padding.
        dict(name="route_batch", op="route", grad=False, dtype="f32", cols=16384, experts=256, copies=8, score="sigmoid",
             groups=8, keep=4, best=2, bias=True, renormalize=True, scale=2.5, pad=0.02, off=0),
        # The backward pass where every expert's score counts, whose products
        # are in bfloat16.
        dict(name="route_grad", op="route", grad=True, dtype="bf16", cols=16384, experts=160, copies=6, score="softmax",
             groups=1, keep=1, best=1, bias=False, renormalize=False, scale=1.0, pad=0.0, off=3),
        # One token's experts are summed, in serving.
        dict(name="combine_token", op="combine", grad=False, dtype="bf16", cols=1, copies=8, d=4096, residual=True),
        # The experts' results of a training batch are summed onto the residual.
        dict(name="combine_batch", op="combine", grad=False, dtype="bf16", cols=8192, copies=8, d=2048, residual=True),
        # Two experts a node of a graph, backward, with the node and feature
        # counts of the message-passing benchmark.
        dict(name="combine_graph_grad", op="combine", grad=True, dtype="f32", cols=200003, copies=2, d=100, residual=False),
        # Dropout of every node's features.
        dict(name="dropout_graph", op="dropout", dtype="f32", cols=200003, d=100, p=0.5, residual=False),
        # A block's output onto its residual, in training.
        dict(name="dropout_train", op="dropout", dtype="bf16", cols=16384, d=4096, p=0.1, residual=True),
        # One new token through a square projection: the weight is read for a
        # single column.
        dict(name="linear8_token", op="linear8", dtype="bf16", cols=1, inp=4096, out=4096, act="none", bias=True,
             residual=True, keep=False),
        # The widening product of a feed-forward block over a batch of prompts:
        # the largest call.
        dict(name="linear8_ffn", op="linear8", dtype="bf16", cols=8192, inp=2048, out=8192, act="gelu", bias=True,
             residual=False, keep=False),
        # A few tokens in flight, two experts each: most experts see one or two
        # columns.
        dict(name="grouped8_tokens", op="linear8", dtype="bf16", cols=12, copies=2, groups=16, inp=2048, out=1024, skew=0.3,
             drop=0.0, act="silu", bias=False, residual=False, keep=False),
        # The experts' first product over a batch of prompts, a quarter of the
        # columns meant for experts that live elsewhere.
        dict(name="grouped8_experts", op="linear8", dtype="f16", cols=8192, copies=2, groups=32, inp=1024, out=2816, skew=0.3,
             drop=0.25, act="silu", bias=True, residual=False, keep=False),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _size(rng, lo, hi):
    """Near a logarithmic draw: a multiple of 64, of 8, or whatever it is."""
    n, unit = _log(rng, lo, hi), rng.choice((64, 64, 8, 1))
    return max(unit, n // unit * unit)


MOST = 8192 * 2048 * 8192       # products of one case: those of the largest listed one


def draw(rng):
    op = rng.choice(("route", "route", "combine", "dropout", "linear8", "linear8"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        experts = groups * max(2, _log(rng, 4, 512) // groups)
        keep = rng.randint(1, groups)
        copies = min(_log(rng, 1, 16), experts // groups * keep)
        score = rng.choice(("softmax", "sigmoid"))
        return dict(op=op, grad=rng.random() < 0.4, dtype=dtype, cols=_log(rng, 1, min(100003, 8388608 // experts)),
                    experts=experts, copies=copies, score=score, groups=groups, keep=keep, best=rng.choice((1, 2)),
                    bias=rng.random() < 0.5, renormalize=rng.random() < 0.6, scale=rng.choice((1.0, 2.5)),
                    pad=rng.choice((0.0, 0.0, 0.1)), off=rng.choice((0, 0, experts // 4)))
    if op == "combine":
        d, copies = _size(rng, 64, 8192), rng.choice((1, 2, 2, 4, 6, 8))
        return dict(op=op, grad=rng.random() < 0.5, dtype=dtype, cols=_log(rng, 1, min(200003, 134217728 // (d * copies))),
                    copies=copies, d=d, residual=rng.random() < 0.5)
    if op == "dropout":
        d = _size(rng, 64, 8192)
        return dict(op=op, dtype=dtype, cols=_log(rng, 1, min(200003, 67108864 // d)), d=d, p=rng.choice((0.1, 0.1, 0.25, 0.5)),
                    residual=rng.random() < 0.5)
    inp, out = _size(rng, 64, 8192), _size(rng, 64, 8192)
    case = dict(op=op, dtype=dtype)
    if rng.random() < 0.5:
        case.update(cols=_log(rng, 1, max(1, min(100003, MOST // (inp * out), 67108864 // max(inp, out)))))
    else:
        groups, copies = _log(rng, 2, 64), rng.choice((1, 2, 4))
        while groups * inp * out > 1 << 28:
            inp, out = max(64, inp // 2), max(64, out // 2)
        cols = _log(rng, 1, max(1, min(50003, MOST // (2 * copies * inp * out), 50000000 // (copies * max(inp, out)))))
        case.update(cols=cols, copies=copies, groups=groups, skew=rng.choice((0.0, 0.3, 0.6)), drop=rng.choice((0.0, 0.0, 0.25)))
    act = rng.choice(("none", "relu", "gelu", "silu"))
    case.update(inp=inp, out=out, act=act, bias=rng.random() < 0.6, residual=rng.random() < 0.4,
                keep=act != "none" and rng.random() < 0.2)
    return case


# ------------------------------------------------------------------ the inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _matrix(g, m, n, dtype, scale=1.0):
    """A column-major m x n matrix of normal values."""
    return torch.randn((n, m), generator=g, device=DEV, dtype=torch.float32).mul_(scale).to(dtype).t()


def _empty(m, n, dtype):
    return torch.empty((n, m), dtype=dtype, device=DEV).t()


def prepare(case, seed):
    g, T, cols = _gen(seed), TYPES[case["dtype"]], case["cols"]
    return {"route": _prepare_route, "combine": _prepare_combine, "dropout": _prepare_dropout,
            "linear8": _prepare_linear8}[case["op"]](case, g, T, cols)


def _prepare_route(case, g, T, cols):
    E, copies = case["experts"], case["copies"]
    L = torch.randn((cols, E), generator=g, device=DEV).mul_(1.5)
    if case["off"]:                             # experts that cannot be chosen now
        L[:, torch.randperm(E, generator=g, device=DEV)[:case["off"]]] = -math.inf
    if case["pad"]:                             # columns that hold no token
        L[torch.rand(cols, generator=g, device=DEV) < case["pad"]] = -math.inf
    s = dict(case=case, L=L.to(T).t(), bias=None, ids=_empty(copies, cols, torch.int32))
    if case["bias"]:
        s["bias"] = 0.1 * torch.randn(E, generator=g, device=DEV)
    if case["grad"]:
        s["ids"] = _plain_route(s, case)[0].t().contiguous().t()
        s.update(dw=_matrix(g, copies, cols, torch.float32), dL=_empty(E, cols, T))
    else:
        s["weights"] = _empty(copies, cols, torch.float32)
    return s


def _prepare_combine(case, g, T, cols):
    d, copies = case["d"], case["copies"]
    w = torch.rand((cols, copies), generator=g, device=DEV) + 0.05
    s = dict(case=case, X=_matrix(g, d, cols * copies, T), weights=(w / w.sum(1, keepdim=True)).t(), R=None)
    if case["grad"]:
        s.update(dY=_matrix(g, d, cols, T), dX=_empty(d, cols * copies, T), dw=_empty(copies, cols, torch.float32))
    else:
        s.update(Y=_empty(d, cols, T), R=_matrix(g, d, cols, T) if case["residual"] else None)
    return s


def _prepare_dropout(case, g, T, cols):
    d = case["d"]
    seed, offset = torch.randint(0, 1 << 62, (2,), generator=g, device=DEV).tolist()
    return dict(case=case, X=_matrix(g, d, cols, T), R=_matrix(g, d, cols, T) if case["residual"] else None,
                Y=_empty(d, cols, T), seed=seed, offset=offset)


def _prepare_linear8(case, g, T, cols):
    inp, out, groups = case["inp"], case["out"], case.get("groups")
    n = cols * case.get("copies", 1)
    W = torch.randn((groups or 1, out, inp), generator=g, device=DEV).mul_(inp ** -0.5)
    q, sw = _quantize(W)                        # the weights are laid out in 8 bits once
    q, sw = q.to(torch.int8).permute(1, 2, 0), sw.t()
    X = torch.randn((cols, inp), generator=g, device=DEV) * (0.5 + torch.rand((cols, 1), generator=g, device=DEV))
    s = dict(case=case, W=q if groups else q[:, :, 0], sw=sw if groups else sw[:, 0], X=X.to(T).t(), bias=None, R=None, Z=None,
             Xq=_empty(inp, cols, torch.int8), sx=torch.empty(cols, device=DEV), Y=_empty(out, n, T))
    if groups:
        share = (case["skew"] * torch.randn(groups, generator=g, device=DEV)).exp()
        ids = torch.multinomial(share, n, replacement=True, generator=g) + 1
        if case["drop"]:
            ids[torch.rand(n, generator=g, device=DEV) < case["drop"]] = 0
        s["ids"] = ids.to(torch.int32)
        if case["copies"] > 1:
            s["ids"] = s["ids"].view(cols, case["copies"]).t()
    if case["bias"]:
        s["bias"] = _matrix(g, out, groups or 1, T, 0.2)
        s["bias"] = s["bias"] if groups else s["bias"][:, 0]
    if case["residual"]:
        s["R"] = _matrix(g, out, n, T)
    if case["keep"]:
        s["Z"] = _empty(out, n, T)
    return s


# ---------------------------------------------------------------- the two forms

def run(state):
    c = state["case"]
    if own:
        return {"route": _own_route, "combine": _own_combine, "dropout": _own_dropout, "linear8": _own_linear8}[c["op"]](state, c)
    return {"route": _plain_route_grad if c.get("grad") else _plain_route, "combine": _plain_combine, "dropout": _plain_dropout,
            "linear8": _plain_grouped8 if c.get("groups") else _plain_linear8}[c["op"]](state, c)


def _own_route(s, c):
    import jlust_amd as J
    if c["grad"]:
        J.execute(J.RouteGradOp, s["L"], s["ids"], s["dw"], s["dL"], score=c["score"], renormalize=c["renormalize"], scale=c["scale"])
        return [s["dL"]]
    J.execute(J.RouteOp, s["L"], s["ids"], s["weights"], bias=s["bias"], score=c["score"], groups=c["groups"], keep=c["keep"],
              best=c["best"], renormalize=c["renormalize"], scale=c["scale"])
    return s["ids"], s["weights"]


def _own_combine(s, c):
    import jlust_amd as J
    if c["grad"]:
        J.execute(J.CombineGradOp, s["X"], s["weights"], s["dY"], dX=s["dX"], dweights=s["dw"])
        return s["dX"], s["dw"]
    J.execute(J.CombineOp, s["X"], s["weights"], s["Y"], residual=s["R"])
    return [s["Y"]]


def _own_dropout(s, c):
    import jlust_amd as J
    J.execute(J.DropoutOp, s["X"], s["Y"], p=c["p"], seed=s["seed"], offset=s["offset"], residual=s["R"])
    return [s["Y"]]


def _own_linear8(s, c):
    import jlust_amd as J
    act = {"none": J.identity_fn, "relu": J.relu_fn, "gelu": J.gelu_fn, "silu": J.silu_fn}[c["act"]]
    J.execute(J.QuantizeOp, s["X"], s["Xq"], s["sx"])
    kw = dict(w_scale=s["sw"], x_scale=s["sx"], bias=s["bias"], act=act, residual=s["R"], preact=s["Z"])
    if c.get("groups"):
        h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, s["ids"], n_groups=c["groups"])
        J.execute(h, s["W"], s["Xq"], s["Y"], **kw)
    else:
        J.execute(J.LinearOp, s["W"], s["Xq"], s["Y"], **kw)
    return [v for v in (s["Y"], s["Z"]) if v is not None]


def _scores(l, score):
    """Scores of rows of logits: 0 for a logit of -inf or NaN."""
    live = l > -math.inf
    if score == "sigmoid":
        return torch.where(live, 1 / (1 + torch.exp(-l)), 0.0), live
    top = torch.where(live, l, -math.inf).amax(1, keepdim=True)
    e = torch.where(live, torch.exp(torch.where(l == top, 0.0, l - top)), 0.0)
    return torch.where(live, e / e.sum(1, keepdim=True), 0.0), live


def _plain_route(s, c):
    """In 64 bits: neighbours in the order of the scores may be close."""
    l = s["L"].t().double()
    n, E, G = l.shape[0], c["experts"], c["groups"]
    p, live = _scores(l, c["score"])
    ranked = p if s["bias"] is None else p + s["bias"].double()
    key = torch.where(live, l if s["bias"] is None else ranked, -math.inf)
    if c["keep"] < G:
        each = (torch.where(live, ranked, -math.inf) if c["best"] == 2 else key).view(n, G, E // G).sort(dim=2, descending=True)[0][:, :, :c["best"]]
        of_group = each[:, :, 0] if c["best"] == 1 else each[:, :, 0] + torch.where(each[:, :, 1] > -math.inf, each[:, :, 1], 0.0)
        kept = of_group.sort(dim=1, descending=True, stable=True)[1][:, :c["keep"]]
        mask = torch.zeros((n, G), dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        key = torch.where(mask[:, :, None].expand(n, G, E // G).reshape(n, E), key, -math.inf)
    best, at = key.sort(dim=1, descending=True, stable=True)
    best, at = best[:, :c["copies"]], at[:, :c["copies"]]
    some = best > -math.inf
    w = torch.where(some, p.gather(1, at), 0.0)
    if c["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return torch.where(some, at + 1, 0).to(torch.int32).t(), (w * c["scale"]).float().t()


def _plain_route_grad(s, c):
    l = s["L"].t().float()
    p, _ = _scores(l, c["score"])
    at = s["ids"].t().long() - 1
    some = at >= 0
    at = at.clamp_min(0)
    t = torch.where(some, s["dw"].t() * c["scale"], 0.0)
    q = torch.where(some, p.gather(1, at), 0.0)
    if c["score"] == "softmax" and not c["renormalize"]:
        dl = p * (torch.zeros_like(l).scatter_add_(1, at, t) - (q * t).sum(1, keepdim=True))
        return [dl.to(s["L"].dtype).t()]
    if c["renormalize"]:
        total = q.sum(1, keepdim=True)
        r = torch.where(total > 0, q / total, 0.0)
        g = r * (t - (r * t).sum(1, keepdim=True))
    else:
        g = t * q
    if c["score"] == "sigmoid":
        g = g * (1 - q)
    return [torch.zeros_like(l).scatter_add_(1, at, torch.where(some, g, 0.0)).to(s["L"].dtype).t()]


def _plain_combine(s, c):
    x = s["X"].t().float().view(c["cols"], c["copies"], c["d"])
    w = s["weights"].t()[:, :, None]
    if c["grad"]:
        dy = s["dY"].t().float()[:, None, :]
        return (w * dy).to(s["X"].dtype).view(-1, c["d"]).t(), (x * dy).sum(2).t()
    y = (w * x).sum(1)
    if s["R"] is not None:
        y = y + s["R"].t().float()
    return [y.to(s["X"].dtype).t()]


LOW = 0xFFFFFFFF


def _fields(seed, offset, d, cols):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): for each column of d
    elements, 8 fields of 16 bits from each counter {i / 8, j, offset}."""
    c0 = torch.arange((d + 7) // 8, device=DEV)[None, :]
    c1 = torch.arange(cols, device=DEV)[:, None]
    c2, c3 = torch.tensor(offset & LOW, device=DEV), torch.tensor(offset >> 32, device=DEV)
    k0, k1 = seed & LOW, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57         # 64 bits of each, whatever the sign
        c0, c1, c2, c3 = (b >> 32 & LOW) ^ c1 ^ k0, b & LOW, (a >> 32 & LOW) ^ c3 ^ k1, a & LOW
        k0, k1 = (k0 + 0x9E3779B9) & LOW, (k1 + 0xBB67AE85) & LOW
    words = torch.stack(torch.broadcast_tensors(c0, c1, c2, c3), 2)
    return torch.stack((words & 0xFFFF, words >> 16), 3).view(cols, -1)[:, :d]


def _plain_dropout(s, c):
    dropped = round(c["p"] * 65536)
    keep = _fields(s["seed"], s["offset"], c["d"], c["cols"]) >= dropped
    y = torch.where(keep, s["X"].t().float() * (65536 / (65536 - dropped)), 0.0)
    if s["R"] is not None:
        y = y + s["R"].t().float()
    return [y.to(s["X"].dtype).t()]


def _quantize(x):
    """Whole numbers within 127 of 0 and a 32-bit scale for the last axis; the
    quotients in 64 bits, where a value halfway between two shows."""
    x = x.double()
    scale = (x.abs().amax(-1) / 127).float()
    return torch.round(x / torch.where(scale > 0, scale, 1.0).double()[..., None]).clamp_(-127, 127), scale


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _plain_linear8(s, c):
    T, (q, sx) = s["X"].dtype, _quantize(s["X"].t())
    z = torch.matmul(q.float(), s["W"].float().t()) * sx[:, None] * s["sw"]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, c["act"])
    if s["R"] is not None:
        y = y + s["R"].t().float()
    return [y.to(T).t()] + ([z.to(T).t()] if s["Z"] is not None else [])


def _plain_grouped8(s, c):
    T, groups, copies = s["X"].dtype, c["groups"], c["copies"]
    q, sx = _quantize(s["X"].t())
    e = s["ids"].t().reshape(-1).long() - 1
    e = torch.where((e >= 0) & (e < groups), e, groups)
    e, order = torch.sort(e, stable=True)
    counts = torch.bincount(e, minlength=groups + 1)
    place = torch.arange(e.numel(), device=e.device) - (torch.cumsum(counts, 0) - counts)[e]
    used = int(counts[:groups].sum())
    order, e, place = order[:used], e[:used], place[:used]
    x = torch.zeros((groups, max(1, int(counts[:groups].max())), c["inp"]), device=e.device)
    x[e, place] = q.float()[order // copies]
    w = s["W"].permute(2, 1, 0).float().contiguous()              # group, inp, out
    z = torch.bmm(x, w)[e, place] * sx[order // copies][:, None] * s["sw"].t()[e]
    if s["bias"] is not None:
        z = z + s["bias"].t().float()[e]
    n = s["ids"].numel()
    y = torch.zeros((n, c["out"]), device=e.device)
    y[order] = _act(z, c["act"])
    if s["R"] is not None:
        y = y + s["R"].t().float()
    got = [y.to(T).t()]
    if s["Z"] is not None:
        kept = torch.zeros((n, c["out"]), device=e.device)
        kept[order] = z
        got.append(kept.to(T).t())
    return got


# ------------------------------------------------------------- work, and 64 bits

def work(case):
    size, cols = TYPES[case["dtype"]].itemsize, case["cols"]
    if case["op"] == "route":
        E, copies = case["experts"], case["copies"]
        pairs = 8 * copies * cols
        if not case["grad"]:
            return dict(bytes=E * cols * size + pairs + 4 * E * case["bias"], flops=4 * E * cols)
        dense = case["score"] == "softmax" and not case["renormalize"]
        return dict(bytes=(E + (E if dense else copies)) * cols * size + pairs, flops=(4 * E if dense else 8 * copies) * cols)
    if case["op"] == "combine":
        d, copies = case["d"], case["copies"]
        columns = 2 * copies + 1 if case["grad"] else copies + 1 + case["residual"]
        return dict(bytes=columns * d * cols * size + (8 if case["grad"] else 4) * copies * cols,
                    flops=(3 if case["grad"] else 2) * copies * d * cols)
    if case["op"] == "dropout":
        return dict(bytes=(2 + case["residual"]) * case["d"] * cols * size, flops=2 * case["d"] * cols)
    inp, out, n = case["inp"], case["out"], cols * case.get("copies", 1)
    weights = min(case.get("groups", 1), n) * inp * out
    live = 1.0 - case.get("drop", 0.0)
    return dict(bytes=cols * inp * size + weights + n * out * size * (1 + case["keep"] + case["residual"]),
                flops=2 * live * n * inp * out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        return (_exact_route_grad if case["grad"] else _exact_route)(s, case)
    if case["op"] == "combine":
        w = s["weights"].double()
        X = s["X"].double().t().reshape(case["cols"], case["copies"], case["d"])
        if case["grad"]:
            dY = s["dY"].double().t()
            per = [w[k][:, None] * dY for k in range(case["copies"])]
            dots = [torch.linalg.vecdot(X[:, k], dY) for k in range(case["copies"])]
            return torch.stack(per, 1).reshape(-1, case["d"]).t(), torch.stack(dots)
        Y = torch.zeros((case["cols"], case["d"]), dtype=torch.float64, device=X.device)
        for k in range(case["copies"]):
            Y += w[k][:, None] * X[:, k]
        return [(Y if s["R"] is None else Y + s["R"].double().t()).t()]
    if case["op"] == "dropout":
        return [_exact_dropout(s, case)]
    return _exact_linear8(s, case)


def _exact_route(s, c):
    L = s["L"].t().double().cpu().numpy()
    n, E = L.shape
    G, size = c["groups"], E // c["groups"]
    P = _exact_scores(L, c["score"])
    bias = None if s["bias"] is None else s["bias"].double().cpu().numpy()
    ids, w = np.zeros((n, c["copies"]), dtype=np.int32), np.zeros((n, c["copies"]))
    value = P if bias is None else P + bias
    order = L if bias is None else value
    value, order = np.where(np.isneginf(L), -np.inf, value), np.where(np.isneginf(L), -np.inf, order)
    if c["keep"] < G:
        parts = (order if c["best"] == 1 else value).reshape(n, G, size)
        top = parts.max(2)
        if c["best"] == 2:
            rest = parts.copy()
            np.put_along_axis(rest, parts.argmax(2)[:, :, None], -np.inf, 2)
            second = rest.max(2)
            top = top + np.where(np.isneginf(second), 0.0, second)
        first = np.argsort(-top, axis=1, kind="stable")[:, :c["keep"]]
        allowed = np.zeros((n, G), dtype=bool)
        np.put_along_axis(allowed, first, True, 1)
        order = np.where(np.repeat(allowed, size, 1), order, -np.inf)
    for k in range(c["copies"]):
        at = order.argmax(1)
        rows = np.nonzero(order[np.arange(n), at] > -np.inf)[0]
        ids[rows, k] = at[rows] + 1
        w[rows, k] = P[rows, at[rows]]
        order[rows, at[rows]] = -np.inf
    if c["renormalize"]:
        total = w.sum(1)
        w = w / np.where(total > 0, total, 1.0)[:, None]
    return torch.from_numpy(ids).t(), torch.from_numpy(w * c["scale"]).t()


def _exact_scores(L, score):
    if score == "sigmoid":
        return np.exp(-np.logaddexp(0.0, -L))
    top = L.max(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.where(np.isneginf(L), 0.0, np.exp(L - top))
    total = e.sum(1, keepdims=True)
    return e / np.where(total > 0, total, 1.0)


def _exact_route_grad(s, c):
    L = s["L"].t().double().cpu().numpy()
    at, t = s["ids"].t().cpu().numpy().astype(np.int64) - 1, s["dw"].t().double().cpu().numpy() * c["scale"]
    P = _exact_scores(L, c["score"])
    rows, ks = np.nonzero(at >= 0)
    es = at[rows, ks]
    chosen, T = np.zeros_like(P), np.zeros_like(P)
    chosen[rows, es], T[rows, es] = 1.0, t[rows, ks]
    if c["renormalize"]:
        Q = chosen * P
        total = Q.sum(1, keepdims=True)
        Q = Q / np.where(total > 0, total, 1.0)
        D = Q * (T - (Q * T).sum(1, keepdims=True))
        return [torch.from_numpy(D * (1 - P) if c["score"] == "sigmoid" else D).t()]
    if c["score"] == "sigmoid":
        return [torch.from_numpy(T * P * (1 - P)).t()]
    return [torch.from_numpy(P * T - P * (P * T).sum(1, keepdims=True)).t()]


def _exact_dropout(s, c):
    d, cols, M = c["d"], c["cols"], np.uint64(LOW)
    x = [np.broadcast_to(np.arange((d + 7) // 8, dtype=np.uint64), (cols, (d + 7) // 8)),
         np.arange(cols, dtype=np.uint64)[:, None], np.uint64(s["offset"]) & M, np.uint64(s["offset"]) >> np.uint64(32)]
    keys = [((s["seed"] + i * 0x9E3779B9) & LOW, ((s["seed"] >> 32) + i * 0xBB67AE85) & LOW) for i in range(10)]
    for a, b in keys:
        p, q = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(q >> np.uint64(32)) ^ x[1] ^ np.uint64(a), q & M, (p >> np.uint64(32)) ^ x[3] ^ np.uint64(b), p & M]
    u = np.stack([np.broadcast_to(v, (cols, (d + 7) // 8)) for v in x], -1).astype("<u4").view("<u2").reshape(cols, -1)[:, :d]
    thr = int(c["p"] * 65536 + 0.5)
    keep = torch.from_numpy((u >= thr)).to(s["X"].device).t()
    Y = s["X"].double() * keep * (65536.0 / (65536 - thr))
    return Y if s["R"] is None else Y + s["R"].double()


def _exact_linear8(s, c):
    X = s["X"].double()
    sx = (X.abs().max(0)[0] / 127).float().double()
    Q = torch.round(X / torch.where(sx > 0, sx, 1.0)).clamp(-127, 127)
    W, sw = s["W"].double(), s["sw"].double()
    if not c.get("groups"):
        W, sw = W[:, :, None], sw[:, None]
    groups, copies, out, n = W.shape[2], c.get("copies", 1), c["out"], c["cols"] * c.get("copies", 1)
    group = s["ids"].t().reshape(-1).long() - 1 if "ids" in s else torch.zeros(n, dtype=torch.long, device=X.device)
    Z = torch.zeros((out, n), dtype=torch.float64, device=X.device)
    Y = torch.zeros_like(Z)
    for k in range(groups):
        at = torch.nonzero(group == k)[:, 0]
        if at.numel():
            z = (W[:, :, k].contiguous() @ Q[:, at // copies]) * sw[:, k][:, None] * sx[at // copies]
            if s["bias"] is not None:
                b = s["bias"].double()
                z = z + (b[:, k] if c.get("groups") else b)[:, None]
            Z[:, at] = z
            Y[:, at] = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0.0), "gelu": lambda: z * torch.special.ndtr(z),
                        "silu": lambda: z * torch.sigmoid(z)}[c["act"]]()
    if s["R"] is not None:
        Y = Y + s["R"].double()
    return [Y] + ([Z] if s["Z"] is not None else [])
