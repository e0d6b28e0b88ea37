"""The products, grouped products and normalisations of a network's layer, as a
program calls them beside the sparse products: what they are measured by.

Every case names an `op`:

  linear    Y = act.(W*X .+ b) .+ R, or with `grad` its gradients dX, dW, db
  grouped   the same with a weight matrix per group: column p of Y takes the
            matrix of group ids[p]; `copies` consecutive columns of Y share one
            column of X (the `copies` experts of a token, ids being copies x
            cols); a column whose id names no group keeps R alone, or zeros
  norm      layer norm of every column of X, or with `grad` its gradients

A column is one token, one node of a graph or one sample.  Dense matrices are
column-major as everywhere in this library: X is `inp` x `cols` with
stride(0) == 1.  `w` says along which side W is contiguous: "out" is a
column-major out x inp matrix, "inp" the transpose of a column-major inp x out
one.  Group ids count from 1.
"""
import math

import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


# ------------------------------------------------------------------- the cases

def listed():
    return [
        # One new token through a square projection with its residual: the
        # whole weight is read for a single column.
        dict(name="linear_token", op="linear", grad=False, dtype="bf16", cols=1, inp=4096, out=4096,
             act="none", bias=True, residual=True, keep=False, w="out"),
        # A graph layer's update over every node: the node and feature counts
        # of the message-passing benchmark, neither of them round.
        dict(name="linear_graph", op="linear", grad=False, dtype="f32", cols=200003, inp=100, out=100,
             act="relu", bias=True, residual=True, keep=False, w="out"),
        # The widening product of a feed-forward block over a training batch,
        # its pre-activation kept for the backward pass.
        dict(name="linear_ffn", op="linear", grad=False, dtype="bf16", cols=8192, inp=2048, out=8192,
             act="gelu", bias=True, residual=False, keep=True, w="out"),
        # The backward pass of that product: the largest call.
        dict(name="linear_ffn_grad", op="linear", grad=True, dtype="bf16", cols=8192, inp=2048, out=8192,
             act="gelu", bias=True, residual=False, keep=True, w="inp"),
        # A few tokens in flight, two experts each: most experts see one or
        # two columns.
        dict(name="grouped_tokens", op="grouped", grad=False, dtype="bf16", cols=12, copies=2, groups=16,
             inp=2048, out=1024, skew=0.3, drop=0.0, act="silu", bias=False, residual=False, keep=False, w="inp"),
        # A weight matrix per node type of a heterogeneous graph.
        dict(name="grouped_types", op="grouped", grad=False, dtype="f32", cols=100003, copies=1, groups=7,
             inp=128, out=96, skew=0.6, drop=0.0, act="relu", bias=True, residual=True, keep=False, w="out"),
        # The experts' first product over a training batch, in half precision,
        # a quarter of the columns meant for experts that live elsewhere.
        dict(name="grouped_experts", op="grouped", grad=False, dtype="f16", cols=8192, copies=2, groups=32,
             inp=1024, out=2816, skew=0.3, drop=0.25, act="gelu", bias=True, residual=False, keep=True, w="inp"),
        # Its backward pass in bfloat16.
        dict(name="grouped_experts_grad", op="grouped", grad=True, dtype="bf16", cols=8192, copies=2, groups=32,
             inp=1024, out=2816, skew=0.3, drop=0.0, act="silu", bias=True, residual=False, keep=True, w="out"),
        # One token's normalisation: nothing but latency.
        dict(name="norm_token", op="norm", grad=False, dtype="bf16", cols=1, inp=4096),
        # Every node of a graph, backward, a feature count that is no power of
        # two.
        dict(name="norm_graph_grad", op="norm", grad=True, dtype="f32", cols=200003, inp=100),
        # A training batch, forward.
        dict(name="norm_train", op="norm", grad=False, dtype="bf16", cols=16384, inp=4096),
        # An odd batch of odd width, backward.
        dict(name="norm_odd_grad", op="norm", grad=True, dtype="f16", cols=9001, inp=2047),
    ]


def _log(rng, lo, hi):
    n = int(round(lo * (hi / lo) ** rng.random()))
    return n + 1 if n in (3072, 6144) else n


def _size(rng, lo, hi):
    """Near a logarithmic draw: a multiple of 64 (of 512 from 1,024 on), of 8,
    or whatever it is."""
    n = _log(rng, lo, hi)
    unit = rng.choice((64, 64, 8, 1))
    if unit == 64 and n >= 1024:
        unit = 512
    n = n // unit * unit
    return n - unit if n in (3072, 6144) else n


MOST = 8192 * 2048 * 8192       # products of one case: those of the largest listed one


def draw(rng):
    op = rng.choice(("linear", "linear", "grouped", "grouped", "norm"))
    grad = rng.random() < 0.4
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op == "norm":
        inp = _size(rng, 64, 8192)
        return dict(op=op, grad=grad, dtype=dtype, cols=_log(rng, 1, min(200003, 67108864 // inp)), inp=inp)
    inp, out = _size(rng, 64, 8192), _size(rng, 64, 8192)
    most = MOST // 4 if dtype == "f32" else MOST
    case = dict(op=op, grad=grad, dtype=dtype)
    if op == "linear":
        case.update(cols=_log(rng, 1, max(1, min(200003, most // (inp * out), 100000000 // max(inp, out)))))
    else:
        groups = _log(rng, 2, 64)
        while groups * inp * out > 1 << 28:
            inp, out = max(64, inp // 2), max(64, out // 2)
        copies = rng.choice((1, 2, 4))
        cols = _log(rng, 1, max(1, min(100003, most // (2 * copies * inp * out), 50000000 // (copies * max(inp, out)))))
        case.update(cols=cols, copies=copies, groups=groups, skew=rng.choice((0.0, 0.3, 0.6)),
                    drop=rng.choice((0.0, 0.0, 0.25)))
    act = rng.choice(("none", "relu", "gelu", "silu"))
    case.update(inp=inp, out=out, act=act, bias=rng.random() < 0.7, residual=not grad and rng.random() < 0.4,
                keep=act != "none" and (grad or rng.random() < 0.3), w=rng.choice(("out", "inp")))
    return case


# ------------------------------------------------------------------ the inputs

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _matrix(g, m, n, dtype, scale=1.0, shift=0.0):
    """A column-major m x n matrix of normal values."""
    t = torch.randn((n, m), generator=g, device=DEV, dtype=torch.float32)
    return t.mul_(scale).add_(shift).to(dtype).t()


def _empty(m, n, dtype):
    return torch.empty((n, m), dtype=dtype, device=DEV).t()


def prepare(case, seed):
    g, T = _gen(seed), TYPES[case["dtype"]]
    cols, inp = case["cols"], case["inp"]
    if case["op"] == "norm":
        s = dict(case=case, X=_matrix(g, inp, cols, T, 1.5, 0.25),
                 weight=(1 + 0.2 * torch.randn(inp, generator=g, device=DEV)).to(T),
                 bias=(0.2 * torch.randn(inp, generator=g, device=DEV)).to(T))
        if case["grad"]:
            x = s["X"].t().double()
            mean = x.mean(1)
            rstd = (x.var(1, unbiased=False) + EPS).rsqrt()
            s.update(dY=_matrix(g, inp, cols, T), stats=torch.stack((mean, rstd), 1).float().t(),
                     dX=_empty(inp, cols, T), dweight=torch.empty_like(s["weight"]), dbias=torch.empty_like(s["bias"]))
        else:
            s.update(Y=_empty(inp, cols, T), stats=_empty(2, cols, torch.float32))
        return s
    out, groups = case["out"], case.get("groups")
    n = cols * case.get("copies", 1)
    a, b = (out, inp) if case["w"] == "out" else (inp, out)
    W = torch.randn((groups or 1, b, a), generator=g, device=DEV, dtype=torch.float32).mul_(inp ** -0.5).to(T)
    W = W.permute(2, 1, 0) if case["w"] == "out" else W.permute(1, 2, 0)
    s = dict(case=case, X=_matrix(g, inp, cols, T), W=W if groups else W[:, :, 0], bias=None, R=None, Z=None)
    if groups:
        share = (case["skew"] * torch.randn(groups, generator=g, device=DEV)).exp()
        ids = torch.multinomial(share, n, replacement=True, generator=g) + 1
        if case["drop"]:
            ids[torch.rand(n, generator=g, device=DEV) < case["drop"]] = 0
        s["ids"] = ids.to(torch.int32)
        if case["copies"] > 1:
            s["ids"] = s["ids"].view(cols, case["copies"]).t()      # a column of ids for each column of X
    if case["bias"]:
        s["bias"] = _matrix(g, out, groups or 1, T, 0.2)
        s["bias"] = s["bias"] if groups else s["bias"][:, 0]
    if case["residual"]:
        s["R"] = _matrix(g, out, n, T)
    if case["grad"]:
        s.update(dY=_matrix(g, out, n, T), dX=_empty(inp, cols, T), dW=torch.empty_like(W) if groups else torch.empty_like(W)[:, :, 0],
                 db=None if s["bias"] is None else torch.empty_like(s["bias"]))
        if case["act"] != "none":
            s["Z"] = _matrix(g, out, n, T)      # what the forward pass kept
    else:
        s["Y"] = _empty(out, n, T)
        if case["keep"]:
            s["Z"] = _empty(out, n, T)
    return s


# ---------------------------------------------------------------- the two forms

def run(state):
    return (_own if own else _plain)(state, state["case"])


def _own(s, c):
    import jlust_amd as J
    if c["op"] == "norm":
        if c["grad"]:
            J.execute(J.LayerNormGradOp, s["X"], s["dY"], s["stats"], weight=s["weight"], dX=s["dX"],
                      dweight=s["dweight"], dbias=s["dbias"])
            return s["dX"], s["dweight"], s["dbias"]
        J.execute(J.LayerNormOp, s["X"], s["Y"], weight=s["weight"], bias=s["bias"], eps=EPS, stats=s["stats"])
        return s["Y"], s["stats"]
    act = {"none": J.identity_fn, "relu": J.relu_fn, "gelu": J.gelu_fn, "silu": J.silu_fn}[c["act"]]
    if c["op"] == "grouped":
        h = J.prepare(J.HIPBackend(), J.GroupedLinearOp, s["ids"], n_groups=c["groups"])
        if c["grad"]:
            J.execute(J.GroupedLinearGradOp, h, s["W"], s["X"], s["dY"], preact=s["Z"], act=act, dX=s["dX"],
                      dW=s["dW"], dbias=s["db"])
        else:
            J.execute(h, s["W"], s["X"], s["Y"], bias=s["bias"], act=act, residual=s["R"], preact=s["Z"])
    elif c["grad"]:
        J.execute(J.LinearGradOp, s["W"], s["X"], s["dY"], preact=s["Z"], act=act, dX=s["dX"], dW=s["dW"],
                  dbias=s["db"])
    else:
        J.execute(J.LinearOp, s["W"], s["X"], s["Y"], bias=s["bias"], act=act, residual=s["R"], preact=s["Z"])
    return _outputs(s, c)


def _outputs(s, c):
    if c["grad"]:
        return [v for v in (s["dX"], s["dW"], s["db"]) if v is not None]
    return [v for v in (s["Y"], s["Z"]) if v is not None]


def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain(s, c):
    """In 32 bits; rows of the working tensors are the columns of the case's."""
    if c["op"] == "norm":
        return _plain_norm(s, c)
    return (_plain_grouped if c["op"] == "grouped" else _plain_linear)(s, c)


def _plain_norm(s, c):
    x, w = s["X"].t().float(), s["weight"].float()
    T = s["X"].dtype
    if not c["grad"]:
        mean = x.mean(1, keepdim=True)
        d = x - mean
        rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
        return (d * rstd * w + s["bias"].float()).to(T).t(), torch.cat((mean, rstd), 1).t()
    mean, rstd = s["stats"][0, :, None], s["stats"][1, :, None]
    h = (x - mean) * rstd
    dy = s["dY"].t().float()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return dx.to(T).t(), (dy * h).sum(0).to(T), dy.sum(0).to(T)


def _plain_linear(s, c):
    T, x, w = s["X"].dtype, s["X"].t().float(), s["W"].float()
    if c["grad"]:
        g = s["dY"].t().float()
        if c["act"] != "none":
            g = g * _act_slope(s["Z"].t().float(), c["act"])
        got = [torch.matmul(g, w).to(T).t(), torch.matmul(g.t(), x).to(T)]
        return got + ([g.sum(0).to(T)] if s["bias"] is not None else [])
    z = torch.matmul(x, w.t())
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, c["act"])
    if s["R"] is not None:
        y = y + s["R"].t().float()
    return [y.to(T).t()] + ([z.to(T).t()] if s["Z"] is not None else [])


def _slots(ids, groups):
    """The columns in the order of their groups, their groups, their places in
    them, and the size of the largest group."""
    e = ids.t().reshape(-1).long() - 1
    e = torch.where((e >= 0) & (e < groups), e, groups)
    e, order = torch.sort(e, stable=True)
    counts = torch.bincount(e, minlength=groups + 1)
    first = torch.cumsum(counts, 0) - counts
    place = torch.arange(e.numel(), device=e.device) - first[e]
    used = int(first[groups])
    return order[:used], e[:used], place[:used], int(counts[:groups].max())


def _padded(v, e, place, groups, width):
    """The rows of v at [group, place] of a tensor that is zero elsewhere."""
    t = torch.zeros((groups, width, v.shape[1]), dtype=v.dtype, device=v.device)
    t[e, place] = v
    return t


def _plain_grouped(s, c):
    T, groups, copies = s["X"].dtype, c["groups"], c["copies"]
    order, e, place, width = _slots(s["ids"], groups)
    x = _padded(s["X"].t().float()[order // copies], e, place, groups, width)
    w = s["W"].permute(2, 0, 1).float()                       # group, out, inp
    n = s["ids"].numel()
    if c["grad"]:
        g = s["dY"].t().float()[order]
        if c["act"] != "none":
            g = g * _act_slope(s["Z"].t().float()[order], c["act"])
        g = _padded(g, e, place, groups, width)
        dx = torch.zeros((n, c["inp"]), device=x.device)
        dx[order] = torch.bmm(g, w.contiguous())[e, place]
        dx = dx.view(c["cols"], copies, c["inp"]).sum(1)
        dw = torch.bmm(g.transpose(1, 2).contiguous(), x)
        got = [dx.to(T).t(), dw.to(T).permute(1, 2, 0)]
        return got + ([g.sum(1).to(T).t()] if s["bias"] is not None else [])
    z = torch.bmm(x, w.transpose(1, 2).contiguous())[e, place]
    if s["bias"] is not None:
        z = z + s["bias"].t().float()[e]
    y = torch.zeros((n, c["out"]), device=x.device)
    y[order] = _act(z, c["act"])
    if s["R"] is not None:
        y = y + s["R"].t().float()
    got = [y.to(T).t()]
    if s["Z"] is not None:
        kept = torch.zeros((n, c["out"]), device=x.device)
        kept[order] = z
        got.append(kept.to(T).t())
    return got


# ------------------------------------------------------------- work, and 64 bits

def work(case):
    size = TYPES[case["dtype"]].itemsize
    cols, inp = case["cols"], case["inp"]
    if case["op"] == "norm":
        passes = 3 if case["grad"] else 2
        return dict(bytes=passes * cols * inp * size + 8 * cols + (3 if case["grad"] else 2) * inp * size,
                    flops=(14 if case["grad"] else 8) * cols * inp)
    out, n = case["out"], cols * case.get("copies", 1)
    weights = min(case.get("groups", 1), n) * inp * out
    live = 1.0 - case.get("drop", 0.0)
    if case["grad"]:
        values = 2 * cols * inp + weights + case.get("groups", 1) * inp * out + n * out * (2 if case["act"] != "none" else 1)
        return dict(bytes=values * size, flops=4 * live * n * inp * out)
    values = cols * inp + weights + n * out * (1 + case["keep"] + case["residual"])
    return dict(bytes=values * size, flops=2 * live * n * inp * out)


def _exact_slope(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, 1.0, 0.0).double()
    if act == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z.square() / 2) * (2 * math.pi) ** -0.5
    s = torch.sigmoid(z)
    return s + z * s * (1 - s)


def _exact_act(z, act):
    return {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, 0.0), "gelu": lambda: z * torch.special.ndtr(z),
            "silu": lambda: z * torch.sigmoid(z)}[act]()


def exact(case, seed):
    s = prepare(case, seed)
    X = s["X"].double()
    if case["op"] == "norm":
        d = case["inp"]
        if not case["grad"]:
            mu = X.sum(0) / d
            var = (X.square().sum(0) - d * mu.square()) / d
            r = (var + EPS).pow(-0.5)
            return (X - mu) * r * s["weight"].double()[:, None] + s["bias"].double()[:, None], torch.stack((mu, r))
        mu, r = s["stats"].double()
        H = (X - mu) * r
        G = s["weight"].double()[:, None] * s["dY"].double()
        dX = r / d * (d * G - G.sum(0) - H * (G * H).sum(0))
        return dX, (s["dY"].double() * H).sum(1), s["dY"].double().sum(1)
    W = s["W"].double() if "groups" in case else s["W"].double()[:, :, None]
    groups, copies, out = W.shape[2], case.get("copies", 1), case["out"]
    n = case["cols"] * copies
    group = s["ids"].t().reshape(-1).long() - 1 if "ids" in s else torch.zeros(n, dtype=torch.long, device=X.device)
    members = [torch.nonzero(group == k)[:, 0] for k in range(groups)]
    if case["grad"]:
        G = s["dY"].double() if s["Z"] is None else s["dY"].double() * _exact_slope(s["Z"].double(), case["act"])
        per = torch.zeros((case["inp"], n), dtype=torch.float64, device=X.device)
        dW, db = torch.zeros_like(W), torch.zeros((out, groups), dtype=torch.float64, device=X.device)
        for k, at in enumerate(members):
            if at.numel():
                per[:, at] = W[:, :, k].t().contiguous() @ G[:, at]
                dW[:, :, k] = G[:, at] @ X[:, at // copies].t().contiguous()
                db[:, k] = G[:, at].sum(1)
        dX = per.view(case["inp"], case["cols"], copies).sum(2)
        got = [dX, dW if "groups" in case else dW[:, :, 0]]
        return got + ([db if "groups" in case else db[:, 0]] if s["bias"] is not None else [])
    Z = torch.zeros((out, n), dtype=torch.float64, device=X.device)
    Y = torch.zeros_like(Z)
    for k, at in enumerate(members):
        if at.numel():
            z = W[:, :, k].contiguous() @ X[:, at // copies]
            if s["bias"] is not None:
                b = s["bias"].double()
                z = z + (b[:, k] if "groups" in case else b)[:, None]
            Z[:, at] = z
            Y[:, at] = _exact_act(z, case["act"])
    if s["R"] is not None:
        Y = Y + s["R"].double()
    return [Y] + ([Z] if s["Z"] is not None else [])
