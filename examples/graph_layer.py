"""Trains a small network on a graph with nodes of several types:

    python examples/graph_layer.py            (on a GPU)

    H  = layer_norm(X)                               one column a node
    M  = A * H'                                      sum over the neighbours (SpMM)
    Z  = W[type] * M' .+ b[type]                     a matrix per node type
    Y  = gelu.(Z) .+ X                               residual
    S  = V * Y .+ c                                  class scores

and every gradient by the operators' own: GroupedLinearGradOp, LinearGradOp,
LayerNormGradOp, and the transposed SpMM (A's arrays as CSC).  The sparse product
takes a column per feature and the layer's products a column per node, so the
features are transposed between them.
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import jlust_amd as J  # noqa: E402


def columns(rows):
    """A column-major matrix of rows.shape that holds `rows`."""
    return J.dense_matrix(*rows.shape, dtype=rows.dtype, device=rows.device).copy_(rows)


class GraphNet:
    def __init__(self, A, types, n_types, d, classes, seed=0, dtype=torch.float32):
        """A: n x n CSR; types: each node's, from 1."""
        g = torch.Generator().manual_seed(seed)
        dev = A.device

        def weights(*shape, scale):
            return (torch.randn(shape, generator=g) * scale).to(dtype).to(dev)

        n = A.extents[0]
        self.A = A
        # A' over the same arrays: rows of A are columns of A'.
        self.At = J.csc_tensor(A.pos_buffers[1], A.crd_buffers[1], A.val, (n, n), A.origin)
        self.plan = J.prepare(J.HIPBackend(), J.GroupedLinearOp, types, n_groups=n_types)
        self.p = dict(W=weights(n_types, d, d, scale=d ** -0.5).permute(2, 1, 0),       # out x inp x types
                      b=weights(n_types, d, scale=0.1).t(), w=torch.ones(d, dtype=dtype, device=dev),
                      s=torch.zeros(d, dtype=dtype, device=dev), V=weights(d, classes, scale=d ** -0.5).t(),
                      c=torch.zeros(classes, dtype=dtype, device=dev))
        self.grad = {k: torch.empty_like(v) for k, v in self.p.items()}

    def forward(self, X):
        p, d, n = self.p, *X.shape
        self.X, self.H, self.stats = X, torch.empty_like(X), J.dense_matrix(2, n, torch.float32, X.device)
        J.execute(J.LayerNormOp, X, self.H, weight=p["w"], bias=p["s"], stats=self.stats)
        M = J.dense_matrix(n, d, X.dtype, X.device)
        J.execute(J.SpMMOp, self.A, columns(self.H.t()), M)
        self.M = columns(M.t())
        self.Z, self.Y = torch.empty_like(X), torch.empty_like(X)
        J.execute(self.plan, p["W"], self.M, self.Y, bias=p["b"], act=J.gelu_fn, residual=X, preact=self.Z)
        S = J.dense_matrix(p["V"].shape[0], n, X.dtype, X.device)
        return J.execute(J.LinearOp, p["V"], self.Y, S, bias=p["c"])

    def backward(self, dS):
        """Fills self.grad from the scores' gradient and returns that of X."""
        p, g, (d, n) = self.p, self.grad, self.X.shape
        dY, dM, dH = torch.empty_like(self.X), torch.empty_like(self.X), J.dense_matrix(n, d, self.X.dtype, self.X.device)
        J.execute(J.LinearGradOp, p["V"], self.Y, dS, dX=dY, dW=g["V"], dbias=g["c"])
        J.execute(J.GroupedLinearGradOp, self.plan, p["W"], self.M, dY, act=J.gelu_fn, preact=self.Z, dX=dM, dW=g["W"],
                  dbias=g["b"])
        J.execute(J.SpMMOp, self.At, columns(dM.t()), dH)
        dX = torch.empty_like(self.X)
        J.execute(J.LayerNormGradOp, self.X, columns(dH.t()), self.stats, weight=p["w"], dX=dX, dweight=g["w"], dbias=g["s"])
        return dX.add_(dY)                       # the residual's path

    def step(self, rate):
        for k, v in self.p.items():
            v.sub_(self.grad[k], alpha=rate)


def random_graph(n, mean, seed=0, dtype=torch.float32, device="cuda"):
    """Rows of `mean` random neighbours, averaged (1-based CSR)."""
    g = torch.Generator().manual_seed(seed)
    cols = torch.sort(torch.randint(1, n + 1, (n, mean), generator=g), 1)[0].reshape(-1)
    rowptr = torch.arange(1, n * mean + 2, mean)
    t = lambda v, T: v.to(T).to(device)  # noqa: E731
    return J.csr_tensor(t(rowptr, torch.int32), t(cols, torch.int32), torch.full((n * mean,), 1.0 / mean, dtype=dtype, device=device),
                        (n, n))


def main(n=20_000, d=96, types=5, classes=10, steps=20):
    g = torch.Generator().manual_seed(1)
    A = random_graph(n, 8)
    kind = torch.randint(1, types + 1, (n,), generator=g).to(torch.int32).cuda()
    X = torch.randn(n, d, generator=g).cuda().t()
    want = torch.randint(0, classes, (n,), generator=g).cuda()
    net = GraphNet(A, kind, types, d, classes)
    for i in range(steps):
        S = net.forward(X)
        P = torch.softmax(S, 0)
        loss = -torch.log(P[want, torch.arange(n, device="cuda")]).mean()
        P[want, torch.arange(n, device="cuda")] -= 1
        net.backward(columns(P / n))
        net.step(1.0)
        if i % 5 == 0 or i == steps - 1:
            print(f"step {i:3d}  loss {float(loss):.4f}", flush=True)
    return float(loss)


if __name__ == "__main__":
    main()
