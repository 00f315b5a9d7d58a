"""Trains a small mixture of experts on the nodes of a graph:

    python -m powersparse_amd.examples.expert_nodes [--nodes N] [--steps K] [--seed S]

Every node carries a token (a community's tokens are more frequent in it); the model
predicts the node's community from its neighbourhood:

    x  = EmbeddingLookup(table, token)          learned features
    h  = SpMM(graph, x)                         mean over the neighbours
    router -> top 2 experts a node              ExpertSort, ExpertDispatch
    expert products, weighted sum               torch, ExpertCombine
    logits -> cross entropy

The gradients run back through ExpertCombineGrad, ExpertDispatchGrad, SpMM of the
transposed graph and EmbeddingGrad, and are clipped by their global norm before the
update. Products of dense matrices are torch's; everything that follows ids or edges is
this framework's, wrapped for autograd below.
"""
import argparse

import numpy as np
import torch

import powersparse_amd as ps


def _stream():
    return torch.cuda.current_stream().cuda_stream


class Lookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, ids, scale):
        out = torch.empty((ids.numel(), table.shape[1]), dtype=table.dtype, device=table.device)
        ps.EmbeddingLookup(table, ids, out, scale=scale, stream=_stream())
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale = table.shape[0], scale
        return out

    @staticmethod
    def backward(ctx, grad_out):
        ids, = ctx.saved_tensors
        grad_out = grad_out.contiguous()
        n, cols = grad_out.shape
        grad = torch.empty((ctx.rows, cols), dtype=grad_out.dtype, device=grad_out.device)
        work = torch.empty(ps.embedding_grad_workspace_bytes(n, cols, ctx.rows),
                           dtype=torch.uint8, device=grad_out.device)
        ps.EmbeddingGrad(ids, grad_out, grad, work, scale=ctx.scale, stream=_stream())
        return grad, None, None


class Aggregate(torch.autograd.Function):
    """graph @ x; `back` is the transposed graph's matrix."""

    @staticmethod
    def forward(ctx, x, graph, back):
        ctx.back, ctx.graph = back, graph
        return Aggregate.spmm(graph, x)

    @staticmethod
    def backward(ctx, grad_out):
        return Aggregate.spmm(ctx.back, grad_out.contiguous()), None, None

    @staticmethod
    def spmm(matrix, b):
        c = torch.zeros((matrix.MatrixRow(), b.shape[1]), device=b.device)
        ps.SpMMAsync(matrix, b.shape[1], b.data_ptr(), c.data_ptr(), stream=_stream())
        return c


class Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position):
        xs = x.new_zeros((position.numel(), x.shape[1]))
        ps.ExpertDispatch(x, position, xs, stream=_stream())
        ctx.save_for_backward(position)
        return xs

    @staticmethod
    def backward(ctx, dxs):
        position, = ctx.saved_tensors
        dx = dxs.new_empty((position.shape[0], dxs.shape[1]))
        ps.ExpertDispatchGrad(dxs.contiguous(), position, dx, stream=_stream())
        return dx, None


class Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, position, weights):
        y = ys.new_empty((position.shape[0], ys.shape[1]))
        ps.ExpertCombine(ys, position, weights, y, stream=_stream())
        ctx.save_for_backward(ys, position, weights)
        return y

    @staticmethod
    def backward(ctx, dy):
        ys, position, weights = ctx.saved_tensors
        dys, dweights = torch.zeros_like(ys), torch.empty_like(weights)
        ps.ExpertCombineGrad(dy.contiguous(), ys, position, weights, dys, dweights,
                             stream=_stream())
        return dys, None, dweights


def sort_slots(ids, experts):
    """(position, slots per expert) of the routed slots."""
    order = torch.empty(ids.numel(), dtype=torch.int32, device=ids.device)
    position = torch.empty(tuple(ids.shape), dtype=torch.int32, device=ids.device)
    offsets = torch.empty(experts + 1, dtype=torch.int32, device=ids.device)
    work = torch.empty(ps.expert_sort_workspace_bytes(ids.numel(), experts), dtype=torch.uint8,
                       device=ids.device)
    ps.ExpertSort(ids, order, position, offsets, work, stream=_stream())
    return position, torch.diff(offsets).tolist()


class Model:
    """Parameters, and the forward pass over all nodes."""

    def __init__(self, tokens, classes, width=64, experts=8, top_k=2, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, std):
            return (torch.randn(shape, generator=g, device="cuda") * std).requires_grad_()

        self.top_k, self.experts, self.scale = top_k, experts, width ** 0.5
        self.table = normal(tokens, width, std=1.0 / width)
        self.router = normal(width, experts, std=0.1)
        self.expert = [normal(width, width, std=width ** -0.5) for _ in range(experts)]
        self.out = normal(width, classes, std=width ** -0.5)

    def parameters(self):
        return [self.table, self.router, self.out] + self.expert

    def logits(self, token, graph, back):
        h = Aggregate.apply(Lookup.apply(self.table, token, self.scale), graph, back)
        top = (h @ self.router).topk(self.top_k, dim=1)
        weights = torch.softmax(top.values, dim=1)
        position, counts = sort_slots(top.indices, self.experts)
        xs = Dispatch.apply(h, position)
        # (no slot is dropped here: the segments are the whole of xs)
        ys = torch.cat([torch.relu(part @ w) for part, w in zip(xs.split(counts), self.expert)])
        return Combine.apply(ys, position, weights) @ self.out + h @ self.out


def graph_and_transpose(csr):
    """Matrices of the row-normalised graph (every node its own neighbour too) and of its
    transpose, and the normalised values as a host COO list."""
    deg = np.diff(csr.row_ptr)
    row = np.concatenate([np.repeat(np.arange(csr.rows), deg), np.arange(csr.rows)])
    col = np.concatenate([csr.col_ind, np.arange(csr.rows)])
    val = (1.0 / (1.0 + deg))[row].astype(np.float32)

    def matrix(r, c):
        order = np.lexsort((c, r))
        ptr = np.concatenate([[0], np.cumsum(np.bincount(r, minlength=csr.rows))])
        return ps.PowerSparseMatrixGPU(csr.rows, csr.rows, r.size, ptr, c[order], val[order])

    return matrix(row, col), matrix(col, row), (row, col, val)


def problem(nodes, classes=16, tokens=2000, seed=0):
    """A community graph, a token for every node and its community."""
    block = max(nodes // classes, 1)
    csr = ps.synth_community(classes, block, min(0.5, 12.0 / block), 2.0, 0.02, 0.02, seed=seed + 1)
    rng = np.random.default_rng(seed)
    label = np.arange(csr.rows) // block
    own = rng.integers(0, tokens // classes, csr.rows) * classes + label
    token = np.where(rng.random(csr.rows) < 0.3, own, rng.integers(0, tokens, csr.rows))
    return csr, torch.from_numpy(token).cuda(), torch.from_numpy(label).cuda(), tokens


def train(nodes=8192, steps=60, seed=0, max_norm=0.1, rate=5.0, say=print):
    """Losses and gradient norms of the steps."""
    csr, token, label, tokens = problem(nodes, seed=seed)
    graph, back, _ = graph_and_transpose(csr)
    model = Model(tokens, int(label.max()) + 1, seed=seed)
    params = model.parameters()
    for p in params:
        p.grad = torch.zeros_like(p)
    grads = ps.GradientList([p.grad for p in params])  # they stay where they are
    norm = torch.empty(1, device="cuda")
    losses, norms = [], []
    for step in range(steps):
        loss = torch.nn.functional.cross_entropy(model.logits(token, graph, back), label)
        with torch.no_grad():
            for p in params:
                p.grad.zero_()
        loss.backward()
        ps.ClipGradNorm(grads, max_norm, norm, stream=_stream())
        with torch.no_grad():
            for p in params:
                p -= rate * p.grad
        losses.append(float(loss.detach()))
        norms.append(float(norm))
        if step % 10 == 0 or step == steps - 1:
            say(f"step {step}: loss {losses[-1]:.4f}, gradient norm {norms[-1]:.4f}")
    return losses, norms


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--nodes", type=int, default=8192)
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--seed", type=int, default=0)
    a = parser.parse_args()
    ps.set_device(0)
    train(a.nodes, a.steps, a.seed)


if __name__ == "__main__":
    main()
