"""Trains a small mixture of experts on the nodes of a graph:

    python -m powersparse_amd.examples.expert_nodes [--nodes N] [--steps K] [--seed S]
        [--norm] [--balance C] [--adamw {32,8}]

Every node carries a token (a community's tokens are more frequent in it); the model
predicts the node's community from its neighbourhood:

    x  = EmbeddingLookup(table, token)          learned features
    h  = SpMM(graph, x)                         mean over the neighbours
    n  = LayerNorm(h)                           with --norm, else h
    router -> top 2 experts a node              ExpertRoute, ExpertSort, ExpertDispatch
    expert products, weighted sum               torch, ExpertCombine
    logits -> cross entropy                     + C times the router's balance loss

The gradients run back through ExpertCombineGrad, ExpertDispatchGrad, ExpertRouteGrad,
LayerNormGrad, SpMM of the transposed graph and EmbeddingGrad, and are clipped by their
global norm before the update, or with --adamw on the way of AdamW's, whose moments are
kept in 32 or 8 bits. Products of dense matrices are torch's; everything else is this
framework's, wrapped for autograd below.
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


class Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        y, mean = torch.empty_like(x), torch.empty(x.shape[0], device=x.device)
        rstd = torch.empty_like(mean)
        ps.LayerNorm(x, weight, bias, y, mean, rstd, stream=_stream())
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dweight, dbias = torch.empty_like(x), torch.empty_like(weight), torch.empty_like(weight)
        work = torch.empty(ps.layer_norm_grad_workspace_bytes(*x.shape), dtype=torch.uint8,
                           device=x.device)
        ps.LayerNormGrad(dy.contiguous(), x, weight, mean, rstd, dx, dweight, dbias, work,
                         stream=_stream())
        return dx, dweight, dbias


class Route(torch.autograd.Function):
    """(ids, weights, balance loss) of the top_k experts by the rows of `logits`."""

    @staticmethod
    def forward(ctx, logits, top_k):
        tokens, experts = logits.shape
        ids = torch.empty((tokens, top_k), dtype=torch.int32, device=logits.device)
        counts = torch.empty(experts + 1, dtype=torch.int32, device=logits.device)
        weights, loss = logits.new_empty((tokens, top_k)), logits.new_empty(1)
        work = torch.empty(ps.expert_route_workspace_bytes(tokens, experts), dtype=torch.uint8,
                           device=logits.device)
        ps.ExpertRoute(logits, ids, weights, counts, loss, work, stream=_stream())
        ctx.save_for_backward(logits, ids, counts)
        ctx.mark_non_differentiable(ids)
        return ids, weights, loss

    @staticmethod
    def backward(ctx, _, dweights, dloss):
        logits, ids, counts = ctx.saved_tensors
        dlogits = torch.empty_like(logits)
        ps.ExpertRouteGrad(logits, ids, dweights.contiguous(), counts, dloss.contiguous(), dlogits,
                           stream=_stream())
        return dlogits, None


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

    def __init__(self, tokens, classes, width=64, experts=8, top_k=2, seed=0, norm=False):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape, std):
            return (torch.randn(shape, generator=g, device="cuda") * std).requires_grad_()

        self.top_k, self.experts, self.scale = top_k, experts, width ** 0.5
        self.table = normal(tokens, width, std=1.0 / width)
        self.router = normal(width, experts, std=0.1)
        self.expert = [normal(width, width, std=width ** -0.5) for _ in range(experts)]
        self.out = normal(width, classes, std=width ** -0.5)
        self.norm = None
        if norm:
            self.norm = [torch.ones(width, device="cuda", requires_grad=True),
                         torch.zeros(width, device="cuda", requires_grad=True)]
        self.balance = None  # the last pass's balance loss

    def parameters(self):
        return [self.table, self.router, self.out] + self.expert + (self.norm or [])

    def logits(self, token, graph, back):
        h = Aggregate.apply(Lookup.apply(self.table, token, self.scale), graph, back)
        if self.norm:
            h = Norm.apply(h, *self.norm)
        ids, weights, self.balance = Route.apply(h @ self.router, self.top_k)
        position, counts = sort_slots(ids, self.experts)
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


class AdamW:
    """AdamW over parameters whose gradients stay where they are: those of matrices decay. Updates
    are counted on the device, where they are made or, by a norm that is not finite, skipped."""

    def __init__(self, params, bits=32):
        state = torch.float32 if bits == 32 else torch.uint8
        m, v = ([torch.zeros(p.shape, dtype=state, device=p.device) for p in params]
                for _ in range(2))
        scales = None
        if bits == 8:
            scales = [torch.zeros((ps.state_blocks(p.numel()), 2), device=p.device) for p in params]
        self.tensors = ps.AdamWList([p.detach() for p in params], [p.grad for p in params], m, v,
                                    scales=scales,
                                    weight_decay=[0.01 if p.dim() > 1 else 0.0 for p in params])
        self.steps = torch.zeros(1, dtype=torch.int32, device=params[0].device)

    def step(self, rate, norm, max_norm):
        self.steps += torch.isfinite(norm)
        ps.AdamWStep(self.tensors, rate, self.steps, norm=norm, max_norm=max_norm, stream=_stream())


def train(nodes=8192, steps=60, seed=0, max_norm=0.1, rate=None, say=print, norm=False,
          balance=0.0, adamw=0):
    """Losses and gradient norms of the steps; `adamw` 32 or 8: by AdamW with moments of so many
    bits, else by plain descent."""
    csr, token, label, tokens = problem(nodes, seed=seed)
    graph, back, _ = graph_and_transpose(csr)
    model = Model(tokens, int(label.max()) + 1, seed=seed, norm=norm)
    params = model.parameters()
    for p in params:
        p.grad = torch.zeros_like(p)
    grads = ps.GradientList([p.grad for p in params])  # they stay where they are
    optimizer = AdamW(params, adamw) if adamw else None
    rate = rate if rate is not None else 0.003 if adamw else 5.0
    size = torch.empty(1, device="cuda")
    losses, norms = [], []
    for step in range(steps):
        loss = torch.nn.functional.cross_entropy(model.logits(token, graph, back), label)
        with torch.no_grad():
            for p in params:
                p.grad.zero_()
        (loss + balance * model.balance.sum()).backward()
        model.balance = model.balance.detach()  # the value alone: its graph goes with the step's
        if optimizer:
            ps.GradNorm(grads, size, stream=_stream())
            optimizer.step(rate, size, max_norm)
        else:
            ps.ClipGradNorm(grads, max_norm, size, stream=_stream())
            with torch.no_grad():
                for p in params:
                    p -= rate * p.grad
        losses.append(float(loss.detach()))
        norms.append(float(size))
        if step % 10 == 0 or step == steps - 1:
            say(f"step {step}: loss {losses[-1]:.4f}, gradient norm {norms[-1]:.4f}")
    return losses, norms


def main():
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--nodes", type=int, default=8192)
    parser.add_argument("--steps", type=int, default=60)
    parser.add_argument("--seed", type=int, default=0)
    parser.add_argument("--norm", action="store_true")
    parser.add_argument("--balance", type=float, default=0.0)
    parser.add_argument("--adamw", type=int, choices=(32, 8), default=0)
    a = parser.parse_args()
    ps.set_device(0)
    train(a.nodes, a.steps, a.seed, norm=a.norm, balance=a.balance, adamw=a.adamw)


if __name__ == "__main__":
    main()
