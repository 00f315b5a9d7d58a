"""The example that trains a mixture of experts on a graph's nodes: its
gradients against the same model in torch's own operations in 64 bits, and a
short training run."""
import pytest
import torch

import powersparse_amd as ps
from gpu_util import setup
from powersparse_amd.examples import expert_nodes as ex

pytestmark = pytest.mark.gpu


def plain_logits(model, params, token, coo, n):
    """The model in 64 bits on the host."""
    table, router, out, *expert = params
    row, col, val = (torch.from_numpy(a) for a in coo)
    x = table[token.cpu()] * model.scale
    h = torch.zeros((n, x.shape[1]), dtype=torch.float64)
    h = h.index_add(0, row, val.double()[:, None] * x[col])
    top = (h @ router).topk(model.top_k, dim=1)
    w = torch.softmax(top.values, dim=1)
    each = torch.stack([torch.relu(h @ e) for e in expert], 1)  # nodes x experts x width
    chosen = torch.gather(each, 1, top.indices[..., None].expand(-1, -1, h.shape[1]))
    y = (w[..., None] * chosen).sum(1)
    return y @ out + h @ out


def test_gradients():
    setup()
    csr, token, label, tokens = ex.problem(512, seed=3)
    graph, back, coo = ex.graph_and_transpose(csr)
    model = ex.Model(tokens, int(label.max()) + 1, seed=3)
    logits = model.logits(token, graph, back)
    loss = torch.nn.functional.cross_entropy(logits, label)
    loss.backward()
    params = [p.detach().cpu().double().requires_grad_() for p in model.parameters()]
    exact = plain_logits(model, params, token, coo, csr.rows)
    exact_loss = torch.nn.functional.cross_entropy(exact, label.cpu())
    exact_loss.backward()
    # products of 64 columns and sums of up to some hundred rows in FP32, several in a row
    torch.testing.assert_close(logits.detach().cpu().double(), exact.detach(), rtol=1e-4, atol=1e-4)
    for got, want in zip(model.parameters(), params):
        scale = float(want.grad.abs().max())
        torch.testing.assert_close(got.grad.cpu().double(), want.grad, rtol=1e-3, atol=1e-4 * scale)


def test_training():
    setup()
    lines = []
    losses, norms = ex.train(nodes=2048, steps=40, seed=1, say=lines.append)
    assert losses[-1] < 0.7 * losses[0] and all(n > 0 for n in norms)
    assert len(lines) == 5
