"""The example's options: the gradients of the model with layer norm and the balance loss against
the same model in torch's own operations in 64 bits, an AdamW update on the way, and runs of all."""
import math

import pytest
import torch

import powersparse_amd as ps
from gpu_util import setup
from powersparse_amd.examples import expert_nodes as ex

pytestmark = pytest.mark.gpu


def plain(model, params, token, coo, n):
    """(logits, balance loss) of the model in 64 bits on the host."""
    table, router, out, *rest = params
    expert, (weight, bias) = rest[:-2], rest[-2:]
    row, col, val = (torch.from_numpy(a) for a in coo)
    x = table[token.cpu()] * model.scale
    h = torch.zeros((n, x.shape[1]), dtype=torch.float64)
    h = h.index_add(0, row, val.double()[:, None] * x[col])
    h = torch.nn.functional.layer_norm(h, h.shape[1:], weight, bias, 1e-5)
    scores = h @ router
    top = scores.topk(model.top_k, dim=1)
    w = torch.softmax(top.values, dim=1)
    each = torch.stack([torch.relu(h @ e) for e in expert], 1)  # nodes x experts x width
    chosen = torch.gather(each, 1, top.indices[..., None].expand(-1, -1, h.shape[1]))
    y = (w[..., None] * chosen).sum(1)
    share = torch.bincount(top.indices.view(-1), minlength=model.experts).double() / top.indices.numel()
    balance = model.experts * (share * torch.softmax(scores, 1).mean(0)).sum()
    return y @ out + h @ out, balance


def test_gradients():
    setup()
    csr, token, label, tokens = ex.problem(512, seed=4)
    graph, back, coo = ex.graph_and_transpose(csr)
    model = ex.Model(tokens, int(label.max()) + 1, seed=4, norm=True)
    with torch.no_grad():
        model.norm[0].mul_(1.5)
        model.norm[1].add_(0.1)
    logits = model.logits(token, graph, back)
    loss = torch.nn.functional.cross_entropy(logits, label) + 0.5 * model.balance.sum()
    loss.backward()
    params = [p.detach().cpu().double().requires_grad_() for p in model.parameters()]
    exact, balance = plain(model, params, token, coo, csr.rows)
    exact_loss = torch.nn.functional.cross_entropy(exact, label.cpu()) + 0.5 * balance
    exact_loss.backward()
    # products of 64 columns and sums of up to some hundred rows in FP32, several in a row
    torch.testing.assert_close(logits.detach().cpu().double(), exact.detach(), rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(float(model.balance.detach()), float(balance.detach()), rtol=1e-5, atol=0)
    for got, want in zip(model.parameters(), params):
        scale = float(want.grad.abs().max())
        torch.testing.assert_close(got.grad.cpu().double(), want.grad, rtol=1e-3, atol=1e-4 * scale)


def test_update():
    """The clipped AdamW step of the example's optimizer is its formula's, on its gradients."""
    setup()
    model = ex.Model(200, 8, seed=1, norm=True)
    params = model.parameters()
    gen = torch.Generator(device="cuda").manual_seed(2)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen, device="cuda")
    grads = ps.GradientList([p.grad for p in params])
    before = [(p.detach().double(), p.grad.double()) for p in params]
    size = torch.empty(1, device="cuda")
    ps.GradNorm(grads, size)
    ex.AdamW(params).step(0.01, size, 1.0)
    norm = math.sqrt(sum(float(g.square().sum()) for _, g in before))
    for p, (old, g) in zip(params, before):
        g = g / (norm + 1e-6)
        decay = 0.01 if p.dim() > 1 else 0.0
        want = old - 0.01 * (decay * old + g / (g.abs() + 1e-8))
        # |update| is 1 at most; some thirty roundings of it, one of the parameter
        assert bool(((p.detach().double() - want).abs() <= 2.0 ** -24 * (0.4 + 2 * old.abs())).all())


@pytest.mark.parametrize("adamw", [0, 32, 8])
def test_runs(adamw):
    setup()
    lines = []
    losses, norms = ex.train(nodes=1024, steps=12, seed=1, say=lines.append, norm=True,
                             balance=0.01, adamw=adamw)
    assert all(math.isfinite(v) for v in losses) and all(n > 0 for n in norms)
    assert len(lines) == 3


@pytest.mark.parametrize("bits", [32, 8])
def test_a_skipped_update_is_not_counted(bits):
    """Updates whose norm is not finite change nothing, and the first one after them is the first
    of the formula: counted as the third, it would be 0.58 of that."""
    setup()
    model = ex.Model(200, 8, seed=1, norm=True)
    params = model.parameters()
    gen = torch.Generator(device="cuda").manual_seed(3)
    for p in params:
        p.grad = torch.randn(p.shape, generator=gen, device="cuda")
    optimizer = ex.AdamW(params, bits)
    before = [p.detach().clone() for p in params]
    size = torch.empty(1, device="cuda")
    for bad in (math.inf, math.nan):
        optimizer.step(0.01, size.fill_(bad), 1.0)
        assert all(torch.equal(p.detach(), old) for p, old in zip(params, before))
    ps.GradNorm(ps.GradientList([p.grad for p in params]), size)
    optimizer.step(0.01, size, 1.0)
    norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
    for p, old in zip(params, before):
        g, old = p.grad.double() / (norm + 1e-6), old.double()
        decay = 0.01 if p.dim() > 1 else 0.0
        want = old - 0.01 * (decay * old + g / (g.abs() + 1e-8))
        off = (p.detach().double() - want).abs()
        assert bool((off <= 2.0 ** -24 * (0.4 + 2 * old.abs())).all())  # as in test_update


def test_a_step_leaves_no_graph(monkeypatch):
    """What the model keeps of a pass holds none of its graph once the step is done."""
    setup()
    made = []

    class Kept(ex.Model):
        def __init__(self, *args, **kwargs):
            super().__init__(*args, **kwargs)
            made.append(self)

    monkeypatch.setattr(ex, "Model", Kept)
    ex.train(nodes=512, steps=1, seed=1, say=lambda line: None, norm=True, balance=0.01)
    assert made[0].balance.grad_fn is None and not made[0].balance.requires_grad
    assert math.isfinite(float(made[0].balance))
