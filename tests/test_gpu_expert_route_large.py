"""The router's kernels for many tokens, and logits that differ in their last bits, against 64-bit
forms on the device."""
import math
import zlib

import pytest
import torch

import more_rows_ref as ref
import powersparse_amd as ps
from gpu_util import say, setup

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    setup()


def generator(*key):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def check(logits, top_k, normalize, mask=None):
    """Forward and gradient of a batch; logits without NaN and infinities but -inf."""
    T, E = logits.shape
    ids = torch.full((T, top_k), 7, dtype=torch.int32, device="cuda")
    weights = torch.full((T, top_k), 7.0, device="cuda")
    counts = torch.full((E + 1,), 7, dtype=torch.int32, device="cuda")
    loss = torch.full((1,), 7.0, device="cuda")
    work = torch.empty(ps.expert_route_workspace_bytes(T, E), dtype=torch.uint8,
                       device="cuda").fill_(255)
    ps.ExpertRoute(logits, ids, weights, counts, loss, work, mask=mask, normalize=normalize)
    l = logits.double()
    if mask is not None:
        l = l.masked_fill(~mask[:, None], -math.inf)
    values, order = torch.sort(l, dim=1, descending=True, stable=True)
    taken = values[:, :top_k] > -math.inf
    want = torch.where(taken, order[:, :top_k], -1)
    assert torch.equal(ids.long(), want)
    freq = torch.bincount(want[taken], minlength=E)
    on = taken[:, 0]
    assert torch.equal(counts.long(), torch.cat([freq, on.sum().view(1)]))
    p = torch.where(on[:, None], torch.softmax(l, 1), 0.0)
    w = torch.where(taken, p.gather(1, order[:, :top_k]), 0.0)
    if normalize:
        w = torch.where(on[:, None], w / w.sum(1, keepdim=True), 0.0)
    low = torch.where(l > -math.inf, l, math.inf).amin(1)
    far = torch.where(on, values[:, 0] - low, 0.0)
    rel = (2.25 * far + E + 12) * ref.U32
    assert bool(((weights.double() - w).abs() <= w * (rel[:, None] + ref.U32) + 2.0 ** -126).all())
    share = freq.double() / freq.sum().clamp(min=1)
    tokens = int(on.sum())
    exact = E * float((share * p.sum(0)).sum()) / max(tokens, 1)
    # sums over the tokens of a lane and of a workgroup's lanes in FP32, then in 64 bits
    off = (float(rel.max()) + (T / 256 + 80) * ref.U32) * exact
    assert abs(float(loss) - exact) <= off + 2.0 ** -120
    again = torch.empty_like(ids), torch.empty_like(weights)
    ps.ExpertRoute(logits, *again, mask=mask, normalize=normalize)
    assert torch.equal(again[0], ids) and torch.equal(again[1], weights)

    dw = torch.randn((T, top_k), generator=generator("dw", T, E), device="cuda")
    dloss = torch.full((1,), float(T), device="cuda")
    got = torch.full_like(logits, 7.0)
    ps.ExpertRouteGrad(logits, ids, dw, counts, dloss, got, normalize=normalize)
    h = (T * E / max(tokens, 1) * share).expand_as(p).clone()
    d = torch.where(taken, dw.double(), 0.0)
    if not normalize:
        h.scatter_add_(1, order[:, :top_k], d)
    inner = (p * h).sum(1, keepdim=True)
    grad, mag = p * (h - inner), p * (h.abs() + (p * h.abs()).sum(1, keepdim=True))
    if normalize:
        inner = (w * d).sum(1, keepdim=True)
        grad.scatter_add_(1, order[:, :top_k], w * (d - inner))
        mag.scatter_add_(1, order[:, :top_k], w * (d.abs() + (w * d.abs()).sum(1, keepdim=True)))
    unit = ref.UNIT[logits.dtype]
    bound = mag * 2 * (rel + (E + 12) * ref.U32)[:, None] * (1 + unit) + unit * grad.abs() + \
        ref.TINY[logits.dtype]
    assert bool(((got.double() - grad).abs() <= bound).all())


@pytest.mark.parametrize("experts", [8, 9, 16, 20, 32, 33, 64, 65, 128, 129, 200, 256, 300, 512, 700,
                                     1024])
def test_many_tokens(experts):
    """Around the 8,192 tokens that change the lanes, and several turns of every workgroup."""
    for k, (tokens, dtype) in enumerate([(8191, torch.float32), (8192, torch.float32),
                                         (40007, torch.bfloat16), (20011, torch.float16)]):
        if experts > 300:
            tokens = min(tokens, 12007)
        say(f"route {tokens} x {experts} {dtype}")
        gen = generator("many", experts, k)
        logits = 2 * torch.randn((tokens, experts), generator=gen, device="cuda")
        if k >= 1:
            logits[torch.rand(logits.shape, generator=gen, device="cuda") < 0.3] = -math.inf
        mask = torch.rand(tokens, generator=gen, device="cuda") < 0.9 if k != 1 else None
        check(logits.to(dtype), min(experts, (1, 3, 8, 5)[k]), k % 2 == 0, mask)


@pytest.mark.parametrize("experts", [5, 16, 64, 128, 300, 1024])
def test_logits_that_differ_in_their_last_bits(experts):
    """Neighbouring FP32 numbers, equal ones among them: what the cut keys cannot tell apart."""
    for tokens in (50, 9001):
        gen = generator("last bits", experts, tokens)
        steps = torch.randint(0, 40, (tokens, experts), generator=gen, device="cuda")
        for base in (1.0, -1.0, 2.0 ** -130, 1e30):
            bits = torch.full_like(steps, base, dtype=torch.float32).view(torch.int32) + \
                steps.to(torch.int32)
            logits = bits.view(torch.float32)
            # some rows have nothing of the kind, and some a few among others
            far = torch.randn(logits.shape, generator=gen, device="cuda")
            rows = torch.rand((tokens, 1), generator=gen, device="cuda")
            if base < 1e3:
                logits = torch.where(rows < 0.3, far, torch.where((rows < 0.6) & (far > 0), far, logits))
            check(logits.contiguous(), min(experts, 4), True)


def test_all_equal():
    """A fresh router: every logit the same."""
    for tokens in (3, 10000):
        check(torch.zeros((tokens, 48), device="cuda"), 4, True)
        check(torch.full((tokens, 130), -2.5, dtype=torch.bfloat16, device="cuda"), 2, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_nan_among_many(dtype):
    """A NaN is its token's first choice and makes its weights NaN; its neighbours' stay."""
    T, E, K = 9001, 96, 4
    gen = generator("nan", dtype)
    clean = torch.randn((T, E), generator=gen, device="cuda").to(dtype)
    bad = torch.rand(T, generator=gen, device="cuda") < 0.05
    at = torch.randint(0, E, (T,), generator=gen, device="cuda")
    logits = clean.clone()
    rows = torch.nonzero(bad).view(-1)
    logits[rows, at[rows]] = float("nan")
    outs = []
    for l in (clean, logits):
        ids, w = torch.empty((T, K), dtype=torch.int32, device="cuda"), torch.empty((T, K), device="cuda")
        ps.ExpertRoute(l, ids, w)
        outs.append((ids, w))
    assert torch.equal(outs[0][0][~bad], outs[1][0][~bad])
    assert torch.equal(outs[0][1][~bad], outs[1][1][~bad])
    ids, w = outs[1]
    assert torch.equal(ids[rows, 0].long(), at[rows]) and bool(torch.isnan(w[rows]).all())
    rest = clean.double()
    rest[rows, at[rows]] = -math.inf
    order = torch.sort(rest, dim=1, descending=True, stable=True).indices[:, :K - 1]
    assert torch.equal(ids[rows, 1:].long(), order[rows])


@pytest.mark.parametrize("experts", [5, 16, 17, 64, 128, 200, 300, 1024])
def test_the_loss_takes_every_token_once(experts):
    """The loss to less than a token's part of it. A probability is off by the exponential, 2 + 2.3
    times the logits' difference of up to 12, the sum of the experts, at most 15 + 6 additions, a
    reciprocal and a product, 3: 54 units; a sum over the tokens has 10 turns of a lane at most, 4
    steps in a wave and 16 waves, then 64-bit sums and one rounding: 86 units together, 5.2e-6. A
    token's part is some 1 / 40,007, 2.5e-5."""
    T, K = 40007, min(experts, 4)
    gen = generator("every token", experts)
    logits = torch.randn((T, experts), generator=gen, device="cuda")
    ids = torch.empty((T, K), dtype=torch.int32, device="cuda")
    w, loss = torch.empty((T, K), device="cuda"), torch.empty(1, device="cuda")
    counts = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
    work = torch.empty(ps.expert_route_workspace_bytes(T, experts), dtype=torch.uint8,
                       device="cuda")
    ps.ExpertRoute(logits, ids, w, counts, loss, work)
    l = logits.double()
    assert float((l.amax(1) - l.amin(1)).max()) <= 12
    p = torch.softmax(l, 1)
    freq = torch.bincount(torch.sort(l, dim=1, descending=True, stable=True).indices[:, :K]
                          .reshape(-1), minlength=experts)
    assert torch.equal(counts.long(), torch.cat([freq, torch.tensor([T], device="cuda")]))
    each = experts * (p * freq.double()).sum(1) / (T * freq.sum())  # a token's part of the loss
    exact = float(each.sum())
    off = 86 * ref.U32 * exact
    assert float(each.min()) > 4 * off and abs(float(loss) - exact) <= off
