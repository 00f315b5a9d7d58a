"""The router and its gradient against 64-bit plain forms: every number of experts where the
kernels change, ties, barred experts, padding, rows that are left empty, NaN, balance loss,
gradients against differences and autograd, streams and graphs, and the way into the sort."""
import math
import zlib

import pytest
import torch

import more_rows_ref as ref
import powersparse_amd as ps
import rows_ref
from gpu_util import say, setup

pytestmark = pytest.mark.gpu

F = rows_ref.DTYPES
EXPERTS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256,
           257, 500, 512, 513, 1023, 1024]


@pytest.fixture(scope="module", autouse=True)
def device():
    setup()


def generator(*key):
    g = torch.Generator()
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def route(logits, top_k, normalize=True, mask=None, losses=True):
    T, E = logits.shape
    ids = torch.full((T, top_k), 7, dtype=torch.int32, device="cuda")
    weights = torch.full((T, top_k), 7.0, device="cuda")
    if not losses:
        ps.ExpertRoute(logits, ids, weights, mask=mask, normalize=normalize)
        return ids, weights
    counts = torch.full((E + 1,), 7, dtype=torch.int32, device="cuda")
    loss = torch.full((1,), 7.0, device="cuda")
    work = torch.empty(ps.expert_route_workspace_bytes(T, E), dtype=torch.uint8,
                       device="cuda").fill_(255)
    ps.ExpertRoute(logits, ids, weights, counts, loss, work, mask=mask, normalize=normalize)
    return ids, weights, counts, loss


def check(logits, top_k, normalize, mask=None):
    ids, weights, counts, loss = route(logits, top_k, normalize, mask)
    torch.cuda.synchronize()
    want = ref.route(logits, top_k, normalize, mask)
    assert torch.equal(ids.cpu(), want["ids"])
    assert torch.equal(counts.cpu(), want["counts"])
    ref.held(weights, want["weights"], want["weights_off"], "weights")
    ref.held(loss, want["loss"], want["loss_off"], "loss")
    again = route(logits, top_k, normalize, mask, losses=False)
    assert torch.equal(again[0], ids) and torch.equal(again[1], weights)
    return ids, weights, counts, loss


def check_grad(gen, logits, ids, counts, normalize):
    dweights = torch.randn(ids.shape, generator=gen).cuda()
    dloss = torch.tensor([3.0], device="cuda")
    for dw, dl in ((dweights, dloss), (dweights, None), (None, dloss)):
        out, whole = rows_ref.strided(*logits.shape, logits.dtype, 3, 1, fill=7.0)
        ps.ExpertRouteGrad(logits, ids, dw, counts, dl, out, normalize=normalize)
        torch.cuda.synchronize()
        ref.held(out, *ref.route_grad(logits, ids, dw, counts, dl, normalize), "dlogits")
        out.fill_(7.0)
        assert bool((whole == 7.0).all())


def some_logits(gen, tokens, experts, dtype, barred=0.0):
    l = 2 * torch.randn((tokens, experts), generator=gen)
    l[torch.rand((tokens, experts), generator=gen) < barred] = -math.inf
    return l.to(F[dtype]).cuda()


@pytest.mark.parametrize("experts", EXPERTS)
def test_experts(experts):
    for k, dtype in enumerate(("f32", "bf16", "f16")):
        gen = generator("experts", experts, dtype)
        top_k = sorted({1, min(experts, 2 + k), min(experts, 8), experts if experts < 40 else 1})
        for n in top_k:
            say(f"route {experts} experts, top {n}, {dtype}")
            logits = some_logits(gen, 37, experts, dtype, barred=(0.0, 0.3, 0.9)[k])
            mask = torch.rand(37, generator=gen).cuda() < 0.8
            ids, _, counts, _ = check(logits, n, k != 1, mask)
            check_grad(gen, logits, ids, counts, k != 1)


@pytest.mark.parametrize("top_k", [1, 63, 64, 65, 300])
def test_many_slots(top_k):
    gen = generator("slots", top_k)
    logits = some_logits(gen, 9, 300, "f32", barred=0.4)
    for normalize in (True, False):
        ids, _, counts, _ = check(logits, top_k, normalize)
        check_grad(gen, logits, ids, counts, normalize)


@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 33, 1000, 4097])
def test_tokens(tokens):
    gen = generator("tokens", tokens)
    logits = some_logits(gen, tokens, 16, "f32")
    ids, _, counts, _ = check(logits, 2, True)
    check_grad(gen, logits, ids, counts, True)


def test_many_tokens():
    """Beyond a turn of every workgroup, against torch on the device in 64 bits."""
    gen = generator("many")
    T, E, K = 200003, 64, 4
    logits = torch.randn((T, E), generator=gen).cuda()
    ids, weights, counts, loss = route(logits, K)
    l = logits.double()
    top = l.topk(K, 1)
    assert torch.equal(ids.long(), top.indices)  # no two of a row are equal
    p = torch.softmax(l, 1)
    freq = torch.bincount(top.indices.view(-1), minlength=E)
    assert torch.equal(counts[:E].long(), freq) and int(counts[E]) == T
    exact = E * float((freq.double() / (T * K) * p.mean(0)).sum())
    assert abs(float(loss) - exact) <= 1e-5 * exact  # some 400 tokens a chain, 64-bit joins
    assert float((weights.double() - torch.softmax(top.values, 1)).abs().max()) <= 60 * ref.U32
    dw, dloss = torch.randn((T, K), generator=gen).cuda(), torch.tensor([float(T)], device="cuda")
    got = torch.empty_like(logits)
    ps.ExpertRouteGrad(logits, ids, dw, counts, dloss, got)
    l.requires_grad_()
    w = torch.softmax(l.gather(1, ids.long()), 1)
    f = freq.double() / (T * K)
    total = (w * dw.double()).sum() + T * E * (f * torch.softmax(l, 1).mean(0)).sum()
    want, = torch.autograd.grad(total, l)
    assert float((got.double() - want).abs().max()) <= 200 * ref.U32 * (1 + float(dw.abs().max()))


def test_ties_go_to_the_lowest_expert():
    for experts in (5, 64, 100, 300, 1024):
        logits = torch.zeros((3, experts), device="cuda")
        logits[1, ::2] = -0.0  # equal to 0
        logits[2, experts // 2:] = 1.0
        k = min(5, experts // 2)
        ids, weights = route(logits, k, losses=False)
        first = list(range(k))
        assert ids.tolist() == [first, first, [experts // 2 + i for i in first]]
        assert float((weights - 1.0 / k).abs().max()) <= 8 * ref.U32


def test_everything_barred_or_masked():
    logits = torch.full((4, 10), -math.inf, device="cuda")
    logits[1, 3] = 1.0
    logits[2] = 0.0
    mask = torch.tensor([1, 1, 0, 1], dtype=torch.uint8, device="cuda")
    for normalize in (True, False):
        ids, weights, counts, loss = route(logits, 2, normalize, mask)
        assert ids.tolist() == [[-1, -1], [3, -1], [-1, -1], [-1, -1]]
        assert weights.tolist() == [[0, 0], [1, 0], [0, 0], [0, 0]]
        assert counts.tolist() == [0, 0, 0, 1] + [0] * 6 + [1] and float(loss) == 10.0
        grad = torch.full_like(logits, 7.0)
        ps.ExpertRouteGrad(logits, ids, torch.ones_like(weights), counts,
                           torch.ones(1, device="cuda"), grad, normalize=normalize)
        assert not bool(grad.any()) and bool(torch.isfinite(grad).all())
        none = torch.zeros(4, dtype=torch.bool, device="cuda")
        ids, weights, counts, loss = route(logits, 2, normalize, none)
        assert bool((ids == -1).all()) and not weights.any() and not counts.any()
        assert float(loss) == 0.0
        ps.ExpertRouteGrad(logits, ids, None, counts, torch.ones(1, device="cuda"), grad)
        assert not bool(grad.any())


def test_lowest_values_of_a_type_are_no_bars():
    for dtype in F.values():
        logits = torch.full((2, 6), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        logits[1, 2] = 0
        ids, weights = route(logits, 3, losses=False)
        assert ids.tolist() == [[0, 1, 2], [2, 0, 1]]
        assert weights[1].tolist() == [1, 0, 0]
        assert float((weights[0] - 1 / 3).abs().max()) <= 8 * ref.U32


def test_nan_and_infinities():
    logits = torch.zeros((5, 70), device="cuda")
    logits[1, 9], logits[1, 65] = float("nan"), 3.0
    logits[2, 8] = math.inf
    logits[3, 7] = -float("nan")
    masked = torch.tensor([True, True, True, True, False], device="cuda")
    logits[4] = float("nan")
    ids, weights, counts, loss = route(logits, 3, False, masked)
    assert ids[:4].tolist() == [[0, 1, 2], [9, 65, 0], [8, 0, 1], [7, 0, 1]]
    assert bool(torch.isnan(weights[1:4]).all()) and math.isnan(float(loss))
    assert float((weights[0] - 1 / 70).abs().max()) <= ref.U32
    assert ids[4].tolist() == [-1] * 3 and not weights[4].any()
    assert counts[:70].sum() == 12 and counts[70] == 4
    grad = torch.full_like(logits, 7.0)
    ps.ExpertRouteGrad(logits, ids, torch.ones_like(weights), counts, None, grad, normalize=False)
    assert torch.isfinite(grad).all(1).tolist() == [True, False, False, False, True]
    assert not grad[4].any()


def test_balance():
    """1 where all is balanced, the number of experts where one has everything."""
    E, T = 8, 64
    even = torch.full((T, E), -30.0, device="cuda")
    even[torch.arange(T), torch.arange(T) % E] = 30.0
    assert abs(float(route(even, 1)[3]) - 1.0) <= 100 * ref.U32
    one = torch.full((T, E), -30.0, device="cuda")
    one[:, 5] = 30.0
    assert abs(float(route(one, 1)[3]) - E) <= 100 * ref.U32 * E


def test_nothing_to_do():
    logits = torch.empty((0, 12), device="cuda")
    ids, weights, counts, loss = route(logits, 3)
    assert not counts.any() and float(loss) == 0.0
    ps.ExpertRouteGrad(logits, ids, weights, counts, loss, torch.empty_like(logits))


def test_gradients_against_differences():
    """Central differences of sum(dw * w) + 2 * loss in 64 bits, the choices as they are."""
    gen = generator("differences")
    logits = torch.randn((6, 9), generator=gen)
    for normalize in (True, False):
        ids, _, counts, _ = route(logits.cuda(), 3, normalize)
        dw = torch.randn((6, 3), generator=gen)
        got = torch.empty((6, 9), device="cuda")
        ps.ExpertRouteGrad(logits.cuda(), ids, dw.cuda(), counts, torch.tensor([2.0]).cuda(), got,
                           normalize=normalize)
        chosen, f = ids.cpu().long(), counts.cpu().double()[:9] / 18

        def total(l):
            p = torch.softmax(l, 1)
            w = p.gather(1, chosen)
            if normalize:
                w = w / w.sum(1, keepdim=True)
            return float((w * dw).sum() + 2 * 9 * (f * p.mean(0)).sum())

        h = 2.0 ** -10
        for t in range(6):
            for e in range(9):
                moved = []
                for s in (h, -h):
                    l = logits.double().clone()
                    l[t, e] += s
                    moved.append(total(l))
                want = (moved[0] - moved[1]) / (2 * h)  # off by h^2 and some third derivative of 1
                assert abs(float(got[t, e]) - want) <= 2e-5


def test_counts_of_several_ranks():
    """With the counts added up over two halves of a batch, their gradients are the batch's."""
    gen = generator("ranks")
    logits = torch.randn((50, 12), generator=gen).cuda()
    whole = route(logits, 2)
    halves = [route(part, 2) for part in (logits[:30], logits[30:])]
    counts = halves[0][2] + halves[1][2]
    assert torch.equal(counts, whole[2])
    dloss = torch.tensor([5.0], device="cuda")
    want, got = torch.empty_like(logits), torch.empty_like(logits)
    ps.ExpertRouteGrad(logits, whole[0], None, whole[2], dloss, want)
    for at, (ids, _, _, _) in zip((slice(0, 30), slice(30, 50)), halves):
        ps.ExpertRouteGrad(logits[at], ids, None, counts, dloss, got[at])
    assert torch.equal(got, want)


def test_the_same_bits_every_time_and_workspaces_made_for_more():
    gen = generator("bits")
    logits = torch.randn((50021, 40), generator=gen).cuda()
    work = torch.empty(ps.expert_route_workspace_bytes(60000, 512), dtype=torch.uint8,
                       device="cuda")
    got = []
    for fill in (0, 255, 1):
        work.fill_(fill)
        outs = [torch.empty((50021, 2), dtype=torch.int32, device="cuda"),
                torch.empty((50021, 2), device="cuda"),
                torch.empty(41, dtype=torch.int32, device="cuda"), torch.empty(1, device="cuda")]
        ps.ExpertRoute(logits, *outs, work)
        got.append(outs)
    assert all(torch.equal(a, b) for other in got[1:] for a, b in zip(got[0], other))


@pytest.mark.parametrize("tokens", [5, 3000])
def test_in_a_graph_on_into_the_sort(tokens):
    """Routed, sorted, dispatched, combined and back, captured and replayed."""
    gen = generator("graph", tokens)
    E, K, D = 20, 3, 48
    logits = torch.empty((tokens, E), device="cuda")
    x = torch.empty((tokens, D), device="cuda")
    mask = torch.empty(tokens, dtype=torch.bool, device="cuda")
    def i32(*shape):
        return torch.zeros(shape, dtype=torch.int32, device="cuda")
    ids, counts, order, position, offsets = (i32(tokens, K), i32(E + 1), i32(tokens * K),
                                             i32(tokens, K), i32(E + 1))
    w, dw, loss = torch.empty((tokens, K), device="cuda"), torch.empty((tokens, K), device="cuda"), \
        torch.empty(1, device="cuda")
    xs, dxs = (torch.zeros((tokens * K, D), device="cuda") for _ in range(2))
    y, dlogits = torch.empty_like(x), torch.empty_like(logits)
    one = torch.ones(1, device="cuda")
    work = [torch.empty(n, dtype=torch.uint8, device="cuda") for n in
            (ps.expert_route_workspace_bytes(tokens, E), ps.expert_sort_workspace_bytes(tokens * K, E))]

    def step():
        s = torch.cuda.current_stream()
        ps.ExpertRoute(logits, ids, w, counts, loss, work[0], mask=mask, stream=s)
        ps.ExpertSort(ids, order, position, offsets, work[1], stream=s)
        ps.ExpertDispatch(x, position, xs, stream=s)
        ps.ExpertCombine(xs, position, w, y, stream=s)
        ps.ExpertCombineGrad(x, xs, position, w, dxs, dw, stream=s)
        ps.ExpertRouteGrad(logits, ids, dw, counts, one, dlogits, stream=s)

    def fill():
        logits.copy_(torch.randn(logits.shape, generator=gen))
        x.copy_(torch.randn(x.shape, generator=gen))
        mask.copy_(torch.rand(tokens, generator=gen) < 0.9)

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        fill()
        graph.replay()
        torch.cuda.synchronize()
        outs = [ids, w, counts, loss, position, offsets, y, dw, dlogits]
        replayed = [o.clone() for o in outs]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, o) for a, o in zip(replayed, outs))
        # every row comes back as its weights' sum of itself, and the experts' shares agree
        assert torch.equal(torch.diff(offsets), counts[:E])
        on = mask[:, None].float()
        assert float((y - x * on).abs().max()) <= 8 * ref.U32 * float(x.abs().max())
        assert torch.equal(position < 0, ~mask[:, None].expand(-1, K))


@pytest.mark.parametrize("tokens,experts,top_k", [(4, 70, 5), (9004, 20, 3), (12, 300, 100)])
def test_places_left_over_beside_a_nan(tokens, experts, top_k):
    """A NaN makes its token's weights NaN, but of the experts that were chosen: places left over
    have id -1 and weight 0 whatever the logits."""
    logits = torch.full((tokens, experts), -math.inf, device="cuda")
    logits[0::4, 2] = 0.5
    logits[1::4, 9], logits[1::4, 4] = float("nan"), 1.0
    logits[2::4, 11] = -float("nan")
    logits[3::4, 1] = math.inf
    for normalize in (True, False):
        for losses in (True, False):
            ids, weights = route(logits, top_k, normalize, losses=losses)[:2]
            want = torch.full_like(ids, -1)
            want[0::4, 0], want[1::4, 0], want[1::4, 1] = 2, 9, 4
            want[2::4, 0], want[3::4, 0] = 11, 1
            assert torch.equal(ids, want)
            assert bool((weights[0::4, 0] == 1).all())
            for k in (1, 2, 3):
                taken = want[k::4] >= 0
                assert bool(torch.isnan(weights[k::4][taken]).all())
            assert not weights[want < 0].any()


@pytest.mark.parametrize("tokens,experts", [(400, 8), (9000, 8), (400, 16), (9000, 20), (400, 64),
                                            (100, 128)])
@pytest.mark.parametrize("std", [1, 8])
def test_weights_of_far_logits(tokens, experts, std):
    """All experts chosen, weights over a hundred powers of two: logits whose differences FP32
    holds, so that what is off is the exponentials, 2^-24 (3 + 0.05 |x|) of a weight's own and 4 of
    the sum's, whose terms are near the largest, additions one behind another, experts / 4 of a lane
    and 6 joins at most, the reciprocal, 2, and a product."""
    gen = generator("far", tokens, experts, std)
    logits = torch.round(std * 64 * torch.randn((tokens, experts), generator=gen)) / 64
    assert float(logits.abs().max()) < 64
    ids, weights = route(logits.cuda(), experts, True, losses=False)
    want = torch.sort(logits.double(), dim=1, descending=True, stable=True)
    assert torch.equal(ids.cpu().long(), want.indices)
    exact = torch.softmax(want.values, 1)
    x = want.values[:, :1] - want.values
    units = 3 + 0.05 * x + 4 + experts / 4 + 6 + 2 + 1
    off = (weights.cpu().double() - exact).abs()
    assert bool((off <= units * ref.U32 * exact + 2.0 ** -126).all())
