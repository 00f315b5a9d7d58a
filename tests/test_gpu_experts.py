"""Tokens sorted by expert and back, and the gradients, against plain forms in
64 bits: one token to many sort tiles, one expert to 1024, dropped slots, tokens
without a slot, types, widths, strides and alignments, positions out of range,
non-finite values in places that take no part, offsets beyond 32 bits, graphs."""
import zlib

import pytest
import torch

import powersparse_amd as ps
import rows_ref as ref
from gpu_util import say, setup

pytestmark = pytest.mark.gpu

F = ref.DTYPES
NAN = float("nan")


@pytest.fixture(scope="module", autouse=True)
def device():
    setup()


def generator(*key):
    g = torch.Generator()
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def sort(ids, experts):
    n = ids.numel()
    order = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    position = torch.full(tuple(ids.shape), -7, dtype=torch.int32, device="cuda")
    offsets = torch.full((experts + 1,), -7, dtype=torch.int32, device="cuda")
    work = torch.full((ps.expert_sort_workspace_bytes(n, experts),), 255, dtype=torch.uint8,
                      device="cuda")
    ps.ExpertSort(ids.cuda(), order, position, offsets, work)
    torch.cuda.synchronize()
    return order, position, offsets


@pytest.mark.parametrize("experts", [1, 2, 17, 64, 255, 256, 1023, 1024])
@pytest.mark.parametrize("tokens,top_k", [(0, 2), (1, 1), (1, 8), (63, 1), (65, 3), (1024, 4),
                                          (4097, 1), (2049, 6), (1024, 8), (8193, 1),
                                          (9000, 8)])
def test_sort(experts, tokens, top_k):
    gen = generator(experts, tokens, top_k)
    for dist, id_t in (("uniform", torch.int64), ("one", torch.int32), ("skewed", torch.int32)):
        say(f"sort experts={experts} tokens={tokens} top_k={top_k} {dist}")
        if dist == "one":
            ids = torch.full((tokens, top_k), experts - 1)
        else:
            u = torch.rand((tokens, top_k), generator=gen)
            ids = (u ** (1 if dist == "uniform" else 4) * (experts + 2)).long() - 1
        order, position, offsets = sort(ids.to(id_t), experts)
        o, p, f = ref.sort(ids, experts)
        assert offsets.tolist() == f
        assert order.tolist() == o
        assert position.view(-1).tolist() == p


@pytest.mark.parametrize("tokens", [8192, 8193, 150000, 540001])
@pytest.mark.parametrize("experts", [3, 200, 1024])
def test_sort_long_lists(experts, tokens):
    gen = generator("long", experts, tokens)
    say(f"sort long list experts={experts} tokens={tokens}")
    ids = torch.randint(-1, experts + 1, (tokens, 8), generator=gen)
    order, position, offsets = sort(ids, experts)
    key = torch.where((ids >= 0) & (ids < experts), ids, experts).view(-1)
    o = torch.sort(key, stable=True).indices
    assert torch.equal(order.cpu().long(), o)
    p = torch.empty_like(o)
    p[o] = torch.arange(o.numel())
    assert torch.equal(position.cpu().view(-1).long(), torch.where(key < experts, p, -1))
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    assert offsets.tolist() == [0] + torch.cumsum(counts, 0).tolist()


def test_sort_all_dropped():
    ids = torch.tensor([[-1, 5], [99, -(1 << 40)]])
    order, position, offsets = sort(ids, 5)
    assert order.tolist() == [0, 1, 2, 3] and position.view(-1).tolist() == [-1] * 4
    assert offsets.tolist() == [0] * 6


def routed(gen, tokens, top_k, experts, drop):
    ids = torch.randint(0, experts, (tokens, top_k), generator=gen)
    ids[torch.rand((tokens, top_k), generator=gen) < drop] = -1
    if tokens > 2 and drop:
        ids[1] = -1  # a token without a slot
    return sort(ids, experts)


@pytest.mark.parametrize("dtype", F)
@pytest.mark.parametrize("cols", [1, 3, 7, 8, 9, 33, 96, 333, 1024, 2056, 4100])
def test_forward_and_gradients(dtype, cols):
    gen = generator(dtype, cols)
    t = F[dtype]
    for tokens, top_k, pad, offset, drop in ((1, 1, 0, 0, 0.0), (1, 8, 3, 1, 0.0),
                                             (37, 3, 0, 3, 0.3), (70, 11, 5, 0, 0.5)):
        say(f"experts {dtype} cols={cols} tokens={tokens} top_k={top_k} drop={drop}")
        order, position, offsets = routed(gen, tokens, top_k, 5, drop)
        slots = tokens * top_k
        filled = int(offsets[-1])

        def matrix(rows, poison=None):
            view, _ = ref.strided(rows, cols, t, pad, offset)
            view.copy_(torch.randn((rows, cols), generator=gen))
            if poison is not None:
                view[poison:] = NAN  # rows that no slot names
            return view

        def output(rows):
            return ref.strided(rows, cols, t, pad, offset, fill=7.0)

        x = matrix(tokens)
        xs, whole = output(slots)
        ps.ExpertDispatch(x, position, xs)
        torch.cuda.synchronize()
        assert torch.equal(xs[:filled], x[order[:filled].long() // top_k])
        assert bool((xs[filled:] == 7.0).all())
        xs.fill_(7.0)
        assert bool((whole == 7.0).all())

        ys = matrix(slots, filled)
        weights = torch.rand((tokens, top_k), generator=gen).cuda()
        weights[position < 0] = NAN  # a dropped slot's weight is not looked at
        y, whole = output(tokens)
        ps.ExpertCombine(ys, position, weights, y)
        torch.cuda.synchronize()
        exact, mag = ref.combine(ys, position, weights)
        ref.close(y, exact, mag, 2 * top_k, "combine")
        y.fill_(7.0)
        assert bool((whole == 7.0).all())

        dxs = matrix(slots, filled)
        dx, whole = output(tokens)
        ps.ExpertDispatchGrad(dxs, position, dx)
        torch.cuda.synchronize()
        exact, mag = ref.combine(dxs, position, None)
        ref.close(dx, exact, mag, top_k, "dispatch gradient")
        dx.fill_(7.0)
        assert bool((whole == 7.0).all())

        dy = matrix(tokens)
        if tokens > 2 and drop:
            dy[1] = float("inf")  # the token without a slot: nothing depends on it
        dys, whole = output(slots)
        dw = torch.full((tokens, top_k), 7.0, device="cuda")
        ps.ExpertCombineGrad(dy, ys, position, weights, dys, dw)
        torch.cuda.synchronize()
        e_dys, e_dw, mag = ref.combine_grad(dy, ys, position, weights)
        ref.close(dys[:filled], e_dys[:filled], e_dys[:filled].abs(), 1, "dys")
        assert bool((dys[filled:] == 7.0).all())
        ref.close(dw, e_dw, mag, cols + 1, "dweights")
        dys.fill_(7.0)
        assert bool((whole == 7.0).all())


def test_positions_out_of_range_are_skipped():
    gen = generator("range")
    x = torch.randn((3, 40), generator=gen).cuda()
    position = torch.tensor([[0, 9], [-5, 2], [1 << 30, -(1 << 31)]], dtype=torch.int32,
                            device="cuda")
    xs = torch.full((4, 40), 7.0, device="cuda")
    ps.ExpertDispatch(x, position, xs)
    assert torch.equal(xs[0], x[0]) and torch.equal(xs[2], x[1])
    assert bool((xs[[1, 3]] == 7.0).all())
    w = torch.tensor([[2.0, NAN], [NAN, 3.0], [NAN, NAN]], device="cuda")
    y = torch.full((3, 40), 7.0, device="cuda")
    ps.ExpertCombine(xs, position, w, y)
    assert torch.equal(y, torch.stack([2 * x[0], 3 * x[1], torch.zeros_like(x[0])]))
    dys, dw = torch.full_like(xs, 7.0), torch.empty((3, 2), device="cuda")
    ps.ExpertCombineGrad(x, xs, position, w, dys, dw)
    assert bool((dys[[1, 3]] == 7.0).all()) and torch.equal(dys[2], 3 * x[1])
    assert dw[0, 1] == dw[1, 0] == dw[2, 0] == dw[2, 1] == 0


def test_column_ranges_of_one_buffer():
    gen = generator("columns")
    whole = torch.randn((50, 33), generator=gen).cuda()
    before = whole.clone()
    x, xs = whole[:25, 3:15], whole[:50, 15:27]
    position = torch.randperm(50, generator=gen).to(torch.int32).view(25, 2).cuda()
    ps.ExpertDispatch(x, position, xs)
    before[position.view(-1).long(), 15:27] = before[:25, 3:15].repeat_interleave(2, 0)
    assert torch.equal(whole, before)
    # a single row, whose own stride is not the buffer's
    one = torch.tensor([[7, 30]], dtype=torch.int32, device="cuda")
    ps.ExpertDispatch(whole[9:10, 3:15], one, xs)
    before[[7, 30], 15:27] = before[9, 3:15]
    assert torch.equal(whole, before)
    ps.ExpertCombine(xs, one, None, whole[11:12, 3:15])
    before[11, 3:15] = before[7, 15:27] + before[30, 15:27]
    assert torch.equal(whole, before)


def test_differences():
    """Combine is linear in ys and in the weights; the gradients are its transposes. Whole
    numbers, so that both sides are exact."""
    gen = generator("differences")
    T, K, D, S = 30, 3, 21, 90
    _, position, _ = routed(gen, T, K, 4, 0.2)

    def whole(*shape):
        return torch.randint(-3, 4, shape, generator=gen).float().cuda()

    ys, d, w, e, r = whole(S, D), whole(S, D), whole(T, K), whole(T, K), whole(T, D)
    e[position < 0] = 0

    def value(ys, w):
        y = torch.empty((T, D), device="cuda")
        ps.ExpertCombine(ys, position, w, y)
        return float((y.double() * r.double()).sum())

    dys, dw = torch.zeros((S, D), device="cuda"), torch.empty((T, K), device="cuda")
    ps.ExpertCombineGrad(r, ys, position, w, dys, dw)
    assert (value(ys + d, w) - value(ys - d, w)) / 2 == float((dys.double() * d.double()).sum())
    assert (value(ys, w + e) - value(ys, w - e)) / 2 == float((dw.double() * e.double()).sum())
    # the dispatch and its gradient are each other's transpose
    x, g, xs, dx = whole(T, D), whole(S, D), torch.zeros((S, D), device="cuda"), whole(T, D)
    ps.ExpertDispatch(x, position, xs)
    ps.ExpertDispatchGrad(g, position, dx)
    assert float((xs.double() * g.double()).sum()) == float((x.double() * dx.double()).sum())


def test_beyond_32_bits():
    T, K, D = 300000, 4, 4096  # 4.9e9 elements in expert order
    ids = torch.randint(0, 6, (T, K))
    order, position, _ = sort(ids, 6)
    x = (torch.arange(T, device="cuda") % 251).to(torch.bfloat16)[:, None].expand(T, D).contiguous()
    xs = torch.empty((T * K, D), dtype=torch.bfloat16, device="cuda")
    ps.ExpertDispatch(x, position, xs)
    col = xs[:, [0, 1000, D - 1]].float()
    assert torch.equal(col, x[:, :3].float()[order.long() // K])
    y = torch.empty_like(x)
    ps.ExpertDispatchGrad(xs, position, y)
    for c in (0, 2047, D - 1):  # sums up to 1000, rounded to 8 bits of mantissa
        assert torch.equal(y[:, c], (4 * x[:, c].float()).to(torch.bfloat16))


def test_in_a_graph():
    gen = generator("graph")
    T, K, E, D = 1500, 4, 9, 72
    ids = torch.empty((T, K), dtype=torch.int64, device="cuda")
    x = torch.empty((T, D), device="cuda")
    w = torch.empty((T, K), device="cuda")
    position = torch.empty((T, K), dtype=torch.int32, device="cuda")
    order = torch.empty(T * K, dtype=torch.int32, device="cuda")
    offsets = torch.empty(E + 1, dtype=torch.int32, device="cuda")
    xs, dys = torch.zeros((T * K, D), device="cuda"), torch.zeros((T * K, D), device="cuda")
    y, dw = torch.empty((T, D), device="cuda"), torch.empty((T, K), device="cuda")
    work = torch.empty(ps.expert_sort_workspace_bytes(T * K, E), dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream().cuda_stream
        ps.ExpertSort(ids, order, position, offsets, work, stream=s)
        ps.ExpertDispatch(x, position, xs, stream=s)
        ps.ExpertCombine(xs, position, w, y, stream=s)
        ps.ExpertCombineGrad(y, xs, position, w, dys, dw, stream=s)

    def contents():
        ids.copy_(torch.randint(-1, E, (T, K), generator=gen))
        x.copy_(torch.randn((T, D), generator=gen))
        w.copy_(torch.rand((T, K), generator=gen))

    contents()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        contents()
        outs = (order, position, offsets, xs, y, dys, dw)
        xs.zero_()
        dys.zero_()
        graph.replay()
        torch.cuda.synchronize()
        replayed = [o.clone() for o in outs]
        xs.zero_()
        dys.zero_()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, outs))


@pytest.mark.parametrize("experts", [5, 1024])
def test_sort_in_a_workspace_for_more(experts):
    gen = generator("workspace", experts)
    for most, count in ((196616, 196608), (4194400, 4194304), (4194400, 8193)):
        say(f"sort of {count} slots in a workspace for {most}, {experts} experts")
        work = torch.full((ps.expert_sort_workspace_bytes(most, experts),), 255,
                          dtype=torch.uint8, device="cuda")
        ids = torch.randint(-1, experts + 1, (count,), generator=gen)
        order, position = (torch.empty(count, dtype=torch.int32, device="cuda") for _ in range(2))
        offsets = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
        ps.ExpertSort(ids.cuda(), order, position, offsets, work)
        key = torch.where((ids >= 0) & (ids < experts), ids, experts)
        assert torch.equal(order.cpu().long(), torch.sort(key, stable=True).indices)
        assert int(offsets[-1]) == int((key < experts).sum())


def test_positions_between_the_rows_of_the_output():
    """Columns that a matrix leaves out of its buffer are nobody's: positions may be there."""
    gen = generator("between")
    whole = torch.zeros((20, 33), device="cuda")
    x, xs = torch.randn((9, 24), generator=gen).cuda(), whole[:, :24]
    position = whole.view(torch.int32)[7, 24:33]
    position.copy_(torch.randperm(20, generator=gen)[:9].to(torch.int32))
    where = position.long()
    ps.ExpertDispatch(x, position, xs)
    assert torch.equal(xs[where], x) and torch.equal(position.long(), where)
    assert int(torch.count_nonzero(xs.any(1))) == 9
