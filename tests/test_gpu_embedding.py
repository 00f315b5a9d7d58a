"""Embedding lookup and its gradient against plain forms in 64 bits: types, id
types, widths from one element to more than a workgroup's pieces, strides and
alignments, ids out of range, runs of equal ids of every length around the
chunks' and the sort tiles' borders, accumulation, padding, offsets beyond 32
bits, streams and graphs."""
import itertools
import zlib

import pytest
import torch

import powersparse_amd as ps
import rows_ref as ref
from gpu_util import say, setup

pytestmark = pytest.mark.gpu

F = ref.DTYPES


@pytest.fixture(scope="module", autouse=True)
def device():
    setup()


def values(gen, rows, cols, dtype, pad=0, offset=0):
    view, whole = ref.strided(rows, cols, dtype, pad, offset)
    view.copy_(torch.randn((rows, cols), generator=gen))
    return view, whole


def generator(*key):
    g = torch.Generator()
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


@pytest.mark.parametrize("table_t,out_t", list(itertools.product(F, F)))
@pytest.mark.parametrize("cols", [1, 2, 3, 7, 8, 9, 33, 96, 333, 1024, 2049])
def test_lookup(table_t, out_t, cols):
    gen = generator(table_t, out_t, cols)
    for count, rows, pad, offset, id_t in ((1, 1, 0, 0, torch.int64), (5, 3, 1, 1, torch.int32),
                                           (300, 77, 0, 3, torch.int64),
                                           (1030, 50, 5, 0, torch.int32)):
        say(f"lookup {table_t}->{out_t} cols={cols} count={count} rows={rows} pad={pad}")
        table, _ = values(gen, rows, cols, F[table_t], pad, offset)
        ids = torch.randint(-1, rows + 1, (count,), generator=gen)
        if id_t is torch.int64 and count > 4:
            ids[1], ids[2] = 1 << 40, -(1 << 40)
        ids = ids.to(id_t).cuda()
        out, whole = ref.strided(count, cols, F[out_t], pad, offset, fill=7.0)
        ps.EmbeddingLookup(table, ids, out, scale=1.25)
        torch.cuda.synchronize()
        exact = ref.lookup(table, ids, 1.25)
        ref.close(out, exact, exact.abs(), 1, "lookup")
        out.fill_(7.0)  # nothing outside the rows was written
        assert bool((whole == 7.0).all())


def test_lookup_special_values():
    table = torch.tensor([[float("inf"), float("nan"), -0.0, 1e-40, 3e38, -65520.0, 65519.0, 1.0]],
                         device="cuda")
    for out_t in F.values():
        out = torch.empty((3, 8), dtype=out_t, device="cuda")
        ps.EmbeddingLookup(table, torch.tensor([0, -1, 0], device="cuda"), out)
        torch.testing.assert_close(out[[0, 2]], table.to(out_t).expand(2, 8), rtol=0, atol=0,
                                   equal_nan=True)
        assert bool((out[1] == 0).all())  # a masked id reads no row, whatever the table holds


def test_lookup_empty():
    table = torch.ones((3, 4), device="cuda")
    ps.EmbeddingLookup(table, torch.empty(0, dtype=torch.int32, device="cuda"),
                       torch.empty((0, 4), device="cuda"))
    out = torch.ones((2, 4), device="cuda")
    ps.EmbeddingLookup(torch.empty((0, 4), device="cuda"),
                       torch.tensor([0, 1], device="cuda"), out)
    assert bool((out == 0).all())


def test_lookup_beyond_32_bits():
    rows, cols = 1100000, 4096  # 4.5e9 elements
    table = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
    ids = torch.tensor([0, rows - 1, rows // 2 + 1, 524288, 524287], device="cuda")
    mark = torch.arange(1, 6, device="cuda", dtype=torch.bfloat16)
    table[ids] = mark[:, None].expand(5, cols)
    out = torch.empty((5, cols), dtype=torch.bfloat16, device="cuda")
    ps.EmbeddingLookup(table, ids, out)
    assert bool((out == mark[:, None]).all())
    # and a gradient whose rows lie beyond 2^32 elements
    dy = out.clone()
    work = ps.DeviceBuffer(ps.embedding_grad_workspace_bytes(5, cols, rows))
    ps.EmbeddingGrad(ids, dy, table, work, scale=2.0)
    torch.cuda.synchronize()
    assert bool((table[ids] == 2 * mark[:, None]).all())
    assert int(torch.count_nonzero(table.view(-1, 1 << 16).any(1))) <= 10
    assert float(table.sum(dtype=torch.float64)) == 2 * 15 * cols


# ids whose sorted runs meet the chunks' borders in every way
def runs(lengths, gen, spread=1):
    ids = torch.cat([torch.full((n,), r * spread) for r, n in enumerate(lengths)])
    return ids[torch.randperm(ids.numel(), generator=gen)]


RUNS = {
    "single": [1], "one_16": [16], "one_17": [17], "one_31": [31], "one_32": [32],
    "one_33": [33], "one_48": [48], "one_49": [49], "one_1000": [1000],
    "shift_32": [1, 32, 3], "shift_33": [1, 33], "shift_16": [15, 16, 17, 16, 16],
    "shift_47": [8, 47, 2], "two_long": [40, 40, 5, 100], "border": [16, 32, 16, 64, 1],
    "ladder": list(range(1, 70)), "ones": [1] * 100, "long_short": [500, 1, 1, 700, 2],
    "tail": [3] * 20 + [90], "5000": [5000, 3, 4000, 1, 1], "empty_rows": [0, 0, 3, 0, 50, 0],
}


def check_grad(ids, cols, rows, dy_t, grad_t, gen, scale=0.75, padding=-1, accumulate=False,
               pad=0, offset=0):
    dy, _ = values(gen, ids.numel(), cols, dy_t, pad, offset)
    grad, whole = ref.strided(rows, cols, grad_t, pad, offset, fill=7.0)
    before = None
    if accumulate:
        grad.copy_(torch.randn((rows, cols), generator=gen))
        before = grad.cpu().double()
    else:
        grad.fill_(float("nan"))
    work = torch.full((ps.embedding_grad_workspace_bytes(ids.numel(), cols, rows),), 255,
                      dtype=torch.uint8, device="cuda")
    again = grad.clone()
    where = ids.cuda()
    ps.EmbeddingGrad(where, dy, grad, work, scale=scale, padding_idx=padding,
                     accumulate=accumulate)
    work.fill_(90)
    ps.EmbeddingGrad(where, dy, again, work, scale=scale, padding_idx=padding,
                     accumulate=accumulate)
    torch.cuda.synchronize()
    exact, mag, most = ref.lookup_grad(ids, dy, rows, scale, padding)
    if accumulate:
        exact, mag = exact + before, mag + before.abs()
    ref.close(grad, exact, mag, most + 2, "gradient")
    assert torch.equal(grad, again)  # the same bits every time
    if accumulate:
        idle = torch.ones(rows, dtype=torch.bool)
        i = ids.long()
        idle[i[(i >= 0) & (i < rows) & (i != padding)]] = False
        assert torch.equal(grad.cpu()[idle].double(), before[idle])
    grad.fill_(7.0)
    assert bool((whole == 7.0).all())


@pytest.mark.parametrize("name", RUNS)
@pytest.mark.parametrize("dy_t,grad_t", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
def test_grad_runs(name, dy_t, grad_t):
    gen = generator(name, dy_t, grad_t)
    for cols, accumulate in ((8, False), (333, False), (37, True)):
        say(f"grad runs {name} {dy_t}->{grad_t} cols={cols} accumulate={accumulate}")
        ids = runs(RUNS[name], gen)
        check_grad(ids, cols, len(RUNS[name]), F[dy_t], F[grad_t], gen, accumulate=accumulate)


@pytest.mark.parametrize("dy_t,grad_t", list(itertools.product(F, F)))
@pytest.mark.parametrize("cols", [1, 3, 7, 8, 9, 33, 128, 1027, 2304])
@pytest.mark.parametrize("accumulate", [False, True])
def test_grad_types_and_widths(dy_t, grad_t, cols, accumulate):
    gen = generator(dy_t, grad_t, cols, accumulate)
    for count, rows, pad, offset, id_t in ((1, 1, 0, 0, torch.int64), (7, 300, 1, 1, torch.int32),
                                           (333, 40, 0, 3, torch.int64)):
        say(f"grad {dy_t}->{grad_t} cols={cols} count={count} rows={rows} accumulate={accumulate}")
        ids = torch.randint(-2, rows + 2, (count,), generator=gen).to(id_t)
        check_grad(ids, cols, rows, F[dy_t], F[grad_t], gen, accumulate=accumulate, pad=pad,
                   offset=offset, padding=rows // 2)


# 1, 2 and 3 passes of the sort; one tile and many
@pytest.mark.parametrize("rows", [2, 1023, 1024, 70001, (1 << 20) + 5, 3000000])
@pytest.mark.parametrize("count", [4095, 4096, 4097, 8192, 8193, 20011, 70001])
def test_grad_sorts(rows, count):
    gen = generator(rows, count)
    say(f"grad sort rows={rows} count={count}")
    u = torch.rand(count, generator=gen, dtype=torch.float64)
    ids = (rows * u * u * u).long()
    ids[::97] = -1
    check_grad(ids, 4, rows, torch.float32, torch.float32, gen)


# tiles added up by groups, tiles of several items a thread, the scanned table
@pytest.mark.parametrize("count", [65536, 65537, 300001, 1048577, 4300003])
def test_grad_long_lists(count):
    gen = generator("long", count)
    for rows in (5, 70001):
        say(f"grad long list rows={rows} count={count}")
        u = torch.rand(count, generator=gen, dtype=torch.float64)
        ids = (rows * u * u).long()
        ids[::97] = -1
        check_grad(ids, 2, rows, torch.float32, torch.float32, gen)


def test_grad_nothing():
    gen = generator("nothing")
    for ids in (torch.empty(0, dtype=torch.int64), torch.full((100,), -1), torch.full((40,), 9)):
        check_grad(ids, 5, 9, torch.float32, torch.float32, gen)
        check_grad(ids, 5, 9, torch.float32, torch.float32, gen, accumulate=True)


def test_grad_masked_rows_may_hold_anything():
    dy = torch.ones((40, 16), device="cuda")
    ids = torch.arange(40, device="cuda") % 4
    dy[ids == 2] = float("nan")
    ids = torch.where(ids == 2, -1, ids)
    dy[ids == 3] = float("inf")
    grad = torch.empty((4, 16), device="cuda")
    work = ps.DeviceBuffer(ps.embedding_grad_workspace_bytes(40, 16, 4))
    ps.EmbeddingGrad(ids, dy, grad, work, padding_idx=3)
    assert grad.cpu()[:, 0].tolist() == [10.0, 10.0, 0.0, 0.0]


def test_grad_against_differences():
    """The lookup is linear: <lookup(table + d) - lookup(table - d), r> / 2 = <grad(r), d>.
    Small whole numbers, so that both sides are exact."""
    gen = generator("differences")
    rows, cols, count = 60, 45, 500
    ids = torch.randint(-1, rows, (count,), generator=gen).cuda()
    table, d = (torch.randint(-4, 5, (rows, cols), generator=gen).float().cuda() for _ in range(2))
    r = torch.randint(-4, 5, (count, cols), generator=gen).float().cuda()
    up, down = torch.empty_like(r), torch.empty_like(r)
    ps.EmbeddingLookup(table + d, ids, up, scale=2.0)
    ps.EmbeddingLookup(table - d, ids, down, scale=2.0)
    grad = torch.empty_like(table)
    work = ps.DeviceBuffer(ps.embedding_grad_workspace_bytes(count, cols, rows))
    ps.EmbeddingGrad(ids, r, grad, work, scale=2.0)
    left = ((up - down).double() * r.double()).sum() / 2
    assert float(left) == float((grad.double() * d.double()).sum())


def test_on_another_stream():
    stream = torch.cuda.Stream()
    table = torch.randn((1000, 64), device="cuda")
    ids = torch.randint(0, 1000, (5000,), device="cuda")
    out, grad = torch.empty((5000, 64), device="cuda"), torch.empty_like(table)
    work = ps.DeviceBuffer(ps.embedding_grad_workspace_bytes(5000, 64, 1000))
    late = torch.zeros_like(table)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(50):
            late.add_(table)  # work before the call on its stream
        late.copy_(table)
    ps.EmbeddingLookup(late, ids, out, stream=stream.cuda_stream)
    ps.EmbeddingGrad(ids, out, grad, work, stream=stream)
    stream.synchronize()
    assert torch.equal(out, table[ids])
    exact, mag, most = ref.lookup_grad(ids, out, 1000, 1.0)
    ref.close(grad, exact, mag, most + 2, "gradient")


def test_in_a_graph():
    """Both calls captured once and replayed on new contents."""
    gen = generator("graph")
    table = torch.empty((3000, 48), device="cuda")
    ids = torch.empty(9000, dtype=torch.int64, device="cuda")
    out, grad = torch.empty((9000, 48), device="cuda"), torch.empty((3000, 48), device="cuda")
    work = torch.empty(ps.embedding_grad_workspace_bytes(9000, 48, 3000), dtype=torch.uint8,
                       device="cuda")

    def step():
        s = torch.cuda.current_stream().cuda_stream
        ps.EmbeddingLookup(table, ids, out, scale=3.0, stream=s)
        ps.EmbeddingGrad(ids, out, grad, work, stream=s)

    def contents():
        table.copy_(torch.randn((3000, 48), generator=gen))
        ids.copy_(torch.randint(-1, 3000, (9000,), generator=gen))

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
        grad.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone(), grad.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(replayed[0], out) and torch.equal(replayed[1], grad)


@pytest.mark.parametrize("most,counts,cols,rows", [
    (16392, (16384, 8191, 1), 1024, 50000),  # chunks of twice the entries
    (196616, (196608, 65537), 8, 1024),      # tiles of twice the items, two digits
    (196616, (196608, 196600), 8, 1023),
    (4194400, (4194304, 800000), 1, 3000)])  # no groups of tiles any more
def test_grad_in_a_workspace_for_more(most, counts, cols, rows):
    gen = generator("workspace", most, rows)
    work = torch.full((ps.embedding_grad_workspace_bytes(most, cols, rows),), 255,
                      dtype=torch.uint8, device="cuda")
    for count in counts:
        say(f"grad of {count} ids in a workspace for {most}")
        ids = torch.randint(-1, rows, (count,), generator=gen)
        dy, _ = values(gen, count, cols, torch.float32)
        grad = torch.full((rows, cols), float("nan"), device="cuda")
        ps.EmbeddingGrad(ids.cuda(), dy, grad, work)
        torch.cuda.synchronize()
        exact, mag, times = ref.lookup_grad(ids, dy, rows, 1.0)
        ref.close(grad, exact, mag, times + 2, "gradient")
