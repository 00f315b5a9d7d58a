"""The row operators where their kernels change with the size: outputs stored with
the non-temporal hint (32 MB and more), long chunks of the lookup's gradient, more
workgroups than one launch takes, tables of almost 2^31 rows. The plain forms run on the device, in 64 bits."""
import zlib

import pytest
import torch

import powersparse_amd as ps
import rows_ref as ref
from gpu_util import say, setup

pytestmark = pytest.mark.gpu

F = ref.DTYPES
MB32 = 32 << 20


@pytest.fixture(scope="module", autouse=True)
def device():
    setup()


def generator(*key):
    g = torch.Generator(device="cuda")
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def matrix(gen, rows, cols, dtype, pad=0, offset=0):
    view, whole = ref.strided(rows, cols, dtype, pad, offset, fill=7.0)
    view.copy_(torch.randn((rows, cols), generator=gen, device="cuda"))
    return view, whole


def untouched(view, whole):
    """Nothing outside the rows was written."""
    view.fill_(7.0)
    assert bool((whole == 7.0).all())


def rows_for(cols, dtype):
    return MB32 // (cols * dtype.itemsize) + 3


@pytest.mark.parametrize("table_t,out_t,cols", [
    ("f32", "f32", 333), ("f32", "f32", 3), ("bf16", "bf16", 333), ("bf16", "f16", 1023),
    ("f16", "f32", 2049), ("f32", "bf16", 65), ("f16", "f16", 8), ("bf16", "f32", 4096)])
def test_lookup_of_large_outputs(table_t, out_t, cols):
    gen = generator(table_t, out_t, cols)
    count, rows = rows_for(cols, F[out_t]), 4001
    table, _ = matrix(gen, rows, cols, F[table_t], 3, 1)
    ids = torch.randint(-1, rows + 1, (count,), generator=gen, device="cuda")
    ok = (ids >= 0) & (ids < rows)
    for pad, offset in ((0, 0), (5, 3)):
        say(f"large lookup {table_t}->{out_t} cols={cols} count={count} pad={pad}")
        out, whole = ref.strided(count, cols, F[out_t], pad, offset, fill=7.0)
        ps.EmbeddingLookup(table, ids, out, scale=1.25)
        exact = torch.where(ok[:, None], table[ids.clamp(0, rows - 1)].double() * 1.25, 0.0).cpu()
        ref.close(out, exact, exact.abs(), 1, "lookup")
        untouched(out, whole)


# 8, 16, 32 and 64 lanes a token, a workgroup a token
@pytest.mark.parametrize("dtype,cols", [("f32", 3), ("bf16", 63), ("f16", 121), ("bf16", 249),
                                        ("f32", 333), ("bf16", 2057), ("f32", 2049)])
def test_experts_of_large_outputs(dtype, cols):
    gen = generator(dtype, cols)
    t = F[dtype]
    tokens, top_k = rows_for(cols, t), 3
    slots = tokens * top_k
    ids = torch.randint(-1, 6, (tokens, top_k), generator=gen, device="cuda")
    order, position = (torch.empty(slots, dtype=torch.int32, device="cuda") for _ in range(2))
    position = position.view(tokens, top_k)
    offsets = torch.empty(7, dtype=torch.int32, device="cuda")
    work = ps.DeviceBuffer(ps.expert_sort_workspace_bytes(slots, 6))
    ps.ExpertSort(ids, order, position, offsets, work)
    filled = int(offsets[-1])
    assert filled == int((ids >= 0).sum())
    on, at = position >= 0, position.clamp(min=0).long()
    weights = torch.rand((tokens, top_k), generator=gen, device="cuda")
    w = torch.where(on, weights, 0.0).double()
    for pad, offset in ((0, 0), (5, 3)):
        say(f"large experts {dtype} cols={cols} tokens={tokens} pad={pad}")
        x, _ = matrix(gen, tokens, cols, t, pad, offset)
        xs, whole = ref.strided(slots, cols, t, pad, offset, fill=7.0)
        ps.ExpertDispatch(x, position, xs)
        assert torch.equal(xs[:filled], x[order[:filled].long() // top_k])
        assert bool((xs[filled:] == 7.0).all())
        untouched(xs, whole)

        ys, _ = matrix(gen, slots, cols, t, pad, offset)
        y, whole = ref.strided(tokens, cols, t, pad, offset, fill=7.0)
        ps.ExpertCombine(ys, position, weights, y)
        exact, mag = (torch.zeros((tokens, cols), dtype=torch.float64, device="cuda")
                      for _ in range(2))
        for k in range(top_k):
            term = w[:, k, None] * ys[at[:, k]].double()
            exact += term
            mag += term.abs()
        ref.close(y, exact.cpu(), mag.cpu(), 2 * top_k, "combine")
        untouched(y, whole)

        dys, whole = ref.strided(slots, cols, t, pad, offset, fill=7.0)
        dw = torch.full((tokens, top_k), 7.0, device="cuda")
        ps.ExpertCombineGrad(x, ys, position, weights, dys, dw)
        for k in range(top_k):
            term = x.double() * ys[at[:, k]].double()
            exact = torch.where(on[:, k], term.sum(1), 0.0)
            ref.close(dw[:, k], exact.cpu(), term.abs().sum(1).cpu(), cols + 1, "dweights")
        token, k = order[:filled].long() // top_k, order[:filled].long() % top_k
        exact = (weights[token, k].double()[:, None] * x[token].double()).cpu()
        ref.close(dys[:filled], exact, exact.abs(), 1, "dys")
        assert bool((dys[filled:] == 7.0).all())
        untouched(dys, whole)


# Chunks of 64, 128 and 256 entries, of many pieces each (4096 columns) and of few.
@pytest.mark.parametrize("chunk,count,cols,dy_t,grad_t", [
    (64, 20000, 4096, "bf16", "f32"), (128, 40000, 4093, "f32", "f32"),
    (256, 100000, 4096, "bf16", "bf16"), (64, 262147, 333, "f16", "f16"),
    (128, 500000, 333, "bf16", "bf16"), (256, 1200000, 333, "f16", "f16"),
    (256, 1200000, 250, "bf16", "f32")])
def test_grad_of_long_chunks(chunk, count, cols, dy_t, grad_t):
    gen = generator(chunk, count, cols)
    say(f"grad of chunks of {chunk}: {count} ids, {cols} columns {dy_t}->{grad_t}")
    pick = torch.Generator().manual_seed(chunk + cols)
    kinds = [1, 2, 3, chunk - 1, chunk, chunk + 1, 2 * chunk - 1, 2 * chunk, 2 * chunk + 1,
             3 * chunk + 2, 63 * chunk, 65 * chunk + 1, 66 * chunk]
    lengths, left = [], count - 70
    while left > 0:
        n = kinds[int(torch.randint(0, len(kinds), (1,), generator=pick))]
        lengths.append(min(n, left))
        left -= lengths[-1]
    ids = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
    ids = torch.cat([ids, torch.full((70,), -1)]).cuda()
    ids = ids[torch.randperm(count, generator=gen, device="cuda")]
    rows = len(lengths) + 2
    dy = torch.randn((count, cols), generator=gen, device="cuda").to(F[dy_t])
    exact, mag = (torch.zeros((rows, cols), dtype=torch.float64, device="cuda") for _ in range(2))
    keep = torch.nonzero(ids >= 0).view(-1)
    for part in keep.split(1 << 16):
        exact.index_add_(0, ids[part], dy[part].double() * 0.75)
        mag.index_add_(0, ids[part], dy[part].double().abs() * 0.75)
    exact, mag, most = exact.cpu(), mag.cpu(), max(lengths)
    work = torch.full((ps.embedding_grad_workspace_bytes(count, cols, rows),), 255,
                      dtype=torch.uint8, device="cuda")
    grad, whole = ref.strided(rows, cols, F[grad_t], 3, 1, fill=7.0)
    ps.EmbeddingGrad(ids, dy, grad, work, scale=0.75)
    ref.close(grad, exact, mag, most + 2, "gradient")
    again = torch.empty((rows, cols), dtype=F[grad_t], device="cuda")
    ps.EmbeddingGrad(ids, dy, again, work, scale=0.75)
    assert torch.equal(grad, again)
    before = again.cpu().double()
    ps.EmbeddingGrad(ids, dy, again, work, scale=0.75, accumulate=True)
    ref.close(again, exact + before, mag + before.abs(), most + 2, "accumulated gradient")
    untouched(grad, whole)


def test_more_workgroups_than_a_launch_takes():
    """Rows of 7 columns are moved an element a thread, 2^21 workgroups of 256 a launch."""
    gen = generator("launches")
    cols = 7
    n = (1 << 29) // cols + 1000
    say(f"{n} rows of {cols} columns")
    table = torch.randn((3001, cols), generator=gen, device="cuda").half()
    ids = torch.randint(0, 3001, (n,), generator=gen, device="cuda", dtype=torch.int32)
    x = torch.full((n, cols), 7.0, dtype=torch.float16, device="cuda")
    ps.EmbeddingLookup(table, ids, x)
    assert torch.equal(x, table[ids])
    position = torch.randperm(n, generator=gen, device="cuda", dtype=torch.int32).view(n, 1)
    xs = torch.full((n, cols), 7.0, dtype=torch.float16, device="cuda")
    ps.ExpertDispatch(x, position, xs)
    assert torch.equal(xs[position.view(-1)], x)
    y = torch.full((n, cols), 7.0, dtype=torch.float16, device="cuda")
    ps.ExpertDispatchGrad(xs, position, y)
    assert torch.equal(y, x)
    # whole numbers, so that the dots are exact
    x.copy_((ids[:, None] % 5).expand(n, cols))
    xs[position.view(-1)] = x
    weights = (ids % 3).float().view(n, 1)
    dys = torch.full((n, cols), 7.0, dtype=torch.float16, device="cuda")
    dw = torch.full((n, 1), 7.0, device="cuda")
    ps.ExpertCombineGrad(x, xs, position, weights, dys, dw)
    assert torch.equal(dw.view(-1), (ids % 5).float().square() * cols)
    assert torch.equal(dys[position.view(-1)], x * weights.half())


@pytest.mark.parametrize("count", [100, 10000])
def test_tables_of_almost_2_to_31_rows(count):
    """Four digits of the ids, offsets beyond 2^33, rows to clear for more than one launch."""
    gen = generator("rows", count)
    rows, cols = (1 << 31) - 2, 5
    say(f"gradient of {count} ids, {rows} rows of {cols} columns")
    ids = torch.randint(0, rows, (count,), generator=gen, device="cuda")
    ids[:6] = torch.tensor([0, rows - 1, rows, -1, 1 << 30, rows - 1], device="cuda")
    ids[6:40] = (1 << 24) + 17
    dy = torch.randint(1, 5, (count, cols), generator=gen, device="cuda").half()
    grad = torch.full((rows, cols), float("nan"), dtype=torch.float16, device="cuda")
    work = torch.full((ps.embedding_grad_workspace_bytes(count, cols, rows),), 255,
                      dtype=torch.uint8, device="cuda")
    ps.EmbeddingGrad(ids, dy, grad, work)
    named, at = torch.unique(ids[(ids >= 0) & (ids < rows)], return_inverse=True)
    exact = torch.zeros((named.numel(), cols), dtype=torch.float64, device="cuda")
    exact.index_add_(0, at, dy[(ids >= 0) & (ids < rows)].double())
    assert torch.equal(grad[named].double(), exact)  # whole numbers below 2^11
    nonzero = sum(int(torch.count_nonzero(part)) for part in grad.split(1 << 27))
    assert nonzero == named.numel() * cols
    out = torch.empty((count, cols), dtype=torch.float16, device="cuda")
    ps.EmbeddingLookup(grad, ids, out, scale=0.5)
    assert bool((out[2:4] == 0).all())
    keep = (ids >= 0) & (ids < rows)
    assert torch.equal(out[keep].double(), exact[at] * 0.5)
