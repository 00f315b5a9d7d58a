"""Layer norm and its gradients against 64-bit plain forms: types, widths from one column to
beyond what registers hold, strides and odd alignments, rows without spread, missing weights,
gradients against differences, workspaces, streams and graphs."""
import zlib

import pytest
import torch

import more_rows_ref as ref
import powersparse_amd as ps
import rows_ref
from gpu_util import say, setup

pytestmark = pytest.mark.gpu

F = rows_ref.DTYPES
# around the pieces, the lanes and the pieces a lane of every kernel
WIDTHS = [1, 2, 3, 4, 5, 7, 8, 9, 31, 32, 33, 63, 64, 65, 128, 255, 257, 333, 512, 513, 1000, 1024,
          1025, 2047, 2048, 2049, 4096, 4100, 8192, 8195, 16384, 16390, 32768, 32777, 50001]


@pytest.fixture(scope="module", autouse=True)
def device():
    setup()


def generator(*key):
    g = torch.Generator()
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def rows_of(gen, rows, cols, dtype, pad=0, offset=0, mean=0.5):
    x = torch.randn((rows, cols), generator=gen) * torch.exp(torch.randn((rows, 1), generator=gen))
    x += mean * torch.randn((rows, 1), generator=gen)
    view, whole = rows_ref.strided(rows, cols, dtype, pad, offset)
    view.copy_(x)
    return view, whole


def vector(gen, cols, dtype, base):
    return (base + 0.2 * torch.randn(cols, generator=gen)).to(dtype).cuda()


def forward(x, w, b, y_dtype, pad=0, offset=0, eps=1e-5):
    y, whole = rows_ref.strided(x.shape[0], x.shape[1], y_dtype, pad, offset, fill=7.0)
    mean, rstd = (torch.full((x.shape[0],), 7.0, device="cuda") for _ in range(2))
    ps.LayerNorm(x, w, b, y, mean, rstd, eps=eps)
    torch.cuda.synchronize()
    want = ref.norm(x, w, b, eps)
    for got, (exact, off), what in zip((y, mean, rstd), want, ("y", "mean", "rstd")):
        ref.held(got, exact, off, what)
    y.fill_(7.0)
    assert bool((whole == 7.0).all())  # nothing outside the rows was written
    return mean, rstd


def backward(gen, x, w, mean, rstd, dy_dtype, sums, pad=0, offset=0, accumulate=False):
    rows, cols = x.shape
    dy, _ = rows_of(gen, rows, cols, dy_dtype, pad, offset, mean=0.1)
    dx, whole = rows_ref.strided(rows, cols, x.dtype, pad, offset, fill=7.0)
    was = [torch.randn(cols, generator=gen).to(sums).cuda() for _ in range(2)]
    dw, db = (v.clone() for v in was)
    work = torch.empty(ps.layer_norm_grad_workspace_bytes(rows, cols), dtype=torch.uint8,
                       device="cuda").fill_(255)
    ps.LayerNormGrad(dy, x, w, mean, rstd, dx, dw, db, work, accumulate=accumulate)
    torch.cuda.synchronize()
    want = ref.norm_grad(dy, x, w, mean, rstd)
    ref.held(dx, *want[0], "dx")
    for got, before, (exact, off), what in zip((dw, db), was, want[1:], ("dweight", "dbias")):
        if accumulate:
            before = before.cpu().double()
            exact = exact + before
            off = off + ref.U32 * exact.abs()
        ref.held(got, exact, off, what)
    dx.fill_(7.0)
    assert bool((whole == 7.0).all())
    return dy, work


@pytest.mark.parametrize("cols", WIDTHS)
def test_widths(cols):
    gen = generator("widths", cols)
    for k, (rows, dtype) in enumerate([(1, "f32"), (7, "bf16"), (37, "f32"), (65, "f16")]):
        if rows * cols > 1 << 20:
            rows = 5
        say(f"layer norm {rows} x {cols} {dtype}")
        x, _ = rows_of(gen, rows, cols, F[dtype])
        w, b = vector(gen, cols, torch.float32, 1.0), vector(gen, cols, torch.float32, 0.0)
        mean, rstd = forward(x, w, b, F[dtype])
        if cols > 1:
            backward(gen, x, w, mean, rstd, F[dtype], torch.float32, accumulate=k == 2)


@pytest.mark.parametrize("x_type", sorted(F))
@pytest.mark.parametrize("y_type", sorted(F))
def test_types(x_type, y_type):
    for cols, w_type in ((40, "f32"), (333, "bf16"), (1028, "f16"), (6, "f32")):
        gen = generator("types", x_type, y_type, cols)
        say(f"layer norm {x_type} {y_type} {cols}")
        x, _ = rows_of(gen, 29, cols, F[x_type])
        w, b = vector(gen, cols, F[w_type], 1.0), vector(gen, cols, F[w_type], 0.1)
        mean, rstd = forward(x, w, b, F[y_type])
        backward(gen, x, w, mean, rstd, F[y_type], F[w_type])


@pytest.mark.parametrize("dtype", sorted(F))
@pytest.mark.parametrize("cols,pad,offset", [(8, 1, 1), (64, 3, 5), (333, 0, 1), (100, 28, 3),
                                             (2048, 7, 1), (5000, 1, 7), (40000, 5, 3)])
def test_strides_and_alignments(dtype, cols, pad, offset):
    gen = generator("strides", dtype, cols)
    x, _ = rows_of(gen, 11, cols, F[dtype], pad, offset)
    w = vector(gen, cols + 1, F[dtype], 1.0)[1:]
    mean, rstd = forward(x, w, None, F[dtype], pad, offset)
    backward(gen, x, w, mean, rstd, F[dtype], torch.float32, pad, offset)


@pytest.mark.parametrize("rows", [1, 2, 3, 63, 64, 65, 1023, 1024, 1025, 4099, 20011])
@pytest.mark.parametrize("cols", [4, 33, 128, 320])
def test_rows(rows, cols):
    """Row counts around the workgroups' shares."""
    gen = generator("rows", rows, cols)
    x, _ = rows_of(gen, rows, cols, torch.float32)
    mean, rstd = forward(x, None, None, torch.float32)
    backward(gen, x, None, mean, rstd, torch.float32, torch.float32)


def test_large_mean():
    """Deviations that are small against the mean: sums of squares would cancel."""
    for cols in (64, 1000, 9000, 70000):
        gen = generator("mean", cols)
        x = 1000.0 + torch.randn((9, cols), generator=gen)
        forward(x.cuda(), None, None, torch.float32)


def test_rows_of_one_value():
    for cols in (1, 5, 64, 1000, 40000):
        x = torch.full((3, cols), 3.25, device="cuda")
        b = torch.randn(cols, device="cuda")
        y, rstd = torch.empty_like(x), torch.empty(3, device="cuda")
        ps.LayerNorm(x, None, b, y, None, rstd, eps=0.0625)
        assert torch.equal(y, b.expand_as(y)) and bool((rstd == 4.0).all())
        ps.LayerNorm(x, None, b, y, eps=0.0)
        assert bool(torch.isnan(y).all())


def test_rows_do_not_meet():
    """A row that holds NaN or infinities makes no other row so."""
    for cols in (8, 100, 3000, 40000):
        x = torch.randn((5, cols), device="cuda")
        x[1, cols // 2], x[3, 0] = float("nan"), float("inf")
        y = torch.empty_like(x)
        ps.LayerNorm(x, None, None, y)
        assert torch.isfinite(y).all(1).tolist() == [True, False, True, False, True]


def test_nothing_to_do():
    x = torch.empty((0, 64), device="cuda")
    ps.LayerNorm(x, None, None, torch.empty_like(x), torch.empty(0, device="cuda"),
                 torch.empty(0, device="cuda"))
    dw, db = torch.full((64,), 7.0, device="cuda"), torch.full((64,), 7.0, device="cuda")
    none = torch.empty(0, device="cuda")
    work = torch.empty(ps.layer_norm_grad_workspace_bytes(0, 64), dtype=torch.uint8, device="cuda")
    ps.LayerNormGrad(x, x, None, none, none, x, dw, db, work, accumulate=True)
    assert bool((dw == 7).all()) and bool((db == 7).all())
    ps.LayerNormGrad(x, x, None, none, none, x, dw, db, work)
    assert bool((dw == 0).all()) and bool((db == 0).all())


def test_sums_that_are_not_wanted():
    gen = generator("unwanted")
    for cols in (40, 40000):
        x, _ = rows_of(gen, 70, cols, torch.float32)
        dy = torch.randn((70, cols), generator=gen).cuda()
        mean, rstd = torch.empty(70, device="cuda"), torch.empty(70, device="cuda")
        ps.LayerNorm(x, None, None, torch.empty_like(x), mean, rstd)
        work = torch.empty(ps.layer_norm_grad_workspace_bytes(70, cols), dtype=torch.uint8,
                           device="cuda")
        outs = [torch.empty_like(x) for _ in range(4)]
        dw, db, dw2, db2 = (torch.empty(cols, device="cuda") for _ in range(4))
        ps.LayerNormGrad(dy, x, None, mean, rstd, outs[0], dw, db, work)
        ps.LayerNormGrad(dy, x, None, mean, rstd, outs[1], None, db2, work)
        ps.LayerNormGrad(dy, x, None, mean, rstd, outs[2], dw2, None, work)
        ps.LayerNormGrad(dy, x, None, mean, rstd, outs[3], None, None, None)
        assert torch.equal(dw, dw2) and torch.equal(db, db2)
        assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_gradients_against_differences():
    """Central differences of sum(dy * y), the forward pass in 64 bits by its formula: with steps of
    2^-10 they are off by some h^2 of the third derivatives."""
    gen = generator("differences")
    x, dy = (torch.randn((3, 24), generator=gen) for _ in range(2))
    w, b = 1 + 0.2 * torch.randn(24, generator=gen), torch.randn(24, generator=gen)

    def loss(x, w, b):
        return float((dy.double() * ref.norm(x, w, b, 1e-5)[0][0]).sum())

    d = [v.cuda() for v in (x, w, b)]
    mean, rstd = torch.empty(3, device="cuda"), torch.empty(3, device="cuda")
    ps.LayerNorm(*d, torch.empty_like(d[0]), mean, rstd)
    dx, dw, db = (torch.empty_like(v) for v in d)
    work = torch.empty(ps.layer_norm_grad_workspace_bytes(3, 24), dtype=torch.uint8, device="cuda")
    ps.LayerNormGrad(dy.cuda(), d[0], d[1], mean, rstd, dx, dw, db, work)
    h = 2.0 ** -10
    args = [x.double(), w.double(), b.double()]
    for k, got in enumerate((dx, dw, db)):
        flat = got.cpu().view(-1)
        for i in range(flat.numel()):
            moved = []
            for s in (h, -h):
                a = [v.clone() for v in args]
                a[k].view(-1)[i] += s
                moved.append(loss(*a))
            want = (moved[0] - moved[1]) / (2 * h)
            assert abs(float(flat[i]) - want) <= 1e-4 * (1 + abs(want)), (k, i, float(flat[i]), want)


def test_the_same_bits_every_time_and_workspaces_made_for_more():
    gen = generator("bits")
    x, _ = rows_of(gen, 5003, 200, torch.bfloat16)
    dy = torch.randn((5003, 200), generator=gen).to(torch.bfloat16).cuda()
    mean, rstd = torch.empty(5003, device="cuda"), torch.empty(5003, device="cuda")
    ps.LayerNorm(x, None, None, torch.empty_like(x), mean, rstd)
    work = torch.empty(ps.layer_norm_grad_workspace_bytes(6000, 1000), dtype=torch.uint8,
                       device="cuda")
    got = []
    for fill in (0, 255, 1):
        work.fill_(fill)
        dx, dw, db = torch.empty_like(dy), torch.empty(200, device="cuda"), \
            torch.empty(200, device="cuda")
        ps.LayerNormGrad(dy, x, None, mean, rstd, dx, dw, db, work)
        got.append((dx, dw, db))
    assert all(torch.equal(a, b) for other in got[1:] for a, b in zip(got[0], other))


@pytest.mark.parametrize("cols", [96, 2048, 40000])
def test_in_a_graph_on_a_stream(cols):
    gen = generator("graph", cols)
    rows = 3000 if cols < 4096 else 9
    x = torch.randn((rows, cols), generator=gen).cuda()
    dy = torch.randn((rows, cols), generator=gen).cuda()
    w, b = torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
    work = torch.empty(ps.layer_norm_grad_workspace_bytes(rows, cols), dtype=torch.uint8,
                       device="cuda")
    outs = [torch.empty_like(x), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"),
            torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")]

    def step():
        s = torch.cuda.current_stream()
        ps.LayerNorm(x, w, b, *outs[:3], stream=s)
        ps.LayerNormGrad(dy, x, w, outs[1], outs[2], *outs[3:], work, stream=s)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        for t in (x, dy):
            t.copy_(torch.randn(t.shape, generator=gen))
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [o.clone() for o in outs]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, o) for a, o in zip(replayed, outs))


def test_offsets_beyond_32_bits():
    """Rows so far apart that their places need 64 bits."""
    rows, cols = 5, 24
    ld = (1 << 30) + 3
    whole = torch.empty(4 * ld + cols, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(whole, (rows, cols), (ld, 1))
    gen = generator("far")
    x.copy_(torch.randn((rows, cols), generator=gen))
    y = torch.empty((rows, cols), device="cuda")
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ps.LayerNorm(x, None, None, y, mean, rstd)
    near = x.contiguous()
    ref.held(y, *ref.norm(near, None, None, 1e-5)[0], "y")
    dy, dx = torch.randn((rows, cols), generator=gen).cuda(), torch.empty_like(near)
    ps.LayerNormGrad(dy, x, None, mean, rstd, dx, None, None, None)
    want = ref.norm_grad(dy, near, None, mean, rstd)[0]
    ref.held(dx, *want, "dx")
    ps.LayerNormGrad(dy, near, None, mean, rstd, x, None, None, None)
    assert torch.equal(x, dx)
