"""The norm over many gradient tensors and clipping, against 64-bit sums: types,
sizes from nothing to several chunks, odd alignments, in place and into other
buffers, norms beyond FP32's squares, zeros, infinities and NaN."""
import math
import zlib

import pytest
import torch

import powersparse_amd as ps
import rows_ref as ref
from gpu_util import say, setup

pytestmark = pytest.mark.gpu

F = ref.DTYPES
SIZES = [1, 0, 7, 2048, 2049, 1, 100003, 8, 4096, 333]


@pytest.fixture(scope="module", autouse=True)
def device():
    setup()


def generator(*key):
    g = torch.Generator()
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def tensors(gen, sizes, dtypes, std=1.0):
    """Views at odd places of larger buffers, so that few are aligned to 16 bytes."""
    out = []
    for i, n in enumerate(sizes):
        whole = torch.full((n + 16,), 7.0, dtype=dtypes[i % len(dtypes)], device="cuda")
        v = whole[i % 5:i % 5 + n]
        v.copy_(torch.randn(n, generator=gen) * std)
        out.append((v, whole, i % 5))
    return out


def norm_of(grads, scale=1.0):
    return abs(scale) * math.sqrt(sum(float(g.double().square().sum()) for g in grads))


def check(grads, outs, before, max_norm, scale, norm, what):
    exact = norm_of(before, scale)
    # 64-bit sums: one rounding to FP32, and far less from the sums themselves
    assert abs(float(norm) - exact) <= 2 * ref.U32 * exact + 2.0 ** -149, (float(norm), exact)
    c = min(1.0, max_norm / (exact + 1e-6)) * scale
    for b, o in zip(before, outs):
        e = b.cpu().double() * c
        ref.close(o, e, e.abs(), 2, what)  # c's rounding and the product's


@pytest.mark.parametrize("dtypes", [("f32",), ("f16",), ("bf16",), ("f32", "bf16", "f16")])
@pytest.mark.parametrize("out", [None, "f32", "bf16", "f16"])
@pytest.mark.parametrize("ratio", [0.5, 3.0])
def test_clip(dtypes, out, ratio):
    gen = generator(dtypes, out, ratio)
    for scale in (1.0, 0.125):
        say(f"clip {dtypes} out={out} ratio={ratio} scale={scale}")
        parts = tensors(gen, SIZES, [F[d] for d in dtypes])
        grads = [p[0] for p in parts]
        before = [g.clone() for g in grads]
        dst = parts if out is None else tensors(gen, SIZES, [F[out]])
        outs = [p[0] for p in dst]
        max_norm = norm_of(before, scale) / ratio
        norm = torch.full((1,), 7.0, device="cuda")
        glist = ps.GradientList(grads, None if out is None else outs)
        ps.GradNorm(glist, norm, grad_scale=scale)
        alone = norm.clone()
        assert all(torch.equal(g, b) for g, b in zip(grads, before))
        ps.ClipGradNorm(glist, max_norm, norm, grad_scale=scale)
        torch.cuda.synchronize()
        assert torch.equal(norm, alone)
        check(grads, outs, before, max_norm, scale, norm, "clip")
        if out is not None:
            assert all(torch.equal(g, b) for g, b in zip(grads, before))
        for v, whole, at in dst:  # nothing outside the tensors was written
            v.fill_(7.0)
            assert bool((whole == 7.0).all())


def test_given_norm():
    gen = generator("given")
    grads = [p[0] for p in tensors(gen, SIZES, [torch.float32])]
    before = [g.clone() for g in grads]
    norm = torch.tensor([1000.0], device="cuda")
    glist = ps.GradientList(grads)
    ps.ClipGrads(glist, 250.0, norm)
    for g, b in zip(grads, before):
        e = b.cpu().double() * (250.0 / (1000.0 + 1e-6))
        ref.close(g, e, e.abs(), 2, "given norm")
    assert float(norm) == 1000.0
    ps.ClipGrads(glist, 2000.0, norm)  # within the bound: the same bits
    for g, b in zip(grads, before):
        e = b.cpu().double() * (250.0 / (1000.0 + 1e-6))
        ref.close(g, e, e.abs(), 2, "given norm")


def test_beyond_squares_in_32_bits():
    """Norms whose squares overflow or vanish in FP32."""
    for value in (1e25, 1e-30):
        g = torch.full((5000,), value, device="cuda")
        norm = torch.empty(1, device="cuda")
        ps.GradNorm(ps.GradientList([g]), norm)
        exact = float(g.double().square().sum().sqrt())
        assert abs(float(norm) - exact) <= 2 * ref.U32 * exact


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_not_finite(bad):
    g = torch.ones(10000, device="cuda")
    g[7777] = bad
    norm = torch.empty(1, device="cuda")
    ps.ClipGradNorm(ps.GradientList([g]), 1.0, norm)
    if math.isnan(bad):
        assert math.isnan(float(norm)) and bool(torch.isnan(g).all())
    else:
        assert float(norm) == math.inf
        assert math.isnan(float(g[7777])) and float(g.nan_to_num().abs().sum()) == 0


def test_zeros_and_bound_zero():
    g = torch.zeros(3000, device="cuda")
    norm = torch.full((1,), 7.0, device="cuda")
    ps.ClipGradNorm(ps.GradientList([g]), 1.0, norm)
    assert float(norm) == 0.0 and bool((g == 0).all())
    g.fill_(1.0)
    ps.ClipGradNorm(ps.GradientList([g]), 0.0, norm)
    assert bool((g == 0).all())


def test_nothing():
    norm = torch.full((1,), 7.0, device="cuda")
    for grads in ([], [torch.empty(0, device="cuda")]):
        norm.fill_(7.0)
        ps.GradNorm(ps.GradientList(grads), norm)
        assert float(norm) == 0.0
        norm.fill_(7.0)
        ps.ClipGradNorm(ps.GradientList(grads), 1.0, norm)
        assert float(norm) == 0.0
        ps.ClipGrads(ps.GradientList(grads), 1.0, norm)


def test_many_tensors_side_by_side():
    """Neighbours in one buffer, in place and into another one."""
    gen = generator("many")
    sizes = [int(n) for n in torch.randint(0, 9000, (700,), generator=gen)]
    whole = torch.randn(sum(sizes), generator=gen).cuda()
    before = whole.cpu().double()
    norm = torch.empty(1, device="cuda")
    out = torch.empty(sum(sizes), dtype=torch.bfloat16, device="cuda")
    ps.ClipGradNorm(ps.GradientList(whole.split(sizes), out.split(sizes)), 2.0, norm)
    e = before * (2.0 / (float(before.square().sum().sqrt()) + 1e-6))
    ref.close(out, e, e.abs(), 2, "into another buffer")
    ps.ClipGradNorm(ps.GradientList(whole.split(sizes)), 2.0, norm)
    ref.close(whole, e, e.abs(), 2, "in place")


def test_large():
    """Several chunks a workgroup, counts beyond 2^32 elements."""
    n = (1 << 32) + 5
    g = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    h = torch.ones(1000, device="cuda")
    norm = torch.empty(1, device="cuda")
    ps.ClipGradNorm(ps.GradientList([g, h]), 1.0, norm)
    exact = math.sqrt(n + 1000)
    assert abs(float(norm) - exact) <= 2 * ref.U32 * exact
    c = torch.tensor(1.0 / (exact + 1e-6))
    assert bool((g == c.to(torch.bfloat16)).all())
    assert abs(float(h[-1]) - float(c)) <= 4 * ref.U32 * float(c)


def test_in_a_graph():
    gen = generator("graph")
    parts = tensors(gen, SIZES, [torch.float32, torch.bfloat16])
    grads = [p[0] for p in parts]
    outs = [torch.empty(g.shape, device="cuda") for g in grads]
    norm = torch.empty(1, device="cuda")
    glist = ps.GradientList(grads, outs)

    def step():
        ps.ClipGradNorm(glist, 1.0, norm, stream=torch.cuda.current_stream().cuda_stream)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(3):
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [norm.clone()] + [o.clone() for o in outs]
        step()
        torch.cuda.synchronize()
        assert torch.equal(replayed[0], norm)
        assert all(torch.equal(a, b) for a, b in zip(replayed[1:], outs))


def test_a_norm_in_a_gradient_is_refused():
    """Workgroups read the gradients while one writes the norm, and read the norm while they
    write the outputs."""
    whole = torch.ones(3000, device="cuda")
    grads = [whole[2000:3000], whole[:1000], whole[1000:1500]]  # two of them side by side
    outs = [torch.ones(g.numel() * 2, device="cuda")[:g.numel()] for g in grads]
    apart = torch.zeros(4, device="cuda")
    for glist, in_place in ((ps.GradientList(grads), True), (ps.GradientList(grads, outs), False)):
        for at in (0, 999, 1000, 1499, 2000, 2999):
            with pytest.raises(ValueError, match="norm lies in"):
                ps.GradNorm(glist, whole[at:at + 1])
            with pytest.raises(ValueError, match="norm lies in"):
                ps.ClipGradNorm(glist, 1.0, whole[at:at + 1])
            if in_place:
                with pytest.raises(ValueError, match="norm lies in"):
                    ps.ClipGrads(glist, 1.0, whole[at:at + 1])
            else:  # it is only read there, and the outputs are elsewhere
                ps.ClipGrads(glist, 1.0, whole[at:at + 1])
        if not in_place:
            for at in (0, 999):
                with pytest.raises(ValueError, match="norm lies in"):
                    ps.ClipGrads(glist, 1.0, outs[0][at:at + 1])
                with pytest.raises(ValueError, match="norm lies in"):
                    ps.ClipGradNorm(glist, 1.0, outs[0][at:at + 1])
        assert bool((whole == 1).all())
        for norm in (whole[1500:1501], whole[1999:2000], apart[1:2]):  # between them, and apart
            norm.zero_()
            ps.GradNorm(glist, norm)
            assert float(norm) == 50.0
            ps.ClipGrads(glist, 100.0, norm)
            ps.ClipGradNorm(glist, 100.0, norm)
            assert float(norm) == 50.0
            norm.fill_(1.0)
    assert bool((whole == 1).all()) and all(bool((o == 1).all()) for o in outs)


@pytest.mark.parametrize("norm_near", [1e-42, 1e-6, 1.0, 3.0, 1e30, 3.4028234e38, 1e40])
def test_one_call_clips_as_two_do(norm_near):
    """ClipGradNorm = GradNorm, then ClipGrads: the same bits, up to norms beyond FP32, where
    both give zeros, as for an infinite one."""
    gen = generator("two calls", norm_near)
    n = 40000
    g = torch.rand(n, generator=gen, dtype=torch.float64) + 0.5
    g = (g * (norm_near / float(g.square().sum().sqrt()))).float().cuda()
    whole = norm_of([g])
    for dtype, ratio, scale in ((torch.float32, 3.0, 1.0), (torch.float32, 1.0000001, 0.7),
                                (torch.bfloat16, 7.0, 0.3)):
        max_norm = min(whole * scale / ratio, 3e38)
        one, two = (torch.full((n,), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        norm, again = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
        ps.ClipGradNorm(ps.GradientList([g], [one]), max_norm, norm, grad_scale=scale)
        glist = ps.GradientList([g], [two])
        ps.GradNorm(glist, again, grad_scale=scale)
        ps.ClipGrads(glist, max_norm, again, grad_scale=scale)
        assert torch.equal(norm, again) and torch.equal(one, two)
        exact = whole * scale
        if exact > torch.finfo(torch.float32).max:
            assert float(norm) == math.inf and bool((one == 0).all())
        else:
            c = min(1.0, max_norm / (float(norm) + 1e-6)) * scale
            e = g.cpu().double() * c
            ref.close(one, e, e.abs() + c * 2.0 ** -149, 3, "clip")


def test_a_list_that_goes_during_a_capture():
    """Its memory is given back without harm to the graph being captured."""
    g = torch.full((5000,), 2.0, device="cuda")
    kept, gone = ps.GradientList([g]), ps.GradientList([torch.ones(100, device="cuda")])
    norm = torch.empty(1, device="cuda")
    ps.GradNorm(kept, norm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ps.GradNorm(kept, norm, stream=torch.cuda.current_stream())
        gone.close()
        norm.add_(1.0)
    for value in (1.0, 3.0, 0.5):
        g.fill_(value)
        norm.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - (value * math.sqrt(5000) + 1)) <= 1e-4 * float(norm)


def test_the_memory_of_lists_goes_back():
    g = torch.empty(1 << 28, dtype=torch.bfloat16, device="cuda")  # lists of half a megabyte
    ps.GradientList([g]).close()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    for _ in range(200):
        ps.GradientList([g]).close()
    assert before - torch.cuda.mem_get_info()[0] < 20 << 20


def test_a_list_that_goes_while_it_works():
    g = torch.full((1 << 27,), 2.0, device="cuda")
    norm = torch.empty(1, device="cuda")
    for _ in range(3):
        glist = ps.GradientList([g])
        for _ in range(20):
            ps.GradNorm(glist, norm)
        glist.close()
        with pytest.raises(ValueError, match="closed"):
            ps.GradNorm(glist, norm)
    assert abs(float(norm) - 2 * 2 ** 13.5) <= 2 * ref.U32 * 2 * 2 ** 13.5
