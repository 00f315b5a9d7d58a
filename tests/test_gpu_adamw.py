"""AdamW over many tensors against 64-bit forms: types, sizes from nothing to several chunks, odd
alignments, moments in 32 and in 8 bits, clipping on the way, rates and steps on the device,
graphs."""
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
SIZES = [1, 0, 3, 4, 5, 255, 256, 257, 1023, 4095, 4096, 4097, 12289, 100003, 7]
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def device():
    setup()


def generator(*key):
    g = torch.Generator()
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


class Place:
    """A view at an odd place of a larger buffer, and whether anything around it changed."""

    def __init__(self, values, dtype, at):
        n = values.numel()
        raw = torch.uint8 if dtype == F8 else dtype
        self.whole = torch.full((n + 16,), 7, dtype=raw, device="cuda")
        self.lo, self.hi = at, at + n
        part = self.whole[at:at + n]
        self.t = part.view(F8) if dtype == F8 else part
        self.t.copy_(values.to(dtype))

    def kept(self):
        return bool((self.whole[:self.lo] == 7).all() and (self.whole[self.hi:] == 7).all())


class Model:
    """Parameters with gradients and moments, on the device and as they are in 64 bits."""

    def __init__(self, gen, sizes, param, grad, copy=None, f8=False, decay=0.1):
        self.f8, self.decay = f8, [decay if n % 2 else 0.0 for n in sizes]
        self.p, self.g, self.m, self.v, self.s, self.c = [], [], [], [], [], []
        for i, n in enumerate(sizes):
            size = torch.exp(2 * torch.randn(n, generator=gen)) * 1e-3
            put = lambda x, dtype: Place(x, dtype, i % 5)  # noqa: E731
            self.p.append(put(0.02 * torch.randn(n, generator=gen), F[param]))
            self.g.append(put(torch.randn(n, generator=gen) * size, F[grad]))
            m = 0.3 * torch.randn(n, generator=gen) * size
            v = (size * torch.rand(n, generator=gen)) ** 2
            if f8:
                m, v = m.double(), v.double().sqrt()
                mc, ms, _, _ = ref.to_8_bits(m, 1, False)
                vc, vs, _, _ = ref.to_8_bits(v, 1, True)
                self.m.append(put((mc * m.sign()).float(), F8))
                self.v.append(put(vc.float(), F8))
                self.s.append(put(torch.stack([ms, vs], 1).float().view(-1)
                                  if n else torch.empty(0), torch.float32))
            else:
                self.m.append(put(m, torch.float32))
                self.v.append(put(v, torch.float32))
            if copy:
                self.c.append(put(torch.zeros(n), F[copy]) if i % 3 else None)

    def list(self):
        t = lambda xs: [x.t if x is not None else None for x in xs]  # noqa: E731
        return ps.AdamWList(t(self.p), t(self.g), t(self.m), t(self.v),
                            scales=t(self.s) if self.f8 else None,
                            copies=t(self.c) if self.c else None, weight_decay=self.decay)

    def exact(self):
        """(p, g, m, v) of every tensor in 64 bits."""
        out = []
        for i in range(len(self.p)):
            p, g, m, v = (x[i].t.cpu().float().double() for x in (self.p, self.g, self.m, self.v))
            if self.f8:
                by = self.s[i].t.cpu().double().view(-1, 2).repeat_interleave(256, 0)[:p.numel()]
                m, v = m * by[:, 0], (v * by[:, 1]) ** 2
            out.append((p, g, m, v))
        return out

    def check(self, before, lr, step, scale=1.0, **more):
        for i, (p, g, m, v) in enumerate(before):
            if not p.numel():
                continue
            new, mm, vv = ref.adamw(p, g, m, v, lr, step, self.decay[i], scale=scale, **more)
            ref.held(self.p[i].t, *new, f"parameter {i}")
            if self.c and self.c[i] is not None:
                ref.held(self.c[i].t, *new, f"copy {i}")
            if not self.f8:
                ref.held(self.m[i].t, *mm, f"exp_avg {i}")
                ref.held(self.v[i].t, *vv, f"exp_avg_sq {i}")
                continue
            root = vv[0].sqrt()
            scales = self.s[i].t.cpu().double().view(-1, 2)
            for k, (x, off, got) in enumerate(((mm[0], mm[1], self.m[i].t),
                                               (root, gamma_root(root), self.v[i].t))):
                code, s, near, steps = ref.to_8_bits(x, step, k == 1)
                top = (off / x.abs().clamp(min=1e-300)).view(-1)
                blocks = s.numel()
                most = torch.zeros(blocks * 256, dtype=torch.float64)
                most[:x.numel()] = off
                # a block's scale is as far off as its largest element may be, and a division
                rel = most.view(-1, 256).amax(1) / 448.0 + 3 * ref.U32 * s
                assert bool(((scales[:, k] - s).abs() <= rel).all()), (i, k)
                got = got.cpu().float().double()
                assert bool(((got < 0) == (x < 0))[got != 0].all())
                # codes by the rule, but where the sum is as near to a whole number as its error
                err = steps * (top + rel.div(s).repeat_interleave(256)[:x.numel()] + 6 * ref.U32)
                err = err + 2.0 ** -19
                wrong = (got.abs() != code) & (near > err)
                assert not wrong.any(), (i, k, torch.nonzero(wrong)[:3].tolist())
                assert float((got.abs() != code).double().mean()) <= 0.01 + 1.0 / x.numel()

        for xs in (self.p, self.g, self.m, self.v, self.s, self.c):
            assert all(x is None or x.kept() for x in xs)


def gamma_root(root):
    return ref.gamma(10) * root


@pytest.mark.parametrize("param", sorted(F))
@pytest.mark.parametrize("grad", sorted(F))
@pytest.mark.parametrize("f8", [False, True])
def test_types(param, grad, f8):
    gen = generator("types", param, grad, f8)
    copy = {"f32": "bf16", "bf16": "f32", "f16": "f16"}[param]
    model = Model(gen, SIZES, param, grad, copy, f8)
    tensors = model.list()
    for step in (1, 2, 3, 1000):
        say(f"adamw {param} {grad} f8={f8} step {step}")
        before = model.exact()
        ps.AdamWStep(tensors, 1e-3, step)
        torch.cuda.synchronize()
        model.check(before, 1e-3, step)


@pytest.mark.parametrize("f8", [False, True])
def test_options(f8):
    gen = generator("options", f8)
    for beta1, beta2, eps, lr, step in ((0.0, 0.9, 1e-3, 0.1, 1), (0.95, 0.0, 1e-6, 1e-2, 7),
                                        (0.99, 0.9999, 0.1, 1e-5, 10 ** 9),
                                        (0.5, 0.5, 1e-8, 0.0, 3)):
        model = Model(gen, SIZES, "f32", "f32", None, f8)
        before = model.exact()
        ps.AdamWStep(model.list(), lr, step, beta1=beta1, beta2=beta2, eps=eps, grad_scale=0.25)
        torch.cuda.synchronize()
        model.check(before, lr, step, 0.25, beta1=beta1, beta2=beta2, eps=eps)


@pytest.mark.parametrize("f8", [False, True])
def test_clipping_on_the_way(f8):
    gen = generator("clip", f8)
    model = Model(gen, SIZES, "f32", "bf16", "bf16", f8)
    grads = ps.GradientList([g.t for g in model.g])
    norm = torch.empty(1, device="cuda")
    tensors = model.list()
    for ratio in (0.5, 4.0):
        ps.GradNorm(grads, norm, grad_scale=0.5)
        n = float(norm)
        before = model.exact()
        ps.AdamWStep(tensors, 1e-3, 5, norm=norm, max_norm=n / ratio, grad_scale=0.5)
        torch.cuda.synchronize()
        model.check(before, 1e-3, 5, 0.5 * min(1.0, (n / ratio) / (n + 1e-6)))
        assert float(norm) == n
    before = model.exact()
    ps.AdamWStep(tensors, 1e-3, 6, norm=norm)  # no bound
    model.check(before, 1e-3, 6)


@pytest.mark.parametrize("f8", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), math.inf])
def test_a_norm_that_is_not_finite_changes_nothing(f8, bad):
    model = Model(generator("skip", f8), SIZES, "f32", "f32", "bf16", f8)
    tensors = model.list()
    model.g[9].t[100] = bad
    norm = torch.empty(1, device="cuda")
    ps.GradNorm(ps.GradientList([g.t for g in model.g]), norm)
    whole = [x.whole.clone() for xs in (model.p, model.m, model.v, model.s) for x in xs]
    ps.AdamWStep(tensors, 1e-3, 1, norm=norm, max_norm=1.0)
    after = [x.whole for xs in (model.p, model.m, model.v, model.s) for x in xs]
    assert all(torch.equal(a, b) for a, b in zip(whole, after))


def test_a_gradient_that_is_not_finite():
    """Without a norm it reaches its own element, in 8 bits its block."""
    for bad in (float("nan"), math.inf):
        for f8 in (False, True):
            model = Model(generator("bad", f8), [5000], "f32", "f32", None, f8)
            model.g[0].t[1000] = bad
            ps.AdamWStep(model.list(), 1e-3, 1)
            ps.AdamWStep(model.list(), 1e-3, 2)
            wrong = torch.nonzero(~torch.isfinite(model.p[0].t)).view(-1).tolist()
            assert 1000 in wrong and all(i // 256 == 1000 // 256 for i in wrong)
            if not f8:
                assert wrong == [1000]
            m = torch.isfinite(model.exact()[0][2])
            assert not m[1000] and bool(m[:768].all()) and bool(m[1024:].all())


def test_rate_and_step_on_the_device():
    gen = generator("device")
    a, b = (Model(generator("same"), SIZES, "f32", "f32", None, True) for _ in range(2))
    lr = torch.tensor(1e-3, device="cuda")
    step = torch.tensor([0], dtype=torch.int32, device="cuda")
    la, lb = a.list(), b.list()
    for t in (1, 2, 3):
        step += 1
        ps.AdamWStep(la, float(lr), t)
        ps.AdamWStep(lb, lr, step)
        for x, y in zip(a.p + a.m + a.v + a.s, b.p + b.m + b.v + b.s):
            assert torch.equal(x.whole, y.whole)
    step.fill_(-5)  # counts as 1
    ps.AdamWStep(la, float(lr), 1)
    ps.AdamWStep(lb, lr, step)
    assert all(torch.equal(x.whole, y.whole) for x, y in zip(a.p, b.p))
    del gen


@pytest.mark.parametrize("f8", [False, True])
def test_in_a_graph_with_the_norm(f8):
    """Norm, rate, step and update captured, replayed on new gradients."""
    a, b = (Model(generator("graph"), SIZES, "f32", "bf16", "bf16", f8) for _ in range(2))
    lr = torch.tensor([1e-2], device="cuda")
    work = []
    for model in (a, b):
        work.append((model.list(), ps.GradientList([g.t for g in model.g]),
                     torch.empty(1, device="cuda"),
                     torch.zeros(1, dtype=torch.int32, device="cuda")))

    def run(model):
        tensors, grads, norm, step = work[0 if model is a else 1]
        s = torch.cuda.current_stream()
        step += 1
        ps.GradNorm(grads, norm, stream=s)
        ps.AdamWStep(tensors, lr, step, norm=norm, max_norm=0.01, stream=s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(a)
    run(b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(a)
    gen = generator("new")
    for k in range(4):
        lr.fill_(1e-2 / (k + 1))
        for x, y in zip(a.g, b.g):
            x.t.copy_(torch.randn(x.t.shape, generator=gen) * 1e-3)
            y.t.copy_(x.t)
        graph.replay()
        run(b)
        torch.cuda.synchronize()
        for x, y in zip(a.p + a.m + a.v + a.s, b.p + b.m + b.v + b.s):
            assert torch.equal(x.whole, y.whole)


def test_zeros_stay_zeros_and_nothing_becomes_zero():
    """Fresh states and no gradient: nothing moves. A second moment far below its block's largest
    stays above zero, and the step by it stays bounded."""
    n = 1000
    p, g = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda")
    m, v = (torch.zeros(n, device="cuda").to(F8) for _ in range(2))
    s = torch.zeros((ps.state_blocks(n), 2), device="cuda")
    tensors = ps.AdamWList([p], [g], [m], [v], scales=[s], weight_decay=0.0)
    ps.AdamWStep(tensors, 1e-3, 1)
    assert bool((p == 1).all()) and not m.float().any() and not v.float().any()
    g.fill_(1e-9)
    g[::256] = 1.0
    for t in range(1, 4):
        ps.AdamWStep(tensors, 1e-3, t)
    assert bool((v.float() > 0).all())
    assert float((p - 1).abs().max()) <= 3 * 1.1e-3  # m / sqrt(v) is 1 at most for equal gradients


@pytest.mark.parametrize("f8", [False, True])
def test_second_moments_below_the_normal_numbers(f8):
    """Gradients of 1e-18 and no eps: the first step goes by one. (1 - beta2) g^2 is 1e-39, where
    FP32 numbers are 2^-149 apart, 1.4e-6 of it: the root is off by 0.7e-6, and some forty FP32
    roundings come to 2.4e-6."""
    n = 1000
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 1e-18, device="cuda")
    g[::2] *= -1
    if f8:
        m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
        scales = [torch.zeros((ps.state_blocks(n), 2), device="cuda")]
    else:
        m, v, scales = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), None
    ps.AdamWStep(ps.AdamWList([p], [g], [m], [v], scales=scales), 1.0, 1, eps=0.0)
    assert float((p + g.sign()).abs().max()) <= 4e-6


def test_moments_in_8_bits_follow_the_gradients():
    """A second moment that gains a part in 1000 a step gains it in its codes too, which rounding to
    nearest would leave at 4.5. 2000 steps of gradients twice as large take the exact root from 1 to
    1.896; the codes around it stand for 1.786 and 2.009, 0.2232 apart. The rule in 64 bits gives
    every element one of these two, the mean being 1.979: within a step of the grid, and within half
    of one."""
    n = 4096
    p = torch.zeros(n, device="cuda")
    g = torch.full((n,), 2.0, device="cuda")
    m, v = torch.zeros(n, device="cuda").to(F8), torch.ones(n, device="cuda").to(F8)
    s = torch.ones((ps.state_blocks(n), 2), device="cuda")
    big = torch.arange(n, device="cuda") % 256 == 0
    g[big] = 100.0  # keeps every block's scale where it is
    s[:, 1] = 100.0 / 448.0
    v.copy_(torch.where(big, 448.0, 4.5))  # 4.5 * 100 / 448 is 1.0045
    tensors = ps.AdamWList([p], [g], [m], [v], scales=[s], weight_decay=0.0)
    for t in range(1, 2001):
        ps.AdamWStep(tensors, 0.0, t)
    root = (v.float().view(-1, 256) * s[:, 1:]).view(-1)[~big]
    exact = math.sqrt(4.0 - (4.0 - 1.0045 ** 2) * 0.999 ** 2000)
    assert bool(((root - exact).abs() <= 0.2233).all()), (float(root.min()), float(root.max()))
    assert abs(float(root.mean()) - exact) <= 0.1117


def test_nothing_to_do():
    for tensors in (ps.AdamWList([], [], [], []),
                    ps.AdamWList(*([torch.empty(0, device="cuda")] for _ in range(4)))):
        ps.AdamWStep(tensors, 1e-3, 1)
        tensors.close()
        tensors.close()
        with pytest.raises(ValueError, match="closed"):
            ps.AdamWStep(tensors, 1e-3, 1)


def test_large():
    """A tensor beyond 2^32 elements: places and thresholds behind it."""
    n = (1 << 32) + 300
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda") for _ in range(2))
    s = torch.zeros((ps.state_blocks(n), 2), device="cuda")
    ps.AdamWStep(ps.AdamWList([p], [g], [m], [v], scales=[s], weight_decay=0.0), 0.5, 1)
    assert bool((p == -0.5).all())
    # All are their blocks' largest: 448 (code 0x7E). The scale is their FP32 product with FP32's
    # 1 / 448, so their quotient is 448 (1 - 3 * 2^-24) at least, 14 (1 - 3 * 2^-24) steps of the
    # grid: where u is below 14 * 3 * 2^-24 < 3 * 2^-20 the code below, 416, is right too.
    for codes in (m, v):
        for k, part in enumerate(codes.split(1 << 30)):
            i = torch.nonzero(part != 0x7E).view(-1) + (k << 30)
            assert bool((codes[i] == 0x7D).all())
            u = (((i * 0x6A09E667) + 0x9E3779B9) & 0xFFFFFFFF) >> 12
            assert bool((u < 3).all())
    assert float((s[-2:, 0] / (0.1 / 448) - 1).abs().max()) <= 8 * ref.U32


def test_values_that_lie_in_what_is_written_are_refused():
    a = torch.zeros(4 * 1000, device="cuda")
    i = torch.zeros(1000, dtype=torch.int32, device="cuda")
    p, m, v, g = a.split(1000)
    tensors = ps.AdamWList([p], [g], [m], [v])
    for at in (p[:1], m[999:], v[5:6]):
        with pytest.raises(ValueError, match="lies in"):
            ps.AdamWStep(tensors, at, 1)
        with pytest.raises(ValueError, match="lies in"):
            ps.AdamWStep(tensors, 1e-3, 1, norm=at, max_norm=1.0)
    with pytest.raises(ValueError, match="lies in"):
        ps.AdamWStep(tensors, 1e-3, p[:1].view(torch.int32))
    ps.AdamWStep(tensors, g[:1], 1)  # a gradient is only read
    del i


def test_a_list_may_go_at_any_time():
    model = Model(generator("gone"), SIZES, "f32", "f32")
    tensors = model.list()
    before = model.exact()
    ps.AdamWStep(tensors, 1e-3, 1)
    tensors.close()
    another = model.list()  # its memory goes back here, when the step has run
    torch.cuda.synchronize()
    model.check(before, 1e-3, 1)
    another.close()


def test_steps_that_are_refused():
    """Numbers on the host that FP32 does not hold, and other options out of range."""
    p, g, m, v = (torch.ones(100, device="cuda") for _ in range(4))
    tensors = ps.AdamWList([p], [g], [m], [v])

    def refused(text, lr=1e-3, step=1, **more):
        with pytest.raises(ValueError, match=text):
            ps.AdamWStep(tensors, lr, step, **more)

    for rate in (math.nan, math.inf, 1e39, -1e39, 1e300):
        refused("the rate is not a number", lr=rate)
    for eps in (math.nan, -1e-8, math.inf, 1e39):
        refused("eps is not a number", eps=eps)
    for beta in (math.nan, -0.1, 1.0):
        refused("betas", beta1=beta)
        refused("betas", beta2=beta)
    for step in (0, -1):
        refused("counted from 1", step=step)
    norm = torch.ones(1, device="cuda")
    for bound in (math.nan, -1.0):
        refused("the bound is not a number", norm=norm, max_norm=bound)
    refused("max_norm needs the norm", max_norm=1.0)
    assert all(bool((x == 1).all()) for x in (p, g, m, v))
    largest = torch.finfo(torch.float32).max
    ps.AdamWStep(tensors, 0.0, 1, eps=largest)
    assert bool((p == 1).all())
    ps.AdamWStep(tensors, largest, 1, eps=largest)
    assert bool(torch.isfinite(p).all())


def test_moments_in_8_bits_under_random_gradients():
    """2000 steps of N(0, 1) gradients from a root of 1, beside the exact course and the rule in 64
    bits. A step moves a root r by d = 0.0005 (g^2 - r^2) / r, 0.00048 r on average, and a code goes
    up with the probability d / q, q its step of the grid, r / 8 at most: the variance of a rounding
    is at most q |d| = 6.1e-5 r^2. What it leaves decays by 0.999 a step: 500 of them are in the
    root, 0.030, whose root is 0.174. They add up in the square, 1000 of them, 0.061, and so the
    root's mean may rise by 0.03. Means of 16,384 elements that walk by themselves are off by
    0.174 / 128 and their spread by 1 / 181."""
    n, beta1, beta2 = 16384, 0.9, 0.999
    gen = generator("walk")
    p, g = torch.zeros(n, device="cuda"), torch.empty(n, device="cuda")
    code, scale, _, _ = ref.to_8_bits(torch.ones(n, dtype=torch.float64), 1, True)
    m, v = torch.zeros(n, device="cuda").to(F8), code.float().cuda().to(F8)
    s = torch.stack([torch.zeros_like(scale), scale], 1).float().cuda()
    tensors = ps.AdamWList([p], [g], [m], [v], scales=[s], weight_decay=0.0)
    exact = torch.ones(n, dtype=torch.float64)
    rule = exact.clone()
    for t in range(1, 2001):
        fresh = torch.randn(n, generator=gen)
        g.copy_(fresh)
        ps.AdamWStep(tensors, 0.0, t, beta1=beta1, beta2=beta2)
        square = fresh.double().square_()
        exact = beta2 * exact + (1 - beta2) * square
        new = (beta2 * rule * rule + (1 - beta2) * square).sqrt()
        code, scale, _, _ = ref.to_8_bits(new, t, True)
        rule = code * scale.repeat_interleave(256)
    got = (v.float().view(-1, 256) * s[:, 1:]).view(-1).cpu().double()
    means, spreads = [], []
    for root in (got, rule):
        off = root / exact.sqrt() - 1
        means.append(float(off.mean()))
        spreads.append(float(off.square().mean().sqrt()))
        assert abs(means[-1]) <= 0.03 and spreads[-1] <= 0.18
        assert -0.01 <= float((root * root / exact).mean()) - 1 <= 0.065
    assert abs(means[0] - means[1]) <= 6 * 0.174 / 128 * math.sqrt(2)
    assert abs(spreads[0] / spreads[1] - 1) <= 6 / 181 * math.sqrt(2)


@pytest.mark.parametrize("f8", [False, True])
def test_skipped_updates_in_a_graph(f8):
    """A step on the device that goes up by whether the norm is finite, captured with the norm and
    the update: replays whose gradients overflow change nothing and are not counted, and those after
    them are the first, second and third updates."""
    a, b = (Model(generator("skipped"), SIZES, "f32", "f16", "bf16", f8) for _ in range(2))
    la, lb = a.list(), b.list()
    grads = ps.GradientList([g.t for g in a.g])
    norm, step = torch.empty(1, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")

    def run():
        s = torch.cuda.current_stream()
        ps.GradNorm(grads, norm, stream=s)
        step.add_(torch.isfinite(norm))
        ps.AdamWStep(la, 1e-2, step, norm=norm, max_norm=0.01, stream=s)

    model_state = [x.whole.clone() for x in a.p + a.m + a.v + a.s]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for x, was in zip(a.p + a.m + a.v + a.s, model_state):
        x.whole.copy_(was)
    step.zero_()
    gen = generator("skipped gradients")
    done = 0
    for bad in (True, True, False, True, False, False):
        for k, (x, y) in enumerate(zip(a.g, b.g)):
            x.t.copy_(torch.randn(x.t.shape, generator=gen) * 1e-2)
            if bad and k == 13:
                x.t[50000] = math.inf
            y.t.copy_(x.t)
        graph.replay()
        torch.cuda.synchronize()
        if not bad:
            done += 1
            ps.AdamWStep(lb, 1e-2, done, norm=norm, max_norm=0.01)
        torch.cuda.synchronize()
        assert int(step) == done and bool(torch.isfinite(norm)) != bad
        for x, y in zip(a.p + a.m + a.v + a.s, b.p + b.m + b.v + b.s):
            assert torch.equal(x.whole, y.whole)
        for x, y in zip(a.c, b.c):
            assert x is None or done == 0 or torch.equal(x.whole, y.whole)
