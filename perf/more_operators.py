"""More operators this framework's performance is followed on, the rest of a training step next
to those of operators.py: layer norm and its gradients, the router of a mixture of experts
(softmax, top-k, balance loss) and its gradient, and the AdamW step over many tensors with states
in 32 or 8 bits.

A case is one pass through one operator as a user's program calls it. Widths and row counts are
those of the framework's graphs (32 to 512 features, a million nodes) and the generic powers of
two of transformer layers, with odd and ragged ones between them. Rows have means and scales of
their own, as activations do; logits prefer some experts; gradients and second moments spread over
some orders of magnitude.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
F8 = torch.float8_e4m3fn
BLOCK = 256  # elements of an 8-bit state that share a scale
BETA1, BETA2, ADAM_EPS, NORM_EPS = 0.9, 0.999, 1e-8, 1e-5

# ------------------------------------------------------------------ cases


def _norm(name, op, rows, cols, x, y, weight, pad=0):
    return dict(name=name, op=op, rows=rows, cols=cols, x=x, y=y, weight=weight, pad=pad)


def _route(name, op, tokens, top_k, experts, dtype, normalize, masked, barred):
    return dict(name=name, op=op, tokens=tokens, top_k=top_k, experts=experts, dtype=dtype,
                normalize=normalize, masked=masked, barred=barred)


def _adamw(name, tensors, total, param, grad, copy, state, ratio, grad_scale):
    return dict(name=name, op="adamw", tensors=tensors, total=total, param=param, grad=grad,
                copy=copy, state=state, ratio=ratio, grad_scale=grad_scale, lr=1e-4, step=1000)


def listed():
    return [
        # One decoding step of a few sequences: latency only.
        _norm("norm_step", "norm", 8, 2048, "bf16", "bf16", "bf16"),
        # A million nodes' features between two layers of a graph model.
        _norm("norm_nodes", "norm", 1000000, 128, "f32", "f32", "f32"),
        # A training batch of a wide layer, the largest.
        _norm("norm_batch", "norm", 32768, 4096, "bf16", "bf16", "f32"),
        # The gradients of a small batch of nodes, odd sizes, columns of a wider buffer.
        _norm("norm_grad_odd", "norm_grad", 30011, 333, "f32", "f32", "f32", pad=3),
        # The gradients of that training batch, an FP32 residual stream and BF16 branches.
        _norm("norm_grad_batch", "norm_grad", 16384, 4096, "f32", "bf16", "f32"),
        # Routing of one decoding step.
        _route("route_step", "route", 8, 8, 64, "bf16", True, 0.0, 0.0),
        # Routing of a padded training batch.
        _route("route_batch", "route", 65536, 8, 128, "f32", True, 0.1, 0.0),
        # Its gradient.
        _route("route_grad_batch", "route_grad", 65536, 8, 128, "f32", True, 0.1, 0.0),
        # Nodes routed by relation, few experts, some barred for a node: odd sizes.
        _route("route_grad_odd", "route_grad", 300007, 3, 17, "f16", False, 0.0, 0.2),
        # A small graph model's step: plain FP32.
        _adamw("adamw_small", 37, 1100003, "f32", "f32", "", "f32", 0.5, 1.0),
        # Mixed precision: BF16 gradients clipped on the way, FP32 weights and their BF16 copy.
        _adamw("adamw_mixed", 291, 400000077, "f32", "bf16", "bf16", "f32", 4.0, 0.125),
        # The same with both moments in 8 bits.
        _adamw("adamw_8bit", 291, 400000077, "f32", "bf16", "bf16", "f8", 4.0, 0.125),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "route", "route_grad", "adamw"])
    kinds = sorted(DTYPES)
    if op in ("norm", "norm_grad"):
        rows = _log_between(rng, 1, 1000000)
        cols = _log_between(rng, 32, max(33, min(16384, 2 ** 26 // rows)))
        if rng.random() < 0.6:
            cols = max(32, cols // 32 * 32)
        return dict(op=op, rows=rows, cols=cols, x=rng.choice(kinds), y=rng.choice(kinds),
                    weight=rng.choice(kinds), pad=rng.choice([0, 0, 0, 64, 3]))
    if op == "adamw":
        total, param = _log_between(rng, 1000, 200000000), rng.choice(["f32", "f32", "bf16"])
        return dict(op=op, tensors=min(_log_between(rng, 1, 400), total), total=total, param=param,
                    grad=rng.choice(kinds), state=rng.choice(["f32", "f8"]),
                    copy=rng.choice(["", "bf16", "f16"]) if param == "f32" else "",
                    ratio=round(math.exp(rng.uniform(-1.5, 2.0)), 3),
                    grad_scale=rng.choice([1.0, 1.0 / 1024, 0.3]), lr=rng.choice([1e-4, 2e-5]),
                    step=_log_between(rng, 1, 100000))
    experts = _log_between(rng, 2, 512)
    return dict(op=op, tokens=_log_between(rng, 1, min(300000, 2 ** 23 // experts)),
                top_k=rng.randint(1, min(8, experts)), experts=experts, dtype=rng.choice(kinds),
                normalize=rng.random() < 0.5,
                masked=round(rng.choice([0.0, rng.uniform(0.0, 0.5)]), 3),
                barred=round(rng.choice([0.0, 0.0, rng.uniform(0.0, 0.9)]), 3))


# ----------------------------------------------------------------- inputs


def _normal(shape, gen, dtype="f32", std=1.0):
    """Normal values, rounded to `dtype`, made a part at a time."""
    out = torch.empty(shape, dtype=DTYPES[dtype], device="cuda")
    for part in out.view(-1).split(1 << 28):
        part.copy_(torch.randn(part.numel(), generator=gen, device="cuda").mul_(std))
    return out


def _activations(case, dtype, gen):
    """Rows with means and scales of their own; columns of a wider buffer with `pad`."""
    rows, cols = case["rows"], case["cols"]
    x = _normal((rows, cols + case["pad"]), gen)
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))
    x += 0.5 * torch.randn((rows, 1), generator=gen, device="cuda")
    return x.to(DTYPES[dtype])[:, :cols]


def _sizes(case):
    """The tensors' element counts: some matrices, many vectors; they add up to `total`."""
    rng = random.Random(case["tensors"] * 7919 + case["total"])
    w = [math.exp(rng.uniform(0.0, 6.0)) for _ in range(case["tensors"])]
    rest = case["total"] - case["tensors"]
    sizes = [1 + int(rest * x / sum(w)) for x in w]
    sizes[-1] += case["total"] - sum(sizes)
    return sizes


def _places(case):
    """Where the tensors lie in one buffer, as an allocator places them: each begins at a multiple
    of BLOCK elements. [(begin, elements)] and the buffer's elements."""
    places, at = [], 0
    for n in _sizes(case):
        places.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return places, at


def _to_blocks(x, positive, u):
    """Codes and scales of the 8-bit form: blocks of 256, the largest of each at 448. Between two
    codes the upper one is taken where the fraction of the step is 1 - u or more. What is above
    zero and `positive` stays there, at the least code or above."""
    blocks = x.view(-1, BLOCK)
    scale = (blocks.abs().amax(1, keepdim=True) / 448.0).clamp(min=2.0 ** -126)
    ratio = blocks.abs() / scale
    # E4M3 has 8 codes between two powers of two, from 2^-6 up, and as many below.
    step = torch.ldexp(torch.ones_like(ratio), torch.frexp(ratio).exponent.clamp(min=-5) - 4)
    ratio = (torch.floor(ratio / step + u) * step).clamp(max=448.0)
    if positive:
        ratio = torch.where(blocks > 0, ratio.clamp(min=2.0 ** -9), ratio)
    return torch.where(blocks < 0, -ratio, ratio).to(F8).view(-1), scale.view(-1)


def _thresholds(first, t):
    """u of _to_blocks for blocks that begin at the elements `first` of their tensors, in step t:
    two Weyl sequences, so that an element's u takes every value alike over the steps."""
    i = first[:, None] + torch.arange(BLOCK, device=first.device)
    u = (i * 0x6A09E667 + t * 0x9E3779B9) & 0xFFFFFFFF
    return (u >> 12).float() * 2.0 ** -20


def _adamw_state(case, gen):
    places, n = _places(case)
    inside = torch.zeros(n, dtype=torch.bool, device="cuda")
    for at, size in places:
        inside[at:at + size] = True
    # Gradients as the second moments have seen them: of scales over three orders of magnitude.
    spread = torch.exp(torch.randn(n, generator=gen, device="cuda"))
    spread *= inside / (case["grad_scale"] * math.sqrt(case["total"]))
    if case["grad"] == "f16":
        spread *= max(1.0, 1e-4 / (float(spread.sum()) / case["total"]))
    grad = _normal((n,), gen).mul_(spread).to(DTYPES[case["grad"]])
    norm = math.sqrt(sum(float(p.double().square().sum()) for p in grad.split(1 << 27)))
    norm *= case["grad_scale"]
    c = case["grad_scale"] * min(1.0, 1.0 / case["ratio"])
    m = _normal((n,), gen).mul_(spread).mul_(0.3 * c)
    r = _normal((n,), gen).mul_(0.2).add_(1.0).abs_().mul_(spread).mul_(c)
    p = _normal((n,), gen, std=0.02).mul_(inside).to(DTYPES[case["param"]])
    s = dict(case=case, places=places, p=p, grad=grad,
             norm=torch.full((1,), norm, device="cuda"), max_norm=norm / case["ratio"],
             decay=[0.0 if size < 4096 else 0.1 for _, size in places])
    # The same for each block of the buffer, and where in its tensor it begins.
    blocks = torch.tensor([-(-size // BLOCK) for _, size in places], device="cuda")
    s["block_decay"] = torch.tensor(s["decay"], device="cuda").repeat_interleave(blocks)
    begin = torch.tensor([at for at, _ in places], device="cuda").repeat_interleave(blocks)
    s["block_first"] = torch.arange(0, n, BLOCK, device="cuda") - begin
    if case["state"] == "f8":
        (m, ms), (r, rs) = _to_blocks(m, False, 0.5), _to_blocks(r, True, 0.5)
        s.update(m=m, v=r, scales=torch.stack([ms, rs], 1).contiguous())
    else:
        s.update(m=m, v=r.square_())
    if case["copy"]:
        s["copy"] = p.to(DTYPES[case["copy"]])
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed) * 1000003 + 29)
    op = case["op"]
    if op in ("norm", "norm_grad"):
        rows, cols = case["rows"], case["cols"]
        w = DTYPES[case["weight"]]
        s = dict(case=case, x=_activations(case, case["x"], gen),
                 weight=(1.0 + 0.2 * torch.randn(cols, generator=gen, device="cuda")).to(w),
                 mean=torch.empty(rows, device="cuda"), rstd=torch.empty(rows, device="cuda"))
        if op == "norm":
            s.update(bias=(0.1 * torch.randn(cols, generator=gen, device="cuda")).to(w),
                     y=torch.empty((rows, cols), dtype=DTYPES[case["y"]], device="cuda"))
            return s
        for at in range(0, rows, 1 << 16):  # the forward pass has left them
            part = s["x"][at:at + (1 << 16)].double()
            var, mean = torch.var_mean(part, 1, correction=0)
            s["mean"][at:at + (1 << 16)] = mean
            s["rstd"][at:at + (1 << 16)] = (var + NORM_EPS).rsqrt()
        s.update(dy=_normal((rows, cols + case["pad"]), gen, case["y"], 0.1)[:, :cols],
                 dx=torch.empty((rows, cols), dtype=DTYPES[case["x"]], device="cuda"),
                 dweight=torch.empty(cols, dtype=w, device="cuda"),
                 dbias=torch.empty(cols, dtype=w, device="cuda"))
        return s
    if op == "adamw":
        return _adamw_state(case, gen)
    T, K, E = case["tokens"], case["top_k"], case["experts"]
    prefer = -0.5 * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    logits = _normal((T, E), gen) + prefer[torch.randperm(E, generator=gen, device="cuda")]
    if case["barred"]:
        logits[torch.rand((T, E), generator=gen, device="cuda") < case["barred"]] = -math.inf
    s = dict(case=case, logits=logits.to(DTYPES[case["dtype"]]), mask=None,
             ids=torch.empty((T, K), dtype=torch.int32, device="cuda"),
             counts=torch.empty(E + 1, dtype=torch.int32, device="cuda"))
    if case["masked"]:
        s["mask"] = torch.rand(T, generator=gen, device="cuda") >= case["masked"]
    if op == "route":
        s.update(weights=torch.empty((T, K), device="cuda"), loss=torch.empty(1, device="cuda"))
        return s
    chosen = _plain_route(s)  # the forward pass has made them
    s.update(ids=chosen["ids"], counts=chosen["counts"],
             dweights=torch.randn((T, K), generator=gen, device="cuda"),
             dloss=torch.full((1,), 0.01 * T, device="cuda"),
             dlogits=torch.empty_like(s["logits"]))
    return s


# ------------------------------------------------------------- plain forms


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    x = x - mean
    rstd = 1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + NORM_EPS)
    y = x * rstd * s["weight"].float() + s["bias"].float()
    return dict(y=y.to(s["y"].dtype), mean=mean.view(-1), rstd=rstd.view(-1))


def _plain_norm_grad(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    xh = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy * s["weight"].float()
    dx = (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)) * rstd
    return dict(dx=dx.to(s["dx"].dtype), dweight=(dy * xh).sum(0).to(s["dweight"].dtype),
                dbias=dy.sum(0).to(s["dbias"].dtype))


def _probabilities(logits, mask):
    """Softmax of every row; zeros in rows that are masked or all -inf."""
    l = logits.float()
    if mask is not None:
        l = torch.where(mask[:, None], l, -math.inf)
    top = l.amax(1, keepdim=True)
    p = torch.exp(l - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(1, keepdim=True)
    return l, p / torch.where(total == 0, 1.0, total)


def _plain_route(s):
    case = s["case"]
    K, E = case["top_k"], case["experts"]
    l, p = _probabilities(s["logits"], s["mask"])
    values, ids = torch.sort(l, dim=1, descending=True, stable=True)
    values, ids = values[:, :K], ids[:, :K]
    taken = values > -math.inf
    weights = torch.where(taken, p.gather(1, ids), 0.0)
    if case["normalize"]:
        w = torch.where(taken, torch.exp(values - torch.where(taken, values, 0.0)[:, :1]), 0.0)
        total = w.sum(1, keepdim=True)
        weights = w / torch.where(total == 0, 1.0, total)
    ids = torch.where(taken, ids, -1)
    counts = torch.zeros(E + 2, dtype=torch.int64, device="cuda")
    counts.index_add_(0, (ids + 1).view(-1), torch.ones_like(ids).view(-1))
    chosen, tokens = counts[1:E + 1], taken[:, 0].sum()
    scale = E / (tokens * chosen.sum()).double().clamp(min=1.0)
    loss = (p.sum(0, dtype=torch.float64) * chosen).sum() * scale
    return dict(ids=ids.to(torch.int32), weights=weights, loss=loss.float().view(1),
                counts=torch.cat([chosen, tokens.view(1)]).to(torch.int32))


def _plain_route_grad(s):
    case = s["case"]
    E = case["experts"]
    taken, ids = s["ids"] >= 0, s["ids"].clamp(min=0).long()
    l, p = _probabilities(s["logits"], taken[:, 0])
    counts = s["counts"].double()
    scale = E / (counts[E] * counts[:E].sum()).clamp(min=1.0) * s["dloss"]
    h = (counts[:E] * scale).float().expand_as(p).contiguous()
    dw = torch.where(taken, s["dweights"], 0.0)
    if not case["normalize"]:
        h.scatter_add_(1, ids, dw)
    grad = p * (h - (p * h).sum(1, keepdim=True))
    if case["normalize"]:
        chosen = l.gather(1, ids)
        w = torch.where(taken, torch.exp(chosen - torch.where(taken, chosen, 0.0)[:, :1]), 0.0)
        w = w / w.sum(1, keepdim=True).clamp(min=1.0)
        grad.scatter_add_(1, ids, w * (dw - (w * dw).sum(1, keepdim=True)))
    return grad.to(s["dlogits"].dtype)


def _plain_adamw(s):
    case = s["case"]
    c = case["grad_scale"] * (s["max_norm"] / (s["norm"] + 1e-6)).clamp(max=1.0)
    g = s["grad"].float() * c
    if case["state"] == "f8":
        scales = s["scales"]
        m = (s["m"].float().view(-1, BLOCK) * scales[:, :1]).view(-1)
        v = (s["v"].float().view(-1, BLOCK) * scales[:, 1:]).view(-1).square()
    else:
        m, v = s["m"], s["v"]
    m = BETA1 * m + (1.0 - BETA1) * g
    v = BETA2 * v + (1.0 - BETA2) * g * g
    t = case["step"]
    p = s["p"].float()
    up = (m / (1.0 - BETA1 ** t)) / (torch.sqrt(v / (1.0 - BETA2 ** t)) + ADAM_EPS)
    up.view(-1, BLOCK).add_(p.view(-1, BLOCK) * s["block_decay"][:, None])
    s["p"].copy_(p - case["lr"] * up)
    if case["state"] == "f8":
        u = _thresholds(s["block_first"], t)
        (mc, ms), (rc, rs) = _to_blocks(m, False, u), _to_blocks(v.sqrt(), True, u)
        s["m"].copy_(mc)
        s["v"].copy_(rc)
        s["scales"].copy_(torch.stack([ms, rs], 1))
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    if case["copy"]:
        s["copy"].copy_(p - case["lr"] * up)
    return {k: s[k] for k in ("p", "m", "v", "scales", "copy") if k in s}


# ---------------------------------------------------- the framework's calls


def _workspace(state, nbytes):
    if "workspace" not in state:
        state["workspace"] = torch.empty(max(nbytes, 1), dtype=torch.uint8, device="cuda")
    return state["workspace"]


def _adamw_list(s, ps):
    """The step's list of tensors, kept as long as they stay where they are."""
    def parts(flat):
        return [flat[at:at + n] for at, n in s["places"]]

    scales = None
    if s["case"]["state"] == "f8":
        scales = [s["scales"][at // BLOCK:(at + n + BLOCK - 1) // BLOCK] for at, n in s["places"]]
    return ps.AdamWList(parts(s["p"]), parts(s["grad"]), parts(s["m"]), parts(s["v"]),
                        scales=scales, copies=parts(s["copy"]) if s["case"]["copy"] else None,
                        weight_decay=s["decay"])


def _own(s):
    import powersparse_amd as ps
    case, op = s["case"], s["case"]["op"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "norm":
        ps.LayerNorm(s["x"], s["weight"], s["bias"], s["y"], s["mean"], s["rstd"], eps=NORM_EPS,
                     stream=stream)
        return {k: s[k] for k in ("y", "mean", "rstd")}
    if op == "norm_grad":
        work = _workspace(s, ps.layer_norm_grad_workspace_bytes(case["rows"], case["cols"]))
        ps.LayerNormGrad(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"], s["dx"],
                         s["dweight"], s["dbias"], work, stream=stream)
        return {k: s[k] for k in ("dx", "dweight", "dbias")}
    if op == "route":
        work = _workspace(s, ps.expert_route_workspace_bytes(case["tokens"], case["experts"]))
        ps.ExpertRoute(s["logits"], s["ids"], s["weights"], s["counts"], s["loss"], work,
                       mask=s["mask"], normalize=case["normalize"], stream=stream)
        return {k: s[k] for k in ("ids", "weights", "counts", "loss")}
    if op == "route_grad":
        ps.ExpertRouteGrad(s["logits"], s["ids"], s["dweights"], s["counts"], s["dloss"],
                           s["dlogits"], normalize=case["normalize"], stream=stream)
        return s["dlogits"]
    if "list" not in s:
        s["list"] = _adamw_list(s, ps)
    ps.AdamWStep(s["list"], case["lr"], case["step"], beta1=BETA1, beta2=BETA2, eps=ADAM_EPS,
                 norm=s["norm"], max_norm=s["max_norm"], grad_scale=case["grad_scale"],
                 stream=stream)
    return {k: s[k] for k in ("p", "m", "v", "scales", "copy") if k in s}


def run(state):
    if own:
        return _own(state)
    plain = dict(norm=_plain_norm, norm_grad=_plain_norm_grad, route=_plain_route,
                 route_grad=_plain_route_grad, adamw=_plain_adamw)
    return plain[state["case"]["op"]](state)


# ------------------------------------------------------------------- work


def _size(dtype):
    return DTYPES[dtype].itemsize


def work(case):
    op = case["op"]
    if op in ("norm", "norm_grad"):
        rows, cols, w = case["rows"], case["cols"], _size(case["weight"])
        cells = rows * cols
        if op == "norm":
            return dict(bytes=cells * (_size(case["x"]) + _size(case["y"])) + 8 * rows +
                        2 * cols * w, flops=8 * cells)
        return dict(bytes=cells * (2 * _size(case["x"]) + _size(case["y"])) + 8 * rows +
                    3 * cols * w, flops=14 * cells)
    if op == "adamw":
        n = case["total"]
        states = 16 * n if case["state"] == "f32" else 4 * n + 16 * -(-n // BLOCK)
        copy = _size(case["copy"]) if case["copy"] else 0
        return dict(bytes=n * (2 * _size(case["param"]) + _size(case["grad"]) + copy) + states,
                    flops=14 * n)
    T, K, E = case["tokens"], case["top_k"], case["experts"]
    logits = T * E * _size(case["dtype"])
    if op == "route":
        return dict(bytes=logits + 8 * T * K + (T if case["masked"] else 0) + 4 * (E + 2),
                    flops=5 * T * E)
    return dict(bytes=2 * logits + 8 * T * K + 4 * (E + 2), flops=8 * T * E)


# ------------------------------------------------------------------ exact


def _exact_route(s, logits):
    """(weights, balance loss) in 64 bits with torch's own softmax, for autograd."""
    case = s["case"]
    E = case["experts"]
    on = torch.isfinite(logits).any(1)
    if s["mask"] is not None:
        on = on & s["mask"]
    part = logits[on]
    p = torch.softmax(part, 1)
    # torch's sort of -logits, stable, puts the lowest index first among equals
    order = (-part.detach()).argsort(dim=1, stable=True)[:, :case["top_k"]]
    barred = part.detach().gather(1, order) == -math.inf
    chosen = part.gather(1, order).masked_fill(barred, -math.inf)
    w = torch.softmax(chosen, 1) if case["normalize"] else p.gather(1, order)
    w = w.masked_fill(barred, 0.0)
    weights = torch.zeros((on.numel(), case["top_k"]), dtype=torch.float64, device="cuda")
    weights = weights.index_put((on.nonzero().view(-1),), w)
    freq = torch.bincount(order[~barred], minlength=E).double()
    loss = E * (freq / freq.sum().clamp(min=1.0) * p.sum(0) / max(int(on.sum()), 1)).sum()
    return weights, loss.view(1)


def _exact_adamw(s):
    case = s["case"]
    scale = case["grad_scale"] * min(1.0, s["max_norm"] / (float(s["norm"]) + 1e-6))
    g = s["grad"].double() * scale
    m, r = s["m"].double(), s["v"].double()
    if case["state"] == "f8":
        by_block = s["scales"].double().repeat_interleave(BLOCK, 0)
        m, r = m * by_block[:, 0], r * by_block[:, 1]
    else:
        r = r.sqrt()
    m = torch.lerp(g, m, BETA1)
    r = torch.hypot(math.sqrt(BETA2) * r, math.sqrt(1.0 - BETA2) * g)
    t, p = case["step"], s["p"].double()
    decay = s["block_decay"].double().repeat_interleave(BLOCK)
    denom = r / math.sqrt(-math.expm1(t * math.log(BETA2))) + ADAM_EPS
    p = p * (1.0 - case["lr"] * decay) - (case["lr"] / -math.expm1(t * math.log(BETA1))) * m / denom
    out = dict(p=p, m=m, v=r * r)
    if case["state"] == "f8":
        # What the codes stand for before their rounding, and the scales.
        top = torch.stack([m.abs().view(-1, BLOCK).amax(1), r.view(-1, BLOCK).amax(1)], 1) / 448.0
        top = top.clamp(min=2.0 ** -126)
        by_block = top.repeat_interleave(BLOCK, 0)
        out.update(m=m / by_block[:, 0], v=r / by_block[:, 1], scales=top)
    if case["copy"]:
        out["copy"] = p
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "adamw":
        return _exact_adamw(s)
    if op in ("norm", "norm_grad"):
        x = s["x"].double().requires_grad_(op == "norm_grad")
        w = s["weight"].double().requires_grad_(op == "norm_grad")
        b = (s["bias"] if op == "norm" else torch.zeros_like(s["weight"])).double()
        b.requires_grad_(op == "norm_grad")
        y = torch.nn.functional.layer_norm(x, (case["cols"],), w, b, NORM_EPS)
        if op == "norm":
            var, mean = torch.var_mean(x, 1, correction=0)
            return dict(y=y, mean=mean, rstd=(var + NORM_EPS).rsqrt())
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return dict(dx=dx, dweight=dw, dbias=db)
    logits = s["logits"].double().requires_grad_(op == "route_grad")
    weights, loss = _exact_route(s, logits)
    if op == "route":
        return dict(ids=None, weights=weights, counts=None, loss=loss)
    total = (weights * s["dweights"].double()).sum() + loss.sum() * s["dloss"].double().sum()
    grad, = torch.autograd.grad(total, logits)
    return torch.where(torch.isfinite(s["logits"]), grad, 0.0)
