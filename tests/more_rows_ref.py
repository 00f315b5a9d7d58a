"""Plain 64-bit forms of layer norm, the router and AdamW on the host, with the bounds that the
operators' results are held to.

u = 2^-24 is FP32's unit roundoff. Each function returns the exact values and, for each, how far
FP32 arithmetic may be off before the result's own rounding: a sum whose longest chain has h
additions is off by at most h u / (1 - h u) times the sum of the magnitudes, each other operation by
u relative (the hardware's square root, reciprocal and exponential by 2 u; FP32 arguments of an
exponential by u times their magnitude)."""
import math

import torch

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def held(got, exact, off, what):
    """|got - exact| <= off, and got's own rounding on top."""
    dtype = got.dtype
    got = got.detach().cpu().double()
    assert got.shape == exact.shape, (what, got.shape, exact.shape)
    bound = off * (1 + UNIT[dtype]) + UNIT[dtype] * exact.abs() + TINY[dtype]
    bad = ~((got - exact).abs() <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound; first at "
        f"{torch.nonzero(bad)[0].tolist()}: {got[bad][0]} for {exact[bad][0]}, "
        f"bound {torch.as_tensor(bound).expand(bad.shape)[bad][0]}")


def gamma(h):
    return h * U32 / (1 - h * U32)


def chain(cols):
    """The longest chain of additions in a row's sum: a lane adds at most 64 elements and some
    more of rows wider than 32,768, then 10 steps join 1,024 lanes."""
    return min(cols, 80 + cols // 512)


def norm(x, weight, bias, eps):
    """((y, off), (mean, off), (rstd, off))."""
    x = x.detach().cpu().double()
    cols = x.shape[1]
    w = torch.ones(cols, dtype=torch.float64) if weight is None else weight.cpu().double()
    b = torch.zeros(cols, dtype=torch.float64) if bias is None else bias.cpu().double()
    mean = x.mean(1, keepdim=True)
    dev = x - mean
    var = (dev * dev).mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    mean_off = gamma(chain(cols) + 2) * x.abs().mean(1, keepdim=True)
    # the deviations' own rounding (twice, squared), the square's, the sum's, the division's; and
    # the mean's error, which adds its square to the variance
    var_off = gamma(chain(cols) + 8) * var + 1.01 * mean_off ** 2
    rstd_rel = 0.5 * var_off / (var + eps) * 1.01 + 5 * U32
    xh = dev * rstd
    y = xh * w + b
    off = rstd * w.abs() * mean_off * 1.01 + (xh * w).abs() * (rstd_rel + 4 * U32) + \
        U32 * (y.abs() + b.abs())
    return (y, off), (mean.view(-1), mean_off.view(-1)), (rstd.view(-1), (rstd * rstd_rel).view(-1))


def norm_grad(dy, x, weight, mean, rstd):
    """((dx, off), (dweight, off), (dbias, off)) by the mean and rstd that are given."""
    dy, x = dy.detach().cpu().double(), x.detach().cpu().double()
    rows, cols = x.shape
    w = torch.ones(cols, dtype=torch.float64) if weight is None else weight.cpu().double()
    rstd = rstd.cpu().double()[:, None]
    xh = (x - mean.cpu().double()[:, None]) * rstd
    g = dy * w
    mg, mgx = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = rstd * (g - mg - xh * mgx)
    h = chain(cols) + 6
    off = rstd * (gamma(h) * (g.abs().mean(1, keepdim=True) +
                              xh.abs() * (g * xh).abs().mean(1, keepdim=True)) +
                  gamma(6) * (g.abs() + mg.abs() + (xh * mgx).abs()))
    return ((dx, off), ((dy * xh).sum(0), gamma(rows + 6) * (dy * xh).abs().sum(0)),
            (dy.sum(0), gamma(rows + 2) * dy.abs().sum(0)))


def route(logits, top_k, normalize, mask=None):
    """A dict of ids, weights, counts, loss, and the bounds weights_off, loss_off; logits
    without NaN and infinities but -inf."""
    l = logits.detach().cpu().double()
    T, E = l.shape
    ids = torch.full((T, top_k), -1, dtype=torch.int32)
    weights = torch.zeros((T, top_k), dtype=torch.float64)
    off = torch.zeros_like(weights)
    p = torch.zeros((T, E), dtype=torch.float64)
    counts = torch.zeros(E + 1, dtype=torch.int64)
    far = torch.zeros(T, dtype=torch.float64)  # of logits from the largest
    for t in range(T):
        row = l[t].tolist()
        open_to = [e for e in range(E) if row[e] != -math.inf]
        if not open_to or (mask is not None and not bool(mask[t])):
            continue
        best = sorted(open_to, key=lambda e: (-row[e], e))[:top_k]
        ids[t, :len(best)] = torch.tensor(best, dtype=torch.int32)
        top = row[best[0]]
        p[t] = torch.softmax(l[t], 0)
        w = p[t][best]
        if normalize:
            w = w / w.sum()
        weights[t, :len(best)] = w
        far[t] = top - min(row[e] for e in open_to)
        counts[best] += 1
        counts[E] += 1
    # exponential by powers of two: the difference of logits is rounded, and its product with
    # log2(e), whose FP32 value is 0.22 U32 off: 2.22 times the difference; its own error; the sum
    # over the experts; two divisions
    rel = (2.25 * far + E + 12) * U32
    off = weights * rel[:, None] + 2.0 ** -126
    chosen, tokens = counts[:E].double(), int(counts[E])
    loss, loss_off = 0.0, 0.0
    if tokens:
        scale = E / (tokens * float(chosen.sum()))
        loss = float((chosen * p.sum(0)).sum()) * scale
        loss_off = float((chosen * (p * (rel + (T + 6) * U32)[:, None]).sum(0)).sum()) * scale
        loss_off += 2.0 ** -120
    return dict(ids=ids, weights=weights, weights_off=off, counts=counts.to(torch.int32), p=p,
                rel=rel, loss=torch.tensor([loss], dtype=torch.float64), loss_off=loss_off)


def route_grad(logits, ids, dweights, counts, dloss, normalize):
    """(dlogits, off)."""
    l, ids = logits.detach().cpu().double(), ids.cpu().long()
    T, E = l.shape
    dw = torch.zeros(ids.shape, dtype=torch.float64) if dweights is None else dweights.cpu().double()
    by_loss = torch.zeros(E, dtype=torch.float64)
    if dloss is not None and int(counts[E]) > 0:
        c = counts.cpu().double()
        by_loss = float(dloss) * E * c[:E] / (c[E] * c[:E].sum())
    out, off = torch.zeros_like(l), torch.zeros_like(l)
    for t in range(T):
        if ids[t, 0] < 0:
            continue
        p = torch.softmax(l[t], 0)
        open_to = l[t][l[t] > -math.inf]
        rel = float(2.25 * (open_to.max() - open_to.min()) + 2 * E + 24) * U32
        chosen = ids[t][ids[t] >= 0]
        d = dw[t][ids[t] >= 0]
        h = by_loss.clone()
        if not normalize:
            h[chosen] += d
        out[t] = p * (h - (p * h).sum())
        off[t] = p * (h.abs() + (p * h.abs()).sum()) * 2 * rel
        if normalize:
            w = p[chosen] / p[chosen].sum()
            out[t][chosen] += w * (d - (w * d).sum())
            off[t][chosen] += w * (d.abs() + (w * d.abs()).sum()) * 2 * rel
    return out, off + 2.0 ** -120


def adamw(p, g, m, v, lr, step, decay, beta1=0.9, beta2=0.999, eps=1e-8, scale=1.0):
    """((p, off), (m, off), (v, off)) after a step, all given and returned in 64 bits."""
    g = g * scale
    M = beta1 * m.abs() + (1 - beta1) * g.abs()
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    root = (v / (1 - beta2 ** step)).sqrt()
    up = m / (1 - beta1 ** step) / (root + eps)
    new = p - lr * (decay * p + up)
    # m: six roundings of its terms; v ten; the update thirty over m's terms; the rate's own
    up_off = gamma(40) * (M / (1 - beta1 ** step) / (root + eps)) + gamma(4) * (decay * p).abs()
    return (new, lr * up_off + 2.0 ** -140), (m, gamma(7) * M + 2.0 ** -140), \
        (v, gamma(11) * v + 2.0 ** -140)


def spacing(a):
    """Of E4M3's grid around magnitudes `a`."""
    _, e = torch.frexp(a)
    return torch.ldexp(torch.ones_like(a), e.clamp(min=-5) - 4)


def thresholds(n, step):
    """u of each of n elements of a tensor in a step."""
    i = torch.arange(n)
    return ((((i * 0x6A09E667) + step * 0x9E3779B9) & 0xFFFFFFFF) >> 12).double() * 2.0 ** -20


def to_8_bits(x, step, positive):
    """(magnitudes of codes, scales, how near each was to the other code) of x in blocks of 256."""
    n = x.numel()
    pad = -n % 256
    full = torch.cat([x.abs(), torch.zeros(pad, dtype=torch.float64)]).view(-1, 256)
    scale = (full.amax(1) / 448.0).clamp(min=2.0 ** -126)
    ratio = (full / scale[:, None]).view(-1)[:n]
    q = spacing(ratio)
    t = ratio / q + thresholds(n, step)
    code = (torch.floor(t) * q).clamp(max=448.0)
    if positive:
        code = torch.where(x > 0, code.clamp(min=2.0 ** -9), code)
    return code, scale, (t - torch.round(t)).abs(), ratio / q
