"""Plain 64-bit forms of the row operators on the host, and the bounds that
the operators' results are held to.

u32 = 2^-24 is FP32's unit roundoff, u its result type's. A sum of m products
in FP32, in any order, is off by at most m * u32 / (1 - m * u32) times the sum
of the magnitudes (m - 1 additions and one rounding per product); a scale adds
one rounding, the result's own rounding u times the result (and half of the
smallest subnormal of the type)."""
import torch

U32 = 2.0 ** -24
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def close(got, exact, magnitude, terms, what):
    """|got - exact| within the bound for `terms` FP32 roundings of values whose
    magnitudes add up to `magnitude`, rounded once to got's type."""
    dtype = got.dtype
    got, exact = got.detach().cpu().double(), exact.double()
    g = terms * U32 / (1 - terms * U32)
    bound = g * magnitude * (1 + UNIT[dtype]) + UNIT[dtype] * exact.abs() + TINY[dtype]
    bad = ~((got - exact).abs() <= bound)
    assert not bad.any(), (
        f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound; first at "
        f"{torch.nonzero(bad)[0].tolist()}: {got[bad][0]} for {exact[bad][0]}, "
        f"bound {torch.as_tensor(bound).expand(bad.shape)[bad][0]}")


def lookup(table, ids, scale):
    t, i = table.cpu().double(), ids.cpu().long().reshape(-1)
    ok = (i >= 0) & (i < t.shape[0])
    return torch.where(ok[:, None], t[i.clamp(0, max(t.shape[0] - 1, 0))] * scale, 0.0)


def lookup_grad(ids, dy, rows, scale, padding=-1):
    """(gradient, sum of magnitudes, most ids of a row)."""
    i, g = ids.cpu().long().reshape(-1), dy.cpu().double()
    ok = (i >= 0) & (i < rows) & (i != padding)
    out = torch.zeros((rows, g.shape[1]), dtype=torch.float64)
    mag = torch.zeros_like(out)
    out.index_add_(0, i[ok], g[ok] * scale)
    mag.index_add_(0, i[ok], (g[ok] * scale).abs())
    most = int(torch.bincount(i[ok], minlength=1).max()) if ok.any() else 0
    return out, mag, most


def sort(ids, experts):
    """(order, position, offsets), slot by slot."""
    flat = ids.cpu().reshape(-1).tolist()
    places = [[] for _ in range(experts + 1)]
    for slot, e in enumerate(flat):
        places[e if 0 <= e < experts else experts].append(slot)
    order = [s for p in places for s in p]
    position = [-1] * len(flat)
    offsets, at = [], 0
    for e in range(experts + 1):
        offsets.append(at)
        for s in places[e]:
            if e < experts:
                position[s] = at
            at += 1
    return order, position, offsets


def combine(ys, position, weights):
    """(y, sum of magnitudes)."""
    v, p = ys.cpu().double(), position.cpu().long()
    w = weights.cpu().double() if weights is not None else torch.ones(p.shape, dtype=torch.float64)
    y = torch.zeros((p.shape[0], v.shape[1]), dtype=torch.float64)
    mag = torch.zeros_like(y)
    for t in range(p.shape[0]):
        for k in range(p.shape[1]):
            if 0 <= p[t, k] < v.shape[0]:
                y[t] += w[t, k] * v[p[t, k]]
                mag[t] += (w[t, k] * v[p[t, k]]).abs()
    return y, mag


def combine_grad(dy, ys, position, weights):
    """(dys with NaN in the rows that no slot names, dweights, its magnitudes)."""
    g, v, p, w = (x.cpu().double() for x in (dy, ys, position, weights))
    dys = torch.full_like(v, float("nan"))
    dw = torch.zeros(p.shape, dtype=torch.float64)
    mag = torch.zeros_like(dw)
    for t in range(p.shape[0]):
        for k in range(p.shape[1]):
            q = int(p[t, k])
            if 0 <= q < v.shape[0]:
                dys[q] = w[t, k] * g[t]
                dw[t, k] = (g[t] * v[q]).sum()
                mag[t, k] = (g[t] * v[q]).abs().sum()
    return dys, dw, mag


def strided(rows, cols, dtype, pad=0, offset=0, fill=None, device="cuda"):
    """A rows x cols view with `pad` elements between rows, `offset` elements into its
    allocation; returns (view, whole allocation)."""
    whole = torch.empty(offset + rows * (cols + pad) + pad + 8, dtype=dtype, device=device)
    whole.fill_(float("nan") if fill is None else fill)
    view = whole[offset:offset + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    return view, whole
