"""Child process of tests/test_gpu_more_rows_guard.py: layer norm, the router and AdamW on
DeviceBuffers of exactly the sizes asked for, workspaces included, with the device allocation
guards on (PS_DEVICE_GUARD set by the parent). Checks the results against numpy in 64 bits and
prints `guard violations: N`."""
import gc
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import powersparse_amd as ps  # noqa: E402
from powersparse_amd import _native  # noqa: E402

U32 = 2.0 ** -24


def say(*a):
    print(*a, flush=True)


class Arr:
    """A host array on the device: the buffer and its description."""

    def __init__(self, host):
        self.dtype, self.shape = host.dtype, host.shape
        self.buf = ps.DeviceBuffer(host=host) if host.size else ps.DeviceBuffer(0)
        self.dev = ps.DeviceArray(self.buf, host.shape, str(host.dtype))

    def back(self):
        return self.buf.download(self.dtype, int(np.prod(self.shape))).reshape(self.shape)


def near(got, exact, off, what):
    unit = 2.0 ** -11 if got.dtype == np.float16 else U32
    bound = 2 * off + unit * np.abs(exact) + 2.0 ** -24
    assert (np.abs(got.astype(np.float64) - exact) <= bound).all(), what


def layer_norm(rng, rows, cols, dtype):
    x = (rng.normal(size=(rows, cols)) + rng.normal(size=(rows, 1))).astype(dtype)
    w, b = rng.normal(size=cols).astype(np.float32), rng.normal(size=cols).astype(dtype)
    d_x, d_w, d_b = Arr(x), Arr(w), Arr(b)
    y = Arr(np.full((rows, cols), 7, dtype))
    mean, rstd = Arr(np.full(rows, 7, np.float32)), Arr(np.full(rows, 7, np.float32))
    ps.LayerNorm(d_x.dev, d_w.dev, d_b.dev, y.dev, mean.dev, rstd.dev, eps=0.01)
    x64 = x.astype(np.float64)
    m = x64.mean(1, keepdims=True)
    s = 1 / np.sqrt(((x64 - m) ** 2).mean(1, keepdims=True) + 0.01)
    # sums of `cols` terms in any order; means are no larger than some 5, 1 / deviation than 10
    off = (cols + 20) * U32 * 100 * (1 + np.abs(w) + np.abs(b.astype(np.float64)))
    near(y.back(), (x64 - m) * s * w + b, off, "y")
    dy = rng.normal(size=(rows, cols)).astype(dtype)
    d_dy, dx = Arr(dy), Arr(np.full((rows, cols), 7, dtype))
    dw, db = Arr(np.full(cols, 7, np.float32)), Arr(np.full(cols, 7, dtype))
    work = ps.DeviceBuffer(ps.layer_norm_grad_workspace_bytes(rows, cols))
    ps.LayerNormGrad(d_dy.dev, d_x.dev, d_w.dev, mean.dev, rstd.dev, dx.dev, dw.dev, db.dev, work)
    ps.synchronize()
    m, s = mean.back().astype(np.float64)[:, None], rstd.back().astype(np.float64)[:, None]
    xh, g = (x64 - m) * s, dy.astype(np.float64) * w
    exact = s * (g - g.mean(1, keepdims=True) - xh * (g * xh).mean(1, keepdims=True))
    near(dx.back(), exact, (cols + 20) * U32 * s * 10 * (1 + np.abs(g) + np.abs(xh)), "dx")
    near(dw.back(), (dy * xh).sum(0), (rows + 8) * U32 * np.abs(dy * xh).sum(0), "dweight")
    near(db.back(), dy.astype(np.float64).sum(0), (rows + 8) * U32 * np.abs(dy.astype(np.float64)).sum(0),
         "dbias")
    say(f"layer norm {rows} x {cols} {np.dtype(dtype)}")


def route(rng, tokens, experts, top_k, dtype):
    logits = rng.normal(size=(tokens, experts)).astype(dtype)
    mask = (rng.random(tokens) < 0.8).astype(np.uint8)
    d_logits, d_mask = Arr(logits), Arr(mask)
    ids, w = Arr(np.zeros((tokens, top_k), np.int32)), Arr(np.zeros((tokens, top_k), np.float32))
    counts, loss = Arr(np.zeros(experts + 1, np.int32)), Arr(np.zeros(1, np.float32))
    work = ps.DeviceBuffer(ps.expert_route_workspace_bytes(tokens, experts))
    ps.ExpertRoute(d_logits.dev, ids.dev, w.dev, counts.dev, loss.dev, work, mask=d_mask.dev)
    grad, dw = Arr(np.full((tokens, experts), 7, dtype)), Arr(rng.normal(size=(tokens, top_k)).astype(np.float32))
    ps.ExpertRouteGrad(d_logits.dev, ids.dev, dw.dev, counts.dev, loss.dev, grad.dev)
    ps.synchronize()
    on = mask.astype(bool)
    order = np.argsort(-logits.astype(np.float64), axis=1, kind="stable")[:, :top_k]
    assert np.array_equal(ids.back(), np.where(on[:, None], order, -1))
    assert np.array_equal(counts.back()[:-1], np.bincount(order[on].reshape(-1), minlength=experts))
    assert counts.back()[-1] == on.sum()
    e = np.exp(logits.astype(np.float64) - logits.max(1, keepdims=True))
    chosen = np.take_along_axis(e, order, 1)
    chosen = chosen / chosen.sum(1, keepdims=True) * on[:, None]
    near(w.back(), chosen, 40 * U32 * chosen, "weights")
    assert np.isfinite(grad.back()).all() and not grad.back()[~on].any()
    assert np.abs(grad.back().astype(np.float64).sum(1)).max() <= 0.05  # of a softmax: zero
    say(f"route {tokens} x {experts} top {top_k} {np.dtype(dtype)}")


def adamw(rng, sizes, grad_dtype, f8):
    p = [rng.normal(size=n).astype(np.float32) for n in sizes]
    g = [rng.normal(size=n).astype(grad_dtype) for n in sizes]
    state = np.uint8 if f8 else np.float32
    d_p, d_g = [Arr(x) for x in p], [Arr(x) for x in g]
    m, v = ([Arr(np.zeros(n, state)) for n in sizes] for _ in range(2))
    scales = [Arr(np.zeros((ps.state_blocks(n), 2), np.float32)) for n in sizes] if f8 else None
    copies = [Arr(np.zeros(n, np.float16)) for n in sizes]
    dev = lambda xs: [x.dev for x in xs] if xs else None  # noqa: E731
    tensors = ps.AdamWList(dev(d_p), dev(d_g), dev(m), dev(v), scales=dev(scales),
                           copies=dev(copies), weight_decay=0.5)
    ps.AdamWStep(tensors, 0.01, 1)
    ps.synchronize()
    for x, grad, got, copy in zip(p, g, d_p, copies):
        g64 = grad.astype(np.float64)
        exact = x - 0.01 * (0.5 * x.astype(np.float64) + g64 / (np.abs(g64) + 1e-8))
        near(got.back(), exact, 0.01 * 40 * U32 * (1 + np.abs(x)), "parameter")
        near(copy.back(), exact, 0.01 * 40 * U32 * (1 + np.abs(x)), "copy")
    tensors.close()
    say(f"adamw {len(sizes)} tensors {np.dtype(grad_dtype)} 8 bits: {f8}")


def main():
    ps.set_device(0)
    lib = _native.hip()
    assert lib.ps_guard_violations() == 0, "guards are off or already tripped"
    rng = np.random.default_rng(5)
    for rows, cols in ((1, 1), (3, 2), (7, 5), (33, 40), (65, 64), (5, 333), (130, 520), (9, 1030),
                       (3, 2100), (2, 5000), (2, 9000), (3, 17000), (2, 40001), (5000, 70)):
        for dtype in (np.float32, np.float16):
            layer_norm(rng, rows, cols, dtype)
    for tokens, experts, top_k in ((1, 1, 1), (5, 3, 2), (40, 17, 3), (33, 64, 8), (9, 100, 5),
                                   (300, 130, 4), (70, 500, 9), (19, 1023, 70), (9000, 20, 2),
                                   (8200, 200, 3)):
        for dtype in (np.float32, np.float16):
            route(rng, tokens, experts, top_k, dtype)
    for dtype in (np.float32, np.float16):
        for f8 in (False, True):
            adamw(rng, [1, 255, 256, 257, 4095, 4096, 4097, 12289, 7], dtype, f8)
    gc.collect()
    say(f"guard violations: {lib.ps_guard_violations()}")


if __name__ == "__main__":
    main()
