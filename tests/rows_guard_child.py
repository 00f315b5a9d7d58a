"""Child process of tests/test_gpu_rows_guard.py: the row operators on
DeviceBuffers of exactly the sizes asked for, workspaces included, with the
device allocation guards on (PS_DEVICE_GUARD set by the parent). Checks the
results against numpy in 64 bits and prints `guard violations: N`."""
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


def near(got, exact, magnitude, terms, what):
    unit = 2.0 ** -11 if got.dtype == np.float16 else U32
    bound = 2 * terms * U32 * magnitude + unit * np.abs(exact) + 2.0 ** -25
    assert (np.abs(got.astype(np.float64) - exact) <= bound).all(), what


def embedding(rng, count, rows, cols, dtype, ids_t):
    table = rng.normal(size=(rows, cols)).astype(dtype)
    ids = rng.integers(-1, rows + 1, count).astype(ids_t)
    if count > 50:
        ids[: count // 2] = rows // 2  # a long run
    out, d_table, d_ids = Arr(np.full((count, cols), 7, dtype)), Arr(table), Arr(ids)
    ps.EmbeddingLookup(d_table.dev, d_ids.dev, out.dev, scale=1.5)
    ps.synchronize()
    ok = (ids >= 0) & (ids < rows)
    exact = np.where(ok[:, None], table[np.clip(ids, 0, rows - 1)].astype(np.float64) * 1.5, 0)
    near(out.back(), exact, np.abs(exact), 1, "lookup")
    dy, grad = rng.normal(size=(count, cols)).astype(dtype), Arr(np.full((rows, cols), 7, np.float32))
    work = ps.DeviceBuffer(ps.embedding_grad_workspace_bytes(count, cols, rows))
    d_dy = Arr(dy)
    exact, mag = np.zeros((rows, cols)), np.zeros((rows, cols))
    np.add.at(exact, ids[ok], dy[ok].astype(np.float64))
    np.add.at(mag, ids[ok], np.abs(dy[ok].astype(np.float64)))
    ps.EmbeddingGrad(d_ids.dev, d_dy.dev, grad.dev, work)
    ps.synchronize()
    near(grad.back(), exact, mag, count, "gradient")
    ps.EmbeddingGrad(d_ids.dev, d_dy.dev, grad.dev, work, accumulate=True)
    ps.synchronize()
    near(grad.back(), 2 * exact, 2 * mag, count, "accumulated gradient")
    say(f"embedding count={count} rows={rows} cols={cols} {np.dtype(dtype)}")


def experts(rng, tokens, top_k, count, cols, dtype):
    ids = rng.integers(-1, count + 1, (tokens, top_k)).astype(np.int64)
    n = tokens * top_k
    order, position = Arr(np.zeros(n, np.int32)), Arr(np.zeros((tokens, top_k), np.int32))
    offsets = Arr(np.zeros(count + 1, np.int32))
    work = ps.DeviceBuffer(ps.expert_sort_workspace_bytes(n, count))
    ps.ExpertSort(Arr(ids).dev, order.dev, position.dev, offsets.dev, work)
    ps.synchronize()
    key = np.where((ids >= 0) & (ids < count), ids, count).reshape(-1)
    o = np.argsort(key, kind="stable")
    assert np.array_equal(order.back(), o)
    p = np.empty(n, np.int64)
    p[o] = np.arange(n)
    p = np.where(key < count, p, -1).reshape(tokens, top_k)
    assert np.array_equal(position.back(), p)
    filled = int((key < count).sum())
    assert offsets.back()[-1] == filled
    # only the filled rows exist: positions never lead beyond them
    x, ys = rng.normal(size=(tokens, cols)).astype(dtype), rng.normal(size=(filled, cols)).astype(dtype)
    w = rng.random((tokens, top_k)).astype(np.float32)
    d_x, d_ys, d_w = Arr(x), Arr(ys), Arr(w)
    xs, y = Arr(np.zeros((filled, cols), dtype)), Arr(np.zeros((tokens, cols), dtype))
    dys, dw = Arr(np.zeros((filled, cols), dtype)), Arr(np.zeros((tokens, top_k), np.float32))
    ps.ExpertDispatch(d_x.dev, position.dev, xs.dev)
    ps.ExpertCombine(d_ys.dev, position.dev, d_w.dev, y.dev)
    ps.ExpertCombineGrad(d_x.dev, d_ys.dev, position.dev, d_w.dev, dys.dev, dw.dev)
    ps.synchronize()
    assert np.array_equal(xs.back(), x[o[:filled] // top_k])
    on = (p >= 0)[..., None]
    rows = np.where(on, ys.astype(np.float64)[np.maximum(p, 0)], 0) if filled else np.zeros((tokens, top_k, cols))
    near(y.back(), (rows * w[..., None]).sum(1), np.abs(rows * w[..., None]).sum(1), 2 * top_k, "combine")
    near(dw.back(), (rows * x[:, None]).sum(2), np.abs(rows * x[:, None]).sum(2), cols + 1, "dweights")
    g = (w[..., None].astype(np.float64) * x[:, None])[p >= 0][np.argsort(p[p >= 0])]
    near(dys.back(), g, np.abs(g), 1, "dys")
    say(f"experts tokens={tokens} top_k={top_k} experts={count} cols={cols} {np.dtype(dtype)}")


def clipping(rng, sizes, dtype):
    grads = [rng.normal(size=n).astype(dtype) for n in sizes]
    dev = [Arr(g) for g in grads]
    norm = Arr(np.zeros(1, np.float32))
    exact = np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in grads))
    glist = ps.GradientList([d.dev for d in dev])
    ps.ClipGradNorm(glist, float(exact) / 2, norm.dev)
    ps.synchronize()
    assert abs(norm.back()[0] - exact) <= 2 * U32 * exact
    for g, d in zip(grads, dev):
        e = g.astype(np.float64) * ((float(exact) / 2) / (exact + 1e-6))
        near(d.back(), e, np.abs(e), 2, "clip")
    glist.close()
    say(f"clipping {len(sizes)} tensors {np.dtype(dtype)}")


def main():
    ps.set_device(0)
    lib = _native.hip()
    assert lib.ps_guard_violations() == 0, "guards are off or already tripped"
    rng = np.random.default_rng(3)
    for count, rows, cols in ((1, 1, 1), (17, 40, 33), (300, 5000, 8), (4096, 1030, 7),
                              (5000, 70000, 40), (70001, 3, 100), (200001, 900, 12),
                              (800001, 2000, 3)):
        for dtype, ids_t in ((np.float32, np.int32), (np.float16, np.int64)):
            embedding(rng, count, rows, cols, dtype, ids_t)
    for tokens, top_k, count, cols in ((1, 1, 1, 1), (3, 8, 64, 333), (700, 7, 1024, 20),
                                       (40000, 6, 130, 9)):
        for dtype in (np.float32, np.float16):
            experts(rng, tokens, top_k, count, cols, dtype)
    for dtype in (np.float32, np.float16):
        clipping(rng, [1, 4095, 4096, 4097, 12289, 7], dtype)
    import gc
    gc.collect()
    say(f"guard violations: {lib.ps_guard_violations()}")


if __name__ == "__main__":
    main()
