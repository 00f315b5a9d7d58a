"""Layer norm's kernels with several turns of every workgroup, against 64-bit plain forms."""
import pytest
import torch

import more_rows_ref as ref
import powersparse_amd as ps
from gpu_util import say, setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,x_type,y_type", [
    (40009, 24, torch.bfloat16, torch.bfloat16), (20011, 128, torch.float32, torch.bfloat16),
    (9001, 333, torch.float32, torch.float32), (9001, 300, torch.float16, torch.float16),
    (4500, 1024, torch.bfloat16, torch.bfloat16), (4500, 2048, torch.bfloat16, torch.float32),
    (2600, 4099, torch.float32, torch.float32), (2600, 4096, torch.float32, torch.bfloat16),
    (1100, 8192, torch.bfloat16, torch.bfloat16), (700, 16384, torch.float32, torch.float32),
    (700, 16384, torch.bfloat16, torch.bfloat16), (130, 32768, torch.float16, torch.float16),
    (130, 50003, torch.float32, torch.float32)])
def test_many_rows(rows, cols, x_type, y_type):
    setup()
    say(f"layer norm {rows} x {cols} {x_type} {y_type}")
    gen = torch.Generator(device="cuda").manual_seed(rows * 7 + cols)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    x = (normal(rows, cols) * torch.exp(normal(rows, 1)) + normal(rows, 1)).to(x_type)
    w, b = 1 + 0.2 * normal(cols), 0.2 * normal(cols)
    y = torch.empty((rows, cols), dtype=y_type, device="cuda")
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    ps.LayerNorm(x, w, b, y, mean, rstd)
    for got, want, what in zip((y, mean, rstd), ref.norm(x, w, b, 1e-5), ("y", "mean", "rstd")):
        ref.held(got, *want, what)
    dy, dx = normal(rows, cols).to(y_type), torch.empty_like(x)
    dw, db = torch.empty_like(w), torch.empty_like(b)
    work = torch.empty(ps.layer_norm_grad_workspace_bytes(rows, cols), dtype=torch.uint8,
                       device="cuda").fill_(255)
    ps.LayerNormGrad(dy, x, w, mean, rstd, dx, dw, db, work)
    for got, want, what in zip((dx, dw, db), ref.norm_grad(dy, x, w, mean, rstd),
                               ("dx", "dweight", "dbias")):
        ref.held(got, *want, what)


@pytest.mark.parametrize("rows,cols,x_type,y_type", [
    (1, 33, torch.float32, torch.float32), (65, 320, torch.float32, torch.bfloat16),
    (1025, 128, torch.float16, torch.float16), (4099, 33, torch.float32, torch.float32),
    (20011, 4, torch.float32, torch.float32), (20011, 128, torch.float32, torch.bfloat16),
    (20011, 320, torch.bfloat16, torch.float32), (40009, 24, torch.bfloat16, torch.bfloat16),
    (40009, 333, torch.float32, torch.float32), (100003, 7, torch.float16, torch.float32),
    (9001, 1024, torch.bfloat16, torch.bfloat16), (9001, 2048, torch.float32, torch.float32),
    (2600, 4099, torch.float32, torch.bfloat16), (1100, 16384, torch.float32, torch.float32),
    (1100, 16384, torch.bfloat16, torch.bfloat16), (1100, 32768, torch.float16, torch.float16),
    (1100, 50003, torch.float32, torch.float32)])
@pytest.mark.parametrize("accumulate", [False, True])
def test_sums_of_whole_numbers(rows, cols, x_type, y_type, accumulate):
    """dweight and dbias take every row once: with whole numbers, a mean of 0 and an rstd of 1 or 2
    every partial sum is below 2^24 and exact in FP32, in any order."""
    setup()
    say(f"layer norm's sums {rows} x {cols} {x_type} {y_type}")
    gen = torch.Generator(device="cuda").manual_seed(rows * 7 + cols)

    def whole(*shape):
        """1 to 8 with either sign."""
        n = torch.randint(1, 9, shape, generator=gen, device="cuda")
        return n * (2 * torch.randint(0, 2, shape, generator=gen, device="cuda") - 1)

    x, dy = whole(rows, cols), whole(rows, cols)
    rstd = torch.randint(1, 3, (rows,), generator=gen, device="cuda")
    was = whole(2, cols)
    assert 128 * rows + 8 < 1 << 24
    dw, db = (v.float() for v in was)
    dx = torch.empty((rows, cols), dtype=x_type, device="cuda")
    work = torch.empty(ps.layer_norm_grad_workspace_bytes(rows, cols), dtype=torch.uint8,
                       device="cuda").fill_(255)
    ps.LayerNormGrad(dy.to(y_type), x.to(x_type), None, torch.zeros(rows, device="cuda"),
                     rstd.float(), dx, dw, db, work, accumulate=accumulate)
    want_w, want_b = (dy * x * rstd[:, None]).sum(0), dy.sum(0)
    if accumulate:
        want_w, want_b = want_w + was[0], want_b + was[1]
    assert torch.equal(dw.long(), want_w) and torch.equal(db.long(), want_b)
    assert torch.equal(dw, dw.round()) and torch.equal(db, db.round())
