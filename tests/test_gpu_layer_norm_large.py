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
