"""The norm of rows that take 4 and 8 spans of 256 values a warp (wider than 8192 and 16384), with three and more rows for each
block: the values asked for a row ahead, the buffers of sums taken in turn, and the weight's gradient over several
rows. The checks and their tolerances are those of test_gpu_norm.py.
"""
import pytest

import test_gpu_norm as norm_tests

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind,weight", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("width,rows", [(9000, 1200), (16500, 700), (20000, 600), (32768, 512)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (8, 0), (3, 1)])
def test_many_wide_rows(cuda, kind, weight, width, rows, pad, offset):
    norm_tests.test_norm(cuda, kind, weight, width, rows, pad, offset)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("width", [20000, 32767, 32768])
def test_in_place(cuda, kind, width):
    """Results in the place of x, the residual and the gradients, the same bits as elsewhere."""
    import torch

    import grouped_gemm_gpu_kernel_b200 as gg
    rows, dt = 500, norm_tests.dtypes()[kind]
    x, r, w, gy, gh = [torch.randn(*s, device=cuda).to(dt) for s in ((rows, width), (rows, width), (width,), (rows, width), (rows, width))]
    norm = gg.RmsNorm(width, dtype=norm_tests.KINDS[kind])
    y, h, rstd, gx, gw = torch.empty_like(x), torch.empty_like(x), torch.empty(rows, device=cuda), torch.empty_like(x), torch.empty(width, device=cuda)
    assert norm.run(x, w, y=y, residual=r, residual_out=h, rstd=rstd) == 0
    assert norm.backward(h, w, rstd, gy, gx, grad_weight=gw, grad_h=gh) == 0
    assert norm.run(x, w, y=x, residual=r, residual_out=r) == 0
    assert torch.equal(x, y) and torch.equal(r, h)
    again = torch.empty_like(gw)
    assert norm.backward(h, w, rstd, gy, gh, grad_weight=again, grad_h=gh) == 0
    assert torch.equal(gh, gx) and torch.equal(again, gw)
