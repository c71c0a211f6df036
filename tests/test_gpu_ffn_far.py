"""Rows whose offsets pass 2^31 elements or 2^32 bytes: the last rows are right, and those before them too where they are cheap to
check. The tolerances are those of test_gpu_norm.py, test_gpu_f8.py and test_gpu_gated.py with their sums written out.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg

pytestmark = [pytest.mark.gpu, pytest.mark.slow]
STEP = 2.0 ** -23


def test_norm(cuda):
    import torch
    rows, width = 66000, 32768
    assert rows * width > 2 ** 31
    x = torch.ones(rows, width, device="cuda", dtype=torch.bfloat16)
    x[-3:] = torch.randn(3, width, device="cuda").bfloat16()
    norm = gg.RmsNorm(width, dtype=gg.OutputType.kBF16)
    q, s, rstd = torch.zeros(rows, width, device="cuda", dtype=torch.float8_e4m3fn), torch.zeros(rows, 256, device="cuda"), torch.zeros(rows, device="cuda")
    assert norm.run(x, y=x, q=q, scales=s, rstd=rstd) == 0  # in place
    h = torch.ones(3, width, device="cuda", dtype=torch.float64)
    assert bool((x[:-3].amin(1) == 1).all()) and bool((x[:-3].amax(1) == 1).all())
    assert bool((q[-9:-3].float() == 448).all()) and float(s[-4, -1]) == pytest.approx(1 / 448, rel=1e-5)
    h = x[-3:].double()
    wide = q[-3:].double() * s[-3:].double().repeat_interleave(128, 1)
    # y is in 16 bits and q from the unrounded one: a half step of each
    assert bool(((wide - h).abs() <= h.abs() * (2.0 ** -4 + 2.0 ** -8 + 1e-4) + 1e-4).all())
    assert bool((h.square().mean(1) - 1).abs().max() < 1e-2)


def test_8bit_product(cuda):
    import torch
    rows, n, k = 36000, 32768, 64
    assert rows * n * 4 > 2 ** 32
    g = torch.Generator(device="cuda").manual_seed(1)
    a = torch.randn(rows, k, device="cuda", generator=g).to(torch.float8_e4m3fn)
    b = torch.randn(2, n, k, device="cuda", generator=g).to(torch.float8_e4m3fn)
    sa, sb = torch.rand(rows, 1, device="cuda", generator=g) + 0.5, torch.rand(2, n // 128, 1, device="cuda", generator=g) + 0.5
    d = torch.full((rows, n), 7.0, device="cuda")
    counts = torch.tensor([rows - 1000, 997], device="cuda", dtype=torch.int32)
    plan = gg.F8Plan(2, n, k, [t.data_ptr() for t in b], k, [t.data_ptr() for t in sb], output_type=gg.OutputType.kF32)
    assert plan.run(a, sa, counts, d) == 0
    torch.cuda.synchronize()
    assert plan.status() == 0
    for at, e in ((slice(0, 50), 0), (slice(rows - 1050, rows - 1000), 0), (slice(rows - 1000, rows - 950), 1), (slice(rows - 53, rows - 3), 1)):
        x, w = a[at].double() * sa[at].double(), b[e].double() * sb[e].double().repeat_interleave(128, 0)
        assert bool(((d[at].double() - x @ w.t()).abs() <= (x.abs() @ w.abs().t()) * (STEP * (128 + 4))).all())
    assert bool((d[-3:] == 7).all())


def test_gated_block(cuda):
    import torch
    rows, n, k = 66000, 32768, 64
    assert rows * n > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(rows, k, device="cuda", generator=g).bfloat16()
    wg, wu = [(torch.randn(1, k, n, device="cuda", generator=g) / 8).bfloat16() for _ in range(2)]
    gate, up, h = [torch.full((rows, n), 7.0, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
    plan = gg.GatedPlan(1, n, k, [wg.data_ptr()], [wu.data_ptr()], n)
    assert plan.run(x, None, h, gate=gate, up=up) == 0
    for at in (slice(0, 40), slice(rows - 40, rows)):
        xx = x[at].double()
        a, b = xx @ wg[0].double(), xx @ wu[0].double()
        want = a * torch.sigmoid(a) * b
        off = (xx.abs() @ wg[0].double().abs()) * (STEP * 66)
        assert bool(((gate[at].double() - a).abs() <= a.abs() * 2.0 ** -8 + 2 * off).all())
        more = (xx.abs() @ wu[0].double().abs()) * (STEP * 66)
        assert bool(((h[at].double() - want).abs() <= want.abs() * (2.0 ** -8 + 1e-4) + 2 * (1.13 * off * b.abs() + more * a.abs()) + 1e-30).all())
    gh = h  # any values
    gx, gw = torch.empty(rows, k, device="cuda", dtype=torch.bfloat16), [torch.empty(1, k, n, device="cuda") for _ in range(2)]
    counts = torch.tensor([rows - 5], device="cuda", dtype=torch.int32)
    gx.fill_(7.0)
    assert plan.backward(x, gate, up, gh, counts, gate, up, grad_x=gx, grad_gate_w=gw[0], grad_up_w=gw[1]) == 0
    torch.cuda.synchronize()
    assert plan.status() == 0 and bool((gx[-5:] == 7).all())
    at = slice(rows - 45, rows - 5)
    dg, du = gate[at].double(), up[at].double()
    want = dg @ wg[0].double().t() + du @ wu[0].double().t()
    size = dg.abs() @ wg[0].double().abs().t() + du.abs() @ wu[0].double().abs().t()
    assert bool(((gx[at].double() - want).abs() <= want.abs() * 2.0 ** -8 + size * (STEP * (2 * n + 2))).all())
    columns = slice(n - 64, n)
    for w, d in zip(gw, (gate, up)):
        part = d[:rows - 5, columns].double()
        want, size = x[:rows - 5].double().t() @ part, x[:rows - 5].double().abs().t() @ part.abs()
        # the sum over 66000 rows in FP32: a step each at most, if none is rounded to nearest
        assert bool(((w[0][:, columns].double() - want).abs() <= size * (STEP * rows)).all())
