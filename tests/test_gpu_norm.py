"""The root-mean-square norm, its 8-bit output and its gradient against the definition in 64 bits.

Tolerances. u = 2^-24 is half a step of FP32. The sum of squares is of positive numbers: its relative error is at most the
longest chain of additions (64 of a thread, 5 + 5 across lanes and warps, an fma each) times u, and with the division, eps,
the root and the reciprocal rstd is off by less than SUM = (64 + 10) u / 2 + 4 u < 41 u. y takes two products more and is
rounded once to its type (half a step). A mean of products of both signs has an error of the chain times the sum of the
magnitudes; 2 CHAIN with CHAIN = 80 u covers the products and rstd. An 8-bit value is off by half a step of its type, or, below
its normal numbers, by half of the smallest one, times the scale.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg
from grouped_gemm_gpu_kernel_b200 import capi

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SUM = 41 * U
CHAIN = 80 * U
KINDS = {"f32": gg.OutputType.kF32, "f16": gg.OutputType.kF16, "bf16": gg.OutputType.kBF16}
TINY = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}  # smallest subnormal


def dtypes():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def half_step(kind):
    import torch
    return 0.0 if kind == "f32" else torch.finfo(dtypes()[kind]).eps / 2


def matrix(rows, width, dtype, pitch=None, offset=0, fill=0):
    """A rows x width view of a larger buffer; the buffer is there to see what is written around it."""
    import torch
    pitch = width if pitch is None else pitch
    size = torch.empty(0, dtype=dtype).element_size()
    buf = torch.full(((rows + 1) * pitch + offset + 64,), fill, device="cuda", dtype=torch.uint8 if size == 1 else dtype)
    return buf, buf.view(dtype)[offset:].as_strided((rows, width), (pitch, 1))


def check(name, got, want, bound):
    import torch
    off = (got.double() - want).abs()
    worst = (off - bound).max()
    assert bool((off <= bound).all()), f"{name}: {float(worst)} past the bound, largest difference {float(off.max())}"
    assert bool(torch.isfinite(got.double()).all())


def reference(h, w, eps):
    rstd = 1.0 / (h.square().mean(1, keepdim=True) + eps).sqrt()
    return rstd, h * rstd * w


WIDTHS = [1, 7, 8, 64, 127, 128, 129, 255, 256, 257, 1000, 1003, 1024, 2048, 4096, 4100, 8192, 8200, 16384, 20000, 32768]


@pytest.mark.parametrize("kind,weight", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows,pad,offset", [(1, 0, 0), (5, 8, 0), (3, 3, 1), (2050, 0, 0)])
def test_norm(cuda, kind, weight, width, rows, pad, offset):
    import torch
    if rows > 100 and width * rows > 2050 * 8200:
        pytest.skip("the team for many rows of this width is that of 8200")
    dt, wdt = dtypes()[kind], dtypes()[weight]
    g = torch.Generator(device="cuda").manual_seed(width * 10 + rows)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    pitch = width + pad
    x, r = [matrix(rows, width, dt, pitch, offset)[1] for _ in range(2)]
    x.copy_(rnd(rows, width) * torch.exp(rnd(rows, 1)))
    r.copy_(rnd(rows, width))
    w = (1.0 + 0.3 * rnd(width)).to(wdt)
    hb, h = matrix(rows, width, dt, pitch, offset, fill=7)
    yb, y = matrix(rows, width, dt, pitch, offset, fill=7)
    qb, q = matrix(rows, width, dtypes()["e4m3"], pitch, offset, fill=7)
    blocks = -(-width // 128)
    sb, s = matrix(rows, blocks, torch.float32, blocks + 1, 0, fill=7)
    rstd = torch.empty(rows, device="cuda")
    eps = 1e-5
    norm = gg.RmsNorm(width, dtype=KINDS[kind], weight_type=KINDS[weight], eps=eps)
    assert norm.run(x, w, y=y, residual=r, residual_out=h, q=q, scales=s, rstd=rstd) == 0
    torch.cuda.synchronize()
    assert torch.equal(h, (x.float() + r.float()).to(dt))
    want_rstd, want = reference(h.double(), w.double(), eps)
    check("rstd", rstd[:, None], want_rstd, want_rstd * SUM)
    check("y", y, want, want.abs() * (half_step(kind) * 1.01 + SUM + 3 * U) + TINY[kind])
    groups = torch.nn.functional.pad(want, (0, blocks * 128 - width)).view(rows, blocks, 128)
    most = groups.abs().amax(2) / 448.0
    check("scales", s, most, most * (SUM + 6 * U))
    wide = s.double().repeat_interleave(128, 1)[:, :width]
    check("q", q.double() * wide, want, want.abs() * (2.0 ** -4 + 1e-4) + wide * 2.0 ** -10)
    # around the rows nothing is written
    for buf, view, size in ((hb, h, width), (yb, y, width), (qb, q, width), (sb, s, blocks)):
        before = buf.clone()
        view.view(torch.uint8 if buf.dtype == torch.uint8 else buf.dtype).fill_(7)
        assert bool((buf == 7).all())
        buf.copy_(before)

    # the gradient
    gy, gh = [matrix(rows, width, dt, pitch, offset)[1] for _ in range(2)]
    gy.copy_(rnd(rows, width)), gh.copy_(rnd(rows, width))
    gxb, gx = matrix(rows, width, dt, pitch, offset, fill=7)
    gw = torch.empty(width, device="cuda")
    assert norm.backward(h, w, rstd, gy, gx, grad_weight=gw, grad_h=gh) == 0
    xhat, gd = h.double() * rstd.double()[:, None], gy.double() * w.double()
    mean, mags = (gd * xhat).mean(1, keepdim=True), (gd * xhat).abs().mean(1, keepdim=True)
    want = rstd.double()[:, None] * (gd - xhat * mean) + gh.double()
    parts = rstd.double()[:, None] * (gd.abs() + xhat.abs() * mags) + gh.double().abs()
    check("grad_x", gx, want, want.abs() * half_step(kind) * 1.01 + 2 * CHAIN * parts + TINY[kind])
    terms = gy.double() * xhat
    check("grad_weight", gw, terms.sum(0), (rows + 128) * U * terms.abs().sum(0) + 1e-30)
    gx.fill_(7)
    assert bool((gxb == 7).all())


@pytest.mark.parametrize("kind", ["e4m3", "e5m2"])
def test_eight_bits(cuda, kind):
    """Blocks of zeros, of very small and of very large values, and with values that are not finite."""
    import torch
    width, rows = 640, 8
    x = torch.randn(rows, width, device="cuda")
    x[0] = 0.0
    x[1, 128:256] = 0.0
    x[2, :128] *= 1e-20
    x[2, 128:256] = 0.0
    x[2, 130] = 1e-37   # below 2^-100 after the norm
    x[3] *= 1e15
    x[4, 300] = float("inf")
    x[5, 10] = float("nan")
    norm = gg.RmsNorm(width, eps=1e-6)
    q = torch.zeros(rows, width, device="cuda", dtype=dtypes()[kind])
    s, y = torch.zeros(rows, 5, device="cuda"), torch.zeros(rows, width, device="cuda")
    assert norm.run(x, y=y, q=q, scales=s) == 0
    back = q.float() * s.repeat_interleave(128, 1)
    fine = torch.ones(rows, dtype=torch.bool, device="cuda")
    fine[4:6] = False
    step, small, top = (2.0 ** -4, 2.0 ** -10, 448.0) if kind == "e4m3" else (2.0 ** -3, 2.0 ** -17, 57344.0)
    wide = s.repeat_interleave(128, 1)
    off = (back - y).abs()[fine]
    assert bool((off <= (y.abs() * (step + 1e-4) + wide * small)[fine] + 2.0 ** -100).all())
    assert bool((s[0] == 0).all()) and bool((q[0].float() == 0).all())
    assert float(s[1, 1]) == 0.0 and float(s[2, 1]) == 0.0
    assert bool((q.float()[fine].abs().amax(1)[1:] == top).all())   # the largest of a block is the type's largest number
    # a row with an infinity or a NaN: y of it is not finite there, and the block's scale says so
    assert not bool(torch.isfinite(s[4, 2])) and not bool(torch.isfinite(s[5]).any())


@pytest.mark.parametrize("kind", ["e4m3", "e5m2"])
@pytest.mark.parametrize("width,aligned", [(4096, True), (1000, True), (387, False)])
def test_eight_bits_of_ties(cuda, kind, width, aligned):
    """With rows and weights in BF16 every 8-bit value is the nearest one, ties to even: rstd falls out of y over the block's
    largest, which leaves a quotient 7 a / b times a power of two, a and b whole numbers below 2^16. One that is no tie is at least
    1 / (b c) away from the tie c, of 5 bits, relative to it: 2^-21, and the kernel's quotient is within 2^-23, the 64-bit one's
    rounding to FP32, which restores ties, within 2^-24."""
    import torch
    gen = torch.Generator("cuda").manual_seed(width)
    rows = 300
    x = torch.randn(rows, width + (0 if aligned else 2), device="cuda", generator=gen).bfloat16()[:, :width]
    w = (1 + 0.1 * torch.randn(width, device="cuda", generator=gen)).bfloat16()
    norm = gg.RmsNorm(width, dtype=gg.OutputType.kBF16)
    q = torch.empty(rows, width, device="cuda", dtype=dtypes()[kind])
    s = torch.empty(rows, -(-width // 128), device="cuda")
    assert norm.run(x, w, q=q, scales=s) == 0
    t = torch.nn.functional.pad(x.double() * w.double(), (0, -width % 128)).view(rows, -1, 128)
    top = 448.0 if kind == "e4m3" else 57344.0
    want = (t * top / t.abs().amax(2, keepdim=True)).float().to(dtypes()[kind]).view(rows, -1)[:, :width]
    assert torch.equal(q.float(), want.float())


def test_optional_parts(cuda):
    """Without weight, residual and 8 bits; without the gradients that are not asked for; no rows at all."""
    import torch
    x = torch.randn(9, 300, device="cuda")
    y, rstd = torch.empty_like(x), torch.empty(9, device="cuda")
    norm = gg.RmsNorm(300, eps=0.0)
    assert norm.run(x, y=y, rstd=rstd) == 0
    want = x.double() / x.double().square().mean(1, keepdim=True).sqrt()
    check("y", y, want, want.abs() * 60 * U)
    only = torch.empty(9, device="cuda")
    assert norm.run(x, rstd=only) == 0 and torch.equal(only, rstd)
    gy = torch.randn_like(x)
    gx, full = torch.empty_like(x), torch.empty_like(x)
    gw = torch.empty(300, device="cuda")
    assert norm.backward(x, None, rstd, gy, gx) == 0
    assert norm.backward(x, torch.ones(300, device="cuda"), rstd, gy, full, grad_weight=gw, grad_h=torch.zeros_like(x)) == 0
    assert torch.equal(gx, full)
    h = torch.empty_like(x)
    assert norm.run(x, residual_out=h) == 0 and torch.equal(h, x)  # no residual: x
    q, s = torch.empty(9, 300, device="cuda", dtype=dtypes()["e5m2"]), torch.empty(9, 3, device="cuda")
    assert norm.run(x, q=q, scales=s) == 0
    check("q", q.double() * s.double().repeat_interleave(128, 1)[:, :300], want, want.abs() * (2.0 ** -3 + 1e-4) + 1e-6)
    none = torch.empty(0, 300, device="cuda")
    gw.fill_(3.0)
    assert norm.run(none, y=none) == 0
    assert norm.backward(none, None, torch.empty(0, device="cuda"), none, none, grad_weight=gw) == 0
    assert bool((gw == 0).all())


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("width", [64, 1003, 4096])
def test_in_place(cuda, kind, width):
    import torch
    dt = dtypes()[kind]
    x, r, w = [torch.randn(*s, device="cuda").to(dt) for s in ((33, width), (33, width), (width,))]
    norm = gg.RmsNorm(width, dtype=KINDS[kind])
    y, h, rstd = torch.empty_like(x), torch.empty_like(x), torch.empty(33, device="cuda")
    assert norm.run(x, w, y=y, residual=r, residual_out=h, rstd=rstd) == 0
    a, b = x.clone(), r.clone()
    assert norm.run(a, w, y=a, residual=b, residual_out=b) == 0
    assert torch.equal(a, y) and torch.equal(b, h)
    gy, gh = torch.randn_like(x), torch.randn_like(x)
    gx = torch.empty_like(x)
    assert norm.backward(h, w, rstd, gy, gx, grad_h=gh) == 0
    for over in (0, 1):
        p = [gy.clone(), gh.clone()]
        assert norm.backward(h, w, rstd, p[0], p[over], grad_h=p[1]) == 0
        assert torch.equal(p[over], gx)


def test_same_bits_captured_and_on_a_stream(cuda):
    import torch
    x, r, w, gy = [torch.randn(*s, device="cuda").bfloat16() for s in ((3000, 1024), (3000, 1024), (1024,), (3000, 1024))]
    norm = gg.RmsNorm(1024, dtype=gg.OutputType.kBF16)
    outs = []

    def call(stream):
        o = [torch.zeros_like(x), torch.zeros_like(x), torch.zeros(3000, device="cuda"), torch.zeros_like(x), torch.zeros(1024, device="cuda")]
        outs.append(o)
        assert norm.run(x, w, y=o[0], residual=r, residual_out=o[1], rstd=o[2], stream=stream) == 0
        assert norm.backward(o[1], w, o[2], gy, o[3], grad_weight=o[4], stream=stream) == 0

    call(None)
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        call(torch.cuda.current_stream())
    for t in outs[1]:
        t.fill_(float("nan"))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    del graph


def test_gradient_against_differences(cuda):
    """The change of <c, y> + <d, h> along a direction, by central differences of the definition in 64 bits."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(4)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    x, w, c, d = rnd(6, 517), rnd(517), rnd(6, 517), rnd(6, 517)
    norm = gg.RmsNorm(517, eps=1e-6)
    rstd, gx, gw = torch.empty(6, device="cuda"), torch.empty_like(x), torch.empty_like(w)
    assert norm.run(x, w, rstd=rstd) == 0
    assert norm.backward(x, w, rstd, c, gx, grad_weight=gw, grad_h=d) == 0
    goal = lambda x, w: float((c.double() * reference(x, w, 1e-6)[1]).sum() + (d.double() * x).sum())  # noqa: E731
    vx, vw = rnd(6, 517).double(), rnd(517).double()
    t = 1e-4
    there = (goal(x.double() + t * vx, w.double() + t * vw) - goal(x.double() - t * vx, w.double() - t * vw)) / (2 * t)
    along = float((gx.double() * vx).sum() + (gw.double() * vw).sum())
    # t^2 of third derivatives, each below 100 here over 3000 terms of size 1: 3e-3 at most
    assert abs(there - along) < 3e-3 + 1e-5 * float((gx.double() * vx).abs().sum())


def test_refusals(cuda):
    import torch
    norm = gg.RmsNorm(64)
    x, y = torch.zeros(4, 64, device="cuda"), torch.zeros(4, 64, device="cuda")
    q, s = torch.zeros(4, 64, device="cuda", dtype=torch.float8_e4m3fn), torch.zeros(4, 1, device="cuda")
    for bad in (dict(x=x[:, :32]), dict(x=x.half()), dict(x=x.cpu()), dict(y=y[:3]), dict(y=y.t().reshape(64, 4)), dict(residual=x.double()),
                dict(weight=torch.zeros(63, device="cuda")), dict(weight=torch.zeros(64, device="cuda").half()), dict(q=q), dict(scales=s),
                dict(q=q.view(torch.uint8), scales=s), dict(q=q, scales=torch.zeros(4, 2, device="cuda")), dict(rstd=torch.zeros(5, device="cuda")),
                dict(y=torch.zeros(4, 128, device="cuda")[:, ::2])):
        with pytest.raises(ValueError):
            norm.run(**(dict(x=x, y=y) | bad))
    rstd = torch.zeros(4, device="cuda")
    for bad in (dict(grad_y=x[:3]), dict(grad_x=y.half()), dict(rstd=rstd[:3]), dict(grad_weight=rstd), dict(grad_h=x[:, :8])):
        with pytest.raises(ValueError):
            norm.backward(**(dict(h=x, weight=None, rstd=rstd, grad_y=x, grad_x=y) | bad))
    # what only the C-ABI can be asked
    lib, ptr = capi.load(), x.data_ptr()
    import ctypes
    ok = dict(x=ptr, y=y.data_ptr(), rows=4, ldx=64, ldy=64)
    for bad in (dict(rows=-1), dict(x=None), dict(ldx=63), dict(ldy=63), dict(residual=ptr, ldr=3), dict(residual_out=ptr, ldro=3),
                dict(q=q.data_ptr(), ldq=64, lds=1, q_type=3), dict(q=q.data_ptr(), scales=s.data_ptr(), ldq=63, lds=1, q_type=3),
                dict(q=q.data_ptr(), scales=s.data_ptr(), ldq=64, lds=0, q_type=3), dict(q=q.data_ptr(), scales=s.data_ptr(), ldq=64, lds=1, q_type=2)):
        assert lib.gg_norm_run(norm._h, ctypes.byref(capi.GGNorm(**(ok | bad))), None) == capi.CUDA_ERROR_INVALID_VALUE
    ok = dict(h=ptr, rstd=rstd.data_ptr(), grad_y=ptr, grad_x=y.data_ptr(), rows=4, ldh=64, ldgy=64, ldgx=64)
    for bad in (dict(rows=-1), dict(h=None), dict(rstd=None), dict(grad_y=None), dict(grad_x=None), dict(ldh=1), dict(ldgy=1), dict(ldgx=1),
                dict(grad_h=ptr, ldgh=1)):
        assert lib.gg_norm_backward(norm._h, ctypes.byref(capi.GGNormGradient(**(ok | bad))), None) == capi.CUDA_ERROR_INVALID_VALUE
    norm.close()
    assert norm.run(x, y=y) == capi.CUDA_ERROR_INVALID_DEVICE_POINTER
