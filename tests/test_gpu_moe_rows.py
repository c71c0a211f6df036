"""moe_dispatch, moe_combine and moe_combine_backward against their definitions in 64 bits.

dispatch copies: equal bits. A sum of top_k products in FP32 is off by at most (top_k + 1) 2^-24 times the
sum of its terms' sizes, a dot product over a row of W by (W + 1) 2^-24 times its own; one rounding to the
output's type comes on top.
"""
import numpy as np
import pytest

import grouped_gemm_gpu_kernel_b200 as gg
from grouped_gemm_gpu_kernel_b200 import capi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {"f32": (U, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def positions_for(t, k, g, cuda, unrouted=0.15, spare=5):
    """Places of t * k slots in random packed rows, some nowhere; (positions, packed rows)."""
    import torch
    rows = t * k + spare
    place = torch.randperm(rows, device=cuda, generator=g)[:t * k].view(t, k)
    gone = torch.rand(t, k, device=cuda, generator=g) < unrouted
    if t > 2:
        gone[1] = True  # a token that goes nowhere
    return torch.where(gone, -1, place).int(), rows


def within(got, want, bound):
    err = (got.double().cpu() - want.cpu()).abs()
    assert (err <= bound.cpu() + 1e-300).all(), float((err / (bound.cpu() + 1e-300)).max())


SIZES = [(1, 1, 1), (1, 2, 4096), (4, 8, 2048), (3, 3, 257), (130, 2, 64), (65, 5, 1000), (33, 32, 72), (1000, 4, 8),
         (257, 1, 14336), (18, 9, 1030)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "u8"])
@pytest.mark.parametrize("t,k,w", SIZES)
def test_dispatch_copies_rows(cuda, t, k, w, dtype):
    import torch
    g = torch.Generator(device=cuda).manual_seed(t * w)
    pos, rows = positions_for(t, k, g, cuda)
    if dtype == "u8":
        x = torch.randint(0, 255, (t, w), dtype=torch.uint8, device=cuda, generator=g)
        packed = torch.full((rows, w), 255, dtype=torch.uint8, device=cuda)
    else:
        x = torch.randn(t, w, device=cuda, generator=g).to(torch_type(dtype))
        packed = torch.full((rows, w), 99.0, device=cuda, dtype=x.dtype)
    want = packed.clone()
    ok = pos >= 0
    want[pos[ok].long()] = x[:, None, :].expand(t, k, w)[ok]
    assert gg.moe_dispatch(x, pos, packed) == 0
    assert torch.equal(packed, want)


@pytest.mark.parametrize("pt,ot", [("f32", "f32"), ("f32", "bf16"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"),
                                   ("bf16", "f16"), ("f32", "f16"), ("f16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("t,k,w", SIZES)
def test_combine_and_its_gradient(cuda, t, k, w, pt, ot):
    import torch
    g = torch.Generator(device=cuda).manual_seed(t + w)
    pos, rows = positions_for(t, k, g, cuda)
    y = torch.randn(rows, w, device=cuda, generator=g).to(torch_type(pt))
    wts = torch.randn(t, k, device=cuda, generator=g)
    ok = pos >= 0
    wts[~ok] = float("nan")  # of a slot that went nowhere: not read
    used = torch.zeros(rows, dtype=torch.bool, device=cuda)
    used[pos[ok].long()] = True
    y[~used] = float("nan")  # rows that nobody names: not read
    wz = torch.where(ok, wts, 0.0).double()
    yg = torch.where(ok[:, :, None], y[pos.clamp(min=0).long()].double(), 0.0)
    rel, least = ROUND[ot]
    for weights in (wts, None):
        out = torch.full((t, w), float("nan"), device=cuda, dtype=torch_type(ot))
        assert gg.moe_combine(y, pos, out, weights) == 0
        terms = yg * (wz[:, :, None] if weights is not None else 1.0)
        size = (k + 1) * U * terms.abs().sum(1)
        within(out, terms.sum(1), size * (1 + rel) + rel * terms.sum(1).abs() + least)

    go = torch.randn(t, w, device=cuda, generator=g).to(torch_type(ot))
    gp = torch.full((rows, w), 99.0, device=cuda, dtype=y.dtype)
    gw = torch.full((t, k), float("nan"), device=cuda)
    assert gg.moe_combine_backward(go, y, pos, wts, gp, gw) == 0
    dots = go.double()[:, None, :] * yg
    within(gw, dots.sum(2), (w + 1) * U * dots.abs().sum(2))
    assert (gw[~ok] == 0).all()
    want = torch.full((rows, w), 99.0, device=cuda, dtype=torch.float64)
    want[pos[ok].long()] = (wz[:, :, None] * go.double()[:, None, :])[ok]
    rel, least = ROUND[pt]
    within(gp, want, (rel + U) * (1 + U) * want.abs() * used[:, None] + least)
    # written over packed itself
    again = torch.full((t, k), float("nan"), device=cuda)
    assert gg.moe_combine_backward(go, y, pos, wts, y, again) == 0
    assert torch.equal(again, gw) and torch.equal(y[used], gp[used])


def test_gradient_matches_differences(cuda):
    """<go, combine(y, w)> is linear in y and in w: its change over any step is the gradient's product."""
    import torch
    t, k, w = 40, 3, 130
    g = torch.Generator(device=cuda).manual_seed(5)
    pos, rows = positions_for(t, k, g, cuda)
    y, wts = torch.randn(rows, w, device=cuda, generator=g), torch.randn(t, k, device=cuda, generator=g)
    go = torch.randn(t, w, device=cuda, generator=g)
    gp, gw = torch.zeros(rows, w, device=cuda), torch.zeros(t, k, device=cuda)
    assert gg.moe_combine_backward(go, y, pos, wts, gp, gw) == 0

    def goal(yy, ww):
        out = torch.zeros(t, w, device=cuda)
        assert gg.moe_combine(yy, pos, out, ww) == 0
        return float((out.double() * go.double()).sum())

    dy, dw = torch.randn(rows, w, device=cuda, generator=g), torch.randn(t, k, device=cuda, generator=g)
    # 5200 products of numbers of size 1 to 4, each off by some 2^-22: below 1e-3 in all
    assert abs(goal(y + dy, wts) - goal(y, wts) - float((gp.double() * dy.double()).sum())) < 2e-2
    assert abs(goal(y, wts + dw) - goal(y, wts) - float((gw.double() * dw.double()).sum())) < 2e-2
    # and of dispatch: <d packed, dispatch(x)>
    x = torch.randn(t, w, device=cuda, generator=g)
    packed, gx = torch.zeros(rows, w, device=cuda), torch.zeros(t, w, device=cuda)
    assert gg.moe_dispatch(x, pos, packed) == 0
    gd = torch.randn(rows, w, device=cuda, generator=g)
    assert gg.moe_combine(gd, pos, gx) == 0
    assert abs(float((packed.double() * gd.double()).sum()) - float((x.double() * gx.double()).sum())) < 2e-2


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("first,pitch", [(0, 520), (1, 515), (4, 516), (2, 514)])
def test_pitches_and_misaligned_rows(cuda, dtype, first, pitch):
    import torch
    t, k, w = 37, 3, 512
    g = torch.Generator(device=cuda).manual_seed(first)
    pos, rows = positions_for(t, k, g, cuda)
    dt = torch_type(dtype)

    def wide(n, fill=float("nan")):
        return torch.full((n, pitch + first), fill, device=cuda, dtype=dt)[:, first:first + w]

    x, go = torch.randn(t, w, device=cuda, generator=g).to(dt), torch.randn(t, w, device=cuda, generator=g).to(dt)
    wts = torch.randn(t, k, device=cuda, generator=g)

    def passes(view):
        xs, packed, out, gos, gp = view(t), view(rows, 0.0), view(t), view(t), view(rows, 0.0)
        xs.copy_(x), gos.copy_(go)
        gw = torch.zeros(t, k, device=cuda)
        assert gg.moe_dispatch(xs, pos, packed) == 0
        assert gg.moe_combine(packed, pos, out, wts) == 0
        assert gg.moe_combine_backward(gos, packed, pos, wts, gp, gw) == 0
        return packed.clone(), out.clone(), gp.clone(), gw

    got = passes(wide)
    want = passes(lambda n, fill=float("nan"): torch.full((n, w), fill, device=cuda, dtype=dt))
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a, b)
    # the dot products may be summed in another order on another load width
    size = (go.double()[:, None, :] * want[0][pos.clamp(min=0).long()].double()).abs().sum(2)
    within(got[3], want[3].double(), 2 * (w + 1) * U * size)


def test_positions_out_of_range_go_nowhere(cuda):
    import torch
    pos = torch.tensor([[0, 9], [-5, 1], [2 ** 31 - 1, -2 ** 31]], dtype=torch.int32, device=cuda)
    x, packed = torch.ones(3, 64, device=cuda), torch.zeros(4, 64, device=cuda)[:2]
    assert gg.moe_dispatch(x, pos, packed) == 0
    assert (packed == 1).all()
    out, gw = torch.zeros(3, 64, device=cuda), torch.full((3, 2), 9.0, device=cuda)
    assert gg.moe_combine(packed, pos, out) == 0
    assert out[:, 0].tolist() == [1.0, 1.0, 0.0]
    assert gg.moe_combine_backward(x, packed, pos, torch.ones(3, 2, device=cuda), packed.clone(), gw) == 0
    assert gw.tolist() == [[64.0, 0.0], [0.0, 64.0], [0.0, 0.0]]


def test_rows_past_two_billion_elements(cuda):
    """Packed rows whose element offsets pass 32 bits (4.3 GB)."""
    import torch
    w, rows = 4096, (1 << 19) + 16
    packed = torch.zeros(rows, w, device=cuda, dtype=torch.bfloat16)
    x = torch.randn(2, w, device=cuda).bfloat16()
    pos = torch.tensor([[rows - 1, 3], [rows - 7, (1 << 19) + 1]], dtype=torch.int32, device=cuda)
    assert gg.moe_dispatch(x, pos, packed) == 0
    assert torch.equal(packed[rows - 1], x[0]) and torch.equal(packed[3], x[0]) and torch.equal(packed[rows - 7], x[1])
    out = torch.zeros_like(x)
    assert gg.moe_combine(packed, pos, out) == 0
    assert torch.equal(out, (x.float() * 2).bfloat16())
    gw = torch.zeros(2, 2, device=cuda)
    assert gg.moe_combine_backward(x, packed, pos, torch.full((2, 2), 0.5, device=cuda), packed, gw) == 0
    assert torch.equal(packed[rows - 7], (x[1].float() * 0.5).bfloat16())
    del packed


def test_empty_calls_and_refusals(cuda):
    import torch
    f = lambda *s: torch.zeros(*s, device=cuda)  # noqa: E731
    i = lambda *s: torch.zeros(*s, device=cuda, dtype=torch.int32)  # noqa: E731
    assert gg.moe_dispatch(f(0, 8), i(0, 2), f(4, 8)) == 0
    assert gg.moe_combine(f(4, 8), i(0, 2), f(0, 8)) == 0
    out = torch.full((3, 8), 7.0, device=cuda)
    assert gg.moe_combine(f(0, 8), i(3, 2), out) == 0  # no packed rows: every token sums nothing
    assert (out == 0).all()
    gw = torch.full((3, 2), 7.0, device=cuda)
    assert gg.moe_combine_backward(f(3, 8), f(0, 8), i(3, 2), f(3, 2), f(0, 8), gw) == 0
    assert (gw == 0).all()
    with pytest.raises(ValueError):
        gg.moe_dispatch(f(3, 8), i(3, 2), f(4, 9))
    with pytest.raises(ValueError):
        gg.moe_dispatch(f(3, 8), i(3, 2).long(), f(4, 8))
    with pytest.raises(ValueError):
        gg.moe_dispatch(f(3, 8), i(4, 2), f(4, 8))
    with pytest.raises(ValueError):
        gg.moe_dispatch(f(3, 8), i(3, 2), f(4, 8).half())
    with pytest.raises(ValueError):
        gg.moe_dispatch(f(8, 3).t(), i(3, 2), f(4, 8))
    with pytest.raises(ValueError):
        gg.moe_combine(f(4, 8).double(), i(3, 2), f(3, 8))
    with pytest.raises(ValueError):
        gg.moe_combine(f(4, 8), i(3, 2), f(3, 8), f(3, 3))
    with pytest.raises(ValueError):
        gg.moe_combine_backward(f(3, 8), f(4, 8), i(3, 2), f(3, 2), f(4, 8).half(), f(3, 2))
    assert gg.moe_dispatch(f(3, 8).double(), i(3, 2), f(4, 8).double()) == capi.CUDA_ERROR_INVALID_VALUE  # 8-byte elements
