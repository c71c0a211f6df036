"""Activations and their slopes of numbers far out, to the ends of BF16, FP16 and FP32, in the gated block and the 8-bit product.

Tolerances. A value is within NEAR = 4e-5 of it up to where exp(-z) is exp(80) (test_gpu_gated.py has the arithmetic). Past that
SiLU and its slope are below 81 exp(-80) = 1.5e-33 in magnitude, GELU (z = -80 at x = -9.6, z' = 21.4 there) and its slope below
9.6 * 22 exp(-80) = 3.9e-33, and both fall from there on: what the kernels give there is 0 or as small, so FAR = 1e-32 bounds the difference,
however large the number is. A result is rounded once, by half a step or half the smallest number.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg

pytestmark = pytest.mark.gpu
NEAR = 4e-5
FAR = 1e-32
ACTS = {"relu": gg.Activation.kReLU, "gelu": gg.Activation.kGELU, "silu": gg.Activation.kSiLU}
PLACES = [0.0, 1e-30, 1.0, 5.0, 9.0, 9.5, 9.75, 10.0, 17.0, 40.0, 79.0, 80.0, 84.0, 87.0, 88.0, 89.0, 100.0, 1000.0, 65504.0, 1e11, 1e13, 4e19, 6e19, 1e30, 3e38]


def both(x, act):
    """act(x) and act'(x) in 64 bits."""
    import torch
    if act == "relu":
        return x.clamp(min=0), (x > 0).double()
    c = 1.5957691216057308
    z, dz = (x, 1.0) if act == "silu" else (c * (x + 0.044715 * x ** 3), c * (1 + 3 * 0.044715 * x ** 2))
    s, other = torch.sigmoid(z), torch.sigmoid(-z)
    return x * s, s + x * s * other * dz


def near(name, got, want):
    import torch
    info = torch.finfo(got.dtype)
    half = 0.0 if got.dtype == torch.float32 else info.eps / 2
    off = (got.double() - want).abs()
    bound = want.abs() * (NEAR * 1.13 + half) * 1.01 + FAR + info.tiny * info.eps
    assert bool((off <= bound).all()), (name, got[~(off <= bound)][:4].tolist(), want[~(off <= bound)][:4].tolist())


def places(cuda, dtype):
    import torch
    x = torch.tensor(PLACES + [-p for p in PLACES], device=cuda, dtype=torch.float64)
    return x[x.abs() <= torch.finfo(dtype).max].to(dtype)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("act", sorted(ACTS))
def test_gated_block(cuda, act, kind):
    """Rows (gate, 1) against gate weights (1, 0) and up weights (0, 1): the gates are the rows' first values, up is 1."""
    import torch
    dt = {"f16": torch.float16, "bf16": torch.bfloat16}[kind]
    gates, n = places(cuda, dt), 40
    rows = gates.numel()
    z = lambda *s: torch.zeros(*s, device=cuda, dtype=dt)  # noqa: E731
    x, wg, wu = z(rows, 8), z(8, n), z(8, n)
    x[:, 0], x[:, 1], wg[0], wu[1] = gates, 1.0, 1.0, 1.0
    plan = gg.GatedPlan(1, n, 2, [wg.data_ptr()], [wu.data_ptr()], n, activation=ACTS[act],
                        input_type=gg.InputType.kF16 if kind == "f16" else gg.InputType.kBF16)
    h, gate, up, dg, du = [z(rows, n) for _ in range(5)]
    assert plan.run(x[:, :2], None, h, gate=gate, up=up) == 0
    wide = gates.double()[:, None].expand(rows, n)
    assert torch.equal(gate.double(), wide) and bool((up == 1).all())
    value, slope = both(wide, act)
    near("h", h, value)
    assert plan.backward(x[:, :2], gate, up, torch.ones_like(h), None, dg, du) == 0
    near("grad_gate", dg, slope)
    near("grad_up", du, value)
    # and value by value, where rows are not aligned
    odd = [torch.empty(rows * n + 1, device=cuda, dtype=dt)[1:].view(rows, n).copy_(t) for t in (gate, up, torch.ones_like(h))]
    dg2, du2 = torch.full_like(dg, float("nan")), torch.full_like(du, float("nan"))
    assert plan.backward(x[:, :2], *odd, None, dg2, du2) == 0
    assert torch.equal(dg2, dg) and torch.equal(du2, du)


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("act", sorted(ACTS))
def test_8bit_product(cuda, act, out):
    """Products of zeros and a bias: act(bias)."""
    import torch
    dt = {"f32": torch.float32, "bf16": torch.bfloat16}[out]
    bias = places(cuda, torch.float32).float()
    n, rows = bias.numel(), 5
    zero = lambda *s: torch.zeros(*s, device=cuda, dtype=torch.uint8).view(torch.float8_e4m3fn)  # noqa: E731
    a, b, s, d = zero(rows, 16), zero(n, 16), torch.ones(rows, 1, device=cuda), torch.empty(rows, n, device=cuda, dtype=dt)
    plan = gg.F8Plan(1, n, 16, [b.data_ptr()], 16, [s.data_ptr()], bias_ptrs=[bias.data_ptr()], activation=ACTS[act],
                     output_type=gg.OutputType.kF32 if out == "f32" else gg.OutputType.kBF16)
    assert plan.run(a, s, None, d) == 0
    near("d", d, both(bias.double(), act)[0][None].expand(rows, n))
