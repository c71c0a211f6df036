"""The gated 8-bit product's 8-bit results are the nearest ones to their quotients, ties to even.

Rows and weights are whole numbers from -3 to 3 and all scales powers of two, so that gate, up and their product v are exact in FP32 on
any way. A quotient 448 v / top (or 57344 v / top) is 7 v / top times a power of two; from a tie c between two 8-bit values, which has
5 bits at most, it is 0 or at least 1 / (7 v) or 1 / (c top) away, relative to it: 2^-23 with v and top below 2^17, 2^-22
where the bound below is reached. An FP32 number nearest to it, or off by 2^-44 more, is on the same side, since its rounding is 2^-24.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg

pytestmark = pytest.mark.gpu


def nearest(x, kind):
    """x (64 bits, within the type) rounded to the type's values, ties to even, by the numbers' definition."""
    import torch
    bits, low = (3, -6) if kind == "e4m3" else (2, -14)
    exponent = torch.frexp(torch.where(x == 0, torch.ones_like(x), x))[1] - 1
    step = torch.ldexp(torch.ones_like(x), exponent.clamp(min=low) - bits)
    return torch.round(x / step) * step


@pytest.mark.parametrize("out,top", [("e4m3", 448.0), ("e5m2", 57344.0)])
@pytest.mark.parametrize("n,k", [(256, 48), (300, 130)])
def test_nearest(cuda, out, top, n, k):
    import torch
    g = torch.Generator(device=cuda).manual_seed(n)
    counts, f8 = [700, 0, 1301], torch.float8_e4m3fn
    rows, e, nb, kb = sum(counts), len(counts), -(-n // 128), -(-k // 128)
    whole = lambda *s: torch.randint(-3, 4, s, device=cuda, generator=g).float()  # noqa: E731
    power = lambda *s: torch.ldexp(torch.ones(s, device=cuda), torch.randint(-3, 4, s, device=cuda, generator=g))  # noqa: E731
    a = torch.zeros(rows, -(-k // 16) * 16, device=cuda, dtype=torch.uint8).view(f8)[:, :k]
    a.copy_(whole(rows, k).to(f8))
    sa = power(rows, 1).expand(rows, kb).contiguous()
    weights, scales = [], []
    for _ in range(2):
        w = torch.zeros(e, n, -(-k // 16) * 16, device=cuda, dtype=torch.uint8).view(f8)[..., :k]
        w.copy_(whole(e, n, k).to(f8))
        weights.append(w), scales.append(power(e, nb, 1).expand(e, nb, kb).contiguous())
    each = lambda t: [x.data_ptr() for x in t]  # noqa: E731
    dt = torch.float8_e4m3fn if out == "e4m3" else torch.float8_e5m2
    d, sd = torch.zeros(rows, n, device=cuda, dtype=torch.uint8).view(dt), torch.zeros(rows, nb, device=cuda)
    plan = gg.F8Plan(e, n, k, each(weights[0]), weights[0].stride(1), each(scales[0]), up_ptrs=each(weights[1]), up_scale_ptrs=each(scales[1]),
                     output_type=gg.OutputType.kE4M3 if out == "e4m3" else gg.OutputType.kE5M2)
    assert plan.run(a, sa, torch.tensor(counts, device=cuda, dtype=torch.int32), d, d_scales=sd) == 0
    torch.cuda.synchronize()
    assert plan.status() == 0
    first = 0
    for x, count in enumerate(counts):
        at = slice(first, first + count)
        first += count
        if not count:
            continue
        v = (a[at].double() @ weights[0][x].double().t()) * (a[at].double() @ weights[1][x].double().t())
        assert float(v.abs().max()) < 2 ** 17
        blocks = torch.nn.functional.pad(v, (0, nb * 128 - n)).view(count, nb, 128)
        most = blocks.abs().amax(2, keepdim=True)
        want = nearest(torch.where(most > 0, blocks * top / most.clamp(min=1), torch.zeros_like(blocks)), out).view(count, -1)[:, :n]
        got = d[at].double()
        assert torch.equal(got, want), f"{int((got != want).sum())} of {got.numel()} are not the nearest"
        factor = sa[at, :1].double() ** 2 * scales[0][x, :, 0].double() * scales[1][x, :, 0].double()
        assert torch.equal(sd[at].double(), (most[..., 0] * factor / top).float().double())
