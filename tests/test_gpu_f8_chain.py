"""Two 8-bit products behind one another, the second on the rows and scales that the first writes, on new rows in the same buffers each
time: the bits of the same calls with a synchronisation between them, whichever kernel is set up while another still runs.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts,hidden,inner", [([3, 0, 5, 1], 256, 384), ([150, 0, 260, 1], 640, 1000 // 16 * 16), ([700, 900, 0, 448], 1024, 512)])
def test_chain(cuda, counts, hidden, inner):
    import torch
    f8, g, e, rows, steps = torch.float8_e4m3fn, torch.Generator(device=cuda).manual_seed(3), len(counts), sum(counts), 24
    blocks = lambda n: -(-n // 128)  # noqa: E731
    rnd = lambda *s: (torch.randn(*s, device=cuda, generator=g).clamp(-4, 4) * 100).to(f8)  # noqa: E731
    scale = lambda *s: (0.5 + torch.rand(*s, device=cuda, generator=g)) * 1e-3  # noqa: E731
    wg, wu, wd = rnd(e, inner, hidden), rnd(e, inner, hidden), rnd(e, hidden, inner)
    sg, su, sd = scale(e, blocks(inner), blocks(hidden)), scale(e, blocks(inner), blocks(hidden)), scale(e, blocks(hidden), blocks(inner))
    each = lambda t: [x.data_ptr() for x in t]  # noqa: E731
    first = gg.F8Plan(e, inner, hidden, each(wg), hidden, each(sg), up_ptrs=each(wu), up_scale_ptrs=each(su), output_type=gg.OutputType.kE4M3,
                      activation=gg.Activation.kSiLU)
    second = gg.F8Plan(e, hidden, inner, each(wd), inner, each(sd), output_type=gg.OutputType.kF32)
    count = torch.tensor(counts, device=cuda, dtype=torch.int32)
    inputs = [(rnd(rows, hidden), scale(rows, blocks(hidden)) * 2.0 ** (i % 7)) for i in range(steps)]
    mid, smid = torch.zeros(rows, inner, device=cuda, dtype=torch.uint8).view(f8), torch.zeros(rows, blocks(inner), device=cuda)
    outs = [[torch.zeros(rows, hidden, device=cuda) for _ in range(steps)] for _ in range(2)]
    for wait, out in zip((True, False), outs):
        torch.cuda.synchronize()
        for (a, sa), d in zip(inputs, out):
            assert first.run(a, sa, count, mid, d_scales=smid) == 0
            if wait:
                torch.cuda.synchronize()
            assert second.run(mid, smid, count, d) == 0
            if wait:
                torch.cuda.synchronize()
    torch.cuda.synchronize()
    assert first.status() == 0 and second.status() == 0
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(torch.isfinite(a).all()) and bool((a != 0).any())
