"""Calls that follow a two-part executor run on one stream, with nothing between them.

An executor with tile classes makes two launches that overlap. The kernels of the mixture-of-experts operators wait on
the GPU for the launch just before them, which is the second; it may be through long before the first. So the first
part is one tile of a long inner dimension here and the second a short one: what follows has to find D
written, and may overwrite A. Results are compared bit by bit with runs that are synchronised in between.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg

pytestmark = pytest.mark.gpu
CONFIGS = [gg.KernelConfig(128, 256, 64, tile_classes=gg.TileClasses.kSmallOnCudaCores),
           gg.KernelConfig(128, 64, 64, tile_classes=gg.TileClasses.kSmallOnCudaCores),
           gg.KernelConfig(256, 256, 64, tile_classes=gg.TileClasses.kPairBlocks),
           gg.KernelConfig(256, 128, 64, tile_classes=gg.TileClasses.kPairBlocks)]


class TwoParts:
    """A 256 x 256 problem of a long inner dimension (the first launch) and a short one (the second)."""

    def __init__(self, cuda, cfg, k=32768):
        import torch
        g = torch.Generator(device=cuda).manual_seed(cfg.cta_n)
        half = lambda *s: torch.randn(*s, device=cuda, generator=g).half()  # noqa: E731
        self.a, self.b, self.d = half(256, k), half(k, 256), torch.zeros(256, 256, device=cuda)
        m = 40 if cfg.tile_classes == gg.TileClasses.kSmallOnCudaCores else 100
        self.small = [half(m, 64), half(64, 64), torch.zeros(m, 64, device=cuda)]
        problems = [gg.ProblemDesc(256, 256, k, self.a.data_ptr(), self.b.data_ptr(), None, self.d.data_ptr(), k, 256, 256, 256),
                    gg.ProblemDesc(m, 64, 64, *(t.data_ptr() for t in self.small[:2]), None, self.small[2].data_ptr(),
                                   64, 64, 64, 64)]
        self.ex = gg.GroupedGemmExecutor()
        assert self.ex.build(gg.prepare_problem_set(problems, cfg, gg.SortMode.kByTiles), cfg) == 0
        assert self.ex.launches() == 2
        assert self.ex.run() == 0
        torch.cuda.synchronize()
        assert self.ex.status() == 0
        self.want = self.d.clone()
        assert torch.isfinite(self.want).all()


@pytest.mark.parametrize("cfg", CONFIGS, ids=lambda c: f"{c.cta_m}x{c.cta_n}-{c.tile_classes}")
def test_combine_reads_all_of_d(cuda, cfg):
    import torch
    p = TwoParts(cuda, cfg)
    places = torch.arange(256, dtype=torch.int32, device=cuda)[:, None].contiguous()
    outs = [torch.zeros_like(p.d) for _ in range(20)]
    for out in outs:
        p.d.fill_(float("nan"))
        assert p.ex.run() == 0
        assert gg.moe_combine(p.d, places, out) == 0
    assert all(torch.equal(out, p.want) for out in outs)
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream(cuda)
    out = torch.zeros_like(p.d)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        p.d.fill_(float("nan"))
        assert p.ex.run(torch.cuda.current_stream()) == 0
        assert gg.moe_combine(p.d, places, out, stream=torch.cuda.current_stream()) == 0
    for _ in range(20):
        out.zero_()
        graph.replay()
        assert torch.equal(out, p.want)
    del graph


@pytest.mark.parametrize("cfg", CONFIGS, ids=lambda c: f"{c.cta_m}x{c.cta_n}-{c.tile_classes}")
def test_dispatch_overwrites_a_behind_the_run(cuda, cfg):
    import torch
    p = TwoParts(cuda, cfg)
    places = torch.arange(256, dtype=torch.int32, device=cuda)[:, None].contiguous()
    kept, other = p.a.clone(), torch.zeros_like(p.a)
    for _ in range(20):
        assert gg.moe_dispatch(kept, places, p.a) == 0
        assert p.ex.run() == 0
        assert gg.moe_dispatch(other, places, p.a) == 0
        assert torch.equal(p.d, p.want)
        p.d.zero_()
