"""The 8-bit product's tile width for a few rows on many experts, as the launch of a captured run shows it: the blocks are the tiles, up to
the SMs.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg

pytestmark = pytest.mark.gpu


def blocks_of(call):
    """Blocks of the one kernel that `call` launches, captured and not run."""
    import torch
    driver = pytest.importorskip("cuda.bindings.driver")
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        assert call(torch.cuda.current_stream()) == 0
    raw = driver.CUgraph(graph.raw_cuda_graph())
    error, _, count = driver.cuGraphGetNodes(raw)
    assert int(error) == 0 and count == 1
    error, nodes, _ = driver.cuGraphGetNodes(raw, count)
    error, params = driver.cuGraphKernelNodeGetParams(nodes[0])
    assert int(error) == 0
    blocks = params.gridDimX
    del graph
    return blocks


@pytest.mark.parametrize("n,k,gated", [(4096, 14336, False), (2048, 7168, True), (7168, 2048, False), (1024, 4096, True)])
def test_few_rows_take_the_tiles_that_there_can_be(cuda, n, k, gated):
    """Rows are on as many experts as there are rows, at most: the experts without any change nothing."""
    import torch
    w = torch.zeros(n, k, device=cuda, dtype=torch.uint8)
    s, d = torch.ones(-(-n // 128), -(-k // 128), device=cuda), torch.zeros(8, n, device=cuda, dtype=torch.bfloat16)
    a, sa = torch.zeros(8, k, device=cuda, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(8, -(-k // 128), device=cuda)

    def blocks(experts, rows):
        up = dict(up_ptrs=[w.data_ptr()] * experts, up_scale_ptrs=[s.data_ptr()] * experts) if gated else {}
        plan = gg.F8Plan(experts, n, k, [w.data_ptr()] * experts, k, [s.data_ptr()] * experts, **up)
        counts = torch.zeros(experts, device=cuda, dtype=torch.int32)
        return blocks_of(lambda stream: plan.run(a[:rows], sa[:rows], counts, d[:rows], stream=stream))

    for rows in range(1, 9):
        few = blocks(rows, rows)
        assert [blocks(experts, rows) for experts in (16, 32, 64, 128)] == [few] * 4, rows
