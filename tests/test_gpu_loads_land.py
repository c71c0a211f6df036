"""A block of the 8-bit product or the gated block ends once its loads have landed, and no later: the wait at its end is limited to
100 ms a stage, so that a stage which it took for one under way, or a round of a stage that it took for another, would show as a run of
100 ms and more. All numbers of stages up to several rounds, on single CTAs and pairs, with and without rows, and many tiles.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg

pytestmark = pytest.mark.gpu
MOST_MS = 50.0


def took(call):
    import torch
    assert call() == 0  # what a first call sets up
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    a.record()
    assert call() == 0
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b)


@pytest.mark.parametrize("rows,n", [(1, 64), (40, 600), (300, 20000), (0, 300)])
@pytest.mark.parametrize("gated", [False, True])
def test_8bit_product(cuda, rows, n, gated):
    import torch
    zero = lambda *s: torch.zeros(*s, device=cuda, dtype=torch.uint8).view(torch.float8_e4m3fn)  # noqa: E731
    counts = torch.tensor([rows, 0], device=cuda, dtype=torch.int32)
    for blocks in list(range(1, 20)) + [31, 32, 33]:
        k = 128 * blocks
        a, b, s = zero(max(rows, 1), k), zero(n, k), torch.ones(-(-n // 128), blocks, device=cuda)
        sa, d = torch.ones(max(rows, 1), blocks, device=cuda), torch.zeros(max(rows, 1), n, device=cuda)
        up = dict(up_ptrs=[b.data_ptr()] * 2, up_scale_ptrs=[s.data_ptr()] * 2) if gated else {}
        plan = gg.F8Plan(2, n, k, [b.data_ptr()] * 2, k, [s.data_ptr()] * 2, output_type=gg.OutputType.kF32, **up)
        assert took(lambda: plan.run(a, sa, counts, d)) < MOST_MS, blocks
        assert plan.status() == 0


@pytest.mark.parametrize("rows,n", [(1, 64), (40, 600), (1024, 72), (1100, 8000), (0, 304)])
def test_gated_block(cuda, rows, n):
    """The outer size is the forward's depth, the rows are the weights' gradients'; 512 rows an expert and more go to pairs."""
    import torch
    z = lambda *s: torch.zeros(*s, device=cuda, dtype=torch.bfloat16)  # noqa: E731
    for k in [8, *range(64, 64 * 15, 64), 64 * 24]:
        for more in (0, 5):
            total = max(1, 2 * rows + more)
            counts = torch.tensor([rows, rows + more], device=cuda, dtype=torch.int32)
            x, w, h, gate, up, gh = z(total, k), z(k, n), z(total, n), z(total, n), z(total, n), z(total, n)
            dg, du, dx, dw = z(total, n), z(total, n), z(total, k), z(2, k, n)
            plan = gg.GatedPlan(2, n, k, [w.data_ptr()] * 2, [w.data_ptr()] * 2, n)
            assert took(lambda: plan.run(x, counts, h, gate=gate, up=up)) < MOST_MS, k
            assert took(lambda: plan.backward(x, gate, up, gh, counts, dg, du, grad_x=dx, grad_gate_w=dw, grad_up_w=dw.clone())) < MOST_MS, k
            assert plan.status() == 0
