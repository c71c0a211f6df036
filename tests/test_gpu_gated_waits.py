"""The limit on waits (GG_WAIT_TIMEOUT_MS) bounds a step of the gated block's kernels, not a tile or a kernel: with one that is many
steps long and much shorter than the kernel, nothing runs out and the results are right. The limit is read when the
library is first used, so each case is a process of its own.

All values are -1, 0 or 1 and there is no activation, so every sum is a whole number below 2^24, exact in FP32 in any order, and a
result is that number rounded to BF16: the comparison is for equality.
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIMIT_MS = 1

HEAD = f"""
import torch
import grouped_gemm_gpu_kernel_b200 as gg
g = torch.Generator(device="cuda").manual_seed(1)
z = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)
sign = lambda *s: z(*s).bernoulli_(0.5, generator=g).mul_(2).sub_(1)
some = lambda *s: sign(*s).mul_(z(*s).bernoulli_(0.5, generator=g))


def equal(got, want):
    assert torch.equal(got, want.float().to(torch.bfloat16)), int((got.double() != want).sum())


def timed(call, plan):
    for _ in range(2):  # the first loads the kernels
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        assert call() == 0
        b.record()
        torch.cuda.synchronize()
        assert plan.status() == 0
    took = a.elapsed_time(b)
    print(round(took, 2), "ms")
    assert took > 3 * {LIMIT_MS}
"""

WEIGHTS = {
    # on pairs of CTAs: the one ragged expert comes last, behind tiles whose stages are all whole
    "ragged_last_pairs": "n, k, counts = 8192, 8192, [4096] * 7 + [4091]",
    # and on single ones
    "ragged_last": "n, k, counts = 24576, 248, [16384] * 7 + [16379]",
    # one tile of many stages
    "one_long_tile_pairs": "n, k, counts = 128, 256, [1 << 20]",
    "one_long_tile": "n, k, counts = 128, 64, [(1 << 20) - 3]",
}


def run(code):
    env = dict(os.environ, GG_WAIT_TIMEOUT_MS=str(LIMIT_MS), PYTHONPATH=REPO)
    p = subprocess.run([sys.executable, "-c", HEAD + code], env=env, cwd=REPO, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stdout + p.stderr
    print(p.stdout)


@pytest.mark.parametrize("name", sorted(WEIGHTS))
def test_gradients_of_the_weights(cuda, name):
    run(WEIGHTS[name] + """
e, rows = len(counts), sum(counts)
x, v, dg, du = some(rows, k), sign(rows, n), z(rows, n), z(rows, n)
w, gwg, gwu = z(k, n), z(e, k, n), z(e, k, n)
plan = gg.GatedPlan(e, n, k, [w.data_ptr()] * e, [w.data_ptr()] * e, n, activation=gg.Activation.kNone)
count = torch.tensor(counts, device="cuda", dtype=torch.int32)
timed(lambda: plan.backward(x, v, v, v, count, dg, du, grad_gate_w=gwg, grad_up_w=gwu), plan)
first = 0
for i, c in enumerate(counts):
    at = slice(n - 64, n)
    for got, d in ((gwg, dg), (gwu, du)):
        equal(got[i][:, at], x[first:first + c].double().t() @ d[first:first + c, at].double())
    first += c
""")


@pytest.mark.parametrize("rows", [16, 520])
def test_forward_of_a_long_outer_size(cuda, rows):
    run(f"n, k, rows = 128, 1 << 20, {rows}" + """
x, wg, wu, h, gate, up = some(rows, k), some(k, n), some(k, n), z(rows, n), z(rows, n), z(rows, n)
plan = gg.GatedPlan(1, n, k, [wg.data_ptr()], [wu.data_ptr()], n, activation=gg.Activation.kNone)
timed(lambda: plan.run(x, None, h, gate=gate, up=up), plan)
for got, w in ((gate, wg), (up, wu)):
    equal(got, sum(x[:, i:i + (1 << 18)].double() @ w[i:i + (1 << 18)].double() for i in range(0, k, 1 << 18)))
""")


@pytest.mark.parametrize("rows", [16, 520])
def test_gradient_of_rows_of_a_long_inner_size(cuda, rows):
    run(f"n, k, rows = 1 << 20, 256, {rows}" + """
wg, wu, gx, gate, up, gh, x = some(k, n), some(k, n), z(rows, k), sign(rows, n), sign(rows, n), sign(rows, n), z(rows, k)
plan = gg.GatedPlan(1, n, k, [wg.data_ptr()], [wu.data_ptr()], n, activation=gg.Activation.kNone)
timed(lambda: plan.backward(x, gate, up, gh, None, gate, up, grad_x=gx), plan)
at = [slice(i, i + (1 << 18)) for i in range(0, n, 1 << 18)]
equal(gx, sum(d[:, a].double() @ w[:, a].double().t() for a in at for d, w in ((gate, wg), (up, wu))))
""")
