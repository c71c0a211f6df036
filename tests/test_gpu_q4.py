"""Experts in 4-bit weights (gg_q4_plan_*) against the product with the unpacked weights in 64 bits.

q - zero is exact and so is its product with an activation. What is rounded is the sums: with R the
root of the sum of the terms' squares of one output, partial sums stay below 4 R and there are
k / 8 + groups + 8 of them in sequence, each off by at most 2^-23 relative:
bound = 4 (k / 8 + groups + 8) 2^-23 R, plus one rounding to the output's type. GELU's slope is
below 1.2; its own arithmetic adds 2^-20 relative.
"""
import math

import pytest

import grouped_gemm_gpu_kernel_b200 as gg
from grouped_gemm_gpu_kernel_b200 import capi

pytestmark = pytest.mark.gpu

ROUND = {"f32": (2.0 ** -24, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}
OUT = {"f32": gg.OutputType.kF32, "f16": gg.OutputType.kF16, "bf16": gg.OutputType.kBF16}
IN = {"f16": gg.InputType.kF16, "bf16": gg.InputType.kBF16}


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Weights:
    def __init__(self, cuda, experts, n, k, group, dtype, zeros=False, bias=False, seed=0, pad=0):
        import torch
        g = torch.Generator(device=cuda).manual_seed(seed)
        self.experts, self.n, self.k, self.group, self.dtype, self.g = experts, n, k, group, dtype, g
        self.groups = -(-k // group)
        # the pad bytes, and the spare half byte of an odd k, hold junk
        self.q = torch.randint(0, 256, (experts, n, (k + 1) // 2 + pad), dtype=torch.uint8, device=cuda, generator=g)
        self.scales = ((0.5 + torch.rand(experts, n, self.groups, device=cuda, generator=g)) / math.sqrt(21.0 * k)).to(
            torch_type(dtype))
        self.zeros = torch.randint(0, 16, (experts, n, self.groups), dtype=torch.uint8, device=cuda,
                                   generator=g) if zeros else None
        self.bias = torch.randn(experts, n, device=cuda, generator=g) if bias else None

    def plan(self, out="f32", act=gg.Activation.kNone, bias_ptrs=None, stream=None):
        each = lambda t: None if t is None else [x.data_ptr() for x in t]  # noqa: E731
        return gg.Q4Plan(self.experts, self.n, self.k, self.group, each(self.q), self.q.shape[2], each(self.scales),
                         each(self.zeros), bias_ptrs or each(self.bias), IN[self.dtype], OUT[out], act, stream=stream)

    def dense(self, e):
        import torch
        q = torch.stack([self.q[e] & 15, self.q[e] >> 4], 2).flatten(1)[:, :self.k].double()
        of = torch.arange(self.k, device=q.device) // self.group
        zero = self.zeros[e].double()[:, of] if self.zeros is not None else 8.0
        return (q - zero) * self.scales[e].double()[:, of]


def check(wt, a, rows, d, out, act=gg.Activation.kNone, row_tokens=None, bias=None):
    import torch
    at = 0
    rel, least = ROUND[out]
    for e, r in enumerate(rows):
        if r == 0:
            continue
        x = (a[at:at + r] if row_tokens is None else a[row_tokens[at:at + r].long()]).double()
        w = wt.dense(e)
        want = x @ w.t()
        tol = 4 * (wt.k / 8 + wt.groups + 8) * 2.0 ** -23 * torch.sqrt((x * x) @ (w * w).t())
        b = bias[e] if bias is not None else (wt.bias[e] if wt.bias is not None else None)
        if b is not None:
            want = want + b.double()
            tol = tol + 2.0 ** -23 * (want.abs() + b.double().abs())
        if act == gg.Activation.kReLU:
            want = want.clamp(min=0)
        elif act == gg.Activation.kGELU:
            pre = want
            want = pre * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (pre + 0.044715 * pre ** 3))
            tol = 1.2 * tol + 2.0 ** -20 * pre.abs()
        tol = tol * (1 + rel) + rel * want.abs() + least
        err = (d[at:at + r].double() - want).abs()
        assert (err <= tol).all(), (e, float((err / tol).max()))
        at += r


def rows_tensor(rows, cuda):
    import torch
    return torch.tensor(rows, dtype=torch.int32, device=cuda)


SHAPES = [(1, 1, 32), (16, 128, 32), (17, 129, 64), (64, 256, 128), (100, 31, 128), (385, 257, 32), (48, 4096, 64),
          (1000, 520, 128), (33, 1000, 256), (8, 2048, 512), (256, 14336, 128)]


@pytest.mark.parametrize("zeros", [False, True], ids=["sym", "zeros"])
@pytest.mark.parametrize("dtype,out", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("n,k,group", SHAPES)
def test_matches_the_unpacked_product(cuda, n, k, group, dtype, out, zeros):
    import torch
    rows = [2, 0, 9, 1, 0, 23]
    wt = Weights(cuda, len(rows), n, k, group, dtype, zeros, seed=n + k, pad=n % 3)
    a = torch.randn(sum(rows), k, device=cuda, generator=wt.g).to(torch_type(dtype))
    d = torch.full((sum(rows) + 3, n), 55.0, device=cuda, dtype=torch_type(out))
    plan = wt.plan(out)
    assert plan.run(a, rows_tensor(rows, cuda), d) == 0
    assert plan.status() == 0
    check(wt, a, rows, d, out)
    assert (d[sum(rows):] == 55.0).all()  # rows past the counts' sum are not written
    plan.close()


@pytest.mark.parametrize("count", [1, 2, 7, 8, 9, 16, 17, 31, 32, 33, 40, 63, 64, 65, 200])
def test_row_counts_of_one_matrix(cuda, count):
    """One expert without counts: a matrix-vector product, then more rows."""
    import torch
    wt = Weights(cuda, 1, 144, 640, 64, "f16", True, bias=True, seed=count)
    a = torch.randn(count, 640, device=cuda, generator=wt.g).half()
    d = torch.full((count, 144), float("nan"), device=cuda)
    plan = wt.plan("f32")
    assert plan.run(a, None, d) == 0
    check(wt, a, [count], d, "f32")


@pytest.mark.parametrize("n,k,group,zeros", [(96, 256, 32, True), (40, 130, 64, False), (64, 1024, 128, True)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_whole_numbers_come_out_exact(cuda, dtype, n, k, group, zeros):
    """Small whole activations and scales that are powers of two: every sum is exact in FP32, so a wrong
    nibble, scale or zero anywhere shows."""
    import torch
    rows = [3, 1, 0, 12]
    wt = Weights(cuda, 4, n, k, group, dtype, zeros, seed=9)
    wt.scales = torch.exp2(torch.randint(-2, 3, wt.scales.shape, device=cuda, generator=wt.g).float()).to(wt.scales.dtype)
    a = torch.randint(-8, 9, (sum(rows), k), device=cuda, generator=wt.g).to(torch_type(dtype))
    d = torch.full((sum(rows), n), float("nan"), device=cuda)
    plan = wt.plan("f32")
    assert plan.run(a, rows_tensor(rows, cuda), d) == 0
    at = 0
    for e, r in enumerate(rows):
        assert torch.equal(d[at:at + r].double(), a[at:at + r].double() @ wt.dense(e).t())
        at += r


@pytest.mark.parametrize("act", [gg.Activation.kNone, gg.Activation.kReLU, gg.Activation.kGELU])
def test_bias_activation_and_gather(cuda, act):
    import torch
    rows = [4, 0, 11]
    wt = Weights(cuda, 3, 200, 384, 128, "bf16", bias=True, seed=2)
    a = torch.randn(6, 384, device=cuda, generator=wt.g).bfloat16()
    tokens = torch.randint(0, 6, (15,), device=cuda, generator=wt.g, dtype=torch.int32)
    for out in ("f32", "bf16", "f16"):
        d = torch.full((15, 200), float("nan"), device=cuda, dtype=torch_type(out))
        plan = wt.plan(out, act)
        assert plan.run(a, rows_tensor(rows, cuda), d, row_tokens=tokens) == 0
        check(wt, a, rows, d, out, act, tokens)
    # experts without a bias, and gathered rows that do not exist (zeros)
    ptrs = [wt.bias[0].data_ptr(), None, None]
    bias = wt.bias.clone()
    bias[1:] = 0
    plan = wt.plan("f32", act, bias_ptrs=ptrs)
    tokens[3], tokens[7] = -1, 6
    d = torch.full((15, 200), float("nan"), device=cuda)
    assert plan.run(a, rows_tensor(rows, cuda), d, row_tokens=tokens) == 0
    more = torch.cat([a, torch.zeros(1, 384, device=cuda, dtype=a.dtype)])
    there = torch.where((tokens < 0) | (tokens > 5), 6, tokens)
    check(wt, more, rows, d, "f32", act, there, bias)


@pytest.mark.parametrize("pitch,first", [(300, 0), (264, 0), (259, 0), (300, 3), (264, 8)])
def test_pitches_and_misaligned_activations(cuda, pitch, first):
    import torch
    rows = [5, 9]
    wt = Weights(cuda, 2, 50, 256, 64, "f16", seed=4)
    a = torch.randn(14, 256, device=cuda, generator=wt.g).half()
    wide = torch.full((14, pitch + first), float("nan"), device=cuda, dtype=torch.float16)[:, first:first + 256]
    wide.copy_(a)
    plan = wt.plan("f32")
    want, got = torch.zeros(14, 50, device=cuda), torch.full((14, 57), 3.0, device=cuda)
    assert plan.run(a, rows_tensor(rows, cuda), want) == 0
    assert plan.run(wide, rows_tensor(rows, cuda), got[:, 5:55]) == 0
    assert torch.equal(got[:, 5:55], want)
    assert (got[:, :5] == 3).all() and (got[:, 55:] == 3).all()


def test_nan_and_infinity_stay_in_their_row(cuda):
    import torch
    wt = Weights(cuda, 2, 64, 200, 32, "f16", seed=5)
    a = torch.randn(12, 200, device=cuda, generator=wt.g).half()
    d0, d1 = torch.zeros(12, 64, device=cuda), torch.zeros(12, 64, device=cuda)
    plan = wt.plan("f32")
    assert plan.run(a, rows_tensor([9, 3], cuda), d0) == 0
    a[4, 17], a[10, 199] = float("nan"), float("inf")
    assert plan.run(a, rows_tensor([9, 3], cuda), d1) == 0
    keep = [i for i in range(12) if i not in (4, 10)]
    assert torch.equal(d1[keep], d0[keep])
    assert torch.isnan(d1[4]).all() and not torch.isfinite(d1[10]).any()


@pytest.mark.parametrize("experts", [1, 40, 300, 1024])
def test_many_experts_few_of_them_busy(cuda, experts):
    import torch
    wt = Weights(cuda, experts, 24, 160, 32, "f16", True, seed=experts)
    rows = [0] * experts
    for e in (0, experts // 2, experts - 1):
        rows[e] += 3 if e else 10
    if experts == 300:
        rows = [e % 3 for e in range(300)]
    a = torch.randn(sum(rows), 160, device=cuda, generator=wt.g).half()
    d = torch.full((sum(rows), 24), float("nan"), device=cuda)
    plan = wt.plan("f32")
    assert plan.run(a, rows_tensor(rows, cuda), d) == 0
    check(wt, a, rows, d, "f32")
    d.fill_(5.0)
    assert plan.run(a, rows_tensor([0] * experts, cuda), d) == 0  # nobody busy
    assert plan.status() == 0 and (d == 5.0).all()


@pytest.mark.parametrize("rows", [[3, -1, 2], [8, 1, 0], [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]])
def test_bad_counts_compute_nothing(cuda, rows):
    import torch
    wt = Weights(cuda, 3, 32, 128, 128, "f16", seed=6)
    a, d = torch.ones(8, 128, device=cuda).half(), torch.full((8, 32), 5.0, device=cuda)
    plan = wt.plan("f32")
    assert plan.run(a, rows_tensor(rows, cuda), d) == 0
    assert plan.status() == capi.GG_STATUS_BAD_ROWS
    assert plan.status() == 0 and (d == 5.0).all()
    # counts that d has room for but a has not
    assert plan.run(a[:4], rows_tensor([3, 0, 3], cuda), d) == 0
    assert plan.status() == capi.GG_STATUS_BAD_ROWS and (d == 5.0).all()


def test_same_bits_again_on_a_side_stream_and_in_a_graph(cuda):
    import torch
    rows = [20, 1, 0, 35]
    wt = Weights(cuda, 4, 1040, 2048, 128, "bf16", bias=True, seed=7)
    a = torch.randn(56, 2048, device=cuda, generator=wt.g).bfloat16()
    s = torch.cuda.Stream(cuda)
    s.wait_stream(torch.cuda.current_stream())
    plan, other = wt.plan("bf16"), wt.plan("bf16", stream=s)
    r = rows_tensor(rows, cuda)
    want, got = (torch.zeros(56, 1040, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    torch.cuda.synchronize()
    assert plan.run(a, r, want) == 0 and other.run(a, r, got, stream=s) == 0
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        assert plan.run(a, r, got, stream=torch.cuda.current_stream()) == 0
    second = [0, 0, 50, 6]
    r.copy_(rows_tensor(second, cuda))
    graph.replay()
    torch.cuda.synchronize()
    check(wt, a, second, got, "bf16")
    del graph


def test_tensors_that_do_not_fit_are_refused(cuda):
    import torch
    wt = Weights(cuda, 2, 32, 128, 128, "f16", seed=6)
    plan = wt.plan("f32")
    a, r, d = torch.ones(8, 128, device=cuda).half(), rows_tensor([4, 4], cuda), torch.zeros(8, 32, device=cuda)
    assert plan.run(a, r, d) == 0
    assert plan.run(a, None, d) == capi.CUDA_ERROR_INVALID_VALUE  # counts are needed with two experts
    for args in ((a.float(), r, d), (a.bfloat16(), r, d), (a[:, :-1], r, d), (a, r.long(), d), (a, r[:1], d), (a, r, d.half()),
                 (a, r, d[:, :-1]), (a.cpu(), r, d), (a, r, d.t().contiguous().t())):
        with pytest.raises(ValueError):
            plan.run(*args)
    with pytest.raises(ValueError):
        plan.run(a, r, d, row_tokens=r)
    plan.close()
    assert plan.run(a, r, d) == capi.CUDA_ERROR_INVALID_DEVICE_POINTER


@pytest.mark.parametrize("act", [gg.Activation.kReLU, gg.Activation.kGELU])
def test_activation_of_nan_is_the_grouped_products(cuda, act):
    """One name, one meaning: GG_ACT_RELU is max(x, 0), which is 0 for a NaN, and GELU of a NaN is a NaN, in the plan
    of 4-bit experts as in the grouped product."""
    import torch
    wt = Weights(cuda, 1, 64, 128, 64, "f16", seed=8)
    a = torch.randn(5, 128, device=cuda, generator=wt.g).half()
    a[2, 7] = float("nan")
    got, want = torch.full((5, 64), 5.0, device=cuda), torch.full((5, 64), 5.0, device=cuda)
    assert wt.plan("f32", act).run(a, None, got) == 0
    dense = wt.dense(0).t().half().contiguous()
    cfg = gg.KernelConfig(128, 128, 64, activation=act)
    problem = gg.ProblemDesc(5, 64, 128, a.data_ptr(), dense.data_ptr(), None, want.data_ptr(), 128, 64, 64, 64)
    assert gg.run_grouped_gemm_once([problem], gg.SortMode.kNone, cfg) == 0
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert (got[2] == 0).all() if act == gg.Activation.kReLU else torch.isnan(got[2]).all()
