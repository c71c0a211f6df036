"""The gated feed-forward of experts and its gradient against the definition in 64 bits.

Tolerances. The products of 16-bit values are exact in FP32; an addition is off by at most a step (2^-23, if it does not round
to nearest) of the sum of the magnitudes, so a product over k is off by at most STEP (k + 2) S with S the sum of
|x w|. Each gradient is compared with what the stored gate, up, grad_gate and grad_up give, so that only its own
arithmetic and its rounding (half a step of the type) count.

act(x) = x / (1 + exp(-z)), z = x or 2 u(x): z is off by at most 4 roundings of 2^-24 of it, __expf by 2 + 1.173 |z| steps
of 2^-23, the sum, the division (2 steps) and the product by 4 steps more. The kernels cap -z at 80, so that is
(2 + 94 + 160 + 4) 2^-23 < 4e-5 relative at most: NEAR. Past the cap act is x exp(-80) < 2e-35 |x| in place of less, and the
slope below 2e-35 (1 + |x| z'(x)) with z' <= 1.6 + 0.22 x^2: FAR (1 + |x|)^3 bounds both. The slope s + x s (1 - s) z' is
at most 1.13, and its error NEAR of that (1 - s is off by 2^-24, and 0 where z > 17.4; |x| z' is below 25 up to there).
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg
from grouped_gemm_gpu_kernel_b200 import capi

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -23
NEAR = 4e-5
FAR = 4e-35
ACTS = {"none": gg.Activation.kNone, "relu": gg.Activation.kReLU, "gelu": gg.Activation.kGELU, "silu": gg.Activation.kSiLU}


def act64(x, name):
    import torch
    return {"none": lambda: x, "relu": lambda: x.clamp(min=0), "silu": lambda: x * torch.sigmoid(x),
            "gelu": lambda: x * torch.sigmoid(1.5957691216057308 * (x + 0.044715 * x ** 3))}[name]()


def slope64(x, name):
    import torch
    x = x.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(act64(x, name).sum(), x)[0] if name != "none" else torch.ones_like(x)


def pitched(shape, dtype, fill, spare=0):
    import torch
    *lead, rows, cols = shape
    return torch.full((*lead, rows, -(-cols // 8) * 8 + spare), fill, device="cuda", dtype=dtype)[..., :cols]


class Case:
    """Experts with `counts` rows. Behind the last row and between columns and pitch stand NaNs (inputs) or 7 (outputs)."""

    def __init__(self, counts, n, k, kind="bf16", act="silu", spare=3, seed=0, wtype=None):
        import torch
        self.counts, self.n, self.k, self.act = counts, n, k, act
        self.dt = {"f16": torch.float16, "bf16": torch.bfloat16}[kind]
        self.half = torch.finfo(self.dt).eps / 2
        self.floor = torch.finfo(self.dt).tiny * torch.finfo(self.dt).eps
        g = torch.Generator(device="cuda").manual_seed(seed + 7 * n + k)
        rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        e, self.total = len(counts), sum(counts)
        self.capacity = self.total + spare
        nan = float("nan")
        self.x, self.grad_h = pitched((self.capacity, k), self.dt, nan, 8), pitched((self.capacity, n), self.dt, nan)
        self.x[:self.total], self.grad_h[:self.total] = rnd(self.total, k).to(self.dt), rnd(self.total, n).to(self.dt)
        self.wg, self.wu = pitched((e, k, n), self.dt, nan, 8), pitched((e, k, n), self.dt, nan, 8)
        self.wg.copy_(rnd(e, k, n) * (1.5 / k ** 0.5)), self.wu.copy_(rnd(e, k, n) / k ** 0.5)
        self.rows = torch.tensor(counts, device="cuda", dtype=torch.int32)
        self.h, self.gate, self.up, self.gg, self.gu = [pitched((self.capacity, n), self.dt, 7) for _ in range(5)]
        self.gx = pitched((self.capacity, k), self.dt, 7)
        self.wtype = self.dt if wtype is None else wtype
        self.gwg, self.gwu = [pitched((e, k, n), self.wtype, 7) for _ in range(2)]
        self.plan = gg.GatedPlan(e, n, k, [w.data_ptr() for w in self.wg], [w.data_ptr() for w in self.wu], self.wg.stride(1),
                                 input_type=gg.InputType.kF16 if kind == "f16" else gg.InputType.kBF16, activation=ACTS[act])

    def forward(self, stream=None, keep=True, rows=True):
        return self.plan.run(self.x, self.rows if rows else None, self.h, **(dict(gate=self.gate, up=self.up) if keep else {}), stream=stream)

    def backward(self, stream=None, rows=True):
        return self.plan.backward(self.x, self.gate, self.up, self.grad_h, self.rows if rows else None, self.gg, self.gu, grad_x=self.gx,
                                  grad_gate_w=self.gwg, grad_up_w=self.gwu, stream=stream)

    def near(self, name, got, want, bound, half=None, floor=None):
        import torch
        half = self.half if half is None else half
        off = (got.double() - want).abs()
        limit = bound * (1 + half) + want.abs() * half + (self.floor if floor is None else floor)
        assert bool(torch.isfinite(got.double()).all()), name
        assert bool((off <= limit).all()), f"{name}: largest difference {float(off.max())}, of the bound {float((off / limit).max())}"

    def spans(self):
        first = 0
        for e, count in enumerate(self.counts):
            yield e, slice(first, first + count)
            first += count

    def untouched(self, *views):
        for v in views:
            assert bool((v[self.total:] == 7).all())
            whole = v.as_strided((v.shape[0], v.stride(0)), (v.stride(0), 1))[:, v.shape[1]:]
            assert bool((whole == 7).all())

    def check_forward(self, kept=True):
        import torch
        torch.cuda.synchronize()
        assert self.plan.status() == 0
        for e, at in self.spans():
            x, wg, wu = self.x[at].double(), self.wg[e].double(), self.wu[e].double()
            g, u = x @ wg, x @ wu
            og, ou = [(x.abs() @ w.abs()) * (STEP * (self.k + 2)) for w in (wg, wu)]
            v = act64(g, self.act)
            if kept:
                self.near("gate", self.gate[at], g, og)
                self.near("up", self.up[at], u, ou)
            ov = 1.13 * og + NEAR * v.abs() + FAR * (1 + g.abs()) ** 3
            self.near("h", self.h[at], v * u, ov * u.abs() + ou * v.abs() + ov * ou)
        self.untouched(self.h, *((self.gate, self.up) if kept else ()))

    def check_backward(self):
        import torch
        torch.cuda.synchronize()
        assert self.plan.status() == 0
        info = torch.finfo(self.wtype)
        half, floor = (0.0, info.tiny) if self.wtype == torch.float32 else (self.half, self.floor)
        for e, at in self.spans():
            g, u, gh, x = [t[at].double() for t in (self.gate, self.up, self.grad_h, self.x)]
            s, v = slope64(g, self.act), act64(g, self.act)
            self.near("grad_gate", self.gg[at], gh * u * s, (NEAR * 1.13 + FAR * (1 + g.abs()) ** 3) * (gh * u).abs())
            self.near("grad_up", self.gu[at], gh * v, (NEAR * v.abs() + FAR * (1 + g.abs()) ** 3) * gh.abs())
            dg, du, wg, wu = self.gg[at].double(), self.gu[at].double(), self.wg[e].double(), self.wu[e].double()
            self.near("grad_x", self.gx[at], dg @ wg.t() + du @ wu.t(), (dg.abs() @ wg.abs().t() + du.abs() @ wu.abs().t()) * (STEP * (2 * self.n + 2)))
            rows = at.stop - at.start
            for name, got, d in (("grad_wg", self.gwg, dg), ("grad_wu", self.gwu, du)):
                self.near(name, got[e], x.t() @ d, (x.abs().t() @ d.abs()) * (STEP * (rows + 2)), half, floor)
        self.untouched(self.gg, self.gu, self.gx)
        for w in (self.gwg, self.gwu):
            assert bool((w.as_strided((w.shape[0], w.shape[1], w.stride(1)), w.stride())[..., self.n:] == 7).all())


@pytest.mark.parametrize("k", [1, 8, 63, 64, 65, 200, 515])
@pytest.mark.parametrize("n", [1, 64, 127, 128, 130, 331])
def test_sizes(cuda, n, k):
    c = Case([3, 0, 129, 1], n, k)
    assert c.forward() == 0
    c.check_forward()
    assert c.backward() == 0
    c.check_backward()


@pytest.mark.parametrize("counts", [[1], [15, 16, 17], [63, 64, 65], [127, 128, 129], [0, 0, 5, 0], [300, 1, 0, 257], [0]])
@pytest.mark.parametrize("kind,wide", [("bf16", False), ("f16", True), ("bf16", True)])
def test_counts(cuda, counts, kind, wide):
    """The last rows of an expert share a stage of the weights' gradient with the next expert's first."""
    import torch
    c = Case(counts, 200, 136, kind=kind, wtype=torch.float32 if wide else None)
    assert c.forward() == 0
    c.check_forward()
    assert c.backward() == 0
    c.check_backward()


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_activations(cuda, act, kind):
    c = Case([40, 100, 0, 7], 264, 72, kind=kind, act=act)
    c.x[3] *= 30.0  # far out on both sides
    c.x[4] = 0.0
    assert c.forward() == 0
    c.check_forward()
    assert c.backward() == 0
    c.check_backward()


@pytest.mark.parametrize("counts", [[512], [513, 700], [1000, 24], [0, 1537, 600], [256 * 3 + 1, 256 * 3 - 1, 640]])
@pytest.mark.parametrize("n,k", [(128, 64), (300, 520), (72, 256), (131, 130)])
def test_rows_in_tiles_of_256(cuda, counts, n, k):
    """Rows and k enough for tiles on pairs of CTAs, with last tiles of which one CTA has no part."""
    c = Case(counts, n, k)
    assert c.forward() == 0
    c.check_forward()
    assert c.backward() == 0
    c.check_backward()


def test_many_tiles(cuda):
    """More tiles than SMs, several stretches of rows of one expert, and experts enough for a full table."""
    c = Case([1000, 300, 0, 2500], 1100, 400)
    assert c.forward() == 0
    c.check_forward()
    assert c.backward() == 0
    c.check_backward()
    import random
    rng = random.Random(5)
    c = Case([rng.choice([0, 0, 1, 3]) for _ in range(1023)] + [2], 24, 16)
    assert c.forward() == 0
    c.check_forward()
    assert c.backward() == 0
    c.check_backward()


def test_parts_and_places(cuda):
    """Without gate and up; without counts; gradients in the place of gate, up and grad_h; and each gradient alone."""
    import torch
    c = Case([50], 136, 80, spare=0)
    assert c.forward(keep=False, rows=False) == 0
    c.check_forward(kept=False)
    assert c.forward(rows=False) == 0
    assert c.backward(rows=False) == 0
    c.check_backward()
    want = [t.clone() for t in (c.gg, c.gu, c.gx, c.gwg, c.gwu)]
    for t in (c.gx, c.gwg, c.gwu):
        t.fill_(7)
    gh = c.grad_h.as_strided(c.grad_h.shape, c.grad_h.stride())
    assert c.plan.backward(c.x, c.gate, c.up, gh, c.rows, c.gate, c.up, grad_x=c.gx) == 0
    torch.cuda.synchronize()
    assert torch.equal(c.gate, want[0]) and torch.equal(c.up, want[1]) and torch.equal(c.gx, want[2])
    assert bool((c.gwg == 7).all())
    assert c.forward(rows=False) == 0
    assert c.plan.backward(c.x, c.gate, c.up, gh, c.rows, gh, c.up, grad_gate_w=c.gwg, grad_up_w=c.gwu) == 0
    torch.cuda.synchronize()
    assert torch.equal(gh, want[0]) and torch.equal(c.up, want[1]) and torch.equal(c.gwg, want[3]) and torch.equal(c.gwu, want[4])


def test_outputs_on_any_alignment(cuda):
    """Outputs that no TMA load reads may start anywhere: h, gate, up, grad_x and the weights' gradients."""
    import torch
    n, k = 131, 77
    c = Case([40, 33], n, k, spare=0)
    assert c.forward() == 0 and c.backward() == 0
    want = [t.clone() for t in (c.h, c.gate, c.up, c.gx, c.gwg, c.gwu)]
    odd = lambda *s, dt=c.dt: torch.full((1 + int(torch.tensor(s).prod()),), 7, device="cuda", dtype=dt)[1:].view(*s)  # noqa: E731
    h, gate, up, gx, gwg, gwu = odd(73, n), odd(73, n), odd(73, n), odd(73, k), odd(2, k, n), odd(2, k, n)
    assert c.plan.run(c.x, c.rows, h, gate=gate, up=up) == 0
    ghd = odd(73, n)
    ghd.copy_(c.grad_h)
    assert c.plan.backward(c.x, gate, up, ghd, c.rows, c.gg, c.gu, grad_x=gx, grad_gate_w=gwg, grad_up_w=gwu) == 0
    torch.cuda.synchronize()
    for a, b in zip((h, gate, up, gx, gwg, gwu), want):
        assert torch.equal(a, b)


def test_no_rows(cuda):
    import torch
    c = Case([0, 0, 0], 72, 40, spare=0)
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    assert c.plan.status() == 0
    assert bool((c.gwg == 0).all()) and bool((c.gwu == 0).all())


@pytest.mark.parametrize("counts", [[5, -1, 3], [20, 20, 20], [2 ** 31 - 1, 2 ** 31 - 1, 2]])
def test_bad_counts_compute_nothing(cuda, counts):
    import torch
    c = Case([10, 10, 9], 64, 64)
    assert c.forward() == 0
    torch.cuda.synchronize()
    c.rows.copy_(torch.tensor(counts, dtype=torch.int32))
    c.h.fill_(7)
    assert c.forward(keep=False) == 0 and c.backward() == 0
    torch.cuda.synchronize()
    assert c.plan.status() == capi.GG_STATUS_BAD_ROWS
    for t in (c.h, c.gg, c.gu, c.gx, c.gwg, c.gwu):
        assert bool((t == 7).all())
    assert c.plan.status() == 0


def test_not_finite_stays_with_its_expert(cuda):
    import torch
    c = Case([30, 18, 41], 96, 80)
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    clean = [t.clone() for t in (c.h, c.gx, c.gwg, c.gwu)]
    c.x[30, 5] = float("nan")       # expert 1's first row
    c.grad_h[47, 9] = float("inf")  # its last
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    keep = torch.ones(89, dtype=torch.bool, device="cuda")
    keep[30] = keep[47] = False
    assert torch.equal(c.h[:89][keep], clean[0][:89][keep]) and bool(torch.isnan(c.h[30]).all())
    assert torch.equal(c.gx[:89][keep], clean[1][:89][keep])
    for e in (0, 2):
        assert torch.equal(c.gwg[e], clean[2][e]) and torch.equal(c.gwu[e], clean[3][e])


@pytest.mark.parametrize("counts,n,k", [([20, 30, 0, 77], 500, 200), ([700, 30, 0, 1400], 200, 300)])
def test_same_bits_captured_on_streams_and_with_new_counts(cuda, counts, n, k):
    import torch
    c = Case(counts, n, k)
    total = sum(counts)
    assert c.forward() == 0 and c.backward() == 0
    c.check_forward()
    c.check_backward()
    want = [t.clone() for t in (c.h, c.gx, c.gwg, c.gwu)]
    other = torch.empty_like(c.h)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):  # one plan on two streams at once
        assert c.plan.run(c.x, c.rows, c.h, stream=streams[0]) == 0
        assert c.plan.run(c.x, c.rows, other, stream=streams[1]) == 0
    torch.cuda.synchronize()
    assert torch.equal(c.h[:total], want[0][:total]) and torch.equal(other[:total], want[0][:total])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        st = torch.cuda.current_stream()
        assert c.forward(stream=st) == 0 and c.backward(stream=st) == 0
    for t in (c.h, c.gx, c.gwg, c.gwu):
        t.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip((c.h, c.gx, c.gwg, c.gwu), want):
        assert torch.equal(a, b)
    c.counts, c.total = [60, 0, total - 67, 7], total
    c.rows.copy_(torch.tensor(c.counts, dtype=torch.int32))
    for t in (c.h, c.gx, c.gwg, c.gwu):
        t.fill_(7)
    graph.replay()
    c.check_forward()
    c.check_backward()
    del graph


def test_gradient_against_differences(cuda):
    """The change of <grad_h, h> along a direction of x and of both weights, by central differences of the definition in 64
    bits. What the kernels round on the way (gate, up, grad_gate, grad_up to 2^-11, the results too) is at most five halves of a
    step of each term: 5 * 2^-11 of the sum of the terms' magnitudes if all had one sign; of random sign, a tenth of that."""
    import torch
    c = Case([25, 0, 40], 72, 48, kind="f16", spare=0)
    assert c.forward() == 0 and c.backward() == 0
    torch.cuda.synchronize()
    g = torch.Generator(device="cuda").manual_seed(9)
    rnd = lambda t: torch.randn(t.shape, device="cuda", generator=g, dtype=torch.float64)  # noqa: E731
    vx, vg, vu = rnd(c.x), rnd(c.wg) / 7, rnd(c.wu) / 7

    def goal(t):
        total = 0.0
        for e, at in c.spans():
            x = c.x[at].double() + t * vx[at]
            total += float((c.grad_h[at].double() * act64(x @ (c.wg[e].double() + t * vg[e]), "silu") * (x @ (c.wu[e].double() + t * vu[e]))).sum())
        return total

    t = 1e-5
    there = (goal(t) - goal(-t)) / (2 * t)
    terms = [c.gx.double() * vx, c.gwg.double() * vg, c.gwu.double() * vu]
    assert abs(there - sum(float(v.sum()) for v in terms)) < 0.5 * 2.0 ** -11 * sum(float(v.abs().sum()) for v in terms)


def test_refusals(cuda):
    import torch
    c = Case([4, 4], 64, 48, spare=0)
    z = lambda *s, dt=c.dt: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    ok = dict(x=c.x, rows=c.rows, h=c.h)
    for bad in (dict(x=z(8, 40)), dict(x=z(8, 48, dt=torch.float16)), dict(h=z(7, 64)), dict(rows=c.rows[:1]), dict(gate=c.gate), dict(up=c.up),
                dict(gate=c.gate, up=z(8, 72)[:, :64]), dict(x=c.x.cpu())):
        with pytest.raises(ValueError):
            c.plan.run(**(ok | bad))
    invalid = capi.CUDA_ERROR_INVALID_VALUE
    assert c.plan.run(z(8, 52)[:, :48], c.rows, c.h) == invalid       # a pitch off 16 bytes
    assert c.plan.run(z(8, 56)[:, 4:52], c.rows, c.h) == invalid      # a base off 16 bytes
    assert c.plan.run(c.x, None, c.h) == invalid                      # two experts need counts
    ok = dict(x=c.x, gate=c.gate, up=c.up, grad_h=c.grad_h, rows=c.rows, grad_gate=c.gg, grad_up=c.gu)
    for bad in (dict(gate=z(8, 72)[:, :64]), dict(grad_up=z(8, 72)[:, :64]), dict(grad_h=z(7, 64)), dict(grad_x=z(8, 40)), dict(grad_gate_w=c.gwg),
                dict(grad_up_w=c.gwu), dict(grad_gate_w=c.gwg, grad_up_w=c.gwu.float()), dict(grad_gate_w=c.gwg.half(), grad_up_w=c.gwu.half()),
                dict(grad_gate_w=c.gwg[:1], grad_up_w=c.gwu[:1]), dict(grad_gate_w=c.gwg.transpose(1, 2), grad_up_w=c.gwu.transpose(1, 2)),
                dict(grad_gate_w=z(1, 48, 64).expand(2, 48, 64), grad_up_w=z(1, 48, 64).expand(2, 48, 64)), dict(grad_gate_w=z(48, 64), grad_up_w=z(48, 64))):
        with pytest.raises(ValueError):
            c.plan.backward(**(ok | bad))
    odd = [z(8, 65)[:, :64] for _ in range(2)]
    assert c.plan.backward(**(ok | dict(grad_gate=odd[0], grad_up=odd[1]))) == invalid
    c.plan.close()
    assert c.plan.run(c.x, c.rows, c.h) == capi.CUDA_ERROR_INVALID_DEVICE_POINTER


@pytest.mark.parametrize("counts", [[5, -1, 3], [20, 20, 20], [2 ** 31 - 1, 2 ** 31 - 1, 2]])
@pytest.mark.parametrize("spare", [3, None])
def test_bad_counts_without_products(cuda, counts, spare):
    """The gradients of gate and up alone, with room for some rows or (None) for none: bad counts are reported too."""
    import torch
    c = Case([10, 10, 9], 64, 64)
    rows = slice(0, None if spare else 0)
    c.rows.copy_(torch.tensor(counts, dtype=torch.int32))
    call = lambda: c.plan.backward(*[t[rows] for t in (c.x, c.gate, c.up, c.grad_h)], c.rows, c.gg[rows], c.gu[rows])  # noqa: E731
    assert call() == 0
    torch.cuda.synchronize()
    assert c.plan.status() == capi.GG_STATUS_BAD_ROWS
    assert bool((c.gg == 7).all()) and bool((c.gu == 7).all())
    assert c.plan.status() == 0
    c.rows.zero_()
    assert call() == 0
    torch.cuda.synchronize()
    assert c.plan.status() == 0
