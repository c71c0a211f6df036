"""The 8-bit product with a scale for each block of 128 against the definition in 64 bits.

Tolerances. The products of 8-bit values are exact; the sum over a block of 128 and the sum over blocks are FP32, each addition
off by at most a step (2^-23, if it does not round to nearest) of the sum of the magnitudes so far: with S the
sum of |sa sb A B|, G is off by at most STEP (128 + blocks + 3) S, the scales' product and their multiplication included. The
activations' slopes are below 1.13 in magnitude, and their own evaluation is within 1e-5 relative. A result is rounded once.
"""
import ctypes

import pytest

import grouped_gemm_gpu_kernel_b200 as gg
from grouped_gemm_gpu_kernel_b200 import capi

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -23
ACTS = {"none": gg.Activation.kNone, "relu": gg.Activation.kReLU, "gelu": gg.Activation.kGELU, "silu": gg.Activation.kSiLU}
OUT = {"f32": gg.OutputType.kF32, "f16": gg.OutputType.kF16, "bf16": gg.OutputType.kBF16, "e4m3": gg.OutputType.kE4M3, "e5m2": gg.OutputType.kE5M2}


def dtypes():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def act64(x, name):
    import torch
    return {"none": lambda: x, "relu": lambda: x.clamp(min=0), "silu": lambda: x * torch.sigmoid(x),
            "gelu": lambda: x * torch.sigmoid(1.5957691216057308 * (x + 0.044715 * x ** 3))}[name]()


def eight(shape, dtype, gen, pitch=None):
    """Random 8-bit values in a view whose rows are `pitch` bytes apart, NaN in the bytes between."""
    import torch
    *lead, rows, cols = shape
    pitch = -(-cols // 16) * 16 if pitch is None else pitch
    buf = torch.full((*lead, rows, pitch), 0x7f, device="cuda", dtype=torch.uint8).view(dtype)
    v = buf[..., :cols]
    top = 448.0 if dtype == torch.float8_e4m3fn else 57344.0
    v.copy_((torch.randn(*shape, device="cuda", generator=gen).clamp(-4, 4) * (top / 4)).to(dtype))
    return v


class Case:
    """Experts with `counts` rows; behind the last row of A and its scales stand NaNs, behind D's a mark."""

    def __init__(self, counts, n, k, out="f32", kind="e4m3", gated=False, act="none", bias=False, spare=3, ldd=None, seed=0, offset=0):
        import torch
        self.counts, self.n, self.k, self.out, self.gated, self.act = counts, n, k, out, gated, act
        g = torch.Generator(device="cuda").manual_seed(seed + n * 7 + k)
        e, total = len(counts), sum(counts)
        self.total, self.capacity = total, total + spare
        dt = dtypes()[kind]
        nb, kb = -(-n // 128), -(-k // 128)
        self.a = eight((self.capacity, k), dt, g)
        self.a[total:].view(torch.uint8).fill_(0x7f)
        self.sa = torch.full((self.capacity, kb + 2), float("nan"), device="cuda")[:, :kb]
        uniform = lambda *s: 0.5 + torch.rand(*s, device="cuda", generator=g)  # noqa: E731
        top = 448.0 if kind == "e4m3" else 57344.0
        self.sa[:total] = uniform(total, kb) * (3.0 / top)
        self.weights, self.scales = [], []
        for _ in range(2 if gated else 1):
            self.weights.append(eight((e, n, k), dt, g))
            self.scales.append(uniform(e, nb, kb) * (4.0 / top / k ** 0.5))
        self.bias = torch.randn(e, n, device="cuda", generator=g) if bias else None
        self.rows = torch.tensor(counts, device="cuda", dtype=torch.int32)
        self.odt = dtypes()[out]
        size = torch.empty(0, dtype=self.odt).element_size()
        ldd = n if ldd is None else ldd
        self.buf = torch.full((offset + self.capacity * ldd + 32,), 7, device="cuda", dtype=torch.uint8 if size == 1 else self.odt)
        self.d = self.buf.view(self.odt)[offset:].as_strided((self.capacity, n), (ldd, 1))
        self.sd = torch.full((self.capacity, nb + 1), 7.0, device="cuda")[:, :nb] if size == 1 else None
        each = lambda t: None if t is None else [x.data_ptr() for x in t]  # noqa: E731
        up = (each(self.weights[1]), each(self.scales[1])) if gated else (None, None)
        self.plan = gg.F8Plan(e, n, k, each(self.weights[0]), self.weights[0].stride(1), each(self.scales[0]), *up, bias_ptrs=each(self.bias),
                              input_type=gg.InputType.kE4M3 if kind == "e4m3" else gg.InputType.kE5M2, output_type=OUT[out], activation=ACTS[act])

    def run(self, stream=None, rows=True):
        return self.plan.run(self.a, self.sa, self.rows if rows else None, self.d, d_scales=self.sd, stream=stream)

    def check(self):
        import torch
        torch.cuda.synchronize()
        assert self.plan.status() == 0
        wide = lambda s, n, dim: s.double().repeat_interleave(128, dim).narrow(dim, 0, n)  # noqa: E731
        a = self.a[:self.total].double() * wide(self.sa[:self.total], self.k, 1)
        want, bound = torch.zeros(self.total, self.n, device="cuda", dtype=torch.float64), torch.zeros(self.total, self.n, device="cuda", dtype=torch.float64)
        first = 0
        steps = STEP * (128 + self.sa.shape[1] + 3)
        for e, count in enumerate(self.counts):
            if not count:
                continue
            rows = slice(first, first + count)
            first += count
            got = []
            for w, s in zip(self.weights, self.scales):
                b = w[e].double() * wide(wide(s[e], self.n, 0), self.k, 1)
                got.append((a[rows] @ b.t(), a[rows].abs() @ b.abs().t() * steps))
            g, off = got[0]
            if self.bias is not None:
                g, off = g + self.bias[e].double(), off + STEP * (g.abs() + self.bias[e].double().abs())
            v = act64(g, self.act)
            off = off if self.act == "none" else 1.13 * off + 1e-5 * v.abs()
            if self.gated:
                u, uoff = got[1]
                off = u.abs() * off + v.abs() * uoff + off * uoff + STEP * (u * v).abs()
                v = v * u
            want[rows], bound[rows] = v, off
        d = self.d[:self.total].double()
        if self.sd is None:
            info = torch.finfo(self.odt)
            half = 0.0 if self.odt == torch.float32 else info.eps / 2
            bound = bound * (1 + half) + want.abs() * half + info.tiny * info.eps / 2
        else:
            s = self.sd[:self.total].double()
            top, half, small = (448.0, 2.0 ** -4, 2.0 ** -10) if self.out == "e4m3" else (57344.0, 2.0 ** -3, 2.0 ** -17)
            pad = lambda t: torch.nn.functional.pad(t, (0, s.shape[1] * 128 - self.n)).view(self.total, -1, 128)  # noqa: E731
            most, most_off = pad(want).abs().amax(2) / top, pad(bound).amax(2) / top
            assert bool(((s - most).abs() <= most_off + 4 * STEP * most).all())
            wide_s = wide(s, self.n, 1)
            d = d * wide_s
            bound = bound * (1 + half) + want.abs() * (half + 1e-4) + wide_s * small
        off = (d - want).abs()
        assert bool(torch.isfinite(d).all())
        assert bool((off <= bound).all()), f"largest difference {float(off.max())}, of the bound {float((off / bound.clamp(min=1e-300)).max())}"
        # behind the rows and between them nothing is written
        keep = self.buf.clone()
        self.d[:self.total].view(self.buf.dtype).fill_(7)
        assert bool((self.buf == 7).all())
        self.buf.copy_(keep)
        if self.sd is not None:
            assert bool((self.sd[self.total:] == 7).all())


@pytest.mark.parametrize("k", [1, 15, 16, 127, 128, 129, 640, 1003, 4096])
@pytest.mark.parametrize("n", [1, 31, 128, 130, 777])
def test_sizes(cuda, n, k):
    c = Case([3, 0, 129, 1], n, k)
    assert c.run() == 0
    c.check()


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 127, 128, 129, 256, 300])
@pytest.mark.parametrize("n", [64, 2368, 9472, 18944 + 5])
def test_tile_widths(cuda, n, rows):
    """One expert: the outputs of a tile are 32 to 256 by how many tiles there are for the GPU's SMs."""
    c = Case([rows], n, 260)
    assert c.run() == 0
    c.check()


@pytest.mark.parametrize("counts", [[513], [300, 724], [0, 1000, 257], [256, 512, 1, 255]])
@pytest.mark.parametrize("n,k,out,gated", [(9472, 260, "bf16", False), (9477, 128, "f32", False), (4736, 700, "bf16", True), (4800, 390, "e4m3", True),
                                           (4737, 1000, "e5m2", True)])
def test_many_rows(cuda, counts, n, k, out, gated):
    """Several tiles of rows of an expert, of the widest kind, and more of them than SMs."""
    c = Case(counts, n, k, out=out, gated=gated, act="silu" if gated else "none", ldd=-(-n // 32) * 32 if out != "f32" else None)
    assert c.run() == 0
    c.check()


@pytest.mark.parametrize("out", ["f32", "f16", "bf16", "e4m3", "e5m2"])
@pytest.mark.parametrize("counts,n,k", [([5, 0, 130, 1, 64], 300, 384), ([1], 128, 128), ([40] * 8, 4736, 200), ([2] * 3, 1, 7), ([200], 127, 33)])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_gated(cuda, counts, n, k, out, act):
    c = Case(counts, n, k, out=out, gated=True, act=act)
    assert c.run() == 0
    c.check()


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("kind", ["e4m3", "e5m2"])
def test_types_bias_and_activation(cuda, kind, act, out):
    c = Case([33, 100, 0, 7], 333, 520, out=out, kind=kind, act=act, bias=True)
    assert c.run() == 0
    c.check()


@pytest.mark.parametrize("out,gated", [("f32", False), ("bf16", False), ("bf16", True), ("e4m3", True)])
@pytest.mark.parametrize("ldd,offset", [(333, 0), (333, 1), (336, 0), (352, 16), (334, 2)])
def test_outputs_on_any_alignment(cuda, out, gated, ldd, offset):
    c = Case([33, 100], 333, 130, out=out, gated=gated, act="silu" if gated else "none", ldd=ldd, offset=offset)
    assert c.run() == 0
    c.check()


def test_many_experts(cuda):
    import random
    rng = random.Random(3)
    counts = [rng.choice([0, 0, 1, 2, 5]) for _ in range(1024)]
    counts[-1] = 3
    c = Case(counts, 40, 48, out="bf16")
    assert c.run() == 0
    c.check()


def test_without_counts(cuda):
    c = Case([77], 200, 300, spare=0)
    assert c.run(rows=False) == 0
    c.check()


def test_no_rows(cuda):
    import torch
    c = Case([0, 0], 64, 64)
    assert c.run() == 0
    c.check()
    a, s, d = c.a[:0], c.sa[:0], c.d[:0]
    assert c.plan.run(a, s, c.rows, d) == 0
    torch.cuda.synchronize()
    assert c.plan.status() == 0


@pytest.mark.parametrize("counts", [[5, -1, 3], [20, 20, 20], [2 ** 31 - 1, 2 ** 31 - 1, 2], [0, 0, 33]])
def test_bad_counts_compute_nothing(cuda, counts):
    import torch
    c = Case([10, 10, 9], 64, 64)
    c.rows.copy_(torch.tensor(counts, dtype=torch.int32))
    assert c.run() == 0
    torch.cuda.synchronize()
    assert c.plan.status() == capi.GG_STATUS_BAD_ROWS
    assert bool((c.buf == 7).all())
    assert c.plan.status() == 0
    c.rows.copy_(torch.tensor([10, 10, 9], dtype=torch.int32))
    assert c.run() == 0
    c.check()


def test_not_finite_stays_in_its_place(cuda):
    """A NaN in a row reaches that row's results, one in a weight that output's, of that expert; nothing else."""
    import torch
    c = Case([40, 50], 200, 256)
    assert c.run() == 0
    torch.cuda.synchronize()
    clean = c.d.clone()
    c.a[7, 100].view(torch.uint8).fill_(0x7f)
    c.weights[0][1, 33, 5].view(torch.uint8).fill_(0x7f)
    assert c.run() == 0
    torch.cuda.synchronize()
    bad = torch.isnan(c.d[:90])
    want = torch.zeros_like(bad)
    want[7] = True
    want[40:90, 33] = True
    assert torch.equal(bad, want) and torch.equal(c.d[:90][~bad], clean[:90][~bad])


def test_same_bits_captured_on_streams_and_with_new_counts(cuda):
    import torch
    c, other = Case([20, 30, 0, 77], 500, 640, out="bf16", seed=1), Case([20, 30, 0, 77], 500, 640, out="bf16", seed=1)
    assert c.run() == 0
    c.check()
    want = c.d.clone()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):  # one plan on two streams at once
        assert c.plan.run(c.a, c.sa, c.rows, c.d, stream=streams[0]) == 0
        assert c.plan.run(c.a, c.sa, c.rows, other.d, stream=streams[1]) == 0
    torch.cuda.synchronize()
    assert torch.equal(c.d[:127], want[:127]) and torch.equal(other.d[:127], want[:127])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        assert c.run(stream=torch.cuda.current_stream()) == 0
    c.counts = [60, 0, 60, 7]
    c.rows.copy_(torch.tensor(c.counts, dtype=torch.int32))
    c.buf.fill_(7)
    graph.replay()
    c.check()
    del graph


def test_refusals(cuda):
    import torch
    c = Case([4, 4], 64, 64, out="bf16")
    z = lambda *s, dt=torch.float32: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    f8 = torch.float8_e4m3fn
    ok = dict(a=c.a, a_scales=c.sa, rows=c.rows, d=c.d)
    for bad in (dict(a=c.a[:, :32]), dict(a=c.a[:5]), dict(a=c.a.view(torch.uint8)), dict(a=c.a.cpu()), dict(a_scales=z(11, 2)), dict(a_scales=c.sa.half()),
                dict(rows=c.rows[:1]), dict(rows=c.rows.long()), dict(d=z(11, 64)), dict(d=z(11, 63, dt=torch.bfloat16)), dict(d_scales=z(11, 1)),
                dict(a=z(11, 128, dt=f8)[:, ::2])):
        with pytest.raises(ValueError):
            c.plan.run(**(ok | bad))
    invalid = capi.CUDA_ERROR_INVALID_VALUE
    assert c.plan.run(z(11, 72, dt=f8)[:, :64], c.sa, c.rows, c.d) == invalid          # a pitch off 16 bytes
    assert c.plan.run(z(11, 80, dt=f8)[:, 8:72], c.sa, c.rows, c.d) == invalid         # a base off 16 bytes
    assert c.plan.run(c.a, c.sa, None, c.d) == invalid                                 # two experts need counts
    lib = capi.load()
    call = lambda **f: lib.gg_f8_plan_run(c.plan._h, *[(dict(a=c.a.data_ptr(), lda=64, s=c.sa.data_ptr(), lds=3, rows=c.rows.data_ptr(), d=c.d.data_ptr(),  # noqa: E731
                                                             ldd=64, ds=None, ldds=0, cap=11) | f)[n] for n in ("a", "lda", "s", "lds", "rows", "d", "ldd", "ds", "ldds", "cap")], None)
    for bad in (dict(a=None), dict(s=None), dict(d=None), dict(lda=48), dict(lds=0), dict(ldd=63), dict(cap=-1), dict(cap=2 ** 31 - 65536)):
        assert call(**bad) == invalid
    g = Case([4, 4], 64, 64, out="e4m3", gated=True, act="silu")
    with pytest.raises(ValueError):
        g.plan.run(g.a, g.sa, g.rows, g.d)
    assert lib.gg_f8_plan_status(c.plan._h, None) == invalid
    c.plan.close()
    assert c.plan.run(**ok) == capi.CUDA_ERROR_INVALID_DEVICE_POINTER
    _ = ctypes
