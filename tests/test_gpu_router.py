"""The mixture-of-experts router (gg_router_*) against its definition in 64 bits.

Whole numbers (indices, counts, positions) have to be equal. Bounds of the floating results, from the
arithmetic: exp(x) in FP32 is off by at most 2^-22 + |x| 2^-23 relative (the fast exponential, and the
rounding of its scaled argument), which is below 6e-6 for the |x| <= 48 that matter to a sum here; a sum
of E positive terms adds (V + 8) 2^-24; so RTOL = 1e-5 bounds p, the weights and the means, and what is
made of them by a few products. A gradient is bounded term by term with the same RTOL.
"""
import math

import numpy as np
import pytest

import grouped_gemm_gpu_kernel_b200 as gg
from grouped_gemm_gpu_kernel_b200 import capi

pytestmark = pytest.mark.gpu

RTOL = 1e-5
TYPES = {"f32": gg.OutputType.kF32, "f16": gg.OutputType.kF16, "bf16": gg.OutputType.kBF16}


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def rounding(name):
    """(relative, absolute) error of one rounding to the type."""
    return {"f32": (2.0 ** -24, 0.0), "f16": (2.0 ** -11, 2.0 ** -25), "bf16": (2.0 ** -8, 0.0)}[name]


class Forward:
    """One run with NaN- or junk-filled outputs, brought to the host."""

    def __init__(self, logits, top_k, normalize=True, mask=None, dtype="f32", router=None, stream=None):
        import torch
        t, e = logits.shape
        dev = logits.device
        self.router = router or gg.MoeRouter(e, top_k, t, logit_type=TYPES[dtype], normalize=normalize)
        junk = lambda *s: torch.full(s, -77, dtype=torch.int32, device=dev)  # noqa: E731
        nan = lambda *s: torch.full(s, float("nan"), device=dev)  # noqa: E731
        self.indices, self.weights, self.positions = junk(t, top_k), nan(t, top_k), junk(t, top_k)
        self.rows, self.losses, self.row_tokens = junk(e), nan(3), junk(t * top_k)
        self.lse, self.prob_mean = nan(t), nan(e)
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        assert self.router.run(logits, self.indices, self.weights, self.positions, self.rows, self.losses,
                               row_tokens=self.row_tokens, lse=self.lse, prob_mean=self.prob_mean, token_mask=mask,
                               stream=stream) == 0


def reference(logits, top_k, normalize, mask):
    """The definition on the host in 64 bits, token by token."""
    l = logits.double().cpu().numpy()
    t, e = l.shape
    m = np.ones(t, bool) if mask is None else mask.cpu().numpy().astype(bool)
    idx = np.full((t, top_k), -1, np.int64)
    w = np.zeros((t, top_k))
    p = np.zeros((t, e))
    lse = np.zeros(t)
    valid = m & (l != -np.inf).any(1)
    for i in np.nonzero(valid)[0]:
        row = l[i]
        key = np.where(np.isnan(row), np.inf, row)
        order = sorted(range(e), key=lambda x: (not np.isnan(row[x]), -key[x], x))
        chosen = [x for x in order if row[x] != -np.inf][:top_k]
        with np.errstate(invalid="ignore"):
            top = row[order[0]]
            ex = np.exp(row - top)
            p[i] = ex / ex.sum()
            lse[i] = top + np.log(ex.sum())
            idx[i, :len(chosen)] = chosen
            w[i, :len(chosen)] = ex[chosen] / ex[chosen].sum() if normalize else p[i, chosen]
    rows = np.bincount(idx[idx >= 0], minlength=e)
    flat = idx.reshape(-1)
    slots = np.array(sorted(np.nonzero(flat >= 0)[0], key=lambda s: (flat[s], s)), dtype=np.int64)
    pos = np.full(t * top_k, -1, np.int64)
    pos[slots] = np.arange(len(slots))
    row_tokens = np.full(t * top_k, -1, np.int64)
    row_tokens[:len(slots)] = slots // top_k
    n = int(valid.sum())
    mean = p.sum(0) / max(1, n)
    f = rows / max(1, rows.sum())
    losses = np.array([e * (f * mean).sum(), (lse ** 2).sum() / max(1, n), n])
    return dict(indices=idx, weights=w, positions=pos.reshape(t, top_k), rows=rows, row_tokens=row_tokens, lse=lse,
                prob_mean=mean, losses=losses, p=p, valid=valid, f=f, n=n)


def check_forward(fw, ref):
    for name in ("indices", "positions", "rows", "row_tokens"):
        np.testing.assert_array_equal(getattr(fw, name).cpu().numpy(), ref[name], err_msg=name)
    close = lambda a, b, atol: np.testing.assert_allclose(a.double().cpu().numpy(), b, rtol=RTOL, atol=atol)  # noqa: E731
    close(fw.weights, ref["weights"], 1e-12)
    close(fw.lse, ref["lse"], RTOL)  # an error of the sum is absolute in its logarithm
    close(fw.prob_mean, ref["prob_mean"], 1e-12)
    scale = np.abs(ref["lse"]).max() if len(ref["lse"]) else 0.0
    assert abs(float(fw.losses[0]) - ref["losses"][0]) <= 2 * RTOL * max(1.0, ref["losses"][0])
    assert abs(float(fw.losses[1]) - ref["losses"][1]) <= 2 * RTOL * (ref["losses"][1] + scale)
    assert float(fw.losses[2]) == ref["losses"][2]


def make(cuda, t, e, dtype, seed, std=2.0):
    import torch
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randn(t, e, device=cuda, generator=g) * std).to(torch_type(dtype)), g


SIZES = [(1, 1, 1), (1, 64, 2), (3, 8, 8), (5, 7, 3), (64, 64, 2), (65, 37, 5), (257, 128, 6), (999, 31, 4), (300, 256, 8),
         (33, 257, 8), (40, 512, 3), (21, 1000, 32), (9, 1024, 10), (2500, 9, 2), (4000, 64, 1)]


@pytest.mark.parametrize("normalize", [True, False], ids=["norm", "raw"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,e,k", SIZES, ids=lambda v: str(v))
def test_forward_matches_the_definition(cuda, t, e, k, dtype, normalize):
    import torch
    logits, g = make(cuda, t, e, dtype, t + e)
    mask = torch.rand(t, device=cuda, generator=g) > 0.2 if t % 2 else None
    fw = Forward(logits, k, normalize, mask, dtype)
    check_forward(fw, reference(logits, k, normalize, mask))


def test_more_slots_than_experts(cuda):
    logits, _ = make(cuda, 50, 3, "f32", 1)
    fw = Forward(logits, 5)
    check_forward(fw, reference(logits, 5, True, None))
    assert (fw.indices[:, 3:] == -1).all() and (fw.weights[:, 3:] == 0).all()


@pytest.mark.parametrize("e", [16, 600])
def test_no_tokens(cuda, e):
    import torch
    fw = Forward(torch.empty(0, e, device=cuda), 2)
    assert fw.rows.tolist() == [0] * e and fw.losses.tolist() == [0.0] * 3 and fw.prob_mean.tolist() == [0.0] * e


@pytest.mark.parametrize("t", [7, 2000])
def test_ties_go_to_the_lowest_expert_and_zeros_tie(cuda, t):
    import torch
    g = torch.Generator(device=cuda).manual_seed(3)
    logits = torch.randint(-2, 3, (t, 70), device=cuda, generator=g).float()
    logits[::3] = 0.0
    logits[::3, 1::2] = -0.0
    fw = Forward(logits, 6)
    check_forward(fw, reference(logits, 6, True, None))
    assert fw.indices[0].tolist() == [0, 1, 2, 3, 4, 5]


@pytest.mark.parametrize("e", [40, 300])
def test_masked_rows_may_hold_anything(cuda, e):
    """Tokens out of the mask with NaN and infinities, closed experts, tokens with every expert closed."""
    import torch
    t, k = 513, 4
    logits, g = make(cuda, t, e, "f32", 8)
    logits[:, 5] = -math.inf
    logits[10:20, :] = -math.inf            # nothing left: as if masked
    logits[20:30, 3:] = -math.inf           # fewer experts left than slots
    mask = torch.ones(t, dtype=torch.uint8, device=cuda)
    mask[100:140] = 0
    logits[100:110] = math.nan
    logits[110:120] = math.inf
    logits[120:130] = -math.inf
    ref = reference(logits, k, True, mask)
    fw = Forward(logits, k, True, mask)
    check_forward(fw, ref)
    grad = torch.full_like(logits, math.nan)
    gw = torch.randn(t, k, device=cuda, generator=g)
    gw[fw.indices < 0] = math.nan           # of slots without an expert: not read
    gl = torch.tensor([0.5, 0.25], device=cuda)
    assert fw.router.backward(logits, fw.indices, fw.weights, fw.rows, fw.losses, fw.lse, gw, gl, grad) == 0
    assert torch.isfinite(grad).all()
    dead = torch.from_numpy(~ref["valid"]).to(cuda)
    assert (grad[dead] == 0).all() and (grad[:, 5] == 0).all()
    all_masked = Forward(logits, k, True, torch.zeros_like(mask))
    assert all_masked.losses.tolist() == [0.0] * 3 and all_masked.rows.sum() == 0
    assert (all_masked.row_tokens == -1).all() and (all_masked.positions == -1).all()
    gw = torch.ones(t, k, device=cuda)
    assert fw.router.backward(logits, all_masked.indices, all_masked.weights, all_masked.rows, all_masked.losses,
                              all_masked.lse, gw, gl, grad) == 0
    assert (grad == 0).all()


def test_nan_and_infinity_stay_in_their_token(cuda):
    import torch
    logits, _ = make(cuda, 100, 64, "f32", 4)
    clean = Forward(logits, 2)
    bad = logits.clone()
    bad[7, 9], bad[8, 3] = math.nan, math.inf
    fw = Forward(bad, 2)
    assert fw.indices[7, 0] == 9 and fw.indices[8, 0] == 3
    assert torch.isnan(fw.weights[7]).all() and torch.isnan(fw.weights[8]).all()
    keep = torch.ones(100, dtype=torch.bool, device=cuda)
    keep[7:9] = False
    assert torch.equal(fw.indices[keep], clean.indices[keep]) and torch.equal(fw.weights[keep], clean.weights[keep])
    assert int(fw.rows.sum()) == 200


@pytest.mark.parametrize("with_weights,with_losses", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("normalize", [True, False], ids=["norm", "raw"])
@pytest.mark.parametrize("t,e,k,dtype", [(1, 1, 1, "f32"), (77, 37, 5, "f32"), (130, 64, 2, "bf16"), (64, 256, 8, "f16"),
                                         (19, 600, 7, "f32"), (500, 8, 12, "f16"), (5000, 96, 4, "bf16")])
def test_gradient_matches_the_formula(cuda, t, e, k, dtype, normalize, with_weights, with_losses):
    import torch
    logits, g = make(cuda, t, e, dtype, 5 * t + e)
    mask = torch.rand(t, device=cuda, generator=g) > 0.1 if t > 1 else None
    fw = Forward(logits, k, normalize, mask, dtype)
    ref = reference(logits, k, normalize, mask)
    gw = torch.randn(t, k, device=cuda, generator=g) if with_weights else None
    gl = torch.tensor([0.7 * t, 0.3 * t], device=cuda) if with_losses else None
    grad = torch.full_like(logits, float("nan"))
    assert fw.router.backward(logits, fw.indices, fw.weights, fw.rows, fw.losses, fw.lse, gw, gl, grad) == 0
    g0, g1 = gl.double().tolist() if with_losses else (0.0, 0.0)
    p, n = ref["p"], max(1, ref["n"])
    c = g0 * e / n * ref["f"]
    dot = p @ c
    want = p * (c - dot[:, None] + (2 * g1 / n * ref["lse"])[:, None])
    size = p * (c + dot[:, None] + np.abs(2 * g1 / n * ref["lse"])[:, None])
    if with_weights:
        ok = ref["indices"] >= 0
        gwn = np.where(ok, gw.double().cpu().numpy(), 0.0)
        part, big = ref["weights"] * gwn, ref["weights"] * np.abs(gwn)
        total, total_big = part.sum(1, keepdims=True), big.sum(1, keepdims=True)
        if normalize:
            part, big = ref["weights"] * (gwn - total), big + ref["weights"] * total_big
        else:
            want, size = want - p * total, size + p * total_big
        r, j = np.nonzero(ok)
        np.add.at(want, (r, ref["indices"][r, j]), part[r, j])
        np.add.at(size, (r, ref["indices"][r, j]), big[r, j])
    rel, least = rounding(dtype)
    got = grad.double().cpu().numpy()
    err, bound = np.abs(got - want), 3 * RTOL * size + rel * np.abs(want) + least + 1e-30
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("normalize", [True, False], ids=["norm", "raw"])
def test_gradient_matches_differences(cuda, normalize):
    """Along random directions: the change of <gw, weights> + g0 balance + g1 z, computed in 64 bits, over a
    step that changes no choice. The difference quotient's own error is of order h^2 = 1e-8."""
    import torch
    t, e, k, h = 60, 24, 3, 1e-4
    logits, g = make(cuda, t, e, "f32", 11, std=1.0)
    fw = Forward(logits, k, normalize)
    gw = torch.randn(t, k, device=cuda, generator=g)
    gl = torch.tensor([3.0, 0.5], device=cuda)
    grad = torch.empty_like(logits)
    assert fw.router.backward(logits, fw.indices, fw.weights, fw.rows, fw.losses, fw.lse, gw, gl, grad) == 0

    def goal(x):
        ref = reference(x, k, normalize, None)
        return float((ref["weights"] * gw.double().cpu().numpy()).sum() + 3.0 * ref["losses"][0] + 0.5 * ref["losses"][1])

    base = reference(logits, k, normalize, None)["indices"]
    for seed in range(4):
        d = torch.randn(t, e, device=cuda, dtype=torch.float64, generator=torch.Generator(device=cuda).manual_seed(seed))
        up, down = logits.double() + h * d, logits.double() - h * d
        for x in (up, down):
            assert (np.sort(reference(x, k, normalize, None)["indices"], 1) == np.sort(base, 1)).all()
        want = (goal(up) - goal(down)) / (2 * h)
        got = float((grad.double() * d).sum())
        assert abs(got - want) <= 1e-4 * max(1.0, abs(want))


def test_pitches_and_misaligned_rows(cuda):
    """Rows with a pitch, and a base that no vector load can take, give the bits of the packed ones."""
    import torch
    t, e, k = 321, 64, 4
    for dtype in ("f32", "f16"):
        logits, g = make(cuda, t, e, dtype, 6)
        gw, gl = torch.randn(t, k, device=cuda, generator=g), torch.tensor([1.0, 1.0], device=cuda)
        want = Forward(logits, k, dtype=dtype)
        want_grad = torch.empty_like(logits)
        args = (want.indices, want.weights, want.rows, want.losses, want.lse, gw, gl)
        assert want.router.backward(logits, *args, want_grad) == 0
        for first, pitch in ((0, 72), (1, 67), (8, 80)):
            wide = torch.full((t, pitch), float("nan"), device=cuda, dtype=logits.dtype)
            view = wide[:, first % 8:first % 8 + e]
            view.copy_(logits)
            fw = Forward(view, k, dtype=dtype)
            out = torch.full((t, pitch), 5.0, device=cuda, dtype=logits.dtype)
            grad = out[:, first % 8:first % 8 + e]
            assert fw.router.backward(view, fw.indices, fw.weights, fw.rows, fw.losses, fw.lse, gw, gl, grad) == 0
            for name in ("indices", "weights", "positions", "rows", "losses", "row_tokens", "lse", "prob_mean"):
                assert torch.equal(getattr(fw, name), getattr(want, name)), name
            assert torch.equal(grad, want_grad)
            rest = torch.ones(pitch, dtype=torch.bool, device=cuda)
            rest[first % 8:first % 8 + e] = False
            assert (out[:, rest] == 5.0).all()


def test_same_bits_again_on_a_side_stream_and_in_a_graph(cuda):
    import torch
    t, e, k = 20000, 64, 4
    logits, _ = make(cuda, t, e, "bf16", 2)
    a = Forward(logits, k, dtype="bf16")
    s = torch.cuda.Stream(cuda)
    b = Forward(logits, k, dtype="bf16", router=a.router, stream=s)
    torch.cuda.synchronize()
    names = ("indices", "weights", "positions", "rows", "losses", "row_tokens", "lse", "prob_mean")
    for name in names:
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    # fewer tokens with the same router, from a captured graph
    few, _ = make(cuda, 700, e, "bf16", 3)
    want = Forward(few, k, dtype="bf16")
    graph = torch.cuda.CUDAGraph()
    outs = [torch.zeros_like(getattr(want, n)) for n in ("indices", "weights", "positions", "rows", "losses")]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        assert a.router.run(few, *outs, stream=torch.cuda.current_stream()) == 0
    graph.replay()
    torch.cuda.synchronize()
    for n, o in zip(("indices", "weights", "positions", "rows", "losses"), outs):
        assert torch.equal(o, getattr(want, n)), n
    del graph


def test_the_plan_takes_the_counts(cuda):
    """rows and positions are what MoePlan wants: dispatched rows of an expert are its packed rows."""
    import torch
    t, e, k = 400, 12, 3
    logits, _ = make(cuda, t, e, "f32", 12)
    fw = Forward(logits, k)
    rows, tokens = fw.rows.tolist(), fw.row_tokens.tolist()
    at = 0
    for x in range(e):
        for r in range(at, at + rows[x]):
            assert x in fw.indices[tokens[r]].tolist()
        at += rows[x]
    assert at == t * k


def test_tensors_that_do_not_fit_are_refused(cuda):
    import torch
    r = gg.MoeRouter(8, 2, 16)
    ok = lambda t=4: (torch.zeros(t, 8, device=cuda), torch.zeros(t, 2, dtype=torch.int32, device=cuda),  # noqa: E731
                      torch.zeros(t, 2, device=cuda), torch.zeros(t, 2, dtype=torch.int32, device=cuda),
                      torch.zeros(8, dtype=torch.int32, device=cuda), torch.zeros(3, device=cuda))
    assert r.run(*ok()) == 0
    assert r.run(*ok(17)) == capi.CUDA_ERROR_INVALID_VALUE  # more tokens than the router was made for
    for i in range(6):
        for wrong in (lambda x: x.double(), lambda x: x.flatten()[:-1] if x.dim() == 1 else x[:, :-1], lambda x: x.cpu()):
            args = list(ok())
            args[i] = wrong(args[i])
            with pytest.raises(ValueError):
                r.run(*args)
    with pytest.raises(ValueError):
        r.run(*ok(), token_mask=torch.ones(3, dtype=torch.uint8, device=cuda))
    with pytest.raises(ValueError):
        r.run(*ok(), token_mask=torch.ones(4, device=cuda))
    r.close()
    assert r.run(*ok()) == capi.CUDA_ERROR_INVALID_DEVICE_POINTER
