"""The router over the range of its logits: a common offset far above their differences, the types' largest and
lowest finite values. Softmax does not change with a common offset, so the bounds of test_gpu_router.py
hold: RTOL for probabilities, weights and means, three of them on each term of a gradient. lse itself is one FP32 number,
off by its rounding, 2^-24 |lse|, the rounding of the sum top + log(...), as much again, and the logarithm's
2^-20 absolute.
"""
import math

import numpy as np
import pytest

from test_gpu_router import RTOL, Forward, check_forward, make, reference, rounding, torch_type

pytestmark = pytest.mark.gpu
LAYOUTS = [(5, 8, 3), (300, 64, 2), (150, 256, 8), (90, 200, 5), (40, 600, 7), (12, 1000, 20)]


def check_lse(fw, ref):
    got = fw.lse.double().cpu().numpy()
    assert (np.abs(got - ref["lse"]) <= 2.0 ** -23 * np.abs(ref["lse"]) + 2.0 ** -20).all()


def gradient(ref, gw, gl, normalize):
    """(the gradient, the sum of its terms' sizes) in 64 bits."""
    e, n = ref["p"].shape[1], max(1, ref["n"])
    p, (g0, g1) = ref["p"], gl
    c = g0 * e / n * ref["f"]
    dot = p @ c
    want = p * (c - dot[:, None] + (2 * g1 / n * ref["lse"])[:, None])
    size = p * (c + dot[:, None] + np.abs(2 * g1 / n * ref["lse"])[:, None])
    gwn = np.where(ref["indices"] >= 0, gw, 0.0)
    part, big = ref["weights"] * gwn, ref["weights"] * np.abs(gwn)
    total, total_big = part.sum(1, keepdims=True), big.sum(1, keepdims=True)
    if normalize:
        part, big = ref["weights"] * (gwn - total), big + ref["weights"] * total_big
    else:
        want, size = want - p * total, size + p * total_big
    r, j = np.nonzero(ref["indices"] >= 0)
    np.add.at(want, (r, ref["indices"][r, j]), part[r, j])
    np.add.at(size, (r, ref["indices"][r, j]), big[r, j])
    return want, size


def check_gradient(cuda, fw, logits, ref, normalize, dtype, g, gl):
    import torch
    gw = torch.randn(*fw.weights.shape, device=cuda, generator=g)
    grad = torch.full_like(logits, float("nan"))
    assert fw.router.backward(logits, fw.indices, fw.weights, fw.rows, fw.losses, fw.lse, gw, torch.tensor(gl, device=cuda), grad) == 0
    want, size = gradient(ref, gw.double().cpu().numpy(), gl, normalize)
    rel, least = rounding(dtype)
    err = np.abs(grad.double().cpu().numpy() - want)
    bound = 3 * RTOL * size + rel * np.abs(want) + least + 1e-30
    assert (err <= bound).all(), float((err / bound).max())


# offsets that the type can hold beside differences of a few units
OFFSETS = [("f32", 1e3), ("f32", -1e4), ("f32", 3e4), ("f16", -1e3), ("f16", 1e4), ("f16", -3e4), ("bf16", 1e3), ("bf16", -1e4)]


@pytest.mark.parametrize("normalize", [True, False], ids=["norm", "raw"])
@pytest.mark.parametrize("dtype,offset", OFFSETS, ids=lambda v: str(v))
@pytest.mark.parametrize("t,e,k", LAYOUTS, ids=lambda v: str(v))
def test_forward_with_a_common_offset(cuda, t, e, k, dtype, offset, normalize):
    logits, _ = make(cuda, t, e, "f32", t + e)
    logits = (logits + offset).to(torch_type(dtype))
    fw = Forward(logits, k, normalize, None, dtype)
    ref = reference(logits, k, normalize, None)
    check_forward(fw, ref)
    check_lse(fw, ref)


@pytest.mark.parametrize("normalize", [True, False], ids=["norm", "raw"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,e,k", LAYOUTS, ids=lambda v: str(v))
def test_forward_at_the_ends_of_the_type(cuda, t, e, k, dtype, normalize):
    """Masks of the type's lowest value in place of -infinity: on some experts, on all of a token's, and beside the
    largest value. A token whose logits are all the lowest is uniform over all experts."""
    import torch
    logits, _ = make(cuda, t, e, dtype, t + e)
    info = torch.finfo(logits.dtype)
    logits[:, ::3] = info.min
    logits[::4] = info.min
    logits[1::4, 1] = info.max
    logits[2::8] = info.max
    fw = Forward(logits, k, normalize, None, dtype)
    ref = reference(logits, k, normalize, None)
    for name in ("indices", "positions", "rows", "row_tokens"):
        np.testing.assert_array_equal(getattr(fw, name).cpu().numpy(), ref[name], err_msg=name)
    close = lambda a, b: np.testing.assert_allclose(a.double().cpu().numpy(), b, rtol=RTOL, atol=1e-12)  # noqa: E731
    close(fw.weights, ref["weights"])
    close(fw.prob_mean, ref["prob_mean"])
    check_lse(fw, ref)
    assert abs(float(fw.losses[0]) - ref["losses"][0]) <= 2 * RTOL * max(1.0, ref["losses"][0])
    z = ref["losses"][1]
    if z > 2 * torch.finfo(torch.float32).max:  # the mean of lse^2 is past FP32
        assert float(fw.losses[1]) == math.inf
    else:
        assert abs(float(fw.losses[1]) - z) <= 2 * RTOL * z
    assert float(fw.losses[2]) == t


@pytest.mark.parametrize("normalize", [True, False], ids=["norm", "raw"])
@pytest.mark.parametrize("dtype,offset", OFFSETS, ids=lambda v: str(v))
@pytest.mark.parametrize("t,e,k", LAYOUTS, ids=lambda v: str(v))
def test_gradient_with_a_common_offset(cuda, t, e, k, dtype, offset, normalize):
    logits, g = make(cuda, t, e, "f32", t + e)
    logits = (logits + offset).to(torch_type(dtype))
    fw = Forward(logits, k, normalize, None, dtype)
    ref = reference(logits, k, normalize, None)
    check_gradient(cuda, fw, logits, ref, normalize, dtype, g, [0.7 * t, 0.0])
    check_gradient(cuda, fw, logits, ref, normalize, dtype, g, [0.7 * t, 0.3 * t / abs(offset)])


@pytest.mark.parametrize("normalize", [True, False], ids=["norm", "raw"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("t,e,k", LAYOUTS, ids=lambda v: str(v))
def test_gradient_at_the_ends_of_the_type(cuda, t, e, k, dtype, normalize):
    import torch
    logits, g = make(cuda, t, e, dtype, t + e)
    info = torch.finfo(logits.dtype)
    logits[:, ::3] = info.min
    logits[::4] = info.min
    logits[1::4, 1] = info.max
    logits[2::8] = info.max
    fw = Forward(logits, k, normalize, None, dtype)
    check_gradient(cuda, fw, logits, reference(logits, k, normalize, None), normalize, dtype, g, [0.7 * t, 0.0])
