"""The layer of examples/moe_layer.py, which runs the router, the row moves, the grouped product and the 4-bit
experts together, against the same layer in 64 bits.

What is rounded: the packed values and gradients to FP16, at most six times between an input and a result
(up, down, combine; combine's gradient, two products, dispatch's), each by 2^-11 of its size; as errors of random
sign that is sqrt(6) 2^-11 = 1.2e-3 of a result's norm. 3e-3 bounds it.
"""
import importlib.util
import os

import pytest

import grouped_gemm_gpu_kernel_b200 as gg

pytestmark = pytest.mark.gpu
BOUND = 3e-3


@pytest.fixture(scope="module")
def layer_module():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "moe_layer.py")
    spec = importlib.util.spec_from_file_location("moe_layer", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def reference(x, gate, up, down, top_k, mask):
    """(y, losses) in 64 bits, differentiable."""
    import torch
    logits = x @ gate.t()
    lse = torch.logsumexp(logits, 1)
    p = torch.exp(logits - lse[:, None])
    top, index = logits.topk(top_k, dim=1)
    w = torch.softmax(top, 1) * mask[:, None]
    y = torch.zeros_like(x)
    experts = up.shape[0]
    rows = torch.zeros(experts, device=x.device, dtype=torch.float64)
    for e in range(experts):
        t, j = ((index == e) & mask[:, None].bool()).nonzero(as_tuple=True)
        rows[e] = len(t)
        y = y.index_add(0, t, torch.relu(x[t] @ up[e]) @ down[e] * w[t, j][:, None])
    n = mask.sum()
    mean = (p * mask[:, None]).sum(0) / n
    balance = experts * (rows / rows.sum() * mean).sum()
    return y, balance, (lse * lse * mask).sum() / n, rows


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k,masked", [(256, 128, 256, 8, 2, False), (333, 264, 136, 5, 3, True)])
def test_training_step(cuda, layer_module, tokens, hidden, inner, experts, top_k, masked):
    import torch
    gate, up, down = layer_module.weights(experts, hidden, inner, seed=tokens)
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(tokens, hidden, device=cuda, generator=g).half()
    mask = (torch.rand(tokens, device=cuda, generator=g) > 0.2).to(torch.uint8) if masked else None
    grad_y = torch.randn(tokens, hidden, device=cuda, generator=g).half()
    layer = layer_module.MoeLayer(gate, up, down, top_k, tokens, balance=0.5, z=0.25)
    y = layer.forward(x, mask)
    grads = layer.backward(grad_y)

    leaf = [t.double().requires_grad_(True) for t in (x, gate, up, down)]
    m = mask.double() if masked else torch.ones(tokens, device=cuda, dtype=torch.float64)
    want, balance, z, rows = reference(*leaf, top_k, m)
    goal = (want * grad_y.double()).sum() + 0.5 * balance + 0.25 * z
    wanted = torch.autograd.grad(goal, leaf)
    assert layer.rows.tolist() == rows.long().tolist()
    assert abs(float(layer.losses[0]) - float(balance.detach())) < 1e-4
    assert abs(float(layer.losses[1]) - float(z.detach())) < 1e-3
    assert off(y, want.detach()) < BOUND
    for name, a, b in zip(("x", "gate", "up", "down"), grads, wanted):
        assert off(a, b) < BOUND, name


@pytest.mark.parametrize("tokens", [1, 3, 16])
def test_decoding_step(cuda, layer_module, tokens):
    import torch
    experts, hidden, inner, group = 8, 256, 512, 64
    gate, up, down = layer_module.weights(experts, hidden, inner, seed=2)
    decoder = layer_module.MoeDecoder(gate, up, down, 2, tokens, group)
    x = torch.randn(tokens, hidden, device=cuda, generator=torch.Generator(device=cuda).manual_seed(tokens)).half()
    dense = []
    for q, scales in decoder.quantized:
        both = torch.stack([q & 15, q >> 4], 3).flatten(2).double() - 8
        dense.append((both * scales.double().repeat_interleave(group, 2)).transpose(1, 2))
    want = reference(x.double(), gate.double(), dense[0], dense[1], 2, torch.ones(tokens, device=cuda, dtype=torch.float64))[0]
    for _ in range(2):
        assert off(decoder.step(x), want) < BOUND
    # captured in a graph, as a decoding loop runs it
    s, graph, y = torch.cuda.Stream(cuda), torch.cuda.CUDAGraph(), torch.zeros_like(x)
    logits = x.float() @ gate.t()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        st = torch.cuda.current_stream()
        d = decoder
        assert d.router.run(logits, d.indices, d.weights, d.positions, d.rows, d.losses, row_tokens=d.row_tokens, stream=st) == 0
        assert d.plans[0].run(x, d.rows, d.h, row_tokens=d.row_tokens, stream=st) == 0
        assert d.plans[1].run(d.h, d.rows, d.out, stream=st) == 0
        assert gg.moe_combine(d.out, d.positions, y, d.weights, stream=st) == 0
    decoder.h.fill_(float("nan")), decoder.out.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert off(y, want) < BOUND
    del graph
