"""The layer of examples/gated_moe_layer.py, which runs the norm, the router, the row moves, the gated block, the grouped product
and the 8-bit products together, against the same layer in 64 bits.

Training: what is rounded to BF16 between an input and a result is at most eight values in a row (h, n, gate or up, mid, out, and
back as many as gradients), each by 2^-8 at most, of random sign: sqrt(8) 2^-8 / sqrt(3) = 6.4e-3 of a result's norm if every one
were uniform in its half step; 1e-2 bounds it. The router's choice is that of the stored n, as the reference takes it.

Serving: E4M3 rounds a value by 2^-4 at most, 2^-4 / sqrt(3) = 0.036 in the mean. A sum of products of random sign is as far
off, relative to its norm, as its factors: gate and up by 0.036 each, their product by sqrt(1.13^2 + 1) times that, 0.054, and rounded
to 8 bits sqrt(0.054^2 + 0.036^2) = 0.065; 0.1 bounds it. The weights of the reference are the 8-bit ones.
"""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def module():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "gated_moe_layer.py")
    spec = importlib.util.spec_from_file_location("gated_moe_layer", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def reference(x, residual, norm, gate, wg, wu, wd, index):
    """(h, y, balance, z) in 64 bits, differentiable; index: the experts of each token."""
    import torch
    h = x + residual
    n = h * (h.square().mean(1, keepdim=True) + 1e-6).rsqrt() * norm
    logits = n @ gate.t()
    lse = torch.logsumexp(logits, 1)
    p = torch.exp(logits - lse[:, None])
    w = torch.softmax(logits.gather(1, index), 1)
    y = torch.zeros_like(x)
    experts = wg.shape[0]
    rows = torch.bincount(index.reshape(-1), minlength=experts).double()
    for e in range(experts):
        t, j = (index == e).nonzero(as_tuple=True)
        g = n[t] @ wg[e]
        y = y.index_add(0, t, (g * torch.sigmoid(g) * (n[t] @ wu[e])) @ wd[e] * w[t, j][:, None])
    balance = experts * (rows / rows.sum() * p.mean(0)).sum()
    return h, y, balance, (lse * lse).mean()


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("tokens,hidden,inner,experts,top_k", [(256, 128, 256, 8, 2), (333, 264, 136, 5, 3), (2048, 256, 384, 4, 2)])
def test_training_step(cuda, module, tokens, hidden, inner, experts, top_k):
    import torch
    w = module.weights(experts, hidden, inner, seed=tokens)
    g = torch.Generator(device=cuda).manual_seed(1)
    x, r, gh, gy = [torch.randn(tokens, hidden, device=cuda, generator=g).bfloat16() for _ in range(4)]
    layer = module.GatedMoeLayer(*w, top_k=top_k, tokens=tokens, balance=0.5, z=0.25)
    h, y = layer.forward(x, r)
    h, y = h.clone(), y.clone()
    index = layer.indices.long()
    grads = layer.backward(gh, gy)
    leaf = [t.double().requires_grad_(True) for t in (x, *w)]
    wh, wy, balance, z = reference(leaf[0], r.double(), *leaf[1:], index)
    goal = (wh * gh.double()).sum() + (wy * gy.double()).sum() + 0.5 * balance + 0.25 * z
    wanted = torch.autograd.grad(goal, leaf)
    assert off(h, wh.detach()) < 1e-2 and off(y, wy.detach()) < 1e-2
    for name, a, b in zip(("x", "norm", "gate", "wg", "wu", "wd"), grads, wanted):
        assert off(a, b) < 1e-2, name


@pytest.mark.parametrize("tokens,hidden,inner", [(1, 256, 512), (7, 272, 400), (64, 1024, 640)])
def test_serving_step(cuda, module, tokens, hidden, inner):
    import torch
    experts, top_k = 8, 2
    w = module.weights(experts, hidden, inner, seed=3)
    server = module.GatedMoeServer(*w, top_k=top_k, tokens=tokens)
    g = torch.Generator(device=cuda).manual_seed(tokens)
    x, r = [torch.randn(tokens, hidden, device=cuda, generator=g).bfloat16() for _ in range(2)]
    h, y = server.step(x, r)
    dense = []
    for q, s in server.quantized:
        wide = s.double().repeat_interleave(128, 1)[:, :q.shape[1]].repeat_interleave(128, 2)[:, :, :q.shape[2]]
        dense.append((q.double() * wide).transpose(1, 2))
    want = reference(x.double(), r.double(), w[0].double(), w[1].double(), *dense, server.indices.long())
    assert off(h, want[0]) < 1e-2 and off(y, want[1]) < 0.1
    # captured in a graph, as a serving loop runs it: the same bits
    first = y.clone()
    logits, out = server.n.float() @ server.gate.t(), torch.zeros_like(x)
    s, graph = torch.cuda.Stream(cuda), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        server.step(x, r, logits=logits, y=out, stream=torch.cuda.current_stream())
    for t in (server.h, server.n, server.out, server.mid_s, server.packed_s):
        t.fill_(float("nan"))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    assert server.gate_up.status() == 0 and server.down.status() == 0
    del graph


@pytest.mark.parametrize("tokens,hidden,inner", [(1, 256, 512), (64, 1024, 640)])
def test_captured_serving_step_routes_its_own_rows(cuda, module, tokens, hidden, inner):
    """A captured step, replayed on rows that it was not captured with, gives what a step on them gives, bit for bit: the logits are
    those of the rows of the replay. With logits of the server's and with the caller's."""
    import torch
    w = module.weights(8, hidden, inner, seed=5)
    server = module.GatedMoeServer(*w, top_k=2, tokens=tokens)
    g = torch.Generator(device=cuda).manual_seed(tokens)
    make = lambda: torch.randn(tokens, hidden, device=cuda, generator=g).bfloat16()  # noqa: E731
    x, r, out = make(), make(), torch.zeros(tokens, hidden, device=cuda, dtype=torch.bfloat16)
    for logits in (None, torch.full((tokens, 8), float("nan"), device=cuda)):
        s, graph = torch.cuda.Stream(cuda), torch.cuda.CUDAGraph()
        server.step(x, r)  # what a first call sets up
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=s):
            server.step(x, r, logits=logits, y=out, stream=torch.cuda.current_stream())
        for _ in range(3):
            x.copy_(make()), r.copy_(make())
            h, y = server.step(x, r)
            h, y, indices, kept = h.clone(), y.clone(), server.indices.clone(), server.logits.clone()
            for t in (server.h, server.n, server.out, server.mid_s, server.packed_s, server.logits):
                t.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(server.logits if logits is None else logits, kept) and torch.equal(server.indices, indices)
            assert torch.equal(server.h, h) and torch.equal(out, y)
        del graph
    assert server.gate_up.status() == 0 and server.down.status() == 0


def test_serving_step_on_a_stream(cuda, module):
    """Without logits from outside, on a stream that is neither torch's current one nor the default, behind work that takes a while:
    the same bits as on the default stream."""
    import torch
    server = module.GatedMoeServer(*module.weights(8, 256, 512, seed=6), top_k=2, tokens=16)
    g = torch.Generator(device=cuda).manual_seed(6)
    x, r = [torch.randn(16, 256, device=cuda, generator=g).bfloat16() for _ in range(2)]
    h, y = [t.clone() for t in server.step(x, r)]
    late_x, late_r = torch.zeros_like(x), torch.zeros_like(r)
    server.step(late_x, late_r)
    torch.cuda.synchronize()
    s = torch.cuda.Stream(cuda)
    with torch.cuda.stream(s):
        torch.cuda._sleep(50_000_000)
        late_x.copy_(x), late_r.copy_(r)
    got = server.step(late_x, late_r, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(got[0], h) and torch.equal(got[1], y)
