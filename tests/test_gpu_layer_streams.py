"""The layers of the examples under `with torch.cuda.stream(...)`, whose work torch puts on that stream: behind work that takes a while
they give the bits of the default stream, where nothing had to wait.
"""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


def example(name):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", name + ".py")
    spec = importlib.util.spec_from_file_location(name, path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def on_a_stream(step, inputs):
    """step(*inputs) on a stream whose inputs are written late, and on the default stream."""
    import torch
    want = [t.clone() for t in step(*inputs)]
    late = [torch.zeros_like(t) for t in inputs]
    step(*late)  # the step's own buffers hold other rows'
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(50_000_000)
        for a, b in zip(late, inputs):
            a.copy_(b)
        got = step(*late)
    torch.cuda.synchronize()
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def rows(cuda, count, *shape):
    import torch
    g = torch.Generator(device=cuda).manual_seed(8)
    return [torch.randn(*shape, device=cuda, generator=g) for _ in range(count)]


def test_gated_training_step(cuda):
    m = example("gated_moe_layer")
    layer = m.GatedMoeLayer(*m.weights(4, 128, 256, seed=1), top_k=2, tokens=200)

    def step(x, r, gh, gy):
        h, y = layer.forward(x, r)
        return (h, y, *layer.backward(gh, gy))

    on_a_stream(step, [t.bfloat16() for t in rows(cuda, 4, 200, 128)])


def test_gated_serving_step(cuda):
    m = example("gated_moe_layer")
    server = m.GatedMoeServer(*m.weights(4, 128, 256, seed=2), top_k=2, tokens=9)
    on_a_stream(server.step, [t.bfloat16() for t in rows(cuda, 2, 9, 128)])


def test_training_step(cuda):
    m = example("moe_layer")
    layer = m.MoeLayer(*m.weights(4, 128, 256, seed=3), top_k=2, tokens=200)

    def step(x, gy):
        y = layer.forward(x)
        return (y, *layer.backward(gy))

    on_a_stream(step, [t.half() for t in rows(cuda, 2, 200, 128)])


def test_decoding_step(cuda):
    m = example("moe_layer")
    decoder = m.MoeDecoder(*m.weights(4, 128, 256, seed=4), top_k=2, tokens=5)
    on_a_stream(lambda x: (decoder.step(x),), [t.half() for t in rows(cuda, 1, 5, 128)])
