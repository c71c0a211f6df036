"""A mixture-of-experts layer on the package's operators: a training step, and decoding with 4-bit experts.

    y[t] = sum over the top_k experts e of token t:  w(t, e) * relu(x[t] @ up[e]) @ down[e]

Training runs router -> dispatch -> grouped product (MoePlan) up and down -> combine, and back: the gradients of
the combine, of both products (the grouped kernel on the transposed weights, read in place as column-major
operands, and on the transposed rows for the weights), of the dispatch and of the router with its balance and
z losses. Row counts stay on the device, but for the products of the weights' gradients, whose inner
dimension they are. Decoding reads the tokens' rows straight into the 4-bit product.

    python examples/moe_layer.py
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import grouped_gemm_gpu_kernel_b200 as gg  # noqa: E402


def _done(status: int) -> None:
    if status != 0:
        raise RuntimeError(f"status {status}")


def _stream():
    """The stream that torch's own operations between the calls run on."""
    return torch.cuda.current_stream()


class MoeLayer:
    """FP16 experts up (experts, hidden, inner) and down (experts, inner, hidden), FP32 gate (experts, hidden)."""

    def __init__(self, gate, up, down, top_k: int, tokens: int, balance: float = 0.01, z: float = 0.001):
        self.gate, self.up, self.down, self.top_k, self.tokens = gate, up, down, top_k, tokens
        self.experts, self.hidden, self.inner = up.shape
        dev, rows = up.device, tokens * top_k
        f32 = lambda *s: torch.empty(*s, device=dev)  # noqa: E731
        f16 = lambda *s: torch.empty(*s, device=dev, dtype=torch.float16)  # noqa: E731
        i32 = lambda *s: torch.empty(*s, device=dev, dtype=torch.int32)  # noqa: E731
        self.router = gg.MoeRouter(self.experts, top_k, tokens)
        self.indices, self.positions, self.rows = i32(tokens, top_k), i32(tokens, top_k), i32(self.experts)
        self.weights, self.losses, self.lse, self.prob_mean = f32(tokens, top_k), f32(3), f32(tokens), f32(self.experts)
        self.grad_losses = torch.tensor([balance, z], device=dev)
        self.packed, self.h, self.out = f16(rows, self.hidden), f16(rows, self.inner), f16(rows, self.hidden)
        self.grad_h, self.grad_packed = f16(rows, self.inner), f16(rows, self.hidden)
        self.grad_weights, self.grad_logits = f32(tokens, top_k), f32(tokens, self.experts)
        self.up_plan = self._plan(self.packed, self.up, self.h, act=gg.Activation.kReLU)
        self.down_plan = self._plan(self.h, self.down, self.out)
        self.down_back = self._plan(self.out, self.down, self.grad_h, transposed=True)
        self.up_back = self._plan(self.grad_h, self.up, self.grad_packed, transposed=True)

    def _plan(self, a, w, d, act=gg.Activation.kNone, transposed=False):
        """d[rows of e] = act(a[rows of e] @ w[e]), or @ w[e]^T: w as it stands, a column-major operand."""
        cfg = gg.KernelConfig(128, 128, 64, output_type=gg.OutputType.kF16, activation=act,
                              b_layout=gg.Layout.kColMajor if transposed else gg.Layout.kRowMajor)
        return gg.MoePlan(self.experts, d.shape[1], a.shape[1], a.shape[0], a.data_ptr(), a.shape[1],
                          [x.data_ptr() for x in w], w.shape[2], d.data_ptr(), d.shape[1], config=cfg)

    def forward(self, x, mask=None):
        """x (tokens, hidden) FP16 -> y; mask: tokens to leave out (0)."""
        self.x, self.logits = x, x.float() @ self.gate.t()
        _done(self.router.run(self.logits, self.indices, self.weights, self.positions, self.rows, self.losses, lse=self.lse,
                              prob_mean=self.prob_mean, token_mask=mask, stream=_stream()))
        _done(gg.moe_dispatch(x, self.positions, self.packed, stream=_stream()))
        _done(self.up_plan.run(self.rows, stream=_stream()))
        _done(self.down_plan.run(self.rows, stream=_stream()))
        y = torch.empty_like(x)
        _done(gg.moe_combine(self.out, self.positions, y, self.weights, stream=_stream()))
        return y

    def backward(self, grad_y):
        """Gradients (x, gate, up, down) of <grad_y, y> + balance * losses[0] + z * losses[1]."""
        # the gradient of the experts' rows takes the place of their values
        _done(gg.moe_combine_backward(grad_y, self.out, self.positions, self.weights, self.out, self.grad_weights, stream=_stream()))
        _done(self.down_back.run(self.rows, stream=_stream()))
        self.grad_h.mul_(self.h > 0)
        _done(self.up_back.run(self.rows, stream=_stream()))
        _done(self.router.backward(self.logits, self.indices, self.weights, self.rows, self.losses, self.lse, self.grad_weights,
                                   self.grad_losses, self.grad_logits, stream=_stream()))
        grad_x = torch.empty_like(self.x)
        _done(gg.moe_combine(self.grad_packed, self.positions, grad_x, stream=_stream()))
        grad_x = (grad_x.float() + self.grad_logits @ self.gate).half()
        counts = self.rows.tolist()
        return (grad_x, self.grad_logits.t() @ self.x.float(), self._weight_gradient(self.packed, self.grad_h, counts),
                self._weight_gradient(self.h, self.out, counts))

    def _weight_gradient(self, a, g, counts):
        """a[rows of e]^T @ g[rows of e] for every expert, FP32, as one grouped launch."""
        d = torch.zeros(self.experts, a.shape[1], g.shape[1], device=a.device)
        problems, at = [], 0
        for e, r in enumerate(counts):
            if r:
                problems.append(gg.ProblemDesc(a.shape[1], g.shape[1], r, a[at:].data_ptr(), g[at:].data_ptr(), None,
                                               d[e].data_ptr(), a.shape[1], g.shape[1], g.shape[1], g.shape[1]))
            at += r
        cfg = gg.KernelConfig(128, 128, 64, a_layout=gg.Layout.kColMajor)
        _done(gg.run_grouped_gemm_once(problems, gg.SortMode.kByTiles, cfg, stream=_stream()))
        return d


def quantize(w, group: int):
    """(packed 4-bit weights, FP16 scales) of w (experts, outputs, inputs): symmetric, zero at 8."""
    e, n, k = w.shape
    groups = w.float().view(e, n, k // group, group)
    scales = (groups.abs().amax(3) / 7.0).clamp(min=1e-6).half()
    q = (torch.round(groups / scales.float()[..., None]) + 8).clamp(0, 15).to(torch.uint8).view(e, n, k)
    return q[:, :, 0::2] | q[:, :, 1::2] << 4, scales


class MoeDecoder:
    """The same layer with experts in 4 bits, for a few tokens at a time; every step is five launches."""

    def __init__(self, gate, up, down, top_k: int, tokens: int, group: int = 64):
        self.gate, self.top_k = gate, top_k
        experts, hidden, inner = up.shape
        dev, rows = up.device, tokens * top_k
        self.quantized = [quantize(w.transpose(1, 2).contiguous(), group) for w in (up, down)]
        each = lambda t: [x.data_ptr() for x in t]  # noqa: E731
        self.plans = [gg.Q4Plan(experts, n, k, group, each(q), k // 2, each(s), output_type=gg.OutputType.kF16, activation=act)
                      for (q, s), n, k, act in zip(self.quantized, (inner, hidden), (hidden, inner),
                                                   (gg.Activation.kReLU, gg.Activation.kNone))]
        i32 = lambda *s: torch.empty(*s, device=dev, dtype=torch.int32)  # noqa: E731
        self.router = gg.MoeRouter(experts, top_k, tokens)
        self.indices, self.positions, self.row_tokens, self.rows = i32(tokens, top_k), i32(tokens, top_k), i32(rows), i32(experts)
        self.weights, self.losses = torch.empty(tokens, top_k, device=dev), torch.empty(3, device=dev)
        self.h = torch.empty(rows, inner, device=dev, dtype=torch.float16)
        self.out = torch.empty(rows, hidden, device=dev, dtype=torch.float16)

    def step(self, x):
        logits = x.float() @ self.gate.t()
        _done(self.router.run(logits, self.indices, self.weights, self.positions, self.rows, self.losses, row_tokens=self.row_tokens, stream=_stream()))
        _done(self.plans[0].run(x, self.rows, self.h, row_tokens=self.row_tokens, stream=_stream()))
        _done(self.plans[1].run(self.h, self.rows, self.out, stream=_stream()))
        y = torch.empty_like(x)
        _done(gg.moe_combine(self.out, self.positions, y, self.weights, stream=_stream()))
        return y


def weights(experts: int, hidden: int, inner: int, device="cuda", seed: int = 0):
    g = torch.Generator(device=device).manual_seed(seed)
    make = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    return (make(experts, hidden) * hidden ** -0.5, (make(experts, hidden, inner) * hidden ** -0.5).half(),
            (make(experts, inner, hidden) * inner ** -0.5).half())


def main() -> None:
    gate, up, down = weights(8, 1024, 2048)
    layer = MoeLayer(gate, up, down, top_k=2, tokens=2048)
    x = torch.randn(2048, 1024, device="cuda").half()
    y = layer.forward(x)
    grad_x, grad_gate, grad_up, grad_down = layer.backward(torch.ones_like(y))
    print("training step: rows per expert", layer.rows.tolist(), "balance loss %.4f, z loss %.4f" % tuple(layer.losses[:2].tolist()),
          "gradient norms", ["%.3g" % g.float().norm() for g in (grad_x, grad_gate, grad_up, grad_down)])
    decoder = MoeDecoder(gate, up, down, top_k=2, tokens=4)
    few = decoder.step(x[:4])
    print("decoding in 4 bits: relative difference to FP16 experts %.3g" % float((few - y[:4]).float().norm() / y[:4].float().norm()))


if __name__ == "__main__":
    main()
