"""A gated mixture-of-experts layer with the norm before it: a training step in BF16, and serving with 8-bit rows and
weights that have a scale for each block of 128.

    h = x + residual,  n = norm(h),  y[t] = sum over the top_k experts e of token t:  w(t, e) * (silu(n Wg_e) * (n Wu_e)) Wd_e

Training runs norm -> router -> dispatch -> gated block (GatedPlan) -> way down (MoePlan) -> combine, and back. Row counts
stay on the device but for the gradient of Wd, whose inner dimension they are. Serving runs norm (rows in 16 bits for the router
and in 8 for the experts) -> router -> dispatch of rows and scales -> gated 8-bit product, into 8 bits -> 8-bit product
-> combine: eight launches a step beside the logits' product, all on one stream, so that a step can be captured in a graph.

    python examples/gated_moe_layer.py
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import grouped_gemm_gpu_kernel_b200 as gg  # noqa: E402

BLOCK = 128
EPS = 1e-6


def _done(status: int) -> None:
    if status != 0:
        raise RuntimeError(f"status {status}")


def _stream():
    """The stream that torch's own operations between the calls run on."""
    return torch.cuda.current_stream()


def _ptrs(t):
    return [x.data_ptr() for x in t]


class GatedMoeLayer:
    """BF16 experts wg, wu (experts, hidden, inner), wd (experts, inner, hidden), norm weight (hidden); FP32 router gate (experts, hidden).
    hidden and inner: multiples of 8."""

    def __init__(self, norm, gate, wg, wu, wd, top_k: int, tokens: int, balance: float = 0.01, z: float = 0.001):
        self.norm_weight, self.gate, self.wg, self.wu, self.wd, self.top_k = norm, gate, wg, wu, wd, top_k
        self.experts, self.hidden, self.inner = wg.shape
        dev, rows = wg.device, tokens * top_k
        f32 = lambda *s: torch.empty(*s, device=dev)  # noqa: E731
        b16 = lambda *s: torch.empty(*s, device=dev, dtype=torch.bfloat16)  # noqa: E731
        i32 = lambda *s: torch.empty(*s, device=dev, dtype=torch.int32)  # noqa: E731
        self.norm = gg.RmsNorm(self.hidden, dtype=gg.OutputType.kBF16, eps=EPS)
        self.router = gg.MoeRouter(self.experts, top_k, tokens)
        self.block = gg.GatedPlan(self.experts, self.inner, self.hidden, _ptrs(wg), _ptrs(wu), self.inner)
        self.h, self.n, self.rstd = b16(tokens, self.hidden), b16(tokens, self.hidden), f32(tokens)
        self.indices, self.positions, self.rows = i32(tokens, top_k), i32(tokens, top_k), i32(self.experts)
        self.weights, self.losses, self.lse = f32(tokens, top_k), f32(3), f32(tokens)
        self.grad_losses = torch.tensor([balance, z], device=dev)
        self.packed, self.out = b16(rows, self.hidden), b16(rows, self.hidden)
        self.mid, self.gate_out, self.up_out, self.grad_mid = (b16(rows, self.inner) for _ in range(4))
        self.grad_packed, self.grad_weights, self.grad_logits = b16(rows, self.hidden), f32(tokens, top_k), f32(tokens, self.experts)
        self.down = self._plan(self.mid, wd, self.out)
        self.down_back = self._plan(self.out, wd, self.grad_mid, transposed=True)

    def _plan(self, a, w, d, transposed=False):
        cfg = gg.KernelConfig(128, 128, 64, input_type=gg.InputType.kBF16, output_type=gg.OutputType.kBF16,
                              b_layout=gg.Layout.kColMajor if transposed else gg.Layout.kRowMajor)
        return gg.MoePlan(self.experts, d.shape[1], a.shape[1], a.shape[0], a.data_ptr(), a.shape[1], _ptrs(w), w.shape[2], d.data_ptr(),
                          d.shape[1], config=cfg)

    def forward(self, x, residual):
        """(tokens, hidden) BF16 -> (h, y)"""
        _done(self.norm.run(x, self.norm_weight, y=self.n, residual=residual, residual_out=self.h, rstd=self.rstd, stream=_stream()))
        self.logits = self.n.float() @ self.gate.t()
        _done(self.router.run(self.logits, self.indices, self.weights, self.positions, self.rows, self.losses, lse=self.lse, stream=_stream()))
        _done(gg.moe_dispatch(self.n, self.positions, self.packed, stream=_stream()))
        _done(self.block.run(self.packed, self.rows, self.mid, gate=self.gate_out, up=self.up_out, stream=_stream()))
        _done(self.down.run(self.rows, stream=_stream()))
        y = torch.empty_like(x)
        _done(gg.moe_combine(self.out, self.positions, y, self.weights, stream=_stream()))
        return self.h, y

    def backward(self, grad_h, grad_y):
        """Gradients (x, norm weight, gate, wg, wu, wd) of <grad_h, h> + <grad_y, y> + balance * losses[0] + z * losses[1]; the
        residual's is x's."""
        _done(gg.moe_combine_backward(grad_y, self.out, self.positions, self.weights, self.out, self.grad_weights, stream=_stream()))
        _done(self.down_back.run(self.rows, stream=_stream()))
        grad_wg, grad_wu = torch.empty_like(self.wg), torch.empty_like(self.wu)
        # grad_gate and grad_up take the places of gate and up
        _done(self.block.backward(self.packed, self.gate_out, self.up_out, self.grad_mid, self.rows, self.gate_out, self.up_out,
                                  grad_x=self.grad_packed, grad_gate_w=grad_wg, grad_up_w=grad_wu, stream=_stream()))
        _done(self.router.backward(self.logits, self.indices, self.weights, self.rows, self.losses, self.lse, self.grad_weights,
                                   self.grad_losses, self.grad_logits, stream=_stream()))
        grad_n = torch.empty_like(self.n)
        _done(gg.moe_combine(self.grad_packed, self.positions, grad_n, stream=_stream()))
        grad_n = (grad_n.float() + self.grad_logits @ self.gate).bfloat16()
        grad_x, grad_norm = torch.empty_like(self.h), torch.empty(self.hidden, device=self.h.device)
        _done(self.norm.backward(self.h, self.norm_weight, self.rstd, grad_n, grad_x, grad_weight=grad_norm, grad_h=grad_h, stream=_stream()))
        return grad_x, grad_norm, self.grad_logits.t() @ self.n.float(), grad_wg, grad_wu, self._down_gradient()

    def _down_gradient(self):
        """mid[rows of e]^T @ grad_out[rows of e] for every expert, FP32, as one grouped launch."""
        d = torch.zeros(self.experts, self.inner, self.hidden, device=self.mid.device)
        problems, at = [], 0
        for e, r in enumerate(self.rows.tolist()):
            if r:
                problems.append(gg.ProblemDesc(self.inner, self.hidden, r, self.mid[at:].data_ptr(), self.out[at:].data_ptr(), None,
                                               d[e].data_ptr(), self.inner, self.hidden, self.hidden, self.hidden))
            at += r
        cfg = gg.KernelConfig(128, 128, 64, input_type=gg.InputType.kBF16, a_layout=gg.Layout.kColMajor)
        _done(gg.run_grouped_gemm_once(problems, gg.SortMode.kByTiles, cfg, stream=_stream()))
        return d


def quantize(w):
    """(8-bit weights (experts, outputs, inputs), FP32 scales for each block of 128 x 128) of w (experts, inputs, outputs)."""
    w = w.transpose(1, 2).float()
    e, n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    pad = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(e, nb, BLOCK, kb, BLOCK)
    scales = (pad.abs().amax((2, 4)) / 448.0).clamp(min=1e-12)
    q = (pad / scales[:, :, None, :, None]).to(torch.float8_e4m3fn).view(e, nb * BLOCK, kb * BLOCK)
    return q[:, :n, :k].contiguous(), scales


class GatedMoeServer:
    """The same layer on 8-bit experts, for up to `tokens` tokens a step. hidden and inner: multiples of 16."""

    def __init__(self, norm, gate, wg, wu, wd, top_k: int, tokens: int):
        self.norm_weight, self.gate = norm, gate
        experts, hidden, inner = wg.shape
        dev, rows = wg.device, tokens * top_k
        f32 = lambda *s: torch.empty(*s, device=dev)  # noqa: E731
        e4m3 = lambda *s: torch.empty(*s, device=dev, dtype=torch.float8_e4m3fn)  # noqa: E731
        b16 = lambda *s: torch.empty(*s, device=dev, dtype=torch.bfloat16)  # noqa: E731
        i32 = lambda *s: torch.empty(*s, device=dev, dtype=torch.int32)  # noqa: E731
        blocks = lambda n: -(-n // BLOCK)  # noqa: E731
        self.quantized = [quantize(w) for w in (wg, wu, wd)]
        (qg, sg), (qu, su), (qd, sd) = self.quantized
        self.norm = gg.RmsNorm(hidden, dtype=gg.OutputType.kBF16, eps=EPS)
        self.router = gg.MoeRouter(experts, top_k, tokens)
        self.gate_up = gg.F8Plan(experts, inner, hidden, _ptrs(qg), hidden, _ptrs(sg), up_ptrs=_ptrs(qu), up_scale_ptrs=_ptrs(su),
                                 output_type=gg.OutputType.kE4M3, activation=gg.Activation.kSiLU)
        self.down = gg.F8Plan(experts, hidden, inner, _ptrs(qd), inner, _ptrs(sd))
        self.h, self.n, self.q, self.s = b16(tokens, hidden), b16(tokens, hidden), e4m3(tokens, hidden), f32(tokens, blocks(hidden))
        self.indices, self.positions, self.rows = i32(tokens, top_k), i32(tokens, top_k), i32(experts)
        self.weights, self.losses, self.logits = f32(tokens, top_k), f32(3), f32(tokens, experts)
        self.packed, self.packed_s = e4m3(rows, hidden), f32(rows, blocks(hidden))
        self.mid, self.mid_s, self.out = e4m3(rows, inner), f32(rows, blocks(inner)), b16(rows, hidden)

    def step(self, x, residual, logits=None, y=None, stream=None):
        """(tokens, hidden) BF16 -> (h, y). logits: (tokens, experts) FP32, where the step puts the router's logits (None: a buffer of
        the server's); y: where it puts y. stream: a torch stream (None: torch's current one). Everything runs on it, the
        logits' product too, so that a captured step routes what its inputs hold when it is replayed."""
        stream = _stream() if stream is None else stream
        with torch.cuda.stream(stream):
            logits = self.logits if logits is None else logits
            _done(self.norm.run(x, self.norm_weight, y=self.n, residual=residual, residual_out=self.h, q=self.q, scales=self.s, stream=stream))
            torch.mm(self.n.float(), self.gate.t(), out=logits)
            _done(self.router.run(logits, self.indices, self.weights, self.positions, self.rows, self.losses, stream=stream))
            _done(gg.moe_dispatch(self.q, self.positions, self.packed, stream))
            _done(gg.moe_dispatch(self.s, self.positions, self.packed_s, stream))
            _done(self.gate_up.run(self.packed, self.packed_s, self.rows, self.mid, d_scales=self.mid_s, stream=stream))
            _done(self.down.run(self.mid, self.mid_s, self.rows, self.out, stream=stream))
            y = torch.empty_like(x) if y is None else y
            _done(gg.moe_combine(self.out, self.positions, y, self.weights, stream))
        return self.h, y


def weights(experts: int, hidden: int, inner: int, device="cuda", seed: int = 0):
    g = torch.Generator(device=device).manual_seed(seed)
    make = lambda *s: torch.randn(*s, device=device, generator=g)  # noqa: E731
    return ((1.0 + 0.2 * make(hidden)).bfloat16(), make(experts, hidden) * hidden ** -0.5, (make(experts, hidden, inner) * hidden ** -0.5).bfloat16(),
            (make(experts, hidden, inner) * hidden ** -0.5).bfloat16(), (make(experts, inner, hidden) * inner ** -0.5).bfloat16())


def main() -> None:
    w = weights(8, 1024, 2048)
    layer = GatedMoeLayer(*w, top_k=2, tokens=2048)
    x, r = torch.randn(2, 2048, 1024, device="cuda").bfloat16()
    h, y = layer.forward(x, r)
    names = ("x", "norm", "gate", "wg", "wu", "wd")
    grads = layer.backward(torch.zeros_like(h), torch.ones_like(y))
    print("training step: rows per expert", layer.rows.tolist(), "gradient norms", {n: float("%.3g" % g.float().norm()) for n, g in zip(names, grads)})
    server = GatedMoeServer(*w, top_k=2, tokens=64)
    few = server.step(x[:64], r[:64])[1]
    print("serving in 8 bits: relative difference to BF16 %.3g" % float((few - y[:64]).float().norm() / y[:64].float().norm()))


if __name__ == "__main__":
    main()
