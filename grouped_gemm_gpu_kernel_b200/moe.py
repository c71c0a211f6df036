"""The parts of a mixture-of-experts layer around the grouped product: the router with its losses and
gradient, the moves of rows into expert order and back, and the experts in 4-bit weights for decoding.

Every call goes through the C-ABI (include/grouped_gemm_b200.h, which states the definitions) and
follows the package's manner: buffers are the caller's, calls enqueue on the given stream (None: the
legacy default stream) without synchronising, functions return the cudaError_t value as an int, and
constructors and tensor mismatches raise ValueError. All tensors are on the current CUDA device, and routers and
plans run on the one that was current when they were made.

    router = gg.MoeRouter(experts=64, top_k=2, capacity_tokens=8192)
    router.run(logits, indices, weights, positions, rows, losses, lse=lse)
    gg.moe_dispatch(x, positions, packed)          # packed: tokens * top_k rows, A of a MoePlan
    plan.run(rows)                                 # MoePlan, or Q4Plan.run(packed, rows, y)
    gg.moe_combine(y, positions, out, weights)
"""
from __future__ import annotations

import ctypes
import importlib
from typing import Optional, Sequence

from . import capi

_calls = None


def _native():
    """The module that checks the tensors and makes the calls (csrc/moe_python.cpp; raises when it has not been built)."""
    global _calls
    if _calls is None:
        capi.load()
        try:
            _calls = importlib.import_module("._moe_native", __package__)
        except ImportError as e:
            raise RuntimeError("the calls of the mixture-of-experts operators are missing; build them with "
                               f"`python -m grouped_gemm_gpu_kernel_b200.build` ({e})") from e
    return _calls


def _stream(stream) -> Optional[int]:
    if stream is None:
        return None
    if isinstance(stream, int):
        return stream or None
    return getattr(stream, "cuda_stream", None) or None


class MoeRouter:
    """Top-k router of `experts` experts for up to capacity_tokens tokens a run (gg_router_*).

    logit_type: OutputType of the logits and their gradient. normalize: a token's weights are the
    softmax over its chosen experts (else the softmax over all, read at the chosen ones). The router
    owns a workspace: one router per concurrent stream.
    """

    def __init__(self, experts: int, top_k: int, capacity_tokens: int, logit_type: int = capi.GG_OUTPUT_F32,
                 normalize: bool = True):
        self._lib = capi.load()
        self._h, self._p = None, 0
        cfg = capi.GGRouterConfig(int(experts), int(top_k), int(capacity_tokens), int(logit_type), 1 if normalize else 0)
        h = ctypes.c_void_p()
        st = self._lib.gg_router_create(ctypes.byref(cfg), ctypes.byref(h))
        if st != 0:
            raise ValueError(f"gg_router_create failed with status {st}")
        self._h = h
        self.experts, self.top_k, self.capacity_tokens = int(experts), int(top_k), int(capacity_tokens)
        self.logit_type = int(logit_type)
        self._run, self._backward = _native().router_run, _native().router_backward
        self._p = h.value

    def run(self, logits, indices, weights, positions, rows, losses, row_tokens=None, lse=None, prob_mean=None,
            token_mask=None, stream=None) -> int:
        """logits (tokens, experts); outputs indices (int32), weights (float32) and positions (int32), each
        (tokens, top_k); rows (int32, experts); losses (float32, 3); optional row_tokens (int32,
        tokens * top_k), lse (float32, tokens), prob_mean (float32, experts). token_mask: uint8 or bool
        (tokens), zero where a token is not routed."""
        return self._run(self._p, self.experts, self.top_k, self.logit_type, logits, indices, weights, positions, rows, losses,
                         row_tokens, lse, prob_mean, token_mask, stream)

    def backward(self, logits, indices, weights, rows, losses, lse, grad_weights, grad_losses, grad_logits,
                 stream=None) -> int:
        """grad_logits from the run's inputs and outputs, the gradient of its weights (float32, tokens x
        top_k, or None) and of losses[0] and losses[1] (float32, 2, or None)."""
        return self._backward(self._p, self.experts, self.top_k, self.logit_type, logits, indices, weights, rows, losses, lse,
                              grad_weights, grad_losses, grad_logits, stream)

    def close(self):
        if self._h:
            self._lib.gg_router_destroy(self._h)
            self._h, self._p = None, 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def moe_dispatch(x, positions, packed, stream=None) -> int:
    """packed[positions[t, j]] = x[t]: x (tokens, width), packed (rows, width), of one dtype of 1, 2 or 4
    bytes; positions (tokens, top_k) int32, entries outside packed's rows go nowhere."""
    return (_calls or _native()).dispatch(x, positions, packed, stream)


def moe_combine(packed, positions, out, weights=None, stream=None) -> int:
    """out[t] = sum over j of weights[t, j] * packed[positions[t, j]] (weights None: 1, the gradient of
    moe_dispatch); weights float32 (tokens, top_k)."""
    return (_calls or _native()).combine(packed, positions, out, weights, stream)


def moe_combine_backward(grad_out, packed, positions, weights, grad_packed, grad_weights, stream=None) -> int:
    """The gradients of moe_combine with weights: grad_packed (like packed) and grad_weights (float32,
    tokens x top_k)."""
    return (_calls or _native()).combine_backward(grad_out, packed, positions, weights, grad_packed, grad_weights, stream)


class Q4Plan:
    """Experts with 4-bit weights and a scale per output and group of k (gg_q4_plan_*).

    q_ptrs: one device pointer per expert to n rows of ceil(k / 2) bytes (pitch ldq bytes), the low 4
    bits first; scale_ptrs: n x ceil(k / group) values of the input type; zero_ptrs: the same shape,
    bytes of 0..15 (None: 8); bias_ptrs: n FP32 values (or None) per expert. The constructor copies the
    weights into the kernel's layout in order on `stream` and synchronises it; the sources may be freed
    afterwards (the biases are read at run time).
    """

    def __init__(self, experts: int, n: int, k: int, group: int, q_ptrs: Sequence[int], ldq: int,
                 scale_ptrs: Sequence[int], zero_ptrs: Optional[Sequence[int]] = None,
                 bias_ptrs: Optional[Sequence[Optional[int]]] = None, input_type: int = capi.GG_INPUT_F16,
                 output_type: int = capi.GG_OUTPUT_F32, activation: int = capi.GG_ACT_NONE, stream=None):
        self._lib = capi.load()
        self._h, self._p = None, 0
        tables = []
        for name, ptrs in (("q", q_ptrs), ("scale", scale_ptrs), ("zero", zero_ptrs), ("bias", bias_ptrs)):
            if ptrs is None:
                tables.append(None)
                continue
            if len(ptrs) != experts:
                raise ValueError(f"one {name} pointer per expert")
            tables.append((ctypes.c_void_p * max(1, experts))(*[ctypes.c_void_p(int(x) if x else None) for x in ptrs]))
        cast = [ctypes.cast(x, ctypes.POINTER(ctypes.c_void_p)) if x is not None else None for x in tables]
        prob = capi.GGQ4Problem(cast[0], cast[1], cast[2], cast[3], int(experts), int(n), int(k), int(group), int(ldq),
                                int(input_type), int(output_type), int(activation))
        h = ctypes.c_void_p()
        st = self._lib.gg_q4_plan_create(ctypes.byref(prob), _stream(stream), ctypes.byref(h))
        if st != 0:
            raise ValueError(f"gg_q4_plan_create failed with status {st}")
        self._h = h
        self.experts, self.n, self.k = int(experts), int(n), int(k)
        self.input_type, self.output_type = int(input_type), int(output_type)
        self._run = _native().q4_run
        self._p = h.value

    def run(self, a, rows, d, row_tokens=None, stream=None) -> int:
        """a (a_rows, k); rows: int32 device tensor of `experts` counts (None with one expert: all rows of
        d); d (capacity rows, n). row_tokens: int32, one per row of d, the row of `a` that it reads."""
        return self._run(self._p, self.experts, self.n, self.k, self.input_type, self.output_type, a, rows, d, row_tokens, stream)

    def status(self) -> int:
        """Synchronises; returns (then clears) the GG_STATUS_* bits of the plan's runs."""
        out = ctypes.c_int(0)
        st = self._lib.gg_q4_plan_status(self._h, ctypes.byref(out))
        if st != 0:
            raise RuntimeError(f"gg_q4_plan_status failed with status {st}")
        return out.value

    def close(self):
        if self._h:
            self._lib.gg_q4_plan_destroy(self._h)
            self._h, self._p = None, 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
