"""What stands between the router and the experts' products, and the experts' feed-forward: the root-mean-square norm
with the residual's addition and an output in 8 bits, the product of 8-bit rows with 8-bit expert weights that have a scale
for each block of 128, and the gated feed-forward of experts with its gradient.

Every call goes through the C-ABI (include/grouped_gemm_b200.h, which states the definitions) in the manner of the
mixture-of-experts calls: buffers are the caller's, calls enqueue on the given stream (None: the legacy default stream)
without synchronising, functions return the cudaError_t value as an int, and constructors and tensor mismatches raise
ValueError. All tensors are on the current CUDA device, which is the one that was current when the handle was made.

    norm = gg.RmsNorm(hidden, dtype=gg.OutputType.kBF16)
    norm.run(x, weight, residual=r, residual_out=h, q=q, scales=s)     # q, s: rows in 8 bits
    gate_up = gg.F8Plan(experts, inner, hidden, gate_ptrs, hidden, gate_scale_ptrs, up_ptrs, up_scale_ptrs,
                        output_type=gg.OutputType.kE4M3, activation=gg.Activation.kSiLU)
    gate_up.run(packed_q, packed_s, rows, hq, hs)                      # rows: MoeRouter's counts
    down = gg.F8Plan(experts, hidden, inner, down_ptrs, inner, down_scale_ptrs)
    down.run(hq, hs, rows, out)
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence

from . import capi
from .moe import _native


def _tables(experts: int, **named):
    """One array of device pointers per name (None: none)."""
    out = []
    for name, ptrs in named.items():
        if ptrs is None:
            out.append(None)
            continue
        if len(ptrs) != experts:
            raise ValueError(f"one {name} pointer per expert")
        table = (ctypes.c_void_p * max(1, experts))(*[ctypes.c_void_p(int(x) if x else None) for x in ptrs])
        out.append(ctypes.cast(table, ctypes.POINTER(ctypes.c_void_p)))
    return out


class _Handle:
    """A handle of the library, closed once."""

    _destroy = ""

    def _make(self, create: str, config) -> None:
        self._lib, self._h, self._p = capi.load(), None, 0
        h = ctypes.c_void_p()
        st = getattr(self._lib, create)(ctypes.byref(config), ctypes.byref(h))
        if st != 0:
            raise ValueError(f"{create} failed with status {st}")
        self._h, self._p = h, h.value

    def _status(self, name: str) -> int:
        out = ctypes.c_int(0)
        st = getattr(self._lib, name)(self._h, ctypes.byref(out))
        if st != 0:
            raise RuntimeError(f"{name} failed with status {st}")
        return out.value

    def close(self):
        if getattr(self, "_h", None):
            getattr(self._lib, self._destroy)(self._h)
            self._h, self._p = None, 0

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class RmsNorm(_Handle):
    """Root-mean-square norm of rows of `width` values (gg_norm_*).

    dtype: OutputType of the rows (kF32, kF16, kBF16); weight_type: the same, or kF32. The handle owns the workspace of
    the weight's gradient: one per concurrent stream of backward passes.
    """

    _destroy = "gg_norm_destroy"

    def __init__(self, width: int, dtype: int = capi.GG_OUTPUT_F32, weight_type: Optional[int] = None, eps: float = 1e-6):
        weight_type = dtype if weight_type is None else weight_type
        self._make("gg_norm_create", capi.GGNormConfig(int(width), int(dtype), int(weight_type), float(eps)))
        self.width, self.dtype, self.weight_type, self.eps = int(width), int(dtype), int(weight_type), float(eps)
        self._run, self._backward = _native().norm_run, _native().norm_backward

    def run(self, x, weight=None, y=None, residual=None, residual_out=None, q=None, scales=None, rstd=None, stream=None) -> int:
        """x (rows, width). Optional: weight (width; None: ones), residual, and the outputs residual_out (x + residual), y, q
        (float8_e4m3fn or float8_e5m2) with scales (float32, rows x ceil(width / 128)), rstd (float32, rows)."""
        return self._run(self._p, self.width, self.dtype, self.weight_type, x, weight, y, residual, residual_out, q, scales, rstd, stream)

    def backward(self, h, weight, rstd, grad_y, grad_x, grad_weight=None, grad_h=None, stream=None) -> int:
        """grad_x (of x and of the residual) and grad_weight (float32, width) from the run's h (its residual_out, or x) and
        rstd, grad_y, and grad_h, the gradient that reaches h past the norm."""
        return self._backward(self._p, self.width, self.dtype, self.weight_type, h, weight, rstd, grad_y, grad_x, grad_weight, grad_h, stream)


class F8Plan(_Handle):
    """Experts with 8-bit weights and a scale for each block of 128 x 128 (gg_f8_plan_*).

    b_ptrs: one device pointer per expert to n rows of k bytes (pitch ldb, 16-byte aligned), scale_ptrs: ceil(n / 128) x
    ceil(k / 128) FP32 values. up_ptrs and up_scale_ptrs: a second matrix, for act(x B^T) * (x Up^T); its result can be
    in 8 bits (output_type kE4M3 or kE5M2). bias_ptrs: n FP32 values (or None) per expert. The weights stay the caller's.
    """

    _destroy = "gg_f8_plan_destroy"

    def __init__(self, experts: int, n: int, k: int, b_ptrs: Sequence[int], ldb: int, scale_ptrs: Sequence[int],
                 up_ptrs: Optional[Sequence[int]] = None, up_scale_ptrs: Optional[Sequence[int]] = None,
                 bias_ptrs: Optional[Sequence[Optional[int]]] = None, input_type: int = capi.GG_INPUT_E4M3,
                 output_type: int = capi.GG_OUTPUT_BF16, activation: int = capi.GG_ACT_NONE):
        tables = _tables(experts, b=b_ptrs, scale=scale_ptrs, up=up_ptrs, up_scale=up_scale_ptrs, bias=bias_ptrs)
        self._make("gg_f8_plan_create", capi.GGF8Problem(*tables, int(experts), int(n), int(k), int(ldb), int(input_type),
                                                         int(output_type), int(activation)))
        self.experts, self.n, self.k = int(experts), int(n), int(k)
        self.input_type, self.output_type = int(input_type), int(output_type)
        self._run = _native().f8_run

    def run(self, a, a_scales, rows, d, d_scales=None, stream=None) -> int:
        """a (capacity rows, k) in the input type with rows on 16-byte boundaries; a_scales (float32, capacity rows x
        ceil(k / 128)); rows: int32 device tensor of `experts` counts (None with one expert: all rows); d (capacity rows, n);
        d_scales (float32, capacity rows x ceil(n / 128)) with a d in 8 bits."""
        return self._run(self._p, self.experts, self.n, self.k, self.input_type, self.output_type, a, a_scales, rows, d, d_scales, stream)

    def status(self) -> int:
        """Synchronises; returns (then clears) the GG_STATUS_* bits of the plan's runs."""
        return self._status("gg_f8_plan_status")


class GatedPlan(_Handle):
    """Gated feed-forward of experts, h = act(x Wg) * (x Wu), and its gradient (gg_gated_plan_*).

    gate_ptrs, up_ptrs: one device pointer per expert to a k x n matrix of the input type (row pitch ldw), rows on 16-byte
    boundaries. The weights stay the caller's.
    """

    _destroy = "gg_gated_plan_destroy"

    def __init__(self, experts: int, n: int, k: int, gate_ptrs: Sequence[int], up_ptrs: Sequence[int], ldw: int,
                 input_type: int = capi.GG_INPUT_BF16, activation: int = capi.GG_ACT_SILU):
        tables = _tables(experts, gate=gate_ptrs, up=up_ptrs)
        self._make("gg_gated_plan_create", capi.GGGatedProblem(*tables, int(experts), int(n), int(k), int(ldw), int(input_type), int(activation)))
        self.experts, self.n, self.k, self.input_type = int(experts), int(n), int(k), int(input_type)
        self._run, self._backward = _native().gated_run, _native().gated_backward

    def run(self, x, rows, h, gate=None, up=None, stream=None) -> int:
        """x (capacity rows, k) with rows on 16-byte boundaries; rows: int32 device tensor of `experts` counts (None with
        one expert: all rows); h (capacity rows, n); gate and up, like h: kept for the backward pass."""
        return self._run(self._p, self.experts, self.n, self.k, self.input_type, x, rows, h, gate, up, stream)

    def backward(self, x, gate, up, grad_h, rows, grad_gate, grad_up, grad_x=None, grad_gate_w=None, grad_up_w=None, stream=None) -> int:
        """grad_gate and grad_up (capacity rows, n; rows on 16-byte boundaries; they may be gate, up or grad_h), grad_x
        (capacity rows, k), grad_gate_w and grad_up_w (experts, k, n; float32 or the plan's type; zeros for an expert without rows)."""
        return self._backward(self._p, self.experts, self.n, self.k, self.input_type, x, gate, up, grad_h, rows, grad_gate, grad_up,
                              grad_x, grad_gate_w, grad_up_w, stream)

    def status(self) -> int:
        """Synchronises; returns (then clears) the GG_STATUS_* bits of the plan's runs."""
        return self._status("gg_gated_plan_status")
