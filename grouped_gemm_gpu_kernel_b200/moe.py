"""The parts of a mixture-of-experts layer around the grouped product: the router with its losses and
gradient, the moves of rows into expert order and back, and the experts in 4-bit weights for decoding.

Every call goes through the C-ABI (include/grouped_gemm_b200.h, which states the definitions) and
follows the package's manner: buffers are the caller's, calls enqueue on the given stream (None: the
legacy default stream) without synchronising, functions return the cudaError_t value as an int, and
constructors and tensor mismatches raise ValueError.

    router = gg.MoeRouter(experts=64, top_k=2, capacity_tokens=8192)
    router.run(logits, indices, weights, positions, rows, losses, lse=lse)
    gg.moe_dispatch(x, positions, packed)          # packed: tokens * top_k rows, A of a MoePlan
    plan.run(rows)                                 # MoePlan, or Q4Plan.run(packed, rows, y)
    gg.moe_combine(y, positions, out, weights)
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional, Sequence

from . import capi

_types = {}  # torch dtype -> GG_OUTPUT_*
_f32 = _i32 = None
_masks = ()

# The checks below run before every launch, which a decoding step makes some ten of: each reads an attribute of a
# tensor once (some 50 to 100 ns apiece), and the C structs are filled by one struct.pack.
_ROUTE = struct.Struct("@10P2i")
_ROUTE_GRADIENT = struct.Struct("@9P3i4x")


def _load_types():
    global _f32, _i32, _masks
    import torch

    _types[torch.float32] = capi.GG_OUTPUT_F32
    _types[torch.float16] = capi.GG_OUTPUT_F16
    _types[torch.bfloat16] = capi.GG_OUTPUT_BF16
    _f32, _i32, _masks = torch.float32, torch.int32, (torch.uint8, torch.bool)


def _type_of(t, name: str) -> int:
    if _f32 is None:
        _load_types()
    v = _types.get(t.dtype)
    if v is None:
        raise ValueError(f"{name}: float32, float16 or bfloat16 expected, got {t.dtype}")
    return v


def _stream(stream) -> Optional[int]:
    if stream is None:
        return None
    if isinstance(stream, int):
        return stream or None
    return getattr(stream, "cuda_stream", None) or None


def _shape(t, name: str):
    s = t.shape
    if len(s) != 2:
        raise ValueError(f"{name}: two dimensions expected, got {tuple(s)}")
    return s


def _pitch(t, rows: int, cols: int, name: str) -> int:
    """The row pitch of a rows x cols device tensor with contiguous columns."""
    if t.shape != (rows, cols):
        raise ValueError(f"{name}: shape ({rows}, {cols}) expected, got {tuple(t.shape)}")
    r, c = t.stride()
    if (c != 1 and cols > 1) or (r < cols and rows > 1) or not t.is_cuda:
        raise ValueError(f"{name}: a CUDA tensor with contiguous columns and rows that do not overlap expected")
    return r if r >= cols and r > 0 else max(1, cols)


def _packed(t, count: int, dtype, name: str) -> int:
    """The address of a contiguous device tensor of `count` elements."""
    if t.dtype is not dtype or t.numel() != count or not t.is_contiguous() or not t.is_cuda:
        raise ValueError(f"{name}: a contiguous CUDA {dtype} tensor of {count} elements expected, got "
                         f"{t.dtype} {tuple(t.shape)}")
    return t.data_ptr()


class MoeRouter:
    """Top-k router of `experts` experts for up to capacity_tokens tokens a run (gg_router_*).

    logit_type: OutputType of the logits and their gradient. normalize: a token's weights are the
    softmax over its chosen experts (else the softmax over all, read at the chosen ones). The router
    owns a workspace: one router per concurrent stream.
    """

    def __init__(self, experts: int, top_k: int, capacity_tokens: int, logit_type: int = capi.GG_OUTPUT_F32,
                 normalize: bool = True):
        self._lib = capi.load()
        self._h = None
        cfg = capi.GGRouterConfig(int(experts), int(top_k), int(capacity_tokens), int(logit_type), 1 if normalize else 0)
        h = ctypes.c_void_p()
        st = self._lib.gg_router_create(ctypes.byref(cfg), ctypes.byref(h))
        if st != 0:
            raise ValueError(f"gg_router_create failed with status {st}")
        self._h = h
        self.experts, self.top_k, self.capacity_tokens = int(experts), int(top_k), int(capacity_tokens)
        self.logit_type = int(logit_type)

    def run(self, logits, indices, weights, positions, rows, losses, row_tokens=None, lse=None, prob_mean=None,
            token_mask=None, stream=None) -> int:
        """logits (tokens, experts); outputs indices (int32), weights (float32) and positions (int32), each
        (tokens, top_k); rows (int32, experts); losses (float32, 3); optional row_tokens (int32,
        tokens * top_k), lse (float32, tokens), prob_mean (float32, experts). token_mask: uint8 or bool
        (tokens), zero where a token is not routed."""
        if not self._h:
            return capi.CUDA_ERROR_INVALID_DEVICE_POINTER
        if _type_of(logits, "logits") != self.logit_type:
            raise ValueError(f"logits: the router was made for another type than {logits.dtype}")
        t, e = _shape(logits, "logits")[0], self.experts
        slots = t * self.top_k
        ld = _pitch(logits, t, e, "logits")
        mask = 0
        if token_mask is not None:
            if token_mask.dtype not in _masks or token_mask.numel() != t or not token_mask.is_contiguous() or not token_mask.is_cuda:
                raise ValueError("token_mask: one contiguous CUDA uint8 or bool per token expected")
            mask = token_mask.data_ptr()
        q = _ROUTE.pack(logits.data_ptr(), mask, _packed(indices, slots, _i32, "indices"),
                        _packed(weights, slots, _f32, "weights"), _packed(positions, slots, _i32, "positions"),
                        _packed(rows, e, _i32, "rows"), _packed(losses, 3, _f32, "losses"),
                        0 if row_tokens is None else _packed(row_tokens, slots, _i32, "row_tokens"),
                        0 if lse is None else _packed(lse, t, _f32, "lse"),
                        0 if prob_mean is None else _packed(prob_mean, e, _f32, "prob_mean"), t, ld)
        return self._lib.gg_router_run(self._h, q, _stream(stream))

    def backward(self, logits, indices, weights, rows, losses, lse, grad_weights, grad_losses, grad_logits,
                 stream=None) -> int:
        """grad_logits from the run's inputs and outputs, the gradient of its weights (float32, tokens x
        top_k, or None) and of losses[0] and losses[1] (float32, 2, or None)."""
        if not self._h:
            return capi.CUDA_ERROR_INVALID_DEVICE_POINTER
        if _type_of(logits, "logits") != self.logit_type or grad_logits.dtype is not logits.dtype:
            raise ValueError("logits, grad_logits: the router's type expected")
        t, e = _shape(logits, "logits")[0], self.experts
        slots = t * self.top_k
        ld, ldg = _pitch(logits, t, e, "logits"), _pitch(grad_logits, t, e, "grad_logits")
        q = _ROUTE_GRADIENT.pack(logits.data_ptr(), _packed(indices, slots, _i32, "indices"),
                                 _packed(weights, slots, _f32, "weights"), _packed(rows, e, _i32, "rows"),
                                 _packed(losses, 3, _f32, "losses"), _packed(lse, t, _f32, "lse"),
                                 0 if grad_weights is None else _packed(grad_weights, slots, _f32, "grad_weights"),
                                 0 if grad_losses is None else _packed(grad_losses, 2, _f32, "grad_losses"),
                                 grad_logits.data_ptr(), t, ld, ldg)
        return self._lib.gg_router_backward(self._h, q, _stream(stream))

    def close(self):
        if self._h:
            self._lib.gg_router_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _slots(positions, tokens: int) -> int:
    t, k = _shape(positions, "positions")
    if t != tokens:
        raise ValueError(f"positions: ({tokens}, top_k) expected, got ({t}, {k})")
    return k


def moe_dispatch(x, positions, packed, stream=None) -> int:
    """packed[positions[t, j]] = x[t]: x (tokens, width), packed (rows, width), of one dtype of 1, 2 or 4
    bytes; positions (tokens, top_k) int32, entries outside packed's rows go nowhere."""
    if _f32 is None:
        _load_types()
    t, w = _shape(x, "x")
    k = _slots(positions, t)
    if packed.dtype is not x.dtype:
        raise ValueError("x, packed: one dtype expected")
    r = _shape(packed, "packed")[0]
    ldx, ldp = _pitch(x, t, w, "x"), _pitch(packed, r, w, "packed")
    return capi.load().gg_moe_dispatch(x.data_ptr(), ldx, _packed(positions, t * k, _i32, "positions"), t, k, w,
                                       x.element_size(), packed.data_ptr(), r, ldp, _stream(stream))


def moe_combine(packed, positions, out, weights=None, stream=None) -> int:
    """out[t] = sum over j of weights[t, j] * packed[positions[t, j]] (weights None: 1, the gradient of
    moe_dispatch); weights float32 (tokens, top_k)."""
    pt, ot = _type_of(packed, "packed"), _type_of(out, "out")
    t, w = _shape(out, "out")
    k = _slots(positions, t)
    r = _shape(packed, "packed")[0]
    ldp, ldo = _pitch(packed, r, w, "packed"), _pitch(out, t, w, "out")
    return capi.load().gg_moe_combine(packed.data_ptr(), pt, r, ldp, _packed(positions, t * k, _i32, "positions"),
                                      None if weights is None else _packed(weights, t * k, _f32, "weights"), t, k, w,
                                      out.data_ptr(), ot, ldo, _stream(stream))


def moe_combine_backward(grad_out, packed, positions, weights, grad_packed, grad_weights, stream=None) -> int:
    """The gradients of moe_combine with weights: grad_packed (like packed) and grad_weights (float32,
    tokens x top_k)."""
    ot, pt = _type_of(grad_out, "grad_out"), _type_of(packed, "packed")
    t, w = _shape(grad_out, "grad_out")
    k = _slots(positions, t)
    r = _shape(packed, "packed")[0]
    if grad_packed.dtype is not packed.dtype:
        raise ValueError("packed, grad_packed: one dtype expected")
    ldo, ldp, ldgp = (_pitch(grad_out, t, w, "grad_out"), _pitch(packed, r, w, "packed"),
                      _pitch(grad_packed, r, w, "grad_packed"))
    return capi.load().gg_moe_combine_backward(
        grad_out.data_ptr(), ot, ldo, packed.data_ptr(), pt, r, ldp, _packed(positions, t * k, _i32, "positions"),
        _packed(weights, t * k, _f32, "weights"), t, k, w, grad_packed.data_ptr(), ldgp,
        _packed(grad_weights, t * k, _f32, "grad_weights"), _stream(stream))


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
        self._h = None
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

    def run(self, a, rows, d, row_tokens=None, stream=None) -> int:
        """a (a_rows, k); rows: int32 device tensor of `experts` counts (None with one expert: all rows of
        d); d (capacity rows, n). row_tokens: int32, one per row of d, the row of `a` that it reads."""
        if not self._h:
            return capi.CUDA_ERROR_INVALID_DEVICE_POINTER
        if _type_of(a, "a") != (capi.GG_OUTPUT_F16 if self.input_type == capi.GG_INPUT_F16 else capi.GG_OUTPUT_BF16):
            raise ValueError(f"a: the plan was made for another type than {a.dtype}")
        if _type_of(d, "d") != self.output_type:
            raise ValueError(f"d: the plan was made for another type than {d.dtype}")
        ar, cap = _shape(a, "a")[0], _shape(d, "d")[0]
        lda, ldd = _pitch(a, ar, self.k, "a"), _pitch(d, cap, self.n, "d")
        return self._lib.gg_q4_plan_run(
            self._h, a.data_ptr(), lda, ar, None if row_tokens is None else _packed(row_tokens, cap, _i32, "row_tokens"),
            None if rows is None else _packed(rows, self.experts, _i32, "rows"), d.data_ptr(), ldd, cap, _stream(stream))

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
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
