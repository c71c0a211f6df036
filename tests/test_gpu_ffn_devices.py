"""The calls of the norm, the 8-bit product and the gated block take tensors of the current device only. One GPU has no tensor
of another, so tensors that say they are on another stand for it: their memory is this GPU's, whatever is done with it.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg
from test_gpu_moe_devices import Elsewhere

pytestmark = pytest.mark.gpu


def calls(cuda):
    """(function, tensors by name) of every call, with all of its optional tensors."""
    import torch
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, device=cuda, dtype=dt)  # noqa: E731
    f32, f8, i32 = torch.float32, torch.float8_e4m3fn, torch.int32
    norm = gg.RmsNorm(64, dtype=gg.OutputType.kBF16)
    yield norm.run, dict(x=z(4, 64), weight=z(64), y=z(4, 64), residual=z(4, 64), residual_out=z(4, 64), q=z(4, 64, dt=f8), scales=z(4, 1, dt=f32),
                         rstd=z(4, dt=f32))
    yield norm.backward, dict(h=z(4, 64), weight=z(64), rstd=z(4, dt=f32), grad_y=z(4, 64), grad_x=z(4, 64), grad_weight=z(64, dt=f32), grad_h=z(4, 64))
    w, s = z(2, 64, 64, dt=f8), z(2, 1, 1, dt=f32)
    ptrs = lambda t: [x.data_ptr() for x in t]  # noqa: E731
    f8_plan = gg.F8Plan(2, 64, 64, ptrs(w), 64, ptrs(s), up_ptrs=ptrs(w), up_scale_ptrs=ptrs(s), output_type=gg.OutputType.kE4M3,
                        activation=gg.Activation.kSiLU)
    keep = [w, s]
    yield f8_plan.run, dict(a=z(4, 64, dt=f8), a_scales=z(4, 1, dt=f32), rows=z(2, dt=i32), d=z(4, 64, dt=f8), d_scales=z(4, 1, dt=f32))
    w16 = z(2, 64, 64)
    keep.append(w16)
    plan = gg.GatedPlan(2, 64, 64, ptrs(w16), ptrs(w16), 64)
    m = lambda: z(4, 64)  # noqa: E731
    yield plan.run, dict(x=m(), rows=z(2, dt=i32), h=m(), gate=m(), up=m())
    yield plan.backward, dict(x=m(), gate=m(), up=m(), grad_h=m(), rows=z(2, dt=i32), grad_gate=m(), grad_up=m(), grad_x=m(), grad_gate_w=z(2, 64, 64),
                              grad_up_w=z(2, 64, 64))
    torch.cuda.synchronize()
    del keep


def test_every_tensor_has_to_be_on_the_current_device(cuda):
    for call, tensors in calls(cuda):
        assert call(**{n: Elsewhere(t, 0) for n, t in tensors.items()}) == 0
        for name in tensors:
            for device in (1, -1):
                with pytest.raises(ValueError):
                    call(**(tensors | {name: Elsewhere(tensors[name], device)}))
        with pytest.raises(ValueError):
            call(**{n: Elsewhere(t, 1) for n, t in tensors.items()})
