"""The Python calls of the mixture-of-experts operators take tensors of the current device only. One GPU has no tensor of
another, so tensors that say they are on another stand for it: their memory is this GPU's, whatever is done with it.
"""
import pytest

import grouped_gemm_gpu_kernel_b200 as gg

pytestmark = pytest.mark.gpu


class Elsewhere:
    """A tensor of this GPU that says it is on GPU `device`."""

    def __init__(self, tensor, device):
        self._tensor, self._device = tensor, device

    def get_device(self):
        return self._device

    @property
    def device(self):
        import torch
        return torch.device("cuda", self._device)

    def __getattr__(self, name):
        return getattr(self._tensor, name)


def calls(cuda):
    """(function, tensors) of every call, with all of its optional tensors."""
    import torch
    t, e, k, width = 6, 8, 2, 64
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)  # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device=cuda)  # noqa: E731
    router = gg.MoeRouter(e, k, t)
    out = [i32(t, k), f32(t, k), i32(t, k), i32(e), f32(3)]
    more = [i32(t * k), f32(t), f32(e), torch.ones(t, dtype=torch.uint8, device=cuda)]
    yield router.run, [f32(t, e), *out, *more]
    yield router.backward, [f32(t, e), out[0], out[1], out[3], out[4], more[1], f32(t, k), f32(2), f32(t, e)]
    places = torch.arange(t * k, dtype=torch.int32, device=cuda).view(t, k)
    yield gg.moe_dispatch, [f32(t, width), places, f32(t * k, width)]
    yield gg.moe_combine, [f32(t * k, width), places, f32(t, width), f32(t, k)]
    yield gg.moe_combine_backward, [f32(t, width), f32(t * k, width), places, f32(t, k), f32(t * k, width), f32(t, k)]
    q, s = torch.zeros(32, 64, dtype=torch.uint8, device=cuda), torch.ones(32, 1, dtype=torch.float16, device=cuda)
    plan = gg.Q4Plan(1, 32, 128, 128, [q.data_ptr()], 64, [s.data_ptr()])
    yield plan.run, [torch.zeros(4, 128, dtype=torch.float16, device=cuda), i32(1), f32(4, 32), i32(4)]


def test_every_tensor_has_to_be_on_the_current_device(cuda):
    for call, tensors in calls(cuda):
        assert call(*(Elsewhere(t, 0) for t in tensors)) == 0
        for i in range(len(tensors)):
            for device in (1, -1):
                args = list(tensors)
                args[i] = Elsewhere(args[i], device)
                with pytest.raises(ValueError):
                    call(*args)
        with pytest.raises(ValueError):
            call(*(Elsewhere(t, 1) for t in tensors))
