"""The host side of the norm, the 8-bit product and the gated feed-forward: what the C-ABI refuses before any device
work, and what the Python classes refuse."""
import ctypes

import pytest

import grouped_gemm_gpu_kernel_b200 as gg
from grouped_gemm_gpu_kernel_b200 import capi

BAD = capi.CUDA_ERROR_INVALID_VALUE
GONE = capi.CUDA_ERROR_INVALID_DEVICE_POINTER
PTR = 0x1000


def table(count=2, change=None):
    t = (ctypes.c_void_p * 1100)(*[PTR] * 1100)
    if change is not None:
        t[count - 1] = change or None
    return ctypes.cast(t, ctypes.POINTER(ctypes.c_void_p)), t


def test_null_handles_and_arguments():
    lib = capi.load()
    for create, config, destroy in (("gg_norm_create", capi.GGNormConfig(8, 0, 0, 1e-6), "gg_norm_destroy"),
                                    ("gg_f8_plan_create", capi.GGF8Problem(), "gg_f8_plan_destroy"),
                                    ("gg_gated_plan_create", capi.GGGatedProblem(), "gg_gated_plan_destroy")):
        out = ctypes.c_void_p(5)
        assert getattr(lib, create)(None, ctypes.byref(out)) == BAD and out.value is None
        assert getattr(lib, create)(ctypes.byref(config), None) == BAD
        getattr(lib, destroy)(None)
    assert lib.gg_norm_run(None, ctypes.byref(capi.GGNorm()), None) == GONE
    assert lib.gg_norm_backward(None, ctypes.byref(capi.GGNormGradient()), None) == GONE
    assert lib.gg_f8_plan_run(None, PTR, 16, PTR, 1, PTR, PTR, 16, None, 0, 1, None) == GONE
    assert lib.gg_f8_plan_status(None, ctypes.byref(ctypes.c_int())) == GONE
    assert lib.gg_gated_plan_run(None, ctypes.byref(capi.GGGated()), None) == GONE
    assert lib.gg_gated_plan_backward(None, ctypes.byref(capi.GGGatedGradient()), None) == GONE
    assert lib.gg_gated_plan_status(None, ctypes.byref(ctypes.c_int())) == GONE


@pytest.mark.parametrize("change", [dict(width=0), dict(width=-4), dict(width=capi.GG_NORM_MAX_WIDTH + 1), dict(dtype=3), dict(dtype=-1),
                                    dict(dtype=0, weight_type=1), dict(dtype=1, weight_type=2), dict(eps=-1e-6), dict(eps=float("nan")),
                                    dict(eps=float("inf"))])
def test_norms_out_of_range_are_refused(change):
    with pytest.raises(ValueError):
        gg.RmsNorm(**(dict(width=64, dtype=0) | change))


F8 = dict(experts=2, n=16, k=64, ldb=64, input_type=capi.GG_INPUT_E4M3, output_type=0, activation=0)


@pytest.mark.parametrize("change", [dict(experts=0), dict(experts=1025), dict(n=0), dict(n=2 ** 30 + 1), dict(k=0), dict(k=-1), dict(k=2 ** 30 + 1, ldb=2 ** 30 + 16), dict(ldb=63), dict(ldb=72), dict(ldb=48),
                                    dict(input_type=0), dict(input_type=1), dict(input_type=4), dict(output_type=-1), dict(output_type=5),
                                    dict(output_type=capi.GG_OUTPUT_E4M3), dict(output_type=capi.GG_OUTPUT_E5M2), dict(activation=4),
                                    dict(activation=-1), dict(b=0), dict(b=PTR + 8), dict(b_scales=0), dict(up=0), dict(up=PTR + 1),
                                    dict(up_scales=0), dict(up="alone"), dict(up_scales="alone"), dict(bias="gated")])
def test_f8_problems_out_of_range_are_refused(change):
    f = F8 | {n: v for n, v in change.items() if n in F8}
    kept = {n: table(2, change[n] if isinstance(change.get(n), int) else None) for n in ("b", "b_scales", "up", "up_scales", "bias")}
    gated = any(n in change for n in ("up", "up_scales")) or change.get("bias") == "gated"
    use = {"b", "b_scales"} | ({"up", "up_scales"} if gated else set()) | ({"bias"} if "bias" in change else set())
    for n in ("up", "up_scales"):
        if change.get(n) == "alone":
            use -= {"up", "up_scales"} - {n}
    out = ctypes.c_void_p()
    prob = capi.GGF8Problem(*[kept[n][0] if n in use else None for n in ("b", "b_scales", "up", "up_scales", "bias")],
                            *[f[n] for n in ("experts", "n", "k", "ldb", "input_type", "output_type", "activation")])
    assert capi.load().gg_f8_plan_create(ctypes.byref(prob), ctypes.byref(out)) == BAD and out.value is None


GATED = dict(experts=2, n=16, k=64, ldw=16, type=0, activation=0)


@pytest.mark.parametrize("change", [dict(experts=0), dict(experts=1025), dict(n=0), dict(n=2 ** 30 + 1, ldw=2 ** 30 + 8), dict(k=0), dict(k=2 ** 30 + 1), dict(ldw=15), dict(ldw=20), dict(type=2), dict(type=-1),
                                    dict(activation=4), dict(activation=-1), dict(gate=0), dict(gate=PTR + 2), dict(up=0), dict(up=PTR + 8)])
def test_gated_problems_out_of_range_are_refused(change):
    f = GATED | {n: v for n, v in change.items() if n in GATED}
    kept = {n: table(2, change.get(n)) for n in ("gate", "up")}
    out = ctypes.c_void_p()
    prob = capi.GGGatedProblem(kept["gate"][0], kept["up"][0], *[f[n] for n in ("experts", "n", "k", "ldw", "type", "activation")])
    assert capi.load().gg_gated_plan_create(ctypes.byref(prob), ctypes.byref(out)) == BAD and out.value is None


def test_tables_have_one_entry_per_expert():
    with pytest.raises(ValueError):
        gg.F8Plan(2, 16, 64, [PTR], 64, [PTR, PTR])
    with pytest.raises(ValueError):
        gg.F8Plan(2, 16, 64, [PTR, PTR], 64, [PTR])
    with pytest.raises(ValueError):
        gg.F8Plan(2, 16, 64, [PTR, PTR], 64, [PTR, PTR], up_ptrs=[PTR, PTR], up_scale_ptrs=[PTR])
    with pytest.raises(ValueError):
        gg.F8Plan(2, 16, 64, [PTR, PTR], 64, [PTR, PTR], bias_ptrs=[PTR])
    with pytest.raises(ValueError):
        gg.GatedPlan(2, 16, 64, [PTR, PTR], [PTR], 16)


def test_other_plans_keep_their_activations():
    """The new activation and output types are the new plans' alone."""
    cfg = gg.KernelConfig(128, 128, 64, activation=gg.Activation.kSiLU).to_c()
    assert capi.load().gg_query_occupancy(ctypes.byref(cfg), ctypes.byref(capi.GGOccupancy())) == BAD
    cfg = gg.KernelConfig(128, 128, 64, output_type=gg.OutputType.kE4M3).to_c()
    assert capi.load().gg_query_occupancy(ctypes.byref(cfg), ctypes.byref(capi.GGOccupancy())) == BAD
