"""The host side of the mixture-of-experts operators: what the C-ABI refuses before any device work."""
import ctypes

import pytest

import grouped_gemm_gpu_kernel_b200 as gg
from grouped_gemm_gpu_kernel_b200 import capi

BAD = capi.CUDA_ERROR_INVALID_VALUE
GONE = capi.CUDA_ERROR_INVALID_DEVICE_POINTER
PTR = 0x1000


@pytest.mark.parametrize("cfg", [(0, 1, 8, 0), (1025, 1, 8, 0), (8, 0, 8, 0), (8, 33, 8, 0), (8, 2, -1, 0), (8, 2, 2 ** 30, 0), (8, 1, 2 ** 31 - 65536, 0),
                                 (8, 2, 8, 3), (8, 2, 8, -1)])
def test_router_sizes_out_of_range_are_refused(cfg):
    with pytest.raises(ValueError):
        gg.MoeRouter(cfg[0], cfg[1], cfg[2], logit_type=cfg[3])


def test_null_handles_and_arguments():
    lib = capi.load()
    out = ctypes.c_void_p(5)
    assert lib.gg_router_create(None, ctypes.byref(out)) == BAD and out.value is None
    assert lib.gg_router_create(ctypes.byref(capi.GGRouterConfig(8, 2, 8, 0, 1)), None) == BAD
    assert lib.gg_router_run(None, ctypes.byref(capi.GGRoute()), None) == GONE
    assert lib.gg_router_backward(None, ctypes.byref(capi.GGRouteGradient()), None) == GONE
    lib.gg_router_destroy(None)
    out = ctypes.c_void_p(5)
    assert lib.gg_q4_plan_create(None, None, ctypes.byref(out)) == BAD and out.value is None
    assert lib.gg_q4_plan_run(None, PTR, 8, 1, None, PTR, PTR, 8, 1, None) == GONE
    assert lib.gg_q4_plan_status(None, ctypes.byref(ctypes.c_int())) == GONE
    lib.gg_q4_plan_destroy(None)


@pytest.mark.parametrize("change", [dict(experts=0), dict(experts=1025), dict(n=0), dict(k=0), dict(k=-3), dict(group=0),
                                    dict(group=16), dict(group=96), dict(group=192), dict(ldq=31), dict(input_type=2),
                                    dict(input_type=-1), dict(output_type=3), dict(activation=3), dict(activation=-1),
                                    dict(q=None), dict(scales=None), dict(zeros=None)])
def test_q4_problems_out_of_range_are_refused(change):
    f = dict(experts=2, n=16, k=64, group=32, ldq=32, input_type=0, output_type=0, activation=0) | {
        n: v for n, v in change.items() if n not in ("q", "scales", "zeros")}
    table = lambda: (ctypes.c_void_p * 1100)(*[PTR] * 1100)  # noqa: E731
    q, scales, zeros = table(), table(), table()
    for name, t in (("q", q), ("scales", scales), ("zeros", zeros)):
        if name in change:
            t[1] = None  # one expert's pointer is missing
    cast = lambda t: ctypes.cast(t, ctypes.POINTER(ctypes.c_void_p))  # noqa: E731
    out = ctypes.c_void_p()
    prob = capi.GGQ4Problem(cast(q), cast(scales), cast(zeros), None, f["experts"], f["n"], f["k"], f["group"], f["ldq"],
                            f["input_type"], f["output_type"], f["activation"])
    assert capi.load().gg_q4_plan_create(ctypes.byref(prob), None, ctypes.byref(out)) == BAD


def test_q4_tables_have_one_entry_per_expert():
    with pytest.raises(ValueError):
        gg.Q4Plan(2, 16, 64, 32, [PTR], 32, [PTR, PTR])
    with pytest.raises(ValueError):
        gg.Q4Plan(2, 16, 64, 32, [PTR, PTR], 32, [PTR, PTR], bias_ptrs=[None])


@pytest.mark.parametrize("change", [dict(tokens=-1), dict(top_k=0), dict(width=-1), dict(width=2 ** 30 + 1, ld=2 ** 30 + 1, ldp=2 ** 30 + 1), dict(rows=-1), dict(ld=7), dict(ldp=7),
                                    dict(x=None), dict(pos=None), dict(packed=None), dict(size=8), dict(size=0)])
def test_row_moves_refuse_what_does_not_fit(change):
    lib = capi.load()
    f = dict(x=PTR, ld=8, pos=PTR, tokens=2, top_k=2, width=8, size=4, packed=PTR, rows=4, ldp=8) | change
    assert lib.gg_moe_dispatch(f["x"], f["ld"], f["pos"], f["tokens"], f["top_k"], f["width"], f["size"], f["packed"],
                               f["rows"], f["ldp"], None) == BAD
    t = 0 if f["size"] == 4 else 3  # an unknown type in the place of an unknown size
    assert lib.gg_moe_combine(f["packed"], t, f["rows"], f["ldp"], f["pos"], None, f["tokens"], f["top_k"], f["width"],
                              f["x"], 0, f["ld"], None) == BAD
    assert lib.gg_moe_combine_backward(f["x"], 0, f["ld"], f["packed"], t, f["rows"], f["ldp"], f["pos"], PTR, f["tokens"],
                                       f["top_k"], f["width"], PTR, 8, PTR, None) == BAD
    if not change.keys() & {"x", "pos", "packed", "size", "ld"}:
        return
    assert lib.gg_moe_combine_backward(PTR, 0, 8, PTR, 0, 4, 8, PTR, None, 2, 2, 8, PTR, 8, PTR, None) == BAD
    assert lib.gg_moe_combine_backward(PTR, 0, 8, PTR, 0, 4, 8, PTR, PTR, 2, 2, 8, PTR, 8, None, None) == BAD
    assert lib.gg_moe_combine_backward(PTR, 0, 8, PTR, 0, 4, 8, PTR, PTR, 2, 2, 8, PTR, 7, PTR, None) == BAD


def test_empty_moves_need_no_device():
    lib = capi.load()
    assert lib.gg_moe_dispatch(None, 8, None, 0, 2, 8, 4, None, 4, 8, None) == 0
    assert lib.gg_moe_combine(None, 0, 0, 8, None, None, 0, 2, 8, None, 0, 8, None) == 0
    assert lib.gg_moe_combine_backward(None, 0, 8, None, 0, 0, 8, None, None, 0, 2, 8, None, 8, None, None) == 0


def test_q4_rows_of_the_longest_k_need_their_bytes():
    """k = 2^31 - 1 takes a pitch of 2^30 bytes like any other takes ceil(k / 2): a shorter one is refused."""
    table = (ctypes.c_void_p * 1)(PTR)
    cast = ctypes.cast(table, ctypes.POINTER(ctypes.c_void_p))
    for k in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 3):
        out = ctypes.c_void_p()
        prob = capi.GGQ4Problem(cast, cast, None, None, 1, 16, k, 128, (k - 1) // 2, 0, 0, 0)
        assert capi.load().gg_q4_plan_create(ctypes.byref(prob), None, ctypes.byref(out)) == BAD


def test_current_device_needs_a_place():
    assert capi.load().gg_current_device(None) == BAD
