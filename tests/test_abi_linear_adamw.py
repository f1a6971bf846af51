"""Host-side checks of the dense-layer and AdamW entry points that need no GPU: bad calls are refused before any device work."""
import ctypes as C
import os
import re

from coconet_amd import capi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "coconet_hip.h")


def test_constants_match_the_header():
    text = open(HEADER).read()
    for name, value in [("ACT_" + k.upper(), v) for k, v in capi.ACTS.items()] + [("TYPE_" + k.upper(), v) for k, v in capi.TYPES.items()]:
        assert int(re.search(rf"#define\s+CCN_{name}\s+(\d+)", text).group(1)) == value


def test_linear_refusals():
    lib = capi.load()
    plan = C.c_void_p(1)
    for dims in ((0, 8, 8), (8, 0, 8), (8, 8, -1)):
        assert lib.ccn_linear_plan_create(*dims, C.byref(plan)) == capi.CCN_EINVAL and not plan.value
    assert lib.ccn_linear_plan_create(8, 8, 8, None) == capi.CCN_EINVAL
    for dims in ((8, (1 << 21) + 1, 8), (8, 8, (1 << 21) + 1), ((1 << 30) + 1, 8, 8)):
        assert lib.ccn_linear_plan_create(*dims, C.byref(plan)) == capi.CCN_ERANGE
    assert lib.ccn_linear_plan_destroy(None) == capi.CCN_OK
    for t in ("bf16", "f16"):
        assert getattr(lib, "ccn_linear_" + t)(None, 0x1000, 8, 0x1000, 8, None, None, 0, 0x1000, 8, None, 0, 8, 8, 8, 0, None) == capi.CCN_EINVAL
        assert getattr(lib, "ccn_linear_backward_" + t)(None, 0x1000, 8, None, 0, 0x1000, 8, 0x1000, 8, 0x1000, 8, 0x1000, 8, 0, 0x1000, 0, 8, 8, 8, 0,
                                                         None) == capi.CCN_EINVAL


def test_adamw_refusals():
    lib = capi.load()
    plan = C.c_void_p(1)
    counts = (C.c_size_t * 2)(10, 20)
    for bits in (0, 4, 16, 64):
        assert lib.ccn_adamw_plan_create(counts, None, 2, bits, C.byref(plan)) == capi.CCN_EINVAL and not plan.value
    assert lib.ccn_adamw_plan_create(None, None, 2, 32, C.byref(plan)) == capi.CCN_EINVAL
    assert lib.ccn_adamw_plan_create(counts, None, 0, 32, C.byref(plan)) == capi.CCN_EINVAL
    assert lib.ccn_adamw_plan_create(counts, None, 2, 32, None) == capi.CCN_EINVAL
    huge = (C.c_size_t * 1)(1 << 62)
    assert lib.ccn_adamw_plan_create(huge, None, 1, 32, C.byref(plan)) == capi.CCN_ERANGE and not plan.value
    many = (C.c_size_t * 3)(1 << 38, 1 << 38, 1)      # 2^31 blocks and one more
    assert lib.ccn_adamw_plan_create(many, None, 3, 32, C.byref(plan)) == capi.CCN_ERANGE and not plan.value
    assert lib.ccn_adamw_plan_destroy(None) == capi.CCN_OK
    assert lib.ccn_adamw_plan_sizes(None, None, None) == capi.CCN_EINVAL
    tbl = (C.c_void_p * 4)(*([0x1000] * 4))
    p = C.cast(tbl, C.POINTER(C.c_void_p))
    assert lib.ccn_adamw_scattered(None, p, 2, 0, p, None, 0, 0x1000, 0x1000, None, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, 1.0, None, None, None) == capi.CCN_EINVAL
