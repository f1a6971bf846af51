"""Host-side checks of the dense-layer and AdamW entry points that need no GPU: bad calls are refused before any device work."""
import ctypes as C
import os
import re

import pytest
import torch

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


class OnGpu(torch.Tensor):
    """A host tensor that says it is on the GPU: what the checks of layouts look at is the same."""
    is_cuda = True


class Pinned(torch.Tensor):
    def is_pinned(self):
        return True


def gpu(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)


BF, F32 = capi._dtypes("bf16"), capi._dtypes("f32")


@pytest.mark.parametrize("x,ld", [
    (gpu(4, 8), 8), (gpu(4, 8), 16), (gpu(32), 8), (gpu(2, 2, 8), 8), (gpu(4, 12)[:, :8], 12), (gpu(4, 12)[:, 3:11], 24), (gpu(2, 2, 12)[..., :8], 12), (gpu(8, 8)[::2], 16),
    (gpu(4, 8, dtype=torch.int16), 8), (gpu(1, 12)[:, :8], 8), (gpu(1, 12)[:, :8], 77), (gpu(5, 1), 1), (gpu(8, 4)[:, 1:2], 4), (gpu(0, 8), 8), (gpu(4, 12)[1:, 4:], 12),
    (gpu(1, 2, 12)[:, :1, :8], 5)])
def test_matrices_that_are_taken(x, ld):
    assert capi._matrix(x, ld, BF, "x") == x.data_ptr()


@pytest.mark.parametrize("x,ld", [
    (gpu(4, 8, dtype=torch.float32), 8), (gpu(4, 8, dtype=torch.float16), 8), (torch.zeros(4, 8, dtype=torch.bfloat16), 8), (gpu(8, 4).t(), 8), (gpu(8, 8).t(), 8),
    (gpu(4, 12)[:, :8], 8), (gpu(2, 3, 12)[:, :2, :8], 12), (gpu(1, 8).expand(4, 8), 8), (gpu(4, 16)[:, ::2], 16), (gpu(16)[::2], 8)])
def test_matrices_that_are_refused(x, ld):
    with pytest.raises(capi.CoconetError) as e:
        capi._matrix(x, ld, BF, "x")
    assert e.value.code == capi.CCN_EINVAL and "x needs" in str(e.value)


def test_arrays():
    for x, n in ((gpu(8, dtype=torch.float32), 8), (gpu(8, dtype=torch.float32), 3), (gpu(2, 4, dtype=torch.float32), 8)):
        assert capi._array(x, n, F32, "b") == x.data_ptr()
    pinned = torch.zeros(4, 8).as_subclass(Pinned)      # host memory that the GPU reads
    assert capi._array(pinned, 32, F32, "b") == pinned.data_ptr() and capi._matrix(pinned, 8, F32, "b") == pinned.data_ptr()
    assert capi._array(None, 8, F32, "b") is None and capi._array(4096, 8, F32, "b") == 4096
    assert capi._matrix(None, 8, BF, "b") is None and capi._matrix(4096, 8, BF, "b") == 4096
    for x, code in ((gpu(8), capi.CCN_EINVAL), (torch.zeros(8), capi.CCN_EINVAL), (gpu(16, dtype=torch.float32)[::2], capi.CCN_EINVAL),
                    (gpu(7, dtype=torch.float32), capi.CCN_ERANGE)):
        with pytest.raises(capi.CoconetError) as e:
            capi._array(x, 8, F32, "b")
        assert e.value.code == code


def adamw_plan(*counts):
    plan = capi.AdamWPlan.__new__(capi.AdamWPlan)      # what tables() looks at; a plan itself is made on the GPU
    plan.counts, plan.h = list(counts), None
    return plan


def test_adamw_tables_that_are_taken():
    f = lambda *s: gpu(*s, dtype=torch.float32)  # noqa: E731
    plan = adamw_plan(12, 0, 5)
    g, w, h = [[gpu(12), None, gpu(5)], [gpu(3, 4), None, gpu(9)]], [f(4, 3), None, f(5)], [gpu(12), None, gpu(5)]
    gt, P, wt, ht = plan.tables(g, w, h)
    assert P == 2 and list(gt) == [None if x is None else x.data_ptr() for r in g for x in r] and list(wt) == [None if x is None else x.data_ptr() for x in w]
    assert gt.names == ["bf16"] and wt.names == ["f32"] and ht.names == ["bf16"]
    assert plan.tables([[4096, 0, 8192]], [4096, 0, 8192])[0].names == ["f32", "bf16", "f16"]
    assert plan.tables([[x if x is None else x.view(torch.int16) for x in g[0]]], w)[0].names == ["bf16", "f16"]
    plan.tables([[gpu(3, 4).t(), None, gpu(5)]], [f(3, 4).t(), None, f(5)], [gpu(3, 4).t(), None, gpu(5)])   # all in the same order


@pytest.mark.parametrize("g,w,h,code", [
    ([gpu(12), gpu(5, dtype=torch.float16)], None, None, capi.CCN_EINVAL), ([gpu(12, dtype=torch.float64), gpu(5, dtype=torch.float64)], None, None, capi.CCN_EINVAL),
    ([torch.zeros(12), torch.zeros(5)], None, None, capi.CCN_EINVAL), ([gpu(11), gpu(5)], None, None, capi.CCN_ERANGE), ([gpu(24)[::2], gpu(5)], None, None, capi.CCN_EINVAL),
    ([gpu(4, 3).t(), gpu(5)], None, None, capi.CCN_EINVAL), (None, [gpu(12), gpu(5)], None, capi.CCN_EINVAL),
    (None, [gpu(3, 4, dtype=torch.float32).t(), gpu(5, dtype=torch.float32)], None, capi.CCN_EINVAL), (None, None, [gpu(12, dtype=torch.float32), gpu(5)], capi.CCN_EINVAL),
    (None, None, [gpu(12), gpu(4)], capi.CCN_ERANGE)])
def test_adamw_tables_that_are_refused(g, w, h, code):
    good = [gpu(12), gpu(5)], [gpu(12, dtype=torch.float32), gpu(5, dtype=torch.float32)], [gpu(12), gpu(5)]
    with pytest.raises(capi.CoconetError) as e:
        adamw_plan(12, 5).tables([g or good[0]], w or good[1], h or good[2])
    assert e.value.code == code
