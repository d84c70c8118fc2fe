"""The kernel that each range of sizes takes, asked without a device."""
import ctypes

import pytest

from tests import dense_plans as dp


@pytest.fixture(scope="module", autouse=True)
def built():
    from nano_ktrans_b200 import build

    build.build()


@pytest.mark.parametrize("gated", [False, True])
def test_ranges(gated):
    assert dp.kernel(0, 64, 64, gated) == "none"
    for m in (1, 7, 32):
        assert dp.kernel(m, 2048, 2048, gated) == "stream"
    for m, n, k in ((33, 2048, 2048), (200, 2048, 1408), (333, 1001, 1000), (700, 330, 256)):
        assert dp.kernel(m, n, k, gated) == "split"
    for m, n, k in ((2048, 4096, 14336), (4000, 5001, 1024), (3765, 5789, 152), (2048, 4096, 4096)):
        assert dp.kernel(m, n, k, gated) == "pair"


@pytest.mark.parametrize("m", [1, 100, 4000])
def test_rows_that_no_wide_load_can_take(m):
    assert dp.kernel(m, 5000, 1023) == "generic"
    for kw in (dict(ldx=1028), dict(x_dev=(1 << 40) + 2), dict(w_dev=(1 << 41) + 8), dict(ldw=1025)):
        assert (dp.kernel(m, 5000, 1024, **kw) == "generic") == (m > 1 or "ldx" not in kw)
    # outputs, biases and residuals may lie anywhere
    assert dp.kernel(m, 5000, 1024, out_dev=(1 << 43) + 2, ldo=5001, bias_dev=(1 << 44) + 6, residual_dev=(1 << 45) + 2) != "generic"


def test_refusals():
    from nano_ktrans_b200 import _lib

    L, err, out = _lib.lib(), ctypes.create_string_buffer(256), _lib.MoeLinearPlan()
    d = _lib.MoeLinearDesc(m=1, n=0, k=1)
    assert L.moe_linear_query(ctypes.byref(d), ctypes.byref(out), err, 256) == _lib.MOE_EINVAL and b"n and k" in err.value
    assert L.moe_linear_query(ctypes.byref(d), None, err, 256) == _lib.MOE_EINVAL
    assert L.moe_linear_query(None, ctypes.byref(out), None, 0) == _lib.MOE_EINVAL
