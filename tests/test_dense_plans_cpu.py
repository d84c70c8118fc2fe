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


# An SM's shared memory; what a block is charged beside its dynamic part: 1024 reserved, and static variables
SM_BYTES, BLOCK_BYTES = 233472, 1024 + 256


def clusters():
    """Plans whose blocks wait for one another, over the whole range of sizes."""
    ms = [33, 40, 64, 80, 100, 128, 129, 136, 200, 256, 257, 333, 600, 1024, 3000]
    ns = [1, 16, 24, 100, 256, 330, 768, 1001, 1408, 2048, 4096, 5000, 9738, 17326, 151936]
    ks = [40, 72, 128, 200, 264, 512, 520, 1024, 1408, 2048, 4096, 14336]
    out = {}
    for gated in (False, True):
        for m in ms:
            for n in ns:
                for k in ks:
                    p = dp.plan(m, n, k, gated)
                    if p["kernel"] == "pair" or (p["kernel"] == "split" and p["splits"] > 1):
                        out[(p["tmem_columns"], p["smem_bytes"])] = (m, n, k, gated, p)
    return out


def test_blocks_that_wait_for_one_another_never_wait_for_tensor_memory():
    """Blocks of clusters that fit an SM together by their shared memory, of the same or of different calls, ask for at
    most the 512 columns that it has: otherwise one could hold some and wait for a block that waits for them."""
    found = clusters()
    assert {t for t, _ in found} == {32, 64, 128, 256, 512} and any(v[4]["kernel"] == "pair" for v in found.values())
    for (columns, smem), case in found.items():
        # in proportion: blocks of more than 512 columns, in steps of 32, together exceed the SM
        assert (smem + BLOCK_BYTES) * 544 > SM_BYTES * columns, case
        assert smem + 272 <= 232448, case
    least = {}
    for columns, smem in found:
        least[columns] = min(smem, least.get(columns, smem))

    def fill(columns, room):
        for c, smem in least.items():
            if smem + BLOCK_BYTES <= room:
                assert columns + c <= 512, (columns, c, least)
                fill(columns + c, room - smem - BLOCK_BYTES)

    fill(0, SM_BYTES)


MOST = (1 << 31) - 256


@pytest.mark.parametrize("name", ["m", "n", "k"])
def test_sizes_whose_tiles_leave_32_bits(name):
    """Row and column numbers are 32 bits in the kernels, a tile's last ones beyond the tensor's end included."""
    from nano_ktrans_b200 import _lib

    L, err, out = _lib.lib(), ctypes.create_string_buffer(256), _lib.MoeLinearPlan()
    for size, code in ((MOST, _lib.MOE_OK), (MOST + 1, _lib.MOE_EINVAL), ((1 << 31) - 1, _lib.MOE_EINVAL)):
        d = dict(m=1, n=8, k=8, x_dev=1 << 50, w_dev=1 << 51, out_dev=1 << 52)
        d[name] = size
        d.update(ldx=d["k"], ldw=d["k"], ldo=d["n"])
        for rows in (1, 33) if name != "m" else (size,):
            d["m"] = rows
            assert L.moe_linear_query(ctypes.byref(_lib.MoeLinearDesc(**d)), ctypes.byref(out), err, 256) == code, err.value
            assert code == _lib.MOE_OK or b"2^31 - 256" in err.value
