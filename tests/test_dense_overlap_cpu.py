"""Which overlaps of an output with other tensors the dense operators refuse, against a plain enumeration of the bytes.
Asked of ``moe_linear_query``, which checks what ``moe_linear`` checks and launches nothing."""
import ctypes
import random

import pytest


@pytest.fixture(scope="module")
def lib():
    from nano_ktrans_b200 import _lib, build

    build.build()
    return _lib.lib()


BASE = 1 << 30


def elements(at, rows, cols, ld):
    return {at + r * ld + c for r in range(rows) for c in range(cols)}


def refused(lib, **kw):
    from nano_ktrans_b200 import _lib

    d = dict(x_dev=1 << 40, w_dev=1 << 41, w_up_dev=None, bias_dev=None, residual_dev=None, ldw=64, ldw_up=64, ldr=64,
             dtype=0, activation=0)
    d.update(kw)
    err, out = ctypes.create_string_buffer(256), _lib.MoeLinearPlan()
    rc = lib.moe_linear_query(ctypes.byref(_lib.MoeLinearDesc(**d)), ctypes.byref(out), err, 256)
    assert rc == _lib.MOE_OK or b"overlaps" in err.value, err.value
    return rc != _lib.MOE_OK


def test_column_ranges_of_one_buffer(lib):
    """x, residual and output side by side in one buffer, as a fused projection's parts lie, are no overlap."""
    m, k, n, ld = 5, 16, 24, 64
    at = dict(x_dev=BASE, ldx=ld, m=m, n=n, k=k, ldo=ld)
    assert not refused(lib, out_dev=BASE + 2 * 16, **at)
    assert not refused(lib, out_dev=BASE + 2 * 40, residual_dev=BASE + 2 * 16, **dict(at, ldr=ld))
    assert refused(lib, out_dev=BASE + 2 * 15, **at)        # a column of x
    assert refused(lib, out_dev=BASE + 2 * 41, **at)        # the last column is x's first one of the next row
    assert refused(lib, out_dev=BASE + 2 * (ld + 8), **at)  # the same columns, a row below
    # rows before, after and between
    assert not refused(lib, out_dev=BASE + 2 * (m * ld), **at)
    assert not refused(lib, out_dev=BASE - 2 * (m * ld), **at)
    assert not refused(lib, out_dev=BASE + 2 * (16 - 2 * ld), **at)


@pytest.mark.parametrize("seed", range(40))
def test_against_the_bytes(lib, seed):
    rng = random.Random(seed)
    for _ in range(50):
        m, k, n = rng.randint(1, 6), rng.randint(1, 9), rng.randint(1, 9)
        step = rng.randint(max(k, n), 24)
        same = rng.random() < 0.7
        ldx = step if same else rng.randint(k, 24)
        ldo = step if same else rng.randint(n, 24)
        ldr = step if same else rng.randint(n, 24)
        out, res = rng.randint(-60, 60), rng.randint(-60, 60)
        o, x, r = elements(out, m, n, ldo), elements(0, m, k, ldx), elements(res, m, n, ldr)
        got = refused(lib, x_dev=BASE, out_dev=BASE + 2 * out, residual_dev=BASE + 2 * res, m=m, n=n, k=k, ldx=ldx, ldo=ldo, ldr=ldr)
        in_place = res == out and ldr == ldo
        met = bool(o & x) or (bool(o & r) and not in_place)
        if met:
            assert got, (m, k, n, ldx, ldo, ldr, out, res)
        elif m == 1 or ldx == ldo == ldr:
            assert not got, (m, k, n, ldx, ldo, ldr, out, res)  # one step: exact; of others, refusing is safe


def test_a_bias_or_weight_within_the_rows_of_the_output(lib):
    """A one-piece operand in the gap between the output's columns and the next row is no overlap."""
    at = dict(m=4, n=16, k=8, ldx=8, ldo=64, out_dev=BASE)
    assert not refused(lib, bias_dev=BASE + 2 * 20, **at)
    assert refused(lib, bias_dev=BASE + 2 * 50, **at)  # reaches into the next row
    assert refused(lib, bias_dev=BASE + 2 * 64, **at)
    assert not refused(lib, w_dev=BASE + 2 * 16, ldw=64, **at)  # [16, 8]: its rows lie between the output's
    assert refused(lib, w_dev=BASE + 2 * 60, ldw=64, **at)
