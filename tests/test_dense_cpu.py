"""Argument checks of the dense operators that need no GPU: the C entry refuses before it launches anything."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nano_ktrans_b200 import _lib, build

    build.build()
    return _lib.lib()


def desc(**kw):
    from nano_ktrans_b200 import _lib

    # addresses that no call here reaches: every one of these descriptions is refused
    d = dict(x_dev=0x10000, w_dev=0x20000, w_up_dev=None, bias_dev=None, residual_dev=None, out_dev=0x90000,
             ldx=64, ldw=64, ldw_up=64, ldr=32, ldo=32, m=4, n=32, k=64, dtype=0, activation=0)
    d.update(kw)
    return _lib.MoeLinearDesc(**d)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(activation=9), "activation"),
    (dict(activation=-1), "activation"), (dict(m=-1), "m must be"), (dict(n=0), "n and k"), (dict(k=0), "n and k"),
    (dict(x_dev=None), "null"), (dict(w_dev=None), "null"), (dict(out_dev=None), "null"),
    (dict(x_dev=0x10001), "aligned"), (dict(ldx=63), "apart"), (dict(ldw=10), "apart"), (dict(ldo=31), "apart"),
    (dict(residual_dev=0x50000, ldr=16), "apart"), (dict(w_up_dev=0x30000, ldw_up=2), "apart"),
    (dict(w_up_dev=0x30000, bias_dev=0x40000), "gated"), (dict(w_up_dev=0x30000, residual_dev=0x40000), "gated"),
    (dict(out_dev=0x10000), "overlaps"), (dict(out_dev=0x20002), "overlaps"),
    (dict(residual_dev=0x90002), "overlaps"), (dict(residual_dev=0x90000, ldr=40), "overlaps"),
    (dict(bias_dev=0x90000), "overlaps"), (dict(w_up_dev=0x90000 - 2), "overlaps"),
])
def test_linear_refuses(lib, kw, needle):
    from nano_ktrans_b200 import _lib

    err = ctypes.create_string_buffer(256)
    d = desc(**kw)
    assert lib.moe_linear(ctypes.byref(d), None, err, len(err)) == _lib.MOE_EINVAL
    assert needle in err.value.decode()
    assert lib.moe_linear(ctypes.byref(d), None, None, 0) == _lib.MOE_EINVAL  # no buffer for the message


def test_linear_without_rows_and_without_description(lib):
    from nano_ktrans_b200 import _lib

    d = desc(m=0, x_dev=None, out_dev=None)
    assert lib.moe_linear(ctypes.byref(d), None, None, 0) == _lib.MOE_OK
    assert lib.moe_linear(None, None, None, 0) == _lib.MOE_EINVAL


def test_host_tensors_are_refused():
    from nano_ktrans_b200 import gated_linear, linear

    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        linear(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        gated_linear(x, w, w)


def test_dense_mlp_checks_its_shapes():
    from nano_ktrans_b200 import DenseMLP

    g = torch.zeros(8, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="gate and up"):
        DenseMLP(g, g, g)
    mlp = DenseMLP(g, g, g.t())
    assert (mlp.hidden_size, mlp.intermediate_size) == (4, 8)
