"""GELU and its tanh approximation where they are small: far out on the negative side the result is a tiny multiple of
its argument, and each of its own bits has to be right, not only its distance on the scale of the argument.

The arguments are made exactly: a zero product plus a bias, or one product by 1.  Bounds, relative to the result, of an
fp32 evaluation at an exact argument v (a unit is 2^-23, an operation half a unit, expf 2 units, erfcf 4):
gelu = v/2 erfc(z), z = -v/sqrt 2 off by a unit, which erfc magnifies by at most 2 z^2 + 2 = v^2 + 2; two products:
(v^2 + 8) units.  gelu_tanh = v s(2 y): 2 y off by 3 units, which exp magnifies by |2 y|; exp 2, quotient 2, sum and
product 2 halves: (6 |y| + 6) units.  Then one rounding to the type."""
import math

import pytest
import torch

from tests import dense_ref as dr

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def expected(v, name, dtype):
    """(exact value at v, allowed distance of the result from it)"""
    v = v.double()
    if name == "gelu":
        out, units = 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5)), v * v + 8
    else:
        y = math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)
        e = torch.exp(-2.0 * y.abs())
        out, units = v * torch.where(y < 0, e, torch.ones_like(e)) / (1.0 + e), 6 * y.abs() + 6
    return out, dr._rounded(out, units * 2.0 ** -23 * out.abs(), dtype)


def arguments(n, dtype, dev):
    """n values of the type, most of them between -9.5 and -2, some positive, some near zero"""
    v = torch.cat([torch.linspace(-9.5, -2.0, 700), torch.linspace(-2.0, 6.0, 150), torch.linspace(-0.01, 0.01, 50)])
    return v.to(dtype).to(dev)[torch.arange(n, device=dev) % 900]


def check(got, v, name):
    dr.assert_within(got, tuple(t.expand_as(got) for t in expected(v, name, got.dtype)), name)


# one token, a few, a prompt, rows that no wide load takes, many tiles of a pair of SMs
SHAPES = [(1, 900, 64), (20, 901, 64), (200, 900, 128), (40, 900, 77), (4000, 5000, 256)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("name", ["gelu", "gelu_tanh"])
@pytest.mark.parametrize("shape", SHAPES)
def test_small_results_of_a_projection(shape, name, dtype, cuda_device):
    from nano_ktrans_b200 import linear

    m, n, k = shape
    x, w = torch.zeros(m, k, dtype=dtype, device=cuda_device), torch.ones(n, k, dtype=dtype, device=cuda_device)
    v = arguments(n, dtype, cuda_device)
    check(linear(x, w, v, activation=name), v, name)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("name", ["gelu", "gelu_tanh"])
@pytest.mark.parametrize("shape", SHAPES)
def test_small_results_of_a_gated_product(shape, name, dtype, cuda_device):
    from nano_ktrans_b200 import gated_linear

    m, n, k = shape
    x, wg, wu = (torch.zeros(r, k, dtype=dtype, device=cuda_device) for r in (m, n, n))
    v = arguments(n, dtype, cuda_device)
    x[:, 0], wg[:, 0], wu[:, 0] = 1, v, 1
    check(gated_linear(x, wg, wu, activation=name), v, name)


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh"])
@pytest.mark.parametrize("m", [1, 200])
def test_ends_of_the_range(m, name, cuda_device):
    """Far arguments: the identity on one side, zero on the other, no overflow on the way; NaN stays."""
    from nano_ktrans_b200 import linear

    v = torch.tensor([-3e38, -1e20, -100.0, -20.0, 20.0, 100.0, 1e20, 3e38, float("inf"), float("nan"), -0.0, 0.0],
                     dtype=BF16, device=cuda_device)
    x, w = torch.zeros(m, 64, dtype=BF16, device=cuda_device), torch.ones(12, 64, dtype=BF16, device=cuda_device)
    out = linear(x, w, v, activation=name)
    assert bool((out[:, :4] == 0).all()) and torch.equal(out[:, 4:9], v[4:9].expand(m, 5))
    assert bool(out[:, 9].isnan().all()) and bool((out[:, 10:] == 0).all())
