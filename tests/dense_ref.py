"""Plain 64-bit forms of the dense operators, with the bound each result has to keep.

Bound of a projection.  Products of two 16-bit values are exact in fp32.  A tensor-core step adds
16 products to an fp32 sum: its terms are aligned to the largest and cut, so the step errs by at
most 2 units of 2^-23 of S = sum |x w|; a K-long sum takes K / 16 such steps, and the joins of
partial sums (at most 64) and the fp32 adds of bias and residual one rounding each.  Hence
|sum - exact| <= (K / 8 + 64) 2^-23 S'.  The activations' slope is at most 1.13 (gelu's maximum
1.129, silu's 1.100) and they cost at most 16 fp32 roundings of values up to 1 + |v|.  The result
is rounded once to its type: half a unit, eps / 2 relative, and 2^-25 absolute where fp16 is
subnormal (2^-134 for bf16).
"""
import math

import torch

SUBNORMAL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
SLOPE = 1.13


def act64(v, name):
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)))
    if name == "relu":
        return v.clamp_min(0.0)
    return v


def _product(x, w):
    x, w = x.double(), w.double()
    return x @ w.t(), (x.shape[1] / 8 + 64) * 2.0 ** -23 * (x.abs() @ w.abs().t())


def _rounded(v, err, dtype):
    err = err * (1 + 2.0 ** -20) + 2.0 ** -22 * v.abs()
    return err + torch.finfo(dtype).eps / 2 * (v.abs() + err) + SUBNORMAL[dtype]


def linear64(x, w, bias=None, activation=None, residual=None):
    """(exact value, allowed distance of the rounded result from it)"""
    v, err = _product(x, w)
    if bias is not None:
        v = v + bias.double()
        err = err + 2.0 ** -23 * v.abs()
    if activation not in (None, "none"):
        err = SLOPE * err + 16 * 2.0 ** -23 * (1 + v.abs())
        v = act64(v, activation)
    if residual is not None:
        v = v + residual.double()
    return v, _rounded(v, err, x.dtype)


def gated64(x, wg, wu, activation="silu"):
    g, eg = _product(x, wg)
    u, eu = _product(x, wu)
    a = act64(g, activation)
    ea = SLOPE * eg + 16 * 2.0 ** -23 * (1 + g.abs())
    v = a * u
    return v, _rounded(v, a.abs() * eu + u.abs() * ea + ea * eu, x.dtype)


def assert_within(got, ref, what=""):
    v, bound = ref
    d = (got.double() - v).abs()
    bad = ~(d <= bound)
    if bad.any():
        i = int(torch.argmax((d - bound).flatten()))
        raise AssertionError(f"{what}: {int(bad.sum())} of {d.numel()} outside; at {i}: got {float(got.flatten()[i])} "
                             f"exact {float(v.flatten()[i])} allowed {float(bound.flatten()[i]):.3e}")
