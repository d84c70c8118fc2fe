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


def route64(logits, top_k, use_softmax, renorm):
    """(ids, weights, values ranked) of logits [T, E] in their type: probabilities are rounded to the type before they
    are ranked, equal ones go to the lowest expert."""
    dt, v = logits.dtype, logits.double()
    if use_softmax:
        p = torch.softmax(v, 1)
        ranked = p.to(dt)
        w, ids = torch.sort(ranked, dim=1, descending=True, stable=True)
        w, ids = w[:, :top_k].double(), ids[:, :top_k]
        if renorm:
            w = w / w.sum(1, keepdim=True).to(dt).double()
        return ids, w.to(dt), p
    w, ids = torch.sort(v, dim=1, descending=True, stable=True)
    return ids[:, :top_k], torch.softmax(w[:, :top_k], 1).to(dt), v


def assert_routing(ids, weights, logits, top_k, use_softmax, renorm):
    """Ids and weights against the 64-bit routing of the same logits.  A probability may be rounded the other way where
    its fp32 value falls beside a border of its type (one unit, eps relative): a pick may differ only where the two
    values lie within two units, and a weight by the roundings of its probability, of the sum and of the quotient."""
    eps = torch.finfo(logits.dtype).eps
    want, w, ranked = route64(logits, top_k, use_softmax, renorm)
    for t in torch.nonzero((ids != want).any(1)).flatten().tolist():
        a, b = ranked[t, ids[t]], ranked[t, want[t]]
        assert len(set(ids[t].tolist())) == top_k, f"token {t}: an expert twice"
        assert bool(((a - b).abs() <= 2 * eps * b.abs()).all()), f"token {t}: {ids[t].tolist()} for {want[t].tolist()}"
        assert use_softmax, f"token {t}: logits are ranked as they are"
    d = (weights.double() - w.double()).abs()
    assert bool((d <= 3 * eps * w.double().abs() + SUBNORMAL[logits.dtype] * 4).all()), float(d.max())


def moe64(x, ids, weights, gate, up, down, shared=None, residual=None):
    """(exact value, allowed distance) of the layer's output on a given routing.

    h = w silu(g) u is kept as two values of the type: (eps / 2)^2 relative and 2^-25 (fp16) absolute are lost.  The down
    projection's sum runs over the high and low parts of every routed expert's h."""
    t, top_k = ids.shape
    dt, hid, inter = x.dtype, gate.shape[2], gate.shape[1]
    xd, half = x.double(), torch.finfo(dt).eps / 2
    v = torch.zeros(t, hid, dtype=torch.float64, device=x.device)
    err, mass = torch.zeros_like(v), torch.zeros_like(v)

    def add(rows, scale, g_w, u_w, d_w):
        nonlocal v, err, mass
        g, eg = _product(x[rows], g_w)
        u, eu = _product(x[rows], u_w)
        a = g * torch.sigmoid(g)
        ea = SLOPE * eg + 16 * 2.0 ** -23 * (1 + g.abs())
        s = scale.double().unsqueeze(1)
        h = s * a * u
        eh = s.abs() * (a.abs() * eu + u.abs() * ea + ea * eu) + 8 * 2.0 ** -23 * h.abs()
        eh = eh + half * half * (h.abs() + eh) + 2 * SUBNORMAL[dt]
        dd = d_w.double()
        v[rows] += h @ dd.t()
        err[rows] += eh @ dd.abs().t()
        mass[rows] += h.abs() @ dd.abs().t()

    for e in sorted(set(ids.flatten().tolist())):
        if e < 0 or e >= gate.shape[0]:
            continue
        hit = ids == e
        rows = torch.nonzero(hit.any(1)).flatten()
        add(rows, (weights.double() * hit).sum(1)[rows], gate[e], up[e], down[e])
    k = 2 * top_k * inter
    if shared is not None:
        every = torch.arange(t, device=x.device)
        gv = xd @ shared["gate_vec"].double()
        scale = torch.sigmoid(gv)
        add(every, scale, shared["gate"], shared["up"], shared["down"])
        # the gate's own sum: K = hidden in fp32 over 128 threads, slope of the sigmoid at most 1/4
        eg = (hid / 8 + 64) * 2.0 ** -23 * (xd.abs() @ shared["gate_vec"].double().abs()) / 4 + 8 * 2.0 ** -23
        g, _ = _product(x, shared["gate"])
        u, _ = _product(x, shared["up"])
        err += eg.unsqueeze(1) * ((g * torch.sigmoid(g) * u).abs() @ shared["down"].double().abs().t())
        k += 2 * shared["gate"].shape[0]
    err = err + (k / 8 + 64) * 2.0 ** -23 * mass
    if residual is not None:
        v = v + residual.double()
    return v, _rounded(v, err, dt)
