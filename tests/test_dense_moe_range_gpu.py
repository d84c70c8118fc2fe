"""fp16 expert layers whose intermediate values h = w silu(g) u lie far above and far below fp16's own range: they are
kept as two fp16 values each, but on a scale of their token and expert, so that the layer's result is what the formula
gives in fp32.

Bound: as dense_ref.moe64's, with the loss of h stated on its scale.  The largest |h| of a token's piece lies in
[2^14, 2^15) there: an h loses 2^-22 of itself or, where its second part is subnormal, 2^-25 of the scale, at most
2^-39 of the largest.  A piece is a part of the expert's rows; the expert's largest bounds every piece's."""
import pytest
import torch

from tests import dense_ref as dr

pytestmark = pytest.mark.gpu

FP16 = torch.float16


def rnd(dev, seed, *shape, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(FP16)


def scaled64(x, ids, weights, gate, up, down):
    """(exact value, allowed distance) of experts_forward"""
    v = torch.zeros(x.shape[0], gate.shape[2], dtype=torch.float64, device=x.device)
    err = torch.zeros_like(v)
    inter, top_k = gate.shape[1], ids.shape[1]
    for e in sorted(set(ids.flatten().tolist())):
        if e < 0:
            continue
        hit = ids == e
        rows = torch.nonzero(hit.any(1)).flatten()
        s = (weights.double() * hit).sum(1)[rows].unsqueeze(1)
        g, eg = dr._product(x[rows], gate[e])
        u, eu = dr._product(x[rows], up[e])
        a = g * torch.sigmoid(g)
        # silu's fp32 roundings are relative to it: exp of g magnifies half a unit by |g|
        ea = dr.SLOPE * eg + (8 + g.abs()) * 2.0 ** -23 * a.abs()
        h = s * a * u
        eh = s.abs() * (a.abs() * eu + u.abs() * ea + ea * eu) + 4 * 2.0 ** -23 * h.abs()
        eh = eh + 2.0 ** -22 * (h.abs() + eh) + 2.0 ** -39 * (h.abs() + eh).amax(1, keepdim=True)
        dd = down[e].double()
        v[rows] += h @ dd.t()
        err[rows] += eh @ dd.abs().t() + (2 * top_k * inter / 8 + 64) * 2.0 ** -23 * (h.abs() @ dd.abs().t())
    return v, dr._rounded(v, err, FP16)


# (tokens, experts, top_k, hidden, inter): every number of column tiles, many experts in a block's rows, several passes
SHAPES = [(1, 8, 2, 128, 256), (3, 40, 8, 64, 16), (6, 8, 2, 128, 208), (12, 5, 2, 256, 144), (16, 60, 16, 64, 16), (16, 256, 16, 64, 16),
          (2, 3, 3, 48, 16400), (16, 8, 2, 64, 16384)]


# products of gate and up around 1e6 times a unit (h beyond 65504, the outputs not), around 1e-6, and one token of each
@pytest.mark.parametrize("level", ["large", "small", "mixed"])
@pytest.mark.parametrize("shape", SHAPES)
def test_h_outside_the_type(shape, level, cuda_device):
    from nano_ktrans_b200 import DenseMoeLayer

    t, e, k, hid, inter = shape
    gate, up = (rnd(cuda_device, n, e, inter, hid, scale=hid ** -0.5) for n in (1, 2))
    d_scale = {"large": 2.0 ** -9, "small": 64.0, "mixed": 1.0}[level] * inter ** -0.5
    down = rnd(cuda_device, 3, e, hid, inter, scale=d_scale)
    x = rnd(cuda_device, 4, t, hid)
    if level == "large":
        x *= 900.0
    elif level == "small":
        x *= 2.0 ** -9
    else:
        x *= torch.tensor([900.0, 2.0 ** -9], device=cuda_device)[torch.arange(t, device=cuda_device) % 2].unsqueeze(1).to(FP16)
    layer = DenseMoeLayer(gate, up, down, top_k=k)
    g = torch.Generator(device=cuda_device).manual_seed(5)
    ids = torch.rand(t, e, generator=g, device=cuda_device).argsort(1)[:, :k].contiguous()
    w = (torch.rand(t, k, generator=g, device=cuda_device) + 0.01).to(FP16)
    if level == "small":
        w *= 0.05  # a small routing weight takes nothing from h's bits either
    want = scaled64(x, ids, w, gate, up, down)
    out = layer.experts_forward(x, ids, w)
    if level != "mixed":
        assert bool(out.isfinite().all()), "the formula's result is finite"
        dr.assert_within(out, want, level)
    else:  # the large tokens' results are beyond fp16 themselves where they are; the others are untouched by them
        fits = want[0].abs() < 60000
        dr.assert_within(out[fits], (want[0][fits], want[1][fits]), level)
        over = want[0].abs() > 70000
        assert bool(out[over].isinf().all())
    assert layer.read_status() == 0


@pytest.mark.parametrize("tokens", [1, 7, 16])
def test_shared_expert_and_router_at_large_h(tokens, cuda_device):
    """The shared expert's piece has its own scale; from hidden states, against the routed part and the shared part
    computed as layers of their own."""
    from nano_ktrans_b200 import DenseMoeLayer

    e, hid, inter, s = 6, 128, 96, 48
    gate, up = (rnd(cuda_device, n, e, inter, hid, scale=hid ** -0.5) for n in (1, 2))
    down = rnd(cuda_device, 3, e, hid, inter, scale=2.0 ** -9 * inter ** -0.5)
    sg, su = (rnd(cuda_device, n, s, hid, scale=hid ** -0.5) for n in (4, 5))
    sd = rnd(cuda_device, 6, hid, s, scale=2.0 ** -9 * s ** -0.5)
    x, wr = rnd(cuda_device, 7, tokens, hid, scale=900.0), rnd(cuda_device, 8, e, hid, scale=2.0 ** -10)
    shared = dict(gate=sg, up=su, down=sd, gate_vec=torch.zeros(hid, dtype=FP16, device=cuda_device))
    layer = DenseMoeLayer(gate, up, down, top_k=2, shared=shared)
    ids = torch.empty(tokens, 2, dtype=torch.int64, device=cuda_device)
    w = torch.empty(tokens, 2, dtype=FP16, device=cuda_device)
    out = layer.forward_x(x, wr, out_ids=ids, out_weights=w)
    v, b = scaled64(x, ids, w, gate, up, down)
    # its gate is sigmoid(0) = 1/2 for every token
    zero, half = torch.zeros(tokens, 1, dtype=torch.int64, device=cuda_device), torch.full((tokens, 1), 0.5, dtype=FP16, device=cuda_device)
    vs, bs = scaled64(x, zero, half, sg[None], su[None], sd[None])
    # both bounds hold a rounding to the type of their own part; the sum's is at most theirs and the sum's own
    dr.assert_within(out, (v + vs, b + bs + torch.finfo(FP16).eps / 2 * (v + vs).abs()), "with the shared expert")
    assert layer.read_status() == 0
