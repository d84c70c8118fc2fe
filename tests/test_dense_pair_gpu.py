"""The projection kernel of SM pairs, plain and gated, with everything its epilogue does: bias, each activation, residual
(aligned, not, in place), ragged and unaligned outputs.  Every test asserts that its sizes reach that kernel."""
import pytest
import torch

from tests import dense_plans as dp
from tests import dense_ref as dr

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def rnd(dev, seed, *shape, dtype=BF16, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


# ragged in tokens and features (a last tile of 137, 157, 185 and 8 columns), short and long K, K off a whole step
SHAPES = [(4000, 5000, 1024), (4000, 5001, 1024), (3765, 5789, 152), (2048, 4096, 4096), (3000, 3001, 4104), (2500, 4104, 512)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", SHAPES)
def test_sizes(shape, dtype, cuda_device):
    from nano_ktrans_b200 import gated_linear, linear

    m, n, k = shape
    assert dp.kernel(m, n, k) == dp.kernel(m, n, k, gated=True) == "pair"
    x, w = rnd(cuda_device, 1, m, k, dtype=dtype), rnd(cuda_device, 2, n, k, dtype=dtype, scale=k ** -0.5)
    b, r = rnd(cuda_device, 3, n, dtype=dtype), rnd(cuda_device, 4, m, n, dtype=dtype)
    dr.assert_within(linear(x, w), dr.linear64(x, w), f"{shape} plain")
    dr.assert_within(linear(x, w, b), dr.linear64(x, w, b), f"{shape} bias")
    dr.assert_within(linear(x, w, b, residual=r), dr.linear64(x, w, b, None, r), f"{shape} bias residual")
    wu = rnd(cuda_device, 5, n, k, dtype=dtype, scale=k ** -0.5)
    dr.assert_within(gated_linear(x, w, wu), dr.gated64(x, w, wu), f"{shape} gated")


@pytest.mark.parametrize("activation", [None, "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("n", [4104, 4101])
def test_activations(n, activation, cuda_device):
    from nano_ktrans_b200 import gated_linear, linear

    m, k = 2500, 512
    assert dp.kernel(m, n, k) == dp.kernel(m, n, k, gated=True) == "pair"
    for dtype in (BF16, FP16):
        x, w = rnd(cuda_device, 8, m, k, dtype=dtype), rnd(cuda_device, 9, n, k, dtype=dtype, scale=0.1)
        b, r = rnd(cuda_device, 10, n, dtype=dtype, scale=3.0), rnd(cuda_device, 11, m, n, dtype=dtype)
        dr.assert_within(linear(x, w, b, activation=activation, residual=r), dr.linear64(x, w, b, activation, r))
        dr.assert_within(linear(x, w, activation=activation), dr.linear64(x, w, None, activation))
        w2 = rnd(cuda_device, 12, n, k, dtype=dtype, scale=0.1)
        dr.assert_within(gated_linear(x, w, w2, activation=activation), dr.gated64(x, w, w2, activation))


@pytest.mark.parametrize("off,pad,bias_off", [(0, 8, 0), (8, 8, 1), (4, 12, 8), (1, 3, 0)])
def test_strided_rows_and_what_lies_around_them(off, pad, bias_off, cuda_device):
    """Outputs and residuals in wider buffers, at offsets down to two bytes; what lies around the output stays."""
    from nano_ktrans_b200 import gated_linear, linear

    m, n, k = 2503, 4104, 512

    def inside(seed, rows, cols, o, p, scale=1.0):
        buf = torch.full((rows + 2, cols + o + p), float("nan"), dtype=BF16, device=cuda_device)
        buf[1:1 + rows, o:o + cols] = rnd(cuda_device, seed, rows, cols, scale=scale)
        return buf[1:1 + rows, o:o + cols]

    x, w, w2 = inside(1, m, k, 8, 8), inside(2, n, k, 16, 8, 0.1), inside(3, n, k, 0, 8, 0.1)
    assert dp.kernel(m, n, k, ldx=x.stride(0), ldw=w.stride(0), ldo=n + off + pad) == "pair"
    assert dp.kernel(m, n, k, True, ldx=x.stride(0), ldw=w.stride(0), ldw_up=w2.stride(0), ldo=n + off + pad) == "pair"
    b = torch.full((n + 16,), float("nan"), dtype=BF16, device=cuda_device)[bias_off:bias_off + n].copy_(rnd(cuda_device, 5, n))
    # the residual lies as the output does, then otherwise
    for r in (inside(4, m, n, off, pad), inside(4, m, n, 8, 8), inside(4, m, n, 1, 2)):
        for fn, ref in ((lambda o: linear(x, w, b, residual=r, out=o), dr.linear64(x, w, b, None, r)),
                        (lambda o: gated_linear(x, w, w2, out=o), dr.gated64(x, w, w2))):
            buf = torch.full((m + 2, n + off + pad), 7.0, dtype=BF16, device=cuda_device)
            out = buf[1:1 + m, off:off + n]
            assert fn(out) is out
            dr.assert_within(out, ref, f"off {off} pad {pad}")
            out.fill_(7.0)
            assert bool((buf == 7.0).all()), "wrote outside its rows"


@pytest.mark.parametrize("n", [4104, 4101])
def test_infinities_and_nan_stay_in_their_row_and_column(n, cuda_device):
    from nano_ktrans_b200 import gated_linear, linear

    m, k = 2500, 520
    assert dp.kernel(m, n, k) == dp.kernel(m, n, k, gated=True) == "pair"
    x, w, w2 = rnd(cuda_device, 1, m, k), rnd(cuda_device, 2, n, k, scale=0.1), rnd(cuda_device, 3, n, k, scale=0.1)
    r = rnd(cuda_device, 4, m, n)
    clean, cleanr, cleang = linear(x, w), linear(x, w, residual=r), gated_linear(x, w, w2)
    x[m - 1, 77] = float("inf")
    x[300, 519] = float("nan")
    w[n - 3, 5] = float("nan")
    w2[11, 519] = float("nan")
    r[1000, 7] = float("nan")
    out, outr, outg = linear(x, w), linear(x, w, residual=r), gated_linear(x, w, w2)
    keep = torch.ones(m, n, dtype=torch.bool, device=cuda_device)
    keep[m - 1] = keep[300] = False
    keep[:, n - 3] = False
    assert torch.equal(out[keep], clean[keep]) and bool(out[:, n - 3].isnan().all()) and bool(out[300].isnan().all())
    assert not bool(out[m - 1].isfinite().any())
    keepr = keep.clone()
    keepr[1000, 7] = False
    assert torch.equal(outr[keepr], cleanr[keepr]) and bool(outr[1000, 7].isnan())
    keep[:, 11] = False
    assert torch.equal(outg[keep], cleang[keep]) and bool(outg[:, 11].isnan().all())


@pytest.mark.parametrize("n,off", [(4104, 0), (4104, 1), (4101, 0)])
def test_residual_in_place_and_repeats_are_bit_equal(n, off, cuda_device):
    from nano_ktrans_b200 import linear

    m, k = 2500, 1408
    assert dp.kernel(m, n, k) == "pair"
    x, w, b = rnd(cuda_device, 1, m, k), rnd(cuda_device, 2, n, k, scale=0.05), rnd(cuda_device, 3, n)
    wide = rnd(cuda_device, 4, m, n + 8)
    r = wide[:, off:off + n]
    want = linear(x, w, b, activation="silu", residual=r)
    for _ in range(3):
        assert torch.equal(linear(x, w, b, activation="silu", residual=r), want)
    around = torch.cat([wide[:, :off], wide[:, off + n:]], 1)
    assert linear(x, w, b, activation="silu", residual=r, out=r) is r
    assert torch.equal(r, want) and torch.equal(torch.cat([wide[:, :off], wide[:, off + n:]], 1), around)


def test_two_streams_and_a_graph(cuda_device):
    """Calls on the pair kernel and on the split kernel in flight at once, and replayed, give each its own result."""
    from nano_ktrans_b200 import linear

    shapes = [(2500, 4104, 512), (100, 1408, 2048), (700, 330, 256)]
    assert [dp.kernel(*s) for s in shapes] == ["pair", "split", "split"]
    xs = [rnd(cuda_device, i, m, k) for i, (m, n, k) in enumerate(shapes)]
    ws = [rnd(cuda_device, 10 + i, n, k, scale=0.05) for i, (m, n, k) in enumerate(shapes)]
    want = [linear(x, w) for x, w in zip(xs, ws)]
    streams = [torch.cuda.Stream() for _ in shapes]
    torch.cuda.synchronize()
    outs = [[linear(x, w, stream=s) for _ in range(20)] for x, w, s in zip(xs, ws, streams)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os_, w in zip(outs, want) for o in os_)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = [linear(x, w) for x, w in zip(xs, ws)]
    for x in xs:
        x.mul_(-0.5)
    want = [linear(x, w) for x, w in zip(xs, ws)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(res, want))
