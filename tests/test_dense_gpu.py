"""linear / gated_linear / DenseMLP against 64-bit forms (tests/dense_ref.py holds the bounds)."""
import pytest
import torch

from tests import dense_ref as dr

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def rnd(dev, seed, *shape, dtype=BF16, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


# (m, n, k): one token, the borders of 8- and 16-token tiles, tile borders, ragged sizes, long prompts
SHAPES = [(1, 2048, 2048), (1, 1, 1), (1, 5, 64), (2, 64, 8), (3, 7, 24), (7, 130, 1000), (8, 2048, 1408), (9, 257, 512),
          (15, 301, 4096), (16, 1024, 2048), (17, 1001, 1000), (31, 64, 14336), (33, 2050, 264), (64, 128, 64),
          (65, 129, 72), (100, 1408, 2048), (128, 2048, 1408), (129, 255, 136), (200, 2048, 1408), (256, 256, 256),
          (257, 513, 520), (333, 1001, 1000), (640, 768, 2048), (1025, 2100, 1032), (2048, 4096, 1024), (3001, 2777, 152),
          # rows that no wide load can take
          (1, 100, 77), (5, 33, 7), (40, 70, 129), (200, 130, 1001)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", SHAPES)
def test_linear_sizes(shape, dtype, cuda_device):
    from nano_ktrans_b200 import linear

    m, n, k = shape
    x, w = rnd(cuda_device, 1, m, k, dtype=dtype), rnd(cuda_device, 2, n, k, dtype=dtype, scale=k ** -0.5)
    b, r = rnd(cuda_device, 3, n, dtype=dtype), rnd(cuda_device, 4, m, n, dtype=dtype)
    dr.assert_within(linear(x, w), dr.linear64(x, w), f"{shape} plain")
    dr.assert_within(linear(x, w, b, residual=r), dr.linear64(x, w, b, None, r), f"{shape} bias residual")


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", SHAPES)
def test_gated_sizes(shape, dtype, cuda_device):
    from nano_ktrans_b200 import gated_linear

    m, n, k = shape
    x = rnd(cuda_device, 5, m, k, dtype=dtype)
    wg, wu = rnd(cuda_device, 6, n, k, dtype=dtype, scale=k ** -0.5), rnd(cuda_device, 7, n, k, dtype=dtype, scale=k ** -0.5)
    dr.assert_within(gated_linear(x, wg, wu), dr.gated64(x, wg, wu), f"{shape}")


@pytest.mark.parametrize("activation", [None, "silu", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("m", [1, 13, 150, 700])
def test_activations(m, activation, cuda_device):
    from nano_ktrans_b200 import gated_linear, linear

    for dtype in (BF16, FP16):
        x, w = rnd(cuda_device, 8, m, 256, dtype=dtype), rnd(cuda_device, 9, 330, 256, dtype=dtype, scale=0.2)
        b, r = rnd(cuda_device, 10, 330, dtype=dtype, scale=3.0), rnd(cuda_device, 11, m, 330, dtype=dtype)
        dr.assert_within(linear(x, w, b, activation=activation, residual=r), dr.linear64(x, w, b, activation, r))
        w2 = rnd(cuda_device, 12, 330, 256, dtype=dtype, scale=0.1)
        dr.assert_within(gated_linear(x, w, w2, activation=activation), dr.gated64(x, w, w2, activation))


@pytest.mark.parametrize("off,pad", [(0, 8), (0, 16), (8, 8), (4, 12), (1, 3)])
@pytest.mark.parametrize("m", [1, 6, 16, 70, 300])
def test_strided_rows_and_what_lies_around_them(m, off, pad, cuda_device):
    """Rows of wider buffers, at offsets down to two bytes; NaN around the inputs reaches nothing, and what
    lies around the output stays as it was."""
    from nano_ktrans_b200 import gated_linear, linear

    n, k = 136, 256

    def inside(seed, rows, cols, scale=1.0):
        buf = torch.full((rows + 2, cols + off + pad), float("nan"), dtype=BF16, device=cuda_device)
        buf[1:1 + rows, off:off + cols] = rnd(cuda_device, seed, rows, cols, scale=scale)
        return buf[1:1 + rows, off:off + cols]

    x, w, w2, r = inside(1, m, k), inside(2, n, k, 0.1), inside(3, n, k, 0.1), inside(4, m, n)
    for fn, ref in ((lambda o: linear(x, w, residual=r, out=o), dr.linear64(x, w, None, None, r)),
                    (lambda o: gated_linear(x, w, w2, out=o), dr.gated64(x, w, w2))):
        buf = torch.full((m + 2, n + off + pad), 7.0, dtype=BF16, device=cuda_device)
        out = buf[1:1 + m, off:off + n]
        assert fn(out) is out
        dr.assert_within(out, ref, f"m {m} off {off} pad {pad}")
        out.fill_(7.0)
        assert bool((buf == 7.0).all()), "wrote outside its rows"


@pytest.mark.parametrize("m", [1, 12, 90, 400])
def test_infinities_and_nan_stay_in_their_row_and_column(m, cuda_device):
    from nano_ktrans_b200 import gated_linear, linear

    n, k = 200, 520
    x, w, w2 = rnd(cuda_device, 1, m, k), rnd(cuda_device, 2, n, k, scale=0.1), rnd(cuda_device, 3, n, k, scale=0.1)
    clean, cleang = linear(x, w), gated_linear(x, w, w2)
    x[m - 1, 77] = float("inf")
    w[n - 3, 5] = float("nan")
    w2[11, 519] = float("nan")
    out, outg = linear(x, w), gated_linear(x, w, w2)
    keep = torch.ones(m, n, dtype=torch.bool, device=cuda_device)
    keep[m - 1] = False
    keep[:, n - 3] = False
    assert torch.equal(out[keep], clean[keep]) and bool(out[:, n - 3].isnan().all())
    assert not bool(out[m - 1].isfinite().any())
    keep[:, 11] = False
    assert torch.equal(outg[keep], cleang[keep]) and bool(outg[:, 11].isnan().all())


@pytest.mark.parametrize("m", [1, 16, 130, 600])
def test_residual_in_place_and_repeats_are_bit_equal(m, cuda_device):
    from nano_ktrans_b200 import linear

    x, w, r = rnd(cuda_device, 1, m, 1408), rnd(cuda_device, 2, 520, 1408, scale=0.05), rnd(cuda_device, 3, m, 520)
    want = linear(x, w, residual=r)
    for _ in range(3):
        assert torch.equal(linear(x, w, residual=r), want)
    assert linear(x, w, residual=r, out=r) is r
    assert torch.equal(r, want)


def test_no_tokens(cuda_device):
    from nano_ktrans_b200 import DenseMLP, gated_linear, linear

    x, w = rnd(cuda_device, 1, 0, 64), rnd(cuda_device, 2, 32, 64)
    assert linear(x, w).shape == (0, 32) and gated_linear(x, w, w).shape == (0, 32)
    assert DenseMLP(w, w, w.t().contiguous())(x).shape == (0, 64)


@pytest.mark.parametrize("m", [1, 5, 40, 300])
def test_two_streams_and_two_graphs(m, cuda_device):
    """Calls in flight on two streams at once, and two captured graphs replayed at once, give each its own result."""
    from nano_ktrans_b200 import DenseMLP

    xs = [rnd(cuda_device, i, m, 512) for i in range(2)]
    g, u, d = (rnd(cuda_device, 5 + i, *s, scale=0.05) for i, s in enumerate([(1408, 512), (1408, 512), (512, 1408)]))
    mlp = DenseMLP(g, u, d)
    want = [mlp(x, residual=x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[mlp(x, residual=x, stream=s) for _ in range(20)] for x, s in zip(xs, streams)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os_, w in zip(outs, want) for o in os_)
    graphs, res = [], []
    for x in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res.append(mlp(x, residual=x))
        graphs.append(gr)
    for x in xs:
        x.mul_(-0.5)
    want = [mlp(x, residual=x) for x in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for gr, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(res, want))


@pytest.mark.parametrize("m", [1, 9, 129])
def test_output_as_the_next_calls_weight(m, cuda_device):
    """A projection whose result is the next projection's weight: the next kernel reads it only once it is written."""
    from nano_ktrans_b200 import linear

    a, b = rnd(cuda_device, 1, 256, 64, scale=0.1), rnd(cuda_device, 2, 512, 64, scale=0.1)
    base, x = rnd(cuda_device, 3, 512, 256, scale=0.1), rnd(cuda_device, 4, m, 256)
    for _ in range(5):
        merged = linear(b, a, residual=base)  # [512, 256] = base + b a^T
        out = linear(x, merged)
        dr.assert_within(out, dr.linear64(x, merged))


@pytest.mark.parametrize("tokens", [1, 8, 150])
def test_dense_mlp(tokens, cuda_device):
    from nano_ktrans_b200 import DenseMLP

    g, u, d = (rnd(cuda_device, 5 + i, *s, scale=0.03) for i, s in enumerate([(1408, 2048), (1408, 2048), (2048, 1408)]))
    x = rnd(cuda_device, 1, tokens, 2048)
    out = DenseMLP(g, u, d)(x, residual=x)
    hv, hb = dr.gated64(x, g, u)
    v, b = dr.linear64(hv.to(BF16), d, None, None, x)
    # the product in between may sit hb away from its 64-bit value, and the plain form rounds it too
    slack = (hb + torch.finfo(BF16).eps / 2 * hv.abs()) @ d.double().abs().t()
    dr.assert_within(out, (v, b + slack * (1 + torch.finfo(BF16).eps)))


def test_refusals(cuda_device):
    from nano_ktrans_b200 import gated_linear, linear
    from nano_ktrans_b200._lib import MoeError

    x, w = rnd(cuda_device, 1, 4, 64), rnd(cuda_device, 2, 32, 64)
    with pytest.raises(ValueError, match="weight"):
        linear(x, w[:, :32])
    with pytest.raises(ValueError, match="weight"):
        linear(x, w.to(FP16))
    with pytest.raises(ValueError, match="bf16 or fp16"):
        linear(x.float(), w.float())
    with pytest.raises(ValueError, match="unit stride"):
        linear(rnd(cuda_device, 1, 64, 4).t(), w)
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="bias"):
        linear(x, w, rnd(cuda_device, 1, 31))
    with pytest.raises(ValueError, match="residual"):
        linear(x, w, residual=rnd(cuda_device, 1, 4, 31))
    with pytest.raises(ValueError, match="out"):
        linear(x, w, out=torch.empty(4, 32, device=cuda_device))
    with pytest.raises(ValueError, match="up_weight"):
        gated_linear(x, w, w[:16])
    with pytest.raises(MoeError, match="apart"):
        linear(x[:1].expand(4, 64), w)
    with pytest.raises(MoeError, match="overlaps"):
        linear(x, rnd(cuda_device, 1, 64, 64), out=x)
    buf = rnd(cuda_device, 3, 8, 32)
    with pytest.raises(MoeError, match="overlaps"):
        linear(x, w, residual=buf[:4], out=buf[1:5])
