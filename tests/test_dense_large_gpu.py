"""Sizes and offsets beyond 32 bits."""
import pytest
import torch

from tests import dense_ref as dr

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_more_rows_than_a_description_holds(cuda_device):
    """2^32 + 5 rows would arrive as 5: refused.  The memory is reserved, not read."""
    from nano_ktrans_b200 import linear

    x = torch.empty(2 ** 32 + 5, 1, dtype=BF16, device=cuda_device)
    w = torch.ones(1, 1, dtype=BF16, device=cuda_device)
    with pytest.raises(ValueError, match="at most"):
        linear(x, w)
    with pytest.raises(ValueError, match="at most"):
        linear(w, x)


@pytest.mark.parametrize("m", [3, 100, 700])
def test_elements_beyond_32_bits(m, cuda_device):
    """Rows so far apart that the last ones of x, weight, residual and output lie beyond 2^31 elements, 2^32 bytes."""
    from nano_ktrans_b200 import gated_linear, linear

    n, k = 264, 128
    g = torch.Generator(device=cuda_device).manual_seed(1)

    def apart(rows, cols):
        ld = (2 ** 31 + 2 ** 20) // (rows - 1) // 8 * 8 + 8
        t = torch.empty((rows - 1) * ld + cols, dtype=BF16, device=cuda_device).as_strided((rows, cols), (ld, 1))
        return t.copy_(torch.randn(rows, cols, generator=g, device=cuda_device) * 0.1)

    x, w, wu, r, out = apart(m, k), apart(n, k), apart(n, k), apart(m, n), apart(m, n)
    linear(x, w, residual=r, out=out)
    dr.assert_within(out.contiguous(), dr.linear64(x.contiguous(), w.contiguous(), None, None, r.contiguous()))
    gated_linear(x, w, wu, out=out)
    dr.assert_within(out.contiguous(), dr.gated64(x.contiguous(), w.contiguous(), wu.contiguous()))
    linear(x[:, 1:], w[:, 1:], out=out)  # rows off 16 bytes
    dr.assert_within(out.contiguous(), dr.linear64(x[:, 1:].contiguous(), w[:, 1:].contiguous()))


def test_expert_layer_beyond_32_bits(cuda_device):
    """Weights of more than 2^31 elements, and rows of x, residual and output that far apart."""
    from nano_ktrans_b200 import DenseMoeLayer

    e, h, i, t = 40, 8192, 8192, 3
    g = torch.Generator(device=cuda_device).manual_seed(1)
    last = [torch.randn(*s, generator=g, device=cuda_device).mul_(s[1] ** -0.5).to(BF16) for s in ((i, h), (i, h), (h, i))]
    weights = [torch.empty(e, *w.shape, dtype=BF16, device=cuda_device) for w in last]
    for w, l in zip(weights, last):
        w[e - 1], w[0] = l, l
    layer = DenseMoeLayer(*weights, top_k=2)
    ld = 2 ** 30 + 8

    def apart():
        return torch.empty(2 * ld + h, dtype=BF16, device=cuda_device).as_strided((t, h), (ld, 1))

    x, r, out = apart(), apart(), apart()
    x.copy_(torch.randn(t, h, generator=g, device=cuda_device))
    r.copy_(torch.randn(t, h, generator=g, device=cuda_device))
    ids = torch.tensor([[e - 1, 0], [0, -1], [-1, e - 1]], device=cuda_device)
    w = torch.rand(t, 2, generator=g, device=cuda_device).to(BF16)
    layer.experts_forward(x, ids, w, residual=r, out=out)
    small = torch.where(ids == e - 1, 1, ids)
    two = [torch.stack([l, l]) for l in last]
    dr.assert_within(out.contiguous(), dr.moe64(x.contiguous(), small, w, *two, None, r.contiguous()))
    assert layer.read_status() == 0
