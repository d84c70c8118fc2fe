"""Inputs and outputs of the dense operators as column ranges of one buffer: a fused projection's parts."""
import pytest
import torch

from tests import dense_plans as dp
from tests import dense_ref as dr

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def rnd(dev, seed, *shape, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(BF16)


@pytest.mark.parametrize("m,n,k,kernel", [(1, 136, 256, "stream"), (9, 136, 256, "stream"), (100, 136, 256, "split"),
                                          (70, 133, 250, "generic"), (2500, 4104, 512, "pair")])
def test_x_residual_and_output_side_by_side(m, n, k, kernel, cuda_device):
    from nano_ktrans_b200 import gated_linear, linear

    assert dp.kernel(m, n, k, ldx=k + 3 * n, ldo=k + 3 * n) == kernel
    buf = rnd(cuda_device, 1, m, k + 3 * n)
    before = buf.clone()
    x, r = buf[:, :k], buf[:, k:k + n]
    w, wu = rnd(cuda_device, 2, n, k, scale=0.1), rnd(cuda_device, 3, n, k, scale=0.1)
    out, gated = buf[:, k + n:k + 2 * n], buf[:, k + 2 * n:]
    linear(x, w, residual=r, out=out)
    gated_linear(x, w, wu, out=gated)
    dr.assert_within(out, dr.linear64(before[:, :k], w, None, None, before[:, k:k + n]))
    dr.assert_within(gated, dr.gated64(before[:, :k], w, wu))
    assert torch.equal(buf[:, :k + n], before[:, :k + n])


@pytest.mark.parametrize("tokens", [2, 16])
def test_expert_layer_writes_beside_its_input(tokens, cuda_device):
    from nano_ktrans_b200 import DenseMoeLayer

    e, h, i = 6, 128, 64
    layer = DenseMoeLayer(rnd(cuda_device, 1, e, i, h, scale=0.1), rnd(cuda_device, 2, e, i, h, scale=0.1),
                          rnd(cuda_device, 3, e, h, i, scale=0.1), top_k=2)
    wr = rnd(cuda_device, 4, e, h, scale=0.1)
    buf = rnd(cuda_device, 5, tokens, 3 * h)
    want = layer.forward_x(buf[:, :h].contiguous(), wr, residual=buf[:, h:2 * h].contiguous())
    before = buf.clone()
    layer.forward_x(buf[:, :h], wr, residual=buf[:, h:2 * h], out=buf[:, 2 * h:])
    assert torch.equal(buf[:, 2 * h:], want) and torch.equal(buf[:, :2 * h], before[:, :2 * h])
