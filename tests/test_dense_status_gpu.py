"""The status word of the dense operators."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def small_layer(dev):
    from nano_ktrans_b200 import DenseMoeLayer

    g, u, d = (torch.zeros(2, *s, dtype=BF16, device=dev) for s in ((16, 64), (16, 64), (64, 16)))
    x = torch.zeros(1, 64, dtype=BF16, device=dev)
    w = torch.ones(1, 1, dtype=BF16, device=dev)
    return DenseMoeLayer(g, u, d, top_k=1), x, w


def test_nothing_is_lost_to_a_read_at_the_same_time(cuda_device):
    """A bad id on another stream is reported by the read that runs meanwhile or by the one after it, never by neither."""
    layer, x, w = small_layer(cuda_device)
    bad = torch.full((1, 1), 5, device=cuda_device)
    side = torch.cuda.Stream()
    out = torch.empty(1, 64, dtype=BF16, device=cuda_device)
    layer.experts_forward(x, bad, w, out=out)
    torch.cuda.synchronize()
    layer.read_status()
    lost = 0
    for i in range(4000):
        with torch.cuda.stream(side):
            torch.cuda._sleep(100 * (i % 400))  # clocks, so that it comes at different moments of the read
        layer.experts_forward(x, bad, w, out=out, stream=side)
        seen = layer.read_status()
        side.synchronize()
        lost += (seen | layer.read_status()) != 1
    assert lost == 0, f"{lost} of 4000 reports lost"
    assert layer.read_status() == 0


def test_read_without_a_layer(cuda_device):
    from nano_ktrans_b200 import read_dense_status

    layer, x, w = small_layer(cuda_device)
    assert read_dense_status() == 0
    layer.experts_forward(x, torch.full((1, 1), 5, device=cuda_device), w)
    assert read_dense_status(cuda_device) == 1 and read_dense_status(torch.device("cuda")) == 0
    side = torch.cuda.Stream()
    layer.experts_forward(x, torch.full((1, 1), 5, device=cuda_device), w, stream=side)
    assert read_dense_status(cuda_device, stream=side) == 1 and layer.read_status() == 0
    with pytest.raises(ValueError, match="CUDA"):
        read_dense_status(torch.device("cpu"))
