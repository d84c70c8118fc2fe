"""A DenseMoeLayer on parameters that are given other memory between its calls: it reads where they are now, never the
memory that they left."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E, K, H, I, S = 6, 2, 128, 64, 32


class Bank(torch.nn.Module):
    def __init__(self, seed, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        for name, shape in (("gate", (E, I, H)), ("up", (E, I, H)), ("down", (E, H, I)), ("s_gate", (S, H)), ("s_up", (S, H)),
                            ("s_down", (H, S)), ("s_vec", (H,))):
            setattr(self, name, torch.nn.Parameter((torch.randn(*shape, generator=g) * 0.1).to(dtype).to(device)))

    def layer(self):
        from nano_ktrans_b200 import DenseMoeLayer

        return DenseMoeLayer(self.gate, self.up, self.down, top_k=K,
                             shared=dict(gate=self.s_gate, up=self.s_up, down=self.s_down, gate_vec=self.s_vec))


def inputs(tokens, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(3)
    return (torch.randn(tokens, H, generator=g, device="cuda").to(dtype),
            (torch.randn(E, H, generator=g, device="cuda") * 0.1).to(dtype))


@pytest.mark.parametrize("name", ["gate", "up", "down", "s_gate", "s_up", "s_down", "s_vec"])
@pytest.mark.parametrize("tokens", [1, 9])
def test_one_weight_given_other_memory(name, tokens, cuda_device):
    bank, other = Bank(1), Bank(2)
    layer = bank.layer()
    x, wr = inputs(tokens)
    before = layer.forward_x(x, wr)
    getattr(bank, name).data = getattr(other, name).data.clone()
    torch.cuda.empty_cache()
    out = layer.forward_x(x, wr)
    assert torch.equal(out, bank.layer().forward_x(x, wr)) and not torch.equal(out, before)


def test_a_module_that_is_moved_and_cast(cuda_device):
    bank = Bank(1)
    layer = bank.layer()
    x, wr = inputs(4)
    before = layer.forward_x(x, wr)
    bank.cpu()
    with pytest.raises(ValueError, match="CUDA"):
        layer.forward_x(x, wr)
    torch.cuda.empty_cache()
    bank.to(cuda_device)
    assert torch.equal(layer.forward_x(x, wr), before)
    bank.half()
    with pytest.raises(ValueError, match="x must be"):
        layer.forward_x(x, wr)
    xh, wh = inputs(4, torch.float16)
    assert torch.equal(layer.forward_x(xh, wh), bank.layer().forward_x(xh, wh))
    bank.up.data = bank.up.data[:, :, :64].contiguous()
    with pytest.raises(ValueError, match="gate and up"):
        layer.forward_x(xh, wh)


def test_a_weight_whose_memory_is_gone(cuda_device):
    """Storage given back, as sharding wrappers do between steps: refused before anything is launched."""
    from nano_ktrans_b200._lib import MoeError

    bank = Bank(1)
    layer = bank.layer()
    x, wr = inputs(2)
    want = layer.forward_x(x, wr)
    keep, storage = bank.gate.data.clone(), bank.gate.untyped_storage()
    size = storage.size()
    storage.resize_(0)
    with pytest.raises(MoeError, match="null"):
        layer.forward_x(x, wr)
    storage.resize_(size)
    bank.gate.data.copy_(keep)
    assert torch.equal(layer.forward_x(x, wr), want)


def test_two_threads_while_a_weight_moves(cuda_device):
    """What a call compares is set after what it then uses, so that a call of another thread meets a whole description."""
    from nano_ktrans_b200 import DenseMoeLayer

    order = []

    class Seen(DenseMoeLayer):
        def __setattr__(self, name, value):
            order.append(name)
            super().__setattr__(name, value)

    bank = Bank(1)
    layer = Seen(bank.gate, bank.up, bank.down, top_k=K)
    x, wr = inputs(2)
    bank.up.data = bank.up.data.clone()
    order.clear()
    out = layer.forward_x(x, wr)
    assert order[-1] == "_at" and {"_space", "_layer_bytes", "dtype"} <= set(order)
    assert torch.equal(out, DenseMoeLayer(bank.gate, bank.up, bank.down, top_k=K).forward_x(x, wr))
