"""ResidentExperts: when the stack is made anew.  On the host, with a stand-in for the layer that keeps the stacks."""
import pytest
import torch

from nano_ktrans_b200.dense_moe import ResidentExperts

H, I = 6, 4
NAMES = ("w1", "w3", "w2")


class Expert(torch.nn.Module):
    def __init__(self, seed, dtype=torch.bfloat16, device="cpu"):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        for n, (o, i) in zip(NAMES, ((I, H), (I, H), (H, I))):
            setattr(self, n, torch.nn.Linear(i, o, bias=False, dtype=dtype))
            getattr(self, n).weight.data.copy_(torch.randn(o, i, generator=g))
        self.to(device)

    def forward(self, x):
        return self.w2(torch.nn.functional.silu(self.w1(x)) * self.w3(x))


class Stacks:
    def __init__(self, gate, up, down, top_k):
        self.stacks = (gate, up, down)


def make(on=(1, 4, 7), device="cpu"):
    mods = torch.nn.ModuleDict({str(n): Expert(n, device=device) for n in on})
    return mods, ResidentExperts(mods, mask_of(on), 2, torch.device("cpu"), make_layer=Stacks)


def mask_of(on):
    mask = torch.zeros(9, dtype=torch.bool)
    mask[list(on)] = True
    return mask


def holds(res, mods, on=(1, 4, 7)):
    """The stack has the modules' weights, and is where they are."""
    layer = res.current(mods, mask_of(on))
    assert res.slot.tolist() == [on.index(n) if n in on else -1 for n in range(9)]
    for j, name in enumerate(NAMES):
        for n in on:
            w = getattr(mods[str(n)], name).weight
            assert torch.equal(layer.stacks[j][on.index(n)], w) and w.data_ptr() == layer.stacks[j][on.index(n)].data_ptr()
    return layer


def test_nothing_changes():
    mods, res = make()
    layer = holds(res, mods)
    with torch.no_grad():
        mods["4"].w3.weight.mul_(2)
    mods.load_state_dict({k: torch.ones_like(v) for k, v in mods.state_dict().items()})
    assert holds(res, mods) is layer


def expert(mods):
    mods["7"] = Expert(20)


def linear(mods):
    mods["4"].w1 = Expert(20).w1


def parameter(mods):
    mods["1"].w2.weight = torch.nn.Parameter(Expert(20).w2.weight.detach())


def data(mods):
    mods["4"].w3.weight.data = Expert(20).w3.weight.data


def assign(mods):
    mods.load_state_dict({k: v.clone() + 1 for k, v in mods.state_dict().items()}, assign=True)


def there_and_back(mods):
    mods.float()
    mods.bfloat16()


@pytest.mark.parametrize("change", [expert, linear, parameter, data, assign, there_and_back])
def test_what_makes_it_anew(change):
    mods, res = make()
    layer = holds(res, mods)
    change(mods)
    again = holds(res, mods)
    assert again is not layer and holds(res, mods) is again


def test_another_dict_of_modules():
    mods, res = make()
    other = torch.nn.ModuleDict({str(n): Expert(30 + n) for n in (1, 4, 7)})
    holds(res, other)
    del other["4"]
    assert res.current(other, mask_of((1, 4, 7))) is not None and res.slot.tolist() == [-1, 0, -1, -1, -1, -1, -1, 1, -1]
    other["4"] = Expert(50)
    holds(res, other)


def test_modules_on_another_device_are_called_themselves():
    mods, res = make(device="meta")
    assert res.current(mods, mask_of((1, 4, 7))) is None
    mods.to_empty(device="cpu")
    mods.load_state_dict({k: torch.randn(v.shape).to(v.dtype) for k, v in mods.state_dict().items()})
    holds(res, mods)
    mods["4"].to("meta")
    assert res.current(mods, mask_of((1, 4, 7))) is None and res.slot is None


def test_modules_that_become_something_else_are_called_themselves():
    mods, res = make()
    holds(res, mods)
    mods["4"].w1 = torch.nn.Linear(H, I, dtype=torch.bfloat16)  # with a bias
    assert res.current(mods, mask_of((1, 4, 7))) is None and res.current(mods, mask_of((1, 4, 7))) is None
    mods["4"].w1.bias = None
    holds(res, mods)
    mods["1"].w2.float()
    assert res.current(mods, mask_of((1, 4, 7))) is None
    mods["1"].w2.bfloat16()
    holds(res, mods)


def test_a_capture_makes_nothing_anew(monkeypatch):
    mods, res = make()
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    layer = res.current(mods, mask_of((1, 4, 7)))
    data(mods)
    with pytest.raises(RuntimeError, match="outside the capture"):
        res.current(mods, mask_of((1, 4, 7)))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert holds(res, mods) is not layer


def test_the_mask_changes():
    mods, res = make()
    layer = holds(res, mods)
    for on in ((1, 4), (7,), (1, 4, 7)):
        mask = mask_of(on)
        again = res.current(mods, mask)
        assert again is not layer and res.some and res.current(mods, mask.clone()) is again
        holds(res, mods, on)
        layer = again
    mask[4] = False  # in place
    assert res.current(mods, mask) is not layer
    holds(res, mods, (1, 7))
    assert res.current(mods, mask_of(())) is None and not res.some
    mods["2"] = Expert(60)
    holds(res, mods, (1, 2))


def test_a_resident_expert_without_a_module():
    """It has no place in the stack, until it gets a module."""
    mods, res = make()
    res.current(mods, mask_of((1, 3, 4)))
    assert res.slot.tolist() == [-1, 0, -1, -1, 1, -1, -1, -1, -1]
    mods["3"] = Expert(70)
    holds(res, mods, (1, 3, 4))


def test_masks_of_other_types_and_of_inference_mode():
    mods, res = make()
    layer = holds(res, mods)
    assert res.current(mods, mask_of((1, 4, 7)).to(torch.uint8)) is layer
    with torch.inference_mode():
        mask = mask_of((1, 4))
    res.current(mods, mask)
    holds(res, mods, (1, 4))
