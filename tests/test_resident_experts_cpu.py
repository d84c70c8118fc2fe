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


def biased(m):
    m.w2.bias = torch.nn.Parameter(torch.ones(H, dtype=torch.bfloat16))


def own_forward(m):
    inner = m.forward
    m.forward = lambda x: 0.5 * inner(x)


def linear_forward(m):
    inner = m.w3.forward
    m.w3.forward = lambda x: inner(x) + 1


class Another(Expert):
    def __init__(self, function):
        super().__init__(80)
        self.function = function

    def forward(self, x):
        return self.function(self, x)


F = torch.nn.functional
OTHERS = dict(
    gelu=lambda m, x: m.w2(F.gelu(m.w1(x)) * m.w3(x)),
    quick_gelu=lambda m, x: m.w2(m.w1(x) * torch.sigmoid(1.702 * m.w1(x)) * m.w3(x)),
    hardswish=lambda m, x: m.w2(F.hardswish(m.w1(x)) * m.w3(x)),
    mish=lambda m, x: m.w2(F.mish(m.w1(x)) * m.w3(x)),
    relu=lambda m, x: m.w2(F.relu(m.w1(x)) * m.w3(x)),
    limited=lambda m, x: m.w2(F.silu(m.w1(x).clamp(max=7)) * m.w3(x)),
    limited_up=lambda m, x: m.w2(F.silu(m.w1(x)) * m.w3(x).clamp(-7, 7)),
    plus_one=lambda m, x: m.w2(F.silu(m.w1(x)) * (m.w3(x) + 1)),
    exchanged=lambda m, x: m.w2(m.w1(x) * F.silu(m.w3(x))),
    not_gated=lambda m, x: m.w2(F.silu(m.w1(x))),
    scaled=lambda m, x: 2.5 * m.w2(F.silu(m.w1(x)) * m.w3(x)),
    skip=lambda m, x: x + m.w2(F.silu(m.w1(x)) * m.w3(x)),
)
SAME = dict(
    sigmoid=lambda m, x: m.w2(m.w1(x) * torch.sigmoid(m.w1(x)) * m.w3(x)),
    wide=lambda m, x: m.w2((F.silu(m.w1(x).float()) * m.w3(x).float()).to(x.dtype)),
    module=lambda m, x: m.w2(torch.nn.SiLU()(m.w1(x)) * m.w3(x)),
)


@pytest.mark.parametrize("name", sorted(OTHERS))
def test_other_functions_are_refused(name):
    mods = torch.nn.ModuleDict({"1": Expert(1), "4": Another(OTHERS[name])})
    with pytest.raises(ValueError, match="silu"):
        ResidentExperts(mods, mask_of((1, 4)), 2, torch.device("cpu"), make_layer=Stacks)


@pytest.mark.parametrize("name", sorted(SAME))
def test_the_same_function_written_otherwise(name):
    mods = torch.nn.ModuleDict({"1": Expert(1), "4": Another(SAME[name])})
    before = [p.detach().clone() for p in mods.parameters()]
    holds(ResidentExperts(mods, mask_of((1, 4)), 2, torch.device("cpu"), make_layer=Stacks), mods, (1, 4))
    assert all(torch.equal(p, q) for p, q in zip(mods.parameters(), before))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_types_that_the_routing_weights_do_not_have(dtype):
    mods = torch.nn.ModuleDict({"1": Expert(1, dtype)})
    with pytest.raises(ValueError, match="bfloat16"):
        ResidentExperts(mods, mask_of((1,)), 2, torch.device("cpu"), make_layer=Stacks)
    mods, res = make()
    mods.half()
    assert res.current(mods, mask_of((1, 4, 7))) is None
    mods.bfloat16()
    holds(res, mods)


@pytest.mark.parametrize("change", [own_forward, linear_forward, biased])
def test_a_function_that_changes(change):
    mods, res = make()
    holds(res, mods)
    change(mods["4"])
    for _ in range(2):
        assert res.current(mods, mask_of((1, 4, 7))) is None
    mods["4"].w2.bias = None
    for m in (mods["4"], mods["4"].w3):
        m.__dict__.pop("forward", None)
    holds(res, mods)


@pytest.mark.parametrize("before", [True, False])
@pytest.mark.parametrize("where", ["expert", "w1", "pre"])
def test_hooks(where, before):
    """While there are any the modules are called themselves; nothing else runs them."""
    mods = torch.nn.ModuleDict({str(n): Expert(n) for n in (1, 4, 7)})
    seen = []

    def hook():
        if where == "pre":
            return mods["4"].register_forward_pre_hook(lambda m, a: seen.append(1))
        return (mods["4"] if where == "expert" else mods["4"].w1).register_forward_hook(lambda m, a, y: seen.append(1))

    h = hook() if before else None
    res = ResidentExperts(mods, mask_of((1, 4, 7)), 2, torch.device("cpu"), make_layer=Stacks)
    h = h or hook()
    assert res.current(mods, mask_of((1, 4, 7))) is None and res.some
    assert res.current(mods, mask_of(())) is None and not res.some  # the mask is followed all the same
    h.remove()
    holds(res, mods)
    assert not seen


@pytest.mark.parametrize("at", ["built", "stacked anew"])
def test_stacking_in_inference_mode(at):
    """It leaves the parameters what they were: usable by autograd afterwards."""
    mods = torch.nn.ModuleDict({str(n): Expert(n) for n in (1, 4, 7)})
    if at == "built":
        with torch.inference_mode():
            res = ResidentExperts(mods, mask_of((1, 4, 7)), 2, torch.device("cpu"), make_layer=Stacks)
    else:
        res = ResidentExperts(mods, mask_of((1, 4, 7)), 2, torch.device("cpu"), make_layer=Stacks)
        with torch.inference_mode():
            data(mods)
            res.current(mods, mask_of((1, 4, 7)))
    holds(res, mods)
    assert not any(p.is_inference() for p in mods["1"].parameters())
    mods["1"](torch.ones(2, H, dtype=torch.bfloat16)).sum().backward()
    assert mods["1"].w1.weight.grad is not None
    holds(res, mods)


def test_stacking_under_autocast():
    mods = torch.nn.ModuleDict({str(n): Expert(n) for n in (1, 4, 7)})
    with torch.autocast("cpu", dtype=torch.float16):
        res = ResidentExperts(mods, mask_of((1, 4, 7)), 2, torch.device("cpu"), make_layer=Stacks)
    holds(res, mods)


def test_a_module_that_takes_no_such_call():
    def fails(m, x):
        raise RuntimeError("not like this")

    mods = torch.nn.ModuleDict({"1": Expert(1), "4": Another(fails)})
    with pytest.raises(ValueError, match="silu"):
        ResidentExperts(mods, mask_of((1, 4)), 2, torch.device("cpu"), make_layer=Stacks)
    mods, res = make()
    mods["4"] = Another(fails)
    assert res.current(mods, mask_of((1, 4, 7))) is None
