"""HybridMoE(resident_experts="dense") when its modules change after it was built: small batches (the stacked weights) and
larger ones (the modules themselves) have to go by the same experts."""
import pytest
import torch

from tests import dense_ref as dr
from tests import helpers as hp

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
E, K, H, I = 12, 4, 256, 128
ON = [1, 4, 7]


class Expert(torch.nn.Module):
    def __init__(self, seed, device, dtype=BF16, act=torch.nn.functional.silu):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        self.act = act
        for name, (o, i) in (("w1", (I, H)), ("w3", (I, H)), ("w2", (H, I))):
            lin = torch.nn.Linear(i, o, bias=False, dtype=dtype)
            lin.weight.data.copy_(torch.randn(o, i, generator=g) * 0.08)
            setattr(self, name, lin.to(device))

    def forward(self, x):
        return self.w2(self.act(self.w1(x)) * self.w3(x))


@pytest.fixture(scope="module")
def codes():
    dev = torch.device("cuda:0")
    return hp.device_layer({n: hp.make_expert(5, n, H, I, 4, 128) for n in range(E)}, E, H, I, 4, 128, dev)


def build(codes, mods, on=ON, resident="dense", mask_device="cpu", **kw):
    from nano_ktrans_b200.hybrid_moe import HybridMoE

    mask = torch.zeros(E, dtype=torch.bool, device=mask_device)
    mask[on] = True
    return HybridMoE(num_experts=E, top_k=K, hidden_size=H, moe_intermediate_size=I, gpu_experts=mods, gpu_experts_mask=mask,
                     layer_idx=0, weight_path="", router_use_softmax=True, normalize_topk_prob=True, resident_experts=resident,
                     offload_backend_kwargs={"device": torch.device("cuda:0"), "max_tokens": 64, "layer_weights": codes}, **kw)


def modules(device, on=ON, **kw):
    return torch.nn.ModuleDict({str(n): Expert(100 + n, device, **kw) for n in on})


def inputs(t, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(t, H, generator=g, device="cuda").to(BF16), torch.randn(t, E, generator=g, device="cuda").to(BF16))


def check(moe, t, on=ON):
    """On the modules' present weights and the present mask: small batches against the 64-bit form over the backend's own
    part, larger ones against the module loop."""
    x, lg = inputs(t)
    out = moe(x, lg)
    if t > 16:
        assert torch.equal(out, build(codes_of(moe), moe.gpu_experts, on, "modules")(x, lg))
        return
    ids, w = moe.last_topk_ids, moe.last_topk_weights
    keep = torch.ones(E, dtype=torch.bool, device="cuda")
    keep[on] = False
    offloaded = moe.offload_backend.layer.experts_forward(x, ids, w, offload_mask=keep)
    slot = torch.full((E,), -1, device="cuda")
    slot[on] = torch.arange(len(on), device="cuda")
    gate, up, down = (torch.stack([getattr(moe.gpu_experts[str(n)], a).weight.detach() for n in on]) for a in ("w1", "w3", "w2"))
    dr.assert_within(out, dr.moe64(x, slot[ids], w, gate, up, down, None, offloaded), f"{t} tokens")


def codes_of(moe):
    return moe.offload_backend.layer.weights


TOKENS = [1, 8, 16, 40]


def refill(moe, seed):
    """New weights for every module, in place."""
    with torch.no_grad():
        for n, m in moe.gpu_experts.items():
            g = torch.Generator().manual_seed(seed + int(n))
            for a in ("w1", "w3", "w2"):
                p = getattr(m, a).weight
                p.copy_(torch.randn(p.shape, generator=g) * 0.08)


@pytest.mark.parametrize("t", TOKENS)
def test_modules_built_on_the_host_and_moved(t, codes, cuda_device):
    moe = build(codes, modules("cpu"))
    moe.to(cuda_device)
    check(moe, t)
    state = {k: torch.randn(v.shape, generator=torch.Generator().manual_seed(7)).to(v.dtype) * 0.08 for k, v in moe.state_dict().items()}
    moe.load_state_dict(state)
    check(moe, t)
    refill(moe, 300)
    check(moe, t)


@pytest.mark.parametrize("t", TOKENS)
@pytest.mark.parametrize("how", ["in place", "data", "parameter", "assign", "linear", "expert", "to and back"])
def test_weights_that_are_replaced(how, t, codes, cuda_device):
    moe = build(codes, modules(cuda_device))
    check(moe, t)
    fresh = {str(n): Expert(500 + n, cuda_device) for n in ON}
    if how == "in place":
        refill(moe, 400)
    elif how == "data":
        moe.gpu_experts["4"].w3.weight.data = fresh["4"].w3.weight.data
    elif how == "parameter":
        moe.gpu_experts["1"].w2.weight = fresh["1"].w2.weight
    elif how == "assign":
        moe.load_state_dict({f"gpu_experts.{n}.{k}": v for n in fresh for k, v in fresh[n].state_dict().items()}, assign=True)
    elif how == "linear":
        moe.gpu_experts["7"].w1 = fresh["7"].w1
    elif how == "expert":
        moe.gpu_experts["4"] = fresh["4"]
    else:
        moe.cpu()
        refill(moe, 600)
        moe.to(cuda_device)
    check(moe, t)
    refill(moe, 700)
    check(moe, t)


@pytest.mark.parametrize("t", TOKENS)
@pytest.mark.parametrize("mask_device", ["cpu", "cuda"])
def test_residency_that_changes(mask_device, t, codes, cuda_device):
    mods = modules(cuda_device, on=[1, 2, 4, 7])
    moe = build(codes, mods, mask_device=mask_device)
    check(moe, t)
    for on in ([1, 4], [1, 2, 4, 7], [2], [1, 4, 7]):
        mask = torch.zeros(E, dtype=torch.bool, device=mask_device)
        mask[on] = True
        moe.gpu_experts_mask = mask
        moe.offload_backend.update_gpu_expert_mask(mask)
        check(moe, t, on)
    mask[[1, 4]] = False  # the same tensor, in place
    moe.offload_backend.update_gpu_expert_mask(mask)
    check(moe, t, [7])


def test_no_host_read_whatever_device_the_mask_is_on(codes, cuda_device):
    for mask_device in ("cpu", "cuda"):
        moe = build(codes, modules(cuda_device), mask_device=mask_device)
        x, lg = inputs(6)
        moe(x, lg)
        torch.cuda.synchronize()
        torch.cuda.set_sync_debug_mode("error")
        try:
            moe(x, lg)
        finally:
            torch.cuda.set_sync_debug_mode(0)


def test_experts_of_another_kind_are_refused(codes, cuda_device):
    with pytest.raises(ValueError, match="hidden_act"):
        build(codes, modules(cuda_device), hidden_act="gelu")
    with pytest.raises(ValueError, match="silu"):
        build(codes, modules(cuda_device, act=torch.nn.functional.gelu))
    with pytest.raises(ValueError, match="silu"):
        build(codes, modules(cuda_device, act=lambda v: torch.nn.functional.silu(v).clamp(max=7)))
    with pytest.raises(ValueError, match="bfloat16"):
        build(codes, modules(cuda_device, dtype=torch.float16))
    with pytest.raises(ValueError, match="bfloat16"):
        build(codes, modules(cuda_device, dtype=torch.float32))


@pytest.mark.parametrize("name", ["silu", "SiLU", "swish"])
def test_names_of_the_activation(name, codes, cuda_device):
    check(build(codes, modules(cuda_device), hidden_act=name), 3)


@pytest.mark.parametrize("where", ["expert", "linear"])
@pytest.mark.parametrize("when", ["before", "after"])
def test_hooks_are_run(when, where, codes, cuda_device):
    """A module with hooks is called, on small batches too."""
    mods = modules(cuda_device)
    seen = []
    target = mods["4"] if where == "expert" else mods["4"].w2
    if when == "before":
        handle = target.register_forward_hook(lambda m, a, y: seen.append(1) or y * 0)
    moe = build(codes, mods)
    if when == "after":
        handle = target.register_forward_hook(lambda m, a, y: seen.append(1) or y * 0)
    x, lg = inputs(8)
    lg[:, 4] = 9.0
    seen.clear()
    got = moe(x, lg)
    want = build(codes, mods, resident="modules")(x, lg)
    assert len(seen) == 2 and torch.equal(got, want)
    handle.remove()
    seen.clear()
    check(moe, 8)
    assert not seen


@pytest.mark.parametrize("t", [1, 8])
def test_a_module_whose_function_changes(t, codes, cuda_device):
    """Its own forward replaced, as adapters do: the module is called."""
    mods = modules(cuda_device)
    moe = build(codes, mods)
    check(moe, t)
    inner = mods["4"].forward
    mods["4"].forward = lambda x: 0.5 * inner(x)
    x, lg = inputs(t)
    lg[:, 4] = 9.0
    assert torch.equal(moe(x, lg), build(codes, mods, resident="modules")(x, lg))
    del mods["4"].forward
    check(moe, t)


def test_a_capture_finds_changed_weights(codes, cuda_device):
    """The stack cannot be made anew inside a capture: refused, and right after one call outside."""
    moe = build(codes, modules(cuda_device))
    x, lg = inputs(4)
    moe(x, lg)
    moe.gpu_experts["4"].w3.weight.data = Expert(900, cuda_device).w3.weight.data
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="outside"):
        with torch.cuda.graph(graph):
            moe(x, lg)
    check(moe, 4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = moe(x, lg)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, moe(x, lg))


def test_hidden_states_at_any_alignment(codes, cuda_device):
    moe = build(codes, modules(cuda_device))
    x, lg = inputs(5)
    want = moe(x, lg)
    for off, width in ((1, H + 3), (8, H + 20), (4, H + 8)):
        wide = torch.zeros(5, width, dtype=BF16, device=cuda_device)
        wide[:, off:off + H] = x
        assert torch.equal(moe(wide[:, off:off + H], lg), want)


@pytest.mark.parametrize("resident", ["dense", "modules", "kernels"])
def test_no_tokens(resident, codes, cuda_device):
    moe = build(codes, modules(cuda_device), resident=resident)
    x, lg = inputs(3)
    assert moe(x[:0], lg[:0]).shape == (0, H)


def test_in_inference_mode(codes, cuda_device):
    """Weights that change and are stacked anew there stay usable by autograd outside."""
    moe = build(codes, modules(cuda_device))
    with torch.inference_mode():
        check(moe, 5)
        moe.gpu_experts["4"].w3.weight.data = Expert(900, cuda_device).w3.weight.data
        check(moe, 5)
    check(moe, 5)
    moe.gpu_experts["4"](inputs(2)[0]).sum().backward()
    assert moe.gpu_experts["4"].w3.weight.grad is not None
    check(moe, 5)
