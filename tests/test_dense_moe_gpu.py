"""DenseMoeLayer against its 64-bit form (tests/dense_ref.py holds the bounds)."""
import pytest
import torch

from tests import dense_ref as dr

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def rnd(dev, seed, *shape, dtype=BF16, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=dev) * scale).to(dtype)


def make(dev, e, top_k, h, i, s=0, dtype=BF16, softmax=True, renorm=True, seed=0):
    from nano_ktrans_b200 import DenseMoeLayer

    gate, up = (rnd(dev, seed + n, e, i, h, dtype=dtype, scale=h ** -0.5) for n in (1, 2))
    down = rnd(dev, seed + 3, e, h, i, dtype=dtype, scale=i ** -0.5)
    shared = None
    if s:
        shared = dict(gate=rnd(dev, seed + 4, s, h, dtype=dtype, scale=h ** -0.5), up=rnd(dev, seed + 5, s, h, dtype=dtype, scale=h ** -0.5),
                      down=rnd(dev, seed + 6, h, s, dtype=dtype, scale=s ** -0.5), gate_vec=rnd(dev, seed + 7, h, dtype=dtype, scale=h ** -0.5))
    layer = DenseMoeLayer(gate, up, down, top_k=top_k, router_use_softmax=softmax, normalize_topk_prob=renorm, shared=shared)
    return layer, shared


def check(layer, shared, out, x, ids, w, residual=None, what=""):
    dr.assert_within(out, dr.moe64(x, ids, w, layer.gate, layer.up, layer.down, shared, residual), what)
    assert layer.read_status() == 0


def run_x(layer, x, wr, **kw):
    dev, t = x.device, x.shape[0]
    ids = torch.empty(t, layer.top_k, dtype=torch.int64, device=dev)
    w = torch.empty(t, layer.top_k, dtype=x.dtype, device=dev)
    lg = torch.empty(t, layer.num_experts, dtype=x.dtype, device=dev)
    out = layer.forward_x(x, wr, out_ids=ids, out_weights=w, out_logits=lg, **kw)
    return out, ids, w, lg


# (tokens, experts, top_k, hidden, inter, shared)
SHAPES = [(1, 128, 8, 2048, 768, 0), (3, 128, 8, 2048, 768, 0), (16, 128, 8, 2048, 768, 0), (6, 60, 4, 2048, 1408, 5632),
          (5, 8, 2, 1024, 3584, 0), (1, 1, 1, 16, 16, 0), (16, 1, 1, 16, 16, 16), (4, 33, 16, 48, 80, 0), (5, 33, 5, 80, 48, 112),
          (16, 40, 16, 272, 144, 0), (8, 1024, 16, 256, 32, 0), (9, 7, 7, 528, 1040, 16), (12, 31, 3, 2064, 16, 0),
          (2, 64, 6, 16, 2064, 32),
          # more intermediate rows than the blocks hold at a time
          (16, 8, 2, 64, 16384, 1600)]


@pytest.mark.parametrize("dtype,softmax,renorm", [(BF16, True, True), (BF16, True, False), (FP16, False, True), (FP16, True, True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_layer_from_hidden_states(shape, dtype, softmax, renorm, cuda_device):
    t, e, k, h, i, s = shape
    layer, shared = make(cuda_device, e, k, h, i, s, dtype, softmax, renorm)
    x, r = rnd(cuda_device, 11, t, h, dtype=dtype), rnd(cuda_device, 12, t, h, dtype=dtype)
    wr = rnd(cuda_device, 13, e, h, dtype=dtype, scale=1.5 * h ** -0.5)
    out, ids, w, lg = run_x(layer, x, wr, residual=r)
    dr.assert_within(lg, dr.linear64(x, wr), "logits")
    dr.assert_routing(ids, w, lg, k, softmax, renorm)
    check(layer, shared, out, x, ids, w, r, "from hidden states")
    # the same logits given: the same bits, with and without the routing wanted
    ids2, w2 = torch.empty_like(ids), torch.empty_like(w)
    assert torch.equal(layer.forward(x, lg, residual=r, out_ids=ids2, out_weights=w2), out)
    assert torch.equal(ids2, ids) and torch.equal(w2, w)
    assert torch.equal(layer.forward(x, lg, residual=r), out)
    # the routing given
    assert torch.equal(layer.experts_forward(x, ids, w, residual=r, add_shared=True), out)
    plain = layer.experts_forward(x, ids, w)
    check(layer, None, plain, x, ids, w, None, "experts alone")


@pytest.mark.parametrize("tokens", range(1, 17))
def test_every_token_count(tokens, cuda_device):
    layer, shared = make(cuda_device, 24, 4, 256, 208, 64)
    x, wr = rnd(cuda_device, tokens, tokens, 256), rnd(cuda_device, 99, 24, 256, scale=0.1)
    out, ids, w, lg = run_x(layer, x, wr)
    dr.assert_routing(ids, w, lg, 4, True, True)
    check(layer, shared, out, x, ids, w)


def test_ties_go_to_the_lowest_expert(cuda_device):
    layer, _ = make(cuda_device, 40, 5, 64, 32)
    lg = torch.zeros(4, 40, dtype=BF16, device=cuda_device)
    lg[1, 30] = 2.0
    lg[2, 3:] = 1.0
    lg[3, ::2] = -0.0  # equal to +0
    ids = torch.empty(4, 5, dtype=torch.int64, device=cuda_device)
    layer.forward(rnd(cuda_device, 1, 4, 64), lg, out_ids=ids)
    assert ids.tolist() == [[0, 1, 2, 3, 4], [30, 0, 1, 2, 3], [3, 4, 5, 6, 7], [0, 1, 2, 3, 4]]


def test_given_routing_odd_cases(cuda_device):
    """No expert for a token, for every token, an expert twice, ids out of range, masked experts."""
    layer, shared = make(cuda_device, 10, 3, 128, 96, 32)
    t = 6
    x, r = rnd(cuda_device, 1, t, 128), rnd(cuda_device, 2, t, 128)
    w = torch.rand(t, 3, device=cuda_device).to(BF16)
    ids = torch.tensor([[0, 1, 2], [-1, -1, -1], [4, 4, 9], [9, -5, 4], [7, 7, 7], [3, -1, 3]], device=cuda_device)
    check(layer, None, layer.experts_forward(x, ids, w, residual=r), x, ids, w, r)
    check(layer, shared, layer.experts_forward(x, ids, w, add_shared=True), x, ids, w)
    none = torch.full_like(ids, -1)
    assert torch.equal(layer.experts_forward(x, none, w, residual=r), r)
    assert not bool(layer.experts_forward(x, none, w).any())
    check(layer, shared, layer.experts_forward(x, none, w, add_shared=True), x, none, w)
    # weights of experts that are left out may be anything
    w2 = w.clone()
    w2[1] = float("nan")
    assert torch.equal(layer.experts_forward(x, ids, w2, residual=r), layer.experts_forward(x, ids, w, residual=r))
    mask = torch.ones(10, dtype=torch.bool, device=cuda_device)
    mask[[4, 7]] = False
    kept = torch.where((ids == 4) | (ids == 7), -1, ids)
    assert torch.equal(layer.experts_forward(x, ids, w, offload_mask=mask), layer.experts_forward(x, kept, w))
    out = layer.experts_forward(x, ids, w, offload_mask=torch.zeros_like(mask), residual=r)
    assert torch.equal(out, r)
    assert layer.read_status() == 0
    bad = ids.clone()
    bad[0, 0] = 10
    bad[2, 2] = 1 << 40
    want = layer.experts_forward(x, torch.where(bad >= 10, -1, bad), w)
    assert torch.equal(layer.experts_forward(x, bad, w), want)
    assert layer.read_status() == 1 and layer.read_status() == 0


@pytest.mark.parametrize("tokens", [2, 7, 16])
def test_a_tokens_infinities_stay_its_own(tokens, cuda_device):
    layer, _ = make(cuda_device, 12, 2, 128, 64, 32)
    x, wr = rnd(cuda_device, 3, tokens, 128), rnd(cuda_device, 4, 12, 128, scale=0.1)
    clean = layer.forward_x(x, wr)
    x[tokens // 2, 9] = float("nan")
    out = layer.forward_x(x, wr)
    keep = [i for i in range(tokens) if i != tokens // 2]
    assert torch.equal(out[keep], clean[keep]) and bool(out[tokens // 2].isnan().all())


@pytest.mark.parametrize("tokens", [1, 5, 13])
def test_strided_rows_in_place_and_repeats(tokens, cuda_device):
    layer, _ = make(cuda_device, 16, 4, 256, 128, 64)
    wr = rnd(cuda_device, 4, 16, 256, scale=0.1)
    x, r = rnd(cuda_device, 5, tokens, 256), rnd(cuda_device, 6, tokens, 256)
    want = layer.forward_x(x, wr, residual=r)
    for _ in range(5):
        assert torch.equal(layer.forward_x(x, wr, residual=r), want)
    wide = torch.full((tokens + 2, 256 + 40), float("nan"), dtype=BF16, device=cuda_device)
    wide[1:-1, 8:264] = x
    buf = torch.full((tokens + 2, 259), 7.0, dtype=BF16, device=cuda_device)
    out = buf[1:-1, 1:257]
    layer.forward_x(wide[1:-1, 8:264], wr, residual=r, out=out)
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert bool((buf == 7.0).all()), "wrote outside its rows"
    a = r.clone()
    assert layer.forward_x(x, wr, residual=a, out=a) is a and torch.equal(a, want)
    b = x.clone()
    layer.forward_x(b, wr, residual=r, out=b)
    assert torch.equal(b, want)
    c = x.clone()
    want2 = layer.forward_x(x, wr, residual=x)
    layer.forward_x(c, wr, residual=c, out=c)
    assert torch.equal(c, want2)


@pytest.mark.parametrize("tokens", [1, 8, 16])
def test_two_streams_and_two_graphs(tokens, cuda_device):
    layer, _ = make(cuda_device, 16, 4, 512, 256, 64)
    wr = rnd(cuda_device, 4, 16, 512, scale=0.1)
    xs = [rnd(cuda_device, 20 + i, tokens, 512) for i in range(2)]
    want = [layer.forward_x(x, wr, residual=x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[layer.forward_x(x, wr, residual=x, stream=s) for _ in range(20)] for x, s in zip(xs, streams)]
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for os_, w in zip(outs, want) for o in os_)
    graphs, res = [], []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = layer.forward_x(x, wr, residual=x)
            res.append(layer.forward_x(y, wr, residual=y))
        graphs.append(g)
    for x in xs:
        x.mul_(-0.5)
    want = []
    for x in xs:
        y = layer.forward_x(x, wr, residual=x)
        want.append(layer.forward_x(y, wr, residual=y))
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(res, want))
    assert layer.read_status() == 0


def test_no_tokens_and_refusals(cuda_device):
    from nano_ktrans_b200 import DenseMoeLayer
    from nano_ktrans_b200._lib import MOE_ERANGE, MoeError

    layer, shared = make(cuda_device, 8, 2, 64, 32, 16)
    wr = rnd(cuda_device, 4, 8, 64)
    assert layer.forward_x(rnd(cuda_device, 1, 0, 64), wr).shape == (0, 64)
    x = rnd(cuda_device, 1, 4, 64)
    with pytest.raises(MoeError, match="at most 16") as e:
        layer.forward_x(rnd(cuda_device, 1, 17, 64), wr)
    assert e.value.code == MOE_ERANGE
    with pytest.raises(ValueError, match="x must be"):
        layer.forward_x(rnd(cuda_device, 1, 4, 48), wr)
    with pytest.raises(ValueError, match="x must be"):
        layer.forward_x(x.to(FP16), wr)
    with pytest.raises(ValueError, match="router_weight"):
        layer.forward_x(x, wr[:4])
    with pytest.raises(ValueError, match="router logits"):
        layer.forward(x, wr)
    with pytest.raises(ValueError, match="out_ids"):
        layer.forward_x(x, wr, out_ids=torch.empty(4, 3, dtype=torch.int64, device=cuda_device))
    with pytest.raises(ValueError, match="topk_weights"):
        layer.experts_forward(x, torch.zeros(4, 2, dtype=torch.int64, device=cuda_device), torch.ones(4, 2, device=cuda_device))
    with pytest.raises(ValueError, match="offload_mask"):
        layer.forward_x(x, wr, offload_mask=torch.ones(7, dtype=torch.bool, device=cuda_device))
    with pytest.raises(MoeError, match="16-byte"):
        layer.forward_x(rnd(cuda_device, 1, 4, 72)[:, 4:68], wr)
    with pytest.raises(MoeError, match="16-byte"):
        layer.forward_x(rnd(cuda_device, 1, 4, 68)[:, :64], wr)
    buf = rnd(cuda_device, 1, 5, 64)
    with pytest.raises(MoeError, match="overlaps"):
        layer.forward_x(buf[:4], wr, out=buf[1:])
    with pytest.raises(MoeError, match="overlaps"):
        layer.forward_x(x, wr, out=wr[:4])
    lg = torch.empty(4, 8, dtype=BF16, device=cuda_device)
    with pytest.raises(MoeError, match="two outputs"):
        layer.forward_x(x, wr, out_logits=lg, out_weights=lg.view(-1)[:8].view(4, 2))
    g, u, d = layer.gate, layer.up, layer.down
    with pytest.raises(ValueError, match="down"):
        DenseMoeLayer(g, u, u, top_k=2)
    with pytest.raises(ValueError, match="contiguous"):
        DenseMoeLayer(g, u, g.transpose(1, 2), top_k=2)
    with pytest.raises(MoeError, match="top_k"):
        DenseMoeLayer(g, u, d, top_k=17)
    with pytest.raises(MoeError, match="top_k"):
        DenseMoeLayer(g, u, d, top_k=9).forward_x(x, wr)
    with pytest.raises(MoeError, match="inter_size"):
        DenseMoeLayer(g[:, :24].contiguous(), u[:, :24].contiguous(), d[:, :, :24].contiguous(), top_k=2)


class Expert(torch.nn.Module):
    """The reference's expert: w2(silu(w1 x) * w3 x)."""

    def __init__(self, gate, up, down):
        super().__init__()
        for name, w in (("w1", gate), ("w3", up), ("w2", down)):
            lin = torch.nn.Linear(w.shape[1], w.shape[0], bias=False, device=w.device, dtype=w.dtype)
            lin.weight.data.copy_(w)
            setattr(self, name, lin)

    def forward(self, x):
        return self.w2(torch.nn.functional.silu(self.w1(x)) * self.w3(x))


@pytest.mark.parametrize("tokens", [1, 6, 16, 40])
@pytest.mark.parametrize("resident", [2, 9])
def test_hybrid_moe_with_dense_resident_experts(tokens, resident, cuda_device):
    """Resident experts from their bf16 modules and the others from their codes, in one forward: the dense path against
    the 64-bit form over the backend's own part, without a host sync; above its token limit the module loop."""
    from nano_ktrans_b200.hybrid_moe import HybridMoE
    from tests import helpers as hp

    e, k, h, i = 16, 4, 256, 128
    lw = hp.device_layer({n: hp.make_expert(5, n, h, i, 4, 128) for n in range(e)}, e, h, i, 4, 128, cuda_device)
    on = list(range(1, 1 + resident))
    mods = torch.nn.ModuleDict()
    for n in on:
        mods[str(n)] = Expert(*(rnd(cuda_device, 100 + 3 * n + j, *s, scale=0.05) for j, s in enumerate([(i, h), (i, h), (h, i)])))
    mask = torch.zeros(e, dtype=torch.bool)
    mask[on] = True
    kw = dict(num_experts=e, top_k=k, hidden_size=h, moe_intermediate_size=i, gpu_experts=mods, gpu_experts_mask=mask,
              layer_idx=0, weight_path="", router_use_softmax=True, normalize_topk_prob=True,
              offload_backend_kwargs={"device": cuda_device, "max_tokens": 64, "layer_weights": lw})
    before = [mods[str(n)].w2.weight.clone() for n in on]
    moe, loop = HybridMoE(resident_experts="dense", **kw), HybridMoE(resident_experts="modules", **kw)
    for n, w in zip(on, before):
        assert torch.equal(mods[str(n)].w2.weight, w), "stacking changed a module's weights"
    assert mods[str(on[0])].w1.weight.data_ptr() == moe._dense.gate.data_ptr()
    x, lg = rnd(cuda_device, 1, tokens, h), rnd(cuda_device, 2, tokens, e)
    want = loop(x, lg)
    moe(x, lg)
    torch.cuda.synchronize()
    if tokens <= 16:
        torch.cuda.set_sync_debug_mode("error")
    try:
        out = moe(x, lg)
    finally:
        torch.cuda.set_sync_debug_mode(0)
    if tokens > 16:
        assert torch.equal(out, want)
        return
    assert torch.equal(moe.last_topk_ids, loop.last_topk_ids)
    offloaded = moe.offload_backend.layer.experts_forward(x, moe.last_topk_ids, moe.last_topk_weights, offload_mask=~mask)
    slots = moe._dense_slot[moe.last_topk_ids]
    d = moe._dense
    dr.assert_within(out, dr.moe64(x, slots, moe.last_topk_weights, d.gate, d.up, d.down, None, offloaded))
    assert d.read_status() == 0


def test_given_routing_on_fewer_experts_than_picks(cuda_device):
    """Two stacked experts under a top-8 routing, as when two of a layer's experts are resident."""
    layer, _ = make(cuda_device, 2, 8, 128, 64)
    x, w = rnd(cuda_device, 1, 3, 128), torch.rand(3, 8, device=cuda_device).to(BF16)
    ids = torch.full((3, 8), -1, device=cuda_device)
    ids[0, 5], ids[2, 0], ids[2, 7] = 1, 1, 0
    check(layer, None, layer.experts_forward(x, ids, w), x, ids, w)
