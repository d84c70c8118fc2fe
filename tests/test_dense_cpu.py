"""Argument checks of the dense operators that need no GPU: the C entry refuses before it launches anything."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nano_ktrans_b200 import _lib, build

    build.build()
    return _lib.lib()


def desc(**kw):
    from nano_ktrans_b200 import _lib

    # addresses that no call here reaches: every one of these descriptions is refused
    d = dict(x_dev=0x10000, w_dev=0x20000, w_up_dev=None, bias_dev=None, residual_dev=None, out_dev=0x90000,
             ldx=64, ldw=64, ldw_up=64, ldr=32, ldo=32, m=4, n=32, k=64, dtype=0, activation=0)
    d.update(kw)
    return _lib.MoeLinearDesc(**d)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(activation=9), "activation"),
    (dict(activation=-1), "activation"), (dict(m=-1), "m must be"), (dict(n=0), "n and k"), (dict(k=0), "n and k"),
    (dict(x_dev=None), "null"), (dict(w_dev=None), "null"), (dict(out_dev=None), "null"),
    (dict(x_dev=0x10001), "aligned"), (dict(ldx=63), "apart"), (dict(ldw=10), "apart"), (dict(ldo=31), "apart"),
    (dict(residual_dev=0x50000, ldr=16), "apart"), (dict(w_up_dev=0x30000, ldw_up=2), "apart"),
    (dict(w_up_dev=0x30000, bias_dev=0x40000), "gated"), (dict(w_up_dev=0x30000, residual_dev=0x40000), "gated"),
    (dict(out_dev=0x10000), "overlaps"), (dict(out_dev=0x20002), "overlaps"),
    (dict(residual_dev=0x90002), "overlaps"), (dict(residual_dev=0x90000, ldr=40), "overlaps"),
    (dict(bias_dev=0x90000), "overlaps"), (dict(w_up_dev=0x90000 - 2), "overlaps"),
])
def test_linear_refuses(lib, kw, needle):
    from nano_ktrans_b200 import _lib

    err = ctypes.create_string_buffer(256)
    d = desc(**kw)
    assert lib.moe_linear(ctypes.byref(d), None, err, len(err)) == _lib.MOE_EINVAL
    assert needle in err.value.decode()
    assert lib.moe_linear(ctypes.byref(d), None, None, 0) == _lib.MOE_EINVAL  # no buffer for the message


def test_linear_without_rows_and_without_description(lib):
    from nano_ktrans_b200 import _lib

    d = desc(m=0, x_dev=None, out_dev=None)
    assert lib.moe_linear(ctypes.byref(d), None, None, 0) == _lib.MOE_OK
    assert lib.moe_linear(None, None, None, 0) == _lib.MOE_EINVAL


def test_host_tensors_are_refused():
    from nano_ktrans_b200 import gated_linear, linear

    x, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        linear(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        gated_linear(x, w, w)


def test_dense_mlp_checks_its_shapes():
    from nano_ktrans_b200 import DenseMLP

    g = torch.zeros(8, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="gate and up"):
        DenseMLP(g, g, g)
    mlp = DenseMLP(g, g, g.t())
    assert (mlp.hidden_size, mlp.intermediate_size) == (4, 8)


def moe_desc(**kw):
    from nano_ktrans_b200 import _lib

    # addresses that no call here reaches: every one of these descriptions is refused
    d = dict(gate_dev=0x100000, up_dev=0x200000, down_dev=0x300000, num_experts=8, top_k=2, hidden_size=64, inter_size=32,
             shared_inter=0, router_use_softmax=1, normalize_topk_prob=1, dtype=0, x_dev=0x400000, router_w_dev=0x500000,
             out_dev=0x600000, workspace_dev=0x1700000, ldx=64, ldr=64, ldo=64, workspace_bytes=1 << 24, num_tokens=4,
             add_shared=1)
    d.update(kw)
    return _lib.MoeDenseDesc(**d)


SHARED = dict(shared_inter=16, shared_gate_dev=0x800000, shared_up_dev=0x810000, shared_down_dev=0x820000,
              shared_gate_vec_dev=0x830000)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=3), "dtype"), (dict(num_experts=0), "num_experts"), (dict(num_experts=1025), "num_experts"),
    (dict(top_k=0), "top_k"), (dict(top_k=9), "top_k"), (dict(num_experts=32, top_k=17), "top_k"),
    (dict(hidden_size=40), "hidden_size"), (dict(hidden_size=0), "hidden_size"), (dict(inter_size=8), "inter_size"),
    (dict(shared_inter=8), "shared_inter"), (dict(num_tokens=-1), "token"), (dict(gate_dev=None), "null"),
    (dict(x_dev=None), "null"), (dict(workspace_dev=None), "null"), (dict(SHARED, shared_up_dev=None), "shared"),
    (dict(router_w_dev=None), "no routing"), (dict(ids_dev=0x900000), "given routing"),
    (dict(ids_dev=0x900000, weights_dev=0x910000), "given routing"),
    (dict(router_w_dev=None, ids_dev=0x900000, weights_dev=0x910000, ids_out_dev=0x920000), "not written"),
    (dict(x_dev=0x400008), "16-byte"), (dict(down_dev=0x300008), "16-byte"), (dict(ldx=68), "16-byte"),
    (dict(SHARED, shared_gate_vec_dev=0x830002), "16-byte"), (dict(out_dev=0x600001), "2-byte"),
    (dict(ids_out_dev=0x900004), "8-byte"), (dict(ldx=48), "apart"), (dict(ldo=63), "apart"),
    (dict(residual_dev=0x900000, ldr=32), "apart"), (dict(workspace_dev=0x1700010), "workspace"),
    (dict(workspace_bytes=100), "workspace"), (dict(out_dev=0x400080), "overlaps"), (dict(out_dev=0x100100), "overlaps"),
    (dict(workspace_dev=0x400000), "overlaps"), (dict(out_dev=0x400000, ldo=80), "overlaps"),
    (dict(weights_out_dev=0x600000), "two outputs"), (dict(logits_dev=0x600010), "two outputs"),
    (dict(SHARED, out_dev=0x820000), "overlaps"),
])
def test_dense_moe_refuses(lib, kw, needle):
    from nano_ktrans_b200 import _lib

    err = ctypes.create_string_buffer(256)
    d = moe_desc(**kw)
    assert lib.moe_dense_forward(ctypes.byref(d), None, err, len(err)) == _lib.MOE_EINVAL
    assert needle in err.value.decode(), err.value


def test_dense_moe_token_limits_and_workspace(lib):
    from nano_ktrans_b200 import _lib

    err = ctypes.create_string_buffer(256)
    n = ctypes.c_int64(-1)
    assert lib.moe_dense_forward(ctypes.byref(moe_desc(num_tokens=0, x_dev=None)), None, err, len(err)) == _lib.MOE_OK
    assert lib.moe_dense_forward(ctypes.byref(moe_desc(num_tokens=17)), None, err, len(err)) == _lib.MOE_ERANGE
    assert lib.moe_dense_workspace(ctypes.byref(moe_desc(num_tokens=17)), ctypes.byref(n), err, len(err)) == _lib.MOE_ERANGE
    assert lib.moe_dense_workspace(ctypes.byref(moe_desc(**SHARED)), ctypes.byref(n), err, len(err)) == _lib.MOE_OK
    # barrier, shared gates, logits, a row of partial sums for every token and piece of the split
    assert n.value >= 8 + 4 * 4 + 2 * 4 * 8 + 148 * 4 * 64 * 4 and n.value % 256 == 0
    assert lib.moe_dense_workspace(None, ctypes.byref(n), err, len(err)) == _lib.MOE_EINVAL
    assert lib.moe_dense_read_status(None, None, err, len(err)) == _lib.MOE_EINVAL


def test_dense_moe_layer_refuses_host_weights():
    from nano_ktrans_b200 import DenseMoeLayer

    g, d = torch.zeros(4, 16, 32, dtype=torch.bfloat16), torch.zeros(4, 32, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        DenseMoeLayer(g, g, d, top_k=2)
    with pytest.raises(ValueError, match="gate and up"):
        DenseMoeLayer(g, d, d, top_k=2)


def test_stack_expert_modules():
    """The stacks hold the modules' weights and the modules keep views of them."""
    from nano_ktrans_b200 import stack_expert_modules

    class Expert(torch.nn.Module):
        def __init__(self, names, bias=False):
            super().__init__()
            for n, (o, i) in zip(names, [(3, 4), (3, 4), (4, 3)]):
                setattr(self, n, torch.nn.Linear(i, o, bias=bias))

    mods = [Expert(("w1", "w3", "w2")), Expert(("gate_proj", "up_proj", "down_proj"))]
    want = [[getattr(m, n).weight.detach().clone() for n in names]
            for m, names in zip(mods, (("w1", "w3", "w2"), ("gate_proj", "up_proj", "down_proj")))]
    gate, up, down = stack_expert_modules(mods)
    for e in range(2):
        for stack, w in zip((gate, up, down), want[e]):
            assert torch.equal(stack[e], w)
    down[1].mul_(2)
    assert torch.equal(mods[1].down_proj.weight, want[1][2] * 2)
    with pytest.raises(ValueError, match="without bias"):
        stack_expert_modules([Expert(("w1", "w3", "w2"), bias=True)])
    with pytest.raises(ValueError, match="gated expert"):
        stack_expert_modules([torch.nn.Linear(2, 2)])
    with pytest.raises(ValueError, match="no expert"):
        stack_expert_modules([])
