"""``DenseMoeLayer``: a whole mixture-of-experts layer on unquantised weights, for a few tokens.

The reference's MoE block with GPU-resident experts (nano_ktrans/models/mixtral.py:212-218,
layers/hybrid_moe.py:3321-3329, :3442-3533): router projection, routing, gated experts, weighted
sum, shared expert and the decoder layer's residual, in two kernel launches and without a host
read.  ``MoeLayer`` is its counterpart on quantised weights.

The layer borrows its weight tensors and goes by where they are when it is called; it keeps no
other state: every call takes its workspace from the caching allocator of the stream it runs on,
so calls on several streams are independent.
"""
from __future__ import annotations

import ctypes
import operator
from typing import Optional

import torch

from . import _lib
from .dense import _DTYPES, _empty_on, _err_buffer, _stream_on, read_dense_status

MAX_TOKENS = _lib.DENSE_MAX_TOKENS


# Attribute names of an expert's gate, up and down projection: the reference's SparseExpertMLP
# (nano_ktrans/layers/expert_mlp.py:9-23), and the checkpoints' own.
_PROJECTIONS = (("w1", "w3", "w2"), ("gate_proj", "up_proj", "down_proj"))


def _projections(module) -> list:
    """An expert module's gate, up and down layers; a ValueError where they are not three linear layers without bias whose
    weights are parameters of their own."""
    names = next((n for n in _PROJECTIONS if all(hasattr(module, a) for a in n)), None)
    layers = [getattr(module, a) for a in names or ()]
    if names is None or any(getattr(p, "bias", None) is not None or "weight" not in getattr(p, "_parameters", ()) for p in layers):
        raise ValueError(f"{type(module).__name__} is not a gated expert of three linear layers without bias")
    return layers


def stack_expert_modules(modules) -> tuple:
    """``(gate [E, I, H], up [E, I, H], down [E, H, I])`` of expert modules with ``w1`` / ``w3`` / ``w2`` (or
    ``gate_proj`` / ``up_proj`` / ``down_proj``) linear layers without bias, of one size, type and device.  The modules'
    parameters are made views of the stacks, so the weights are held once."""
    parts = [_projections(m) for m in modules]
    if not parts:
        raise ValueError("no expert modules")
    weights = [[p.weight for p in layers] for layers in parts]
    kind = {(w.dtype, w.device) for ws in weights for w in ws}
    if len(kind) > 1 or any(ws[j].shape != weights[0][j].shape for ws in weights for j in range(3)):
        raise ValueError("the experts differ in size, type or device: one stack cannot hold them")
    if len({id(w) for ws in weights for w in ws}) < 3 * len(weights):
        raise ValueError("two experts share a weight: it cannot be a view of two places")
    # Copies that autocast leaves alone, into tensors that autograd may use: the parameters become views of them.
    with torch.inference_mode(False), torch.no_grad():
        stacks = tuple(torch.empty(len(weights), *w.shape, dtype=w.dtype, device=w.device) for w in weights[0])
        for e, ws in enumerate(weights):
            for stack, w in zip(stacks, ws):
                stack[e].copy_(w)
        for e, ws in enumerate(weights):
            for stack, w in zip(stacks, ws):
                w.data = stack[e]
    return stacks


# A shared expert's weights, in the order of the layer's description.
_SHARED = ("gate", "up", "down", "gate_vec")


class DenseMoeLayer:
    """``gate`` / ``up`` [E, I, H], ``down`` [E, H, I] (bf16 or fp16, contiguous, on one CUDA device; H and I
    multiples of 16); ``shared``: ``{"gate", "up": [S, H], "down": [H, S], "gate_vec": [H]}`` or None."""

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, *, top_k: int,
                 router_use_softmax: bool = True, normalize_topk_prob: bool = True, shared: Optional[dict] = None):
        self.top_k = int(top_k)
        self.router_use_softmax, self.normalize_topk_prob = bool(router_use_softmax), bool(normalize_topk_prob)
        self.gate, self.up, self.down = gate, up, down
        self.shared = dict(shared) if shared is not None else None
        self._bind()

    def _weights(self) -> list:
        """The weight tensors as they are now, in the order of the description's pointers."""
        held = [self.gate, self.up, self.down]
        if self.shared is not None:
            held += [self.shared[n] for n in _SHARED]
        return held

    def _bind(self) -> None:
        """Check the weights and describe the layer by their present addresses.  Done again by the first call that finds
        a weight elsewhere (a parameter given another ``data``, a module moved): the memory it left may be freed."""
        gate, up, down, shared = self.gate, self.up, self.down, self.shared
        if gate.dim() != 3 or up.shape != gate.shape or down.shape != (gate.shape[0], gate.shape[2], gate.shape[1]):
            raise ValueError(f"gate and up must be [E, I, H] and down [E, H, I], got {tuple(gate.shape)}, "
                             f"{tuple(up.shape)}, {tuple(down.shape)}")
        if gate.dtype not in _DTYPES or not gate.is_cuda:
            raise ValueError(f"expert weights must be bf16 or fp16 CUDA tensors, got {gate.dtype} on {gate.device}")
        self.num_experts, self.inter_size, self.hidden_size = gate.shape
        self.dtype, self.device, self._dev = gate.dtype, gate.device, gate.get_device()
        self.shared_inter = 0
        h = self.hidden_size
        named = [("gate", gate), ("up", up), ("down", down)]
        if shared is not None:
            s = self.shared_inter = int(shared["gate"].shape[0])
            for name, shape in zip(_SHARED, ((s, h), (s, h), (h, s), (h,))):
                if tuple(shared[name].shape) != shape or s < 1:
                    raise ValueError(f"shared {name} must be {shape}, got {tuple(shared[name].shape)}")
                named.append((f"shared {name}", shared[name]))
        for name, w in named:
            if w.dtype is not gate.dtype or w.device != gate.device or not w.is_contiguous():
                raise ValueError(f"{name} must be a contiguous {gate.dtype} tensor on {gate.device}")
        at = [w.data_ptr() for w in self._weights()]
        desc = _lib.MoeDenseDesc(*at, *([None] * (3 + len(_SHARED) - len(at))), self.num_experts, self.top_k, h,
                                 self.inter_size, self.shared_inter, int(self.router_use_softmax),
                                 int(self.normalize_topk_prob), _DTYPES[gate.dtype])
        space = []  # workspace bytes by token count
        err = _err_buffer()
        with torch.cuda.device(self._dev):  # the workspace goes by the device's SMs
            for t in range(MAX_TOKENS + 1):
                desc.num_tokens = t
                n = ctypes.c_int64(0)
                rc = _lib.lib().moe_dense_workspace(ctypes.byref(desc), ctypes.byref(n), err, 512)
                if rc != _lib.MOE_OK:
                    raise _lib.MoeError(rc, err.value.decode(errors="replace"))
                space.append(n.value)
        self._space, self._layer_bytes = space, bytes(desc)
        self._at = at  # last: what another thread compares before it uses the others

    # ------------------------------------------------------------------
    def _rows(self, t: torch.Tensor, name: str, rows: Optional[int], cols: int) -> int:
        """Row stride of a [rows, cols] tensor of the layer's type, after its checks."""
        if t.dim() != 2 or t.shape[1] != cols or (rows is not None and t.shape[0] != rows):
            raise ValueError(f"{name} must be [{'T' if rows is None else rows}, {cols}], got {tuple(t.shape)}")
        if t.dtype is not self.dtype or t.get_device() != self._dev:
            raise ValueError(f"{name} must be {self.dtype} on {self.device}, got {t.dtype} on {t.device}")
        ld, inner = t.stride()
        if inner != 1:
            raise ValueError(f"{name} must have unit stride along its rows")
        return ld if t.shape[0] > 1 else cols

    def _exact(self, t: torch.Tensor, name: str, shape: tuple, dtype) -> int:
        if t.shape != shape or t.dtype is not dtype or t.get_device() != self._dev or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dtype} {shape} tensor on {self.device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        return t.data_ptr()

    def _run(self, x, residual, out, offload_mask, add_shared, stream, *, router=None, logits=None, ids=None,
             weights=None, out_ids=None, out_weights=None) -> torch.Tensor:
        if [w.data_ptr() for w in self._weights()] != self._at:
            self._bind()
        ldx = self._rows(x, "x", None, self.hidden_size)
        t = x.shape[0]
        d = _lib.MoeDenseDesc.from_buffer_copy(self._layer_bytes)
        # a count above the limit is refused, whatever its low 32 bits
        d.x_dev, d.ldx, d.num_tokens, d.add_shared = x.data_ptr(), ldx, min(t, MAX_TOKENS + 1), add_shared
        if router is not None:
            d.router_w_dev = self._exact(router, "router_weight", (self.num_experts, self.hidden_size), self.dtype)
        if logits is not None:
            d.logits_dev = self._exact(logits, "router logits", (t, self.num_experts), self.dtype)
        routing = (t, self.top_k)
        if ids is not None:
            d.ids_dev = self._exact(ids, "topk_ids", routing, torch.int64)
            d.weights_dev = self._exact(weights, "topk_weights", routing, self.dtype)
        if out_ids is not None:
            d.ids_out_dev = self._exact(out_ids, "out_ids", routing, torch.int64)
        if out_weights is not None:
            d.weights_out_dev = self._exact(out_weights, "out_weights", routing, self.dtype)
        if offload_mask is not None:
            if offload_mask.dtype not in (torch.bool, torch.uint8):
                raise ValueError(f"offload_mask must be bool or uint8, got {offload_mask.dtype}")
            d.offload_mask_dev = self._exact(offload_mask, "offload_mask", (self.num_experts,), offload_mask.dtype)
        if residual is not None:
            d.ldr = self._rows(residual, "residual", t, self.hidden_size)
            d.residual_dev = residual.data_ptr()
        if out is None:
            out = _empty_on((t, self.hidden_size), self.dtype, self.device, stream)
        d.ldo = self._rows(out, "out", t, self.hidden_size)
        d.out_dev = out.data_ptr()
        if t == 0:
            return out
        ws = None
        if t <= MAX_TOKENS:
            n = d.workspace_bytes = self._space[t]
            ws = _empty_on(n, torch.uint8, self.device, stream)
            d.workspace_dev = ws.data_ptr()
        err = _err_buffer()
        if self._dev == torch._C._cuda_getDevice():
            rc = _lib.lib().moe_dense_forward(ctypes.byref(d), _stream_on(self._dev, stream), err, 512)
        else:
            with torch.cuda.device(self._dev):
                rc = _lib.lib().moe_dense_forward(ctypes.byref(d), _stream_on(self._dev, stream), err, 512)
        if rc != _lib.MOE_OK:
            raise _lib.MoeError(rc, err.value.decode(errors="replace"))
        return out

    def forward_x(self, x: torch.Tensor, router_weight: torch.Tensor, *, residual=None, out=None, out_ids=None,
                  out_weights=None, out_logits=None, offload_mask=None, add_shared: bool = True,
                  stream=None) -> torch.Tensor:
        """The layer from hidden states ``x`` [T, H], T <= 16: routes from ``x @ router_weight.T`` (rounded to the
        layer's type; ``out_logits`` receives it), returns ``residual +`` the layer's output, rounded once.  ``out``
        may be ``x`` or ``residual`` itself."""
        return self._run(x, residual, out, offload_mask, add_shared, stream, router=router_weight, logits=out_logits,
                         out_ids=out_ids, out_weights=out_weights)

    def forward(self, x: torch.Tensor, router_logits: torch.Tensor, *, residual=None, out=None, out_ids=None,
                out_weights=None, offload_mask=None, add_shared: bool = True, stream=None) -> torch.Tensor:
        """The layer from given router logits [T, E]."""
        return self._run(x, residual, out, offload_mask, add_shared, stream, logits=router_logits, out_ids=out_ids,
                         out_weights=out_weights)

    def experts_forward(self, x: torch.Tensor, topk_ids: torch.Tensor, topk_weights: torch.Tensor, *, residual=None,
                        out=None, offload_mask=None, add_shared: bool = False, stream=None) -> torch.Tensor:
        """The experts on a given routing: ids [T, top_k] int64, negative ones mean no expert."""
        return self._run(x, residual, out, offload_mask, add_shared, stream, ids=topk_ids, weights=topk_weights)

    __call__ = forward

    def read_status(self, stream=None) -> int:
        """``read_dense_status`` of the layer's device."""
        return read_dense_status(self._dev, stream)


def _version(t: torch.Tensor) -> int:
    return 0 if t.is_inference() else t._version  # tensors made in inference mode count no changes


def _shows_silu(module, layers) -> bool:
    """Whether the module, whatever its weights, computes ``down(silu(gate(x)) * up(x))``: called on weights that show its
    activation value by value (gate and up hold a value each in the column that x picks, down is the identity), so that an
    activation of another kind, a limit, a scale or a term beside the product is seen."""
    names = {p: n for n, p in module.named_children()}
    if any(type(p).forward is not torch.nn.Linear.forward or "forward" in p.__dict__ or p not in names for p in layers):
        return False
    w = layers[0].weight
    inter, hidden = w.shape
    gate, up = torch.zeros_like(w, requires_grad=False), torch.zeros_like(w, requires_grad=False)
    gate[:, 0] = torch.linspace(-12.0, 12.0, inter, device=w.device)
    up[:, 0] = torch.linspace(-9.0, 10.0, inter, device=w.device).roll(inter // 3)
    down = torch.eye(hidden, inter, dtype=w.dtype, device=w.device)
    x = torch.zeros(3, hidden, dtype=w.dtype, device=w.device)
    x[0, 0], x[1, 0] = 1.0, -1.0
    probe = {f"{names[p]}.weight": v for p, v in zip(layers, (gate, up, down))}
    with torch.no_grad(), torch.autocast(w.device.type, enabled=False):
        try:
            out = torch.func.functional_call(module, probe, (x,))
        except Exception:  # whatever a module makes of a call that it does not take
            return False
    n = min(hidden, inter)
    g, u = gate[:n, 0].double(), up[:n, 0].double()
    want = torch.zeros(3, hidden, dtype=torch.float64, device=w.device)
    want[0, :n], want[1, :n] = g * torch.sigmoid(g) * u, g * torch.sigmoid(-g) * u
    # roundings to the type of sigmoid, silu and the product, half a unit each
    return out.shape == want.shape and bool(((out.double() - want).abs() <= 2 * torch.finfo(w.dtype).eps * want.abs()).all())


class ResidentExperts:
    """Expert modules run by a ``DenseMoeLayer``: their weights are stacked (``stack_expert_modules``) and stacked anew by the
    first call that finds one of them to be elsewhere than in the stack, whatever put it there: a module moved or cast, a
    parameter given other ``data`` or replaced, a layer or an expert exchanged, another residency mask."""

    def __init__(self, modules, mask: torch.Tensor, top_k: int, device, make_layer=DenseMoeLayer):
        self._modules, self._top_k = modules, top_k
        self._device, self._make_layer = device, make_layer
        self.layer = None                          # None: the modules are to be called themselves
        self.slot: Optional[torch.Tensor] = None   # expert -> its place in the stack, -1: not in it
        self._read(mask)
        self._stack()

    @property
    def some(self) -> bool:
        """Whether the mask of the last call named any expert as resident."""
        return len(self._resident) > 0

    def current(self, modules, mask: torch.Tensor):
        """The layer on the present weights of ``modules``, or None where they have to be called themselves: on another
        device, with hooks, or since they have become something else than bf16 experts of the layer's function."""
        same = self._same_mask(mask)
        if (not same or modules is not self._modules or not self._unchanged()
                or (self._put_off and not any(self._hooks))):
            if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the resident experts' weights or mask have changed since they were stacked: call the "
                                   "layer once outside the capture first")
            if not same:
                self._read(mask)
            self._modules = modules
            try:
                self._stack()
            except (ValueError, _lib.MoeError):
                pass
        return None if any(self._hooks) else self.layer

    def _read(self, mask: torch.Tensor) -> None:
        self._mask, self._mask_version = mask, _version(mask)
        self._mask_host = mask.bool().cpu().clone()
        self._resident = torch.nonzero(self._mask_host).flatten().tolist()

    def _same_mask(self, mask: torch.Tensor) -> bool:
        """Without a host read: a mask on a device is the same while the tensor is and counts no change."""
        if mask.device.type == "cpu":
            return torch.equal(mask.bool(), self._mask_host)
        return mask is self._mask and _version(mask) == self._mask_version

    def _stack(self) -> None:
        self.layer = self.slot = None
        here = [e for e in self._resident if str(e) in self._modules]
        experts = [self._modules[str(e)] for e in here]
        self._watch(experts)
        self._put_off = any(self._hooks)  # the check below would run them
        if self._put_off:
            return
        try:
            parts = [_projections(m) for m in experts]
            weights = [p.weight for layers in parts for p in layers]
            if weights and all(w.device == self._device for w in weights):
                if any(w.dtype is not torch.bfloat16 for w in weights):
                    raise ValueError("resident experts must be torch.bfloat16, the type of the routing weights")
                for m, layers in zip(experts, parts):
                    if not _shows_silu(m, layers):
                        raise ValueError(f"{type(m).__name__} does not compute w2(silu(w1 x) * w3 x) of its weights")
                layer = self._make_layer(*stack_expert_modules(experts), top_k=self._top_k)
                slot = torch.full((self._mask_host.numel(),), -1, dtype=torch.int64)
                slot[here] = torch.arange(len(here))
                self.layer, self.slot = layer, slot.to(self._device)
        finally:
            self._watch(experts)

    def _watch(self, experts) -> None:
        """What has to stay the same: objects under their names, and addresses.  Kept as columns, so that the comparison
        of a call runs in a few C loops."""
        children = [c for m in experts for c in m._modules.values() if c is not None]
        held = [(getattr(self._modules, "_modules", self._modules), str(e)) for e in self._resident]
        held += [(m._modules, n) for m in experts for n in m._modules]
        held += [(c._parameters, n) for c in children for n in c._parameters]
        held += [(m.__dict__, "forward") for m in experts + children]  # an instance's own, as wrappers set it
        self._dicts, self._names = [d for d, _ in held], [n for _, n in held]
        self._objects = list(map(dict.get, self._dicts, self._names))
        self._params = [w for c in children for w in c._parameters.values() if w is not None]
        self._at = list(map(torch.Tensor.data_ptr, self._params))
        self._hooks = [h for m in experts + children for h in (m._forward_hooks, m._forward_pre_hooks)]

    def _unchanged(self) -> bool:
        return (all(map(operator.is_, map(dict.get, self._dicts, self._names), self._objects))
                and list(map(torch.Tensor.data_ptr, self._params)) == self._at)
