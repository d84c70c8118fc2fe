"""Dense (unquantised bf16 / fp16) projections and the MLP built from them.

``linear``        ``act(x W^T + b) + residual`` in one kernel
``gated_linear``  ``act(x Wg^T) * (x Wu^T)`` in one kernel
``DenseMLP``      ``w2(silu(w1 x) * w3 x)``: the reference's ``SparseExpertMLP``
                  (nano_ktrans/layers/expert_mlp.py:9-25) of a dense decoder layer or a
                  GPU-resident expert, as two launches

The quantised counterpart is ``QuantizedDenseMLP``.  Sums are fp32 and each result is
rounded once.  Calls only enqueue on the stream (the tensors' device's current stream unless
one is given) and keep nothing between calls.
"""
from __future__ import annotations

import ctypes
import threading
from typing import Optional

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_tls = threading.local()


def _err_buffer():
    buf = getattr(_tls, "err", None)
    if buf is None:
        buf = _tls.err = ctypes.create_string_buffer(512)
    return buf


def _stream_on(device_index: int, stream) -> int:
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device_index)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _empty_on(shape, dtype, device, stream) -> torch.Tensor:
    """A new tensor that belongs to the stream the kernels run on: allocated for another
    stream, its memory could be handed out again while they still write it."""
    if stream is None or _stream_on(device.index, stream) == torch._C._cuda_getCurrentRawStream(device.index):
        return torch.empty(shape, dtype=dtype, device=device)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _matrix(t: torch.Tensor, name: str, rows: Optional[int], cols: int, like: torch.Tensor) -> int:
    """Row stride of a [rows, cols] tensor after its checks."""
    if t.dim() != 2 or t.shape[1] != cols or (rows is not None and t.shape[0] != rows):
        raise ValueError(f"{name} must be [{'n' if rows is None else rows}, {cols}], got {tuple(t.shape)}")
    if t.dtype is not like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    ld, inner = t.stride()
    if inner != 1 and cols > 1:
        raise ValueError(f"{name} must have unit stride along its rows")
    return ld if t.shape[0] > 1 else cols


def _project(x, weight, up, bias, activation, residual, out, stream) -> torch.Tensor:
    dtype = _DTYPES.get(x.dtype)
    if dtype is None or not x.is_cuda or x.dim() != 2:
        raise ValueError(f"x must be a bf16 or fp16 [m, k] CUDA tensor, got {x.dtype} {tuple(x.shape)} on {x.device}")
    act = _lib.ACTIVATIONS.get(activation, -1)
    if act < 0:
        raise ValueError(f"unknown activation {activation!r}: one of {sorted(k for k in _lib.ACTIVATIONS if k)}")
    m, k = x.shape
    ldx = _matrix(x, "x", m, k, x)
    ldw = _matrix(weight, "weight" if up is None else "gate_weight", None, k, x)
    n = weight.shape[0]
    if n < 1 or k < 1:
        raise ValueError(f"empty weight {tuple(weight.shape)}")
    ldu = 0 if up is None else _matrix(up, "up_weight", n, k, x)
    if bias is not None and (bias.shape != (n,) or bias.dtype is not x.dtype or bias.device != x.device
                             or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous {x.dtype} [{n}] tensor on {x.device}")
    ldr = 0 if residual is None else _matrix(residual, "residual", m, n, x)
    if out is None:
        out = _empty_on((m, n), x.dtype, x.device, stream)
    ldo = _matrix(out, "out", m, n, x)
    if m == 0:
        return out
    dev = x.get_device()
    desc = _lib.MoeLinearDesc(x.data_ptr(), weight.data_ptr(), None if up is None else up.data_ptr(),
                              None if bias is None else bias.data_ptr(),
                              None if residual is None else residual.data_ptr(), out.data_ptr(),
                              ldx, ldw, ldu, ldr, ldo, m, n, k, dtype, act)
    err = _err_buffer()
    if dev == torch.cuda.current_device():
        rc = _lib.lib().moe_linear(ctypes.byref(desc), _stream_on(dev, stream), err, 512)
    else:
        with torch.cuda.device(dev):
            rc = _lib.lib().moe_linear(ctypes.byref(desc), _stream_on(dev, stream), err, 512)
    if rc != _lib.MOE_OK:
        raise _lib.MoeError(rc, err.value.decode(errors="replace"))
    return out


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
           activation: Optional[str] = None, residual: Optional[torch.Tensor] = None,
           out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``, rounded once.

    ``x`` [m, k], ``weight`` [n, k], ``bias`` [n], ``residual`` / ``out`` [m, n]: one of bf16 or fp16
    for all, unit stride along rows, any row stride.  ``activation``: None, "silu", "gelu",
    "gelu_tanh" or "relu".  ``out`` may be ``residual`` itself and no other input."""
    return _project(x, weight, None, bias, activation, residual, out, stream)


def gated_linear(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, *,
                 activation: Optional[str] = "silu", out: Optional[torch.Tensor] = None,
                 stream=None) -> torch.Tensor:
    """``act(x @ gate_weight.T) * (x @ up_weight.T)``, rounded once: the first half of a gated MLP."""
    return _project(x, gate_weight, up_weight, None, activation, None, out, stream)


class DenseMLP:
    """``forward(x [T, H]) -> [T, H]`` = ``down(silu(gate(x)) * up(x))`` (+ residual) on unquantised
    weights ``gate`` / ``up`` [I, H] and ``down`` [H, I] (the reference's ``w1`` / ``w3`` / ``w2``).
    The product between the two launches is rounded to the weights' type, as between the
    reference's modules."""

    def __init__(self, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor, *, activation: str = "silu"):
        if gate.dim() != 2 or up.shape != gate.shape or down.shape != (gate.shape[1], gate.shape[0]):
            raise ValueError(f"gate and up must be [I, H] and down [H, I], got {tuple(gate.shape)}, "
                             f"{tuple(up.shape)}, {tuple(down.shape)}")
        self.gate, self.up, self.down, self.activation = gate, up, down, activation
        self.intermediate_size, self.hidden_size = gate.shape

    def forward(self, x: torch.Tensor, *, residual: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
        h = gated_linear(x, self.gate, self.up, activation=self.activation, stream=stream)
        return linear(h, self.down, residual=residual, out=out, stream=stream)

    __call__ = forward
