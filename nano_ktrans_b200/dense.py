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
_MOST = 2 ** 31 - 256  # the description's sizes are 32 bits: a larger one would arrive as another
_tls = threading.local()
_Desc = _lib.MoeLinearDesc
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # a torch built without CUDA has none
_entry = None


def _moe_linear():
    """The library's entry point, looked up once."""
    global _entry
    if _entry is None:
        _entry = _lib.lib().moe_linear
    return _entry


def _err_buffer():
    buf = getattr(_tls, "err", None)
    if buf is None:
        buf = _tls.err = ctypes.create_string_buffer(512)
    return buf


def _stream_on(device_index: int, stream) -> int:
    if stream is None:
        return _raw_stream(device_index)
    return stream if isinstance(stream, int) else stream.cuda_stream


def _empty_on(shape, dtype, device, stream) -> torch.Tensor:
    """A new tensor that belongs to the stream the kernels run on: allocated for another
    stream, its memory could be handed out again while they still write it."""
    if stream is None or _stream_on(device.index, stream) == _raw_stream(device.index):
        return torch.empty(shape, dtype=dtype, device=device)
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _row_stride(t: torch.Tensor, name: str, rows: Optional[int], cols: int, dtype, dev: int) -> int:
    """Row stride of a [rows, cols] tensor after its checks.  The first test is the usual case in as few attribute
    reads as it takes: these checks are most of what a small call costs on the host."""
    shape = t.shape
    if len(shape) == 2 and shape[1] == cols and shape[0] == rows and t.dtype is dtype and t.get_device() == dev \
            and t.is_contiguous():
        return cols
    if t.dim() != 2 or shape[1] != cols or (rows is not None and shape[0] != rows):
        raise ValueError(f"{name} must be [{'n' if rows is None else rows}, {cols}], got {tuple(shape)}")
    if t.dtype is not dtype or t.get_device() != dev:
        raise ValueError(f"{name} must be {dtype} on cuda:{dev}, got {t.dtype} on {t.device}")
    ld, inner = t.stride()
    if inner != 1 and cols > 1:
        raise ValueError(f"{name} must have unit stride along its rows")
    return ld if shape[0] > 1 else cols


def _project(x, weight, up, bias, activation, residual, out, stream) -> torch.Tensor:
    dtype = x.dtype
    code = _DTYPES.get(dtype)
    if code is None or not x.is_cuda or x.dim() != 2 or weight.dim() != 2:
        raise ValueError(f"x must be a bf16 or fp16 [m, k] CUDA tensor and the weight [n, k], got {x.dtype} "
                         f"{tuple(x.shape)} on {x.device} and {tuple(weight.shape)}")
    act = _lib.ACTIVATIONS.get(activation, -1)
    if act < 0:
        raise ValueError(f"unknown activation {activation!r}: one of {sorted(k for k in _lib.ACTIVATIONS if k)}")
    dev = x.get_device()
    m, k = x.shape
    n = weight.shape[0]
    ldx = _row_stride(x, "x", m, k, dtype, dev)
    ldw = _row_stride(weight, "weight" if up is None else "gate_weight", n, k, dtype, dev)
    if n < 1 or k < 1:
        raise ValueError(f"empty weight {tuple(weight.shape)}")
    if m > _MOST or n > _MOST or k > _MOST:
        raise ValueError(f"m, n and k are at most {_MOST}, got {m}, {n}, {k}")
    up_ptr = bias_ptr = res_ptr = None
    ldu = ldr = 0
    if up is not None:
        ldu, up_ptr = _row_stride(up, "up_weight", n, k, dtype, dev), up.data_ptr()
    if bias is not None:
        if bias.shape != (n,) or bias.dtype is not dtype or bias.get_device() != dev or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous {dtype} [{n}] tensor on {x.device}")
        bias_ptr = bias.data_ptr()
    if residual is not None:
        ldr, res_ptr = _row_stride(residual, "residual", m, n, dtype, dev), residual.data_ptr()
    if out is None:
        out = _empty_on((m, n), dtype, x.device, stream)
        ldo = n
    else:
        ldo = _row_stride(out, "out", m, n, dtype, dev)
    if m == 0:
        return out
    desc = _Desc(x.data_ptr(), weight.data_ptr(), up_ptr, bias_ptr, res_ptr, out.data_ptr(), ldx, ldw, ldu, ldr, ldo,
                 m, n, k, code, act)
    err = _err_buffer()
    if dev == torch._C._cuda_getDevice():
        rc = _moe_linear()(desc, _raw_stream(dev) if stream is None else _stream_on(dev, stream), err, 512)
    else:
        with torch.cuda.device(dev):
            rc = _moe_linear()(desc, _stream_on(dev, stream), err, 512)
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
    if up_weight is None:
        raise ValueError("up_weight is missing: linear is the product with one weight")
    return _project(x, gate_weight, up_weight, None, activation, None, out, stream)


def read_dense_status(device=None, stream=None) -> int:
    """Status bits (as ``MoeLayer.read_status``) of the dense calls on a device (the current one) since the last read,
    whichever operator or layer made them and whoever reads; synchronises the stream."""
    dev = torch.device("cuda" if device is None else device) if not isinstance(device, int) else torch.device("cuda", device)
    if dev.type != "cuda":
        raise ValueError(f"the dense operators run on CUDA devices, not on {dev}")
    st, err = ctypes.c_int32(0), _err_buffer()
    index = torch.cuda.current_device() if dev.index is None else dev.index
    with torch.cuda.device(index):
        rc = _lib.lib().moe_dense_read_status(ctypes.byref(st), _stream_on(index, stream), err, 512)
    if rc != _lib.MOE_OK:
        raise _lib.MoeError(rc, err.value.decode(errors="replace"))
    return int(st.value)


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
