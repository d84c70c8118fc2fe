"""nano_ktrans_b200 — B200 (sm_100a) device backend for nano-ktrans's routed-expert MoE path.

Public API (mirrors the reference's names):

* ``GPTQLinearWeight``, ``quantize_symmetric`` — quantized-weight container
* ``ExpertOffloadBackend``, ``normalize_offload_backend_name`` — plugin interface
* ``CudaMoEBackend`` — the ``"cuda"`` expert backend
* ``HybridMoE`` — the MoE layer using it
* ``MoeLayer`` — direct access to the C-ABI handle (route / experts / fused forward)
* ``linear``, ``gated_linear``, ``DenseMLP`` — unquantised (bf16 / fp16) projections with their
  bias, activation, gating and residual in the same kernel; ``read_dense_status``
* ``DenseMoeLayer`` — a whole expert layer on unquantised weights for a few tokens: router
  projection, routing, experts, shared expert and residual in two kernels
* ``EpMoeLayer``, ``plan_placement``, ``shard_layer``, ``TorchDistComm``,
  ``PeerExchange`` — expert parallelism over the ranks of a process group (NCCL
  all-to-alls, or the library's kernels over peer memory)
"""
from .offload_backend import ExpertOffloadBackend, normalize_offload_backend_name
from .weights import GPTQLinearWeight, LayerWeights, quantize_symmetric, stack_layer

__all__ = [
    "ExpertOffloadBackend", "normalize_offload_backend_name", "GPTQLinearWeight", "LayerWeights",
    "quantize_symmetric", "stack_layer", "CudaMoEBackend", "HybridMoE", "MoeLayer",
    "EpMoeLayer", "plan_placement", "shard_layer", "TorchDistComm", "PeerExchange",
    "linear", "gated_linear", "DenseMLP", "DenseMoeLayer", "stack_expert_modules",
    "read_dense_status",
]


_MODULES = {
    "CudaMoEBackend": "cuda_moe", "HybridMoE": "hybrid_moe", "MoeLayer": "moe_layer",
    "EpMoeLayer": "expert_parallel", "plan_placement": "expert_parallel", "shard_layer": "expert_parallel",
    "TorchDistComm": "expert_parallel", "PeerExchange": "expert_parallel",
    "linear": "dense", "gated_linear": "dense", "DenseMLP": "dense", "DenseMoeLayer": "dense_moe",
    "stack_expert_modules": "dense_moe", "read_dense_status": "dense",
}


def __getattr__(name):
    module = _MODULES.get(name)
    if module is None:
        raise AttributeError(name)
    from importlib import import_module

    # kept as a plain attribute: the next use is not looked up again
    value = globals()[name] = getattr(import_module("." + module, __name__), name)
    return value
