// dense.h — host-side launchers of the dense (unquantised) kernels.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/moe_b200.h"

namespace moe {
namespace dense {

// One projection: out = act(x W^T + b) + r, or with w_up set
// out = act(x W^T) * (x Wup^T).  Strides are elements between rows.
struct LinearArgs {
  const uint16_t* x;
  const uint16_t* w;
  const uint16_t* w_up;  // gated product when not null
  const uint16_t* bias;
  const uint16_t* res;
  uint16_t* out;
  int64_t ldx, ldw, ldwu, ldr, ldo;
  int m, n, k;
  int act;
};

// Every shape, stride and alignment.
cudaError_t launch_generic(const LinearArgs& a, int dtype, cudaStream_t st);

}  // namespace dense
}  // namespace moe
