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

// Whether every row of x and of the weights lies on a 16-byte boundary and
// holds whole 16-byte pieces: what all kernels but the generic one need.
bool wide_rows(const LinearArgs& a);
// Up to kStreamTokens tokens, wide rows.
constexpr int kStreamTokens = 32;
cudaError_t launch_stream_linear(const LinearArgs& a, int dtype, int sms, cudaStream_t st);

// More tokens than that, wide rows: tcgen05 kernels.
cudaError_t launch_gemm(const LinearArgs& a, int dtype, int dev, int sms, cudaStream_t st);
// Which of them, on a device of `sms` SMs (dev < 0: none at hand, every cluster is taken to fit).
void plan_gemm(const LinearArgs& a, int dev, int sms, moe_linear_plan& out);
// Copy a status word to the host and clear the bits that were copied; waits for `st`.
cudaError_t take_status(const void* symbol, int* status, cudaStream_t st);
cudaError_t read_gemm_status(int* status, cudaStream_t st);

// A whole expert layer for up to kMoeTokens tokens.
constexpr int kMoeTokens = 16;
constexpr int kMoeTopK = 16;
constexpr int kMoePairs = kMoeTokens * kMoeTopK;
constexpr int kMoeExperts = 1024;
struct MoeArgs {
  const uint16_t* x;
  const uint16_t* router_w;  // logits are computed when set, else read (or unused with ids_in)
  uint16_t* logits;          // [tokens][experts]
  const int64_t* ids_in;     // given routing [tokens][top_k], or null
  const uint16_t* w_in;
  const uint8_t* mask;       // [experts], null: all
  const uint16_t *gate, *up, *down;  // [experts][inter][hidden] twice, [experts][hidden][inter]
  const uint16_t *shared_gate, *shared_up, *shared_down, *shared_gate_vec;
  const uint16_t* res;
  uint16_t* out;
  int64_t* ids_out;
  uint16_t* w_out;
  // workspace of the call
  unsigned long long* bar;
  float* shared_open;        // [tokens]
  float* partial;            // [moe_pieces][tokens][hidden]
  int h_cap;                 // set by the launcher, as is
  uint64_t inter_inverse;    // 2^64 / inter
  int64_t ldx, ldr, ldo;
  int tokens, experts, top_k, hidden, inter, shared_inter, use_softmax, renorm;
};
constexpr int kHBytes = 26624;  // of a block's h in shared memory
int64_t moe_pieces(const MoeArgs& a, int sms);
cudaError_t launch_dense_moe(MoeArgs a, int dtype, int sms, cudaStream_t st);
cudaError_t read_dense_status(int* status, cudaStream_t st);

}  // namespace dense
}  // namespace moe
