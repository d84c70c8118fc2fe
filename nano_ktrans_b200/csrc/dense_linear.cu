// dense_linear.cu — dense projections out = act(x W^T + b) + r and the gated
// product act(x Wg^T) * (x Wu^T): the kernel for every shape and alignment.
//
// The reference computes these with nn.Linear modules: the dense decoder
// layer's and the GPU-resident experts' w2(silu(w1 x) * w3 x)
// (nano_ktrans/layers/expert_mlp.py:9-25) and the router
// (nano_ktrans/models/mixtral.py:127).
#include "dense_common.cuh"

namespace moe {
namespace dense {

// ---------------------------------------------------------------------------
// Generic tile kernel: 64 tokens x 64 features per CTA, K in steps of 32
// staged element by element in shared memory, warp-level mma with fp32
// accumulators.  It serves what the wide-load kernels do not take (K not a
// multiple of 8, rows off their 16-byte boundaries), so it makes no
// assumption on sizes, strides or alignment beyond the 2 bytes of an element.
// ---------------------------------------------------------------------------
constexpr int kGT = 64, kGK = 32, kGPad = kGK + 8;

template <typename T, bool GATED>
__global__ void __launch_bounds__(256) generic_kernel(LinearArgs a) {
  __shared__ uint16_t xs[kGT][kGPad];
  __shared__ uint16_t ws[GATED ? 2 : 1][kGT][kGPad];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kGT;
  const int wm = (warp & 3) * 16, wn = (warp >> 2) * 32;  // warp tile: 16 tokens x 32 features
  const int mtiles = (a.m + kGT - 1) / kGT;
  for (int mt = blockIdx.y; mt < mtiles; mt += gridDim.y) {
    const int m0 = mt * kGT;
    float acc[GATED ? 2 : 1][4][4] = {};
    for (int k0 = 0; k0 < a.k; k0 += kGK) {
      __syncthreads();
      for (int i = tid; i < kGT * kGK; i += 256) {
        const int r = i / kGK, c = i % kGK, k = k0 + c;
        xs[r][c] = (m0 + r < a.m && k < a.k) ? a.x[(m0 + r) * a.ldx + k] : 0;
        const bool in = n0 + r < a.n && k < a.k;
        ws[0][r][c] = in ? a.w[(n0 + r) * a.ldw + k] : 0;
        if constexpr (GATED) ws[1][r][c] = in ? a.w_up[(n0 + r) * a.ldwu + k] : 0;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < kGK; kk += 16) {
        auto ld = [&](const uint16_t* row, int c) { return *reinterpret_cast<const uint32_t*>(row + kk + c + 2 * t); };
        const uint32_t a0 = ld(xs[wm + g], 0), a1 = ld(xs[wm + g + 8], 0), a2 = ld(xs[wm + g], 8),
                       a3 = ld(xs[wm + g + 8], 8);
#pragma unroll
        for (int p = 0; p < (GATED ? 2 : 1); ++p)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint16_t* row = ws[p][wn + 8 * j + g];
            T::mma(acc[p][j], a0, a1, a2, a3, ld(row, 0), ld(row, 8));
          }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + wm + g + (i >> 1) * 8;
        const int n = n0 + wn + 8 * j + 2 * t + (i & 1);
        if (m >= a.m || n >= a.n) continue;
        float v = acc[0][j][i];
        if constexpr (GATED) {
          v = activate_rt(a.act, v) * acc[1][j][i];
        } else {
          if (a.bias) v += T::to_f32(a.bias[n]);
          v = activate_rt(a.act, v);
          if (a.res) v += T::to_f32(a.res[m * a.ldr + n]);
        }
        a.out[m * a.ldo + n] = T::from_f32(v);
      }
  }
}

template <typename T>
static cudaError_t generic(const LinearArgs& a, cudaStream_t st) {
  const int mt = (a.m + kGT - 1) / kGT;
  const dim3 grid((a.n + kGT - 1) / kGT, mt < 65535 ? mt : 65535);
  if (a.w_up)
    generic_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else
    generic_kernel<T, false><<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_generic(const LinearArgs& a, int dtype, cudaStream_t st) {
  return dtype == MOE_DTYPE_FP16 ? generic<Fp16>(a, st) : generic<Bf16>(a, st);
}

}  // namespace dense
}  // namespace moe
