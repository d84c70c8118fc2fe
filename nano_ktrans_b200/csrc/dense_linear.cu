// dense_linear.cu — dense projections out = act(x W^T + b) + r and the gated
// product act(x Wg^T) * (x Wu^T): the kernel for every shape and alignment,
// and the weight-streaming kernel for a few tokens.
//
// The reference computes these with nn.Linear modules: the dense decoder
// layer's and the GPU-resident experts' w2(silu(w1 x) * w3 x)
// (nano_ktrans/layers/expert_mlp.py:9-25) and the router
// (nano_ktrans/models/mixtral.py:127).
#include "dense_stream.cuh"
#include "kernels.h"

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

// Its time is the staging loads that are under way at once.  Left to the compiler,
// their number changed with the size of the epilogue (512 x 4096 x 4095, 312 to
// 595 us): the loads are unrolled here and the activation is a template argument
// (242 us; 7 x 4096 x 4095 136 us, gated 280).
template <typename T, bool GATED, int ACT>
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
#pragma unroll
      for (int j = 0; j < kGT * kGK / 256; ++j) {
        const int i = tid + 256 * j, r = i / kGK, c = i % kGK, k = k0 + c;
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
          v = activate<ACT>(v) * acc[1][j][i];
        } else {
          if (a.bias) v += T::to_f32(a.bias[n]);
          v = activate<ACT>(v);
          if (a.res) v += T::to_f32(a.res[m * a.ldr + n]);
        }
        a.out[m * a.ldo + n] = T::from_f32(v);
      }
  }
}

template <typename T, int ACT>
static cudaError_t generic(const LinearArgs& a, cudaStream_t st) {
  const int mt = (a.m + kGT - 1) / kGT;
  const dim3 grid((a.n + kGT - 1) / kGT, mt < 65535 ? mt : 65535);
  if (a.w_up)
    generic_kernel<T, true, ACT><<<grid, 256, 0, st>>>(a);
  else
    generic_kernel<T, false, ACT><<<grid, 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t generic_act(const LinearArgs& a, cudaStream_t st) {
  switch (a.act) {
    case MOE_ACT_SILU: return generic<T, MOE_ACT_SILU>(a, st);
    case MOE_ACT_GELU: return generic<T, MOE_ACT_GELU>(a, st);
    case MOE_ACT_GELU_TANH: return generic<T, MOE_ACT_GELU_TANH>(a, st);
    case MOE_ACT_RELU: return generic<T, MOE_ACT_RELU>(a, st);
    default: return generic<T, MOE_ACT_NONE>(a, st);
  }
}

cudaError_t launch_generic(const LinearArgs& a, int dtype, cudaStream_t st) {
  return dtype == MOE_DTYPE_FP16 ? generic_act<Fp16>(a, st) : generic_act<Bf16>(a, st);
}

// ---------------------------------------------------------------------------
// A few tokens: weight rows streamed past the token columns (dense_stream.cuh).
// One block per SM, each with a range of features; the ranges differ by one
// feature at most.  A plain tile is 16 features; a
// gated tile is 8 gate rows (mma rows 0-7) and the same 8 up rows (mma rows
// 8-15), so gate and up of a feature meet in one thread.
// ---------------------------------------------------------------------------
template <bool GATED, int NT>
struct LinearSrc {
  struct Tile {
    const uint16_t *p, *u;  // this lane's first row (the block's last one where there is none), of each weight when gated
    int left;               // rows from there to the block's end
  };
  const LinearArgs& a;
  int r0, r1, t8;
  const uint16_t* xrow[NT];
  MOE_DEV LinearSrc(const LinearArgs& args, int lo, int hi) : a(args), r0(lo), r1(hi) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
    t8 = 8 * (lane & 3);
#pragma unroll
    for (int j = 0; j < NT; ++j) xrow[j] = 8 * j + g < a.m ? a.x + (8 * j + g) * a.ldx + t8 : nullptr;
  }
  MOE_DEV int length() const { return a.k; }
  MOE_DEV Tile tile(int i) const {
    const int r = r0 + (GATED ? 8 : 16) * i + ((threadIdx.x & 31) >> 3), in = min(r, r1 - 1);
    return {a.w + in * a.ldw, GATED ? a.w_up + in * a.ldwu : nullptr, r1 - r};
  }
  MOE_DEV void rows(const Tile& t, int k, const uint16_t* (&p)[4], uint32_t& valid) const {
    if constexpr (GATED) {
      const bool two = t.left > 4;
      p[0] = t.p + k;
      p[1] = p[0] + (two ? 4 * a.ldw : 0);
      p[2] = t.u + k;
      p[3] = p[2] + (two ? 4 * a.ldwu : 0);
      valid = (t.left > 0 ? 5u : 0u) | (two ? 10u : 0u);
    } else {
      p[0] = t.p + k;
      valid = t.left > 0 ? 1u : 0u;
#pragma unroll
      for (int i = 1; i < 4; ++i) {
        const bool in = t.left > 4 * i;
        p[i] = p[0] + (in ? 4 * i * a.ldw : 0);
        valid |= in ? 1u << i : 0u;
      }
    }
  }
  MOE_DEV void tokens(int k, bool two, int j, uint4& x0, uint4& x1) const {
    const uint4 z = make_uint4(0, 0, 0, 0);
    x0 = xrow[j] != nullptr && k + t8 < a.k ? ld_tokens(xrow[j] + k) : z;
    x1 = two && xrow[j] != nullptr && k + 32 + t8 < a.k ? ld_tokens(xrow[j] + k + 32) : z;
  }
};

template <typename T, bool GATED, int NT, int RT>
__global__ void __launch_bounds__(kSThreads, 1) stream_linear_kernel(const __grid_constant__ LinearArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  // A launch that may start early reads nothing before its predecessor is done
  // (weights too: they may be that kernel's output), and lets none start early.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // the first n % blocks blocks have a row more (one 32-bit division: this is on the way to the first load)
  const uint32_t blocks = gridDim.x, b = blockIdx.x, each = static_cast<uint32_t>(a.n) / blocks, more = a.n - each * blocks;
  const int r0 = static_cast<int>(each * b + min(b, more)), r1 = r0 + static_cast<int>(each + (b < more ? 1u : 0u));
  constexpr int kRows = GATED ? 8 : 16;
  const int tiles = (r1 - r0 + kRows - 1) / kRows;
  const LinearSrc<GATED, NT> src(a, r0, r1);
  Streamer<T, NT, RT, kRows, LinearSrc<GATED, NT>> s(src, smem);
  s.prologue(tiles);
  s.run(a.m, [&](int tile, int row, int col, auto sum) {
    const int n = r0 + kRows * tile + row;
    if (n >= r1) return;
    float v = sum(row, col);
    if constexpr (GATED) {
      v = activate_rt(a.act, v) * sum(row + 8, col);
    } else {
      if (a.bias) v += T::to_f32(a.bias[n]);
      v = activate_rt(a.act, v);
      if (a.res) v += T::to_f32(a.res[col * a.ldr + n]);
    }
    a.out[col * a.ldo + n] = T::from_f32(v);
  }, [] {});
}

template <typename T, bool GATED, int NT, int RT>
static cudaError_t stream_launch(const LinearArgs& a, int sms, cudaStream_t st) {
  const void* kern = reinterpret_cast<const void*>(stream_linear_kernel<T, GATED, NT, RT>);
  constexpr size_t smem = kStreamBytes;
  if (!ensure_dynamic_smem(kern, smem, kSThreads)) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.n < sms ? a.n : sms);
  cfg.blockDim = dim3(kSThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, stream_linear_kernel<T, GATED, NT, RT>, a);
}

template <typename T, bool GATED, int NT>
static cudaError_t stream_tiles(const LinearArgs& a, int sms, cudaStream_t st) {
  const int rows = (a.n + sms - 1) / sms, tile = GATED ? 8 : 16;  // a block's rows
  const int rt = tiles_at_once<NT>((rows + tile - 1) / tile, a.k);
  if constexpr (NT == 1)
    if (rt == 4) return stream_launch<T, GATED, NT, 4>(a, sms, st);
  if constexpr (NT <= 2)
    if (rt == 2) return stream_launch<T, GATED, NT, 2>(a, sms, st);
  return stream_launch<T, GATED, NT, 1>(a, sms, st);
}

template <typename T, bool GATED>
static cudaError_t stream_cols(const LinearArgs& a, int sms, cudaStream_t st) {
  return a.m <= 8 ? stream_tiles<T, GATED, 1>(a, sms, st)
         : a.m <= 16 ? stream_tiles<T, GATED, 2>(a, sms, st)
                     : stream_tiles<T, GATED, 4>(a, sms, st);
}

bool wide_rows(const LinearArgs& a) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) |
                      reinterpret_cast<uintptr_t>(a.w_up);
  // a single row has no stride to respect
  const int64_t l = (a.m > 1 ? a.ldx : 0) | (a.n > 1 ? a.ldw : 0) | (a.n > 1 && a.w_up ? a.ldwu : 0) | a.k;
  return p % 16 == 0 && l % 8 == 0;
}

cudaError_t launch_stream_linear(const LinearArgs& a, int dtype, int sms, cudaStream_t st) {
  if (dtype == MOE_DTYPE_FP16) return a.w_up ? stream_cols<Fp16, true>(a, sms, st) : stream_cols<Fp16, false>(a, sms, st);
  return a.w_up ? stream_cols<Bf16, true>(a, sms, st) : stream_cols<Bf16, false>(a, sms, st);
}

}  // namespace dense
}  // namespace moe
