// dense_common.cuh — device helpers of the dense (unquantised bf16 / fp16)
// projections and expert layers: element types, warp-level mma, wide loads,
// activations and the epilogue arithmetic every dense kernel shares.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "common.cuh"
#include "dense.h"

namespace moe {
namespace dense {

// 16-bit element types.  Tensors are addressed as raw 16-bit patterns; the
// tag selects the conversion and the mma operand type.
struct Bf16 {
  static constexpr bool kBf16 = true;
  static MOE_DEV float to_f32(uint16_t b) { return bf16_to_f32(b); }
  static MOE_DEV uint16_t from_f32(float f) { return f32_to_bf16(f); }
  static MOE_DEV float2 unpack(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static MOE_DEV uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static MOE_DEV void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

struct Fp16 {
  static constexpr bool kBf16 = false;
  static MOE_DEV float to_f32(uint16_t b) { return __half2float(__ushort_as_half(b)); }
  static MOE_DEV uint16_t from_f32(float f) { return __half_as_ushort(__float2half_rn(f)); }
  static MOE_DEV float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
  static MOE_DEV uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static MOE_DEV void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
};

// Activations in fp32 (the accumulator's type); the result is rounded once,
// after the residual.  Where a GELU is small its factor is computed as the small
// number that it is: 1 + erf and 1 + tanh cancel there, down to nothing below -5.5.
template <int ACT>
MOE_DEV float activate(float v) {
  if constexpr (ACT == MOE_ACT_SILU) return silu_f32(v);
  if constexpr (ACT == MOE_ACT_GELU) return 0.5f * v * erfcf(v * -0.70710678118654752f);
  if constexpr (ACT == MOE_ACT_GELU_TANH) {
    // (1 + tanh y) / 2 = 1 / (1 + e^-2y), the exponential of the negative side on both, which cannot overflow
    const float y = 0.79788456080286536f * (v + 0.044715f * v * v * v), e = expf(-2.0f * fabsf(y));
    return v * __fdividef(y < 0.0f ? e : 1.0f, 1.0f + e);  // of 1 .. 2: within 2 units
  }
  if constexpr (ACT == MOE_ACT_RELU) return v < 0.0f ? 0.0f : v;  // NaN stays NaN
  return v;
}

MOE_DEV float activate_rt(int act, float v) {
  switch (act) {
    case MOE_ACT_SILU: return activate<MOE_ACT_SILU>(v);
    case MOE_ACT_GELU: return activate<MOE_ACT_GELU>(v);
    case MOE_ACT_GELU_TANH: return activate<MOE_ACT_GELU_TANH>(v);
    case MOE_ACT_RELU: return activate<MOE_ACT_RELU>(v);
    default: return v;
  }
}

}  // namespace dense
}  // namespace moe
