// dense_api.cu — extern "C" entry points of the dense (unquantised) operators.
//
// Stateless calls: no handle, nothing kept between calls, so calls on
// different streams or in different graphs do not meet.  The error convention
// is moe_create's: int status, message in the caller's buffer.
#include <cstdarg>
#include <cstdio>

#include "../../include/moe_b200.h"
#include "dense.h"

namespace {

using moe::dense::LinearArgs;

int refuse(char* buf, size_t len, int code, const char* f, ...) {
  if (buf != nullptr && len > 0) {
    va_list ap;
    va_start(ap, f);
    vsnprintf(buf, len, f, ap);
    va_end(ap);
  }
  return code;
}

// Bytes [lo, hi) that `rows` rows of `cols` 16-bit elements, `ld` apart, lie in.
struct Span {
  uintptr_t lo, hi;
};
Span span(const void* p, int64_t rows, int64_t cols, int64_t ld) {
  const uintptr_t b = reinterpret_cast<uintptr_t>(p);
  return {b, rows > 0 ? b + 2 * static_cast<uintptr_t>((rows - 1) * ld + cols) : b};
}
bool meet(const Span& a, const Span& b) { return a.lo < b.hi && b.lo < a.hi; }

}  // namespace

extern "C" {

int moe_linear(const moe_linear_desc* d, void* stream, char* err, size_t err_len) {
  const char* me = "moe_linear";
  if (d == nullptr) return refuse(err, err_len, MOE_EINVAL, "%s: null argument", me);
  if (d->dtype != MOE_DTYPE_BF16 && d->dtype != MOE_DTYPE_FP16)
    return refuse(err, err_len, MOE_EINVAL, "%s: dtype must be MOE_DTYPE_BF16 or MOE_DTYPE_FP16", me);
  if (d->activation < MOE_ACT_NONE || d->activation > MOE_ACT_RELU)
    return refuse(err, err_len, MOE_EINVAL, "%s: unknown activation %d", me, d->activation);
  if (d->m < 0 || d->n < 1 || d->k < 1)
    return refuse(err, err_len, MOE_EINVAL, "%s: m must be >= 0, n and k >= 1 (got %d, %d, %d)", me, d->m, d->n, d->k);
  if (d->m == 0) return MOE_OK;
  if (d->x_dev == nullptr || d->w_dev == nullptr || d->out_dev == nullptr)
    return refuse(err, err_len, MOE_EINVAL, "%s: null device pointer", me);
  const void* ptrs[] = {d->x_dev, d->w_dev, d->w_up_dev, d->bias_dev, d->residual_dev, d->out_dev};
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % 2) return refuse(err, err_len, MOE_EINVAL, "%s: pointers must be 2-byte aligned", me);
  if (d->w_up_dev && (d->bias_dev || d->residual_dev))
    return refuse(err, err_len, MOE_EINVAL, "%s: a gated product takes no bias and no residual", me);
  if (d->ldx < d->k || d->ldw < d->k || (d->w_up_dev && d->ldw_up < d->k))
    return refuse(err, err_len, MOE_EINVAL, "%s: the rows of x and of the weights must be at least k apart", me);
  if (d->ldo < d->n || (d->residual_dev && d->ldr < d->n))
    return refuse(err, err_len, MOE_EINVAL, "%s: the rows of out and residual must be at least n apart", me);
  // Every block writes its part of out while others still read the inputs.
  // The residual may be out itself: each element is read by the thread that
  // then writes it.
  const Span out = span(d->out_dev, d->m, d->n, d->ldo);
  const bool in_place = d->residual_dev == d->out_dev && d->ldr == d->ldo;
  if (meet(out, span(d->x_dev, d->m, d->k, d->ldx)) || meet(out, span(d->w_dev, d->n, d->k, d->ldw)) ||
      (d->w_up_dev && meet(out, span(d->w_up_dev, d->n, d->k, d->ldw_up))) ||
      (d->bias_dev && meet(out, span(d->bias_dev, 1, d->n, d->n))) ||
      (d->residual_dev && !in_place && meet(out, span(d->residual_dev, d->m, d->n, d->ldr))))
    return refuse(err, err_len, MOE_EINVAL, "%s: out overlaps an input (only residual may be out itself)", me);
  LinearArgs a{};
  a.x = static_cast<const uint16_t*>(d->x_dev);
  a.w = static_cast<const uint16_t*>(d->w_dev);
  a.w_up = static_cast<const uint16_t*>(d->w_up_dev);
  a.bias = static_cast<const uint16_t*>(d->bias_dev);
  a.res = static_cast<const uint16_t*>(d->residual_dev);
  a.out = static_cast<uint16_t*>(d->out_dev);
  a.ldx = d->ldx;
  a.ldw = d->ldw;
  a.ldwu = d->ldw_up;
  a.ldr = d->ldr;
  a.ldo = d->ldo;
  a.m = d->m;
  a.n = d->n;
  a.k = d->k;
  a.act = d->activation;
  const cudaError_t e = moe::dense::launch_generic(a, d->dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return refuse(err, err_len, MOE_ECUDA, "%s: %s", me, cudaGetErrorString(e));
  return MOE_OK;
}

}  // extern "C"
