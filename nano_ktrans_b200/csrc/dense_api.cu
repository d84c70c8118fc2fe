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

// `rows` rows of `cols` 16-bit elements, `ld` elements apart: bytes [lo, hi) hold
// them, in pieces of `row` bytes `step` apart.
struct Span {
  uintptr_t lo, hi;
  uintptr_t row, step;  // step 0: one piece
};
Span span(const void* p, int64_t rows, int64_t cols, int64_t ld) {
  const uintptr_t b = reinterpret_cast<uintptr_t>(p);
  return {b, rows > 0 ? b + 2 * static_cast<uintptr_t>((rows - 1) * ld + cols) : b, 2 * static_cast<uintptr_t>(cols),
          rows > 1 ? 2 * static_cast<uintptr_t>(ld) : 0};
}
// Whether they have a byte in common.  Two column ranges of one buffer have not,
// though each lies between the other's first and last byte; rows of two different
// steps are taken to meet where their whole extents do.
bool meet(const Span& a, const Span& b) {
  if (!(a.lo < b.hi && b.lo < a.hi)) return false;
  const uintptr_t step = a.step ? a.step : b.step;
  if (step == 0 || (a.step && b.step && a.step != b.step)) return true;
  // where b's pieces start between two of a's: they fit if they end before the next one
  const uintptr_t off = b.lo >= a.lo ? (b.lo - a.lo) % step : (step - (a.lo - b.lo) % step) % step;
  return off < a.row || off + b.row > step;
}

int sm_count(int* device = nullptr) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (device != nullptr) *device = dev;
  return cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? sms : 0;
}

// A few tokens are bound by the weights' bytes (streaming kernel); more go to
// the tensor-core GEMMs (NONE here: which of them goes by their plans).  Rows that
// no 16-byte load can take, to the generic kernel.
int kernel_of(const LinearArgs& a) {
  if (!moe::dense::wide_rows(a)) return MOE_LINEAR_GENERIC;
  return a.m <= moe::dense::kStreamTokens ? MOE_LINEAR_STREAM : MOE_LINEAR_NONE;
}

cudaError_t launch_linear(const LinearArgs& a, int dtype, cudaStream_t st) {
  int dev = 0;
  const int sms = sm_count(&dev);
  if (sms < 1) return cudaErrorInvalidDevice;
  switch (kernel_of(a)) {
    case MOE_LINEAR_GENERIC: return moe::dense::launch_generic(a, dtype, st);
    case MOE_LINEAR_STREAM: return moe::dense::launch_stream_linear(a, dtype, sms, st);
    default: return moe::dense::launch_gemm(a, dtype, dev, sms, st);
  }
}

constexpr int kB200Sms = 148;  // for the checks of a call on a host without a device

// The description of a projection, checked; what it says, in `a`.
int read_linear(const char* me, const moe_linear_desc* d, LinearArgs& a, char* err, size_t err_len) {
  if (d == nullptr) return refuse(err, err_len, MOE_EINVAL, "%s: null argument", me);
  if (d->dtype != MOE_DTYPE_BF16 && d->dtype != MOE_DTYPE_FP16)
    return refuse(err, err_len, MOE_EINVAL, "%s: dtype must be MOE_DTYPE_BF16 or MOE_DTYPE_FP16", me);
  if (d->activation < MOE_ACT_NONE || d->activation > MOE_ACT_RELU)
    return refuse(err, err_len, MOE_EINVAL, "%s: unknown activation %d", me, d->activation);
  if (d->m < 0 || d->n < 1 || d->k < 1)
    return refuse(err, err_len, MOE_EINVAL, "%s: m must be >= 0, n and k >= 1 (got %d, %d, %d)", me, d->m, d->n, d->k);
  // a tile's last row and column number, up to 255 beyond the tensor's, have to fit 32 bits
  const int32_t most = INT32_MAX - 255;
  if (d->m > most || d->n > most || d->k > most)
    return refuse(err, err_len, MOE_EINVAL, "%s: m, n and k are at most 2^31 - 256 (got %d, %d, %d)", me, d->m, d->n, d->k);
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
  return MOE_OK;
}

}  // namespace

extern "C" {

int moe_linear(const moe_linear_desc* d, void* stream, char* err, size_t err_len) {
  LinearArgs a{};
  const int rc = read_linear("moe_linear", d, a, err, err_len);
  if (rc != MOE_OK || a.m == 0) return rc;
  const cudaError_t e = launch_linear(a, d->dtype, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return refuse(err, err_len, MOE_ECUDA, "moe_linear: %s", cudaGetErrorString(e));
  return MOE_OK;
}

int moe_linear_query(const moe_linear_desc* d, moe_linear_plan* plan, char* err, size_t err_len) {
  if (plan == nullptr) return refuse(err, err_len, MOE_EINVAL, "moe_linear_query: null argument");
  LinearArgs a{};
  const int rc = read_linear("moe_linear_query", d, a, err, err_len);
  if (rc != MOE_OK) return rc;
  *plan = {};
  if (a.m == 0) return MOE_OK;
  int dev = -1;
  int sms = sm_count(&dev);
  if (sms < 1) {
    cudaGetLastError();
    dev = -1;
    sms = kB200Sms;
  }
  plan->kernel = kernel_of(a);
  if (plan->kernel == MOE_LINEAR_NONE) moe::dense::plan_gemm(a, dev, sms, *plan);
  return MOE_OK;
}

namespace {

struct MoeSpace {
  size_t bar, open, logits, partial, bytes;
};
MoeSpace moe_space(const moe_dense_desc& d, int sms) {
  const auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
  const size_t t = d.num_tokens;
  moe::dense::MoeArgs a{};
  a.tokens = d.num_tokens;
  a.experts = d.num_experts;
  a.top_k = d.top_k;
  a.inter = d.inter_size;
  a.shared_inter = d.shared_inter;
  MoeSpace s{};
  s.bar = 0;
  s.open = 256;
  s.logits = s.open + up(4 * t);
  s.partial = s.logits + up(2 * t * d.num_experts);
  s.bytes = s.partial + (t ? 4 * t * d.hidden_size * static_cast<size_t>(moe::dense::moe_pieces(a, sms)) : 0);
  return s;
}

// nullptr, or what is wrong with the layer's description.
const char* check_layer(const moe_dense_desc& d) {
  if (d.dtype != MOE_DTYPE_BF16 && d.dtype != MOE_DTYPE_FP16) return "dtype must be MOE_DTYPE_BF16 or MOE_DTYPE_FP16";
  if (d.num_experts < 1 || d.num_experts > moe::dense::kMoeExperts) return "num_experts must be in [1, 1024]";
  if (d.top_k < 1 || d.top_k > moe::dense::kMoeTopK) return "top_k must be in [1, 16]";
  const int32_t big = 1 << 16;
  if (d.hidden_size < 16 || d.hidden_size % 16 || d.hidden_size > big) return "hidden_size must be a positive multiple of 16";
  if (d.inter_size < 16 || d.inter_size % 16 || d.inter_size > big) return "inter_size must be a positive multiple of 16";
  if (d.shared_inter < 0 || d.shared_inter % 16 || d.shared_inter > big) return "shared_inter must be a multiple of 16";
  if (d.num_tokens < 0) return "negative token count";
  return nullptr;
}

}  // namespace

int moe_dense_workspace(const moe_dense_desc* d, int64_t* bytes, char* err, size_t err_len) {
  if (d == nullptr || bytes == nullptr) return refuse(err, err_len, MOE_EINVAL, "moe_dense_workspace: null argument");
  if (const char* why = check_layer(*d)) return refuse(err, err_len, MOE_EINVAL, "moe_dense_workspace: %s", why);
  if (d->num_tokens > MOE_DENSE_MAX_TOKENS)
    return refuse(err, err_len, MOE_ERANGE, "moe_dense_workspace: %d tokens, at most %d", d->num_tokens, MOE_DENSE_MAX_TOKENS);
  const int sms = sm_count();
  *bytes = static_cast<int64_t>(moe_space(*d, sms > 0 ? sms : kB200Sms).bytes);
  return MOE_OK;
}

int moe_dense_forward(const moe_dense_desc* d, void* stream, char* err, size_t err_len) {
  const char* me = "moe_dense_forward";
  if (d == nullptr) return refuse(err, err_len, MOE_EINVAL, "%s: null argument", me);
  if (const char* why = check_layer(*d)) return refuse(err, err_len, MOE_EINVAL, "%s: %s", me, why);
  if (d->num_tokens > MOE_DENSE_MAX_TOKENS)
    return refuse(err, err_len, MOE_ERANGE, "%s: %d tokens, at most %d", me, d->num_tokens, MOE_DENSE_MAX_TOKENS);
  if (d->num_tokens == 0) return MOE_OK;
  const bool shared = d->shared_inter > 0 && d->add_shared;
  const int64_t t = d->num_tokens, E = d->num_experts, H = d->hidden_size, I = d->inter_size;
  const int64_t S = shared ? d->shared_inter : 0;
  const void* need[] = {d->gate_dev, d->up_dev, d->down_dev, d->x_dev, d->out_dev, d->workspace_dev};
  for (const void* p : need)
    if (p == nullptr) return refuse(err, err_len, MOE_EINVAL, "%s: null device pointer", me);
  if (shared && (!d->shared_gate_dev || !d->shared_up_dev || !d->shared_down_dev || !d->shared_gate_vec_dev))
    return refuse(err, err_len, MOE_EINVAL, "%s: null shared-expert pointer", me);
  const bool given = d->ids_dev != nullptr || d->weights_dev != nullptr;
  if (given && (d->ids_dev == nullptr || d->weights_dev == nullptr || d->router_w_dev || d->logits_dev))
    return refuse(err, err_len, MOE_EINVAL, "%s: given routing needs ids and weights, and no router or logits", me);
  if (!given && d->router_w_dev == nullptr && d->logits_dev == nullptr)
    return refuse(err, err_len, MOE_EINVAL, "%s: no routing: router weights, logits or ids", me);
  if (!given && d->top_k > E) return refuse(err, err_len, MOE_EINVAL, "%s: top_k above num_experts", me);
  if (given && (d->ids_out_dev || d->weights_out_dev))
    return refuse(err, err_len, MOE_EINVAL, "%s: given routing is not written out again", me);
  const void* wide[] = {d->gate_dev, d->up_dev, d->down_dev, d->x_dev, d->router_w_dev,
                        shared ? d->shared_gate_dev : nullptr, shared ? d->shared_up_dev : nullptr,
                        shared ? d->shared_down_dev : nullptr, shared ? d->shared_gate_vec_dev : nullptr};
  for (const void* p : wide)
    if (reinterpret_cast<uintptr_t>(p) % 16)
      return refuse(err, err_len, MOE_EINVAL, "%s: x and the weights must start on 16-byte boundaries", me);
  if (t > 1 && d->ldx % 8) return refuse(err, err_len, MOE_EINVAL, "%s: the rows of x must lie on 16-byte boundaries", me);
  const void* even[] = {d->logits_dev, d->weights_dev, d->residual_dev, d->out_dev, d->weights_out_dev};
  for (const void* p : even)
    if (reinterpret_cast<uintptr_t>(p) % 2) return refuse(err, err_len, MOE_EINVAL, "%s: pointers must be 2-byte aligned", me);
  if (reinterpret_cast<uintptr_t>(d->ids_dev) % 8 || reinterpret_cast<uintptr_t>(d->ids_out_dev) % 8)
    return refuse(err, err_len, MOE_EINVAL, "%s: ids must be 8-byte aligned", me);
  if (d->ldx < H || d->ldo < H || (d->residual_dev && d->ldr < H))
    return refuse(err, err_len, MOE_EINVAL, "%s: the rows of x, residual and out must be at least hidden_size apart", me);
  const int sms = sm_count();
  const MoeSpace ws = moe_space(*d, sms > 0 ? sms : kB200Sms);
  if (reinterpret_cast<uintptr_t>(d->workspace_dev) % 256 || d->workspace_bytes < static_cast<int64_t>(ws.bytes))
    return refuse(err, err_len, MOE_EINVAL, "%s: the workspace must be 256-byte aligned and hold %lld bytes", me,
                  static_cast<long long>(ws.bytes));
  // What is written: out, the routing, the logits, the workspace.  Nothing of
  // it may meet anything that is read, nor each other; out may be x (which is
  // read no more once the first output is stored) or residual.
  const auto whole = [](const void* p, int64_t n, int64_t bytes_each) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(p);
    const uintptr_t size = static_cast<uintptr_t>(n * bytes_each);
    return p ? Span{b, b + size, size, 0} : Span{};
  };
  const Span x = span(d->x_dev, t, H, d->ldx), out = span(d->out_dev, t, H, d->ldo);
  const Span res = d->residual_dev ? span(d->residual_dev, t, H, d->ldr) : Span{};
  const Span lg = whole(d->logits_dev, t * E, 2);
  const Span written[] = {out, whole(d->workspace_dev, ws.bytes, 1), whole(d->ids_out_dev, t * d->top_k, 8),
                          whole(d->weights_out_dev, t * d->top_k, 2), d->router_w_dev ? lg : Span{}};
  const Span read[] = {x, res, whole(d->gate_dev, E * I * H, 2), whole(d->up_dev, E * I * H, 2),
                       whole(d->down_dev, E * I * H, 2), whole(shared ? d->shared_gate_dev : nullptr, S * H, 2),
                       whole(shared ? d->shared_up_dev : nullptr, S * H, 2),
                       whole(shared ? d->shared_down_dev : nullptr, S * H, 2),
                       whole(shared ? d->shared_gate_vec_dev : nullptr, H, 2), whole(d->router_w_dev, E * H, 2),
                       d->router_w_dev ? Span{} : lg, whole(d->ids_dev, t * d->top_k, 8),
                       whole(d->weights_dev, t * d->top_k, 2), whole(d->offload_mask_dev, E, 1)};
  const bool on_x = d->out_dev == d->x_dev && (t == 1 || d->ldo == d->ldx);
  const bool on_res = d->out_dev == d->residual_dev && (t == 1 || d->ldo == d->ldr);
  for (int i = 0; i < 5; ++i) {
    for (int j = 0; j < 14; ++j)
      if (meet(written[i], read[j]) && !(i == 0 && ((j == 0 && on_x) || (j == 1 && on_res))))
        return refuse(err, err_len, MOE_EINVAL, "%s: an output overlaps an input (only x or residual may be out itself)", me);
    for (int j = 0; j < i; ++j)
      if (meet(written[i], written[j])) return refuse(err, err_len, MOE_EINVAL, "%s: two outputs overlap", me);
  }
  if (sms < 1) return refuse(err, err_len, MOE_ECUDA, "%s: no device", me);
  char* w = static_cast<char*>(d->workspace_dev);
  moe::dense::MoeArgs a{};
  a.x = static_cast<const uint16_t*>(d->x_dev);
  a.router_w = static_cast<const uint16_t*>(d->router_w_dev);
  a.logits = d->logits_dev ? static_cast<uint16_t*>(d->logits_dev) : reinterpret_cast<uint16_t*>(w + ws.logits);
  a.ids_in = d->ids_dev;
  a.w_in = static_cast<const uint16_t*>(d->weights_dev);
  a.mask = d->offload_mask_dev;
  a.gate = static_cast<const uint16_t*>(d->gate_dev);
  a.up = static_cast<const uint16_t*>(d->up_dev);
  a.down = static_cast<const uint16_t*>(d->down_dev);
  if (shared) {
    a.shared_gate = static_cast<const uint16_t*>(d->shared_gate_dev);
    a.shared_up = static_cast<const uint16_t*>(d->shared_up_dev);
    a.shared_down = static_cast<const uint16_t*>(d->shared_down_dev);
    a.shared_gate_vec = static_cast<const uint16_t*>(d->shared_gate_vec_dev);
  }
  a.res = static_cast<const uint16_t*>(d->residual_dev);
  a.out = static_cast<uint16_t*>(d->out_dev);
  a.ids_out = d->ids_out_dev;
  a.w_out = static_cast<uint16_t*>(d->weights_out_dev);
  a.bar = reinterpret_cast<unsigned long long*>(w + ws.bar);
  a.shared_open = reinterpret_cast<float*>(w + ws.open);
  a.partial = reinterpret_cast<float*>(w + ws.partial);
  a.ldx = d->ldx;
  a.ldr = d->ldr;
  a.ldo = d->ldo;
  a.tokens = d->num_tokens;
  a.experts = d->num_experts;
  a.top_k = d->top_k;
  a.hidden = d->hidden_size;
  a.inter = d->inter_size;
  a.shared_inter = static_cast<int>(S);
  a.use_softmax = d->router_use_softmax != 0;
  a.renorm = d->normalize_topk_prob != 0;
  const cudaError_t e = moe::dense::launch_dense_moe(a, d->dtype, sms, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return refuse(err, err_len, MOE_ECUDA, "%s: %s", me, cudaGetErrorString(e));
  return MOE_OK;
}

int moe_dense_read_status(int32_t* status, void* stream, char* err, size_t err_len) {
  if (status == nullptr) return refuse(err, err_len, MOE_EINVAL, "moe_dense_read_status: null argument");
  int v = 0;
  int g = 0;
  cudaError_t e = moe::dense::read_dense_status(&v, static_cast<cudaStream_t>(stream));
  if (e == cudaSuccess) e = moe::dense::read_gemm_status(&g, static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return refuse(err, err_len, MOE_ECUDA, "moe_dense_read_status: %s", cudaGetErrorString(e));
  *status = v | g;
  return MOE_OK;
}

}  // extern "C"
