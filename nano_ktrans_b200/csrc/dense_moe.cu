// dense_moe.cu — a whole mixture-of-experts layer on unquantised bf16 / fp16
// expert weights for a few tokens, in two kernels.
//
// The reference's MoE block (nano_ktrans/models/mixtral.py:212-218) with
// GPU-resident experts: router nn.Linear, routing
// (layers/hybrid_moe.py:3321-3329), the per-expert module loop with its host
// reads of the routed ids (:3501-3533) or the batch-1 stacked bmm
// (:3442-3500), weighted sum, shared expert, and the decoder layer's residual.
//
//   l     = round(x Wr^T);  ids, w = top-k of l as the router kernel ranks it
//   h_te  = w_te * silu(x_t G_e^T) * (x_t U_e^T)            (fp32)
//   out_t = round(r_t + sum_e D_e h_te + D_s h_ts),  h_ts weighted by sigmoid(x_t . g_s)
//
// With the weight inside h the weighted sum over experts is part of the down
// projection's K loop: out = [D_e1 | D_e2 | ...] [h_e1; h_e2; ...], one
// accumulator per output.  h is kept as hi + lo, two values of the layer's
// type (hi = round(h), lo = round(h - hi): relative error 2^-16 for bf16,
// 2^-22 for fp16), each a token column of its own: the tensor cores have room,
// since the kernel is bound by reading each routed expert's weights once.
//
// dense_router_kernel: one block per expert, logits of all tokens; one more
// block for the shared expert's gate; zeroes the grid barrier of the call.
// dense_moe_kernel: one block per SM, cooperative.  Every block routes all
// tokens by itself (one warp a token) and lists the routed experts in
// ascending order; then the gate / up rows of all of them, and after one grid
// barrier the output rows, are split evenly over the blocks by rows and
// streamed (dense_stream.cuh).  The first down-projection steps are loaded
// before the barrier, so its latency passes with 128 KB per SM in flight.
#include "async_copy.cuh"
#include "dense_stream.cuh"
#include "kernels.h"

namespace moe {
namespace dense {

__device__ int g_dense_status;  // kStatus* bits of this device's dense calls since the last read

constexpr int kRouterThreads = 256;

// Block e < num_experts: logits[t][e]; block num_experts: the shared gate.
template <typename T>
__global__ void __launch_bounds__(kRouterThreads) dense_router_kernel(const __grid_constant__ MoeArgs a) {
  __shared__ float part[kRouterThreads / 32][kMoeTokens];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x == 0 && tid == 0) *a.bar = 0;
  const int e = a.router_w ? blockIdx.x : a.experts;  // without a projection the only block is the gate's
  const uint16_t* w = e < a.experts ? a.router_w + static_cast<int64_t>(e) * a.hidden : a.shared_gate_vec;
  if (w == nullptr) return;
  float acc[kMoeTokens];
#pragma unroll
  for (int t = 0; t < kMoeTokens; ++t) acc[t] = 0.0f;
  for (int k = tid * 8; k < a.hidden; k += kRouterThreads * 8) {
    const uint4 wq = *reinterpret_cast<const uint4*>(w + k);
    const uint32_t wv[4] = {wq.x, wq.y, wq.z, wq.w};
#pragma unroll
    for (int t0 = 0; t0 < kMoeTokens; t0 += 4) {
      if (t0 >= a.tokens) break;
      uint4 xq[4];  // four tokens' loads under way at once
#pragma unroll
      for (int i = 0; i < 4; ++i) xq[i] = *reinterpret_cast<const uint4*>(a.x + min(t0 + i, a.tokens - 1) * a.ldx + k);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t xv[4] = {xq[i].x, xq[i].y, xq[i].z, xq[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 p = T::unpack(wv[j]), q = T::unpack(xv[j]);
          acc[t0 + i] = fmaf(p.x, q.x, acc[t0 + i]);
          acc[t0 + i] = fmaf(p.y, q.y, acc[t0 + i]);
        }
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kMoeTokens; ++t)
    if (t < a.tokens) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) acc[t] += __shfl_xor_sync(kFullMask, acc[t], off);
      if (lane == 0) part[warp][t] = acc[t];
    }
  __syncthreads();
  if (tid < a.tokens) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kRouterThreads / 32; ++i) v += part[i][tid];
    if (e < a.experts) a.logits[tid * a.experts + e] = T::from_f32(v);
    else a.shared_open[tid] = sigmoid_f32(v);
  }
}

// Order-preserving 16-bit image of a 16-bit float: NaN on top, -0 equal to +0.
template <typename T>
MOE_DEV uint32_t key16(float v) {
  if (isnan(v)) return 0xffffu;
  uint32_t b = T::from_f32(v);
  if (b == 0x8000u) b = 0;
  return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
}
template <typename T>
MOE_DEV float key16_value(uint32_t k) {
  return T::to_f32(static_cast<uint16_t>((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu)));
}

// One warp routes one token: lane j < top_k returns the j-th pick.  keys: this
// warp's scratch of `E` words.  Values are rounded to the layer's type before
// they are ranked, equal ones go to the lowest expert.
template <typename T>
MOE_DEV void route_warp(const uint16_t* row, const MoeArgs& a, uint32_t* keys, int& id, float& wt) {
  const int lane = threadIdx.x & 31, E = a.experts;
  float m = -INFINITY, s = 0.0f;
  if (a.use_softmax) {
    for (int e = lane; e < E; e += 32) {
      const float v = T::to_f32(__ldcg(row + e));
      keys[e] = __float_as_uint(v);
      m = fmaxf(m, v);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, off));
    for (int e = lane; e < E; e += 32) {
      const float p = expf(__uint_as_float(keys[e]) - m);
      keys[e] = __float_as_uint(p);
      s += p;
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(kFullMask, s, off);
    for (int e = lane; e < E; e += 32)
      keys[e] = (key16<T>(__uint_as_float(keys[e]) / s) << 16) | static_cast<uint32_t>(0xffff - e);
  } else {
    for (int e = lane; e < E; e += 32)
      keys[e] = (key16<T>(T::to_f32(__ldcg(row + e))) << 16) | static_cast<uint32_t>(0xffff - e);
  }
  float val = 0.0f, sum = 0.0f, v0 = 0.0f, exsum = 0.0f;
  id = -1;
  for (int j = 0; j < a.top_k; ++j) {
    uint32_t best = 0;
    for (int e = lane; e < E; e += 32) best = max(best, keys[e]);
    best = __reduce_max_sync(kFullMask, best);
    const int e = 0xffff - static_cast<int>(best & 0xffffu);
    if ((e & 31) == lane) keys[e] = 0;  // valid keys are never 0; each lane reads back only its own words
    const float v = key16_value<T>(best >> 16);
    if (lane == j) {
      val = v;
      id = e;
    }
    sum += v;
    if (j == 0) v0 = v;
    if (!a.use_softmax) exsum += expf(v - v0);
  }
  if (a.use_softmax)
    wt = a.renorm ? val / T::to_f32(T::from_f32(sum)) : val;
  else
    wt = expf(val - v0) / exsum;
  wt = T::to_f32(T::from_f32(wt));
}

// Routing tables of a call, in shared memory.
struct Tables {
  int16_t pair[kMoePairs][kMoeTokens];  // [active expert][token]: t * top_k + slot, -1 when not routed there
  float weight[kMoePairs][kMoeTokens];
  int active[kMoePairs];                // routed experts, ascending
  int id[kMoeTokens][kMoeTopK];
  float w[kMoeTokens][kMoeTopK];
  int n_active;
  int ok;
};

// Gate and up rows of the routed experts, then of the shared expert, as one
// list of rows; `lo` to `hi` are this block's.  Tile i is the list's group of
// 8 rows number lo / 8 + i (a group never spans two experts: their sizes are
// multiples of 16), rows outside the block's range masked.
template <int NT>
struct GateUpSrc {
  static constexpr bool kWhole = false;
  struct Tile {
    const uint16_t *g, *u;  // this lane's first gate and up row
    bool first, second;     // whether that row and the one 4 below are this block's
  };
  struct Step {
    int k;
  };
  const MoeArgs& a;
  const Tables& tb;
  int lo, hi, routed, q, t8;
  const uint16_t* xrow[NT];
  MOE_DEV GateUpSrc(const MoeArgs& args, const Tables& tables, int lo_, int hi_)
      : a(args), tb(tables), lo(lo_), hi(hi_), routed(tables.n_active * args.inter) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
    q = lane >> 3;
    t8 = 8 * (lane & 3);
#pragma unroll
    for (int j = 0; j < NT; ++j) xrow[j] = 8 * j + g < a.tokens ? a.x + (8 * j + g) * a.ldx + t8 : nullptr;
  }
  MOE_DEV int halves() const { return (a.hidden + 31) / 32; }
  MOE_DEV const uint16_t* any() const { return a.gate; }
  MOE_DEV Tile tile(int i) const {
    const int v0 = (lo / 8 + i) * 8, v = v0 + q;
    Tile t{a.gate, a.up, v >= lo && v < hi, v + 4 >= lo && v + 4 < hi};
    if (v0 < routed) {
      const int s = v0 / a.inter;
      const int64_t at = (static_cast<int64_t>(tb.active[s]) * a.inter + (v - s * a.inter)) * a.hidden;
      t.g = a.gate + at;
      t.u = a.up + at;
    } else {
      const int64_t at = static_cast<int64_t>(v - routed) * a.hidden;
      t.g = a.shared_gate + at;
      t.u = a.shared_up + at;
    }
    return t;
  }
  MOE_DEV Step step(int half) const { return {32 * half}; }
  MOE_DEV void row(const Tile& t, const Step& s, int i, const uint16_t*& p, int& n) const {
    n = a.hidden - s.k;
    p = ((i & 1) ? t.second : t.first) ? (i < 2 ? t.g : t.u) + (i & 1) * 4 * a.hidden + s.k : nullptr;
  }
  MOE_DEV void tokens(const Step& s, int j, uint4& x0, uint4& x1) const {
    const uint4 z = make_uint4(0, 0, 0, 0);
    x0 = xrow[j] != nullptr && s.k + t8 < a.hidden ? ld_tokens(xrow[j] + s.k) : z;
    x1 = xrow[j] != nullptr && s.k + 32 + t8 < a.hidden ? ld_tokens(xrow[j] + s.k + 32) : z;
  }
};

// Output rows [r0, r1); K runs over the routed experts' h, then the shared
// expert's.  Columns: hi of token c for c < half, then lo of token c - half.
template <int NT>
struct DownSrc {
  static constexpr bool kWhole = true;  // a step of 64 elements lies in one expert
  static constexpr int kHalf = 4 * NT;
  struct Tile {
    int row, left;  // this lane's first row, rows from there to the block's end
  };
  struct Step {
    const uint16_t* w;  // row 0 of the expert at the step's first element
    int ld, k, slot;    // row length, place in the row, place in the active list (-1: shared)
  };
  const MoeArgs& a;
  const Tables& tb;
  int r0, r1, ue, routed_units, q, g, t8;
  MOE_DEV DownSrc(const MoeArgs& args, const Tables& tables, int lo, int hi) : a(args), tb(tables), r0(lo), r1(hi) {
    const int lane = threadIdx.x & 31;
    q = lane >> 3;
    g = lane >> 2;
    t8 = 8 * (lane & 3);
    ue = (a.inter + 63) / 64;
    routed_units = tables.n_active * ue;
  }
  MOE_DEV int halves() const { return 2 * (routed_units + (a.shared_inter + 63) / 64); }
  MOE_DEV const uint16_t* any() const { return a.down; }
  MOE_DEV Tile tile(int i) const { return {r0 + 16 * i + q, r1 - (r0 + 16 * i + q)}; }
  MOE_DEV Step step(int half) const {
    const int unit = half / 2;
    if (unit < routed_units) {
      const int s = unit / ue, k = (unit - s * ue) * 64;
      return {a.down + static_cast<int64_t>(tb.active[s]) * a.hidden * a.inter + k, a.inter, k, s};
    }
    const int k = (unit - routed_units) * 64;
    return {a.shared_down + k, a.shared_inter, k, -1};
  }
  MOE_DEV void row(const Tile& t, const Step& s, int i, const uint16_t*& p, int& n) const {
    n = s.ld - s.k;
    p = t.left > 4 * i ? s.w + static_cast<int64_t>(t.row + 4 * i) * s.ld : nullptr;
  }
  MOE_DEV void tokens(const Step& s, int j, uint4& x0, uint4& x1) const {
    const int col = 8 * j + g, part = col >= kHalf ? 1 : 0, tok = col - part * kHalf, k = s.k + t8;
    int pair = -1;
    if (tok < a.tokens) pair = s.slot < 0 ? tok : tb.pair[s.slot][tok];
    const uint16_t* p = (s.slot < 0 ? a.h_shared : a.h) + static_cast<int64_t>(2 * pair + part) * s.ld + k;
    const uint4 z = make_uint4(0, 0, 0, 0);
    x0 = pair >= 0 && k < s.ld ? ld_l2(p) : z;
    x1 = pair >= 0 && k + 32 < s.ld ? ld_l2(p + 32) : z;
  }
};

// h = hi + lo in the layer's type.  An h beyond fp16's range stays infinite.
template <typename T>
MOE_DEV void store_split(uint16_t* hi, uint16_t* lo, float h) {
  const uint16_t b = T::from_f32(h);
  const float rest = h - T::to_f32(b);
  *hi = b;
  *lo = T::from_f32(isfinite(rest) ? rest : 0.0f);
}

// NT column tiles hold the tokens of the gate / up phase, ND those of the down phase (hi and lo).
template <typename T, int NT, int ND>
__global__ void __launch_bounds__(kSThreads, 1) dense_moe_kernel(const __grid_constant__ MoeArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Tables tb;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- routing, in every block ----
  uint32_t* keys = reinterpret_cast<uint32_t*>(smem);  // [16][E] words, then used[E] bytes: before the ring is in use
  uint8_t* used = reinterpret_cast<uint8_t*>(keys + kMoeTokens * a.experts);
  for (int i = tid; i < a.experts; i += kSThreads) used[i] = 0;
  for (int i = tid; i < kMoePairs * kMoeTokens; i += kSThreads) {
    (&tb.pair[0][0])[i] = -1;
    (&tb.weight[0][0])[i] = 0.0f;
  }
  __syncthreads();
  if (warp < a.tokens) {
    int id = -1;
    float wt = 0.0f;
    if (a.ids_in == nullptr) {
      route_warp<T>(a.logits + warp * a.experts, a, keys + warp * a.experts, id, wt);
    } else if (lane < a.top_k) {
      const int64_t given = a.ids_in[warp * a.top_k + lane];
      wt = T::to_f32(a.w_in[warp * a.top_k + lane]);
      id = given >= 0 && given < a.experts ? static_cast<int>(given) : -1;
      if (given >= a.experts && blockIdx.x == 0) atomicOr(&g_dense_status, kStatusBadExpertId);
    }
    if (lane < a.top_k) {
      if (blockIdx.x == 0 && a.ids_in == nullptr) {
        if (a.ids_out) a.ids_out[warp * a.top_k + lane] = id;
        if (a.w_out) a.w_out[warp * a.top_k + lane] = T::from_f32(wt);
      }
      if (id >= 0 && a.mask != nullptr && a.mask[id] == 0) id = -1;
      if (id >= 0) used[id] = 1;
      tb.id[warp][lane] = id;
      tb.w[warp][lane] = wt;
    }
  }
  __syncthreads();
  int16_t* slot = reinterpret_cast<int16_t*>(keys);  // [E] place of an expert in the active list
  if (warp == 0) {
    int n = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const bool on = e0 + lane < a.experts && used[e0 + lane] != 0;
      const uint32_t b = __ballot_sync(kFullMask, on);
      if (on) {
        const int s = n + __popc(b & ((1u << lane) - 1u));
        tb.active[s] = e0 + lane;
        slot[e0 + lane] = static_cast<int16_t>(s);
      }
      n += __popc(b);
    }
    if (lane == 0) tb.n_active = n;
    __syncwarp();
    if (lane < a.tokens)
      for (int j = 0; j < a.top_k; ++j) {  // an expert given twice for a token counts with both weights
        const int id = tb.id[lane][j];
        if (id < 0) continue;
        const int s = slot[id];
        if (tb.pair[s][lane] < 0) tb.pair[s][lane] = static_cast<int16_t>(lane * a.top_k + j);
        tb.weight[s][lane] += tb.w[lane][j];
      }
  }
  __syncthreads();

  // ---- h = w silu(gate) up ----
  const int64_t rows = static_cast<int64_t>(tb.n_active) * a.inter + a.shared_inter;
  const int lo = static_cast<int>(rows * blockIdx.x / gridDim.x), hi = static_cast<int>(rows * (blockIdx.x + 1) / gridDim.x);
  {
    const GateUpSrc<NT> src(a, tb, lo, hi);
    const int tiles = hi > lo ? (hi + 7) / 8 - lo / 8 : 0;
    Streamer<T, NT, 8, GateUpSrc<NT>> s(src, smem);
    s.prologue(tiles);
    s.run(a.tokens, [&](int tile, int row, int col, auto sum) {
      const int v0 = (lo / 8 + tile) * 8, v = v0 + row;
      if (v < lo || v >= hi) return;
      if (v0 < src.routed) {
        const int e = v0 / a.inter, pair = tb.pair[e][col];
        if (pair < 0) return;
        const float h = tb.weight[e][col] * (silu_f32(sum(row, col)) * sum(row + 8, col));
        uint16_t* p = a.h + static_cast<int64_t>(2 * pair) * a.inter + (v - e * a.inter);
        store_split<T>(p, p + a.inter, h);
      } else {
        const float h = __ldcg(a.shared_open + col) * (silu_f32(sum(row, col)) * sum(row + 8, col));
        uint16_t* p = a.h_shared + static_cast<int64_t>(2 * col) * a.shared_inter + (v - src.routed);
        store_split<T>(p, p + a.shared_inter, h);
      }
    });
  }

  // ---- out = r + sum over experts of D h ----
  const int r0 = static_cast<int>(static_cast<int64_t>(a.hidden) * blockIdx.x / gridDim.x);
  const int r1 = static_cast<int>(static_cast<int64_t>(a.hidden) * (blockIdx.x + 1) / gridDim.x);
  const DownSrc<ND> src(a, tb, r0, r1);
  const bool none = src.halves() == 0;  // every expert masked and no shared expert
  Streamer<T, ND, 16, DownSrc<ND>> s(src, smem);
  s.prologue(none ? 0 : (r1 - r0 + 15) / 16);  // weights only: they do not wait for h
  if (!ac::grid_sync_zeroed(a.bar, &tb.ok)) {
    if (tid == 0) atomicOr(&g_dense_status, kStatusTimeout);
    return;
  }
  auto store = [&](int n, int col, float v) {
    if (a.res) v += T::to_f32(a.res[col * a.ldr + n]);
    a.out[col * a.ldo + n] = T::from_f32(v);
  };
  if (none) {
    for (int i = tid; i < (r1 - r0) * a.tokens; i += kSThreads) store(r0 + i % (r1 - r0), i / (r1 - r0), 0.0f);
    return;
  }
  s.run(a.tokens, [&](int tile, int row, int col, auto sum) {
    const int n = r0 + 16 * tile + row;
    if (n < r1) store(n, col, sum(row, col) + sum(row, col + 4 * ND));
  });
}

template <typename T, int NT, int ND>
static cudaError_t moe_main(const MoeArgs& a, int sms, cudaStream_t st) {
  const void* kern = reinterpret_cast<const void*>(dense_moe_kernel<T, NT, ND>);
  constexpr size_t smem = kStreamBytes;
  static_assert((sizeof(uint32_t) * kMoeTokens + 1) * kMoeExperts <= smem, "routing scratch");
  if (!ensure_dynamic_smem(kern, smem, kSThreads)) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(sms);
  cfg.blockDim = dim3(kSThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, dense_moe_kernel<T, NT, ND>, a);
}

template <typename T>
static cudaError_t moe_both(const MoeArgs& a, int sms, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.router_w ? a.experts + (a.shared_gate_vec ? 1 : 0) : 1);
  cfg.blockDim = dim3(kRouterThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, dense_router_kernel<T>, a);
  if (e != cudaSuccess) return e;
  if (a.tokens <= 4) return moe_main<T, 1, 1>(a, sms, st);
  if (a.tokens <= 8) return moe_main<T, 1, 2>(a, sms, st);
  return moe_main<T, 2, 4>(a, sms, st);
}

cudaError_t launch_dense_moe(const MoeArgs& a, int dtype, int sms, cudaStream_t st) {
  return dtype == MOE_DTYPE_FP16 ? moe_both<Fp16>(a, sms, st) : moe_both<Bf16>(a, sms, st);
}

cudaError_t read_dense_status(int* status, cudaStream_t st) {
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, g_dense_status);
  if (e == cudaSuccess) e = cudaMemcpyAsync(status, p, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaMemsetAsync(p, 0, sizeof(int), st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  return e;
}

}  // namespace dense
}  // namespace moe
