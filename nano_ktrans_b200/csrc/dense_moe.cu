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
// dense_router_kernel: one block per expert, logits of all tokens; one more
// block for the shared expert's gate; zeroes the grid barrier of the call.
// dense_moe_kernel: one block per SM, cooperative.  Every block routes all
// tokens by itself (one warp a token) and lists the routed experts in
// ascending order.  Their intermediate rows (and the shared expert's), one
// after the other, are split evenly over the blocks, and a block does both
// halves of its rows' work: it streams their gate and up rows
// (dense_stream.cuh), keeps h in shared memory, and streams the down
// projection's columns of just these rows past it.  So h never leaves the SM
// and no block waits for another between the projections; a block's partial
// outputs (fp32, per expert piece and token) go to the workspace, and after one
// grid barrier every block adds up its share of the outputs over the pieces,
// in order (no atomics).  Splitting the down projection by output rows instead
// needs the barrier between the projections and all of h in every block, read
// from L2 step by step: 16 tokens, 128 x 768 experts, 190 us.
//
// h is kept as hi + lo, two values of the layer's type (hi = round(h), lo =
// round(h - hi): relative error 2^-16 for bf16, 2^-22 for fp16), each a column
// of its own: the tensor cores have room, since the kernel is bound by reading
// each routed expert's weights once.  bf16 has fp32's range.  fp16 has not: there
// h is first multiplied by a power of two that brings the largest |h| of a
// token's piece into [2^14, 2^15) and that the partial sums are divided by, so an
// h of any size is kept to 2^-22 of itself or 2^-39 of that largest one.
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

// One warp routes one token: lane j < top_k returns the j-th pick.  Values are
// rounded to the layer's type before they are ranked, equal ones go to the
// lowest expert.  EPL: experts per lane, in registers.
template <typename T, int EPL>
MOE_DEV void route_warp(const uint16_t* row, const MoeArgs& a, int& id, float& wt) {
  const int lane = threadIdx.x & 31, E = a.experts;
  float v[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) v[i] = i * 32 + lane < E ? T::to_f32(__ldcg(row + i * 32 + lane)) : -INFINITY;
  if (a.use_softmax) {
    float m = -INFINITY, s = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) m = fmaxf(m, v[i]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(kFullMask, m, off));
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      if (i * 32 + lane < E) {
        v[i] = expf(v[i] - m);
        s += v[i];
      }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(kFullMask, s, off);
#pragma unroll
    for (int i = 0; i < EPL; ++i) v[i] = v[i] / s;
  }
  // unique 32-bit keys, each lane's in descending order (valid keys are never 0)
  uint32_t key[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    key[i] = i * 32 + lane < E ? (key16<T>(v[i]) << 16) | static_cast<uint32_t>(0xffff - (i * 32 + lane)) : 0u;
#pragma unroll
  for (int p = 0; p < EPL - 1; ++p)
#pragma unroll
    for (int i = 0; i < EPL - 1 - p; ++i) {
      const uint32_t hi = max(key[i], key[i + 1]), lo = min(key[i], key[i + 1]);
      key[i] = hi;
      key[i + 1] = lo;
    }
  float val = 0.0f, sum = 0.0f, v0 = 0.0f, exsum = 0.0f;
  id = -1;
#pragma unroll 1
  for (int j = 0; j < a.top_k; ++j) {
    const uint32_t best = __reduce_max_sync(kFullMask, key[0]);
    if (key[0] == best) {
#pragma unroll
      for (int i = 0; i < EPL - 1; ++i) key[i] = key[i + 1];
      key[EPL - 1] = 0;
    }
    const float x = key16_value<T>(best >> 16);
    if (lane == j) {
      val = x;
      id = 0xffff - static_cast<int>(best & 0xffffu);
    }
    sum += x;
    if (j == 0) v0 = x;
    if (!a.use_softmax) exsum += expf(x - v0);
  }
  if (a.use_softmax)
    wt = a.renorm ? val / T::to_f32(T::from_f32(sum)) : val;
  else
    wt = expf(val - v0) / exsum;
  wt = T::to_f32(T::from_f32(wt));
}

// Routing of a call, in shared memory.
struct Tables {
  float weight[kMoePairs + 1][kMoeTokens];  // [place in the active list][i]: the expert's i-th token's weight,
  uint8_t list[kMoePairs + 1][kMoeTokens];  // and which token that is
  uint32_t tokens[kMoePairs + 1];           // tokens of an active expert, one bit each; the shared expert's come last
  int active[kMoePairs];                    // routed experts, ascending
  uint32_t used[kMoeExperts / 32];          // routed experts, one bit each
  int n_places[kMoeTokens];                 // a token's experts in ascending order: place in the active list,
  int place[kMoeTokens][kMoeTopK + 1];      // first range of its rows,
  int range[kMoeTokens][kMoeTopK + 1];
  int pieces[kMoeTokens][kMoeTopK + 2];     // and pieces of the experts before it
  // fp16: bits of the largest finite |h| of a range's [piece][i-th token of its expert].  Experts have 16 rows at least,
  // so a range of cap rows meets cap / 16 + 2 of them at most.
  uint32_t top[kHBytes / 64 + 2 * kMoeTokens];
  int n_active;
  int ok;
};

// How the intermediate rows are split: `groups` groups of 8 rows over `ranges`
// ranges, block b working on ranges [b * per_block, (b + 1) * per_block).
struct Split {
  uint32_t groups;
  int ranges, per_block;
  MOE_DEV Split(int64_t rows, int cap) : groups(static_cast<uint32_t>(rows / 8)) {
    const uint32_t blocks = gridDim.x, most = blocks * (cap / 8);
    per_block = groups > most ? static_cast<int>((groups + most - 1) / most) : 1;
    ranges = groups < blocks ? static_cast<int>(groups) : static_cast<int>(blocks) * per_block;  // none is empty
  }
  // a / b; the 64-bit division only where it takes one
  static MOE_DEV uint32_t quotient(uint64_t a, uint32_t b) {
    return (a >> 32) == 0 ? static_cast<uint32_t>(a) / b : static_cast<uint32_t>(a / b);
  }
  MOE_DEV int begin(int r) const { return static_cast<int>(8 * quotient(static_cast<uint64_t>(groups) * r, ranges)); }
  // range of the row (a multiple of 8)
  MOE_DEV int of_row(int row) const {
    return static_cast<int>(quotient(static_cast<uint64_t>(row / 8 + 1) * ranges + groups - 1, groups)) - 1;
  }
};

// Expert (place in the active list) of an intermediate row.
MOE_DEV int place_of(const MoeArgs& a, int row) { return static_cast<int>(__umul64hi(static_cast<uint64_t>(row), a.inter_inverse)); }

// Gate and up rows [lo, hi) of the list of intermediate rows (multiples of 8).
// Tile i is its i-th group of 8 (a group never spans two experts: their sizes
// are multiples of 16).  Column c is token list[c], or token c without a list.
struct GateUpSrc {
  struct Tile {
    const uint16_t *g, *u;  // this lane's first gate and up row
  };
  const MoeArgs& a;
  const Tables& tb;
  int lo, hi, routed, t8;
  const uint16_t* xrow;
  MOE_DEV GateUpSrc(const MoeArgs& args, const Tables& tables, int lo_, int hi_, const uint8_t* list, int cols)
      : a(args), tb(tables), lo(lo_), hi(hi_), routed(tables.n_active * args.inter) {
    const int lane = threadIdx.x & 31, g = lane >> 2;
    t8 = 8 * (lane & 3);
    xrow = g < cols ? a.x + (list != nullptr ? list[g] : g) * a.ldx + t8 : nullptr;
  }
  MOE_DEV int length() const { return a.hidden; }
  MOE_DEV int tiles() const { return (hi - lo) / 8; }
  MOE_DEV Tile tile(int i) const {
    const int v = lo + 8 * i, q = (threadIdx.x & 31) >> 3;
    if (v < routed) {
      const int s = place_of(a, v);
      const int64_t at = (static_cast<int64_t>(tb.active[s]) * a.inter + (v - s * a.inter) + q) * a.hidden;
      return {a.gate + at, a.up + at};
    }
    const int64_t at = static_cast<int64_t>(v - routed + q) * a.hidden;
    return {a.shared_gate + at, a.shared_up + at};
  }
  MOE_DEV void rows(const Tile& t, int k, const uint16_t* (&p)[4], uint32_t& valid) const {
    p[0] = t.g + k;
    p[1] = p[0] + 4 * a.hidden;
    p[2] = t.u + k;
    p[3] = p[2] + 4 * a.hidden;
    valid = 15u;
  }
  MOE_DEV void tokens(int k, bool two, int, uint4& x0, uint4& x1) const {
    const uint4 z = make_uint4(0, 0, 0, 0);
    x0 = xrow != nullptr && k + t8 < a.hidden ? ld_tokens(xrow + k) : z;
    x1 = two && xrow != nullptr && k + 32 + t8 < a.hidden ? ld_tokens(xrow + k + 32) : z;
  }
};

// Power of two that brings a largest |h| (its bits) into [2^14, 2^15), and its
// inverse.  Below 2^-111 the scale stays at 2^125: both are normal numbers then.
MOE_DEV float h_scale(uint32_t top) { return __uint_as_float((268u - max(top >> 23, 16u)) << 23); }
MOE_DEV float h_unscale(uint32_t top) { return __uint_as_float((max(top >> 23, 16u) - 14u) << 23); }

// The down projection's columns of rows [lo, hi), all output rows: every warp
// takes whole tiles of 16 output rows (tile w, w + 16, ...), RT at a time, over
// the K of one expert's piece after the other.  Column 2 i of the mma is hi and
// column 2 i + 1 lo of the expert's i-th token, so that one thread holds both
// sums of an output; of ND column tiles (4 tokens each) only those that the
// expert has tokens for are worked on.  The ring is the Streamer's.
template <typename T, int ND, int RT>
struct DownStreamer {
  static constexpr int D = kSlots, PD = D / RT;
  struct Piece {
    const uint16_t* w;  // row 0 at the piece's first column
    int ld, len, place, v;
  };
  const MoeArgs& a;
  const Tables& tb;
  const uint16_t* hs;  // [hi, lo][token of the expert][cap] from row lo on
  int lo, hi, routed, cap, range;
  uint32_t ring;
  int count;        // this warp's tiles
  Piece lp;         // next to load: piece, first tile of its group, step
  int lg, ls;

  MOE_DEV DownStreamer(const MoeArgs& args, const Tables& tables, unsigned char* smem, const uint16_t* h, int cap_, int range_,
                       int lo_, int hi_)
      : a(args), tb(tables), hs(h), lo(lo_), hi(hi_), routed(tables.n_active * args.inter), cap(cap_), range(range_) {
    const int warp = threadIdx.x >> 5, tiles = a.hidden / 16;
    ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + warp * (D * kStepBytes);
    count = warp < tiles ? (tiles - warp + kSW - 1) / kSW : 0;
  }
  MOE_DEV Piece piece(int v) const {
    if (v < routed) {
      const int s = place_of(a, v), off = v - s * a.inter;
      return {a.down + static_cast<int64_t>(tb.active[s]) * a.hidden * a.inter + off, a.inter, min(hi, (s + 1) * a.inter) - v,
              s, v};
    }
    return {a.shared_down + (v - routed), a.shared_inter, hi - v, tb.n_active, v};
  }
  MOE_DEV void load(int turn, int i) {
    if (lp.v < hi && lg + i < count) {
      const int lane = threadIdx.x & 31, c = lane & 7, row = lane >> 3;
      const uint32_t dst = ring + (turn * RT + i) * kStepBytes + row * 128 + ((c ^ ((row & 1) << 2)) << 4);
      const int r = 16 * ((threadIdx.x >> 5) + kSW * (lg + i)) + row, k = 64 * ls + 8 * c;
      const bool take = k < lp.len;
      const uint16_t* p = take ? lp.w + static_cast<int64_t>(r) * lp.ld + k : a.down;
      const int64_t four = take ? 4 * static_cast<int64_t>(lp.ld) : 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) copy16(dst + q * 512, p + q * four, take ? 16u : 0u);
    }
    copy_commit();
  }
  MOE_DEV void next_step() {
    if (64 * ++ls >= lp.len) {
      ls = 0;
      lg += RT;
      if (lg >= count) {
        lg = 0;
        const int v = lp.v + lp.len;
        if (v < hi) lp = piece(v);
        else lp.v = v;
      }
    }
  }
  MOE_DEV void prologue() {
    lg = ls = 0;
    if (count == 0 || lo >= hi) return;
    lp = piece(lo);
#pragma unroll
    for (int p = 0; p < PD; ++p) {
#pragma unroll
      for (int i = 0; i < RT; ++i) load(p, i);
      next_step();
    }
  }
  MOE_DEV void run() {
    if (count == 0) return;
    const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const uint32_t frag0 = g * 128 + ((t4 ^ ((g & 1) << 2)) << 4), frag1 = g * 128 + ((t4 ^ 4 ^ ((g & 1) << 2)) << 4);
    int turn = 0;
    const int first = lo < routed ? place_of(a, lo) : tb.n_active;  // place of the range's first piece
    for (int v = lo; v < hi;) {
      const Piece p = piece(v);
      const int n = __popc(tb.tokens[p.place]);  // the expert's tokens
      const uint16_t* hrow[ND];
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        const int i = 4 * j + (g >> 1);
        hrow[j] = i < n ? hs + ((g & 1) * a.tokens + i) * cap + (v - lo) + 8 * t4 : nullptr;
      }
      float* out = a.partial + (static_cast<int64_t>(range + p.place) * a.tokens + t4) * a.hidden + g;
      float back[ND];  // what the scale of the 4 j + t4-th token's h is undone by
#pragma unroll
      for (int j = 0; j < ND; ++j) {
        back[j] = 1.0f;
        if constexpr (!T::kBf16)
          if (4 * j + t4 < n) back[j] = h_unscale(tb.top[(p.place - first) * a.tokens + 4 * j + t4]);
      }
      for (int grp = 0; grp < count; grp += RT) {
        float acc[RT][ND][4];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < ND; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.0f;
#pragma unroll 1
        for (int k = 0; k < p.len; k += 64) {
          uint4 x[ND][2];
          const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < ND; ++j)
            if (4 * j < n) {
              x[j][0] = hrow[j] != nullptr && k + 8 * t4 < p.len ? *reinterpret_cast<const uint4*>(hrow[j] + k) : z;
              x[j][1] = hrow[j] != nullptr && k + 32 + 8 * t4 < p.len ? *reinterpret_cast<const uint4*>(hrow[j] + k + 32) : z;
            }
          constexpr int P = RT >= 2 ? 2 : 1;  // slots at a time, as in the Streamer
#pragma unroll
          for (int i = 0; i < RT; i += P) {
            copy_wait<D - P>();
            __syncwarp();
            uint4 a0[P], a1[P], b0[P], b1[P];
#pragma unroll
            for (int q = 0; q < P; ++q) {
              const uint32_t from = ring + (turn * RT + i + q) * kStepBytes;
              a0[q] = ld_shared(from + frag0);
              b0[q] = ld_shared(from + frag0 + 1024);
              a1[q] = ld_shared(from + frag1);
              b1[q] = ld_shared(from + frag1 + 1024);
            }
            // a slot past the warp's last tile holds other bytes: its sums are not stored
#pragma unroll
            for (int j = 0; j < ND; ++j)
              if (4 * j < n) {
#pragma unroll
                for (int q = 0; q < P; ++q) T::mma(acc[i + q][j], a0[q].x, b0[q].x, a0[q].y, b0[q].y, x[j][0].x, x[j][0].y);
#pragma unroll
                for (int q = 0; q < P; ++q) T::mma(acc[i + q][j], a0[q].z, b0[q].z, a0[q].w, b0[q].w, x[j][0].z, x[j][0].w);
#pragma unroll
                for (int q = 0; q < P; ++q) T::mma(acc[i + q][j], a1[q].x, b1[q].x, a1[q].y, b1[q].y, x[j][1].x, x[j][1].y);
#pragma unroll
                for (int q = 0; q < P; ++q) T::mma(acc[i + q][j], a1[q].z, b1[q].z, a1[q].w, b1[q].w, x[j][1].z, x[j][1].w);
              }
            __syncwarp();
#pragma unroll
            for (int q = 0; q < P; ++q) load(turn, i + q);
          }
          next_step();
          turn = turn + 1 == PD ? 0 : turn + 1;
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
          if (grp + i < count) {
            float* o = out + 16 * ((threadIdx.x >> 5) + kSW * (grp + i));
#pragma unroll
            for (int j = 0; j < ND; ++j)
              if (4 * j + t4 < n) {
                __stcg(o + static_cast<int64_t>(4 * j) * a.hidden, (acc[i][j][0] + acc[i][j][1]) * back[j]);
                __stcg(o + static_cast<int64_t>(4 * j) * a.hidden + 8, (acc[i][j][2] + acc[i][j][3]) * back[j]);
              }
          }
      }
      v += p.len;
    }
  }
};

// h = hi + lo in the layer's type; infinities and NaN stay what they are.
template <typename T>
MOE_DEV void store_split(uint16_t* hi, uint16_t* lo, float h) {
  const uint16_t b = T::from_f32(h);
  const float rest = h - T::to_f32(b);
  *hi = b;
  *lo = T::from_f32(isfinite(rest) ? rest : 0.0f);
}

// fp16: the fp32 values h [token of the expert][cap] of rows [lo, hi) become scaled
// hi [token][cap] and lo [token][cap] in the same bytes.  The whole block's, which
// holds all of h in registers between the two (13 values a thread).
template <typename T>
MOE_DEV void split_scaled(const MoeArgs& a, Tables& tb, float* hf, int cap, int lo, int hi) {
  constexpr int kEach = kHBytes / 4 / kSThreads;
  static_assert(kEach * 4 * kSThreads == kHBytes, "h is shared out evenly");
  const int routed = tb.n_active * a.inter, first = lo < routed ? place_of(a, lo) : tb.n_active;
  float h[kEach];
  int slot[kEach];  // of the largest |h|, -1: no element here
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int e = threadIdx.x + kSThreads * j, i = e / cap, v = lo + e - i * cap;
    slot[j] = -1;
    h[j] = 0.0f;
    if (i < a.tokens && v < hi) {
      const int place = v < routed ? place_of(a, v) : tb.n_active;
      if (i < __popc(tb.tokens[place])) {
        slot[j] = (place - first) * a.tokens + i;
        h[j] = hf[e];
        if (isfinite(h[j])) atomicMax(&tb.top[slot[j]], __float_as_uint(fabsf(h[j])));
      }
    }
  }
  __syncthreads();
  uint16_t* out = reinterpret_cast<uint16_t*>(hf);
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (slot[j] >= 0) {
      uint16_t* p = out + threadIdx.x + kSThreads * j;
      store_split<T>(p, p + a.tokens * cap, h[j] * h_scale(tb.top[slot[j]]));
    }
  __syncthreads();
}

// The gate / up phase takes RG row tiles at once, the down phase RD, with up to ND column tiles of 4 tokens.
template <typename T, int ND, int RG, int RD>
__global__ void __launch_bounds__(kSThreads, 1) dense_moe_kernel(const __grid_constant__ MoeArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Tables tb;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // ---- routing, in every block ----
  if (tid < kMoeExperts / 32) tb.used[tid] = 0;
  if (tid <= kMoePairs) tb.tokens[tid] = 0;
  __syncthreads();
  int id = -1;
  float wt = 0.0f;
  if (warp < a.tokens) {
    if (a.ids_in == nullptr) {
      const uint16_t* row = a.logits + warp * a.experts;
      if (a.experts <= 64) route_warp<T, 2>(row, a, id, wt);
      else if (a.experts <= 128) route_warp<T, 4>(row, a, id, wt);
      else if (a.experts <= 256) route_warp<T, 8>(row, a, id, wt);
      else route_warp<T, 32>(row, a, id, wt);
      if (blockIdx.x == 0 && lane < a.top_k) {
        if (a.ids_out) a.ids_out[warp * a.top_k + lane] = id;
        if (a.w_out) a.w_out[warp * a.top_k + lane] = T::from_f32(wt);
      }
    } else {
      int64_t given = -1;
      if (lane < a.top_k) {
        given = a.ids_in[warp * a.top_k + lane];
        wt = T::to_f32(a.w_in[warp * a.top_k + lane]);
      }
      if (given >= a.experts && blockIdx.x == 0) atomicOr(&g_dense_status, kStatusBadExpertId);
      id = given >= 0 && given < a.experts ? static_cast<int>(given) : -1;
      // an expert given twice for a token counts once, with both weights
      float total = 0.0f;
      bool first = true;
      for (int j = 0; j < a.top_k; ++j) {
        const int other = __shfl_sync(kFullMask, id, j);
        const float w = __shfl_sync(kFullMask, wt, j);
        if (other == id) {
          total += w;
          first = first && j >= lane;
        }
      }
      wt = total;
      if (!first) id = -1;
    }
    if (lane >= a.top_k || (id >= 0 && a.mask != nullptr && a.mask[id] == 0)) id = -1;
    if (id >= 0) atomicOr(&tb.used[id >> 5], 1u << (id & 31));
  }
  __syncthreads();
  int place = -1;
  if (id >= 0) {
    place = __popc(tb.used[id >> 5] & ((1u << (id & 31)) - 1u));
    for (int i = 0; i < id >> 5; ++i) place += __popc(tb.used[i]);
    tb.active[place] = id;
    atomicOr(&tb.tokens[place], 1u << warp);
  }
  if (warp == kSW - 1) {  // 32 words of 32 experts
    int n = __popc(tb.used[lane]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) n += __shfl_xor_sync(kFullMask, n, off);
    if (lane == 0) tb.n_active = n;
    if (a.shared_inter > 0) {  // every token's, in the place after the last routed expert
      if (lane == 0) tb.tokens[n] = (1u << a.tokens) - 1u;
      if (lane < a.tokens) {
        tb.weight[n][lane] = __ldcg(a.shared_open + lane);
        tb.list[n][lane] = static_cast<uint8_t>(lane);
      }
    }
  }
  __syncthreads();
  if (place >= 0) {
    const int i = __popc(tb.tokens[place] & ((1u << warp) - 1u));
    tb.weight[place][i] = wt;
    tb.list[place][i] = static_cast<uint8_t>(warp);
  }
  __syncthreads();

  // ---- this block's rows: h, then their part of the outputs ----
  const Split split(static_cast<int64_t>(tb.n_active) * a.inter + a.shared_inter, a.h_cap);
  uint16_t* hs = reinterpret_cast<uint16_t*>(smem + kStreamBytes);
  const int first = min(static_cast<int>(blockIdx.x) * split.per_block, split.ranges);
  const int last = min(first + split.per_block, split.ranges);
  for (int r = first; r < last; ++r) {
    const int lo = split.begin(r), hi = split.begin(r + 1);
    DownStreamer<T, ND, RD> down(a, tb, smem, hs, a.h_cap, r, lo, hi);
    const auto put = [&](int place, int i, int v, float gate, float up) {
      const float h = tb.weight[place][i] * (silu_f32(gate) * up);
      const int at = i * a.h_cap + (v - lo);
      if constexpr (T::kBf16) store_split<T>(hs + at, hs + at + a.tokens * a.h_cap, h);
      else reinterpret_cast<float*>(hs)[at] = h;
    };
    if constexpr (!T::kBf16)  // read again after the barriers of the gate / up phase
      for (int i = tid; i < static_cast<int>(sizeof(tb.top) / sizeof(tb.top[0])); i += kSThreads) tb.top[i] = 0;
    if constexpr (ND <= 2) {
      // at most 8 tokens: one column tile holds them all, for all rows of the range at once
      const GateUpSrc src(a, tb, lo, hi, nullptr, a.tokens);
      Streamer<T, 1, RG, 8, GateUpSrc> up(src, smem);
      up.prologue(src.tiles());
      up.run(a.tokens, [&](int tile, int row, int col, auto sum) {
        const int v = lo + 8 * tile, place = v < src.routed ? place_of(a, v) : tb.n_active;
        const uint32_t toks = tb.tokens[place], bit = 1u << col;
        if (toks & bit) put(place, __popc(toks & (bit - 1u)), v + row, sum(row, col), sum(row + 8, col));
      }, [&] { down.prologue(); });
    } else {
      // Expert by expert, only the tokens routed there as columns, 8 at a time:
      // with all 16 as columns of every expert the token fragments were as many
      // bytes as the weights (16 tokens, 128 x 768 experts: 178 us).
      const int routed = tb.n_active * a.inter;
      for (int v = lo; v < hi;) {
        const int place = v < routed ? place_of(a, v) : tb.n_active;
        const int end = v < routed ? min(hi, (place + 1) * a.inter) : hi, n = __popc(tb.tokens[place]);
        for (int c0 = 0; c0 < n; c0 += 8) {
          const int cols = min(8, n - c0);
          const GateUpSrc src(a, tb, v, end, &tb.list[place][c0], cols);
          Streamer<T, 1, RG, 8, GateUpSrc> up(src, smem);
          up.prologue(src.tiles());
          up.run(cols, [&](int tile, int row, int col, auto sum) {
            put(place, c0 + col, v + 8 * tile + row, sum(row, col), sum(row + 8, col));
          }, [&] {
            if (end == hi && c0 + 8 >= n) down.prologue();
          });
          __syncthreads();  // the partials may be overwritten
        }
        v = end;
      }
    }
    __syncthreads();  // h is complete
    if constexpr (!T::kBf16) split_scaled<T>(a, tb, reinterpret_cast<float*>(hs), a.h_cap, lo, hi);
    down.run();
    __syncthreads();  // h may be written again
  }
  // This block's partial sums are written; while the others finish, each token's
  // list of pieces, by the warp that routed it.
  ac::grid_arrive(a.bar);
  if (warp < a.tokens) {
    if (lane == a.top_k && a.shared_inter > 0) place = tb.n_active;
    int rank = 0, before = 0, r0 = 0, count = 0;
    if (place >= 0) {
      const int begin = place * a.inter, len = place < tb.n_active ? a.inter : a.shared_inter;
      r0 = split.of_row(begin);
      count = split.of_row(begin + len - 8) - r0 + 1;
    }
    for (int j = 0; j <= a.top_k; ++j) {
      const int other = __shfl_sync(kFullMask, place, j), c = __shfl_sync(kFullMask, count, j);
      if (other >= 0 && other < place) {
        ++rank;
        before += c;
      }
    }
    const int n = __popc(__ballot_sync(kFullMask, place >= 0));
    if (lane == 0) tb.n_places[warp] = n;
    if (place >= 0) {
      tb.place[warp][rank] = place;
      tb.range[warp][rank] = r0;
      tb.pieces[warp][rank] = before;
      if (rank == n - 1) tb.pieces[warp][n] = before + count;
    }
  }
  if (!ac::grid_wait(a.bar, &tb.ok)) {
    if (tid == 0) atomicOr(&g_dense_status, kStatusTimeout);
    return;
  }

  // ---- out = r + the pieces' sums ----
  // `lanes` neighbouring lanes add up a quad, four outputs of a token: lane l of
  // them takes pieces l, l + lanes, ... (experts ascending), four reads under way
  // at once, then their sums are added in a fixed tree.  As many lanes as let the
  // block take all its quads in one pass, but 8 at least.
  const int quads = a.hidden / 4;
  const uint32_t all = static_cast<uint32_t>(quads) * a.tokens, b = blockIdx.x;  // at most 16384 x 16
  const int q0 = static_cast<int>(all * b / gridDim.x), q1 = static_cast<int>(all * (b + 1) / gridDim.x);
  int lanes = 32;
  while (lanes > 8 && kSThreads / lanes < q1 - q0) lanes /= 2;
  for (int qb = q0; qb < q1; qb += kSThreads / lanes) {
    const int q = qb + tid / lanes, tok = min(q, q1 - 1) / quads, col = min(q, q1 - 1) - tok * quads;
    const int total = q < q1 && tb.n_places[tok] > 0 ? tb.pieces[tok][tb.n_places[tok]] : 0;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    int j = 0;  // place in the token's list
    for (int p0 = tid & (lanes - 1); p0 < total; p0 += 4 * lanes) {
      float4 f[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int p = p0 + u * lanes;
        f[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (p < total) {
          while (p >= tb.pieces[tok][j + 1]) ++j;
          const int at_place = tb.place[tok][j], at = tb.range[tok][j] + p - tb.pieces[tok][j] + at_place;
          const int i = __popc(tb.tokens[at_place] & ((1u << tok) - 1u));
          f[u] = __ldcg(reinterpret_cast<const float4*>(a.partial + (static_cast<int64_t>(at) * a.tokens + i) * a.hidden +
                                                        4 * col));
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        s.x += f[u].x;
        s.y += f[u].y;
        s.z += f[u].z;
        s.w += f[u].w;
      }
    }
    __syncwarp();
    for (int off = lanes / 2; off > 0; off >>= 1) {
      s.x += __shfl_xor_sync(kFullMask, s.x, off);
      s.y += __shfl_xor_sync(kFullMask, s.y, off);
      s.z += __shfl_xor_sync(kFullMask, s.z, off);
      s.w += __shfl_xor_sync(kFullMask, s.w, off);
    }
    if (q < q1 && (tid & (lanes - 1)) == 0) {
      const float v[4] = {s.x, s.y, s.z, s.w};
      uint16_t* o = a.out + tok * a.ldo + 4 * col;
      float r[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (a.res != nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = T::to_f32(a.res[tok * a.ldr + 4 * col + i]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = T::from_f32(v[i] + r[i]);
    }
  }
}

// Rows of h that a block holds at a time: 32 more than a multiple of 64, so
// that the fragment reads of two token rows fall into different banks.
int moe_h_cap(int tokens) {
  const int rows = kHBytes / (4 * tokens);
  return (rows - 32) / 64 * 64 + 32;
}
// Partial rows [tokens][hidden] of the largest split: a piece per range and
// expert boundary.
int64_t moe_pieces(const MoeArgs& a, int sms) {
  const int most = a.tokens * a.top_k < a.experts ? a.tokens * a.top_k : a.experts;
  const int64_t groups = (static_cast<int64_t>(most) * a.inter + a.shared_inter) / 8, cap = moe_h_cap(a.tokens) / 8;
  const int64_t per_block = (groups + sms * cap - 1) / (sms * cap);
  return sms * (per_block > 0 ? per_block : 1) + most + 1;
}

template <typename T, int ND, int RG, int RD>
static cudaError_t moe_main(const MoeArgs& a, int sms, cudaStream_t st) {
  const void* kern = reinterpret_cast<const void*>(dense_moe_kernel<T, ND, RG, RD>);
  constexpr size_t smem = kStreamBytes + kHBytes;
  static_assert(smem + sizeof(Tables) + 1024 <= 232448, "shared-memory plan");
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
  return cudaLaunchKernelEx(&cfg, dense_moe_kernel<T, ND, RG, RD>, a);
}

template <typename T, int ND, int RG>
static cudaError_t moe_down(const MoeArgs& a, int sms, cudaStream_t st) {
  const int rd = tiles_at_once<ND>((a.hidden / 16 + kSW - 1) / kSW, kLongK);  // a warp's tiles
  if constexpr (ND == 1)
    if (rd == 4) return moe_main<T, ND, RG, 4>(a, sms, st);
  if constexpr (ND <= 2)
    if (rd == 2) return moe_main<T, ND, RG, 2>(a, sms, st);
  return moe_main<T, ND, RG, 1>(a, sms, st);
}

template <typename T, int ND>
static cudaError_t moe_tiles(const MoeArgs& a, int sms, cudaStream_t st) {
  return tiles_at_once<1>(kSlots, a.hidden) == 4 ? moe_down<T, ND, 4>(a, sms, st) : moe_down<T, ND, 2>(a, sms, st);
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
  if (a.tokens <= 4) return moe_tiles<T, 1>(a, sms, st);
  if (a.tokens <= 8) return moe_tiles<T, 2>(a, sms, st);
  return moe_tiles<T, 4>(a, sms, st);
}

cudaError_t launch_dense_moe(MoeArgs a, int dtype, int sms, cudaStream_t st) {
  a.h_cap = moe_h_cap(a.tokens);
  a.inter_inverse = ~0ull / static_cast<uint64_t>(a.inter) + 1;  // floor(row / inter) = high word of row * this, rows < 2^32
  return dtype == MOE_DTYPE_FP16 ? moe_both<Fp16>(a, sms, st) : moe_both<Bf16>(a, sms, st);
}

cudaError_t read_dense_status(int* status, cudaStream_t st) { return take_status(&g_dense_status, status, st); }

}  // namespace dense
}  // namespace moe
