// dense_gemm.cu — dense projections on the tcgen05 tensor cores, for more
// tokens than the weight-streaming kernel takes: out = act(x W^T + b) + r and
// act(x Wg^T) * (x Wu^T), accumulated in tensor memory in fp32, the epilogue
// in the same kernel.  A = token rows (the MMA's M), B = weight rows (its N),
// both K-major, TMA-loaded in 64-element K steps with the 128-byte swizzle;
// rows and K beyond the tensors arrive as zeros.
//
// pair_gemm_kernel: many tokens.  A pair of SMs (cta_group::2) works on 256
//   tokens x 256 weight rows: each SM stages half of both operands, so a byte
//   brought into shared memory is used for 256 rows of the other operand.
//   Gated: the first SM's half of B is 128 gate rows, the second's the same 128
//   up rows, so gate and up of a feature are 128 accumulator columns apart.
//   Persistent; two accumulators of 256 columns (all of tensor memory), so the
//   epilogue of one tile runs under the next tile's MMAs.
// split_gemm_kernel: a few hundred tokens, or too few tiles for every SM.  One
//   SM per tile of up to 256 tokens x a slice of the features whose width is
//   chosen so that the slices cover the SMs evenly, optionally with K split
//   over a cluster of 2, 4 or 8 SMs that add their partial sums through
//   distributed shared memory in rank order (no workspace, no atomics).
//
// Waits are bounded: one that runs out records kStatusTimeout and the kernel
// unwinds, waiting (bounded) for what it has in flight.
#include <cuda.h>

#include <mutex>

#include "dense_common.cuh"
#include "kernels.h"

namespace moe {
namespace dense {

__device__ int g_gemm_status;  // kStatus* bits of this device's GEMM launches since the last read

namespace {

constexpr uint32_t kSpin = 1u << 22;
constexpr int kBK = 64;                 // K elements per stage: one 128-byte swizzled row
constexpr size_t kSmemLimit = 232448;
// A block of a cluster holds tensor memory while it waits for the cluster's
// other blocks, so it must never wait for some itself: two such blocks of two
// clusters could wait for each other for good.  It therefore takes shared memory
// in proportion, 512 columns all of it, and the blocks of clusters that an SM can
// hold never come to more than its 512 columns, whatever calls they belong to.
// (Blocks without a cluster may have to wait, but nothing waits in them.)
constexpr size_t kTmemShare = (kSmemLimit - 512) / 512;  // bytes a column

MOE_DEV uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
MOE_DEV void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
MOE_DEV void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Arrive on a barrier of any block of the cluster.
MOE_DEV void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
MOE_DEV bool mbar_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < kSpin; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}
MOE_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Address, in the cluster's shared window, of block `rank`'s copy of `addr`.
MOE_DEV uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
MOE_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;" ::: "memory"); }
MOE_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
MOE_DEV void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}
MOE_DEV void st_cluster(uint32_t addr, float x, float y, float z, float w) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(x), "f"(y), "f"(z), "f"(w) : "memory");
}

// 2-D tiled load into this block's shared memory (no multicast).  With PAIR the
// barrier may be the pair's other block's.
template <bool PAIR>
MOE_DEV void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
        "[%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}

// K-major tile, 128-byte swizzle: rows of 128 bytes, 8-row groups 1024 bytes apart.
MOE_DEV uint64_t tile_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
// Instruction descriptor: D fp32, A and B of the element type, K-major, M x n.
template <typename T>
MOE_DEV uint32_t instr_desc(int m, int n) {
  constexpr uint32_t type = T::kBf16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
template <int GROUP>
MOE_DEV void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (GROUP == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// One arrival on `bar` (of both blocks of a pair) once the MMAs issued so far are done.
MOE_DEV void commit_one(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
MOE_DEV void commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
MOE_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
MOE_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 consecutive fp32 columns of this warp's 32 lanes; the values are there after tmem_wait.
MOE_DEV void tmem_ld16(uint32_t taddr, float* v) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// 8 columns.
MOE_DEV void tmem_ld8(uint32_t taddr, float (&v)[8]) {
  uint32_t r[8];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}

// N groups of 8 columns, `apart` columns from one to the next, in one round trip.
template <int N>
MOE_DEV void tmem_ld8_all(uint32_t taddr, int apart, float (&v)[N][8]) {
  uint32_t r[N][8];
#pragma unroll
  for (int g = 0; g < N; ++g)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[g][0]), "=r"(r[g][1]), "=r"(r[g][2]), "=r"(r[g][3]), "=r"(r[g][4]), "=r"(r[g][5]), "=r"(r[g][6]),
                   "=r"(r[g][7])
                 : "r"(taddr + g * apart));
  // the registers pass through the wait, so that nothing uses them before it
#pragma unroll
  for (int g = 0; g < N; ++g)
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[g][0]), "+r"(r[g][1]), "+r"(r[g][2]), "+r"(r[g][3]), "+r"(r[g][4]), "+r"(r[g][5]), "+r"(r[g][6]),
                   "+r"(r[g][7])::"memory");
#pragma unroll
  for (int g = 0; g < N; ++g)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[g][i] = __uint_as_float(r[g][i]);
}

template <int N>
MOE_DEV void activate_all(int act, float (&v)[N]) {
  switch (act) {
    case MOE_ACT_SILU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate<MOE_ACT_SILU>(v[i]);
      break;
    case MOE_ACT_GELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate<MOE_ACT_GELU>(v[i]);
      break;
    case MOE_ACT_GELU_TANH:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate<MOE_ACT_GELU_TANH>(v[i]);
      break;
    case MOE_ACT_RELU:
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = activate<MOE_ACT_RELU>(v[i]);
      break;
    default:
      break;
  }
}

MOE_DEV void give_up(volatile int* flag) {
  if (!*flag) {
    *flag = 1;
    atomicOr(&g_gemm_status, kStatusTimeout);
  }
}

// ---------------------------------------------------------------------------
// pair_gemm_kernel
// ---------------------------------------------------------------------------
constexpr int kPStages = 6, kPTile = 128 * 128, kPStage = 2 * kPTile;  // A and B half of one SM: 16 KB each
constexpr int kPBarOff = kPStages * kPStage;
constexpr int kPTurnOff = kPBarOff + 8 * (2 * kPStages + 4) + 16;  // 32 rows x 16 columns of each epilogue warp
constexpr int kPTurnRow = 17;
constexpr size_t kPSmem = kPTurnOff + 4 * 32 * kPTurnRow * sizeof(float) + 1024;
constexpr int kPThreads = 256;
constexpr size_t kPTake = 512 * kTmemShare;  // what a block asks for
static_assert(kPSmem <= kPTake && kPTake <= kSmemLimit, "shared-memory plan");

// Residual of 64 columns of a row, read well ahead of the sums it joins: a read
// per 16 columns when they are stored waits out a memory latency each time
// (4000 x 5000 outputs, K = 1024, with bias: 148 us, so 76).
struct Ahead64 {
  uint4 r[8];
  MOE_DEV void load(const LinearArgs& a, int64_t m, int n, bool row) {
    const uint16_t* p = a.res + m * a.ldr + n;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      r[i] = row && n + 8 * i + 8 <= a.n ? *reinterpret_cast<const uint4*>(p + 8 * i) : make_uint4(0, 0, 0, 0);
  }
};

// 16 output columns of one row from n on, all of them there, rows on 16-byte
// boundaries; r0 and r1: their residual (zeros without one).
template <typename T>
MOE_DEV void store16(const LinearArgs& a, int64_t m, int n, float (&v)[16], uint4 r0, uint4 r1) {
  uint4* o = reinterpret_cast<uint4*>(a.out + m * a.ldo + n);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint4 q = h == 0 ? r0 : r1;
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = T::unpack(w[i]);
      p[i] = T::pack(v[8 * h + 2 * i] + f.x, v[8 * h + 2 * i + 1] + f.y);
    }
    o[h] = make_uint4(p[0], p[1], p[2], p[3]);
  }
}

// The same for any row alignment and a ragged last column, by the whole warp:
// 32 rows from m0 on, this lane's row in v.  The values are turned through
// `turn` (32 x kPTurnRow), so that 16 lanes write neighbouring elements of a row;
// a store of one element in each of 32 rows cost 32 sectors (3765 x 5789 gated outputs
// of K = 152: 245 us, so 169).
template <typename T>
MOE_DEV void store_any(const LinearArgs& a, int64_t m0, int n, const float (&v)[16], float* turn) {
  const int lane = threadIdx.x & 31, col = lane & 15;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 16; ++i) turn[lane * kPTurnRow + i] = v[i];
  __syncwarp();
  // this lane's 16 elements: rows lane / 16, + 2, ...; all residuals are read before anything is stored
  const int64_t first = m0 + (lane >> 4);
  const int rows = n + col < a.n ? static_cast<int>(min(static_cast<int64_t>(16), (a.m - first + 1) / 2)) : 0;
  const float* mine = turn + (lane >> 4) * kPTurnRow + col;
  uint16_t* o = a.out + first * a.ldo + n + col;
  const int64_t step = 2 * a.ldo;
  if (a.res != nullptr) {
    const uint16_t* p = a.res + first * a.ldr + n + col;
    uint16_t r[16];
#pragma unroll
    for (int i = 0; i < 16; ++i, p += 2 * a.ldr) r[i] = i < rows ? *p : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i, o += step)
      if (i < rows) *o = T::from_f32(mine[2 * i * kPTurnRow] + T::to_f32(r[i]));
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i, o += step)
      if (i < rows) *o = T::from_f32(mine[2 * i * kPTurnRow]);
  }
}

template <typename T, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPThreads, 1)
    pair_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                     const __grid_constant__ CUtensorMap tm_u, const __grid_constant__ LinearArgs a, int wide) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int abort_s;
  volatile int* aborted = &abort_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kPBarOff);
  uint64_t* full = bars;                      // [stages] of the first block: both blocks' tiles landed
  uint64_t* empty = bars + kPStages;          // [stages] of each block: the MMAs that read the stage are done
  uint64_t* acc_full = empty + kPStages;      // [2] of each block
  uint64_t* acc_empty = acc_full + 2;         // [2] of the first block: both blocks' epilogue warps have read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);

  if (tid == 0) {
    for (int s = 0; s < kPStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&acc_full[s]), 1);
      mbar_init(smem_u32(&acc_empty[s]), 8);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *aborted = 0;
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  cluster_sync();  // the peer's barriers are initialised, both have their tensor memory
  fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  constexpr int kTN = GATED ? 128 : 256;  // features per tile
  const int mt = (a.m + 255) / 256, nt = (a.n + kTN - 1) / kTN, nk = (a.k + kBK - 1) / kBK;
  const int pairs = gridDim.x / 2, pair = blockIdx.x / 2;
  // Tiles in groups of up to 16 row tiles, rows fastest: the pairs at work share
  // few weight tiles and a block of tokens that stays in L2.
  const int total = mt * nt;
  auto place = [&](int i, int& m, int& n) {
    const int per = 16 * nt, gidx = i / per, in = i - gidx * per, rows = min(16, mt - 16 * gidx);
    n = in / rows;
    m = 16 * gidx + in - n * rows;
  };

  if (warp == 0) {
    if (lane == 0) {
      int it = 0, s = 0;
      uint32_t phase = 1;  // a stage's first use waits for nothing
      const uint32_t full0 = map_rank(smem_u32(&full[0]), 0);
      bool ok = true;
      for (int i = pair; i < total && ok; i += pairs) {
        int m, n;
        place(i, m, n);
        const int xr = m * 256 + 128 * static_cast<int>(rank);
        const int wr = GATED ? n * 128 : n * 256 + 128 * static_cast<int>(rank);
        const CUtensorMap* tw = GATED && rank == 1 ? &tm_u : &tm_w;
        for (int kc = 0; kc < nk; ++kc, ++it) {
          if (it >= kPStages && !mbar_wait(smem_u32(&empty[s]), phase)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_expect_tx(smem_u32(&full[s]), 2 * kPStage);
          const uint32_t bar = full0 + 8 * s, dst = smem_u32(smem) + s * kPStage;
          tma_load<true>(dst, &tm_x, kc * kBK, xr, bar);
          tma_load<true>(dst + kPTile, tw, kc * kBK, wr, bar);
          if (++s == kPStages) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) give_up(aborted);
      // nothing of this block's stages is in flight or being read when it exits
      for (int j = max(0, it - kPStages); j < it; ++j) mbar_wait(smem_u32(&empty[j % kPStages]), (j / kPStages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = instr_desc<T>(256, 256);
      const uint64_t da0 = tile_desc(smem_u32(smem)), db0 = tile_desc(smem_u32(smem) + kPTile);
      int s = 0, ti = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = pair; i < total && ok; i += pairs, ++ti) {
        const int acc = ti & 1;
        if (ti >= 2 && !mbar_wait(smem_u32(&acc_empty[acc]), ((ti >> 1) - 1) & 1)) {
          ok = false;
          break;
        }
        fence_after();
        for (int kc = 0; kc < nk; ++kc) {
          if (!mbar_wait(smem_u32(&full[s]), phase)) {
            ok = false;
            break;
          }
          fence_after();
          const uint64_t da = da0 + static_cast<uint64_t>(s) * (kPStage >> 4);
          const uint64_t db = db0 + static_cast<uint64_t>(s) * (kPStage >> 4);
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk)
            umma<2>(tmem + acc * 256, da + 2 * kk, db + 2 * kk, idesc, kc > 0 || kk > 0);
          commit_pair(smem_u32(&empty[s]));
          if (++s == kPStages) {
            s = 0;
            phase ^= 1;
          }
        }
        commit_pair(smem_u32(&acc_full[acc]));
      }
      if (!ok) give_up(aborted);
    }
  } else if (warp >= 4) {
    const int q = warp & 3;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    float* turn = reinterpret_cast<float*>(smem + kPTurnOff) + q * 32 * kPTurnRow;
    const bool wide_bias = reinterpret_cast<uintptr_t>(a.bias) % 16 == 0;
    int ti = 0;
    for (int i = pair; i < total; i += pairs, ++ti) {
      int mi, ni;
      place(i, mi, ni);
      const int acc = ti & 1, n0 = ni * kTN;
      const int64_t m = static_cast<int64_t>(mi) * 256 + 128 * rank + q * 32 + lane;
      const bool ahead = !GATED && wide != 0 && a.res != nullptr;
      Ahead64 cur, next;
#pragma unroll
      for (int j = 0; j < 8; ++j) cur.r[j] = next.r[j] = make_uint4(0, 0, 0, 0);
      if (ahead) cur.load(a, m, n0, m < a.m);  // while the tile's MMAs still run
      const bool ok = mbar_wait(smem_u32(&acc_full[acc]), (ti >> 1) & 1);
      if (!__all_sync(kFullMask, ok)) {
        give_up(aborted);
        break;
      }
      fence_after();
      const uint32_t base = tmem + acc * 256 + lanes;
#pragma unroll 1
      for (int c = 0; c < kTN && n0 + c < a.n; c += 64) {  // warp-uniform
        if (ahead && c + 64 < kTN) next.load(a, m, n0 + c + 64, m < a.m);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = n0 + c + 16 * j;
          if (n >= a.n) break;
          float v[16];
          tmem_ld16(base + c + 16 * j, v);
          if constexpr (GATED) {
            float u[16];
            tmem_ld16(base + 128 + c + 16 * j, u);
            activate_all(a.act, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] *= u[i];
          } else {
            if (a.bias && wide_bias && n + 16 <= a.n) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint4 q = __ldg(reinterpret_cast<const uint4*>(a.bias + n + 8 * h));
                const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 f = T::unpack(w[i]);
                  v[8 * h + 2 * i] += f.x;
                  v[8 * h + 2 * i + 1] += f.y;
                }
              }
            } else if (a.bias) {
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (n + i < a.n) v[i] += T::to_f32(__ldg(a.bias + n + i));
            }
            activate_all(a.act, v);
          }
          if (wide != 0 && n + 16 <= a.n) {
            if (m < a.m) store16<T>(a, m, n, v, cur.r[2 * j], cur.r[2 * j + 1]);
          } else {
            store_any<T>(a, m - lane, n, v, turn);
          }
        }
        cur = next;
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_rank(smem_u32(&acc_empty[acc]), 0));
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  cluster_sync();
  fence_after();
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// ---------------------------------------------------------------------------
// split_gemm_kernel
// ---------------------------------------------------------------------------
struct SplitPlan {
  int rows;     // token rows per tile: 128 or 256
  int splits;   // blocks of a cluster that share a tile, each with a part of K
  int slices;   // feature slices, in groups of 8 features
  int width;    // features of the widest slice, padded (gated: multiple of 8, else of 16)
  int box_x;    // token rows loaded per stage
  int stages;
  int smem;
  int tmem;     // columns of tensor memory
  int wide;     // out and residual rows allow 16-byte accesses
};
constexpr int kQThreads = 320;  // producer, MMA, 8 epilogue warps
constexpr int kQTail = 1024 + 16384;  // alignment, and what an MMA reads past a tile of fewer than 128 rows

// Bias and residual of 8 columns of a row, read ahead of the sums they join.
template <typename T>
struct Extra8 {
  uint32_t b[4], r[4];
  MOE_DEV void load(const LinearArgs& a, int64_t m, int n, bool row, bool wide) {
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = r[i] = 0;
    const auto pick = [&](const uint16_t* p, uint32_t (&o)[4], bool vec) {
      if (vec) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        o[0] = q.x;
        o[1] = q.y;
        o[2] = q.z;
        o[3] = q.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (n + i < a.n) o[i / 2] |= static_cast<uint32_t>(p[i]) << (16 * (i & 1));
      }
    };
    if (a.bias) pick(a.bias + n, b, false);
    if (a.res && row) pick(a.res + m * a.ldr + n, r, wide && n + 8 <= a.n);
  }
};

// Epilogue of 8 columns of a row.
template <typename T, bool GATED>
MOE_DEV void finish8(const LinearArgs& a, int64_t m, int n, float (&v)[8], const float (&u)[8], const Extra8<T>& e, bool wide) {
  if constexpr (GATED) {
    activate_all(a.act, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= u[i];
  } else {
    if (a.bias) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = T::unpack(e.b[i]);
        v[2 * i] += f.x;
        v[2 * i + 1] += f.y;
      }
    }
    activate_all(a.act, v);
    if (a.res) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = T::unpack(e.r[i]);
        v[2 * i] += f.x;
        v[2 * i + 1] += f.y;
      }
    }
  }
  uint16_t* o = a.out + m * a.ldo + n;
  if (wide && n + 8 <= a.n) {
    *reinterpret_cast<uint4*>(o) =
        make_uint4(T::pack(v[0], v[1]), T::pack(v[2], v[3]), T::pack(v[4], v[5]), T::pack(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (n + i < a.n) o[i] = T::from_f32(v[i]);
  }
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(kQThreads, 1)
    split_gemm_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                      const __grid_constant__ CUtensorMap tm_u, const __grid_constant__ LinearArgs a,
                      const __grid_constant__ SplitPlan p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[16], empty[16], acc_full;
  __shared__ uint32_t tmem_s;
  __shared__ int abort_s;
  volatile int* aborted = &abort_s;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = p.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int slice = blockIdx.x / p.splits;
  const int64_t eights = (a.n + 7) / 8;
  const int n0 = static_cast<int>(8 * (eights * slice / p.slices));
  const int n1 = min(a.n, static_cast<int>(8 * (eights * (slice + 1) / p.slices)));
  const int m0 = blockIdx.y * p.rows, valid = min(p.rows, a.m - m0);
  const int nk = (a.k + kBK - 1) / kBK;
  const int k_lo = nk * rank / p.splits, k_hi = nk * (rank + 1) / p.splits, steps = k_hi - k_lo;
  const int cols = GATED ? 2 * p.width : p.width;  // the MMA's N
  const int row_tiles = (valid + 127) / 128;
  const int x_bytes = p.box_x * 128, stage_bytes = x_bytes + cols * 128;
  const uint32_t tmem_cols = static_cast<uint32_t>(p.tmem);

  if (tid == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(&acc_full), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *aborted = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)),
                 "r"(tmem_cols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_s;
  if (p.splits > 1) cluster_arrive();  // this block runs: its shared memory may be written (waited for before the exchange)
  asm volatile("griddepcontrol.wait;" ::: "memory");

  // One thread walks the stages in each role, so what it does per step is paid in
  // full latency: positions and descriptors are carried along, not worked out
  // (with divisions by the stage count a step took 500 ns whatever its size).
  if (warp == 0) {
    if (lane == 0) {
      uint32_t bar = smem_u32(&full[0]), gone = smem_u32(&empty[0]), dst = smem_u32(smem);
      int s = 0, it = 0, k = k_lo * kBK;
      uint32_t phase = 1;  // a stage's first use waits for nothing
      for (; it < steps; ++it, k += kBK) {
        if (it >= p.stages && !mbar_wait(gone, phase)) {
          give_up(aborted);
          break;
        }
        mbar_expect_tx(bar, stage_bytes);
        tma_load<false>(dst, &tm_x, k, m0, bar);
        tma_load<false>(dst + x_bytes, &tm_w, k, n0, bar);
        if constexpr (GATED) tma_load<false>(dst + x_bytes + p.width * 128, &tm_u, k, n0, bar);
        bar += 8;
        gone += 8;
        dst += stage_bytes;
        if (++s == p.stages) {
          s = 0;
          phase ^= 1;
          bar = smem_u32(&full[0]);
          gone = smem_u32(&empty[0]);
          dst = smem_u32(smem);
        }
      }
      if (*aborted)  // no copy may still be landing when the block exits
        for (int j = max(0, it - p.stages); j < it; ++j) mbar_wait(smem_u32(&full[j % p.stages]), (j / p.stages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = instr_desc<T>(128, cols);
      const uint64_t da0 = tile_desc(smem_u32(smem)), db0 = tile_desc(smem_u32(smem + x_bytes));
      const uint64_t next = static_cast<uint64_t>(stage_bytes >> 4);
      uint64_t da = da0, db = db0;
      uint32_t bar = smem_u32(&full[0]), gone = smem_u32(&empty[0]), phase = 0;
      int s = 0;
      for (int it = 0; it < steps; ++it) {
        if (!mbar_wait(bar, phase)) {
          give_up(aborted);
          break;
        }
        fence_after();
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk) umma<1>(tmem, da + 2 * kk, db + 2 * kk, idesc, it > 0 || kk > 0);
        // A tile of fewer than 128 rows: the MMA reads on into other bytes of the
        // stages; those accumulator lanes are never read.
        if (row_tiles > 1) {
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk)
            umma<1>(tmem + cols, da + 1024 + 2 * kk, db + 2 * kk, idesc, it > 0 || kk > 0);
        }
        commit_one(gone);
        bar += 8;
        gone += 8;
        da += next;
        db += next;
        if (++s == p.stages) {
          s = 0;
          phase ^= 1;
          bar = smem_u32(&full[0]);
          gone = smem_u32(&empty[0]);
          da = da0;
          db = db0;
        }
      }
      commit_one(smem_u32(&acc_full));
      if (!mbar_wait(smem_u32(&acc_full), 0)) give_up(aborted);  // every MMA is done before tensor memory is freed
    }
  }
  __syncwarp();

  // ---- epilogue: a lane is a token row, columns in chunks of 8 ----
  // Items (chunk, 32 rows): warp e takes item e, e + 8, ... of a lane quarter it may read.
  const int chunks = (n1 - n0 + 7) / 8, q = warp & 3, half = (warp - 2) >> 2;
  bool good = true;
  if (warp >= 2) {
    Extra8<T> next;
    if (p.splits == 1) {
      if (half < chunks) next.load(a, m0 + q * 32 + lane, n0 + 8 * half, q * 32 + lane < valid, p.wide);
    }
    good = __all_sync(kFullMask, mbar_wait(smem_u32(&acc_full), 0));
    if (!good) give_up(aborted);
    fence_after();
    if (good && p.splits == 1 && !*aborted) {
      for (int r = 0; r < row_tiles; ++r) {
        const int row = r * 128 + q * 32 + lane;
        for (int c = half; c < chunks; c += 2) {
          const Extra8<T> e = next;
          // the next item's bias and residual are under way while this one's sums are worked on
          const int nc = c + 2 < chunks ? c + 2 : half, nrow = c + 2 < chunks ? row : row + 128;
          next.load(a, m0 + nrow, n0 + 8 * nc, nrow < valid, p.wide);
          const uint32_t at = tmem + r * cols + 8 * c + (static_cast<uint32_t>(q * 32) << 16);
          float v[8], u[8];
          tmem_ld8(at, v);
          if constexpr (GATED) tmem_ld8(at + p.width, u);
          if (row < valid) finish8<T, GATED>(a, m0 + row, n0 + 8 * c, v, u, e, p.wide);
        }
      }
    }
    fence_before();
  }
  if (p.splits > 1) {
    // Chunk c belongs to block c % splits of the cluster.  Every block sends its
    // partial sums of a chunk to the owner's shared memory, [sender][chunk]
    // [4 columns][row], beside the owner's stages; the owner adds them in sender
    // order.
    constexpr int kSub = GATED ? 4 : 2;  // quads of columns of a chunk
    const int log = __ffs(p.splits) - 1, own = (chunks + p.splits - 1) >> log, quad_bytes = valid * 16;
    unsigned char* exchange = smem + p.stages * stage_bytes;
    __syncwarp();
    cluster_wait();
    if (warp >= 2 && !*aborted) {
      fence_after();
      const uint32_t mine = smem_u32(exchange) + static_cast<uint32_t>(rank * own * kSub * quad_bytes);
      constexpr int kAtOnce = GATED ? 2 : 4;  // chunks read from tensor memory in one round trip
      for (int r = 0; r < row_tiles; ++r) {
        const int row = r * 128 + q * 32 + lane;
        if (r * 128 + q * 32 >= valid) continue;  // warp-uniform
        for (int c0 = half; c0 < chunks; c0 += 2 * kAtOnce) {
          // chunks past the last one are padding of the tile: read and not sent
          const int last = (cols - 8) / 8;
          const uint32_t at = tmem + r * cols + (static_cast<uint32_t>(q * 32) << 16);
          float v[kAtOnce][8], u[kAtOnce][8];
          if (c0 + 2 * (kAtOnce - 1) <= (GATED ? p.width / 8 - 1 : last)) {
            tmem_ld8_all<kAtOnce>(at + 8 * c0, 16, v);
            if constexpr (GATED) tmem_ld8_all<kAtOnce>(at + p.width + 8 * c0, 16, u);
          } else {
            for (int g = 0; g < kAtOnce; ++g) {
              const int c = min(c0 + 2 * g, chunks - 1);
#pragma unroll
              for (int h = 0; h < kAtOnce; ++h)
                if (h == g) {
                  tmem_ld8(at + 8 * c, v[h]);
                  if constexpr (GATED) tmem_ld8(at + p.width + 8 * c, u[h]);
                }
            }
          }
          if (row < valid) {
#pragma unroll
            for (int g = 0; g < kAtOnce; ++g) {
              const int c = c0 + 2 * g;
              if (c < chunks) {
                const uint32_t to = map_rank(mine + (c >> log) * kSub * quad_bytes + row * 16, c & (p.splits - 1));
                st_cluster(to, v[g][0], v[g][1], v[g][2], v[g][3]);
                st_cluster(to + quad_bytes, v[g][4], v[g][5], v[g][6], v[g][7]);
                if constexpr (GATED) {
                  st_cluster(to + 2 * quad_bytes, u[g][0], u[g][1], u[g][2], u[g][3]);
                  st_cluster(to + 3 * quad_bytes, u[g][4], u[g][5], u[g][6], u[g][7]);
                }
              }
            }
          }
        }
      }
      fence_before();
    }
    // items of this block's chunks: 32 rows x a chunk per warp
    const int groups = (valid + 31) / 32, mine_chunks = rank < chunks ? (chunks - rank + p.splits - 1) / p.splits : 0;
    const int items = groups * mine_chunks;
    Extra8<T> next;
    const auto fetch = [&](int i) {
      const int row = (i % groups) * 32 + lane, c = rank + (i / groups) * p.splits;
      next.load(a, m0 + row, n0 + 8 * c, row < valid, p.wide);
    };
    if (warp < items) fetch(warp);
    __syncwarp();
    cluster_sync();
    if (!*aborted) {
      for (int i = warp; i < items; i += kQThreads / 32) {
        const Extra8<T> e = next;
        if (i + kQThreads / 32 < items) fetch(i + kQThreads / 32);
        const int row = (i % groups) * 32 + lane, slot = i / groups;
        if (row >= valid) continue;
        float v[8] = {}, u[8] = {};
        for (int s = 0; s < p.splits; ++s) {
          const unsigned char* from = exchange + static_cast<size_t>((s * own + slot) * kSub) * quad_bytes + row * 16;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 f = *reinterpret_cast<const float4*>(from + h * quad_bytes);
            v[4 * h] += f.x;
            v[4 * h + 1] += f.y;
            v[4 * h + 2] += f.z;
            v[4 * h + 3] += f.w;
            if constexpr (GATED) {
              const float4 g = *reinterpret_cast<const float4*>(from + (2 + h) * quad_bytes);
              u[4 * h] += g.x;
              u[4 * h + 1] += g.y;
              u[4 * h + 2] += g.z;
              u[4 * h + 3] += g.w;
            }
          }
        }
        finish8<T, GATED>(a, m0 + row, n0 + 8 * (rank + slot * p.splits), v, u, e, p.wide);
      }
    }
  }
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(tmem_cols));
  }
}

// ---------------------------------------------------------------------------
// Plans
// ---------------------------------------------------------------------------

// Blocks of the split kernel that run at once, by cluster size (asked of the
// driver once per device: how many clusters fit depends on the SMs per GPC).
int resident_blocks(int dev, int splits, int sms) {
  static std::mutex mu;
  static int known[64][9];
  if (splits == 1 || dev < 0 || dev >= 64) return sms;
  std::lock_guard<std::mutex> lock(mu);
  int& v = known[dev][splits];
  if (v == 0) {
    if (!ensure_dynamic_smem(reinterpret_cast<const void*>(split_gemm_kernel<Bf16, false>), kSmemLimit - 2048, kQThreads)) {
      v = -1;
      return 0;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(splits);
    cfg.blockDim = dim3(kQThreads);
    cfg.dynamicSmemBytes = kSmemLimit - 2048;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, split_gemm_kernel<Bf16, false>, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      v = -1;
    } else {
      v = n * splits < sms ? n * splits : sms;
    }
  }
  return v < 0 ? 0 : v;
}

// Estimated clocks of a plan; the best of the candidates is taken.  Per K step
// a block brings box_x + cols rows of 128 bytes into shared memory (about 50
// bytes a clock and SM) and its MMAs take 2 clocks a column and row tile; the
// epilogue, and where K is split the exchange of the partial sums, come once
// per wave.
SplitPlan plan_split(const LinearArgs& a, int dev, int sms, double& clocks) {
  const bool gated = a.w_up != nullptr;
  const int nk = (a.k + kBK - 1) / kBK, pad = gated ? 8 : 16, mul = gated ? 2 : 1;
  SplitPlan best{};
  clocks = 1e30;
  for (int rows = 128; rows <= 256; rows += 128) {
    if (rows == 256 && a.m <= 128) break;
    const int mg = (a.m + rows - 1) / rows;
    if (mg > 65535) continue;
    const int box = a.m >= rows ? rows : (a.m + 7) / 8 * 8;
    for (int splits = 1; splits <= 8; splits *= 2) {
      if (splits > nk) break;
      const int cap = resident_blocks(dev, splits, sms);
      for (int waves = 1; waves <= 4; ++waves) {
        int slices = cap * waves / (splits * mg);
        if (slices < 1) continue;
        const int most = (a.n + pad - 1) / pad;  // no narrower than the padding
        if (slices > most) slices = most;
        const int eights = (a.n + 7) / 8, width = (8 * ((eights + slices - 1) / slices) + pad - 1) / pad * pad;
        const int cols = width * mul;
        if (cols > 256 || rows / 128 * cols > 512) continue;
        const int stage = (box + cols) * 128;
        const int steps = (nk + splits - 1) / splits, real_waves = (slices * mg * splits + cap - 1) / cap;
        // partial sums that a block receives, beside its stages: its chunks of 8 columns from every block
        const int valid = a.m < rows ? a.m : rows, own = ((width + 7) / 8 + splits - 1) / splits;
        const int64_t part = splits > 1 ? 32LL * mul * valid * own * splits : 0;
        const int64_t room = static_cast<int64_t>(kSmemLimit) - 2048 - kQTail - part;
        int stages = room > 0 ? static_cast<int>(room / stage) : 0;
        if (stages > 16) stages = 16;
        if (stages > steps) stages = steps;
        if (stages < steps && stages < 3) continue;
        int64_t smem = static_cast<int64_t>(stages) * stage + part + kQTail;
        const double load = stage / 50.0, mma = 2.0 * cols * (box > 128 ? 2 : 1);
        const double items = (valid + 31) / 32 * ((width + 7) / 8) * mul / 8.0;  // 32 rows x 8 columns a warp
        const double join = splits > 1 ? 2500.0 + 90.0 * items + 60.0 * items : 110.0 * items;
        const double t = real_waves * (steps * (load > mma ? load : mma) + join + 3000.0);
        if (t < clocks) {
          clocks = t;
          const int need = rows / 128 * cols, tmem = need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512;
          if (splits > 1 && smem < static_cast<int64_t>(tmem * kTmemShare)) smem = static_cast<int64_t>(tmem * kTmemShare);
          best = SplitPlan{rows, splits, slices, width, box, stages, static_cast<int>(smem), tmem, 0};
        }
      }
    }
  }
  return best;
}

// A tensor map wants a stride of whole 16 bytes even where there is one row.
uint64_t row_stride(int64_t ld, int rows, int k) { return static_cast<uint64_t>(rows > 1 ? ld : k); }

// 16-byte accesses to the rows of out and residual.
int wide_output(const LinearArgs& a) {
  const auto aligned = [&](const void* p, int64_t ld) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (a.m == 1 || ld % 8 == 0);
  };
  return aligned(a.out, a.ldo) && (a.res == nullptr || aligned(a.res, a.ldr));
}

template <typename T, bool GATED>
cudaError_t launch_split(const LinearArgs& a, SplitPlan p, cudaStream_t st) {
  p.wide = wide_output(a);
  alignas(64) CUtensorMap tx, tw, tu;
  if (!make_tmap_rows(&tx, a.x, T::kBf16, a.k, a.m, a.ldx, p.box_x) ||
      !make_tmap_rows(&tw, a.w, T::kBf16, a.k, a.n, row_stride(a.ldw, a.n, a.k), p.width) ||
      !make_tmap_rows(&tu, GATED ? a.w_up : a.w, T::kBf16, a.k, a.n,
                      row_stride(GATED ? a.ldwu : a.ldw, a.n, a.k), p.width))
    return cudaErrorInvalidValue;
  const void* kern = reinterpret_cast<const void*>(split_gemm_kernel<T, GATED>);
  if (!ensure_dynamic_smem(kern, p.smem, kQThreads)) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(p.slices * p.splits, (a.m + p.rows - 1) / p.rows);
  cfg.blockDim = dim3(kQThreads);
  cfg.dynamicSmemBytes = p.smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.splits;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, split_gemm_kernel<T, GATED>, tx, tw, tu, a, p);
}

template <typename T, bool GATED>
cudaError_t launch_pair(const LinearArgs& a, int sms, cudaStream_t st) {
  alignas(64) CUtensorMap tx, tw, tu;
  if (!make_tmap_rows(&tx, a.x, T::kBf16, a.k, a.m, a.ldx, 128) ||
      !make_tmap_rows(&tw, a.w, T::kBf16, a.k, a.n, row_stride(a.ldw, a.n, a.k), 128) ||
      !make_tmap_rows(&tu, GATED ? a.w_up : a.w, T::kBf16, a.k, a.n,
                      row_stride(GATED ? a.ldwu : a.ldw, a.n, a.k), 128))
    return cudaErrorInvalidValue;
  const void* kern = reinterpret_cast<const void*>(pair_gemm_kernel<T, GATED>);
  if (!ensure_dynamic_smem(kern, kPTake, kPThreads)) return cudaErrorInvalidConfiguration;
  const int wide = wide_output(a);
  const int64_t tiles = static_cast<int64_t>((a.m + 255) / 256) * ((a.n + (GATED ? 127 : 255)) / (GATED ? 128 : 256));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * static_cast<unsigned>(tiles < sms / 2 ? tiles : sms / 2));
  cfg.blockDim = dim3(kPThreads);
  cfg.dynamicSmemBytes = kPTake;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, pair_gemm_kernel<T, GATED>, tx, tw, tu, a, wide);
}

// Whether the split kernel takes a projection, and then its plan.
bool takes_split(const LinearArgs& a, int dev, int sms, SplitPlan& p) {
  double split_clocks = 0;
  p = plan_split(a, dev, sms, split_clocks);
  const int wide = a.w_up != nullptr ? 128 : 256;
  const int64_t tiles = static_cast<int64_t>((a.m + 255) / 256) * ((a.n + wide - 1) / wide);
  const int pairs = sms / 2, nk = (a.k + kBK - 1) / kBK;
  const double pair_clocks = static_cast<double>((tiles + pairs - 1) / pairs) * nk * 600.0 + 8000.0;
  return split_clocks < pair_clocks;
}

template <typename T, bool GATED>
cudaError_t gemm(const LinearArgs& a, int dev, int sms, cudaStream_t st) {
  SplitPlan p;
  return takes_split(a, dev, sms, p) ? launch_split<T, GATED>(a, p, st) : launch_pair<T, GATED>(a, sms, st);
}

}  // namespace

cudaError_t launch_gemm(const LinearArgs& a, int dtype, int dev, int sms, cudaStream_t st) {
  if (dtype == MOE_DTYPE_FP16) return a.w_up ? gemm<Fp16, true>(a, dev, sms, st) : gemm<Fp16, false>(a, dev, sms, st);
  return a.w_up ? gemm<Bf16, true>(a, dev, sms, st) : gemm<Bf16, false>(a, dev, sms, st);
}

void plan_gemm(const LinearArgs& a, int dev, int sms, moe_linear_plan& out) {
  SplitPlan p;
  if (takes_split(a, dev, sms, p)) {
    out = {MOE_LINEAR_SPLIT, p.rows, p.splits, p.slices, p.width, p.stages, p.smem, p.tmem};
  } else {
    out = {MOE_LINEAR_PAIR, 256, 1, 1, a.w_up != nullptr ? 128 : 256, kPStages, static_cast<int>(kPTake), 512};
  }
}

__global__ void clear_bits_kernel(int* word, int bits) { atomicAnd(word, ~bits); }

// Only what was read is cleared: a kernel of another stream may set a bit meanwhile.
cudaError_t take_status(const void* symbol, int* status, cudaStream_t st) {
  void* p = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&p, symbol);
  if (e == cudaSuccess) e = cudaMemcpyAsync(status, p, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess || *status == 0) return e;
  clear_bits_kernel<<<1, 1, 0, st>>>(static_cast<int*>(p), *status);
  e = cudaGetLastError();
  return e == cudaSuccess ? cudaStreamSynchronize(st) : e;
}
cudaError_t read_gemm_status(int* status, cudaStream_t st) { return take_status(&g_gemm_status, status, st); }

}  // namespace dense
}  // namespace moe
