// dense_stream.cuh — streaming a block's weight rows past a few token columns
// on the warp-level tensor cores.
//
// With a handful of tokens a projection is bound by reading its weights once.
// A block owns a range of weight rows, cut into tiles of 16 (the mma's M;
// tokens are its N, 8 per column tile).  The 16 warps share K: in a step they
// cover 16 adjacent stretches of 64 elements of every row, one a warp, and what
// K leaves over is shared out in halves of 32, so that the warps differ by one
// half at most.  (Fewer warps on a tile and several tiles at once need fewer
// sums, but read DRAM in shorter runs: 8 experts of 14336, 5 tokens, 419 us with
// 16 warps on a tile, 447 with 4.)  For a step a warp takes up to RT tiles, so a
// token fragment is loaded once for RT weight tiles; the first step's, the same
// in every round of tiles, is kept.  Lane (g, t) feeds the mma with 8 consecutive
// elements at 8 t and at 32 + 8 t of rows g and g + 8 (A) and of token column g
// (B): an mma is unchanged by a permutation of K that both operands share, so
// nothing is shuffled.
//
// Weights in flight: a warp copies a step's 16 rows x 128 bytes of each tile
// into its own ring of D = PD x RT slots in shared memory with cp.async, whole
// 128-byte lines at a time, PD steps ahead, and waits for its own copies only;
// 16 warps x D x 2 KB = 128 KB per SM are under way (7 TB/s x 1 us / 148 SMs
// is 47 KB).  Rows are stored with the 64-byte halves of odd rows swapped, so
// that the fragment reads (two rows a phase) meet no bank conflict.  Addresses
// are split into a part per tile (kept in registers for a round of RT tiles)
// and a part per step, so that a slot costs a few tens of instructions: with
// both worked out per slot the issue slots, not the memory, were the limit.
//
// Partial sums: a warp keeps RT tiles in registers over its part of K, puts the
// 16 x 8 partial tiles into shared memory, and the block adds the 16 partials
// of each output in warp order (no atomics: the same bits every run) while the
// next tiles' copies are in flight.
#pragma once

#include "dense_common.cuh"

namespace moe {
namespace dense {

constexpr int kSW = 16;                 // warps of a block
constexpr int kSThreads = 32 * kSW;
constexpr int kPartCol = 20;            // floats per column of a partial tile: 16 rows, padded so that the 8 x 4 lanes
                                        // of a store fall into different banks
constexpr int kPartTile = 8 * kPartCol;

// 16 bytes global -> shared, past L1; zeros where bytes is 0 instead of 16.
MOE_DEV void copy16(uint32_t dst, const uint16_t* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
MOE_DEV void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
MOE_DEV void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
MOE_DEV uint4 ld_shared(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
  return r;
}
// Activations are read by every tile: through L1.
MOE_DEV uint4 ld_tokens(const uint16_t* p) {
  uint4 r;
  asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
constexpr int kStepBytes = 2048;  // 16 rows x 64 elements

constexpr int kSlots = 4;  // of a warp's ring

// Tiles that a warp keeps in registers when its block has `tiles` of K `k`: as
// many as share a token fragment, but no more than there are, since a ring slot
// of a tile that does not exist is a copy less in flight (2048 x 2048, one token:
// 4.0 us, with slots for four tiles where there is one 5.0); and two where a
// round of four would be over after two steps (128 x 768 experts, hidden 2048,
// 16 tokens: 149 us with two, 164 with four; 8 x 14336, hidden 4096: 439 and 424;
// sizes between were not measured).
constexpr int kLongK = 2 * 64 * kSW + 1;
template <int NT>
inline int tiles_at_once(int tiles, int k) {
  const int most = kSlots / NT;
  return tiles >= 3 && most >= 4 && k >= kLongK ? 4 : tiles >= 2 && most >= 2 ? 2 : 1;
}

// Dynamic shared memory of a Streamer: the ring of four slots a warp, then the partials.
constexpr size_t kStreamBytes = static_cast<size_t>(kSW) * kSlots * kStepBytes + sizeof(float) * 4 * kSW * kPartTile;

// NT column tiles of 8 tokens (1, 2 or 4), RT row tiles (RT * NT <= 4).  Src:
//   length()                 K
//   Tile tile(int)           what copying a tile's rows needs
//   rows(Tile, k, p, valid)  addresses at element k of rows (lane / 8) + 4 i, i < 4, and a bit for each that exists (every
//                            address has to be readable for k < K)
//   tokens(k, two, j, x0, x1) column 8 j + g at elements k + 8 t and, with `two`, k + 32 + 8 t (zeros otherwise: that
//                            half is the next warp's, and 0 x inf must not appear here)
//   fin(tile, row, col, sum) one output; sum(row, col) adds the partials
// FROWS outputs per column and tile (16, or 8 where rows g and g + 8 belong to
// one output), `cols` columns.
template <typename T, int NT, int RT, int FROWS, class Src>
struct Streamer {
  static constexpr int D = kSlots, PD = D / RT;  // steps ahead
  static_assert(RT * NT <= 4, "partials");
  using Tile = typename Src::Tile;
  const Src& src;
  uint32_t ring;      // the warp's ring
  float* part;
  int halves, steps;  // of K; the warp's steps
  int tiles;
  int lb, ls;         // next to load: first tile of its round, step
  Tile lt[RT];
  uint4 first[NT][2]; // token fragments of the first step: the same in every round

  MOE_DEV Streamer(const Src& source, unsigned char* smem) : src(source) {
    ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + (threadIdx.x >> 5) * (D * kStepBytes);
    part = reinterpret_cast<float*>(smem + kSW * D * kStepBytes);
  }

  MOE_DEV void load_round() {
#pragma unroll
    for (int i = 0; i < RT; ++i) lt[i] = src.tile(min(lb + i, tiles - 1));
  }

  // Where this lane's pieces of step s are: element offset (0 where there is
  // nothing to copy), and whether there is.
  struct At {
    int k;
    uint32_t bytes;
  };
  MOE_DEV At at_step(int s) const {
    const int piece = threadIdx.x & 7, k = 32 * half_at(s) + 8 * piece;
    const bool ok = (piece < 4 || both(s)) && k < src.length();
    return {ok ? k : 0, ok ? 16u : 0u};
  }
  // Slot i of the ring's `turn`: one group, empty past the last tile, so that the groups count the slots.
  MOE_DEV void load(const At& at, int turn, int i) {
    if (lb + i < tiles) {
      const int lane = threadIdx.x & 31, piece = lane & 7, row = lane >> 3;
      const uint32_t dst = ring + (turn * RT + i) * kStepBytes + row * 128 + ((piece ^ ((row & 1) << 2)) << 4);
      const uint16_t* p[4];
      uint32_t valid;
      src.rows(lt[i], at.k, p, valid);
#pragma unroll
      for (int r = 0; r < 4; ++r) copy16(dst + r * 512, p[r], (valid >> r & 1u) ? at.bytes : 0u);
    }
    copy_commit();
  }
  // First half of this warp's step s (the last step shares out what is left, one
  // half a warp if that is enough), and whether the step has a second.
  MOE_DEV int half_at(int s) const {
    const int w = threadIdx.x >> 5, base = 2 * kSW * s, left = halves - base;
    if (left >= 2 * kSW) return base + 2 * w;
    const int twos = max(left - kSW, 0);
    return base + (w < twos ? 2 * w : twos + w);
  }
  MOE_DEV bool both(int s) const {
    const int w = threadIdx.x >> 5, left = halves - 2 * kSW * s;
    return left >= 2 * kSW || w < left - kSW;
  }
  MOE_DEV void fetch(int s, uint4 (&x)[NT][2]) const {
    const int k = 32 * half_at(s);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      src.tokens(k, both(s), j, x[j][0], x[j][1]);
    }
  }
  MOE_DEV void next_step() {
    if (++ls == steps) {
      ls = 0;
      lb += RT;
      if (lb < tiles) load_round();
    }
  }

  MOE_DEV void prologue(int n_tiles) {
    halves = (src.length() + 31) / 32;
    const int w = threadIdx.x >> 5, full = halves / (2 * kSW);
    steps = full + (halves - 2 * kSW * full > w ? 1 : 0);
    tiles = n_tiles;
    lb = ls = 0;
#pragma unroll
    for (int j = 0; j < NT; ++j) first[j][0] = first[j][1] = make_uint4(0, 0, 0, 0);
    if (steps == 0 || tiles == 0) return;
    fetch(0, first);  // ahead of the weights, or it would queue behind 128 KB of them (3.6 us at the start of a kernel)
    load_round();
#pragma unroll
    for (int p = 0; p < PD; ++p) {
      const At at = at_step(ls);
#pragma unroll
      for (int i = 0; i < RT; ++i) load(at, p, i);
      next_step();
    }
  }

  // `ahead` runs once the last step is consumed, before the partials are added: the next stage's first copies.
  template <class Fin, class Ahead>
  MOE_DEV void run(int cols, const Fin& fin, const Ahead& ahead) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const uint32_t frag0 = g * 128 + ((t4 ^ ((g & 1) << 2)) << 4);      // first half of row g in a step
    const uint32_t frag1 = g * 128 + ((t4 ^ 4 ^ ((g & 1) << 2)) << 4);  // second half
    int turn = 0;
    for (int base = 0; base < tiles; base += RT) {
      float acc[RT][NT][4];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.0f;
      uint4 next[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        next[j][0] = first[j][0];
        next[j][1] = first[j][1];
      }
#pragma unroll 1
      for (int s = 0; s < steps; ++s) {
        uint4 x[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          x[j][0] = next[j][0];
          x[j][1] = next[j][1];
        }
        if (s + 1 < steps) fetch(s + 1, next);
        const At at = at_step(ls);
        // Two slots at a time where there are two: their reads and mma chains overlap,
        // and one pair of warp barriers serves both.
        constexpr int P = RT >= 2 ? 2 : 1;
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
          // a slot past the last tile holds an earlier tile's bytes: its sums are never read
#pragma unroll
          for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int q = 0; q < P; ++q) T::mma(acc[i + q][j], a0[q].x, b0[q].x, a0[q].y, b0[q].y, x[j][0].x, x[j][0].y);
#pragma unroll
            for (int q = 0; q < P; ++q) T::mma(acc[i + q][j], a0[q].z, b0[q].z, a0[q].w, b0[q].w, x[j][0].z, x[j][0].w);
#pragma unroll
            for (int q = 0; q < P; ++q) T::mma(acc[i + q][j], a1[q].x, b1[q].x, a1[q].y, b1[q].y, x[j][1].x, x[j][1].y);
#pragma unroll
            for (int q = 0; q < P; ++q) T::mma(acc[i + q][j], a1[q].z, b1[q].z, a1[q].w, b1[q].w, x[j][1].z, x[j][1].w);
          }
          __syncwarp();  // every lane has read the slots
#pragma unroll
          for (int q = 0; q < P; ++q) load(at, turn, i + q);
        }
        next_step();
        turn = turn + 1 == PD ? 0 : turn + 1;
      }
      const int nt = min(RT, tiles - base);
      if (base + RT >= tiles) ahead();
      if (base > 0) __syncthreads();  // the last round's partials have been added
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        if (i < nt) {
          float* p = part + (i * kSW + warp) * (NT * kPartTile) + 2 * t4 * kPartCol + g;
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            float* q = p + j * kPartTile;
            q[0] = acc[i][j][0];
            q[kPartCol] = acc[i][j][1];
            q[8] = acc[i][j][2];
            q[kPartCol + 8] = acc[i][j][3];
          }
        }
      }
      __syncthreads();
      // o = (tile, column, row); o / cols by a 16-bit reciprocal, exact while (o / FROWS) cols < 2^16 (at most 4 x 32 x 32)
      const uint32_t inverse = 65536u / static_cast<uint32_t>(cols) + 1u;
      for (int o = threadIdx.x; o < nt * cols * FROWS; o += kSThreads) {
        const int oc = o / FROWS, row = o % FROWS, tl = static_cast<int>((oc * inverse) >> 16), col = oc - tl * cols;
        fin(base + tl, row, col, [&](int r, int c) {
          const float* p = part + tl * kSW * (NT * kPartTile) + (c >> 3) * kPartTile + (c & 7) * kPartCol + r;
          float v = 0.0f;
#pragma unroll
          for (int w = 0; w < kSW; ++w) v += p[w * (NT * kPartTile)];
          return v;
        });
      }
    }
  }
};

}  // namespace dense
}  // namespace moe
