// dense_stream.cuh — streaming a block's weight rows past a few token columns
// on the warp-level tensor cores.
//
// With a handful of tokens a projection is bound by reading its weights once.
// A block owns a range of weight rows, cut into tiles of 16 (the mma's M;
// tokens are its N, 8 per column tile).  The 16 warps split K evenly, in halves
// of 32 elements, and each walks its part in steps of 64 elements; for a step
// it takes up to RT tiles one after the other, so a token fragment is loaded
// once for RT weight tiles (loading it for every tile cost 8 of 31 us at 118
// MB of weights and 7 tokens: those loads queue behind the weights').  Lane
// (g, t) feeds the mma with 8 consecutive elements at 8 t and at 32 + 8 t of
// rows g and g + 8 (A) and of token column g (B): an mma is unchanged by a
// permutation of K that both operands share, so nothing is shuffled.
//
// Weights in flight: a warp copies a step's 16 rows x 128 bytes of each tile
// into its own ring of D = PD x RT slots in shared memory with cp.async, whole
// 128-byte lines at a time, PD steps ahead, and waits for its own copies only;
// 16 warps x D x 2 KB = 128 KB per SM are under way (6.5 TB/s x 1 us / 148 SMs
// is 44 KB).  Rows are stored with the 64-byte halves of odd rows swapped, so
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

// 16 bytes global -> shared, past L1; zeros where !take (nothing is read then).
MOE_DEV void copy16(uint32_t dst, const uint16_t* src, bool take) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
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
// Written by other blocks of the same launch: from L2, where they are coherent.
MOE_DEV uint4 ld_l2(const uint16_t* p) {
  uint4 r;
  asm volatile("ld.global.cg.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
  return r;
}

constexpr int kStepBytes = 2048;  // 16 rows x 64 elements

constexpr int kSlots = 4;  // of a warp's ring

// Tiles a warp keeps in registers when its block has `tiles`: as many as share
// a token fragment, but no more than there are, since a ring slot of a tile
// that does not exist is a copy less in flight (2048 x 2048, one token: 4.0 us,
// with slots for four tiles where there is one 5.0).
template <int NT>
inline int tiles_at_once(int tiles) {
  const int most = kSlots / NT;
  return tiles >= 3 && most >= 4 ? 4 : tiles >= 2 && most >= 2 ? 2 : 1;
}
// Dynamic shared memory of a Streamer: the ring of four slots a warp, then the partials.
constexpr size_t kStreamBytes = static_cast<size_t>(kSW) * kSlots * kStepBytes + sizeof(float) * 4 * kSW * kPartTile;

// NT column tiles of 8 tokens (1, 2 or 4), RT row tiles (RT * NT <= 4).  Src:
//   halves()                  K in halves of 32 elements; kWhole: a warp's part starts on an even half
//   Tile tile(int)            what copying a tile's rows needs, rows (lane / 8) + 4 i
//   Step step(int half)       what a step needs: where it is in K
//   row(Tile, Step, i, p, n)  row i's address at the step's first element (null: zeros), elements from there to its end
//   tokens(Step, j, x0, x1)   column 8 j + g at 8 t and 32 + 8 t of the step (zeros outside)
//   fin(tile, row, col, sum)  one output; sum(row, col) adds the partials
// FROWS outputs per column and tile (16, or 8 where rows g and g + 8 belong to
// one output), `cols` columns.
template <typename T, int NT, int RT, int FROWS, class Src>
struct Streamer {
  static constexpr int D = kSlots, PD = D / RT;  // steps ahead
  static_assert(RT * NT <= 4, "partials");
  using Tile = typename Src::Tile;
  using Step = typename Src::Step;
  const Src& src;
  uint32_t ring;      // the warp's ring
  float* part;
  int h0, h1, steps;  // the warp's halves and steps
  int tiles;
  int lb, ls;         // next to load: first tile of its round, step
  Tile lt[RT];

  MOE_DEV Streamer(const Src& source, unsigned char* smem) : src(source) {
    ring = static_cast<uint32_t>(__cvta_generic_to_shared(smem)) + (threadIdx.x >> 5) * (D * kStepBytes);
    part = reinterpret_cast<float*>(smem + kSW * D * kStepBytes);
  }

  MOE_DEV void load_round() {
#pragma unroll
    for (int i = 0; i < RT; ++i) lt[i] = src.tile(min(lb + i, max(tiles - 1, 0)));
  }

  // Slot i of the ring's `turn`: one group, empty past the last tile, so that the groups count the slots.
  MOE_DEV void load(const Step& at, bool both, int turn, int i) {
    if (lb + i < tiles) {
      const int lane = threadIdx.x & 31, piece = lane & 7, row = lane >> 3;
      const uint32_t dst = ring + (turn * RT + i) * kStepBytes + row * 128 + ((piece ^ ((row & 1) << 2)) << 4);
      const bool mine = piece < 4 || both;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint16_t* p;
        int n;
        src.row(lt[i], at, r, p, n);
        const bool take = p != nullptr && 8 * piece < n && mine;
        copy16(dst + r * 512, take ? p + 8 * piece : src.any(), take);
      }
    }
    copy_commit();
  }
  // The second half of a warp's last step may belong to the next warp.
  MOE_DEV bool both(int s) const { return h0 + 2 * s + 1 < h1; }
  MOE_DEV void next_step() {
    if (++ls == steps) {
      ls = 0;
      lb += RT;
      if (lb < tiles) load_round();
    }
  }

  MOE_DEV void prologue(int n_tiles) {
    const int warp = threadIdx.x >> 5, halves = src.halves();
    h0 = static_cast<int>(static_cast<int64_t>(halves) * warp / kSW);
    h1 = static_cast<int>(static_cast<int64_t>(halves) * (warp + 1) / kSW);
    if constexpr (Src::kWhole) {
      h0 = (h0 + 1) & ~1;
      h1 = warp == kSW - 1 ? halves : (h1 + 1) & ~1;
    }
    steps = h1 > h0 ? (h1 - h0 + 1) / 2 : 0;
    tiles = n_tiles;
    lb = ls = 0;
    if (steps == 0) return;
    load_round();
#pragma unroll
    for (int p = 0; p < PD; ++p) {
      const Step at = src.step(h0 + 2 * ls);
#pragma unroll
      for (int i = 0; i < RT; ++i) load(at, both(ls), p, i);
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
      auto fetch = [&](int s) {
        const Step at = src.step(h0 + 2 * s);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          src.tokens(at, j, next[j][0], next[j][1]);
          if (!both(s)) next[j][1] = make_uint4(0, 0, 0, 0);  // the next warp's half: 0 x inf must not appear here
        }
      };
      if (steps > 0) fetch(0);
#pragma unroll 1
      for (int s = 0; s < steps; ++s) {
        uint4 x[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          x[j][0] = next[j][0];
          x[j][1] = next[j][1];
        }
        if (s + 1 < steps) fetch(s + 1);
        const Step at = src.step(h0 + 2 * ls);
        const bool whole = both(ls);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          copy_wait<D - 1>();
          __syncwarp();
          const uint32_t from = ring + (turn * RT + i) * kStepBytes;
          const uint4 a0 = ld_shared(from + frag0), b0 = ld_shared(from + frag0 + 1024);
          const uint4 a1 = ld_shared(from + frag1), b1 = ld_shared(from + frag1 + 1024);
          // a slot past the last tile holds an earlier tile's bytes: its sums are never read
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            T::mma(acc[i][j], a0.x, b0.x, a0.y, b0.y, x[j][0].x, x[j][0].y);
            T::mma(acc[i][j], a0.z, b0.z, a0.w, b0.w, x[j][0].z, x[j][0].w);
            T::mma(acc[i][j], a1.x, b1.x, a1.y, b1.y, x[j][1].x, x[j][1].y);
            T::mma(acc[i][j], a1.z, b1.z, a1.w, b1.w, x[j][1].z, x[j][1].w);
          }
          __syncwarp();  // every lane has read the slot
          load(at, whole, turn, i);
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
      const int per = FROWS * cols;
      for (int o = threadIdx.x; o < nt * per; o += kSThreads) {
        const int tl = o / per, rc = o - tl * per, col = rc / FROWS, row = rc % FROWS;
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
