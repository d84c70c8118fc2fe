// dense_stream.cuh — streaming a block's weight rows past a few token columns
// on the warp-level tensor cores.
//
// With a handful of tokens a projection is bound by reading its weights once.
// A block owns a range of weight rows, cut into tiles of 16 (the mma's M;
// tokens are its N, 8 per column tile).  K is cut into units of 4 * VEC
// elements, and step s = tile * units + unit goes to warp s % 16: every warp
// has the same number of steps to within one, whatever the sizes.  In a step
// lane (g, t) of a warp takes VEC consecutive elements at unit + t * VEC of
// rows g and g + 8, straight from global memory into mma A registers, and the
// same K positions of token column g into B registers: an mma is unchanged by
// a permutation of K that both operands share, so nothing is staged in shared
// memory or shuffled.  Each warp keeps D steps of weights in flight in
// registers (512 threads x 4 x 64 bytes = 128 KB per SM, about three times
// what 6.5 TB/s x 1 us / 148 needs).
//
// Partial sums: a warp adds up its steps of a tile in registers, puts the
// 16 x 8 partial tiles into shared memory, and once per round of tiles the
// block adds the 16 partials of each output in warp order (no atomics: the
// same bits every run).  Partials are double buffered, and the next round's
// loads are in flight meanwhile.
#pragma once

#include "dense_common.cuh"

namespace moe {
namespace dense {

constexpr int kSW = 16;                 // warps of a block
constexpr int kSThreads = 32 * kSW;
constexpr int kPartCol = 20;            // floats per column of a partial tile: 16 rows, padded so that the 8 x 4 lanes
                                        // of a store fall into different banks
constexpr int kPartTile = 8 * kPartCol;

// Weights are read once: they pass L1 by.
MOE_DEV void ld_weights(uint32_t (&r)[8], const uint16_t* p) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}
MOE_DEV void ld_weights(uint32_t (&r)[4], const uint16_t* p) {
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "l"(p));
}
// Activations are read by every tile: through L1.
MOE_DEV void ld_tokens(uint32_t (&r)[8], const uint16_t* p) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}
MOE_DEV void ld_tokens(uint32_t (&r)[4], const uint16_t* p) {
  asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "l"(p));
}
// Written by other blocks of the same launch: from L2, where they are coherent.
MOE_DEV void ld_l2(uint32_t (&r)[8], const uint16_t* p) {
  asm volatile("ld.global.cg.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}
template <int N>
MOE_DEV void zero(uint32_t (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = 0;
}

// Tiles whose partials one round holds (per buffer: R * 16 * NT * 640 bytes).
template <int NT>
constexpr int round_tiles() {
  return NT >= 4 ? 1 : 4 / NT;
}
template <int NT>
constexpr size_t part_bytes() {
  return sizeof(float) * 2 * round_tiles<NT>() * kSW * NT * kPartTile;
}

// NT column tiles of 8 tokens, VEC elements per lane and row, D steps in flight.
//   src.load(tile, unit, a, b)   rows g and g + 8 of the tile (zero outside)
//   src.tokens(unit, j, x)       column 8 j + g (zero outside)
//   fin(tile, row, col, sum)     one output; sum(row, col) adds the partials
// FROWS outputs per column and tile (16, or 8 where rows g and g + 8 belong to
// one output), `cols` columns.
template <typename T, int NT, int VEC, int D, int FROWS>
struct Streamer {
  static constexpr int R = round_tiles<NT>();
  uint32_t fa[D][VEC / 2], fb[D][VEC / 2];
  int lt, lu;  // next step to load

  MOE_DEV void step(int& t, int& u, int units) const {
    u += kSW;
    while (u >= units) {
      u -= units;
      ++t;
    }
  }

  template <class Src>
  MOE_DEV void prologue(const Src& src, int tiles, int units) {
    lt = 0;
    lu = (threadIdx.x >> 5) - kSW;
    step(lt, lu, units);
#pragma unroll
    for (int i = 0; i < D; ++i)
      if (lt < tiles) {
        src.load(lt, lu, fa[i], fb[i]);
        step(lt, lu, units);
      }
  }

  template <class Src, class Fin>
  MOE_DEV void run(const Src& src, int tiles, int units, int cols, const Fin& fin, float* part) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    int ct = 0, cu = warp - kSW;
    step(ct, cu, units);
    float acc[NT][4];
    int cur = -1, round = 0;
    auto slot = [&](int tile, int w) {
      return part + static_cast<size_t>((((tile / R) & 1) * R + tile % R) * kSW + w) * (NT * kPartTile);
    };
    auto flush = [&]() {
      if (cur < 0) return;
      float* p = slot(cur, warp);
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float* q = p + j * kPartTile + 2 * t4 * kPartCol + g;
        q[0] = acc[j][0];
        q[kPartCol] = acc[j][1];
        q[8] = acc[j][2];
        q[kPartCol + 8] = acc[j][3];
      }
    };
    auto end_round = [&]() {
      __syncthreads();
      const int t0 = round * R, nt = min(R, tiles - t0), per = FROWS * cols;
      for (int i = threadIdx.x; i < nt * per; i += kSThreads) {
        const int tl = i / per, rc = i - tl * per, col = rc / FROWS, row = rc % FROWS, tile = t0 + tl;
        // warps that have a step of this tile: all of them once a tile has 16 units
        const int first = static_cast<int>((static_cast<int64_t>(tile) * units) % kSW);
        fin(tile, row, col, [&](int r, int c) {
          const float* p = slot(tile, 0) + (c >> 3) * kPartTile + (c & 7) * kPartCol + r;
          float s = 0.0f;
#pragma unroll
          for (int w = 0; w < kSW; ++w)
            if (units >= kSW || ((w - first + kSW) & (kSW - 1)) < units) s += p[w * (NT * kPartTile)];
          return s;
        });
      }
      ++round;
    };
    while (ct < tiles) {
#pragma unroll
      for (int i = 0; i < D; ++i) {
        if (ct < tiles) {
          if (ct != cur) {
            flush();
            cur = ct;
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;
            while (ct >= (round + 1) * R) end_round();
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            uint32_t x[VEC / 2];
            src.tokens(cu, j, x);
#pragma unroll
            for (int q = 0; q < VEC / 4; ++q)
              T::mma(acc[j], fa[i][2 * q], fb[i][2 * q], fa[i][2 * q + 1], fb[i][2 * q + 1], x[2 * q], x[2 * q + 1]);
          }
          if (lt < tiles) {
            src.load(lt, lu, fa[i], fb[i]);
            step(lt, lu, units);
          }
          step(ct, cu, units);
        }
      }
    }
    flush();
    while (round * R < tiles) end_round();
  }
};

}  // namespace dense
}  // namespace moe
