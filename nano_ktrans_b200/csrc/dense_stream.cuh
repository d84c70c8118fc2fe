// dense_stream.cuh — streaming a block's weight rows past a few token columns
// on the warp-level tensor cores.
//
// With a handful of tokens a projection is bound by reading its weights once.
// A block owns a range of weight rows, cut into tiles of 16 (the mma's M;
// tokens are its N, 8 per column tile).  K is cut into units of 64 elements,
// and step s = tile * units + unit goes to warp s % 16: every warp has the same
// number of steps to within one, whatever the sizes.  In a step lane (g, t) of
// a warp takes 8 consecutive elements at 8 t and at 32 + 8 t of rows g and g + 8
// as the mma's A registers and the same K positions of token column g as B: an
// mma is unchanged by a permutation of K that both operands share, so nothing
// is shuffled.
//
// Weights in flight: every lane copies its own four 16-byte pieces of a step
// into a ring of D steps in shared memory with cp.async and reads back what it
// copied itself, so the ring needs no barrier between threads; 16 warps x D x
// 2 KB = 128 KB per SM are under way (6.5 TB/s x 1 us / 148 SMs is 44 KB).
// Loading straight into registers instead kept one step in flight, not D: the
// hardware's scoreboards were shared between the loads (118 MB of weights, 7
// tokens: 29.5 us; every step of a warp waited out a whole memory latency).
//
// Partial sums: a warp adds up its steps of a tile in registers, puts the
// 16 x 8 partial tiles into shared memory, and once per round of tiles the
// block adds the 16 partials of each output in warp order (no atomics: the
// same bits every run).  Partials are double buffered, and the next round's
// copies are in flight meanwhile.
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

// Tiles whose partials one round holds.
template <int NT>
constexpr int round_tiles() {
  return NT == 1 ? 2 : 1;
}
template <int NT>
constexpr int part_floats() {
  return 2 * round_tiles<NT>() * kSW * NT * kPartTile;
}
// Dynamic shared memory of a Streamer: the ring, then the partials.
template <int NT, int D>
constexpr size_t stream_bytes() {
  return static_cast<size_t>(kSW) * D * kStepBytes + sizeof(float) * part_floats<NT>();
}

// NT column tiles of 8 tokens, D steps in flight.
//   src.rows(tile, unit, pa, pb, len)  rows g and g + 8 of the tile at the unit's first element (null: zeros), and the
//                                      elements from there to the end of the row
//   src.tokens(unit, j, x0, x1)        column 8 j + g at 8 t and 32 + 8 t of the unit (zeros outside)
//   fin(tile, row, col, sum)           one output; sum(row, col) adds the partials
// FROWS outputs per column and tile (16, or 8 where rows g and g + 8 belong to
// one output), `cols` columns.
template <typename T, int NT, int D, int FROWS>
struct Streamer {
  static constexpr int R = round_tiles<NT>();
  uint32_t ring;  // this lane's 16 bytes of the warp's first piece
  float* part;
  int lt, lu;     // next step to load

  MOE_DEV explicit Streamer(unsigned char* smem) {
    const uint32_t base = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    ring = base + (threadIdx.x >> 5) * (D * kStepBytes) + (threadIdx.x & 31) * 16;
    part = reinterpret_cast<float*>(smem + kSW * D * kStepBytes);
  }

  static MOE_DEV void step(int& t, int& u, int units) {
    u += kSW;
    while (u >= units) {
      u -= units;
      ++t;
    }
  }

  // One group, empty past the last step, so that the groups count the steps.
  template <class Src>
  MOE_DEV void load(const Src& src, int slot, int tiles, int units) {
    if (lt < tiles) {
      const uint16_t *pa, *pb;
      int len;
      src.rows(lt, lu, pa, pb, len);
      const int t8 = 8 * (threadIdx.x & 3);
      const uint32_t dst = ring + slot * kStepBytes;
      const uint16_t* safe = src.any();
      const bool in0 = t8 < len, in1 = 32 + t8 < len;
      copy16(dst, pa != nullptr && in0 ? pa + t8 : safe, pa != nullptr && in0);
      copy16(dst + 512, pb != nullptr && in0 ? pb + t8 : safe, pb != nullptr && in0);
      copy16(dst + 1024, pa != nullptr && in1 ? pa + 32 + t8 : safe, pa != nullptr && in1);
      copy16(dst + 1536, pb != nullptr && in1 ? pb + 32 + t8 : safe, pb != nullptr && in1);
      step(lt, lu, units);
    }
    copy_commit();
  }

  template <class Src>
  MOE_DEV void prologue(const Src& src, int tiles, int units) {
    lt = 0;
    lu = (threadIdx.x >> 5) - kSW;
    step(lt, lu, units);
#pragma unroll
    for (int i = 0; i < D; ++i) load(src, i, tiles, units);
  }

  template <class Src, class Fin>
  MOE_DEV void run(const Src& src, int tiles, int units, int cols, const Fin& fin) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    int ct = 0, cu = warp - kSW;
    step(ct, cu, units);
    float acc[NT][4];
    int cur = -1, round = 0, slot = 0;
    auto place = [&](int tile, int w) {
      return part + static_cast<size_t>((((tile / R) & 1) * R + tile % R) * kSW + w) * (NT * kPartTile);
    };
    auto flush = [&]() {
      if (cur < 0) return;
      float* p = place(cur, warp);
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
          const float* p = place(tile, 0) + (c >> 3) * kPartTile + (c & 7) * kPartCol + r;
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
      if (ct != cur) {
        flush();
        cur = ct;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[j][c] = 0.0f;
        while (ct >= (round + 1) * R) end_round();
      }
      uint4 x[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) src.tokens(cu, j, x[j][0], x[j][1]);
      copy_wait<D - 1>();
      const uint32_t from = ring + slot * kStepBytes;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 wa = ld_shared(from + 1024 * h), wb = ld_shared(from + 1024 * h + 512);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          T::mma(acc[j], wa.x, wb.x, wa.y, wb.y, x[j][h].x, x[j][h].y);
          T::mma(acc[j], wa.z, wb.z, wa.w, wb.w, x[j][h].z, x[j][h].w);
        }
      }
      load(src, slot, tiles, units);
      slot = slot + 1 == D ? 0 : slot + 1;
      step(ct, cu, units);
    }
    flush();
    while (round * R < tiles) end_round();
  }
};

}  // namespace dense
}  // namespace moe
