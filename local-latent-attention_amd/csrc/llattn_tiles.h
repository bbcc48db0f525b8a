// What the products over 64-k steps of the head loss (llattn_head.hip) and of the gated feed-forward (llattn_gated.hip)
// share: the shapes of workgroups, operands in LDS, and which shape and how many splits a product takes.
#pragma once

#include <algorithm>

#include "llattn_gemm.h"

namespace llattn {
namespace tiles {

using namespace gemm;

// A shape of workgroup: WR x WC waves, each 16 MB x 16 NB of the tile, NST LDS stages of 64 k.
template <int MB_, int NB_, int WR_, int WC_, int NST_>
struct Shape {
  static constexpr int MB = MB_, NB = NB_, WR = WR_, WC = WC_, NST = NST_;
  static constexpr int W = WR * WC, THREADS = 64 * W, TM = 16 * MB * WR, TN = 16 * NB * WC, STAGE = (TM + TN) * 128;
};

// T rows of a step with its 64 k along them (128 bytes each), loaded by W waves.  Chunk c (8 k) of row o at c ^ swz(o).
// PERM: lane r of fragment block j reads row 32 (j / 2) + 4 (j % 2) + 8 (r / 4) + r % 4, so that as the first operand a pair of
// blocks gives each lane 8 consecutive columns of the product.
template <int T, int W, bool PERM>
struct RowOp {
  static constexpr int BYTES = T * 128, LOADS = BYTES / 1024 / W;
  uint32_t off[LOADS], base[2];  // base: of this lane's fragments, by 32-k half
  int kc[LOADS];                 // first k of this lane's chunks
  __device__ __forceinline__ void init(int64_t ld, int w, int lane, int o0) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = 8 * (w * LOADS + i) + (lane >> 3), c = (lane & 7) ^ pswz<PERM>(row);
      off[i] = step_off((int64_t)row * ld * 2 + 16 * c);
      kc[i] = 8 * c;
    }
    const int r = lane & 15, g = lane >> 4, row = PERM ? 8 * (r >> 2) + (r & 3) : r;
#pragma unroll
    for (int h = 0; h < 2; ++h) base[h] = (o0 + row) * 128 + (((4 * h + g) ^ pswz<PERM>(row)) << 4);
  }
  // load i of a step with `left` k to the contraction's end: chunks past it read zero
  __device__ __forceinline__ uint32_t at(int i, int left) const { return kmask(off[i], kc[i], left); }
  // rows o0 + 16 i + r (PERM: as above), k 32 half + 8 g .. of the stage at st; o0 a multiple of 32
  __device__ __forceinline__ bf16x8 frag(const unsigned char* st, int i, int half) const {
    // PERM: the swizzle's third bit is bit 3 of the row and its low two those of r, so 4 and 32 rows on leave it alone
    return *reinterpret_cast<const bf16x8*>(st + base[half] + (PERM ? (i >> 1) * 4096 + (i & 1) * 512 : i * 2048));
  }
};

// 64 k-rows of a step, T columns of them (2 T bytes each).  Chunk c (8 columns) of k-row k at c ^ swz(k): the 32 lanes
// that read at a time (eight k-rows of 16 columns) take 16 different chunks of 256 bytes.
template <int T, int W>
struct ColOp {
  static constexpr int BYTES = T * 128, LOADS = BYTES / 1024 / W, PER = T / 8;
  uint32_t off[LOADS], base[4];  // base: by the 16-column block's place in its four
  static __device__ __forceinline__ int swz(int k) { return 2 * (k & 3) + 8 * ((k >> 3) & 1); }
  __device__ __forceinline__ void init(int64_t ld, int w, int lane, int o0) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int q = (w * LOADS + i) * 64 + lane, k = q / PER;
      off[i] = step_off((int64_t)k * ld * 2 + 16 * ((q % PER) ^ swz(k)));
    }
    // transposing reads: the 16 lanes of group g supply k-rows 8 g + r / 4 (and 4 further), 8 bytes at column 4 (r % 4)
    const int r = lane & 15, g = lane >> 4, k = 8 * g + (r >> 2);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int byte = 2 * (o0 + 16 * u) + 8 * (r & 3);  // o0 is a multiple of 64: the swizzle stays within 128 columns
      base[u] = k * (2 * T) + (((byte >> 4) ^ swz(k)) << 4) + (byte & 15);
    }
  }
  __device__ __forceinline__ uint32_t at(int i, int) const { return off[i]; }  // k-rows past the end lie past the extent
  // columns o0 + 16 j + r, k 32 half + 8 g ..
  __device__ __forceinline__ bf16x8 frag(const unsigned char* st, int j, int half) const {
    bf16x4 hv[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      // blocks j >= 4 lie 128 bytes further: bit 3 of their chunk is that of base's flipped
      const unsigned char* p = st + (base[j & 3] ^ ((j >> 2) << 7)) + (32 * half + 4 * q) * (2 * T);
      hv[q] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(p));
    }
    return bf16x8{hv[0][0], hv[0][1], hv[0][2], hv[0][3], hv[1][0], hv[1][1], hv[1][2], hv[1][3]};
  }
};

constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Workgroups: tiles of 64 x 128, 128 x 128 and 256 x 256.
enum Kind { THIN = 0, SQUARE = 1, BIG = 2, KINDS = 3 };
typedef Shape<2, 4, 2, 2, 3> ThinShape;
typedef Shape<4, 4, 2, 2, 2> SquareShape;
typedef Shape<4, 8, 4, 2, 2> BigShape;
constexpr int kTm[KINDS] = {64, 128, 256}, kTn[KINDS] = {128, 128, 256}, kPerCu[KINDS] = {2, 2, 1};
// us of a 64-k step of a workgroup with 1 or 2 of them on a CU, and of a tile beside its steps.  Products alone, us (taken: *;
// S: splits):
//                            64 x 128   128 x 128                256 x 256
//   64 x 128 x 509       l     5.2 *      6.2                      9.4
//   512 x 256 x 4000     l     6.0        7.2 *                   12.5     (64 x 128 is for up to 64 rows)
//                        dh               35 S 1, 13 S 4           71 S 1  (* 128, S 13)
//                        dW               7.4 *                   15.0
//   333 x 1408 x 50257   l    71.8       55.4 *                   65.4
//                        dh              118 S 4, 68 S 8, 50 S 15 * 222 S 4, 120 S 8
//                        dW              75.4                     76.2 *
//   2048 x 1408 x 131072 l               753                      583 *
//   4096 x 1408 x 32000  l               331                      293 *
//                        q               416                      306 *
//                        dh              413 S 1                  605 S 1, 334 S 2, 488 S 3, 355 S 5 *
//                        dW              342                      317 *
//   8192 x 1536 x 32768  l               719                      622 *
//                        q               844                      654 *
//                        dh              878 S 1                  698 S 1, 749 S 2, 620 S 4 *
//                        dW              739                      623 *
// The model misses the best by 6% in dh of 4096 x 1408 x 32000 and by 1 us at 512 rows.
constexpr double kStep[KINDS][2] = {{0.45, 0.60}, {0.60, 1.00}, {1.55, 1.55}};
constexpr double kTile[KINDS] = {5.0, 6.0, 10.0};

struct Tiling { int kind, splits; double us; };

// The tiles of an M x N product over `steps` 64-wide k steps, and the splits of its contraction (at most `most`): the least
// expected time, in rounds of whole tiles over the 256 CUs, the partial sums written and read at 4.5 TB/s.
constexpr Tiling tiling(int64_t M, int64_t N, int steps, int most) {
  Tiling best{SQUARE, 1, 1e30};
  for (int kind = M <= 64 ? THIN : SQUARE; kind < KINDS; ++kind) {
    if (most > 1 && kind == THIN) continue;  // gradients: 128 x 128 and larger
    const int64_t tiles = ceil_div(M, kTm[kind]) * ceil_div(N, kTn[kind]), slots = 256 * kPerCu[kind];
    for (int S = 1; S <= most && (S == 1 || steps / S >= 4); ++S) {
      const int64_t n = tiles * S, rest = n % slots;
      const double per = (double)ceil_div(steps, S);
      double t = (double)(n / slots) * (per * kStep[kind][kPerCu[kind] - 1] + kTile[kind]);
      if (rest) t += per * kStep[kind][rest > 256 ? 1 : 0] + kTile[kind];
      if (S > 1) t += 6.0 + 8.0 * S * (double)M * (double)N / 4.5e6;
      if (t < best.us) best = Tiling{kind, S, t};
    }
  }
  return best;
}

}  // namespace tiles
}  // namespace llattn
