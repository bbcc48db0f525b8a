// Softmax cross entropy of h Wᵀ over a vocabulary of any size without keeping the logits (include/llattn_train.h).
//
//   l[n][v] = sum_d h[n][d] W[v][d],   lse[n] = log sum_v exp l[n][v],   loss[n] = lse[n] - l[n][t_n]
//   dl[n][v] = (exp(l[n][v] - lse[n]) - [v == t_n]) s_n,   dh = dl W,   dW = dlᵀ h
//
// Forward: a tile of l lives in the accumulators alone; its epilogue leaves, per row and wave, the maximum m of the
// wave's columns and the sum of exp(l - m), and the target's logit.  A second launch joins them:
//   M = max m,   S = sum (sum of the part) exp(m - M),   lse = M + log S.
// Exponentials run in base 2 on x = l log2(e): c = m log2(e) rounded once is subtracted from every term of a part and
// given back to the joined sum, so its rounding cancels; loss = ((C - l_t log2 e) + log2 S) ln 2 takes the small
// difference first.
//
// Backward: a piece of the vocabulary at a time, the same product again with q = softmax - onehot (bf16) in its epilogue,
// then dh (+)= q W and dW = qᵀ h, times the scale that every row shares.  q is bf16 because the matrix cores take 16 bits: off
// by half a step of 2^-8 of each entry, which averages out over the contraction.  What it leaves, with dW in fp32: 5e-5 of dW at
// 333 x 1408 x 50256, 1.7e-4 at 4096 x 256 x 8000, 1.5e-3 where single entries make up a row (333 x 128 x 512); results in
// bf16 are off by 1.7e-3 from their own rounding (2.2e-3 in the last case).  The shared scale stays
// out of q: within it, the entries near -1, which are one value in all rows, would round alike (1 / 4096 rows: 0.4% of
// the whole gradient).  Gradients row by row are divided by the largest of them, which is shared in the same way: rows
// of one gradient (a mean taken outside) then round as if there were none.  Their ratios to it are multiplied in.
//
// What bounds it: 2 rows V D operations for each of the four products on the matrix cores; with few rows the reads of
// W.
#include <algorithm>

#include "llattn_gemm.h"
#include "llattn_train.h"

namespace llattn {
namespace {

using namespace gemm;

enum Epilogue { STATS = 0, STATS_PRED = 1, GRAD = 2, SUM = 3, OUT_BF16 = 4, OUT_F32 = 5 };

struct HeadArgs {
  int M, N, K;              // rows, columns, contraction
  int steps, per;           // 64-wide k steps, of a split
  int tiles_m, tiles_n, total;  // total: with the splits
  const uint16_t* A; int64_t lda;
  const uint16_t* B; int64_t ldb;
  // logits
  int v0;                   // first column of the piece in the vocabulary
  int64_t V;                // targets outside [0, V) are errors
  const int64_t* targets;
  int64_t ignore_index;
  float2* part;             // STATS: parts [slots][M] and the target's logit [M]
  int32_t* part_i;
  float* tgt;
  const float* lse2;        // GRAD
  uint16_t* p; int64_t p_block; int p_cols;  // q, its columns and the elements of 64 of them
  // gradients: alpha = *scale * (inv ? *inv : 1) of the products, and grad[row] / *scale within q (grad null: 1)
  const float* grad;
  const float* scale;
  const float* inv;
  void* C;                  // SUM: fp32 [splits][M][N]
  int accumulate;
};

// (value, index) maximum with the smaller index on ties
__device__ __forceinline__ void max_first(float& m, int& i, float m2, int i2) {
  if (m2 > m || (m2 == m && i2 < i)) {
    m = m2;
    i = i2;
  }
}

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

// The same for q: 64 k-rows of T columns, whose blocks of 64 lie ld elements apart, a row of one in 128 bytes.
template <int T, int W>
struct BlockOp : ColOp<T, W> {
  using ColOp<T, W>::LOADS, ColOp<T, W>::PER, ColOp<T, W>::off;
  int k_of[LOADS];
  __device__ __forceinline__ void init(int64_t ld, int w, int lane, int o0) {
    ColOp<T, W>::init(0, w, lane, o0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int q = (w * LOADS + i) * 64 + lane, k = q / PER, c = (q % PER) ^ this->swz(k);
      off[i] = (uint32_t)((c >> 3) * ld * 2 + k * 128 + 16 * (c & 7));
      k_of[i] = k;
    }
  }
  __device__ __forceinline__ uint32_t at(int i, int left) const { return kmask(off[i], k_of[i], left); }
};

// Tiles of a product.  A 64-k step is two rounds of products, each beside the fragment reads of the next: k 0..31
// (reads k 32..63), a barrier, k 32..63 (reads the next step's k 0..31 and issues the loads of step kt + NST into the
// stage just read).  Waves whose part of the tile lies outside load and wait like the others and do nothing else.
// Offsets are taken from the tile's first row and step, so operands may be of any size.
//
// The logits' products take tile after tile (2048 x 1408 x 131072: 614 us, so 583); the gradients' one tile a workgroup
// (128 steps a tile of dW: the longer loop cost 586 -> 636 us a piece of 8192 x 1536 x 32768).
//
// Measured, 8192 rows, D 1536: l of 131072 columns 2420 us (1360 TFLOP/s), a piece of 32768 of them: q 683 us (1210; it
// writes 537 MB), dh 630 us (1310) and 680 where it adds to the piece's before, dW 604 us (1370).  256 x 256 tiles: matrix
// cores 59-68% busy at a clock of 1.9 GHz that these products themselves bring down.
template <int EPI, bool AT, bool BT, typename S, int WGS>
__global__ __launch_bounds__(S::THREADS, WGS * S::W / 4) void head_kernel(const HeadArgs a) {
  constexpr int MB = S::MB, NB = S::NB, TM = S::TM, TN = S::TN, NST = S::NST, STAGE = S::STAGE, W = S::W;
  constexpr bool LOSS = EPI == STATS || EPI == STATS_PRED || EPI == GRAD;  // else A is q, in blocks of 64 columns
  typedef std::conditional_t<AT, BlockOp<TM, W>, RowOp<TM, W, false>> OpA;
  typedef std::conditional_t<BT, ColOp<TN, W>, RowOp<TN, W, true>> OpB;
  constexpr int LOADS = OpA::LOADS + OpB::LOADS;
  static_assert(LOADS <= MB + NB, "the second round's reads carry the loads");
  static_assert((!AT || (16 * MB) % 64 == 0) && (!BT || (16 * NB) % 64 == 0), "ColOp::base");
  __shared__ __align__(1024) unsigned char smem[NST * STAGE];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  static_assert(S::WC == 2 && (S::WR == 2 || S::WR == 4), "wave layouts");
  // eight waves: those of one SIMD (w, w + 4) lie in opposite halves of both sides
  const int wm = W == 8 ? (w & 3) ^ (w >> 2 << 1) : w >> 1, wn = W == 8 ? (w & 1) ^ (w >> 2) : w & 1;
  // Workgroup b takes tiles b, b + gridDim.x, ... of the launch's order (its XCD's share of them, a run of the tiles).
  struct Tile { int m0, n0, split, steps; };  // steps: of the split (none or less: zeros)
  auto tile_at = [&](int v) {
    int t = xcd_remap(v, a.total);
    const int tiles = a.tiles_m * a.tiles_n, split = t / tiles;
    t -= split * tiles;
    constexpr int GM = 8;
    const int group = t / (GM * a.tiles_n), first_m = group * GM, gm = min(a.tiles_m - first_m, GM);
    const int tm = first_m + (t % (GM * a.tiles_n)) % gm, tn = t % (GM * a.tiles_n) / gm;
    const int steps = min(a.steps - split * a.per, a.per);
    return Tile{__builtin_amdgcn_readfirstlane(tm * TM), __builtin_amdgcn_readfirstlane(tn * TN),
                __builtin_amdgcn_readfirstlane(split), __builtin_amdgcn_readfirstlane(steps)};
  };
  OpA oa;
  OpB ob;
  oa.init(LOSS || AT ? a.lda : 64, w, lane, wm * 16 * MB);
  ob.init(a.ldb, w, lane, wn * 16 * NB);
  auto source = [&](const uint16_t* p, int64_t ld, bool t, int o, int n, int k0) {  // n of the operand's rows (t: columns) from o on
    StepSrc s;
    s.addr = reinterpret_cast<uint64_t>(p + (t ? o + (int64_t)k0 * 64 * ld : o * ld + (int64_t)k0 * 64));
    s.full = t ? extent_of(64, ld, n) : extent_of(n, ld, 64);  // not t: chunks past the last k are masked (RowOp::at)
    s.tail = t ? extent_of(a.K & 63 ? a.K & 63 : 64, ld, n) : s.full;
    s.inc = t ? (uint32_t)(128 * ld) : 128u;
    return s;
  };
  auto source_a = [&](const Tile& t) {
    const int n = min(TM, a.M - t.m0), k0 = t.split * a.per;
    if constexpr (LOSS) return source(a.A, a.lda, false, t.m0, n, k0);
    StepSrc s;
    s.addr = reinterpret_cast<uint64_t>(a.A + (AT ? t.m0 / 64 : k0) * a.lda + (AT ? (int64_t)k0 * 64 : t.m0) * 64);
    const uint32_t blocks = AT ? (uint32_t)((n - 1) / 64 * a.lda * 2) : 0;  // up to the last block's
    s.full = blocks + (AT ? 64 : n) * 128;
    s.tail = AT && a.K & 63 ? blocks + (a.K & 63) * 128 : s.full;
    s.inc = AT ? 64 * 128 : (uint32_t)(a.lda * 2);
    return s;
  };
  auto source_b = [&](const Tile& t) { return source(a.B, a.ldb, BT, t.n0, min(TN, a.N - t.n0), t.split * a.per); };
  auto k_of = [&](const Tile& t) { return min(a.K - t.split * a.per * 64, t.steps * 64); };
  int v = blockIdx.x;
  Tile tile = tile_at(v);
  StepSrc sa = source_a(tile), sb = source_b(tile);
  int ahead = k_of(tile);  // k from the step that ra and rb describe to the end of its tile's
  i32x4 ra = sa.rsrc(ahead, 64), rb = sb.rsrc(ahead, 64);
  auto advance = [&]() {
    sa.addr += sa.inc;
    sb.addr += sb.inc;
    ahead -= 64;
    ra = sa.rsrc(ahead, 64);
    rb = sb.rsrc(ahead, 64);
  };
  const uint32_t lds_a = __builtin_amdgcn_readfirstlane(lds_addr(smem) + w * OpA::LOADS * 1024);
  const uint32_t lds_b = __builtin_amdgcn_readfirstlane(lds_addr(smem) + OpA::BYTES + w * OpB::LOADS * 1024);
  auto load = [&](auto stage, auto q) {
    constexpr int s = decltype(stage)::value, n = decltype(q)::value;
    if constexpr (n < OpA::LOADS) dma_at<s * STAGE + n * 1024>(ra, oa.at(n, ahead), lds_a);
    else dma_at<s * STAGE + (n - OpA::LOADS) * 1024>(rb, ob.at(n - OpA::LOADS, ahead), lds_b);
  };
  bf16x8 a0[MB], a1[MB], b0[NB], b1[NB];  // k 0..31 and 32..63
  f32x4 acc[MB][NB];
  // MB NB products, B first: lane (r, g) accumulates C[r][4 g + e]; io(q), q < MB + NB, spread over them
  auto round = [&](const bf16x8 (&x)[MB], const bf16x8 (&y)[NB], auto io) {
    constexpr int N = MB + NB, P = MB * NB;
    unroll<N>([&](auto qt) {
      constexpr int q = decltype(qt)::value;
      io(qt);
#pragma unroll
      for (int n = q * P / N; n < (q + 1) * P / N; ++n)
        acc[n / NB][n % NB] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[n % NB], x[n / NB], acc[n / NB][n % NB], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // What the epilogue of a tile reads of the wave's rows, a row a lane: read ahead of it, it costs no latency there.
  int64_t read_tg = a.ignore_index;
  float read_l2 = 0.f;
  auto read_rows = [&](const Tile& t) {
    if constexpr (LOSS) {
      const int row = t.m0 + wm * 16 * MB + lane % (16 * MB);
      read_tg = a.ignore_index;
      read_l2 = 0.f;
      if (row < a.M) {
        read_tg = a.targets[row];
        if constexpr (EPI == GRAD) read_l2 = a.lse2[row];
      }
    }
  };
  float lane_l2 = 0.f;
  int lane_tc = -1;  // the target's column within the piece; -1: it has none, -2: an ignored row
  auto settle_rows = [&]() {
    if constexpr (LOSS) {
      const int64_t t = read_tg;
      lane_tc = t == a.ignore_index ? -2 : t >= a.v0 && t < a.v0 + a.N ? (int)(t - a.v0) : -1;
      lane_l2 = t != a.ignore_index && (t < 0 || t >= a.V) ? __builtin_nanf("") : read_l2;
    }
  };
  read_rows(tile);
  unroll<NST>([&](auto st) {
    if constexpr (decltype(st)::value > 0) advance();
    unroll<LOADS>([&](auto q) { load(st, q); });
  });
  __builtin_amdgcn_s_waitcnt(wait_vm((NST - 1) * LOADS));  // loads complete in issue order: step 0 has landed
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  auto first_frags = [&]() {
#pragma unroll
    for (int j = 0; j < NB; ++j) b0[j] = ob.frag(smem + OpA::BYTES, j, 0);
#pragma unroll
    for (int i = 0; i < MB; ++i) a0[i] = oa.frag(smem, i, 0);
  };
  bool own = tile.m0 + wm * 16 * MB < a.M && tile.n0 + wn * 16 * NB < a.N;  // part of the tile is this wave's
  if (own) first_frags();
  for (;;) {
    // The next tile's first steps are loaded, and its first fragments read, in this one's last steps: no step of the
    // pipeline waits for the epilogue between them.  A tile before another takes whole turns of the stages.
    const bool more = LOSS && v + (int)gridDim.x < a.total;
    const Tile next = more ? tile_at(v + gridDim.x) : tile;
    const StepSrc next_a = source_a(next), next_b = source_b(next);
    const int next_k = more ? k_of(next) : 0;
    const int steps = more ? (max(tile.steps, 1) + NST - 1) / NST * NST : tile.steps;
    const int row0 = tile.m0 + wm * 16 * MB, n0 = tile.n0, col0 = n0 + wn * 16 * NB, tn = n0 / TN;
    settle_rows();
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    int kt = 0;
    auto next_step = [&]() {
      if (LOSS && kt + NST == steps) {
        sa = next_a;
        sb = next_b;
        ahead = next_k;
        ra = sa.rsrc(ahead, 64);
        rb = sb.rsrc(ahead, 64);
      } else {
        advance();
      }
    };
    auto step = [&](auto st, auto live_tag) {
      constexpr int ST = decltype(st)::value, NEXT = (ST + 1) % NST;
      constexpr bool LIVE = decltype(live_tag)::value;
      const unsigned char* cur = smem + ST * STAGE;
      const unsigned char* nxt = smem + NEXT * STAGE;
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (LIVE)
        round(a0, b0, [&](auto qt) {
          constexpr int q = decltype(qt)::value;
          if constexpr (q < NB) b1[q] = ob.frag(cur + OpA::BYTES, q, 1);
          else a1[q - NB] = oa.frag(cur, q - NB, 1);
          if constexpr (q == 0) next_step();
        });
      else next_step();
      // this wave's loads of step kt + 1 have landed and its fragments of step kt are read; then every wave's
      __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0((NST - 2) * LOADS));
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (LIVE)
        round(a1, b1, [&](auto qt) {
          constexpr int q = decltype(qt)::value;
          if constexpr (q < NB) b0[q] = ob.frag(nxt + OpA::BYTES, q, 0);
          else a0[q - NB] = oa.frag(nxt, q - NB, 0);
          if constexpr (q < LOADS) load(st, qt);
        });
      else unroll<LOADS>([&](auto q) { load(st, q); });
    };
    auto all_steps = [&](auto live_tag) {
      while (kt < steps) {
        unroll<NST>([&](auto st) {
          if (kt < steps) {
            step(st, live_tag);
            ++kt;
          }
        });
      }
    };
    if (own) all_steps(std::true_type{});
    else all_steps(std::false_type{});
    const bool next_own = next.m0 + wm * 16 * MB < a.M && next.n0 + wn * 16 * NB < a.N;
    if (more && next_own && !own) first_frags();
    if (more) read_rows(next);

    if constexpr (EPI == SUM || EPI == OUT_BF16 || EPI == OUT_F32) {
      if constexpr (EPI == SUM) {
        // What is added to is read a row of blocks ahead of the stores (read one by one behind them: 34 us a tile).
        float* const c = static_cast<float*>(a.C) + (int64_t)tile.split * a.M * a.N;
        const auto at = [&](int i, int j, int64_t& o) {
          const int row = row0 + 16 * i + r, col = col0 + 16 * j + 4 * g;
          o = (int64_t)row * a.N + col;
          return row < a.M && col < a.N;
        };
        f32x4 before[2][NB];
        auto fetch = [&](int i) {
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            int64_t o;
            before[i & 1][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (at(i, j, o) && a.accumulate) before[i & 1][j] = *reinterpret_cast<const f32x4*>(c + o);
          }
        };
        fetch(0);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if (i + 1 < MB) fetch(i + 1);
#pragma unroll
          for (int j = 0; j < NB; ++j) {
            int64_t o;
            if (at(i, j, o)) *reinterpret_cast<f32x4*>(c + o) = acc[i][j] + before[i & 1][j];
          }
        }
      } else {
        const float alpha = *a.scale * (a.inv ? *a.inv : 1.f);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          const int row = row0 + 16 * i + r;
#pragma unroll
          for (int j = 0; j < NB; j += 2) {
            f32x4 u = acc[i][j] * alpha, v = acc[i][j + 1] * alpha;
            if constexpr (EPI == OUT_F32) {
              const int col = col0 + 16 * j + 4 * g;
              float* c = static_cast<float*>(a.C) + (int64_t)row * a.N + col;
              if (row < a.M && col < a.N) *reinterpret_cast<f32x4*>(c) = u;
              if (row < a.M && col + 16 < a.N) *reinterpret_cast<f32x4*>(c + 16) = v;
            } else {
              // Neighbouring blocks swap halves between their lanes: 8 consecutive columns of one of them each, 16 bytes.
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(u[e]), __float_as_uint(v[e]), false, false);
                u[e] = __uint_as_float(x[0]);
                v[e] = __uint_as_float(x[1]);
              }
              const int col = col0 + 16 * (j + (g & 1)) + 4 * (g & 2);
              if (row < a.M && col < a.N)
                st16(static_cast<uint16_t*>(a.C) + (int64_t)row * a.N + col,
                     make_uint4(pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3]), pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])));
            }
          }
        }
      }
    } else {
      const auto column = [&](int j) { return col0 + 32 * (j >> 1) + 8 * g + 4 * (j & 1); };  // of block j's element 0, within the piece
      // What few elements need stands behind branches that few waves take: the target's element and the columns past the
      // piece.  (An exponential takes 16 cycles of its SIMD and any other instruction 4; 128 elements a lane, two waves.)
      const bool ragged = n0 + TN > a.N;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const int row = row0 + 16 * i + r;
        const bool live = row < a.M;
        const int tc = __shfl(lane_tc, 16 * i + r);
        const bool has = tc >= col0 && tc < col0 + 16 * NB && ((tc - col0) >> 3 & 3) == g;  // among this lane's columns
        if constexpr (EPI == GRAD) {
          const float l2 = __shfl(lane_l2, 16 * i + r);
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = fast_exp2(fmaf(acc[i][j][e], kLog2e, -l2));
          if (has) {
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][e] -= column(j) + e == tc ? 1.f : 0.f;
          }
          if (a.grad) {
            const float s = live ? a.grad[row] / *a.scale : 0.f;  // the largest gives exactly 1
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] *= s;
          }
          if (ragged) {  // columns past the piece are zero: the products contract over them
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][e] = column(j) + e < a.N ? acc[i][j][e] : 0.f;
          }
#pragma unroll
          for (int j = 0; j < NB; j += 2) {
            const int c = column(j);
            const f32x4 u = acc[i][j], v = acc[i][j + 1];
            uint4 q = make_uint4(pack_bf16x2(u[0], u[1]), pack_bf16x2(u[2], u[3]), pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
            if (tc == -2) q = make_uint4(0, 0, 0, 0);
            if (live && c < a.p_cols) st16(a.p + (c >> 6) * a.p_block + (int64_t)row * 64 + (c & 63), q);  // 16 rows x 64 bytes a store
          }
        } else {
          float m = kNegInf;
          int mi = 0x7fffffff;
          if (ragged) {
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][e] = column(j) + e < a.N ? acc[i][j][e] : kNegInf;
          }
          if (has) {
            float v = 0.f;
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) v = column(j) + e == tc ? acc[i][j][e] : v;
            a.tgt[row] = v;
          }
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              if constexpr (EPI == STATS_PRED) {  // a lane's columns ascend: the first of equal ones stays
                if (acc[i][j][e] > m) {
                  m = acc[i][j][e];
                  mi = 32 * (j >> 1) + 4 * (j & 1) + e;
                }
              } else {
                m = fmaxf(m, acc[i][j][e]);
              }
            }
          if (EPI == STATS_PRED && mi != 0x7fffffff) mi += a.v0 + col0 + 8 * g;
          if constexpr (EPI == STATS_PRED) {
            max_first(m, mi, __shfl_xor(m, 16), __shfl_xor(mi, 16));
            max_first(m, mi, __shfl_xor(m, 32), __shfl_xor(mi, 32));
          } else {
            m = max_groups(m);
          }
          const float c0 = m == kNegInf ? 0.f : __fmul_rn(m, kLog2e);
          float s = 0.f;
#pragma unroll
          for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s += fast_exp2(fmaf(acc[i][j][e], kLog2e, -c0));
          s = sum_groups(s);
          if (live && g == 0) {
            const int64_t o = (int64_t)(2 * tn + wn) * a.M + row;
            a.part[o] = make_float2(m, s);
            if constexpr (EPI == STATS_PRED) a.part_i[o] = mi;
          }
        }
      }
    }
    if (!more) break;
    v += gridDim.x;
    tile = next;
    own = next_own;
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // no DMA may land after the workgroup exits
}

// Joins the parts of R rows: Q = 256 / R threads a row take every Q-th part, first the maxima, then the sums against the
// row's maximum; the Q in a fixed order, behind what the columns before left (`run`, where `more`).  FINAL: the loss, else
// `run`.  (16 rows a workgroup read whole cache lines, 4 fill the chip where rows are few: 8192 rows of 1024 parts 34 us
// against 80, 333 rows of 786 parts 17 against 8.  Latency and 2 TB/s: the parts are read twice, 134 MB.)
struct JoinArgs {
  const float2* part; const int32_t* part_i;
  int slots, M, more;
  float2* run; int32_t* run_i;
  const float* tgt; const int64_t* targets; int64_t ignore_index, V;
  float *loss, *lse2;
  int32_t* pred;
};

template <bool FINAL, int R>
__global__ __launch_bounds__(256) void head_join_kernel(const JoinArgs a) {
  constexpr int Q = 256 / R;
  __shared__ float sm[Q][R], ss[Q][R];
  __shared__ int si[Q][R];
  const int lr = threadIdx.x % R, q = threadIdx.x / R, row = blockIdx.x * R + lr;
  const bool live = row < a.M;
  float m = kNegInf;
  int mi = 0x7fffffff;
  float2 before = make_float2(kNegInf, 0.f);
  if (live && a.more) {
    before = a.run[row];
    if (q == 0) {
      m = before.x;
      if (a.part_i) mi = a.run_i[row];
    }
  }
  if (live) {
    if (a.part_i) {
      for (int k = q; k < a.slots; k += Q) max_first(m, mi, a.part[(int64_t)k * a.M + row].x, a.part_i[(int64_t)k * a.M + row]);
    } else {
#pragma unroll 8
      for (int k = q; k < a.slots; k += Q) m = fmaxf(m, a.part[(int64_t)k * a.M + row].x);
    }
  }
  sm[q][lr] = m;
  si[q][lr] = mi;
  __syncthreads();
  for (int o = Q / 2; o > 0; o >>= 1) {
    if (q < o) {
      float m1 = sm[q][lr];
      int i1 = si[q][lr];
      if (a.part_i) max_first(m1, i1, sm[q + o][lr], si[q + o][lr]);
      else m1 = fmaxf(m1, sm[q + o][lr]);
      sm[q][lr] = m1;
      si[q][lr] = i1;
    }
    __syncthreads();
  }
  m = sm[0][lr];
  // a part's sum is in units of exp2(its maximum's rounded multiple of log2 e), as the tile took it
  const float C = m == kNegInf ? 0.f : __fmul_rn(m, kLog2e);
  const auto in_units = [&](float2 x) { return x.x == kNegInf ? (x.y == x.y ? 0.f : x.y) : x.y * fast_exp2(__fmul_rn(x.x, kLog2e) - C); };
  float s = live && a.more && q == 0 ? in_units(before) : 0.f;
  if (live) {
#pragma unroll 8
    for (int k = q; k < a.slots; k += Q) s += in_units(a.part[(int64_t)k * a.M + row]);
  }
  ss[q][lr] = s;
  __syncthreads();
  for (int o = Q / 2; o > 0; o >>= 1) {
    if (q < o) ss[q][lr] += ss[q + o][lr];
    __syncthreads();
  }
  if (q != 0 || !live) return;
  s = ss[0][lr];
  mi = si[0][lr];
  if constexpr (!FINAL) {
    a.run[row] = make_float2(m, s);
    if (a.part_i) a.run_i[row] = mi;
    return;
  }
  const float lg = __builtin_amdgcn_logf(s);  // base 2
  const int64_t t = a.targets[row];
  a.lse2[row] = C + lg;
  a.loss[row] = t == a.ignore_index ? 0.f
              : t < 0 || t >= a.V ? __builtin_nanf("") : (fmaf(-a.tgt[row], kLog2e, C) + lg) * kLn2;
  if (a.pred) a.pred[row] = mi == 0x7fffffff ? 0 : mi;  // a row of NaN has no maximum
}

// total = sum of loss; with inv, its mean, and inv = 1 / rows that count: one workgroup, a fixed order, 64-bit sums.
__global__ __launch_bounds__(1024) void head_total_kernel(const float* loss, const int64_t* targets, int64_t ignore_index,
                                                          int M, float* total, float* inv) {
  __shared__ double sl[1024];
  __shared__ int sn[1024];
  double l = 0.0;
  int n = 0;
  for (int i = threadIdx.x; i < M; i += 1024) {
    l += (double)loss[i];
    n += targets[i] != ignore_index;
  }
  sl[threadIdx.x] = l;
  sn[threadIdx.x] = n;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) {
      sl[threadIdx.x] += sl[threadIdx.x + o];
      sn[threadIdx.x] += sn[threadIdx.x + o];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    *total = (float)(inv ? sl[0] / (double)sn[0] : sl[0]);  // the mean of no rows is NaN
    if (inv) *inv = sn[0] ? 1.f / (float)sn[0] : 0.f;  // and its gradients are zero
  }
}

// What q leaves to the products' scale: the first of the largest gradients by size among the finite ones of rows that count
// (1 where all are zero), with its sign, so that rows of one gradient have q = softmax - onehot exactly.
__global__ __launch_bounds__(1024) void head_scale_kernel(const float* grad, const int64_t* targets, int64_t ignore_index, int M,
                                                          float* scale) {
  __shared__ float sm[1024];
  __shared__ int si[1024];
  float m = 0.f;
  int mi = 0x7fffffff;
  for (int i = threadIdx.x; i < M; i += 1024) {
    const float g = fabsf(grad[i]);
    if (targets[i] != ignore_index && g > m && g < __builtin_inff()) {
      m = g;
      mi = i;
    }
  }
  sm[threadIdx.x] = m;
  si[threadIdx.x] = mi;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) max_first(sm[threadIdx.x], si[threadIdx.x], sm[threadIdx.x + o], si[threadIdx.x + o]);
    __syncthreads();
  }
  if (threadIdx.x == 0) *scale = sm[0] > 0.f ? grad[si[0]] : 1.f;
}

// out = alpha * sum over splits of the partial sums, in order (bandwidth: 8192 x 1536 from 4 splits in 40 us, 5.6 TB/s)
template <typename T>
__global__ __launch_bounds__(256) void head_reduce_kernel(const float* x, int splits, int64_t n, T* y, const float* scale,
                                                          const float* inv) {
  const float alpha = *scale * (inv ? *inv : 1.f);
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
    float v[4];
    load4<float>(x + i, v);
    for (int s = 1; s < splits; ++s) {
      float u[4];
      load4<float>(x + s * n + i, u);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += u[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= alpha;
    store4<T>(y + i, v);
  }
}

constexpr size_t up(size_t n) { return (n + 255) & ~size_t(255); }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

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
Tiling tiling(int64_t M, int64_t N, int steps, int most) {
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

int32_t check(const llattn_head_cfg* c) {
  if (!c) return fail(LLATTN_ERR_SHAPE, "llattn_head: null configuration");
  if (c->rows <= 0 || c->rows >= (1 << 23) || c->V <= 0 || c->D <= 0 || c->D % 8 || c->V > 0x7fffff00)
    return fail(LLATTN_ERR_SHAPE, "llattn_head: rows %d, V %d, D %d: must be positive, rows below 2^23, D a multiple of 8",
                c->rows, c->V, c->D);
  if (c->piece < 0 || c->piece % 256)
    return fail(LLATTN_ERR_SHAPE, "llattn_head: piece %d must be 0 or a multiple of 256", c->piece);
  if (c->dw_dtype != LLATTN_F32 && c->dw_dtype != LLATTN_BF16)
    return fail(LLATTN_ERR_DTYPE, "llattn_head: unknown dW dtype %d", c->dw_dtype);
  return LLATTN_OK;
}

// forward: columns whose parts are joined at once, so that those stay within 256 MB
struct FwdPlan { int kind, range; size_t slots, bytes; };
FwdPlan fwd_plan(const llattn_head_cfg* c) {
  FwdPlan f;
  f.kind = tiling(c->rows, c->V, (c->D + 63) / 64, 1).kind;
  const int64_t most = std::max<int64_t>(1, (int64_t)(256 << 20) / (24 * (int64_t)c->rows));  // tile columns, two parts of 12 bytes each
  const int64_t tiles = ceil_div(c->V, kTn[f.kind]);
  f.range = (int)(std::min(tiles, most) * kTn[f.kind]);
  f.slots = 2 * (size_t)std::min(tiles, most);
  const size_t r = (size_t)c->rows;
  f.bytes = up(f.slots * r * 8) + up(f.slots * r * 4) + up(r * 8) + 2 * up(r * 4);
  return f;
}

// backward: columns of a piece
int piece_of(const llattn_head_cfg* c) {
  int64_t p = c->piece;
  if (p == 0) p = std::max<int64_t>(256, (int64_t(1) << 28) / c->rows / 256 * 256);
  return (int)std::min<int64_t>(p, ceil_div(c->V, 256) * 256);
}

// q of a piece [rows][piece], the sums of dh over pieces and splits, the partial sums of dW, the shared scale
struct BwdPlan {
  int piece, pieces;
  Tiling logits, dh, dw;
  size_t p, dh_part, dw_part;
  bool dh_direct() const { return pieces == 1 && dh.splits == 1; }
  size_t bytes() const { return p + dh_part + dw_part + up(4); }
};
BwdPlan bwd_plan(const llattn_head_cfg* c) {
  BwdPlan b{};
  b.piece = piece_of(c);
  b.pieces = (int)ceil_div(c->V, b.piece);
  const int nv = std::min(b.piece, c->V);
  b.logits = tiling(c->rows, nv, (c->D + 63) / 64, 1);
  b.dh = tiling(c->rows, c->D, (nv + 63) / 64, 16);
  b.dw = tiling(nv, c->D, (c->rows + 63) / 64, 16);
  b.p = up((size_t)c->rows * b.piece * 2);
  b.dh_part = b.dh_direct() ? 0 : up((size_t)b.dh.splits * c->rows * c->D * 4);
  b.dw_part = b.dw.splits > 1 ? up((size_t)b.dw.splits * ((nv + 7) / 8 * 8) * c->D * 4) : 0;
  return b;
}

template <int EPI, bool AT, bool BT>
void launch(HeadArgs& a, int kind, int splits, hipStream_t st) {
  a.steps = (a.K + 63) / 64;
  a.per = (a.steps + splits - 1) / splits;
  a.tiles_m = (a.M + kTm[kind] - 1) / kTm[kind];
  a.tiles_n = (a.N + kTn[kind] - 1) / kTn[kind];
  a.total = a.tiles_m * a.tiles_n * splits;
  const bool loss = EPI == STATS || EPI == STATS_PRED || EPI == GRAD;
  const dim3 grid((unsigned)(loss ? std::min(a.total, 256 * kPerCu[kind]) : a.total));
  if (kind == BIG) hipLaunchKernelGGL((head_kernel<EPI, AT, BT, BigShape, 1>), grid, dim3(BigShape::THREADS), 0, st, a);
  else if (kind == SQUARE) hipLaunchKernelGGL((head_kernel<EPI, AT, BT, SquareShape, 2>), grid, dim3(SquareShape::THREADS), 0, st, a);
  else if constexpr (!AT && !BT) hipLaunchKernelGGL((head_kernel<EPI, AT, BT, ThinShape, 2>), grid, dim3(ThinShape::THREADS), 0, st, a);
}

// l of `cols` columns from v0 on: h [rows][D] by W [cols][D]
void logits_of(HeadArgs& a, const llattn_head_cfg* c, const void* h, int64_t ldh, const void* W, int64_t ldw, int v0, int cols) {
  a.M = c->rows; a.N = cols; a.K = c->D;
  a.A = static_cast<const uint16_t*>(h); a.lda = ldh;
  a.B = static_cast<const uint16_t*>(W) + v0 * ldw; a.ldb = ldw;
  a.v0 = v0; a.V = c->V;
}

template <typename T>
void launch_reduce(const float* x, int splits, int64_t n, T* y, const HeadArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(head_reduce_kernel<T>, dim3((unsigned)std::min<int64_t>(ceil_div(n, 1024), 8192)), dim3(256), 0, st, x, splits,
                     n, y, a.scale, a.inv);
}

int32_t check_operands(const char* who, const llattn_head_cfg* c, const void* h, int64_t ldh, const void* W, int64_t ldw,
                       const void* targets, const void* ws, size_t ws_bytes, size_t need) {
  if (!h || !W || !targets) return fail(LLATTN_ERR_LAYOUT, "%s: null h, W or targets", who);
  if (ldh < c->D || ldw < c->D || ldh % 8 || ldw % 8 || !aligned16(h) || !aligned16(W) || ldh >= (1 << 23) || ldw >= (1 << 23))
    return fail(LLATTN_ERR_LAYOUT, "%s: rows of h and W must be 16-byte aligned, of strides in [D, 2^23) elements (ldh %lld, "
                "ldw %lld)", who, (long long)ldh, (long long)ldw);
  if (!ws || ws_bytes < need || !aligned16(ws))
    return fail(LLATTN_ERR_WORKSPACE, "%s: needs %zu workspace bytes (got %zu)", who, need, ws_bytes);
  return LLATTN_OK;
}

}  // namespace
}  // namespace llattn

using namespace llattn;

extern "C" size_t llattn_head_bytes(const llattn_head_cfg* c, int32_t which) {
  if (check(c) != LLATTN_OK) return 0;
  if (which == 0) return fwd_plan(c).bytes;
  if (which == 1) return bwd_plan(c).bytes();
  fail(LLATTN_ERR_SHAPE, "llattn_head_bytes: unknown workspace %d", which);
  return 0;
}

extern "C" int32_t llattn_head_fwd(const llattn_head_cfg* c, const void* h, int64_t ldh, const void* W, int64_t ldw,
                                   const int64_t* targets, int64_t ignore_index, float* loss, float* lse2, int32_t* pred,
                                   float* total, float* inv, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int32_t rc = check(c)) return rc;
  const FwdPlan f = fwd_plan(c);
  if (const int32_t rc = check_operands("llattn_head_fwd", c, h, ldh, W, ldw, targets, workspace, workspace_bytes, f.bytes))
    return rc;
  if (!loss || !lse2 || (inv && !total)) return fail(LLATTN_ERR_LAYOUT, "llattn_head_fwd: null loss, lse2 or total");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const size_t r = (size_t)c->rows;
  char* p = static_cast<char*>(workspace);
  HeadArgs a{};
  a.part = reinterpret_cast<float2*>(p); p += up(f.slots * r * 8);
  a.part_i = reinterpret_cast<int32_t*>(p); p += up(f.slots * r * 4);
  JoinArgs j{};
  j.run = reinterpret_cast<float2*>(p); p += up(r * 8);
  j.run_i = reinterpret_cast<int32_t*>(p); p += up(r * 4);
  a.tgt = reinterpret_cast<float*>(p);
  a.targets = targets; a.ignore_index = ignore_index;
  j.M = c->rows; j.tgt = a.tgt; j.targets = targets; j.ignore_index = ignore_index; j.V = c->V;
  j.loss = loss; j.lse2 = lse2; j.pred = pred;
  const bool many = c->rows >= 2048;
  const dim3 jgrid(many ? (c->rows + 15) / 16 : (c->rows + 3) / 4), block(256);
  j.part = a.part; j.part_i = pred ? a.part_i : nullptr;
  for (int64_t v0 = 0; v0 < c->V; v0 += f.range) {
    logits_of(a, c, h, ldh, W, ldw, (int)v0, (int)std::min<int64_t>(f.range, c->V - v0));
    if (pred) launch<STATS_PRED, false, false>(a, f.kind, 1, st);
    else launch<STATS, false, false>(a, f.kind, 1, st);
    j.slots = 2 * a.tiles_n;
    j.more = v0 > 0;
    const bool last = v0 + f.range >= c->V;
    if (many && last) hipLaunchKernelGGL((head_join_kernel<true, 16>), jgrid, block, 0, st, j);
    else if (many) hipLaunchKernelGGL((head_join_kernel<false, 16>), jgrid, block, 0, st, j);
    else if (last) hipLaunchKernelGGL((head_join_kernel<true, 4>), jgrid, block, 0, st, j);
    else hipLaunchKernelGGL((head_join_kernel<false, 4>), jgrid, block, 0, st, j);
  }
  if (total) hipLaunchKernelGGL(head_total_kernel, dim3(1), dim3(1024), 0, st, loss, targets, ignore_index, c->rows, total, inv);
  return check_launch("llattn_head_fwd");
}

extern "C" int32_t llattn_head_bwd(const llattn_head_cfg* c, const void* h, int64_t ldh, const void* W, int64_t ldw,
                                   const int64_t* targets, int64_t ignore_index, const float* lse2, const float* grad,
                                   int32_t grad_stride, const float* inv, void* dh, void* dW, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (const int32_t rc = check(c)) return rc;
  const BwdPlan b = bwd_plan(c);
  if (const int32_t rc = check_operands("llattn_head_bwd", c, h, ldh, W, ldw, targets, workspace, workspace_bytes, b.bytes()))
    return rc;
  if (!lse2 || !grad || grad_stride < 0 || grad_stride > 1)
    return fail(LLATTN_ERR_LAYOUT, "llattn_head_bwd: null lse2 or grad, or a grad stride other than 0 and 1 (%d)", grad_stride);
  if ((dh && !aligned16(dh)) || (dW && !aligned16(dW)))
    return fail(LLATTN_ERR_LAYOUT, "llattn_head_bwd: dh and dW must be 16-byte aligned");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (!dh && !dW) return LLATTN_OK;
  char* ws = static_cast<char*>(workspace);
  float* dh_part = reinterpret_cast<float*>(ws + b.p);
  float* dw_part = reinterpret_cast<float*>(ws + b.p + b.dh_part);
  float* scale = reinterpret_cast<float*>(ws + b.p + b.dh_part + b.dw_part);
  HeadArgs a{};
  a.p = reinterpret_cast<uint16_t*>(ws); a.p_block = (int64_t)c->rows * 64; a.p_cols = b.piece;
  a.targets = targets; a.ignore_index = ignore_index;
  a.lse2 = lse2; a.inv = inv;
  a.grad = grad_stride ? grad : nullptr;
  a.scale = grad_stride ? scale : grad;
  if (grad_stride) hipLaunchKernelGGL(head_scale_kernel, dim3(1), dim3(1024), 0, st, grad, targets, ignore_index, c->rows, scale);
  const int64_t dw_size = c->dw_dtype == LLATTN_F32 ? 4 : 2;
  for (int q = 0; q < b.pieces; ++q) {
    const int v0 = (int)((int64_t)q * b.piece), cols = std::min(b.piece, c->V - v0);
    logits_of(a, c, h, ldh, W, ldw, v0, cols);
    launch<GRAD, false, false>(a, b.logits.kind, 1, st);
    HeadArgs d = a;
    d.A = a.p; d.lda = a.p_block;
    d.N = c->D;
    if (dh) {  // q W: q's chunk that reaches past the piece's columns holds zeros there, W's rows past them read zero
      d.M = c->rows; d.K = cols;
      d.accumulate = q > 0;
      d.C = b.dh_direct() ? dh : dh_part;
      if (b.dh_direct()) launch<OUT_BF16, false, true>(d, b.dh.kind, 1, st);
      else launch<SUM, false, true>(d, b.dh.kind, b.dh.splits, st);
    }
    if (dW) {  // qᵀ h
      d.M = (cols + 7) / 8 * 8; d.K = c->rows;
      d.B = a.A; d.ldb = a.lda;
      d.accumulate = 0;
      void* out = static_cast<char*>(dW) + (int64_t)v0 * c->D * dw_size;
      d.C = b.dw.splits > 1 ? static_cast<void*>(dw_part) : out;
      if (b.dw.splits > 1) {
        launch<SUM, true, true>(d, b.dw.kind, b.dw.splits, st);
        const int64_t n = (int64_t)d.M * c->D;
        if (c->dw_dtype == LLATTN_F32) launch_reduce(dw_part, b.dw.splits, n, static_cast<float*>(out), a, st);
        else launch_reduce(dw_part, b.dw.splits, n, static_cast<uint16_t*>(out), a, st);
      } else if (c->dw_dtype == LLATTN_F32) {
        launch<OUT_F32, true, true>(d, b.dw.kind, 1, st);
      } else {
        launch<OUT_BF16, true, true>(d, b.dw.kind, 1, st);
      }
    }
  }
  if (dh && !b.dh_direct())
    launch_reduce(dh_part, b.dh.splits, (int64_t)c->rows * c->D, static_cast<uint16_t*>(dh), a, st);
  return check_launch("llattn_head_bwd");
}
