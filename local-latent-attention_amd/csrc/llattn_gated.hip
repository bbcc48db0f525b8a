// Gated feed-forward (include/llattn_lm.h):
//
//   a = x W1ᵀ + b1,  u = x W3ᵀ + b3,  h = act(a) u,  y = h W2ᵀ + b2
//   dh = dy W2,  da = dh u act'(a),  du = dh act(a),  dx = da W1 + du W3,  dW1 = daᵀ x,  dW3 = duᵀ x,  dW2 = dyᵀ h
//
// Both projections and the gate are one product: half of a tile's columns are rows of W1 and half the same rows of W3, laid out
// so that a lane's accumulators hold a and u of the same elements; its epilogue writes h and, for a backward, p = act(a) and
// s = act'(a) u.  The backward's first product leaves da = dh s and du = dh p in the two halves of one matrix, so that dx is
// one product over their columns (W1's rows, then W3's) and dW1 and dW3 together another.
//
// Rounded to bf16 besides the results: h, da and du, which the matrix cores take in 16 bits.  They are off by half a step
// of each value at most, independently, so results are about sqrt 2 times as far from the exact ones as their own rounding
// leaves them.  Up to 64 rows, where single results stray further and there is room in the tiles, they are held as the sums of two bf16
// values.  p and s are kept in 24 bits (16 of the significand: their rounding in bf16 would make that sqrt 3, at 8192 x 1536 x 4096
// for 2% of the time), the upper two bytes and the third in planes of their own.
//
// Backward, two products share a launch where both take 128 x 128 tiles (the gate's gradients with dW2, dx with dW1 and dW3): small
// ones fill the chip together.  Forward alone with few rows, two kernels of their own read every weight once, along k.
//
// What bounds it: the matrix cores (2 rows D F operations for each of the three products, twice that backward) and epilogues that no
// other tile's products cover; with few rows the reads of the weights.  8192 x 1536 x 4096: gate 206 us (1.0 PFLOP/s), y 89 (1.16),
// the gate's gradients and dW2 237 (0.87), dx 178 (1.16), dW1 and dW3 174 (1.18); 8192 cubed runs at 1.32 in this library's plain product.
#include <algorithm>

#include "llattn_lm.h"
#include "llattn_tiles.h"

namespace llattn {
namespace {

using namespace tiles;

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// OUT: C, or fp32 parts of it
enum Epilogue { GATE = 0, DGATE = 1, OUT = 2 };

struct GatedArgs {
  int M, N, K;                  // GATE: N columns of h
  int steps, per;               // 64-wide k steps, of a split
  int tiles_m, tiles_n, total;  // total: with the splits
  const uint16_t *A, *A2; int64_t lda;  // A2: the matrix from step `half` on, where A lies along k and there are two
  const uint16_t *B, *B2; int64_t ldb;  // B2: the other matrix of a gate, or the one from step `half` on
  int half, k_half;             // two matrices along k: steps and k of the first, k of either
  int low;                      // few rows: the lower halves of h (GATE), da and du (DGATE) lie that many rows on; or 0
  int fold;                     // OUT in parts: rows [fold, 2 fold) of the product are added to the first; or 0
  const float *bias, *bias2;
  uint16_t* h;                  // GATE: [M][N]
  int act;
  unsigned char *p, *s;         // [M][N] as Float24 lays them out, or null (GATE)
  uint16_t* d; int64_t ldd;     // DGATE: [M][ldd], da in its columns, du from column ldd / 2 on
  void *C, *C2; int64_t ldc;    // rows [0, m_live) of each of the two halves of m_half rows (one half: m_half = M)
  int m_half, m_live;
  int f32;                      // C is fp32 (else bf16)
  float* part;                  // OUT in splits: [splits][M][N]
};

// act(a) and act'(a).  SiLU: a g and g (1 + a (1 - g)), g = 1 / (1 + exp(-a)).  GELU: a Phi and Phi + a phi with
// Phi(-z sqrt 2) = erfc(z) / 2, erfc(z) = t P(t) exp(-z²), t = 1 / (1 + 3 z / 8), P fitted here to 9e-7 of itself over z in
// [0, 12]: the tail keeps its relative accuracy, as products with u make it count.
__device__ __forceinline__ void activation(int act, float a, float& f, float& df) {
  if (act == LLATTN_GATE_SILU) {
    const float g = __builtin_amdgcn_rcpf(1.f + fast_exp2(-kLog2e * a));
    f = a * g;
    df = fmaf(f, 1.f - g, g);
  } else {
    const float z = fabsf(a) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(fmaf(0.375f, z, 1.f));
    float P = -0.133229989f;
    P = fmaf(P, t, 0.381471619f);
    P = fmaf(P, t, -0.120644021f);
    P = fmaf(P, t, 0.276750286f);
    P = fmaf(P, t, 0.169042397f);
    P = fmaf(P, t, 0.215237073f);
    P = fmaf(P, t, 0.211373235f);
    const float e = fast_exp2(-0.5f * kLog2e * a * a), q = 0.5f * t * P * e, cdf = a >= 0.f ? 1.f - q : q;
    f = a * cdf;
    df = fmaf(a, e * 0.39894228040143268f, cdf);
  }
}

// Eight values in 24 bits, cut off: the upper halves in one plane, the next bytes in the plane behind it.  (Cut off, not rounded: no
// NaN turns into another value.)  Pieces of eight columns lie by blocks of 16 rows, then by column, then by row: what a wave writes
// or reads at a time (four pieces of 16 rows) is one run of memory, in the gate's tiles and in those of its gradients
// (row by row instead, training passes of 8192 x 1536 x 4096 took 897 us for 872, of 333 rows 195 for 174), and past the caches,
// which it would empty of the operands: the gate's product 220 -> 209 us there, its gradients' beside dW2 258 -> 240, the next
// products, which read h and d, 98 -> 92 and 198 -> 182.
struct Float24 {
  static __host__ __device__ constexpr int64_t elements(int64_t rows, int cols) { return (rows + 15) / 16 * 16 * cols; }
  static __device__ __forceinline__ int64_t place(int row, int col, int cols) {
    return (((int64_t)(row >> 4) * (cols >> 3) + (col >> 3)) * 16 + (row & 15)) * 8;
  }
  u32x4 hi;
  u32x2 lo;
  static __device__ __forceinline__ uint32_t lows(const f32x4& x) {  // byte 1 of each
    const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x0c0c0501);
    const uint32_t b = __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x05010c0c);
    return a | b;
  }
  static __device__ __forceinline__ void store(unsigned char* plane, int64_t plane_bytes, int64_t at, const f32x4& x, const f32x4& y) {
    const auto hi2 = [](float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302); };
    __builtin_nontemporal_store(u32x4{hi2(x[0], x[1]), hi2(x[2], x[3]), hi2(y[0], y[1]), hi2(y[2], y[3])}, reinterpret_cast<u32x4*>(plane + 2 * at));
    __builtin_nontemporal_store(u32x2{lows(x), lows(y)}, reinterpret_cast<u32x2*>(plane + plane_bytes + at));
  }
  __device__ __forceinline__ void load(const unsigned char* plane, int64_t plane_bytes, int64_t at) {
    hi = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(plane + 2 * at));
    lo = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(plane + plane_bytes + at));
  }
  __device__ __forceinline__ void get(f32x4& x, f32x4& y) const {
    const auto four = [](uint32_t h0, uint32_t h1, uint32_t l) {  // (upper half, byte) -> the upper three bytes
      return f32x4{__uint_as_float(__builtin_amdgcn_perm(h0, l, 0x0504000c)), __uint_as_float(__builtin_amdgcn_perm(h0, l, 0x0706010c)),
                   __uint_as_float(__builtin_amdgcn_perm(h1, l, 0x0504020c)), __uint_as_float(__builtin_amdgcn_perm(h1, l, 0x0706030c))};
    };
    x = four(hi.x, hi.y, lo.x);
    y = four(hi.z, hi.w, lo.y);
  }
};

// Rows of two matrices, T / 2 of each, as RowOp<T, W, true> holds them; a wave's fragments: blocks j < NB / 2 of the first, the
// same rows of the second behind them.
template <int T, int W, int NB>
struct GateOp : RowOp<T, W, true> {
  using Base = RowOp<T, W, true>;
  using Base::off, Base::kc, Base::base, Base::LOADS;
  __device__ __forceinline__ void init(int64_t ld, int w, int lane, int o0) {
    Base::init(ld, w, lane, o0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {  // rows of the matrix that this wave loads
      const int row = 8 * (w * LOADS + i) + (lane >> 3), c = (lane & 7) ^ pswz<true>(row);
      off[i] = step_off((int64_t)(row % (T / 2)) * ld * 2 + 16 * c);
    }
  }
  __device__ __forceinline__ bf16x8 frag(const unsigned char* st, int j, int half) const {
    const int i = j % (NB / 2);
    return *reinterpret_cast<const bf16x8*>(st + base[half] + (j >= NB / 2 ? T / 2 * 128 : 0) + (i >> 1) * 4096 + (i & 1) * 512);
  }
};

// Column blocks of a tile that is not a power of two wide: V columns in rows of T (2 T bytes in LDS, as ColOp<T, W> lays them out;
// chunks past V are not loaded), NB blocks from o0 on, a multiple of 16.
template <int T, int V, int W, int NB>
struct ColsOp {
  static constexpr int BYTES = T * 128, LOADS = BYTES / 1024 / W, PER = T / 8;
  uint32_t off[LOADS], base[NB];
  static __device__ __forceinline__ int swz(int k) { return ColOp<T, W>::swz(k); }
  __device__ __forceinline__ void init(int64_t ld, int w, int lane, int o0) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int q = (w * LOADS + i) * 64 + lane, k = q / PER, c = (q % PER) ^ swz(k);
      off[i] = 8 * c < V ? step_off((int64_t)k * ld * 2 + 16 * c) : kOffPastK;
    }
    const int r = lane & 15, g = lane >> 4, k = 8 * g + (r >> 2);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int byte = 2 * (o0 + 16 * j) + 8 * (r & 3);
      base[j] = k * (2 * T) + (((byte >> 4) ^ swz(k)) << 4) + (byte & 15);
    }
  }
  __device__ __forceinline__ uint32_t at(int i, int) const { return off[i]; }
  __device__ __forceinline__ bf16x8 frag(const unsigned char* st, int j, int half) const {
    bf16x4 hv[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const unsigned char* p = st + base[j] + (32 * half + 4 * q) * (2 * T);
      hv[q] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(p));
    }
    return bf16x8{hv[0][0], hv[0][1], hv[0][2], hv[0][3], hv[1][0], hv[1][1], hv[1][2], hv[1][3]};
  }
};

// T columns along k: the operand that holds them
template <int T, int W, int NB> struct Cols { typedef ColOp<T, W> Op; };
template <int W, int NB> struct Cols<192, W, NB> { typedef ColsOp<256, 192, W, NB> Op; };

// Tiles of a product, as those of the head loss: a 64-k step is two rounds of products, each beside the fragment reads of the
// next: k 0..31 (reads k 32..63), a barrier, k 32..63 (reads the next step's k 0..31 and issues the loads of step
// kt + NST into the stage just read).  Waves whose part of the tile lies outside load and wait like the others and do
// nothing else.  The gate's workgroups take tile after tile, the next one's first steps loaded in the last ones of this.
// AT: A stored with its rows along k.  BT: B likewise.  TWO: a second matrix B from step `half` on, and with AT a second A.
// What a product is made of: EPI, AT, BT and TWO as above
template <int EPI_, bool AT_, bool BT_, bool TWO_>
struct Product {
  static constexpr int EPI = EPI_;
  static constexpr bool AT = AT_, BT = BT_, TWO = TWO_;
};
typedef Product<GATE, false, false, false> GateProduct;
typedef Product<OUT, false, false, false> OutProduct;   // y
typedef Product<DGATE, false, true, false> DGateProduct;
typedef Product<OUT, false, true, true> DxProduct;
typedef Product<OUT, true, true, false> DwProduct;
typedef Product<OUT, true, true, true> DwHalvesProduct;  // of few rows

template <typename P, typename S>
struct Operands {
  static constexpr int W = S::W;
  typedef std::conditional_t<P::AT, typename Cols<S::TM, W, S::MB>::Op, RowOp<S::TM, W, false>> A;
  typedef std::conditional_t<P::EPI == GATE, GateOp<S::TN, W, S::NB>, std::conditional_t<P::BT, typename Cols<S::TN, W, S::NB>::Op, RowOp<S::TN, W, true>>> B;
  static constexpr int STAGE = A::BYTES + B::BYTES, LDS = S::NST * STAGE;
};

// The tiles v, v + stride, ... of a product (one tile where it does not persist)
template <typename P, typename S>
__device__ __forceinline__ void gated_tiles(const GatedArgs& a, unsigned char* smem, int v, int stride) {
  constexpr int EPI = P::EPI;
  constexpr bool AT = P::AT, BT = P::BT, TWO = P::TWO, PERSIST = EPI == GATE;
  constexpr int MB = S::MB, NB = S::NB, TM = S::TM, TN = S::TN, NST = S::NST, W = S::W;
  constexpr int TC = EPI == GATE ? TN / 2 : TN;      // columns of the result in a tile,
  constexpr int WCOLS = EPI == GATE ? 8 * NB : 16 * NB;  // and of a wave
  typedef typename Operands<P, S>::A OpA;
  typedef typename Operands<P, S>::B OpB;
  constexpr int LOADS = OpA::LOADS + OpB::LOADS, STAGE = OpA::BYTES + OpB::BYTES;
  static_assert(LOADS <= MB + NB, "the second round's reads carry the loads");
  static_assert((!AT || TM == 192 || (16 * MB) % 64 == 0) && (!BT || TN == 192 || (16 * NB) % 64 == 0), "ColOp::base");
  static_assert(S::WC == 2 && (S::WR == 2 || S::WR == 4), "wave layouts");
  static_assert(EPI != GATE || (TN / 2) % (8 * OpB::LOADS) == 0, "a wave loads rows of one of the two matrices");
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // eight waves: those of one SIMD (w, w + 4) lie in opposite halves of both sides
  const int wm = W == 8 ? (w & 3) ^ (w >> 2 << 1) : w >> 1, wn = W == 8 ? (w & 1) ^ (w >> 2) : w & 1;
  struct Tile { int m0, n0, split, steps; };  // steps: of the split (none or less: zeros)
  auto tile_at = [&](int v) {
    int t = xcd_remap(v, a.total);
    const int tiles = a.tiles_m * a.tiles_n, split = t / tiles;
    t -= split * tiles;
    constexpr int GM = 8;
    const int group = t / (GM * a.tiles_n), first_m = group * GM, gm = min(a.tiles_m - first_m, GM);
    const int tm = first_m + (t % (GM * a.tiles_n)) % gm, tn = t % (GM * a.tiles_n) / gm;
    const int steps = min(a.steps - split * a.per, a.per);
    return Tile{__builtin_amdgcn_readfirstlane(tm * TM), __builtin_amdgcn_readfirstlane(tn * TC),
                __builtin_amdgcn_readfirstlane(split), __builtin_amdgcn_readfirstlane(steps)};
  };
  OpA oa;
  OpB ob;
  oa.init(a.lda, w, lane, wm * 16 * MB);
  ob.init(a.ldb, w, lane, wn * WCOLS);
  // n of the operand's rows (t: columns) from o on, from step k on of K
  auto source = [&](const uint16_t* p, int64_t ld, bool t, int o, int n, int k, int K) {
    StepSrc s;
    s.addr = reinterpret_cast<uint64_t>(p + (t ? o + (int64_t)k * 64 * ld : o * ld + (int64_t)k * 64));
    s.full = t ? extent_of(64, ld, n) : rows_extent(n, ld, K);  // not t: chunks past the last k are masked (RowOp::at)
    s.tail = t ? extent_of(K & 63 ? K & 63 : 64, ld, n) : s.full;
    s.inc = t ? (uint32_t)(128 * ld) : 128u;
    return s;
  };
  auto source_a = [&](const Tile& t, int k) {
    const int n = min(TM, a.M - t.m0);
    if constexpr (TWO && AT) return k < a.half ? source(a.A, a.lda, AT, t.m0, n, k, a.k_half) : source(a.A2, a.lda, AT, t.m0, n, k - a.half, a.k_half);
    return source(a.A, a.lda, AT, t.m0, n, k, a.K);
  };
  auto source_b = [&](const Tile& t, int k) {  // from step k on
    const int n = min(TC, a.N - t.n0);
    if constexpr (TWO) return k < a.half ? source(a.B, a.ldb, BT, t.n0, n, k, a.k_half) : source(a.B2, a.ldb, BT, t.n0, n, k - a.half, a.k_half);
    return source(EPI == GATE && 2 * w >= W ? a.B2 : a.B, a.ldb, BT, t.n0, n, k, a.K);
  };
  auto k_of = [&](const Tile& t) { return min(a.K - t.split * a.per * 64, t.steps * 64); };
  Tile tile = tile_at(v);
  StepSrc sa = source_a(tile, tile.split * a.per), sb = source_b(tile, tile.split * a.per);
  int ahead = k_of(tile);  // k from the step that ra and rb describe to the end of its tile's
  int kb = tile.split * a.per;  // that step, among all
  const auto left_b = [&]() { return TWO ? min(ahead, a.k_half - 64 * (kb < a.half ? kb : kb - a.half)) : ahead; };
  int bleft = left_b();
  const auto left_a = [&]() { return TWO && AT ? bleft : ahead; };
  i32x4 ra = sa.rsrc(left_a(), 64), rb = sb.rsrc(bleft, 64);
  auto advance = [&]() {
    sa.addr += sa.inc;
    sb.addr += sb.inc;
    ahead -= 64;
    if constexpr (TWO) {
      if (++kb == a.half) {
        sb = source_b(tile, kb);
        if constexpr (AT) sa = source_a(tile, kb);
      }
    }
    bleft = left_b();
    ra = sa.rsrc(left_a(), 64);
    rb = sb.rsrc(bleft, 64);
  };
  const uint32_t lds_a = __builtin_amdgcn_readfirstlane(lds_addr(smem) + w * OpA::LOADS * 1024);
  const uint32_t lds_b = __builtin_amdgcn_readfirstlane(lds_addr(smem) + OpA::BYTES + w * OpB::LOADS * 1024);
  auto load = [&](auto stage, auto q) {
    constexpr int s = decltype(stage)::value, n = decltype(q)::value;
    if constexpr (n < OpA::LOADS) dma_at<s * STAGE + n * 1024>(ra, oa.at(n, ahead), lds_a);
    else dma_at<s * STAGE + (n - OpA::LOADS) * 1024>(rb, ob.at(n - OpA::LOADS, bleft), lds_b);
  };
  bf16x8 a0[MB], a1[MB], b0[NB], b1[NB];  // k 0..31 and 32..63
  f32x4 acc[MB][NB];
  // MB NB products, B first: lane (r, g) accumulates C[r][4 g + e]; io(q), q < MB + NB, spread over them
  auto round = [&](const bf16x8 (&x)[MB], const bf16x8 (&y)[NB], auto io) {
    constexpr int N = MB + NB, ALL = MB * NB;
    unroll<N>([&](auto qt) {
      constexpr int q = decltype(qt)::value;
      io(qt);
#pragma unroll
      for (int n = q * ALL / N; n < (q + 1) * ALL / N; ++n)
        acc[n / NB][n % NB] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(y[n % NB], x[n / NB], acc[n / NB][n % NB], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
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
  bool own = tile.m0 + wm * 16 * MB < a.M && tile.n0 + wn * WCOLS < a.N;  // part of the tile is this wave's
  if (own) first_frags();
  for (;;) {
    // A tile before another takes whole turns of the stages.
    const bool more = PERSIST && v + stride < a.total;
    const Tile next = more ? tile_at(v + stride) : tile;
    const StepSrc next_a = source_a(next, next.split * a.per), next_b = source_b(next, next.split * a.per);
    const int next_k = more ? k_of(next) : 0;
    const int steps = more ? (max(tile.steps, 1) + NST - 1) / NST * NST : tile.steps;
    const int row0 = tile.m0 + wm * 16 * MB, col0 = tile.n0 + wn * WCOLS;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    int kt = 0;
    auto next_step = [&]() {
      if (PERSIST && kt + NST == steps) {
        sa = next_a;
        sb = next_b;
        bleft = ahead = next_k;
        ra = sa.rsrc(ahead, 64);
        rb = sb.rsrc(bleft, 64);
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
    const bool next_own = next.m0 + wm * 16 * MB < a.M && next.n0 + wn * WCOLS < a.N;
    if (more && next_own && !own) first_frags();

    // The columns of a pair of blocks (j, j + 1): as they lie, 8 in a row from `pair` on (B's rows along the lanes), or once
    // the two blocks have swapped halves between their lanes.
    const auto column = [&](int j) { return BT ? col0 + 16 * j + 4 * g : col0 + 32 * (j >> 1) + 8 * g + 4 * (j & 1); };
    const auto pair = [&](int j) { return BT ? col0 + 16 * (j + (g & 1)) + 4 * (g & 2) : col0 + 32 * (j >> 1) + 8 * g; };
    const auto swap = [&](f32x4& x, f32x4& y) {
      if constexpr (BT) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[e]), __float_as_uint(y[e]), false, false);
          x[e] = __uint_as_float(t[0]);
          y[e] = __uint_as_float(t[1]);
        }
      }
    };
    const auto bf16s = [](const f32x4& x, const f32x4& y) {
      return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    };
    // what bf16s leaves of finite values
    const auto rests = [&](const f32x4& x, const f32x4& y, uint4 h) {
      const uint32_t v[4] = {h.x, h.y, h.z, h.w};
      f32x4 q[2] = {x, y};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = q[e >> 2][e & 3] - __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
        q[e >> 2][e & 3] = fabsf(d) < __builtin_inff() ? d : 0.f;
      }
      return bf16s(q[0], q[1]);
    };
    const auto add_bias = [&](f32x4& x, f32x4& y, const float* bias, int c) {
      const float4 u = *reinterpret_cast<const float4*>(bias + c), t = *reinterpret_cast<const float4*>(bias + c + 4);
      x += f32x4{u.x, u.y, u.z, u.w};
      y += f32x4{t.x, t.y, t.z, t.w};
    };
    if constexpr (EPI == GATE) {
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const int row = row0 + 16 * i + r;
#pragma unroll
        for (int j = 0; j < NB / 2; j += 2) {
          const int c = pair(j);
          if (row >= a.M || c >= a.N) continue;
          f32x4 x = acc[i][j], y = acc[i][j + 1], u = acc[i][j + NB / 2], t = acc[i][j + 1 + NB / 2], fx, fy;
          if (a.bias) add_bias(x, y, a.bias, c);
          if (a.bias2) add_bias(u, t, a.bias2, c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float f, df;
            activation(a.act, x[e], f, df);
            fx[e] = f;
            x[e] = df;
            activation(a.act, y[e], f, df);
            fy[e] = f;
            y[e] = df;
          }
          const int64_t o = (int64_t)row * a.N + c;
          const uint4 h = bf16s(fx * u, fy * t);
          st16(a.h + o, h);
          if (a.low) st16(a.h + o + (int64_t)a.low * a.N, rests(fx * u, fy * t, h));
          if (a.p) {
            const int64_t plane = 2 * Float24::elements(a.M, a.N), at = Float24::place(row, c, a.N);
            Float24::store(a.p, plane, at, fx, fy);
            Float24::store(a.s, plane, at, x * u, y * t);
          }
        }
      }
    } else if constexpr (EPI == DGATE) {
      // p and s of a row of blocks are read a row ahead: left to the compiler, each pair of blocks waited for its own
      const int64_t plane = 2 * Float24::elements(a.M, a.N);
      Float24 p[2][NB / 2], s[2][NB / 2];
      const auto fetch = [&](auto it) {
        constexpr int i = decltype(it)::value;
        const int row = row0 + 16 * i + r;
#pragma unroll
        for (int j = 0; j < NB; j += 2) {
          const int c = pair(j);
          const int64_t at = Float24::place(row, c, a.N);
          p[i & 1][j / 2] = s[i & 1][j / 2] = Float24{u32x4{0, 0, 0, 0}, u32x2{0, 0}};
          if (row < a.M && c < a.N) {
            p[i & 1][j / 2].load(a.p, plane, at);
            s[i & 1][j / 2].load(a.s, plane, at);
          }
        }
      };
      fetch(std::integral_constant<int, 0>{});
      unroll<MB>([&](auto it) {
        constexpr int i = decltype(it)::value;
        if constexpr (i + 1 < MB) fetch(std::integral_constant<int, i + 1>{});
        const int row = row0 + 16 * i + r;
#pragma unroll
        for (int j = 0; j < NB; j += 2) {
          f32x4 x = acc[i][j], y = acc[i][j + 1], m, n;
          swap(x, y);
          const int c = pair(j);
          if (row >= (a.low ? a.low : a.M) || 2 * c >= a.ldd) continue;  // few rows: zeros behind the last, for the bias gradients' sums
          if (c >= a.N) x = y = f32x4{0.f, 0.f, 0.f, 0.f};  // the next product contracts over these columns too
          uint16_t* o = a.d + (int64_t)row * a.ldd + c;
          const auto put = [&](uint16_t* o, const Float24& f) {
            f.get(m, n);
            const uint4 v = bf16s(x * m, y * n);
            st16(o, v);
            if (a.low) st16(o + a.low * a.ldd, rests(x * m, y * n, v));
          };
          put(o, s[i & 1][j / 2]);
          put(o + a.ldd / 2, p[i & 1][j / 2]);
        }
      });
    } else if (a.part) {
      float* const c = a.part + (int64_t)tile.split * a.M * a.N;
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const int row = row0 + 16 * i + r;
#pragma unroll
        for (int j = 0; j < NB; ++j)
          if (row < a.M && column(j) < a.N) *reinterpret_cast<f32x4*>(c + (int64_t)row * a.N + column(j)) = acc[i][j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const int row = row0 + 16 * i + r, f = row < a.m_half ? row : row - a.m_half;
        const bool live = row < a.M && f < a.m_live;
        void* const C = row < a.m_half ? a.C : a.C2;
#pragma unroll
        for (int j = 0; j < NB; j += 2) {
          f32x4 x = acc[i][j], y = acc[i][j + 1];
          if (AT && a.f32) {
            float* c = static_cast<float*>(C) + (int64_t)f * a.ldc;
            if (live && column(j) < a.N) *reinterpret_cast<f32x4*>(c + column(j)) = x;
            if (live && column(j + 1) < a.N) *reinterpret_cast<f32x4*>(c + column(j + 1)) = y;
          } else {
            swap(x, y);
            const int c = pair(j);
            if (!live || c >= a.N) continue;
            if (!BT && a.bias) add_bias(x, y, a.bias, c);
            st16(static_cast<uint16_t*>(C) + (int64_t)f * a.ldc + c, bf16s(x, y));
          }
        }
      }
    }
    if (!more) break;
    v += stride;
    tile = next;
    own = next_own;
  }
  // No DMA may land after the workgroup exits.  (Waiting for the loads before the epilogue, so that the next workgroup begins beside
  // its stores, took longer: the gate's gradients of 8192 x 4096 161 -> 177 us.)
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));
}

template <typename P, typename S, int WGS>
__global__ __launch_bounds__(S::THREADS, WGS * S::W / 4) void gated_kernel(const GatedArgs a) {
  __shared__ __align__(1024) unsigned char smem[Operands<P, S>::LDS];
  gated_tiles<P, S>(a, smem, blockIdx.x, gridDim.x);
}
// Two products in one launch, of 128 x 128 tiles: the `first` workgroups of the one with the longer contraction (P0 where `lead`), a
// multiple of 8 (so that the other's are dealt to the XCDs as alone), then the other's.
template <typename P0, typename P1>
__global__ __launch_bounds__(SquareShape::THREADS, SquareShape::W / 2) void gated_pair_kernel(const GatedArgs a, const GatedArgs b, int first,
                                                                                             int lead) {
  __shared__ __align__(1024) unsigned char smem[std::max(Operands<P0, SquareShape>::LDS, Operands<P1, SquareShape>::LDS)];
  const bool ahead = (int)blockIdx.x < first;
  const int v = ahead ? blockIdx.x : blockIdx.x - first;
  if (ahead == (lead != 0)) {
    if (v < a.total) gated_tiles<P0, SquareShape>(a, smem, v, 0);
  } else {
    if (v < b.total) gated_tiles<P1, SquareShape>(b, smem, v, 0);
  }
}

// C = the sum over splits of the parts [splits][M][N], in order, plus the bias; rows as GatedArgs has them.  Up to three products
// in a launch.
struct ReduceArgs {
  GatedArgs a[3];
  int splits[3], first[4];  // first workgroup of each
};
__global__ __launch_bounds__(256) void gated_reduce_kernel(const ReduceArgs q) {
  const int k = ((int)blockIdx.x >= q.first[1]) + ((int)blockIdx.x >= q.first[2]);
  const GatedArgs& a = q.a[k];
  const int64_t n = (int64_t)a.M * a.N, i = ((int64_t)(blockIdx.x - q.first[k]) * 256 + threadIdx.x) * 4;
  if (i >= (a.fold ? (int64_t)a.fold * a.N : n)) return;
  const int row = (int)(i / a.N), col = (int)(i - (int64_t)row * a.N), f = row < a.m_half ? row : row - a.m_half;
  if (f >= a.m_live) return;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 8;
  for (int s = 0; s < q.splits[k]; s += U) {
    float y[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u < q.splits[k]) load4<float>(a.part + (s + u) * n + i, y[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s + u < q.splits[k]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += y[u][e];
      }
  }
  for (int s = 0; a.fold && s < q.splits[k]; ++s) {
    float y[4];
    load4<float>(a.part + s * n + (int64_t)a.fold * a.N + i, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += y[e];
  }
  if (a.bias) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += a.bias[col + e];
  }
  void* const C = row < a.m_half ? a.C : a.C2;
  if (a.f32) store4<float>(static_cast<float*>(C) + (int64_t)f * a.ldc + col, x);
  else store4<uint16_t>(static_cast<uint16_t*>(C) + (int64_t)f * a.ldc + col, x);
}

// ---- few rows, forward alone ------------------------------------------------------------
//
// A workgroup takes ROWS = 16 / SEG rows of the weights (of both, GATED) and all of x; its W waves take the 32-k steps w,
// w + W, ...: every weight is read once, straight into the operand of the matrix cores (lane (r, g): k 8 g .. of a row).  With
// SEG > 1 the operand's 16 rows are SEG segments of k of each row; a product with x's segment s counts in the rows of segment s
// alone, so that few rows of weights still take whole loads, and there are enough workgroups for the chip's bandwidth.  The waves'
// sums are added in LDS.  (Whole rows for both projections, halves for the last: D 1408, F 4096, one row 6.2 and 6.7 us; the last one
// 10.4 by whole rows, 8.7 by quarters.)  h goes from one launch to the next as two bf16 values (16 bits of its significand), so y carries its own
// rounding alone.  What bounds it: latency, and the reads of the weights.
struct ThinArgs {
  int M, N, K;                     // rows (up to 16 NT); rows of the weights, their length
  const uint16_t* x; int64_t ldx;  // [M][K]; the other kernel: h
  uint16_t* h;                     // [2][M][F]: upper and lower part
  const uint16_t *W, *W3;
  const float *bias, *bias3;
  int act;
  uint16_t* y;
};
template <bool GATED, int NT, int SEG, int W, int U>
__global__ __launch_bounds__(64 * W) void gated_thin_kernel(const ThinArgs a) {
  constexpr int MATS = GATED ? 2 : 1, PARTS = GATED ? 1 : 2, ROWS = 16 / SEG;
  __shared__ f32x4 sums[W][MATS][NT][64];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, w = threadIdx.x >> 6;
  const int f0 = blockIdx.x * ROWS, row = f0 + r % ROWS, seg = (a.K + 32 * SEG - 1) / (32 * SEG), k0 = 32 * seg * (r / ROWS);  // steps of a segment
  const uint16_t* p[2] = {a.W + (int64_t)row * a.K + k0 + 8 * g, GATED ? a.W3 + (int64_t)row * a.K + k0 + 8 * g : nullptr};
  const int64_t low = (int64_t)a.M * a.K;  // from h's upper part to its lower one
  f32x4 acc[MATS][NT][SEG];
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int q = 0; q < SEG; ++q) acc[m][t][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = w; s0 < seg; s0 += U * W) {
    bf16x8 v[U][MATS], x[U][NT][SEG][PARTS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + u * W;
      const uint4 zero = make_uint4(0, 0, 0, 0);
      const bool ok = s < seg && row < a.N && k0 + 32 * s + 8 * g < a.K;
#pragma unroll
      for (int m = 0; m < MATS; ++m) v[u][m] = __builtin_bit_cast(bf16x8, ok ? ld16(p[m] + 32 * s) : zero);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int q = 0; q < SEG; ++q) {
          const int n = 16 * t + r, k = 32 * (q * seg + s) + 8 * g;
          const bool live = s < seg && n < a.M && k < a.K;
#pragma unroll
          for (int e = 0; e < PARTS; ++e) x[u][t][q][e] = __builtin_bit_cast(bf16x8, live ? ld16(a.x + e * low + n * a.ldx + k) : zero);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int q = 0; q < SEG; ++q)
#pragma unroll
          for (int e = 0; e < PARTS; ++e)
#pragma unroll
            for (int m = 0; m < MATS; ++m) acc[m][t][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v[u][m], x[u][t][q][e], acc[m][t][q], 0, 0, 0);
  }
  // lane (r, g) holds the operand's rows 4 g + e: segment (4 g) / ROWS counts
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      f32x4 x = acc[m][t][0];
#pragma unroll
      for (int q = 1; q < SEG; ++q)
        if (4 * g / ROWS == q) x = acc[m][t][q];
      sums[w][m][t][lane] = x;
    }
  __syncthreads();
  if (w >= NT) return;
  // wave t: rows 16 t + r of x, weights' rows f0 + (4 g + e) % ROWS
  const int t = w, n = 16 * t + r, f = f0 + 4 * g % ROWS;
  f32x4 out[MATS];
#pragma unroll
  for (int m = 0; m < MATS; ++m) {
    out[m] = sums[0][m][t][lane];
    for (int q = 1; q < W; ++q) out[m] += sums[q][m][t][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // the segments
      if (SEG == 4) out[m][e] += __shfl_xor(out[m][e], 16);
      if (SEG >= 2) out[m][e] += __shfl_xor(out[m][e], 32);
    }
  }
  if (n >= a.M || f >= a.N || 4 * g >= ROWS) return;
  if (a.bias) out[0] += *reinterpret_cast<const f32x4*>(a.bias + f);
  if constexpr (GATED) {
    if (a.bias3) out[1] += *reinterpret_cast<const f32x4*>(a.bias3 + f);
    f32x4 rest;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v, dv;
      activation(a.act, out[0][e], v, dv);
      out[0][e] = v * out[1][e];
      const float d = out[0][e] - bf2f(f2bf(out[0][e]));
      rest[e] = fabsf(d) < __builtin_inff() ? d : 0.f;  // an infinity has no rest
    }
    uint16_t* const h = a.h + (int64_t)n * a.N + f;
    *reinterpret_cast<uint2*>(h) = make_uint2(pack_bf16x2(out[0][0], out[0][1]), pack_bf16x2(out[0][2], out[0][3]));
    *reinterpret_cast<uint2*>(h + (int64_t)a.M * a.N) = make_uint2(pack_bf16x2(rest[0], rest[1]), pack_bf16x2(rest[2], rest[3]));
  } else {
    *reinterpret_cast<uint2*>(a.y + (int64_t)n * a.N + f) =
        make_uint2(pack_bf16x2(out[0][0], out[0][1]), pack_bf16x2(out[0][2], out[0][3]));
  }
}
template <int NT, int S0, int U0, int S1, int W1, int U1>
void launch_thin(const ThinArgs& gate, const ThinArgs& out, hipStream_t st) {
  constexpr int R0 = 16 / S0, R1 = 16 / S1;
  hipLaunchKernelGGL((gated_thin_kernel<true, NT, S0, 8, U0>), dim3((gate.N + R0 - 1) / R0), dim3(512), 0, st, gate);
  hipLaunchKernelGGL((gated_thin_kernel<false, NT, S1, W1, U1>), dim3((out.N + R1 - 1) / R1), dim3(64 * W1), 0, st, out);
}

// ---- launches ------------------------------------------------------------------------------
constexpr size_t up(size_t n) { return (n + 255) & ~size_t(255); }

// 256 x 192 beside the shapes of the head's products: 1536 and 1408 columns are 8 tiles of it, and 8192 rows with them 256, one a CU
// (8192 x 1536 over 4096 k 99 us with 192 tiles of 256 x 256, so 89; over 8192 k 193 and 185, 180 and 173)
constexpr int WIDE = KINDS;
typedef Shape<4, 6, 4, 2, 2> WideShape;
constexpr double kWideStep = 1.38, kWideTile = 9.0;
constexpr int tile_m(int kind) { return kind == WIDE ? 256 : kTm[kind]; }
constexpr int tile_n(int kind) { return kind == WIDE ? 192 : kTn[kind]; }

// As tiling(), without thin tiles and with wide ones
constexpr Tiling choose(int64_t M, int64_t N, int steps, int most, bool wide) {
  Tiling best = tiling(std::max<int64_t>(M, 65), N, steps, most);
  for (int S = 1; wide && S <= most && (S == 1 || steps / S >= 4); ++S) {
    const int64_t tiles = ceil_div(M, 256) * ceil_div(N, 192) * S;
    double t = (double)ceil_div(tiles, 256) * ((double)ceil_div(steps, S) * kWideStep + kWideTile);
    if (S > 1) t += 6.0 + 8.0 * S * (double)M * (double)N / 4.5e6;
    if (t < best.us) best = Tiling{WIDE, S, t};
  }
  return best;
}

// Sizes that follow from the tiling; the number of workgroups
template <typename P>
int prepare(GatedArgs& a, const Tiling& t) {
  a.steps = (a.K + 63) / 64;
  a.per = (a.steps + t.splits - 1) / t.splits;
  a.tiles_m = (a.M + tile_m(t.kind) - 1) / tile_m(t.kind);
  const int tn = P::EPI == GATE ? tile_n(t.kind) / 2 : tile_n(t.kind);
  a.tiles_n = (a.N + tn - 1) / tn;
  a.total = a.tiles_m * a.tiles_n * t.splits;
  return a.total;
}
template <typename P>
void launch(GatedArgs& a, const Tiling& t, hipStream_t st) {
  int n = prepare<P>(a, t);
  if (P::EPI == GATE) n = std::min(n, 256 * (t.kind == SQUARE ? kPerCu[SQUARE] : 1));
  const dim3 grid((unsigned)n);
  if (t.kind == BIG) hipLaunchKernelGGL((gated_kernel<P, BigShape, 1>), grid, dim3(BigShape::THREADS), 0, st, a);
  else if (t.kind == SQUARE) hipLaunchKernelGGL((gated_kernel<P, SquareShape, 2>), grid, dim3(SquareShape::THREADS), 0, st, a);
  else if constexpr (P::EPI == OUT) hipLaunchKernelGGL((gated_kernel<P, WideShape, 1>), grid, dim3(WideShape::THREADS), 0, st, a);
}
template <typename P>
void launch_square(GatedArgs& a, const Tiling& t, hipStream_t st) {
  hipLaunchKernelGGL((gated_kernel<P, SquareShape, 2>), dim3((unsigned)prepare<P>(a, t)), dim3(SquareShape::THREADS), 0, st, a);
}
template <typename P0, typename P1>
void launch_pair(GatedArgs& a, const Tiling& ta, GatedArgs& b, const Tiling& tb, hipStream_t st) {
  const int na = prepare<P0>(a, ta), nb = prepare<P1>(b, tb), lead = a.per >= b.per, first = ((lead ? na : nb) + 7) / 8 * 8;
  hipLaunchKernelGGL((gated_pair_kernel<P0, P1>), dim3((unsigned)(first + (lead ? nb : na))), dim3(SquareShape::THREADS), 0, st, a, b, first,
                     lead);
}
// Adds up the parts of those products that have some
void launch_reduce(const GatedArgs* const* a, const Tiling* const* t, int n, hipStream_t st) {
  ReduceArgs q{};
  int k = 0;
  int64_t blocks = 0;
  for (int i = 0; i < n; ++i) {
    if (!a[i]->part) continue;
    q.a[k] = *a[i];
    q.splits[k] = t[i]->splits;
    blocks += ceil_div((int64_t)(a[i]->fold ? a[i]->fold : a[i]->M) * a[i]->N, 1024);
    q.first[++k] = (int)blocks;
  }
  if (!k) return;
  for (int i = k; i < 3; ++i) q.first[i + 1] = q.first[i];
  hipLaunchKernelGGL(gated_reduce_kernel, dim3((unsigned)blocks), dim3(256), 0, st, q);
}

constexpr int kSplits = 16;
// Rows of a forward alone that the kernels for few of them take (two operands of 16 rows).  us in a graph, D 1408, F 4096, by these and by
// tiles: 1 row 12.1 and 30.8, 16 rows 18.2 and 31.3, 32 rows 27.4 and 32.3; D and F 256: 6.8 and 13.0, 6.9 and 13.8, 7.2 and 14.4
constexpr int kThinRows = 32;
// Rows up to which h, da and du are held as two bf16 values (16 bits of significand), the lower ones kLow rows behind the upper: as more
// rows of the products with the weights, whose 128 x 128 tiles have room for them, and as a second step of those over the rows.  With
// few values their rounding shows: rms errors of single results then lay up to 1.55 times as far out as their own rounding puts them.
// us of a training pass in a graph, D 1408, F 4096, so and in bf16: 1 row 77 and 64, 64 rows 83 and 73 (the host takes 160 without one).
constexpr int kLow = 64;
struct Plan {
  int low, rows;            // kLow or 0; rows of h and d
  int half;                 // columns of da (and of du): F rounded up to 64
  Tiling gate, out, dgate, dx, dw, dw2;
  size_t h, d, part[4];     // h; da and du; parts of out, dx, dw, dw2
  size_t plane;             // p and s, of three bytes
  size_t colsum;
};
// The sizes, and the tilings of a direction's products and what follows from them (a microsecond or two of the host's for each)
enum { SIZES = 0, OF_FORWARD = 1, OF_BACKWARD = 2 };
constexpr Plan tilings_of(const llattn_gated_cfg* c, int which) {
  Plan p{};
  const auto steps = [](int k) { return (k + 63) / 64; };
  const auto part = [](const Tiling& t, int64_t m, int64_t n, bool folded) { return t.splits > 1 || folded ? up((size_t)t.splits * m * n * 4) : 0; };
  p.low = c->rows <= kLow ? kLow : 0;
  p.rows = p.low ? 2 * kLow : c->rows;
  p.half = (c->F + 63) / 64 * 64;
  p.h = up((size_t)p.rows * c->F * 2);
  p.plane = up((size_t)Float24::elements(c->rows, c->F) * 3);
  p.d = up((size_t)p.rows * 2 * p.half * 2);
  if (which == OF_FORWARD) {
    p.gate = choose(c->rows, 2 * (int64_t)c->F, steps(c->D), 1, false);
    p.out = choose(p.rows, c->D_out, steps(c->F), kSplits, true);
    p.part[0] = part(p.out, p.rows, c->D_out, p.low);
  } else if (which == OF_BACKWARD) {
    p.dgate = choose(c->rows, c->F, steps(c->D_out), 1, false);
    p.dx = choose(p.rows, c->D, 2 * steps(c->F), kSplits, true);
    if (p.low) {
      p.dw = p.dw2 = Tiling{SQUARE, 1, 0.0};
    } else {
      p.dw = choose(2 * (int64_t)p.half, c->D, steps(c->rows), kSplits, true);
      p.dw2 = choose(c->D_out, c->F, steps(c->rows), kSplits, true);
    }
    // The gate's gradients wait for memory at the end of a tile, dW2 hardly: side by side on a CU they take less (8192 x 1536 x 4096, before
    // p and s went past the caches: 277 us in a launch of 128 x 128 tiles, apart 121 and 184, or 183 with 128 x 128; 237 since)
    if (p.dw2.kind == SQUARE) p.dgate.kind = SQUARE;
    p.part[1] = part(p.dx, p.rows, c->D, p.low);
    p.part[2] = part(p.dw, 2 * (int64_t)p.half, c->D, false);
    p.part[3] = part(p.dw2, c->D_out, c->F, false);
  }
  return p;
}
Plan plan_of(const llattn_gated_cfg* c, int which) {
  Plan p = tilings_of(c, which);
  if (which == OF_BACKWARD)
    p.colsum = up(std::max(llattn_colsum_workspace_size(p.rows, c->F), llattn_colsum_workspace_size(c->rows, c->D_out)));
  return p;
}
// Forward with a backward to follow, forward alone (h in it, as two bf16 values where rows are few), backward, what is kept between them
enum Space { FORWARD = LLATTN_GATED_FORWARD, ALONE = LLATTN_GATED_ALONE, BACKWARD = LLATTN_GATED_BACKWARD, KEPT = LLATTN_GATED_KEPT };
size_t bytes_of(const llattn_gated_cfg* c, const Plan& p, int which) {
  switch (which) {
    case FORWARD: return std::max<size_t>(p.part[0], 1);
    case ALONE: return c->rows <= kThinRows ? up((size_t)c->rows * c->F * 4) : p.h + p.part[0];
    case BACKWARD: return p.d + p.part[1] + p.part[2] + p.part[3] + p.colsum;
    default: return p.h + 2 * p.plane;
  }
}

int32_t check(const char* who, const llattn_gated_cfg* c) {
  if (!c) return fail(LLATTN_ERR_SHAPE, "%s: null configuration", who);
  const auto width = [](int n) { return n > 0 && n % 8 == 0 && n < 1 << 22; };
  if (c->rows <= 0 || c->rows >= 1 << 23 || !width(c->D) || !width(c->F) || !width(c->D_out))
    return fail(LLATTN_ERR_SHAPE, "%s: rows %d (in [1, 2^23)), D %d, F %d, D_out %d (positive multiples of 8 below 2^22)", who, c->rows,
                c->D, c->F, c->D_out);
  if (c->act != LLATTN_GATE_SILU && c->act != LLATTN_GATE_GELU) return fail(LLATTN_ERR_UNSUPPORTED, "%s: unknown activation %d", who, c->act);
  for (const int32_t t : {c->dw_dtype, c->dw2_dtype})
    if (t != LLATTN_F32 && t != LLATTN_BF16) return fail(LLATTN_ERR_DTYPE, "%s: unknown dtype %d of a weight gradient", who, t);
  return LLATTN_OK;
}

int32_t check_operands(const char* who, const llattn_gated_cfg* c, const void* x, int64_t ldx, const llattn_gated_weights* w,
                       const void* ws, size_t bytes, size_t need) {
  if (!x || !w || !w->W1 || !w->W3 || !w->W2) return fail(LLATTN_ERR_LAYOUT, "%s: null x or weights", who);
  for (const void* p : {x, w->W1, w->W3, w->W2, (const void*)w->b1, (const void*)w->b3, (const void*)w->b2})
    if (!aligned16(p)) return fail(LLATTN_ERR_LAYOUT, "%s: x, weights and biases must be 16-byte aligned", who);
  if (ldx < c->D || ldx % 8 || ldx >= 1 << 23)
    return fail(LLATTN_ERR_LAYOUT, "%s: rows of x: a stride of %lld elements (a multiple of 8 in [D, 2^23))", who, (long long)ldx);
  if (need > 1 && (!ws || bytes < need || !aligned16(ws)))
    return fail(LLATTN_ERR_WORKSPACE, "%s: needs %zu workspace bytes (got %zu)", who, need, bytes);
  return LLATTN_OK;
}

const uint16_t* bf16(const void* p) { return static_cast<const uint16_t*>(p); }

}  // namespace
}  // namespace llattn

using namespace llattn;

extern "C" size_t llattn_gated_bytes(const llattn_gated_cfg* c, int32_t which) {
  if (check("llattn_gated_bytes", c) != LLATTN_OK) return 0;
  if (which < FORWARD || which > KEPT) {
    fail(LLATTN_ERR_SHAPE, "llattn_gated_bytes: unknown buffer %d", which);
    return 0;
  }
  const bool thin = which == ALONE && c->rows <= kThinRows;
  return bytes_of(c, plan_of(c, which == BACKWARD ? OF_BACKWARD : which == KEPT || thin ? SIZES : OF_FORWARD), which);
}

extern "C" int32_t llattn_gated_fwd(const llattn_gated_cfg* c, const void* x, int64_t ldx, const llattn_gated_weights* w, void* kept,
                                    void* y, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int32_t rc = check("llattn_gated_fwd", c)) return rc;
  const bool thin = !kept && c->rows <= kThinRows;
  const Plan plan = plan_of(c, thin ? SIZES : OF_FORWARD);
  const size_t need = bytes_of(c, plan, kept ? FORWARD : ALONE);
  if (const int32_t rc = check_operands("llattn_gated_fwd", c, x, ldx, w, workspace, workspace_bytes, need)) return rc;
  if (!y || !aligned16(y) || !aligned16(kept)) return fail(LLATTN_ERR_LAYOUT, "llattn_gated_fwd: null y, or y or kept not 16-byte aligned");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  if (thin) {
    ThinArgs gate{}, out{};
    gate.M = out.M = c->rows;
    gate.N = out.K = c->F; gate.K = c->D; out.N = c->D_out;
    gate.x = bf16(x); gate.ldx = ldx;
    gate.W = bf16(w->W1); gate.W3 = bf16(w->W3); out.W = bf16(w->W2);
    gate.bias = w->b1; gate.bias3 = w->b3; out.bias = w->b2;
    gate.act = c->act;
    gate.h = reinterpret_cast<uint16_t*>(ws);
    out.x = gate.h; out.ldx = c->F;
    out.y = static_cast<uint16_t*>(y);
    if (c->rows <= 16) launch_thin<1, 1, 6, 2, 8, 8>(gate, out, st);
    else launch_thin<2, 1, 4, 2, 8, 2>(gate, out, st);
    return check_launch("llattn_gated_fwd");
  }
  GatedArgs a{};
  a.M = c->rows; a.N = c->F; a.K = c->D;
  a.A = bf16(x); a.lda = ldx;
  a.B = bf16(w->W1); a.B2 = bf16(w->W3); a.ldb = c->D;
  a.bias = w->b1; a.bias2 = w->b3;
  a.act = c->act;
  a.h = reinterpret_cast<uint16_t*>(kept ? static_cast<char*>(kept) : ws);
  a.low = plan.low;
  if (kept) {
    a.p = static_cast<unsigned char*>(kept) + plan.h;
    a.s = a.p + plan.plane;
  } else {
    ws += plan.h;
  }
  launch<GateProduct>(a, plan.gate, st);
  GatedArgs o{};
  o.M = plan.rows; o.fold = plan.low; o.N = c->D_out; o.K = c->F;
  o.A = a.h; o.lda = c->F;
  o.B = bf16(w->W2); o.ldb = c->F;
  o.bias = w->b2;
  o.C = y; o.ldc = c->D_out; o.m_half = plan.rows; o.m_live = c->rows;
  o.part = plan.part[0] ? reinterpret_cast<float*>(ws) : nullptr;
  launch<OutProduct>(o, plan.out, st);
  const GatedArgs* args[] = {&o};
  const Tiling* tilings[] = {&plan.out};
  launch_reduce(args, tilings, 1, st);
  return check_launch("llattn_gated_fwd");
}

extern "C" int32_t llattn_gated_bwd(const llattn_gated_cfg* c, const void* x, int64_t ldx, const llattn_gated_weights* w,
                                    const void* kept, const void* dy, const llattn_gated_grads* g, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  if (const int32_t rc = check("llattn_gated_bwd", c)) return rc;
  const Plan plan = plan_of(c, OF_BACKWARD);
  if (const int32_t rc = check_operands("llattn_gated_bwd", c, x, ldx, w, workspace, workspace_bytes, bytes_of(c, plan, BACKWARD))) return rc;
  if (!kept || !dy || !g) return fail(LLATTN_ERR_LAYOUT, "llattn_gated_bwd: null kept, dy or gradients");
  for (const void* q : {kept, dy, (const void*)g->dx, (const void*)g->dW1, (const void*)g->dW3, (const void*)g->dW2})
    if (!aligned16(q)) return fail(LLATTN_ERR_LAYOUT, "llattn_gated_bwd: kept, dy and the gradients must be 16-byte aligned");
  if (!g->dW1 != !g->dW3) return fail(LLATTN_ERR_LAYOUT, "llattn_gated_bwd: dW1 and dW3 come together");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  char* at = static_cast<char*>(workspace);
  const auto take = [&](size_t n) { char* q = at; at += n; return q; };
  uint16_t* const d = reinterpret_cast<uint16_t*>(take(plan.d));
  float* part[4] = {};
  for (int k = 1; k < 4; ++k) {
    char* q = take(plan.part[k]);
    if (plan.part[k]) part[k] = reinterpret_cast<float*>(q);
  }
  const int ldd = 2 * plan.half;
  unsigned char* const p = static_cast<unsigned char*>(const_cast<void*>(kept)) + plan.h;

  GatedArgs gate{}, dx{}, dw{}, dw2{};
  const bool on_gate = g->dx || g->dW1 || g->db1 || g->db3, on_dx = g->dx, on_dw = g->dW1, on_dw2 = g->dW2;
  gate.M = c->rows; gate.N = c->F; gate.K = c->D_out;
  gate.A = bf16(dy); gate.lda = c->D_out;
  gate.B = bf16(w->W2); gate.ldb = c->F;
  gate.p = p; gate.s = p + plan.plane;
  gate.d = d; gate.ldd = ldd; gate.low = plan.low;

  dw2.M = c->D_out; dw2.N = c->F; dw2.K = c->rows;
  dw2.A = bf16(dy); dw2.lda = c->D_out;
  dw2.B = bf16(kept); dw2.ldb = c->F;
  dw2.C = g->dW2; dw2.ldc = c->F; dw2.m_half = dw2.m_live = c->D_out;
  dw2.f32 = c->dw2_dtype == LLATTN_F32;
  dw2.part = on_dw2 ? part[3] : nullptr;

  dx.M = plan.rows; dx.fold = plan.low; dx.N = c->D; dx.K = ldd;
  dx.A = d; dx.lda = ldd;
  dx.B = bf16(w->W1); dx.B2 = bf16(w->W3); dx.ldb = c->D;
  dx.half = plan.half / 64; dx.k_half = c->F;
  dx.C = g->dx; dx.ldc = c->D; dx.m_half = plan.rows; dx.m_live = c->rows;
  dx.part = on_dx ? part[1] : nullptr;

  dw.M = ldd; dw.N = c->D; dw.K = c->rows;
  dw.A = d; dw.lda = ldd;
  dw.B = bf16(x); dw.ldb = ldx;
  dw.C = g->dW1; dw.C2 = g->dW3; dw.ldc = c->D; dw.m_half = plan.half; dw.m_live = c->F;
  dw.f32 = c->dw_dtype == LLATTN_F32;
  dw.part = on_dw ? part[2] : nullptr;

  if (plan.low) {  // two steps over the rows: of the upper and the lower halves
    for (GatedArgs* q : {&dw, &dw2}) { q->K = 2 * kLow; q->half = kLow / 64; q->k_half = c->rows; }
    dw.A2 = d + (int64_t)kLow * ldd; dw.B2 = dw.B;
    dw2.A2 = dw2.A; dw2.B2 = dw2.B + (int64_t)kLow * c->F;
  }
  // independent products of 128 x 128 tiles share a launch
  if (on_gate && on_dw2 && plan.dgate.kind == SQUARE && plan.dw2.kind == SQUARE) {
    if (plan.low) launch_pair<DGateProduct, DwHalvesProduct>(gate, plan.dgate, dw2, plan.dw2, st);
    else launch_pair<DGateProduct, DwProduct>(gate, plan.dgate, dw2, plan.dw2, st);
  } else {
    if (on_gate) launch<DGateProduct>(gate, plan.dgate, st);
    if (on_dw2 && plan.low) launch_square<DwHalvesProduct>(dw2, plan.dw2, st);
    else if (on_dw2) launch<DwProduct>(dw2, plan.dw2, st);
  }
  if (on_dx && on_dw && plan.dx.kind == SQUARE && plan.dw.kind == SQUARE) {
    if (plan.low) launch_pair<DxProduct, DwHalvesProduct>(dx, plan.dx, dw, plan.dw, st);
    else launch_pair<DxProduct, DwProduct>(dx, plan.dx, dw, plan.dw, st);
  } else {
    if (on_dx) launch<DxProduct>(dx, plan.dx, st);
    if (on_dw && plan.low) launch_square<DwHalvesProduct>(dw, plan.dw, st);
    else if (on_dw) launch<DwProduct>(dw, plan.dw, st);
  }
  const GatedArgs* args[] = {&dx, &dw, &dw2};
  const Tiling* tilings[] = {&plan.dx, &plan.dw, &plan.dw2};
  launch_reduce(args, tilings, 3, st);
  const auto bias = [&](float* out, const uint16_t* from, int64_t ld, int rows, int n) -> int32_t {
    return out ? llattn_colsum(from, ld, rows, n, out, at, plan.colsum, stream) : LLATTN_OK;
  };
  if (const int32_t rc = bias(g->db1, d, ldd, plan.rows, c->F)) return rc;
  if (const int32_t rc = bias(g->db3, d + plan.half, ldd, plan.rows, c->F)) return rc;
  if (const int32_t rc = bias(g->db2, bf16(dy), c->D_out, c->rows, c->D_out)) return rc;
  return check_launch("llattn_gated_bwd");
}
