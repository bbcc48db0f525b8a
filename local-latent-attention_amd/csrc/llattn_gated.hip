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
// leaves them.  p and s are kept in 24 bits (16 of the significand: their rounding in bf16 would make that sqrt 3, at 8192 x 1536
// x 4096 for 2% of the time), the upper two bytes and the third in planes of their own.
//
// What bounds it: the matrix cores (2 rows D F operations for each of the three products, twice that backward); with few
// rows the reads of the weights.
#include <algorithm>

#include "llattn_lm.h"
#include "llattn_tiles.h"

namespace llattn {
namespace {

using namespace tiles;

// OUT: C (bf16 or fp32); SUM: fp32 parts of it
enum Epilogue { GATE = 0, DGATE = 1, OUT_BF16 = 2, OUT_F32 = 3, SUM = 4 };

struct GatedArgs {
  int M, N, K;                  // GATE: N columns of h
  int steps, per;               // 64-wide k steps, of a split
  int tiles_m, tiles_n, total;  // total: with the splits
  const uint16_t* A; int64_t lda;
  const uint16_t *B, *B2; int64_t ldb;  // B2: the other matrix of a gate, or the one from step `half` on
  int half, k_half;             // two matrices along k: steps and k of the first, k of either
  const float *bias, *bias2;
  uint16_t* h;                  // GATE: [M][N]
  int act;
  unsigned char *p, *s;         // [M][N] of three bytes (Float24), or null (GATE)
  uint16_t* d; int64_t ldd;     // DGATE: [M][ldd], da in its columns, du from column ldd / 2 on
  void *C, *C2; int64_t ldc;    // rows [0, m_live) of each of the two halves of m_half rows (one half: m_half = M)
  int m_half, m_live;
  float* part;                  // SUM: [splits][M][N]
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
// NaN turns into another value.)
struct Float24 {
  uint4 hi;
  uint2 lo;
  static __device__ __forceinline__ uint32_t lows(const f32x4& x) {  // byte 1 of each
    const uint32_t a = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x0c0c0501);
    const uint32_t b = __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x05010c0c);
    return a | b;
  }
  static __device__ __forceinline__ void store(unsigned char* plane, int64_t plane_bytes, int64_t at, const f32x4& x, const f32x4& y) {
    const auto hi2 = [](float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302); };
    st16(plane + 2 * at, make_uint4(hi2(x[0], x[1]), hi2(x[2], x[3]), hi2(y[0], y[1]), hi2(y[2], y[3])));
    *reinterpret_cast<uint2*>(plane + plane_bytes + at) = make_uint2(lows(x), lows(y));
  }
  __device__ __forceinline__ void load(const unsigned char* plane, int64_t plane_bytes, int64_t at) {
    hi = ld16(plane + 2 * at);
    lo = *reinterpret_cast<const uint2*>(plane + plane_bytes + at);
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

// Tiles of a product, as those of the head loss: a 64-k step is two rounds of products, each beside the fragment reads of the
// next: k 0..31 (reads k 32..63), a barrier, k 32..63 (reads the next step's k 0..31 and issues the loads of step
// kt + NST into the stage just read).  Waves whose part of the tile lies outside load and wait like the others and do
// nothing else.  PERSIST: a workgroup takes tile after tile, the next one's first steps loaded in the last ones of this.
// AT: A stored with its rows along k.  BT: B likewise.  TWO: a second matrix B from step `half` on.
template <int EPI, bool AT, bool BT, bool TWO, bool PERSIST, typename S, int WGS>
__global__ __launch_bounds__(S::THREADS, WGS * S::W / 4) void gated_kernel(const GatedArgs a) {
  constexpr int MB = S::MB, NB = S::NB, TM = S::TM, TN = S::TN, NST = S::NST, STAGE = S::STAGE, W = S::W;
  constexpr int TC = EPI == GATE ? TN / 2 : TN;      // columns of the result in a tile,
  constexpr int WCOLS = EPI == GATE ? 8 * NB : 16 * NB;  // and of a wave
  typedef std::conditional_t<AT, ColOp<TM, W>, RowOp<TM, W, false>> OpA;
  typedef std::conditional_t<EPI == GATE, GateOp<TN, W, NB>, std::conditional_t<BT, ColOp<TN, W>, RowOp<TN, W, true>>> OpB;
  constexpr int LOADS = OpA::LOADS + OpB::LOADS;
  static_assert(LOADS <= MB + NB, "the second round's reads carry the loads");
  static_assert((!AT || (16 * MB) % 64 == 0) && (!BT || (16 * NB) % 64 == 0), "ColOp::base");
  static_assert(S::WC == 2 && (S::WR == 2 || S::WR == 4), "wave layouts");
  static_assert(EPI != GATE || (TN / 2) % (8 * OpB::LOADS) == 0, "a wave loads rows of one of the two matrices");
  __shared__ __align__(1024) unsigned char smem[NST * STAGE];
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
    s.full = t ? extent_of(64, ld, n) : extent_of(n, ld, 64);  // not t: chunks past the last k are masked (RowOp::at)
    s.tail = t ? extent_of(K & 63 ? K & 63 : 64, ld, n) : s.full;
    s.inc = t ? (uint32_t)(128 * ld) : 128u;
    return s;
  };
  auto source_a = [&](const Tile& t) { return source(a.A, a.lda, AT, t.m0, min(TM, a.M - t.m0), t.split * a.per, a.K); };
  auto source_b = [&](const Tile& t, int k) {  // from step k on
    const int n = min(TC, a.N - t.n0);
    if constexpr (TWO) return k < a.half ? source(a.B, a.ldb, BT, t.n0, n, k, a.k_half) : source(a.B2, a.ldb, BT, t.n0, n, k - a.half, a.k_half);
    return source(EPI == GATE && 2 * w >= W ? a.B2 : a.B, a.ldb, BT, t.n0, n, k, a.K);
  };
  auto k_of = [&](const Tile& t) { return min(a.K - t.split * a.per * 64, t.steps * 64); };
  int v = blockIdx.x;
  Tile tile = tile_at(v);
  StepSrc sa = source_a(tile), sb = source_b(tile, tile.split * a.per);
  int ahead = k_of(tile);  // k from the step that ra and rb describe to the end of its tile's
  int kb = tile.split * a.per;  // that step, among all
  const auto left_b = [&]() { return TWO ? min(ahead, a.k_half - 64 * (kb < a.half ? kb : kb - a.half)) : ahead; };
  int bleft = left_b();
  i32x4 ra = sa.rsrc(ahead, 64), rb = sb.rsrc(bleft, 64);
  auto advance = [&]() {
    sa.addr += sa.inc;
    sb.addr += sb.inc;
    ahead -= 64;
    if constexpr (TWO) {
      if (++kb == a.half) sb = source_b(tile, kb);
    }
    bleft = left_b();
    ra = sa.rsrc(ahead, 64);
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
    const bool more = PERSIST && v + (int)gridDim.x < a.total;
    const Tile next = more ? tile_at(v + gridDim.x) : tile;
    const StepSrc next_a = source_a(next), next_b = source_b(next, next.split * a.per);
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
          st16(a.h + o, bf16s(fx * u, fy * t));
          if (a.p) {
            const int64_t plane = 2 * (int64_t)a.M * a.N;
            Float24::store(a.p, plane, o, fx, fy);
            Float24::store(a.s, plane, o, x * u, y * t);
          }
        }
      }
    } else if constexpr (EPI == DGATE) {
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const int row = row0 + 16 * i + r;
#pragma unroll
        for (int j = 0; j < NB; j += 2) {
          f32x4 x = acc[i][j], y = acc[i][j + 1];
          swap(x, y);
          const int c = pair(j);
          if (row >= a.M || 2 * c >= a.ldd) continue;
          uint16_t* o = a.d + (int64_t)row * a.ldd + c;
          uint4 da = make_uint4(0, 0, 0, 0), du = da;  // past the last column: zeros, which the products contract over
          if (c < a.N) {
            const int64_t plane = 2 * (int64_t)a.M * a.N, at = (int64_t)row * a.N + c;
            Float24 p, s;
            p.load(a.p, plane, at);
            s.load(a.s, plane, at);
            const auto times = [&](const Float24& q) {
              f32x4 m, n;
              q.get(m, n);
              return bf16s(x * m, y * n);
            };
            da = times(s);
            du = times(p);
          }
          st16(o, da);
          st16(o + a.ldd / 2, du);
        }
      }
    } else if constexpr (EPI == SUM) {
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
          if constexpr (EPI == OUT_F32) {
            float* c = static_cast<float*>(C) + (int64_t)f * a.ldc;
            if (live && column(j) < a.N) *reinterpret_cast<f32x4*>(c + column(j)) = x;
            if (live && column(j + 1) < a.N) *reinterpret_cast<f32x4*>(c + column(j + 1)) = y;
          } else {
            swap(x, y);
            const int c = pair(j);
            if (!live || c >= a.N) continue;
            if (a.bias) add_bias(x, y, a.bias, c);
            st16(static_cast<uint16_t*>(C) + (int64_t)f * a.ldc + c, bf16s(x, y));
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

// C = the sum over splits of the parts [splits][M][N], in order, plus the bias; rows as GatedArgs has them
template <typename T>
__global__ __launch_bounds__(256) void gated_reduce_kernel(const GatedArgs a, int splits) {
  const int64_t n = (int64_t)a.M * a.N;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
    const int row = (int)(i / a.N), col = (int)(i - (int64_t)row * a.N), f = row < a.m_half ? row : row - a.m_half;
    if (f >= a.m_live) continue;
    float x[4];
    load4<float>(a.part + i, x);
    for (int s = 1; s < splits; ++s) {
      float y[4];
      load4<float>(a.part + s * n + i, y);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += y[e];
    }
    if (a.bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += a.bias[col + e];
    }
    store4<T>(static_cast<T*>(row < a.m_half ? a.C : a.C2) + (int64_t)f * a.ldc + col, x);
  }
}

constexpr size_t up(size_t n) { return (n + 255) & ~size_t(255); }

template <int EPI, bool AT, bool BT, bool TWO, bool PERSIST>
void launch(GatedArgs& a, const Tiling& t, hipStream_t st) {
  a.steps = (a.K + 63) / 64;
  a.per = (a.steps + t.splits - 1) / t.splits;
  a.tiles_m = (a.M + kTm[t.kind] - 1) / kTm[t.kind];
  const int tn = EPI == GATE ? kTn[t.kind] / 2 : kTn[t.kind];
  a.tiles_n = (a.N + tn - 1) / tn;
  a.total = a.tiles_m * a.tiles_n * t.splits;
  const dim3 grid((unsigned)(PERSIST ? std::min(a.total, 256 * kPerCu[t.kind]) : a.total));
  if (t.kind == BIG) hipLaunchKernelGGL((gated_kernel<EPI, AT, BT, TWO, PERSIST, BigShape, 1>), grid, dim3(BigShape::THREADS), 0, st, a);
  else if (t.kind == SQUARE) hipLaunchKernelGGL((gated_kernel<EPI, AT, BT, TWO, PERSIST, SquareShape, 2>), grid, dim3(SquareShape::THREADS), 0, st, a);
  else if constexpr (EPI == GATE || EPI == DGATE) hipLaunchKernelGGL((gated_kernel<EPI, AT, BT, TWO, PERSIST, ThinShape, 2>), grid, dim3(ThinShape::THREADS), 0, st, a);
}

// A product into C, whole or in splits
template <bool AT, bool BT, bool TWO>
void product(GatedArgs& a, const Tiling& t, int dtype, float* part, hipStream_t st) {
  if (t.splits > 1) {
    a.part = part;
    launch<SUM, AT, BT, TWO, false>(a, t, st);
    const dim3 grid((unsigned)std::min<int64_t>(ceil_div((int64_t)a.M * a.N, 1024), 8192));
    if (dtype == LLATTN_F32) hipLaunchKernelGGL(gated_reduce_kernel<float>, grid, dim3(256), 0, st, a, t.splits);
    else hipLaunchKernelGGL(gated_reduce_kernel<uint16_t>, grid, dim3(256), 0, st, a, t.splits);
  } else if (dtype == LLATTN_F32) {
    if constexpr (AT) launch<OUT_F32, AT, BT, TWO, false>(a, t, st);
  } else {
    launch<OUT_BF16, AT, BT, TWO, false>(a, t, st);
  }
}

constexpr int kSplits = 16;
struct Plan {
  int half;                 // columns of da (and of du): F rounded up to 64
  Tiling gate, out, dgate, dx, dw, dw2;
  size_t h, d, part[2];     // forward: h, parts; backward: da and du, parts
  size_t colsum;
};
Plan plan_of(const llattn_gated_cfg* c) {
  Plan p{};
  const auto steps = [](int k) { return (k + 63) / 64; };
  const auto part = [](const Tiling& t, int64_t m, int64_t n) { return t.splits > 1 ? up((size_t)t.splits * m * n * 4) : 0; };
  p.half = (c->F + 63) / 64 * 64;
  p.gate = tiling(c->rows, 2 * (int64_t)c->F, steps(c->D), 1);
  p.out = tiling(c->rows, c->D_out, steps(c->F), kSplits);
  p.dgate = tiling(c->rows, c->F, steps(c->D_out), 1);
  p.dx = tiling(c->rows, c->D, 2 * steps(c->F), kSplits);
  p.dw = tiling(2 * (int64_t)p.half, c->D, steps(c->rows), kSplits);
  p.dw2 = tiling(c->D_out, c->F, steps(c->rows), kSplits);
  p.h = up((size_t)c->rows * c->F * 2);
  p.d = up((size_t)c->rows * 2 * p.half * 2);
  p.part[0] = part(p.out, c->rows, c->D_out);
  p.part[1] = std::max({part(p.dx, c->rows, c->D), part(p.dw, 2 * (int64_t)p.half, c->D), part(p.dw2, c->D_out, c->F)});
  p.colsum = up(std::max(llattn_colsum_workspace_size(c->rows, c->F), llattn_colsum_workspace_size(c->rows, c->D_out)));
  return p;
}
size_t bytes_of(const Plan& p, int which) { return which == 0 ? p.h + p.part[0] : p.d + p.part[1] + p.colsum; }

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
  if (ldx < c->D || ldx % 8 || ldx >= 1 << 23) return fail(LLATTN_ERR_LAYOUT, "%s: rows of x: a stride of %lld elements (a multiple of 8 in [D, 2^23))", who, (long long)ldx);
  if (!ws || bytes < need || !aligned16(ws)) return fail(LLATTN_ERR_WORKSPACE, "%s: needs %zu workspace bytes (got %zu)", who, need, bytes);
  return LLATTN_OK;
}

const uint16_t* half_floats(const void* p) { return static_cast<const uint16_t*>(p); }

}  // namespace
}  // namespace llattn

using namespace llattn;

extern "C" size_t llattn_gated_bytes(const llattn_gated_cfg* c, int32_t which) {
  if (check("llattn_gated_bytes", c) != LLATTN_OK) return 0;
  if (which != 0 && which != 1) {
    fail(LLATTN_ERR_SHAPE, "llattn_gated_bytes: unknown workspace %d", which);
    return 0;
  }
  return bytes_of(plan_of(c), which);
}

extern "C" int32_t llattn_gated_fwd(const llattn_gated_cfg* c, const void* x, int64_t ldx, const llattn_gated_weights* w, void* h,
                                    void* p, void* s, void* y, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int32_t rc = check("llattn_gated_fwd", c)) return rc;
  const Plan plan = plan_of(c);
  if (const int32_t rc = check_operands("llattn_gated_fwd", c, x, ldx, w, workspace, workspace_bytes, bytes_of(plan, 0))) return rc;
  if (!y || !p != !s || (p && !h)) return fail(LLATTN_ERR_LAYOUT, "llattn_gated_fwd: y, and for a backward h, p and s");
  for (const void* q : {h, p, s, y})
    if (!aligned16(q)) return fail(LLATTN_ERR_LAYOUT, "llattn_gated_fwd: h, p, s and y must be 16-byte aligned");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  GatedArgs a{};
  a.M = c->rows; a.N = c->F; a.K = c->D;
  a.A = half_floats(x); a.lda = ldx;
  a.B = half_floats(w->W1); a.B2 = half_floats(w->W3); a.ldb = c->D;
  a.bias = w->b1; a.bias2 = w->b3;
  a.act = c->act;
  a.h = static_cast<uint16_t*>(h ? h : ws); a.p = static_cast<unsigned char*>(p); a.s = static_cast<unsigned char*>(s);
  launch<GATE, false, false, false, true>(a, plan.gate, st);
  GatedArgs o{};
  o.M = c->rows; o.N = c->D_out; o.K = c->F;
  o.A = a.h; o.lda = c->F;
  o.B = half_floats(w->W2); o.ldb = c->F;
  o.bias = w->b2;
  o.C = y; o.ldc = c->D_out; o.m_half = o.m_live = c->rows;
  product<false, false, false>(o, plan.out, LLATTN_BF16, reinterpret_cast<float*>(ws + plan.h), st);
  return check_launch("llattn_gated_fwd");
}

extern "C" int32_t llattn_gated_bwd(const llattn_gated_cfg* c, const void* x, int64_t ldx, const llattn_gated_weights* w,
                                    const void* h, const void* p, const void* s, const void* dy, const llattn_gated_grads* g,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  if (const int32_t rc = check("llattn_gated_bwd", c)) return rc;
  const Plan plan = plan_of(c);
  if (const int32_t rc = check_operands("llattn_gated_bwd", c, x, ldx, w, workspace, workspace_bytes, bytes_of(plan, 1))) return rc;
  if (!h || !p || !s || !dy || !g) return fail(LLATTN_ERR_LAYOUT, "llattn_gated_bwd: null h, p, s, dy or gradients");
  for (const void* q : {h, p, s, dy, (const void*)g->dx, (const void*)g->dW1, (const void*)g->dW3, (const void*)g->dW2})
    if (!aligned16(q)) return fail(LLATTN_ERR_LAYOUT, "llattn_gated_bwd: h, p, s, dy and the gradients must be 16-byte aligned");
  if (!g->dW1 != !g->dW3) return fail(LLATTN_ERR_LAYOUT, "llattn_gated_bwd: dW1 and dW3 come together");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  uint16_t* const d = reinterpret_cast<uint16_t*>(ws);
  float* const part = reinterpret_cast<float*>(ws + plan.d);
  void* const sums = ws + plan.d + plan.part[1];
  const int ldd = 2 * plan.half;
  if (g->dx || g->dW1 || g->db1 || g->db3) {
    GatedArgs a{};
    a.M = c->rows; a.N = c->F; a.K = c->D_out;
    a.A = half_floats(dy); a.lda = c->D_out;
    a.B = half_floats(w->W2); a.ldb = c->F;
    a.p = static_cast<unsigned char*>(const_cast<void*>(p)); a.s = static_cast<unsigned char*>(const_cast<void*>(s));
    a.d = d; a.ldd = ldd;
    launch<DGATE, false, true, false, true>(a, plan.dgate, st);
  }
  if (g->dx) {
    GatedArgs a{};
    a.M = c->rows; a.N = c->D; a.K = ldd;
    a.A = d; a.lda = ldd;
    a.B = half_floats(w->W1); a.B2 = half_floats(w->W3); a.ldb = c->D;
    a.half = plan.half / 64; a.k_half = c->F;
    a.C = g->dx; a.ldc = c->D; a.m_half = a.m_live = c->rows;
    product<false, true, true>(a, plan.dx, LLATTN_BF16, part, st);
  }
  if (g->dW1) {
    GatedArgs a{};
    a.M = ldd; a.N = c->D; a.K = c->rows;
    a.A = d; a.lda = ldd;
    a.B = half_floats(x); a.ldb = ldx;
    a.C = g->dW1; a.C2 = g->dW3; a.ldc = c->D; a.m_half = plan.half; a.m_live = c->F;
    product<true, true, false>(a, plan.dw, c->dw_dtype, part, st);
  }
  if (g->dW2) {
    GatedArgs a{};
    a.M = c->D_out; a.N = c->F; a.K = c->rows;
    a.A = half_floats(dy); a.lda = c->D_out;
    a.B = half_floats(h); a.ldb = c->F;
    a.C = g->dW2; a.ldc = c->F; a.m_half = a.m_live = c->D_out;
    product<true, true, false>(a, plan.dw2, c->dw2_dtype, part, st);
  }
  const auto bias = [&](float* out, const uint16_t* from, int64_t ld, int n) -> int32_t {
    return out ? llattn_colsum(from, ld, c->rows, n, out, sums, plan.colsum, stream) : LLATTN_OK;
  };
  if (const int32_t rc = bias(g->db1, d, ldd, c->F)) return rc;
  if (const int32_t rc = bias(g->db3, d + plan.half, ldd, c->F)) return rc;
  if (const int32_t rc = bias(g->db2, half_floats(dy), c->D_out, c->D_out)) return rc;
  return check_launch("llattn_gated_bwd");
}
