// Newton-Schulz orthogonalisation and the weight update made of it (include/llattn_train.h).
//
//   X = U / (|U|_F + eps)  (m x n, m <= n)
//   A = X Xᵀ,  B = b A + c A A,  X <- a X + B X        (steps times)
//
// Precision.  A step multiplies small singular values by a = 3.4445, five steps by 485, and with them whatever the
// roundings of X, A and B leave there: bf16 matrices (half a step of 2^-8) leave order-1 errors in directions that a
// gradient hardly has, fp32 ones nothing.  Matrices are held as hi + lo, two fp16 halves (22 bits), and a product as
// hi hi + hi lo + lo hi on the fp16 matrix cores with fp32 accumulation: what is left out, lo lo, is 2^-22 of it.
// Against float64 that is as exact as fp32 products are (64 x 64 to 1408 x 1408, flat, decaying and low-rank spectra:
// within 2% of fp32's own error; two bf16 halves: 10 to 20 times that), at a third of the 16-bit rate, five times the
// fp32 one.  Scales are powers of two: X is held times S_X ~ sqrt(m n) (its entries average 1 / sqrt(m n)), A and B times
// 2^12 (their entries are at most a few).
//
// Storage: a row holds, for each block of 32 columns, its 32 hi and then its 32 lo halves: 128 bytes, one cache line.
// A k step of 32 is then laid out like a 64-k step of the bf16 products, and their loads and fragment reads serve.
// Rows and columns are padded to whole tiles with zeros, which the iteration keeps, so the loops know no edges.
//
// A and B are symmetric: tiles on and above the diagonal are computed and written to both sides.
#include <algorithm>
#include <cmath>

#include "llattn_gemm.h"
#include "llattn_train.h"

namespace llattn {
namespace {

using namespace gemm;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

constexpr float kSA = 4096.f;  // scale of A and B

template <typename P>
struct Table { P p[LLATTN_MUON_BATCH]; };

__device__ __forceinline__ float load_as(const void* p, int64_t i, int dtype) {
  return dtype == LLATTN_F32 ? static_cast<const float*>(p)[i] : bf2f(static_cast<const uint16_t*>(p)[i]);
}

// ---- momentum and |U|^2 -----------------------------------------------------------
struct PrepArgs {
  Table<const void*> g;
  Table<const float*> m;
  Table<float*> m_out;
  int64_t n;       // elements of a matrix
  int g_dtype, momentum, nesterov, blocks;
  float mu, one_mu;
  double* part;    // [batch][blocks]
};

__device__ __forceinline__ float direction(float g, float m, float mu, float one_mu, int nesterov) {
  return nesterov ? fmaf(mu, m, one_mu * g) : m;
}

// Sum of a workgroup's 256 values, in a fixed order, in every thread.
__device__ __forceinline__ double block_sum(double v, double* s) {
  s[threadIdx.x] = v;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if ((int)threadIdx.x < o) s[threadIdx.x] += s[threadIdx.x + o];
    __syncthreads();
  }
  return s[0];
}

// m_out = mu m + (1 - mu) g and the workgroup's share of |U|^2, in 64 bits (any fp32 values, squares included).
__global__ __launch_bounds__(256) void muon_prep_kernel(const PrepArgs a) {
  __shared__ double s[256];
  const int b = blockIdx.y;
  const void* g = a.g.p[b];
  const float* m = a.m.p[b];
  float* mo = a.m_out.p[b];
  double sum = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.n; i += (int64_t)a.blocks * 256) {
    float u = load_as(g, i, a.g_dtype);
    if (a.momentum) {
      const float v = fmaf(a.mu, m[i], a.one_mu * u);
      mo[i] = v;
      u = direction(u, v, a.mu, a.one_mu, a.nesterov);
    }
    sum += (double)u * (double)u;
  }
  sum = block_sum(sum, s);
  if (threadIdx.x == 0) a.part[(int64_t)b * a.blocks + blockIdx.x] = sum;
}

// ---- X = U / (|U| + eps) as halves, transposed if rows > cols -----------------------
struct SplitArgs {
  Table<const void*> g;
  Table<const float*> m;   // the new momentum
  int rows, cols, flip, g_dtype, momentum, nesterov, blocks;
  float mu, one_mu, eps, scale;
  const double* part;
  uint16_t* x; int64_t ld, batch_stride;  // 16-bit elements
  int mp, np;
};

__device__ __forceinline__ uint16_t h_bits(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }
__device__ __forceinline__ float h_val(uint16_t v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }

// position of column c within a row
__device__ __forceinline__ int hi_at(int c) { return (c >> 5) * 64 + (c & 31); }

__device__ __forceinline__ void store_halves4(uint16_t* row, int c, const float v[4]) {
  uint16_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    h[e] = h_bits(v[e]);
    l[e] = h_bits(v[e] - h_val(h[e]));
  }
  uint16_t* p = row + hi_at(c);
  *reinterpret_cast<uint2*>(p) = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
  *reinterpret_cast<uint2*>(p + 32) = make_uint2(l[0] | (uint32_t)l[1] << 16, l[2] | (uint32_t)l[3] << 16);
}
__device__ __forceinline__ void load_halves4(const uint16_t* row, int c, float v[4]) {
  const uint16_t* p = row + hi_at(c);
  const f16x4 h = *reinterpret_cast<const f16x4*>(p), l = *reinterpret_cast<const f16x4*>(p + 32);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)h[e] + (float)l[e];
}

// One 64 x 64 tile of X per workgroup, through LDS (the reads run along U's rows either way).
__global__ __launch_bounds__(256) void muon_split_kernel(const SplitArgs a) {
  __shared__ double s[256];
  __shared__ float tile[64][65];
  const int b = blockIdx.y, tn = a.np / 64, r0 = blockIdx.x / tn * 64, c0 = blockIdx.x % tn * 64;
  double sum = 0.0;
  for (int i = threadIdx.x; i < a.blocks; i += 256) sum += a.part[(int64_t)b * a.blocks + i];
  const double f = (double)a.scale / (sqrt(block_sum(sum, s)) + (double)a.eps);
  const void* g = a.g.p[b];
  const float* m = a.m.p[b];
  const int u0 = a.flip ? c0 : r0, v0 = a.flip ? r0 : c0;  // the tile's origin in U
  for (int q = threadIdx.x; q < 4096; q += 256) {
    const int lr = q >> 6, lc = q & 63, r = u0 + lr, c = v0 + lc;
    float u = 0.f;
    if (r < a.rows && c < a.cols) {
      const int64_t i = (int64_t)r * a.cols + c;
      u = load_as(g, i, a.g_dtype);
      if (a.momentum) u = direction(u, m[i], a.mu, a.one_mu, a.nesterov);
      u = (float)((double)u * f);
    }
    tile[lr][lc] = u;
  }
  __syncthreads();
  uint16_t* x = a.x + b * a.batch_stride;
  for (int q = threadIdx.x; q < 1024; q += 256) {
    const int lr = q >> 4, lc = (q & 15) * 4;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a.flip ? tile[lc + e][lr] : tile[lr][lc + e];
    store_halves4(x + (int64_t)(r0 + lr) * a.ld, c0 + lc, v);
  }
}

// ---- the products -------------------------------------------------------------------
enum NsMode { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3 };

struct NsArgs {
  const uint16_t* A; int64_t lda, a_stride;  // rows of the tile, k along them
  const uint16_t* B; int64_t ldb, b_stride;  // GRAM, POLY: rows = columns of the tile; APPLY, LAST: rows = k
  const uint16_t* D; int64_t ldd, d_stride;  // POLY: A; APPLY, LAST: X
  uint16_t* C; int64_t ldc, c_stride;
  int steps;                                 // of 32 k
  int tiles, tiles_n;                        // of one matrix; GRAM, POLY: of the upper triangle, and its side
  float alpha, beta;                         // C = alpha D + beta (products), in stored scales
  // LAST
  int rows, cols, flip, w_dtype, update;
  float keep, step;
  Table<const void*> w;
  Table<void*> out;
};

// k-major operand of a step: 32 k-rows of T columns (4 T bytes each); chunk c (16 bytes) of k-row k at c ^ 2 (k & 3).
template <int T>
struct ColOp {
  static constexpr int BYTES = T * 128, NB = BYTES / 1024 / 4, PER = T / 4;
  uint32_t off[NB];
  __device__ __forceinline__ void init(int64_t ld, int w4, int lane) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int q = (w4 * NB + i) * 64 + lane, k = q / PER, c = (q % PER) ^ (2 * (k & 3));
      off[i] = (uint32_t)((int64_t)k * ld * 2 + 16 * c);
    }
  }
  __device__ __forceinline__ void dma(const i32x4& rs, unsigned char* st, int w4, int i) const {
    dma_block(rs, off[i], st + (w4 * NB + i) * 1024);
  }
  // columns o16 + r, k 8 g .. 8 g + 7; half 0: hi, 1: lo
  static __device__ __forceinline__ f16x8 frag(const unsigned char* st, int o16, int r, int g, int half) {
    const int byte = (o16 >> 5) * 128 + half * 64 + (o16 & 31) * 2 + 8 * (r & 3), chunk = byte >> 4, inner = byte & 15;
    bf16x4 hv[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = 8 * g + 4 * q + (r >> 2);
      const unsigned char* p = st + k * (4 * T) + ((chunk ^ (2 * (k & 3))) << 4) + inner;
      hv[q] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(p));
    }
    return __builtin_bit_cast(f16x8, bf16x8{hv[0][0], hv[0][1], hv[0][2], hv[0][3], hv[1][0], hv[1][1], hv[1][2], hv[1][3]});
  }
};

// T x T tiles, four waves (2 x 2), NST stages of 32 k, loads NST - 1 steps ahead, one barrier a step (as in
// llattn_gemm_tile.hip).
template <int MODE, int T, int NST>
__global__ __launch_bounds__(256) void ns_kernel(const NsArgs a) {
  constexpr bool SYM = MODE == GRAM || MODE == POLY;
  constexpr int NBK = T / 32;  // 16 x 16 blocks of a wave per side
  typedef TileOp<true, false, T> OpA;
  typedef std::conditional_t<SYM, OpA, ColOp<T>> OpB;
  constexpr int STAGE = OpA::BYTES + OpB::BYTES, LOADS = OpA::NB + OpB::NB;
  __shared__ __align__(1024) unsigned char smem[NST * STAGE];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  const int v = xcd_remap(blockIdx.x, gridDim.x), b = v / a.tiles, t = v % a.tiles;
  int tm, tn;
  if constexpr (SYM) {  // t = tn (tn + 1) / 2 + tm, tm <= tn
    tn = (int)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while (tn * (tn + 1) / 2 > t) --tn;
    while ((tn + 1) * (tn + 2) / 2 <= t) ++tn;
    tm = t - tn * (tn + 1) / 2;
  } else {  // groups of 8 tile rows
    const int tiles_m = a.tiles / a.tiles_n, group = t / (8 * a.tiles_n), gm = min(tiles_m - group * 8, 8);
    tm = group * 8 + t % (8 * a.tiles_n) % gm;
    tn = t % (8 * a.tiles_n) / gm;
  }
  const int m0 = __builtin_amdgcn_readfirstlane(tm * T), n0 = __builtin_amdgcn_readfirstlane(tn * T);
  const uint16_t* A = a.A + b * a.a_stride + m0 * a.lda;
  const uint16_t* B = a.B + b * a.b_stride + (SYM ? n0 * a.ldb : (int64_t)n0 * 2);
  OpA oa;
  OpB ob;
  oa.init(a.lda, 0, T, wave, lane);
  if constexpr (SYM) ob.init(a.ldb, 0, T, wave, lane);
  else ob.init(a.ldb, wave, lane);
  auto rsrc = [](const uint16_t* p) {  // operands are padded to whole tiles and steps: every offset lies inside
    const uint64_t addr = reinterpret_cast<uint64_t>(p);
    return i32x4{(int)(uint32_t)addr, (int)((addr >> 32) & 0xffff), (int)kOffPastK, kRsrcWord3};
  };
  auto fetch = [&](int kt) {  // step kt (the last one again past the end: never read) into stage kt % NST
    const int k = min(kt, a.steps - 1);
    const i32x4 ra = rsrc(A + (int64_t)k * 64), rb = rsrc(SYM ? B + (int64_t)k * 64 : B + (int64_t)k * 32 * a.ldb);
    unsigned char* st = smem + (kt % NST) * STAGE;
#pragma unroll
    for (int i = 0; i < OpA::NB; ++i) oa.dma(ra, st, wave, i, SK);
#pragma unroll
    for (int i = 0; i < OpB::NB; ++i) {
      if constexpr (SYM) ob.dma(rb, st + OpA::BYTES, wave, i, SK);
      else ob.dma(rb, st + OpA::BYTES, wave, i);
    }
  };
  f32x4 acc[NBK][NBK];
#pragma unroll
  for (int i = 0; i < NBK; ++i)
#pragma unroll
    for (int j = 0; j < NBK; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) fetch(s);
  for (int kt = 0; kt < a.steps; ++kt) {
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0((NST - 2) * LOADS));  // this wave's loads of step kt have landed
    __builtin_amdgcn_s_barrier();  // every wave's; and every wave has read step kt - 1, whose stage is free
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    fetch(kt + NST - 1);
    const unsigned char* st = smem + (kt % NST) * STAGE;
    f16x8 fa[2][NBK], fb[2][NBK];  // hi, lo
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < NBK; ++j) fb[h][j] = __builtin_bit_cast(f16x8, OpB::frag(st + OpA::BYTES, wn * 16 * NBK + 16 * j, r, g, h));
#pragma unroll
      for (int i = 0; i < NBK; ++i) fa[h][i] = __builtin_bit_cast(f16x8, OpA::frag(st, wm * 16 * NBK + 16 * i, r, g, h));
    }
#pragma unroll
    for (int p = 0; p < 3; ++p)  // hi hi, hi lo, lo hi; B first: lane (r, g) accumulates C[r][4 g + e]
#pragma unroll
      for (int i = 0; i < NBK; ++i)
#pragma unroll
        for (int j = 0; j < NBK; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[p == 1][j], fa[p == 2][i], acc[i][j], 0, 0, 0);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // no DMA may land after the workgroup exits

  const uint16_t* D = MODE == GRAM ? nullptr : a.D + b * a.d_stride;
  uint16_t* C = MODE == LAST ? nullptr : a.C + b * a.c_stride;
#pragma unroll
  for (int i = 0; i < NBK; ++i) {
    const int row = m0 + wm * 16 * NBK + 16 * i + r;
#pragma unroll
    for (int j = 0; j < NBK; ++j) {
      const int col = n0 + wn * 16 * NBK + 16 * j + 4 * g;
      float x[4] = {a.beta * acc[i][j][0], a.beta * acc[i][j][1], a.beta * acc[i][j][2], a.beta * acc[i][j][3]};
      if constexpr (MODE != GRAM) {
        float d[4];
        load_halves4(D + row * a.ldd, col, d);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf(a.alpha, d[e], x[e]);
      }
      if constexpr (MODE != LAST) {
        store_halves4(C + row * a.ldc, col, x);
        if (SYM && tm != tn) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint16_t h = h_bits(x[e]);
            uint16_t* p = C + (col + e) * a.ldc + hi_at(row);
            p[0] = h;
            p[32] = h_bits(x[e] - h_val(h));
          }
        }
      } else {
        const int M = a.flip ? a.cols : a.rows, N = a.flip ? a.rows : a.cols;
        if (row >= M) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (col + e >= N) continue;
          const int64_t o = a.flip ? (int64_t)(col + e) * a.cols + row : (int64_t)row * a.cols + col + e;
          float y = x[e];
          if (a.update) y = fmaf(-a.step, y, a.keep * load_as(a.w.p[b], o, a.w_dtype));
          if (a.w_dtype == LLATTN_F32) static_cast<float*>(a.out.p[b])[o] = y;
          else static_cast<uint16_t*>(a.out.p[b])[o] = f2bf(y);
        }
      }
    }
  }
}

// ---- host -----------------------------------------------------------------------------
constexpr size_t up(size_t n) { return (n + 255) & ~size_t(255); }

struct Plan {
  int m, n, T, mp, np, blocks;
  size_t x, a, part;  // bytes of one X, of one A (whole batch), of the partial sums
  size_t bytes() const { return 2 * x + 2 * a + part; }
};

// 128 x 128 tiles where X has at least one for every CU, else 64 x 64.
Plan plan_of(const llattn_muon_cfg* c) {
  Plan p{};
  p.m = std::min(c->rows, c->cols);
  p.n = std::max(c->rows, c->cols);
  const int64_t t128 = (int64_t)c->batch * ((p.m + 127) / 128) * ((p.n + 127) / 128);
  p.T = t128 >= 256 ? 128 : 64;
  p.mp = (p.m + p.T - 1) / p.T * p.T;
  p.np = (p.n + p.T - 1) / p.T * p.T;
  p.blocks = (int)std::min<int64_t>(256, ((int64_t)p.m * p.n + 4095) / 4096);
  p.x = up((size_t)c->batch * p.mp * p.np * 4);
  p.a = up((size_t)c->batch * p.mp * p.mp * 4);
  p.part = up((size_t)c->batch * p.blocks * 8);
  return p;
}

// Largest |p(s)| over s in [0, top] of p(s) = a s + b s^3 + c s^5, and of b s^2 + c s^4 into `poly`.
double grow(double a, double b, double c, double top, double* poly) {
  const auto p = [&](double s) { return std::fabs(s * (a + s * s * (b + s * s * c))); };
  double best = p(top);
  const double disc = 9.0 * b * b - 20.0 * a * c;  // p'(s) = a + 3 b s^2 + 5 c s^4
  if (c != 0.0 && disc >= 0.0) {
    for (const double sign : {-1.0, 1.0}) {
      const double y = (-3.0 * b + sign * std::sqrt(disc)) / (10.0 * c);
      if (y > 0.0 && y < top * top) best = std::max(best, p(std::sqrt(y)));
    }
  } else if (c == 0.0 && b != 0.0 && -a / (3.0 * b) > 0.0 && -a / (3.0 * b) < top * top) {
    best = std::max(best, p(std::sqrt(-a / (3.0 * b))));
  }
  const auto q = [&](double y) { return std::fabs(y * (b + y * c)); };
  double most = q(top * top);
  if (c != 0.0 && -b / (2.0 * c) > 0.0 && -b / (2.0 * c) < top * top) most = std::max(most, q(-b / (2.0 * c)));
  *poly = std::max(*poly, most);
  return best;
}

int32_t check(const llattn_muon_cfg* c) {
  if (!c) return fail(LLATTN_ERR_SHAPE, "llattn_muon: null configuration");
  if (c->batch <= 0 || c->batch > LLATTN_MUON_BATCH || c->rows <= 0 || c->cols <= 0 || c->rows > 32768 || c->cols > 32768)
    return fail(LLATTN_ERR_SHAPE, "llattn_muon: batch %d (1 to %d), %d x %d matrices (1 to 32768)", c->batch,
                LLATTN_MUON_BATCH, c->rows, c->cols);
  for (const int d : {c->g_dtype, c->w_dtype})
    if (d != LLATTN_F32 && d != LLATTN_BF16) return fail(LLATTN_ERR_DTYPE, "llattn_muon: unknown dtype %d", d);
  if (c->steps < 1 || c->steps > 100) return fail(LLATTN_ERR_SHAPE, "llattn_muon: %d steps (1 to 100)", c->steps);
  if (!(c->eps >= 0.f) || !std::isfinite(c->eps)) return fail(LLATTN_ERR_SHAPE, "llattn_muon: eps %g must not be negative", c->eps);
  double s = 1.0, poly = 0.0;  // singular values start in [0, 1]: the Frobenius norm bounds the largest
  for (int i = 0; i < c->steps; ++i) {
    s = grow(c->a, c->b, c->c, s, &poly);
    if (!(s < 3.8) || !(poly < 15.0))
      return fail(LLATTN_ERR_UNSUPPORTED, "llattn_muon: with coefficients (%g, %g, %g) singular values reach %g and the "
                  "polynomial %g in step %d (below 3.8 and 15 are held)", c->a, c->b, c->c, s, poly, i + 1);
  }
  return LLATTN_OK;
}

template <int MODE>
void launch_ns(NsArgs& a, const Plan& p, int batch, hipStream_t st) {
  const int tm = p.mp / p.T, tn = p.np / p.T;
  a.tiles_n = MODE == GRAM || MODE == POLY ? tm : tn;
  a.tiles = MODE == GRAM || MODE == POLY ? tm * (tm + 1) / 2 : tm * tn;
  const dim3 grid((unsigned)(a.tiles * batch)), block(256);
  if (p.T == 128) hipLaunchKernelGGL((ns_kernel<MODE, 128, 2>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((ns_kernel<MODE, 64, 3>), grid, block, 0, st, a);
}

int32_t run(const char* who, const llattn_muon_cfg* c, const void* const* g, const float* const* m, const void* const* w,
            float* const* m_out, void* const* out, void* workspace, size_t workspace_bytes, hipStream_t st) {
  if (const int32_t rc = check(c)) return rc;
  const Plan p = plan_of(c);
  if (!workspace || workspace_bytes < p.bytes() || !aligned16(workspace))
    return fail(LLATTN_ERR_WORKSPACE, "%s: needs %zu workspace bytes (got %zu)", who, p.bytes(), workspace_bytes);
  const bool update = m != nullptr;
  if (!g || !out || (update && (!w || !m_out))) return fail(LLATTN_ERR_LAYOUT, "%s: null pointer array", who);
  const auto misplaced = [](const void* q, int dtype) { return !q || (uintptr_t)q % (size_t)elem_size(dtype); };
  for (int i = 0; i < c->batch; ++i)
    if (misplaced(g[i], c->g_dtype) || misplaced(out[i], c->w_dtype) ||
        (update && (misplaced(m[i], LLATTN_F32) || misplaced(m_out[i], LLATTN_F32) || misplaced(w[i], c->w_dtype))))
      return fail(LLATTN_ERR_LAYOUT, "%s: matrix %d has a null or misaligned pointer", who, i);
  char* ws = static_cast<char*>(workspace);
  uint16_t* X[2] = {reinterpret_cast<uint16_t*>(ws), reinterpret_cast<uint16_t*>(ws + p.x)};
  uint16_t* A = reinterpret_cast<uint16_t*>(ws + 2 * p.x);
  uint16_t* B = reinterpret_cast<uint16_t*>(ws + 2 * p.x + p.a);
  double* part = reinterpret_cast<double*>(ws + 2 * p.x + 2 * p.a);
  const float sx = std::exp2f((float)std::min(14, (int)(0.5 * std::log2((double)p.m * p.n))));
  const float one_mu = (float)(1.0 - (double)c->mu);

  PrepArgs pa{};
  SplitArgs sa{};
  NsArgs na{};
  for (int i = 0; i < c->batch; ++i) {
    pa.g.p[i] = sa.g.p[i] = g[i];
    na.out.p[i] = out[i];
    if (!update) continue;
    pa.m.p[i] = m[i];
    pa.m_out.p[i] = m_out[i];
    sa.m.p[i] = m_out[i];
    na.w.p[i] = w[i];
  }
  pa.n = (int64_t)c->rows * c->cols;
  pa.g_dtype = sa.g_dtype = c->g_dtype;
  pa.momentum = sa.momentum = update;
  pa.nesterov = sa.nesterov = c->nesterov;
  pa.blocks = sa.blocks = p.blocks;
  pa.mu = sa.mu = c->mu;
  pa.one_mu = sa.one_mu = one_mu;
  pa.part = part;
  hipLaunchKernelGGL(muon_prep_kernel, dim3(p.blocks, c->batch), dim3(256), 0, st, pa);
  sa.rows = c->rows; sa.cols = c->cols; sa.flip = c->rows > c->cols;
  sa.eps = c->eps; sa.scale = sx; sa.part = part;
  sa.x = X[0]; sa.ld = 2 * (int64_t)p.np; sa.batch_stride = (int64_t)p.mp * p.np * 2;
  sa.mp = p.mp; sa.np = p.np;
  hipLaunchKernelGGL(muon_split_kernel, dim3((p.mp / 64) * (p.np / 64), c->batch), dim3(256), 0, st, sa);

  const int64_t lx = sa.ld, sx_stride = sa.batch_stride, la = 2 * (int64_t)p.mp, sa_stride = (int64_t)p.mp * p.mp * 2;
  na.rows = c->rows; na.cols = c->cols; na.flip = sa.flip; na.w_dtype = c->w_dtype; na.update = update;
  na.keep = c->keep; na.step = c->step;
  for (int i = 0; i < c->steps; ++i) {
    const uint16_t* x = X[i & 1];
    na.A = na.B = x; na.lda = na.ldb = lx; na.a_stride = na.b_stride = sx_stride;
    na.C = A; na.ldc = la; na.c_stride = sa_stride;
    na.steps = p.np / 32; na.beta = kSA / (sx * sx);
    launch_ns<GRAM>(na, p, c->batch, st);
    na.A = na.B = na.D = A; na.lda = na.ldb = na.ldd = la; na.a_stride = na.b_stride = na.d_stride = sa_stride;
    na.C = B;
    na.steps = p.mp / 32; na.alpha = c->b; na.beta = c->c / kSA;
    launch_ns<POLY>(na, p, c->batch, st);
    na.A = B;
    na.B = na.D = x; na.ldb = na.ldd = lx; na.b_stride = na.d_stride = sx_stride;
    na.C = X[(i + 1) & 1]; na.ldc = lx; na.c_stride = sx_stride;
    na.alpha = c->a; na.beta = 1.f / kSA;
    if (i + 1 < c->steps) {
      launch_ns<APPLY>(na, p, c->batch, st);
    } else {
      na.alpha /= sx;
      na.beta /= sx;
      launch_ns<LAST>(na, p, c->batch, st);
    }
  }
  return check_launch(who);
}

}  // namespace
}  // namespace llattn

using namespace llattn;

extern "C" size_t llattn_muon_bytes(const llattn_muon_cfg* c) { return check(c) == LLATTN_OK ? plan_of(c).bytes() : 0; }

extern "C" int32_t llattn_orthogonalize(const llattn_muon_cfg* c, const void* const* g, void* const* out, void* workspace,
                                        size_t workspace_bytes, void* stream) {
  return run("llattn_orthogonalize", c, g, nullptr, nullptr, nullptr, out, workspace, workspace_bytes,
             static_cast<hipStream_t>(stream));
}

extern "C" int32_t llattn_muon_update(const llattn_muon_cfg* c, const void* const* g, const float* const* m,
                                      const void* const* w, float* const* m_out, void* const* w_out, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  if (!m) return fail(LLATTN_ERR_LAYOUT, "llattn_muon_update: null momentum array");
  if (c && !(c->mu >= 0.f && c->mu < 1.f)) return fail(LLATTN_ERR_SHAPE, "llattn_muon_update: momentum %g outside [0, 1)", c->mu);
  return run("llattn_muon_update", c, g, m, w, m_out, w_out, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}
