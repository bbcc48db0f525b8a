// Newton-Schulz orthogonalisation and the weight update made of it (include/llattn_train.h).
//
//   X = U / (|U|_F + eps)  (m x n, m <= n)
//   A = X Xᵀ,  B = b A + c A A,  X <- a X + B X        (steps times)
//
// Precision.  A step multiplies small singular values by a = 3.4445, five steps by 485, and with them whatever the
// roundings of X, A and B leave there: bf16 matrices (half a step of 2^-8) leave order-1 errors in directions that a
// gradient hardly has, fp32 ones nothing.  Matrices are held as hi + lo, two fp16 halves (22 bits), and a product as
// hi hi + hi lo + lo hi on the fp16 matrix cores with fp32 accumulation: what is left out, lo lo, is 2^-22 of it.
// Against float64 that is as exact as fp32 products are from 64 rows on (64 x 64 to 1408 x 1408, flat, decaying and low-rank
// spectra: within 2% of fp32's own error, below it from 100 on; two bf16 halves: 10 to 20 times that) and 1.2 times
// as far off down to 17 rows (fewer: ns_thin_kernel), at a third of the 16-bit rate, five times the
// fp32 one.  Scales are powers of two: X is held times S_X ~ sqrt(m n) (its entries average 1 / sqrt(m n)), A and B times
// 2^12 (their entries are at most a few).
//
// Storage: a row holds, for each block of 32 columns, its 32 hi and then its 32 lo halves: 128 bytes, one cache line.
// A k step of 32 is then laid out like a 64-k step of the bf16 products, and their loads and fragment reads serve.
// Rows and columns are padded to multiples of 64 with zeros, which the iteration keeps; rows of a tile past them are past
// the operand's extent and read zero.
//
// A and B are symmetric: blocks on and above the diagonal are computed and written to both sides.
//
// Matrices of several shapes share a launch: workgroups find their group, matrix and tile.
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

// 16-bit elements of a row of n columns.
__host__ __device__ constexpr int64_t row_elems(int n) { return 2 * (int64_t)n; }

// ---- momentum and |U|^2 -----------------------------------------------------------
// A group's share of a launch over elements: workgroups [b0, b0 + batch blocks), `blocks` a matrix.
struct ElemGroup {
  int b0, blocks, first, rows, cols, flip, g_dtype, mp, np;
  float scale;
  int64_t x_off;   // of the group's first X
  int part0;       // of its first partial sum
  int parts;       // partial sums a matrix
};
struct ElemArgs {
  Table<const void*> g;
  Table<const float*> m;
  int n_groups, momentum, nesterov;
  float mu, one_mu, eps;
  double* part;
  uint16_t* x;
  ElemGroup grp[LLATTN_MUON_GROUPS];
};
struct PrepArgs {
  ElemArgs e;
  Table<float*> m_out;
};

static_assert(sizeof(PrepArgs) <= 4096, "kernel arguments");

template <typename G>
__device__ __forceinline__ const G& group_of(const G* g, int n, int block) {
  int i = 0;
  while (i + 1 < n && block >= g[i + 1].b0) ++i;
  return g[i];
}

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

__device__ __forceinline__ bool by4(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == LLATTN_F32 ? 15u : 7u)) == 0; }
__device__ __forceinline__ void load4_as(const void* p, int64_t i, int dtype, float v[4]) {
  if (dtype == LLATTN_F32) load4<float>(static_cast<const float*>(p) + i, v);
  else load4<uint16_t>(static_cast<const uint16_t*>(p) + i, v);
}

// m_out = mu m + (1 - mu) g and the workgroup's share of |U|^2, in 64 bits (any fp32 values, squares included).  Bandwidth:
// 22 x 4096 x 1408, fp32: 1.5 GB in 300 us, 5.1 TB/s.
__global__ __launch_bounds__(256) void muon_prep_kernel(const PrepArgs pa) {
  __shared__ double s[256];
  const ElemArgs& a = pa.e;
  const ElemGroup& G = group_of(a.grp, a.n_groups, blockIdx.x);
  const int at = blockIdx.x - G.b0, mat = at / G.blocks, blk = at % G.blocks, id = G.first + mat;
  const void* g = a.g.p[id];
  const float* m = a.m.p[id];
  float* mo = pa.m_out.p[id];
  const int64_t n = (int64_t)G.rows * G.cols, quads = n / 4;
  const bool vec = by4(g, G.g_dtype) && (!a.momentum || (by4(m, LLATTN_F32) && by4(mo, LLATTN_F32)));
  const int64_t q_end = vec ? quads : 0, stride = (int64_t)G.blocks * 256;
  double sum = 0.0;
  for (int64_t q = (int64_t)blk * 256 + threadIdx.x; q < q_end; q += stride) {
    float u[4];
    load4_as(g, 4 * q, G.g_dtype, u);
    if (a.momentum) {
      float v[4];
      load4<float>(m + 4 * q, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = fmaf(a.mu, v[e], a.one_mu * u[e]);
        u[e] = direction(u[e], v[e], a.mu, a.one_mu, a.nesterov);
      }
      store4<float>(mo + 4 * q, v);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum += (double)u[e] * (double)u[e];
  }
  for (int64_t i = 4 * q_end + (int64_t)blk * 256 + threadIdx.x; i < n; i += stride) {
    float u = load_as(g, i, G.g_dtype);
    if (a.momentum) {
      const float v = fmaf(a.mu, m[i], a.one_mu * u);
      mo[i] = v;
      u = direction(u, v, a.mu, a.one_mu, a.nesterov);
    }
    sum += (double)u * (double)u;
  }
  sum = block_sum(sum, s);
  if (threadIdx.x == 0) a.part[G.part0 + mat * G.parts + blk] = sum;
}

// ---- X = U / (|U| + eps) as halves, transposed if rows > cols -----------------------
__device__ __forceinline__ uint16_t h_bits(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }
__device__ __forceinline__ float h_val(uint16_t v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }

// position of column c within a row
__device__ __forceinline__ int hi_at(int c) { return (c >> 5) * 64 + (c & 31); }

// two values' hi and lo halves
__device__ __forceinline__ void halves2(float v0, float v1, uint32_t& h, uint32_t& l) {
  const uint16_t h0 = h_bits(v0), h1 = h_bits(v1);
  h = h0 | (uint32_t)h1 << 16;
  l = h_bits(v0 - h_val(h0)) | (uint32_t)h_bits(v1 - h_val(h1)) << 16;
}
__device__ __forceinline__ void store_halves4(uint16_t* row, int c, const float v[4]) {
  uint2 h, l;
  halves2(v[0], v[1], h.x, l.x);
  halves2(v[2], v[3], h.y, l.y);
  uint16_t* p = row + hi_at(c);
  *reinterpret_cast<uint2*>(p) = h;
  *reinterpret_cast<uint2*>(p + 32) = l;
}
__device__ __forceinline__ void store_halves8(uint16_t* row, int c, const float v[8]) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) halves2(v[2 * e], v[2 * e + 1], h[e], l[e]);
  uint16_t* p = row + hi_at(c);
  st16(p, make_uint4(h[0], h[1], h[2], h[3]));
  st16(p + 32, make_uint4(l[0], l[1], l[2], l[3]));
}
// One 64 x 64 tile of X per workgroup, through LDS (the reads run along U's rows either way).  a.m: the new momentum.
// Bandwidth: 22 x 4096 x 1408, fp32: 1.5 GB in 298 us, 5.1 TB/s.
__global__ __launch_bounds__(256) void muon_split_kernel(const ElemArgs a) {
  __shared__ double s[256];
  __shared__ float tile[64][65];
  const ElemGroup& G = group_of(a.grp, a.n_groups, blockIdx.x);
  const int at = blockIdx.x - G.b0, mat = at / G.blocks, blk = at % G.blocks, id = G.first + mat;
  const int tn = G.np / 64, r0 = blk / tn * 64, c0 = blk % tn * 64;
  double sum = 0.0;
  for (int i = threadIdx.x; i < G.parts; i += 256) sum += a.part[G.part0 + mat * G.parts + i];
  const double f = (double)G.scale / (sqrt(block_sum(sum, s)) + (double)a.eps);
  const void* g = a.g.p[id];
  const float* m = a.m.p[id];
  const int u0 = G.flip ? c0 : r0, v0 = G.flip ? r0 : c0;  // the tile's origin in U
  const bool vec = G.cols % 4 == 0 && by4(g, G.g_dtype) && (!a.momentum || by4(m, LLATTN_F32));
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int q = threadIdx.x + 256 * k, lr = q >> 4, lc = (q & 15) * 4, r = u0 + lr, c = v0 + lc;
    float u[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
    const int64_t i = (int64_t)r * G.cols + c;
    if (r < G.rows && vec) {
      if (c < G.cols) {
        load4_as(g, i, G.g_dtype, u);
        if (a.momentum) load4<float>(m + i, v);
      }
    } else if (r < G.rows) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c + e >= G.cols) continue;
        u[e] = load_as(g, i + e, G.g_dtype);
        if (a.momentum) v[e] = m[i + e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (a.momentum) u[e] = direction(u[e], v[e], a.mu, a.one_mu, a.nesterov);
      tile[lr][lc + e] = r < G.rows && c + e < G.cols ? (float)((double)u[e] * f) : 0.f;  // eps 0: f may be infinite
    }
  }
  __syncthreads();
  const int64_t ld = row_elems(G.np);
  uint16_t* x = a.x + G.x_off + mat * G.mp * ld;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int q = threadIdx.x + 256 * k, lr = q >> 4, lc = (q & 15) * 4;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = G.flip ? tile[lc + e][lr] : tile[lr][lc + e];
    store_halves4(x + (r0 + lr) * ld, c0 + lc, v);
  }
}

// ---- the products -------------------------------------------------------------------
enum NsMode { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3 };

// A group's share of a launch over tiles: workgroups [b0, b0 + count), then padding to a multiple of 8 (the XCDs).
struct TileGroup {
  int b0, count, tiles, tiles_n;  // tiles a matrix, tile columns
  int steps;                      // of 32 k
  int mp, np, first, rows, cols, w_dtype;
  int64_t x_off, a_off;           // of the group's first X and A
  float alpha, beta;              // C = alpha D + beta (products), in stored scales
  float keep, step;               // LAST
};
struct NsArgs {
  const uint16_t* x;   // X
  uint16_t* y;         // the next X (APPLY)
  uint16_t *a, *b;     // A, B
  int n_groups, update;
  TileGroup grp[LLATTN_MUON_GROUPS];
};
struct LastArgs {
  NsArgs n;
  Table<const void*> w;
  Table<void*> out;
};

static_assert(sizeof(LastArgs) <= 4096, "kernel arguments");

// T rows of a step with k along them (128 bytes each: 32 hi, 32 lo), loaded by W waves.  Chunk c of row o at c ^ (o & 7).
template <int T, int W>
struct RowOp {
  static constexpr int BYTES = T * 128, LOADS = BYTES / 1024 / W;
  uint32_t off[LOADS], base[2];  // base: of this lane's fragments, hi and lo
  __device__ __forceinline__ void init(int64_t ld, int w, int lane, int o0) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = 8 * (w * LOADS + i) + (lane >> 3);
      off[i] = (uint32_t)((int64_t)row * ld * 2 + 16 * ((lane & 7) ^ (row & 7)));
    }
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) base[h] = (o0 + r) * 128 + (((4 * h + g) ^ (r & 7)) << 4);
  }
  // rows o0 + 16 i + r, k 8 g .. 8 g + 7 of the stage at st
  __device__ __forceinline__ f16x8 frag(const unsigned char* st, int i, int half) const {
    return *reinterpret_cast<const f16x8*>(st + base[half] + i * 2048);
  }
};

// 32 rows of a step, T columns of them (4 T bytes each).  Chunk c of k-row k at c ^ 2 (k & 3).
template <int T, int W>
struct ColOp {
  static constexpr int BYTES = T * 128, LOADS = BYTES / 1024 / W, PER = T / 4;
  uint32_t off[LOADS], base[4];  // base: by half and the parity of the 16-column block
  __device__ __forceinline__ void init(int64_t ld, int w, int lane, int o0) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int q = (w * LOADS + i) * 64 + lane, k = q / PER, c = (q % PER) ^ (2 * (k & 3));
      off[i] = (uint32_t)((int64_t)k * ld * 2 + 16 * c);
    }
    // transposing reads: the 16 lanes of group g supply k-rows 8 g + r / 4 (and 4 further), 8 bytes at column 4 (r % 4)
    const int r = lane & 15, g = lane >> 4, k = 8 * g + (r >> 2);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int byte = (o0 >> 5) * 128 + (u >> 1) * 64 + (u & 1) * 32 + 8 * (r & 3);
      base[u] = k * (4 * T) + (((byte >> 4) ^ (2 * (k & 3))) << 4) + (byte & 15);
    }
  }
  // columns o0 + 16 j + r (o0 a multiple of 32), k 8 g .. 8 g + 7
  __device__ __forceinline__ f16x8 frag(const unsigned char* st, int j, int half) const {
    const unsigned char* p = st + base[2 * half + (j & 1)] + (j >> 1) * 128;
    bf16x4 hv[2];
#pragma unroll
    for (int q = 0; q < 2; ++q)
      hv[q] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(p + q * 16 * T));
    return __builtin_bit_cast(f16x8, bf16x8{hv[0][0], hv[0][1], hv[0][2], hv[0][3], hv[1][0], hv[1][1], hv[1][2], hv[1][3]});
  }
};

// 4 x 4 transpose within each group of four lanes: lane l gives v[e] and receives lane e's v[l].
__device__ __forceinline__ float quad_swap1(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xB1, 0xf, 0xf, true));
}
__device__ __forceinline__ float quad_swap2(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x4E, 0xf, 0xf, true));
}
__device__ __forceinline__ void quad_transpose(float v[4], int lane) {
  const bool b0 = lane & 1, b1 = lane & 2;
#pragma unroll
  for (int e = 0; e < 4; e += 2) {
    const float t = quad_swap1(b0 ? v[e] : v[e + 1]);
    if (b0) v[e] = t;
    else v[e + 1] = t;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float t = quad_swap2(b1 ? v[e] : v[e + 2]);
    if (b1) v[e] = t;
    else v[e + 2] = t;
  }
}

// Lanes r and r ^ 4 of each eight: those with bit 2 set give x and receive y, the others give y and receive x.
__device__ __forceinline__ void swap4(uint32_t& x, uint32_t& y, int lane) {
  const bool odd = lane & 4;
  const int t = __builtin_amdgcn_update_dpp(0, (int)(odd ? x : y), 0x141, 0xf, 0xf, true);        // lane 7 - r of the eight
  const uint32_t u = (uint32_t)__builtin_amdgcn_update_dpp(0, t, 0x1B, 0xf, 0xf, true);           // and 3 - r of the four
  if (odd) x = u;
  else y = u;
}

// A shape of workgroup: KG groups of WR x WC waves, each wave 16 MB x 16 NB of the tile, NST LDS stages of 32 k a group.
template <int MB_, int NB_, int WR_, int WC_, int KG_, int NST_>
struct Shape {
  static constexpr int MB = MB_, NB = NB_, WR = WR_, WC = WC_, KG = KG_, NST = NST_;
  static constexpr int W = WR * WC, THREADS = 64 * W * KG, TM = 16 * MB * WR, TN = 16 * NB * WC, STAGE = (TM + TN) * 128;
};

// One tile.  A step is three rounds of products, each beside the fragment reads of the next: lo hi (reads A hi), hi hi
// (reads B lo), then a barrier, hi lo (reads B hi and A lo of the next step, and issues the loads of step kt + NST into
// the stage just read).  One set of fragment registers serves, and no round waits for reads of its own.  Waves whose
// part of the tile is not stored load and wait like the others but read and multiply nothing.  Each of the KG groups
// takes a share of the steps; their sums are added through LDS in order.
//
// Measured, 22 matrices 1408 x 4096: X Xᵀ 468 us (1140 TFLOP/s of fp16 products), the polynomial 205 us (900), B X 902 us
// (1190), its last 956 us, 1105 with the weights read.  Matrix cores 59-61% busy at a clock of 1.9 GHz that the products
// themselves bring down; a step of 256 x 256 alone stands at 1500 TFLOP/s, the rest goes into tiles' ends and part rounds.
template <int MODE, typename S>
__device__ __forceinline__ void ns_tile(const NsArgs& a, const Table<const void*>* wt, const Table<void*>* ot,
                                        unsigned char* smem) {
  constexpr bool SYM = MODE == GRAM || MODE == POLY;
  constexpr int MB = S::MB, NB = S::NB, TM = S::TM, TN = S::TN, NST = S::NST, KG = S::KG, W = S::W, STAGE = S::STAGE;
  typedef RowOp<TM, W> OpA;
  typedef std::conditional_t<SYM, RowOp<TN, W>, ColOp<TN, W>> OpB;
  constexpr int LOADS = OpA::LOADS + OpB::LOADS;
  static_assert(LOADS <= MB + NB, "the third round's reads carry the loads");
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kg = wave / W, w = wave % W;
  // eight waves: those of one SIMD (w, w + 4) lie in opposite halves of both sides, so that a tile half outside the
  // matrix takes half the time
  static_assert(S::WC == 2 && (S::WR == 2 || S::WR == 4), "wave layouts");
  const int wm = W == 8 ? (w & 3) ^ (w >> 2 << 1) : w >> 1, wn = W == 8 ? (w & 1) ^ (w >> 2) : w & 1;
  const TileGroup& G = group_of(a.grp, a.n_groups, blockIdx.x);
  if ((int)blockIdx.x - G.b0 >= G.count) return;
  const int v = xcd_remap(blockIdx.x - G.b0, G.count), mat = v / G.tiles;
  int t = v % G.tiles, tm = 0, tn;
  if constexpr (SYM) {  // tile rows from the diagonal on
    int skip = 0;
    while (t >= G.tiles_n - skip) {
      t -= G.tiles_n - skip;
      ++tm;
      skip = tm * TM / TN;
    }
    tn = skip + t;
  } else {  // groups of 8 tile rows
    const int tiles_m = G.tiles / G.tiles_n, group = t / (8 * G.tiles_n), gm = min(tiles_m - group * 8, 8);
    tm = group * 8 + t % (8 * G.tiles_n) % gm;
    tn = t % (8 * G.tiles_n) / gm;
  }
  const int m0 = __builtin_amdgcn_readfirstlane(tm * TM), n0 = __builtin_amdgcn_readfirstlane(tn * TN);
  const int64_t lx = row_elems(G.np), la = row_elems(G.mp);
  const uint16_t* X = a.x + G.x_off + mat * G.mp * lx;
  uint16_t* Am = a.a + G.a_off + mat * G.mp * la;
  uint16_t* Bm = a.b + G.a_off + mat * G.mp * la;
  // operands: rows of the tile with k along them; SYM: the same for its columns, else X with k along its rows
  const uint16_t* opa = MODE == GRAM ? X : MODE == POLY ? Am : Bm;
  const uint16_t* opb = SYM ? opa : X;
  const int64_t lda = MODE == GRAM ? lx : la, ldb = SYM ? lda : lx;
  // first row and column of this wave's part
  const int row0 = m0 + wm * 16 * MB, col0 = n0 + wn * 16 * NB, lim = SYM ? G.mp : G.np;
  const int per = (G.steps + KG - 1) / KG;  // steps of a group: this one's are [kg per, kg per + own)
  const int own = row0 < G.mp && col0 < lim && !(SYM && col0 + 16 * NB <= row0) ? min(max(G.steps - kg * per, 0), per) : 0;
  OpA oa;
  OpB ob;
  oa.init(lda, w, lane, wm * 16 * MB);
  ob.init(ldb, w, lane, wn * 16 * NB);
  // Rows of a ragged tile and steps past the last read zero.  Columns past the end of a k-major row read the next row's:
  // products that are never stored.
  const int first = kg * per;
  int left = G.steps - first;  // steps from the next one to load on
  StepSrc sa, sb;
  sa.addr = reinterpret_cast<uint64_t>(opa + m0 * lda + (int64_t)first * 64);
  sa.full = extent_of(min(TM, G.mp - m0), lda, 64);
  sa.inc = 128;
  if constexpr (SYM) {
    sb.addr = reinterpret_cast<uint64_t>(opb + n0 * ldb + (int64_t)first * 64);
    sb.full = extent_of(min(TN, G.mp - n0), ldb, 64);
    sb.inc = 128;
  } else {
    sb.addr = reinterpret_cast<uint64_t>(opb + (int64_t)n0 * 2 + first * 32 * ldb);
    sb.full = extent_of(32, ldb, 2 * min(TN, G.np - n0));
    sb.inc = (uint32_t)(64 * ldb);
  }
  sa.tail = sb.tail = 0;
  i32x4 ra = sa.rsrc(left, 1), rb = sb.rsrc(left, 1);
  auto next_step = [&]() {
    sa.addr += sa.inc;
    sb.addr += sb.inc;
    left -= 1;
    ra = sa.rsrc(left, 1);
    rb = sb.rsrc(left, 1);
  };
  unsigned char* sm = smem + kg * NST * STAGE;
  const uint32_t lds_a = __builtin_amdgcn_readfirstlane(lds_addr(sm) + w * OpA::LOADS * 1024);
  const uint32_t lds_b = __builtin_amdgcn_readfirstlane(lds_addr(sm) + OpA::BYTES + w * OpB::LOADS * 1024);
  auto load = [&](auto stage, auto q) {
    constexpr int s = decltype(stage)::value, n = decltype(q)::value;
    if constexpr (n < OpA::LOADS) dma_at<s * STAGE + n * 1024>(ra, oa.off[n], lds_a);
    else dma_at<s * STAGE + (n - OpA::LOADS) * 1024>(rb, ob.off[n - OpA::LOADS], lds_b);
  };
  f16x8 ah[MB], al[MB], bh[NB], bl[NB];
  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // MB NB products, B first: lane (r, g) accumulates C[r][4 g + e]; io(q) for q < N spread over them
  auto round = [&](const f16x8 (&x)[MB], const f16x8 (&y)[NB], auto n_tag, auto io) {
    constexpr int N = decltype(n_tag)::value, P = MB * NB;
    unroll<N>([&](auto qt) {
      constexpr int q = decltype(qt)::value;
      io(qt);
#pragma unroll
      for (int n = q * P / N; n < (q + 1) * P / N; ++n)
        acc[n / NB][n % NB] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y[n % NB], x[n / NB], acc[n / NB][n % NB], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  unroll<NST>([&](auto st) {
    if constexpr (decltype(st)::value > 0) next_step();
    unroll<LOADS>([&](auto q) { load(st, q); });
  });
  __builtin_amdgcn_s_waitcnt(wait_vm((NST - 1) * LOADS));  // loads complete in issue order: step 0 has landed
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (own > 0) {
#pragma unroll
    for (int j = 0; j < NB; ++j) bh[j] = ob.frag(sm + OpA::BYTES, j, 0);
#pragma unroll
    for (int i = 0; i < MB; ++i) al[i] = oa.frag(sm, i, 1);
  }
  // a step in stage ST; LIVE: this wave multiplies in it
  auto step = [&](auto st, auto live_tag) {
    constexpr int ST = decltype(st)::value, NEXT = (ST + 1) % NST;
    constexpr bool LIVE = decltype(live_tag)::value;
    const unsigned char* cur = sm + ST * STAGE;
    const unsigned char* nxt = sm + NEXT * STAGE;
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (LIVE) {
      round(al, bh, std::integral_constant<int, MB>{}, [&](auto q) { ah[q] = oa.frag(cur, q, 0); });
      round(ah, bh, std::integral_constant<int, NB>{}, [&](auto q) {
        bl[q] = ob.frag(cur + OpA::BYTES, q, 1);
        if constexpr (decltype(q)::value == 0) next_step();
      });
    } else {
      next_step();
    }
    // this wave's loads of step kt + 1 have landed and its fragments of step kt are read; then every wave's
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0((NST - 2) * LOADS));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (LIVE) {
      round(ah, bl, std::integral_constant<int, MB + NB>{}, [&](auto qt) {
        constexpr int q = decltype(qt)::value;
        if constexpr (q < NB) bh[q] = ob.frag(nxt + OpA::BYTES, q, 0);
        else al[q - NB] = oa.frag(nxt, q - NB, 1);
        if constexpr (q < LOADS) load(st, qt);
      });
    } else {
      unroll<LOADS>([&](auto q) { load(st, q); });
    }
  };
  // a wave multiplies in all of the group's steps, in none, or (in the last k group) in all but the last ones
  auto steps = [&](auto live_tag) {
    int kt = 0;
    while (kt < per) {
      unroll<NST>([&](auto st) {
        if (kt < per) step(st, live_tag);
        ++kt;
      });
    }
  };
  if (own == 0) {
    steps(std::false_type{});
  } else if (KG == 1 || own == per) {
    steps(std::true_type{});
  } else {
    int kt = 0;
    while (kt < per) {
      unroll<NST>([&](auto st) {
        if (kt < own) step(st, std::true_type{});
        else if (kt < per) step(st, std::false_type{});
        ++kt;
      });
    }
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // no DMA may land after the workgroup exits

  const void* w_ptr = nullptr;
  void* out = nullptr;
  bool vec = false, flip = false;
  if constexpr (MODE == LAST) {
    w_ptr = wt->p[G.first + mat];
    out = ot->p[G.first + mat];
    flip = G.rows > G.cols;
    vec = G.cols % 4 == 0 && by4(out, G.w_dtype) && (!a.update || by4(w_ptr, G.w_dtype));
  }
  // The epilogue takes two neighbouring blocks at a time and swaps halves between their lanes, so that a lane holds 8
  // consecutive columns of one of them (g even: the left, g odd: the right) and moves 16 bytes at a time.
  // What it reads, D and the weight that LAST updates (as it is stored), is loaded DEPTH pairs ahead of the stores: taken
  // one by one behind them, each cost its latency (22 x 1408 x 1408, POLY: 34 of 139 us a tile).
  constexpr int PAIRS = MB * NB / 2, DEPTH = KG > 1 ? 1 : PAIRS < 4 ? PAIRS : 4;
  struct Extra { uint4 h, l, w[2]; };
  struct Spot { int rb, cb, row, col; };  // the lane's block, and its row and first column
  // Pairs run down two rows of blocks before the next columns, where one group of waves has both.
  auto block_row = [](int p) { return KG > 1 ? p / (NB / 2) : 2 * (p / NB) + (p & 1); };
  auto block_col = [](int p) { return 2 * (KG > 1 ? p % (NB / 2) : (p / 2) % (NB / 2)); };
  auto spot = [&](int p) {
    const int rb = row0 + 16 * block_row(p), cb = col0 + 16 * block_col(p) + 16 * (g & 1);
    return Spot{rb, cb, rb + r, cb + 4 * (g & 2)};
  };
  auto outside = [&](const Spot& s) { return s.rb >= G.mp || s.cb >= lim || (SYM && s.cb < s.rb); };
  auto at = [&](const Spot& s, int q, int& orow, int& ocol) {  // of LAST's output: first of this lane's q-th four columns
    orow = flip ? s.col + 4 * q + (r & 3) : s.row;
    ocol = flip ? s.rb + (r & 12) : s.col + 4 * q;
  };
  auto fetch = [&](int p, Extra& x) {
    const Spot s = spot(p);
    if (MODE == GRAM || outside(s)) return;
    const uint16_t* d = (MODE == POLY ? Am + s.row * la : X + s.row * lx) + hi_at(s.col);
    x.h = *reinterpret_cast<const uint4*>(d);
    x.l = *reinterpret_cast<const uint4*>(d + 32);
    if constexpr (MODE == LAST) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        int orow, ocol;
        at(s, q, orow, ocol);
        if (!a.update || !vec || orow >= G.rows || ocol >= G.cols) continue;
        const int64_t o = (int64_t)orow * G.cols + ocol;
        if (G.w_dtype == LLATTN_F32) {
          x.w[q] = *reinterpret_cast<const uint4*>(static_cast<const float*>(w_ptr) + o);
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(w_ptr) + o);
          x.w[q].x = v.x;
          x.w[q].y = v.y;
        }
      }
    }
  };
  uint2 below_h[2][2], below_l[2][2];  // two rows of blocks' halves for below the diagonal
  // pair p, its sums in left and right; then(): once x is read
  auto finish = [&](int p, const f32x4& left, const f32x4& right, const Extra& xt, auto then) {
    const Spot s = spot(p);
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const auto v = __builtin_amdgcn_permlane16_swap(__float_as_uint(left[e]), __float_as_uint(right[e]), false, false);
      x[e] = G.beta * __uint_as_float(v[0]);
      x[4 + e] = G.beta * __uint_as_float(v[1]);
    }
    if constexpr (MODE != GRAM) {
      const f16x8 h = __builtin_bit_cast(f16x8, xt.h), l = __builtin_bit_cast(f16x8, xt.l);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fmaf(G.alpha, (float)h[e] + (float)l[e], x[e]);
    }
    const uint4 w0 = xt.w[0], w1 = xt.w[1];
    then();
    if (outside(s)) return;
    if constexpr (MODE == APPLY) {
      store_halves8(a.y + G.x_off + (mat * G.mp + s.row) * lx, s.col, x);
    } else if constexpr (SYM) {
      uint16_t* C = MODE == GRAM ? Am : Bm;
      store_halves8(C + s.row * la, s.col, x);
      if (s.cb <= s.rb) return;
      // and below the diagonal: this lane's columns col + 4 q + r % 4, rows 4 (r / 4) ..
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float* y = x + 4 * q;
        quad_transpose(y, lane);
        uint16_t* c = C + (s.col + 4 * q + (r & 3)) * la;
        if constexpr (KG > 1) {
          store_halves4(c, s.rb + (r & 12), y);
        } else {
          halves2(y[0], y[1], below_h[p & 1][q].x, below_l[p & 1][q].x);
          halves2(y[2], y[3], below_h[p & 1][q].y, below_l[p & 1][q].y);
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float* y = x + 4 * q;
        int orow, ocol;
        at(s, q, orow, ocol);
        if (flip) quad_transpose(y, lane);
        const int n = min(4, G.cols - ocol);
        if (orow >= G.rows || n <= 0) continue;
        const int64_t o = (int64_t)orow * G.cols + ocol;
        const bool f32 = G.w_dtype == LLATTN_F32;
        if (a.update) {
          uint4 u = q ? w1 : w0;
          if (!f32) u = make_uint4(u.x << 16, u.x & 0xffff0000u, u.y << 16, u.y & 0xffff0000u);
          float c4[4] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (!vec) c4[e] = e < n ? load_as(w_ptr, o + e, G.w_dtype) : 0.f;
            y[e] = fmaf(-G.step, y[e], G.keep * c4[e]);
          }
        }
        if (vec) {
          if (f32) store4<float>(static_cast<float*>(out) + o, y);
          else store4<uint16_t>(static_cast<uint16_t*>(out) + o, y);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (e >= n) continue;
            if (f32) static_cast<float*>(out)[o + e] = y[e];
            else static_cast<uint16_t*>(out)[o + e] = f2bf(y[e]);
          }
        }
      }
    }
  };
  Extra xt[DEPTH];
  if constexpr (KG == 1) {
#pragma unroll
    for (int p = 0; p < DEPTH; ++p) fetch(p, xt[p]);
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) {
      const int i = block_row(p), j = block_col(p);
      finish(p, acc[i][j], acc[i][j + 1], xt[p % DEPTH], [&]() {
        if (p + DEPTH < PAIRS) fetch(p + DEPTH, xt[p % DEPTH]);
      });
      if constexpr (SYM) {
        // Both blocks' halves for below the diagonal: lanes of r / 4 even take 8 rows of the upper one, the odd of the lower.
        const Spot s = spot(p - 1);
        if (p % 2 == 0 || outside(s) || s.cb <= s.rb) continue;
        uint16_t* C = MODE == GRAM ? Am : Bm;
        const int rb = s.rb + 4 * (r & 4);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint2 *h0 = &below_h[0][q], *h1 = &below_h[1][q], *l0 = &below_l[0][q], *l1 = &below_l[1][q];
          swap4(h0->x, h1->x, lane);
          swap4(h0->y, h1->y, lane);
          swap4(l0->x, l1->x, lane);
          swap4(l0->y, l1->y, lane);
          uint16_t* c = C + (s.col + 4 * q + (r & 3)) * la + hi_at(rb + (r & 8));
          if (s.cb <= rb) continue;
          st16(c, make_uint4(h0->x, h0->y, h1->x, h1->y));
          st16(c + 32, make_uint4(l0->x, l0->y, l1->x, l1->y));
        }
      }
    }
  } else {
    static_assert(KG * W * MB * NB * 1024 <= KG * NST * STAGE, "the groups' sums fit their stages");
    __builtin_amdgcn_s_barrier();  // every wave has read its fragments and its loads have landed
    asm volatile("" ::: "memory");
    f32x4* sum = reinterpret_cast<f32x4*>(smem);  // [KG][W][MB NB][64]
#pragma unroll
    for (int u = 0; u < MB * NB; ++u) sum[(wave * MB * NB + u) * 64 + lane] = acc[u / NB][u % NB];
    __syncthreads();
#pragma unroll
    for (int p = 0; p < PAIRS; ++p) {  // pairs are shared out among the groups
      if (p % KG != kg) continue;
      fetch(p, xt[0]);
      f32x4 c[2];
#pragma unroll
      for (int k = 0; k < KG; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const f32x4 v = sum[((k * W + w) * MB * NB + block_row(p) * NB + block_col(p) + u) * 64 + lane];
          c[u] = k ? c[u] + v : v;
        }
      finish(p, c[0], c[1], xt[0], []() {});
    }
  }
}

template <int MODE, typename S, int WGS>
__global__ __launch_bounds__(S::THREADS, WGS * S::W * S::KG / 4) void ns_kernel(const NsArgs a) {
  __shared__ __align__(1024) unsigned char smem[S::KG * S::NST * S::STAGE];
  ns_tile<MODE, S>(a, nullptr, nullptr, smem);
}
template <typename S, int WGS>
__global__ __launch_bounds__(S::THREADS, WGS * S::W * S::KG / 4) void ns_last_kernel(const LastArgs a) {
  __shared__ __align__(1024) unsigned char smem[S::KG * S::NST * S::STAGE];
  ns_tile<LAST, S>(a.n, &a.w, &a.out, smem);
}

// ---- small matrices: the whole call in one workgroup each ---------------------------------------------------------------
// Up to 64 rows of X (the smaller side) and kSmallCols columns: X, A and B stay in LDS, as blocks of 32 columns (64 rows
// of 128 bytes, chunk c of row o at c ^ (o & 7)).  The chain of 2 + 3 steps launches that it replaces waits for launches
// and for its own tail 15 times; here it is the latency of LDS reads and barriers of 15 dependent products, which grows
// with the columns and with launches one behind the other.  A call in us, here and by the chain's best tiles:
//   4 of 64 x 64: 24, 70   x 128: 40, 73   x 256: 70, 78   x 448: 115, 84     128 of 64 x 128: 82, 86   x 448: 234, 120
// so up to kSmallCols columns times launches.
constexpr int kSmall = 64;         // matrices a launch
constexpr int kSmallCols = 256;    // X: 64 KB of LDS beside 32 KB for A and B

struct SmallGroup {
  int first, rows, cols, np, g_dtype, w_dtype;
  float scale, keep, step;
};
struct SmallArgs {
  const void* g[kSmall];
  const float* m[kSmall];
  float* m_out[kSmall];
  const void* w[kSmall];
  void* out[kSmall];
  int n_groups, update, nesterov, steps;
  float mu, one_mu, eps, a, b, c;
  SmallGroup grp[LLATTN_MUON_GROUPS];
};
static_assert(sizeof(SmallArgs) <= 4096, "kernel arguments");

__device__ __forceinline__ int small_at(int row, int col) {  // byte of the hi half
  return (col >> 5) * 8192 + row * 128 + ((((col & 31) >> 3) ^ (row & 7)) << 4) + (col & 7) * 2;
}
__device__ __forceinline__ int lo_of(int byte) { return byte ^ 64; }  // its lo half: four chunks further

__global__ __launch_bounds__(256) void ns_small_kernel(const SmallArgs a) {
  extern __shared__ __align__(1024) unsigned char lds[];  // A, B, X
  __shared__ double red[256];
  unsigned char *As = lds, *Bs = lds + 16384, *Xs = lds + 32768;
  int gi = 0;
  while (gi + 1 < a.n_groups && (int)blockIdx.x >= a.grp[gi + 1].first) ++gi;
  const SmallGroup& G = a.grp[gi];
  const int id = blockIdx.x, tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), r0 = (wave >> 1) * 32, c0 = (wave & 1) * 32;
  const bool flip = G.rows > G.cols;
  const int n = G.rows * G.cols, blocks = G.np / 32;
  for (int i = tid; i < blocks * 512; i += 256) *reinterpret_cast<uint4*>(Xs + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
  const void* gp = a.g[id];
  double sum = 0.0;
  for (int i = tid; i < n; i += 256) {
    float u = load_as(gp, i, G.g_dtype);
    if (a.update) {
      const float v = fmaf(a.mu, a.m[id][i], a.one_mu * u);
      a.m_out[id][i] = v;
      u = direction(u, v, a.mu, a.one_mu, a.nesterov);
    }
    sum += (double)u * (double)u;
  }
  const double f = (double)G.scale / (sqrt(block_sum(sum, red)) + (double)a.eps);
  for (int i = tid; i < n; i += 256) {  // each thread reads back what it wrote itself
    float u = load_as(gp, i, G.g_dtype);
    if (a.update) u = direction(u, a.m_out[id][i], a.mu, a.one_mu, a.nesterov);
    u = (float)((double)u * f);
    const int ur = i / G.cols, uc = i - ur * G.cols;
    const int at = small_at(flip ? uc : ur, flip ? ur : uc);
    const uint16_t h = h_bits(u);
    *reinterpret_cast<uint16_t*>(Xs + at) = h;
    *reinterpret_cast<uint16_t*>(Xs + lo_of(at)) = h_bits(u - h_val(h));
  }
  __syncthreads();
  // fragment of rows o16 + r of block kb (half 0: hi, 1: lo), k along the block's columns
  auto row_frag = [&](const unsigned char* M, int kb, int o16, int half) {
    const int row = o16 + r;
    return *reinterpret_cast<const f16x8*>(M + kb * 8192 + row * 128 + (((4 * half + g) ^ (row & 7)) << 4));
  };
  // of columns o16 + r, k along X's rows k0 ..
  auto col_frag = [&](int k0, int o16, int half) {
    bf16x4 hv[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = k0 + 8 * g + 4 * q + (r >> 2), at = small_at(k, o16 + 4 * (r & 3));
      hv[q] = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(Xs + (half ? lo_of(at) : at)));
    }
    return __builtin_bit_cast(f16x8, bf16x8{hv[0][0], hv[0][1], hv[0][2], hv[0][3], hv[1][0], hv[1][1], hv[1][2], hv[1][3]});
  };
  f32x4 acc[2][2];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  auto products = [&](const f16x8 (&x)[2][2], const f16x8 (&y)[2][2]) {  // [half][block]
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(y[p == 1][j], x[p == 2][i], acc[i][j], 0, 0, 0);
  };
  auto get4 = [&](const unsigned char* M, int row, int col, float (&v)[4]) {
    const int at = small_at(row, col);
    const f16x4 h = *reinterpret_cast<const f16x4*>(M + at), l = *reinterpret_cast<const f16x4*>(M + lo_of(at));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)h[e] + (float)l[e];
  };
  auto put4 = [&](unsigned char* M, int row, int col, const float (&v)[4]) {
    const int at = small_at(row, col);
    f16x4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      h[e] = (_Float16)v[e];
      l[e] = (_Float16)(v[e] - (float)h[e]);
    }
    *reinterpret_cast<f16x4*>(M + at) = h;
    *reinterpret_cast<f16x4*>(M + lo_of(at)) = l;
  };
  const float ga = kSA / (G.scale * G.scale), pb = a.c / kSA;
  for (int step = 0; step < a.steps; ++step) {
    const bool last = step + 1 == a.steps;
    clear();
    for (int kb = 0; kb < blocks; ++kb) {
      f16x8 x[2][2], y[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[h][i] = row_frag(Xs, kb, r0 + 16 * i, h);
          y[h][i] = row_frag(Xs, kb, c0 + 16 * i, h);
        }
      products(x, y);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float v[4] = {ga * acc[i][j][0], ga * acc[i][j][1], ga * acc[i][j][2], ga * acc[i][j][3]};
        put4(As, r0 + 16 * i + r, c0 + 16 * j + 4 * g, v);
      }
    __syncthreads();
    clear();
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f16x8 x[2][2], y[2][2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[h][i] = row_frag(As, kb, r0 + 16 * i, h);
          y[h][i] = row_frag(As, kb, c0 + 16 * i, h);
        }
      products(x, y);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int row = r0 + 16 * i + r, col = c0 + 16 * j + 4 * g;
        float v[4];
        get4(As, row, col, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = fmaf(a.b, v[e], pb * acc[i][j][e]);
        put4(Bs, row, col, v);
      }
    __syncthreads();
    f16x8 bf[2][2][2];  // [k block][half][row block] of B
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) bf[kb][h][i] = row_frag(Bs, kb, r0 + 16 * i, h);
    for (int cb = 0; cb < G.np; cb += 64) {
      clear();
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        f16x8 y[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 2; ++j) y[h][j] = col_frag(32 * kb, cb + c0 + 16 * j, h);
        products(bf[kb], y);
      }
      float v[2][2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          get4(Xs, r0 + 16 * i + r, cb + c0 + 16 * j + 4 * g, v[i][j]);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][j][e] = fmaf(a.a, v[i][j][e], acc[i][j][e] / kSA);
        }
      if (!last) __syncthreads();  // every wave has read these columns
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = r0 + 16 * i + r, col = cb + c0 + 16 * j + 4 * g;
          if (!last) {
            put4(Xs, row, col, v[i][j]);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int ur = flip ? col + e : row, uc = flip ? row : col + e;
            if (ur >= G.rows || uc >= G.cols) continue;
            const int o = ur * G.cols + uc;
            float y = v[i][j][e] / G.scale;
            if (a.update) y = fmaf(-G.step, y, G.keep * load_as(a.w[id], o, G.w_dtype));
            if (G.w_dtype == LLATTN_F32) static_cast<float*>(a.out[id])[o] = y;
            else static_cast<uint16_t*>(a.out[id])[o] = f2bf(y);
          }
        }
    }
    __syncthreads();
  }
}

// ---- thin matrices: the iteration on the smaller side's Gram matrix, in 64 bits -----------------------------------------
// Up to kThin rows of X (the smaller side), any number of columns.  Sums over so few rows are short, and what fp32 products
// round is then less than what the halves do: 82 x 1 was off by 2.3e-6 and fp32 by 3.3e-7, sides of 1 to 10 by 1.5 to 3
// times fp32's; from 17 to 32 by 1.2 times (500 matrices: 1.6 at most), from 33 on 1.1.  X after the steps is Q X0 with
//   A = X0 X0ᵀ,  P = a + b A + c A A,  Q <- P Q,  A <- P A P        (steps times)
// so X is read twice and written once, and all else is a 16 x 16 matrix: with fp64 products what is left is one rounding.
// One workgroup a matrix, 16 waves: bound by the latency of their loads.  Against the products on halves, a call: 16 x 448 at
// most 20 us (the host's) and 72, 16 x 4096 58 and 164, 16 x 32768 409 and 799, 128 of 16 x 4096 128 and 557.
constexpr int kThin = 16;
typedef double f64x4 __attribute__((ext_vector_type(4)));

__global__ __launch_bounds__(1024) void ns_thin_kernel(const SmallArgs a) {
  __shared__ double part[16][256];
  __shared__ double A[16][17], P[16][17], Q[16][17], T[16][17];
  int gi = 0;
  while (gi + 1 < a.n_groups && (int)blockIdx.x >= a.grp[gi + 1].first) ++gi;
  const SmallGroup& G = a.grp[gi];
  const int id = blockIdx.x, tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4, wave = tid >> 6;
  const bool flip = G.rows > G.cols;
  const int m = flip ? G.cols : G.rows, n = flip ? G.rows : G.cols;
  const auto at = [&](int row, int col) { return flip ? col * m + row : row * n + col; };  // of X: at most 16 x 32768
  const void* gp = a.g[id];
  // A lane gives row r, columns k0 + 4 e + g: as both operands, X Xᵀ.  Each element is one lane's, which updates its momentum.
  f64x4 acc = {0.0, 0.0, 0.0, 0.0};
  for (int k0 = 16 * wave; k0 < n; k0 += 256) {
    double u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + 4 * e + g;
      float v = 0.f;
      if (r < m && k < n) {
        const int i = at(r, k);
        v = load_as(gp, i, G.g_dtype);
        if (a.update) {
          const float mo = fmaf(a.mu, a.m[id][i], a.one_mu * v);
          a.m_out[id][i] = mo;
          v = direction(v, mo, a.mu, a.one_mu, a.nesterov);
        }
      }
      u[e] = (double)v;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(u[e], u[e], acc, 0, 0, 0);
  }
#pragma unroll
  for (int v = 0; v < 4; ++v) part[wave][(4 * v + g) * 16 + r] = acc[v];  // lane (r, g): rows 4 v + g of column r
  __syncthreads();
  const int i = tid >> 4 & 15, j = tid & 15;
  const bool mine = tid < 256;
  if (mine) {
    double s = 0.0;
    for (int w = 0; w < 16; ++w) s += part[w][tid];
    T[i][j] = s;
  }
  __syncthreads();
  double f = 0.0;
  if (mine) {
    double s = 0.0;
    for (int d = 0; d < 16; ++d) s += T[d][d];  // |U|^2
    f = 1.0 / (sqrt(s) + (double)a.eps);
    A[i][j] = T[i][j] * f * f;
    Q[i][j] = i == j ? f : 0.0;
  }
  __syncthreads();
  const auto dot = [&](const double (&x)[16][17], const double (&y)[16][17]) {
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < 16; ++k) s = fma(x[i][k], y[k][j], s);
    return s;
  };
  for (int step = 0; step < a.steps; ++step) {
    if (mine) P[i][j] = fma((double)a.c, dot(A, A), (double)a.b * A[i][j]) + (i == j ? (double)a.a : 0.0);
    __syncthreads();
    double q = 0.0;
    if (mine) {
      q = dot(P, Q);
      T[i][j] = dot(P, A);
    }
    __syncthreads();
    if (mine) {
      Q[i][j] = q;
      A[i][j] = dot(T, P);
    }
    __syncthreads();
  }
  double qf[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) qf[s] = Q[r][4 * s + g];
  // 16 columns at a time, all read before any is written
  for (int c0 = 16 * wave; c0 < n; c0 += 256) {
    const int k = c0 + r;
    f64x4 y = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float v = 0.f;
      if (4 * s + g < m && k < n) {
        const int e = at(4 * s + g, k);
        v = load_as(gp, e, G.g_dtype);
        if (a.update) v = direction(v, a.m_out[id][e], a.mu, a.one_mu, a.nesterov);
      }
      y = __builtin_amdgcn_mfma_f64_16x16x4f64(qf[s], (double)v, y, 0, 0, 0);
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      if (4 * v + g >= m || k >= n) continue;
      const int e = at(4 * v + g, k);
      float x = (float)y[v];
      if (a.update) x = fmaf(-G.step, x, G.keep * load_as(a.w[id], e, G.w_dtype));
      if (G.w_dtype == LLATTN_F32) static_cast<float*>(a.out[id])[e] = x;
      else static_cast<uint16_t*>(a.out[id])[e] = f2bf(x);
    }
  }
}

// ---- host -----------------------------------------------------------------------------
constexpr size_t up(size_t n) { return (n + 255) & ~size_t(255); }

// Workgroups of a launch.
enum Kind { SMALL = 0, SPLIT = 1, SQUARE = 2, BIG = 3, KINDS = 4 };
typedef Shape<2, 2, 2, 2, 1, 3> SmallShape;
typedef Shape<2, 2, 2, 2, 2, 3> SplitShape;
typedef Shape<4, 4, 2, 2, 1, 2> SquareShape;
typedef Shape<4, 8, 4, 2, 1, 2> BigShape;
constexpr int kTm[KINDS] = {SmallShape::TM, SplitShape::TM, SquareShape::TM, BigShape::TM};
constexpr int kTn[KINDS] = {SmallShape::TN, SplitShape::TN, SquareShape::TN, BigShape::TN};
constexpr int kPerCu[KINDS] = {3, 1, 2, 1};
// us of a 32-k step of a workgroup with 1, 2, 3 of them on a CU, and of a tile beside its steps.
constexpr double kStep[KINDS][3] = {{0.33, 0.50, 0.80}, {0.28, 0.28, 0.28}, {0.67, 1.37, 1.37}, {2.15, 2.15, 2.15}};
constexpr double kTile[KINDS] = {3.5, 4.0, 7.0, 16.0};

struct GroupPlan {
  int m, n, mp, np, parts, first, part0;
  size_t x_off, a_off;  // 16-bit elements
};
struct Plan {
  int matrices;
  GroupPlan g[LLATTN_MUON_GROUPS];
  size_t x, a, part;    // bytes of one X, of one A, of the partial sums
  size_t bytes() const { return 2 * x + 2 * a + part; }
};

Plan plan_of(const llattn_muon_cfg* c, const llattn_muon_group* groups) {
  Plan p{};
  size_t x = 0, a = 0, part = 0;
  for (int i = 0; i < c->n_groups; ++i) {
    const llattn_muon_group& q = groups[i];
    GroupPlan& g = p.g[i];
    g.m = std::min(q.rows, q.cols);
    g.n = std::max(q.rows, q.cols);
    g.mp = (g.m + 63) / 64 * 64;
    g.np = (g.n + 63) / 64 * 64;
    g.parts = (int)std::min<int64_t>(256, ((int64_t)g.m * g.n + 4095) / 4096);
    g.first = p.matrices;
    g.part0 = (int)part;
    g.x_off = x;
    g.a_off = a;
    p.matrices += q.batch;
    part += (size_t)q.batch * g.parts;
    x += (size_t)q.batch * g.mp * row_elems(g.np);
    a += (size_t)q.batch * g.mp * row_elems(g.mp);
  }
  p.x = up(2 * x);
  p.a = up(2 * a);
  p.part = up(8 * part);
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

int32_t check(const llattn_muon_cfg* c, const llattn_muon_group* groups) {
  if (!c || !groups) return fail(LLATTN_ERR_SHAPE, "llattn_muon: null configuration");
  if (c->n_groups < 1 || c->n_groups > LLATTN_MUON_GROUPS)
    return fail(LLATTN_ERR_SHAPE, "llattn_muon: %d groups (1 to %d)", c->n_groups, LLATTN_MUON_GROUPS);
  int64_t total = 0;
  for (int i = 0; i < c->n_groups; ++i) {
    const llattn_muon_group& q = groups[i];
    if (q.batch <= 0 || q.rows <= 0 || q.cols <= 0 || q.rows > 32768 || q.cols > 32768)
      return fail(LLATTN_ERR_SHAPE, "llattn_muon: group %d: %d matrices of %d x %d (1 to 32768)", i, q.batch, q.rows, q.cols);
    for (const int d : {q.g_dtype, q.w_dtype})
      if (d != LLATTN_F32 && d != LLATTN_BF16) return fail(LLATTN_ERR_DTYPE, "llattn_muon: unknown dtype %d", d);
    total += q.batch;
  }
  if (total > LLATTN_MUON_BATCH)
    return fail(LLATTN_ERR_SHAPE, "llattn_muon: %lld matrices (at most %d a call)", (long long)total, LLATTN_MUON_BATCH);
  if (c->tiles < 0 || c->tiles > KINDS) return fail(LLATTN_ERR_SHAPE, "llattn_muon: tiles %d (0 to 4)", c->tiles);
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

// Tiles of a matrix: all of an m x n one, or those of a symmetric one that reach the diagonal.
int tiles_of(bool sym, int kind, int m, int n) {
  const int tm = (m + kTm[kind] - 1) / kTm[kind], tn = (n + kTn[kind] - 1) / kTn[kind];
  if (!sym) return tm * tn;
  int t = 0;
  for (int i = 0; i < tm; ++i) t += tn - i * kTm[kind] / kTn[kind];
  return t;
}

struct Call {
  const llattn_muon_cfg* c;
  const llattn_muon_group* groups;
  Plan p;
  hipStream_t st;
  uint16_t *X[2], *A, *B;
  bool update;
  int kind[3];  // workgroups of GRAM, POLY, APPLY and LAST
};

template <int MODE, typename S, int WGS>
void launch_shape(const LastArgs& a, int blocks, hipStream_t st) {
  if constexpr (MODE == LAST) hipLaunchKernelGGL((ns_last_kernel<S, WGS>), dim3((unsigned)blocks), dim3(S::THREADS), 0, st, a);
  else hipLaunchKernelGGL((ns_kernel<MODE, S, WGS>), dim3((unsigned)blocks), dim3(S::THREADS), 0, st, a.n);
}
template <int MODE>
void launch_kind(int kind, const LastArgs& a, int blocks, hipStream_t st) {
  if (kind == SMALL) launch_shape<MODE, SmallShape, kPerCu[SMALL]>(a, blocks, st);
  else if (kind == SPLIT) launch_shape<MODE, SplitShape, kPerCu[SPLIT]>(a, blocks, st);
  else if (kind == SQUARE) launch_shape<MODE, SquareShape, kPerCu[SQUARE]>(a, blocks, st);
  else launch_shape<MODE, BigShape, kPerCu[BIG]>(a, blocks, st);
}

float scale_of(const GroupPlan& g) { return std::exp2f((float)std::min(14, (int)(0.5 * std::log2((double)g.m * g.n)))); }

// The workgroups that a launch takes: the least expected time.  A launch of one shape runs in rounds of whole tiles over
// the 256 CUs, the last with fewer workgroups on each; of several, its work is shared out and ends with a part of the
// longest tile.  Measured in us (G: X Xᵀ, P: A A, A: B X):
//                                   64 x 64        64 x 64, 2 k groups   128 x 128       256 x 256
//   3 of 333 x 1001     G P A     11   8  10         10   8  13          23  15  15      57  34  34
//   1 of 512 x 1408     G P A     14   9   9         12   9   9          33  17  17      78  44  41
//   1 of 1408 x 4096    G P A     37  17  60         32  15  70          76  36  55     191  86  85
//   6 of 1000 x 1500    G P A     47  35  73          -                  38  30  65      87  72  71
//   22 of 1408 x 1408   G P A    252 259 475          -                 204 209 343     188 201 365
//   22 of 1408 x 4096   G P A    833 257 1353         -                 495 218 934     479 215 897
//   8 of 4096 x 4096    G P A   3212 3217 3808        -                1393 1469 2636  1387 1391 2194
// What it takes is the best of its row but for G and P of the 22 matrices, where 128 x 128 is taken and 256 x 256 would be
// quicker (G 9% and 3%, P 4% and 1%): the epilogues became faster after the constants were fitted.
// (128 x 256 tiles on eight waves lay between the last two throughout.)
template <bool SYM>
int choose(const llattn_muon_cfg* c, const llattn_muon_group* groups, const Plan& p, bool gram) {
  if (c->tiles > 0) return c->tiles - 1;
  int best = SMALL;
  double best_t = 0.0;
  for (int kind = 0; kind < KINDS; ++kind) {
    const auto count = [&](int i) {
      return (int64_t)groups[i].batch * tiles_of(SYM, kind, p.g[i].mp, SYM ? p.g[i].mp : p.g[i].np);
    };
    const auto tile_us = [&](int i, int64_t on) { return (gram ? p.g[i].np : p.g[i].mp) / 32 * kStep[kind][on - 1] + kTile[kind]; };
    int64_t tiles = 0;
    for (int i = 0; i < c->n_groups; ++i) tiles += count(i);
    if (kind == SPLIT && tiles > 256) continue;
    const int64_t slots = 256 * kPerCu[kind], on = std::min<int64_t>(kPerCu[kind], (tiles + 255) / 256);
    double t;
    if (c->n_groups == 1) {
      const int64_t rest = tiles % slots;
      t = (double)(tiles / slots) * tile_us(0, kPerCu[kind]) + (rest ? tile_us(0, (rest + 255) / 256) : 0.0);
    } else {
      double work = 0.0, longest = 0.0;
      for (int i = 0; i < c->n_groups; ++i) {
        work += tile_us(i, on) * (double)count(i);
        longest = std::max(longest, tile_us(i, on));
      }
      const double rounds = work / (256.0 * (double)on) / longest;
      t = longest * (rounds < 2.0 ? std::ceil(rounds) : rounds + 0.3);
    }
    if (kind == 0 || t < best_t) {
      best = kind;
      best_t = t;
    }
  }
  return best;
}

template <int MODE>
void launch_products(const Call& k, LastArgs& a) {
  constexpr bool SYM = MODE == GRAM || MODE == POLY;
  int order[LLATTN_MUON_GROUPS];  // long contractions first: the short ones fill up behind them
  for (int i = 0; i < k.c->n_groups; ++i) order[i] = i;
  std::stable_sort(order, order + k.c->n_groups, [&](int i, int j) {
    return MODE == GRAM ? k.p.g[i].np > k.p.g[j].np : k.p.g[i].mp > k.p.g[j].mp;
  });
  const int kind = k.kind[MODE == LAST ? APPLY : MODE];
  int blocks = 0;
  for (int o = 0; o < k.c->n_groups; ++o) {
    const int i = order[o];
    const GroupPlan& g = k.p.g[i];
    const llattn_muon_group& q = k.groups[i];
    TileGroup& t = a.n.grp[o];
    t = TileGroup{};
    t.b0 = blocks;
    t.tiles = tiles_of(SYM, kind, g.mp, SYM ? g.mp : g.np);
    t.tiles_n = ((SYM ? g.mp : g.np) + kTn[kind] - 1) / kTn[kind];
    t.count = t.tiles * q.batch;
    t.steps = (MODE == GRAM ? g.np : g.mp) / 32;
    t.mp = g.mp; t.np = g.np; t.first = g.first; t.rows = q.rows; t.cols = q.cols; t.w_dtype = q.w_dtype;
    t.x_off = (int64_t)g.x_off; t.a_off = (int64_t)g.a_off;
    t.keep = q.keep; t.step = q.step;
    const float sx = scale_of(g);
    t.alpha = MODE == POLY ? k.c->b : MODE == LAST ? k.c->a / sx : k.c->a;
    t.beta = MODE == GRAM ? kSA / (sx * sx) : MODE == POLY ? k.c->c / kSA : MODE == LAST ? 1.f / (kSA * sx) : 1.f / kSA;
    blocks += (t.count + 7) / 8 * 8;
  }
  a.n.n_groups = k.c->n_groups;
  launch_kind<MODE>(kind, a, blocks, k.st);
}

// ns_thin_kernel's matrices.  A singular value of zero is an eigenvalue of 1e-17 or so of A, of either sign, which every step
// multiplies by a^2: a negative one that has grown to order 1 runs away (rank 4 of 10 x 40: five steps differ from the
// iteration on X by 2e-16, 15 steps by 1e-9, 20 overflow).  Up to 1e10 of growth, 9 steps of a = 3.4445, it stays below 1e-4
// beside sums of any length here.
bool thin(const llattn_muon_cfg* c, const llattn_muon_group& g) {
  return std::min(g.rows, g.cols) <= kThin && std::pow(std::fabs((double)c->a), 2.0 * c->steps) <= 1e10;
}

// All of the call in one workgroup a matrix (ns_small_kernel), where every matrix fits and its launches are the quicker ones.
bool all_small(const llattn_muon_cfg* c, const Plan& p) {
  if (c->tiles) return false;
  const int launches = (p.matrices + kSmall - 1) / kSmall;
  for (int i = 0; i < c->n_groups; ++i)
    if (p.g[i].mp > 64 || p.g[i].np * launches > kSmallCols) return false;
  return true;
}

// One workgroup a matrix: ns_small_kernel or ns_thin_kernel.
int32_t run_single(const char* who, const llattn_muon_cfg* c, const llattn_muon_group* groups, const Plan& p, const void* const* g,
                   const float* const* m, const void* const* w, float* const* m_out, void* const* out, bool update, bool thin,
                   hipStream_t st) {
  SmallArgs a{};
  a.update = update; a.nesterov = c->nesterov; a.steps = c->steps;
  a.mu = c->mu; a.one_mu = (float)(1.0 - (double)c->mu); a.eps = c->eps;
  a.a = c->a; a.b = c->b; a.c = c->c;
  int np = 0, held = 0;
  const auto launch = [&]() {
    if (thin) hipLaunchKernelGGL(ns_thin_kernel, dim3(held), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL(ns_small_kernel, dim3(held), dim3(256), 32768 + (size_t)np * 256, st, a);
    a.n_groups = held = np = 0;
  };
  for (int i = 0; i < c->n_groups; ++i) {
    int b = p.g[i].first;
    const int end = b + groups[i].batch;
    while (b < end) {
      SmallGroup& t = a.grp[a.n_groups++];
      t = SmallGroup{held, groups[i].rows, groups[i].cols, p.g[i].np, groups[i].g_dtype, groups[i].w_dtype, scale_of(p.g[i]),
                     groups[i].keep, groups[i].step};
      np = std::max(np, t.np);
      for (; b < end && held < kSmall; ++b, ++held) {
        a.g[held] = g[b];
        a.out[held] = out[b];
        if (!update) continue;
        a.m[held] = m[b];
        a.m_out[held] = m_out[b];
        a.w[held] = w[b];
      }
      if (held == kSmall) launch();
    }
  }
  if (held) launch();
  return check_launch(who);
}

// The launches of matrices that need not be thin; k.p is their plan.
int32_t run_chain(const char* who, Call& k, const void* const* g, const float* const* m, const void* const* w, float* const* m_out,
                  void* const* out, void* workspace) {
  const llattn_muon_cfg* c = k.c;
  const llattn_muon_group* groups = k.groups;
  const Plan& p = k.p;
  const hipStream_t st = k.st;
  if (all_small(c, p)) return run_single(who, c, groups, p, g, m, w, m_out, out, k.update, false, st);
  char* ws = static_cast<char*>(workspace);
  k.X[0] = reinterpret_cast<uint16_t*>(ws);
  k.X[1] = reinterpret_cast<uint16_t*>(ws + p.x);
  k.A = reinterpret_cast<uint16_t*>(ws + 2 * p.x);
  k.B = reinterpret_cast<uint16_t*>(ws + 2 * p.x + p.a);

  PrepArgs pa{};
  LastArgs na{};
  ElemArgs& e = pa.e;
  e.n_groups = c->n_groups;
  e.momentum = k.update;
  e.nesterov = c->nesterov;
  e.mu = c->mu;
  e.one_mu = (float)(1.0 - (double)c->mu);
  e.eps = c->eps;
  e.part = reinterpret_cast<double*>(ws + 2 * p.x + 2 * p.a);
  e.x = k.X[0];
  int blocks = 0;
  for (int i = 0; i < c->n_groups; ++i) {
    const GroupPlan& q = p.g[i];
    for (int b = q.first; b < q.first + groups[i].batch; ++b) {
      e.g.p[b] = g[b];
      na.out.p[b] = out[b];
      if (!k.update) continue;
      e.m.p[b] = m[b];
      pa.m_out.p[b] = m_out[b];
      na.w.p[b] = w[b];
    }
    ElemGroup& t = e.grp[i];
    t.b0 = blocks;
    t.blocks = t.parts = q.parts;
    t.first = q.first; t.rows = groups[i].rows; t.cols = groups[i].cols; t.flip = t.rows > t.cols;
    t.g_dtype = groups[i].g_dtype; t.mp = q.mp; t.np = q.np;
    t.scale = scale_of(q);
    t.x_off = (int64_t)q.x_off;
    t.part0 = q.part0;
    blocks += groups[i].batch * q.parts;
  }
  k.kind[GRAM] = choose<true>(c, groups, p, true);
  k.kind[POLY] = choose<true>(c, groups, p, false);
  k.kind[APPLY] = choose<false>(c, groups, p, false);
  hipLaunchKernelGGL(muon_prep_kernel, dim3(blocks), dim3(256), 0, st, pa);
  blocks = 0;
  for (int i = 0; i < c->n_groups; ++i) {  // one workgroup per 64 x 64 tile of X
    e.grp[i].b0 = blocks;
    e.grp[i].blocks = (p.g[i].mp / 64) * (p.g[i].np / 64);
    blocks += groups[i].batch * e.grp[i].blocks;
  }
  for (int b = 0; b < p.matrices; ++b) e.m.p[b] = pa.m_out.p[b];
  hipLaunchKernelGGL(muon_split_kernel, dim3(blocks), dim3(256), 0, st, e);

  na.n.a = k.A;
  na.n.b = k.B;
  na.n.update = k.update;
  for (int i = 0; i < c->steps; ++i) {
    na.n.x = k.X[i & 1];
    na.n.y = k.X[(i + 1) & 1];
    launch_products<GRAM>(k, na);
    launch_products<POLY>(k, na);
    if (i + 1 < c->steps) launch_products<APPLY>(k, na);
    else launch_products<LAST>(k, na);
  }
  return check_launch(who);
}

// A part of a call's matrices.
struct Part {
  llattn_muon_cfg c;
  llattn_muon_group groups[LLATTN_MUON_GROUPS];
  const void* g[LLATTN_MUON_BATCH];
  const float* m[LLATTN_MUON_BATCH];
  const void* w[LLATTN_MUON_BATCH];
  float* m_out[LLATTN_MUON_BATCH];
  void* out[LLATTN_MUON_BATCH];
};

int32_t run(const char* who, const llattn_muon_cfg* c, const llattn_muon_group* groups, const void* const* g,
            const float* const* m, const void* const* w, float* const* m_out, void* const* out, void* workspace,
            size_t workspace_bytes, hipStream_t st) {
  if (const int32_t rc = check(c, groups)) return rc;
  Call k{c, groups, plan_of(c, groups), st, {}, nullptr, nullptr, m != nullptr, {}};
  if (!workspace || workspace_bytes < k.p.bytes() || !aligned16(workspace))
    return fail(LLATTN_ERR_WORKSPACE, "%s: needs %zu workspace bytes (got %zu)", who, k.p.bytes(), workspace_bytes);
  if (!g || !out || (k.update && (!w || !m_out))) return fail(LLATTN_ERR_LAYOUT, "%s: null pointer array", who);
  const auto misplaced = [](const void* q, int dtype) { return !q || (uintptr_t)q % (size_t)elem_size(dtype); };
  int thin_groups = 0;
  for (int i = 0; i < c->n_groups; ++i) {
    thin_groups += thin(c, groups[i]);
    for (int b = k.p.g[i].first; b < k.p.g[i].first + groups[i].batch; ++b)
      if (misplaced(g[b], groups[i].g_dtype) || misplaced(out[b], groups[i].w_dtype) ||
          (k.update && (misplaced(m[b], LLATTN_F32) || misplaced(m_out[b], LLATTN_F32) || misplaced(w[b], groups[i].w_dtype))))
        return fail(LLATTN_ERR_LAYOUT, "%s: matrix %d has a null or misaligned pointer", who, b);
  }
  if (c->tiles || !thin_groups) return run_chain(who, k, g, m, w, m_out, out, workspace);
  if (thin_groups == c->n_groups) return run_single(who, c, groups, k.p, g, m, w, m_out, out, k.update, true, st);
  // both: each with its own launches
  for (const bool want : {true, false}) {
    Part q{};
    q.c = *c;
    q.c.n_groups = 0;
    int held = 0;
    for (int i = 0; i < c->n_groups; ++i) {
      if (thin(c, groups[i]) != want) continue;
      q.groups[q.c.n_groups++] = groups[i];
      for (int b = k.p.g[i].first; b < k.p.g[i].first + groups[i].batch; ++b, ++held) {
        q.g[held] = g[b];
        q.out[held] = out[b];
        if (!k.update) continue;
        q.m[held] = m[b];
        q.w[held] = w[b];
        q.m_out[held] = m_out[b];
      }
    }
    Call part{&q.c, q.groups, plan_of(&q.c, q.groups), st, {}, nullptr, nullptr, k.update, {}};
    const int32_t rc = want ? run_single(who, &q.c, q.groups, part.p, q.g, q.m, q.w, q.m_out, q.out, k.update, true, st)
                            : run_chain(who, part, q.g, q.m, q.w, q.m_out, q.out, workspace);
    if (rc) return rc;
  }
  return LLATTN_OK;
}

}  // namespace
}  // namespace llattn

using namespace llattn;

extern "C" size_t llattn_muon_bytes(const llattn_muon_cfg* c, const llattn_muon_group* groups) {
  return check(c, groups) == LLATTN_OK ? plan_of(c, groups).bytes() : 0;
}

extern "C" int32_t llattn_orthogonalize(const llattn_muon_cfg* c, const llattn_muon_group* groups, const void* const* g,
                                        void* const* out, void* workspace, size_t workspace_bytes, void* stream) {
  return run("llattn_orthogonalize", c, groups, g, nullptr, nullptr, nullptr, out, workspace, workspace_bytes,
             static_cast<hipStream_t>(stream));
}

extern "C" int32_t llattn_muon_update(const llattn_muon_cfg* c, const llattn_muon_group* groups, const void* const* g,
                                      const float* const* m, const void* const* w, float* const* m_out, void* const* w_out,
                                      void* workspace, size_t workspace_bytes, void* stream) {
  if (!m) return fail(LLATTN_ERR_LAYOUT, "llattn_muon_update: null momentum array");
  if (c && !(c->mu >= 0.f && c->mu < 1.f)) return fail(LLATTN_ERR_SHAPE, "llattn_muon_update: momentum %g outside [0, 1)", c->mu);
  return run("llattn_muon_update", c, groups, g, m, w, m_out, w_out, workspace, workspace_bytes,
             static_cast<hipStream_t>(stream));
}
