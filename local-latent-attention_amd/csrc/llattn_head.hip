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
// Backward: a piece of the vocabulary at a time, the same product again with dl (bf16) in its epilogue, then dh (+)=
// dl W and dW = dlᵀ h on the GEMM kernels.  Rounding dl to bf16 is as far off as rounding the results to bf16 is (half
// a step of 2^-8 each), and those errors average out over the contraction.
//
// What bounds it: 2 rows V D operations for each of the four products on the matrix cores; with few rows the reads of
// W.
#include <algorithm>

#include "llattn_gemm.h"
#include "llattn_train.h"

namespace llattn {
namespace {

using namespace gemm;

struct HeadArgs {
  int M, N, D;     // rows, columns of this piece, hidden size
  int v0;          // first column of the piece in the vocabulary
  int64_t V;       // vocabulary: targets outside [0, V) are errors
  const uint16_t* h; int64_t ldh;
  const uint16_t* w; int64_t ldw;  // at the piece's first row
  int tiles_m, tiles_n;
  const int64_t* targets;
  int64_t ignore_index;
  // forward: parts [slots][M] and the target's logit [M]
  float2* part;
  int32_t* part_i;
  float* tgt;
  // backward
  const float* lse2;
  const float* grad;
  int grad_stride;
  const float* inv;
  uint16_t* p; int64_t ldp;
};

enum Mode { STATS = 0, STATS_PRED = 1, GRAD = 2 };

// (value, index) maximum with the smaller index on ties
__device__ __forceinline__ void max_first(float& m, int& i, float m2, int i2) {
  if (m2 > m || (m2 == m && i2 < i)) {
    m = m2;
    i = i2;
  }
}

// One (32 MB) x (32 NB) tile of l per workgroup, as tile_product of llattn_gemm_tile.hip: four waves, NST stages of
// 64 k, loads NST - 1 steps ahead.  Offsets are taken from the tile's first row, so h and W may be of any size.
template <int MODE, int MB, int NB, int NST>
__global__ __launch_bounds__(256) void head_tile_kernel(const HeadArgs a) {
  constexpr int TM = 32 * MB, TN = 32 * NB;
  typedef TileOp<true, false, TM> OpA;
  typedef TileOp<true, false, TN> OpB;
  constexpr int STAGE = OpA::BYTES + OpB::BYTES, LOADS = OpA::NB + OpB::NB;
  __shared__ __align__(1024) unsigned char smem[NST * STAGE];
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  constexpr int GM = 8;
  const int group = t / (GM * a.tiles_n), first_m = group * GM, gm = min(a.tiles_m - first_m, GM);
  const int tm = first_m + (t % (GM * a.tiles_n)) % gm, tn = t % (GM * a.tiles_n) / gm;
  const int m0 = tm * TM, n0 = tn * TN;
  const int rows = min(TM, a.M - m0), cols = min(TN, a.N - n0);
  const uint16_t* hb = a.h + (int64_t)m0 * a.ldh;
  const uint16_t* wb = a.w + (int64_t)n0 * a.ldw;
  const int64_t hbytes = ((int64_t)(rows - 1) * a.ldh + a.D) * 2, wbytes = ((int64_t)(cols - 1) * a.ldw + a.D) * 2;
  OpA oa;
  OpB ob;
  oa.init(a.ldh, 0, rows, wave, lane);
  ob.init(a.ldw, 0, cols, wave, lane);
  const int nk = (a.D + SK - 1) / SK;
  auto fetch = [&](int kt) {
    const int k0 = min(kt, nk - 1) * SK, klim = a.D - k0;
    const i32x4 ra = step_rsrc<true>(hb, a.ldh, hbytes, k0), rb = step_rsrc<true>(wb, a.ldw, wbytes, k0);
    unsigned char* st = smem + (kt % NST) * STAGE;
#pragma unroll
    for (int i = 0; i < OpA::NB; ++i) oa.dma(ra, st, wave, i, klim);
#pragma unroll
    for (int i = 0; i < OpB::NB; ++i) ob.dma(rb, st + OpA::BYTES, wave, i, klim);
  };
  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) fetch(s);
  for (int kt = 0; kt < nk; ++kt) {
    __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0((NST - 2) * LOADS));  // this wave's loads of step kt have landed
    __builtin_amdgcn_s_barrier();  // every wave's; and every wave has read step kt - 1, whose stage is free
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    fetch(kt + NST - 1);
    const unsigned char* st = smem + (kt % NST) * STAGE;
    bf16x8 fa[2][MB], fb[2][NB];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < NB; ++j) fb[h][j] = OpB::frag(st + OpA::BYTES, wn * 16 * NB + 16 * j, r, g, h);
#pragma unroll
      for (int i = 0; i < MB; ++i) fa[h][i] = OpA::frag(st, wm * 16 * MB + 16 * i, r, g, h);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)  // B first: lane (r, g) accumulates l[row r][column 4 g + e]
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[h][j], fa[h][i], acc[i][j], 0, 0, 0);
  }
  __builtin_amdgcn_s_waitcnt(wait_vm_lgkm0(0));  // no DMA may land after the workgroup exits
  const int colw = n0 + wn * 16 * NB + 4 * g;    // first column of this lane within the piece
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int row = m0 + wm * 16 * MB + 16 * i + r;
    const bool live = row < a.M;
    const int64_t tg = live ? a.targets[row] : a.ignore_index;
    const int64_t tc = tg - a.v0;  // the target's column within the piece
    if constexpr (MODE == GRAD) {
      const float l2 = live ? a.lse2[row] : 0.f;
      const bool ignored = tg == a.ignore_index;
      float s = 0.f;
      if (live && !ignored)
        s = tg < 0 || tg >= a.V ? __builtin_nanf("") : a.grad[(int64_t)row * a.grad_stride] * (a.inv ? *a.inv : 1.f);
      uint16_t* out = a.p + (int64_t)row * a.ldp;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int c = colw + 16 * j;
        float d[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float q = fast_exp2(fmaf(acc[i][j][e], kLog2e, -l2)) - (c + e == tc ? 1.f : 0.f);
          d[e] = ignored || c + e >= a.N ? 0.f : q * s;  // columns past the piece are zero: the products contract over them
        }
        if (live && c < a.ldp) store4<uint16_t>(out + c, d);
      }
    } else {
      float m = kNegInf;
      int mi = 0x7fffffff;
#pragma unroll
      for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = colw + 16 * j + e;
          const float v = c < a.N ? acc[i][j][e] : kNegInf;
          acc[i][j][e] = v;
          if constexpr (MODE == STATS_PRED) {
            if (c < a.N) max_first(m, mi, v, a.v0 + c);
          } else {
            m = fmaxf(m, v);
          }
          if (c == tc && live && c < a.N) a.tgt[row] = v;
        }
      if constexpr (MODE == STATS_PRED) {
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
        if constexpr (MODE == STATS_PRED) a.part_i[o] = mi;
      }
    }
  }
}

// Joins the parts of 8 rows: 32 threads a row take every 32nd part, then the 32 in order, behind what the columns before
// left (`run`, where `more`).  FINAL: the loss, else `run`.
struct JoinArgs {
  const float2* part; const int32_t* part_i;
  int slots, M, more;
  float2* run; int32_t* run_i;
  const float* tgt; const int64_t* targets; int64_t ignore_index, V;
  float *loss, *lse2;
  int32_t* pred;
};

__device__ __forceinline__ void join(float& m, float& s, int& i, float m2, float s2, int i2) {
  const float M = fmaxf(m, m2);
  const float C = M == kNegInf ? 0.f : __fmul_rn(M, kLog2e);
  const float c1 = m == kNegInf ? C : __fmul_rn(m, kLog2e), c2 = m2 == kNegInf ? C : __fmul_rn(m2, kLog2e);
  s = s * fast_exp2(c1 - C) + s2 * fast_exp2(c2 - C);
  max_first(m, i, m2, i2);
  m = M;
}

template <bool FINAL>
__global__ __launch_bounds__(256) void head_join_kernel(const JoinArgs a) {
  __shared__ float sm[32][8], ss[32][8];
  __shared__ int si[32][8];
  const int lr = threadIdx.x & 7, q = threadIdx.x >> 3, row = blockIdx.x * 8 + lr;
  float m = kNegInf, s = 0.f;
  int mi = 0x7fffffff;
  if (row < a.M) {
    if (a.more && q == 0) {
      const float2 x = a.run[row];
      m = x.x;
      s = x.y;
      if (a.part_i) mi = a.run_i[row];
    }
    for (int k = q; k < a.slots; k += 32) {
      const float2 x = a.part[(int64_t)k * a.M + row];
      join(m, s, mi, x.x, x.y, a.part_i ? a.part_i[(int64_t)k * a.M + row] : 0);
    }
  }
  sm[q][lr] = m;
  ss[q][lr] = s;
  si[q][lr] = mi;
  __syncthreads();
  if (threadIdx.x >= 8 || row >= a.M) return;
  for (int k = 1; k < 32; ++k) join(m, s, mi, sm[k][lr], ss[k][lr], si[k][lr]);
  if constexpr (!FINAL) {
    a.run[row] = make_float2(m, s);
    if (a.part_i) a.run_i[row] = mi;
    return;
  }
  const float C = m == kNegInf ? 0.f : __fmul_rn(m, kLog2e), lg = __builtin_amdgcn_logf(s);  // base 2
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
    if (inv) *inv = 1.f / (float)sn[0];
  }
}

__global__ __launch_bounds__(256) void head_cast_kernel(const float* x, uint16_t* y, int64_t quads) {
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < quads; q += (int64_t)gridDim.x * 256) {
    float v[4];
    load4<float>(x + 4 * q, v);
    store4<uint16_t>(y + 4 * q, v);
  }
}

constexpr size_t up(size_t n) { return (n + 255) & ~size_t(255); }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Tile { int tm, tn; };
Tile tile_of(int rows) { return rows <= 64 ? Tile{64, 128} : Tile{128, 128}; }

int32_t check(const llattn_head_cfg* c) {
  if (!c) return fail(LLATTN_ERR_SHAPE, "llattn_head: null configuration");
  if (c->rows <= 0 || c->V <= 0 || c->D <= 0 || c->D % 8 || c->V > 0x7fffff00)
    return fail(LLATTN_ERR_SHAPE, "llattn_head: rows %d, V %d, D %d: must be positive, D a multiple of 8", c->rows, c->V,
                c->D);
  if (c->piece < 0 || c->piece % 256)
    return fail(LLATTN_ERR_SHAPE, "llattn_head: piece %d must be 0 or a multiple of 256", c->piece);
  if (c->dw_dtype != LLATTN_F32 && c->dw_dtype != LLATTN_BF16)
    return fail(LLATTN_ERR_DTYPE, "llattn_head: unknown dW dtype %d", c->dw_dtype);
  return LLATTN_OK;
}

// forward: columns whose parts are joined at once, so that those stay within 256 MB
struct FwdPlan { Tile t; int range; size_t slots, bytes; };
FwdPlan fwd_plan(const llattn_head_cfg* c) {
  FwdPlan f;
  f.t = tile_of(c->rows);
  const int64_t most = std::max<int64_t>(1, (int64_t)(256 << 20) / (24 * (int64_t)c->rows));  // tile columns, two parts of 12 bytes each
  const int64_t tiles = ceil_div(c->V, f.t.tn);
  f.range = (int)(std::min(tiles, most) * f.t.tn);
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

llattn_gemm_desc dh_desc(const llattn_head_cfg* c, const void* p, int64_t ldp, const void* w, int64_t ldw, int nv, void* out,
                         bool f32, bool add) {
  llattn_gemm_desc d{};
  d.M = c->rows; d.N = c->D; d.K = (nv + 7) / 8 * 8;
  d.A = p; d.lda = ldp;
  d.B = w; d.ldb = ldw; d.b_trans = 1;
  d.C = out; d.ldc = c->D; d.c_dtype = f32 ? LLATTN_F32 : LLATTN_BF16; d.accumulate = add;
  return d;
}
llattn_gemm_desc dw_desc(const llattn_head_cfg* c, const void* p, int64_t ldp, const void* h, int64_t ldh, int nv, void* out) {
  llattn_gemm_desc d{};
  d.M = (nv + 7) / 8 * 8; d.N = c->D; d.K = c->rows;
  d.A = p; d.lda = ldp; d.a_trans = 1;
  d.B = h; d.ldb = ldh; d.b_trans = 1;
  d.C = out; d.ldc = c->D; d.c_dtype = c->dw_dtype;
  return d;
}

struct BwdPlan { int piece, pieces; size_t p, acc, gemm; size_t bytes() const { return p + acc + gemm; } };
BwdPlan bwd_plan(const llattn_head_cfg* c) {
  BwdPlan b{};
  b.piece = piece_of(c);
  b.pieces = (int)ceil_div(c->V, b.piece);
  b.p = up((size_t)c->rows * b.piece * 2);
  b.acc = b.pieces > 1 ? up((size_t)c->rows * c->D * 4) : 0;
  const int last = c->V - (b.pieces - 1) * b.piece;
  for (int nv : {std::min(b.piece, c->V), last}) {
    const llattn_gemm_desc d0 = dh_desc(c, nullptr, b.piece, nullptr, c->D, nv, nullptr, b.pieces > 1, false);
    const llattn_gemm_desc d1 = dw_desc(c, nullptr, b.piece, nullptr, c->D, nv, nullptr);
    b.gemm = std::max({b.gemm, up(llattn_gemm_workspace_size(&d0)), up(llattn_gemm_workspace_size(&d1))});
  }
  return b;
}

template <int MODE>
void launch_tiles(HeadArgs& a, const Tile& t, hipStream_t st) {
  a.tiles_m = (a.M + t.tm - 1) / t.tm;
  a.tiles_n = (a.N + t.tn - 1) / t.tn;
  const dim3 grid(a.tiles_m * a.tiles_n), block(256);
  if (t.tm == 64) hipLaunchKernelGGL((head_tile_kernel<MODE, 2, 4, 3>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((head_tile_kernel<MODE, 4, 4, 2>), grid, block, 0, st, a);
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
  a.M = c->rows; a.D = c->D; a.V = c->V;
  a.h = static_cast<const uint16_t*>(h); a.ldh = ldh; a.ldw = ldw;
  a.targets = targets; a.ignore_index = ignore_index;
  j.M = c->rows; j.tgt = a.tgt; j.targets = targets; j.ignore_index = ignore_index; j.V = c->V;
  j.loss = loss; j.lse2 = lse2; j.pred = pred;
  const dim3 jgrid((c->rows + 7) / 8), block(256);
  j.part = a.part; j.part_i = pred ? a.part_i : nullptr;
  for (int64_t v0 = 0; v0 < c->V; v0 += f.range) {
    a.v0 = (int)v0;
    a.N = std::min(f.range, c->V - a.v0);
    a.w = static_cast<const uint16_t*>(W) + (int64_t)a.v0 * ldw;
    if (pred) launch_tiles<STATS_PRED>(a, f.t, st);
    else launch_tiles<STATS>(a, f.t, st);
    j.slots = 2 * a.tiles_n;
    j.more = v0 > 0;
    if (v0 + f.range < c->V) hipLaunchKernelGGL(head_join_kernel<false>, jgrid, block, 0, st, j);
    else hipLaunchKernelGGL(head_join_kernel<true>, jgrid, block, 0, st, j);
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
  char* ws = static_cast<char*>(workspace);
  HeadArgs a{};
  a.p = reinterpret_cast<uint16_t*>(ws); a.ldp = b.piece;
  float* acc = reinterpret_cast<float*>(ws + b.p);
  void* gws = ws + b.p + b.acc;
  a.M = c->rows; a.D = c->D; a.V = c->V;
  a.h = static_cast<const uint16_t*>(h); a.ldh = ldh; a.ldw = ldw;
  a.targets = targets; a.ignore_index = ignore_index;
  a.lse2 = lse2; a.grad = grad; a.grad_stride = grad_stride; a.inv = inv;
  const int64_t dwsz = c->dw_dtype == LLATTN_F32 ? 4 : 2;
  if (!dh && !dW) return LLATTN_OK;
  for (int q = 0; q < b.pieces; ++q) {
    a.v0 = (int)((int64_t)q * b.piece);
    a.N = std::min(b.piece, c->V - a.v0);
    a.w = static_cast<const uint16_t*>(W) + (int64_t)a.v0 * ldw;
    launch_tiles<GRAD>(a, tile_of(c->rows), st);
    if (dh) {
      const bool f32 = b.pieces > 1;
      const llattn_gemm_desc d = dh_desc(c, a.p, a.ldp, a.w, ldw, a.N, f32 ? static_cast<void*>(acc) : dh, f32, q > 0);
      if (const int32_t rc = gemm::product(&d, a.N, gws, b.gemm, st)) return rc;
    }
    if (dW) {
      const llattn_gemm_desc d = dw_desc(c, a.p, a.ldp, h, ldh, a.N, static_cast<char*>(dW) + (int64_t)a.v0 * c->D * dwsz);
      if (const int32_t rc = gemm::product(&d, c->rows, gws, b.gemm, st)) return rc;
    }
  }
  if (dh && b.pieces > 1) {
    const int64_t quads = (int64_t)c->rows * c->D / 4;
    hipLaunchKernelGGL(head_cast_kernel, dim3((unsigned)std::min<int64_t>((quads + 255) / 256, 4096)), dim3(256), 0, st, acc,
                       static_cast<uint16_t*>(dh), quads);
  }
  return check_launch("llattn_head_bwd");
}
