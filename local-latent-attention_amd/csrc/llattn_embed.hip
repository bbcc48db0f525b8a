// Token rows, scaled, plus position rows, and the gradients of both tables (include/llattn_lm.h).
//
//   out[n] = s W[id_n] + Pos[pos_n],   dW[v] = s sum_{id_n = v} dout[n],   dPos[p] = sum_{pos_n = p} dout[n]
//
// The gradients are sums over the rows of one key (a token or a position), so the rows are ordered by key first: one
// launch, a workgroup for each residue class of keys (key mod buckets), which reads all keys, keeps its own in their
// order and counts them out by key.  The order of the keys among themselves is of no use here; the residues spread a
// text's frequent tokens, whose numbers are close, over the workgroups.  Where positions are n % T the order is known.
//
// A run (the rows of one key, of length L) is summed in a tree of its own: blocks of 32 rows from its first row on, 32 of
// these blocks to one of 1024 rows, then the blocks of 1024, the blocks of 32 behind them and the rows behind those in
// order.  One launch adds the blocks of 32, one (from 1024 rows on) those of 1024, and the last one writes every row of the
// tables, zeros where a run is empty.  Nothing depends on where the run lies in the order, so neither atomics nor other tokens
// change a bit.  A block of 32 that starts within positions [32 c, 32 c + 32) of the order is the only one that does
// (it covers position 32 c + 31), which makes c its number.
//
// What bounds it: memory.  Forward: a table row read and a row written per token; backward: dout read once for each
// table, the tables' gradients written whole.
#include <algorithm>

#include "llattn_abi.h"
#include "llattn_device.h"
#include "llattn_lm.h"

namespace llattn {
namespace {

constexpr int kLeaf = 32;          // rows of a block; as many blocks make one of the next level
constexpr int kKeys = 512;         // keys of a bucket at most
constexpr int kWaves = 16;         // of a sorting workgroup
constexpr int kList = 4096;        // rows of a bucket held in LDS
constexpr int kMostRows = 1 << 22; // of a table: 8192 buckets

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_f __attribute__((aligned(4)));
typedef u32x4 u32x4_h __attribute__((aligned(2)));

// 16 bytes of a row at any alignment of whole elements; `left` elements remain in the row
template <typename T>
__device__ __forceinline__ u32x4 load_piece(const T* p, int left) {
  constexpr int N = Vec16<T>::N;
  if (left >= N) {
    if constexpr (N == 4) return *reinterpret_cast<const u32x4_f*>(p);
    else return *reinterpret_cast<const u32x4_h*>(p);
  }
  u32x4 v = {0, 0, 0, 0};
  for (int e = 0; e < left; ++e) {
    if constexpr (N == 4) v[e] = __float_as_uint(p[e]);
    else v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void store_piece(T* p, u32x4 v, int left) {
  constexpr int N = Vec16<T>::N;
  if (left >= N) {
    if constexpr (N == 4) *reinterpret_cast<u32x4_f*>(p) = v;
    else *reinterpret_cast<u32x4_h*>(p) = v;
    return;
  }
  for (int e = 0; e < left; ++e) {
    if constexpr (N == 4) p[e] = __uint_as_float(v[e]);
    else p[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
  }
}
template <typename T>
__device__ __forceinline__ void unpack(u32x4 v, float (&o)[Vec16<T>::N]) {
  if constexpr (std::is_same_v<T, float>) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = __uint_as_float(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[2 * e] = __uint_as_float(v[e] << 16);
      o[2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
    }
  }
}
template <typename T>
__device__ __forceinline__ u32x4 pack(const float (&o)[Vec16<T>::N]) {
  u32x4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (std::is_same_v<T, float>) v[e] = __float_as_uint(o[e]);
    else v[e] = pack_bf16x2(o[2 * e], o[2 * e + 1]);
  }
  return v;
}

// A row's 16-byte pieces are shared by `width` lanes (8 to 64) of a wave, in `parts` tasks of `per` pieces each.
struct Split { int pieces, width, parts, per; };
// Threads of a launch whose workgroups may pass 2^32 threads in one dimension
__device__ __forceinline__ int64_t thread_of() { return ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; }
struct Task { int row, from, to, lane; };
__device__ __forceinline__ Task task_of(const Split& s, int64_t task, int lane) {
  const int row = (int)(task / s.parts), part = (int)(task - (int64_t)row * s.parts);
  return Task{row, part * s.per, min((part + 1) * s.per, s.pieces), lane};
}

__device__ __forceinline__ int64_t index_at(const void* p, int bytes, int64_t n) {
  return bytes == 8 ? static_cast<const int64_t*>(p)[n] : (int64_t)static_cast<const int32_t*>(p)[n];
}

struct FwdArgs {
  int rows, T, V, P, D, index_bytes;
  const void *ids, *pos;
  const void *W, *Pos;
  int64_t ldw, ldp;
  void* out;
  float scale;
  Split split;
};

template <typename T>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const FwdArgs a) {
  constexpr int N = Vec16<T>::N;
  const int64_t t = thread_of() / a.split.width;
  if (t >= (int64_t)a.rows * a.split.parts) return;
  const Task k = task_of(a.split, t, threadIdx.x % a.split.width);
  const int64_t id = index_at(a.ids, a.index_bytes, k.row);
  const int64_t p = a.P ? a.pos ? index_at(a.pos, a.index_bytes, k.row) : k.row % a.T : 0;
  const bool ok = id >= 0 && id < a.V && (!a.P || (p >= 0 && p < a.P));
  const T* w = static_cast<const T*>(a.W) + (ok ? id : 0) * a.ldw;
  const T* q = static_cast<const T*>(a.Pos) + (ok ? p : 0) * a.ldp;
  T* o = static_cast<T*>(a.out) + (int64_t)k.row * a.D;
  for (int c = k.from + k.lane; c < k.to; c += a.split.width) {
    const int d = c * N, left = a.D - d;
    float x[N], y[N];
    unpack<T>(load_piece(w + d, left), x);
    if (a.P) unpack<T>(load_piece(q + d, left), y);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      x[e] = a.P ? fmaf(a.scale, x[e], y[e]) : a.scale * x[e];
      if (!ok) x[e] = __builtin_nanf("");
    }
    store_piece(o + d, pack<T>(x), left);
  }
}

// Rows by key.  order: rows, the runs of a bucket one after another; runs[key]: first and one past the last position of its run.
struct Keys {
  const void* keys;       // null: row n has key n % T, and nothing is written (runs of `alike` rows)
  int index_bytes;
  int T, alike;
  int R;                  // keys outside [0, R) and `padding` have no run
  int64_t padding;
  int buckets;            // a power of two, R <= kKeys buckets
  int32_t* order;
  int2* runs;
  int2* list;             // scratch [rows]
};
__device__ __forceinline__ int row_at(const Keys& s, int i) {
  return s.keys ? s.order[i] : (i % s.alike) * s.T + i / s.alike;
}
__device__ __forceinline__ int2 run_of(const Keys& s, int key) {
  if (s.keys) return s.runs[key];
  return key < s.T ? make_int2(key * s.alike, (key + 1) * s.alike) : make_int2(0, 0);
}
__device__ __forceinline__ int key_at(const Keys& s, int i) {  // of position i < the number of rows that have runs
  return s.keys ? (int)index_at(s.keys, s.index_bytes, s.order[i]) : i / s.alike;
}

struct SortArgs {
  Keys set[2];
  int first[3];  // workgroups of each set
  int rows;
  int32_t* counted;  // rows that have runs, of each set
};

// What a workgroup reads of 16 waves x 64 keys at a time: latency-bound, so several such pieces are in flight.
__global__ __launch_bounds__(64 * kWaves) void embed_sort_kernel(const SortArgs a) {
  __shared__ int2 list[kList];
  __shared__ int count[kWaves][kKeys];
  __shared__ int eq_of[kWaves], lt_of[kWaves], all_of[kWaves], sums[kKeys / 64];
  const int which = (int)blockIdx.x >= a.first[1];
  const Keys& s = a.set[which];
  const int b = blockIdx.x - a.first[which], mask = s.buckets - 1, shift = 31 - __builtin_clz(s.buckets);
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t seg = ((a.rows + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int64_t lo = min((int64_t)a.rows, w * seg), hi = min((int64_t)a.rows, lo + seg);
  const auto key_of = [&](int64_t n) -> int {  // or -1
    if (n >= hi) return -1;
    const int64_t k = index_at(s.keys, s.index_bytes, n);
    return k >= 0 && k < s.R && k != s.padding ? (int)k : -1;
  };
  constexpr int U = 8;
  int eq = 0, lt = 0, all = 0;
  for (int64_t n = lo; n < hi; n += 64 * U) {
    int k[U];
#pragma unroll
    for (int u = 0; u < U; ++u) k[u] = key_of(n + 64 * u + lane);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      eq += k[u] >= 0 && (k[u] & mask) == b;
      lt += k[u] >= 0 && (k[u] & mask) < b;
      all += k[u] >= 0;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    eq += __shfl_xor(eq, o);
    lt += __shfl_xor(lt, o);
    all += __shfl_xor(all, o);
  }
  if (lane == 0) {
    eq_of[w] = eq;
    lt_of[w] = lt;
    all_of[w] = all;
  }
  for (int i = threadIdx.x; i < kWaves * kKeys; i += 64 * kWaves) (&count[0][0])[i] = 0;
  __syncthreads();
  int base = 0, n_list = 0, at = 0, total = 0;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    base += lt_of[v];
    if (v < w) at += eq_of[v];
    n_list += eq_of[v];
    total += all_of[v];
  }
  if (b == 0 && threadIdx.x == 0) a.counted[which] = total;
  // this bucket's rows in their order
  int2* const kept = n_list <= kList ? list : s.list + base;
  if (eq) {
    for (int64_t n = lo; n < hi; n += 64 * U) {
      int k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) k[u] = key_of(n + 64 * u + lane);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool mine = k[u] >= 0 && (k[u] & mask) == b;
        const uint64_t m = __ballot(mine);
        if (mine) kept[at + __popcll(m & ((1ull << lane) - 1))] = make_int2((int)(n + 64 * u + lane), k[u] >> shift);
        at += __popcll(m);
      }
    }
  }
  __syncthreads();
  // counted out by key: each wave counts a stretch of the list, the counts are added up by key and, within a key, by wave
  const int step = ((n_list + kWaves - 1) / kWaves + 63) / 64 * 64;
  const int from = min(n_list, w * step), to = min(n_list, from + step);
  for (int i = from + lane; i < to; i += 64) atomicAdd(&count[w][kept[i].y], 1);
  __syncthreads();
  if (threadIdx.x < kKeys) {
    const int k = threadIdx.x;
    int c[kWaves], mine = 0;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      c[v] = mine;
      mine += count[v][k];
    }
    int before = mine;  // inclusive scan over the 64 keys of this wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(before, o);
      if (lane >= o) before += x;
    }
    if (lane == 63) sums[w] = before;
    before -= mine;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) count[v][k] = before + c[v];
    // waves of the keys before are added below, once their sums are there
    eq = mine;
    lt = before;
  }
  __syncthreads();
  if (threadIdx.x < kKeys) {
    int more = 0;
    for (int v = 0; v < w; ++v) more += sums[v];
#pragma unroll
    for (int v = 0; v < kWaves; ++v) count[v][threadIdx.x] += more;
    const int64_t key = b + ((int64_t)threadIdx.x << shift);
    if (key < s.R) s.runs[key] = eq ? make_int2(base + more + lt, base + more + lt + eq) : make_int2(0, 0);
  }
  __syncthreads();
  for (int i = from; i < to; i += 64) {
    const bool live = i + lane < to;
    const int2 x = live ? kept[i + lane] : make_int2(0, 0);
    uint64_t m = __ballot(live);  // the lanes of the same key
#pragma unroll
    for (int bit = 0; bit < 9; ++bit) {
      const bool one = x.y >> bit & 1;
      const uint64_t v = __ballot(one);
      m &= one ? v : ~v;
    }
    if (live) {
      const int rank = __popcll(m & ((1ull << lane) - 1)), first = __ffsll((unsigned long long)m) - 1;
      int at0 = 0;
      if (rank == 0) at0 = atomicAdd(&count[w][x.y], __popcll(m));
      at0 = __shfl(at0, first);
      s.order[base + at0 + rank] = x.x;
    }
  }
}
static_assert(kKeys == 1 << 9, "bits of a key within its bucket");

struct BwdArgs {
  Keys set[2];
  int64_t tasks[3];        // first task of each set
  int rows, D;
  const int32_t* counted;  // rows that have runs, of the sorted sets
  const void* dout;
  float* leaf[2];          // sums of 32 rows [rows / 32][Dp], and of 1024
  float* node[2];
  void* out[2];            // dW, dPos
  float scale[2];
  Split split, fsplit;     // of a row of dout, of a row of sums
  int Dp;
};

// acc += the rows at `get(i)`, i < n, in order
template <typename T, typename F>
__device__ __forceinline__ void add_rows(float (&acc)[Vec16<T>::N], int n, int left, F&& get) {
  constexpr int N = Vec16<T>::N, U = 8;
  int i = 0;
  for (; i + U <= n; i += U) {
    u32x4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load_piece(get(i + u), left);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[N];
      unpack<T>(v[u], x);
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += x[e];
    }
  }
  for (; i < n; ++i) {
    float x[N];
    unpack<T>(load_piece(get(i), left), x);
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] += x[e];
  }
}

// The first position of the block of `size` positions that starts in [c size, (c + 1) size), or -1
__device__ __forceinline__ int block_start(const Keys& s, int counted, int c, int size) {
  const int64_t last = (int64_t)c * size + size - 1;
  if (last >= counted) return -1;
  const int2 r = run_of(s, key_at(s, (int)last));
  const int at = r.x + ((int)last - r.x) / size * size;
  return at + size <= r.y ? at : -1;
}

template <typename T>
__global__ __launch_bounds__(256) void embed_leaf_kernel(const BwdArgs a) {
  constexpr int N = Vec16<T>::N;
  const int64_t t = thread_of() / a.split.width;
  const int set = t >= a.tasks[1];
  if (t >= a.tasks[2]) return;
  const Keys& s = a.set[set];
  const Task k = task_of(a.split, t - a.tasks[set], threadIdx.x % a.split.width);
  const int at = block_start(s, s.keys ? a.counted[set] : a.rows, k.row, kLeaf);
  if (at < 0) return;
  float* const o = a.leaf[set] + (int64_t)k.row * a.Dp;
  for (int c = k.from + k.lane; c < k.to; c += a.split.width) {
    const int d = c * N, left = a.D - d;
    float acc[N] = {};
    add_rows<T>(acc, kLeaf, left, [&](int i) { return static_cast<const T*>(a.dout) + (int64_t)row_at(s, at + i) * a.D + d; });
#pragma unroll
    for (int e = 0; e < N; e += 4) *reinterpret_cast<float4*>(o + d + e) = make_float4(acc[e], acc[e + 1], acc[e + 2], acc[e + 3]);
  }
}

__global__ __launch_bounds__(256) void embed_node_kernel(const BwdArgs a) {
  const int64_t t = thread_of() / a.fsplit.width;
  const int set = t >= a.tasks[1];
  if (t >= a.tasks[2]) return;
  const Keys& s = a.set[set];
  const Task k = task_of(a.fsplit, t - a.tasks[set], threadIdx.x % a.fsplit.width);
  const int at = block_start(s, s.keys ? a.counted[set] : a.rows, k.row, kLeaf * kLeaf);
  if (at < 0) return;
  float* const o = a.node[set] + (int64_t)k.row * a.Dp;
  for (int c = k.from + k.lane; c < k.to; c += a.fsplit.width) {
    float acc[4] = {};
    add_rows<float>(acc, kLeaf, 4, [&](int i) { return a.leaf[set] + (int64_t)(at / kLeaf + i) * a.Dp + 4 * c; });
    *reinterpret_cast<float4*>(o + 4 * c) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  }
}

// Rows of sums, of a whole run: the blocks of 1024, those of 32 behind them, the rows behind those
template <typename T>
__global__ __launch_bounds__(256) void embed_bwd_kernel(const BwdArgs a) {
  constexpr int N = Vec16<T>::N;
  const int64_t t = thread_of() / a.split.width;
  const int set = t >= a.tasks[1];
  if (t >= a.tasks[2]) return;
  const Keys& s = a.set[set];
  const Task k = task_of(a.split, t - a.tasks[set], threadIdx.x % a.split.width);
  const int2 run = run_of(s, k.row);
  const int L = run.y - run.x, nodes = L / (kLeaf * kLeaf), leaves = L / kLeaf - nodes * kLeaf, rest = L % kLeaf;
  T* const o = static_cast<T*>(a.out[set]) + (int64_t)k.row * a.D;
  const int leaf0 = run.x + nodes * kLeaf * kLeaf, row0 = run.y - rest;
  for (int c = k.from + k.lane; c < k.to; c += a.split.width) {
    const int d = c * N, left = a.D - d;
    float acc[N] = {};
    for (int e = 0; e < N && nodes; e += 4) {
      float x[4] = {};
      add_rows<float>(x, nodes, 4, [&](int i) { return a.node[set] + (int64_t)(run.x / (kLeaf * kLeaf) + i) * a.Dp + d + e; });
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[e + q] += x[q];
    }
    for (int e = 0; e < N && leaves; e += 4) {
      float x[4] = {};
      add_rows<float>(x, leaves, 4, [&](int i) { return a.leaf[set] + (int64_t)(leaf0 / kLeaf + i) * a.Dp + d + e; });
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[e + q] += x[q];
    }
    if (rest) {
      float x[N] = {};
      add_rows<T>(x, rest, left, [&](int i) { return static_cast<const T*>(a.dout) + (int64_t)row_at(s, row0 + i) * a.D + d; });
#pragma unroll
      for (int e = 0; e < N; ++e) acc[e] += x[e];
    }
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] *= a.scale[set];
    store_piece(o + d, pack<T>(acc), left);
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr size_t up(size_t n) { return (n + 255) & ~size_t(255); }

// Lanes and tasks of a row of D elements: up to four pieces a lane, fewer where there are too few rows to fill the chip.
Split split_of(int D, int n, int64_t rows) {
  Split s;
  s.pieces = (int)ceil_div(D, n);
  s.width = s.pieces > 32 ? 64 : s.pieces > 16 ? 32 : s.pieces > 8 ? 16 : 8;
  const int turns = (int)ceil_div(s.pieces, s.width), most = rows * s.width >= 64 * 4096 ? 4 : 1;
  s.parts = (int)ceil_div(turns, most);
  s.per = (int)ceil_div(turns, s.parts) * s.width;
  s.parts = (int)ceil_div(s.pieces, s.per);
  return s;
}

dim3 grid_of(int64_t tasks, const Split& s) {
  const int64_t n = ceil_div(tasks * s.width, 256), x = std::min<int64_t>(n, 1 << 20);
  return dim3((unsigned)x, (unsigned)ceil_div(n, x));
}

int32_t check(const char* who, const llattn_embed_cfg* c, bool has_pos) {
  if (!c) return fail(LLATTN_ERR_SHAPE, "%s: null configuration", who);
  if (c->rows < 0 || c->rows > 0x7fffffff || c->V <= 0 || c->V > kMostRows || c->P < 0 || c->P > kMostRows || c->D <= 0 || c->D > 1 << 20)
    return fail(LLATTN_ERR_SHAPE, "%s: rows %lld (below 2^31), V %d, P %d (at most 2^22), D %d", who, (long long)c->rows, c->V, c->P, c->D);
  if (c->P && !has_pos && (c->T <= 0 || c->T > c->P || c->rows % c->T))
    return fail(LLATTN_ERR_SHAPE, "%s: T %d must be in [1, P %d] and divide the rows (%lld)", who, c->T, c->P, (long long)c->rows);
  if (c->dtype != LLATTN_F32 && c->dtype != LLATTN_BF16) return fail(LLATTN_ERR_DTYPE, "%s: unknown dtype %d", who, c->dtype);
  if (c->index_bytes != 4 && c->index_bytes != 8) return fail(LLATTN_ERR_DTYPE, "%s: indices of %d bytes", who, c->index_bytes);
  if (c->padding < -1 || c->padding >= c->V) return fail(LLATTN_ERR_SHAPE, "%s: padding %lld outside [-1, V)", who, (long long)c->padding);
  return LLATTN_OK;
}

bool whole(const void* p, int64_t size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) == 0; }

int buckets_of(int R) {
  int b = 256;  // a workgroup for every CU
  while ((int64_t)b * kKeys < R) b *= 2;
  return b;
}

// Workspace: for a sorted set order, runs and list; for every set the sums of 32 and of 1024 rows; counted
struct Plan {
  int64_t rows, leaves, nodes;
  int Dp;
  int trees;
  size_t set_bytes[2], tree_bytes;
  size_t bytes() const { return 256 + set_bytes[0] + set_bytes[1] + trees * tree_bytes; }
};
Plan plan_of(const llattn_embed_cfg* c, bool has_pos) {
  Plan p{};
  p.rows = c->rows;
  p.leaves = c->rows / kLeaf;
  p.nodes = c->rows / (kLeaf * kLeaf);
  p.Dp = (c->D + 7) / 8 * 8;
  p.trees = c->P ? 2 : 1;
  const auto sorted = [&](int R) { return up((size_t)c->rows * 4) + up((size_t)R * 8) + up((size_t)c->rows * 8); };
  p.set_bytes[0] = sorted(c->V);
  p.set_bytes[1] = c->P && has_pos ? sorted(c->P) : 0;
  p.tree_bytes = up((size_t)p.leaves * p.Dp * 4) + up((size_t)p.nodes * p.Dp * 4);
  return p;
}

template <typename T>
void launch_bwd(BwdArgs& a, const Plan& p, const int64_t (&table)[2], hipStream_t st) {
  const auto tasks = [&](const Split& s, int64_t n0, int64_t n1) {
    a.tasks[0] = 0;
    a.tasks[1] = n0 * s.parts;
    a.tasks[2] = (n0 + n1) * s.parts;
    return a.tasks[2];
  };
  const int64_t on0 = table[0] > 0, on1 = table[1] > 0;
  if (p.leaves) {
    a.split = split_of(a.D, Vec16<T>::N, p.leaves);
    const int64_t n = tasks(a.split, on0 * p.leaves, on1 * p.leaves);
    hipLaunchKernelGGL(embed_leaf_kernel<T>, grid_of(n, a.split), dim3(256), 0, st, a);
  }
  if (p.nodes) {
    a.fsplit = split_of(a.Dp, 4, p.nodes);
    const int64_t n = tasks(a.fsplit, on0 * p.nodes, on1 * p.nodes);
    hipLaunchKernelGGL(embed_node_kernel, grid_of(n, a.fsplit), dim3(256), 0, st, a);
  }
  a.split = split_of(a.D, Vec16<T>::N, table[0] + table[1]);
  const int64_t n = tasks(a.split, table[0], table[1]);
  hipLaunchKernelGGL(embed_bwd_kernel<T>, grid_of(n, a.split), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace llattn

using namespace llattn;

extern "C" int32_t llattn_embed_fwd(const llattn_embed_cfg* c, const void* ids, const void* pos, const void* W, int64_t ldw,
                                    const void* Pos, int64_t ldp, void* out, void* stream) {
  if (const int32_t rc = check("llattn_embed_fwd", c, pos != nullptr)) return rc;
  if (c->rows == 0) return LLATTN_OK;
  const int64_t size = elem_size(c->dtype);
  if (!ids || !W || !out || (c->P && !Pos)) return fail(LLATTN_ERR_LAYOUT, "llattn_embed_fwd: null ids, table or output");
  if (!whole(ids, c->index_bytes) || !whole(pos, c->index_bytes) || !whole(W, size) || !whole(Pos, size) || !whole(out, size))
    return fail(LLATTN_ERR_LAYOUT, "llattn_embed_fwd: a tensor is not aligned to its elements");
  if (ldw < c->D || (c->P && ldp < c->D) || ldw > (int64_t)1 << 40 || ldp > (int64_t)1 << 40)
    return fail(LLATTN_ERR_LAYOUT, "llattn_embed_fwd: row strides %lld, %lld under D %d, or past 2^40", (long long)ldw, (long long)ldp, c->D);
  FwdArgs a{(int)c->rows, c->T, c->V, c->P, c->D, c->index_bytes, ids, c->P ? pos : nullptr, W, Pos, ldw, ldp, out, c->scale, {}};
  a.split = split_of(c->D, (int)(16 / size), c->rows);
  const dim3 grid = grid_of(c->rows * a.split.parts, a.split);
  if (c->dtype == LLATTN_F32) hipLaunchKernelGGL(embed_fwd_kernel<float>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
  else hipLaunchKernelGGL(embed_fwd_kernel<uint16_t>, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return check_launch("llattn_embed_fwd");
}

extern "C" size_t llattn_embed_bytes(const llattn_embed_cfg* c, int32_t has_pos) {
  if (check("llattn_embed_bytes", c, has_pos != 0) != LLATTN_OK) return 0;
  return plan_of(c, has_pos != 0).bytes();
}

extern "C" int32_t llattn_embed_bwd(const llattn_embed_cfg* c, const void* ids, const void* pos, const void* dout, void* dW,
                                    void* dPos, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int32_t rc = check("llattn_embed_bwd", c, pos != nullptr)) return rc;
  if (dPos && !c->P) return fail(LLATTN_ERR_SHAPE, "llattn_embed_bwd: a gradient of no position rows");
  if (!dW && !dPos) return LLATTN_OK;
  const int64_t size = elem_size(c->dtype);
  if (c->rows && (!ids || !dout)) return fail(LLATTN_ERR_LAYOUT, "llattn_embed_bwd: null ids or gradient");
  if (!whole(ids, c->index_bytes) || !whole(pos, c->index_bytes) || !whole(dout, size) || !whole(dW, size) || !whole(dPos, size))
    return fail(LLATTN_ERR_LAYOUT, "llattn_embed_bwd: a tensor is not aligned to its elements");
  const Plan p = plan_of(c, pos != nullptr);
  if (!workspace || workspace_bytes < p.bytes() || !aligned16(workspace))
    return fail(LLATTN_ERR_WORKSPACE, "llattn_embed_bwd: needs %zu workspace bytes (got %zu)", p.bytes(), workspace_bytes);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  char* at = static_cast<char*>(workspace);
  const auto take = [&](size_t n) { char* x = at; at += up(n); return x; };
  const size_t r = (size_t)c->rows;
  SortArgs s{};
  s.rows = (int)c->rows;
  s.counted = reinterpret_cast<int32_t*>(take(256));
  const auto sorted = [&](Keys& k, const void* keys, int R, int64_t padding) {
    k.keys = keys; k.index_bytes = c->index_bytes; k.R = R; k.padding = padding; k.buckets = buckets_of(R);
    k.order = reinterpret_cast<int32_t*>(take(4 * r));
    k.runs = reinterpret_cast<int2*>(take(8 * (size_t)R));
    k.list = reinterpret_cast<int2*>(take(8 * r));
  };
  sorted(s.set[0], ids, c->V, c->padding);
  if (c->P && pos) sorted(s.set[1], pos, c->P, -1);
  else if (c->P) { s.set[1].T = c->T; s.set[1].alike = (int)(c->rows / c->T); }
  BwdArgs a{};
  a.rows = s.rows; a.D = c->D; a.Dp = p.Dp; a.dout = dout;
  for (int k = 0; k < p.trees; ++k) {
    a.leaf[k] = reinterpret_cast<float*>(take((size_t)p.leaves * p.Dp * 4));
    a.node[k] = reinterpret_cast<float*>(take((size_t)p.nodes * p.Dp * 4));
  }
  s.first[1] = dW ? s.set[0].buckets : 0;
  s.first[2] = s.first[1] + (dPos && pos ? s.set[1].buckets : 0);
  if (s.first[2]) hipLaunchKernelGGL(embed_sort_kernel, dim3(s.first[2]), dim3(64 * kWaves), 0, st, s);
  a.set[0] = s.set[0]; a.set[1] = s.set[1];
  a.counted = s.counted;
  a.out[0] = dW; a.out[1] = dPos;
  a.scale[0] = c->scale; a.scale[1] = 1.f;
  const int64_t table[2] = {dW ? c->V : 0, dPos ? c->P : 0};
  if (c->dtype == LLATTN_F32) launch_bwd<float>(a, p, table, st);
  else launch_bwd<uint16_t>(a, p, table, st);
  return check_launch("llattn_embed_bwd");
}
