// Token rows, scaled, plus position rows, and the gradients of both tables (include/llattn_lm.h).
//
//   out[n] = s W[id_n] + Pos[pos_n],   dW[v] = s sum_{id_n = v} dout[n],   dPos[p] = sum_{pos_n = p} dout[n]
//
// The gradients are sums over the rows of one key (a token or a position), so the rows are ordered by key first.  That waits for no
// gradient, so a training pass does it behind the forward, where the chip is idle until the host has come to the backward (packed
// rows, 8192 x 1536: 143 us with it in the backward, 128; the sort was 19 us then, 12 now).  One launch, a workgroup for each residue class of keys
// (key mod buckets), which reads all keys, keeps its own in their order and counts them out by key.  The order of the keys among
// themselves is of no use here; the residues spread a text's frequent tokens, whose numbers are close, over the workgroups.  Where
// positions are n % T the order is known.
//
// A run (the rows of one key, of length L) is summed in a tree of its own: blocks of 32 rows from its first row on, 32 of
// these blocks to one of 1024 rows, then the blocks of 1024, the blocks of 32 behind them and the rows behind those in
// order.  One launch adds the blocks of 32, one (from 1024 rows on) those of 1024, and the last one writes every row of the
// tables, zeros where a run is empty.  Nothing depends on where the run lies in the order, so neither atomics nor other tokens
// change a bit.  A block of 32 that starts within positions [32 c, 32 c + 32) of the order is the only one that does
// (it covers position 32 c + 31), which makes c its number.
//
// What bounds it: memory.  Forward: a table row read and a row written per token; backward: dout read once for each
// table, the tables' gradients written whole.  us in training passes of 32768 rows x 1408 fp32, 32000 tokens, 2048 positions: forward
// 57 (250 MB), order 20 (latency: half of it the reading of the keys by 256 workgroups), sums of 32 rows 20, of 1024 5, the tables
// 68 (380 MB); a copy runs at 5.0 TB/s.  Few tokens take none but the last of these launches (embed_scan_kernel).
#include <algorithm>
#include <cmath>

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

// What each of a sorting workgroup's waves takes of n entries, in whole steps of 64.  n is anything below 2^31: unsigned, for the
// sum of n and the waves, the waves' ends and the steps past the last entry go beyond that.
__host__ __device__ constexpr uint32_t share_of(uint32_t n) { return ((n + kWaves - 1) / kWaves + 63) / 64 * 64; }
static_assert(share_of(0x7fffffff) == 1u << 27 && share_of(0x7ffffff0) == 1u << 27 && share_of(0) == 0 && share_of(1) == 64,
              "the waves' shares of the most rows");

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_f __attribute__((aligned(4)));
typedef u32x4 u32x4_h __attribute__((aligned(2)));

// Pieces of a lane, all held at the same time (1 and 4 were no quicker, rows of 5632 bytes)
constexpr int kTurns = 2;

// 16 bytes of a row at any alignment of whole elements; `left` elements remain in the row.  RAGGED: rows of not a whole
// number of pieces
template <typename T, bool RAGGED>
__device__ __forceinline__ u32x4 load_piece(const T* p, int left) {
  constexpr int N = Vec16<T>::N;
  if (!RAGGED || left >= N) {
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
// Non-temporal: what is written does not push out of the caches what is read (the tables' rows, dout: in training passes of 32768 x
// 1408 the forward took 71 us otherwise against 57, the last launch backward 137 against 83; a norm that reads the rows right
// behind takes as long either way, within 2%).
template <typename T, bool RAGGED>
__device__ __forceinline__ void store_piece(T* p, u32x4 v, int left) {
  constexpr int N = Vec16<T>::N;
  if (!RAGGED || left >= N) {
    if constexpr (N == 4) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_f*>(p));
    else __builtin_nontemporal_store(v, reinterpret_cast<u32x4_h*>(p));
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

// A row's 16-byte pieces are shared by 2^shift lanes (8 to 64) of a wave, in `parts` tasks of `per` pieces each, up to kTurns a
// lane.  A workgroup takes one part of 256 / 2^shift rows; workgroups of neighbouring parts follow one another, all those of one
// set of rows (`blocks`) before the next set's.  (Divisions by workgroup, in scalar registers: by thread they took longer than the
// memory.)
struct Split { int pieces, shift, parts, per; };
struct Task { int row, from, to, lane, width; };
__device__ __forceinline__ int64_t block_of() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
__device__ __forceinline__ Task task_of(const Split& s, int64_t block) {
  const uint32_t group = (uint32_t)block / (uint32_t)s.parts, part = (uint32_t)block - group * s.parts;
  const int lw = s.shift, from = (int)part * s.per;
  return Task{(int)((group << (8 - lw)) + (threadIdx.x >> lw)), from, min(from + s.per, s.pieces), (int)threadIdx.x & ((1 << lw) - 1), 1 << lw};
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

template <typename T, bool RAGGED>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const FwdArgs a) {
  constexpr int N = Vec16<T>::N;
  const Task k = task_of(a.split, block_of());
  if ((uint32_t)k.row >= (uint32_t)a.rows) return;
  const int64_t id = index_at(a.ids, a.index_bytes, k.row);
  const int64_t p = a.P ? a.pos ? index_at(a.pos, a.index_bytes, k.row) : (uint32_t)k.row % (uint32_t)a.T : 0;
  const bool ok = id >= 0 && id < a.V && (!a.P || (p >= 0 && p < a.P));
  const T* w = static_cast<const T*>(a.W) + (ok ? id : 0) * a.ldw;
  const T* q = static_cast<const T*>(a.Pos) + (ok ? p : 0) * a.ldp;
  T* o = static_cast<T*>(a.out) + (int64_t)k.row * a.D;
  u32x4 x[kTurns], y[kTurns];  // every load before the first store
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int c = k.from + k.lane + u * k.width, d = c * N;
    if (c < k.to) {
      x[u] = load_piece<T, RAGGED>(w + d, a.D - d);
      if (a.P) y[u] = load_piece<T, RAGGED>(q + d, a.D - d);
    }
  }
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int c = k.from + k.lane + u * k.width, d = c * N;
    if (c >= k.to) continue;
    float f[N], g[N];
    unpack<T>(x[u], f);
    unpack<T>(y[u], g);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      f[e] = a.P ? fmaf(a.scale, f[e], g[e]) : a.scale * f[e];
      if (!ok) f[e] = __builtin_nanf("");
    }
    store_piece<T, RAGGED>(o + d, pack<T>(f), a.D - d);
  }
}

// Rows by key.  order: rows, the runs of a bucket one after another; runs: first and one past the last position of each key's run.
struct Keys {
  const void* keys;       // null: row n has key n % T, and nothing is written (runs of `alike` rows)
  int index_bytes;
  int T, alike;
  int R;                  // keys outside [0, R) and `padding` have no run
  int64_t padding;
  int buckets, per;       // buckets: a power of two, of `per` keys at most (R <= per buckets, per <= kKeys)
  int32_t* order;
  int2* runs;             // by bucket, then by key
  int2* list;             // scratch [rows]
};
// The run of a key, and the row that stands j-th in it
__device__ __forceinline__ int2 run_of(const Keys& s, int key) {
  if (s.keys) return s.runs[(key & (s.buckets - 1)) * s.per + (key >> (31 - __builtin_clz(s.buckets)))];
  return key < s.T ? make_int2(key * s.alike, (key + 1) * s.alike) : make_int2(0, 0);
}
__device__ __forceinline__ int row_at(const Keys& s, int2 run, int key, int j) { return s.keys ? s.order[run.x + j] : j * s.T + key; }
__device__ __forceinline__ int key_at(const Keys& s, int i) {  // of position i < the number of rows that have runs
  return s.keys ? (int)index_at(s.keys, s.index_bytes, s.order[i]) : i / s.alike;
}

struct SortArgs {
  Keys set[2];
  int first[3];  // workgroups of each set
  int rows;
  int32_t* counted;  // rows that have runs, of each set
};

// The keys of a workgroup's waves, 64 at a time, stay in registers between the counting and the collecting where they are no
// more than STEPS times 64 a wave (16384 rows, 32768 rows); others are read again.  With 16 steps in 64 registers, two workgroups on a CU:
// those of both sets at a time.  (8192 rows in two sets 12.0 us, 14.8 with 32 steps, 19.4 with those in 76 registers; 32768 rows 25.4 with
// 16 steps, 20.4 with 32.  In 64 registers these spill, and a launch with scratch memory slows its neighbours: forward 58 -> 61 us, the
// tables' gradients 68 -> 72.)
template <int STEPS>
__global__ __launch_bounds__(64 * kWaves, STEPS <= 16 ? 8 : 4) void embed_sort_kernel(const SortArgs a) {
  __shared__ int2 list[kList];
  __shared__ int count[kWaves][kKeys];
  __shared__ int eq_of[kWaves], lt_of[kWaves], all_of[kWaves], sums[kKeys / 64];
  const int which = (int)blockIdx.x >= a.first[1];
  const Keys& s = a.set[which];
  const int b = blockIdx.x - a.first[which], mask = s.buckets - 1, shift = 31 - __builtin_clz(s.buckets);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t seg = share_of(a.rows);
  const int64_t lo = min((int64_t)a.rows, w * seg), hi = min((int64_t)a.rows, lo + seg);
  constexpr uint32_t kNone = 0xffffffffu;
  const uint32_t padding = s.padding < 0 ? kNone : (uint32_t)s.padding;
  uint32_t key[STEPS];
  const auto read = [&](int64_t n0) {  // the keys n0 + 64 u + lane; kNone: none that has a run
#pragma unroll
    for (int u0 = 0; u0 < STEPS; u0 += 8) {
      if (n0 + 64 * u0 >= hi) {
#pragma unroll
        for (int u = 0; u < 8; ++u) key[u0 + u] = kNone;
        continue;
      }
      uint2 raw[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int64_t n = n0 + 64 * (u0 + u) + lane;
        raw[u] = make_uint2(kNone, 0);
        if (n < hi) {
          if (s.index_bytes == 8) raw[u] = static_cast<const uint2*>(s.keys)[n];
          else raw[u].x = static_cast<const uint32_t*>(s.keys)[n];
        }
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
        key[u0 + u] = raw[u].y == 0 && raw[u].x < (uint32_t)s.R && raw[u].x != padding ? raw[u].x : kNone;
    }
  };
  // a key's residue class; past every one for none (keys are below 2^31)
  const auto bucket = [&](uint32_t k) { return k & ((uint32_t)mask | 0x80000000u); };
  int eq = 0, lt = 0, all = 0;
  for (int64_t n = lo; n < hi; n += 64 * STEPS) {
    read(n);
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
      if (n + 64 * u >= hi) continue;
      const uint32_t k = bucket(key[u]);
      eq += __popcll(__ballot(k == (uint32_t)b));
      lt += __popcll(__ballot(k < (uint32_t)b));
      // by the key: a residue class of none is not kNone.  Positions of the order past these rows are never written
      if (b == 0) all += __popcll(__ballot(key[u] != kNone));
    }
  }
  if (lane == 0) {
    eq_of[w] = eq;
    lt_of[w] = lt;
    all_of[w] = all;
  }
  for (int i = lane; i < s.per; i += 64) count[w][i] = 0;
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
    for (int64_t n = lo; n < hi; n += 64 * STEPS) {
      if (seg > 64 * STEPS) read(n);
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        const bool mine = bucket(key[u]) == (uint32_t)b;
        const uint64_t m = __ballot(mine);
        if (!m) continue;
        if (mine) kept[at + __popcll(m & ((1ull << lane) - 1))] = make_int2((int)(n + 64 * u + lane), (int)(key[u] >> shift));
        at += __popcll(m);
      }
    }
  }
  __syncthreads();
  // counted out by key: each wave counts a stretch of the list, the counts are added up by key and, within a key, by wave
  const uint32_t listed = n_list, step = share_of(listed), from = min(listed, w * step), to = min(listed, from + step);
  for (uint32_t i = from + lane; i < to; i += 64) atomicAdd(&count[w][kept[i].y], 1);
  __syncthreads();
  const int k = threadIdx.x;
  if (w * 64 < s.per) {
    int c[kWaves], mine = 0;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      c[v] = mine;
      mine += k < s.per ? count[v][k] : 0;
    }
    int before = mine;  // inclusive scan over the 64 keys of this wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(before, o);
      if (lane >= o) before += x;
    }
    if (lane == 63) sums[w] = before;
    lt = before - mine;
    eq = mine;
    if (k < s.per) {
#pragma unroll
      for (int v = 0; v < kWaves; ++v) count[v][k] = lt + c[v];
    }
  }
  __syncthreads();
  if (k < s.per) {
    int more = 0;  // the keys of the waves before
    for (int v = 0; v < w; ++v) more += sums[v];
    if (more) {
#pragma unroll
      for (int v = 0; v < kWaves; ++v) count[v][k] += more;
    }
    const int first = base + more + lt;
    s.runs[b * s.per + k] = eq ? make_int2(first, first + eq) : make_int2(0, 0);
  }
  __syncthreads();
  for (uint32_t i = from; i < to; i += 64) {
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
  int64_t blocks, total;   // workgroups of the first set, and of both
  int n_rows[2];           // rows of this launch's results, of each set
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

// The pieces of one lane of a row of sums
template <typename T>
struct Sum {
  static constexpr int N = Vec16<T>::N;
  float v[kTurns][N];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int u = 0; u < kTurns; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) v[u][e] = 0.f;
  }
  __device__ __forceinline__ void add(const Sum& x) {
#pragma unroll
    for (int u = 0; u < kTurns; ++u)
#pragma unroll
      for (int e = 0; e < N; ++e) v[u][e] += x.v[u][e];
  }
};

// sum += the rows of T that start at get(i), i < n, in order, U at a time
template <typename T, bool RAGGED, int U, typename F>
__device__ __forceinline__ void add_rows(Sum<T>& sum, int n, const Task& k, int D, F&& get) {
  constexpr int N = Vec16<T>::N;
  for (int i = 0; i < n; i += U) {
    u32x4 v[U][kTurns];
#pragma unroll
    for (int q = 0; q < U; ++q) {
      const T* p = i + q < n ? get(i + q) : nullptr;
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        const int c = k.from + k.lane + u * k.width;
        v[q][u] = u32x4{0, 0, 0, 0};
        if (p && c < k.to) v[q][u] = load_piece<T, RAGGED>(p + c * N, D - c * N);
      }
    }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (i + q >= n) break;
#pragma unroll
      for (int u = 0; u < kTurns; ++u) {
        float x[N];
        unpack<T>(v[q][u], x);
#pragma unroll
        for (int e = 0; e < N; ++e) sum.v[u][e] += x[e];
      }
    }
  }
}

// sum += the rows of fp32 sums that start at get(i), i < n, in order
template <typename T, typename F>
__device__ __forceinline__ void add_sums(Sum<T>& sum, int n, const Task& k, F&& get) {
  constexpr int N = Vec16<T>::N, U = 2;
  for (int i = 0; i < n; i += U) {
    float4 v[U][kTurns][N / 4];
#pragma unroll
    for (int q = 0; q < U; ++q)
#pragma unroll
      for (int u = 0; u < kTurns; ++u)
#pragma unroll
        for (int e = 0; e < N / 4; ++e) {
          const int c = k.from + k.lane + u * k.width;
          v[q][u][e] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (i + q < n && c < k.to) v[q][u][e] = *reinterpret_cast<const float4*>(get(i + q) + c * N + 4 * e);
        }
#pragma unroll
    for (int q = 0; q < U; ++q) {
      if (i + q >= n) break;
#pragma unroll
      for (int u = 0; u < kTurns; ++u)
#pragma unroll
        for (int e = 0; e < N / 4; ++e) {
          sum.v[u][4 * e] += v[q][u][e].x;
          sum.v[u][4 * e + 1] += v[q][u][e].y;
          sum.v[u][4 * e + 2] += v[q][u][e].z;
          sum.v[u][4 * e + 3] += v[q][u][e].w;
        }
    }
  }
}

// The block of `size` positions that starts in [c size, (c + 1) size): its run and key, and where in the run it starts (-1: there
// is none)
struct Block { int2 run; int key, at; };
__device__ __forceinline__ Block block_at(const Keys& s, int counted, int c, int size) {
  const int64_t last = (int64_t)c * size + size - 1;
  if (last >= counted) return Block{make_int2(0, 0), 0, -1};
  const int key = key_at(s, (int)last);
  // the keys lie in the caller's memory: one written to since the rows were ordered changes sums, and reads nothing outside
  if (s.keys && (uint32_t)key >= (uint32_t)s.R) return Block{make_int2(0, 0), 0, -1};
  const int2 run = run_of(s, key);
  const int at = ((int)last - run.x) / size * size;
  return Block{run, key, at + size <= run.y - run.x ? at : -1};
}

// This workgroup's set and task
__device__ __forceinline__ Task task_in(const BwdArgs& a, const Split& split, int& set) {
  int64_t b = block_of();
  set = b >= a.blocks;
  if (set) b -= a.blocks;
  Task k = task_of(split, b);
  if ((uint32_t)k.row >= (uint32_t)a.n_rows[set]) k.row = -1;
  return k;
}

template <typename T>
__device__ __forceinline__ void store_sums(float* o, const Sum<T>& x, const Task& k) {
  constexpr int N = Vec16<T>::N;
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int c = k.from + k.lane + u * k.width;
    if (c >= k.to) continue;
#pragma unroll
    for (int e = 0; e < N; e += 4)
      *reinterpret_cast<float4*>(o + c * N + e) = make_float4(x.v[u][e], x.v[u][e + 1], x.v[u][e + 2], x.v[u][e + 3]);
  }
}

template <typename T, bool RAGGED>
__global__ __launch_bounds__(256) void embed_leaf_kernel(const BwdArgs a) {
  int set;
  const Task k = task_in(a, a.split, set);
  if (k.row < 0 || block_of() >= a.total) return;
  const Keys& s = a.set[set];
  const Block b = block_at(s, s.keys ? a.counted[set] : a.rows, k.row, kLeaf);
  if (b.at < 0) return;
  Sum<T> sum;
  sum.zero();
  // 8 rows ahead (32768 x 1408: 20.6 us; 4 21.2, 16 31.6, with fewer waves)
  add_rows<T, RAGGED, 8>(sum, kLeaf, k, a.D,
                         [&](int i) { return static_cast<const T*>(a.dout) + (int64_t)row_at(s, b.run, b.key, b.at + i) * a.D; });
  store_sums(a.leaf[set] + (int64_t)k.row * a.Dp, sum, k);
}

__global__ __launch_bounds__(256) void embed_node_kernel(const BwdArgs a) {
  int set;
  const Task k = task_in(a, a.fsplit, set);
  if (k.row < 0 || block_of() >= a.total) return;
  const Keys& s = a.set[set];
  const Block b = block_at(s, s.keys ? a.counted[set] : a.rows, k.row, kLeaf * kLeaf);
  if (b.at < 0) return;
  const float* const leaf = a.leaf[set] + (int64_t)((b.run.x + b.at) / kLeaf) * a.Dp;
  float* const o = a.node[set] + (int64_t)k.row * a.Dp;
  for (int c = k.from + k.lane; c < k.to; c += k.width) {
    float4 v[kLeaf];
#pragma unroll
    for (int i = 0; i < kLeaf; ++i) v[i] = *reinterpret_cast<const float4*>(leaf + (int64_t)i * a.Dp + 4 * c);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kLeaf; ++i) x = make_float4(x.x + v[i].x, x.y + v[i].y, x.z + v[i].z, x.w + v[i].w);
    *reinterpret_cast<float4*>(o + 4 * c) = x;
  }
}

template <typename T, bool RAGGED>
__device__ __forceinline__ void store_row(const BwdArgs& a, int set, const Task& k, const Sum<T>& sum) {
  constexpr int N = Vec16<T>::N;
  T* const o = static_cast<T*>(a.out[set]) + (int64_t)k.row * a.D;
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int c = k.from + k.lane + u * k.width;
    if (c >= k.to) continue;
    float x[N];
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = sum.v[u][e] * a.scale[set];
    store_piece<T, RAGGED>(o + c * N, pack<T>(x), a.D - c * N);
  }
}

// Rows of the tables' gradients, of a whole run each: the blocks of 1024, those of 32 behind them, the rows behind those.  Most runs are
// empty or short, so what counts is the number of waves at work and not what each has in flight: with 8 (bf16: 6) on a SIMD
// instead of 6 (4), two sums and two rows (bf16: four) ahead instead of four, 52305 rows x 1536 bf16 take 43 us for 49, 34048 x 1408
// fp32 68 for 71.  (One register of the bf16 form spills then, 11 where rows are ragged; 5 waves, without that, 46.)
template <typename T> constexpr bool kWide = std::is_same_v<T, float>;
template <typename T, bool RAGGED>
__global__ __launch_bounds__(256, kWide<T> ? 8 : 6) void embed_bwd_kernel(const BwdArgs a) {
  int set;
  const Task k = task_in(a, a.split, set);
  if (k.row < 0 || block_of() >= a.total) return;
  const Keys& s = a.set[set];
  const int2 run = run_of(s, k.row);
  const int L = run.y - run.x, nodes = L / (kLeaf * kLeaf), leaves = L / kLeaf - nodes * kLeaf, rest = L % kLeaf;
  Sum<T> sum;
  sum.zero();
  if (nodes) add_sums<T>(sum, nodes, k, [&](int i) { return a.node[set] + (int64_t)(run.x / (kLeaf * kLeaf) + i) * a.Dp; });
  if (leaves) {
    Sum<T> x;
    x.zero();
    const int leaf0 = (run.x + nodes * kLeaf * kLeaf) / kLeaf;
    add_sums<T>(x, leaves, k, [&](int i) { return a.leaf[set] + (int64_t)(leaf0 + i) * a.Dp; });
    sum.add(x);
  }
  if (rest) {
    Sum<T> x;
    x.zero();
    add_rows<T, RAGGED, kWide<T> ? 2 : 4>(x, rest, k, a.D,
                           [&](int i) { return static_cast<const T*>(a.dout) + (int64_t)row_at(s, run, k.row, L - rest + i) * a.D; });
    sum.add(x);
  }
  store_row<T, RAGGED>(a, set, k, sum);
}

// Few tokens: a wave for every row of the tables looks through the keys itself and adds up what it finds, in the same tree; no
// other launch and no workspace.
template <typename T, bool RAGGED>
__global__ __launch_bounds__(256) void embed_scan_kernel(const BwdArgs a) {
  constexpr int N = Vec16<T>::N, U = 8;
  int set;
  const Task k = task_in(a, a.split, set);
  if (k.row < 0 || block_of() >= a.total) return;
  const Keys& s = a.set[set];
  const int lane = k.lane;
  const int c = k.from + lane, d = c * N;
  const bool live = c < k.to;
  float rest[N] = {}, leaf[N] = {}, node[N] = {};
  int n = 0;
  const auto add = [&](const u32x4& v) {
    float x[N];
    unpack<T>(v, x);
#pragma unroll
    for (int e = 0; e < N; ++e) rest[e] += x[e];
    ++n;
    if (n % kLeaf == 0) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        leaf[e] += rest[e];
        rest[e] = 0.f;
      }
      if (n % (kLeaf * kLeaf) == 0) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          node[e] += leaf[e];
          leaf[e] = 0.f;
        }
      }
    }
  };
  const auto load = [&](int row) {
    u32x4 v = {0, 0, 0, 0};
    if (live) v = load_piece<T, RAGGED>(static_cast<const T*>(a.dout) + (int64_t)row * a.D + d, a.D - d);
    return v;
  };
  if (s.keys) {
    for (int n0 = 0; n0 < a.rows; n0 += 64) {
      const int i = n0 + lane;
      bool mine = false;
      if (i < a.rows) {
        const int64_t key = index_at(s.keys, s.index_bytes, i);
        mine = key == k.row && key != s.padding;
      }
      uint64_t m = __ballot(mine);
      while (m) {
        u32x4 v[U];
        int found = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (!m) break;
          v[u] = load(n0 + __builtin_ctzll(m));
          m &= m - 1;
          ++found;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u < found) add(v[u]);
      }
    }
  } else {
    const int2 run = run_of(s, k.row);
    for (int i = run.x; i < run.y; i += U) {
      u32x4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u < run.y) v[u] = load(row_at(s, run, k.row, i + u - run.x));
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + u < run.y) add(v[u]);
    }
  }
  if (!live) return;
#pragma unroll
  for (int e = 0; e < N; ++e) rest[e] = ((node[e] + leaf[e]) + rest[e]) * a.scale[set];
  store_piece<T, RAGGED>(static_cast<T*>(a.out[set]) + (int64_t)k.row * a.D + d, pack<T>(rest), a.D - d);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr size_t up(size_t n) { return (n + 255) & ~size_t(255); }

// Lanes and tasks of a row of D elements: up to kTurns pieces a lane, fewer where there are too few rows to fill the chip.
Split split_of(int D, int n, int64_t rows) {
  Split s;
  s.pieces = (int)ceil_div(D, n);
  s.shift = s.pieces > 32 ? 6 : s.pieces > 16 ? 5 : s.pieces > 8 ? 4 : 3;
  const int width = 1 << s.shift, turns = (int)ceil_div(s.pieces, width), most = rows * width >= 64 * 4096 ? kTurns : 1;
  s.parts = (int)ceil_div(turns, most);
  s.per = (int)ceil_div(turns, s.parts) * width;
  s.parts = (int)ceil_div(s.pieces, s.per);
  return s;
}

// Workgroups of `rows` rows; their grid (a launch holds fewer than 2^32 threads in a dimension)
int64_t blocks_of(const Split& s, int64_t rows) { return ceil_div(rows, 256 >> s.shift) * s.parts; }
dim3 grid_of(int64_t blocks) {
  const int64_t x = std::min<int64_t>(blocks, 1 << 20);
  return dim3((unsigned)x, (unsigned)ceil_div(blocks, x));
}

int32_t check(const char* who, const llattn_embed_cfg* c, bool has_pos) {
  if (!c) return fail(LLATTN_ERR_SHAPE, "%s: null configuration", who);
  if (c->rows < 0 || c->rows > 0x7fffffff || c->V <= 0 || c->V > kMostRows || c->P < 0 || c->P > kMostRows || c->D <= 0 || c->D > 1 << 20)
    return fail(LLATTN_ERR_SHAPE, "%s: rows %lld (below 2^31), V %d, P %d (at most 2^22), D %d", who, (long long)c->rows, c->V, c->P, c->D);
  if (c->P && !has_pos && (c->T <= 0 || c->T > c->P || c->rows % c->T))
    return fail(LLATTN_ERR_SHAPE, "%s: T %d must be in [1, P %d] and divide the rows (%lld)", who, c->T, c->P, (long long)c->rows);
  if (c->dtype != LLATTN_F32 && c->dtype != LLATTN_BF16) return fail(LLATTN_ERR_DTYPE, "%s: unknown dtype %d", who, c->dtype);
  if (c->index_bytes != 4 && c->index_bytes != 8) return fail(LLATTN_ERR_DTYPE, "%s: indices of %d bytes", who, c->index_bytes);
  if (!std::isfinite(c->scale)) return fail(LLATTN_ERR_SHAPE, "%s: scale %g is not finite", who, (double)c->scale);
  if (c->padding < -1 || c->padding >= c->V) return fail(LLATTN_ERR_SHAPE, "%s: padding %lld outside [-1, V)", who, (long long)c->padding);
  return LLATTN_OK;
}

bool whole(const void* p, int64_t size) { return (reinterpret_cast<uintptr_t>(p) & (size - 1)) == 0; }

int buckets_of(int R) {
  int b = 256;  // a workgroup for every CU
  while ((int64_t)b * kKeys < R) b *= 2;
  return b;
}

// Few tokens: pieces shared by whole waves, one a lane
Split scan_split(int D, int n) {
  Split s;
  s.pieces = (int)ceil_div(D, n);
  s.shift = 6;
  s.per = 64;
  s.parts = (int)ceil_div(s.pieces, 64);
  return s;
}
// What the scan takes grows with the keys that its waves read, (V + P) ceil(D / 256) rows.  us in a graph, lookup and gradients, by the scan
// and by the order, at 2^20 of them 7.8 and 16.0, at 2^21.6 9.1 and 18.3, 2^23.3 11.4 and 20.0, 2^24.1 16.9 and 18.1, 2^24.6 44.5 and 45.0
bool scans(const llattn_embed_cfg* c) {
  return c->rows <= 1024 && ((int64_t)c->V + c->P) * ceil_div(c->D, 256) * c->rows <= 1 << 24;
}

// What a backward reads besides dout (the order): counted; for each sorted set the rows in order, the runs and the list.  Its
// workspace: for each table the sums of 32 and of 1024 rows.
struct Plan {
  int64_t leaves, nodes;
  int Dp;
  size_t order, trees;  // bytes; 1: none needed
};
Plan plan_of(const llattn_embed_cfg* c, bool has_pos) {
  Plan p{};
  p.order = p.trees = 1;
  if (scans(c)) return p;
  p.leaves = c->rows / kLeaf;
  p.nodes = c->rows / (kLeaf * kLeaf);
  p.Dp = (c->D + 7) / 8 * 8;
  const auto sorted = [&](int R) {
    const size_t b = buckets_of(R);
    return up((size_t)c->rows * 4) + up(b * ceil_div(R, b) * 8) + up((size_t)c->rows * 8);
  };
  p.order = 256 + sorted(c->V) + (c->P && has_pos ? sorted(c->P) : 0);
  p.trees = std::max<size_t>((c->P ? 2 : 1) * (up((size_t)p.leaves * p.Dp * 4) + up((size_t)p.nodes * p.Dp * 4)), 1);
  return p;
}
// The sets of tokens and of positions, and where in the order they lie (it is null: nowhere)
SortArgs sets_of(const llattn_embed_cfg* c, const void* ids, const void* pos, void* order) {
  SortArgs s{};
  s.rows = (int)c->rows;
  char* at = static_cast<char*>(order);
  const auto take = [&](size_t n) { char* x = at; at += up(n); return x; };
  if (order) s.counted = reinterpret_cast<int32_t*>(take(256));
  const size_t r = (size_t)c->rows;
  const auto keyed = [&](Keys& k, const void* keys, int R, int64_t padding) {
    k.keys = keys; k.index_bytes = c->index_bytes; k.R = R; k.padding = padding; k.buckets = buckets_of(R); k.per = (int)ceil_div(R, k.buckets);
    if (!order) return;
    k.order = reinterpret_cast<int32_t*>(take(4 * r));
    k.runs = reinterpret_cast<int2*>(take(8 * (size_t)k.per * k.buckets));
    k.list = reinterpret_cast<int2*>(take(8 * r));
  };
  keyed(s.set[0], ids, c->V, c->padding);
  if (c->P && pos) keyed(s.set[1], pos, c->P, -1);
  else if (c->P) { s.set[1].T = c->T; s.set[1].alike = (int)(c->rows / c->T); }
  return s;
}

// The workgroups of n0 rows of one set and n1 of the other
dim3 blocks_for(BwdArgs& a, const Split& s, int64_t n0, int64_t n1) {
  a.blocks = blocks_of(s, n0);
  a.total = a.blocks + blocks_of(s, n1);
  a.n_rows[0] = (int)n0;
  a.n_rows[1] = (int)n1;
  return grid_of(a.total);
}

template <typename T, bool RAGGED>
void launch_bwd(BwdArgs& a, const Plan& p, const int64_t (&table)[2], hipStream_t st) {
  const int64_t on0 = table[0] > 0, on1 = table[1] > 0;
  if (p.leaves) {
    a.split = split_of(a.D, Vec16<T>::N, p.leaves);
    hipLaunchKernelGGL((embed_leaf_kernel<T, RAGGED>), blocks_for(a, a.split, on0 * p.leaves, on1 * p.leaves), dim3(256), 0, st, a);
  }
  if (p.nodes) {
    a.fsplit = split_of(a.Dp, 4, p.nodes);
    hipLaunchKernelGGL(embed_node_kernel, blocks_for(a, a.fsplit, on0 * p.nodes, on1 * p.nodes), dim3(256), 0, st, a);
  }
  a.split = split_of(a.D, Vec16<T>::N, table[0] + table[1]);
  hipLaunchKernelGGL((embed_bwd_kernel<T, RAGGED>), blocks_for(a, a.split, table[0], table[1]), dim3(256), 0, st, a);
}
template <typename T, bool RAGGED>
void launch_scan(BwdArgs& a, const int64_t (&table)[2], hipStream_t st) {
  a.split = scan_split(a.D, Vec16<T>::N);
  hipLaunchKernelGGL((embed_scan_kernel<T, RAGGED>), blocks_for(a, a.split, table[0], table[1]), dim3(256), 0, st, a);
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
  const dim3 grid = grid_of(blocks_of(a.split, c->rows));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const bool ragged = c->D % (16 / size) != 0;
  if (c->dtype == LLATTN_F32 && ragged) hipLaunchKernelGGL((embed_fwd_kernel<float, true>), grid, dim3(256), 0, st, a);
  else if (c->dtype == LLATTN_F32) hipLaunchKernelGGL((embed_fwd_kernel<float, false>), grid, dim3(256), 0, st, a);
  else if (ragged) hipLaunchKernelGGL((embed_fwd_kernel<uint16_t, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((embed_fwd_kernel<uint16_t, false>), grid, dim3(256), 0, st, a);
  return check_launch("llattn_embed_fwd");
}

extern "C" size_t llattn_embed_bytes(const llattn_embed_cfg* c, int32_t has_pos, int32_t which) {
  if (check("llattn_embed_bytes", c, has_pos != 0) != LLATTN_OK) return 0;
  if (which != LLATTN_EMBED_ORDER && which != LLATTN_EMBED_BACKWARD) {
    fail(LLATTN_ERR_SHAPE, "llattn_embed_bytes: unknown buffer %d", which);
    return 0;
  }
  const Plan p = plan_of(c, has_pos != 0);
  return which == LLATTN_EMBED_ORDER ? p.order : p.trees;
}

extern "C" int32_t llattn_embed_order(const llattn_embed_cfg* c, const void* ids, const void* pos, int32_t tokens, int32_t positions,
                                      void* order, size_t order_bytes, void* stream) {
  if (const int32_t rc = check("llattn_embed_order", c, pos != nullptr)) return rc;
  if ((c->rows && tokens && !ids) || (positions && c->P && !pos)) return fail(LLATTN_ERR_LAYOUT, "llattn_embed_order: null ids or positions");
  if (!whole(ids, c->index_bytes) || !whole(pos, c->index_bytes))
    return fail(LLATTN_ERR_LAYOUT, "llattn_embed_order: a tensor is not aligned to its elements");
  const Plan p = plan_of(c, pos != nullptr);
  if (p.order == 1) return LLATTN_OK;
  if (!order || order_bytes < p.order || !aligned16(order))
    return fail(LLATTN_ERR_WORKSPACE, "llattn_embed_order: needs %zu bytes (got %zu)", p.order, order_bytes);
  SortArgs s = sets_of(c, ids, pos, order);
  s.first[1] = tokens ? s.set[0].buckets : 0;
  s.first[2] = s.first[1] + (positions && c->P ? s.set[1].buckets : 0);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (s.first[2] && c->rows <= 16 * 64 * kWaves) hipLaunchKernelGGL(embed_sort_kernel<16>, dim3(s.first[2]), dim3(64 * kWaves), 0, st, s);
  else if (s.first[2]) hipLaunchKernelGGL(embed_sort_kernel<32>, dim3(s.first[2]), dim3(64 * kWaves), 0, st, s);
  return check_launch("llattn_embed_order");
}

extern "C" int32_t llattn_embed_bwd(const llattn_embed_cfg* c, const void* ids, const void* pos, const void* order, const void* dout,
                                    void* dW, void* dPos, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int32_t rc = check("llattn_embed_bwd", c, pos != nullptr)) return rc;
  if (dPos && !c->P) return fail(LLATTN_ERR_SHAPE, "llattn_embed_bwd: a gradient of no position rows");
  if (!dW && !dPos) return LLATTN_OK;
  const int64_t size = elem_size(c->dtype);
  if (c->rows && (!ids || !dout)) return fail(LLATTN_ERR_LAYOUT, "llattn_embed_bwd: null ids or gradient");
  if (!whole(ids, c->index_bytes) || !whole(pos, c->index_bytes) || !whole(dout, size) || !whole(dW, size) || !whole(dPos, size))
    return fail(LLATTN_ERR_LAYOUT, "llattn_embed_bwd: a tensor is not aligned to its elements");
  const Plan p = plan_of(c, pos != nullptr);
  if (p.order > 1 && (dW || pos) && (!order || !aligned16(order)))
    return fail(LLATTN_ERR_LAYOUT, "llattn_embed_bwd: null order, or one not 16-byte aligned");
  if (p.trees > 1 && (!workspace || workspace_bytes < p.trees || !aligned16(workspace)))
    return fail(LLATTN_ERR_WORKSPACE, "llattn_embed_bwd: needs %zu workspace bytes (got %zu)", p.trees, workspace_bytes);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t table[2] = {dW ? c->V : 0, dPos ? c->P : 0};
  const bool f32 = c->dtype == LLATTN_F32, ragged = c->D % (16 / size) != 0;
  const SortArgs s = sets_of(c, ids, pos, p.order > 1 ? const_cast<void*>(order) : nullptr);
  BwdArgs a{};
  a.set[0] = s.set[0]; a.set[1] = s.set[1];
  a.rows = s.rows; a.D = c->D; a.Dp = p.Dp; a.dout = dout;
  a.counted = s.counted;
  a.out[0] = dW; a.out[1] = dPos;
  a.scale[0] = c->scale; a.scale[1] = 1.f;
  if (p.order == 1) {
    if (f32 && ragged) launch_scan<float, true>(a, table, st);
    else if (f32) launch_scan<float, false>(a, table, st);
    else if (ragged) launch_scan<uint16_t, true>(a, table, st);
    else launch_scan<uint16_t, false>(a, table, st);
    return check_launch("llattn_embed_bwd");
  }
  char* at = static_cast<char*>(workspace);
  for (int k = 0; k < (c->P ? 2 : 1); ++k) {
    a.leaf[k] = reinterpret_cast<float*>(at);
    at += up((size_t)p.leaves * p.Dp * 4);
    a.node[k] = reinterpret_cast<float*>(at);
    at += up((size_t)p.nodes * p.Dp * 4);
  }
  if (f32 && ragged) launch_bwd<float, true>(a, p, table, st);
  else if (f32) launch_bwd<float, false>(a, p, table, st);
  else if (ragged) launch_bwd<uint16_t, true>(a, p, table, st);
  else launch_bwd<uint16_t, false>(a, p, table, st);
  return check_launch("llattn_embed_bwd");
}
