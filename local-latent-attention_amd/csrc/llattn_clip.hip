// The norm over a list of gradients, and the gradients scaled to a largest norm (include/llattn_lm.h).
//
//   norm = sqrt(sum g^2),   c = min(1, max_norm / (norm + 1e-6)),   out = c g
//
// Squares, sums and products in 64 bits: a square of an fp32 value neither overflows nor vanishes there, and 64-bit
// arithmetic at the rate that memory delivers elements is a twentieth of what the chip has.  One launch per 128 tensors sums
// squares, a workgroup over its share of all tensors' chunks; the scaling launch adds the workgroups' sums up again
// in every workgroup, in one order, so that no launch stands between them.
//
// What bounds it: memory.  Gradients are read twice (a norm has to be known before anything is scaled) and written once, past the
// caches (non-temporal), which are left to what the norm has read last.  The 540 M fp32 gradients of the 0.55b model: squares
// 0.36 ms (6.0 TB/s), scaling 0.85 ms (5.1 TB/s; a copy 5.0).  Eight loads ahead instead of four took 7% off the squares; chunks of
// 65536, 1024 to 4096 workgroups and one workgroup a chunk were no quicker (the last 50% slower, as each adds up the parts).
#include <algorithm>
#include <new>
#include <vector>

#include "llattn_abi.h"
#include "llattn_device.h"
#include "llattn_lm.h"

namespace llattn {
namespace {

constexpr int kGroup = 128;        // tensors of a launch: their table travels in the kernel's arguments
constexpr int kChunk = 16384;      // elements of a chunk; a workgroup takes chunk after chunk
constexpr int kWgs = 2048;       // 8 workgroups of 256 on each of 256 CUs
constexpr int kAhead = 8;          // 16-byte loads a thread has in flight
constexpr double kEps = 1e-6;

struct Table {
  const void* g[kGroup];
  void* out[kGroup];
  int64_t numel[kGroup];
  int32_t first[kGroup + 1];       // first chunk of each tensor, and their number
  uint8_t bf16[kGroup];
  int32_t n;
};
static_assert(sizeof(Table) <= 3900, "kernel arguments");

// 16 bytes at any alignment of whole elements
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_f __attribute__((aligned(4)));
typedef u32x4 u32x4_h __attribute__((aligned(2)));

template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ u32x4 load(const float* p) { return *reinterpret_cast<const u32x4_f*>(p); }
  static __device__ __forceinline__ void store(float* p, u32x4 v) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4_f*>(p)); }
  static __device__ __forceinline__ double square(u32x4 v, double s) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double x = __uint_as_float(v[e]);
      s = fma(x, x, s);
    }
    return s;
  }
  static __device__ __forceinline__ u32x4 times(u32x4 v, double c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __float_as_uint((float)((double)__uint_as_float(v[e]) * c));
    return v;
  }
};
template <> struct Piece<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ u32x4 load(const uint16_t* p) { return *reinterpret_cast<const u32x4_h*>(p); }
  static __device__ __forceinline__ void store(uint16_t* p, u32x4 v) { __builtin_nontemporal_store(v, reinterpret_cast<u32x4_h*>(p)); }
  static __device__ __forceinline__ double square(u32x4 v, double s) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double x = __uint_as_float(v[e] << 16), y = __uint_as_float(v[e] & 0xffff0000u);
      s = fma(x, x, s);
      s = fma(y, y, s);
    }
    return s;
  }
  static __device__ __forceinline__ u32x4 times(u32x4 v, double c) {
    // the product in 64 bits is rounded to fp32 and then to bf16: a value that the first rounding puts on the middle between
    // two bf16 values (one in 2^16) may go to the farther one, by 2^-16 of a step
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[e] = pack_bf16x2((float)((double)__uint_as_float(v[e] << 16) * c),
                         (float)((double)__uint_as_float(v[e] & 0xffff0000u) * c));
    return v;
  }
};

// Adds up the 256 threads' values in a fixed order; the sum in every thread.
__device__ __forceinline__ double block_sum(double s) {
  __shared__ double sm[4];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
  __syncthreads();
  return (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

// The tensor that holds chunk c
__device__ __forceinline__ int tensor_of(const Table& t, int c) {
  int lo = 0, hi = t.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ double chunk_square(const T* g, int64_t n, double s) {
  constexpr int N = Piece<T>::N, STEP = 256 * N;
  const int full = (int)(n / N) * N;
  int i = threadIdx.x * N;
  for (; i + (kAhead - 1) * STEP < full; i += kAhead * STEP) {
    u32x4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) v[k] = Piece<T>::load(g + i + k * STEP);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) s = Piece<T>::square(v[k], s);
  }
  for (; i < full; i += STEP) s = Piece<T>::square(Piece<T>::load(g + i), s);
  if (full + (int)threadIdx.x < n) {
    const double x = to_f<T>(g[full + threadIdx.x]);
    s = fma(x, x, s);
  }
  return s;
}

__global__ __launch_bounds__(256) void grad_square_kernel(const Table t, double* part) {
  double s = 0.0;
  for (int c = blockIdx.x; c < t.first[t.n]; c += gridDim.x) {
    const int k = __builtin_amdgcn_readfirstlane(tensor_of(t, c));
    const int64_t at = (int64_t)(c - t.first[k]) * kChunk, n = min(t.numel[k] - at, (int64_t)kChunk);
    if (t.bf16[k]) s = chunk_square(static_cast<const uint16_t*>(t.g[k]) + at, n, s);
    else s = chunk_square(static_cast<const float*>(t.g[k]) + at, n, s);
  }
  s = block_sum(s);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double joined(const double* part, int parts) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) s += part[i];
  return block_sum(s);
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const double* part, int parts, float* norm) {
  const double s = joined(part, parts);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* g, T* out, int64_t n, double c) {
  constexpr int N = Piece<T>::N, STEP = 256 * N;
  const int full = (int)(n / N) * N;
  int i = threadIdx.x * N;
  for (; i + (kAhead - 1) * STEP < full; i += kAhead * STEP) {
    u32x4 v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) v[k] = Piece<T>::load(g + i + k * STEP);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) Piece<T>::store(out + i + k * STEP, Piece<T>::times(v[k], c));
  }
  for (; i < full; i += STEP) Piece<T>::store(out + i, Piece<T>::times(Piece<T>::load(g + i), c));
  if (full + (int)threadIdx.x < n) out[full + threadIdx.x] = from_f<T>((float)((double)to_f<T>(g[full + threadIdx.x]) * c));
}

// Chunks from the last to the first: what the norm read last lies in the caches still.
__global__ __launch_bounds__(256) void grad_scale_kernel(const Table t, const double* part, int parts, const float* norm_in,
                                                         float* norm, double max_norm) {
  double n;
  if (norm_in) {
    n = *norm_in;
  } else {
    n = sqrt(joined(part, parts));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  }
  double c = max_norm / (n + kEps);
  c = c > 1.0 ? 1.0 : c;  // NaN stays
  for (int b = t.first[t.n] - 1 - (int)blockIdx.x; b >= 0; b -= gridDim.x) {
    const int k = __builtin_amdgcn_readfirstlane(tensor_of(t, b));
    if (c == 1.0 && t.out[k] == t.g[k]) continue;
    const int64_t at = (int64_t)(b - t.first[k]) * kChunk, m = min(t.numel[k] - at, (int64_t)kChunk);
    if (t.bf16[k]) chunk_scale(static_cast<const uint16_t*>(t.g[k]) + at, static_cast<uint16_t*>(t.out[k]) + at, m, c);
    else chunk_scale(static_cast<const float*>(t.g[k]) + at, static_cast<float*>(t.out[k]) + at, m, c);
  }
}

int grid_of(const Table& t) { return std::min(t.first[t.n], kWgs); }

// Cuts the list into tables of tensors that hold something.
template <typename F>
void tables(int32_t n, const void* const* g, void* const* out, const int64_t* numel, const int32_t* dtype, F&& launch) {
  Table t;
  t.n = 0;
  t.first[0] = 0;
  for (int i = 0; i < n; ++i) {
    if (numel[i] == 0) continue;
    const int64_t chunks = (numel[i] + kChunk - 1) / kChunk;
    if (t.n == kGroup || t.first[t.n] + chunks > 0x7fffffff) {
      launch(t);
      t.n = 0;
    }
    if (g) {
      t.g[t.n] = g[i];
      t.out[t.n] = out ? out[i] : const_cast<void*>(g[i]);
      t.bf16[t.n] = dtype[i] == LLATTN_BF16;
    }
    t.numel[t.n] = numel[i];
    t.first[t.n + 1] = t.first[t.n] + (int32_t)chunks;
    ++t.n;
  }
  if (t.n) launch(t);
}

int32_t check_sizes(const char* who, int32_t n, const int64_t* numel) {
  if (n < 0 || (n > 0 && !numel)) return fail(LLATTN_ERR_SHAPE, "%s: %d tensors, or no sizes", who, n);
  for (int i = 0; i < n; ++i)
    if (numel[i] < 0 || numel[i] > (int64_t)1 << 44) return fail(LLATTN_ERR_SHAPE, "%s: tensor %d has %lld elements", who, i, (long long)numel[i]);
  return LLATTN_OK;
}

int64_t parts_of(int32_t n, const int64_t* numel) {
  int64_t parts = 0;
  tables(n, nullptr, nullptr, numel, nullptr, [&](const Table& t) { parts += grid_of(t); });
  return parts;
}

int32_t check_lists(const char* who, int32_t n, const void* const* g, void* const* out, const int64_t* numel, const int32_t* dtype) {
  if (const int32_t rc = check_sizes(who, n, numel)) return rc;
  if (n > 0 && (!g || !dtype)) return fail(LLATTN_ERR_LAYOUT, "%s: no pointers or types", who);
  for (int i = 0; i < n; ++i) {
    if (dtype[i] != LLATTN_F32 && dtype[i] != LLATTN_BF16) return fail(LLATTN_ERR_DTYPE, "%s: tensor %d: unknown dtype %d", who, i, dtype[i]);
    if (numel[i] == 0) continue;
    const uintptr_t mask = elem_size(dtype[i]) - 1;
    if (!g[i] || (out && !out[i])) return fail(LLATTN_ERR_LAYOUT, "%s: tensor %d: null pointer", who, i);
    if ((reinterpret_cast<uintptr_t>(g[i]) & mask) || (out && (reinterpret_cast<uintptr_t>(out[i]) & mask)))
      return fail(LLATTN_ERR_LAYOUT, "%s: tensor %d is not aligned to its elements", who, i);
  }
  return LLATTN_OK;
}

// What is written overlaps nothing else: neither another output nor an input but its own in place, nor the norm that is read.
int32_t check_apart(const char* who, int32_t n, const void* const* g, void* const* out, const int64_t* numel, const int32_t* dtype,
                    const float* norm_in) {
  struct Span { uintptr_t at, end; int i; };
  std::vector<Span> w;
  w.reserve(n);
  for (int i = 0; i < n; ++i) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(out ? out[i] : g[i]);
    if (numel[i]) w.push_back({at, at + (uintptr_t)numel[i] * elem_size(dtype[i]), i});
  }
  std::sort(w.begin(), w.end(), [](const Span& a, const Span& b) { return a.at < b.at; });
  for (size_t k = 1; k < w.size(); ++k)
    if (w[k].at < w[k - 1].end) return fail(LLATTN_ERR_LAYOUT, "%s: tensors %d and %d, which are written, overlap", who, w[k - 1].i, w[k].i);
  const auto first = [&](uintptr_t at) {  // the first that ends past it
    return std::upper_bound(w.begin(), w.end(), at, [](uintptr_t v, const Span& s) { return v < s.end; });
  };
  const uintptr_t norm = reinterpret_cast<uintptr_t>(norm_in);
  if (const auto k = first(norm); norm && k != w.end() && k->at < norm + sizeof(float))
    return fail(LLATTN_ERR_LAYOUT, "%s: tensor %d, which is written, holds the norm", who, k->i);
  if (!out) return LLATTN_OK;
  for (int i = 0; i < n; ++i) {
    if (!numel[i]) continue;
    const uintptr_t at = reinterpret_cast<uintptr_t>(g[i]), end = at + (uintptr_t)numel[i] * elem_size(dtype[i]);
    for (auto k = first(at); k != w.end() && k->at < end; ++k)
      if (k->i != i || k->at != at) return fail(LLATTN_ERR_LAYOUT, "%s: output %d overlaps gradient %d", who, k->i, i);
  }
  return LLATTN_OK;
}

// Squares of all tables; the number of parts.
int64_t launch_squares(int32_t n, const void* const* g, const int64_t* numel, const int32_t* dtype, double* part, hipStream_t st) {
  int64_t parts = 0;
  tables(n, g, nullptr, numel, dtype, [&](const Table& t) {
    const int grid = grid_of(t);
    hipLaunchKernelGGL(grad_square_kernel, dim3(grid), dim3(256), 0, st, t, part + parts);
    parts += grid;
  });
  return parts;
}

int32_t check_workspace(const char* who, const void* ws, size_t bytes, size_t need) {
  if (!ws || bytes < need || (reinterpret_cast<uintptr_t>(ws) & 7)) return fail(LLATTN_ERR_WORKSPACE, "%s: needs %zu workspace bytes (got %zu)", who, need, bytes);
  return LLATTN_OK;
}

}  // namespace
}  // namespace llattn

using namespace llattn;

extern "C" size_t llattn_grad_norm_bytes(int32_t n, const int64_t* numel) {
  if (check_sizes("llattn_grad_norm_bytes", n, numel) != LLATTN_OK) return 0;
  const int64_t parts = parts_of(n, numel);
  if (parts > 0x7fffffff) {
    fail(LLATTN_ERR_SHAPE, "llattn_grad_norm_bytes: too many tensors");
    return 0;
  }
  return std::max<size_t>(8, 8 * (size_t)parts);
}

extern "C" int32_t llattn_grad_norm(int32_t n, const void* const* g, const int64_t* numel, const int32_t* dtype, float* norm,
                                    void* workspace, size_t workspace_bytes, void* stream) {
  if (const int32_t rc = check_lists("llattn_grad_norm", n, g, nullptr, numel, dtype)) return rc;
  if (!norm) return fail(LLATTN_ERR_LAYOUT, "llattn_grad_norm: null norm");
  const size_t need = llattn_grad_norm_bytes(n, numel);
  if (need == 0) return LLATTN_ERR_SHAPE;
  if (const int32_t rc = check_workspace("llattn_grad_norm", workspace, workspace_bytes, need)) return rc;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  const int parts = (int)launch_squares(n, g, numel, dtype, part, st);
  hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, st, part, parts, norm);
  return check_launch("llattn_grad_norm");
}

extern "C" int32_t llattn_clip_grads(int32_t n, const void* const* g, void* const* out, const int64_t* numel, const int32_t* dtype,
                                     double max_norm, const float* norm_in, float* norm, void* workspace, size_t workspace_bytes,
                                     void* stream) {
  if (const int32_t rc = check_lists("llattn_clip_grads", n, g, out, numel, dtype)) return rc;
  if (!norm_in == !norm) return fail(LLATTN_ERR_LAYOUT, "llattn_clip_grads: one of norm_in and norm");
  std::vector<Table> all;
  try {  // both need memory of the host's, before anything is launched
    if (const int32_t rc = check_apart("llattn_clip_grads", n, g, out, numel, dtype, norm_in)) return rc;
    tables(n, g, out, numel, dtype, [&](const Table& t) { all.push_back(t); });
  } catch (const std::bad_alloc&) {
    return fail(LLATTN_ERR_SHAPE, "llattn_clip_grads: no memory for the tables of %d tensors", n);
  }
  const hipStream_t st = static_cast<hipStream_t>(stream);
  double* part = static_cast<double*>(workspace);
  int parts = 0;
  if (!norm_in) {
    const size_t need = llattn_grad_norm_bytes(n, numel);
    if (need == 0) return LLATTN_ERR_SHAPE;
    if (const int32_t rc = check_workspace("llattn_clip_grads", workspace, workspace_bytes, need)) return rc;
    parts = (int)launch_squares(n, g, numel, dtype, part, st);
    if (parts == 0) hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, st, part, 0, norm);
  }
  // the last table first, as its gradients were read last
  for (size_t k = all.size(); k-- > 0;)
    hipLaunchKernelGGL(grad_scale_kernel, dim3(grid_of(all[k])), dim3(256), 0, st, all[k], part, parts, norm_in,
                       k == 0 ? norm : nullptr, max_norm);
  return check_launch("llattn_clip_grads");
}
