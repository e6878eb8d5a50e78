// The global norm of a list of gradient tensors and the gradients scaled to it:
//   norm = scale sqrt(sum g^2),  factor = scale min(1, max_norm / (norm + 1e-6)),  out = factor g
//
// Two walks over the tensors, both cut into pieces of kPiece elements that the workgroups take in turn:
// the first leaves a sum of squares per workgroup, the second adds those up again in every workgroup (a
// fixed order, so all get the same factor) and scales.  The second walks the pieces backwards: what the
// first read last is still in the 256 MB cache.  Squares and sums are in 64 bits: in 32, gradients above
// 2^64 or below 2^-63 would give an infinite or a zero norm.  The tensors' addresses travel in the kernel
// arguments (kBatch of them a launch), so a captured call holds no pointer to host memory and the device
// keeps no table.
//
// Bound: reading and writing the gradients.  233 million fp16 elements into fp32 105 to 117 + 272 us (4.0 to
// 4.4 TB/s beside the write-back of the previous call's output, 5.9 without one; 5.1 TB/s, a copy's rate);
// 112 tensors of 2.2 million elements in place 4.7 + 3.9 us, and 38 us of host time for their addresses and
// checks.  512 workgroups or pieces of half the size read slower (117 and 96 us alone against 79), 2048 the
// same with twice the sums to add up again; stores past the caches 387 -> 422 us.
//
// Scaling by a number on the device is the second walk alone: 9.6 us for those 112 tensors behind a backward.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "dk_common.h"

namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;                          // elements of a lane's piece of work
constexpr int kRuns = 4;
constexpr int kPiece = kThreads * kVec * kRuns;  // 8192 elements
constexpr int kBatch = 128;                      // tensors of a launch: the most, in powers of two, whose
                                                 // table and the other arguments stay under 4 KB
constexpr int kGroups = 1024;                    // workgroups of a launch, four to a CU

typedef __bf16 bf16;
// 16-byte accesses at any element's address
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x8u __attribute__((ext_vector_type(8), aligned(2)));

struct Table {
  const void* src[kBatch];
  void* dst[kBatch];
  int64_t numel[kBatch];
  uint32_t first[kBatch + 1];     // the tensors' first pieces
  uint8_t type[kBatch];           // source type | destination type << 4
  int n;
};
static_assert(sizeof(Table) + 64 + 256 <= 4096, "kernel arguments, the launch's own 256 bytes among them");

struct Piece {
  int tensor;
  int64_t begin;
  int count;
};

__device__ __forceinline__ Piece piece_of(const Table& t, uint32_t c) {
  int lo = 0, hi = t.n - 1;       // the last tensor whose first piece is at most c
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  const int64_t begin = (int64_t)(c - t.first[lo]) * kPiece, left = t.numel[lo] - begin;
  return {lo, begin, (int)(left < kPiece ? left : kPiece)};
}

template <int TYPE>
__device__ __forceinline__ float from_bits(uint16_t u) {
  if (TYPE == DK_TYPE_F16) return (float)__builtin_bit_cast(f16, u);
  return __builtin_bit_cast(float, (uint32_t)u << 16);
}

template <int TYPE>
__device__ __forceinline__ uint16_t to_bits(float v) {
  if (TYPE == DK_TYPE_F16) return __builtin_bit_cast(uint16_t, (f16)v);
  return __builtin_bit_cast(uint16_t, (bf16)v);
}

template <int TYPE>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (TYPE == DK_TYPE_F32) return static_cast<const float*>(p)[i];
  else return from_bits<TYPE>(static_cast<const uint16_t*>(p)[i]);
}

template <int TYPE>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (TYPE == DK_TYPE_F32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = to_bits<TYPE>(v);
}

// kVec elements as loaded, and as numbers
template <int TYPE>
struct Raw {
  f32x4u a, b;
};
template <>
struct Raw<DK_TYPE_F16> {
  u16x8u a;
};
template <>
struct Raw<DK_TYPE_BF16> {
  u16x8u a;
};

template <int TYPE>
__device__ __forceinline__ Raw<TYPE> load8(const void* p, int64_t i) {
  if constexpr (TYPE == DK_TYPE_F32) {
    const float* q = static_cast<const float*>(p) + i;
    return {*reinterpret_cast<const f32x4u*>(q), *reinterpret_cast<const f32x4u*>(q + 4)};
  } else {
    return {*reinterpret_cast<const u16x8u*>(static_cast<const uint16_t*>(p) + i)};
  }
}

template <int TYPE>
__device__ __forceinline__ float number(const Raw<TYPE>& r, int k) {
  if constexpr (TYPE == DK_TYPE_F32) return k < 4 ? r.a[k] : r.b[k - 4];
  else return from_bits<TYPE>(r.a[k]);
}

template <int TYPE>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&v)[kVec]) {
  if constexpr (TYPE == DK_TYPE_F32) {
    f32x4u a, b;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a[k] = v[k];
      b[k] = v[k + 4];
    }
    *reinterpret_cast<f32x4u*>(static_cast<float*>(p) + i) = a;
    *reinterpret_cast<f32x4u*>(static_cast<float*>(p) + i + 4) = b;
  } else {
    u16x8u a;
#pragma unroll
    for (int k = 0; k < 8; ++k) a[k] = to_bits<TYPE>(v[k]);
    *reinterpret_cast<u16x8u*>(static_cast<uint16_t*>(p) + i) = a;
  }
}

// f with the type as a constant
template <class F>
__device__ __forceinline__ void with_type(int type, F&& f) {
  if (type == DK_TYPE_F32) f(std::integral_constant<int, DK_TYPE_F32>{});
  else if (type == DK_TYPE_F16) f(std::integral_constant<int, DK_TYPE_F16>{});
  else f(std::integral_constant<int, DK_TYPE_BF16>{});
}

// A piece: vec(raw elements, place) for each run of kVec, all loads of a whole piece before the first use;
// one(element's place) for the last elements of a tensor.
template <int TYPE, class V, class O>
__device__ __forceinline__ void walk(const void* src, const Piece& q, V&& vec, O&& one) {
  const int i0 = kVec * threadIdx.x;
  if (q.count == kPiece) {
    Raw<TYPE> r[kRuns];
#pragma unroll
    for (int u = 0; u < kRuns; ++u) r[u] = load8<TYPE>(src, q.begin + i0 + u * kVec * kThreads);
#pragma unroll
    for (int u = 0; u < kRuns; ++u) vec(r[u], q.begin + i0 + u * kVec * kThreads);
    return;
  }
  int i = i0;
  for (; i + kVec <= q.count; i += kVec * kThreads) vec(load8<TYPE>(src, q.begin + i), q.begin + i);
  for (; i < q.count; ++i) one(q.begin + i);   // one lane, fewer than kVec
}

// the workgroup's sum in a fixed order; every thread gets it
__device__ __forceinline__ double block_sum(double s, double* red) {
#pragma unroll
  for (int x = 1; x < 64; x *= 2) s += __shfl_xor(s, x);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  double total = red[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) total += red[w];
  return total;
}

__global__ __launch_bounds__(kThreads) void squares_kernel(Table t, uint32_t pieces, double* part) {
  __shared__ double red[kThreads / 64];
  double s = 0.0;
  for (uint32_t c = blockIdx.x; c < pieces; c += gridDim.x) {
    const Piece q = piece_of(t, c);
    const void* src = t.src[q.tensor];
    with_type(t.type[q.tensor] & 15, [&](auto type) {
      constexpr int T = decltype(type)::value;
      auto add = [&](double v) { s = __builtin_fma(v, v, s); };
      walk<T>(
          src, q,
          [&](const Raw<T>& r, int64_t) {
#pragma unroll
            for (int k = 0; k < kVec; ++k) add((double)number<T>(r, k));
          },
          [&](int64_t i) { add((double)load1<T>(src, i)); });
    });
  }
  const double total = block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = total;
}

// dst = factor src over all pieces, the last one first
__device__ __forceinline__ void scale_pieces(const Table& t, uint32_t pieces, float factor) {
  for (uint32_t b = blockIdx.x; b < pieces; b += gridDim.x) {
    const Piece q = piece_of(t, pieces - 1 - b);
    const void* src = t.src[q.tensor];
    void* dst = t.dst[q.tensor];
    if (src == dst && factor == 1.0f) continue;   // nothing changes in place
    with_type(t.type[q.tensor] & 15, [&](auto type) {
      with_type(t.type[q.tensor] >> 4, [&](auto to) {
        constexpr int T = decltype(type)::value, U = decltype(to)::value;
        walk<T>(
            src, q,
            [&](const Raw<T>& r, int64_t i) {
              float v[kVec];
#pragma unroll
              for (int k = 0; k < kVec; ++k) v[k] = number<T>(r, k) * factor;
              store8<U>(dst, i, v);
            },
            [&](int64_t i) { store1<U>(dst, i, load1<T>(src, i) * factor); });
      });
    });
  }
}

__global__ __launch_bounds__(kThreads) void scale_kernel(Table t, uint32_t pieces, const double* part,
                                                         int parts, double max_norm, double scale,
                                                         float* norm_out) {
  __shared__ double red[kThreads / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += kThreads) s += part[i];
  const double norm = scale * sqrt(block_sum(s, red));
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double ratio = max_norm / (norm + 1e-6);
  // a NaN norm gives NaN; no largest norm: `scale` alone, whatever the norm
  const float factor = (float)(scale * (ratio > 1.0 || max_norm == INFINITY ? 1.0 : ratio));
  scale_pieces(t, pieces, factor);
}

// every element times scale by[0]
__global__ __launch_bounds__(kThreads) void times_kernel(Table t, uint32_t pieces, const float* by, double scale) {
  scale_pieces(t, pieces, (float)(scale * (double)*by));
}

int64_t type_size(int type) {
  return type == DK_TYPE_F32 ? 4 : type == DK_TYPE_F16 || type == DK_TYPE_BF16 ? 2 : 0;
}

int groups_of(int64_t pieces) { return (int)(pieces < kGroups ? pieces : kGroups); }

}  // namespace

extern "C" int64_t dk_grad_clip_workspace(int64_t n) {
  return n <= 0 ? 0 : (n + kBatch - 1) / kBatch * kGroups * (int64_t)sizeof(double);
}

namespace {

struct Lists {
  const void* const* src;
  void* const* dst;            // null: nothing is written
  const int64_t* numel;
  const int32_t *types, *dst_types;
  int64_t n;
};

int check_lists(const Lists& l) {
  for (int64_t i = 0; i < l.n; ++i) {
    const int64_t from = type_size(l.types[i]), to = l.dst ? type_size(l.dst_types[i]) : from;
    if (!from || !to || l.numel[i] < 0 || l.numel[i] > (int64_t)1 << 40) return DK_ERR_INVALID;
    if (l.numel[i] && (!l.src[i] || (l.dst && !l.dst[i]))) return DK_ERR_INVALID;
    if (!dk_aligned(l.src[i], from) || (l.dst && !dk_aligned(l.dst[i], to))) return DK_ERR_ALIGN;
    if (l.dst && l.dst[i] == l.src[i] && l.numel[i] && l.types[i] != l.dst_types[i]) return DK_ERR_INVALID;
  }
  if (!l.dst) return 0;
  // what is written overlaps nothing else that is read or written: in place, its own source alone
  struct Range {
    uintptr_t begin, end;
    bool write;
  };
  try {
    std::vector<Range> all;
    all.reserve(2 * l.n);
    for (int64_t i = 0; i < l.n; ++i) {
      if (!l.numel[i]) continue;
      const uintptr_t s = (uintptr_t)l.src[i], d = (uintptr_t)l.dst[i];
      all.push_back({d, d + l.numel[i] * type_size(l.dst_types[i]), true});
      if (s != d) all.push_back({s, s + l.numel[i] * type_size(l.types[i]), false});
    }
    std::sort(all.begin(), all.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    uintptr_t written = 0, touched = 0;
    for (const Range& r : all) {
      if (r.begin < written || (r.write && r.begin < touched)) return DK_ERR_INVALID;
      if (r.write) written = std::max(written, r.end);
      touched = std::max(touched, r.end);
    }
  } catch (...) {
    return DK_ERR_INVALID;
  }
  return 0;
}

// the batch of tensors from `i` on (advanced past it) and its pieces; tensors without elements skipped
int64_t fill(const Lists& l, Table& t, int64_t& i) {
  int64_t pieces = 0;
  t.n = 0;
  for (; i < l.n && t.n < kBatch; ++i) {
    const int64_t c = (l.numel[i] + kPiece - 1) / kPiece;
    if (pieces + c > UINT32_MAX / 2) break;
    if (!c) continue;
    t.src[t.n] = l.src[i];
    t.dst[t.n] = l.dst ? l.dst[i] : nullptr;
    t.numel[t.n] = l.numel[i];
    t.type[t.n] = (uint8_t)(l.types[i] | (l.dst ? l.dst_types[i] : 0) << 4);
    t.first[t.n] = (uint32_t)pieces;
    ++t.n;
    pieces += c;
  }
  t.first[t.n] = (uint32_t)pieces;
  return pieces;
}

}  // namespace

extern "C" int dk_grad_clip(const void* const* src, void* const* dst, const int64_t* numel,
                            const int32_t* types, const int32_t* dst_types, int64_t n, double max_norm,
                            double scale, float* norm, void* ws, int64_t ws_bytes, hipStream_t stream) {
  if (n < 1 || n > (int64_t)1 << 20 || !src || !numel || !types || (dst && !dst_types) || !norm ||
      !(max_norm > 0.0) || !(scale > 0.0) || scale - scale != 0.0)
    return DK_ERR_INVALID;
  if (!dk_aligned(norm, 4)) return DK_ERR_ALIGN;
  const Lists l{src, dst, numel, types, dst_types, n};
  if (const int rc = check_lists(l)) return rc;
  if (!ws || ws_bytes < dk_grad_clip_workspace(n) || !dk_aligned(ws, 8)) return DK_ERR_WORKSPACE;
  double* part = static_cast<double*>(ws);
  Table t;
  int parts = 0;
  for (int64_t i = 0; i < n;) {
    const int64_t pieces = fill(l, t, i);
    if (!pieces) continue;
    const int g = groups_of(pieces);
    hipLaunchKernelGGL(squares_kernel, dim3(g), dim3(kThreads), 0, stream, t, (uint32_t)pieces, part + parts);
    DK_CHECK_LAUNCH();
    parts += g;
  }
  bool said = false;
  for (int64_t i = 0; dst && i < n;) {
    const int64_t pieces = fill(l, t, i);
    if (!pieces) continue;
    hipLaunchKernelGGL(scale_kernel, dim3(groups_of(pieces)), dim3(kThreads), 0, stream, t, (uint32_t)pieces,
                       part, parts, max_norm, scale, said ? nullptr : norm);
    DK_CHECK_LAUNCH();
    said = true;
  }
  if (!said) {   // the norm alone (or no elements)
    t.n = 0;
    hipLaunchKernelGGL(scale_kernel, dim3(1), dim3(kThreads), 0, stream, t, 0u, part, parts, max_norm, scale,
                       norm);
    DK_CHECK_LAUNCH();
  }
  return 0;
}

extern "C" int dk_grad_scale(void* const* tensors, const int64_t* numel, const int32_t* types, int64_t n,
                             const float* factor, double scale, hipStream_t stream) {
  if (n < 1 || n > (int64_t)1 << 20 || !tensors || !numel || !types || !factor) return DK_ERR_INVALID;
  if (!dk_aligned(factor, 4)) return DK_ERR_ALIGN;
  const Lists l{(const void* const*)tensors, tensors, numel, types, types, n};
  if (const int rc = check_lists(l)) return rc;
  for (int64_t i = 0; i < n; ++i)   // (workgroups read the factor while others write)
    if ((uintptr_t)factor + 4 > (uintptr_t)tensors[i] &&
        (uintptr_t)factor < (uintptr_t)tensors[i] + numel[i] * type_size(types[i]))
      return DK_ERR_INVALID;
  Table t;
  for (int64_t i = 0; i < n;) {
    const int64_t pieces = fill(l, t, i);
    if (!pieces) continue;
    hipLaunchKernelGGL(times_kernel, dim3(groups_of(pieces)), dim3(kThreads), 0, stream, t, (uint32_t)pieces,
                       factor, scale);
    DK_CHECK_LAUNCH();
  }
  return 0;
}
