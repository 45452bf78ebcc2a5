// Global norm of a list of tensors, and their scaling to a largest norm
// (sm_100a).
//
//   norm_partial_kernel  each block walks units of 32 KB over all tensors and
//                        writes one f64 partial;
//   norm_finish_kernel   one block adds the partials in order: the norm (f32);
//   clip_kernel          out = in * min(1, max_norm / (norm + 1e-6)), rounded
//                        once to out's type; on short lists its blocks add
//                        the partials themselves, which saves the finish
//                        launch.  One launch per pair of types in the list.
//
// HBM-bound: the tensors are read once for the norm and once for the scaling
// (from L2 where they fit: the scaling walks the units backwards, so that it
// starts with what the norm read last).  A launch carries its list of tensors
// in its arguments - no copy to the device, nothing kept between calls; a list
// longer than kGradSlots takes several launches, whose partials follow one
// another.
//
// Sums: 32 elements at a time in f32 (each step rounds by 2^-24), then f64.
// Squares of elements outside [2^-63, 2^60] leave the f32 range: where the
// largest of the 32 is outside [2^-40, 2^60], all of them are summed in f64.
// (Squares that vanish beside a largest element of at least 2^-40 are below
// 2^-46 of its square.)  No atomics: a result repeats bit for bit.
#pragma once
#include <cstdint>
#include <type_traits>

#include "ptx.cuh"
#include "router_train.cuh"

namespace moe {

constexpr int kNormThreads = 256;
constexpr int kNormChunks = 8;                          // 16-byte chunks of input a thread has in flight
constexpr int kNormBlocksPerSm = 4;
// Blocks of a launch.  Lists of up to kNormLarge units run on the blocks that
// are resident, and every block of the scaling adds up the partials for
// itself.  Above that (155 MB of input) a block takes one unit and the hardware
// hands them out: with resident blocks in a fixed order, the slowest of them
// set the pace (scaling 2 x 470 M f32 to bf16: 951 us on 592 blocks, 838 on
// 9472, 798 with one unit each; below, the third launch costs what that gives:
// three launches ran 30 M bf16 21% slower than two, 60 M 5% slower, 120 M 2%
// faster).  A norm's blocks are kept to as many partials as one block then adds
// up in a few microseconds.
constexpr int kNormResident = 148 * kNormBlocksPerSm;
constexpr uint32_t kNormLarge = 8 * kNormResident;
constexpr int kNormMaxBlocks = 16384;

// Elements of a chunk and of a unit (32 KB of input).
__host__ __device__ constexpr int chunk_elems(int type) { return type == kElemF32 ? 4 : 8; }
__host__ __device__ constexpr int64_t unit_elems(int type) { return kNormThreads * kNormChunks * chunk_elems(type); }

// rows x cols elements, rows in_ld / out_ld elements apart (a dense tensor is
// one row).  head: elements before the first one that is 16-byte aligned in
// `in` and in `out` aligned to the store of a chunk (0 for every tensor of
// several rows); -1: no such element, the tensor is read one element at a
// time.
struct GradEntry {
  const void* in;
  void* out;
  int64_t rows, cols, in_ld, out_ld;
  int16_t in_type, out_type;
  int16_t head;
};

constexpr int kGradSlotsSmall = 48;   // launch arguments of 3 KB
constexpr int kGradSlots = 500;       // 32 KB (the most that a launch takes is 32,764 bytes)
template <int SLOTS>
struct GradList {
  GradEntry e[SLOTS];
  uint32_t unit0[SLOTS];  // first unit of each tensor; apart from the entries, so that a search reads few lines
  int32_t n;
  uint32_t units;
};
static_assert(sizeof(GradList<kGradSlots>) < 32000, "launch arguments end at 32,764 bytes");

enum : int { kNormL1 = 1, kNormL2 = 2, kNormInf = 3 };

// The tensor that a unit belongs to: the last one whose first unit is not past it.
template <int SLOTS>
__device__ __forceinline__ int entry_of(const GradList<SLOTS>& list, uint32_t unit) {
  int lo = 0, hi = list.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.unit0[mid] <= unit) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Element i of the tensor (row-major over rows x cols) as an offset.
__device__ __forceinline__ int64_t entry_at(int64_t i, int64_t rows, int64_t cols, int64_t ld) {
  if (rows == 1) return i;
  const int64_t r = (i | cols) >> 32 ? i / cols : (int64_t)((uint32_t)i / (uint32_t)cols);
  return r * ld + (i - r * cols);
}

// The 16-bit and f32 types' values of a chunk.
template <int TYPE>
__device__ __forceinline__ void chunk_values(const uint4& r, float* v) {
  if (TYPE == kElemF32) {
    v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
  } else {
    unpack16(r.x, TYPE, v[0], v[1]);
    unpack16(r.y, TYPE, v[2], v[3]);
    unpack16(r.z, TYPE, v[4], v[5]);
    unpack16(r.w, TYPE, v[6], v[7]);
  }
}
// Plain loads throughout: the scaling may run in place, and the read-only
// path is for memory that nobody writes during the kernel.
template <int TYPE>
__device__ __forceinline__ float single_value(const void* p, int64_t i) {
  if (TYPE == kElemF32) return static_cast<const float*>(p)[i];
  const uint16_t u = static_cast<const uint16_t*>(p)[i];
  return TYPE == kElemBF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}
template <int TYPE>
__device__ __forceinline__ const uint4* chunk_ptr(const void* p, int64_t i) {
  return reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + i * (TYPE == kElemF32 ? 4 : 2));
}

// A block's pass over one unit: all of a thread's chunks are loaded, then
// chunks(raw, index of the first, number in the tensor, whether the tensor is
// dense and the unit whole) takes them (zeros past the end); single(in offset, out offset) takes the elements outside chunks:
// those before and after (in a tensor's first unit), or all where head < 0.
// WHOLE: whole units have a body of their own (the scaling: 41 -> 39 us for 60 M
// bf16; the norm's sums, twice in one kernel, spill: 27 -> 40 us).
template <int TYPE, bool WHOLE, class Chunks, class Single>
__device__ __forceinline__ void walk_unit(const GradEntry& e, int64_t u, Chunks&& chunks, Single&& single) {
  constexpr int CE = chunk_elems(TYPE);
  const int64_t rows = e.rows, cols = e.cols, total = rows * cols;
  if (e.head < 0) {
    const int64_t hi = min(total, (u + 1) * unit_elems(TYPE));
    for (int64_t i = u * unit_elems(TYPE) + threadIdx.x; i < hi; i += kNormThreads)
      single(entry_at(i, rows, cols, e.in_ld), entry_at(i, rows, cols, e.out_ld));
    return;
  }
  const int64_t n = (total - e.head) / CE;  // chunks
  const int64_t first = u * (kNormThreads * kNormChunks) + threadIdx.x;
  uint4 raw[kNormChunks];
  const bool whole = WHOLE && rows == 1 && (u + 1) * (kNormThreads * kNormChunks) <= n;
  if (whole) {  // most units: nothing to ask per chunk
    const uint4* q = chunk_ptr<TYPE>(e.in, e.head) + first;
#pragma unroll
    for (int s = 0; s < kNormChunks; ++s) raw[s] = q[s * kNormThreads];
    chunks(raw, first, n, std::true_type());
  } else if (rows == 1) {
    const uint4* q = chunk_ptr<TYPE>(e.in, e.head) + first;
#pragma unroll
    for (int s = 0; s < kNormChunks; ++s)
      raw[s] = first + s * kNormThreads < n ? q[s * kNormThreads] : make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll
    for (int s = 0; s < kNormChunks; ++s)
      raw[s] = first + s * kNormThreads < n
                   ? *chunk_ptr<TYPE>(e.in, entry_at((first + s * kNormThreads) * CE, rows, cols, e.in_ld))
                   : make_uint4(0, 0, 0, 0);
  }
  if (!whole) chunks(raw, first, n, std::false_type());
  if (u == 0) {
    const int64_t tail = e.head + CE * n;
    const int64_t i = threadIdx.x < 8 ? (int64_t)threadIdx.x : tail + threadIdx.x - 8;
    if (threadIdx.x < 8 ? i < e.head : threadIdx.x < 16 && i < total) single(i, i);
  }
}

// ---------------------------------------------------------------- norm
template <int NORM>
__device__ __forceinline__ double big_term(float x) {
  return NORM == kNormL2 ? (double)x * (double)x : (double)fabsf(x);
}

// The part of one thread: f64 sum of |x|^p, or the bits of the largest |x|
// (as integers, which order NaN above infinity, so that a NaN comes through).
struct NormAcc {
  double sum;
  uint32_t top;
};

template <int NORM, int N>
__device__ __forceinline__ void norm_add(const float (&v)[N], NormAcc& acc) {
  if (NORM == kNormInf) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc.top = max(acc.top, __float_as_uint(fabsf(v[i])));
    return;
  }
  float part[4] = {0.f, 0.f, 0.f, 0.f}, top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    part[i & 3] = NORM == kNormL2 ? fmaf(v[i], v[i], part[i & 3]) : part[i & 3] + fabsf(v[i]);
    top = fmaxf(top, fabsf(v[i]));
  }
  // A largest of 0 leaves a sum of 0 or, where all are NaN, NaN.
  if (top <= 0x1p60f && (NORM == kNormL1 || top >= 0x1p-40f || top == 0.f)) {
    acc.sum += (double)((part[0] + part[1]) + (part[2] + part[3]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) acc.sum += big_term<NORM>(v[i]);
  }
}

template <int NORM, int TYPE>
__device__ __forceinline__ void norm_unit(const GradEntry& e, int64_t u, NormAcc& acc) {
  constexpr int CE = chunk_elems(TYPE), PER = 32 / CE;  // chunks of 32 elements
  walk_unit<TYPE, false>(
      e, u,
      [&](const uint4 (&raw)[kNormChunks], int64_t, int64_t, auto) {
#pragma unroll
        for (int s = 0; s < kNormChunks; s += PER) {
          float v[32];
#pragma unroll
          for (int c = 0; c < PER; ++c) chunk_values<TYPE>(raw[s + c], v + c * CE);
          norm_add<NORM>(v, acc);
        }
      },
      [&](int64_t in, int64_t) {
        const float v[1] = {single_value<TYPE>(e.in, in)};
        norm_add<NORM>(v, acc);
      });
}

template <int NORM, int SLOTS>
__global__ void __launch_bounds__(kNormThreads, kNormBlocksPerSm) norm_partial_kernel(const __grid_constant__ GradList<SLOTS> list,
                                                                    double* __restrict__ partial) {
  __shared__ double s_w[kNormThreads / 32];
  NormAcc acc{0.0, 0u};
  int at = entry_of(list, blockIdx.x);
  for (uint32_t unit = blockIdx.x; unit < list.units; unit += gridDim.x) {
    while (at + 1 < list.n && list.unit0[at + 1] <= unit) ++at;
    const GradEntry& e = list.e[at];
    const int64_t u = unit - list.unit0[at];
    if (e.in_type == kElemF32) norm_unit<NORM, kElemF32>(e, u, acc);
    else if (e.in_type == kElemBF16) norm_unit<NORM, kElemBF16>(e, u, acc);
    else norm_unit<NORM, kElemF16>(e, u, acc);
  }
  if (NORM == kNormInf) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, acc.top);
    if ((threadIdx.x & 31) == 0) s_w[threadIdx.x >> 5] = (double)top;
    __syncthreads();
    if (threadIdx.x == 0) {
      double m = 0.0;
      for (int w = 0; w < kNormThreads / 32; ++w) m = fmax(m, s_w[w]);
      partial[blockIdx.x] = m;
    }
  } else {
    const double sum = block_sum(acc.sum, s_w);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
  }
}

// The norm from n partials, the same value in every thread of the block.
__device__ __forceinline__ float norm_of(int norm_type, const double* partial, int n, double* s_w) {
  double v = 0.0;
  if (norm_type == kNormInf) {
    for (int i = threadIdx.x; i < n; i += kNormThreads) v = fmax(v, partial[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) s_w[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < kNormThreads / 32; ++w) v = fmax(v, s_w[w]);
    return __uint_as_float((uint32_t)v);  // the bits of |x|: whole numbers below 2^32
  }
#pragma unroll 8
  for (int i = threadIdx.x; i < n; i += kNormThreads) v += partial[i];
  v = block_sum(v, s_w);
  return (float)(norm_type == kNormL2 ? sqrt(v) : v);
}

__global__ void __launch_bounds__(kNormThreads) norm_finish_kernel(int norm_type, const double* partial, int n,
                                                                   float* norm) {
  __shared__ double s_w[kNormThreads / 32];
  const float v = norm_of(norm_type, partial, n, s_w);
  if (threadIdx.x == 0) *norm = v;
}

// ---------------------------------------------------------------- clip
template <int IN, int OUT>
__device__ __forceinline__ void clip_unit(const GradEntry& e, int64_t u, float coef) {
  constexpr int CE = chunk_elems(IN);
  const int64_t rows = e.rows;
  walk_unit<IN, true>(
      e, u,
      [&](const uint4 (&raw)[kNormChunks], int64_t first, int64_t n, auto whole) {
#pragma unroll
        for (int s = 0; s < kNormChunks; ++s) {
          const int64_t c = first + s * kNormThreads;
          if (!decltype(whole)::value && c >= n) continue;
          float v[CE];
          chunk_values<IN>(raw[s], v);
#pragma unroll
          for (int x = 0; x < CE; ++x) v[x] *= coef;
          const int64_t at = decltype(whole)::value || rows == 1 ? e.head + c * CE : entry_at(c * CE, rows, e.cols, e.out_ld);
          if (OUT == kElemF32) {
#pragma unroll
            for (int x = 0; x < CE; x += 4)
              *reinterpret_cast<float4*>(static_cast<float*>(e.out) + at + x) =
                  make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
          } else if (CE == 4) {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(e.out) + at) =
                make_uint2(pack16(v[0], v[1], OUT), pack16(v[2], v[3], OUT));
          } else {
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(e.out) + at) =
                make_uint4(pack16(v[0], v[1], OUT), pack16(v[2], v[3], OUT), pack16(v[4 % CE], v[5 % CE], OUT),
                           pack16(v[6 % CE], v[7 % CE], OUT));
          }
        }
      },
      [&](int64_t in, int64_t out) { elem_store(e.out, OUT, out, single_value<IN>(e.in, in) * coef); });
}

struct ClipNorm {
  const double* partial;  // n partials of the norm, or
  int32_t n;
  int32_t norm_type;
  const float* given;     // the norm itself
  float* norm;            // written by block 0 from the partials
  double max_norm;
};

// One pair of types per launch: a switch over all pairs around this body
// spilled 2 KB a thread and ran the 2 x 470 M element case at 1625 us.
template <int IN, int OUT, int SLOTS>
__global__ void __launch_bounds__(kNormThreads, kNormBlocksPerSm) clip_kernel(const __grid_constant__ GradList<SLOTS> list,
                                                            const ClipNorm c) {
  __shared__ double s_w[kNormThreads / 32];
  float norm;
  if (c.given) {
    norm = *c.given;
  } else {
    norm = norm_of(c.norm_type, c.partial, c.n, s_w);
    if (c.norm && blockIdx.x == 0 && threadIdx.x == 0) *c.norm = norm;
  }
  const double ratio = c.max_norm / ((double)norm + 1e-6);
  const float coef = ratio >= 1.0 ? 1.f : (float)ratio;  // a NaN ratio stays
  int at = entry_of(list, list.units - 1 - blockIdx.x);
  for (uint32_t i = blockIdx.x; i < list.units; i += gridDim.x) {
    const uint32_t unit = list.units - 1 - i;
    while (list.unit0[at] > unit) --at;
    const GradEntry& e = list.e[at];
    if (IN == OUT && coef == 1.f && e.in == e.out) continue;  // in place, nothing to scale
    clip_unit<IN, OUT>(e, unit - list.unit0[at], coef);
  }
}

}  // namespace moe
