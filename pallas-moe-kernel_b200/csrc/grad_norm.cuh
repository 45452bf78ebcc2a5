// Global norm of a list of tensors, and their scaling to a largest norm
// (sm_100a).
//
//   norm_partial_kernel  each block walks units of kNormUnit elements over all
//                        tensors and writes one f64 partial;
//   norm_finish_kernel   one block adds the partials in order: the norm (f32);
//   clip_kernel          out = in * min(1, max_norm / (norm + 1e-6)), rounded
//                        once to out's type; its blocks add the partials
//                        themselves, which saves the finish launch.
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

#include "ptx.cuh"
#include "router_train.cuh"

namespace moe {

constexpr int kNormThreads = 256;
constexpr int kNormVecs = 4;                                // 8-element vectors a thread takes per unit
constexpr int kNormUnit = kNormThreads * kNormVecs * 8;     // elements
constexpr int kNormBlocksPerSm = 4;
constexpr int kNormMaxBlocks = 148 * kNormBlocksPerSm;      // most blocks (partials) of one launch

// rows x cols elements, rows in_ld / out_ld elements apart (a dense tensor is
// one row).  head: elements before the first one that is 16-byte aligned in
// `in` and in `out` (0 for every tensor of several rows); -1: no such element,
// the tensor is read one element at a time.
struct GradEntry {
  const void* in;
  void* out;
  int64_t rows, cols, in_ld, out_ld;
  int32_t in_type, out_type;
  int32_t head;
  uint32_t unit0;  // first unit of this tensor in its launch
};

constexpr int kGradSlotsSmall = 48;   // launch arguments of 3 KB
constexpr int kGradSlots = 500;       // 32 KB (the most that a launch takes is 32,764 bytes)
template <int SLOTS>
struct GradList {
  GradEntry e[SLOTS];
  int32_t n;
  uint32_t units;
};

enum : int { kNormL1 = 1, kNormL2 = 2, kNormInf = 3 };

// The entry of a unit: the last one whose first unit is not past it.
template <int SLOTS>
__device__ __forceinline__ int entry_of(const GradList<SLOTS>& list, uint32_t unit) {
  int lo = 0, hi = list.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.e[mid].unit0 <= unit) lo = mid;
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

// A block's pass over one unit: f8(in offset, out offset) per vector of 8 and
// f1(...) per single element.  The first unit of a tensor also takes the
// elements before and after the vectors.
template <class F8, class F1>
__device__ __forceinline__ void walk_unit(const GradEntry& e, int64_t u, F8&& f8, F1&& f1) {
  const int64_t total = e.rows * e.cols, rows = e.rows, cols = e.cols;
  if (e.head < 0) {
    const int64_t hi = min(total, (u + 1) * kNormUnit);
    for (int64_t i = u * kNormUnit + threadIdx.x; i < hi; i += kNormThreads)
      f1(entry_at(i, rows, cols, e.in_ld), entry_at(i, rows, cols, e.out_ld));
    return;
  }
  const int64_t nvec = (total - e.head) >> 3;
  f8(u * (kNormUnit / 8) + threadIdx.x, nvec);
  if (u == 0) {
    const int64_t tail = e.head + 8 * nvec;
    int64_t i = threadIdx.x < 8 ? threadIdx.x : tail + threadIdx.x - 8;
    if (threadIdx.x < 8 ? i < e.head : threadIdx.x < 16 && i < total) f1(i, i);
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
  walk_unit(
      e, u,
      [&](int64_t first, int64_t nvec) {
        float v[kNormVecs * 8];
#pragma unroll
        for (int s = 0; s < kNormVecs; ++s) {
          const int64_t i = first + s * kNormThreads;
          if (i < nvec) {
            elem_load8(e.in, TYPE, entry_at(e.head + 8 * i, e.rows, e.cols, e.in_ld), v + 8 * s);
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x) v[8 * s + x] = 0.f;
          }
        }
        norm_add<NORM>(v, acc);
      },
      [&](int64_t in, int64_t) {
        const float v[1] = {elem_load(e.in, TYPE, in)};
        norm_add<NORM>(v, acc);
      });
}

template <int NORM, int SLOTS>
__global__ void __launch_bounds__(kNormThreads) norm_partial_kernel(const __grid_constant__ GradList<SLOTS> list,
                                                                    double* __restrict__ partial) {
  __shared__ double s_w[kNormThreads / 32];
  NormAcc acc{0.0, 0u};
  for (uint32_t unit = blockIdx.x; unit < list.units; unit += gridDim.x) {
    const GradEntry& e = list.e[entry_of(list, unit)];
    const int64_t u = unit - e.unit0;
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
template <int NORM>
__device__ __forceinline__ float norm_of(const double* partial, int n, double* s_w) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) v = NORM == kNormInf ? fmax(v, partial[i]) : v + partial[i];
  if (NORM == kNormInf) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) s_w[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x >> 5; ++w) v = fmax(v, s_w[w]);
    return __uint_as_float((uint32_t)v);  // the bits of |x|: whole numbers below 2^32
  }
  v = block_sum(v, s_w);
  return (float)(NORM == kNormL2 ? sqrt(v) : v);
}

template <int NORM>
__global__ void __launch_bounds__(kNormThreads) norm_finish_kernel(const double* partial, int n, float* norm) {
  __shared__ double s_w[kNormThreads / 32];
  const float v = norm_of<NORM>(partial, n, s_w);
  if (threadIdx.x == 0) *norm = v;
}

// ---------------------------------------------------------------- clip
// in may be out: plain loads (the read-only path is for memory that nobody
// writes during the kernel).
template <int TYPE>
__device__ __forceinline__ void clip_load8(const void* p, int64_t i, float* v) {
  if (TYPE == kElemF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = q[0], b = q[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    unpack16(a.x, TYPE, v[0], v[1]);
    unpack16(a.y, TYPE, v[2], v[3]);
    unpack16(a.z, TYPE, v[4], v[5]);
    unpack16(a.w, TYPE, v[6], v[7]);
  }
}
template <int TYPE>
__device__ __forceinline__ float clip_load(const void* p, int64_t i) {
  if (TYPE == kElemF32) return static_cast<const float*>(p)[i];
  const uint16_t u = static_cast<const uint16_t*>(p)[i];
  return TYPE == kElemBF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}

template <int IN, int OUT>
__device__ __forceinline__ void clip_unit(const GradEntry& e, int64_t u, float coef) {
  walk_unit(
      e, u,
      [&](int64_t first, int64_t nvec) {
        float v[kNormVecs * 8];
#pragma unroll
        for (int s = 0; s < kNormVecs; ++s) {
          const int64_t i = first + s * kNormThreads;
          if (i < nvec) clip_load8<IN>(e.in, entry_at(e.head + 8 * i, e.rows, e.cols, e.in_ld), v + 8 * s);
        }
#pragma unroll
        for (int s = 0; s < kNormVecs; ++s) {
          const int64_t i = first + s * kNormThreads;
          if (i >= nvec) continue;
#pragma unroll
          for (int x = 0; x < 8; ++x) v[8 * s + x] *= coef;
          elem_store8(e.out, OUT, entry_at(e.head + 8 * i, e.rows, e.cols, e.out_ld), v + 8 * s);
        }
      },
      [&](int64_t in, int64_t out) { elem_store(e.out, OUT, out, clip_load<IN>(e.in, in) * coef); });
}

struct ClipNorm {
  const double* partial;  // n partials of the norm, or
  int32_t n;
  const float* given;     // the norm itself
  float* norm;            // written by block 0 from the partials
  double max_norm;
};

template <int NORM, int SLOTS>
__global__ void __launch_bounds__(kNormThreads) clip_kernel(const __grid_constant__ GradList<SLOTS> list,
                                                            const ClipNorm c) {
  __shared__ double s_w[kNormThreads / 32];
  float norm;
  if (c.given) {
    norm = *c.given;
  } else {
    norm = norm_of<NORM>(c.partial, c.n, s_w);
    if (c.norm && blockIdx.x == 0 && threadIdx.x == 0) *c.norm = norm;
  }
  const double ratio = c.max_norm / ((double)norm + 1e-6);
  const float coef = ratio < 1.0 ? (float)ratio : ratio >= 1.0 ? 1.f : (float)ratio;  // NaN stays
  for (uint32_t i = blockIdx.x; i < list.units; i += gridDim.x) {
    const uint32_t unit = list.units - 1 - i;
    const GradEntry& e = list.e[entry_of(list, unit)];
    if (coef == 1.f && e.in == e.out && e.in_type == e.out_type) continue;  // in place, nothing to scale
    const int64_t u = unit - e.unit0;
    switch (e.in_type * 3 + e.out_type) {
      case 0: clip_unit<0, 0>(e, u, coef); break;
      case 1: clip_unit<0, 1>(e, u, coef); break;
      case 2: clip_unit<0, 2>(e, u, coef); break;
      case 3: clip_unit<1, 0>(e, u, coef); break;
      case 4: clip_unit<1, 1>(e, u, coef); break;
      case 5: clip_unit<1, 2>(e, u, coef); break;
      case 6: clip_unit<2, 0>(e, u, coef); break;
      case 7: clip_unit<2, 1>(e, u, coef); break;
      case 8: clip_unit<2, 2>(e, u, coef); break;
    }
  }
}

}  // namespace moe
