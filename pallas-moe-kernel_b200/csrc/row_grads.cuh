// Backward of the row movement around the expert MLP (sm_100a): gather_rows
// and combine_rows of router.cuh.
//
//   combine_bwd_kernel  Y[t] = sum_j w[t, j] Ys[inverse[t, j]] gives
//                       dYs[inverse[t, j]] = w[t, j] dY[t] and
//                       dw[t, j] = <dY[t], Ys[inverse[t, j]]>; rows of dYs
//                       that no entry maps to are 0.
//   gather_bwd_kernel   Xs[inverse[t, j]] = X[t] gives
//                       dX[t] = sum_j dXs[inverse[t, j]], in slot order.
//
// Both are HBM-bound: every row is read or written once, a token's dY row is
// read once for its k slots.  TPT threads share a token and walk its row in
// 4-element vectors (16 bytes of f32, 8 of the 16-bit types); dot products are
// summed in f32 per thread and then across the threads in a fixed order.
// Measured against the 6547 GB/s of a copy: combine at T = 8192, k = 8,
// D = 7168 (f32, bf16 out) 461 to 475 us = 0.98 to 1.01, gather at T = 16384,
// k = 2, D = 4096 (f32, bf16 out) 100 us = 1.02.
#pragma once
#include <cstdint>

#include "ptx.cuh"
#include "router_train.cuh"

namespace moe {

constexpr int kRowThreads = 256;
constexpr int kRowSlots = 8;  // vectors of expert rows in flight per thread: 8 slots, or fewer with more vectors each

template <int TYPE>
__device__ __forceinline__ float4 row_load4(const void* p, int64_t i4) {
  if (TYPE == kElemF32) return __ldg(static_cast<const float4*>(p) + i4);
  const uint2 u = __ldg(static_cast<const uint2*>(p) + i4);
  float4 v;
  unpack16(u.x, TYPE, v.x, v.y);
  unpack16(u.y, TYPE, v.z, v.w);
  return v;
}
template <int TYPE>
__device__ __forceinline__ void row_store4(void* p, int64_t i4, float4 v) {
  if (TYPE == kElemF32) static_cast<float4*>(p)[i4] = v;
  else static_cast<uint2*>(p)[i4] = make_uint2(pack16(v.x, v.y, TYPE), pack16(v.z, v.w, TYPE));
}

struct CombineBwd {
  const void* dy;           // (T, D)
  const float* y_sorted;    // (rows, D)
  const int32_t* inverse;   // (T, k)
  const float* weights;     // (T, k)
  void* dys;                // (rows, D)
  float* dw;                // (T, k)
  int64_t T, rows;
  int32_t k, D;
  int32_t zero_blocks;      // the first blocks, 0 or 2^zero_shift: zero the rows that no entry maps to
  int32_t zero_shift;
};

constexpr int kZeroRows = 32768;  // most rows of a zeroing block: a bit each in shared memory (4 KB)

// Zeroing blocks where kZeroRows allows as few: 2^this.  Each reads all of
// `inverse`, so fewer for short rows (T = 32768, k = 16: D = 128 to bf16 94 us
// without any, 101 with 32, 108 with 64, 122 with one per SM; D = 256 to f32 185,
// 193, 199, 262); long rows need more for their stores (T = 4096, k = 8, D = 512,
// nine tokens in ten dropped: 45 us with 32, 29 with 64; T = 8192, D = 7168 481
// and 318, with none dropped 461 like without).
constexpr int zero_shift_most(int D) { return D >= 512 ? 6 : 5; }

// The rows of dys that no entry maps to (behind the last routed row, or dropped
// after the permutation): zero.  A zeroing block looks through all of `inverse`
// and marks what falls into its rows, beside the tokens' blocks; blocks take 32
// rows in turn, so that a tail of padding is shared.  A call, not inlined: with
// it in the kernel the tokens' loop got 30 registers less and ran 15% longer.
template <int DYS>
__device__ __noinline__ void zero_unmapped(const CombineBwd& p, uint32_t* s_map) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int shift = p.zero_shift;
  const int64_t n = p.T * p.k;
  const uint32_t me = blockIdx.x, all = (uint32_t)((p.rows + 31) >> 5);          // words of 32 rows
  const uint32_t words = all > me ? (all - me - 1 >> shift) + 1 : 0;             // this block's: me, me + 2^shift, ...
  for (uint32_t w = threadIdx.x; w < words; w += kRowThreads) s_map[w] = 0;
  __syncthreads();
  const auto mark = [&](int r) {
    const uint32_t w = (uint32_t)r >> 5;
    if ((w & ((1u << shift) - 1u)) == me && (uint32_t)r < (uint32_t)p.rows)
      atomicOr(s_map + (w >> shift), 1u << (r & 31));
  };
  // Entries in fours from the first 16-byte boundary on, eight fours in flight.
  const int64_t head = min(n, (int64_t)((0 - (reinterpret_cast<uintptr_t>(p.inverse) >> 2)) & 3));
  const int64_t fours = (n - head) / 4, tail = head + 4 * fours;
  if (threadIdx.x < head) mark(__ldg(p.inverse + threadIdx.x));
  if (threadIdx.x < n - tail) mark(__ldg(p.inverse + tail + threadIdx.x));
  const int4* body = reinterpret_cast<const int4*>(p.inverse + head);
  constexpr int kAhead = 8;
  for (int64_t i0 = threadIdx.x; i0 < fours; i0 += kAhead * kRowThreads) {
    int4 r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      r[u] = i0 + u * kRowThreads < fours ? __ldg(body + i0 + u * kRowThreads) : make_int4(-1, -1, -1, -1);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) mark(r[u].x), mark(r[u].y), mark(r[u].z), mark(r[u].w);
  }
  __syncthreads();
  // Stores of 16 bytes where a row is made of them, else of 8 (the 16-bit types).
  const int64_t row_bytes = (int64_t)p.D * (DYS == kElemF32 ? 4 : 2);
  const bool wide = ((row_bytes | reinterpret_cast<intptr_t>(p.dys)) & 15) == 0;
  for (uint32_t w = warp; w < words; w += kRowThreads / 32) {
    uint32_t left = ~s_map[w];
    const int64_t row0 = (int64_t)((w << shift) + me) * 32;
    if (row0 + 32 > p.rows) left &= (1u << (p.rows & 31)) - 1u;
    for (; left; left &= left - 1) {
      uint8_t* row = static_cast<uint8_t*>(p.dys) + (row0 + __ffs(left) - 1) * row_bytes;
      if (wide) {
#pragma unroll 4
        for (int c = lane; c < (int)(row_bytes >> 4); c += 32) reinterpret_cast<uint4*>(row)[c] = make_uint4(0, 0, 0, 0);
      } else {
        for (int c = lane; c < (int)(row_bytes >> 3); c += 32) reinterpret_cast<uint2*>(row)[c] = make_uint2(0, 0);
      }
    }
  }
}

// The sum over a token's TPT threads, valid in the first of them.
template <int TPT>
__device__ __forceinline__ float token_sum(float v, float* s_w) {
#pragma unroll
  for (int o = (TPT < 32 ? TPT : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (TPT > 32) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    if (lane == 0) s_w[warp] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TPT / 32; ++w) v += s_w[(threadIdx.x / TPT) * (TPT / 32) + w];
  }
  return v;
}

template <int TPT, int DY, int DYS, int SLOTS>
__global__ void __launch_bounds__(kRowThreads) combine_bwd_kernel(const __grid_constant__ CombineBwd p) {
  constexpr int U = kRowSlots / SLOTS;
  __shared__ float s_w[kRowThreads / 32];
  __shared__ uint32_t s_map[kZeroRows / 32];
  const int n4 = p.D >> 2;
  if (blockIdx.x < p.zero_blocks) {
    zero_unmapped<DYS>(p, s_map);
    return;
  }
  const int k = p.k, me = threadIdx.x % TPT;
  const int64_t t = (int64_t)(blockIdx.x - p.zero_blocks) * (kRowThreads / TPT) + threadIdx.x / TPT;
  const bool inside = t < p.T;
  for (int j0 = 0; j0 < k; j0 += SLOTS) {
    int64_t row[SLOTS];
    float w[SLOTS], dot[SLOTS];
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      const bool on = inside && j0 + j < k;
      const int r = on ? __ldg(p.inverse + t * k + j0 + j) : -1;
      row[j] = r >= 0 && r < p.rows ? (int64_t)r * n4 : -1;
      w[j] = row[j] >= 0 ? __ldg(p.weights + t * k + j0 + j) : 0.f;
      dot[j] = 0.f;
    }
    for (int c0 = me; inside && c0 < n4; c0 += U * TPT) {
      float4 g[U], y[SLOTS][U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + u * TPT < n4) g[u] = row_load4<DY>(p.dy, t * n4 + c0 + u * TPT);
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (row[j] >= 0 && c0 + u * TPT < n4) y[j][u] = row_load4<kElemF32>(p.y_sorted, row[j] + c0 + u * TPT);
      }
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        if (row[j] < 0) continue;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (c0 + u * TPT >= n4) continue;
          dot[j] += g[u].x * y[j][u].x + g[u].y * y[j][u].y + (g[u].z * y[j][u].z + g[u].w * y[j][u].w);
          row_store4<DYS>(p.dys, row[j] + c0 + u * TPT,
                          make_float4(w[j] * g[u].x, w[j] * g[u].y, w[j] * g[u].z, w[j] * g[u].w));
        }
      }
    }
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
      if (j0 + j >= k) break;
      const float sum = token_sum<TPT>(dot[j], s_w);
      if (inside && me == 0) p.dw[t * k + j0 + j] = sum;
    }
  }
}

struct GatherBwd {
  const void* dxs;         // (rows, D)
  const int32_t* inverse;  // (T, k)
  void* dx;                // (T, D)
  int64_t T, rows;
  int32_t k, D;
};

// VEC elements of a row, as they are in memory until they are added: 4, or 8
// of the 16-bit types where rows allow 16-byte loads (8-byte loads ran the
// bf16 gather at k = 8, D = 7168 at 5.3 TB/s, these at 6.5).
template <int TYPE, int VEC>
struct RawVec {
  uint4 r;
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    if (TYPE == kElemF32 || VEC == 8) {
      r = __ldg(static_cast<const uint4*>(p) + i);
    } else {
      const uint2 u = __ldg(static_cast<const uint2*>(p) + i);
      r = make_uint4(u.x, u.y, 0, 0);
    }
  }
  __device__ __forceinline__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void add_to(float (&acc)[VEC]) const {
    float v[8];
    if (TYPE == kElemF32) {
      v[0] = __uint_as_float(r.x), v[1] = __uint_as_float(r.y), v[2] = __uint_as_float(r.z), v[3] = __uint_as_float(r.w);
    } else {
      unpack16(r.x, TYPE, v[0], v[1]);
      unpack16(r.y, TYPE, v[2], v[3]);
      unpack16(r.z, TYPE, v[4], v[5]);
      unpack16(r.w, TYPE, v[6], v[7]);
    }
#pragma unroll
    for (int x = 0; x < VEC; ++x) acc[x] += v[x];
  }
};
template <int TYPE, int VEC>
__device__ __forceinline__ void vec_store(void* p, int64_t i, const float (&v)[VEC]) {
  if (TYPE != kElemF32 && VEC == 8) {
    static_cast<uint4*>(p)[i] = make_uint4(pack16(v[0], v[1], TYPE), pack16(v[2], v[3], TYPE),
                                           pack16(v[4 % VEC], v[5 % VEC], TYPE), pack16(v[6 % VEC], v[7 % VEC], TYPE));
  } else {
#pragma unroll
    for (int x = 0; x < VEC; x += 4)
      row_store4<TYPE>(p, i * (VEC / 4) + x / 4, make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]));
  }
}

// SLOTS rows of a token and 8 / SLOTS vectors of each are in flight per thread.
template <int TPT, int DXS, int DX, int SLOTS, int VEC>
__global__ void __launch_bounds__(kRowThreads) gather_bwd_kernel(const GatherBwd p) {
  constexpr int U = VEC == 8 && SLOTS == 2 ? 2 : kRowSlots / SLOTS;
  const int n = p.D / VEC, k = p.k, me = threadIdx.x % TPT;
  const int64_t t = (int64_t)blockIdx.x * (kRowThreads / TPT) + threadIdx.x / TPT;
  if (t >= p.T) return;
  for (int c0 = me; c0 < n; c0 += U * TPT) {
    float acc[U][VEC] = {};
    for (int j0 = 0; j0 < k; j0 += SLOTS) {
      RawVec<DXS, VEC> v[SLOTS][U];
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
        const int r = j0 + j < k ? __ldg(p.inverse + t * k + j0 + j) : -1;
        const bool on = r >= 0 && r < p.rows;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (on && c0 + u * TPT < n) v[j][u].load(p.dxs, (int64_t)r * n + c0 + u * TPT);
          else v[j][u].zero();
        }
      }
#pragma unroll
      for (int j = 0; j < SLOTS; ++j) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[j][u].add_to(acc[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (c0 + u * TPT < n) vec_store<DX, VEC>(p.dx, t * n + c0 + u * TPT, acc[u]);
  }
}

}  // namespace moe
