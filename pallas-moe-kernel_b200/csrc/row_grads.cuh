// Backward of the row movement around the expert MLP (sm_100a): gather_rows
// and combine_rows of router.cuh.
//
//   combine_bwd_kernel  Y[t] = sum_j w[t, j] Ys[inverse[t, j]] gives
//                       dYs[inverse[t, j]] = w[t, j] dY[t] and
//                       dw[t, j] = <dY[t], Ys[inverse[t, j]]>.
//   gather_bwd_kernel   Xs[inverse[t, j]] = X[t] gives
//                       dX[t] = sum_j dXs[inverse[t, j]], in slot order.
//
// Both are HBM-bound: every row is read or written once, a token's dY row is
// read once for its k slots.  TPT threads share a token and walk its row in
// 4-element vectors (16 bytes of f32, 8 of the 16-bit types); dot products are
// summed in f32 per thread and then across the threads in a fixed order.
#pragma once
#include <cstdint>

#include "ptx.cuh"
#include "router_train.cuh"

namespace moe {

constexpr int kRowThreads = 256;
constexpr int kRowSlots = 8;  // slots whose rows are in flight together

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
  const int32_t* group_sizes;  // (E,)
  void* dys;                // (rows, D)
  float* dw;                // (T, k)
  int64_t T, rows;
  int32_t k, D, E;
  int32_t token_blocks;     // blocks past these zero the rows behind sum(group_sizes)
};

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

template <int TPT, int DY, int DYS>
__global__ void __launch_bounds__(kRowThreads) combine_bwd_kernel(const CombineBwd p) {
  __shared__ float s_w[kRowThreads / 32];
  const int n4 = p.D >> 2;
  if (blockIdx.x >= p.token_blocks) {
    // Rows behind the last routed one take no part: zero.
    __shared__ int s_total;
    if (threadIdx.x < 32) {
      int64_t sum = 0;
      for (int e = threadIdx.x; e < p.E; e += 32) {
        const int g = __ldg(p.group_sizes + e);
        sum += g > 0 ? g : 0;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (threadIdx.x == 0) s_total = (int)(sum < p.rows ? sum : p.rows);
    }
    __syncthreads();
    const int zb = gridDim.x - p.token_blocks;
    for (int64_t i = (int64_t)s_total * n4 + (blockIdx.x - p.token_blocks) * kRowThreads + threadIdx.x; i < p.rows * n4;
         i += (int64_t)zb * kRowThreads)
      row_store4<DYS>(p.dys, i, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  const int k = p.k, me = threadIdx.x % TPT;
  const int64_t t = (int64_t)blockIdx.x * (kRowThreads / TPT) + threadIdx.x / TPT;
  const bool inside = t < p.T;
  for (int j0 = 0; j0 < k; j0 += kRowSlots) {
    int64_t row[kRowSlots];
    float w[kRowSlots], dot[kRowSlots];
#pragma unroll
    for (int j = 0; j < kRowSlots; ++j) {
      const bool on = inside && j0 + j < k;
      const int r = on ? __ldg(p.inverse + t * k + j0 + j) : -1;
      row[j] = r >= 0 && r < p.rows ? (int64_t)r * n4 : -1;
      w[j] = row[j] >= 0 ? __ldg(p.weights + t * k + j0 + j) : 0.f;
      dot[j] = 0.f;
    }
    for (int c = me; c < n4; c += TPT) {
      const float4 g = inside ? row_load4<DY>(p.dy, t * n4 + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      float4 y[kRowSlots];
#pragma unroll
      for (int j = 0; j < kRowSlots; ++j)
        if (row[j] >= 0) y[j] = row_load4<kElemF32>(p.y_sorted, row[j] + c);
#pragma unroll
      for (int j = 0; j < kRowSlots; ++j) {
        if (row[j] < 0) continue;
        dot[j] += g.x * y[j].x + g.y * y[j].y + (g.z * y[j].z + g.w * y[j].w);
        row_store4<DYS>(p.dys, row[j] + c, make_float4(w[j] * g.x, w[j] * g.y, w[j] * g.z, w[j] * g.w));
      }
    }
#pragma unroll
    for (int j = 0; j < kRowSlots; ++j) {
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

template <int TPT, int DXS, int DX>
__global__ void __launch_bounds__(kRowThreads) gather_bwd_kernel(const GatherBwd p) {
  const int n4 = p.D >> 2, k = p.k, me = threadIdx.x % TPT;
  const int64_t t = (int64_t)blockIdx.x * (kRowThreads / TPT) + threadIdx.x / TPT;
  if (t >= p.T) return;
  for (int c = me; c < n4; c += TPT) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < k; j0 += kRowSlots) {
      float4 v[kRowSlots];
#pragma unroll
      for (int j = 0; j < kRowSlots; ++j) {
        const int r = j0 + j < k ? __ldg(p.inverse + t * k + j0 + j) : -1;
        v[j] = r >= 0 && r < p.rows ? row_load4<DXS>(p.dxs, (int64_t)r * n4 + c) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < kRowSlots; ++j) {
        acc.x += v[j].x;
        acc.y += v[j].y;
        acc.z += v[j].z;
        acc.w += v[j].w;
      }
    }
    row_store4<DX>(p.dx, t * n4 + c, acc);
  }
}

}  // namespace moe
