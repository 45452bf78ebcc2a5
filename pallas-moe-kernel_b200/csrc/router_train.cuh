// Top-k routing for training (sm_100a): expert choice, weights, per-expert
// counts, the balance loss and the z loss in one pass over the router logits,
// and the gradient of all of them in a second pass.
//
// With l the logits of a token (a row), p = softmax(l), s = sigmoid(l):
//   q        p (softmax scoring) or s / sum(s) (sigmoid scoring)
//   ids      the k largest logits, ties to the lower expert id; -1 where no
//            logit above -inf is left (or the ids the caller chose)
//   w_j      normalised: score_j / sum over the chosen scores; else the score
//            (p or s) itself
//   c_e, N   chosen entries per expert and tokens of a sequence
//   balance  mean over sequences of sum_e (c_e E / (k N)) (sum_t q_te / N)
//   z        mean over tokens of lse(l)^2
// A token that the mask leaves out, or whose logits are all -inf, takes no
// part: ids -1, weights 0, no share in any sum, gradient 0.
//
// Gradient: with f' = c_e E / (k N) - 1 (sum(q) = 1, so the constant drops
// out; c E - k N is formed in integers, which keeps the few bits that matter),
//   dl += dB / (S' N) q (f' - <f', q>) [(1 - s) for sigmoid scoring]
//       + dZ 2 lse p / N_all
//       + the weights' part on the chosen experts (route_backward_kernel).
//
// Layout: G lanes hold one row, V consecutive experts each (G V >= E), so
// small E packs 32 / G tokens in a warp and the expert order is the lane
// order: among equal maxima the lowest lane, then the lowest element, is the
// lowest id.  Sums over tokens stay in registers, then go warp by warp and
// block by block in a fixed order: no float atomics, results repeat bit for
// bit.  A block's tokens belong to one sequence.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "abi_util.h"
#include "ptx.cuh"

namespace moe {

enum : int { kElemF32 = 0, kElemBF16 = 1, kElemF16 = 2 };

constexpr int kRouteThreads = 256;
constexpr int kRouteWarps = kRouteThreads / 32;

struct RouteParams {
  const void* logits;      // (T, E), rows `ld` elements apart
  const uint8_t* mask;     // (T,) or null: 0 = the token takes no part
  const int32_t* given;    // (T, k) or null: ids chosen by the caller
  int32_t* ids;            // (T, k)
  float* weights;          // (T, k)
  float* part_q;           // [blocks][E] sums of q
  int32_t* part_c;         // [blocks][E] counts
  float* part_z;           // [blocks] sums of lse^2
  int32_t* part_n;         // [blocks] tokens
  uint32_t* ticket;        // zeroed here for route_finish_kernel
  int64_t ld;
  int64_t seq_len;         // tokens per sequence
  int32_t chunks;          // blocks per sequence
  int32_t E, k;
  int32_t type;            // kElem* of the logits
  int32_t vec;             // rows can be read in 16-byte vectors (8 elements at a time)
  int32_t sigmoid, normalize;
};

// ---------------------------------------------------------------- elements
__device__ __forceinline__ float elem_load(const void* p, int type, int64_t i) {
  if (type == kElemF32) return __ldg(static_cast<const float*>(p) + i);
  const uint16_t u = __ldg(static_cast<const uint16_t*>(p) + i);
  return type == kElemBF16 ? __uint_as_float((uint32_t)u << 16) : __half2float(__ushort_as_half(u));
}
__device__ __forceinline__ uint16_t elem_bits16(float v, int type) {
  return type == kElemBF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ void unpack16(uint32_t u, int type, float& a, float& b) {
  if (type == kElemBF16) {
    a = __uint_as_float(u << 16);
    b = __uint_as_float(u & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    a = f.x;
    b = f.y;
  }
}
// Eight consecutive elements from a 16-byte aligned address.
__device__ __forceinline__ void elem_load8(const void* p, int type, int64_t i, float* v) {
  if (type == kElemF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
    unpack16(a.x, type, v[0], v[1]);
    unpack16(a.y, type, v[2], v[3]);
    unpack16(a.z, type, v[4], v[5]);
    unpack16(a.w, type, v[6], v[7]);
  }
}
__device__ __forceinline__ uint32_t pack16(float a, float b, int type) {
  return (uint32_t)elem_bits16(a, type) | ((uint32_t)elem_bits16(b, type) << 16);
}
__device__ __forceinline__ void elem_store8(void* p, int type, int64_t i, const float* v) {
  if (type == kElemF32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(pack16(v[0], v[1], type), pack16(v[2], v[3], type), pack16(v[4], v[5], type),
                   pack16(v[6], v[7], type));
  }
}
__device__ __forceinline__ void elem_store(void* p, int type, int64_t i, float v) {
  if (type == kElemF32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = elem_bits16(v, type);
}

// Experts [e0, e0 + V) of the row at element offset `row`; -inf past E.
template <int V>
__device__ __forceinline__ void row_load(const void* p, int type, int vec, int64_t row, int e0, int E, bool live,
                                         float (&v)[V]) {
#pragma unroll
  for (int c = 0; c < V; c += 8) {
    if (live && vec && e0 + c < E) {
      elem_load8(p, type, row + e0 + c, v + c);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[c + i] = live && e0 + c + i < E ? elem_load(p, type, row + e0 + c + i) : -INFINITY;
    }
  }
}

template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// s_e e^-m with m = min(row maximum, 0): sigmoid scores of a row scaled so
// that a row of very negative logits keeps its ratios (unscaled, all of them
// would leave the f32 range).  r = e^(m - l) is kept for the slope.
struct SigmoidRow {
  float m, em;
  __device__ __forceinline__ explicit SigmoidRow(float mx) : m(fminf(mx, 0.f)), em(expf(fminf(mx, 0.f))) {}
  __device__ __forceinline__ float r(float l) const { return expf(m - l); }
  __device__ __forceinline__ float scaled(float r_) const { return 1.f / (em + r_); }
  // 1 - s = r / (e^m + r); r is infinite far below the maximum, where it is 1.
  __device__ __forceinline__ float slope(float r_) const { return r_ > 1e37f ? 1.f : r_ / (em + r_); }
};

// ---------------------------------------------------------------- forward
// Bounded by instruction issue rather than HBM at E = 256, k = 8 (k rounds of
// a maximum over the row); see the launch code for the group sizes.
template <int G, int V, int KMAX>
__global__ void __launch_bounds__(kRouteThreads) route_train_kernel(const RouteParams p) {
  constexpr int TPW = 32 / G;  // tokens per warp and step
  extern __shared__ int s_cnt[];  // [E] counts, then [warps][G V] sums of q
  __shared__ float s_z[kRouteWarps];
  __shared__ int s_n[kRouteWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % G;
  const uint32_t gmask = (G == 32 ? 0xffffffffu : ((1u << G) - 1u) << (lane / G * G));
  const int e0 = gl * V, E = p.E, k = p.k;
  for (int e = threadIdx.x; e < E; e += kRouteThreads) s_cnt[e] = 0;
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
  __syncthreads();

  const int64_t seq = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  const int64_t lo = seq * p.seq_len + p.seq_len * chunk / p.chunks;
  const int64_t hi = seq * p.seq_len + p.seq_len * (chunk + 1) / p.chunks;
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  float z = 0.f;
  int n = 0;
  for (int64_t base = lo + warp * TPW; base < hi; base += kRouteWarps * TPW) {
    const int64_t t = base + lane / G;
    const bool inside = t < hi;
    const bool live = inside && (!p.mask || __ldg(p.mask + t));
    float v[V];
    row_load<V>(p.logits, p.type, p.vec, t * p.ld, e0, E, live, v);
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < V; ++i) mx = fmaxf(mx, v[i]);
    mx = group_max<G>(mx);
    const bool keep = mx > -INFINITY;
    float ex[V], total = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      ex[i] = keep && e0 + i < E ? expf(v[i] - mx) : 0.f;
      total += ex[i];
    }
    total = group_sum<G>(total);
    const float lse = keep ? mx + logf(total) : 0.f;
    const SigmoidRow sg(mx);
    float norm = total;  // what the scores are divided by to give q
    if (p.sigmoid) {
      norm = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        ex[i] = keep && e0 + i < E ? sg.scaled(sg.r(v[i])) : 0.f;
        norm += ex[i];
      }
      norm = group_sum<G>(norm);
    }
    const float inv = keep ? 1.f / norm : 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += ex[i] * inv;
    if (gl == 0 && keep) {
      z += lse * lse;
      ++n;
    }

    // Choice: k rounds of the row's maximum, or the caller's ids.
    float sel[KMAX];
    if (!p.given) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = v[i] > -INFINITY ? v[i] : -INFINITY;  // NaN is never chosen
#pragma unroll
      for (int j = 0; j < KMAX; ++j) {
        if (j >= k) break;
        float m = v[0];
#pragma unroll
        for (int i = 1; i < V; ++i) m = fmaxf(m, v[i]);
        const float M = group_max<G>(m);
        const bool any = M > -INFINITY;
        const uint32_t owners = __ballot_sync(0xffffffffu, m == M) & gmask;
        int id = -1;
        if (lane == __ffs(owners) - 1) {
          if (any) {
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
              if (v[i] == M) id = i;
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (i == id) v[i] = -INFINITY;
            id += e0;
            atomicAdd(&s_cnt[id], 1);
          }
          if (inside) p.ids[t * k + j] = id;
        }
        sel[j] = M;
      }
    } else {
#pragma unroll
      for (int j = 0; j < KMAX; ++j) {
        if (j >= k) break;
        int id = live ? __ldg(p.given + t * k + j) : -1;
        if (!keep || id < 0 || id >= E) id = -1;
        sel[j] = id >= 0 ? elem_load(p.logits, p.type, t * p.ld + id) : -INFINITY;
        if (gl == 0 && inside) {
          p.ids[t * k + j] = id;
          if (id >= 0) atomicAdd(&s_cnt[id], 1);
        }
      }
    }
    // Weights of the chosen logits, on the row's own scale; normalised, the
    // softmax is taken relative to the largest chosen logit.
    float top = mx, sum = 0.f;
    if (p.normalize) {
      top = -INFINITY;
#pragma unroll
      for (int j = 0; j < KMAX; ++j)
        if (j < k) top = fmaxf(top, sel[j]);
    }
    const SigmoidRow sw(top);
#pragma unroll
    for (int j = 0; j < KMAX; ++j) {
      if (j >= k) break;
      // A chosen -inf (the caller's choice) has score 0; a slot without an
      // expert has sel = -inf as well.
      if (sel[j] == -INFINITY) sel[j] = 0.f;
      else sel[j] = p.sigmoid ? sw.scaled(sw.r(sel[j])) : expf(sel[j] - top);
      sum += sel[j];
    }
    const float scale = p.normalize ? (sum == 0.f ? 0.f : 1.f / sum) : p.sigmoid ? sw.em : inv;
#pragma unroll
    for (int j = 0; j < KMAX; ++j) {
      if (j >= k) break;
      if (gl == j % G && inside) p.weights[t * k + j] = sel[j] * scale;
    }
  }

  // Block sums: lanes of equal gl, then warps, in order.
#pragma unroll
  for (int o = G; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    z += __shfl_xor_sync(0xffffffffu, z, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  float* s_q = reinterpret_cast<float*>(s_cnt + E);
  if (lane < G) {
#pragma unroll
    for (int i = 0; i < V; ++i) s_q[warp * (G * V) + e0 + i] = acc[i];
  }
  if (lane == 0) {
    s_z[warp] = z;
    s_n[warp] = n;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) sum += s_q[w * (G * V) + e];
    p.part_q[(int64_t)blockIdx.x * E + e] = sum;
    p.part_c[(int64_t)blockIdx.x * E + e] = s_cnt[e];
  }
  if (threadIdx.x == 0) {
    float zs = 0.f;
    int ns = 0;
    for (int w = 0; w < kRouteWarps; ++w) {
      zs += s_z[w];
      ns += s_n[w];
    }
    p.part_z[blockIdx.x] = zs;
    p.part_n[blockIdx.x] = ns;
  }
}

// ---------------------------------------------------------------- finish
// Block (s, b): experts [32 b, 32 b + 32) of sequence s: counts, and the
// block's part of sum_e c_e P_e.  The block that finishes last adds the parts
// of all sequences in order (f64: the sums run over every block).
struct RouteFinish {
  const float* part_q;
  const int32_t* part_c;
  const float* part_z;
  const int32_t* part_n;
  uint32_t* ticket;
  double* seq_part;   // [S][blocks per sequence]
  int32_t* counts;    // (S, E)
  int32_t* tokens;    // (S,)
  float* balance;
  float* z;
  int32_t S, chunks, E, k, eblocks;
};

constexpr int kFinishThreads = 512;

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the block, valid in every thread; s_w holds one value per warp.
__device__ __forceinline__ double block_sum(double v, double* s_w) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  v = warp_sum(v);
  __syncthreads();
  if (lane == 0) s_w[warp] = v;
  __syncthreads();
  double sum = 0.0;
  for (int w = 0; w < nw; ++w) sum += s_w[w];
  return sum;
}

__global__ void __launch_bounds__(kFinishThreads) route_finish_kernel(const RouteFinish p) {
  constexpr int R = kFinishThreads / 32;  // partial rows read at a time
  __shared__ double s_q[R][32];
  __shared__ int s_c[R][32];
  __shared__ double s_w[R];
  __shared__ int s_last;
  const int lane = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int s = blockIdx.x / p.eblocks, eb = blockIdx.x % p.eblocks;
  const int e = eb * 32 + lane;
  const int64_t b0 = (int64_t)s * p.chunks;
  double q = 0.0;
  int c = 0;
  if (e < p.E) {
    for (int i = r; i < p.chunks; i += R) {
      q += (double)p.part_q[(b0 + i) * p.E + e];
      c += p.part_c[(b0 + i) * p.E + e];
    }
  }
  double n = 0.0;
  for (int i = threadIdx.x; i < p.chunks; i += kFinishThreads) n += p.part_n[b0 + i];
  n = block_sum(n, s_w);
  s_q[r][lane] = q;
  s_c[r][lane] = c;
  __syncthreads();
  if (r == 0) {
    for (int i = 1; i < R; ++i) {
      q += s_q[i][lane];
      c += s_c[i][lane];
    }
    if (e < p.E) p.counts[(int64_t)s * p.E + e] = c;
    const double sum = warp_sum(n > 0.0 ? (double)c * p.E / (p.k * n) * (q / n) : 0.0);
    if (lane == 0) {
      p.seq_part[blockIdx.x] = sum;
      if (eb == 0) p.tokens[s] = (int)n;
      __threadfence();
      s_last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
    }
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double bal = 0.0, z = 0.0, tokens = 0.0, live = 0.0;
  for (int64_t i = threadIdx.x; i < (int64_t)p.S * p.eblocks; i += kFinishThreads) bal += __ldcg(p.seq_part + i);
  for (int64_t i = threadIdx.x; i < (int64_t)p.S * p.chunks; i += kFinishThreads) z += p.part_z[i];
  for (int i = threadIdx.x; i < p.S; i += kFinishThreads) {
    const int ns = __ldcg(p.tokens + i);
    tokens += ns;
    live += ns > 0;
  }
  bal = block_sum(bal, s_w);
  z = block_sum(z, s_w);
  tokens = block_sum(tokens, s_w);
  live = block_sum(live, s_w);
  if (threadIdx.x == 0) {
    *p.balance = (float)(live > 0.0 ? bal / live : 0.0);
    *p.z = (float)(tokens > 0.0 ? z / tokens : 0.0);
  }
}

// ---------------------------------------------------------------- backward
struct RouteBackward {
  const void* logits;
  const uint8_t* mask;
  const int32_t* ids;      // (T, k) from the forward
  const float* weights;    // (T, k) from the forward
  const int32_t* counts;   // (S, E)
  const int32_t* tokens;   // (S,)
  const float* d_weights;  // (T, k) or null
  const float* d_balance;  // scalar or null
  const float* d_z;        // scalar or null
  void* d_logits;          // (T, E), contiguous, the logits' type
  int64_t ld, seq_len;
  int32_t S, chunks, E, k, type, vec, vec_out;
  int32_t sigmoid, normalize;
};

// The weights' part, on the chosen experts (j, with <.> over the row's slots):
//   normalised                   w_j (dw_j - <dw, w>) (times 1 - s_j, sigmoid)
//   plain softmax probability    w_j dw_j, and -p_e <dw, w> on every expert
//   plain sigmoid                w_j dw_j (1 - s_j)
template <int G, int V>
__global__ void __launch_bounds__(kRouteThreads) route_backward_kernel(const RouteBackward p) {
  constexpr int TPW = 32 / G;
  __shared__ int s_sum[2][kRouteWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % G;
  const int e0 = gl * V, E = p.E, k = p.k;
  const int64_t seq = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
  const int64_t lo = seq * p.seq_len + p.seq_len * chunk / p.chunks;
  const int64_t hi = seq * p.seq_len + p.seq_len * (chunk + 1) / p.chunks;

  // Tokens in all sequences and sequences with any.
  int all = 0, live_seqs = 0;
  for (int i = threadIdx.x; i < p.S; i += kRouteThreads) {
    const int ns = __ldg(p.tokens + i);
    all += ns;
    live_seqs += ns > 0;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    live_seqs += __shfl_xor_sync(0xffffffffu, live_seqs, o);
  }
  if (lane == 0) {
    s_sum[0][warp] = all;
    s_sum[1][warp] = live_seqs;
  }
  __syncthreads();
  all = live_seqs = 0;
  for (int w = 0; w < kRouteWarps; ++w) {
    all += s_sum[0][w];
    live_seqs += s_sum[1][w];
  }
  const int ns = __ldg(p.tokens + seq);
  // dB / (S' N) (1 / (k N)) (c E - k N): the integer part is exact.
  const float db = p.d_balance && ns > 0 ? __ldg(p.d_balance) / ((float)live_seqs * (float)ns) : 0.f;
  const float dz = p.d_z && all > 0 ? 2.f * __ldg(p.d_z) / (float)all : 0.f;
  float f[V];
  const float kn = (float)((int64_t)k * (ns > 0 ? ns : 1));
#pragma unroll
  for (int i = 0; i < V; ++i)
    f[i] = e0 + i < E ? (float)((int64_t)__ldg(p.counts + seq * E + e0 + i) * E - (int64_t)k * ns) / kn : 0.f;

  for (int64_t base = lo + warp * TPW; base < hi; base += kRouteWarps * TPW) {
    const int64_t t = base + lane / G;
    const bool inside = t < hi;
    const bool live = inside && (!p.mask || __ldg(p.mask + t));
    float v[V];
    row_load<V>(p.logits, p.type, p.vec, t * p.ld, e0, E, live, v);
    float mx = v[0];
#pragma unroll
    for (int i = 1; i < V; ++i) mx = fmaxf(mx, v[i]);
    mx = group_max<G>(mx);
    const bool keep = mx > -INFINITY;
    float d[V], slope[V];
    // Softmax part: p, and with softmax scoring q = p.
    float total = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      d[i] = keep && e0 + i < E ? expf(v[i] - mx) : 0.f;
      total += d[i];
    }
    total = group_sum<G>(total);
    const float inv = keep ? 1.f / total : 0.f;
    const float zl = keep ? dz * (mx + logf(total)) : 0.f;
    // <dw, w> over the slots in use.
    float dot = 0.f;
    if (p.d_weights && inside) {
      for (int j = 0; j < k; ++j)
        if (__ldg(p.ids + t * k + j) >= 0) dot += __ldg(p.d_weights + t * k + j) * __ldg(p.weights + t * k + j);
    }
    if (!p.sigmoid) {
      float fq = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        d[i] *= inv;
        fq += f[i] * d[i];
        slope[i] = 1.f;
      }
      fq = group_sum<G>(fq);
      const float extra = zl - (p.normalize ? 0.f : dot);
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] *= db * (f[i] - fq) + extra;
    } else {
      const SigmoidRow sg(mx);
      float q[V], norm = 0.f, fq = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float r = sg.r(v[i]);
        q[i] = keep && e0 + i < E ? sg.scaled(r) : 0.f;
        slope[i] = sg.slope(r);
        norm += q[i];
        fq += f[i] * q[i];
      }
      norm = group_sum<G>(norm);
      fq = group_sum<G>(fq);
      const float qi = keep ? 1.f / norm : 0.f;
      fq *= qi;
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = d[i] * inv * zl + db * (q[i] * qi) * (f[i] - fq) * slope[i];
    }
    if (p.d_weights && keep) {
      const float off = p.normalize ? dot : 0.f;
      for (int j = 0; j < k; ++j) {
        const int at = __ldg(p.ids + t * k + j) - e0;
        if (at < 0 || at >= V) continue;
        const float g = __ldg(p.weights + t * k + j) * (__ldg(p.d_weights + t * k + j) - off);
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (i == at) d[i] += g * slope[i];
      }
    }
    if (!inside) continue;
#pragma unroll
    for (int c = 0; c < V; c += 8) {
      if (!keep) {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[c + i] = 0.f;
      }
      if (p.vec_out) {
        if (e0 + c < E) elem_store8(p.d_logits, p.type, t * E + e0 + c, d + c);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e0 + c + i < E) elem_store(p.d_logits, p.type, t * E + e0 + c + i, d[c + i]);
      }
    }
  }
}

}  // namespace moe
