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
// lowest id.  Slot j of a row (its j-th choice) lives in lane j % G, so that
// ids, weights and their gradients move coalesced and their exponentials run
// side by side.  Exponentials are 2^(x log2 e) with the row maximum taken off
// before the rounding.
//
// Sums over tokens stay in registers, then go warp by warp and block by block
// in a fixed order: no float atomics, results repeat bit for bit.  A block's
// tokens belong to one sequence.  The blocks that finish last add up what the
// others wrote - 16 blocks, then a sequence, then all - found by counters that
// are zero between calls, which saves a second launch (9 us of a 15 us
// forward at T = 16384, E = 8).
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
constexpr int kRouteGroup = 16;  // blocks whose sums are added first

struct RouteParams {
  const void* logits;      // (T, E), rows `ld` elements apart
  const uint8_t* mask;     // (T,) or null: 0 = the token takes no part
  const int32_t* given;    // (T, k) or null: ids chosen by the caller
  int32_t* ids;            // (T, k)
  float* weights;          // (T, k)
  int32_t* counts;         // (S, E)
  int32_t* tokens;         // (S,)
  float* balance;
  float* z;
  float* part_q;           // [blocks][E] sums of q
  int32_t* part_c;         // [blocks][E] counts
  double* part_z;          // [blocks] sums of lse^2
  int32_t* part_n;         // [blocks] tokens
  double* seq_part;        // [S] sum of c_e P_e terms
  uint32_t* counters;      // [S groups][S][1], zero before and after
  int64_t ld;
  int64_t seq_len;         // tokens per sequence
  int32_t S, chunks;       // sequences, blocks per sequence
  int32_t E, k;
  int32_t type;            // kElem* of the logits
  int32_t vec;             // elements of a row read at a time: 8, 4 or 1
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
__device__ __forceinline__ uint32_t pack16(float a, float b, int type) {
  uint32_t r;
  if (type == kElemBF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ void elem_store(void* p, int type, int64_t i, float v) {
  if (type == kElemF32) static_cast<float*>(p)[i] = v;
  else static_cast<uint16_t*>(p)[i] = elem_bits16(v, type);
}

// Rows are held as pairs: sm_100 adds and multiplies two f32 at a time.
template <int V>
struct Row {
  float2 p[V / 2];
};

// Experts [e0, e0 + V) of the row at element offset `row`; -inf past E, and
// throughout for a row that is not live.  The types are told apart once per
// row: a choice inside the conversions costs more than they do.
// `vec`: elements that every row can be read and written in at a time: 8 (16
// bytes of the 16-bit types, two times 16 of f32), 4 or 1.
template <int TYPE, int V>
__device__ __forceinline__ void row_load_t(const void* p, int vec, int64_t row, int e0, int E, bool live, Row<V>& v) {
  constexpr uint32_t none = TYPE == kElemBF16 ? 0xff80ff80u : 0xfc00fc00u;  // -inf twice
  if (vec == 8 && TYPE != kElemF32) {
#pragma unroll
    for (int c = 0; c < V; c += 8) {
      uint4 a = make_uint4(none, none, none, none);
      if (live && e0 + c < E) a = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + row + e0 + c));
      unpack16(a.x, TYPE, v.p[c / 2].x, v.p[c / 2].y);
      unpack16(a.y, TYPE, v.p[c / 2 + 1].x, v.p[c / 2 + 1].y);
      unpack16(a.z, TYPE, v.p[c / 2 + 2].x, v.p[c / 2 + 2].y);
      unpack16(a.w, TYPE, v.p[c / 2 + 3].x, v.p[c / 2 + 3].y);
    }
  } else if (vec >= 4) {
#pragma unroll
    for (int c = 0; c < V; c += 4) {
      const bool on = live && e0 + c < E;
      if (TYPE == kElemF32) {
        float4 a = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (on) a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + row + e0 + c));
        v.p[c / 2] = make_float2(a.x, a.y), v.p[c / 2 + 1] = make_float2(a.z, a.w);
      } else {
        uint2 a = make_uint2(none, none);
        if (on) a = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + row + e0 + c));
        unpack16(a.x, TYPE, v.p[c / 2].x, v.p[c / 2].y);
        unpack16(a.y, TYPE, v.p[c / 2 + 1].x, v.p[c / 2 + 1].y);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float x = live && e0 + i < E ? elem_load(p, TYPE, row + e0 + i) : -INFINITY;
      (i & 1 ? v.p[i / 2].y : v.p[i / 2].x) = x;
    }
  }
}
template <int V>
__device__ __forceinline__ void row_load(const void* p, int type, int vec, int64_t row, int e0, int E, bool live,
                                         Row<V>& v) {
  if (type == kElemF32) row_load_t<kElemF32>(p, vec, row, e0, E, live, v);
  else if (type == kElemBF16) row_load_t<kElemBF16>(p, vec, row, e0, E, live, v);
  else row_load_t<kElemF16>(p, vec, row, e0, E, live, v);
}
// A warp's rows in shared memory, 32 V floats in fours: four q of lane l lies
// at q * 32 + (l ^ q * 32 / V), which neither the lanes' own fours (one q, all
// lanes) nor fours in the order of the experts (all q of a lane, next lane)
// find in one bank.
template <int V>
__device__ __forceinline__ int four_at(int l, int q) {
  return q * 32 + (l ^ (q * (32 / V)));
}

// Stores the warp's 32 / G rows from shared memory, neighbouring lanes
// neighbouring experts: a lane's own V experts written in 16-byte pieces are
// half sectors, twice as many requests.
template <int TYPE, int G, int V>
__device__ __forceinline__ void rows_store_t(const float4* s_fours, void* p, int vec, int64_t t0, int64_t hi, int E,
                                             int lane) {
  if (vec == 8 && TYPE != kElemF32) {
#pragma unroll
    for (int i = 0; i < V / 8; ++i) {
      const int at = i * 32 + lane, l = at / (V / 8), e = 8 * (at % (G * V / 8));
      const int64_t t = t0 + l / G;
      if (t >= hi || e >= E) continue;
      const float4 x = s_fours[four_at<V>(l, 2 * (at % (V / 8)))], y = s_fours[four_at<V>(l, 2 * (at % (V / 8)) + 1)];
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + t * E + e) =
          make_uint4(pack16(x.x, x.y, TYPE), pack16(x.z, x.w, TYPE), pack16(y.x, y.y, TYPE), pack16(y.z, y.w, TYPE));
    }
  } else if (vec >= 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const int at = i * 32 + lane, l = at / (V / 4), e = 4 * (at % (G * V / 4));
      const int64_t t = t0 + l / G;
      if (t >= hi || e >= E) continue;
      const float4 x = s_fours[four_at<V>(l, at % (V / 4))];
      if (TYPE == kElemF32)
        *reinterpret_cast<float4*>(static_cast<float*>(p) + t * E + e) = x;
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + t * E + e) =
            make_uint2(pack16(x.x, x.y, TYPE), pack16(x.z, x.w, TYPE));
    }
  } else {
    for (int i = 0; i < V; ++i) {
      const int at = i * 32 + lane, l = at / V, e = at % (G * V);
      const int64_t t = t0 + l / G;
      if (t < hi && e < E)
        elem_store(p, TYPE, t * E + e, reinterpret_cast<const float*>(s_fours + four_at<V>(l, at % V / 4))[at % 4]);
    }
  }
}
template <int G, int V>
__device__ __forceinline__ void rows_store(const float4* s_fours, void* p, int type, int vec, int64_t t0, int64_t hi,
                                           int E, int lane) {
  if (type == kElemF32) rows_store_t<kElemF32, G, V>(s_fours, p, vec, t0, hi, E, lane);
  else if (type == kElemBF16) rows_store_t<kElemBF16, G, V>(s_fours, p, vec, t0, hi, E, lane);
  else rows_store_t<kElemF16, G, V>(s_fours, p, vec, t0, hi, E, lane);
}
template <int V>
__device__ __forceinline__ void row_fill(Row<V>& v, float x) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) v.p[i] = make_float2(x, x);
}

// Brings the next step's row on its way to L1 while this one is computed; it
// takes no registers, which a load ahead of time would (16 a lane).
template <int V>
__device__ __forceinline__ void row_prefetch(const void* p, int type, int64_t row, int e0, int E, bool live) {
  if (!live || e0 >= E) return;
  const uint8_t* q = static_cast<const uint8_t*>(p) + (row + e0) * (type == kElemF32 ? 4 : 2);
  asm volatile("prefetch.global.L1 [%0];" ::"l"(q));
}

template <int G>
__device__ __forceinline__ float group_max(float v) {
  if constexpr (G == 32) {
    float m;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
  } else {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  }
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---------------------------------------------------------------- scores
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// Flushing forms: a result below 2^-126 is 0, which spares the rescaling that
// the others spend three instructions on.
__device__ __forceinline__ float lg2_ftz(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float ex2_ftz(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_ftz(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int V>
__device__ __forceinline__ float lane_max(const Row<V>& v) {
  float m = fmaxf(v.p[0].x, v.p[0].y);
#pragma unroll
  for (int i = 1; i < V / 2; ++i) m = fmaxf(m, fmaxf(v.p[i].x, v.p[i].y));
  return m;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// e_i = 2^(l_i log2 e - mxl), mxl = the row maximum times log2 e, rounded by
// up to d = 2^-24 |mxl|: a factor 2^d in all of them, which the ratios p = e /
// sum(e) and lse = (mxl + log2 sum(e)) ln 2 are free of while 2^d is near 1.
// Rows that are not kept have l = -inf throughout, mx = 0 and e = 0.  Where the
// maximum is beyond 2^20 (d reaches 0.09 there, and 128 at 1.5e9: every e inf
// or 0; mx log2 e itself ends at 2.4e38), it is taken off first: a difference
// of two logits that close has no rounding that matters.
__device__ __forceinline__ bool far_out(float mx) { return fabsf(mx) > 0x1p20f; }
template <int V>
__device__ __forceinline__ float row_exp(const Row<V>& v, float mx, float mxl, Row<V>& e) {
  float2 total = both(0.f);
  if (far_out(mx)) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      e.p[i] = make_float2(ex2_ftz((v.p[i].x - mx) * kLog2e), ex2_ftz((v.p[i].y - mx) * kLog2e));
      total = __fadd2_rn(total, e.p[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 x = __ffma2_rn(v.p[i], both(kLog2e), both(-mxl));
      e.p[i] = make_float2(ex2_ftz(x.x), ex2_ftz(x.y));
      total = __fadd2_rn(total, e.p[i]);
    }
  }
  return total.x + total.y;
}
__device__ __forceinline__ float row_lse(float mx, float mxl, float total) {
  return far_out(mx) ? fmaf(lg2_ftz(total), kLn2, mx) : (mxl + lg2_ftz(total)) * kLn2;
}

// Sigmoid scores from the same exponentials.  For a maximum mx >= 0,
// s = e / (e + 2^-mxl); for mx < 0 every s is small and is kept as
// s' = s 2^-mxl = e / (e 2^mxl + 1), so that a row of very negative logits has
// ratios at all.  Both are s' = e t with t = 1 / (e a + b), and 1 - s = b t.
// Above mx = 40, e would lose scores near 0 logits: they get exponentials of
// their own.  f(i, s', s' (1 - s)) takes a pair at a time.
template <int V, class F>
__device__ __forceinline__ void row_sigmoid(const Row<V>& v, const Row<V>& e, float mx, float mxl, F&& f) {
  if (mx > 40.f) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 r = make_float2(ex2_ftz(-kLog2e * v.p[i].x), ex2_ftz(-kLog2e * v.p[i].y));
      const float2 s = make_float2(rcp_ftz(1.f + r.x), rcp_ftz(1.f + r.y));
      f(i, s, make_float2(r.x > 1e18f ? s.x : r.x * s.x * s.x, r.y > 1e18f ? s.y : r.y * s.y * s.y));
    }
    return;
  }
  const float other = ex2_ftz(-fabsf(mxl));
  const float2 a = both(mx >= 0.f ? 1.f : other), b = both(mx >= 0.f ? other : 1.f);
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    const float2 x = __ffma2_rn(e.p[i], a, b);
    const float2 t = make_float2(rcp_ftz(x.x), rcp_ftz(x.y));
    const float2 s = __fmul2_rn(e.p[i], t);
    f(i, s, __fmul2_rn(s, __fmul2_rn(b, t)));
  }
}

// The score of a chosen logit relative to `top`: e^(l - top), or a sigmoid
// times e^-min(top, 0).
__device__ __forceinline__ float slot_score(float l, float top, bool sigmoid) {
  if (!sigmoid) return ex2_ftz((l - top) * kLog2e);  // normalised: top is one of the row's chosen
  const float m = fminf(top, 0.f);
  return rcp_ftz(ex2_ftz(m * kLog2e) + ex2_ftz((m - l) * kLog2e));
}

// ---------------------------------------------------------------- forward
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


// Three of them at once; s_w holds three values per warp.
__device__ __forceinline__ void block_sum3(double& a, double& b, double& c, double* s_w) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  a = warp_sum(a);
  b = warp_sum(b);
  c = warp_sum(c);
  __syncthreads();
  if (lane == 0) {
    s_w[warp] = a;
    s_w[nw + warp] = b;
    s_w[2 * nw + warp] = c;
  }
  __syncthreads();
  a = b = c = 0.0;
  for (int w = 0; w < nw; ++w) {
    a += s_w[w];
    b += s_w[nw + w];
    c += s_w[2 * nw + w];
  }
}

// Whether this block is the last of `n` to come to `counter`, which it then
// sets back to 0.  Called by the whole block after its global writes.
__device__ __forceinline__ bool last_block(uint32_t* counter, uint32_t n, int* s_flag) {
  if (n == 1) {
    __syncthreads();
    return true;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = atomicAdd(counter, 1u) == n - 1;
    if (last) *counter = 0;
    *s_flag = last;
  }
  __syncthreads();
  __threadfence();
  return *s_flag != 0;
}

// Groups of blocks whose sums are added first: where a sequence has so many
// blocks and experts that its last block alone would read more than 8 rows a
// thread, which it has in flight together.
__host__ __device__ __forceinline__ int route_groups(int64_t chunks, int E) {
  return chunks * E > 8 * kRouteThreads ? (int)((chunks + kRouteGroup - 1) / kRouteGroup) : 1;
}

// Tokens of a block: whole steps of the block, the last one takes what is left.
__device__ __forceinline__ int64_t route_share(int64_t seq_len, int chunks, int step) {
  const int64_t steps = (seq_len + step - 1) / step;
  return (steps + chunks - 1) / chunks * step;
}

// The end of a sequence, by one block whose threads hold parts of
// sum_e c_e sum_t q_te, sum lse^2 and the number of tokens; the block that
// ends the last sequence ends the call.
__device__ __forceinline__ void route_close(const RouteParams& p, int64_t seq, double sum, double z, double n,
                                            uint32_t* counter, double* s_w, int* s_flag) {
  const int E = p.E, tid = threadIdx.x;
  const int64_t b0 = seq * p.chunks;
  block_sum3(sum, z, n, s_w);
  if (tid == 0) {
    p.tokens[seq] = (int)n;
    sum = n > 0.0 ? sum * E / (p.k * n * n) : 0.0;
    if (p.S == 1) {
      *p.balance = (float)sum;
      *p.z = (float)(n > 0.0 ? z / n : 0.0);
    } else {
      p.seq_part[seq] = sum;
      p.part_z[b0] = z;
    }
  }
  if (p.S == 1 || !last_block(counter, p.S, s_flag)) return;
  double bal = 0.0, live = 0.0;
  z = n = 0.0;
  for (int64_t i = tid; i < p.S; i += kRouteThreads) {
    const int ns = __ldcg(p.tokens + i);
    bal += __ldcg(p.seq_part + i);
    z += __ldcg(p.part_z + i * p.chunks);
    n += ns;
    live += ns > 0;
  }
  live = block_sum(live, s_w);
  block_sum3(bal, z, n, s_w);
  if (tid == 0) {
    *p.balance = (float)(live > 0.0 ? bal / live : 0.0);
    *p.z = (float)(n > 0.0 ? z / n : 0.0);
  }
}

// Adds up blocks' sums, as far as this block is the last one to finish.
__device__ __forceinline__ void route_finish(const RouteParams& p, int64_t seq, int chunk, double* s_w, double* s_q, int* s_c,
                                             int* s_flag) {
  const int E = p.E, tid = threadIdx.x;
  const int groups = route_groups(p.chunks, E);
  const int64_t b0 = seq * p.chunks;
  uint32_t* seq_counters = p.counters + (int64_t)p.S * groups;
  int stride = 1, rows = p.chunks;
  if (groups > 1) {
    const int g = chunk / kRouteGroup;
    const int64_t r0 = b0 + (int64_t)g * kRouteGroup;
    const int n = min(kRouteGroup, p.chunks - g * kRouteGroup);
    if (!last_block(p.counters + seq * groups + g, n, s_flag)) return;
    for (int e = tid; e < E; e += kRouteThreads) {
      float q[kRouteGroup];
      int c[kRouteGroup];
#pragma unroll
      for (int i = 0; i < kRouteGroup; ++i) {
        q[i] = i < n ? __ldcg(p.part_q + (r0 + i) * E + e) : 0.f;
        c[i] = i < n ? __ldcg(p.part_c + (r0 + i) * E + e) : 0;
      }
#pragma unroll
      for (int i = 1; i < kRouteGroup; ++i) {
        q[0] += q[i];
        c[0] += c[i];
      }
      p.part_q[r0 * E + e] = q[0];
      p.part_c[r0 * E + e] = c[0];
    }
    if (tid < 32) {
      double z = tid < n ? __ldcg(p.part_z + r0 + tid) : 0.0;
      int m = tid < n ? __ldcg(p.part_n + r0 + tid) : 0;
#pragma unroll
      for (int o = 8; o; o >>= 1) {
        z += __shfl_xor_sync(0xffffffffu, z, o);
        m += __shfl_xor_sync(0xffffffffu, m, o);
      }
      if (tid == 0) {
        p.part_z[r0] = z;
        p.part_n[r0] = m;
      }
    }
    stride = kRouteGroup;
    rows = groups;
  }
  if (!last_block(seq_counters + seq, rows, s_flag)) return;
  double z = 0.0, n = 0.0, sum = 0.0;
  for (int i = tid; i < rows; i += kRouteThreads) {
    z += __ldcg(p.part_z + b0 + (int64_t)i * stride);
    n += __ldcg(p.part_n + b0 + (int64_t)i * stride);
  }
  // `parts` threads take an expert's rows in turn (few experts: many threads
  // each), neighbouring threads neighbouring experts.
  int width = 1;
  while (width < E && width < kRouteThreads) width *= 2;
  const int parts = kRouteThreads / width, part = tid / width;
  for (int e = tid % width; e < E; e += width) {
    double q = 0.0;
    int c = 0;
    for (int i0 = part; i0 < rows; i0 += 8 * parts) {
      float qs[8];
      int cs[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * parts;
        qs[u] = i < rows ? __ldcg(p.part_q + (b0 + (int64_t)i * stride) * E + e) : 0.f;
        cs[u] = i < rows ? __ldcg(p.part_c + (b0 + (int64_t)i * stride) * E + e) : 0;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        q += (double)qs[u];
        c += cs[u];
      }
    }
    if (parts > 1) {  // then E <= width: every thread comes by at most once
      s_q[tid] = q;
      s_c[tid] = c;
    } else {
      p.counts[seq * E + e] = c;
      sum += (double)c * q;
    }
  }
  if (parts > 1) {
    __syncthreads();
    if (tid < E) {
      double q = 0.0;
      int c = 0;
      for (int i = 0; i < parts; ++i) {
        q += s_q[i * width + tid];
        c += s_c[i * width + tid];
      }
      p.counts[seq * E + tid] = c;
      sum = (double)c * q;
    }
  }
  route_close(p, seq, sum, z, n, seq_counters + p.S, s_w, s_flag);
}

// Blocks per SM that the register budget is cut for.  E = 1024, T = 32768, f32,
// forward: 139 us at one block of 190 registers a thread, 83 at two of 128;
// E = 256, T = 131072: no gain from a fourth block at 64 (spills).
template <int G, int V, int KMAX>
constexpr int route_residents() {
  return V == 32 ? 2 : (KMAX + G - 1) / G <= 4 ? 3 : 2;
}

// T = 131072, E = 256, k = 8, f32: 101 us; with given experts, bf16, sigmoid 62
// (HBM's share 22 and 11).  Bounded by latency: 24 warps an SM with one row per
// group of lanes in flight leave half of the issue slots empty while loads,
// shuffles and special functions are waited for.
template <int G, int V, int KMAX>
__global__ void __launch_bounds__(kRouteThreads, route_residents<G, V, KMAX>()) route_train_kernel(const RouteParams p) {
  constexpr int TPW = 32 / G;                // tokens per warp and step
  constexpr int KS = (KMAX + G - 1) / G;     // slots per lane
  // [warps][V / 4][32] fours of the rows in work; after them [warps][G V] sums
  // of q; then [E] counts.
  extern __shared__ float4 s_quads[];
  int* s_cnt = reinterpret_cast<int*>(s_quads + kRouteWarps * 8 * V);
  __shared__ double s_w[3 * kRouteWarps];
  __shared__ double s_fq[kRouteThreads];
  __shared__ int s_fc[kRouteThreads];
  __shared__ double s_z[kRouteWarps];
  __shared__ int s_n[kRouteWarps];
  __shared__ int s_flag;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % G;
  const uint32_t gmask = (G == 32 ? 0xffffffffu : ((1u << (G & 31)) - 1u) << (lane / G * G));
  const int e0 = gl * V, E = p.E, k = p.k;
  for (int e = threadIdx.x; e < E; e += kRouteThreads) s_cnt[e] = 0;
  __syncthreads();

  const int64_t seq = blockIdx.x / p.chunks;
  const int chunk = blockIdx.x % p.chunks;
  const int64_t per = route_share(p.seq_len, p.chunks, kRouteWarps * TPW);
  const int64_t lo = seq * p.seq_len + chunk * per;
  const int64_t hi = seq * p.seq_len + min(p.seq_len, (chunk + 1) * per);
  Row<V> acc;
  row_fill(acc, 0.f);
  float z = 0.f;
  int n = 0;
  for (int64_t base = lo + warp * TPW; base < hi; base += kRouteWarps * TPW) {
    const int64_t t = base + lane / G;
    const bool inside = t < hi;
    const bool live = inside && (!p.mask || __ldg(p.mask + t));
    Row<V> v;
    row_load(p.logits, p.type, p.vec, t * p.ld, e0, E, live, v);
    const int64_t next = t + kRouteWarps * TPW;
    row_prefetch<V>(p.logits, p.type, next * p.ld, e0, E, next < hi);
    int id[KS];
    float sel[KS];
    if (p.given) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int j = s * G + gl;
        id[s] = live && j < k ? __ldg(p.given + t * k + j) : -1;
        if (id[s] < 0 || id[s] >= E) id[s] = -1;
        sel[s] = id[s] >= 0 ? elem_load(p.logits, p.type, t * p.ld + id[s]) : -INFINITY;
      }
    }
    float m = lane_max(v);
    const float mx = group_max<G>(m);
    const bool keep = mx > -INFINITY;
    if (!keep) row_fill(v, -INFINITY);  // a row of NaN takes no part either
    const float mxl = keep ? mx * kLog2e : 0.f;
    Row<V> ex;
    const float total = group_sum<G>(row_exp(v, keep ? mx : 0.f, mxl, ex));
    const float lse = keep ? row_lse(mx, mxl, total) : 0.f;
    z += lse * lse;
    n += keep;
    float inv;  // 1 / the sum of the scores
    if (!p.sigmoid) {
      inv = keep ? rcp_ftz(total) : 0.f;
    } else {
      float2 sum = both(0.f);
      row_sigmoid(v, ex, mx, mxl, [&](int i, float2 s, float2) {
        ex.p[i] = s;
        sum = __fadd2_rn(sum, s);
      });
      const float norm = group_sum<G>(sum.x + sum.y);  // by every lane: other rows of the warp may be kept
      inv = keep ? rcp_ftz(norm) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) acc.p[i] = __ffma2_rn(ex.p[i], both(inv), acc.p[i]);

    // Choice: k rounds of the row's maximum.  A lane's logits lie in shared
    // memory in fours with the maxima of the fours in registers: taking one
    // out costs a search of the maxima and of one four (searching V registers
    // took twice the instructions).  NaN equals no maximum.
    if (!p.given) {
      constexpr int Q = V / 4;
      float4* quads = s_quads + warp * 32 * Q + lane;
      float qm[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const float4 x = make_float4(v.p[2 * q].x, v.p[2 * q].y, v.p[2 * q + 1].x, v.p[2 * q + 1].y);
        quads[q * 32] = x;
        qm[q] = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        id[s] = -1;
        sel[s] = -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < KMAX; ++j) {
        if (j >= k) break;
        const float M = group_max<G>(m);
        const uint32_t owners = __ballot_sync(0xffffffffu, m == M && M > -INFINITY) & gmask;
        const int owner = __ffs(owners) - 1;
        int at = -1;
        if (lane == owner) {
          int q = 0;
#pragma unroll
          for (int i = Q - 1; i > 0; --i)
            if (qm[i] == M) q = i;
          if (qm[0] == M) q = 0;
          float4 x = quads[q * 32];
          const int i = x.x == M ? 0 : x.y == M ? 1 : x.z == M ? 2 : 3;
          if (i == 0) x.x = -INFINITY;
          if (i == 1) x.y = -INFINITY;
          if (i == 2) x.z = -INFINITY;
          if (i == 3) x.w = -INFINITY;
          quads[q * 32] = x;
          const float left = fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w));
          m = -INFINITY;
#pragma unroll
          for (int z = 0; z < Q; ++z) {
            if (z == q) qm[z] = left;
            m = fmaxf(m, qm[z]);
          }
          at = e0 + 4 * q + i;
        }
        at = __shfl_sync(0xffffffffu, at, owner < 0 ? lane : owner);
        if (gl == j % G) {
          id[j / G] = at;
          sel[j / G] = M;
        }
      }
    }
    // Weights of the chosen logits, on the row's own scale; those that the
    // caller chose, normalised, relative to the largest of them.
    float top = mx;
    if (p.given && p.normalize) {
      top = sel[0];
#pragma unroll
      for (int s = 1; s < KS; ++s) top = fmaxf(top, sel[s]);
      top = group_max<G>(top);
    }
    float w[KS], sum = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      // -inf: no expert in this slot, or one chosen by the caller with score 0.
      w[s] = 0.f;
      if (keep && sel[s] > -INFINITY) {
        // A plain softmax probability is one of the row's e over their sum,
        // mxl's rounding included (at |mx| = 65504 that is 2e-3), or formed as
        // row_exp forms them beyond its range.
        if (!p.sigmoid && !p.normalize && !far_out(mx)) w[s] = ex2_ftz(fmaf(sel[s], kLog2e, -mxl));
        else w[s] = slot_score(sel[s], top, p.sigmoid);
      }
      if (sel[s] != sel[s]) w[s] = sel[s];
      sum += w[s];
    }
    float scale = p.sigmoid ? ex2_ftz(fminf(mx, 0.f) * kLog2e) : inv;
    if (p.normalize) {
      sum = group_sum<G>(sum);
      scale = sum == 0.f ? 0.f : rcp_ftz(sum);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int j = s * G + gl;
      if (inside && j < k) {
        if (!keep) id[s] = -1;
        p.ids[t * k + j] = id[s];
        p.weights[t * k + j] = keep ? w[s] * scale : 0.f;
        if (id[s] >= 0) atomicAdd(&s_cnt[id[s]], 1);
      }
    }
  }

  // Block sums: lanes of equal gl, then warps, in order.
#pragma unroll
  for (int o = G; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      acc.p[i].x += __shfl_xor_sync(0xffffffffu, acc.p[i].x, o);
      acc.p[i].y += __shfl_xor_sync(0xffffffffu, acc.p[i].y, o);
    }
    z += __shfl_xor_sync(0xffffffffu, z, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  float* s_q = reinterpret_cast<float*>(s_quads);
  __syncthreads();  // the rows in work are done with
  if (lane < G) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      s_q[warp * (G * V) + e0 + 2 * i] = acc.p[i].x;
      s_q[warp * (G * V) + e0 + 2 * i + 1] = acc.p[i].y;
    }
  }
  if (lane == 0) {
    s_z[warp] = z;
    s_n[warp] = n;
  }
  __syncthreads();
  if (p.chunks == 1) {  // a sequence of its own: nothing to wait for, nothing by way of memory
    const int tid = threadIdx.x;
    double sum = 0.0;
    for (int e = tid; e < E; e += kRouteThreads) {
      float qs = 0.f;
#pragma unroll
      for (int w = 0; w < kRouteWarps; ++w) qs += s_q[w * (G * V) + e];
      p.counts[seq * E + e] = s_cnt[e];
      sum += (double)s_cnt[e] * (double)qs;
    }
    route_close(p, seq, sum, tid < kRouteWarps ? s_z[tid] : 0.0, tid < kRouteWarps ? s_n[tid] : 0,
                p.counters + 2 * (int64_t)p.S, s_w, &s_flag);
    return;
  }
  for (int e = threadIdx.x; e < E; e += kRouteThreads) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) sum += s_q[w * (G * V) + e];
    p.part_q[(int64_t)blockIdx.x * E + e] = sum;
    p.part_c[(int64_t)blockIdx.x * E + e] = s_cnt[e];
  }
  if (threadIdx.x == 0) {
    double zs = 0.0;
    int ns = 0;
    for (int w = 0; w < kRouteWarps; ++w) {
      zs += s_z[w];
      ns += s_n[w];
    }
    p.part_z[blockIdx.x] = zs;
    p.part_n[blockIdx.x] = ns;
  }
  route_finish(p, seq, chunk, s_w, s_fq, s_fc, &s_flag);
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
// Normalised weights sum to 1 but for their rounding, which times what all dw of
// a row share would stay over where the formula cancels; the first slot's dw is
// taken off all of them before (one weight alone gets exactly 0).
// It is formed in the slots' lanes and added to the row in shared memory, on
// its way to the store (a register exchange takes k V compares a lane).
// WEIGHTS: there is such a part (the losses alone spare its registers).
template <int G, int V, int KMAX, bool WEIGHTS>
__global__ void __launch_bounds__(kRouteThreads, route_residents<G, V, KMAX>()) route_backward_kernel(const RouteBackward p) {
  constexpr int TPW = 32 / G;
  constexpr int KS = (KMAX + G - 1) / G;
  __shared__ float4 s_rows[kRouteWarps][8 * V];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gl = lane % G;
  const int e0 = gl * V, E = p.E, k = p.k;
  float4* fours = s_rows[warp];

  // Tokens in all sequences and sequences with any: by each warp where that is
  // one load a lane, else by the block, to wait in shared memory.  So does the
  // run of tokens in work: registers are what the rows need.
  __shared__ int s_all, s_live;
  __shared__ uint32_t s_unit;
  if (threadIdx.x == 0) s_unit = blockIdx.x;
  if (p.S > 32) {
    __shared__ int s_n[2][kRouteWarps];
    int all = 0, live_seqs = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < p.S; i += kRouteThreads) {
      const int m = __ldg(p.tokens + i);
      all += m;
      live_seqs += m > 0;
    }
    all = __reduce_add_sync(0xffffffffu, all);
    live_seqs = __reduce_add_sync(0xffffffffu, live_seqs);
    if (lane == 0) s_n[0][warp] = all, s_n[1][warp] = live_seqs;
    __syncthreads();
    if (threadIdx.x == 0) {
      all = live_seqs = 0;
      for (int w = 0; w < kRouteWarps; ++w) all += s_n[0][w], live_seqs += s_n[1][w];
      s_all = all, s_live = live_seqs;
    }
    __syncthreads();
  }

  // A block's runs of tokens: one, or with very many sequences several.
  for (uint32_t unit = blockIdx.x;;) {
    const int64_t seq = unit / p.chunks;
    const int chunk = unit % p.chunks;
    const int64_t per = route_share(p.seq_len, p.chunks, kRouteWarps * TPW);
    const int64_t lo = seq * p.seq_len + chunk * per;
    const int64_t hi = seq * p.seq_len + min(p.seq_len, (chunk + 1) * per);
    {  // the first rows come while the experts' factors are made
      const int64_t t = lo + warp * TPW + lane / G;
      row_prefetch<V>(p.logits, p.type, t * p.ld, e0, E, t < hi);
    }
    const int ns = __ldg(p.tokens + seq);
    int all = ns, live_seqs = ns > 0;
    if (p.S > 32) {
      all = s_all, live_seqs = s_live;
    } else if (p.S > 1) {
      const int m = lane < p.S ? __ldg(p.tokens + lane) : 0;
      all = __reduce_add_sync(0xffffffffu, m);
      live_seqs = __reduce_add_sync(0xffffffffu, (int)(m > 0));
    }
    // dB / (S' N) (1 / (k N)) (c E - k N): the integer part is exact (in 32 bits
    // where k N E, which bounds c E, fits).
    const float db = p.d_balance && ns > 0 ? __ldg(p.d_balance) / ((float)live_seqs * (float)ns) : 0.f;
    const float dz = p.d_z && all > 0 ? 2.f * __ldg(p.d_z) / (float)all : 0.f;
    // They lie in shared memory, a lane's experts in fours: the registers that
    // they would take hold more rows instead.
    __shared__ float4 s_f[V / 4][32];
    const float kn = db / (float)((int64_t)k * (ns > 0 ? ns : 1));
    const bool narrow = (int64_t)k * ns * E < (int64_t)1 << 31;
    for (int i = threadIdx.x; i < 32 * V; i += kRouteThreads) {
      const int l = i / V, x = i % V, e = l % G * V + x;
      const int c = e < E ? __ldg(p.counts + seq * E + e) : 0;
      const float over = narrow ? (float)(c * E - k * ns) : (float)((int64_t)c * E - (int64_t)k * ns);
      reinterpret_cast<float*>(&s_f[x / 4][l])[x % 4] = e < E ? over * kn : 0.f;
    }
    __syncthreads();
    const auto f = [&](int i) {  // pair i of the lane's experts
      return reinterpret_cast<const float2*>(&s_f[i / 2][lane])[i % 2];
    };

    for (int64_t base = lo + warp * TPW; base < hi; base += kRouteWarps * TPW) {
      const int64_t t = base + lane / G;
      const bool inside = t < hi;
      const bool live = inside && (!p.mask || __ldg(p.mask + t));
      Row<V> v;
      row_load(p.logits, p.type, p.vec, t * p.ld, e0, E, live, v);
      const int64_t next = t + kRouteWarps * TPW;
      row_prefetch<V>(p.logits, p.type, next * p.ld, e0, E, next < hi);
      // The weights' part per slot.
      int id[KS];
      float g[KS], w[KS], dot = 0.f;
      if constexpr (WEIGHTS) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int j = s * G + gl;
          const bool on = live && j < k;  // the three loads do not wait for one another
          id[s] = on ? __ldg(p.ids + t * k + j) : -1;
          w[s] = on ? __ldg(p.weights + t * k + j) : 0.f;
          g[s] = on ? __ldg(p.d_weights + t * k + j) : 0.f;
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          if (id[s] < 0 || id[s] >= E) {  // dropped, whatever its gradient holds
            id[s] = -1;
            w[s] = g[s] = 0.f;
          }
        }
        float first = __shfl_sync(0xffffffffu, g[0], lane / G * G);
        if (!p.normalize) first = 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          if (id[s] >= 0) g[s] -= first;
          dot = fmaf(w[s], g[s], dot);
          // 1 - sigmoid of the slot's logit, into its weight: w is done with.
          if (p.sigmoid && id[s] >= 0)
            w[s] *= rcp_ftz(1.f + ex2_ftz(elem_load(p.logits, p.type, t * p.ld + id[s]) * kLog2e));
        }
      }
      const float mx = group_max<G>(lane_max(v));
      const bool keep = mx > -INFINITY;
      const float mxl = keep ? mx * kLog2e : 0.f;
      Row<V> d;
      float total = row_exp(v, keep ? mx : 0.f, mxl, d);
      if (WEIGHTS) dot = group_sum<G>(dot);
      if (!p.sigmoid) {
        float2 fs = both(0.f);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) fs = __ffma2_rn(f(i), d.p[i], fs);
        total = group_sum<G>(total);
        const float fq = group_sum<G>(fs.x + fs.y);
        const float inv = keep ? rcp_ftz(total) : 0.f;
        // A row's share of every p: the z loss, the centring, the weights' dot.
        const float every = dz * row_lse(mx, mxl, total) - fq * inv - (p.normalize ? 0.f : dot);
        const float2 x = both(inv), y = both(every * inv);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) d.p[i] = __fmul2_rn(d.p[i], __ffma2_rn(f(i), x, y));
      } else {
        Row<V> ds;
        float2 ns2 = both(0.f), fs = both(0.f);
        row_sigmoid(v, d, mx, mxl, [&](int i, float2 s, float2 slope) {
          ns2 = __fadd2_rn(ns2, s);
          fs = __ffma2_rn(f(i), s, fs);
          ds.p[i] = slope;
        });
        const float norm = group_sum<G>(ns2.x + ns2.y), fq = group_sum<G>(fs.x + fs.y);
        const float qi = keep ? rcp_ftz(norm) : 0.f;
        float zl = 0.f;
        if (p.d_z) {
          total = group_sum<G>(total);
          zl = keep ? dz * row_lse(mx, mxl, total) * rcp_ftz(total) : 0.f;
        }
        const float2 x = both(qi), y = both(-fq * qi * qi), w2 = both(zl);
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
          d.p[i] = __ffma2_rn(ds.p[i], __ffma2_rn(f(i), x, y), __fmul2_rn(d.p[i], w2));
      }
      if (!keep) row_fill(d, 0.f);
      if (!WEIGHTS && p.type != kElemF32 && p.vec_out == 8) {
        // Nothing to add, and a lane's 16 or 32 bytes are whole sectors or
        // halves that its next store fills: straight out (45 us against 54
        // through shared memory at T = 131072, E = 256, sigmoid).
#pragma unroll
        for (int c = 0; c < V; c += 8) {
          const float2* x = d.p + c / 2;
          if (inside && e0 + c < E)
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.d_logits) + t * E + e0 + c) =
                make_uint4(pack16(x[0].x, x[0].y, p.type), pack16(x[1].x, x[1].y, p.type),
                           pack16(x[2].x, x[2].y, p.type), pack16(x[3].x, x[3].y, p.type));
        }
        continue;
      }
      __syncwarp();  // the last step's rows are stored
#pragma unroll
      for (int q = 0; q < V / 4; ++q)
        fours[four_at<V>(lane, q)] = make_float4(d.p[2 * q].x, d.p[2 * q].y, d.p[2 * q + 1].x, d.p[2 * q + 1].y);
      __syncwarp();
      if constexpr (WEIGHTS) {
        const float off = p.normalize ? dot : 0.f;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          g[s] = w[s] * (g[s] - off);
          // Slots of one expert (the caller's choice may repeat it) are added
          // in slot order by the lowest of their lanes.
          const int l = lane / G * G + id[s] / V;
          const int key = id[s] >= 0 ? l * V + id[s] % V : -1 - lane;
          const uint32_t peers = __match_any_sync(0xffffffffu, key);
          bool mine = true;
          if (__any_sync(0xffffffffu, peers != 1u << lane)) {
            float sum = 0.f;
            for (int x = 0; x < 32; ++x) {
              const float other = __shfl_sync(0xffffffffu, g[s], x);
              if (peers >> x & 1u) sum += other;
            }
            g[s] = sum;
            mine = lane == __ffs(peers) - 1;
          }
          if (id[s] >= 0 && mine && keep)
            reinterpret_cast<float*>(fours + four_at<V>(l, id[s] % V / 4))[id[s] % 4] += g[s];
          __syncwarp();
        }
      }
      rows_store<G, V>(fours, p.d_logits, p.type, p.vec_out, base, hi, E, lane);
    }
    if (gridDim.x == (uint32_t)p.S * p.chunks) return;
    __syncthreads();
    if (threadIdx.x == 0) s_unit += gridDim.x;
    __syncthreads();
    unit = s_unit;
    if (unit >= (uint32_t)p.S * p.chunks) return;
  }
}

}  // namespace moe
