// C ABI of the steps that train a whole MoE layer around its expert MLP:
// top-k routing with the balance and z losses, the backward of the row
// movement, and gradient norms and clipping.  Declarations:
// include/moe_b200.h.
#include <algorithm>
#include <cstdint>
#include <cstdlib>
#include <utility>

#include "abi_util.h"
#include "grad_norm.cuh"
#include "router_train.cuh"
#include "row_grads.cuh"

namespace moe {

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
static size_t elem_bytes(int type) { return type == MOE_ELEM_F32 ? 4 : 2; }
static bool elem_ok(int type) { return type == MOE_ELEM_F32 || type == MOE_ELEM_BF16 || type == MOE_ELEM_F16; }

// ------------------------------------------------------------------ routing
// Lanes per row: 8 experts a lane up to 16 experts, then 16, and the whole
// warp with 32 above 512.
static int route_lanes(int E) {
  int g = 1;
  while (g < 32 && g * (E <= 16 ? 8 : 16) < E) g *= 2;
  return g;
}

// Blocks per sequence: one for every step (a token per row group of the block)
// while all of them are resident, else as few as share the steps evenly: a block
// with one token more than its neighbours, or a second, short wave, costs a
// whole step.  Resident is counted as 3 blocks an SM (80 registers a thread), 2
// above 512 experts (128); the variants of up to 32 experts whose lanes hold
// more than four slots have 2 as well and run what is over in a second wave.  A
// sequence has a whole number of blocks: from 223 sequences on one each, which
// leaves up to half of the slots empty.
static int64_t route_chunks(int64_t seq_len, int64_t sequences, int E) {
  const int64_t step = kRouteWarps * (32 / route_lanes(E));
  const int64_t steps = std::max<int64_t>(1, (seq_len + step - 1) / step);
  const int64_t resident = std::max<int64_t>(1, 148 * (E > 512 ? 2 : 3) / std::max<int64_t>(1, sequences));
  const int64_t each = (steps + resident - 1) / resident;
  return (steps + each - 1) / each;
}

struct RouteSpace {
  size_t q, c, z, n, seq, bytes;
};
static RouteSpace route_space(int64_t chunks, int64_t sequences, int E) {
  const int64_t blocks = chunks * sequences, sums = chunks > 1 ? blocks : 0;  // one block: nothing to hand over
  RouteSpace s;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += align256(bytes);
    return here;
  };
  s.q = take((size_t)sums * E * sizeof(float));
  s.c = take((size_t)sums * E * sizeof(int32_t));
  s.z = take((size_t)blocks * sizeof(double));
  s.n = take((size_t)blocks * sizeof(int32_t));
  s.seq = take((size_t)sequences * sizeof(double));
  s.bytes = at;
  return s;
}
static int64_t route_counters(int64_t chunks, int64_t sequences, int E) {
  return sequences * route_groups(chunks, E) + sequences + 1;
}

template <int G, int V, int KMAX>
static int launch_route(const RouteParams& p, int64_t blocks, cudaStream_t st) {
  const size_t smem = (size_t)kRouteWarps * 32 * V * sizeof(float) + (size_t)p.E * sizeof(int);
  route_train_kernel<G, V, KMAX><<<(unsigned)blocks, kRouteThreads, smem, st>>>(p);
  MOE_CUDA_TRY(cudaGetLastError());
  return 0;
}
template <int G, int V>
static int launch_route_k(const RouteParams& p, int64_t blocks, cudaStream_t st) {
  if (p.k <= 2) return launch_route<G, V, 2>(p, blocks, st);
  if (p.k <= 8) return launch_route<G, V, 8>(p, blocks, st);
  return launch_route<G, V, 16>(p, blocks, st);
}
template <int G, int V, int KMAX, bool WEIGHTS>
static int launch_backward(const RouteBackward& p, int64_t blocks, cudaStream_t st) {
  route_backward_kernel<G, V, KMAX, WEIGHTS><<<(unsigned)blocks, kRouteThreads, 0, st>>>(p);
  MOE_CUDA_TRY(cudaGetLastError());
  return 0;
}
template <int G, int V>
static int launch_backward_k(const RouteBackward& p, int64_t blocks, cudaStream_t st) {
  if (!p.d_weights) return launch_backward<G, V, G, false>(p, blocks, st);
  if constexpr (G >= kRouteMaxK) {
    return launch_backward<G, V, kRouteMaxK, true>(p, blocks, st);  // one slot a lane
  } else {
    if (p.k <= 2) return launch_backward<G, V, 2, true>(p, blocks, st);
    if (p.k <= 8) return launch_backward<G, V, 8, true>(p, blocks, st);
    return launch_backward<G, V, kRouteMaxK, true>(p, blocks, st);
  }
}

static int check_route(int elem_type, int64_t ld, int64_t T, int E, int k, int64_t sequences, int scoring) {
  if (T < 0 || E < 1 || E > kRouteMaxExperts || k < 1 || k > kRouteMaxK || k > E || T > (int64_t)0x7fffffff / k)
    return fail(MOE_ERR_INVALID_ARG, "T=%lld E=%d k=%d (1 <= k <= min(%d, E), E <= %d, T k < 2^31)", (long long)T, E,
                k, kRouteMaxK, kRouteMaxExperts);
  if (sequences < 1 || sequences > (int64_t)0x7fffffff || T % sequences)
    return fail(MOE_ERR_INVALID_ARG, "%lld tokens are not %lld sequences of equal length", (long long)T,
                (long long)sequences);
  if (ld < E) return fail(MOE_ERR_INVALID_ARG, "row stride %lld < E=%d", (long long)ld, E);
  if (!elem_ok(elem_type)) return fail(MOE_ERR_UNSUPPORTED_DTYPE, "logits type %d", elem_type);
  if (scoring != MOE_SCORE_SOFTMAX && scoring != MOE_SCORE_SIGMOID)
    return fail(MOE_ERR_INVALID_ARG, "scoring %d (0 softmax, 1 sigmoid)", scoring);
  return 0;
}

// Elements of a row that can be read or written at a time: 8, 4 or 1.
static int route_vec(const void* base, int64_t ld, int E, int type) {
  for (int v = 8; v > 1; v /= 2) {
    const size_t bytes = std::min<size_t>(16, v * elem_bytes(type));
    if (E % v == 0 && ld % v == 0 && reinterpret_cast<uintptr_t>(base) % bytes == 0) return v;
    if (v == 4) break;
  }
  return 1;
}

// ------------------------------------------------------------------ rows
// Threads per token: as few as a row has vectors for, a block where it has
// many.
static int row_threads(int D) { return D >= 1024 ? 256 : D >= 128 ? 32 : 8; }

template <int TPT, int DY, int DYS>
static int launch_combine(const CombineBwd& p, cudaStream_t st) {
  const unsigned blocks = (unsigned)((p.T + kRowThreads / TPT - 1) / (kRowThreads / TPT) + p.zero_blocks);
  if (p.k <= 2) combine_bwd_kernel<TPT, DY, DYS, 2><<<blocks, kRowThreads, 0, st>>>(p);
  else if (p.k <= 4) combine_bwd_kernel<TPT, DY, DYS, 4><<<blocks, kRowThreads, 0, st>>>(p);
  else combine_bwd_kernel<TPT, DY, DYS, kRowSlots><<<blocks, kRowThreads, 0, st>>>(p);
  MOE_CUDA_TRY(cudaGetLastError());
  return 0;
}
template <int TPT>
static int launch_combine_t(const CombineBwd& p, int dy, int dys, cudaStream_t st) {
  switch (dy * 3 + dys) {
    case 0: return launch_combine<TPT, 0, 0>(p, st);
    case 1: return launch_combine<TPT, 0, 1>(p, st);
    case 2: return launch_combine<TPT, 0, 2>(p, st);
    case 3: return launch_combine<TPT, 1, 0>(p, st);
    case 4: return launch_combine<TPT, 1, 1>(p, st);
    case 5: return launch_combine<TPT, 1, 2>(p, st);
    case 6: return launch_combine<TPT, 2, 0>(p, st);
    case 7: return launch_combine<TPT, 2, 1>(p, st);
  }
  return launch_combine<TPT, 2, 2>(p, st);
}
template <int TPT, int DXS, int DX, int VEC>
static int launch_gather_v(const GatherBwd& p, cudaStream_t st) {
  const int64_t blocks = (p.T + kRowThreads / TPT - 1) / (kRowThreads / TPT);
  if (p.k <= 2) gather_bwd_kernel<TPT, DXS, DX, 2, VEC><<<(unsigned)blocks, kRowThreads, 0, st>>>(p);
  else gather_bwd_kernel<TPT, DXS, DX, kRowSlots, VEC><<<(unsigned)blocks, kRowThreads, 0, st>>>(p);
  MOE_CUDA_TRY(cudaGetLastError());
  return 0;
}
template <int TPT, int DXS, int DX>
static int launch_gather(const GatherBwd& p, cudaStream_t st) {
  if constexpr (DXS != kElemF32)
    if (p.D % 8 == 0 && aligned16(p.dxs) && aligned16(p.dx)) return launch_gather_v<TPT, DXS, DX, 8>(p, st);
  return launch_gather_v<TPT, DXS, DX, 4>(p, st);
}
template <int TPT>
static int launch_gather_t(const GatherBwd& p, int dxs, int dx, cudaStream_t st) {
  switch (dxs * 3 + dx) {
    case 0: return launch_gather<TPT, 0, 0>(p, st);
    case 1: return launch_gather<TPT, 0, 1>(p, st);
    case 2: return launch_gather<TPT, 0, 2>(p, st);
    case 3: return launch_gather<TPT, 1, 0>(p, st);
    case 4: return launch_gather<TPT, 1, 1>(p, st);
    case 5: return launch_gather<TPT, 1, 2>(p, st);
    case 6: return launch_gather<TPT, 2, 0>(p, st);
    case 7: return launch_gather<TPT, 2, 1>(p, st);
  }
  return launch_gather<TPT, 2, 2>(p, st);
}

static int check_rows(int64_t T, int k, int D, int64_t rows, int type_a, int type_b) {
  if (T < 0 || T > 0x7fffffff || k < 1 || D <= 0 || (D & 3) || rows < 0 || rows > 0x7fffffff)
    return fail(MOE_ERR_INVALID_ARG, "T=%lld k=%d D=%d rows=%lld (D a positive multiple of 4, T and rows < 2^31)",
                (long long)T, k, D, (long long)rows);
  if (!elem_ok(type_a) || !elem_ok(type_b))
    return fail(MOE_ERR_UNSUPPORTED_DTYPE, "row types %d, %d", type_a, type_b);
  return 0;
}
static bool row_aligned(const void* p, int type) {
  return reinterpret_cast<uintptr_t>(p) % (4 * elem_bytes(type)) == 0;
}

// ------------------------------------------------------------------ gradient lists
static int check_tensors(const moe_tensor_desc* t, int n, int norm_type, bool with_out) {
  if (n < 0 || (n && !t)) return fail(MOE_ERR_INVALID_ARG, "n=%d tensors=%p", n, (const void*)t);
  if (norm_type < MOE_NORM_L1 || norm_type > MOE_NORM_INF)
    return fail(MOE_ERR_INVALID_ARG, "norm type %d (1, 2 or 3 = infinity)", norm_type);
  int64_t total = 0;
  for (int i = 0; i < n; ++i) {
    if (!elem_ok(t[i].in_type) || (with_out && !elem_ok(t[i].out_type)))
      return fail(MOE_ERR_UNSUPPORTED_DTYPE, "tensor %d: types %d, %d", i, t[i].in_type, t[i].out_type);
    if (t[i].rows < 0 || t[i].cols < 0 ||
        (t[i].rows > 1 && (t[i].in_ld < t[i].cols || (with_out && t[i].out_ld < t[i].cols))))
      return fail(MOE_ERR_INVALID_ARG, "tensor %d: %lld x %lld, strides %lld, %lld", i, (long long)t[i].rows,
                  (long long)t[i].cols, (long long)t[i].in_ld, (long long)t[i].out_ld);
    if (t[i].rows == 0 || t[i].cols == 0) continue;
    constexpr int64_t kMost = (int64_t)1 << 40;  // so that units count in 32 bits
    if (t[i].rows > kMost / t[i].cols || (total += t[i].rows * t[i].cols) > kMost)
      return fail(MOE_ERR_UNSUPPORTED_SHAPE, "more than 2^40 elements at tensor %d", i);
    if (!t[i].in || (with_out && !t[i].out)) return fail(MOE_ERR_INVALID_ARG, "tensor %d: null pointer", i);
    if (reinterpret_cast<uintptr_t>(t[i].in) % elem_bytes(t[i].in_type) ||
        (with_out && reinterpret_cast<uintptr_t>(t[i].out) % elem_bytes(t[i].out_type)))
      return fail(MOE_ERR_MISALIGNED, "tensor %d is not aligned to its elements", i);
  }
  return 0;
}

// Bytes of a tensor: `rows` runs of `bytes`, `ld` apart.
struct Span {
  uintptr_t lo;
  uint64_t rows, bytes, ld;
  uintptr_t end() const { return lo + (rows - 1) * ld + bytes; }
};
static Span in_span(const moe_tensor_desc& d) {
  const uint64_t eb = elem_bytes(d.in_type);
  return {reinterpret_cast<uintptr_t>(d.in), (uint64_t)d.rows, d.cols * eb, d.rows > 1 ? d.in_ld * eb : 0};
}
static Span out_span(const moe_tensor_desc& d) {
  const uint64_t eb = elem_bytes(d.out_type);
  return {reinterpret_cast<uintptr_t>(d.out), (uint64_t)d.rows, d.cols * eb, d.rows > 1 ? d.out_ld * eb : 0};
}

// Whether two tensors have a byte in common: slices of one matrix interleave
// without.
static bool spans_meet(Span a, Span b) {
  if (a.lo >= b.end() || b.lo >= a.end()) return false;
  if (a.rows > 1 && b.rows > 1 && a.ld == b.ld) {
    // Row j of b starts at byte `off` of a's row `first` + j, and may run into the next.
    if (a.lo > b.lo) std::swap(a, b);
    const uint64_t first = (b.lo - a.lo) / a.ld, off = (b.lo - a.lo) % a.ld;
    return (off < a.bytes && first < a.rows) || (off + b.bytes > a.ld && first + 1 < a.rows);
  }
  if (a.rows > b.rows) std::swap(a, b);
  for (uint64_t r = 0; r < a.rows; ++r) {
    const uintptr_t lo = a.lo + r * a.ld, hi = lo + a.bytes;
    // The first row of b that ends past lo.
    const uint64_t j = b.rows == 1 || lo < b.lo + b.bytes ? 0 : (lo - b.lo - b.bytes) / b.ld + 1;
    if (j < b.rows && b.lo + j * b.ld < hi && b.lo + j * b.ld + b.bytes > lo) return true;
  }
  return false;
}

// Outputs that share memory would be scaled twice, and a gradient that shares
// it with another's output read before or after that: neither has an order.
// Lists come in the order of their addresses more often than not: that needs
// no sorting.
static int check_outputs(const moe_tensor_desc* t, int n) {
  auto live = [&](int i) { return t[i].rows && t[i].cols; };
  uintptr_t last = 0, out_lo = UINTPTR_MAX, out_hi = 0, in_lo = UINTPTR_MAX, in_hi = 0;
  bool sorted = true;
  for (int i = 0; i < n; ++i) {
    if (!live(i)) continue;
    const bool in_place = t[i].out == t[i].in;
    if (in_place && (t[i].in_type != t[i].out_type || (t[i].rows > 1 && t[i].in_ld != t[i].out_ld)))
      return fail(MOE_ERR_INVALID_ARG, "tensor %d is scaled in place with another type or stride", i);
    const Span o = out_span(t[i]);
    sorted = sorted && o.lo >= last;
    last = o.end();
    out_lo = std::min(out_lo, o.lo);
    out_hi = std::max(out_hi, o.end());
    if (!in_place) {
      const Span g = in_span(t[i]);
      in_lo = std::min(in_lo, g.lo);
      in_hi = std::max(in_hi, g.end());
    }
  }
  if (sorted && (in_lo >= out_hi || out_lo >= in_hi)) return 0;
  struct Item {
    Span s;
    uintptr_t end;
    int tensor;
    bool out;
  };
  // All of them by first byte; those that still run when one starts are compared with it.
  Item* items = static_cast<Item*>(malloc(sizeof(Item) * 2 * (size_t)n));
  int* open = static_cast<int*>(malloc(sizeof(int) * 2 * (size_t)n));
  int m = 0, first = -1, second = -1;
  if (items && open) {
    for (int i = 0; i < n; ++i) {
      if (!live(i)) continue;
      const Span o = out_span(t[i]), g = in_span(t[i]);
      items[m++] = Item{o, o.end(), i, true};
      if (t[i].out != t[i].in) items[m++] = Item{g, g.end(), i, false};
    }
    std::sort(items, items + m, [](const Item& x, const Item& y) { return x.s.lo < y.s.lo; });
    int opened = 0;
    for (int x = 0; x < m && first < 0; ++x) {
      int kept = 0;
      for (int y = 0; y < opened; ++y) {
        const Item& o = items[open[y]];
        if (o.end <= items[x].s.lo) continue;
        open[kept++] = open[y];
        if ((o.out || items[x].out) && spans_meet(o.s, items[x].s)) first = open[y], second = x;
      }
      opened = kept;
      open[opened++] = x;
    }
  }
  const bool memory = items && open, outs = first >= 0 && items[first].out && items[second].out;
  const int a = first >= 0 ? items[first].tensor : -1, b = first >= 0 ? items[second].tensor : -1;
  free(items);
  free(open);
  if (!memory) return fail(MOE_ERR_INVALID_ARG, "no memory for a list of %d tensors", n);
  if (first < 0) return 0;
  if (outs)
    return fail(MOE_ERR_INVALID_ARG, "an output is in the list twice, or two of them share memory: tensors %d and %d",
                a, b);
  return fail(MOE_ERR_INVALID_ARG, "an output shares memory with a gradient: tensors %d and %d", a, b);
}

// A norm inside the list would be scaled, or written while the list is read.
static int check_norm_place(const moe_tensor_desc* t, int n, const float* given, const float* norm) {
  const Span g{reinterpret_cast<uintptr_t>(given), 1, given ? sizeof(float) : 0, 0};
  const Span w{reinterpret_cast<uintptr_t>(norm), 1, norm && norm != given ? sizeof(float) : 0, 0};
  for (int i = 0; i < n; ++i) {
    if (!t[i].rows || !t[i].cols) continue;
    const Span o = out_span(t[i]);
    if ((g.bytes && spans_meet(g, o)) || (w.bytes && (spans_meet(w, o) || spans_meet(w, in_span(t[i])))))
      return fail(MOE_ERR_INVALID_ARG, "the norm lies in tensor %d", i);
  }
  return 0;
}

static int entry_head(const GradEntry& e) {
  const size_t in = reinterpret_cast<uintptr_t>(e.in), out = reinterpret_cast<uintptr_t>(e.out);
  const size_t ib = elem_bytes(e.in_type), ob = elem_bytes(e.out_type);
  const size_t ce = chunk_elems(e.in_type), store = std::min<size_t>(16, ce * ob);
  if (e.rows > 1)
    return e.cols % ce == 0 && in % 16 == 0 && out % store == 0 && e.in_ld * ib % 16 == 0 && e.out_ld * ob % store == 0
               ? 0
               : -1;
  for (int h = 0; h < 8 && h <= e.cols; ++h)
    if ((in + h * ib) % 16 == 0 && (out + h * ob) % store == 0) return h;
  return -1;
}

// Fills `list` with tensors from *at on (of the pair of types `pair`, or all:
// -1); false when none is left.
static int type_pair(const moe_tensor_desc& d) { return d.in_type * 3 + d.out_type; }
template <int SLOTS>
static bool fill_list(GradList<SLOTS>& list, const moe_tensor_desc* t, int n, int* at, int pair) {
  const bool with_out = pair >= 0;
  list.n = 0;
  uint64_t units = 0;
  for (; *at < n && list.n < SLOTS; ++*at) {
    const moe_tensor_desc& d = t[*at];
    if (d.rows == 0 || d.cols == 0 || (with_out && type_pair(d) != pair)) continue;
    GradEntry& e = list.e[list.n];
    e = GradEntry{d.in, with_out ? d.out : const_cast<void*>(d.in), d.rows, d.cols, d.in_ld,
                  with_out ? d.out_ld : d.in_ld, (int16_t)d.in_type, (int16_t)(with_out ? d.out_type : d.in_type), 0};
    e.head = (int16_t)entry_head(e);
    list.unit0[list.n] = (uint32_t)units;
    const uint64_t per = unit_elems(d.in_type), more = ((uint64_t)d.rows * d.cols + per - 1) / per;
    units += more;
    ++list.n;
  }
  list.units = (uint32_t)units;
  return list.n > 0;
}

static bool norm_large(const moe_tensor_desc* t, int n) {
  uint64_t units = 0;
  for (int i = 0; i < n; ++i) units += ((uint64_t)t[i].rows * t[i].cols) / unit_elems(t[i].in_type) + 1;
  return units > kNormLarge;
}

template <int NORM, int SLOTS>
static int launch_partials(const moe_tensor_desc* t, int n, bool large, double* partial, int* count, cudaStream_t st) {
  int at = 0;
  *count = 0;
  GradList<SLOTS> list;
  while (fill_list(list, t, n, &at, -1)) {
    const int blocks = (int)std::min<uint32_t>(list.units, large ? kNormMaxBlocks : kNormResident);
    norm_partial_kernel<NORM, SLOTS><<<blocks, kNormThreads, 0, st>>>(list, partial + *count);
    MOE_CUDA_TRY(cudaGetLastError());
    *count += blocks;
  }
  return 0;
}
template <int NORM>
static int run_partials(const moe_tensor_desc* t, int n, bool large, double* partial, int* count, cudaStream_t st) {
  if (n <= kGradSlotsSmall) return launch_partials<NORM, kGradSlotsSmall>(t, n, large, partial, count, st);
  return launch_partials<NORM, kGradSlots>(t, n, large, partial, count, st);
}
// The partials of all tensors; their number.
static int norm_partials(int norm_type, const moe_tensor_desc* t, int n, bool large, double* partial, int* count,
                         cudaStream_t st) {
  if (norm_type == MOE_NORM_L1) return run_partials<kNormL1>(t, n, large, partial, count, st);
  if (norm_type == MOE_NORM_L2) return run_partials<kNormL2>(t, n, large, partial, count, st);
  return run_partials<kNormInf>(t, n, large, partial, count, st);
}

template <int SLOTS, int IN, int OUT>
static int launch_clip_pair(const moe_tensor_desc* t, int n, bool large, ClipNorm* c, cudaStream_t st) {
  int at = 0;
  GradList<SLOTS> list;
  while (fill_list(list, t, n, &at, IN * 3 + OUT)) {
    const uint32_t blocks = large ? list.units : std::min<uint32_t>(list.units, kNormResident);
    clip_kernel<IN, OUT, SLOTS><<<blocks, kNormThreads, 0, st>>>(list, *c);
    MOE_CUDA_TRY(cudaGetLastError());
    c->norm = nullptr;  // the first launch writes it
  }
  return 0;
}
template <int SLOTS>
static int launch_clip(const moe_tensor_desc* t, int n, bool large, ClipNorm c, cudaStream_t st) {
  unsigned pairs = 0;
  for (int i = 0; i < n; ++i)
    if (t[i].rows && t[i].cols) pairs |= 1u << type_pair(t[i]);
  int r = 0;
  if (!r && (pairs & 1u)) r = launch_clip_pair<SLOTS, 0, 0>(t, n, large, &c, st);
  if (!r && (pairs & 2u)) r = launch_clip_pair<SLOTS, 0, 1>(t, n, large, &c, st);
  if (!r && (pairs & 4u)) r = launch_clip_pair<SLOTS, 0, 2>(t, n, large, &c, st);
  if (!r && (pairs & 8u)) r = launch_clip_pair<SLOTS, 1, 0>(t, n, large, &c, st);
  if (!r && (pairs & 16u)) r = launch_clip_pair<SLOTS, 1, 1>(t, n, large, &c, st);
  if (!r && (pairs & 32u)) r = launch_clip_pair<SLOTS, 1, 2>(t, n, large, &c, st);
  if (!r && (pairs & 64u)) r = launch_clip_pair<SLOTS, 2, 0>(t, n, large, &c, st);
  if (!r && (pairs & 128u)) r = launch_clip_pair<SLOTS, 2, 1>(t, n, large, &c, st);
  if (!r && (pairs & 256u)) r = launch_clip_pair<SLOTS, 2, 2>(t, n, large, &c, st);
  return r;
}

static int run_clip(const moe_tensor_desc* t, int n, int norm_type, double max_norm, const float* given, float* norm,
                    double* partial, cudaStream_t st) {
  const bool large = norm_large(t, n);
  ClipNorm c{partial, 0, norm_type, given, norm, max_norm};
  if (!given) {
    if (int r = norm_partials(norm_type, t, n, large, partial, &c.n, st)) return r;
    if (c.n == 0) {  // no elements: the norm is 0 and there is nothing to scale
      MOE_CUDA_TRY(cudaMemsetAsync(norm, 0, sizeof(float), st));
      return 0;
    }
    if (large) {
      norm_finish_kernel<<<1, kNormThreads, 0, st>>>(norm_type, partial, c.n, norm);
      MOE_CUDA_TRY(cudaGetLastError());
      c.given = norm;
    }
  } else if (norm && norm != given) {
    MOE_CUDA_TRY(cudaMemcpyAsync(norm, given, sizeof(float), cudaMemcpyDeviceToDevice, st));
  }
  return n <= kGradSlotsSmall ? launch_clip<kGradSlotsSmall>(t, n, large, c, st)
                              : launch_clip<kGradSlots>(t, n, large, c, st);
}

}  // namespace moe

using namespace moe;

extern "C" {

// ------------------------------------------------------------------ routing
int64_t moe_route_train_counters(int64_t T, int32_t E, int64_t sequences) {
  if (T < 0 || E < 1 || E > kRouteMaxExperts || sequences < 1 || T % sequences) return 0;
  return route_counters(route_chunks(T / sequences, sequences, E), sequences, E);
}

size_t moe_route_train_workspace_size(int64_t T, int32_t E, int64_t sequences) {
  if (T < 0 || E < 1 || E > kRouteMaxExperts || sequences < 1 || T % sequences) return 0;
  return route_space(route_chunks(T / sequences, sequences, E), sequences, E).bytes;
}

int moe_route_train(const void* logits, int32_t elem_type, int64_t ld, int64_t T, int32_t E, int32_t k,
                    int64_t sequences, const uint8_t* mask, const int32_t* given_ids, int32_t scoring,
                    int32_t normalize, int32_t* ids, float* weights, int32_t* counts, int32_t* tokens, float* balance,
                    float* z, void* workspace, size_t workspace_bytes, uint32_t* counters, void* stream) {
  t_err[0] = 0;
  if (int r = check_route(elem_type, ld, T, E, k, sequences, scoring)) return r;
  if (!counts || !tokens || !balance || !z) return fail(MOE_ERR_INVALID_ARG, "null pointer");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    MOE_CUDA_TRY(cudaMemsetAsync(counts, 0, (size_t)sequences * E * sizeof(int32_t), st));
    MOE_CUDA_TRY(cudaMemsetAsync(tokens, 0, (size_t)sequences * sizeof(int32_t), st));
    MOE_CUDA_TRY(cudaMemsetAsync(balance, 0, sizeof(float), st));
    MOE_CUDA_TRY(cudaMemsetAsync(z, 0, sizeof(float), st));
    return 0;
  }
  if (!logits || !ids || !weights || !counters) return fail(MOE_ERR_INVALID_ARG, "null pointer");
  if (reinterpret_cast<uintptr_t>(logits) % elem_bytes(elem_type))
    return fail(MOE_ERR_MISALIGNED, "logits are not aligned to their elements");
  const int64_t seq_len = T / sequences, chunks = route_chunks(seq_len, sequences, E), blocks = chunks * sequences;
  const RouteSpace s = route_space(chunks, sequences, E);
  if (!workspace || workspace_bytes < s.bytes)
    return fail(MOE_ERR_WORKSPACE_TOO_SMALL, "workspace %zu bytes < required %zu", workspace_bytes, s.bytes);
  if (reinterpret_cast<uintptr_t>(workspace) & 255u)
    return fail(MOE_ERR_MISALIGNED, "workspace must be 256-byte aligned");
  int dev;
  DevInfo* di;
  if (int r = device_info(&dev, &di)) return r;
  uint8_t* w = static_cast<uint8_t*>(workspace);
  RouteParams p{};
  p.logits = logits;
  p.mask = mask;
  p.given = given_ids;
  p.ids = ids;
  p.weights = weights;
  p.part_q = reinterpret_cast<float*>(w + s.q);
  p.part_c = reinterpret_cast<int32_t*>(w + s.c);
  p.part_z = reinterpret_cast<double*>(w + s.z);
  p.part_n = reinterpret_cast<int32_t*>(w + s.n);
  p.seq_part = reinterpret_cast<double*>(w + s.seq);
  p.counts = counts;
  p.tokens = tokens;
  p.balance = balance;
  p.z = z;
  p.counters = counters;
  p.S = (int32_t)sequences;
  p.ld = ld;
  p.seq_len = seq_len;
  p.chunks = (int32_t)chunks;
  p.E = E;
  p.k = k;
  p.type = elem_type;
  p.vec = route_vec(logits, ld, E, elem_type);
  p.sigmoid = scoring == MOE_SCORE_SIGMOID;
  p.normalize = normalize != 0;
  if (E > 512) return launch_route_k<32, 32>(p, blocks, st);
  if (E <= 8) return launch_route_k<1, 8>(p, blocks, st);
  if (E <= 16) return launch_route_k<2, 8>(p, blocks, st);
  switch (route_lanes(E)) {
    case 2: return launch_route_k<2, 16>(p, blocks, st);
    case 4: return launch_route_k<4, 16>(p, blocks, st);
    case 8: return launch_route_k<8, 16>(p, blocks, st);
    case 16: return launch_route_k<16, 16>(p, blocks, st);
  }
  return launch_route_k<32, 16>(p, blocks, st);
}

int moe_route_backward(const void* logits, int32_t elem_type, int64_t ld, int64_t T, int32_t E, int32_t k,
                       int64_t sequences, const uint8_t* mask, int32_t scoring, int32_t normalize, const int32_t* ids,
                       const float* weights, const int32_t* counts, const int32_t* tokens, const float* d_weights,
                       const float* d_balance, const float* d_z, void* d_logits, void* stream) {
  t_err[0] = 0;
  if (int r = check_route(elem_type, ld, T, E, k, sequences, scoring)) return r;
  if (T == 0) return 0;
  if (!logits || !ids || !weights || !counts || !tokens || !d_logits) return fail(MOE_ERR_INVALID_ARG, "null pointer");
  if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(d_logits)) % elem_bytes(elem_type))
    return fail(MOE_ERR_MISALIGNED, "logits or d_logits are not aligned to their elements");
  int dev;
  DevInfo* di;
  if (int r = device_info(&dev, &di)) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  RouteBackward p{};
  p.logits = logits;
  p.mask = mask;
  p.ids = ids;
  p.weights = weights;
  p.counts = counts;
  p.tokens = tokens;
  p.d_weights = d_weights;
  p.d_balance = d_balance;
  p.d_z = d_z;
  p.d_logits = d_logits;
  p.ld = ld;
  p.seq_len = T / sequences;
  p.chunks = (int32_t)route_chunks(p.seq_len, sequences, E);
  p.S = (int32_t)sequences;
  p.E = E;
  p.k = k;
  p.type = elem_type;
  p.vec = route_vec(logits, ld, E, elem_type);
  p.vec_out = route_vec(d_logits, E, E, elem_type);
  p.sigmoid = scoring == MOE_SCORE_SIGMOID;
  p.normalize = normalize != 0;
  // Every block adds up the sequences' tokens: with more sequences than this,
  // only as many blocks as are resident do, and take several sequences each
  // (131072 of one token each, E = 8: 23 ms with all blocks and each warp's own
  // sum, 0.7 so).
  int64_t blocks = p.chunks * sequences;
  if (sequences > 4096) blocks = std::min<int64_t>(blocks, 148 * (E > 512 ? 2 : 3));
  if (E > 512) return launch_backward_k<32, 32>(p, blocks, st);
  if (E <= 8) return launch_backward_k<1, 8>(p, blocks, st);
  if (E <= 16) return launch_backward_k<2, 8>(p, blocks, st);
  switch (route_lanes(E)) {
    case 2: return launch_backward_k<2, 16>(p, blocks, st);
    case 4: return launch_backward_k<4, 16>(p, blocks, st);
    case 8: return launch_backward_k<8, 16>(p, blocks, st);
    case 16: return launch_backward_k<16, 16>(p, blocks, st);
  }
  return launch_backward_k<32, 16>(p, blocks, st);
}

// ------------------------------------------------------------------ rows
int moe_combine_rows_backward(const void* dy, int32_t dy_type, const float* y_sorted, const int32_t* inverse,
                              const float* weights, const int32_t* group_sizes, int64_t T, int32_t k, int32_t D,
                              int64_t rows, int32_t E, void* dys, int32_t dys_type, float* dw, void* stream) {
  t_err[0] = 0;
  if (int r = check_rows(T, k, D, rows, dy_type, dys_type)) return r;
  if (E < 1) return fail(MOE_ERR_INVALID_ARG, "E=%d", E);
  if (T == 0 && rows == 0) return 0;
  if (!group_sizes || (T && (!dy || !inverse || !weights || !dw)) || (rows && (!y_sorted || !dys)))
    return fail(MOE_ERR_INVALID_ARG, "null pointer");
  if (!row_aligned(dy, dy_type) || !aligned16(y_sorted) || !row_aligned(dys, dys_type))
    return fail(MOE_ERR_MISALIGNED, "rows must be aligned to 4 elements");
  int dev;
  DevInfo* di;
  if (int r = device_info(&dev, &di)) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  CombineBwd p{dy, y_sorted, inverse, weights, dys, dw, T, rows, k, D, 0, 0};
  // Rows that no entry maps to are found by blocks that read all of `inverse`
  // each, beside the others' work, unless that reads more than zeroing all of
  // dys beforehand writes (very many short rows).
  const int64_t row_bytes = (int64_t)D * elem_bytes(dys_type);
  int shift = 0;
  while (shift < zero_shift_most(D) && ((int64_t)kRowThreads << shift) < rows * (D / 4)) ++shift;
  while (((int64_t)kZeroRows << shift) < rows) ++shift;
  if (((T * k * 4) << shift) <= std::max<int64_t>(rows * row_bytes, 8 << 20)) {
    p.zero_blocks = rows ? 1 << shift : 0;
    p.zero_shift = shift;
  } else {
    MOE_CUDA_TRY(cudaMemsetAsync(dys, 0, (size_t)(rows * row_bytes), st));
  }
  const int tpt = row_threads(D);
  if (tpt == 256) return launch_combine_t<256>(p, dy_type, dys_type, st);
  if (tpt == 32) return launch_combine_t<32>(p, dy_type, dys_type, st);
  return launch_combine_t<8>(p, dy_type, dys_type, st);
}

int moe_gather_rows_backward(const void* dxs, int32_t dxs_type, const int32_t* inverse, int64_t T, int32_t k,
                             int32_t D, int64_t rows, void* dx, int32_t dx_type, void* stream) {
  t_err[0] = 0;
  if (int r = check_rows(T, k, D, rows, dxs_type, dx_type)) return r;
  if (T == 0) return 0;
  if (!inverse || !dx || (rows && !dxs)) return fail(MOE_ERR_INVALID_ARG, "null pointer");
  if (!row_aligned(dxs, dxs_type) || !row_aligned(dx, dx_type))
    return fail(MOE_ERR_MISALIGNED, "rows must be aligned to 4 elements");
  int dev;
  DevInfo* di;
  if (int r = device_info(&dev, &di)) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const GatherBwd p{dxs, inverse, dx, T, rows, k, D};
  const int tpt = row_threads(D);
  if (tpt == 256) return launch_gather_t<256>(p, dxs_type, dx_type, st);
  if (tpt == 32) return launch_gather_t<32>(p, dxs_type, dx_type, st);
  return launch_gather_t<8>(p, dxs_type, dx_type, st);
}

// ------------------------------------------------------------------ gradient lists
size_t moe_grad_norm_workspace_size(int32_t n) {
  if (n < 0) return 0;
  const size_t launches = (size_t)std::max(1, (n + kGradSlots - 1) / kGradSlots);
  return align256(launches * kNormMaxBlocks * sizeof(double));
}

static int check_norm_space(int n, const void* ws, size_t bytes) {
  const size_t need = moe_grad_norm_workspace_size(n);
  if (!ws || bytes < need) return fail(MOE_ERR_WORKSPACE_TOO_SMALL, "workspace %zu bytes < required %zu", bytes, need);
  if (reinterpret_cast<uintptr_t>(ws) & 255u) return fail(MOE_ERR_MISALIGNED, "workspace must be 256-byte aligned");
  return 0;
}

int moe_grad_norm(const moe_tensor_desc* tensors, int32_t n, int32_t norm_type, float* norm, void* workspace,
                  size_t workspace_bytes, void* stream) {
  t_err[0] = 0;
  if (int r = check_tensors(tensors, n, norm_type, false)) return r;
  if (!norm) return fail(MOE_ERR_INVALID_ARG, "null norm");
  if (int r = check_norm_space(n, workspace, workspace_bytes)) return r;
  int dev;
  DevInfo* di;
  if (int r = device_info(&dev, &di)) return r;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  int count = 0;
  if (int r = norm_partials(norm_type, tensors, n, norm_large(tensors, n), partial, &count, st)) return r;
  norm_finish_kernel<<<1, kNormThreads, 0, st>>>(norm_type, partial, count, norm);
  MOE_CUDA_TRY(cudaGetLastError());
  return 0;
}

int moe_clip_grads(const moe_tensor_desc* tensors, int32_t n, int32_t norm_type, double max_norm,
                   const float* given_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  t_err[0] = 0;
  if (int r = check_tensors(tensors, n, norm_type, true)) return r;
  if (int r = check_outputs(tensors, n)) return r;
  if (!(max_norm >= 0.0)) return fail(MOE_ERR_INVALID_ARG, "max_norm %g", max_norm);
  if (!given_norm && !norm) return fail(MOE_ERR_INVALID_ARG, "null norm");
  if (!given_norm)
    if (int r = check_norm_space(n, workspace, workspace_bytes)) return r;
  if (int r = check_norm_place(tensors, n, given_norm, norm)) return r;
  int dev;
  DevInfo* di;
  if (int r = device_info(&dev, &di)) return r;
  return run_clip(tensors, n, norm_type, max_norm, given_norm, norm, static_cast<double*>(workspace),
                  static_cast<cudaStream_t>(stream));
}

}  // extern "C"
