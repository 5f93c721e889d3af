// Router of a mixture-of-experts block: top-k of the router's logits with softmax weights, and the dispatch
// plan that the grouped products read (rows sorted by expert).
//
// Per token t with logits l[0..E):
//   candidates   the experts with l > -inf (NaN counts as -inf); ids[t, 0..k) are the k largest in falling order,
//                equal logits by lower index; -1 with weight 0 where fewer than k candidates exist
//   weights      p_s = exp(l_s - m) / sum, m = max l, the sum over the chosen (renormalize) or over all candidates,
//                times `scale`; l = +inf counts as exp(0) against m = +inf, the softmax's limit
// Plan for the local experts [e_begin, e_begin + e_count): the (token, slot) pairs whose id is local, sorted by
// expert and inside an expert by t * k + s (so the plan is the same on every run):
//   offsets[e] .. offsets[e + 1]   rows of local expert e
//   row_token[r]                   token of row r, -1 past offsets[e_count]
//   slot_row[t, s]                 row of the pair, -1 when its expert is not local
//
// All of it is latency: T * E logits are read once (2 MB at T = 8192, E = 128). One warp owns a token: each lane
// keeps E / 32 logits as ordered integer keys, and a round of the selection is two warp reductions (redux: the
// maximum, then the lowest index that has it). The plan is a counting sort over CTAs that own contiguous token
// ranges: k_moe_route counts per CTA and expert, k_moe_place adds the counts of the earlier CTAs and places its
// own pairs, ranked inside a warp by match_any. Up to kRouteFuse tokens one CTA does both in one launch.
#pragma once
#include "bs_common.cuh"

namespace bs {

constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 32;
constexpr int kRouteThreads = 1024;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteFuse = 32;   // tokens up to which one CTA counts and places (one round of its 32 warps)
constexpr int kRouteBatch = 256; // pairs ranked at a time: 8 warps' counts in shared memory

struct RouteParams {
  const void* logits;   // [T, ldl] bf16 or fp32; nullptr: ids are given
  const int* ids_in;    // [T, k] when logits == nullptr
  long long ldl;
  int T, E, k;          // E: all experts
  int renormalize;
  float scale;
  int e_begin, e_count; // local experts
  int per_cta;          // tokens per CTA
  float* weights;       // [T, k] (with logits)
  int* ids;             // [T, k] (with logits)
  int* offsets;         // [e_count + 1]
  int* row_token;       // [T * k]
  int* slot_row;        // [T, k]
  int* hist;            // [grid, e_count] counts per CTA (grid > 1)
};

struct RouteSmem {
  int base[kMaxExperts];   // next row of each expert for this CTA
  int count[kMaxExperts];  // this CTA's pairs per expert; later all CTAs'
  int wcnt[kRouteBatch / 32][kMaxExperts];
  int total;
};

// Unsigned key that orders like the float, 0 for what can never be chosen (-inf, NaN). -0 and +0 are one key.
__device__ __forceinline__ uint32_t route_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  const uint32_t key = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (x > -INFINITY) ? key : 0u;  // false for NaN too
}
__device__ __forceinline__ float route_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}
// exp(x - m) for x <= m, with the limit 1 at x == m == +inf.
__device__ __forceinline__ float route_exp(float x, float m) { return x == m ? 1.0f : expf(x - m); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Top-k of one token by one warp; lane s < k leaves with id (-1: none) and weight of slot s.
template <int VPL>
__device__ __forceinline__ void route_token(const RouteParams& p, bool f32, int t, int lane, int& id, float& w) {
  uint32_t key[VPL];
  const long long row = static_cast<long long>(t) * p.ldl;
#pragma unroll
  for (int j = 0; j < VPL; ++j) {
    const int e = lane + 32 * j;
    float x = -INFINITY;
    if (e < p.E)
      x = f32 ? __ldg(static_cast<const float*>(p.logits) + row + e)
              : __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p.logits) + row + e));
    key[j] = route_key(x);
  }
  float m = 0.f, all = 0.f;
  if (!p.renormalize) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j) top = max(top, key[j]);
    m = route_value(__reduce_max_sync(0xffffffffu, top));
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (key[j]) all += route_exp(route_value(key[j]), m);
    all = warp_sum(all);
  }
  id = -1;
  uint32_t mine = 0;
  for (int s = 0; s < p.k; ++s) {
    uint32_t best = 0;
    int at = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (key[j] > best) {
        best = key[j];
        at = lane + 32 * j;
      }
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    if (top == 0) break;
    const int won = static_cast<int>(__reduce_min_sync(0xffffffffu, best == top ? static_cast<uint32_t>(at) : 0x7fffffffu));
    if (s == 0) m = route_value(top);
    if (lane == s) {
      id = won;
      mine = top;
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j)
      if (won == lane + 32 * j) key[j] = 0;
  }
  w = mine ? route_exp(route_value(mine), m) : 0.f;
  const float sum = p.renormalize ? warp_sum(w) : all;
  w = mine ? __fmul_rn(__fdiv_rn(w, sum), p.scale) : 0.f;
}

// Exclusive prefix of sm.count over the local experts into `base` (added to what base holds), by warp 0.
__device__ __forceinline__ void route_scan(RouteSmem& sm, const RouteParams& p, bool write_offsets) {
  const int lane = threadIdx.x & 31;
  int run = 0;
  for (int e0 = 0; e0 < p.e_count; e0 += 32) {
    const int e = e0 + lane;
    const int c = e < p.e_count ? sm.count[e] : 0;
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (e < p.e_count) {
      sm.base[e] += run + inc - c;
      if (write_offsets) p.offsets[e] = run + inc - c;
    }
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) {
    sm.total = run;
    if (write_offsets) p.offsets[p.e_count] = run;
  }
}

// Places the pairs of tokens [t0, t1): sm.base holds each expert's next row.
__device__ __forceinline__ void route_place(RouteSmem& sm, const RouteParams& p, const int* ids, int t0, int t1) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long n0 = static_cast<long long>(t0) * p.k, n1 = static_cast<long long>(t1) * p.k;
  for (long long b = n0; b < n1; b += kRouteBatch) {
    const int nw = static_cast<int>(min(static_cast<long long>(kRouteBatch), n1 - b) + 31) / 32;
    __syncthreads();  // the counts of the previous batch are used up; the first batch's base is there
    for (int w = 0; w < nw; ++w)
      for (int e = tid; e < p.e_count; e += kRouteThreads) sm.wcnt[w][e] = 0;
    __syncthreads();
    const long long i = b + tid;
    int e = -1, rank = 0;
    if (warp < nw) {
      if (i < n1) e = ids[i] - p.e_begin;
      if (static_cast<unsigned>(e) >= static_cast<unsigned>(p.e_count)) e = -1;
      const uint32_t same = __match_any_sync(0xffffffffu, e);
      rank = __popc(same & ((1u << lane) - 1));
      if (e >= 0 && rank == 0) sm.wcnt[warp][e] = __popc(same);
    }
    __syncthreads();
    for (int x = tid; x < p.e_count; x += kRouteThreads) {
      int run = sm.base[x];
      for (int w = 0; w < nw; ++w) {
        const int c = sm.wcnt[w][x];
        sm.wcnt[w][x] = run;
        run += c;
      }
      sm.base[x] = run;
    }
    __syncthreads();
    if (warp < nw && i < n1) {
      int r = -1;
      if (e >= 0) {
        r = sm.wcnt[warp][e] + rank;
        p.row_token[r] = static_cast<int>(i / p.k);
      }
      p.slot_row[i] = r;
    }
  }
}

__device__ __forceinline__ void route_fill(const RouteSmem& sm, const RouteParams& p) {
  const long long R = static_cast<long long>(p.T) * p.k;
  for (long long i = sm.total + static_cast<long long>(blockIdx.x) * kRouteThreads + threadIdx.x; i < R;
       i += static_cast<long long>(gridDim.x) * kRouteThreads)
    p.row_token[i] = -1;
}

// CTA b owns tokens [b * per_cta, (b + 1) * per_cta). VPL = 0: ids are given.
template <int VPL>
__global__ void __launch_bounds__(kRouteThreads) k_moe_route(const RouteParams p, const int f32) {
  __shared__ RouteSmem sm;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) grid_dep_launch();
  for (int e = tid; e < p.e_count; e += kRouteThreads) sm.count[e] = sm.base[e] = 0;
  __syncthreads();
  grid_dep_wait();  // the logits may be the previous kernel's output, the plan its input
  const int t0 = blockIdx.x * p.per_cta, t1 = min(p.T, t0 + p.per_cta);
  if constexpr (VPL > 0) {
    for (int t = t0 + warp; t < t1; t += kRouteWarps) {
      int id;
      float w;
      route_token<VPL>(p, f32 != 0, t, lane, id, w);
      if (lane < p.k) {
        const long long i = static_cast<long long>(t) * p.k + lane;
        p.ids[i] = id;
        p.weights[i] = w;
        const int e = id - p.e_begin;
        if (id >= 0 && static_cast<unsigned>(e) < static_cast<unsigned>(p.e_count)) atomicAdd(&sm.count[e], 1);
      }
    }
  } else {
    const long long n1 = static_cast<long long>(t1) * p.k;
    for (long long i = static_cast<long long>(t0) * p.k + tid; i < n1; i += kRouteThreads) {
      const int e = p.ids_in[i] - p.e_begin;
      if (static_cast<unsigned>(e) < static_cast<unsigned>(p.e_count)) atomicAdd(&sm.count[e], 1);
    }
  }
  __syncthreads();
  if (gridDim.x > 1) {
    for (int e = tid; e < p.e_count; e += kRouteThreads) p.hist[static_cast<size_t>(blockIdx.x) * p.e_count + e] = sm.count[e];
    return;
  }
  if (warp == 0) route_scan(sm, p, true);
  // (the barrier also makes this CTA's ids, written above, visible to all of its threads)
  route_place(sm, p, VPL > 0 ? p.ids : p.ids_in, t0, t1);
  __syncthreads();
  route_fill(sm, p);
}

// Second launch of a plan over several CTAs: same token ranges as the k_moe_route that wrote p.hist.
__global__ void __launch_bounds__(kRouteThreads) k_moe_place(const RouteParams p) {
  __shared__ RouteSmem sm;
  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) grid_dep_launch();
  for (int e = tid; e < p.e_count; e += kRouteThreads) sm.count[e] = sm.base[e] = 0;
  __syncthreads();
  grid_dep_wait();
  // thread (part, e): the counts of CTAs part, part + parts, ... of expert e; integer sums, so the order is free
  int width = 32;
  while (width < p.e_count) width <<= 1;
  const int parts = kRouteThreads / width, e = tid & (width - 1), part = tid / width;
  if (e < p.e_count) {
    int all = 0, before = 0;
    for (int b = part; b < static_cast<int>(gridDim.x); b += parts) {
      const int c = __ldcg(p.hist + static_cast<size_t>(b) * p.e_count + e);
      all += c;
      if (b < static_cast<int>(blockIdx.x)) before += c;
    }
    if (all) atomicAdd(&sm.count[e], all);
    if (before) atomicAdd(&sm.base[e], before);
  }
  __syncthreads();
  if (warp == 0) route_scan(sm, p, blockIdx.x == 0);
  const int t0 = blockIdx.x * p.per_cta, t1 = min(p.T, t0 + p.per_cta);
  route_place(sm, p, p.ids ? p.ids : p.ids_in, t0, t1);
  __syncthreads();
  route_fill(sm, p);
}

}  // namespace bs
