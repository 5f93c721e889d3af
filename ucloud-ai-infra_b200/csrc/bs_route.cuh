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
// ranges: k_moe_route ranks each CTA's pairs inside the CTA (match_any inside a warp, a prefix over warps) and leaves
// its counts per expert, k_moe_place adds the counts of the earlier CTAs and the lower experts. (Ranking in the second
// kernel instead: 25 us at 8192 tokens against 17.) Up to kRouteCluster tokens one launch does both: its CTAs, up to 16,
// are one cluster and read each other's counts in shared memory.
#pragma once
#include "bs_common.cuh"

namespace bs {

constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 32;
constexpr int kRouteThreads = 1024;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteRound = 32;   // tokens of one round of a CTA's 32 warps
constexpr int kRouteCluster = 512; // tokens up to which one cluster counts and places in one launch: 16 CTAs, or 8 by two rounds
constexpr int kRouteBatch = 256; // pairs ranked at a time: 8 warps' counts in shared memory
constexpr int kRouteRankWarps = kRouteBatch / 32;

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
  int* hist;            // [grid, e_count] counts per CTA for k_moe_place; nullptr: the grid is one cluster
};

struct RouteSmem {
  int count[kMaxExperts];                   // this CTA's pairs per expert so far; k_moe_place: all CTAs'
  int base[kMaxExperts];                    // rows before this CTA's, by expert
  int wcnt[kRouteRankWarps][kMaxExperts];
  int wsum[kMaxExperts / 32];
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

// sm.base[e] += the pairs of the experts below e (all CTAs' in sm.count); sm.total. Every thread of the CTA calls it, after
// a barrier; the result is there after the one inside.
__device__ __forceinline__ void route_scan(RouteSmem& sm, const RouteParams& p, bool write_offsets) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int c = tid < p.e_count ? sm.count[tid] : 0;  // kMaxExperts <= threads
  int inc = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31 && warp < kMaxExperts / 32) sm.wsum[warp] = inc;
  __syncthreads();
  if (tid < p.e_count) {
    int before = inc - c;
    for (int w = 0; w < warp; ++w) before += sm.wsum[w];
    sm.base[tid] += before;
    if (write_offsets) p.offsets[tid] = before;
    if (tid == p.e_count - 1) {
      sm.total = before + c;
      if (write_offsets) p.offsets[p.e_count] = before + c;
    }
  }
  __syncthreads();
}

// Ranks pairs [b, min(b + kRouteBatch, n1)) of this CTA by expert, in order, after those ranked before (sm.count, which
// it brings up to date): slot_row gets the rank inside the CTA, -1 without a local expert. A barrier has to stand between
// two batches: the end of one reads the counts that the start of the next one zeroes.
__device__ __forceinline__ void route_rank(RouteSmem& sm, const RouteParams& p, const int* ids, long long b, long long n1) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nw = static_cast<int>(min(static_cast<long long>(kRouteBatch), n1 - b) + 31) / 32;
  for (int i = tid; i < kRouteRankWarps * p.e_count; i += kRouteThreads) sm.wcnt[i / p.e_count][i % p.e_count] = 0;
  __syncthreads();  // (also: the ids that this CTA has written are visible to all of it)
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
  if (tid < p.e_count) {
    int c[kRouteRankWarps];
#pragma unroll
    for (int w = 0; w < kRouteRankWarps; ++w) c[w] = sm.wcnt[w][tid];
    int run = sm.count[tid];
#pragma unroll
    for (int w = 0; w < kRouteRankWarps; ++w) {
      sm.wcnt[w][tid] = run;
      run += c[w];
    }
    sm.count[tid] = run;
  }
  __syncthreads();
  if (warp < nw && i < n1) p.slot_row[i] = e >= 0 ? sm.wcnt[warp][e] + rank : -1;
}

// Rank -> row: adds the rows before this CTA's and writes both directions of the plan for tokens [t0, t1).
__device__ __forceinline__ void route_place(const RouteSmem& sm, const RouteParams& p, const int* ids, int t0, int t1) {
  const long long n1 = static_cast<long long>(t1) * p.k;
  for (long long i = static_cast<long long>(t0) * p.k + threadIdx.x; i < n1; i += kRouteThreads) {
    const int rank = p.slot_row[i];
    if (rank < 0) continue;
    const int r = sm.base[ids[i] - p.e_begin] + rank;
    p.slot_row[i] = r;
    p.row_token[r] = static_cast<int>(i / p.k);
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
  static_assert(kMaxExperts <= kRouteThreads, "a thread per expert");
  if (tid == 0) grid_dep_launch();
  if (tid < p.e_count) sm.count[tid] = sm.base[tid] = 0;
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
      }
    }
  }
  const int* ids = VPL > 0 ? p.ids : p.ids_in;
  const long long n1 = static_cast<long long>(t1) * p.k;
  for (long long b = static_cast<long long>(t0) * p.k; b < n1; b += kRouteBatch) {
    route_rank(sm, p, ids, b, n1);
    __syncthreads();  // every warp has used this batch's counts
  }
  if (p.hist) {
    if (tid < p.e_count) p.hist[static_cast<size_t>(blockIdx.x) * p.e_count + tid] = sm.count[tid];
    return;
  }
  if (gridDim.x > 1) {
    cluster_sync_all();  // every CTA's counts are final
    int all = 0, before = 0;
    if (tid < p.e_count)
      for (uint32_t b = 0; b < gridDim.x; ++b) {
        int c;
        asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c) : "r"(mapa_shared(&sm.count[tid], b)) : "memory");
        all += c;
        before += b < blockIdx.x ? c : 0;
      }
    cluster_sync_all();  // and read by everyone, so they may change and their CTA may end
    if (tid < p.e_count) {
      sm.count[tid] = all;
      sm.base[tid] = before;
    }
    __syncthreads();
  }
  route_scan(sm, p, blockIdx.x == 0);
  route_place(sm, p, ids, t0, t1);
  route_fill(sm, p);
}

// Second launch of a plan over several CTAs: same token ranges as the k_moe_route that wrote p.hist.
__global__ void __launch_bounds__(kRouteThreads) k_moe_place(const RouteParams p) {
  __shared__ RouteSmem sm;
  const int tid = threadIdx.x;
  if (tid == 0) grid_dep_launch();
  if (tid < p.e_count) sm.count[tid] = sm.base[tid] = 0;
  __syncthreads();
  grid_dep_wait();
  // thread (part, e): the counts of CTAs part, part + parts, ... of expert e; integer sums, so the order is free
  int width = 32;
  while (width < p.e_count) width <<= 1;
  const int parts = kRouteThreads / width, e = tid & (width - 1), part = tid / width;
  if (e < p.e_count) {
    const int G = static_cast<int>(gridDim.x), me = static_cast<int>(blockIdx.x);
    int all = 0, before = 0;
#pragma unroll 8
    for (int b = part; b < G; b += parts) {
      const int c = __ldcg(p.hist + static_cast<size_t>(b) * p.e_count + e);
      all += c;
      before += b < me ? c : 0;
    }
    if (all) atomicAdd(&sm.count[e], all);
    if (before) atomicAdd(&sm.base[e], before);
  }
  __syncthreads();
  route_scan(sm, p, blockIdx.x == 0);
  const int t0 = blockIdx.x * p.per_cta, t1 = min(p.T, t0 + p.per_cta);
  route_place(sm, p, p.ids ? p.ids : p.ids_in, t0, t1);
  route_fill(sm, p);
}

}  // namespace bs
