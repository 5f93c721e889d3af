// C-ABI entry points of the mixture-of-experts operators: argument checks, kernel selection and launch. Part of
// bs_capi.cu's translation unit (its helpers and the status word).
#pragma once

namespace {

// CTAs that a cluster of the route kernel may have on the current device: 16 where such a cluster can run, else the
// portable 8.
template <int VPL>
int route_cluster() {
  struct State {
    std::once_flag once[kMaxDevices];
    int n[kMaxDevices];
  };
  static State st;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 8;
  std::call_once(st.once[dev], [&] {
    st.n[dev] = 8;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(bs::kRouteThreads);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 16;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaFuncSetAttribute(bs::k_moe_route<VPL>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&n, bs::k_moe_route<VPL>, &cfg) == cudaSuccess && n > 0)
      st.n[dev] = 16;
    cudaGetLastError();
  });
  return st.n[dev];
}

// Tokens per CTA of the two-launch form: one round of a CTA's warps, more when that would take more CTAs than fit on the
// device at once, two per SM (k_moe_place reads every CTA's counts).
int route_tokens_per_cta(int T, int num_sms) {
  const int at_once = bs::kRouteRound * 2 * num_sms;
  return bs::kRouteRound * (T / at_once + (T % at_once != 0));
}
int route_grid(int T, int num_sms) {
  const int per = route_tokens_per_cta(T, num_sms);
  return (T + per - 1) / per;
}

template <int VPL>
int launch_route(bs::RouteParams& p, int f32, int num_sms, cudaStream_t s) {
  if (!p.hist) {
    const int rounds = p.T <= bs::kRouteRound * route_cluster<VPL>() ? 1 : 2;  // kRouteCluster: two rounds of eight CTAs
    p.per_cta = bs::kRouteRound * rounds;
    const int grid = p.T > 0 ? (p.T + p.per_cta - 1) / p.per_cta : 1;
    return launch_pdl_cluster(bs::k_moe_route<VPL>, grid, bs::kRouteThreads, 0, grid, s, "k_moe_route launch", p, f32);
  }
  p.per_cta = route_tokens_per_cta(p.T, num_sms);
  const int grid = route_grid(p.T, num_sms);
  const int rc = launch_pdl(bs::k_moe_route<VPL>, grid, bs::kRouteThreads, 0, s, "k_moe_route launch", p, f32);
  return rc != BS_OK ? rc : launch_pdl(bs::k_moe_place, grid, bs::kRouteThreads, 0, s, "k_moe_place launch", p);
}

int run_route(bs::RouteParams& p, int f32, void* scratch, size_t scratch_bytes, void* stream) {
  if (p.T < 0 || p.k <= 0 || p.k > bs::kMaxTopK || p.E <= 0 || p.E > bs::kMaxExperts) return BS_ERR_ARG;
  if (p.e_begin < 0 || p.e_count <= 0 || p.e_count > p.E - p.e_begin) return BS_ERR_ARG;
  if (static_cast<long long>(p.T) * p.k > (1ll << 30)) return BS_ERR_ARG;  // 32-bit rows, with room for a CTA's tokens
  if (!p.offsets || (p.T > 0 && (!p.row_token || !p.slot_row))) return BS_ERR_ARG;
  DeviceState* d = device_state();
  if (!d) return BS_ERR_CUDA;
  if (p.T > bs::kRouteCluster) {
    if (!scratch || scratch_bytes < static_cast<size_t>(route_grid(p.T, d->num_sms)) * p.e_count * sizeof(int))
      return BS_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(scratch) & 3u) return BS_ERR_ALIGN;
    p.hist = static_cast<int*>(scratch);
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (!p.logits) return launch_route<0>(p, 0, d->num_sms, s);
  if (p.E <= 32) return launch_route<1>(p, f32, d->num_sms, s);
  if (p.E <= 64) return launch_route<2>(p, f32, d->num_sms, s);
  if (p.E <= 128) return launch_route<4>(p, f32, d->num_sms, s);
  if (p.E <= 256) return launch_route<8>(p, f32, d->num_sms, s);
  return launch_route<16>(p, f32, d->num_sms, s);
}

// How a grouped product runs.
struct GroupedPlan {
  int nt;     // rows per tile of k_grouped_tokens; 0: k_grouped_rows
  int log_s;  // k_grouped_tokens: log2 of the CTAs per tile
};

// Chosen by the mean rows per expert. Measured with router-like skew (times in us; 64 experts, 5120 -> 2 x 1024 fused,
// 1024 -> 5120 plain; 128 experts, 2048 -> 2 x 768, 768 -> 2048; token tiles of 16 and 32 rows, row tiles):
//   fused  mean 4.0: 97.8, 98.3, 125 (64 experts)    4.7: 58.7, 57.3, 72 (128)    12.5: -, 111, 125 (64)
//          mean 14.1: -, 76.3, 76.6 (128)   17.5: -, 115, 127 (64)   19.7: -, 88.5, 81.6 (128)   20: -, 127, 127 (64)
//   plain  mean 4.0: 53.0, 54.4, 57.4 (64)   4.7: 38.3, 35.6, 38.0 (128)   12.5: -, 63.6, 66.9 (64)
//          mean 14.1: -, 44.7, 44.1 (128)    15: -, 67.4, 67.1 (64)        17.5: -, 69.2, 67.7 (64)
// (token tiles of 64 rows were never more than 1 us ahead of the better of 32 and row tiles: not built).
// CTAs per tile: a call with fewer tiles than SMs takes as many as fill them, with at least 8 K blocks each (36 tiles of
// 16 K blocks: 14.6 us on one CTA each, 11.2 on two, 12.0 on four; 64 tiles of 40: 27.7, 19.3, 19.4). With more
// tiles than SMs the fused product is faster on two (its last wave is half as long: 61 tokens 114 -> 101 us, 32
// tokens 109 -> 98 us), the plain one on one (its tiles are too short for the exchange: 240 tokens 43.3 -> 65 us).
GroupedPlan grouped_plan(bool fused, int E, int nblk, int KB, int rows, int num_sms) {
  GroupedPlan g = {0, 0};
  const long long r = rows;
  if (r <= 4ll * E) g.nt = 16;
  else if (r <= (fused ? 16ll : 14ll) * E) g.nt = 32;
  if (!g.nt) return g;
  const long long tiles = static_cast<long long>(rows < E ? rows : E) * (fused ? nblk / 2 : nblk);
  if (tiles > num_sms)
    g.log_s = fused && KB >= 16 ? 1 : 0;
  else
    while (g.log_s < 3 && (16 << g.log_s) <= KB && (tiles << (g.log_s + 1)) <= num_sms) ++g.log_s;
  return g;
}

template <bool FUSED, int NT>
int launch_grouped_tokens(const CUtensorMap& tmW, const CUtensorMap& tmX, const bs::GroupedParams& p, int log_s,
                          int num_sms, cudaStream_t s) {
  using Cfg = bs::GroupedTokensCfg<FUSED, NT>;
  constexpr auto kern = bs::k_grouped_tokens<FUSED, NT>;
  const int rc = prepare_kernel<kern>(Cfg::kSmemBytes, 0);
  if (rc != BS_OK) return rc;
  const int clusters = max_clusters<kern>(Cfg::kThreads, Cfg::kSmemBytes, log_s, num_sms);
  if (clusters <= 0) return BS_ERR_CUDA;
  return launch_pdl_cluster(kern, clusters << log_s, Cfg::kThreads, Cfg::kSmemBytes, 1 << log_s, s,
                            "k_grouped_tokens launch", tmW, tmX, p, log_s);
}

template <bool FUSED, bool BOX>
int launch_grouped_rows(const CUtensorMap& tmA, const CUtensorMap& tmB, const CUtensorMap& tmO, const bs::GroupedParams& p,
                        int num_sms, cudaStream_t s) {
  using Cfg = bs::GroupedRowsCfg<FUSED, BOX>;
  constexpr auto kern = bs::k_grouped_rows<FUSED, BOX>;
  const int rc = prepare_kernel<kern>(Cfg::kSmemBytes, Cfg::Regs::kLaunch);
  if (rc != BS_OK) return rc;
  return launch_pdl(kern, num_sms, Cfg::kThreads, Cfg::kSmemBytes, s, "k_grouped_rows launch", tmA, tmB, tmO, p);
}

template <bool FUSED>
int run_grouped(const void* A, const void* B, const bs::GroupedParams& p, int rows_hint, cudaStream_t s, int num_sms) {
  const int K = p.KB * 128;
  const GroupedPlan g = grouped_plan(FUSED, p.E, p.nblk, p.KB, rows_hint, num_sms);
  const bool gather = p.row_token != nullptr;
  CUtensorMap tmA, tmB;
  if (make_weight_map(&tmB, B, p.E * p.nblk * 128, K, p.b_tiled, FUSED && !g.nt ? 64 : 128) != BS_OK) return BS_ERR_TMAP;
  if (make_map(&tmA, A, K, p.rows_a, K, 128, gather ? 1 : g.nt ? g.nt : 128) != BS_OK) return BS_ERR_TMAP;
  switch (g.nt) {
    case 16: return launch_grouped_tokens<FUSED, 16>(tmB, tmA, p, g.log_s, num_sms, s);
    case 32: return launch_grouped_tokens<FUSED, 32>(tmB, tmA, p, g.log_s, num_sms, s);
    default: break;
  }
  if constexpr (!FUSED) {
    // measured at the kernel: boxes pay from about 128 rows per expert on
    if (!p.out_f32 && rows_hint > 128ll * p.E) {
      CUtensorMap tmO;
      if (make_map(&tmO, p.out, static_cast<uint64_t>(p.nblk) * 256, p.R, static_cast<uint64_t>(p.ldc) * 2, 128, 32) != BS_OK)
        return BS_ERR_TMAP;
      return launch_grouped_rows<false, true>(tmA, tmB, tmO, p, num_sms, s);
    }
  }
  return launch_grouped_rows<FUSED, false>(tmA, tmB, tmA, p, num_sms, s);
}

int validate_grouped(const void* A, const void* B, const void* out, const float* As, const float* Bs, const float* qs,
                     const int* offsets, const int* row_token, int rows_a, int R, int rows_hint, int E, int N, int K,
                     int ldc, int b_tiled, int out_dtype, bool fused) {
  if (rows_a < 0 || R < 0 || rows_hint < 0 || rows_hint > R || E <= 0 || E > bs::kMaxExperts) return BS_ERR_ARG;
  const int rc = validate_gemm(fused, A, B, out, As, Bs, qs, R, N, K, ldc, b_tiled, out_dtype);
  if (rc != BS_OK || R == 0) return rc;
  if (!offsets || rows_a == 0 || (!row_token && rows_a < R)) return BS_ERR_ARG;
  // 32-bit tile counts and TMA coordinates
  // (one weight block past the last expert's is addressed, and read as zeros, where N / 128 is odd)
  if ((static_cast<long long>(E) * N + 128) * (b_tiled ? K / 128 : 1) >= (1ll << 31)) return BS_ERR_ARG;
  if (static_cast<long long>(rows_a) * (K / 16) >= (1ll << 32)) return BS_ERR_ARG;
  if ((static_cast<long long>(R) / 16 + E) * (N / 128) >= (1ll << 31)) return BS_ERR_ARG;
  return BS_OK;
}

bs::GroupedParams grouped_params(const void* A, const float* As, const float* Bs, const int* offsets, const int* row_token, int rows_a,
                                 int R, int E, int N, int K, int b_tiled, int* status) {
  bs::GroupedParams p = {};
  p.E = E;
  p.R = R;
  p.rows_a = rows_a;
  p.nblk = N / 128;
  p.KB = K / 128;
  p.b_tiled = b_tiled;
  p.offsets = offsets;
  p.row_token = row_token;
  p.A = static_cast<const uint8_t*>(A);
  p.As = As;
  p.Bs = Bs;
  p.status = status;
  return p;
}

template <typename Shape, bool WIDE>
int launch_block(bs::BlockParams& p, int num_sms, cudaStream_t s) {
  constexpr auto kern = bs::k_block_norm<Shape, WIDE>;
  const int res_bytes = p.residual ? (WIDE ? 4 : 2) * p.H : 0;
  p.ring = bs::block_ring(p.weights ? p.k : 1, p.H, res_bytes, Shape::kRingBytes);
  const int smem = p.ring.bytes(p.H);
  const int rc = prepare_kernel<kern>(Shape::kRingBytes, 0);
  if (rc != BS_OK) return rc;
  const int threads = ((p.H / 8 + Shape::C - 1) / Shape::C + 31) / 32 * 32;
  int grid = p.T;  // a CTA per token, or as many as fit, with equal numbers of tokens
  if (p.T > num_sms) {
    int per_sm = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, threads + 32, smem) != cudaSuccess || per_sm < 1)
      per_sm = 1;
    cudaGetLastError();
    const int rounds = (p.T - 1) / (per_sm * num_sms) + 1;
    grid = (p.T - 1) / rounds + 1;
  }
  return launch_pdl(kern, grid, threads + 32, smem, s, "k_block_norm launch", p);
}

template <typename Shape>
int launch_block_shape(bs::BlockParams& p, bool wide, int num_sms, cudaStream_t s) {
  return wide ? launch_block<Shape, true>(p, num_sms, s) : launch_block<Shape, false>(p, num_sms, s);
}

}  // namespace

extern "C" {

int bs_fp8_moe_route(const void* logits, int dtype, long long ldl, int T, int n_experts, int top_k, int renormalize,
                     float scale, int e_begin, int e_count, float* weights, int* ids, int* offsets, int* row_token,
                     int* slot_row, void* scratch, size_t scratch_bytes, void* stream) {
  if ((dtype != 0 && dtype != 1) || ldl < n_experts || top_k > n_experts) return BS_ERR_ARG;
  if (T > 0 && (!logits || !weights || !ids)) return BS_ERR_ARG;
  if (reinterpret_cast<uintptr_t>(logits) & (dtype ? 3u : 1u)) return BS_ERR_ALIGN;
  bs::RouteParams p = {};
  static const float none = 0.f;  // T == 0: a pointer that says "logits", never read
  p.logits = logits ? logits : &none;
  p.ldl = ldl;
  p.T = T;
  p.E = n_experts;
  p.k = top_k;
  p.renormalize = renormalize;
  p.scale = scale;
  p.e_begin = e_begin;
  p.e_count = e_count;
  p.weights = weights;
  p.ids = ids;
  p.offsets = offsets;
  p.row_token = row_token;
  p.slot_row = slot_row;
  return run_route(p, dtype, scratch, scratch_bytes, stream);
}

int bs_fp8_moe_dispatch(const int* ids, int T, int n_experts, int top_k, int e_begin, int e_count, int* offsets,
                        int* row_token, int* slot_row, void* scratch, size_t scratch_bytes, void* stream) {
  if (T > 0 && !ids) return BS_ERR_ARG;
  bs::RouteParams p = {};
  p.ids_in = ids;
  p.T = T;
  p.E = n_experts;
  p.k = top_k;
  p.e_begin = e_begin;
  p.e_count = e_count;
  p.offsets = offsets;
  p.row_token = row_token;
  p.slot_row = slot_row;
  return run_route(p, 0, scratch, scratch_bytes, stream);
}

size_t bs_fp8_moe_scratch_bytes(int T, int e_count) {
  if (T <= bs::kRouteCluster || e_count <= 0) return 0;
  DeviceState* d = device_state();
  return static_cast<size_t>(route_grid(T, d ? d->num_sms : 148)) * e_count * sizeof(int);
}

int bs_fp8_grouped_gemm(const void* A, const void* B, void* C, const float* As, const float* Bs, const int* offsets,
                        const int* row_token, int rows_a, int R, int rows_hint, int E, int N, int K, int ldc,
                        int b_tiled, int out_dtype, void* stream) {
  const int rc = validate_grouped(A, B, C, As, Bs, nullptr, offsets, row_token, rows_a, R, rows_hint, E, N, K, ldc,
                                  b_tiled, out_dtype, false);
  if (rc != BS_OK || R == 0) return rc;
  DeviceState* d = device_state();
  if (!d) return BS_ERR_CUDA;
  bs::GroupedParams p = grouped_params(A, As, Bs, offsets, row_token, rows_a, R, E, N, K, b_tiled, d->status);
  p.ldc = ldc;
  p.out_f32 = out_dtype;
  p.out = C;
  return run_grouped<false>(A, B, p, rows_hint ? rows_hint : R, static_cast<cudaStream_t>(stream), d->num_sms);
}

int bs_fp8_grouped_gemm_silu_quant(const void* A, const void* B, void* Q, const float* As, const float* Bs, float* Qs,
                                   const int* offsets, const int* row_token, int rows_a, int R, int rows_hint, int E,
                                   int N2, int K, int b_tiled, void* stream) {
  const int rc = validate_grouped(A, B, Q, As, Bs, Qs, offsets, row_token, rows_a, R, rows_hint, E, N2, K, N2 / 2,
                                  b_tiled, 0, true);
  if (rc != BS_OK || R == 0) return rc;
  DeviceState* d = device_state();
  if (!d) return BS_ERR_CUDA;
  bs::GroupedParams p = grouped_params(A, As, Bs, offsets, row_token, rows_a, R, E, N2, K, b_tiled, d->status);
  p.ldc = N2 / 2;
  p.out = Q;
  p.qs = Qs;
  return run_grouped<true>(A, B, p, rows_hint ? rows_hint : R, static_cast<cudaStream_t>(stream), d->num_sms);
}

int bs_fp8_grouped_plan(int rows_hint, int E, int N, int K, int fused, int* plan, int n) {
  if (!plan || n < BS_GROUPED_FIELDS) return BS_ERR_ARG;
  if (rows_hint <= 0 || E <= 0 || E > bs::kMaxExperts || N <= 0 || N % (fused ? 256 : 128) || K <= 0 || K % 128) return BS_ERR_ARG;
  DeviceState* d = device_state();
  const GroupedPlan g = grouped_plan(fused != 0, E, N / 128, K / 128, rows_hint, d ? d->num_sms : 148);
  for (int i = 0; i < n; ++i) plan[i] = 0;
  plan[BS_GROUPED_KIND] = g.nt ? 1 : 2;
  plan[BS_GROUPED_TILE_ROWS] = g.nt ? g.nt : 128;
  plan[BS_GROUPED_CLUSTER] = 1 << g.log_s;
  return BS_OK;
}

int bs_fp8_block_norm_quant(const void* y, long long ldy, int rows_y, const float* weights, const int* slot_row,
                            int top_k, const void* residual, long long ldr, void* out, long long ldo, int wide,
                            const void* post_weight, const void* gate, int gate_kind, long long ldg, float scale,
                            float residual_scale, const void* pre_weight, float eps, void* A, float* As, void* V, int T,
                            int H, void* stream) {
  if (T < 0 || H <= 0 || H % 128 || H > bs::kBlockMaxH) return BS_ERR_ARG;
  if (wide != 0 && wide != 1) return BS_ERR_ARG;
  const int per16 = wide ? 4 : 8;  // elements of the residual per 16 bytes
  if (ldy < H || ldy % 8 || (residual && (ldr < H || ldr % per16)) || ldo < H || ldo % per16 || rows_y < 0) return BS_ERR_ARG;
  if (!(eps >= 0.f) || gate_kind < 0 || gate_kind > 3 || (gate_kind != 0) != (gate != nullptr)) return BS_ERR_ARG;
  if ((gate_kind == 3 && (ldg < H || ldg % 8)) || (gate_kind == 2 && ldg < 1)) return BS_ERR_ARG;
  if ((weights == nullptr) != (slot_row == nullptr) || (weights && (top_k <= 0 || top_k > bs::kMaxTopK)) || (!weights && rows_y < T)) return BS_ERR_ARG;
  if (T == 0) return BS_OK;
  if (!y || !out || (pre_weight && (!A || !As)) || (V && !pre_weight)) return BS_ERR_ARG;
  if (!aligned16(y) || !aligned16(residual) || !aligned16(out) || !aligned16(post_weight) || !aligned16(pre_weight) ||
      !aligned16(A) || !aligned16(V) || (gate_kind != 2 && !aligned16(gate)))
    return BS_ERR_ALIGN;
  DeviceState* d = device_state();
  if (!d) return BS_ERR_CUDA;
  bs::BlockParams p = {};
  p.y = static_cast<const __nv_bfloat16*>(y);
  p.ldy = ldy;
  p.rows_y = rows_y;
  p.weights = weights;
  p.slot_row = slot_row;
  p.k = top_k;
  p.residual = residual;
  p.ldr = ldr;
  p.out = out;
  p.ldo = ldo;
  p.post = static_cast<const __nv_bfloat16*>(post_weight);
  p.gate = static_cast<const __nv_bfloat16*>(gate);
  p.gate_kind = gate_kind;
  p.ldg = ldg;
  p.scale = scale;
  p.residual_scale = residual_scale;
  p.pre = static_cast<const __nv_bfloat16*>(pre_weight);
  p.eps = eps;
  p.inv_h = 1.0f / static_cast<float>(H);
  p.A = static_cast<uint8_t*>(A);
  p.As = As;
  p.V = static_cast<__nv_bfloat16*>(V);
  p.T = T;
  p.H = H;
  p.status = d->status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (H <= bs::BlockShape1::kMaxH) return launch_block_shape<bs::BlockShape1>(p, wide != 0, d->num_sms, s);
  if (H <= bs::BlockShape2::kMaxH) return launch_block_shape<bs::BlockShape2>(p, wide != 0, d->num_sms, s);
  if (H <= bs::BlockShape3::kMaxH) return launch_block_shape<bs::BlockShape3>(p, wide != 0, d->num_sms, s);
  if (H <= bs::BlockShape4::kMaxH) return launch_block_shape<bs::BlockShape4>(p, wide != 0, d->num_sms, s);
  return launch_block_shape<bs::BlockShape5>(p, wide != 0, d->num_sms, s);
}

}  // extern "C"
