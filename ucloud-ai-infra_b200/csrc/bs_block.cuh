// The end of a transformer block and the start of the next one in one pass over the rows:
//   z   = y[t]                                             (dense block output)
//       = sum_s weights[t, s] * y[slot_row[t, s]]          (experts' rows; slots with row -1 add nothing)
//   n   = z * (1 / sqrt(mean(z^2) + eps)) * post           (norm after the block; optional)
//   h   = residual_scale * residual + scale * gate * n     (residual, and gate per channel, token or element: optional)
//   v   = h * (1 / sqrt(mean(h^2) + eps)) * pre            (norm before the next block)
//   As  = max(amax(v over 128) / 448, 1e-12),  A = e4m3_rn(v / As)
// Every step is fp32; h is rounded once to the residual's type when it is stored, and v is taken from the unrounded
// h and goes to e4m3 without a rounding to bf16 between (V, if asked for, is bf16_rn(v): a router's input).
//
// Bound: HBM. Per token k (or 1) rows of bf16 and the residual are read, the residual and the e4m3 row written; what
// costs is keeping enough of those reads in flight beside two reductions per row, in few instructions per element. A
// producer warp brings the rows of the CTA's next tokens into a ring in shared memory by bulk copies, up to four rows
// per stage, whatever the other warps are doing; the CTAs of an SM share about 200 KB of ring. The other warps own C
// 16-byte chunks of a row each (chunk c = t + threads * j), add the ring's rows up as they land, and keep z and h in
// registers between the two norms; a 128-group is the 16 chunks of a half-warp. Measured on the way (T = 8192,
// H = 5120, k = 8): loads into registers by four CTAs of 320 threads 218 us; the ring with a stage per row 201 us, bound
// by the issue of 1600 instructions per warp and token (waits, IEEE divisions and square roots among them).
#pragma once
#include "bs_common.cuh"
#include "bs_quant.cuh"

namespace bs {

constexpr int kBlockMaxH = 16384;

enum : int { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };

constexpr int kBlockMaxStages = 16;

constexpr int kBlockResSlots = 2;

// Shapes of the kernel: chunks per thread, most threads that own chunks (a producer warp comes on top), CTAs per SM that
// its registers and its ring leave room for. By the row's length: some 20 warps per SM always, in as many CTAs as that
// gives, since one CTA's reductions hide behind another's rows. Measured (T = 8192; us, dense and k = 8; H and two shapes):
//   1024   <1, 128, 5> 25, 35   <2, 64, 8> 21, 32 (but 512: 15, 22 and 20, 26)   <1, 320, 2> 24, 51
//   2048   <2, 160, 4> 38, 62   <1, 320, 2> 48, 67         2560   <2, 160, 4> 48, 77   <1, 320, 2> 56, 78
//   8192   <2, 640, 1> 147, 221   <4, 320, 1> 179, 349     12288  <4, 512, 1> 295, 466     16384  <4, 512, 1> 323, 575
// Spills: <4, 512, 1> 52 bytes (92 with an fp32 residual), the others none (8 to 16 with an fp32 residual and C = 2).
// With an fp32 residual: 2048 45, 71; 5120 105, 190; 16384 376, 749.
template <int C_, int THREADS, int CTAS>
struct BlockShape {
  static constexpr int C = C_, kThreads = THREADS, kCtas = CTAS;
  static constexpr int kMaxH = C * THREADS * 8;
  static constexpr int kRingBytes = 200 * 1024 / CTAS;
  static constexpr int kSums = (THREADS / 32 + 3) / 4 * 4;  // warp totals; those of warps that do not exist are 0
  static_assert(kBlockResSlots * 4 * kMaxH + 2 * 2 * kMaxH <= kRingBytes, "fp32 residual rows and two stages");
};
using BlockShape1 = BlockShape<1, 128, 5>;
using BlockShape2 = BlockShape<2, 160, 4>;
using BlockShape3 = BlockShape<2, 320, 2>;
using BlockShape4 = BlockShape<2, 640, 1>;
using BlockShape5 = BlockShape<4, 512, 1>;
static_assert(BlockShape5::kMaxH == kBlockMaxH, "every row has a shape");

// The ring of a launch: two residual rows, and stages of G rows (a power of two), two at least.
struct BlockRing {
  int G, stages, res_bytes;  // res_bytes: a residual row's, 0 without one
  int bytes(int H) const { return kBlockResSlots * res_bytes + stages * G * 2 * H; }
};
inline BlockRing block_ring(int k, int H, int res_bytes, int ring_bytes) {
  BlockRing r = {k >= 3 ? 4 : k, 0, res_bytes};
  const int room = ring_bytes - kBlockResSlots * res_bytes;
  while (r.G > 1 && 2 * r.G * 2 * H > room) r.G >>= 1;
  const int n = room / (r.G * 2 * H);
  // Two stages of several rows keep enough reads in flight, and more of them cost (7168 x 8192 rows, k = 8: 200 us with
  // two stages of four rows, 225 with three); of single rows 3, 6 and 16 are equal within 2 %.
  const int most = r.G > 1 ? 2 : kBlockMaxStages;
  r.stages = n < 2 ? 2 : n > most ? most : n;
  return r;
}
struct BlockParams {
  const __nv_bfloat16* y;    // [rows_y, ldy]
  long long ldy;
  int rows_y;
  const float* weights;      // [T, k]; nullptr: dense
  const int* slot_row;       // [T, k]
  int k;
  const void* residual;      // [T, ldr] bf16 or fp32; nullptr: none
  long long ldr;
  void* out;                 // [T, ldo] of the residual's type; may be the residual itself
  long long ldo;
  const __nv_bfloat16* post; // [H] or nullptr
  const __nv_bfloat16* gate; // by gate_kind
  int gate_kind;
  long long ldg;             // row stride of a token or full gate
  float scale, residual_scale;
  const __nv_bfloat16* pre;  // [H] or nullptr: no A, As
  float eps, inv_h;          // inv_h: 1 / H
  uint8_t* A;                // [T, H]
  float* As;                 // [T, H / 128]
  __nv_bfloat16* V;          // [T, H] or nullptr
  int T, H;
  BlockRing ring;
  int* status;
};

// Sum over the `threads` consumer threads in a fixed order, in two halves so that other work can stand between them: a
// butterfly per warp and its total in `buf`; then, after the barrier, every thread adds the warp totals. `buf` is not
// reused before the next barrier.
__device__ __forceinline__ void block_sum_begin(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
}
template <int SUMS>
__device__ __forceinline__ float block_sum_end(const float (&buf)[SUMS], int threads) {
  named_bar_sync(1, threads);
  const ulonglong2* b = reinterpret_cast<const ulonglong2*>(buf);
  uint64_t s = fadd2(b[0].x, b[0].y);
#pragma unroll
  for (int i = 1; i < SUMS / 4; ++i) s = fadd2(s, fadd2(b[i].x, b[i].y));
  return lo_f(s) + hi_f(s);
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(
          smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// amax / 448, correctly rounded by one correction step (bs_quant.cuh, group_scale), without its floor.
__device__ __forceinline__ float amax_div_448(float amax) {
  constexpr float kInv448 = 1.0f / 448.0f;
  const float q0 = __fmul_rn(amax, kInv448);
  return __fmaf_rn(__fmaf_rn(-448.0f, q0, amax), kInv448, q0);
}

// blockDim = threads that own chunks + the producer warp.
template <typename Shape, bool WIDE>
__global__ void __launch_bounds__(Shape::kThreads + 32, Shape::kCtas) k_block_norm(const BlockParams p) {
  constexpr int C = Shape::C;
  extern __shared__ __align__(128) uint8_t block_smem[];  // residual rows, then [stages][G rows][2 H]
  __shared__ __align__(16) float sums[2][2][Shape::kSums];  // by row parity and norm
  __shared__ uint64_t full[kBlockMaxStages], empty[kBlockMaxStages];
  __shared__ uint64_t rfull[kBlockResSlots], rempty[kBlockResSlots];
  __shared__ float4 weight[kBlockMaxStages];
  __shared__ int there[kBlockMaxStages];  // bit g: row g of the stage is one (its slot has a row)
  __shared__ volatile int abort_flag;
  const int t = threadIdx.x, nt = static_cast<int>(blockDim.x) - 32, lane = t & 31;
  const int nch = p.H / 8, row_bytes = 2 * p.H;
  const int k = p.weights ? p.k : 1;
  const int G = p.ring.G, stages = p.ring.stages, res_bytes = p.ring.res_bytes;
  uint8_t* ring = block_smem + kBlockResSlots * res_bytes;
  for (int i = t; i < 4 * Shape::kSums; i += blockDim.x) (&sums[0][0][0])[i] = 0.f;
  if (t == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 2);  // both by the producer: the bytes to come, and the weights
      mbar_init(&empty[i], nt / 32);
    }
    for (int i = 0; i < kBlockResSlots; ++i) {
      mbar_init(&rfull[i], 1);
      mbar_init(&rempty[i], nt / 32);
    }
    abort_flag = 0;
    fence_mbar_init();
    grid_dep_launch();
  }
  __syncthreads();
  grid_dep_wait();

  if (t >= nt) {
    // ------------------------------------------------------------ producer
    const uint64_t policy = policy_evict_first();
    int st = 0, rs = 0;
    uint32_t ph = 0, rph = 0;
    bool ok = true;
    // lane s holds slot s of the next token
    auto slot = [&](int row, int& r, float& w) {
      r = -1;
      w = 1.f;
      if (row >= p.T || lane >= k) return;
      if (p.weights) {
        r = __ldg(p.slot_row + static_cast<long long>(row) * k + lane);
        w = __ldg(p.weights + static_cast<long long>(row) * k + lane);
      } else {
        r = row;
      }
    };
    int next_r;
    float next_w;
    slot(blockIdx.x, next_r, next_w);
    for (int row = blockIdx.x; ok && row < p.T; row += gridDim.x) {
      const int my_r = next_r;
      const float my_w = next_w;
      slot(row + gridDim.x, next_r, next_w);
      if (res_bytes) {
        if (lane == 0) {
          ok = mbar_wait(&rempty[rs], rph ^ 1, &abort_flag, p.status, kErrTimeoutEmpty);
          if (ok) {
            mbar_arrive_expect_tx(&rfull[rs], res_bytes);
            bulk_load(block_smem + rs * res_bytes,
                      static_cast<const uint8_t*>(p.residual) + static_cast<long long>(row) * p.ldr * (WIDE ? 4 : 2), res_bytes,
                      &rfull[rs], policy);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        if (++rs == kBlockResSlots) {
          rs = 0;
          rph ^= 1;
        }
      }
      const uint32_t has = __ballot_sync(0xffffffffu, static_cast<unsigned>(my_r) < static_cast<unsigned>(p.rows_y));
      for (int s = 0; s < k; s += G) {
        if (lane == 0) ok = mbar_wait(&empty[st], ph ^ 1, &abort_flag, p.status, kErrTimeoutEmpty);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        __syncwarp();  // the other lanes too come after the readers of this stage: the shuffle orders no memory
        if (!ok) break;
        // lanes s .. s + G - 1 bring their slots' rows (lanes from k on have none)
        const uint32_t mask = (has >> s) & ((1u << G) - 1);
        const int g = lane - s;
        if (lane == 0) {
          there[st] = static_cast<int>(mask);
          mbar_arrive_expect_tx(&full[st], __popc(mask) * row_bytes);
        }
        if (g >= 0 && g < G) {
          reinterpret_cast<float*>(&weight[st])[g] = my_w;
          if ((mask >> g) & 1) {
            bulk_load(ring + static_cast<size_t>(st * G + g) * row_bytes, p.y + static_cast<long long>(my_r) * p.ldy,
                      row_bytes, &full[st], policy);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]);  // the weights are there too
        if (++st == stages) {
          st = 0;
          ph ^= 1;
        }
      }
    }
    if (!ok) pause_ns(2000000ull);  // copies in flight land within microseconds
    return;
  }

  // -------------------------------------------------------------- rows
  // What every row uses, the norm weights' and a channel gate's chunks of this thread, is read again for each row (from
  // L1), always ahead of a reduction: kept in registers it spills (8192 x 2560, one chunk a thread,
  // k = 8: 83 us, and 78 so).
  auto chunk = [&](const __nv_bfloat16* w, int c) {
    return w && c < nch ? __ldg(reinterpret_cast<const uint4*>(w + c * 8)) : make_uint4(0, 0, 0, 0);
  };
  const __nv_bfloat16* channel = p.gate_kind == kGateChannel ? p.gate : nullptr;
  int st = 0, rs = 0;
  uint32_t ph = 0, rph = 0;
  bool ok = true;
  for (int row = blockIdx.x, parity = 0; row < p.T; row += gridDim.x, parity ^= 1) {
    float gt = p.scale;
    if (p.gate_kind == kGateToken) gt = __bfloat162float(__ldg(p.gate + row * p.ldg)) * p.scale;

    uint64_t z[C][4];  // pairs of this thread's elements
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) z[j][e] = 0;
    auto add = [&](int j, const uint4& v, float w) {
      const uint64_t w2 = pack_f2(w, w);
      z[j][0] = ffma2r(w2, bf16x2_to_f2(v.x), z[j][0]);
      z[j][1] = ffma2r(w2, bf16x2_to_f2(v.y), z[j][1]);
      z[j][2] = ffma2r(w2, bf16x2_to_f2(v.z), z[j][2]);
      z[j][3] = ffma2r(w2, bf16x2_to_f2(v.w), z[j][3]);
    };
    for (int s = 0; s < k; s += G) {
      if (ok) ok = mbar_wait_warp(&full[st], ph, &abort_flag, p.status, kErrTimeoutFull);
      if (ok) {
        const int mask = there[st];
        const float4 w4 = weight[st];
        const float w[4] = {w4.x, w4.y, w4.z, w4.w};
        const uint8_t* src = ring + static_cast<size_t>(st * G) * row_bytes + t * 16;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          if (t + nt * j < nch) {
            if (G == 1) {
              if (mask) add(j, *reinterpret_cast<const uint4*>(src + nt * j * 16), w4.x);
              continue;
            }
            uint4 v[4];
#pragma unroll
            for (int g = 0; g < 4; ++g)
              if ((mask >> g) & 1) v[g] = *reinterpret_cast<const uint4*>(src + g * row_bytes + nt * j * 16);
#pragma unroll
            for (int g = 0; g < 4; ++g)
              if ((mask >> g) & 1) add(j, v[g], w[g]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++st == stages) {
        st = 0;
        ph ^= 1;
      }
    }
    auto squares = [&]() {
      uint64_t ss2 = 0;
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) ss2 = ffma2r(z[j][e], z[j][e], ss2);  // zero past the row's end
      return lo_f(ss2) + hi_f(ss2);
    };
    // The gate's chunks are on the way during the first reduction, the next norm's weight during what follows it.
    uint4 g4[C];
#pragma unroll
    for (int j = 0; j < C; ++j) g4[j] = chunk(p.gate_kind == kGateFull ? p.gate + row * p.ldg : channel, t + nt * j);
    if (p.post) {
      uint4 w4[C];
#pragma unroll
      for (int j = 0; j < C; ++j) w4[j] = chunk(p.post, t + nt * j);
      block_sum_begin(squares(), sums[parity][0]);
      const float rs = rsqrtf(fmaf(block_sum_end(sums[parity][0], nt), p.inv_h, p.eps));
      const uint64_t rs2 = pack_f2(rs, rs);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&w4[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[j][e] = fmul2(fmul2(z[j][e], rs2), bf16x2_to_f2(w[e]));
      }
    }
    uint4 next[C];
#pragma unroll
    for (int j = 0; j < C; ++j) next[j] = chunk(p.pre, t + nt * j);
    if (res_bytes && ok) ok = mbar_wait_warp(&rfull[rs], rph, &abort_flag, p.status, kErrTimeoutFull);
    const uint4* res = reinterpret_cast<const uint4*>(block_smem + rs * res_bytes);
    const uint64_t gs2 = pack_f2(gt, gt), a2 = pack_f2(p.residual_scale, p.residual_scale);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int c = t + nt * j;
      if (c < nch) {
        const uint32_t* gw = reinterpret_cast<const uint32_t*>(&g4[j]);
        uint4 rv[WIDE ? 2 : 1];
#pragma unroll
        for (int i = 0; i < (WIDE ? 2 : 1); ++i) rv[i] = res_bytes && ok ? res[WIDE ? 2 * c + i : c] : make_uint4(0, 0, 0, 0);
        const uint32_t* rw = reinterpret_cast<const uint32_t*>(&rv[0]);
        const bool per_element = p.gate_kind == kGateChannel || p.gate_kind == kGateFull;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t g = per_element ? fmul2(bf16x2_to_f2(gw[e]), gs2) : gs2;
          uint64_t r;
          if constexpr (WIDE) {
            const uint32_t* ww = reinterpret_cast<const uint32_t*>(&rv[e >> 1]);
            r = static_cast<uint64_t>(ww[(2 * e) & 3]) | (static_cast<uint64_t>(ww[(2 * e + 1) & 3]) << 32);
          } else {
            r = bf16x2_to_f2(rw[e]);
          }
          z[j][e] = ffma2r(g, z[j][e], fmul2(a2, r));
        }
        if (ok) {
          if constexpr (WIDE) {
            float4* oo = reinterpret_cast<float4*>(static_cast<float*>(p.out) + row * p.ldo + c * 8);
            oo[0] = make_float4(lo_f(z[j][0]), hi_f(z[j][0]), lo_f(z[j][1]), hi_f(z[j][1]));
            oo[1] = make_float4(lo_f(z[j][2]), hi_f(z[j][2]), lo_f(z[j][3]), hi_f(z[j][3]));
          } else {
            *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row * p.ldo + c * 8) =
                make_uint4(pack_bf16x2(lo_f(z[j][0]), hi_f(z[j][0])), pack_bf16x2(lo_f(z[j][1]), hi_f(z[j][1])),
                           pack_bf16x2(lo_f(z[j][2]), hi_f(z[j][2])), pack_bf16x2(lo_f(z[j][3]), hi_f(z[j][3])));
          }
        }
      }
    }
    if (res_bytes) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&rempty[rs]);
      if (++rs == kBlockResSlots) {
        rs = 0;
        rph ^= 1;
      }
    }
    if (p.pre) {
      // v = u * rs with u = h * pre. The quotient v / As is u / (amax(u) / 448), so the row's 1 / sqrt only enters As:
      // the bytes are made while the sum is on its way, and see one rounding (of u) before the division. Groups so
      // small that As is at its floor divide u * rs by the floor instead.
      block_sum_begin(squares(), sums[parity][1]);
      uint32_t q[C][2];
      float su[C];
      auto quant = [&](const uint64_t (&u)[4], float div, uint32_t (&out)[2]) {
        const float nr = -__frcp_rn(div);
        const uint64_t d2 = pack_f2(div, div), nr2 = pack_f2(nr, nr);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint64_t q0 = neg_div_by_scale2(u[2 * h], d2, nr2);
          const uint64_t q1 = neg_div_by_scale2(u[2 * h + 1], d2, nr2);
          out[h] = (f2_to_e4m3x2(lo_f(q0), hi_f(q0)) | (f2_to_e4m3x2(lo_f(q1), hi_f(q1)) << 16)) ^ 0x80808080u;
        }
      };
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(&next[j]);
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          z[j][e] = fmul2(z[j][e], bf16x2_to_f2(w[e]));  // u
          amax = fmaxf(amax, fmaxf(fabsf(lo_f(z[j][e])), fabsf(hi_f(z[j][e]))));
        }
        // of this half-warp: never NaN, and floats from 0 up order like their bits
        const uint32_t bits = __float_as_uint(amax);
        const uint32_t lo = __reduce_max_sync(0xffffffffu, lane < 16 ? bits : 0u);
        const uint32_t hi = __reduce_max_sync(0xffffffffu, lane < 16 ? 0u : bits);
        su[j] = amax_div_448(__uint_as_float(lane < 16 ? lo : hi));
        quant(z[j], su[j], q[j]);
      }
      const float rs = rsqrtf(fmaf(block_sum_end(sums[parity][1], nt), p.inv_h, p.eps));
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int c = t + nt * j;
        float as = __fmul_rn(su[j], rs);
        if (!(as >= 1e-12f)) {
          as = 1e-12f;
          uint64_t v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmul2(z[j][e], pack_f2(rs, rs));
          quant(v, as, q[j]);
        }
        if (c < nch && ok) {
          *reinterpret_cast<uint2*>(p.A + static_cast<size_t>(row) * p.H + c * 8) = make_uint2(q[j][0], q[j][1]);
          if ((lane & 15) == 0) p.As[static_cast<size_t>(row) * (p.H / 128) + c / 16] = as;
          if (p.V) {
            const uint64_t rs2 = pack_f2(rs, rs);
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint64_t x = fmul2(z[j][e], rs2);
              v[e] = pack_bf16x2(lo_f(x), hi_f(x));
            }
            *reinterpret_cast<uint4*>(p.V + static_cast<size_t>(row) * p.H + c * 8) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    }
  }
}

}  // namespace bs
