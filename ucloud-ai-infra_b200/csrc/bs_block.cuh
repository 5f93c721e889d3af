// The end of a transformer block and the start of the next one in one pass over the rows:
//   z   = y[t]                                             (dense block output)
//       = sum_s weights[t, s] * y[slot_row[t, s]]          (experts' rows; slots with row -1 add nothing)
//   n   = z * (1 / sqrt(mean(z^2) + eps)) * post           (norm after the block; optional)
//   h   = residual_scale * residual + scale * gate * n     (gate per channel, token or element; optional)
//   v   = h * (1 / sqrt(mean(h^2) + eps)) * pre            (norm before the next block)
//   As  = max(amax(v over 128) / 448, 1e-12),  A = e4m3_rn(v / As)
// Every step is fp32; h is rounded once to the residual's type when it is stored, and v is taken from the unrounded
// h and goes to e4m3 without a rounding to bf16 between.
//
// Bound: HBM. Per token k (or 1) rows of bf16 and the residual are read, the residual and the e4m3 row written. A CTA
// owns a row, a thread C 16-byte chunks of it (chunk c = t + blockDim * j), so z and h stay in registers between the
// two norms, and a 128-group is the 16 chunks of a half-warp.
#pragma once
#include "bs_common.cuh"
#include "bs_quant.cuh"

namespace bs {

constexpr int kBlockMaxThreads = 512;
constexpr int kBlockMaxChunks = 4;  // rows of at most 512 * 4 * 8 = 16384 elements

enum : int { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };

struct BlockParams {
  const __nv_bfloat16* y;    // [rows_y, ldy]
  long long ldy;
  int rows_y;
  const float* weights;      // [T, k]; nullptr: dense
  const int* slot_row;       // [T, k]
  int k;
  const void* residual;      // [T, ldr] bf16 or fp32
  long long ldr;
  void* out;                 // [T, ldo] of the residual's type; may be the residual itself
  long long ldo;
  const __nv_bfloat16* post; // [H] or nullptr
  const __nv_bfloat16* gate; // by gate_kind
  int gate_kind;
  long long ldg;             // row stride of a token or full gate
  float scale, residual_scale;
  const __nv_bfloat16* pre;  // [H] or nullptr: no A, As
  float eps;
  uint8_t* A;                // [T, H]
  float* As;                 // [T, H / 128]
  int T, H;
};

// Sum over the CTA in a fixed order: a butterfly per warp, then the warp totals in warp order. `buf` is not reused
// before the next barrier of the caller.
__device__ __forceinline__ float block_sum(float v, float* buf) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = buf[0];
  for (int i = 1; i < static_cast<int>(blockDim.x >> 5); ++i) s += buf[i];
  return s;
}

template <int C, bool WIDE>
__global__ void __launch_bounds__(kBlockMaxThreads) k_block_norm(const BlockParams p) {
  __shared__ float sums[2][2][kBlockMaxThreads / 32];  // by row parity and norm
  const int t = threadIdx.x, nt = blockDim.x, lane = t & 31;
  const int nch = p.H / 8;
  if (t == 0) grid_dep_launch();
  grid_dep_wait();
  for (int row = blockIdx.x, parity = 0; row < p.T; row += gridDim.x, parity ^= 1) {
    float z[C][8];
    if (p.weights) {
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[j][e] = 0.f;
      const long long at = static_cast<long long>(row) * p.k;
#pragma unroll 4
      for (int s = 0; s < p.k; ++s) {
        const int r = __ldg(p.slot_row + at + s);
        if (static_cast<unsigned>(r) >= static_cast<unsigned>(p.rows_y)) continue;
        const float w = __ldg(p.weights + at + s);
        const __nv_bfloat16* src = p.y + static_cast<long long>(r) * p.ldy;
#pragma unroll
        for (int j = 0; j < C; ++j) {
          const int c = t + nt * j;
          if (c < nch) {
            float v[8];
            unpack_bf16x8(__ldg(reinterpret_cast<const uint4*>(src + c * 8)), v);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[j][e] = fmaf(w, v[e], z[j][e]);
          }
        }
      }
    } else {
      const __nv_bfloat16* src = p.y + static_cast<long long>(row) * p.ldy;
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int c = t + nt * j;
#pragma unroll
        for (int e = 0; e < 8; ++e) z[j][e] = 0.f;
        if (c < nch) unpack_bf16x8(__ldg(reinterpret_cast<const uint4*>(src + c * 8)), z[j]);
      }
    }
    if (p.post) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < C; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(z[j][e], z[j][e], ss);
      ss = block_sum(ss, sums[parity][0]);
      const float rs = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, static_cast<float>(p.H)) + p.eps));
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int c = t + nt * j;
        if (c < nch) {
          float w[8];
          unpack_bf16x8(__ldg(reinterpret_cast<const uint4*>(p.post + c * 8)), w);
#pragma unroll
          for (int e = 0; e < 8; ++e) z[j][e] = z[j][e] * rs * w[e];
        }
      }
    }
    const float gt = p.gate_kind == kGateToken ? __bfloat162float(__ldg(p.gate + row * p.ldg)) * p.scale : p.scale;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < C; ++j) {
      const int c = t + nt * j;
      if (c < nch) {
        float g[8], r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = gt;
        if (p.gate_kind == kGateChannel || p.gate_kind == kGateFull) {
          const __nv_bfloat16* gr = p.gate + (p.gate_kind == kGateFull ? row * p.ldg : 0) + c * 8;
          unpack_bf16x8(__ldg(reinterpret_cast<const uint4*>(gr)), g);
#pragma unroll
          for (int e = 0; e < 8; ++e) g[e] *= p.scale;
        }
        if constexpr (WIDE) {
          const float4* rr = reinterpret_cast<const float4*>(static_cast<const float*>(p.residual) + row * p.ldr + c * 8);
          const float4 a = rr[0], b = rr[1];
          r[0] = a.x, r[1] = a.y, r[2] = a.z, r[3] = a.w, r[4] = b.x, r[5] = b.y, r[6] = b.z, r[7] = b.w;
        } else {
          unpack_bf16x8(*reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.residual) + row * p.ldr + c * 8), r);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          z[j][e] = fmaf(g[e], z[j][e], p.residual_scale * r[e]);
          ss = fmaf(z[j][e], z[j][e], ss);
        }
        if constexpr (WIDE) {
          float4* oo = reinterpret_cast<float4*>(static_cast<float*>(p.out) + row * p.ldo + c * 8);
          oo[0] = make_float4(z[j][0], z[j][1], z[j][2], z[j][3]);
          oo[1] = make_float4(z[j][4], z[j][5], z[j][6], z[j][7]);
        } else {
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + row * p.ldo + c * 8) =
              make_uint4(pack_bf16x2(z[j][0], z[j][1]), pack_bf16x2(z[j][2], z[j][3]), pack_bf16x2(z[j][4], z[j][5]),
                         pack_bf16x2(z[j][6], z[j][7]));
        }
      }
    }
    if (p.pre) {
      ss = block_sum(ss, sums[parity][1]);
      const float rs = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, static_cast<float>(p.H)) + p.eps));
#pragma unroll
      for (int j = 0; j < C; ++j) {
        if (nt * j >= nch) break;  // uniform across the CTA
        const int c = t + nt * j;
        const bool active = c < nch;
        float amax = 0.f;
        if (active) {
          float w[8];
          unpack_bf16x8(__ldg(reinterpret_cast<const uint4*>(p.pre + c * 8)), w);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            z[j][e] = z[j][e] * rs * w[e];
            amax = fmaxf(amax, fabsf(z[j][e]));
          }
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float sc = group_scale(amax);
        if (active) {
          const float r = __frcp_rn(sc);
          uint32_t q[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            q[h] = f2_to_e4m3x2(div_by_scale(z[j][4 * h], sc, r), div_by_scale(z[j][4 * h + 1], sc, r)) |
                   (f2_to_e4m3x2(div_by_scale(z[j][4 * h + 2], sc, r), div_by_scale(z[j][4 * h + 3], sc, r)) << 16);
          *reinterpret_cast<uint2*>(p.A + static_cast<size_t>(row) * p.H + c * 8) = make_uint2(q[0], q[1]);
          if ((lane & 15) == 0) p.As[static_cast<size_t>(row) * (p.H / 128) + c / 16] = sc;
        }
      }
    }
  }
}

}  // namespace bs
