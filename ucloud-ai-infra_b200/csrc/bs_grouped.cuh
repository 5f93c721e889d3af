// Block-scaled FP8 products grouped by expert, ragged row counts, for sm_100a:
//     C[r, n] = sum_kb P_kb[r, n] * (As[src(r), kb] * Bs[e, n / 128, kb]),  offsets[e] <= r < offsets[e + 1]
// P_kb the fp32 product of one 128-wide K block of e4m3 rows and expert e's e4m3 weights, promoted as in
// bs_prefill.cuh. src(r) = row_token[r] (the rows are read in place, no copy in row order is made) or r. FUSED: the
// weights are [gate; up], and the output is Q, Qs of silu(g) * u per 128-column group (bs_prefill.cuh).
//
// The row counts are known on the device only: every CTA turns the offsets into a table of the experts that have
// rows, with the first tile of each, and walks tiles blockIdx.x, blockIdx.x + gridDim.x, ... of the whole list. Tiles
// of one expert are adjacent, row tiles fastest, so an expert's weights come from HBM once and its row tiles
// share them in L2.
//
// Two kernels (the choice between them, with both measured: grouped_plan in bs_moe_entry.cuh).
//   k_grouped_rows    128 rows x 256 weight columns per tile, rows on the MMA's 128 lanes, for experts with many rows. Bound
//                     by the promotion of each K block's partial and by power: 8192 tokens x 8 of 64 experts, fused
//                     5120 -> 2 x 1024 858 us, plain 1024 -> 5120 475 us (1.5 PFLOP/s, at 1.45-1.65 GHz under the
//                     1000 W limit; a tile costs 128 rows whatever it holds). The plain product with fp32 output, whose
//                     threads write 16 bytes of a row each, takes 1086 us. The fused form spills 8 bytes (68 reloaded).
//   k_grouped_tokens  128 weight rows on the lanes, up to 16 or 32 rows on the columns, for experts with few rows. Bound by
//                     the weights' stream: 61 tokens x 8 of 64 experts, the same products: 100 us (6.7 TB/s), 58 us;
//                     one token: 18.7 us for 84 MB, of which some 6 us are the start (the plan, the first boxes) and end
#pragma once
#include "bs_common.cuh"
#include "bs_prefill.cuh"
#include "bs_route.cuh"

namespace bs {

struct GroupedParams {
  int E, R;             // local experts; rows of the output
  int rows_a;           // rows of A
  int nblk;             // 128-row weight blocks per expert
  int KB;
  int ldc;              // plain: row stride of the output, in elements
  int b_tiled, out_f32;
  const int* offsets;   // [E + 1]
  const int* row_token; // [R]: row of A for each row; nullptr: the row itself
  const uint8_t* A;     // [rows_a, K]
  const float* As;      // [rows_a, KB]
  const float* Bs;      // [E, nblk, KB]
  void* out;            // plain: [R, ldc]; fused: Q [R, I]
  float* qs;            // fused: [R, I / 128]
  int* status;
};

// 4 rows x 128 bytes: rows y0..y3 of a map whose box is one row high, 128-byte swizzle.
__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* map, uint64_t* bar, int x, const int4& y,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w),
      "l"(policy)
      : "memory");
}

// The experts that have rows, in order.
struct GroupTable {
  int n, tiles;
  int expert[kMaxExperts];
  int row0[kMaxExperts], rows[kMaxExperts];
  int tile0[kMaxExperts];  // first tile of the expert
};

// One warp. An offset outside [0, R] or below its predecessor counts as that bound, so a bad plan reads and writes
// nothing outside the buffers.
__device__ __forceinline__ void build_table(GroupTable& g, const GroupedParams& p, int tile_rows, int num_n) {
  const int lane = threadIdx.x & 31;
  int n = 0, tiles = 0;
  for (int e0 = 0; e0 < p.E; e0 += 32) {
    const int e = e0 + lane;
    int lo = 0, rows = 0;
    if (e < p.E) {
      lo = min(max(__ldcg(p.offsets + e), 0), p.R);
      rows = max(min(__ldcg(p.offsets + e + 1), p.R) - lo, 0);
    }
    const uint32_t has = __ballot_sync(0xffffffffu, rows > 0);
    const int mine = (rows + tile_rows - 1) / tile_rows * num_n;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (rows > 0) {
      const int i = n + __popc(has & ((1u << lane) - 1));
      g.expert[i] = e;
      g.row0[i] = lo;
      g.rows[i] = rows;
      g.tile0[i] = tiles + inc - mine;
    }
    n += __popc(has);
    tiles += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (lane == 0) {
    g.n = n;
    g.tiles = tiles;
  }
}

struct GroupTile {
  int expert, tn;
  int row, rows;  // first row, rows of this tile (1 .. tile_rows)
};

// Tile -> expert (binary search), weight column tile and row tile.
__device__ __forceinline__ GroupTile find_tile(const GroupTable& g, int tile, int tile_rows) {
  int lo = 0, hi = g.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (g.tile0[mid] <= tile) lo = mid;
    else hi = mid;
  }
  const int in = tile - g.tile0[lo];
  const int tm = (g.rows[lo] + tile_rows - 1) / tile_rows;
  GroupTile t;
  t.expert = g.expert[lo];
  t.tn = in / tm;
  const int m = in - t.tn * tm;
  t.row = g.row0[lo] + m * tile_rows;
  t.rows = min(g.rows[lo] - m * tile_rows, tile_rows);
  return t;
}

// Row of A behind output row r.
__device__ __forceinline__ int source_row(const GroupedParams& p, int r) {
  if (!p.row_token) return r < p.rows_a ? r : 0;
  const int t = __ldg(p.row_token + r);
  return static_cast<unsigned>(t) < static_cast<unsigned>(p.rows_a) ? t : 0;
}

// 16 bytes from global to shared memory, not through L1, tracked by the thread's cp.async groups.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// 16 bytes of zeros, by the same way.
__device__ __forceinline__ void cp_async16_zero(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, 0;" ::"r"(dst), "l"(src) : "memory");
}
// One arrival on `bar` when every copy this thread has issued so far has landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---------------------------------------------------------------- many rows per expert
// Roles, stages, TMEM buffers and the promotion are those of k_prefill (bs_prefill.cuh). When the rows are gathered,
// warps 10 and 11 bring them, 64 rows each, with 16-byte cp.async copies written where the 128-byte swizzle of a TMA
// load would put them (chunk c of row r at chunk c ^ (r % 8)). 8192 tokens x 8 of 64 experts, K = 5120, N = 2048, plain:
// 1894 us with gathering TMA loads (four rows each, one every 50 ns), 819 us with the loaders, 790 us with the rows
// already in order. The loaders share the promotion warps' issue slots, so their instructions per copy count: 971 us with
// 64-bit row products and a shared-memory load for each copy.
// BOX (plain bf16 output): whole 32-row pieces of a tile leave by TMA from 64 KB of shared memory, at three stages. Measured
// (64 experts, K = 1024, N = 5120; without and with): mean 30 rows per expert 68 and 75 us, 125 rows 102 and 102, 1024
// rows 516 and 493.
template <bool FUSED, bool BOX>
struct GroupedRowsCfg {
  using Regs = RegSplit<384, 168, 40, 232>;
  static constexpr int kThreads = Regs::kThreads;
  static constexpr int kStages = BOX ? 3 : 4;
  static constexpr int kABytes = 128 * 128;
  static constexpr int kStageBytes = kABytes + 256 * 128;
  static constexpr int kXchOff = kStages * kStageBytes;
  // amax halves; plain: 2 or 8 KB per promotion warp
  static constexpr int kXchBytes = FUSED ? 128 * 2 * 4 : BOX ? 8 * 8192 : 8 * 2048;
  static constexpr int kTokOff = kXchOff + kXchBytes;               // gathered rows of the loaders' tile
  static constexpr int kBarOff = kTokOff + 128 * 4;
  static constexpr int kTableOff = kBarOff + 256;
  static constexpr int kSmemBytes = kTableOff + static_cast<int>(sizeof(GroupTable)) + 1024;
  static constexpr int kTmemCols = 512;
};

template <bool FUSED, bool BOX = false>
__global__ void __launch_bounds__(GroupedRowsCfg<FUSED, BOX>::kThreads, 1)
    k_grouped_rows(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmO, const GroupedParams p) {
  static_assert(!(FUSED && BOX), "the fused output is written by its threads");
  using Cfg = GroupedRowsCfg<FUSED, BOX>;
  constexpr int S = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOff);  // [S] TMA -> MMA
  uint64_t* empty = full + S;                                         // [S] MMA -> TMA
  uint64_t* pfull = empty + S;                                        // [2] MMA -> promotion
  uint64_t* pempty = pfull + 2;                                       // [2] promotion -> MMA
  uint64_t* drain = pempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* amax_x = reinterpret_cast<float*>(smem + Cfg::kXchOff);  // fused: [128 rows][2 halves]
  uint32_t* tok = reinterpret_cast<uint32_t*>(smem + Cfg::kTokOff);
  const bool gather = p.row_token != nullptr;
  GroupTable& table = *reinterpret_cast<GroupTable*>(smem + Cfg::kTableOff);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], gather ? 1 + 64 : 1);  // the producer, and the loader threads
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&pfull[i], 1);
      mbar_init(&pempty[i], 256);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    grid_dep_launch();
  }
  const int KB = p.KB, nblk = p.nblk;
  const int I_blk = FUSED ? nblk / 2 : 0;
  const int num_n = FUSED ? I_blk : (nblk + 1) / 2;
  if (warp == 9) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  grid_dep_wait();  // the plan, the rows and the output may belong to the previous kernel
  if (warp == 0) build_table(table, p, 128, num_n);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int num_tiles = table.tiles;

  if (warp >= 8) {
    regs_decrease<Cfg::Regs::kProducer>();
    if (warp == 8 && lane == 0) {
      // ------------------------------------------------------------ TMA producer
      const uint64_t pol_a = policy_evict_last(), pol_b = policy_evict_normal();
      int s = 0;
      uint32_t ph = 0, issued = 0, parity_bits = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        const GroupTile t = find_tile(table, tile, 128);
        const int nb = t.expert * nblk;
        for (int kb = 0; kb < KB; ++kb) {
          ok = mbar_wait(&empty[s], ph ^ 1, abort_flag, p.status, kErrTimeoutEmpty);
          if (!ok) break;
          uint8_t* st = smem + s * Cfg::kStageBytes;
          mbar_arrive_expect_tx(&full[s], gather ? Cfg::kStageBytes - Cfg::kABytes : Cfg::kStageBytes);
          if constexpr (FUSED) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              load_weight_half(st + Cfg::kABytes + 16384 * h, &tmB, &full[s], nb + t.tn, h, kb, KB, p.b_tiled, pol_b);
              load_weight_half(st + Cfg::kABytes + 16384 * h + 8192, &tmB, &full[s], nb + t.tn + I_blk, h, kb, KB,
                               p.b_tiled, pol_b);
            }
          } else {
            load_weight_box(st + Cfg::kABytes, &tmB, &full[s], nb + 2 * t.tn, kb, KB, p.b_tiled, pol_b);
            load_weight_box(st + Cfg::kABytes + 16384, &tmB, &full[s], nb + 2 * t.tn + 1, kb, KB, p.b_tiled, pol_b);
          }
          if (!gather) tma_load_2d(st, &tmA, &full[s], kb * 128, t.row, pol_a);
          issued |= 1u << s;
          parity_bits = (parity_bits & ~(1u << s)) | (ph << s);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      if (!ok) {
        // Leave no copy in flight. (With loaders the barrier also waits for them, and one that gave up never
        // arrives: the copies land within microseconds.)
        if (gather) pause_ns(2000000ull);
        for (int i = 0; i < S && !gather; ++i)
          if (issued & (1u << i))
            mbar_wait(&full[i], (parity_bits >> i) & 1u, abort_flag, p.status, kErrTimeoutDrain, 100000000ull);
      }
    } else if (warp >= 10 && gather) {
      // ------------------------------------------------------------ row loaders
      // Copy i of a lane: chunk lane % 8 of row 64 w + 4 i + lane / 8. The stage's barrier hears from every loader thread
      // when its copies have landed; the MMA issuer makes them visible to the tensor core (its fence), so a loader
      // never waits for its own copies.
      const int w = warp - 10, c = lane & 7, sub = lane >> 3;
      uint32_t* mine = tok + 64 * w;  // start of row 4 i + sub in 16-byte units, at [16 sub + i]
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      const uint32_t row16 = static_cast<uint32_t>(KB) * 8;
      // of the rows at mine[lane] and mine[lane + 32]
      auto sources = [&](int tile, uint32_t& a, uint32_t& b) {
        if (tile >= num_tiles) return;
        const GroupTile t = find_tile(table, tile, 128);
        const int ra = 64 * w + 4 * (lane & 15) + (lane >> 4);
        a = static_cast<uint32_t>(source_row(p, t.row + min(ra, t.rows - 1))) * row16;
        b = static_cast<uint32_t>(source_row(p, t.row + min(ra + 2, t.rows - 1))) * row16;
      };
      uint32_t src0 = 0, src1 = 0;
      sources(blockIdx.x, src0, src1);
      const uint32_t even = 128 * sub + 16 * (c ^ sub), odd = 128 * sub + 16 * (c ^ (sub + 4));  // rows 8 j + sub, + 4
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        __syncwarp();
        mine[lane] = src0;
        mine[lane + 32] = src1;
        __syncwarp();
        // Rows past the tile's, in sixteens, are zeros, written once into each stage: their results are never read, but
        // the tensor core's power goes by the values.
        const int rows = find_tile(table, tile, 128).rows - 64 * w;
        sources(tile + gridDim.x, src0, src1);  // the next tile's, a whole tile ahead
        const uint8_t* src = p.A + c * 16;
        for (int kb = 0; kb < KB; ++kb, src += 128) {
          ok = mbar_wait_warp(&empty[s], ph ^ 1, abort_flag, p.status, kErrTimeoutEmpty);
          if (!ok) break;
          const uint32_t st = smem_u32(smem + s * Cfg::kStageBytes) + 8192 * w;
#pragma unroll
          for (int i = 0; i < 16; i += 4) {
            if (4 * i >= rows) {
              if (kb < S) {
#pragma unroll
                for (int j = 0; j < 4; ++j) cp_async16_zero(st + ((j & 1) ? odd : even) + 512 * (i + j), src);
              }
              continue;
            }
            const uint4 o = *reinterpret_cast<const uint4*>(mine + 16 * sub + i);
            cp_async16(st + even + 512 * i, src + static_cast<uint64_t>(o.x) * 16);
            cp_async16(st + odd + 512 * (i + 1), src + static_cast<uint64_t>(o.y) * 16);
            cp_async16(st + even + 512 * (i + 2), src + static_cast<uint64_t>(o.z) * 16);
            cp_async16(st + odd + 512 * (i + 3), src + static_cast<uint64_t>(o.w) * 16);
          }
          cp_async_arrive(&full[s]);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      cp_async_wait_all();
    } else if (warp == 9 && lane == 0) {
      // ------------------------------------------------------------ MMA issuer
      constexpr uint32_t idesc = idesc_e4m3_f32(128, 256);
      int s = 0, b = 0;
      uint32_t ph = 0, pph = 0;
      bool ok = true;
      for (int tile = blockIdx.x; ok && tile < num_tiles; tile += gridDim.x) {
        for (int kb = 0; kb < KB; ++kb) {
          ok = mbar_wait(&full[s], ph, abort_flag, p.status, kErrTimeoutFull) &&
               mbar_wait(&pempty[b], pph ^ 1, abort_flag, p.status, kErrTimeoutPEmpty);
          if (!ok) break;
          if (gather) fence_proxy_async_smem();  // the loaders' rows, written by ordinary copies
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + s * Cfg::kStageBytes);
          const uint32_t b0 = a0 + Cfg::kABytes;
          const uint32_t d = tmem + static_cast<uint32_t>(b * 256);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_e4m3(d, desc_kmajor_sw128(a0 + 32 * k), desc_kmajor_sw128(b0 + 32 * k), idesc, k > 0 ? 1u : 0u);
          mma_commit(&empty[s]);
          mma_commit(&pfull[b]);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
          if (++b == 2) {
            b = 0;
            pph ^= 1;
          }
        }
      }
      mma_commit(drain);
      mbar_wait(drain, 0, abort_flag, p.status, kErrTimeoutDrain, 100000000ull);
    }
  } else {
    regs_increase<Cfg::Regs::kConsumer>();
    // ------------------------------------------------------------ promotion + epilogue (as in k_prefill)
    const int wg = warp >> 2;
    const int q = warp & 3;
    const int r = q * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    int b = 0;
    uint32_t pph = 0;
    bool ok = true;
    auto source_of = [&](int tile) {
      if (tile >= num_tiles) return 0;
      const GroupTile t = find_tile(table, tile, 128);
      return source_row(p, t.row + (r < t.rows ? r : 0));
    };
    int src = source_of(blockIdx.x);
    for (int tile = blockIdx.x; tile < num_tiles; tile += gridDim.x) {
      const GroupTile t = find_tile(table, tile, 128);
      const bool row_ok = r < t.rows;
      const int row = t.row + (row_ok ? r : 0);
      const int nb = FUSED ? t.tn : 2 * t.tn + wg;  // block inside the expert; fused: the gate's
      const bool col_ok = nb < nblk;
      const float* as_row = p.As + static_cast<size_t>(src) * KB;
      src = source_of(tile + gridDim.x);  // a whole tile ahead
      const float* bs_row = p.Bs + (static_cast<size_t>(t.expert) * nblk + (col_ok ? nb : 0)) * KB;
      const float* bu_row = bs_row + static_cast<size_t>(FUSED ? I_blk : 0) * KB;

      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
      auto promote = [&](uint64_t sc2, uint64_t scu2) {
        if (ok && !mbar_wait_warp(&pfull[b], pph, abort_flag, p.status, kErrTimeoutPFull)) ok = false;
        if (ok) {
          tc_fence_after();
          const uint32_t tbase = tmem + lane_addr + static_cast<uint32_t>(b * 256 + wg * 128);
          uint32_t v[64];
          tmem_ld64(tbase, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) ffma2(acc[i], v[2 * i], v[2 * i + 1], sc2);
          tmem_ld64(tbase + 64, v);
          tmem_ld_wait();
          mbar_arrive(&pempty[b]);
#pragma unroll
          for (int i = 0; i < 32; ++i) ffma2(acc[32 + i], v[2 * i], v[2 * i + 1], scu2);
        }
        if (++b == 2) {
          b = 0;
          pph ^= 1;
        }
      };
      if constexpr (FUSED) {
        constexpr int D = 4;  // scales in groups of four K blocks, one group ahead
        float sa[D], sg[D], su[D];
#pragma unroll
        for (int j = 0; j < D; ++j) {
          const int k = j < KB ? j : KB - 1;
          sa[j] = ldg_f32(as_row + k);
          sg[j] = ldg_f32(bs_row + k);
          su[j] = ldg_f32(bu_row + k);
        }
        for (int kb0 = 0; kb0 < KB; kb0 += D) {
          float na[D], ng[D], nu[D];
#pragma unroll
          for (int j = 0; j < D; ++j) {
            const int kn = kb0 + D + j < KB ? kb0 + D + j : KB - 1;
            na[j] = ldg_f32(as_row + kn);
            ng[j] = ldg_f32(bs_row + kn);
            nu[j] = ldg_f32(bu_row + kn);
          }
#pragma unroll
          for (int j = 0; j < D; ++j) {
            if (kb0 + j >= KB) break;
            const float scg = __fmul_rn(sa[j], sg[j]), scu = __fmul_rn(sa[j], su[j]);
            promote(pack_f2(scg, scg), pack_f2(scu, scu));
          }
#pragma unroll
          for (int j = 0; j < D; ++j) {
            sa[j] = na[j];
            sg[j] = ng[j];
            su[j] = nu[j];
          }
        }
      } else {
        const int kn1 = KB > 1 ? 1 : 0;
        float a_n0 = ldg_f32(as_row), b_n0 = ldg_f32(bs_row);
        float a_n1 = ldg_f32(as_row + kn1), b_n1 = ldg_f32(bs_row + kn1);
        for (int kb = 0; kb < KB; ++kb) {
          const float sa = a_n0, sb = b_n0;
          a_n0 = a_n1;
          b_n0 = b_n1;
          if (kb + 2 < KB) {
            a_n1 = ldg_f32(as_row + kb + 2);
            b_n1 = ldg_f32(bs_row + kb + 2);
          }
          const float sc = __fmul_rn(sa, sb);
          promote(pack_f2(sc, sc), pack_f2(sc, sc));
        }
      }

      if constexpr (!FUSED) {
        if (ok && col_ok) {
          if (p.out_f32) {
            if (row_ok) {
              float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + static_cast<size_t>(row) * p.ldc +
                                                      static_cast<size_t>(nb) * 128);
#pragma unroll
              for (int j = 0; j < 32; ++j)
                dst[j] = make_float4(lo_f(acc[2 * j]), hi_f(acc[2 * j]), lo_f(acc[2 * j + 1]), hi_f(acc[2 * j + 1]));
            }
          } else if constexpr (BOX) {
            // A warp's 32 rows x 128 columns leave as two boxes of 64 columns by TMA, from 8 KB of shared memory laid
            // out as the map's 128-byte swizzle has it (a row of a box at 128 bytes, chunk c at c ^ (row % 8)). Rows
            // of the tile that do not exist belong to the next expert: such a warp stores its rows itself, 128
            // bytes of four rows at a time.
            uint8_t* buf = smem + Cfg::kXchOff + warp * 8192;
            const int rows = t.rows - q * 32;
            bulk_wait_read_all();  // lane 0: the boxes of the previous tile
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; ++j)
              *reinterpret_cast<uint4*>(buf + (j >> 3) * 4096 + lane * 128 + (((j & 7) ^ (lane & 7)) * 16)) =
                  make_uint4(pack_bf16x2(lo_f(acc[4 * j]), hi_f(acc[4 * j])),
                             pack_bf16x2(lo_f(acc[4 * j + 1]), hi_f(acc[4 * j + 1])),
                             pack_bf16x2(lo_f(acc[4 * j + 2]), hi_f(acc[4 * j + 2])),
                             pack_bf16x2(lo_f(acc[4 * j + 3]), hi_f(acc[4 * j + 3])));
            if (rows >= 32) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&tmO, buf, nb * 256, t.row + q * 32);
                tma_store_2d(&tmO, buf + 4096, nb * 256 + 128, t.row + q * 32);
                bulk_commit();
              }
            } else if (rows > 0) {
              __syncwarp();
              __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(t.row + q * 32) * p.ldc +
                                   static_cast<size_t>(nb) * 128 + (lane & 7) * 8;
#pragma unroll 4
              for (int i = 0; i < 16; ++i) {
                const int rr = 4 * (i >> 1) + (lane >> 3);
                const uint4 v = *reinterpret_cast<const uint4*>(buf + (i & 1) * 4096 + rr * 128 + (((lane & 7) ^ (rr & 7)) * 16));
                if (rr < rows) *reinterpret_cast<uint4*>(dst + static_cast<size_t>(rr) * p.ldc + (i & 1) * 64) = v;
              }
            }
          } else {
            // A warp's 32 rows x 32 columns at a time through 2 KB of shared memory (chunks of 16 bytes, swizzled), so
            // that a store writes whole 64-byte pieces of eight rows instead of 16 bytes of 32 rows.
            uint4* buf = reinterpret_cast<uint4*>(smem + Cfg::kXchOff) + warp * 128;
            __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(p.out) + static_cast<size_t>(t.row + q * 32) * p.ldc +
                                 static_cast<size_t>(nb) * 128 + (lane & 3) * 8;
#pragma unroll
            for (int h = 0; h < 4; ++h) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const int j = 16 * h + 4 * c;  // columns 2j .. 2j + 7
                buf[lane * 4 + (c ^ ((lane >> 1) & 3))] =
                    make_uint4(pack_bf16x2(lo_f(acc[j]), hi_f(acc[j])), pack_bf16x2(lo_f(acc[j + 1]), hi_f(acc[j + 1])),
                               pack_bf16x2(lo_f(acc[j + 2]), hi_f(acc[j + 2])),
                               pack_bf16x2(lo_f(acc[j + 3]), hi_f(acc[j + 3])));
              }
              __syncwarp();
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int rr = 8 * i + (lane >> 2);
                const uint4 v = buf[rr * 4 + ((lane & 3) ^ ((rr >> 1) & 3))];
                if (q * 32 + rr < t.rows) *reinterpret_cast<uint4*>(dst + static_cast<size_t>(rr) * p.ldc + 32 * h) = v;
              }
              __syncwarp();
            }
          }
        }
      } else {
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float y0 = silu_mul(lo_f(acc[i]), lo_f(acc[32 + i]));
          const float y1 = silu_mul(hi_f(acc[i]), hi_f(acc[32 + i]));
          acc[i] = pack_f2(y0, y1);
          amax = fmaxf(amax, fmaxf(fabsf(y0), fabsf(y1)));
        }
        amax_x[r * 2 + wg] = amax;
        named_bar_sync(1, 256);
        amax = fmaxf(amax_x[r * 2], amax_x[r * 2 + 1]);
        const float scale = __fdiv_rn(fmaxf(amax, 1e-10f), 448.0f);
        const float inv = __fdiv_rn(1.0f, scale);
        if (ok && row_ok) {
          if (wg == 0) p.qs[static_cast<size_t>(row) * I_blk + t.tn] = scale;
          uint4* dst = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + static_cast<size_t>(row) * I_blk * 128 +
                                                static_cast<size_t>(t.tn) * 128 + wg * 64);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const int e = 8 * j + 2 * h;
              w[h] = f2_to_e4m3x2(__fmul_rn(lo_f(acc[e]), inv), __fmul_rn(hi_f(acc[e]), inv)) |
                     (f2_to_e4m3x2(__fmul_rn(lo_f(acc[e + 1]), inv), __fmul_rn(hi_f(acc[e + 1]), inv)) << 16);
            }
            dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        named_bar_sync(1, 256);  // amax_x is free for the next tile
      }
    }
    if constexpr (BOX) bulk_wait_read_all();  // the last boxes have left shared memory
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::kTmemCols);
  }
}

// ---------------------------------------------------------------- few rows per expert
// Swap-AB as in bs_decode.cuh: the weight block's 128 rows are the MMA's M, up to NT output rows ("tokens") its N. A
// cluster of S CTAs takes a tile together: CTA j of it streams the j-th 1/S of the K blocks, then every CTA sends its
// fp32 partial of token tt to CTA tt % S through distributed shared memory, which adds the S partials in CTA order and
// finishes its tokens. So a call with few tiles still uses every SM, the sum's order is fixed, and no partial goes
// through global memory.
//
// CTA layout (384 threads): warps 0-7 promotion (warpgroup g: tokens [g * NT/2, ...)) and epilogue, warp 8 TMA
// producer, warp 9 TMEM + MMA issuer, warp 10 scale products As[src, kb] * Bs[nb, kb] into a ring of eight slots, warp 11
// hands the exchange buffer back to the cluster.
// A unit of the pipeline is kKu K blocks of a tile (32 KB of weights): gate and up of one K block, or two K blocks of
// one weight block, each set of partials in TMEM columns of its own.
template <bool FUSED, int NT>
struct GroupedTokensCfg {
  static constexpr int kThreads = 384;
  static constexpr int kNwg = FUSED ? 2 : 1;
  static constexpr int kKu = FUSED ? 1 : 2;
  static constexpr int kSets = kNwg * kKu;
  static constexpr int kTr = NT / 2;
  static_assert(NT <= 32, "a lane of the scale warp per token");
  static constexpr int kWBytes = 16384 * kNwg;  // per K block
  static constexpr int kXBytes = NT * 128;
  static constexpr int kBlockBytes = kWBytes + ((kXBytes + 1023) / 1024) * 1024;
  static constexpr int kStageBytes = kKu * kBlockBytes;
  static constexpr int kBufCols = kSets * NT;
  // 4 and 8 buffers: 69.0 and 67.5 us where a CTA has several tiles (fused, 128 experts, 160 tokens), equal elsewhere.
  static constexpr int kBufs = 8;
  static constexpr int kTmemCols = kBufs * kBufCols;
  static_assert((kTmemCols & (kTmemCols - 1)) == 0 && kTmemCols >= 32 && kTmemCols <= 512, "TMEM columns");
  static constexpr int kSlots = 8;
  static constexpr int kRingBytes = kSlots * kSets * NT * 4;
  static constexpr int kXchBytes = kNwg * NT * 128 * 4;     // [S][kNwg][NT / S][128] partials
  static constexpr int kAmaxBytes = FUSED ? NT * 4 * 4 : 0;  // [own token][4 warps]
  static constexpr int kBarBytes = 512;
  static constexpr int kTail = kRingBytes + kXchBytes + kAmaxBytes + kBarBytes + static_cast<int>(sizeof(GroupTable));
  static constexpr int kStagesRaw = (232448 - 1024 - kTail) / kStageBytes;
  static constexpr int kStages = kStagesRaw > 10 ? 10 : kStagesRaw;
  static_assert(kStages >= 3, "pipeline depth");
  static constexpr int kXchOff = kStages * kStageBytes;
  static constexpr int kRingOff = kXchOff + kXchBytes;
  static constexpr int kAmaxOff = kRingOff + kRingBytes;
  static constexpr int kBarOff = kAmaxOff + kAmaxBytes;
  static constexpr int kTableOff = kBarOff + kBarBytes;
  static constexpr int kUsed = kTableOff + static_cast<int>(sizeof(GroupTable));
  // more than half of the SM's shared memory, so that a second CTA (and its TMEM) never lands on the SM
  static constexpr int kSmemBytes = (kUsed > 120 * 1024 ? kUsed : 120 * 1024) + 1024;
};

// A word into a CTA of the cluster; its 4 bytes are counted on that CTA's barrier `bar` when they have arrived.
__device__ __forceinline__ void st_async_f32(uint32_t addr, float v, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(addr),
               "r"(__float_as_uint(v)), "r"(bar)
               : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// Remote arrival that releases what the thread has read and written, and what it has acquired, to the cluster.
__device__ __forceinline__ void mbar_arrive_remote_release(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// mbar_wait_warp that also acquires what CTAs of the cluster published.
__device__ __forceinline__ bool mbar_wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort, int* status) {
  if (__all_sync(0xffffffffu, mbar_try_wait_cluster(bar, parity))) return true;
  const uint64_t t0 = globaltimer_ns();
  uint32_t spins = 0;
  while (true) {
    if (__all_sync(0xffffffffu, mbar_try_wait_cluster(bar, parity))) return true;
    if ((spins++ & 63u) == 0) {
      const bool late = globaltimer_ns() - t0 > kWaitLimitNs;
      if (late) {
        atomicCAS(status, 0, kErrTimeoutCluster);
        *abort = 1;
      }
      if (__any_sync(0xffffffffu, late || *abort)) return false;
    }
  }
}

// log_s: log2 of the cluster size S (1, 2, 4, 8).
template <bool FUSED, int NT>
__global__ void __launch_bounds__(GroupedTokensCfg<FUSED, NT>::kThreads, 1)
    k_grouped_tokens(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                     const GroupedParams p, const int log_s) {
  using Cfg = GroupedTokensCfg<FUSED, NT>;
  constexpr int ST = Cfg::kStages, NWG = Cfg::kNwg, KU = Cfg::kKu, NSET = Cfg::kSets, NB = Cfg::kBufs, NS = Cfg::kSlots,
                TR = Cfg::kTr;
  extern __shared__ uint8_t smem_raw[];
  // (the offset of the aligned base is the same in every CTA: mapped addresses of the cluster's CTAs agree)
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* xch = reinterpret_cast<float*>(smem + Cfg::kXchOff);
  float* ring = reinterpret_cast<float*>(smem + Cfg::kRingOff);  // [NS][KU][NWG][NT] scale products
  float* amx = reinterpret_cast<float*>(smem + Cfg::kAmaxOff);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + Cfg::kBarOff);
  uint64_t* empty = full + ST;
  uint64_t* pfull = empty + ST;
  uint64_t* pempty = pfull + NB;
  uint64_t* sfull = pempty + NB;
  uint64_t* sempty = sfull + NS;
  uint64_t* drain = sempty + NS;
  uint64_t* rfull = drain + 1;   // every CTA's partials of this CTA's tokens are here
  uint64_t* rempty = rfull + 1;  // every CTA has read the partials of the previous tile
  uint64_t* rread = rempty + 1;  // this CTA's warps have
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rread + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * ST + 2 * NB + 2 * NS + 4) * 8 + 8 <= Cfg::kBarBytes, "barrier area");
  GroupTable& table = *reinterpret_cast<GroupTable*>(smem + Cfg::kTableOff);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int S = 1 << log_s;
  const int rank = static_cast<int>(cluster_ctarank());
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < NB; ++i) {
      mbar_init(&pfull[i], 1);
      mbar_init(&pempty[i], 256);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&sfull[i], 32);
      mbar_init(&sempty[i], 256);
    }
    mbar_init(drain, 1);
    mbar_init(rfull, 1);
    mbar_init(rempty, S);
    mbar_init(rread, 8);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
    grid_dep_launch();
  }
  const int KB = p.KB, nblk = p.nblk;
  const int I_blk = FUSED ? nblk / 2 : 0;
  const int num_n = FUSED ? I_blk : nblk;
  if (warp == 9) {
    tmem_alloc(tmem_slot, Cfg::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // every CTA's barriers exist before a remote arrival
  tc_fence_after();
  grid_dep_wait();  // what follows may read the previous kernel's output
  if (warp == 0) build_table(table, p, NT, num_n);
  __syncthreads();
  const uint32_t tmem = *tmem_slot;
  const int num_tiles = table.tiles;
  const int first = static_cast<int>(blockIdx.x) >> log_s, step = static_cast<int>(gridDim.x) >> log_s;
  const int kb0 = KB * rank >> log_s, kb1 = KB * (rank + 1) >> log_s;

  if (warp == 8) {
    // ------------------------------------------------------------ TMA producer
    const uint64_t pol_w = policy_evict_first(), pol_x = policy_evict_last();
    const bool gather = p.row_token != nullptr;
    int s = 0;
    uint32_t ph = 0, issued = 0, parity_bits = 0;
    bool ok = true;
    for (int tile = first; ok && tile < num_tiles; tile += step) {
      const GroupTile t = find_tile(table, tile, NT);
      const int quads = (t.rows + 3) / 4;
      int4 rows = make_int4(0, 0, 0, 0);
      if (gather && lane < quads) {
        const int last = t.row + t.rows - 1, r = t.row + 4 * lane;
        rows = make_int4(source_row(p, r), source_row(p, min(r + 1, last)), source_row(p, min(r + 2, last)),
                         source_row(p, min(r + 3, last)));
      }
      const int nb = t.expert * nblk + t.tn;
      for (int kb = kb0; kb < kb1; kb += KU) {
        if (lane == 0) ok = mbar_wait(&empty[s], ph ^ 1, abort_flag, p.status, kErrTimeoutEmpty);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        uint8_t* st = smem + s * Cfg::kStageBytes;
        const int nk = min(KU, kb1 - kb);
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[s], nk * (Cfg::kWBytes + (gather ? quads * 512 : Cfg::kXBytes)));
#pragma unroll
          for (int h = 0; h < KU; ++h) {
            if (h >= nk) break;
            uint8_t* sh = st + h * Cfg::kBlockBytes;
#pragma unroll
            for (int w = 0; w < NWG; ++w)
              load_weight_box(sh + w * 16384, &tmW, &full[s], w == 0 ? nb : nb + I_blk, kb + h, KB, p.b_tiled, pol_w);
            if (!gather) tma_load_2d(sh + Cfg::kWBytes, &tmX, &full[s], (kb + h) * 128, t.row, pol_x);
          }
        }
        __syncwarp();
        if (gather && lane < quads) {
#pragma unroll
          for (int h = 0; h < KU; ++h)
            if (h < nk)
              tma_gather4(st + h * Cfg::kBlockBytes + Cfg::kWBytes + 512 * lane, &tmX, &full[s], (kb + h) * 128, rows, pol_x);
        }
        issued |= 1u << s;
        parity_bits = (parity_bits & ~(1u << s)) | (ph << s);
        if (++s == ST) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    if (!ok && lane == 0)
      for (int i = 0; i < ST; ++i)
        if (issued & (1u << i))
          mbar_wait(&full[i], (parity_bits >> i) & 1u, abort_flag, p.status, kErrTimeoutDrain, 100000000ull);
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      int s = 0, b = 0;
      uint32_t ph = 0, pph = 0;
      bool ok = true;
      for (int tile = first; ok && tile < num_tiles; tile += step) {
        const GroupTile t = find_tile(table, tile, NT);
        // Columns past the tile's rows are computed from whatever the stage holds (or skipped) and never read.
        const uint32_t idesc = idesc_e4m3_f32(128, (t.rows + 15) / 16 * 16);
        for (int kb = kb0; kb < kb1; kb += KU) {
          ok = mbar_wait(&full[s], ph, abort_flag, p.status, kErrTimeoutFull) &&
               mbar_wait(&pempty[b], pph ^ 1, abort_flag, p.status, kErrTimeoutPEmpty);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int h = 0; h < KU; ++h) {
            if (kb + h >= kb1) break;
            const uint32_t st = smem_u32(smem + s * Cfg::kStageBytes + h * Cfg::kBlockBytes);
            const uint32_t xs = st + Cfg::kWBytes;
#pragma unroll
            for (int w = 0; w < NWG; ++w) {
              const uint32_t d = tmem + static_cast<uint32_t>(b * Cfg::kBufCols + (h * NWG + w) * NT);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_e4m3(d, desc_kmajor_sw128(st + w * 16384 + 32 * k), desc_kmajor_sw128(xs + 32 * k), idesc,
                         k > 0 ? 1u : 0u);
            }
          }
          mma_commit(&empty[s]);
          mma_commit(&pfull[b]);
          if (++s == ST) {
            s = 0;
            ph ^= 1;
          }
          if (++b == NB) {
            b = 0;
            pph ^= 1;
          }
        }
      }
      mma_commit(drain);
      mbar_wait(drain, 0, abort_flag, p.status, kErrTimeoutDrain, 100000000ull);
    }
  } else if (warp == 11) {
    // ------------------------------------------------------------ the exchange buffer, back to the cluster
    // What the promotion warps have read and written there is behind this CTA's barrier, and the arrivals release it to
    // the CTAs that write the next partials. A warp of its own, since a release to the cluster takes its time and the
    // next tile needs it only at its end: with the promotion warps releasing, 61 tokens take 103.5 us instead of 100.0,
    // 128 experts and 160 tokens 79.5 instead of 67.4.
    if (log_s > 0) {
      uint32_t ph = 0;
      for (int tile = first; tile < num_tiles; tile += step, ph ^= 1) {
        if (!mbar_wait_warp(rread, ph, abort_flag, p.status, kErrTimeoutCluster)) break;
        if (lane < S) mbar_arrive_remote_release(mapa_shared(rempty, lane));
      }
    }
  } else if (warp == 10) {
    // ------------------------------------------------------------ scale products
    int slot = 0;
    uint32_t sph = 0;
    bool ok = true;
    for (int tile = first; ok && tile < num_tiles; tile += step) {
      const GroupTile t = find_tile(table, tile, NT);
      const float* arow = p.As + static_cast<size_t>(source_row(p, t.row + (lane < t.rows ? lane : 0))) * KB;
      const float* brow = p.Bs + (static_cast<size_t>(t.expert) * nblk + t.tn) * KB;
      const float* urow = brow + static_cast<size_t>(I_blk) * KB;
      float a[2][KU], bw[2][KU][NWG];  // operands of this unit and the next
      auto load = [&](int u, int kb) {
#pragma unroll
        for (int h = 0; h < KU; ++h) {
          const int k = min(kb + h, kb1 - 1);
          a[u][h] = ldg_f32(arow + k);
#pragma unroll
          for (int w = 0; w < NWG; ++w) bw[u][h][w] = ldg_f32((w == 0 ? brow : urow) + k);
        }
      };
      auto write = [&](int u, int kb_next) {
        if (!mbar_wait(&sempty[slot], sph ^ 1, abort_flag, p.status, kErrTimeoutPEmpty)) {
          ok = false;
          return;
        }
        float* dst = ring + slot * (NSET * NT);
        if (lane < NT) {
#pragma unroll
          for (int h = 0; h < KU; ++h)
#pragma unroll
            for (int w = 0; w < NWG; ++w) dst[(h * NWG + w) * NT + lane] = lane < t.rows ? __fmul_rn(a[u][h], bw[u][h][w]) : 0.f;
        }
        mbar_arrive(&sfull[slot]);
        load(u, kb_next);
        if (++slot == NS) {
          slot = 0;
          sph ^= 1;
        }
      };
      if (kb0 < kb1) {
        load(0, kb0);
        load(1, min(kb0 + KU, kb1 - 1));
      }
      for (int kb = kb0; kb < kb1 && ok; kb += 2 * KU) {
        write(0, min(kb + 2 * KU, kb1 - 1));
        if (kb + KU < kb1 && ok) write(1, min(kb + 3 * KU, kb1 - 1));
      }
    }
  } else {
    // ------------------------------------------------------------ promotion + epilogue
    const int wg = warp >> 2;
    const int q = warp & 3;
    const int tok0 = wg * TR;
    const int r = q * 32 + lane;  // weight row inside the block
    const uint32_t lane_addr = static_cast<uint32_t>(q * 32) << 16;
    const int own = NT >> log_s;  // tokens a CTA finishes
    int b = 0, slot = 0;
    uint32_t pph = 0, sph = 0, rph = 0;
    bool ok = true;
    for (int tile = first; tile < num_tiles; tile += step) {
      const GroupTile t = find_tile(table, tile, NT);
      const int n = t.rows;
      uint64_t acc[NWG][TR / 2];
#pragma unroll
      for (int w = 0; w < NWG; ++w)
#pragma unroll
        for (int i = 0; i < TR / 2; ++i) acc[w][i] = 0;
      for (int kb = kb0; kb < kb1; kb += KU) {
        if (ok && !(mbar_wait_warp(&pfull[b], pph, abort_flag, p.status, kErrTimeoutPFull) &&
                    mbar_wait_warp(&sfull[slot], sph, abort_flag, p.status, kErrTimeoutPFull)))
          ok = false;
        if (ok) {
          tc_fence_after();
          const uint32_t tb = tmem + lane_addr + static_cast<uint32_t>(b * Cfg::kBufCols + tok0);
          const ulonglong2* sc = reinterpret_cast<const ulonglong2*>(ring + slot * (NSET * NT) + tok0);
          constexpr int CH = TR < 16 ? TR : 16;  // columns skipped together when the tile has no such tokens
          uint32_t v[NSET][TR];
#pragma unroll
          for (int c0 = 0; c0 < TR; c0 += CH)
            if (tok0 + c0 < n) {
#pragma unroll
              for (int w = 0; w < NSET; ++w) tmem_ld_run<CH>(tb + w * NT + c0, v[w] + c0);
            }
          tmem_ld_wait();
          mbar_arrive(&pempty[b]);
          const bool whole = kb + KU <= kb1;  // else the unit's last sets hold an earlier unit's values
#pragma unroll
          for (int c0 = 0; c0 < TR; c0 += CH)
            if (tok0 + c0 < n) {
#pragma unroll
              for (int w = 0; w < NSET; ++w)
                if (w < NWG || whole) {
#pragma unroll
                  for (int i = c0; i < c0 + CH; i += 4) {
                    const ulonglong2 s2 = sc[(w * NT + i) / 4];
                    ffma2(acc[w % NWG][i / 2], v[w][i], v[w][i + 1], s2.x);
                    ffma2(acc[w % NWG][i / 2 + 1], v[w][i + 2], v[w][i + 3], s2.y);
                  }
                }
            }
          mbar_arrive(&sempty[slot]);
        }
        if (++b == NB) {
          b = 0;
          pph ^= 1;
        }
        if (++slot == NS) {
          slot = 0;
          sph ^= 1;
        }
      }

      const int n_own = n > rank ? (n - rank + S - 1) >> log_s : 0;  // tokens this CTA finishes: rank, rank + S, ...
      // ---------------- partials to the tokens' owners. Alone, a CTA needs no more than its own barrier for it.
      if (log_s == 0) {
        named_bar_sync(3, 256);  // every warp has read the previous tile's
        if (ok) {
#pragma unroll
          for (int i = 0; i < TR; ++i)
            if (tok0 + i < n) {
#pragma unroll
              for (int w = 0; w < NWG; ++w)
                xch[(w * NT + tok0 + i) * 128 + r] = (i & 1) ? hi_f(acc[w][i / 2]) : lo_f(acc[w][i / 2]);
            }
        }
        named_bar_sync(3, 256);
      } else if (ok) {
        // The owner's barrier counts the bytes, so no fence stands between the words and their reader.
        if (threadIdx.x == 0) mbar_arrive_expect_tx(rfull, n_own * S * NWG * 512);
        ok = mbar_wait_cluster(rempty, rph ^ 1, abort_flag, p.status);
        if (ok) {
#pragma unroll
          for (int i = 0; i < TR; ++i) {
            const int tok = tok0 + i;
            if (tok < n) {
              const int to = tok & (S - 1);
              const uint32_t bar = mapa_shared(rfull, to);
#pragma unroll
              for (int w = 0; w < NWG; ++w)
                st_async_f32(mapa_shared(xch + ((rank * NWG + w) * own + (tok >> log_s)) * 128 + r, to),
                             (i & 1) ? hi_f(acc[w][i / 2]) : lo_f(acc[w][i / 2]), bar);
            }
          }
          ok = mbar_wait_cluster(rfull, rph, abort_flag, p.status);
        }
      }
      // ---------------- this CTA's tokens
      if constexpr (!FUSED) {
        if (ok) {
          for (int j = warp; j < n_own; j += 8) {
            float4 c = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int s = 0; s < S; ++s) {
              const float4 v = *reinterpret_cast<const float4*>(xch + (s * own + j) * 128 + lane * 4);
              c.x += v.x, c.y += v.y, c.z += v.z, c.w += v.w;
            }
            const size_t at = static_cast<size_t>(t.row + (j << log_s) + rank) * p.ldc + static_cast<size_t>(t.tn) * 128 + lane * 4;
            if (p.out_f32)
              *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = c;
            else
              *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + at) =
                  make_uint2(pack_bf16x2(c.x, c.y), pack_bf16x2(c.z, c.w));
          }
        }
      } else {
        // y = silu(g) * u per (token, weight row), kept in this thread's own word of the gate partial; the group's
        // amax is a warp maximum (|y| orders like its bits) and four warps' through shared memory. A NaN counts as 0
        // there, as in the row tiles (whose fmaxf drops it): it stays one NaN among well-scaled values.
        if (ok) {
          for (int j = wg; j < n_own; j += 2) {
            float g = 0.f, u = 0.f;
            for (int s = 0; s < S; ++s) {
              g += xch[((s * 2 + 0) * own + j) * 128 + r];
              u += xch[((s * 2 + 1) * own + j) * 128 + r];
            }
            const float y = silu_mul(g, u);
            xch[j * 128 + r] = y;
            const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(y), 0.f)));
            if (lane == 0) amx[j * 4 + q] = __uint_as_float(m);
          }
        }
        named_bar_sync(1 + wg, 128);
        if (ok) {
          for (int j = wg + 2 * q; j < n_own; j += 8) {
            const float4 a4 = *reinterpret_cast<const float4*>(amx + j * 4);
            const float amax = fmaxf(fmaxf(a4.x, a4.y), fmaxf(a4.z, a4.w));
            const float scale = __fdiv_rn(fmaxf(amax, 1e-10f), 448.0f);
            const float inv = __fdiv_rn(1.0f, scale);
            const size_t row = static_cast<size_t>(t.row + (j << log_s) + rank);
            if (lane == 0) p.qs[row * I_blk + t.tn] = scale;
            const float4 y = *reinterpret_cast<const float4*>(xch + j * 128 + lane * 4);
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.out) + (row * I_blk + t.tn) * 128 + lane * 4) =
                f2_to_e4m3x2(__fmul_rn(y.x, inv), __fmul_rn(y.y, inv)) |
                (f2_to_e4m3x2(__fmul_rn(y.z, inv), __fmul_rn(y.w, inv)) << 16);
          }
        }
      }
      if (ok && log_s > 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive(rread);
      }
      rph ^= 1;
    }
  }
  // No CTA leaves while another of its cluster may still write to it or arrive on its barriers.
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 9) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::kTmemCols);
  }
}

}  // namespace bs
