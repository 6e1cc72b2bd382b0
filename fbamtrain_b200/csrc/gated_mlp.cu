// Gated feed-forward block: the two projections, the activation and the product in one kernel,
//   (v, g) = x W_inᵀ + b_in     h = v act(g)          W_in (2 F, D): value rows first, gate rows behind them
// and its backward, the product of the output gradient with W_out and the derivative of the gating in one kernel,
//   dh = dy W_out     dv = dh act(g)     dg = dh v act'(g).
// The other products of the block are plain ones.
//
// Forward: the B tile of a CTA is the value rows and the gate rows of the same hidden columns, so a lane that reads an
// accumulator row back finds both factors of its results there.  On a CTA pair (one 256 x 256 tile, tcgen05 cta_group::2) the
// leader's half of B is the value rows and its peer's the gate rows; a single CTA loads both.  For a backward v and g are kept in
// fp32: 16-bit ones would add as much error to dv and dg as the rounding of those does, and the extra bytes leave while the
// tensor cores work.
//
// Backward: v and g come back through shared memory by TMA (a lane's own 128-byte rows through the load unit would take 32
// look-ups per instruction), one chunk of 32 columns ahead in the epilogue warp that needs them.
//
// Measured (bf16, 8192 rows): forward 1024 -> 4096 86 us (1 600 TFLOP/s), with the factors kept 127, gradient 95 (a floor of 62 by its
// bytes, 43 by its operations); 2048 -> 8192 318, 401, 262.  Keeping costs more than its bytes alone: they share L2 with the
// operands (neither an eviction hint, nor stores past the TMA unit, nor reading back without it changed that).  Stages: six where
// nothing is kept; four fit beside the kept chunks' staging (three: 8 to 15 % slower).
//
// Epilogue values are fp32; h, dv and dg are rounded once.  What leaves goes through shared memory and TMA tiled stores, which
// also clip rows and columns behind the end.
#include <cuda_runtime.h>
#include <stdint.h>

#include "elem16.cuh"
#include "gelu_math.cuh"
#include "gemm_epilogue.cuh"
#include "gemm_tcgen05.h"
#include "tc05.cuh"
#include "tc05_pair.cuh"
#include "tensor_map.h"

extern int g_fbam_reserved_sms;        // defined in gemm_tcgen05.cu
extern int g_fbam_last_driver_error;   // defined in gemm_tcgen05.cu

namespace {

using namespace tc05;

enum { GATE_GELU = 0, GATE_SILU = 1 };
enum { FORWARD = 0, FORWARD_KEEP = 1, BACKWARD = 2 };

constexpr int BM = 128, BK = 64, UMMA_K = 16;     // rows per CTA
constexpr int kEpiWarps = 8, kThreads = 32 * (2 + kEpiWarps);

// act(g) and act'(g) of two values
__device__ __forceinline__ float2 act2(float2 g, int act) {
  if (act == GATE_GELU) return gelu_math::gelu2(g);
  const float2 e = __fmul2_rn(g, gelu_math::f2(-1.4426950408889634f));
  const float2 d = __fadd2_rn(make_float2(gelu_math::ex2_approx(e.x), gelu_math::ex2_approx(e.y)), gelu_math::f2(1.0f));
  return __fmul2_rn(g, make_float2(gelu_math::rcp_approx(d.x), gelu_math::rcp_approx(d.y)));
}
__device__ __forceinline__ void act_and_grad2(float2 g, int act, float2& a, float2& da) {
  if (act == GATE_GELU) {
    float2 e;
    const float2 er = gelu_math::erf_core2(g, e);
    const float2 cdf = __ffma2_rn(er, gelu_math::f2(0.5f), gelu_math::f2(0.5f));
    a = __fmul2_rn(g, cdf);
    da = __ffma2_rn(__fmul2_rn(g, gelu_math::f2(0.3989422804014327f)), e, cdf);
  } else {
    // 1 - s = e s, to its last bits however large g is; e stays finite for its product with 0
    const float2 x = __fmul2_rn(g, gelu_math::f2(-1.4426950408889634f));
    const float2 e = make_float2(gelu_math::ex2_approx(fminf(x.x, 126.0f)), gelu_math::ex2_approx(fminf(x.y, 126.0f)));
    const float2 d = __fadd2_rn(e, gelu_math::f2(1.0f));
    const float2 s = make_float2(gelu_math::rcp_approx(d.x), gelu_math::rcp_approx(d.y));
    a = __fmul2_rn(g, s);
    // s + a (1 - s)
    da = __ffma2_rn(a, __fmul2_rn(e, s), s);
  }
}

struct Params {
  const elem_t* bias;       // [2 inner], or null
  float* col_sums;          // backward: [rows / 32, upwards][2 inner] sums over 32 rows, or null
  int* status;
  int rows, inner, depth;   // depth: the products' K
  int act;
};

// BN: columns of the accumulator.  Forward: BN / 2 hidden columns, values then gates; backward: BN hidden columns.
template <int BN, bool PAIR, int MODE>
struct Smem {
  static constexpr int kABytes = BM * BK * 2;
  static constexpr int kBBytes = (PAIR ? BN / 2 : BN) * BK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // per epilogue warp, chunks of 32 rows x 32 columns: h twice | v, g in fp32 and h | v, g in fp32 and dv, dg
  static constexpr int kWarpStage = MODE == FORWARD ? 4096 : MODE == FORWARD_KEEP ? 10240 : 12288;
  static constexpr int kFixed = kEpiWarps * kWarpStage + 512 + 1024;
  static constexpr int kStages = (227 * 1024 - kFixed) / kStageBytes > 6 ? 6 : (227 * 1024 - kFixed) / kStageBytes;
  static constexpr int kTotal = kStages * kStageBytes + kFixed;
  static_assert(kStages >= 3, "");
};

// 32 fp32 values of this lane's row in the layout of CU_TENSOR_MAP_SWIZZLE_128B; the buffer is 1024-byte aligned.
__device__ __forceinline__ void put_row128(uint8_t* buffer, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  float4* row = reinterpret_cast<float4*>(buffer + lane * 128);
#pragma unroll
  for (int j = 0; j < 8; ++j) row[j ^ (lane & 7)] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
}
__device__ __forceinline__ void get_row128(const uint8_t* buffer, float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  const float4* row = reinterpret_cast<const float4*>(buffer + lane * 128);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float4 t = row[j ^ (lane & 7)];
    v[4 * j] = t.x; v[4 * j + 1] = t.y; v[4 * j + 2] = t.z; v[4 * j + 3] = t.w;
  }
}

// v += bias[n0 .. n0 + 32), of `left` columns that there are; the same addresses in all lanes
__device__ __forceinline__ void add_bias(float (&v)[32], const elem_t* bias, int left) {
  if (left >= 32 && (reinterpret_cast<uintptr_t>(bias) & 15) == 0) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint4 raw = __ldg(reinterpret_cast<const uint4*>(bias) + q);
      const elem2_t* h = reinterpret_cast<const elem2_t*>(&raw);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = e22ff(h[e]);
        v[8 * q + 2 * e] += f.x;
        v[8 * q + 2 * e + 1] += f.y;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < left) v[j] += e2f(bias[j]);
  }
}

// Tiles in panels of kPanel columns of tiles, row by row inside a panel: what runs at the same time then shares few rows of A
// and of B, which stay in L2 (8192 x 2048 x 8192, forward that keeps: 472 -> 401 us; without keeping 336 -> 318).
constexpr int kPanel = 16;
struct Tile { int m, n; };
__device__ __forceinline__ Tile tile_at(int t, int tiles_m, int tiles_n) {
  const int panel = t / (kPanel * tiles_m), in = t - panel * kPanel * tiles_m;
  const int width = min(kPanel, tiles_n - panel * kPanel);
  return {in / width, panel * kPanel + in % width};
}

// Forward: map_0 h, map_1 v, map_2 g (stores).  Backward: map_0 v, map_1 g (loads), map_2 dv, map_3 dg (stores).
template <int BN, bool PAIR, int MODE>
__device__ __forceinline__ void
gated_body(const CUtensorMap& map_a, const CUtensorMap& map_b, const CUtensorMap& map_0, const CUtensorMap& map_1,
           const CUtensorMap& map_2, const CUtensorMap& map_3, const Params& p) {
  using L = Smem<BN, PAIR, MODE>;
  constexpr bool kBack = MODE == BACKWARD;
  constexpr int kCols = kBack ? BN : BN / 2;           // hidden columns of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_stage = smem + L::kStages * L::kStageBytes;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(epi_stage + kEpiWarps * L::kWarpStage);
  uint64_t* empty_bar = full_bar + L::kStages;
  uint64_t* tmem_full = empty_bar + L::kStages;
  uint64_t* tmem_empty = tmem_full + 2;
  uint64_t* side_bar = tmem_empty + 2;                 // one for each epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(side_bar + kEpiWarps);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = PAIR ? (int)cluster_ctarank() : 0;  // 0 = leader
  const int first_tile = PAIR ? blockIdx.x / 2 : blockIdx.x, stride = PAIR ? gridDim.x / 2 : gridDim.x;
  constexpr int kTileRows = PAIR ? 2 * BM : BM;
  const int tiles_m = (p.rows + kTileRows - 1) / kTileRows, tiles_n = (p.inner + kCols - 1) / kCols;
  const int num_tiles = tiles_m * tiles_n, k_blocks = (p.depth + BK - 1) / BK;
  constexpr uint32_t kTmemCols = 2 * BN;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_b);
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tmem_full[a], 1);
      mbar_init(&tmem_empty[a], (PAIR ? 2 : 1) * kEpiWarps);
    }
    for (int w = 0; w < kEpiWarps; ++w) mbar_init(&side_bar[w], 1);
    mbar_fence_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc2(tmem_slot, kTmemCols);
      tmem_relinquish2();
    } else {
      tmem_alloc(tmem_slot, kTmemCols);
      tmem_relinquish();
    }
  }
  fence_before_sync();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();
  fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += stride) {
        const Tile at = tile_at(tile, tiles_m, tiles_n);
        const int row0 = at.m * kTileRows + rank * BM, n0 = at.n * kCols;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1)) { ok = false; break; }
          uint8_t* sa = smem + stage * L::kStageBytes;
          uint8_t* sb = sa + L::kABytes;
          if constexpr (PAIR) {
            const uint32_t bar = map_to_cta(smem_u32(&full_bar[stage]), 0);
            if (rank == 0) mbar_expect_tx(&full_bar[stage], 2 * L::kStageBytes);
            tma2_load_2d(sa, &map_a, bar, kb * BK, row0);
            if constexpr (kBack) {
#pragma unroll
              for (int j = 0; j < BN / 128; ++j)
                tma2_load_2d(sb + j * BK * 128, &map_b, bar, n0 + rank * (BN / 2) + j * 64, kb * BK);
            } else {
              tma2_load_2d(sb, &map_b, bar, kb * BK, rank * p.inner + n0);
            }
          } else {
            mbar_expect_tx(&full_bar[stage], L::kStageBytes);
            tma_load_2d(sa, &map_a, &full_bar[stage], kb * BK, row0);
            if constexpr (kBack) {
#pragma unroll
              for (int j = 0; j < BN / 64; ++j) tma_load_2d(sb + j * BK * 128, &map_b, &full_bar[stage], n0 + j * 64, kb * BK);
            } else {
              tma_load_2d(sb, &map_b, &full_bar[stage], kb * BK, n0);
              tma_load_2d(sb + kCols * 128, &map_b, &full_bar[stage], kb * BK, p.inner + n0);
            }
          }
          if (++stage == L::kStages) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) atomicExch(p.status, GEMM_ERR_PRODUCER_TIMEOUT);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (of a pair: the leader)
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = make_idesc_f16kind(PAIR ? 256 : 128, BN, false, kBack);
      constexpr uint32_t b_lbo = kBack ? BK * 128 : 16, b_kstep = kBack ? UMMA_K * 128 : UMMA_K * 2;
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += stride) {
        if (!mbar_wait(&tmem_empty[acc], acc_phase ^ 1)) { ok = false; break; }
        fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase)) { ok = false; break; }
          fence_after_sync();
          const uint32_t sa = smem_u32(smem + stage * L::kStageBytes), sb = sa + L::kABytes;
#pragma unroll
          for (int k = 0; k < BK / UMMA_K; ++k) {
            const uint64_t da = make_smem_desc_sw128(sa + k * UMMA_K * 2, 16, 1024);
            const uint64_t db = make_smem_desc_sw128(sb + k * b_kstep, b_lbo, 1024);
            if constexpr (PAIR) mma2_f16_ss(d_tmem, da, db, idesc, (kb | k) != 0);
            else mma_f16_ss(d_tmem, da, db, idesc, (kb | k) != 0);
          }
          if constexpr (PAIR) mma2_commit_both(&empty_bar[stage]);
          else mma_commit(&empty_bar[stage]);
          if (++stage == L::kStages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        if constexpr (PAIR) mma2_commit_both(&tmem_full[acc]);
        else mma_commit(&tmem_full[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1; }
      }
      if (!ok) atomicExch(p.status, GEMM_ERR_MMA_TIMEOUT);
    }
  } else {
    // ------------------------------------------------------------------ epilogue warps: 32 rows, every other run of columns
    const int lane_group = warp % 4, second = (warp - 2) / 4;
    constexpr int kShare = kCols >= 64 ? kCols / 2 : kCols;         // columns of a warp; of 32 the second warp has none
    const int c_first = second * kShare, c_last = c_first + kShare <= kCols ? c_first + kShare : c_first;
    uint8_t* buf_0 = epi_stage + (warp - 2) * L::kWarpStage;
    uint64_t* side = &side_bar[warp - 2];
    int acc = 0;
    uint32_t acc_phase = 0, side_phase = 0, turn = 0;
    bool ok = true;

    // backward: tile and column of the chunk whose v and g are fetched next; behind the last one it stays where it is
    int ahead_tile = first_tile, ahead_c = c_first;
    Tile ahead = tile_at(first_tile, tiles_m, tiles_n);
    auto fetch_next = [&]() {
      if constexpr (kBack) {
        while (ahead_c >= c_last || ahead.n * kCols + ahead_c >= p.inner) {
          ahead_tile += stride;
          if (ahead_tile >= num_tiles) return;
          ahead = tile_at(ahead_tile, tiles_m, tiles_n);
          ahead_c = c_first;
        }
        if (lane == 0) {
          const int x = ahead.n * kCols + ahead_c, y = ahead.m * kTileRows + rank * BM + lane_group * 32;
          mbar_expect_tx(side, 8192);
          tma_load_2d(buf_0, &map_0, side, x, y);
          tma_load_2d(buf_0 + 4096, &map_1, side, x, y);
        }
        ahead_c += 32;
      }
    };
    if (c_first < c_last) fetch_next();
    for (int tile = first_tile; tile < num_tiles && ok; tile += stride) {
      const Tile at = tile_at(tile, tiles_m, tiles_n);
      const int row0 = at.m * kTileRows + rank * BM + lane_group * 32, col0 = at.n * kCols;
      const bool box_in = row0 < p.rows;                            // else there is nothing to store
      if (!mbar_wait(&tmem_full[acc], acc_phase)) { ok = false; break; }
      fence_after_sync();
      const uint32_t taddr = tmem_base + (uint32_t(lane_group * 32) << 16) + acc * BN;
#pragma unroll 1
      for (int c = c_first; c < c_last; c += 32) {
        const int n0 = col0 + c;
        if (n0 >= p.inner) break;                                   // the same for the whole warp
        if constexpr (kBack) {
          if (!mbar_wait(side, side_phase)) { ok = false; break; }
          side_phase ^= 1;
          float v[32], g[32];
          get_row128(buf_0, v);
          get_row128(buf_0 + 4096, g);
          uint32_t r[32];
          tmem_ld_32x32(taddr + c, r);
          __syncwarp();
          fetch_next();
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float2 a, da;
            act_and_grad2(make_float2(g[j], g[j + 1]), p.act, a, da);
            const float2 dh = make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
            const float2 dg = __fmul2_rn(__fmul2_rn(dh, make_float2(v[j], v[j + 1])), da);
            const float2 dv = __fmul2_rn(dh, a);
            v[j] = dv.x; v[j + 1] = dv.y;
            g[j] = dg.x; g[j + 1] = dg.y;
          }
          if (lane == 0) bulk_wait_group_read<0>();
          __syncwarp();
          gemm_epi::stage_row64(buf_0 + 8192, v);
          gemm_epi::stage_row64(buf_0 + 10240, g);
          if (p.col_sums != nullptr && box_in) {                    // rows behind the end are 0
            float* sums = p.col_sums + (long long)(row0 / 32) * 2 * p.inner + n0;
            gemm_epi::segment_sums<32>(v, nullptr);
            gemm_epi::segment_sums<32>(g, nullptr);
            if (n0 + lane < p.inner) {
              sums[lane] = v[0];
              sums[p.inner + lane] = g[0];
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (box_in) {
              tma_store_2d(&map_2, buf_0 + 8192, n0, row0);
              tma_store_2d(&map_3, buf_0 + 10240, n0, row0);
            }
            bulk_commit_group();
          }
        } else {
          float v[32], g[32], h[32];
          {
            uint32_t rv[32], rg[32];
            tmem_ld_32x32(taddr + c, rv);
            tmem_ld_32x32(taddr + kCols + c, rg);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              v[j] = __uint_as_float(rv[j]);
              g[j] = __uint_as_float(rg[j]);
            }
          }
          if (p.bias != nullptr) {
            add_bias(v, p.bias + n0, p.inner - n0);
            add_bias(g, p.bias + p.inner + n0, p.inner - n0);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 t = __fmul2_rn(make_float2(v[j], v[j + 1]), act2(make_float2(g[j], g[j + 1]), p.act));
            h[j] = t.x;
            h[j + 1] = t.y;
          }
          uint8_t* out = MODE == FORWARD ? buf_0 + (turn++ & 1) * 2048 : buf_0 + 8192;
          if (lane == 0) {
            if constexpr (MODE == FORWARD) bulk_wait_group_read<1>();
            else bulk_wait_group_read<0>();
          }
          __syncwarp();
          gemm_epi::stage_row64(out, h);
          if constexpr (MODE == FORWARD_KEEP) {
            put_row128(buf_0, v);
            put_row128(buf_0 + 4096, g);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (box_in) {
              tma_store_2d(&map_0, out, n0, row0);
              if constexpr (MODE == FORWARD_KEEP) {
                tma_store_2d(&map_1, buf_0, n0, row0);
                tma_store_2d(&map_2, buf_0 + 4096, n0, row0);
              }
            }
            bulk_commit_group();
          }
        }
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (!PAIR || rank == 0) mbar_arrive(&tmem_empty[acc]);
        else remote_arrive(map_to_cta(smem_u32(&tmem_empty[acc]), 0));
      }
      if (++acc == 2) { acc = 0; acc_phase ^= 1; }
    }
    if (!ok && lane == 0) atomicExch(p.status, GEMM_ERR_EPILOGUE_TIMEOUT);
    if (lane == 0) bulk_wait_group_all();
  }

  fence_before_sync();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();              // neither CTA leaves while the other may still touch it
  if (warp == 1) {
    fence_after_sync();
    if constexpr (PAIR) tmem_dealloc2(tmem_base, kTmemCols);
    else tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// A few rows: the weights are streamed once, and a 128-row tile would be padding.  A CTA has 8 output columns (and, gated, the 8
// gate columns of the same hidden ones), its warps take runs of 32 along K in turn; mma.sync.m16n8k16 with the 8 columns as N and
// 16 rows as M.  The order of K inside a run does not matter to a product, so lane t of a quad takes K = 8 t .. 8 t + 7 of both
// operands: one 16-byte load feeds two instructions.
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32." ELEM_PTX "." ELEM_PTX ".f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct FewParams {
  const elem_t *x, *w, *bias, *residual;      // w: gated (2 cols, depth), else (cols, depth)
  elem_t* out;                                // [rows][cols] dense
  long long ldx, ldw, ldr;
  int rows, cols, depth, act;                 // depth: a multiple of 8; all rows of x and w on 16-byte boundaries
};

// The second product's CTAs start while the first one's still run, fetch their first weights and wait for its results there.
template <int MT, bool GATED>
__global__ void __launch_bounds__(GATED ? 256 : 512)
few_rows_kernel(const FewParams p) {
  constexpr int kB = GATED ? 2 : 1, kAhead = 4, kFewWarps = GATED ? 8 : 16;
  __shared__ float sums[kFewWarps][kB][MT][16][8];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = lane % 4, grp = lane / 4;
  const int n0 = blockIdx.x * 8, n = n0 + grp;
  const elem_t* w[kB];
#pragma unroll
  for (int i = 0; i < kB; ++i) w[i] = p.w + (long long)((n < p.cols ? n : p.cols - 1) + i * p.cols) * p.ldw;
  const elem_t* x[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = m * 16 + i * 8 + grp;
      x[m][i] = p.x + (long long)(row < p.rows ? row : p.rows - 1) * p.ldx;      // rows behind the last one are not stored
    }
  float acc[kB][MT][4] = {};
  if constexpr (GATED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  bool waited = GATED;
  for (int k0 = warp * 32; k0 < p.depth; k0 += kFewWarps * 32 * kAhead) {
    uint4 b[kAhead][kB];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int k = k0 + u * kFewWarps * 32 + quad * 8;
#pragma unroll
      for (int i = 0; i < kB; ++i)
        b[u][i] = k < p.depth ? __ldcs(reinterpret_cast<const uint4*>(w[i] + k)) : make_uint4(0, 0, 0, 0);
    }
    if (!waited) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      waited = true;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int k = k0 + u * kFewWarps * 32 + quad * 8;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint4 a[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          a[i] = k < p.depth ? *reinterpret_cast<const uint4*>(x[m][i] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kB; ++i) {
          mma_16x8x16(acc[i][m], a[0].x, a[1].x, a[0].y, a[1].y, b[u][i].x, b[u][i].y);
          mma_16x8x16(acc[i][m], a[0].z, a[1].z, a[0].w, a[1].w, b[u][i].z, b[u][i].w);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kB; ++i)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int q = 0; q < 4; ++q) sums[warp][i][m][grp + q / 2 * 8][quad * 2 + q % 2] = acc[i][m][q];
  if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");      // a warp without a part of K
  __syncthreads();
  for (int o = threadIdx.x; o < MT * 128; o += kFewWarps * 32) {
    const int row = o / 8, c = o % 8, col = n0 + c;
    if (row >= p.rows || col >= p.cols) continue;
    float s[kB] = {};
#pragma unroll
    for (int i = 0; i < kB; ++i) {
#pragma unroll
      for (int v = 0; v < kFewWarps; ++v) s[i] += sums[v][i][row / 16][row % 16][c];
      if (p.bias != nullptr) s[i] += e2f(p.bias[col + i * p.cols]);
    }
    if constexpr (GATED) s[0] *= act2(make_float2(s[1], 0.0f), p.act).x;
    else if (p.residual != nullptr) s[0] += e2f(p.residual[row * p.ldr + col]);
    p.out[(long long)row * p.cols + col] = f2e(s[0]);
  }
}

template <bool GATED>
int launch_few(const FewParams& p, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.cols + 7) / 8));
  cfg.blockDim = dim3(GATED ? 256 : 512);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = GATED ? 0 : 1;
  return cudaLaunchKernelEx(&cfg, p.rows <= 16 ? few_rows_kernel<1, GATED> : few_rows_kernel<2, GATED>, p) == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

template <int BN, int MODE>
__global__ void __launch_bounds__(kThreads, 1)
gated_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
             const __grid_constant__ CUtensorMap map_0, const __grid_constant__ CUtensorMap map_1,
             const __grid_constant__ CUtensorMap map_2, const __grid_constant__ CUtensorMap map_3, const Params p) {
  gated_body<BN, false, MODE>(map_a, map_b, map_0, map_1, map_2, map_3, p);
}
template <int BN, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
gated_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                  const __grid_constant__ CUtensorMap map_0, const __grid_constant__ CUtensorMap map_1,
                  const __grid_constant__ CUtensorMap map_2, const __grid_constant__ CUtensorMap map_3, const Params p) {
  gated_body<BN, true, MODE>(map_a, map_b, map_0, map_1, map_2, map_3, p);
}

// out[c] = sum over `parts` rows of part[r][c], in a fixed order: eight threads a column, every eighth row each.
__global__ void __launch_bounds__(256) add_sums_kernel(const float* __restrict__ part, elem_t* __restrict__ out, int parts, int cols) {
  __shared__ float sums[8][33];
  const int c = blockIdx.x * 32 + threadIdx.x % 32, r = threadIdx.x / 32;
  float sum = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int i = r; i < parts; i += 8) sum += part[(long long)i * cols + c];
  }
  sums[r][threadIdx.x % 32] = sum;
  __syncthreads();
  if (r == 0 && c < cols) {
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += sums[i][threadIdx.x];
    out[c] = f2e(sum);
  }
}

// rows x cols of pitch ld; fp32 in boxes of 32 x 32 with 128-byte swizzle, elements in boxes of box_rows x box_cols with
// box_cols * 2 bytes of swizzle
int encode(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld, int box_rows, int box_cols, bool fp32) {
  auto enc = fbam_encode_tiled();
  if (!enc) return GEMM_ERR_DRIVER;
  fbam_bind_context_to_thread();
  const int size = fp32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(base) & 15) || (ld * size) % 16) return GEMM_ERR_ALIGNMENT;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * size};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows}, ones[2] = {1, 1};
  const CUresult r = enc(map, fp32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : ELEM_TMAP, 2, const_cast<void*>(base), dims, strides, box, ones,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, box_cols * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) g_fbam_last_driver_error = (int)r;
  return r == CUDA_SUCCESS ? 0 : GEMM_ERR_TENSORMAP;
}

template <typename K>
int launch(K kernel, int smem, bool pair, long long tiles, const CUtensorMap (&m)[6], const Params& p, cudaStream_t s) {
  static int sms = 0;
  if (sms == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  }
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return GEMM_ERR_LAUNCH;
  const int usable = sms - g_fbam_reserved_sms > 2 ? sms - g_fbam_reserved_sms : 2;
  const long long slots = pair ? usable / 2 : usable, blocks = (tiles < slots ? tiles : slots) * (pair ? 2 : 1);
  kernel<<<(unsigned)blocks, kThreads, smem, s>>>(m[0], m[1], m[2], m[3], m[4], m[5], p);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

long long tiles_of(int rows, int tile_rows, int cols, int tile_cols) {
  return (long long)((rows + tile_rows - 1) / tile_rows) * ((cols + tile_cols - 1) / tile_cols);
}

// Accumulator width and pairing: 0: single CTAs with 64 columns, 1: with 128, 2: pairs with 256.  Pairs where their tiles reach
// every SM; below that the wider tile that still does.  us of the whole block's forward, 64 | 128 | pairs: 8192 x 1024 x 4096
// 261 | 179 | 146, 2048 x 1024 x 4096 83 | 63 | 58, 1001 x 1000 x 2736 54 | 48 | 44, 300 x 1024 x 4096 38 | 36 | 36, 64 x 1024 x
// 4096 30 | 32 | 34.  `pairs` below 0: by this rule, 0: never, 1: always.
int pick(int rows, int inner, bool back, int pairs) {
  const int h = back ? 2 : 1;
  if (pairs < 0 ? tiles_of(rows, 256, inner, 128 * h) >= 74 : pairs > 0) return 2;
  return tiles_of(rows, 128, inner, 64 * h) >= 148 ? 1 : 0;
}

template <int MODE>
int run(int which, int rows, int inner, const CUtensorMap (&m)[6], const Params& p, cudaStream_t s) {
  constexpr int h = MODE == BACKWARD ? 2 : 1;
  if (which == 2)
    return launch(gated_pair_kernel<256, MODE>, Smem<256, true, MODE>::kTotal, true, tiles_of(rows, 256, inner, 128 * h), m, p, s);
  if (which == 1)
    return launch(gated_kernel<128, MODE>, Smem<128, false, MODE>::kTotal, false, tiles_of(rows, 128, inner, 64 * h), m, p, s);
  return launch(gated_kernel<64, MODE>, Smem<64, false, MODE>::kTotal, false, tiles_of(rows, 128, inner, 32 * h), m, p, s);
}

}  // namespace

// x (rows, depth) pitch ldx, w_in (2 inner, depth) pitch ldw, bias (2 inner) elements or null -> h (rows, inner) dense and, where v
// is not null, v and g (rows, inner) dense fp32.  inner is a multiple of 8, all rows start on 16-byte boundaries.
extern "C" int fbam_gated_fwd(const void* x, long long ldx, const void* w_in, long long ldw, const void* bias, void* h, float* v,
                              float* g, int rows, int inner, int depth, int act, int pairs, int* status, void* stream) {
  if (rows <= 0 || inner <= 0 || depth <= 0 || inner % 8 != 0 || inner > 0x3fffffff || act < 0 || act > 1 || (v == nullptr) != (g == nullptr))
    return GEMM_ERR_SHAPE;
  const int which = pick(rows, inner, false, pairs), box = which == 2 ? 128 : which == 1 ? 64 : 32;
  CUtensorMap m[6];
  int e = encode(&m[0], x, rows, depth, ldx, BM, BK, false);
  if (!e) e = encode(&m[1], w_in, 2ll * inner, depth, ldw, box, BK, false);
  if (!e) e = encode(&m[2], h, rows, inner, inner, 32, 32, false);
  if (!e && v) e = encode(&m[3], v, rows, inner, inner, 32, 32, true);
  if (!e && v) e = encode(&m[4], g, rows, inner, inner, 32, 32, true);
  if (e) return e;
  if (!v) m[3] = m[4] = m[2];
  m[5] = m[2];
  const Params p{(const elem_t*)bias, nullptr, status, rows, inner, depth, act};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return v ? run<FORWARD_KEEP>(which, rows, inner, m, p, s) : run<FORWARD>(which, rows, inner, m, p, s);
}

// dy (rows, depth) pitch ldy, w_out (depth, inner) pitch ldw, v and g as the forward left them -> d_vg (rows, 2 inner) dense, and
// where col_sums is not null its column sums in db (2 inner) elements; col_sums is the workspace, 2 inner fp32 values for every 32 rows.
extern "C" int fbam_gated_bwd(const void* dy, long long ldy, const void* w_out, long long ldw, const float* v, const float* g, void* d_vg,
                              float* col_sums, void* db, int rows, int inner, int depth, int act, int pairs, int* status, void* stream) {
  if (rows <= 0 || inner <= 0 || depth <= 0 || inner % 8 != 0 || inner > 0x3fffffff || act < 0 || act > 1 ||
      (col_sums == nullptr) != (db == nullptr))
    return GEMM_ERR_SHAPE;
  CUtensorMap m[6];
  int e = encode(&m[0], dy, rows, depth, ldy, BM, BK, false);
  if (!e) e = encode(&m[1], w_out, depth, inner, ldw, BK, 64, false);
  if (!e) e = encode(&m[2], v, rows, inner, inner, 32, 32, true);
  if (!e) e = encode(&m[3], g, rows, inner, inner, 32, 32, true);
  if (!e) e = encode(&m[4], d_vg, rows, inner, 2ll * inner, 32, 32, false);
  if (!e) e = encode(&m[5], (elem_t*)d_vg + inner, rows, inner, 2ll * inner, 32, 32, false);
  if (e) return e;
  const Params p{nullptr, col_sums, status, rows, inner, depth, act};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  e = run<BACKWARD>(pick(rows, inner, true, pairs), rows, inner, m, p, s);
  if (e || db == nullptr) return e;
  add_sums_kernel<<<(2 * inner + 31) / 32, 256, 0, s>>>(col_sums, (elem_t*)db, (rows + 31) / 32, 2 * inner);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

// Up to 32 rows, the whole block: x (rows, depth) pitch ldx -> h (rows, inner), a workspace, -> y (rows, out_dim), both dense.
// depth and inner are multiples of 8; rows of x, w_in and w_out start on 16-byte boundaries; biases and residual may be null.
extern "C" int fbam_gated_few_rows(const void* x, long long ldx, const void* w_in, long long ld_in, const void* b_in, const void* w_out,
                                   long long ld_out, const void* b_out, const void* residual, long long ldr, void* h, void* y, int rows,
                                   int depth, int inner, int out_dim, int act, void* stream) {
  if (rows <= 0 || rows > 32 || depth <= 0 || inner <= 0 || out_dim <= 0 || depth % 8 || inner % 8 || inner > 0x3fffffff || act < 0 || act > 1)
    return GEMM_ERR_SHAPE;
  if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w_in) | reinterpret_cast<uintptr_t>(w_out) | reinterpret_cast<uintptr_t>(h)) & 15) ||
      ((ldx | ld_in | ld_out) & 7))
    return GEMM_ERR_ALIGNMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int e = launch_few<true>({(const elem_t*)x, (const elem_t*)w_in, (const elem_t*)b_in, nullptr, (elem_t*)h, ldx, ld_in, 0, rows,
                                  inner, depth, act}, s);
  if (e) return e;
  return launch_few<false>({(const elem_t*)h, (const elem_t*)w_out, (const elem_t*)b_out, (const elem_t*)residual, (elem_t*)y, inner,
                            ld_out, ldr, rows, out_dim, inner, act}, s);
}

extern "C" int fbam_product(const void* A, long long lda, int a_mn_major, const void* B, long long ldb, int b_mn_major, int M, int N,
                            int K, void* D, long long ldd, const void* bias, const void* residual, long long ldr, float* slabs,
                            int splits, int* status, void* stream);                                  // gemm_tcgen05.cu
extern "C" int fbam_colsum_to(const void* x, const void* z, void* dz, void* out, int out_elem, float* work, long long rows, int cols,
                              void* stream);                                                         // kernels_simt.cu

// The block's forward: fbam_gated_fwd, and where y is not null y (rows, out_dim) = h W_outᵀ + b_out + residual, dense.  `pairs`, here and
// in the backward: whether the fused product runs on pairs of CTAs, below 0 by its size, 0 never, 1 always.
extern "C" int fbam_gated_block_fwd(const void* x, long long ldx, const void* w_in, long long ld_in, const void* b_in, const void* w_out,
                                    long long ld_out, const void* b_out, const void* residual, void* h, float* v, float* g, void* y,
                                    int rows, int inner, int depth, int out_dim, int act, int pairs, int* status, void* stream) {
  const int e = fbam_gated_fwd(x, ldx, w_in, ld_in, b_in, h, v, g, rows, inner, depth, act, pairs, status, stream);
  if (e || y == nullptr) return e;
  return fbam_product(h, inner, 0, w_out, ld_out, 0, rows, out_dim, inner, y, out_dim, b_out, residual, out_dim, nullptr, 0, status, stream);
}

// The block's backward; a gradient whose pointer is null is not wanted.  slabs: [splits][..] fp32 for a weight gradient
// that is split along the rows.  d_b_out: out_dim rounded up to 8, dy then dense and that wide; col_work as fbam_colsum_partials says.
extern "C" int fbam_gated_block_bwd(const void* dy, long long ldy, const void* x, long long ldx, const void* w_in, long long ld_in,
                                    const void* w_out, long long ld_out, const float* v, const float* g, const void* h, void* d_vg,
                                    float* col_sums, void* d_b_in, void* dx, void* d_w_in, void* d_w_out, void* d_b_out, float* col_work,
                                    float* slabs_in, int splits_in, float* slabs_out, int splits_out, int rows, int inner, int depth,
                                    int out_dim, int act, int pairs, int* status, void* stream) {
  int e = 0;
  if (d_vg != nullptr)
    e = fbam_gated_bwd(dy, ldy, w_out, ld_out, v, g, d_vg, col_sums, d_b_in, rows, inner, out_dim, act, pairs, status, stream);
  if (!e && dx != nullptr)
    e = fbam_product(d_vg, 2ll * inner, 0, w_in, ld_in, 1, rows, depth, 2 * inner, dx, depth, nullptr, nullptr, 0, nullptr, 0, status, stream);
  if (!e && d_w_in != nullptr)
    e = fbam_product(d_vg, 2ll * inner, 1, x, ldx, 1, 2 * inner, depth, rows, d_w_in, depth, nullptr, nullptr, 0, slabs_in, splits_in, status,
                     stream);
  if (!e && d_w_out != nullptr)
    e = fbam_product(dy, ldy, 1, h, inner, 1, out_dim, inner, rows, d_w_out, inner, nullptr, nullptr, 0, slabs_out, splits_out, status,
                     stream);
  if (!e && d_b_out != nullptr) e = fbam_colsum_to(dy, nullptr, nullptr, d_b_out, 1, col_work, rows, (out_dim + 7) / 8 * 8, stream);
  return e;
}

namespace {
// U: elements a thread moves at once
template <int U>
__global__ void __launch_bounds__(256)
refit_kernel(const elem_t* __restrict__ src, uint32_t ld, elem_t* __restrict__ dst, uint32_t src_rows, uint32_t src_cols, uint32_t dst_rows,
             uint32_t dst_cols, uint32_t units) {
  struct alignas(2 * U) Unit { elem_t e[U]; };
  constexpr int kAhead = 4;
  const uint32_t across = dst_cols / U, step = gridDim.x * 256;
  for (uint32_t i0 = blockIdx.x * 256 + threadIdx.x; i0 < units; i0 += kAhead * step) {
    Unit x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint32_t i = i0 + k * step, row = i / across, c = (i - row * across) * U, block = row / dst_rows, r = row - block * dst_rows;
#pragma unroll
      for (int j = 0; j < U; ++j) x[k].e[j] = f2e(0.0f);
      if (i < units && r < src_rows && c < src_cols)
        x[k] = *reinterpret_cast<const Unit*>(src + (long long)(block * src_rows + r) * ld + c);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint32_t i = i0 + k * step;
      if (i < units) *reinterpret_cast<Unit*>(dst + (long long)i * U) = x[k];
    }
  }
}
}  // namespace

// blocks of src_rows x src_cols (pitch ld) -> dense blocks of dst_rows x dst_cols: padded with zeros, or cut.  In pieces of 16, 8, 4
// or 2 bytes, whichever all rows begin and end on: 5460 rows of 1000 bf16 to 5472 in
// 6.4 us, 1000 of 2730 to 2736 in 6.5 (element by element, with a division of 64 bits for each, 24 and 14).
extern "C" int fbam_refit(const void* src, long long ld, void* dst, int blocks, int src_rows, int src_cols, int dst_rows, int dst_cols,
                          void* stream) {
  if (blocks <= 0 || src_rows < 0 || src_cols < 0 || dst_rows <= 0 || dst_cols <= 0 || ld < 0 || ld > 0x7fffffff ||
      (long long)blocks * src_rows > 0x7fffffff)
    return GEMM_ERR_SHAPE;
  const uintptr_t odd = reinterpret_cast<uintptr_t>(src) / 2 | reinterpret_cast<uintptr_t>(dst) / 2 | (uintptr_t)ld | src_cols | dst_cols;
  auto part = [&](auto kernel, int u, const elem_t* from, elem_t* to, long long count, int from_rows, int to_rows) {
    const long long units = count * to_rows * dst_cols / u, need = (units + 1023) / 1024;
    kernel<<<(unsigned)(need < 148 * 8 ? need : 148 * 8), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        from, (uint32_t)ld, to, from_rows, src_cols, to_rows, dst_cols, (uint32_t)units);
  };
  // The kernel counts in 32 bits: blocks one by one, and a block in runs of rows, where there are more values than that.
  constexpr long long kMost = 1ll << 31;
  auto go = [&](auto kernel, int u) {
    const elem_t* from = (const elem_t*)src;
    elem_t* to = (elem_t*)dst;
    if ((long long)blocks * dst_rows * dst_cols <= kMost) return part(kernel, u, from, to, blocks, src_rows, dst_rows);
    const int run = (int)(kMost / dst_cols);
    for (int b = 0; b < blocks; ++b)
      for (long long r = 0; r < dst_rows; r += run) {
        const long long left = src_rows - r, rows = dst_rows - r < run ? dst_rows - r : run;
        part(kernel, u, from + (b * (long long)src_rows + r) * ld, to + (b * (long long)dst_rows + r) * dst_cols, 1,
             (int)(left < 0 ? 0 : left < rows ? left : rows), (int)rows);
      }
  };
  if (odd % 8 == 0) go(refit_kernel<8>, 8);
  else if (odd % 4 == 0) go(refit_kernel<4>, 4);
  else if (odd % 2 == 0) go(refit_kernel<2>, 2);
  else go(refit_kernel<1>, 1);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}
