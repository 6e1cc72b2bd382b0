// Backward of the attention over a sliding window and the first tokens (forward and definition in window_attention.cu).
//
//   P = 2^(S scale log2(e) - lse),  dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta) scale,  dQ = dS K,  dK = dS^T Q,
//   delta = rowsum(dO O)
//
// One thread block owns 128 keys of a key head and walks the tiles of queries that see any of them; a tile's 128 rows are tokens x
// the query heads that share the key head, so dK and dV, which sum over those heads, are summed in tensor memory.  Five tcgen05
// products a tile; roles and barriers as in the backward of the plain causal kernel:
//   warp 21     TMA: K, V once; Q two tiles deep; dO two deep (D = 64) or one (D = 128: shared memory is full)
//   warp 20     MMA issue: S(i+1), dV(i) once P(i) is stored, then dP(i+1), dQ(i), dK(i) (D = 64) or dQ(i), dK(i), dP(i+1)
//               (D = 128, where dQ borrows dP's columns) once dS(i) is stored
//   warps 4-19  point-wise: four threads per row, 32 keys each
//   warps 0-3   add dQ to its tile's sum
//
// dQ of a tile is a sum over the key blocks that it sees.  They add to it in one fixed order, so that the result does not depend on
// which block runs when: the blocks of the first tokens, then the others from the last one down.  The first one stores, those between
// add, the last one adds and writes the rounded gradient, so there is neither a zero fill nor a pass behind the kernel.  Each tile
// has a counter per draining warp; a warp waits until the contributions before its own are in.  Blocks start in an order (a ticket)
// in which every contribution waits for earlier tickets only, so a wait always ends; and each walks its tiles so that it meets a
// tile one step after the block in front of it did: the blocks of the first tokens from the last tile back, the others from their
// first tile on.
#include "attention_tile.cuh"

namespace {

using namespace tc05;
using namespace attn;

constexpr int kRows = 128, kKeys = 128, kNoWindow = 0x3fffffff;
enum { ATT_ERR_TIMEOUT = 501 };

struct BwdParams {
  int T, B, kv_heads, group, tile_tokens, tiles;
  int window, sinks;
  const int* lengths;    // (B) or null
  float scale_log2, scale;
  const float* lse;      // (B, kv_heads, T, group), log2
  const float* delta;    // the same
  float4* sums;          // (B, kv_heads, tile, D / 4, 128) fp32: written before it is read
  int* counters;         // (B, kv_heads, tile, 4): contributions that are in; zeroed
  int* ticket;           // zeroed
  elem_t* dq;
  elem_t* dk;
  elem_t* dv;
  long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  int* status;
};

// delta, and what else has to be there before the main kernel: counters at zero, dQ of the rows behind a sequence's end.
template <int D>
__global__ void __launch_bounds__(256) window_delta_kernel(const elem_t* __restrict__ o, const elem_t* __restrict__ d_o, long long do_sb,
                                                           long long do_st, long long do_sh, float* __restrict__ delta, int* counters,
                                                           int n_counters, const BwdParams p) {
  constexpr int kLanes = D / 8;
  const long long thread = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (thread < n_counters) counters[thread] = 0;
  const int heads = p.kv_heads * p.group;
  const long long idx = thread / kLanes;                     // (b, t, h) row
  const int part = threadIdx.x % kLanes;
  const bool on = idx < (long long)p.B * p.T * heads;
  float s = 0.0f;
  const int h = (int)(idx % heads);
  const long long bt = idx / heads;
  const int t = (int)(bt % p.T), b = (int)(bt / p.T);
  bool there = on;
  if (on) {
    there = p.lengths == nullptr || t < p.lengths[b];
    if (there) {
      const uint4 ov = *reinterpret_cast<const uint4*>(o + idx * D + part * 8);
      const uint4 gv = *reinterpret_cast<const uint4*>(d_o + b * do_sb + t * do_st + h * do_sh + part * 8);
      const elem2_t* oe = reinterpret_cast<const elem2_t*>(&ov);
      const elem2_t* ge = reinterpret_cast<const elem2_t*>(&gv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = e22ff(oe[i]), y = e22ff(ge[i]);
        s += x.x * y.x + x.y * y.y;
      }
    } else {
      *reinterpret_cast<uint4*>(p.dq + b * p.q_sb + t * p.q_st + h * p.q_sh + part * 8) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
#pragma unroll
  for (int off = kLanes / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if (there && part == 0) delta[(((long long)b * p.kv_heads + h / p.group) * p.T + t) * p.group + h % p.group] = s;
}

constexpr int kBwdWarps = 22, kBwdThreads = kBwdWarps * 32;
template <int D>
constexpr int kDoStages = D == 64 ? 2 : 1;
template <int D>
constexpr int kPBuffers = D == 64 ? 2 : 1;
template <int D>
constexpr int bwd_smem_bytes() { return (4 + kDoStages<D>) * 128 * D * 2 + (1 + kPBuffers<D>) * 128 * 128 * 2 + 256 + 1024; }

__device__ __forceinline__ int load_acquire(const int* at) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
  return v;
}
__device__ __forceinline__ void store_release(int* at, int v) {
  asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(at), "r"(v) : "memory");
}

template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
window_bwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do,
                  const __grid_constant__ BwdParams p) {
  constexpr int DP = D / 64;
  constexpr int kTile = 128 * D * 2;           // a 128-row x D operand tile
  constexpr int kSq = 128 * 128 * 2;           // P / dS tiles
  constexpr int DOS = kDoStages<D>, PB = kPBuffers<D>;
  constexpr bool kOwnDq = D == 64;             // dQ has tensor-memory columns of its own
  constexpr uint32_t kTmemCols = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + kTile;
  uint8_t* sQ = sV + kTile;                    // two stages
  uint8_t* sDO = sQ + 2 * kTile;               // DOS stages
  uint8_t* sP = sDO + DOS * kTile;
  uint8_t* sDS = sP + PB * kSq;                // P: PB buffers
  uint64_t* bars = reinterpret_cast<uint64_t*>(sDS + kSq);
  uint64_t* kv_full = bars;
  uint64_t* q_full = bars + 1;      // [2]
  uint64_t* do_full = bars + 3;     // [2]
  uint64_t* q_free = bars + 5;      // [2] dK(i) has read the stage
  uint64_t* do_free = bars + 7;     // [2] dV(i) has read the stage
  uint64_t* s_full = bars + 9;      // S(i) in tensor memory
  uint64_t* dp_full = bars + 10;    // dP(i) in tensor memory
  uint64_t* p_ready = bars + 11;    // P(i) stored, S(i) read (16 warps)
  uint64_t* ds_ready = bars + 12;   // dS(i) stored, dP(i) read (16 warps)
  uint64_t* dv_done = bars + 13;    // [2] dV(i) has read the P buffer
  uint64_t* dq_full = bars + 15;    // dQ(i) in tensor memory
  uint64_t* dq_read = bars + 16;    // dQ(i) drained (4 warps)
  uint64_t* dk_done = bars + 17;    // dQ(i) and dK(i) have read dS; all products so far are complete
  uint64_t* kv_clean = bars + 18;   // K and V rows behind the sequence's end are zeros (16 warps)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 19);
  int* my_ticket = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    *my_ticket = atomicAdd(p.ticket, 1);
    prefetch_tensormap(&map_q); prefetch_tensormap(&map_k); prefetch_tensormap(&map_v); prefetch_tensormap(&map_do);
    for (int i = 0; i < 19; ++i) mbar_init(&bars[i], i == 11 || i == 12 || i == 18 ? 16 : i == 16 ? 4 : 1);
    mbar_fence_init();
  }
  __syncthreads();
  const int ticket = *my_ticket;
  const int bhs = p.B * p.kv_heads, nkb = (p.T + kKeys - 1) / kKeys;
  const int ns = min((p.sinks + kKeys - 1) / kKeys, nkb);          // blocks of first tokens
  const int nth = ticket / bhs, bh = ticket % bhs;
  const int kb = nth < ns ? nth : nkb - 1 - (nth - ns);
  const int b = bh / p.kv_heads, kvh = bh % p.kv_heads;
  const int k0 = kb * kKeys;
  const int len = p.lengths == nullptr ? p.T : min(max(p.lengths[b], 0), p.T);
  const bool first_block = kb < ns;
  const int m_lo = k0 / p.tile_tokens, tok_end = first_block ? len : min(len, k0 + kKeys - 1 + p.window);
  const int m_hi = (tok_end + p.tile_tokens - 1) / p.tile_tokens;
  const int n = k0 < len ? m_hi - m_lo : 0;                        // tiles that see the block
  auto tile_of = [&](int i) { return first_block ? m_hi - 1 - i : m_lo + i; };
  if (n <= 0) {                                                    // keys behind the sequence's end
    for (int i = threadIdx.x; i < kKeys * (D / 8) * 2; i += kBwdThreads) {
      const int which = i & 1, r = (i >> 1) / (D / 8), d = (i >> 1) % (D / 8) * 8;
      if (k0 + r < p.T) {
        elem_t* at = which ? p.dv + b * p.v_sb + (long long)(k0 + r) * p.v_st + kvh * p.v_sh
                           : p.dk + b * p.k_sb + (long long)(k0 + r) * p.k_st + kvh * p.k_sh;
        *reinterpret_cast<uint4*>(at + d) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    return;
  }
  const int used = p.tile_tokens * p.group;                        // rows of a tile
  if (used < kRows) {
    // the copies never write the rows behind them; they are operands of the transposed products
    const int rows = kRows - used, per = (2 + DOS) * DP * rows * 8;
    for (int i = threadIdx.x; i < per; i += kBwdThreads) {
      const int chunk = i & 7, r = used + (i >> 3) % rows, panel = (i >> 3) / rows;    // Q stages and dO stages lie in a row
      *reinterpret_cast<uint4*>(sQ + panel * 128 * 128 + r * 128 + chunk * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
  }
  if (warp == 20) { tmem_alloc(tmem_slot, kTmemCols); tmem_relinquish(); }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tm_s = tmem, tm_dp = tmem + 128, tm_dv = tmem + 256, tm_dk = tmem + 256 + D;
  const uint32_t tm_dq = kOwnDq ? tmem + 256 + 2 * D : tm_dp;

  if (warp == 21) {
    if (elect_one()) {
      bool ok = true;
      auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int t) {
#pragma unroll
        for (int j = 0; j < DP; ++j) tma_load_4d(dst + j * 128 * 128, map, bar, j * 64, head, t, b);
      };
      auto load_q = [&](int i) {
        if (i >= 2 && !mbar_wait(&q_free[i & 1], ((i >> 1) - 1) & 1)) { ok = false; return; }
        mbar_expect_tx(&q_full[i & 1], used * D * 2);
        load(sQ + (i & 1) * kTile, &map_q, &q_full[i & 1], kvh * p.group, tile_of(i) * p.tile_tokens);
      };
      auto load_do = [&](int i) {
        const int s = i % DOS;
        if (i >= DOS && !mbar_wait(&do_free[s], (i / DOS - 1) & 1)) { ok = false; return; }
        mbar_expect_tx(&do_full[s], used * D * 2);
        load(sDO + s * kTile, &map_do, &do_full[s], kvh * p.group, tile_of(i) * p.tile_tokens);
      };
      mbar_expect_tx(kv_full, 2 * kTile);
      load(sK, &map_k, kv_full, kvh, k0);
      load_q(0);
      load(sV, &map_v, kv_full, kvh, k0);
      load_do(0);
      if (n > 1) load_q(1);
      for (int i = 1; i < n && ok; ++i) {
        load_do(i);
        if (ok && i + 1 < n) load_q(i + 1);
      }
      if (!ok) atomicExch(p.status, ATT_ERR_TIMEOUT);
    }
  } else if (warp == 20) {
    if (elect_one()) {
      bool ok = true;
      const uint32_t id_s = make_idesc_f16kind(128, 128, false, false);   // S = Q K^T, dP = dO V^T
      const uint32_t id_t = make_idesc_f16kind(128, D, true, true);       // dV = P^T dO, dK = dS^T Q (A, B MN-major)
      const uint32_t id_q = make_idesc_f16kind(128, D, false, true);      // dQ = dS K (B MN-major)
      const uint32_t aK = smem_u32(sK), aV = smem_u32(sV), aP = smem_u32(sP), aDS = smem_u32(sDS);
      auto scores = [&](uint32_t d, uint32_t a, uint32_t bb) {            // both operands K-major over D
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k / 4) * 128 * 128 + (k % 4) * 32;
          mma_f16_ss(d, make_smem_desc_sw128(a + off, 16, 1024), make_smem_desc_sw128(bb + off, 16, 1024), id_s, k != 0);
        }
      };
      auto transposed = [&](uint32_t d, uint32_t a, uint32_t bb, bool first) {
        // K dimension = queries, 16 rows per step.  A (P or dS) is [query rows][keys]: as an MN-major operand its M = keys
#pragma unroll
        for (int k = 0; k < 128 / 16; ++k)
          mma_f16_ss(d, make_smem_desc_sw128(a + k * 16 * 128, 128 * 128, 1024),
                     make_smem_desc_sw128(bb + k * 16 * 128, 128 * 128, 1024), id_t, !first || k != 0);
      };
      auto issue_s = [&](int i) {
        if (!mbar_wait(&q_full[i & 1], (i >> 1) & 1)) { ok = false; return; }
        fence_after_sync();
        scores(tm_s, smem_u32(sQ + (i & 1) * kTile), aK);
        mma_commit(s_full);
      };
      auto issue_dp = [&](int i) {
        if (!mbar_wait(&do_full[i % DOS], (i / DOS) & 1)) { ok = false; return; }
        fence_after_sync();
        scores(tm_dp, smem_u32(sDO + (i % DOS) * kTile), aV);
        mma_commit(dp_full);
      };
      ok = mbar_wait(kv_full, 0) && mbar_wait(kv_clean, 0);
      if (ok) issue_s(0);
      if (ok) issue_dp(0);
      for (int i = 0; i < n && ok; ++i) {
        if (!mbar_wait(p_ready, i & 1)) { ok = false; break; }
        fence_after_sync();
        if (i + 1 < n) issue_s(i + 1);
        if (!ok) break;
        transposed(tm_dv, aP + (i % PB) * kSq, smem_u32(sDO + (i % DOS) * kTile), i == 0);
        mma_commit(&dv_done[i % PB]);
        mma_commit(&do_free[i % DOS]);
        if (!mbar_wait(ds_ready, i & 1)) { ok = false; break; }
        fence_after_sync();
        if (kOwnDq) {
          if (i + 1 < n) issue_dp(i + 1);
          if (!ok || (i > 0 && !mbar_wait(dq_read, (i - 1) & 1))) { ok = false; break; }
          fence_after_sync();
        }
#pragma unroll
        for (int k = 0; k < 128 / 16; ++k) {   // dQ = dS (K-major over keys) · K (MN-major: key rows, D contiguous)
          const uint64_t a_ds = make_smem_desc_sw128(aDS + (k / 4) * 128 * 128 + (k % 4) * 32, 16, 1024);
          const uint64_t b_k = make_smem_desc_sw128(aK + k * 16 * 128, 128 * 128, 1024);
          mma_f16_ss(tm_dq, a_ds, b_k, id_q, k != 0);
        }
        mma_commit(dq_full);
        transposed(tm_dk, aDS, smem_u32(sQ + (i & 1) * kTile), i == 0);
        mma_commit(dk_done);
        mma_commit(&q_free[i & 1]);
        if (!kOwnDq && i + 1 < n) {
          if (!mbar_wait(dq_read, i & 1)) { ok = false; break; }
          fence_after_sync();
          issue_dp(i + 1);
        }
      }
      if (!ok) atomicExch(p.status, ATT_ERR_TIMEOUT);
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- point-wise: one row, 32 keys per thread
    const int lane_group = warp & 3, part = (warp - 4) >> 2;
    const int row = lane_group * 32 + lane;
    const int token = row / p.group;                 // tile_tokens or more: no row
    const uint32_t lane_addr = uint32_t(lane_group * 32) << 16;
    const long long stat0 = (long long)bh * p.T * p.group;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
    uint8_t* pRow = sP + (part >> 1) * 128 * 128;      // the 64-key panel
    uint8_t* dsRow = sDS + (part >> 1) * 128 * 128;
    const int chunk0 = (part & 1) * 4;                 // first 16-byte piece of the panel row
    bool ok = true;
    if (k0 + kKeys > len && len < p.T) {
      // K and V behind the sequence's end may hold anything: 0 x NaN is NaN in the products over keys
      ok = mbar_wait(kv_full, 0);
      if (ok && k0 + row >= len) {
#pragma unroll
        for (int j = part; j < DP * 8; j += 4) {
          const int at = (j / 8) * 128 * 128 + row * 128 + (j % 8) * 16;
          *reinterpret_cast<uint4*>(sK + at) = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(sV + at) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      fence_proxy_async_smem();
    }
    warp_arrive(kv_clean);
    float lse_next = 0.0f, dl_next = 0.0f;             // statistics of the next tile: fetched one tile ahead
    auto fetch = [&](int i) {
      const int t = tile_of(i) * p.tile_tokens + token;
      if (i < n && token < p.tile_tokens && t < len) {
        const long long at = stat0 + (long long)t * p.group + (row - token * p.group);
        lse_next = p.lse[at];
        dl_next = p.delta[at];
      } else {
        lse_next = dl_next = 0.0f;
      }
    };
    fetch(0);
    for (int i = 0; i < n && ok; ++i) {
      const int t0 = tile_of(i) * p.tile_tokens, t_q = t0 + token;
      const bool row_ok = token < p.tile_tokens && t_q < len;
      const float nl = -lse_next, dl = dl_next;
      fetch(i + 1);
      const float2 nl2 = make_float2(nl, nl);
      // which of its 32 keys the row sees
      uint32_t seen = 0xffffffffu;
      if (k0 + kKeys - 1 > t0 || (k0 <= t0 + p.tile_tokens - 1 - p.window && k0 + kKeys > p.sinks) || t0 + p.tile_tokens > len ||
          used < kRows) {
        const int kk = k0 + part * 32;
        auto below = [](int c) { return c <= 0 ? 0u : c >= 32 ? 0xffffffffu : (1u << c) - 1u; };
        seen = row_ok ? below(t_q + 1 - kk) & (~below(t_q - p.window + 1 - kk) | below(p.sinks - kk)) : 0u;
      }
      if (!mbar_wait(s_full, i & 1)) { ok = false; break; }
      fence_after_sync();
      if (t0 + p.tile_tokens > len && len < p.T) {
        // Q and dO behind the sequence's end, operands of the products over queries.  S(i) has read Q; dP(i) may be reading dO, but
        // only rows whose dS is set to zero below.
        if (!mbar_wait(&do_full[i % DOS], (i / DOS) & 1)) { ok = false; break; }
        if (!row_ok) {
#pragma unroll
          for (int j = part; j < DP * 8; j += 4) {
            const int at = (j / 8) * 128 * 128 + row * 128 + (j % 8) * 16;
            *reinterpret_cast<uint4*>(sQ + (i & 1) * kTile + at) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(sDO + (i % DOS) * kTile + at) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
      }
      uint32_t r[32];
      float pr[32];
      tmem_ld_32x32(tm_s + lane_addr + part * 32, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; j += 2) {
        const float2 e = __ffma2_rn(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])), sc2, nl2);
        pr[j] = fast_exp2(e.x);
        pr[j + 1] = fast_exp2(e.y);
      }
      if (seen != 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!(seen >> j & 1u)) pr[j] = 0.0f;
      }
      // dV(i - PB) has read the buffer
      if (i >= PB && !mbar_wait(&dv_done[i % PB], (i / PB - 1) & 1)) { ok = false; break; }
      // P and dS are rounded to 16 bits as operands of the products
#pragma unroll
      for (int j8 = 0; j8 < 4; ++j8) {
        __align__(16) elem2_t hp[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) hp[q] = ff2e2(pr[j8 * 8 + 2 * q], pr[j8 * 8 + 2 * q + 1]);
        *reinterpret_cast<uint4*>(pRow + (i % PB) * kSq + swz(row, chunk0 + j8)) = *reinterpret_cast<uint4*>(hp);
      }
      fence_proxy_async_smem();
      fence_before_sync();
      warp_arrive(p_ready);
      if (!mbar_wait(dp_full, i & 1)) { ok = false; break; }
      fence_after_sync();
      tmem_ld_32x32(tm_dp + lane_addr + part * 32, r);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) pr[j] = pr[j] * (__uint_as_float(r[j]) - dl) * p.scale;
      if (seen != 0xffffffffu) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (!(seen >> j & 1u)) pr[j] = 0.0f;
      }
      if (i > 0 && !mbar_wait(dk_done, (i - 1) & 1)) { ok = false; break; }   // dQ(i-1), dK(i-1) have read dS
#pragma unroll
      for (int j8 = 0; j8 < 4; ++j8) {
        __align__(16) elem2_t hd[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) hd[q] = ff2e2(pr[j8 * 8 + 2 * q], pr[j8 * 8 + 2 * q + 1]);
        *reinterpret_cast<uint4*>(dsRow + swz(row, chunk0 + j8)) = *reinterpret_cast<uint4*>(hd);
      }
      fence_proxy_async_smem();
      fence_before_sync();
      warp_arrive(ds_ready);
    }
    // dV (parts 0, 1) and dK (parts 2, 3) of this key block, half of the columns each
    if (ok && mbar_wait(dk_done, (n - 1) & 1)) {
      fence_after_sync();
      const int t_k = k0 + row;
      elem_t* dst = part < 2 ? p.dv + b * p.v_sb + t_k * p.v_st + kvh * p.v_sh : p.dk + b * p.k_sb + t_k * p.k_st + kvh * p.k_sh;
      const uint32_t src = part < 2 ? tm_dv : tm_dk;
#pragma unroll 1
      for (int c0 = (part & 1) * (D / 2); c0 < ((part & 1) + 1) * (D / 2); c0 += 32) {
        uint32_t r[32];
        tmem_ld_32x32(src + lane_addr + c0, r);
        tmem_ld_wait();
        if (t_k < p.T) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            __align__(16) elem2_t hh[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) hh[q] = ff2e2(__uint_as_float(r[j + 2 * q]), __uint_as_float(r[j + 2 * q + 1]));
            *reinterpret_cast<uint4*>(dst + c0 + j) = *reinterpret_cast<uint4*>(hh);
          }
        }
      }
    } else {
      ok = false;
    }
    if (!ok && lane == 0) atomicExch(p.status, ATT_ERR_TIMEOUT);
  } else {
    // ---------------------------------------------------------------- dQ: one row per thread
    const int row = warp * 32 + lane, token = row / p.group;
    const uint32_t lane_addr = uint32_t(warp * 32) << 16;
    const int h = kvh * p.group + (row - token * p.group);
    bool ok = true;
    for (int i = 0; i < n && ok; ++i) {
      const int m = tile_of(i), t0 = m * p.tile_tokens, t1 = min(t0 + p.tile_tokens, len) - 1, t_q = t0 + token;
      const bool row_ok = token < p.tile_tokens && t_q < len;
      // the key blocks that add to this tile: [0, firsts), then hi down to lo
      const int hi = t1 / kKeys, firsts = min(ns, hi + 1), lo = max(max(0, t0 - p.window + 1) / kKeys, firsts);
      const int rank = first_block ? kb : firsts + hi - kb, last = firsts + (hi - lo + 1) - 1;
      int* counter = p.counters + ((long long)bh * p.tiles + m) * 4 + warp;
      float4* sum = p.sums + ((long long)bh * p.tiles + m) * (D / 4) * kRows + row;
      elem_t* dst = p.dq + b * p.q_sb + t_q * p.q_st + h * p.q_sh;
      if (!mbar_wait(dq_full, i & 1)) { ok = false; break; }
      fence_after_sync();
      if (rank > 0) {
        bool in = false;
        for (uint32_t spin = 0; spin < kSpinLimit && !in; ++spin) in = load_acquire(counter) >= rank;
        if (!__all_sync(0xffffffffu, in)) { ok = false; break; }
      }
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t r[32];
        tmem_ld_32x32(tm_dq + lane_addr + c0, r);
        tmem_ld_wait();
        if (c0 + 32 == D) {      // all of dQ(i) has been read: the columns may be written again
          fence_before_sync();
          warp_arrive(dq_read);
        }
        float4* at = sum + c0 / 4 * kRows;
        if (rank == last) {
          if (rank > 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 v = __ldcg(at + j * kRows);
              r[4 * j] = __float_as_uint(__uint_as_float(r[4 * j]) + v.x);
              r[4 * j + 1] = __float_as_uint(__uint_as_float(r[4 * j + 1]) + v.y);
              r[4 * j + 2] = __float_as_uint(__uint_as_float(r[4 * j + 2]) + v.z);
              r[4 * j + 3] = __float_as_uint(__uint_as_float(r[4 * j + 3]) + v.w);
            }
          }
          if (row_ok) {
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
              __align__(16) elem2_t hh[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) hh[q] = ff2e2(__uint_as_float(r[j + 2 * q]), __uint_as_float(r[j + 2 * q + 1]));
              *reinterpret_cast<uint4*>(dst + c0 + j) = *reinterpret_cast<uint4*>(hh);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 v = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]),
                                         __uint_as_float(r[4 * j + 3]));
            if (rank == 0) __stcg(at + j * kRows, v); else atomicAdd(at + j * kRows, v);
          }
        }
      }
      if (rank != last) {
        __threadfence();
        __syncwarp();
        if (lane == 0) store_release(counter, rank + 1);
      }
    }
    if (!ok && lane == 0) atomicExch(p.status, ATT_ERR_TIMEOUT);
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 20) { fence_after_sync(); tmem_dealloc(tmem, kTmemCols); }
}

// Floats of the parts of the workspace: sums of dQ (none where no tile has two key blocks), counters and the ticket, delta.
struct Workspace {
  long long sums, counters, delta;
};
Workspace workspace(long long B, long long T, long long kv_heads, long long group, int D) {
  const long long tile_tokens = kRows / group, tiles = (T + tile_tokens - 1) / tile_tokens;
  Workspace w;
  w.sums = T <= kKeys ? 0 : B * kv_heads * tiles * kRows * D;
  w.counters = (B * kv_heads * tiles * 4 + 1 + 3) / 4 * 4;
  w.delta = B * kv_heads * T * group;
  return w;
}

}  // namespace

extern "C" {

long long fbam_window_bwd_workspace(int B, int T, int kv_heads, int group, int D) {
  if (group < 1 || group > kRows) return 0;
  const Workspace w = workspace(B, T, kv_heads, group, D);
  return w.sums + w.counters + w.delta;
}

// Operands as in fbam_window_fwd; out contiguous, as the forward wrote it; d_o (B, T, heads, D) with strides; the gradients with
// strides each; work: fp32 workspace of fbam_window_bwd_workspace values, 16-byte aligned.
int fbam_window_bwd(const void* q, long long q_sb, long long q_st, long long q_sh, const void* k, const void* v, long long k_sb,
                    long long k_st, long long k_sh, long long v_sb, long long v_st, long long v_sh, const void* out, const void* d_o,
                    long long do_sb, long long do_st, long long do_sh, const float* lse, const int* lengths, float* work,
                    long long work_floats, void* dq, long long dq_sb, long long dq_st, long long dq_sh, void* dk, long long dk_sb,
                    long long dk_st, long long dk_sh, void* dv, long long dv_sb, long long dv_st, long long dv_sh, int B, int T,
                    int kv_heads, int group, int D, int window, int sinks, float scale, int* status, void* stream) {
  if ((D != 64 && D != 128) || B < 1 || T < 1 || kv_heads < 1 || group < 1 || group > kRows || sinks < 0) return 1;
  const Workspace w = workspace(B, T, kv_heads, group, D);
  if (work_floats < w.sums + w.counters + w.delta) return 1;
  const uintptr_t outs = (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)out | (uintptr_t)work;
  if ((outs & 15) || dq_sb % 8 || dq_st % 8 || dq_sh % 8 || dk_sb % 8 || dk_st % 8 || dk_sh % 8 || dv_sb % 8 || dv_st % 8 || dv_sh % 8)
    return 2;
  BwdParams p = {};
  p.T = T; p.B = B; p.kv_heads = kv_heads; p.group = group;
  p.tile_tokens = kRows / group;
  p.tiles = (T + p.tile_tokens - 1) / p.tile_tokens;
  p.window = window < 1 || window > kNoWindow ? kNoWindow : window;   // 0: none
  p.sinks = p.window == kNoWindow ? 0 : sinks < kNoWindow ? sinks : kNoWindow;
  p.lengths = lengths;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.scale = scale;
  p.sums = (float4*)work;
  p.counters = (int*)(work + w.sums);
  p.ticket = p.counters + w.counters - 1;
  p.lse = lse;
  float* delta = work + w.sums + w.counters;
  p.delta = delta;
  p.dq = (elem_t*)dq; p.dk = (elem_t*)dk; p.dv = (elem_t*)dv;
  p.q_sb = dq_sb; p.q_st = dq_st; p.q_sh = dq_sh;
  p.k_sb = dk_sb; p.k_st = dk_st; p.k_sh = dk_sh;
  p.v_sb = dv_sb; p.v_st = dv_st; p.v_sh = dv_sh;
  p.status = status;
  const long long nkb = (T + kKeys - 1) / kKeys, blocks = nkb * B * kv_heads;
  const long long rows = (long long)B * T * kv_heads * group;
  long long threads = rows * (D / 8);
  if (threads < w.counters) threads = w.counters;
  if (blocks > 0x7fffffffll || w.counters > 0x7fffffffll || (threads + 255) / 256 > 0x7fffffffll) return 1;
  CUtensorMap mq, mk, mv, mdo;
  int e;
  if ((e = encode_heads(&mq, q, D, kv_heads * group, T, B, q_sh, q_st, q_sb, group, p.tile_tokens))) return e;
  if ((e = encode_heads(&mk, k, D, kv_heads, T, B, k_sh, k_st, k_sb, 1, kKeys))) return e;
  if ((e = encode_heads(&mv, v, D, kv_heads, T, B, v_sh, v_st, v_sb, 1, kKeys))) return e;
  if ((e = encode_heads(&mdo, d_o, D, kv_heads * group, T, B, do_sh, do_st, do_sb, group, p.tile_tokens))) return e;
  cudaStream_t s = (cudaStream_t)stream;
  const unsigned pre = (unsigned)((threads + 255) / 256);
  if (D == 64)
    window_delta_kernel<64><<<pre, 256, 0, s>>>((const elem_t*)out, (const elem_t*)d_o, do_sb, do_st, do_sh, delta, p.counters, (int)w.counters, p);
  else
    window_delta_kernel<128><<<pre, 256, 0, s>>>((const elem_t*)out, (const elem_t*)d_o, do_sb, do_st, do_sh, delta, p.counters, (int)w.counters, p);
  auto kernel = D == 64 ? window_bwd_kernel<64> : window_bwd_kernel<128>;
  const int smem = D == 64 ? bwd_smem_bytes<64>() : bwd_smem_bytes<128>();
  if (set_smem(kernel, smem)) return 5;
  kernel<<<(unsigned)blocks, kBwdThreads, smem, s>>>(mq, mk, mv, mdo, p);
  return cudaGetLastError() == cudaSuccess ? 0 : 5;
}

}  // extern "C"
