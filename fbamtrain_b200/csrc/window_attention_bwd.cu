// Backward of the attention over a sliding window and the first tokens (forward and definition in window_attention.cu).
//
//   P = 2^(S scale log2(e) - lse),  dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta) scale,  dQ = dS K,  dK = dS^T Q,
//   delta = rowsum(dO O), from the output and what its rounding took off
//
// One thread block owns 128 keys of a key head and walks the tiles of queries that see any of them; a tile's 128 rows are tokens x
// the query heads that share the key head, so dK and dV, which sum over those heads, are summed in tensor memory.  All scores are
// TRANSPOSED, a key a row: S^T = K Q^T and dP^T = V dO^T.  Then P^T is the first operand of dV as it stands and goes over S^T in tensor
// memory; dS^T goes to shared memory once, where dK reads it as it lies and dQ transposed (an MN-major operand).  Roles:
//   warp 13     TMA: K, V once; Q with lse two tiles deep; dO with delta two deep (D = 64) or one (D = 128: shared memory is full)
//   warp 12     MMA issue: dV(i), S(i+1) once P(i) is stored; dQ(i), dK(i) once dS(i) is; dP in front of dQ(i-1) (D = 64), or, where
//               dQ borrows its columns (D = 128), behind dV(i) once dQ(i-1) is read
//   warps 4-11  point-wise: 32 keys and 64 queries each
//   warps 0-3   take dQ out of tensor memory and pass it through shared memory, 16 columns at a time
//   warps 14-15 have the copy engine add those to the tile's sum, in turns: a tile's are complete long after the next one's begin
// Sixteen warps leave 128 registers a thread: with four threads a key (80 registers) a hundred bytes a thread were spilled, more than
// the L1 that shared memory leaves holds, and each step waited for L2 (T 30011, 16 over 4 heads of 128, window 2048: 3 037 us).
// Every barrier that a role waits on can complete its next phase only after that role has gone on, so a wait by phase parity cannot
// miss a phase.
//
// dQ of a tile is a sum over the key blocks that it sees.  They add to it in one fixed order, the last key block first, so that the
// result does not depend on which block runs when.  The first one stores, those between add, the last one adds and writes the rounded
// gradient, so there is neither a zero fill nor a pass behind the kernel.  Each tile has a counter of the contributions that are in.
// Thread blocks take their work by a ticket, the last keys first, in which every contribution waits for earlier tickets only, so a wait
// always ends; and all walk their tiles forward, so that a thread block meets a tile one step after the one with the keys behind its own
// did.
//
// The first tokens are seen by all tiles behind them, a window's keys by those of a window only: a walk over all tiles by one thread
// block would last as long as everything else together (3 817 against 3 216 us at T 30011, 16 over 4 heads of 128, window 2048).  It is
// divided into parts, behind all others: run ahead of them instead, they held up the walks behind (1 947 against 2 117 us).  Long walks
// over a window are divided as well, into halves of what a multiprocessor has to do.  The parts of a walk write their dK and dV in
// fp32, and a last kernel adds them up in their order.
//
// T 30011, 16 over 4 heads of 128, window 2048: 1 592 us, 770 TFLOP/s of the products that the masks leave; a tile takes 6 400 cycles, its
// five products 2 600: they wait for the point-wise warps and those for them, and shared memory carries operands, dS and dQ for 4 350.
// 8 x 1024, 16 heads of 64, window 256: 116 us, of which a thread block's start and end, 14 000 cycles that nothing overlaps, are most.
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
  const float* lse;      // (B, kv_heads, tile, 128): minus log2 of the sum of 2^(s scale log2(e))
  const float* delta;    // the same: minus delta scale
  float* sums;           // (B, kv_heads, tile, D / 4, 128, 4) fp32: written before it is read
  int* counters;         // (B, kv_heads, tile): contributions that are in; zeroed
  int* ticket;           // zeroed
  float4* kv_parts;      // (part of a divided walk, dV | dK, D / 4, 128) fp32
  int blocks, firsts;    // key blocks, and those of them with first tokens
  int parts, part_tiles, first_parts, first_part_tiles;   // parts of a walk and their tiles; the same of the first tokens' blocks
  elem_t* dq;
  elem_t* dk;
  elem_t* dv;
  long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  int* status;
};

// delta, and what else has to be there before the main kernel: counters at zero, dQ of the rows behind a sequence's end.  D / 8 threads
// a row, four rows a thread whose loads are on their way together; four of a row's threads place one of its sums each, since where they
// go takes divisions.
// 8 x 1024, 16 heads of 64: 11.4 us, 4.4 TB/s; 30 011 x 16 heads of 128: 65 us, 5.7 TB/s.
template <int D>
__global__ void __launch_bounds__(256) window_delta_kernel(const elem_t* __restrict__ o, const elem_t* __restrict__ low,
                                                           const elem_t* __restrict__ d_o, long long do_sb, long long do_st, long long do_sh,
                                                           float* __restrict__ delta, int* counters, int n_counters, const BwdParams p) {
  constexpr int kLanes = D / 8, kRowsEach = 4, kStep = 256 / kLanes;
  const long long thread = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (thread < n_counters) counters[thread] = 0;
  const int heads = p.kv_heads * p.group, part = threadIdx.x % kLanes;
  const long long all = (long long)p.B * p.T * heads, row0 = (long long)blockIdx.x * kStep * kRowsEach + threadIdx.x / kLanes;   // (b, t, h)
  uint4 ov[kRowsEach], lv[kRowsEach], gv[kRowsEach];
  int h[kRowsEach], t[kRowsEach], b[kRowsEach];
  bool there[kRowsEach];
  int h_at, t_at, b_at;                              // divided once: the next rows are counted on
  if (all < 0x80000000ll) {
    const unsigned bt = (unsigned)row0 / (unsigned)heads;
    h_at = (int)((unsigned)row0 - bt * heads);
    b_at = (int)(bt / (unsigned)p.T);
    t_at = (int)(bt - (unsigned)b_at * p.T);
  } else {
    const long long bt = row0 / heads;
    h_at = (int)(row0 - bt * heads);
    b_at = (int)(bt / p.T);
    t_at = (int)(bt - (long long)b_at * p.T);
  }
  const int step_t = kStep / heads, step_h = kStep - step_t * heads;
#pragma unroll
  for (int u = 0; u < kRowsEach; ++u) {
    const long long idx = row0 + u * kStep;
    h[u] = h_at;
    t[u] = t_at;
    b[u] = b_at;
    h_at += step_h;
    t_at += step_t;
    if (h_at >= heads) {
      h_at -= heads;
      ++t_at;
    }
    while (t_at >= p.T) {
      t_at -= p.T;
      ++b_at;
    }
    there[u] = idx < all;
    if (!there[u]) continue;
    if (p.lengths != nullptr && t[u] >= p.lengths[b[u]]) {
      there[u] = false;
      *reinterpret_cast<uint4*>(p.dq + b[u] * p.q_sb + t[u] * p.q_st + h[u] * p.q_sh + part * 8) = make_uint4(0u, 0u, 0u, 0u);
    } else {
      ov[u] = *reinterpret_cast<const uint4*>(o + idx * D + part * 8);
      lv[u] = *reinterpret_cast<const uint4*>(low + idx * D + part * 8);
      gv[u] = *reinterpret_cast<const uint4*>(d_o + b[u] * do_sb + t[u] * do_st + h[u] * do_sh + part * 8);
    }
  }
  static_assert(kLanes >= kRowsEach, "a lane a row");
  float sum = 0.0f;
  int h_of = 0, t_of = 0, b_of = 0;
  bool placed = false;
#pragma unroll
  for (int u = 0; u < kRowsEach; ++u) {
    float s = 0.0f;
    if (there[u]) {
      const elem2_t* oe = reinterpret_cast<const elem2_t*>(&ov[u]);
      const elem2_t* le = reinterpret_cast<const elem2_t*>(&lv[u]);
      const elem2_t* ge = reinterpret_cast<const elem2_t*>(&gv[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 x = e22ff(oe[i]), z = e22ff(le[i]), y = e22ff(ge[i]);
        s += (x.x + z.x) * y.x + (x.y + z.y) * y.y;
      }
    }
#pragma unroll
    for (int off = kLanes / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (part == u) {
      sum = s;
      h_of = h[u];
      t_of = t[u];
      b_of = b[u];
      placed = there[u];
    }
  }
  if (placed) {
    const unsigned kvh = (unsigned)h_of / p.group, tile = (unsigned)t_of / p.tile_tokens;
    delta[(((long long)b_of * p.kv_heads + kvh) * p.tiles + tile) * kRows + (t_of - tile * p.tile_tokens) * p.group + (h_of - kvh * p.group)] =
        -sum * p.scale;
  }
}

constexpr int kBwdWarps = 16, kBwdThreads = kBwdWarps * 32;
template <int D>
constexpr int kDoStages = D == 64 ? 2 : 1;
constexpr int kStage = 128 * 16 * 4, kStages = 4;   // 16 columns of dQ on their way to the sum
template <int D>
constexpr int bwd_smem_bytes() {
  return (4 + kDoStages<D>) * 128 * D * 2 + 128 * 128 * 2 + kStages * kStage + (2 + kDoStages<D>) * 512 + 256 + 1024;
}

// 16 rows x 64 columns of fp32 in the layout of matrix fragments: thread t receives, for each 8 columns j, columns 8 j + 2 (t % 4) and
// the one behind it of row t / 4 (x[4 j], x[4 j + 1]) and of row t / 4 + 8 (x[4 j + 2], x[4 j + 3]).
__device__ __forceinline__ void tmem_ld_16x64(uint32_t taddr, uint32_t (&x)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]), "=r"(x[8]), "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15]), "=r"(x[16]), "=r"(x[17]), "=r"(x[18]), "=r"(x[19]), "=r"(x[20]), "=r"(x[21]), "=r"(x[22]), "=r"(x[23]), "=r"(x[24]), "=r"(x[25]), "=r"(x[26]), "=r"(x[27]), "=r"(x[28]), "=r"(x[29]), "=r"(x[30]), "=r"(x[31])
      : "r"(taddr)
      : "memory");
}
// 16 rows x 32 columns of pairs of 16-bit values: thread t gives, for each 4 columns j, column 4 j + t % 4 of row t / 4 (x[2 j]) and of
// row t / 4 + 8 (x[2 j + 1]): the pairs that tmem_ld_16x64 gave it.
__device__ __forceinline__ void tmem_st_16x32(uint32_t taddr, const uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]), "r"(x[8]), "r"(x[9]), "r"(x[10]), "r"(x[11]), "r"(x[12]), "r"(x[13]), "r"(x[14]), "r"(x[15])
      : "memory");
}
// Four 8 x 8 matrices of 16-bit values in the same layout to shared memory; lane l names row l % 8 of matrix l / 8.
__device__ __forceinline__ void store_matrices(const void* row, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(row)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint32_t pack(uint32_t a, uint32_t b) {
  const elem2_t h = ff2e2(__uint_as_float(a), __uint_as_float(b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
// `bytes` of shared memory to global memory, or added to fp32 values there; both addresses on 16-byte boundaries.
__device__ __forceinline__ void bulk_store(float* dst, const void* smem_src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(__cvta_generic_to_global(dst)), "r"(smem_u32(smem_src)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bulk_add(float* dst, const void* smem_src, uint32_t bytes) {
  asm volatile("cp.reduce.async.bulk.global.shared::cta.bulk_group.add.f32 [%0], [%1], %2;" ::"l"(__cvta_generic_to_global(dst)),
               "r"(smem_u32(smem_src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void fence_proxy_async_all() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ int load_acquire(const int* at) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(at) : "memory");
  return v;
}
__device__ __forceinline__ void store_release(int* at, int v) {
  asm volatile("st.release.gpu.global.s32 [%0], %1;" ::"l"(at), "r"(v) : "memory");
}

// Sums of several thread blocks in a fixed order, by whole warps: wait until `rank` contributions are in, add, hand on to the next.
__device__ __forceinline__ bool reached(const int* counter, int rank) {
  for (uint32_t spin = 0; spin < kSpinLimit; ++spin)
    if (load_acquire(counter) >= rank) return true;
  return false;
}
__device__ __forceinline__ bool wait_for(const int* counter, int rank) { return __all_sync(0xffffffffu, reached(counter, rank)); }
// N columns of a row; a thread's 16-byte pieces lie PITCH pieces apart, so that a warp's are side by side.
template <int PITCH, int N>
__device__ __forceinline__ void store_part(float4* sum, const uint32_t (&r)[N]) {
#pragma unroll
  for (int j = 0; j < N / 4; ++j)
    __stcg(sum + j * PITCH, make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]),
                                        __uint_as_float(r[4 * j + 3])));
}
template <int N>
__device__ __forceinline__ void store_row(elem_t* dst, const uint32_t (&r)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 8) {
    __align__(16) elem2_t hh[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) hh[q] = ff2e2(__uint_as_float(r[j + 2 * q]), __uint_as_float(r[j + 2 * q + 1]));
    *reinterpret_cast<uint4*>(dst + j) = *reinterpret_cast<uint4*>(hh);
  }
}

// The tiles that see a key block, and of which of them the parts of its walk consist.
struct Walk {
  int first, tiles, last_part;
};
__device__ __forceinline__ Walk walk_of(const BwdParams& p, int kb, int len) {
  const int k0 = kb * kKeys, end = kb < p.firsts ? len : min(len, k0 + kKeys - 1 + p.window);
  Walk w;
  w.first = k0 / p.tile_tokens;
  w.tiles = k0 < len ? (end + p.tile_tokens - 1) / p.tile_tokens - w.first : 0;
  const int part = kb < p.firsts ? p.first_part_tiles : p.part_tiles;
  w.last_part = w.tiles > 0 ? (w.tiles + part - 1) / part - 1 : 0;
  return w;
}
__device__ __forceinline__ long long slot_of(const BwdParams& p, int bh, int kb, int part) {
  if (kb < p.firsts) return ((long long)bh * p.firsts + kb) * p.first_parts + part;
  const long long behind = p.first_parts > 1 ? (long long)p.B * p.kv_heads * p.firsts * p.first_parts : 0;
  return behind + ((long long)bh * (p.blocks - p.firsts) + kb - p.firsts) * p.parts + part;
}

template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
window_bwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const __grid_constant__ CUtensorMap map_dk,
                  const __grid_constant__ CUtensorMap map_dv, const __grid_constant__ BwdParams p) {
  constexpr int DP = D / 64;
  constexpr int kTile = 128 * D * 2;           // a 128-row x D operand tile
  constexpr int kSq = 128 * 128 * 2;           // dS tile
  constexpr int DOS = kDoStages<D>;
  constexpr bool kOwnDq = D == 64;             // dQ has tensor-memory columns of its own
  constexpr uint32_t kTmemCols = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + kTile;
  uint8_t* sQ = sV + kTile;                    // two stages
  uint8_t* sDO = sQ + 2 * kTile;               // DOS stages
  uint8_t* sDS = sDO + DOS * kTile;
  uint8_t* sStage = sDS + kSq;                 // kStages
  float* sL = reinterpret_cast<float*>(sStage + kStages * kStage);   // two stages of 128: minus lse
  float* sD = sL + 2 * 128;                    // DOS stages: minus delta scale
  uint64_t* bars = reinterpret_cast<uint64_t*>(sD + DOS * 128);
  uint64_t* kv_full = bars;
  uint64_t* q_full = bars + 1;      // [2]
  uint64_t* do_full = bars + 3;     // [2]
  uint64_t* q_free = bars + 5;      // [2] dK(i) has read the stage
  uint64_t* do_free = bars + 7;     // [2] dP(i) and dV(i) have read the stage, and the point-wise warps delta (9)
  uint64_t* s_full = bars + 9;      // S(i) in tensor memory
  uint64_t* dp_full = bars + 10;    // dP(i) in tensor memory
  uint64_t* p_ready = bars + 11;    // P(i) stored over S(i) (8 warps)
  uint64_t* ds_ready = bars + 12;   // dS(i) stored, dP(i) read (8 warps)
  uint64_t* dq_full = bars + 13;    // dQ(i) in tensor memory
  uint64_t* dq_read = bars + 14;    // dQ(i) taken out (4 warps)
  uint64_t* dk_done = bars + 15;    // dQ(i) and dK(i) have read dS; all products so far are complete
  uint64_t* kv_clean = bars + 16;   // K and V rows behind the sequence's end are zeros (8 warps)
  uint64_t* staged = bars + 17;     // [tile's turn][kStages] a stage is full (4 warps)
  uint64_t* stage_free = staged + 2 * kStages;   // [kStages] the copy engine has read it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(stage_free + kStages);
  int* my_ticket = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int used = p.tile_tokens * p.group;                        // rows of a tile
  if (threadIdx.x == 0) {
    *my_ticket = atomicAdd(p.ticket, 1);
    prefetch_tensormap(&map_q); prefetch_tensormap(&map_k); prefetch_tensormap(&map_v); prefetch_tensormap(&map_do);
  }
  if (warp == 12) { tmem_alloc(tmem_slot, kTmemCols); tmem_relinquish(); }
  if (threadIdx.x == 13 * 32) {
    for (int i = 0; i < 17 + 3 * kStages; ++i)
      mbar_init(&bars[i], i == 7 || i == 8 ? 9 : i == 11 || i == 12 || i == 16 ? 8 : i == 14 || (i >= 17 && i < 17 + 2 * kStages) ? 4 : 1);
    mbar_fence_init();
  }
  if (used < kRows) {
    // the copies never write the rows behind them; they are operands of the transposed products
    const int rows = kRows - used, per = (2 + DOS) * DP * rows * 8;
    for (int i = threadIdx.x; i < per; i += kBwdThreads) {
      const int chunk = i & 7, r = used + (i >> 3) % rows, panel = (i >> 3) / rows;    // Q stages and dO stages lie in a row
      *reinterpret_cast<uint4*>(sQ + panel * 128 * 128 + r * 128 + chunk * 16) = make_uint4(0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const int ticket = __shfl_sync(0xffffffffu, *my_ticket, 0);      // the same in all lanes: what follows from it takes uniform registers
  const int bhs = p.B * p.kv_heads, ns = p.firsts;
  const int bh = ticket % bhs, behind = ticket / bhs - (p.blocks - ns) * p.parts;   // 0 or more: a block of first tokens
  const int kb = behind < 0 ? p.blocks - 1 - ticket / bhs / p.parts : ns - 1 - behind / p.first_parts;
  const int part_at = behind < 0 ? ticket / bhs % p.parts : behind % p.first_parts;
  const int part_tiles = behind < 0 ? p.part_tiles : p.first_part_tiles;
  const int b = bh / p.kv_heads, kvh = bh % p.kv_heads;
  const int k0 = kb * kKeys;
  const int len = p.lengths == nullptr ? p.T : min(max(p.lengths[b], 0), p.T);
  const Walk walk = walk_of(p, kb, len);
  const int last_part = walk.last_part;
  if (part_at > last_part) {
    if (warp == 12) tmem_dealloc(tmem, kTmemCols);
    return;
  }
  const int m0 = walk.first + part_at * part_tiles, n = min(part_tiles, walk.tiles - part_at * part_tiles);   // the tiles of this part
  if (walk.tiles <= 0) {                                           // keys behind the sequence's end
    for (int i = threadIdx.x; i < kKeys * (D / 8) * 2; i += kBwdThreads) {
      const int which = i & 1, r = (i >> 1) / (D / 8), d = (i >> 1) % (D / 8) * 8;
      if (k0 + r < p.T) {
        elem_t* at = which ? p.dv + b * p.v_sb + (long long)(k0 + r) * p.v_st + kvh * p.v_sh
                           : p.dk + b * p.k_sb + (long long)(k0 + r) * p.k_st + kvh * p.k_sh;
        *reinterpret_cast<uint4*>(at + d) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    if (warp == 12) tmem_dealloc(tmem, kTmemCols);
    return;
  }
  const uint32_t tm_s = tmem, tm_dp = tmem + 128, tm_dv = tmem + 256, tm_dk = tmem + 256 + D;
  const uint32_t tm_dq = kOwnDq ? tmem + 256 + 2 * D : tm_dp;

  // the key blocks that add to a tile: hi down to lo, then those of the first tokens; ours is number `rank` of 0 to `last`
  auto order = [&](int m, int& rank, int& last) {
    const int t0 = m * p.tile_tokens, t1 = min(t0 + p.tile_tokens, len) - 1;
    const int hi = t1 / kKeys, firsts = min(ns, hi + 1), near = hi + 1 - max(max(0, t0 - p.window + 1) / kKeys, firsts);
    rank = kb >= ns ? hi - kb : near + firsts - 1 - kb;
    last = near + firsts - 1;
  };

  // Registers go where the scores are: four warps of 96, four of 144 and eight of 136 of the 128 a thread that the block was launched with.
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 13) {
      if (elect_one()) {
        bool ok = true;
        auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int t) {
#pragma unroll
          for (int j = 0; j < DP; ++j) tma_load_4d(dst + j * 128 * 128, map, bar, j * 64, head, t, b);
        };
        auto load_q = [&](int i) {
          if (i >= 2 && !mbar_wait(&q_free[i & 1], ((i >> 1) - 1) & 1)) { ok = false; return; }
          mbar_expect_tx(&q_full[i & 1], used * D * 2 + 512);
          bulk_load(sL + (i & 1) * 128, p.lse + ((long long)bh * p.tiles + m0 + i) * kRows, 512, &q_full[i & 1]);
          load(sQ + (i & 1) * kTile, &map_q, &q_full[i & 1], kvh * p.group, (m0 + i) * p.tile_tokens);
        };
        auto load_do = [&](int i) {
          const int s = i % DOS;
          if (i >= DOS && !mbar_wait(&do_free[s], (i / DOS - 1) & 1)) { ok = false; return; }
          mbar_expect_tx(&do_full[s], used * D * 2 + 512);
          bulk_load(sD + s * 128, p.delta + ((long long)bh * p.tiles + m0 + i) * kRows, 512, &do_full[s]);
          load(sDO + s * kTile, &map_do, &do_full[s], kvh * p.group, (m0 + i) * p.tile_tokens);
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
    } else if (warp == 12) {
      if (elect_one()) {
        bool ok = true;
        const uint32_t id_s = make_idesc_f16kind(128, 128, false, false);   // S^T = K Q^T, dP^T = V dO^T
        const uint32_t id_t = make_idesc_f16kind(128, D, false, true);      // dV = P^T dO, dK = dS^T Q (B MN-major)
        const uint32_t id_q = make_idesc_f16kind(128, D, true, true);       // dQ = dS K (A, B MN-major)
        const uint64_t kK = k_major(smem_u32(sK)), kV = k_major(smem_u32(sV)), kQ = k_major(smem_u32(sQ)), kDO = k_major(smem_u32(sDO));
        const uint64_t mK = mn_major(smem_u32(sK)), mQ = mn_major(smem_u32(sQ)), mDO = mn_major(smem_u32(sDO));
        const uint64_t kDS = k_major(smem_u32(sDS)), mDS = mn_major(smem_u32(sDS));
        constexpr uint64_t kNext = kTile >> 4;                              // to the next stage
        auto issue_s = [&](int i) {
          if (!mbar_wait(&q_full[i & 1], (i >> 1) & 1)) { ok = false; return; }
          fence_after_sync();
          const uint64_t b = kQ + (i & 1) * kNext;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) mma_f16_ss(tm_s, kK + k_step(k), b + k_step(k), id_s, k != 0);
          mma_commit(s_full);
        };
        auto issue_dp = [&](int i) {
          if (!mbar_wait(&do_full[i % DOS], (i / DOS) & 1)) { ok = false; return; }
          fence_after_sync();
          const uint64_t b = kDO + (i % DOS) * kNext;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) mma_f16_ss(tm_dp, kV + k_step(k), b + k_step(k), id_s, k != 0);
          mma_commit(dp_full);
        };
        ok = mbar_wait(kv_full, 0) && mbar_wait(kv_clean, 0);
        if (ok) issue_s(0);
        if (ok) issue_dp(0);
        for (int i = 0; i < n && ok; ++i) {
          if (!mbar_wait(p_ready, i & 1) || !mbar_wait(&do_full[i % DOS], (i / DOS) & 1)) { ok = false; break; }
          fence_after_sync();
          const uint64_t bDO = mDO + (i % DOS) * kNext, bQ = mQ + (i & 1) * kNext;
#pragma unroll
          for (int k = 0; k < 128 / 16; ++k)     // the 16-bit values of 64 queries lie in the first 32 columns of their scores
            mma_f16_ts(tm_dv, tm_s + (k / 4) * 64 + (k % 4) * 8, bDO + mn_step(k), id_t, i != 0 || k != 0);
          mma_commit(&do_free[i % DOS]);
          if (ok && i + 1 < n) issue_s(i + 1);
          if (!ok || !mbar_wait(ds_ready, i & 1)) { ok = false; break; }
          fence_after_sync();
          if (kOwnDq) {
            if (i + 1 < n) issue_dp(i + 1);
            if (!ok || (i > 0 && !mbar_wait(dq_read, (i - 1) & 1))) { ok = false; break; }
            fence_after_sync();
          }
#pragma unroll
          for (int k = 0; k < 128 / 16; ++k)     // K dimension = keys; M = queries, two panels of 64
            mma_f16_ss(tm_dq, mDS + mn_step(k), mK + mn_step(k), id_q, k != 0);
          mma_commit(dq_full);
#pragma unroll
          for (int k = 0; k < 128 / 16; ++k)     // K dimension = queries
            mma_f16_ss(tm_dk, kDS + k_step(k), bQ + mn_step(k), id_t, i != 0 || k != 0);
          mma_commit(dk_done);
          mma_commit(&q_free[i & 1]);
          if (!kOwnDq && i + 1 < n) {
            if (!mbar_wait(dq_read, i & 1)) { ok = false; break; }
            issue_dp(i + 1);
          }
        }
        if (!ok) atomicExch(p.status, ATT_ERR_TIMEOUT);
      }
    } else if (warp >= 14) {
      // ---------------------------------------------------------------- dQ to its tile's sum: every other tile that is not finished here
      bool ok = true;
      if (elect_one()) {
        const int turn = warp - 14;
        int nth = 0;                               // tiles of both turns so far
        for (int i = 0; i < n && ok; ++i) {
          int rank, last;
          order(m0 + i, rank, last);
          if (rank == last || (nth++ & 1) != turn) continue;
          const long long tile = (long long)bh * p.tiles + m0 + i;
          if (rank > 0) {
            if (!reached(p.counters + tile, rank)) { ok = false; break; }
            fence_proxy_async_all();
          }
          for (int c = 0; c < D / 16; ++c) {
            if (!mbar_wait(&staged[turn * kStages + c % kStages], ((nth - 1 >> 1) * (D / 64) + c / kStages) & 1)) { ok = false; break; }
            float* dst = p.sums + (tile * (D / 16) + c) * (kStage / 4);
            const uint8_t* src = sStage + c % kStages * kStage;
            if (rank == 0) bulk_store(dst, src, kStage); else bulk_add(dst, src, kStage);
            bulk_commit_group();
            if (c > 1) {                           // all copies but the last two have read their stages
              bulk_wait_group_read<2>();
              mbar_arrive(&stage_free[(c - 2) % kStages]);
            }
          }
          if (!ok) break;
          bulk_wait_group_read<1>();
          mbar_arrive(&stage_free[kStages - 2]);
          bulk_wait_group_read<0>();
          mbar_arrive(&stage_free[kStages - 1]);
          bulk_wait_group_all();
          fence_proxy_async_all();
          __threadfence();
          store_release(p.counters + tile, rank + 1);
        }
        if (!ok) atomicExch(p.status, ATT_ERR_TIMEOUT);
      }
    }
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    // ---------------------------------------------------------------- point-wise: 32 keys and 64 queries per warp
    // In the fragment layout a thread has 16 of the 64 queries (of four keys), so it fetches 16 values of lse and of delta.  With a key a
    // thread it needed all 64, the same in all lanes: 1 024 cycles of shared memory a tile, which the products keep busy.
    const int lane_group = warp & 3, part = (warp - 4) >> 2;
    const int row = lane_group * 32 + lane;
    const uint32_t lane_addr = uint32_t(lane_group * 32) << 16;
    const float2 sc2 = make_float2(p.scale_log2, p.scale_log2), scale2 = make_float2(p.scale, p.scale);
    uint8_t* dsPanel = sDS + part * 128 * 128;         // 64 queries
    const int my_row = lane_group * 32 + (lane >> 3 & 1) * 8 + (lane & 7), my_chunk = lane >> 4;   // as an address of store_matrices
    bool ok = true;
    if (k0 + kKeys > len && len < p.T) {
      // K and V behind the sequence's end may hold anything: 0 x NaN is NaN in the products over keys
      ok = mbar_wait(kv_full, 0);
      if (ok && k0 + row >= len) {
#pragma unroll
        for (int j = part; j < DP * 8; j += 2) {
          const int at = (j / 8) * 128 * 128 + row * 128 + (j % 8) * 16;
          *reinterpret_cast<uint4*>(sK + at) = make_uint4(0u, 0u, 0u, 0u);
          *reinterpret_cast<uint4*>(sV + at) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      fence_proxy_async_smem();
    }
    warp_arrive(kv_clean);
    // lse is fetched a tile ahead, and delta before P is handed to the products.
    float2 ahead[8];
    auto fetch = [&](const float* from) {
#pragma unroll
      for (int j = 0; j < 8; ++j) ahead[j] = *reinterpret_cast<const float2*>(from + part * 64 + j * 8 + (lane & 3) * 2);
    };
    if (ok) ok = mbar_wait(&q_full[0], 0);               // lse comes with Q
    if (ok) fetch(sL);
    for (int i = 0; i < n && ok; ++i) {
      const int t0 = (m0 + i) * p.tile_tokens;
      const int rows = min(p.tile_tokens, len - t0) * p.group;     // rows of the tile that are queries
      const bool edge = k0 + kKeys - 1 > t0 || (k0 <= t0 + p.tile_tokens - 1 - p.window && k0 + kKeys > p.sinks) || rows < kRows;
      if (!mbar_wait(s_full, i & 1)) { ok = false; break; }
      fence_after_sync();
      if (t0 + p.tile_tokens > len && len < p.T) {
        // Q and dO behind the sequence's end, operands of the products over queries.  S(i) has read Q; dP(i) may be reading dO, but
        // only rows whose dS is set to zero below.
        if (!mbar_wait(&do_full[i % DOS], (i / DOS) & 1)) { ok = false; break; }
        if (row >= rows) {
#pragma unroll
          for (int j = part; j < DP * 8; j += 2) {
            const int at = (j / 8) * 128 * 128 + row * 128 + (j % 8) * 16;
            *reinterpret_cast<uint4*>(sQ + (i & 1) * kTile + at) = make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(sDO + (i % DOS) * kTile + at) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
      }
      // sets what a query does not see to zero: of the thread's 64 values those of key k and query c that are not in [from, to)
      auto mask = [&](uint32_t (&x)[2][32]) {
        auto below = [](int c) { return c <= 0 ? 0u : c >= 32 ? 0xffffffffu : (1u << c) - 1u; };
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int k = k0 + lane_group * 32 + r4 * 8 + (lane >> 2);
          const int from = max(0, k - t0) * p.group;                                     // t >= k
          const int to = k < p.sinks ? rows : min(rows, max(0, min(k - t0 + p.window, p.tile_tokens)) * p.group);   // t < k + window
#pragma unroll
          for (int w = 0; w < 2; ++w) {                    // 32 queries
            const uint32_t seen = (below(to - part * 64 - w * 32) & ~below(from - part * 64 - w * 32)) >> (lane & 3) * 2;
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t& v = x[r4 >> 1][(w * 4 + j) * 4 + (r4 & 1) * 2 + e];
                v = seen & (1u << (j * 8 + e)) ? v : 0u;
              }
          }
        }
      };
      uint32_t pr[2][32];                                // scores, then P, then dS, as fp32 bits: 16 keys each
#pragma unroll
      for (int h = 0; h < 2; ++h) tmem_ld_16x64(tm_s + lane_addr + (uint32_t(h * 16) << 16) + part * 64, pr[h]);
      tmem_ld_wait();
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 e = __ffma2_rn(make_float2(__uint_as_float(pr[h][j]), __uint_as_float(pr[h][j + 1])), sc2, ahead[j / 4]);
          pr[h][j] = __float_as_uint(fast_exp2(e.x));
          pr[h][j + 1] = __float_as_uint(fast_exp2(e.y));
        }
      if (edge) mask(pr);
      // P and dS are rounded to 16 bits as operands of the products
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t packed[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) packed[j] = pack(pr[h][2 * j], pr[h][2 * j + 1]);
        tmem_st_16x32(tm_s + lane_addr + (uint32_t(h * 16) << 16) + part * 64, packed);
      }
      tmem_st_wait();
      if (!mbar_wait(&do_full[i % DOS], (i / DOS) & 1)) { ok = false; break; }   // delta comes with dO
      fetch(sD + (i % DOS) * 128);
      fence_before_sync();
      warp_arrive(p_ready);
      warp_arrive(&do_free[i % DOS]);
      if (!mbar_wait(dp_full, i & 1)) { ok = false; break; }
      fence_after_sync();
      if (i > 0 && !mbar_wait(dk_done, (i - 1) & 1)) { ok = false; break; }      // dQ(i-1), dK(i-1) have read dS
      {
        uint32_t dp[2][32];
#pragma unroll
        for (int h = 0; h < 2; ++h) tmem_ld_16x64(tm_dp + lane_addr + (uint32_t(h * 16) << 16) + part * 64, dp[h]);
        tmem_ld_wait();
        // dS with its scale, in one multiply-add a pair: P (dP - delta) alone is infinite in half 8 (D = 64) to 11.3 (D = 128) times
        // earlier than dS.  In half dS itself has to be finite, and below 2^-14 it keeps an absolute error of 2^-25.
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 d = __fmul2_rn(make_float2(__uint_as_float(pr[h][j]), __uint_as_float(pr[h][j + 1])),
                                        __ffma2_rn(make_float2(__uint_as_float(dp[h][j]), __uint_as_float(dp[h][j + 1])), scale2, ahead[j / 4]));
            pr[h][j] = __float_as_uint(d.x);
            pr[h][j + 1] = __float_as_uint(d.y);
          }
      }
      if (rows < kRows) mask(pr);                        // behind the last query dO and delta may be anything
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 8; j += 2)                   // 8 queries j and the next 8
          store_matrices(dsPanel + swz(my_row + h * 16, j + my_chunk), pack(pr[h][4 * j], pr[h][4 * j + 1]), pack(pr[h][4 * j + 2], pr[h][4 * j + 3]),
                         pack(pr[h][4 * j + 4], pr[h][4 * j + 5]), pack(pr[h][4 * j + 6], pr[h][4 * j + 7]));
      fence_proxy_async_smem();
      fence_before_sync();
      warp_arrive(ds_ready);
      if (i + 1 < n) {
        if (!mbar_wait(&q_full[(i + 1) & 1], ((i + 1) >> 1) & 1)) { ok = false; break; }
        fetch(sL + ((i + 1) & 1) * 128);
      }
    }
    // dV (part 0) and dK (part 1) of this key block.  A wait may expire in some of a part's four warps only: they meet all the same.
    ok = ok && mbar_wait(dk_done, (n - 1) & 1);
    fence_after_sync();
    const uint32_t src = part == 0 ? tm_dv : tm_dk;
    if (last_part > 0) {
      float4* to = p.kv_parts + (slot_of(p, bh, kb, part_at) * 2 + part) * (D / 4) * kKeys + row;
#pragma unroll 1
      for (int c0 = 0; ok && c0 < D; c0 += 32) {
        uint32_t r[32];
        tmem_ld_32x32(src + lane_addr + c0, r);
        tmem_ld_wait();
        store_part<kKeys>(to + c0 / 4 * kKeys, r);
      }
    } else {
      // through the stages of Q, which nothing reads any more, and out by the copy engine: as rows from registers they took 4 400
      // (D = 64) to 9 000 cycles of every thread block
      uint8_t* tile = sQ + part * kTile;
#pragma unroll 1
      for (int c0 = 0; ok && c0 < D; c0 += 32) {
        uint32_t r[32];
        tmem_ld_32x32(src + lane_addr + c0, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          __align__(16) elem2_t hh[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) hh[q] = ff2e2(__uint_as_float(r[j * 8 + 2 * q]), __uint_as_float(r[j * 8 + 2 * q + 1]));
          *reinterpret_cast<uint4*>(tile + c0 / 64 * 128 * 128 + swz(row, c0 % 64 / 8 + j)) = *reinterpret_cast<uint4*>(hh);
        }
      }
      fence_proxy_async_smem();
      if (part == 0) asm volatile("bar.sync 1, 128;" ::: "memory"); else asm volatile("bar.sync 2, 128;" ::: "memory");   // four warps
      if (ok && lane_group == 0 && elect_one()) {
#pragma unroll
        for (int j = 0; j < DP; ++j) tma_store_4d(part == 0 ? &map_dv : &map_dk, tile + j * 128 * 128, j * 64, kvh, k0, b);   // rows behind T are cut
        bulk_commit_group();
        bulk_wait_group_read<0>();
      }
    }
    if (!ok && lane == 0) atomicExch(p.status, ATT_ERR_TIMEOUT);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    // ---------------------------------------------------------------- dQ: one row per thread
    const int row = warp * 32 + lane, token = row / p.group;
    const uint32_t lane_addr = uint32_t(warp * 32) << 16;
    const int h = kvh * p.group + (row - token * p.group);
    bool ok = true;
    int f = 0;                                           // tiles that went through the stages so far: the finishing warps take turns
    for (int i = 0; i < n && ok; ++i) {
      const int t_q = (m0 + i) * p.tile_tokens + token;
      int rank, last;
      order(m0 + i, rank, last);
      if (rank < last) {
        if (!mbar_wait(dq_full, i & 1)) { ok = false; break; }
        fence_after_sync();
        // all columns go into registers, so that they are free again before anything has left
        uint32_t r[D / 32][32];
#pragma unroll
        for (int c = 0; c < D / 32; ++c) tmem_ld_32x32(tm_dq + lane_addr + c * 32, r[c]);
        tmem_ld_wait();
        fence_before_sync();
        warp_arrive(dq_read);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          const int fill = f * (D / 64) + c / kStages;
          if (fill > 0 && !mbar_wait(&stage_free[c % kStages], (fill - 1) & 1)) { ok = false; break; }
          uint8_t* at = sStage + c % kStages * kStage + row * 16;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t* x = r[c / 2] + c % 2 * 16 + 4 * j;
            *reinterpret_cast<uint4*>(at + j * 2048) = make_uint4(x[0], x[1], x[2], x[3]);
          }
          fence_proxy_async_smem();
          warp_arrive(&staged[(f & 1) * kStages + c % kStages]);
        }
        ++f;
      } else {
        // the last one: the sum so far is fetched, 64 columns at a time, while its own part is on its way
        const long long tile = (long long)bh * p.tiles + m0 + i;
        const float4* sum = reinterpret_cast<const float4*>(p.sums) + tile * (D / 4) * kRows + row;
        elem_t* dst = p.dq + b * p.q_sb + t_q * p.q_st + h * p.q_sh;
        if (rank > 0) {
          if (!wait_for(p.counters + tile, rank)) { ok = false; break; }
          fence_proxy_async_all();
        }
        float4 v[16];
        auto fetch = [&](int half) {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = rank > 0 ? __ldcg(sum + (half * 16 + j) * kRows) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        };
        fetch(0);
        if (!mbar_wait(dq_full, i & 1)) { ok = false; break; }
        fence_after_sync();
#pragma unroll
        for (int half = 0; half < D / 64; ++half) {
          uint32_t r[2][32];
#pragma unroll
          for (int c = 0; c < 2; ++c) tmem_ld_32x32(tm_dq + lane_addr + half * 64 + c * 32, r[c]);
          tmem_ld_wait();
          if (half + 1 == D / 64) {
            fence_before_sync();
            warp_arrive(dq_read);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            uint32_t* x = r[j / 8] + j % 8 * 4;
            x[0] = __float_as_uint(v[j].x + __uint_as_float(x[0]));
            x[1] = __float_as_uint(v[j].y + __uint_as_float(x[1]));
            x[2] = __float_as_uint(v[j].z + __uint_as_float(x[2]));
            x[3] = __float_as_uint(v[j].w + __uint_as_float(x[3]));
          }
          if (half + 1 < D / 64) fetch(half + 1);
          if (token < p.tile_tokens && t_q < len) {
#pragma unroll
            for (int c = 0; c < 2; ++c) store_row(dst + half * 64 + c * 32, r[c]);
          }
        }
      }
    }
    if (!ok && lane == 0) atomicExch(p.status, ATT_ERR_TIMEOUT);
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 12) { fence_after_sync(); tmem_dealloc(tmem, kTmemCols); }
}

// dK and dV of the key blocks whose walks were divided: the parts' sums in their order.  A thread a row's four columns.
template <int D>
__global__ void __launch_bounds__(256) window_parts_kernel(const __grid_constant__ BwdParams p, int kb0, int count) {
  const int kb = kb0 + blockIdx.x % count, bh = blockIdx.x / count, which = blockIdx.y;      // which: dV, dK
  const int b = bh / p.kv_heads, kvh = bh % p.kv_heads;
  const int len = p.lengths == nullptr ? p.T : min(max(p.lengths[b], 0), p.T);
  const Walk walk = walk_of(p, kb, len);
  if (walk.last_part == 0) return;                   // one part, or none: written by the main kernel
  const int i = blockIdx.z * 256 + threadIdx.x, row = i % kKeys, piece = i / kKeys, key = kb * kKeys + row;
  const float4* at = p.kv_parts + slot_of(p, bh, kb, 0) * 2 * (D / 4) * kKeys + which * (D / 4) * kKeys + i;
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int part = 0; part <= walk.last_part; ++part) {
    const float4 v = __ldcg(at + (long long)part * 2 * (D / 4) * kKeys);
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  }
  if (key >= p.T) return;
  elem_t* dst = which ? p.dk + b * p.k_sb + key * p.k_st + kvh * p.k_sh : p.dv + b * p.v_sb + key * p.v_st + kvh * p.v_sh;
  __align__(8) elem2_t out[2] = {ff2e2(sum.x, sum.y), ff2e2(sum.z, sum.w)};
  *reinterpret_cast<uint2*>(dst + piece * 4) = *reinterpret_cast<uint2*>(out);
}

// How the walks are divided, and the workspace in units of four bytes: sums of dQ (none where no tile has two key blocks), dK and dV
// of the parts of divided walks, counters with the ticket, delta.
struct Plan {
  int tile_tokens, tiles, window, sinks, blocks, firsts, parts, part_tiles, first_parts, first_part_tiles;
  long long sums, kv_parts, counters, delta, thread_blocks;
};
Plan make_plan(long long B, long long T, long long kv_heads, int group, int D, int window, int sinks) {
  Plan a;
  a.tile_tokens = kRows / group;
  a.tiles = (int)((T + a.tile_tokens - 1) / a.tile_tokens);
  a.window = window < 1 || window > kNoWindow ? kNoWindow : window;   // 0: none
  a.sinks = a.window == kNoWindow ? 0 : sinks < kNoWindow ? sinks : kNoWindow;
  a.blocks = (int)((T + kKeys - 1) / kKeys);
  const long long first_blocks = ((long long)a.sinks + kKeys - 1) / kKeys;
  a.firsts = (int)(first_blocks < a.blocks ? first_blocks : a.blocks);
  // tiles of the longest walks, and how many of them the machine's 148 multiprocessors take each
  const long long reach = ((long long)kKeys - 1 + a.window) / a.tile_tokens + 2;
  const long long walk = a.tiles < reach ? a.tiles : reach;
  const long long steps = (((long long)a.blocks - a.firsts) * walk + (long long)a.firsts * a.tiles) * B * kv_heads / 148;
  auto divide = [](long long longest, long long share, int& parts, int& tiles) {
    tiles = (int)(share < 8 ? 8 : share < longest ? share : longest);
    parts = (int)((longest + tiles - 1) / tiles);
  };
  divide(walk, steps / 2, a.parts, a.part_tiles);
  divide(a.tiles, (long long)a.firsts * a.tiles * B * kv_heads / 296, a.first_parts, a.first_part_tiles);     // two a multiprocessor
  const long long bh = B * kv_heads;
  a.sums = a.blocks < 2 ? 0 : bh * a.tiles * kRows * D;
  a.kv_parts = ((a.first_parts > 1 ? (long long)a.firsts * a.first_parts : 0) + (a.parts > 1 ? (long long)(a.blocks - a.firsts) * a.parts : 0)) *
               bh * 2 * kKeys * D;
  a.counters = bh * a.tiles;
  a.delta = bh * a.tiles * kRows;
  a.thread_blocks = bh * ((long long)(a.blocks - a.firsts) * a.parts + (long long)a.firsts * a.first_parts);
  return a;
}
long long zeroed(const Plan& a) { return (a.counters + 1 + 3) / 4 * 4; }     // counters and the ticket

}  // namespace

extern "C" {

long long fbam_window_bwd_workspace(int B, int T, int kv_heads, int group, int D, int window, int sinks) {
  if (group < 1 || group > kRows || B < 1 || T < 1 || kv_heads < 1 || sinks < 0) return 0;
  const Plan a = make_plan(B, T, kv_heads, group, D, window, sinks);
  return a.sums + a.kv_parts + zeroed(a) + a.delta;
}

// Operands as in fbam_window_fwd; out and low contiguous, as the forward wrote them; d_o (B, T, heads, D) with strides; the gradients with
// strides each; work: fp32 workspace of fbam_window_bwd_workspace values, 16-byte aligned.
int fbam_window_bwd(const void* q, long long q_sb, long long q_st, long long q_sh, const void* k, const void* v, long long k_sb,
                    long long k_st, long long k_sh, long long v_sb, long long v_st, long long v_sh, const void* out, const void* low, const void* d_o,
                    long long do_sb, long long do_st, long long do_sh, const float* lse, const int* lengths, float* work,
                    long long work_floats, void* dq, long long dq_sb, long long dq_st, long long dq_sh, void* dk, long long dk_sb,
                    long long dk_st, long long dk_sh, void* dv, long long dv_sb, long long dv_st, long long dv_sh, int B, int T,
                    int kv_heads, int group, int D, int window, int sinks, float scale, int* status, void* stream) {
  if ((D != 64 && D != 128) || B < 1 || T < 1 || kv_heads < 1 || group < 1 || group > kRows || sinks < 0) return 1;
  const Plan a = make_plan(B, T, kv_heads, group, D, window, sinks);
  if (work_floats < a.sums + a.kv_parts + zeroed(a) + a.delta) return 1;
  const uintptr_t outs = (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv | (uintptr_t)out | (uintptr_t)low | (uintptr_t)work;
  if ((outs & 15) || dq_sb % 8 || dq_st % 8 || dq_sh % 8 || dk_sb % 8 || dk_st % 8 || dk_sh % 8 || dv_sb % 8 || dv_st % 8 || dv_sh % 8)
    return 2;
  BwdParams p = {};
  p.T = T; p.B = B; p.kv_heads = kv_heads; p.group = group;
  p.tile_tokens = a.tile_tokens; p.tiles = a.tiles;
  p.window = a.window; p.sinks = a.sinks;
  p.blocks = a.blocks; p.firsts = a.firsts;
  p.parts = a.parts; p.part_tiles = a.part_tiles; p.first_parts = a.first_parts; p.first_part_tiles = a.first_part_tiles;
  p.lengths = lengths;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.scale = scale;
  p.sums = work;
  p.kv_parts = (float4*)(work + a.sums);
  p.counters = (int*)(work + a.sums + a.kv_parts);
  p.ticket = p.counters + a.counters;
  p.lse = lse;
  float* delta = work + a.sums + a.kv_parts + zeroed(a);
  p.delta = delta;
  p.dq = (elem_t*)dq; p.dk = (elem_t*)dk; p.dv = (elem_t*)dv;
  p.q_sb = dq_sb; p.q_st = dq_st; p.q_sh = dq_sh;
  p.k_sb = dk_sb; p.k_st = dk_st; p.k_sh = dk_sh;
  p.v_sb = dv_sb; p.v_st = dv_st; p.v_sh = dv_sh;
  p.status = status;
  const long long rows = (long long)B * T * kv_heads * group;
  long long threads = (rows + 3) / 4 * (D / 8);
  if (threads < zeroed(a)) threads = zeroed(a);
  if (a.thread_blocks > 0x7fffffffll || zeroed(a) > 0x7fffffffll || (threads + 255) / 256 > 0x7fffffffll) return 1;
  CUtensorMap mq, mk, mv, mdo, mdk, mdv;
  int e;
  if ((e = encode_heads(&mq, q, D, kv_heads * group, T, B, q_sh, q_st, q_sb, group, p.tile_tokens))) return e;
  if ((e = encode_heads(&mk, k, D, kv_heads, T, B, k_sh, k_st, k_sb, 1, kKeys))) return e;
  if ((e = encode_heads(&mv, v, D, kv_heads, T, B, v_sh, v_st, v_sb, 1, kKeys))) return e;
  if ((e = encode_heads(&mdo, d_o, D, kv_heads * group, T, B, do_sh, do_st, do_sb, group, p.tile_tokens))) return e;
  if ((e = encode_heads(&mdk, dk, D, kv_heads, T, B, dk_sh, dk_st, dk_sb, 1, kKeys))) return e;
  if ((e = encode_heads(&mdv, dv, D, kv_heads, T, B, dv_sh, dv_st, dv_sb, 1, kKeys))) return e;
  cudaStream_t s = (cudaStream_t)stream;
  const unsigned pre = (unsigned)((threads + 255) / 256);
  if (D == 64)
    window_delta_kernel<64><<<pre, 256, 0, s>>>((const elem_t*)out, (const elem_t*)low, (const elem_t*)d_o, do_sb, do_st, do_sh, delta, p.counters,
                                               (int)zeroed(a), p);
  else
    window_delta_kernel<128><<<pre, 256, 0, s>>>((const elem_t*)out, (const elem_t*)low, (const elem_t*)d_o, do_sb, do_st, do_sh, delta, p.counters,
                                                (int)zeroed(a), p);
  auto kernel = D == 64 ? window_bwd_kernel<64> : window_bwd_kernel<128>;
  const int smem = D == 64 ? bwd_smem_bytes<64>() : bwd_smem_bytes<128>();
  if (D == 64 ? set_smem_once<window_bwd_kernel<64>>(smem) : set_smem_once<window_bwd_kernel<128>>(smem)) return 5;
  kernel<<<(unsigned)a.thread_blocks, kBwdThreads, smem, s>>>(mq, mk, mv, mdo, mdk, mdv, p);
  auto parts = D == 64 ? window_parts_kernel<64> : window_parts_kernel<128>;
  const int kb0 = a.first_parts > 1 ? 0 : a.firsts, kb1 = a.parts > 1 ? a.blocks : a.firsts;      // the blocks whose walks are divided
  if (kb1 > kb0) parts<<<dim3((unsigned)(B * kv_heads * (kb1 - kb0)), 2, D / 4 * kKeys / 256), 256, 0, s>>>(p, kb0, kb1 - kb0);
  return cudaGetLastError() == cudaSuccess ? 0 : 5;
}

}  // extern "C"
