// Causal attention that sees a sliding window and the first few tokens, over whole sequences (with its backward pass in
// window_attention_bwd.cu) and for new tokens over a paged cache; query heads may share key heads.
//
// A query at position i sees key j iff j <= i and (i - j < window or j < sinks), j within the sequence.
//
//   o_i = sum_j p_ij v_j,  p_ij = 2^(s_ij scale log2(e) - m_i) / l_i,  s = q k^T,  m the running maximum, l the running sum
//
// One thread block takes one or two tiles of queries of one key head.  A tile's 128 rows are TOKENS x the query heads that share the
// key head, so a key block is read once for all of them and one token of a shared head fills as many rows as there are heads.
// Key blocks of 128 pass through a ring in shared memory, K and V in turn; only blocks that some row of the tiles sees are
// visited (those of the first tokens, then those of the window).  Per block and tile: S = Q K^T into tensor memory
// (tcgen05.mma); four softmax warps, one row a thread, read S, form the exponentials and write P over S as 16-bit values; the
// second product takes P from tensor memory and adds P V to the tile's output there, which is rescaled only when a row's
// maximum has grown by more than 2^8.  Two tiles take turns on the tensor cores.
//
// Over a cache the ring is filled page by page: the lanes of the loading warp each look up one page (or part of one of 128 slots
// or more) and issue its copy.  Entries that are no page, slots behind the sequence and pages that nothing sees are filled with
// zeros by the copy engine (a coordinate behind the last page).  With few rows the keys are split over several thread blocks,
// whose partial sums a second kernel joins.
//
// Rows of V that no query of the block sees may hold anything (slots never written): they are zeroed in shared memory, since
// 0 x NaN is NaN in a product.
//
// 8192 new tokens of two sequences over 32768, 32 over 8 heads of 128: 2 770 us, 1.29 PFLOP/s, where the power limit holds the clock.
// 30 011 tokens, window 2048, 16 over 4 heads of 128: 542 us, 900 TFLOP/s of what the masks leave; 8 x 1024, window 256, 16 heads of 64:
// 43 us, a softmax step of 64 keys of two tiles 1 900 cycles (1 024 of exponentials) and 5 us of a thread block's start and end.  64
// single tokens over 16384, 32 over 4 heads of 128: 272 us, 5.8 TB/s, and 6 for joining five shares.
#include "attention_tile.cuh"

namespace {

using namespace tc05;
using namespace attn;

constexpr int kRows = 128;       // rows of a tile (TMEM lanes)
constexpr int kKeys = 128;       // keys of a block
constexpr int kNoWindow = 0x3fffffff;
enum { ATT_ERR_TIMEOUT = 501 };

struct FwdParams {
  int T;                  // dense: tokens of a sequence; paged: rows of q
  int B, kv_heads, group, tile_tokens;
  int window, sinks;
  const int* lengths;     // (B); null: T everywhere
  // paged
  const int* offsets;     // (B + 1); null: one new token each
  const int* tables;      // (B, max_pages)
  long long t_sb;
  int max_pages, page, pages, piece;
  int splits;
  float scale_log2;
  elem_t* out;            // (B, T, heads, D) or (rows, heads, D), contiguous
  float* lse;             // (B, kv_heads, tiles, 128): minus log2 of the sum of 2^(s scale log2(e)); null where no gradient is wanted
  int tiles;              // of a sequence
  float* part_o;          // (splits, rows, heads, D) and (splits, rows, heads): sums of a split and (reference, total)
  float2* part_ml;
  int* status;
};

// TILES = 2: two tiles a thread block, one thread block a multiprocessor: they share each key block.
// TILES = 1: one tile a thread block, two thread blocks a multiprocessor, where all of them fit at once (296).  One tile and two, heads of
// 64: 3 x 696 with a window of 2, 8 heads, 8.8 and 10.9 us; 150 tiles, window 256, 11.2 and 13.7, no window 26.6 and 33.2; 296 tiles 14.0 and
// 15.1, 18.6 and 22.5; 8 x 1024, window 256, 16 heads, where they do not fit, 59 and 43.  Heads of 128: 150 tiles 13.7 and 16.1, 33.4 and
// 32.7; 296 tiles 17.1 and 18.4, 24.2 and 24.8.  (With six slots of 64 channels a multiprocessor took one of them: 20.5 us for 296 tiles,
// window 256.)  Over a cache heads of 128 have no room for a page's way (two slots): 145 new tokens of ten sequences over 900, 16 over 8
// heads of 64 22.1 and 37.3, 8 over 4 of 128 26 and 23, which stay with two tiles.
// ONE: that tile is one token with up to 16 heads.  It has little to do for each key block that arrives, and two of them hide each
// other's waits.  Its Q keeps 16 rows a panel; what the product reads behind them are other buffers, in rows that nobody looks at.
constexpr int kResident = 296;
template <int D, int TILES, bool ONE>
constexpr int kSlots = TILES == 2 ? (D == 64 ? 8 : 5) : (D == 64 ? (ONE ? 6 : 5) : ONE ? 3 : 2);
template <bool ONE>
constexpr int kQPanel = ONE ? 16 * 128 : kRows * 128;              // bytes of 64 channels of a tile
template <int D, int TILES, bool ONE>
constexpr int fwd_smem_bytes() { return TILES * (D / 64) * kQPanel<ONE> + kSlots<D, TILES, ONE> * kKeys * D * 2 + 256 + 1024; }
// of a multiprocessor, which takes 1 KB for itself with each thread block
template <int D, int TILES, bool ONE>
constexpr bool kAllFit = (TILES == 2 ? 1 : 2) * (fwd_smem_bytes<D, TILES, ONE>() + 1024) <= 228 * 1024;
// STEP: keys whose scores a softmax thread has at a time.  64: the next 64 are scored meanwhile, beside them, and less is scored that
// the masks take away.  128: a product of 128 keys reads Q half as often, but the tensor memory has no room to score ahead; P V starts
// with the first 96 keys.  With heads of 128 the products count where the keys are many: 4 x 4096, 16 over 4 heads of 128, STEP 64 and
// 128: window 256 97 and 109 us, 1024 163 and 164, none 265 and 247; 32 over 8 heads of 128: 512 new tokens of eight sequences over 512
// 53 and 54, over 1024 70 and 68, over 2048 120 and 110, 2048 of two over 16384 893 and 777.
// Single tokens (ONE) have one warp at work and wait for memory: the fewer steps the better (64 sequences of 16384 tokens, 32 over 4
// heads of 128: 268 against 273 us; 100 of up to 2000, 16 over 4 heads of 64: 50 against 53).
template <int TILES, int STEP>
constexpr int kFwdThreads = TILES * 128 + (STEP == 128 ? 128 : 64);     // four softmax warps a tile; MMA issue; loads; for setmaxnreg two more
constexpr int kMost = 96;                                               // STEP 128: keys whose P V starts early

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// Queries of one tile, or of both, as the kernel needs them: token numbers within the sequence's new tokens.
struct Span {
  int p0, p1;      // positions of the first and the last valid query; p1 < p0: none
  int lo, hi;      // steps of keys of the window (first tokens apart)
};

template <int STEP>
__device__ __forceinline__ Span make_span(int i0, int i1, int base, int key_end, int window) {
  Span s;
  s.p0 = max(0, base + i0);
  s.p1 = base + i1 - 1;
  const int end = min(s.p1 + 1, key_end);
  if (i1 <= i0 || end <= 0) { s.p1 = s.p0 - 1; s.lo = 0; s.hi = -1; return s; }
  s.lo = max(0, s.p0 - window + 1) / STEP;
  s.hi = (end - 1) / STEP;
  return s;
}

template <int D, bool PAGED, int TILES, bool ONE, int STEP>
__global__ void __launch_bounds__(kFwdThreads<TILES, STEP>, TILES == 2 ? 1 : 2)
window_fwd_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                  const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out,
                  const __grid_constant__ CUtensorMap map_low, const __grid_constant__ FwdParams p) {
  constexpr int DP = D / 64;                 // 64-wide panels per row
  constexpr int kQBytes = DP * kQPanel<ONE>; // one tile
  constexpr int kKVBytes = kKeys * D * 2;
  constexpr int NS = kSlots<D, TILES, ONE>;
  constexpr uint32_t kTmemO = TILES * 128, kTmemCols = TILES * 256;   // S/P of each tile, 128 columns; then O of each, D
  constexpr int kMma = TILES * 4, kLoad = kMma + 1;   // warps
  constexpr int AHEAD = kKeys / STEP;        // steps of a block: so many are scored ahead, in so many places
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                        // TILES tiles
  uint8_t* sKV = sQ + TILES * kQBytes;       // NS slots: K and V of the blocks in turn
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + NS * kKVBytes);
  uint64_t* q_full = bars;
  uint64_t* full = bars + 1;                 // [NS]
  uint64_t* empty = full + NS;               // [NS]
  uint64_t* s_full = empty + NS;             // [tile][2]: of the steps in turn (STEP 128: the first)
  uint64_t* p_ready = s_full + 2 * TILES;    // [tile][2]: of the steps in turn (STEP 128: of the first 96 keys, of all)
  uint64_t* pv_full = p_ready + 2 * TILES;   // [tile][2]: as s_full
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_full + 2 * TILES);
  int* found = reinterpret_cast<int*>(tmem_slot + 1);   // sequence, pair

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.kv_heads * p.group;
  int b, pair, kvh, split = 0;
  const bool partial = PAGED && p.splits > 1;
  // rows that see nothing: zeros, or a part that adds nothing
  auto clear = [&](long long row0, int rows) {
    const int per = p.group * (D / 8);
    for (int i = threadIdx.x; i < rows * per; i += kFwdThreads<TILES, STEP>) {
      const int r = i % per;
      const long long at = (row0 + i / per) * heads + kvh * p.group + r / (D / 8);
      if (partial) {
        if (r % (D / 8) == 0) p.part_ml[(long long)split * p.T * heads + at] = make_float2(-INFINITY, 0.0f);
      } else {
        *reinterpret_cast<uint4*>(p.out + at * D + r % (D / 8) * 8) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  if constexpr (PAGED) {
    kvh = blockIdx.y;
    split = blockIdx.z;
    if (p.offsets == nullptr) {
      b = blockIdx.x;
      pair = 0;
    } else {
      if (blockIdx.x == 0) {             // rows in front of the first sequence: none, as a rule
        const int front = min(p.offsets[0], p.T);
        for (int t = 0; t < front; t += kRows) clear(t, min(kRows, front - t));
      }
      // which sequence this block's pair of tiles belongs to; the rows behind the last sequence count as one more, without keys
      if (warp == 0) {
        int before = 0, at = -1, which = 0;
        for (int b0 = 0; b0 <= p.B && at < 0; b0 += 32) {
          const int i = b0 + lane;
          int pairs = 0;
          if (i <= p.B) {
            const int r0 = min(max(p.offsets[i], 0), p.T), r1 = i < p.B ? min(max(p.offsets[i + 1], r0), p.T) : p.T;
            pairs = (r1 - r0 + TILES * p.tile_tokens - 1) / (TILES * p.tile_tokens);
          }
          int sum = pairs;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += v;
          }
          const unsigned hit = __ballot_sync(0xffffffffu, (int)blockIdx.x < before + sum);
          if (hit) {
            const int first = __ffs(hit) - 1;
            at = b0 + first;
            which = (int)blockIdx.x - (before + __shfl_sync(0xffffffffu, sum - pairs, first));
          }
          before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) { found[0] = at; found[1] = which; }
      }
      __syncthreads();
      b = found[0];
      pair = found[1];
      if (b < 0) return;
    }
  } else {
    // the last tokens of all sequences first: without a window they see the most keys
    const int bh = blockIdx.x % (p.B * p.kv_heads);
    b = bh / p.kv_heads;
    kvh = bh % p.kv_heads;
    pair = (p.T + TILES * p.tile_tokens - 1) / (TILES * p.tile_tokens) - 1 - blockIdx.x / (p.B * p.kv_heads);
  }
  // this sequence: its rows, where its queries stand, where its keys end
  int row0 = 0, n_rows = p.T, n_valid = p.T, base = 0, key_end;
  if constexpr (PAGED) {
    if (p.offsets == nullptr) {
      row0 = b;
      n_rows = 1;
    } else {
      row0 = min(max(p.offsets[b], 0), p.T);
      n_rows = (b < p.B ? min(max(p.offsets[b + 1], row0), p.T) : p.T) - row0;
    }
    n_valid = n_rows;
    const int length = b < p.B ? max(p.lengths[b], 0) : 0;
    base = length - n_rows;
    key_end = (int)min((long long)length, (long long)p.max_pages * p.page);
  } else {
    if (p.lengths != nullptr) n_valid = min(max(p.lengths[b], 0), p.T);
    key_end = n_valid;
  }
  const int tok0 = pair * TILES * p.tile_tokens;
  Span span[TILES];
#pragma unroll
  for (int g = 0; g < TILES; ++g)
    span[g] = make_span<STEP>(tok0 + g * p.tile_tokens, min(tok0 + (g + 1) * p.tile_tokens, n_valid), base, key_end, p.window);
  const Span both = make_span<STEP>(tok0, min(tok0 + TILES * p.tile_tokens, n_valid), base, key_end, p.window);
  const int near = max(0, both.p0 - p.window + 1), end = min(both.p1 + 1, key_end);       // what both tiles see together:
  const int sink_end = min(p.sinks, end);                                                  // [0, sink_end) and [near, end)
  const int lo = both.lo * STEP / kKeys, hi = both.hi < 0 ? -1 : both.hi * STEP / kKeys;  // blocks of its window
  const int ns = min((p.sinks + kKeys - 1) / kKeys, hi + 1);                               // blocks with first tokens
  const int range0 = max(lo, ns);
  const int listed = ns + max(0, hi - range0 + 1);                                    // a table may end in front of the window
  int c0 = 0, c1 = listed;
  if (PAGED && p.splits > 1) {
    c0 = (int)((long long)listed * split / p.splits);
    c1 = (int)((long long)listed * (split + 1) / p.splits);
  }
  auto block_of = [&](int c) { return c < ns ? c : c - ns + range0; };
  const int sink_steps = (p.sinks + STEP - 1) / STEP;
  auto needed = [&](const Span& s, int step) { return step <= s.hi && (step < sink_steps || step >= s.lo); };

  if (c0 >= c1) {                              // no keys
    clear((PAGED ? (long long)row0 : (long long)b * p.T) + tok0, min(tok0 + TILES * p.tile_tokens, n_rows) - tok0);
    return;
  }

  if (threadIdx.x == 0) {
    prefetch_tensormap(&map_q);
    prefetch_tensormap(&map_k);
    prefetch_tensormap(&map_v);
    mbar_init(q_full, 1);
    for (int s = 0; s < NS; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int g = 0; g < 2 * TILES; ++g) {
      mbar_init(&s_full[g], 1);
      mbar_init(&p_ready[g], 4);
      mbar_init(&pv_full[g], 1);
    }
    mbar_fence_init();
  }
  if (warp == kMma) { tmem_alloc(tmem_slot, kTmemCols); tmem_relinquish(); }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  // With 128 scores a thread registers go where the scores are, four warps at a time (launched with 168 a thread for
  // two tiles, with 128 for one).
  if (warp >= kMma) {
    if constexpr (STEP == 128 && TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if constexpr (STEP == 128 && TILES == 1) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == kLoad) {
      // ---------------------------------------------------------------- loads
      bool ok = true;
      if (lane == 0) {
        const int tiles = span[TILES - 1].hi >= 0 ? TILES : 1;
        mbar_expect_tx(q_full, tiles * p.tile_tokens * p.group * D * 2);
        for (int g = 0; g < tiles; ++g)
#pragma unroll
          for (int j = 0; j < DP; ++j)           // rows beyond the tensor are filled with zeros
            tma_load_4d(sQ + g * kQBytes + j * kQPanel<ONE>, &map_q, q_full, j * 64, kvh * p.group, row0 + tok0 + g * p.tile_tokens,
                        PAGED ? 0 : b);
      }
      // the page (or part of it) that this lane fetches of a block; the number of pages where there is nothing to fetch
      auto look_up = [&](int kb) {
        const int key = kb * kKeys + lane * p.piece;
        int id = -1;
        if (lane * p.piece < kKeys && key < end && (key < sink_end || key + p.piece > near)) {
          const int at = key / p.page;
          if (at < p.max_pages) id = p.tables[b * p.t_sb + at];
        }
        return id < 0 || id >= p.pages ? p.pages : id;
      };
      int next = 0;
      if (PAGED) next = look_up(block_of(c0));
      for (int c = c0; c < c1 && ok; ++c) {
        const int kb = block_of(c), id = next;
        if (PAGED && c + 1 < c1) next = look_up(block_of(c + 1));
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const int f = 2 * (c - c0) + kv, s = f % NS;
          if (f >= NS && !mbar_wait(&empty[s], (f / NS - 1) & 1)) { ok = false; break; }
          const CUtensorMap* map = kv ? &map_v : &map_k;
          if (lane == 0) mbar_expect_tx(&full[s], kKVBytes);
          __syncwarp();
          if constexpr (PAGED) {
            if (lane * p.piece < kKeys) {
              const int slot = (kb * kKeys + lane * p.piece) % p.page;
#pragma unroll
              for (int j = 0; j < DP; ++j)
                tma_load_4d(sKV + s * kKVBytes + j * kKeys * 128 + lane * p.piece * 128, map, &full[s], j * 64, kvh, slot, id);
            }
          } else if (lane == 0) {
#pragma unroll
            for (int j = 0; j < DP; ++j) tma_load_4d(sKV + s * kKVBytes + j * kKeys * 128, map, &full[s], j * 64, kvh, kb * kKeys, b);
          }
        }
      }
      if (!ok && lane == 0) atomicExch(p.status, ATT_ERR_TIMEOUT);
    } else if (warp == kMma) {
      // ---------------------------------------------------------------- products
      if (elect_one()) {
        const uint32_t idesc_s = make_idesc_f16kind(128, STEP, false, false);
        const uint32_t idesc_pv = make_idesc_f16kind(128, D, false, true);   // B = V is MN-major
        auto wait_full = [&](int f) { return mbar_wait(&full[f % NS], (f / NS) & 1); };
        const uint64_t kQ = k_major(smem_u32(sQ)), kKV = k_major(smem_u32(sKV)), mKV = mn_major(smem_u32(sKV));
        int scored[TILES] = {}, added[TILES] = {};   // steps of each tile whose S, whose P V has been issued
        auto issue_s = [&](int g, int t) {       // S_g = Q_g K^T, 64 keys
          const int f = 2 * (t / AHEAD), turn = scored[g]++ % AHEAD;
          const uint64_t a = kQ + g * (kQBytes >> 4), bk = kKV + ((f % NS * kKVBytes + t % AHEAD * (STEP * 128)) >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_f16_ss(tmem + g * 128 + turn * STEP, a + ((k / 4 * kQPanel<ONE> + k % 4 * 32) >> 4), bk + k_step(k), idesc_s, k != 0);
          mma_commit(&s_full[2 * g + turn]);
        };
        auto issue_pv = [&](int g, int t) {      // O_g (+)= P_g V
          const int f = 2 * (t / AHEAD) + 1, nth = added[g]++;
          const uint64_t bv = mKV + (f % NS * kKVBytes >> 4);
#pragma unroll
          for (int k = 0; k < (STEP == 128 ? kMost : STEP) / 16; ++k)
            mma_f16_ts(tmem + kTmemO + g * D, tmem + g * 128 + nth % AHEAD * STEP + k * 8, bv + mn_step(t % AHEAD * (STEP / 16) + k), idesc_pv,
                       nth != 0 || k != 0);
          if constexpr (STEP == 128) {
            if (!mbar_wait(&p_ready[2 * g + 1], nth & 1)) return false;
            fence_after_sync();
#pragma unroll
            for (int k = kMost / 16; k < STEP / 16; ++k)
              mma_f16_ts(tmem + kTmemO + g * D, tmem + g * 128 + k * 8, bv + mn_step(k), idesc_pv, true);
          }
          mma_commit(&pv_full[2 * g + nth % AHEAD]);
          return true;
        };
        const int steps = AHEAD * (c1 - c0);
        auto wants = [&](int g, int t) { return t < steps && needed(g == 0 ? span[0] : span[TILES - 1], block_of(c0 + t / AHEAD) * AHEAD + t % AHEAD); };
        bool ok = mbar_wait(q_full, 0) && wait_full(0);
        if (ok) {
          fence_after_sync();
          for (int t = 0; t < AHEAD; ++t)
            for (int g = 0; g < TILES; ++g)
              if (wants(g, t)) issue_s(g, t);
          mma_commit(&empty[0]);
        }
        // S of a tile's next step is there before the softmax is done with this one: two steps' scores lie beside each other.
        for (int t = 0; t < steps && ok; ++t) {
          const int f = 2 * (t / AHEAD);
          if (t % AHEAD == 0 && !wait_full(f + 1)) { ok = false; break; }
#pragma unroll
          for (int g = 0; g < TILES; ++g) {
            if (wants(g, t)) {
              if (!mbar_wait(&p_ready[2 * g + added[g] % AHEAD], (added[g] / AHEAD) & 1)) { ok = false; break; }
              fence_after_sync();
              if (!issue_pv(g, t)) { ok = false; break; }
            }
            if (g == 0 && t % AHEAD == 0 && t + AHEAD < steps) {
              if (!wait_full(f + 2)) { ok = false; break; }
              fence_after_sync();
            }
            if (wants(g, t + AHEAD)) issue_s(g, t + AHEAD);      // over P of the step that has been added
          }
          if (ok && t % AHEAD == AHEAD - 1) {
            mma_commit(&empty[(f + 1) % NS]);
            if (t + AHEAD < steps) mma_commit(&empty[(f + 2) % NS]);
          }
        }
        if (!ok) atomicExch(p.status, ATT_ERR_TIMEOUT);
      }
    }
  } else {
    if constexpr (STEP == 128 && TILES == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    if constexpr (STEP == 128 && TILES == 1) asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ---------------------------------------------------------------- softmax / output threads of one tile
    const int g = warp >> 2;                         // tile of this warp group
    const int lane_group = warp & 3;                 // TMEM lane quarter this warp may access
    const int row = lane_group * 32 + lane;
    const int token = row / p.group;
    const int i = tok0 + g * p.tile_tokens + token;  // the row's token among the sequence's new ones
    const int pos = base + i;
    const bool stored = token < p.tile_tokens && i < n_rows;
    const bool valid = stored && i < n_valid && pos >= 0;
    const uint32_t lane_addr = uint32_t(lane_group * 32) << 16;
    const uint32_t tmem_pv = tmem + kTmemO + g * D;
    const Span mine = g == 0 ? span[0] : span[TILES - 1];
    const bool idle = ONE && lane_group * 32 >= p.group;   // rows that nobody looks at
    // m is the reference of the exponentials accumulated so far: p = 2^((s - m) scale).  It follows the running row maximum only
    // when that has moved by more than 2^8 past it, so that the output accumulator is rescaled on a few blocks only (values of p
    // stay below 2^8, far inside the 16-bit range; the final division by the row sum uses the same reference).
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    int it = 0;
    for (int t = 0; t < AHEAD * (c1 - c0); ++t) {
      const int step = block_of(c0 + t / AHEAD) * AHEAD + t % AHEAD;
      if (!needed(mine, step)) continue;
      const int k0 = step * STEP;
      const uint32_t tmem_s = tmem + g * 128 + it % AHEAD * STEP;
      if (!mbar_wait(&s_full[2 * g + it % AHEAD], (it / AHEAD) & 1)) { ok = false; break; }
      fence_after_sync();
      if ((k0 + STEP > end || (k0 < near && k0 + STEP > sink_end)) && (g == 0 || !needed(span[0], step))) {
        // rows of V that no query of this block sees; the first tile's P V goes ahead of the second's.  S of this step is there, so V of
        // the block before has been: a wait on V's barrier any earlier could take the phase before for this one.  Eight lanes a row:
        // with a row a lane all lanes met in the same banks, 4 000 cycles a block.
        const int f = 2 * (t / AHEAD) + 1;
        if (!mbar_wait(&full[f % NS], (f / NS) & 1)) { ok = false; break; }
#pragma unroll
        for (int at = 0; at < STEP / 4; at += 4) {
          const int r = lane_group * (STEP / 4) + at + lane / 8, key = k0 + r;
          if (key >= end || (key < near && key >= sink_end)) {
#pragma unroll
            for (int j = 0; j < DP; ++j)
              *reinterpret_cast<uint4*>(sKV + f % NS * kKVBytes + (j * kKeys + t % AHEAD * STEP + r) * 128 + lane % 8 * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        fence_proxy_async_smem();
      }
      if (idle) {
        warp_arrive(&p_ready[2 * g + it % AHEAD]);
        if (STEP == 128) warp_arrive(&p_ready[2 * g + 1]);
        ++it;
        continue;
      }
      uint32_t r[STEP];
#pragma unroll
      for (int j = 0; j < STEP; j += 32) tmem_ld_32x32(tmem_s + lane_addr + j, *reinterpret_cast<uint32_t(*)[32]>(r + j));
      tmem_ld_wait();
      // Masking is a pass of its own that only steps on an edge take.
      if (k0 + STEP > min(mine.p0 + 1, key_end) || (k0 <= mine.p1 - p.window && k0 + STEP > p.sinks)) {
        const int hi = min(pos + 1, key_end) - k0, lo = pos - p.window + 1 - k0, first = p.sinks - k0;
        auto below = [](int c) { return c <= 0 ? 0u : c >= 32 ? 0xffffffffu : (1u << c) - 1u; };
#pragma unroll
        for (int w = 0; w < STEP / 32; ++w) {
          const uint32_t seen = below(hi - w * 32) & (~below(lo - w * 32) | below(first - w * 32));
#pragma unroll
          for (int j = 0; j < 32; ++j) r[w * 32 + j] = seen & (1u << j) ? r[w * 32 + j] : 0xff800000u;      // -inf
        }
      }
      // The maximum is NaN where a score is: then the reference, and with it every exponential of the row, is NaN.
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < STEP; j += 2) mx4[j / 2 & 3] = max3_nan(mx4[j / 2 & 3], __uint_as_float(r[j]), __uint_as_float(r[j + 1]));
      const float m_blk = max3_nan(max3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]);
      const bool grow = valid && !((m_blk - m) * p.scale_log2 <= 8.0f);      // true on the first block of any visible key
      float alpha = 1.0f;
      if (grow) {
        alpha = (m == -INFINITY) ? 0.0f : fast_exp2((m - m_blk) * p.scale_log2);
        m = m_blk;
      }
      const float m_use = (m == -INFINITY) ? 0.0f : m;
      if (it > 0 && __any_sync(0xffffffffu, grow)) {
        // some row of this warp moved its reference: scale the accumulated output rows, once the step before has been added
        if (!mbar_wait(&pv_full[2 * g + (it - 1) % AHEAD], ((it - 1) / AHEAD) & 1)) { ok = false; break; }
        fence_after_sync();
        const float2 a2 = make_float2(alpha, alpha);
#pragma unroll 1
        for (int d0 = 0; d0 < D; d0 += 32) {
          uint32_t ro[32];
          tmem_ld_32x32(tmem_pv + lane_addr + d0, ro);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 v = __fmul2_rn(make_float2(__uint_as_float(ro[j]), __uint_as_float(ro[j + 1])), a2);
            ro[j] = __float_as_uint(v.x);
            ro[j + 1] = __float_as_uint(v.y);
          }
          tmem_st_32x32(tmem_pv + lane_addr + d0, ro);
        }
      }
      // p = 2^(s scale - m scale): one packed multiply-add per pair, then the exponential; the row sum is taken over the fp32
      // values.  P is rounded to 16 bits as an operand of the second product (half a step of its type, relative to values whose
      // largest is near 1).  The special-function units form four exponentials a cycle and quarter of a
      // multiprocessor: 1 024 cycles for 64 keys of two tiles, of the 1 900 that a step takes.  A part of them by a polynomial on the
      // other units gained nothing with two warps a quarter, and where the power limit holds the clock it lost (3 420 against 3 120 us
      // for 8192 tokens over 32768).
      const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
      const float nm = -m_use * p.scale_log2;
      const float2 nm2 = make_float2(nm, nm);
      float2 rs2 = make_float2(0.0f, 0.0f), rs2b = make_float2(0.0f, 0.0f);
#pragma unroll
      for (int part = 0; part < STEP / 32; ++part) {
        uint32_t packed[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int at = part * 32 + 2 * j;
          const float2 e = __ffma2_rn(make_float2(__uint_as_float(r[at]), __uint_as_float(r[at + 1])), sc2, nm2);
          const float2 pe = make_float2(fast_exp2(e.x), fast_exp2(e.y));
          if (j & 1) rs2b = __fadd2_rn(rs2b, pe); else rs2 = __fadd2_rn(rs2, pe);
          elem2_t h = f22e2(pe);
          packed[j] = *reinterpret_cast<uint32_t*>(&h);
        }
        tmem_st_32x16(tmem_s + lane_addr + part * 16, packed);
        if (STEP == 128 && part == kMost / 32 - 1) {
          tmem_st_wait();
          fence_before_sync();
          warp_arrive(&p_ready[2 * g]);
        }
      }
      l = l * alpha + ((rs2.x + rs2.y) + (rs2b.x + rs2b.y));
      tmem_st_wait();
      fence_before_sync();
      warp_arrive(&p_ready[STEP == 128 ? 2 * g + 1 : 2 * g + it % AHEAD]);
      ++it;
    }
    // the last product completes the output rows in tensor memory: divide by the row sum and store
    if (it > 0 && ok && !mbar_wait(&pv_full[2 * g + (it - 1) % AHEAD], ((it - 1) / AHEAD) & 1)) ok = false;
    fence_after_sync();
    {                                            // also after a wait that expired: the tile's warps meet below
      const long long at_row = (PAGED ? (long long)row0 : (long long)b * p.T) + i;
      const long long at = at_row * heads + kvh * p.group + (row - token * p.group);
      if (!valid) l = 0.0f;
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      const float2 inv2 = make_float2(inv, inv);
      if constexpr (PAGED) {
#pragma unroll 1
        for (int d0 = 0; d0 < D; d0 += 32) {
          uint32_t r[32];
          if (it > 0) {
            tmem_ld_32x32(tmem_pv + lane_addr + d0, r);
            tmem_ld_wait();
          }
          if (it == 0 || l == 0.0f) {            // nothing seen
#pragma unroll
            for (int j = 0; j < 32; ++j) r[j] = 0u;
          }
          if (stored) {
            if (partial) {
              float4* dst = reinterpret_cast<float4*>(p.part_o + ((long long)split * p.T * heads + at) * D + d0);
#pragma unroll
              for (int j = 0; j < 8; ++j)
                dst[j] = make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]),
                                     __uint_as_float(r[4 * j + 3]));
            } else {
#pragma unroll
              for (int d = 0; d < 32; d += 8) {
                __align__(16) elem2_t hh[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  hh[q] = f22e2(__fmul2_rn(make_float2(__uint_as_float(r[d + 2 * q]), __uint_as_float(r[d + 2 * q + 1])), inv2));
                *reinterpret_cast<uint4*>(p.out + at * D + d0 + d) = *reinterpret_cast<uint4*>(hh);
              }
            }
          }
        }
      } else {
        // Whole tiles go out by the copy engine, from the tile's Q, which its products have read; rows behind T are cut off.  With a
        // gradient to come, what the rounding took off goes out as well: delta = sum dO O from the rounded output alone was the largest
        // error of the gradients where few keys are seen.
        const int passes = p.lse != nullptr ? 2 : 1;
        for (int pass = 0; pass < passes; ++pass) {
#pragma unroll 1
          for (int d0 = 0; d0 < D; d0 += 32) {
            uint32_t r[32];
            if (it > 0) {
              tmem_ld_32x32(tmem_pv + lane_addr + d0, r);
              tmem_ld_wait();
            }
            if (it == 0 || l == 0.0f) {
#pragma unroll
              for (int j = 0; j < 32; ++j) r[j] = 0u;
            }
#pragma unroll
            for (int d = 0; d < 32; d += 8) {
              __align__(16) elem2_t hh[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float2 o = __fmul2_rn(make_float2(__uint_as_float(r[d + 2 * q]), __uint_as_float(r[d + 2 * q + 1])), inv2);
                hh[q] = f22e2(o);
                if (pass) {
                  const float2 rounded = e22ff(hh[q]);
                  hh[q] = ff2e2(o.x - rounded.x, o.y - rounded.y);
                }
              }
              *reinterpret_cast<uint4*>(sQ + g * kQBytes + d0 / 64 * kQPanel<ONE> + swz(row, d0 % 64 / 8 + d / 8)) = *reinterpret_cast<uint4*>(hh);
            }
          }
          fence_proxy_async_smem();
          asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");   // the tile's warps
          if (lane_group == 0 && tok0 + g * p.tile_tokens < p.T && elect_one()) {
#pragma unroll
            for (int j = 0; j < DP; ++j)
              tma_store_4d(pass ? &map_low : &map_out, sQ + g * kQBytes + j * kQPanel<ONE>, j * 64, kvh * p.group, tok0 + g * p.tile_tokens, b);
            bulk_commit_group();
            bulk_wait_group_read<0>();
          }
          if (pass + 1 < passes) {
            asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory");
          }
        }
      }
      if (stored) {
        if (partial) {
          p.part_ml[(long long)split * p.T * heads + at] = make_float2(l == 0.0f ? -INFINITY : m * p.scale_log2, l);
        } else if (!PAGED && p.lse != nullptr) {
          p.lse[(((long long)b * p.kv_heads + kvh) * p.tiles + pair * TILES + g) * kRows + row] = l == 0.0f ? 0.0f : -(m * p.scale_log2 + log2f(l));
        }
      }
    }
    fence_before_sync();
    if (!ok && lane == 0) atomicExch(p.status, ATT_ERR_TIMEOUT);
  }
  fence_before_sync();
  __syncthreads();
  if (warp == kMma) { fence_after_sync(); tmem_dealloc(tmem, kTmemCols); }
}

// Partial sums of a row's splits to its output: a warp a row.  With each split's reference m_s and total l_s,
// o = sum o_s 2^(m_s - M) / sum l_s 2^(m_s - M).  The order of the sums is that of the splits.
template <int D>
__global__ void __launch_bounds__(256) window_join_kernel(const float* part_o, const float2* part_ml, elem_t* out, long long rows, int splits) {
  constexpr int V = D / 32;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, part_ml[s * rows + row].x);
  float total = 0.0f, o[V];
#pragma unroll
  for (int v = 0; v < V; ++v) o[v] = 0.0f;
  for (int s = 0; s < splits; ++s) {
    const float2 ml = part_ml[s * rows + row];
    if (ml.y == 0.0f) continue;                // its sums were not written
    const float w = exp2f(ml.x - top);
    total += ml.y * w;
    const float* src = part_o + (s * rows + row) * D + lane * V;
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] += src[v] * w;
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  elem_t* dst = out + row * D + lane * V;
#pragma unroll
  for (int v = 0; v < V; v += 2) *reinterpret_cast<elem2_t*>(dst + v) = ff2e2(o[v] * inv, o[v + 1] * inv);
}

template <int D, bool PAGED, int TILES, bool ONE, int STEP>
int launch(dim3 grid, cudaStream_t s, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& out, const CUtensorMap& low,
           const FwdParams& p) {
  constexpr int smem = fwd_smem_bytes<D, TILES, ONE>();
  static_assert(kAllFit<D, TILES, ONE>, "as many thread blocks a multiprocessor as the launch bounds say");
  if (set_smem_once<window_fwd_kernel<D, PAGED, TILES, ONE, STEP>>(smem)) return 5;
  window_fwd_kernel<D, PAGED, TILES, ONE, STEP><<<grid, kFwdThreads<TILES, STEP>, smem, s>>>(q, k, v, out, low, p);
  return 0;
}

// STEP 128: by the keys that a pair of tiles sees at most.
bool far_enough(long long keys, int D) { return D == 128 && keys >= 1536; }

}  // namespace

extern "C" {

// q (B, T, heads, D), k and v (B, T, kv_heads, D) with element strides each; out contiguous; lse fp32 (B, kv_heads, tiles, 128) or
// null, where a tile has 128 / group tokens, and with it low like out: what rounding took off out; lengths (B) or null.
int fbam_window_fwd(const void* q, long long q_sb, long long q_st, long long q_sh, const void* k, const void* v, long long k_sb,
                    long long k_st, long long k_sh, long long v_sb, long long v_st, long long v_sh, void* out, void* low, float* lse,
                    const int* lengths, int B, int T, int kv_heads, int group, int D, int window, int sinks, float scale, int* status,
                    void* stream) {
  if ((D != 64 && D != 128) || B < 1 || T < 1 || kv_heads < 1 || group < 1 || group > kRows || sinks < 0) return 1;
  FwdParams p = {};
  p.T = T; p.B = B; p.kv_heads = kv_heads; p.group = group;
  p.tile_tokens = kRows / group;
  p.window = window < 1 || window > kNoWindow ? kNoWindow : window;   // 0: none
  p.sinks = p.window == kNoWindow ? 0 : sinks < kNoWindow ? sinks : kNoWindow;
  p.lengths = lengths;
  p.splits = 1;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = (elem_t*)out;
  p.lse = lse;
  p.tiles = (T + p.tile_tokens - 1) / p.tile_tokens;
  p.status = status;
  const long long tiles = (long long)p.tiles * B * kv_heads;
  const bool one_tile = tiles <= kResident;
  const int per = (one_tile ? 1 : 2) * p.tile_tokens;
  const long long blocks = (long long)((T + per - 1) / per) * B * kv_heads;
  if (blocks > 0x7fffffffll) return 1;
  const int heads = kv_heads * group;
  const long long o_sb = (long long)T * heads * D;
  CUtensorMap mq, mk, mv, mo, ml;
  int e;
  if ((e = encode_heads(&mq, q, D, kv_heads * group, T, B, q_sh, q_st, q_sb, group, p.tile_tokens))) return e;
  if ((e = encode_heads(&mk, k, D, kv_heads, T, B, k_sh, k_st, k_sb, 1, kKeys))) return e;
  if ((e = encode_heads(&mv, v, D, kv_heads, T, B, v_sh, v_st, v_sb, 1, kKeys))) return e;
  if ((e = encode_heads(&mo, out, D, heads, T, B, D, heads * D, o_sb, group, p.tile_tokens))) return e;
  if ((e = encode_heads(&ml, lse != nullptr ? low : out, D, heads, T, B, D, heads * D, o_sb, group, p.tile_tokens))) return e;
  const unsigned grid = (unsigned)blocks;
  cudaStream_t s = (cudaStream_t)stream;
  const bool wide = far_enough((long long)p.window + per < T ? p.window + per : T, D);
  if (one_tile ? (D == 64 ? launch<64, false, 1, false, 64>(grid, s, mq, mk, mv, mo, ml, p) : launch<128, false, 1, false, 64>(grid, s, mq, mk, mv, mo, ml, p))
      : D == 64 ? launch<64, false, 2, false, 64>(grid, s, mq, mk, mv, mo, ml, p)
      : wide    ? launch<128, false, 2, false, 128>(grid, s, mq, mk, mv, mo, ml, p)
                : launch<128, false, 2, false, 64>(grid, s, mq, mk, mv, mo, ml, p))
    return 5;
  return cudaGetLastError() == cudaSuccess ? 0 : 5;
}

// q (rows, heads, D) with strides; pages (pages, page, kv_heads, D) with strides; tables (B, max_pages) with stride t_sb; lengths
// (B); offsets (B + 1) or null (rows == B); out contiguous.  With splits > 1 part_o (splits, rows, heads, D) and part_ml (splits,
// rows, heads, 2) fp32.
int fbam_cache_attention(const void* q, long long q_st, long long q_sh, const void* k_pages, long long k_sp, long long k_ss, long long k_sh,
                         const void* v_pages, long long v_sp, long long v_ss, long long v_sh, const int* tables, long long t_sb,
                         const int* lengths, const int* offsets, void* out, float* part_o, void* part_ml, int splits, int rows, int B,
                         int max_pages, int page, int pages, int kv_heads, int group, int D, int window, int sinks, float scale,
                         int* status, void* stream) {
  if ((D != 64 && D != 128) || B < 1 || rows < 1 || kv_heads < 1 || group < 1 || group > kRows || sinks < 0 || splits < 1 || pages < 1 ||
      page < 8 || page % 8 || max_pages < 0 || splits > 65535 || kv_heads > 65535)
    return 1;
  FwdParams p = {};
  p.T = rows; p.B = B; p.kv_heads = kv_heads; p.group = group;
  p.tile_tokens = kRows / group;
  p.window = window < 1 || window > kNoWindow ? kNoWindow : window;   // 0: none
  p.sinks = p.window == kNoWindow ? 0 : sinks < kNoWindow ? sinks : kNoWindow;
  p.lengths = lengths; p.offsets = offsets; p.tables = tables; p.t_sb = t_sb;
  p.max_pages = max_pages; p.page = page; p.pages = pages;
  p.piece = page;                            // slots of one copy: the largest power of two in a page, 128 at most
  for (int r = 128; r >= 8; r >>= 1)
    if (page % r == 0) { p.piece = r; break; }
  p.splits = splits;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.out = (elem_t*)out;
  p.part_o = part_o;
  p.part_ml = (float2*)part_ml;
  p.status = status;
  if (((uintptr_t)out | (uintptr_t)part_o | (uintptr_t)part_ml) & 15) return 2;
  // pairs of tiles: one a sequence without offsets; with them, at most one that is not full of each sequence
  const bool single = offsets == nullptr && group <= 16;
  if (single) p.tile_tokens = 1;
  const long long spare = (rows < B ? rows : B) + 1;
  const bool one_tile = D == 64 && !single && splits == 1 && (rows / p.tile_tokens + spare) * kv_heads <= kResident;
  const int per = (one_tile ? 1 : 2) * p.tile_tokens;
  const long long pairs = offsets == nullptr ? B : rows / per + spare;
  int e;
  CUtensorMap mq, mk, mv;
  if ((e = encode_heads(&mq, q, D, kv_heads * group, rows, 1, q_sh, q_st, (long long)rows * q_st, group, p.tile_tokens))) return e;
  if ((e = encode_heads(&mk, k_pages, D, kv_heads, page, pages, k_sh, k_ss, k_sp, 1, p.piece))) return e;
  if ((e = encode_heads(&mv, v_pages, D, kv_heads, page, pages, v_sh, v_ss, v_sp, 1, p.piece))) return e;
  cudaStream_t s = (cudaStream_t)stream;
  const dim3 grid((unsigned)pairs, kv_heads, splits);
  const long long most = (long long)max_pages * page;
  const bool wide = far_enough((long long)p.window + per < most ? p.window + per : most, D);
  if (single     ? (D == 64 ? launch<64, true, 1, true, 128>(grid, s, mq, mk, mv, mq, mq, p) : launch<128, true, 1, true, 128>(grid, s, mq, mk, mv, mq, mq, p))
      : one_tile ? launch<64, true, 1, false, 64>(grid, s, mq, mk, mv, mq, mq, p)
      : D == 64  ? launch<64, true, 2, false, 64>(grid, s, mq, mk, mv, mq, mq, p)
      : wide     ? launch<128, true, 2, false, 128>(grid, s, mq, mk, mv, mq, mq, p)
                 : launch<128, true, 2, false, 64>(grid, s, mq, mk, mv, mq, mq, p))
    return 5;
  if (splits > 1) {
    const long long all = (long long)rows * kv_heads * group;
    const unsigned blocks = (unsigned)((all + 7) / 8);
    if (D == 64)
      window_join_kernel<64><<<blocks, 256, 0, s>>>(part_o, p.part_ml, p.out, all, splits);
    else
      window_join_kernel<128><<<blocks, 256, 0, s>>>(part_o, p.part_ml, p.out, all, splits);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 5;
}

}  // extern "C"
