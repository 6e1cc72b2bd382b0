// Token embedding: out[i] = scale * table[id_i], and the table's gradient
//   d_table[v] = scale * sum over { i : id_i = v } of d_out[i],
// summed in fp32 in an order that the ids alone fix, so equal inputs give equal bits.  An id outside [0, vocab) gives a
// row of zeros and has no gradient.
//
// Gradient:
//   1. embed_sort_kernel  stable radix sort of (id, position) by one cluster of CTAs.  Meanwhile the other clusters of the same
//                         launch write the rows that no id names;
//   2. embed_sum_kernel   the sorted order is cut into pieces of kPiece entries; a piece sums its runs of equal ids.  A run
//                         that lies inside the piece is the row's gradient, one that crosses an edge leaves a partial sum;
//   3. the same kernel on the partial sums, two entries a piece in the order of the pieces, until there is one piece.  A
//      piece leaves two entries of its 32, so that takes log16 of the number of tokens steps, however common an id is.
//
// Bound by memory, and below some ten thousand tokens by the latency of four launches.  Four rows are on their way at once in a
// look-up (65536 rows of 2048 from fp32 to bf16: 86 us, 4.9 TB/s of DRAM traffic); a piece's keys and positions come through
// shared memory so that eight rows can be.  The gradient of the same, 100003 rows of fp32, takes 220 us: sort and 655 MB of zeros,
// then the first sums (73 us: 270 MB read, 150 written) and their partial sums, a sixteenth of the rows at most and taken 32 at a
// time by few CTAs (14 + 8 + 7 us).  Each step of the sums starts while the one before it ends.
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "elem16.cuh"
#include "gemm_tcgen05.h"

namespace {

constexpr int kPiece = 32;        // sorted positions of one piece
constexpr int kSumThreads = 128, kMinLanes = 8;
constexpr int kDigitBits = 10;
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kMaxSortCtas = 16;
constexpr int kAbsentWords = 4096;      // of 32 ids each, that a cluster looks for at once

template <int N>
struct Vals { float v[N]; };

// N values as they lie in memory
template <typename T, int N>
struct Raw {
  static constexpr int kWords = sizeof(T) * N / 16;
  uint4 w[kWords];
  // SHARED: the memory is written while kernels that read it are already resident, so it is read from L2
  template <bool SHARED = false>
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i)
      w[i] = SHARED ? __ldcg(reinterpret_cast<const uint4*>(p) + i) : __ldg(reinterpret_cast<const uint4*>(p) + i);
  }
  __device__ __forceinline__ Vals<N> get() const {
    Vals<N> r;
    if constexpr (sizeof(T) == 2) {
      const elem2_t* h = reinterpret_cast<const elem2_t*>(w);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 f = e22ff(h[i]);
        r.v[2 * i] = f.x; r.v[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) r.v[i] = reinterpret_cast<const float*>(w)[i];
    }
    return r;
  }
};
template <typename T>
struct Raw<T, 1> {
  T v;
  template <bool SHARED = false>
  __device__ __forceinline__ void load(const T* p) { v = SHARED ? __ldcg(p) : __ldg(p); }
  __device__ __forceinline__ Vals<1> get() const {
    if constexpr (sizeof(T) == 2) return {{e2f(v)}};
    else return {{v}};
  }
};
template <int N>
__device__ __forceinline__ void store_vals(float* p, const Vals<N>& r) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(r.v[i], r.v[i + 1], r.v[i + 2], r.v[i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = r.v[i];
  }
}
template <int N>
__device__ __forceinline__ void store_vals(elem_t* p, const Vals<N>& r) {
  if constexpr (N % 4 == 0) {
    __align__(16) elem2_t h[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) h[i] = ff2e2(r.v[2 * i], r.v[2 * i + 1]);
    if constexpr (N == 8) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
    else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(h);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = f2e(r.v[i]);
  }
}

// id -> key in [0, vocab]: vocab stands for every id outside the table and sorts behind all others
template <typename Id>
__device__ __forceinline__ int key_of(const Id* ids, long long i, int vocab) {
  const Id id = ids[i];
  return id >= 0 && id < (Id)vocab ? (int)id : vocab;
}

// ---------------------------------------------------------------------------------------------------------------
// forward: `lanes` threads (a power of two) share kFwdRows neighbouring rows
// ---------------------------------------------------------------------------------------------------------------
constexpr int kFwdRows = 4;

template <typename Id, typename T, typename O, int VEC>
__global__ void __launch_bounds__(256)
embed_fwd_kernel(const Id* __restrict__ ids, const T* __restrict__ table, long long ld, O* __restrict__ out, long long n, int vocab,
                 int dim, float scale, int lanes) {
  const int lane = threadIdx.x % lanes;
  const long long row0 = ((long long)blockIdx.x * (256 / lanes) + threadIdx.x / lanes) * kFwdRows;
  int key[kFwdRows];
#pragma unroll
  for (int r = 0; r < kFwdRows; ++r) key[r] = row0 + r < n ? key_of(ids, row0 + r, vocab) : vocab;
  for (int c = lane * VEC; c < dim; c += lanes * VEC) {
    Raw<T, VEC> x[kFwdRows];
#pragma unroll
    for (int r = 0; r < kFwdRows; ++r)
      if (key[r] < vocab) x[r].load(table + (long long)key[r] * ld + c);
#pragma unroll
    for (int r = 0; r < kFwdRows; ++r) {
      if (row0 + r >= n) break;
      Vals<VEC> v = {};
      if (key[r] < vocab) {
        v = x[r].get();
#pragma unroll
        for (int j = 0; j < VEC; ++j) v.v[j] *= scale;
      }
      store_vals<VEC>(out + (row0 + r) * dim + c, v);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// stable radix sort of the positions by id, one cluster
// ---------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int cluster_read(const int* smem, uint32_t rank) {
  const uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
  int v;
  asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.s32 %0, [a];\n\t}"
               : "=r"(v) : "r"(addr), "r"(rank) : "memory");
  return v;
}

// Zeros for the rows of ids that do not come up, next to the sort and without anything of it.  Cluster c of `clusters` has words
// c, c + clusters, ... of 32 ids (neighbouring ids are about as common as one another); each of its CTAs looks through its part of
// the ids for them, and then writes its part of the rows that none of them has found.
// (By further CTAs of the first sums instead, from bits that the sort left: gradient of 131072 of 262144 x 768 bf16 201 us, not 161.)
template <typename Id>
__device__ __forceinline__ void absent_rows(const Id* __restrict__ ids, uint8_t* d_table, long long row_bytes, int n, int vocab, int cluster,
                                            int clusters) {
  __shared__ int found[kAbsentWords];                           // by this CTA
  __shared__ uint32_t there[kAbsentWords];                      // of the words that this CTA writes the rows of
  constexpr int kAhead = 16;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, rank = (int)cluster_rank(), ranks = (int)cluster_size();
  const int words = (vocab + 31) / 32, ours = (words - cluster + clusters - 1) / clusters;
  const long long begin = (long long)n * rank / ranks, end = (long long)n * (rank + 1) / ranks;
  for (int w0 = 0; w0 < ours; w0 += kAbsentWords) {
    const int count = min(ours - w0, kAbsentWords);
    for (int w = threadIdx.x; w < count; w += kSortThreads) found[w] = 0;
    __syncthreads();
    for (long long i0 = begin + threadIdx.x; i0 < end; i0 += kAhead * kSortThreads) {
      int key[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const long long i = i0 + u * kSortThreads;
        key[u] = i < end ? key_of(ids, i, vocab) : vocab;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t word = (uint32_t)key[u] / 32, turn = word / (uint32_t)clusters, w = turn - w0;
        if (key[u] < vocab && word - turn * clusters == (uint32_t)cluster && w < (uint32_t)count) {
          const int bit = 1 << key[u] % 32;
          if (!(*(volatile int*)&found[w] & bit)) atomicOr(&found[w], bit);      // common ids come up again and again
        }
      }
    }
    cluster_sync();
    const int mine = (count - rank + ranks - 1) / ranks;
    for (int l = threadIdx.x; l < mine; l += kSortThreads) {
      int any = 0;
#pragma unroll 8
      for (int r = 0; r < ranks; ++r) any |= cluster_read(&found[l * ranks + rank], r);
      there[l] = any;
    }
    cluster_sync();                                             // and nobody reads `found` any more
    for (int r = warp; r < mine * 32; r += kSortWarps) {
      const long long v = ((long long)(w0 + r / 32 * ranks + rank) * clusters + cluster) * 32 + r % 32;
      if (v >= vocab || (there[r / 32] >> r % 32 & 1)) continue;
      uint8_t* row = d_table + v * row_bytes;
      // up to the first 16-byte boundary, pieces of 16 bytes, and the rest
      const long long lead = min((long long)(-reinterpret_cast<uintptr_t>(row) & 15), row_bytes), body = (row_bytes - lead) & ~15ll;
      if (2 * lane < lead) *reinterpret_cast<uint16_t*>(row + 2 * lane) = 0;
      for (long long at = lead + 16 * lane; at < lead + body; at += 16 * 32) *reinterpret_cast<uint4*>(row + at) = make_uint4(0, 0, 0, 0);
      if (lead + body + 2 * lane < row_bytes) *reinterpret_cast<uint16_t*>(row + lead + body + 2 * lane) = 0;
    }
    __syncthreads();
  }
}

// Every warp owns a contiguous part of the input, so (CTA, warp, round, lane) is the input's order.  Per pass over `bits`
// bits: count the digits of each warp's part, turn the counts into first output places (digits before, then CTAs before,
// then warps before), and place the elements in order.  counts: [kSortWarps][bins] in shared memory.  A warp has the elements of
// eight rounds on their way at once, and keeps them from the counting to the placing where that is all there are.  What takes
// the time is placing single 8-byte entries from sixteen SMs (131072 ids of 262144: 35 us, with keys and positions apart and
// eight CTAs 65).
template <typename Id>
__global__ void __launch_bounds__(kSortThreads, 1)
embed_sort_kernel(const Id* __restrict__ ids, int2* list_a, int2* list_b, uint8_t* d_table, long long row_bytes, int n, int vocab, int bits,
                  int passes) {
  if (blockIdx.x >= cluster_size()) {
    absent_rows(ids, d_table, row_bytes, n, vocab, (int)(blockIdx.x / cluster_size()) - 1, (int)(gridDim.x / cluster_size()) - 1);
    return;
  }
  extern __shared__ int counts[];
  __shared__ int totals[1 << kDigitBits];
  __shared__ int warp_sums[kSortWarps];
  constexpr int kRounds = 8;
  const int bins = 1 << bits;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = (int)cluster_rank(), ranks = (int)cluster_size();
  const int parts = ranks * kSortWarps;
  const int per_warp = ((n + parts - 1) / parts + 31) / 32 * 32;
  const long long begin_ll = (long long)(rank * kSortWarps + warp) * per_warp;
  const int begin = begin_ll < n ? (int)begin_ll : n;
  const int end = begin + per_warp < n ? begin + per_warp : n;
  const bool kept = per_warp <= kRounds * 32;
  int* mine = counts + warp * bins;
  const uint32_t before = (1u << lane) - 1;

  int2 entry[kRounds];              // key and position
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    const bool to_a = (passes - pass) % 2 != 0;                  // the last pass writes list_a
    const int2* from = to_a ? list_b : list_a;
    int2* to = to_a ? list_a : list_b;
    auto fetch = [&](int i0) {
#pragma unroll
      for (int u = 0; u < kRounds; ++u) {
        const int i = i0 + u * 32 + lane;
        if (i < end) entry[u] = pass == 0 ? make_int2(key_of(ids, i, vocab), i) : __ldcg(from + i);
      }
    };
    if (kept) fetch(begin);
    for (int d = lane; d < bins; d += 32) mine[d] = 0;
    __syncwarp();
    for (int i0 = begin; i0 < end; i0 += kRounds * 32) {
      if (!kept) fetch(i0);
#pragma unroll
      for (int u = 0; u < kRounds; ++u) {
        const bool there = i0 + u * 32 + lane < end;
        const uint32_t active = __ballot_sync(0xffffffffu, there);
        if (there) {
          const int d = (entry[u].x >> shift) & (bins - 1);
          const uint32_t same = __match_any_sync(active, d);
          if ((same & before) == 0) mine[d] += __popc(same);
        }
        __syncwarp();
      }
    }
    __syncthreads();
    // thread d < bins: digit d
    const int d = threadIdx.x;
    int total = 0;
    if (d < bins) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = counts[w * bins + d];
        counts[w * bins + d] = total;
        total += c;
      }
      totals[d] = total;
    }
    if (ranks > 1) cluster_sync();
    int all = total, earlier = 0;
    if (ranks > 1 && d < bins) {
      int t[kMaxSortCtas];
#pragma unroll
      for (int r = 0; r < kMaxSortCtas; ++r) t[r] = r < ranks ? cluster_read(&totals[d], r) : 0;
      all = 0;
#pragma unroll
      for (int r = 0; r < kMaxSortCtas; ++r) {
        if (r < rank) earlier += t[r];
        all += t[r];
      }
    }
    int incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    int below = lane < warp ? warp_sums[lane] : 0;               // kSortWarps = 32
    below = __reduce_add_sync(0xffffffffu, below);
    const int base = incl - all + earlier + below;
    if (d < bins) {
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) counts[w * bins + d] += base;
    }
    __syncthreads();
    for (int i0 = begin; i0 < end; i0 += kRounds * 32) {
      if (!kept) fetch(i0);
#pragma unroll
      for (int u = 0; u < kRounds; ++u) {
        const bool there = i0 + u * 32 + lane < end;
        const uint32_t active = __ballot_sync(0xffffffffu, there);
        if (there) {
          const int digit = (entry[u].x >> shift) & (bins - 1);
          const uint32_t same = __match_any_sync(active, digit);
          const int place = mine[digit] + __popc(same & before);
          __syncwarp(active);
          if ((same & before) == 0) mine[digit] += __popc(same);
          to[place] = entry[u];
        }
        __syncwarp();
      }
    }
    if (ranks > 1) cluster_sync(); else __syncthreads();         // the next pass reads what all CTAs placed, and overwrites totals
  }
}

// ---------------------------------------------------------------------------------------------------------------
// sums of the pieces
// ---------------------------------------------------------------------------------------------------------------
// Entries in the order of their keys: key, and the row of `in` that is added (below 0: none).  A CTA has kSumThreads / lanes
// groups of `lanes` threads; a group takes one piece and VEC columns per thread of the CTA's column slab (blockIdx.y).
// What crosses the edges of a piece is left as two entries of the next step, with their rows in `partial`: the run that came in,
// and the run that begins here and goes on; a run that covers the piece from edge to edge is the former.
// AHEAD: entries of a thread on their way at once.  PARTIAL: `in` is the `partial` of the step before.  That and `list` are written
// while this kernel is already resident, so they are read by loads that go to L2; only d_out is read-only for its whole life.
template <typename I, typename T, int VEC, int AHEAD, bool PARTIAL>
__global__ void __launch_bounds__(kSumThreads)
embed_sum_kernel(const int2* list, const I* in, T* d_table, float* partial, int2* next, int n, int vocab, int dim, float scale,
                 int lanes) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");            // for the sort, or for the step before
  __shared__ int keys[kSumThreads / kMinLanes][kPiece + 2], rows[kSumThreads / kMinLanes][kPiece];
  const int groups = kSumThreads / lanes, group = threadIdx.x / lanes;
  for (int i = threadIdx.x; i < groups * (kPiece + 2); i += kSumThreads) {
    const int g = i / (kPiece + 2), k = i % (kPiece + 2);
    const long long e = ((long long)blockIdx.x * groups + g) * kPiece + k - 1;
    const bool in_list = e >= 0 && e < n;
    const int2 entry = in_list ? __ldcg(list + e) : make_int2(-1, -1);
    keys[g][k] = entry.x;
    if (k >= 1 && k <= kPiece) rows[g][k - 1] = entry.y;
  }
  __syncthreads();
  const int piece = (int)blockIdx.x * groups + group;
  const long long lo = (long long)piece * kPiece;
  if (lo >= n) return;
  const int* my_key = keys[group] + 1;
  const int* my_row = rows[group];
  const int count = n - lo < kPiece ? (int)(n - lo) : kPiece;
  const int first = my_key[0], last = my_key[count - 1];
  const bool came_in = my_key[-1] == first && first < vocab, goes_on = my_key[count] == last && last < vocab;
  const bool leads = threadIdx.x % lanes == 0 && blockIdx.y == 0 && next != nullptr;
  const int col = ((int)blockIdx.y * lanes + (int)threadIdx.x % lanes) * VEC;
  Vals<VEC> sum = {};
  int run = first;
  bool begins = !came_in, any = false;
  int left[2] = {-1, -1};                       // rows of `partial` that hold what came in and what goes on
  auto flush = [&](bool ends) {
    if (any) {
      if (begins && ends) {
        if (col < dim) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) sum.v[j] *= scale;
          store_vals<VEC>(d_table + (long long)run * dim + col, sum);
        }
      } else {
        const int row = piece * 2 + (begins ? 1 : 0);
        if (begins) left[1] = row; else left[0] = row;
        if (col < dim) store_vals<VEC>(partial + (long long)row * dim + col, sum);
      }
    }
    sum = Vals<VEC>{};
    begins = true;
    any = false;
  };
  for (int i0 = 0; i0 < count; i0 += AHEAD) {
    Raw<I, VEC> x[AHEAD];
    int k[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const bool valid = i0 + u < count && my_key[i0 + u] < vocab;
      k[u] = valid ? my_key[i0 + u] : -1;
      const int row = valid ? my_row[i0 + u] : -1;
      if (row >= 0 && col < dim) x[u].template load<PARTIAL>(in + (long long)row * dim + col);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (k[u] < 0) continue;                   // behind the last valid one
      if (k[u] != run) { flush(true); run = k[u]; }
      if (my_row[i0 + u] < 0) continue;
      any = true;
      const Vals<VEC> v = x[u].get();
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum.v[j] += v.v[j];
    }
  }
  if (first < vocab) flush(!(goes_on && run == last));
  if (leads) {
    next[2 * piece] = make_int2(first, left[0]);
    next[2 * piece + 1] = make_int2(last, left[1]);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// threads that share a row of `vecs` vectors: a power of two, 256 at most
int row_lanes(int vecs) {
  int lanes = 1;
  while (lanes < vecs && lanes < 256) lanes *= 2;
  return lanes;
}

template <typename Id, typename T, typename O>
void launch_fwd(const void* ids, const void* table, long long ld, void* out, long long n, int vocab, int dim, float scale,
                cudaStream_t s) {
  constexpr int V = 16 / sizeof(T);                             // 16 bytes of the table a thread
  const bool vec = dim % V == 0 && (ld * sizeof(T)) % 16 == 0 && aligned16(table) && aligned16(out);
  const int lanes = row_lanes(vec ? dim / V : dim), rows = 256 / lanes * kFwdRows;
  const unsigned blocks = (unsigned)((n + rows - 1) / rows);
  if (vec)
    embed_fwd_kernel<Id, T, O, V><<<blocks, 256, 0, s>>>((const Id*)ids, (const T*)table, ld, (O*)out, n, vocab, dim, scale, lanes);
  else
    embed_fwd_kernel<Id, T, O, 1><<<blocks, 256, 0, s>>>((const Id*)ids, (const T*)table, ld, (O*)out, n, vocab, dim, scale, lanes);
}

template <typename Id>
int launch_sort(const void* ids, int2* list, int2* list_b, void* d_table, long long row_bytes, int n, int vocab, cudaStream_t s) {
  int total_bits = 1;
  while ((1ll << total_bits) <= vocab) ++total_bits;      // keys run up to vocab
  const int passes = (total_bits + kDigitBits - 1) / kDigitBits, bits = (total_bits + passes - 1) / passes;
  static std::atomic<int> held[kMaxSortCtas + 1];   // clusters of 1, 2, 4, 8 and 16 CTAs that the machine holds at once; -1: none
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kSortThreads);
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  auto clusters_of = [&](int ctas, int clusters, int smem) {
    cfg.gridDim = dim3((unsigned)(ctas * clusters));
    cfg.dynamicSmemBytes = smem;
    attr.val.clusterDim = {(unsigned)ctas, 1, 1};
  };
  if (held[1] == 0) {
    const int most = kSortWarps * (1 << kDigitBits) * (int)sizeof(int);
    if (cudaFuncSetAttribute(embed_sort_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess ||
        cudaFuncSetAttribute(embed_sort_kernel<Id>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return GEMM_ERR_LAUNCH;
    for (int ctas = kMaxSortCtas; ctas > 0; ctas /= 2) {
      int k = 0;
      clusters_of(ctas, 1, most);
      if (cudaOccupancyMaxActiveClusters(&k, embed_sort_kernel<Id>, &cfg) != cudaSuccess) {      // sixteen are for the device to grant
        cudaGetLastError();
        k = 0;
      }
      held[ctas] = k > 0 ? k : -1;
    }
    if (held[1] < 0) return GEMM_ERR_LAUNCH;
  }
  int ctas = 1;
  while (ctas < kMaxSortCtas && n > ctas * kSortThreads && held[2 * ctas] > 0) ctas *= 2;      // one round per warp and pass where that is enough
  // Clusters of sixteen leave a third of the machine unused, so where the zeros that are certain to come take longer than the sort
  // takes with eight CTAs (0.29 ns an entry and pass; sixteen's six other clusters write 4.8 TB/s), eight it is.  us of the gradient
  // with 16 | 8: 65536 of 100003 x 2048 fp32 238 | 220; 30000 of 50021 x 1029 bf16 113 | 111; 131072 of 262144 x 768 bf16 161 | 205;
  // 131072 of 4096 x 1024 bf16 120 | 142
  if (ctas == kMaxSortCtas && held[ctas / 2] > 0 && (double)(vocab - n) * row_bytes > 1400.0 * passes * n) ctas /= 2;
  const int others = held[ctas] - 1, words = (vocab + 31) / 32;
  clusters_of(ctas, 1 + (others < 1 ? 1 : others < words ? others : words), kSortWarps * (1 << bits) * (int)sizeof(int));
  return cudaLaunchKernelEx(&cfg, embed_sort_kernel<Id>, (const Id*)ids, list, list_b, (uint8_t*)d_table, row_bytes, n, vocab, bits,
                            passes) == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

// A launch that starts while the kernel before it ends
template <typename K, typename... Args>
cudaError_t launch_early(K kernel, dim3 grid, int threads, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The sums of one step
template <typename I, typename T, int VEC, int AHEAD, bool PARTIAL>
cudaError_t launch_step(const int2* list, const void* in, void* d_table, float* partial, int2* next, int n, int vocab, int dim, float scale,
                        cudaStream_t s) {
  int lanes = row_lanes((dim + VEC - 1) / VEC);
  lanes = lanes > kSumThreads ? kSumThreads : lanes < kMinLanes ? kMinLanes : lanes;
  const int pieces = (n + kPiece - 1) / kPiece, per_block = kSumThreads / lanes;
  const dim3 grid((pieces + per_block - 1) / per_block, (dim + lanes * VEC - 1) / (lanes * VEC));
  return launch_early(embed_sum_kernel<I, T, VEC, AHEAD, PARTIAL>, grid, kSumThreads, s, list, (const I*)in, (T*)d_table, partial,
                      pieces > 1 ? next : nullptr, n, vocab, dim, scale, lanes);
}

// Of the first step there is a machine full, of the later ones a few CTAs: those take a piece's entries all at once.
template <typename O, typename T, int VEC>
int launch_sums(const int2* list, const void* d_out, void* d_table, float* partial, int2* next, int n, int vocab, int dim,
                float scale, cudaStream_t s) {
  cudaError_t e = launch_step<O, T, VEC, 8, false>(list, d_out, d_table, partial, next, n, vocab, dim, scale, s);
  for (int pieces = (n + kPiece - 1) / kPiece; pieces > 1 && e == cudaSuccess; pieces = (n + kPiece - 1) / kPiece) {
    n = 2 * pieces;
    const float* in = partial;
    partial += (long long)n * dim;
    list = next;
    next += n;
    e = launch_step<float, T, VEC == 1 ? 1 : 4, kPiece, true>(list, in, d_table, partial, next, n, vocab, dim, scale, s);
  }
  return e == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

template <typename Id, typename O, typename T>
int backward(const void* ids, int2* list, int2* list_b, const void* d_out, void* d_table, float* partial, int2* next, int n, int vocab,
             int dim, float scale, cudaStream_t s) {
  if (const int e = launch_sort<Id>(ids, list, list_b, d_table, (long long)dim * (int)sizeof(T), n, vocab, s)) return e;
  const bool vec = dim % 8 == 0 && aligned16(d_out) && aligned16(d_table) && aligned16(partial);
  return vec ? launch_sums<O, T, 16 / sizeof(O)>(list, d_out, d_table, partial, next, n, vocab, dim, scale, s)
             : launch_sums<O, T, 1>(list, d_out, d_table, partial, next, n, vocab, dim, scale, s);
}

}  // namespace

// ids: int64 (ids64) or int32, n of them; table [vocab] rows of pitch ld, fp32 or elements; out [n][dim], fp32 (only with an
// fp32 table) or elements.
extern "C" int fbam_embed_fwd(const void* ids, int ids64, const void* table, long long ld, int table_fp32, void* out,
                              int out_fp32, long long n, int vocab, int dim, float scale, void* stream) {
  if (n <= 0 || vocab <= 0 || dim <= 0 || (out_fp32 && !table_fp32) || n > 0x7fffffffll) return GEMM_ERR_SHAPE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto go = [&](auto id) {
    using Id = decltype(id);
    if (!table_fp32) launch_fwd<Id, elem_t, elem_t>(ids, table, ld, out, n, vocab, dim, scale, s);
    else if (out_fp32) launch_fwd<Id, float, float>(ids, table, ld, out, n, vocab, dim, scale, s);
    else launch_fwd<Id, float, elem_t>(ids, table, ld, out, n, vocab, dim, scale, s);
  };
  if (ids64) go((long long)0); else go(0);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

// 8-byte words and fp32 values of the workspaces of fbam_embed_bwd
extern "C" void fbam_embed_bwd_workspace(long long n, int dim, long long* words, long long* floats) {
  *words = 2 * n;
  *floats = 0;
  for (long long pieces = (n + kPiece - 1) / kPiece; pieces > 1; pieces = (2 * pieces + kPiece - 1) / kPiece) {
    *words += 2 * pieces;
    *floats += 2 * pieces * dim;
  }
}

extern "C" int fbam_embed_bwd(const void* ids, int ids64, const void* d_out, int out_fp32, void* d_table, int table_fp32,
                              long long n, int vocab, int dim, float scale, void* words, float* partial, void* stream) {
  if (n <= 0 || vocab <= 0 || dim <= 0 || (out_fp32 && !table_fp32) || n > 0x3fffffffll || vocab > 0x3fffffff) return GEMM_ERR_SHAPE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int2 *list = reinterpret_cast<int2*>(words), *list_b = list + n, *next = list_b + n;
  auto go = [&](auto id) {
    using Id = decltype(id);
    const auto run = !table_fp32 ? backward<Id, elem_t, elem_t> : out_fp32 ? backward<Id, float, float> : backward<Id, elem_t, float>;
    return run(ids, list, list_b, d_out, d_table, partial, next, (int)n, vocab, dim, scale, s);
  };
  return ids64 ? go((long long)0) : go(0);
}
