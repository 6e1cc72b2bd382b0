// Token embedding: out[i] = scale * table[id_i], and the table's gradient
//   d_table[v] = scale * sum over { i : id_i = v } of d_out[i],
// summed in fp32 in an order that the ids alone fix, so equal inputs give equal bits.  An id outside [0, vocab) gives a
// row of zeros and has no gradient.
//
// Gradient in three launches:
//   1. embed_sort_kernel   stable radix sort of (id, position) by one cluster of CTAs;
//   2. embed_sum_kernel    the sorted order is cut into pieces of kPiece positions; a piece sums its runs of equal ids.
//                          A run that lies inside the piece is the row's gradient, one that crosses an edge leaves a
//                          partial sum.  Further CTAs of the launch write the rows that no id names;
//   3. embed_join_kernel   adds up the partial sums of the runs that cross edges.
#include <cuda_runtime.h>
#include <stdint.h>

#include "elem16.cuh"
#include "gemm_tcgen05.h"

namespace {

constexpr int kPiece = 32;        // sorted positions of one piece
constexpr int kZeroRows = 32;     // table rows per CTA that looks for absent ids
constexpr int kDigitBits = 10;
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;

template <int N>
struct Vals { float v[N]; };

template <int N>
__device__ __forceinline__ Vals<N> load_vals(const float* p) {
  Vals<N> r;
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 t = *reinterpret_cast<const float4*>(p + i);
      r.v[i] = t.x; r.v[i + 1] = t.y; r.v[i + 2] = t.z; r.v[i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = p[i];
  }
  return r;
}
template <int N>
__device__ __forceinline__ Vals<N> load_vals(const elem_t* p) {
  Vals<N> r;
  if constexpr (N == 8) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const elem2_t* h = reinterpret_cast<const elem2_t*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = e22ff(h[i]);
      r.v[2 * i] = f.x; r.v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.v[i] = e2f(p[i]);
  }
  return r;
}
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
  if constexpr (N == 8) {
    __align__(16) elem2_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = ff2e2(r.v[2 * i], r.v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
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
// forward: `lanes` threads (a power of two) share a row
// ---------------------------------------------------------------------------------------------------------------
template <typename Id, typename T, typename O, int VEC>
__global__ void embed_fwd_kernel(const Id* __restrict__ ids, const T* __restrict__ table, long long ld, O* __restrict__ out,
                                 long long n, int vocab, int dim, float scale, int lanes) {
  const int rows_per_block = blockDim.x / lanes, lane = threadIdx.x % lanes;
  const long long row = (long long)blockIdx.x * rows_per_block + threadIdx.x / lanes;
  if (row >= n) return;
  const int key = key_of(ids, row, vocab);
  const T* src = table + (long long)key * ld;
  O* dst = out + row * dim;
#pragma unroll 4
  for (int c = lane * VEC; c < dim; c += lanes * VEC) {
    Vals<VEC> r = {};
    if (key < vocab) r = load_vals<VEC>(src + c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) r.v[j] *= scale;
    store_vals<VEC>(dst + c, r);
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

// Every warp owns a contiguous part of the input, so (CTA, warp, round, lane) is the input's order.  Per pass over `bits`
// bits: count the digits of each warp's part, turn the counts into first output places (digits before, then CTAs before,
// then warps before), and place the elements in order.  counts: [kSortWarps][bins] in shared memory.
template <typename Id>
__global__ void __launch_bounds__(kSortThreads, 1)
embed_sort_kernel(const Id* __restrict__ ids, int* key_a, int* pos_a, int* key_b, int* pos_b, int* list_count, int n,
                  int vocab, int bits, int passes) {
  extern __shared__ int counts[];
  __shared__ int totals[1 << kDigitBits];
  __shared__ int warp_sums[kSortWarps];
  const int bins = 1 << bits;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int parts = ranks * kSortWarps;
  const int per_warp = ((n + parts - 1) / parts + 31) / 32 * 32;
  const long long begin_ll = (long long)(rank * kSortWarps + warp) * per_warp;
  const int begin = begin_ll < n ? (int)begin_ll : n;
  const int end = begin + per_warp < n ? begin + per_warp : n;
  int* mine = counts + warp * bins;
  const uint32_t before = (1u << lane) - 1;
  if (rank == 0 && threadIdx.x == 0) *list_count = 0;

  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    const int* key_in = (passes - pass) % 2 ? key_b : key_a;     // the last pass writes key_a / pos_a ...
    const int* pos_in = (passes - pass) % 2 ? pos_b : pos_a;
    int* key_out = (passes - pass) % 2 ? key_a : key_b;
    int* pos_out = (passes - pass) % 2 ? pos_a : pos_b;
    auto fetch = [&](int i) { return pass == 0 ? key_of(ids, i, vocab) : __ldcg(key_in + i); };

    for (int d = lane; d < bins; d += 32) mine[d] = 0;
    __syncwarp();
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t active = __ballot_sync(0xffffffffu, i < end);
      if (i < end) {
        const int d = (fetch(i) >> shift) & (bins - 1);
        const uint32_t same = __match_any_sync(active, d);
        if ((same & before) == 0) mine[d] += __popc(same);
      }
      __syncwarp();
    }
    __syncthreads();
    // thread d < bins: digit d
    const int d = threadIdx.x;
    int total = 0;
    if (d < bins) {
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = counts[w * bins + d];
        counts[w * bins + d] = total;
        total += c;
      }
      totals[d] = total;
    }
    cluster_sync();
    int all = 0, earlier = 0;
    if (d < bins) {
      for (uint32_t r = 0; r < ranks; ++r) {
        const int t = cluster_read(&totals[d], r);
        if (r < rank) earlier += t;
        all += t;
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
    int base = incl - all + earlier;
    for (int w = 0; w < warp; ++w) base += warp_sums[w];
    if (d < bins)
      for (int w = 0; w < kSortWarps; ++w) counts[w * bins + d] += base;
    __syncthreads();
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t active = __ballot_sync(0xffffffffu, i < end);
      if (i < end) {
        const int key = fetch(i);
        const int digit = (key >> shift) & (bins - 1);
        const uint32_t same = __match_any_sync(active, digit);
        const int place = mine[digit] + __popc(same & before);
        __syncwarp(active);
        if ((same & before) == 0) mine[digit] += __popc(same);
        key_out[place] = key;
        pos_out[place] = pass == 0 ? i : __ldcg(pos_in + i);
      }
      __syncwarp();
    }
    cluster_sync();       // the next pass reads what all CTAs placed, and overwrites totals
  }
}

// ---------------------------------------------------------------------------------------------------------------
// sums of the pieces, and the rows without an id
// ---------------------------------------------------------------------------------------------------------------
// A CTA has blockDim.x / lanes groups of `lanes` threads; a group takes one piece and VEC columns per thread of the CTA's
// column slab (blockIdx.y).  partial: [pieces][2][dim] fp32; slot 0: the run that came in from the previous piece, slot 1:
// the run that begins here and goes on.  Where one run covers the piece from edge to edge it is in slot 0.
template <typename O, typename T, int VEC>
__global__ void embed_sum_kernel(const int* __restrict__ key, const int* __restrict__ pos, const O* __restrict__ d_out,
                                 T* __restrict__ d_table, float* __restrict__ partial, int* __restrict__ list_count,
                                 int* __restrict__ list, int n, int vocab, int dim, float scale, int lanes, int piece_blocks) {
  if ((int)blockIdx.x >= piece_blocks) {
    __shared__ int there[kZeroRows];
    if (blockIdx.y != 0) return;
    const int v0 = ((int)blockIdx.x - piece_blocks) * kZeroRows;
    if ((int)threadIdx.x < kZeroRows) {
      const int v = v0 + (int)threadIdx.x;
      int lo = 0, hi = n;                       // first place whose key is not below v
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (key[mid] < v) lo = mid + 1; else hi = mid;
      }
      there[threadIdx.x] = v >= vocab || (lo < n && key[lo] == v);
    }
    __syncthreads();
    const Vals<VEC> zero = {};
    for (int r = 0; r < kZeroRows; ++r) {
      if (there[r]) continue;
      T* row = d_table + (long long)(v0 + r) * dim;
      for (int c = threadIdx.x * VEC; c < dim; c += blockDim.x * VEC) store_vals<VEC>(row + c, zero);
    }
    return;
  }
  const int piece = (int)blockIdx.x * (blockDim.x / lanes) + (int)threadIdx.x / lanes;
  const int lo = piece * kPiece;
  if (lo >= n) return;
  const int hi = lo + kPiece < n ? lo + kPiece : n;
  const int first = key[lo], prev = lo > 0 ? key[lo - 1] : -1;
  const int last = key[hi - 1], next = hi < n ? key[hi] : -1;
  if (first >= vocab) return;
  const bool came_in = prev == first, goes_on = next == last && last < vocab;
  const int col = ((int)blockIdx.y * lanes + (int)threadIdx.x % lanes) * VEC;
  if (goes_on && blockIdx.y == 0 && threadIdx.x % lanes == 0 && !(came_in && first == last))
    list[atomicAdd(list_count, 1)] = piece;     // the order of the list decides nothing
  if (col >= dim) return;
  Vals<VEC> sum = {};
  int run = first;
  bool begins = !came_in;
  auto flush = [&](bool ends) {
    if (begins && ends) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum.v[j] *= scale;
      store_vals<VEC>(d_table + (long long)run * dim + col, sum);
    } else {
      store_vals<VEC>(partial + ((long long)piece * 2 + (begins ? 1 : 0)) * dim + col, sum);
    }
    sum = Vals<VEC>{};
    begins = true;
  };
  constexpr int kAhead = 8;
  for (int i0 = lo; i0 < hi; i0 += kAhead) {
    int k[kAhead];
    Vals<VEC> x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      k[u] = i0 + u < hi ? key[i0 + u] : vocab;
      if (k[u] < vocab) x[u] = load_vals<VEC>(d_out + (long long)pos[i0 + u] * dim + col);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (k[u] >= vocab) continue;              // behind the last valid one
      if (k[u] != run) { flush(true); run = k[u]; }
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum.v[j] += x[u].v[j];
    }
  }
  flush(!(goes_on && run == last));
}

// A work item is one run that crosses pieces and 8 x VEC of its columns: 32 rows of threads add up every 32nd partial sum,
// then one row of threads adds the 32 sums in order.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
embed_join_kernel(const int* __restrict__ key, const float* __restrict__ partial, T* __restrict__ d_table,
                  const int* __restrict__ list_count, const int* __restrict__ list, int n, int dim, float scale) {
  __shared__ float sums[32][8 * VEC + 1];
  const int slabs = (dim + 8 * VEC - 1) / (8 * VEC);
  const long long items = (long long)*list_count * slabs;
  const int r = threadIdx.x / 8, c = threadIdx.x % 8;
  for (long long w = blockIdx.x; w < items; w += gridDim.x) {
    const int piece = list[w / slabs], col = (int)(w % slabs) * 8 * VEC + c * VEC;
    const int v = key[(long long)piece * kPiece + kPiece - 1];
    int more = 0;                               // pieces behind this one that the run reaches
    for (;;) {
      const long long at = ((long long)piece + 1 + more + threadIdx.x) * kPiece;
      const int got = __syncthreads_count(at < n && key[at] == v);
      more += got;
      if (got < (int)blockDim.x) break;
    }
    Vals<VEC> sum = {};
    if (col < dim) {
#pragma unroll 4
      for (int i = r; i <= more; i += 32) {
        const Vals<VEC> x = load_vals<VEC>(partial + ((long long)(piece + i) * 2 + (i == 0 ? 1 : 0)) * dim + col);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum.v[j] += x.v[j];
      }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) sums[r][c * VEC + j] = sum.v[j];
    __syncthreads();
    if (r == 0 && col < dim) {
      const int rows = more + 1 < 32 ? more + 1 : 32;
      for (int q = 1; q < rows; ++q)
#pragma unroll
        for (int j = 0; j < VEC; ++j) sum.v[j] += sums[q][c * VEC + j];
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum.v[j] *= scale;
      store_vals<VEC>(d_table + (long long)v * dim + col, sum);
    }
    __syncthreads();
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
  const bool vec = dim % 8 == 0 && (ld * sizeof(T)) % 16 == 0 && aligned16(table) && aligned16(out);
  const int lanes = row_lanes(vec ? dim / 8 : dim), rows = 256 / lanes;
  const unsigned blocks = (unsigned)((n + rows - 1) / rows);
  if (vec)
    embed_fwd_kernel<Id, T, O, 8><<<blocks, 256, 0, s>>>((const Id*)ids, (const T*)table, ld, (O*)out, n, vocab, dim, scale, lanes);
  else
    embed_fwd_kernel<Id, T, O, 1><<<blocks, 256, 0, s>>>((const Id*)ids, (const T*)table, ld, (O*)out, n, vocab, dim, scale, lanes);
}

template <typename Id>
int launch_sort(const void* ids, int* key, int* pos, int* key_b, int* pos_b, int* list_count, int n, int vocab, cudaStream_t s) {
  int total_bits = 1;
  while ((1ll << total_bits) <= vocab) ++total_bits;      // keys run up to vocab
  const int passes = (total_bits + kDigitBits - 1) / kDigitBits, bits = (total_bits + passes - 1) / passes;
  // One CTA sorts 8192 ids (eight rounds per warp and pass); more CTAs where there are more ids, eight at most.
  int ctas = 1;
  while (ctas < 8 && n > ctas * 8192) ctas *= 2;
  const int smem = kSortWarps * (1 << bits) * (int)sizeof(int);
  if (cudaFuncSetAttribute(embed_sort_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           kSortWarps * (1 << kDigitBits) * (int)sizeof(int)) != cudaSuccess)
    return GEMM_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {(unsigned)ctas, 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, embed_sort_kernel<Id>, (const Id*)ids, key, pos, key_b, pos_b, list_count, n, vocab, bits,
                            passes) == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

template <typename O, typename T, int VEC>
int launch_sums(const int* key, const int* pos, const void* d_out, void* d_table, float* partial, int* list_count, int* list,
                int n, int vocab, int dim, float scale, cudaStream_t s) {
  constexpr int threads = 128;
  int lanes = row_lanes((dim + VEC - 1) / VEC);
  if (lanes > threads) lanes = threads;
  const int pieces = (n + kPiece - 1) / kPiece, per_block = threads / lanes;
  const int piece_blocks = (pieces + per_block - 1) / per_block;
  const dim3 grid(piece_blocks + (vocab + kZeroRows - 1) / kZeroRows, (dim + lanes * VEC - 1) / (lanes * VEC));
  embed_sum_kernel<O, T, VEC><<<grid, threads, 0, s>>>(key, pos, (const O*)d_out, (T*)d_table, partial, list_count, list, n,
                                                       vocab, dim, scale, lanes, piece_blocks);
  if (pieces > 1) {
    constexpr int JV = VEC == 8 ? 4 : 1;
    embed_join_kernel<T, JV><<<592, 256, 0, s>>>(key, partial, (T*)d_table, list_count, list, n, dim, scale);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

template <typename O, typename T>
int launch_sums_vec(const int* key, const int* pos, const void* d_out, void* d_table, float* partial, int* list_count,
                    int* list, int n, int vocab, int dim, float scale, cudaStream_t s) {
  const bool vec = dim % 8 == 0 && aligned16(d_out) && aligned16(d_table) && aligned16(partial);
  return vec ? launch_sums<O, T, 8>(key, pos, d_out, d_table, partial, list_count, list, n, vocab, dim, scale, s)
             : launch_sums<O, T, 1>(key, pos, d_out, d_table, partial, list_count, list, n, vocab, dim, scale, s);
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

// int32 words and fp32 values of the workspaces of fbam_embed_bwd
extern "C" void fbam_embed_bwd_workspace(long long n, int dim, long long* words, long long* floats) {
  const long long pieces = (n + kPiece - 1) / kPiece;
  *words = 4 * n + pieces + 1;
  *floats = pieces > 1 ? pieces * 2 * dim : 0;
}

extern "C" int fbam_embed_bwd(const void* ids, int ids64, const void* d_out, int out_fp32, void* d_table, int table_fp32,
                              long long n, int vocab, int dim, float scale, int* words, float* partial, void* stream) {
  if (n <= 0 || vocab <= 0 || dim <= 0 || (out_fp32 && !table_fp32) || n > 0x3fffffffll || vocab > 0x3fffffff) return GEMM_ERR_SHAPE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  int *key = words, *pos = key + n, *key_b = pos + n, *pos_b = key_b + n, *list_count = pos_b + n, *list = list_count + 1;
  const int e = ids64 ? launch_sort<long long>(ids, key, pos, key_b, pos_b, list_count, (int)n, vocab, s)
                      : launch_sort<int>(ids, key, pos, key_b, pos_b, list_count, (int)n, vocab, s);
  if (e) return e;
  if (!table_fp32) return launch_sums_vec<elem_t, elem_t>(key, pos, d_out, d_table, partial, list_count, list, (int)n, vocab, dim, scale, s);
  if (out_fp32) return launch_sums_vec<float, float>(key, pos, d_out, d_table, partial, list_count, list, (int)n, vocab, dim, scale, s);
  return launch_sums_vec<elem_t, float>(key, pos, d_out, d_table, partial, list_count, list, (int)n, vocab, dim, scale, s);
}
