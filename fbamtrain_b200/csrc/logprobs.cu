// Log probabilities of given tokens with the entropy of their distribution and the most likely alternatives, from rows of
// logits; and the gradient of the first two.  With x = logit / temperature, m = max x, S = sum exp(x - m),
// U = sum exp(x - m) (x - m):
//   log p_t = x_t - m - log S          entropy = log S - U / S
//   d x_j = dlogp (1[j = t] - p_j) - dH p_j (log p_j + H)
// m, S and U are kept by every thread in fp32 over one pass of the row, rescaled when the maximum moves and joined at the
// end.  Alternatives are ordered by (value falling, index rising).
//
// A logit of -inf has probability 0.  A row of nothing else has entropy 0, log probabilities of -inf and no gradient.  A
// target outside [0, vocab) has log probability 0 and no gradient.  A NaN makes the row's results NaN and counts as -inf
// among the alternatives.
#include <cuda_runtime.h>
#include <stdint.h>

#include "elem16.cuh"
#include "gemm_tcgen05.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLowest = -3.402823466e38f;   // stands for a maximum of -inf, so that no difference is inf - inf
constexpr float kFar = -1e30f;                // differences go no lower: exp gives 0 and the product with 0 stays 0

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(elem_t x) { return e2f(x); }
__device__ __forceinline__ void from_f(float* p, float x) { *p = x; }
__device__ __forceinline__ void from_f(elem_t* p, float x) { *p = f2e(x); }

// VEC logits as they lie in memory, 16 bytes.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Raw {
  T v[VEC];
  __device__ __forceinline__ void get(float (&x)[VEC]) const {
    if constexpr (sizeof(T) == 2) {
      const elem2_t* a = reinterpret_cast<const elem2_t*>(v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = e22ff(a[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = to_f(v[i]);
    }
  }
  __device__ __forceinline__ void set(const float (&x)[VEC]) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<elem2_t*>(v)[i] = ff2e2(x[2 * i], x[2 * i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) from_f(&v[i], x[i]);
    }
  }
  // of two vectors, the larger of each place; a NaN is not taken where there is a number
  __device__ __forceinline__ Raw max(const Raw& o) const {
    Raw r;
    if constexpr (sizeof(T) == 2) {
      const elem2_t *a = reinterpret_cast<const elem2_t*>(v), *b = reinterpret_cast<const elem2_t*>(o.v);
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<elem2_t*>(r.v)[i] = __hmax2(a[i], b[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) from_f(&r.v[i], fmaxf(to_f(v[i]), to_f(o.v[i])));
    }
    return r;
  }
  __device__ __forceinline__ float top() const {
    if constexpr (sizeof(T) == 2) {
      const elem2_t* a = reinterpret_cast<const elem2_t*>(v);
      const float2 f = e22ff(__hmax2(__hmax2(a[0], a[1]), __hmax2(a[2], a[3])));
      return fmaxf(f.x, f.y);
    } else {
      float t = to_f(v[0]);
#pragma unroll
      for (int i = 1; i < VEC; ++i) t = fmaxf(t, to_f(v[i]));
      return t;
    }
  }
};
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load_raw(const T* p) {
  Raw<T, VEC> r;
  *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(p));
  return r;
}
// The same without a line in L1, which the forward's one reading of a row has no use for (1001 x 100003 fp32: 84 -> 76 us,
// 16384 x 6000 80 -> 70; the backward is no faster with it).
template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> stream_raw(const T* p) {
  Raw<T, VEC> r;
  uint4 t;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(t.x), "=r"(t.y), "=r"(t.z), "=r"(t.w) : "l"(p));
  *reinterpret_cast<uint4*>(&r) = t;
  return r;
}

// Packed pairs (sm_100 computes on two fp32 values per instruction)
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// Sums of part of a row relative to its maximum.
struct Stats {
  float m, s, u;
  // the same sums relative to a maximum that is no lower
  __device__ __forceinline__ void move_to(float top, float c) {
    const float d = fmaxf(fmaxf(m, kLowest) - fmaxf(top, kLowest), kFar);
    const float f = ex2(d * c);
    u = f * fmaf(s, d, u);
    s *= f;
    m = top;
  }
  __device__ __forceinline__ void join(Stats o, float c) {
    const float top = fmaxf(m, o.m);
    move_to(top, c);
    o.move_to(top, c);
    s += o.s;
    u += o.u;
  }
};

// A key that orders floats by value; NaN counts as -inf.  0 is below every key: no logit.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) x = -INFINITY;
  x += 0.0f;                        // -0 and 0 are one value
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}

// Vectors of a row start on 16-byte boundaries whatever the row's start: `lead` places of the first one lie in front of the row.
template <typename T, int VEC>
struct Row {
  const T* p;
  int vocab, lead;
  __device__ __forceinline__ Row(const T* row, int n) : p(row), vocab(n), lead((int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T))) {}
  __device__ __forceinline__ bool has(long long j) const { return j >= 0 && j < vocab; }
  // the VEC logits from j on; -inf outside the row
  __device__ __forceinline__ Raw<T, VEC> load(long long j) const {
    if (j >= 0 && j + VEC <= vocab) return load_raw<T, VEC>(p + j);
    Raw<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (has(j + i)) r.v[i] = p[j + i];
      else from_f(&r.v[i], -INFINITY);
    }
    return r;
  }
};

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
__device__ __forceinline__ uint32_t in_cta(const void* smem, uint32_t rank) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(smem)), "r"(rank));
  return at;
}
__device__ __forceinline__ float cluster_read(const float* smem, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(in_cta(smem, rank)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long cluster_read(const unsigned long long* smem, uint32_t rank) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(in_cta(smem, rank)) : "memory");
  return v;
}

template <int VEC>
constexpr int kBatchOf = 32 / VEC;  // vectors that a thread has on their way at once
constexpr int kMaxTop = 32, kMaxCtas = 8;
constexpr uint32_t kNothing = 0x007fffffu;    // order_key(-inf)

// One row per cluster of CTAs (mostly of one), WARPS warps each.  Vector v of a row belongs to thread v mod (threads of the
// cluster).
//
// Alternatives: a thread keeps the key of the best logit of each of its batches (of 2^fold of them, where shared memory has no room
// for all).  The k-th best of the CTA's threads' best keys
// bounds the k-th best of its logits from below, so only batches whose best reaches that bound are looked at again; what
// reaches it goes on a list, and a place on the list is the count of those that come before by (value falling, id rising).
// Where the list overflows, equal logits are taken in order, or each alternative is looked for in a pass of its own.
//
// Bound: reading the logits once, with the special-function unit close behind for 16-bit ones (one exponential a logit, 0.7 of
// the time of the reading).  8192 x 4096 bf16 20 us (3.4 TB/s), 1001 x 100003 fp32 72 us (5.5 TB/s), 16384 x 6000 fp32 66 us
// (6.0 TB/s).  Packed arithmetic, a whole batch of loads before the first use, 32 warps per SM; fetching a batch ahead in
// registers cost more warps than it hid (8192 x 4096: 24 -> 31).
// With one warp a row, a CTA has ROWS rows, which share nothing.
template <typename T, int VEC, int WARPS, int ROWS>
__global__ void __launch_bounds__(WARPS * ROWS * 32, 1024 / (WARPS * ROWS * 32))
logprobs_fwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ targets, float* __restrict__ logprob,
                    float* __restrict__ entropy, float* __restrict__ stats, float* __restrict__ top_logprobs,
                    long long* __restrict__ top_ids, long long rows, int vocab, int top, float inv_t, int batches, int folded, int candidates) {
  static_assert(WARPS == 1 || ROWS == 1, "rows of a CTA do not wait for one another");
  constexpr int kThreads = WARPS * 32, kBatch = kBatchOf<VEC>;
  const int fold = WARPS == 1 ? 0 : folded;                   // a warp alone has 32 batches at most (launch_fwd)
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ Stats parts[WARPS];
  __shared__ float whole[3];
  __shared__ int list_lengths[ROWS];
  __shared__ float final[ROWS][2];                            // maximum and log of the sum, of rank 0
  const int ctas = (int)cluster_size(), rank = (int)cluster_rank();
  const int sub = ROWS > 1 ? threadIdx.x / 32 : 0;
  const long long r = ROWS > 1 ? (long long)blockIdx.x * ROWS + sub : blockIdx.x / ctas;
  if (r >= rows) return;                                      // a whole warp of several rows
  const int tid = ROWS > 1 ? threadIdx.x % 32 : threadIdx.x, warp = tid / 32, lane = tid % 32;
  unsigned long long* sorted = reinterpret_cast<unsigned long long*>(smem_raw) + sub * (kMaxTop + candidates);
  unsigned long long* list = sorted + kMaxTop;                // [candidates]
  uint32_t* best_of = reinterpret_cast<uint32_t*>(reinterpret_cast<unsigned long long*>(smem_raw) + ROWS * (kMaxTop + candidates)) +
                      sub * (((batches - 1) >> fold) + 1) * kThreads;       // [batches >> fold, upwards][kThreads]
  int& list_length = list_lengths[sub];
  const Row<T, VEC> row(logits + r * ld, vocab);
  const float c = inv_t * kLog2e;
  const long long hop = (long long)ctas * kThreads * VEC;     // from one vector of a thread to its next
  const long long first = (long long)(rank * kThreads + tid) * VEC - row.lead;

  Stats st{-INFINITY, 0.0f, 0.0f};
  uint32_t best = 0;
  auto fetch = [&](Raw<T, VEC> (&to)[kBatch], long long j) {
    if (j >= 0 && j + (kBatch - 1) * hop + VEC <= vocab) {
      const T* p = row.p + j;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) to[b] = stream_raw<T, VEC>(p + b * hop);
    } else {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) to[b] = row.load(j + b * hop);
    }
  };
  for (int i = 0; i < batches; ++i) {
    const long long j = first + i * kBatch * hop;
    Raw<T, VEC> raw[kBatch];
    fetch(raw, j);
    Raw<T, VEC> highest = raw[0];
#pragma unroll
    for (int b = 1; b < kBatch; ++b) highest = highest.max(raw[b]);
    const float top_x = highest.top();
    if (top > 0) {
      const uint32_t key = j < vocab ? order_key(top_x) : 0;
      uint32_t& of = best_of[(i >> fold) * kThreads + tid];
      of = i & ((1 << fold) - 1) ? max(of, key) : key;
      best = max(best, key);
    }
    if (top_x > st.m) st.move_to(top_x, c);
    const float m = fmaxf(st.m, kLowest);
    float2 s2 = both(0.0f), u2 = both(0.0f);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      float x[VEC];
      raw[b].get(x);
#pragma unroll
      for (int q = 0; q < VEC; q += 2) {
        const float2 d = __fadd2_rn(make_float2(x[q], x[q + 1]), both(-m));
        const float2 w = __fmul2_rn(d, both(c));
        const float2 e = make_float2(ex2(w.x), ex2(w.y));        // NaN for a NaN, 0 for -inf
        s2 = __fadd2_rn(s2, e);
        u2 = __ffma2_rn(e, make_float2(fmaxf(d.x, kFar), fmaxf(d.y, kFar)), u2);
      }
    }
    st.s += s2.x + s2.y;
    st.u += u2.x + u2.y;
  }
  // of the warp: one move to its maximum, then sums
  float top_m = st.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top_m = fmaxf(top_m, __shfl_xor_sync(0xffffffffu, top_m, o));
  st.move_to(top_m, c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
    st.u += __shfl_xor_sync(0xffffffffu, st.u, o);
  }
  if constexpr (WARPS > 1) {
    if (lane == 0) parts[warp] = st;
    __syncthreads();
    if (warp == 0) {
      st = parts[lane % WARPS];
#pragma unroll
      for (int o = WARPS / 2; o > 0; o >>= 1)
        st.join({__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.u, o)}, c);
    }
  }
  if (ctas > 1) {
    if (tid == 0) { whole[0] = st.m; whole[1] = st.s; whole[2] = st.u; }
    cluster_sync();
    if (rank == 0 && warp == 0)
      for (int q = 1; q < ctas; ++q) st.join({cluster_read(&whole[0], q), cluster_read(&whole[1], q), cluster_read(&whole[2], q)}, c);
  }
  // the first warp of rank 0: st is of the whole row
  const bool nothing = st.m == -INFINITY && st.s == 0.0f;       // a NaN shows in s
  const float log_s = nothing ? 0.0f : log2f(st.s) * kLn2;
  if (tid == 0 && rank == 0) {
    if (logprob != nullptr) {
      const long long t = targets[r];
      logprob[r] = t < 0 || t >= vocab ? 0.0f : nothing ? -INFINITY : (to_f(row.p[t]) - st.m) * inv_t - log_s;
    }
    entropy[r] = nothing ? 0.0f : log_s - st.u / st.s * inv_t;
    if (stats != nullptr) {
      stats[2 * r] = st.m;
      stats[2 * r + 1] = nothing ? 0.0f : log2f(st.s);
    }
  }
  if (top == 0) {
    if (ctas > 1) cluster_sync();     // no CTA leaves while another reads its sums
    return;
  }

  auto sync = [&]() {
    if constexpr (WARPS > 1) __syncthreads();
    else __syncwarp();
  };
  // The highest bound, in the upper 16 bits of a key, that `top` threads reach (0 where there are not so many); finer bounds of
  // fp32 take more barriers than they leave out candidates.
  uint32_t bound = 0;
  auto settle = [&](int bit) {
    const bool reaches = best >= (bound | (1u << bit));
    int reached;
    if constexpr (WARPS > 1) reached = __syncthreads_count(reaches);
    else reached = __popc(__ballot_sync(0xffffffffu, reaches));
    if (reached >= top) bound |= 1u << bit;
  };
  for (int bit = 31; bit >= 16; --bit) settle(bit);
  if (tid == 0) {
    list_length = 0;
    final[sub][0] = st.m;
    final[sub][1] = log_s;
  }
  sync();
  auto entry = [](float x, long long j) { return (unsigned long long)order_key(x) << 32 | (uint32_t)(0xffffffffu - (uint32_t)j); };
  const float least = key_value(bound);                       // no logit that reaches the bound is below it
  for (int i = 0; i < batches; ++i) {
    if (best_of[(i >> fold) * kThreads + tid] < max(bound, 1u)) continue;
    if (*reinterpret_cast<volatile int*>(&list_length) > candidates) break;    // too many anyway
    const long long j0 = first + (long long)i * kBatch * hop;
    Raw<T, VEC> raw[kBatch];
    fetch(raw, j0);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const long long j = j0 + b * hop;
      uint32_t reach = 0;                                     // one bit for each logit of the vector
      if (bound > kNothing) {
        float x[VEC];
        raw[b].get(x);
#pragma unroll
        for (int q = 0; q < VEC; ++q) reach |= x[q] >= least ? 1u << q : 0u;
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) reach |= row.has(j + q) ? 1u << q : 0u;
      }
      while (reach != 0) {
        const int q = __ffs(reach) - 1;
        reach &= reach - 1;
        const int at = atomicAdd(&list_length, 1);
        if (at < candidates) list[at] = entry(to_f(row.p[j + q]), j + q);
      }
    }
  }
  sync();
  const int length = list_length;
  if (tid < kMaxTop) sorted[tid] = 0;
  sync();
  auto place_all = [&](int n) {
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long mine = list[i];
      int place = 0;
      for (int q = 0; q < n && place < top; ++q) place += list[q] > mine;
      if (place < top) sorted[place] = mine;
    }
  };
  int found = top;
  if (length <= candidates) {
    place_all(length);
  } else {
    // Many logits reach the bound: mostly equal ones.  With the bound exact, those above it go on the list, and of those that
    // equal it the first ones are taken in order.
    for (int bit = 15; bit >= 0; --bit) settle(bit);
    if (tid == 0) list_length = 0;
    sync();
    for (int i = 0; i < batches; ++i) {
      if (best_of[(i >> fold) * kThreads + tid] <= bound) continue;
      for (int b = 0; b < kBatch; ++b) {
        const long long j = first + (long long)(i * kBatch + b) * hop;
        float x[VEC];
        row.load(j).get(x);
#pragma unroll
        for (int q = 0; q < VEC; ++q)
          if (row.has(j + q) && order_key(x[q]) > bound) {
            const int at = atomicAdd(&list_length, 1);
            if (at < candidates) list[at] = entry(x[q], j + q);
          }
      }
    }
    sync();
    found = list_length;
    sync();
    if (found <= candidates) {
      place_all(found);
      sync();                                                 // the list is free
      uint32_t* totals = reinterpret_cast<uint32_t*>(list);
      for (long long base = first - tid * VEC; base < vocab && found < top; base += hop) {
        const long long j = base + tid * VEC;
        float x[VEC];
        row.load(j).get(x);
        uint32_t equal = 0;
#pragma unroll
        for (int q = 0; q < VEC; ++q) equal |= row.has(j + q) && order_key(x[q]) == bound ? 1u << q : 0u;
        const int mine = __popc(equal);
        int upto = mine;                                      // of this warp's lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int t = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += t;
        }
        if (lane == 31) totals[warp] = upto;
        sync();
        int place = found + upto - mine;
        for (int w = 0; w < WARPS; ++w) {
          if (w < warp) place += totals[w];
          found += totals[w];
        }
        for (; equal != 0 && place < top; equal &= equal - 1, ++place) {
          const int q = __ffs(equal) - 1;
          sorted[place] = (unsigned long long)bound << 32 | (uint32_t)(0xffffffffu - (uint32_t)(j + q));
        }
        sync();
      }
      found = top;
    }
  }
  if (found > candidates) {                                   // one pass for each
    unsigned long long last = ~0ull;
    for (int k = 0; k < top && last != 0; ++k) {
      unsigned long long mine = 0;
      for (long long j = first; j < vocab; j += hop) {
        float x[VEC];
        row.load(j).get(x);
#pragma unroll
        for (int q = 0; q < VEC; ++q) {
          const unsigned long long e = row.has(j + q) ? entry(x[q], j + q) : 0;
          if (e < last && e > mine) mine = e;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long e = __shfl_xor_sync(0xffffffffu, mine, o);
        if (e > mine) mine = e;
      }
      if (lane == 0) list[warp] = mine;
      sync();
      for (int w = 0; w < WARPS; ++w)
        if (list[w] > mine) mine = list[w];
      sync();
      if (tid == 0) sorted[k] = mine;
      last = mine;
    }
  }
  if (ctas > 1) cluster_sync(); else sync();
  if (rank == 0) {
    auto put = [&](int k, unsigned long long e) {
      top_ids[r * top + k] = (long long)(0xffffffffu - (uint32_t)e);
      const float m = final[sub][0], x = key_value((uint32_t)(e >> 32));
      top_logprobs[r * top + k] = m == -INFINITY && final[sub][1] == 0.0f ? -INFINITY : (x - m) * inv_t - final[sub][1];
    };
    if (ctas == 1) {
      if (tid < top) put(tid, sorted[tid]);
    } else {
      // the place of an entry: how many of all CTAs' entries come before it
      for (int i = tid; i < ctas * top; i += kThreads) list[i] = cluster_read(&sorted[i % top], i / top);
      __syncthreads();
      for (int i = tid; i < ctas * top; i += kThreads) {
        const unsigned long long mine = list[i];
        int place = 0;
        for (int q = 0; q < ctas * top; ++q) place += list[q] > mine;
        if (place < top && mine != 0) put(place, mine);
      }
    }
  }
  if (ctas > 1) cluster_sync();
}

// d_logits: a warp takes 32 * VEC * kBatch logits of one row.  Bound: reading the logits and writing the gradient;
// 1001 x 100003 fp32 120 us (6.6 TB/s), 400 x 250001 bf16 70 us (5.7 TB/s), 8192 x 4096 bf16 31 us (4.3 TB/s).
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
logprobs_bwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ targets, const float* __restrict__ stats,
                    const float* __restrict__ entropy, const float* __restrict__ d_logprob, const float* __restrict__ d_entropy,
                    T* __restrict__ d_logits, long long d_ld, long long rows, int vocab, float inv_t, unsigned parts) {
  constexpr int kBatch = 4;
  const unsigned long long w = ((unsigned long long)blockIdx.x * 256 + threadIdx.x) / 32;
  const long long r = w / parts;
  if (r >= rows) return;
  const Row<T, VEC> row(logits + r * ld, vocab);
  const int j0 = (int)(w % parts) * (32 * VEC * kBatch) + threadIdx.x % 32 * VEC - row.lead;
  Raw<T, VEC> raw[kBatch];
  if (j0 >= 0 && j0 + (kBatch - 1) * 32 * VEC + VEC <= vocab) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) raw[b] = load_raw<T, VEC>(row.p + j0 + b * 32 * VEC);
  } else {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) raw[b] = row.load(j0 + b * 32 * VEC);
  }
  T* out = d_logits + r * d_ld;
  const bool whole = (reinterpret_cast<uintptr_t>(out - row.lead) & 15) == 0;      // its vectors lie as the logits' do
  const float c = inv_t * kLog2e, m = stats[2 * r], log2_s = stats[2 * r + 1];
  const bool nothing = m == -INFINITY && log2_s == 0.0f;
  const long long t = targets != nullptr ? targets[r] : -1;
  const bool valid = t >= 0 && t < vocab && !nothing;
  const float dl = valid && d_logprob != nullptr ? d_logprob[r] * inv_t : 0.0f;
  const float dh = d_entropy != nullptr ? d_entropy[r] * inv_t : 0.0f;
  // d x = p (a + b log2 p) + dl 1[target]
  const float a = -fmaf(dh, entropy[r], dl), b2 = -dh * kLn2, mm = fmaxf(m, kLowest);
#pragma unroll
  for (int b = 0; b < kBatch; ++b) {
    const int j = j0 + b * 32 * VEC;
    float x[VEC];
    raw[b].get(x);
    if (nothing) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = 0.0f;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        const float2 lp = __ffma2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), both(-mm)), both(c), both(-log2_s));
        const float2 p = make_float2(ex2(lp.x), ex2(lp.y));
        const float2 g = __fmul2_rn(p, __ffma2_rn(both(b2), make_float2(fmaxf(lp.x, kFar), fmaxf(lp.y, kFar)), both(a)));
        x[i] = g.x;
        x[i + 1] = g.y;
      }
    }
    if (valid && t - j < VEC && t >= j) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (t == j + i) x[i] += dl;
    }
    Raw<T, VEC> g;
    g.set(x);
    if (whole && j >= 0 && j + VEC <= vocab) {
      *reinterpret_cast<uint4*>(out + j) = *reinterpret_cast<const uint4*>(&g);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (row.has(j + i)) out[j + i] = g.v[i];
    }
  }
}

// The largest Row::lead
template <typename T>
int most_lead(const void* p, long long ld) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * sizeof(T) % 16 == 0 ? 0 : 16 / sizeof(T) - 1;
}

struct FwdArgs {
  const void* logits;
  long long ld;
  const long long* targets;
  float *logprob, *entropy, *stats, *top_logprobs;
  long long *top_ids, rows;
  int vocab, top;
  float inv_t;
};

template <typename T, int VEC, int WARPS, int ROWS>
int launch_fwd_w(const FwdArgs& a, int ctas, cudaStream_t s) {
  const long long step = (long long)ctas * WARPS * 32 * VEC * kBatchOf<VEC>, batches = (a.vocab + most_lead<T>(a.logits, a.ld) + step - 1) / step;
  const long long candidates = ROWS > 1 ? 256 : 1024, blocks = ROWS > 1 ? (a.rows + ROWS - 1) / ROWS : a.rows * ctas;
  int fold = 0;
  auto smem_of = [&]() { return a.top > 0 ? ROWS * ((candidates + kMaxTop) * 8 + (((batches - 1) >> fold) + 1) * WARPS * 32 * 4) : 0; };
  while (WARPS > 1 && smem_of() > 220 * 1024) ++fold;
  const long long smem = smem_of();
  if (blocks > 0x7fffffffll || smem > 220 * 1024) return GEMM_ERR_SHAPE;
  auto kernel = logprobs_fwd_kernel<T, VEC, WARPS, ROWS>;
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return GEMM_ERR_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(WARPS * ROWS * 32);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {(unsigned)ctas, 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, (const T*)a.logits, a.ld, a.targets, a.logprob, a.entropy, a.stats, a.top_logprobs, a.top_ids,
                            a.rows, a.vocab, a.top, a.inv_t, (int)batches, fold, (int)candidates) == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

// Warps of a row: one where the rows alone fill half the machine's warp slots, more for fewer rows and for long ones, whose
// last ones would run alone.  CTAs of a row where sixteen warps of each are not two CTAs per SM.  us without | with alternatives
// (5, 20, 32) by warps, and CTAs of sixteen:
//   8192 x 4096 bf16      1: 24 | 36    4: 29 | 49     16: 118 | 205
//   4096 x 1000 fp16      1: 10 | 14    4: 20 | 34     16: 57 | 96
//   1001 x 100003 fp32    4: 86 | 104   16: 88 | 115
//   400 x 250001 bf16     4: 80 | 104   16: 61 | 79
//   16 x 262144 bf16      4: 63 | 84    16: 27 | 35    2 CTAs: 18 | 31    8 CTAs: 13 | 23
// (all with the logits going through L1)
template <typename T, int VEC>
int launch_fwd(const FwdArgs& a, cudaStream_t s) {
  constexpr int unit = 32 * VEC * kBatchOf<VEC>;
  const long long units = ((long long)a.vocab + unit - 1) / unit;      // batches of a warp
  long long warps = 1, ctas = 1;
  while (warps < 16 && warps < units && (a.rows * warps < 148 * 16 || units > 32 * warps)) warps *= 4;
  if (warps == 16)
    while (ctas < kMaxCtas && ctas * 16 < units && a.rows * ctas * 2 <= 2 * 148) ctas *= 2;
  return warps == 1 ? launch_fwd_w<T, VEC, 1, 4>(a, 1, s) : warps == 4 ? launch_fwd_w<T, VEC, 4, 1>(a, (int)ctas, s)
                                                                      : launch_fwd_w<T, VEC, 16, 1>(a, (int)ctas, s);
}

template <typename T, int VEC>
int launch_bwd(const void* logits, long long ld, const long long* targets, const float* stats, const float* entropy,
               const float* d_logprob, const float* d_entropy, void* d_logits, long long d_ld, long long rows, int vocab,
               float inv_t, cudaStream_t s) {
  const long long parts = ((long long)vocab + most_lead<T>(logits, ld) + 32 * VEC * 4 - 1) / (32 * VEC * 4), blocks = (rows * parts + 7) / 8;
  if (blocks > 0x7fffffffll) return GEMM_ERR_SHAPE;
  logprobs_bwd_kernel<T, VEC><<<(unsigned)blocks, 256, 0, s>>>((const T*)logits, ld, targets, stats, entropy, d_logprob, d_entropy,
                                                               (T*)d_logits, d_ld, rows, vocab, inv_t, (unsigned)parts);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

}  // namespace

// logits: rows of pitch ld, elements or fp32.  targets and logprob may be null together; top = 0 takes no alternatives.
// stats: two floats a row for the backward, or null.
extern "C" int fbam_logprobs_fwd(const void* logits, int fp32, long long ld, const long long* targets, float* logprob,
                                 float* entropy, float* stats, float* top_logprobs, long long* top_ids, long long rows,
                                 int vocab, int top, float inv_temperature, void* stream) {
  if (rows <= 0 || rows > 0x7fffffffll || vocab <= 0 || vocab > 0x3fffffff || top < 0 || top > vocab || top > kMaxTop) return GEMM_ERR_SHAPE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto f = fp32 ? launch_fwd<float, 4> : launch_fwd<elem_t, 8>;
  return f({logits, ld, targets, logprob, entropy, stats, top_logprobs, top_ids, rows, vocab, top, inv_temperature}, s);
}

extern "C" int fbam_logprobs_bwd(const void* logits, int fp32, long long ld, const long long* targets, const float* stats,
                                 const float* entropy, const float* d_logprob, const float* d_entropy, void* d_logits,
                                 long long d_ld, long long rows, int vocab, float inv_temperature, void* stream) {
  if (rows <= 0 || vocab <= 0 || vocab > 0x3fffffff) return GEMM_ERR_SHAPE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  auto f = fp32 ? launch_bwd<float, 4> : launch_bwd<elem_t, 8>;
  return f(logits, ld, targets, stats, entropy, d_logprob, d_entropy, d_logits, d_ld, rows, vocab, inv_temperature, s);
}
