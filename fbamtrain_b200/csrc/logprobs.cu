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
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(elem_t x) { return e2f(x); }

template <int N>
__device__ __forceinline__ void load_row(const float* p, float (&v)[N]) {
  if constexpr (N == 4) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = p[i];
  }
}
template <int N>
__device__ __forceinline__ void load_row(const elem_t* p, float (&v)[N]) {
  if constexpr (N == 8) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const elem2_t* h = reinterpret_cast<const elem2_t*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = e22ff(h[i]);
      v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = e2f(p[i]);
  }
}
template <int N>
__device__ __forceinline__ void store_row(float* p, const float (&v)[N]) {
  if constexpr (N == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = v[i];
  }
}
template <int N>
__device__ __forceinline__ void store_row(elem_t* p, const float (&v)[N]) {
  if constexpr (N == 8) {
    __align__(16) elem2_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = ff2e2(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(h);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = f2e(v[i]);
  }
}

// Sums of part of a row relative to its maximum; t = (x - m) in units of the logits.
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

// A key that orders floats by value; NaN counts as -inf.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) x = -INFINITY;
  if (x == 0.0f) x = 0.0f;          // -0 and 0 are one value
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}

template <typename T, int VEC>
struct Row {
  const T* p;
  int vocab;
  // the VEC logits from j on; -inf behind the end of the row
  __device__ __forceinline__ void load(int j, float (&v)[VEC]) const {
    if (j + VEC <= vocab) {
      load_row<VEC>(p + j, v);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = j + i < vocab ? to_f(p[j + i]) : -INFINITY;
    }
  }
};

// One row per CTA of WARPS warps.  A group is what one warp reads at once, 32 * VEC neighbouring logits; group_key keeps the
// key of the best logit of each that was not taken (0: none is left) for the alternatives.
template <typename T, int VEC, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
logprobs_fwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ targets, float* __restrict__ logprob,
                    float* __restrict__ entropy, float* __restrict__ stats, float* __restrict__ top_logprobs,
                    long long* __restrict__ top_ids, int vocab, int top, float inv_t) {
  extern __shared__ uint32_t group_key[];
  __shared__ Stats parts[WARPS];
  constexpr int kGroup = 32 * VEC, kBatch = 4;
  const long long r = blockIdx.x;
  const Row<T, VEC> row{logits + r * ld, vocab};
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int groups = (vocab + kGroup - 1) / kGroup;
  const float c = inv_t * kLog2e;

  Stats st{-INFINITY, 0.0f, 0.0f};
  for (int g0 = warp; g0 < groups; g0 += kBatch * WARPS) {
    float x[kBatch][VEC], gm[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) row.load((g0 + b * WARPS) * kGroup + lane * VEC, x[b]);
    float top_x = st.m;
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      gm[b] = -INFINITY;
#pragma unroll
      for (int i = 0; i < VEC; ++i) gm[b] = fmaxf(gm[b], x[b][i]);
      top_x = fmaxf(top_x, gm[b]);
    }
    if (top > 0) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) gm[b] = fmaxf(gm[b], __shfl_xor_sync(0xffffffffu, gm[b], o));
        if (lane == 0 && g0 + b * WARPS < groups) group_key[g0 + b * WARPS] = order_key(gm[b]);
      }
    }
    if (top_x > st.m) st.move_to(top_x, c);
    const float m = fmaxf(st.m, kLowest);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = max_nan(x[b][i] - m, kFar);
        const float e = ex2(d * c);
        st.s += e;
        st.u = fmaf(e, d, st.u);
      }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o), __shfl_xor_sync(0xffffffffu, st.u, o)};
    st.join(other, c);
  }
  if (lane == 0) parts[warp] = st;
  __syncthreads();
  if (warp != 0) return;
  st = parts[0];
  for (int w = 1; w < WARPS; ++w) st.join(parts[w], c);
  const bool nothing = st.m == -INFINITY && st.s == 0.0f;       // a NaN shows in s
  const float log_s = nothing ? 0.0f : log2f(st.s) * kLn2;
  auto log_p = [&](float x) { return nothing ? -INFINITY : (x - st.m) * inv_t - log_s; };
  if (lane == 0) {
    if (logprob != nullptr) {
      const long long t = targets[r];
      logprob[r] = t >= 0 && t < vocab ? log_p(to_f(row.p[t])) : 0.0f;
    }
    entropy[r] = nothing ? 0.0f : log_s - st.u / st.s * inv_t;
    stats[2 * r] = st.m;
    stats[2 * r + 1] = nothing ? 0.0f : log2f(st.s);
  }
  // The alternatives: what comes next is the best of the groups' best, and its group's best is then looked for again among
  // what comes behind it.
  for (int k = 0; k < top; ++k) {
    uint32_t best = 0;
    int best_g = 0;
    for (int g = lane; g < groups; g += 32) {
      const uint32_t key = group_key[g];
      if (key > best) { best = key; best_g = g; }
    }
    const uint32_t all = __reduce_max_sync(0xffffffffu, best);
    best_g = __reduce_min_sync(0xffffffffu, best == all ? best_g : 0x7fffffff);
    // the place of the group's best: the first logit of that value that was not taken
    float v[VEC];
    const int j0 = best_g * kGroup + lane * VEC;
    row.load(j0, v);
    int at = 0x7fffffff;
#pragma unroll
    for (int i = VEC - 1; i >= 0; --i) {
      bool taken = j0 + i >= vocab;
      for (int q = 0; q < k; ++q) taken |= top_ids[r * top + q] == j0 + i;
      if (!taken && order_key(v[i]) == all) at = j0 + i;
    }
    at = min(__reduce_min_sync(0xffffffffu, at), vocab - 1);
    float rest = -INFINITY;
    bool any = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      bool taken = j0 + i >= vocab || j0 + i == at;
      for (int q = 0; q < k; ++q) taken |= top_ids[r * top + q] == j0 + i;
      if (!taken) { rest = fmaxf(rest, v[i]); any = true; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) rest = fmaxf(rest, __shfl_xor_sync(0xffffffffu, rest, o));
    any = __any_sync(0xffffffffu, any);
    if (lane == 0) {
      top_ids[r * top + k] = at;
      top_logprobs[r * top + k] = log_p(to_f(row.p[at]));
      group_key[best_g] = any ? order_key(rest) : 0;
    }
    __syncwarp();
  }
}

// d_logits of one row part per CTA.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
logprobs_bwd_kernel(const T* __restrict__ logits, long long ld, const long long* __restrict__ targets, const float* __restrict__ stats,
                    const float* __restrict__ entropy, const float* __restrict__ d_logprob, const float* __restrict__ d_entropy,
                    T* __restrict__ d_logits, long long d_ld, int vocab, float inv_t, int parts) {
  const long long r = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const Row<T, VEC> row{logits + r * ld, vocab};
  T* out = d_logits + r * d_ld;
  const float c = inv_t * kLog2e, m = stats[2 * r], log2_s = stats[2 * r + 1];
  const bool nothing = m == -INFINITY && log2_s == 0.0f;
  const long long t = targets != nullptr ? targets[r] : -1;
  const bool valid = t >= 0 && t < vocab && !nothing;
  const float dl = valid && d_logprob != nullptr ? d_logprob[r] * inv_t : 0.0f;
  const float dh = d_entropy != nullptr ? d_entropy[r] * inv_t : 0.0f;
  // d x = p (a + b log2 p) + dl 1[target]
  const float a = -fmaf(dh, entropy[r], dl), b = -dh * kLn2, mm = fmaxf(m, kLowest);
  for (int j = (part * 256 + threadIdx.x) * VEC; j < vocab; j += parts * 256 * VEC) {
    float x[VEC];
    row.load(j, x);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float lp = fmaf(max_nan(x[i] - mm, kFar), c, -log2_s);
      const float p = nothing ? 0.0f : ex2(lp);
      x[i] = p * fmaf(b, lp, a) + (j + i == t ? dl : 0.0f);
      if (nothing) x[i] = 0.0f;
    }
    if (j + VEC <= vocab) {
      store_row<VEC>(out + j, x);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (j + i < vocab) {
          float one[1] = {x[i]};
          store_row<1>(out + j + i, one);
        }
    }
  }
}

bool aligned16(const void* p, long long ld, int size) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * size % 16 == 0; }

template <typename T, int VEC, int WARPS>
int launch_fwd_w(const void* logits, long long ld, const long long* targets, float* logprob, float* entropy, float* stats,
                 float* top_logprobs, long long* top_ids, long long rows, int vocab, int top, float inv_t, cudaStream_t s) {
  const int smem = top > 0 ? (vocab + 32 * VEC - 1) / (32 * VEC) * (int)sizeof(float) : 0;
  if (smem > 48 * 1024) {
    if (smem > 200 * 1024) return GEMM_ERR_SHAPE;
    if (cudaFuncSetAttribute(logprobs_fwd_kernel<T, VEC, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
      return GEMM_ERR_LAUNCH;
  }
  logprobs_fwd_kernel<T, VEC, WARPS><<<(unsigned)rows, WARPS * 32, smem, s>>>((const T*)logits, ld, targets, logprob, entropy,
                                                                              stats, top_logprobs, top_ids, vocab, top, inv_t);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

template <typename T, int VEC>
int launch_fwd(const void* logits, long long ld, const long long* targets, float* logprob, float* entropy, float* stats,
               float* top_logprobs, long long* top_ids, long long rows, int vocab, int top, float inv_t, cudaStream_t s) {
  const int groups = (vocab + 32 * VEC - 1) / (32 * VEC);
  auto f = groups <= 4 ? launch_fwd_w<T, VEC, 1> : groups <= 32 ? launch_fwd_w<T, VEC, 4> : launch_fwd_w<T, VEC, 16>;
  return f(logits, ld, targets, logprob, entropy, stats, top_logprobs, top_ids, rows, vocab, top, inv_t, s);
}

template <typename T, int VEC>
int launch_bwd(const void* logits, long long ld, const long long* targets, const float* stats, const float* entropy,
               const float* d_logprob, const float* d_entropy, void* d_logits, long long d_ld, long long rows, int vocab,
               float inv_t, cudaStream_t s) {
  int parts = (vocab + 256 * VEC * 4 - 1) / (256 * VEC * 4);
  if (rows * parts > 0x7fffffffll) return GEMM_ERR_SHAPE;
  logprobs_bwd_kernel<T, VEC><<<(unsigned)(rows * parts), 256, 0, s>>>((const T*)logits, ld, targets, stats, entropy, d_logprob,
                                                                       d_entropy, (T*)d_logits, d_ld, vocab, inv_t, parts);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

}  // namespace

// logits: rows of pitch ld, elements or fp32.  targets and logprob may be null together; top = 0 takes no alternatives.
// stats: two floats a row for the backward.
extern "C" int fbam_logprobs_fwd(const void* logits, int fp32, long long ld, const long long* targets, float* logprob,
                                 float* entropy, float* stats, float* top_logprobs, long long* top_ids, long long rows,
                                 int vocab, int top, float inv_temperature, void* stream) {
  if (rows <= 0 || rows > 0x7fffffffll || vocab <= 0 || vocab > 0x3fffffff || top < 0 || top > vocab) return GEMM_ERR_SHAPE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool vec = aligned16(logits, ld, fp32 ? 4 : 2);
  auto f = fp32 ? (vec ? launch_fwd<float, 4> : launch_fwd<float, 1>) : (vec ? launch_fwd<elem_t, 8> : launch_fwd<elem_t, 1>);
  return f(logits, ld, targets, logprob, entropy, stats, top_logprobs, top_ids, rows, vocab, top, inv_temperature, s);
}

extern "C" int fbam_logprobs_bwd(const void* logits, int fp32, long long ld, const long long* targets, const float* stats,
                                 const float* entropy, const float* d_logprob, const float* d_entropy, void* d_logits,
                                 long long d_ld, long long rows, int vocab, float inv_temperature, void* stream) {
  if (rows <= 0 || vocab <= 0 || vocab > 0x3fffffff) return GEMM_ERR_SHAPE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const bool vec = aligned16(logits, ld, fp32 ? 4 : 2) && aligned16(d_logits, d_ld, fp32 ? 4 : 2);
  auto f = fp32 ? (vec ? launch_bwd<float, 4> : launch_bwd<float, 1>) : (vec ? launch_bwd<elem_t, 8> : launch_bwd<elem_t, 1>);
  return f(logits, ld, targets, stats, entropy, d_logprob, d_entropy, d_logits, d_ld, rows, vocab, inv_temperature, s);
}
