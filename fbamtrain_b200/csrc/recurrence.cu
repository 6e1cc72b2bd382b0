// Gated linear recurrence over sequences (batch, steps, 3, dim): candidates z, gates g and output gates o,
//   f = sigmoid(g)     h_t = f_t (reset_t ? 0 : h_{t-1}) + (1 - f_t) z_t     y_t = sigmoid(o_t) h_t
// and its gradient, with e_t = what step t hands to the step before it:
//   dh_t = dy_t sigmoid(o_t) + e_{t+1}      e_t = (reset_t ? 0 : f_t) dh_t
//   dz = (1 - f) dh     dg = (h_{t-1} - z) f (1 - f) dh     do = dy h sigmoid(o) (1 - sigmoid(o))
// Both directions are scans of x -> a x + b: a warp takes 32 x VEC channels of kSteps consecutive steps, all warps of a CTA
// take consecutive chunks, and what a chunk does to a value that comes in, (product of a, result from 0), is passed on in
// shared memory before every warp walks its chunk again from the true value.  The state is fp32 throughout; the forward leaves
// the state in front of every chunk for the backward, which rebuilds h from it in registers.
#include <cuda_runtime.h>
#include <stdint.h>

#include "elem16.cuh"
#include "gemm_tcgen05.h"

namespace {

constexpr int kSteps = 16;        // steps of a chunk

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// sigmoid(x) and sigmoid(-x), both to full relative accuracy
__device__ __forceinline__ void gate(float x, float& f, float& f1) {
  const float e = ex2(-1.4426950408889634f * fabsf(x));
  const float p = rcp(1.0f + e), q = e * p;
  f = x >= 0.0f ? p : q;
  f1 = x >= 0.0f ? q : p;
  if (x != x) f = f1 = x;
}

template <int VEC>
struct Vec { float v[VEC]; };
template <int VEC>
__device__ __forceinline__ Vec<VEC> load(const elem_t* p) {
  Vec<VEC> r;
  if constexpr (VEC == 2) {
    const float2 f = e22ff(*reinterpret_cast<const elem2_t*>(p));
    r.v[0] = f.x; r.v[1] = f.y;
  } else {
    r.v[0] = e2f(*p);
  }
  return r;
}
template <int VEC>
__device__ __forceinline__ void store(elem_t* p, const Vec<VEC>& r) {
  if constexpr (VEC == 2) *reinterpret_cast<elem2_t*>(p) = ff2e2(r.v[0], r.v[1]);
  else *p = f2e(r.v[0]);
}

// What a chunk makes of a value that comes in.  A gain below 0 marks a chunk with a reset: nothing of what comes in goes on,
// not even as a product of 0 with an infinity or a NaN of the sequence before.
template <int VEC>
__device__ __forceinline__ Vec<VEC> drops() {
  Vec<VEC> r;
#pragma unroll
  for (int j = 0; j < VEC; ++j) r.v[j] = -1.0f;
  return r;
}
__device__ __forceinline__ float pass(float gain, float from0, float x) { return gain < 0.0f ? from0 : fmaf(gain, x, from0); }

struct Shape {
  int batch, steps, dim, chunks;
  long long zb, zt, zk;             // strides of zgo: sequence, step, member
  long long yb, yt;                 // of y, or of dy in the backward
  long long rb, rt;                 // of the resets
};

// The reset flags of a chunk, one bit a step; the same in all lanes.
__device__ __forceinline__ uint32_t reset_bits(const uint8_t* resets, const Shape& s, int b, int t0, int n) {
  if (resets == nullptr) return 0;
  const int lane = threadIdx.x % 32;
  const bool r = lane < n && resets[b * s.rb + (t0 + lane) * s.rt] != 0;
  return __ballot_sync(0xffffffffu, r);
}

template <int VEC, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
recurrence_fwd_kernel(const elem_t* __restrict__ zgo, const float* __restrict__ state_in, const uint8_t* __restrict__ resets,
                      elem_t* __restrict__ y, float* __restrict__ state_out, float* __restrict__ saved, const Shape s) {
  __shared__ Vec<VEC> gain[WARPS][32], from0[WARPS][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int b = blockIdx.y, ch = (blockIdx.x * 32 + lane) * VEC;
  const bool in = ch < s.dim;
  const elem_t* src = zgo + b * s.zb + ch;
  Vec<VEC> h_in = {};
  if (in && state_in != nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) h_in.v[j] = state_in[(long long)b * s.dim + ch + j];
  }
  for (int c0 = 0; c0 < s.chunks; c0 += WARPS) {
    const int chunk = c0 + warp, t0 = chunk * kSteps;
    const int n = min(kSteps, s.steps - t0);                // may be below 0
    const uint32_t bits = reset_bits(resets, s, b, t0, n);
    Vec<VEC> z[kSteps], q[kSteps], o[kSteps];
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
      z[t] = q[t] = o[t] = Vec<VEC>{};
      if (in && t < n) {
        const elem_t* p = src + (t0 + t) * s.zt;
        z[t] = load<VEC>(p);
        q[t] = load<VEC>(p + s.zk);
        o[t] = load<VEC>(p + 2 * s.zk);
      }
    }
    Vec<VEC> a, h;
#pragma unroll
    for (int j = 0; j < VEC; ++j) { a.v[j] = 1.0f; h.v[j] = 0.0f; }
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
      const bool reset = (bits >> t) & 1;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float f, f1;
        gate(q[t].v[j], f, f1);
        if (t >= n) f1 = 0.0f;                              // steps behind the end change nothing
        q[t].v[j] = f1;
        // h - (1 - f) (h - z): 1 - f is known to its last bits where f is near 1
        if (reset) h.v[j] = 0.0f;
        h.v[j] = fmaf(f1, z[t].v[j] - h.v[j], h.v[j]);
        a.v[j] = fmaf(-f1, a.v[j], a.v[j]);
      }
    }
    gain[warp][lane] = bits ? drops<VEC>() : a;
    from0[warp][lane] = h;
    __syncthreads();
    Vec<VEC> mine = h_in;
    h = h_in;
    for (int w = 0; w < WARPS; ++w) {
      if (w == warp) mine = h;
#pragma unroll
      for (int j = 0; j < VEC; ++j) h.v[j] = pass(gain[w][lane].v[j], from0[w][lane].v[j], h.v[j]);
    }
    h_in = h;
    __syncthreads();
    h = mine;
    if (in && saved != nullptr && n > 0) {
      float* at = saved + ((long long)b * s.chunks + chunk) * s.dim + ch;
#pragma unroll
      for (int j = 0; j < VEC; ++j) at[j] = h.v[j];
    }
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
      Vec<VEC> out;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if ((bits >> t) & 1) h.v[j] = 0.0f;
        h.v[j] = fmaf(q[t].v[j], z[t].v[j] - h.v[j], h.v[j]);
        float f, f1;
        gate(o[t].v[j], f, f1);
        out.v[j] = f * h.v[j];
      }
      if (in && t < n) store<VEC>(y + b * s.yb + (t0 + t) * s.yt + ch, out);
    }
    if (in && t0 + kSteps >= s.steps && n > 0) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) state_out[(long long)b * s.dim + ch + j] = h.v[j];
    }
  }
}

template <int VEC, int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
recurrence_bwd_kernel(const elem_t* __restrict__ zgo, const uint8_t* __restrict__ resets, const float* __restrict__ saved,
                      const elem_t* __restrict__ dy, const float* __restrict__ d_state_out, elem_t* __restrict__ d_zgo,
                      float* __restrict__ d_state_in, const Shape s, long long db, long long dt) {
  __shared__ Vec<VEC> gain[WARPS][32], from0[WARPS][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int b = blockIdx.y, ch = (blockIdx.x * 32 + lane) * VEC;
  const bool in = ch < s.dim;
  const elem_t* src = zgo + b * s.zb + ch;
  Vec<VEC> e_in = {};
  if (in && d_state_out != nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) e_in.v[j] = d_state_out[(long long)b * s.dim + ch + j];
  }
  const int rounds = (s.chunks + WARPS - 1) / WARPS;
  for (int round = rounds - 1; round >= 0; --round) {
    const int chunk = round * WARPS + warp, t0 = chunk * kSteps;
    const int n = min(kSteps, s.steps - t0);
    const uint32_t bits = reset_bits(resets, s, b, t0, n);
    Vec<VEC> h[kSteps], z[kSteps], q[kSteps], o[kSteps], d[kSteps], h0 = {};
#pragma unroll
    for (int t = 0; t < kSteps; ++t) {
      z[t] = q[t] = o[t] = d[t] = Vec<VEC>{};
      if (in && t < n) {
        const elem_t* p = src + (t0 + t) * s.zt;
        z[t] = load<VEC>(p);
        q[t] = load<VEC>(p + s.zk);
        o[t] = load<VEC>(p + 2 * s.zk);
        d[t] = load<VEC>(dy + b * s.yb + (t0 + t) * s.yt + ch);
      }
    }
    if (in && n > 0) {
      const float* at = saved + ((long long)b * s.chunks + chunk) * s.dim + ch;
#pragma unroll
      for (int j = 0; j < VEC; ++j) h0.v[j] = at[j];
    }
    Vec<VEC> a, e = h0;
#pragma unroll
    for (int t = 0; t < kSteps; ++t)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if ((bits >> t) & 1) e.v[j] = 0.0f;
        float f, f1;
        gate(q[t].v[j], f, f1);
        e.v[j] = fmaf(f1, z[t].v[j] - e.v[j], e.v[j]);
        h[t].v[j] = e.v[j];
      }
#pragma unroll
    for (int j = 0; j < VEC; ++j) { a.v[j] = 1.0f; e.v[j] = 0.0f; }
#pragma unroll
    for (int t = kSteps - 1; t >= 0; --t)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (t >= n) continue;
        float f, f1, so, so1;
        gate(q[t].v[j], f, f1);
        gate(o[t].v[j], so, so1);
        e.v[j] = (bits >> t) & 1 ? 0.0f : f * fmaf(d[t].v[j], so, e.v[j]);
        a.v[j] *= f;
      }
    gain[warp][lane] = bits ? drops<VEC>() : a;
    from0[warp][lane] = e;
    __syncthreads();
    Vec<VEC> mine = e_in;
    e = e_in;
    for (int w = WARPS - 1; w >= 0; --w) {
      if (w == warp) mine = e;
#pragma unroll
      for (int j = 0; j < VEC; ++j) e.v[j] = pass(gain[w][lane].v[j], from0[w][lane].v[j], e.v[j]);
    }
    e_in = e;
    __syncthreads();
    e = mine;
#pragma unroll
    for (int t = kSteps - 1; t >= 0; --t) {
      if (t >= n) continue;
      Vec<VEC> dz, dg, dout;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const bool reset = (bits >> t) & 1;
        float f, f1, so, so1;
        gate(q[t].v[j], f, f1);
        gate(o[t].v[j], so, so1);
        const float dh = fmaf(d[t].v[j], so, e.v[j]);
        const float before = reset ? 0.0f : t > 0 ? h[t > 0 ? t - 1 : 0].v[j] : h0.v[j];
        dz.v[j] = f1 * dh;
        dg.v[j] = (before - z[t].v[j]) * f * f1 * dh;
        dout.v[j] = d[t].v[j] * h[t].v[j] * so * so1;
        e.v[j] = reset ? 0.0f : f * dh;
      }
      if (in) {
        elem_t* p = d_zgo + b * db + (t0 + t) * dt + ch;
        store<VEC>(p, dz);
        store<VEC>(p + s.dim, dg);
        store<VEC>(p + 2 * s.dim, dout);
      }
    }
  }
  if (in && warp == 0 && d_state_in != nullptr) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) d_state_in[(long long)b * s.dim + ch + j] = e_in.v[j];
  }
}

// Two neighbouring channels per lane where they lie on 4-byte boundaries
bool pairs(const void* p, int dim, long long a, long long b, long long c) {
  return dim % 2 == 0 && ((a | b | c) & 1) == 0 && (reinterpret_cast<uintptr_t>(p) & 3) == 0;
}

template <int VEC, int WARPS>
int launch_fwd(const void* zgo, const float* state_in, const uint8_t* resets, void* y, float* state_out, float* saved,
               const Shape& s, cudaStream_t stream) {
  const dim3 grid((s.dim + 32 * VEC - 1) / (32 * VEC), s.batch);
  recurrence_fwd_kernel<VEC, WARPS><<<grid, WARPS * 32, 0, stream>>>((const elem_t*)zgo, state_in, resets, (elem_t*)y, state_out, saved, s);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

template <int VEC, int WARPS>
int launch_bwd(const void* zgo, const uint8_t* resets, const float* saved, const void* dy, const float* d_state_out,
               void* d_zgo, float* d_state_in, const Shape& s, long long db, long long dt, cudaStream_t stream) {
  const dim3 grid((s.dim + 32 * VEC - 1) / (32 * VEC), s.batch);
  recurrence_bwd_kernel<VEC, WARPS><<<grid, WARPS * 32, 0, stream>>>((const elem_t*)zgo, resets, saved, (const elem_t*)dy, d_state_out,
                                                                     (elem_t*)d_zgo, d_state_in, s, db, dt);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}

}  // namespace

// Steps of a chunk: the forward's `saved` has [batch][ceil(steps / this)][dim] fp32 values (null where no backward follows).
extern "C" int fbam_recurrence_chunk() { return kSteps; }

// zgo: strides zb, zt, zk (sequence, step, member; channels dense); y: yb, yt; resets (bytes, or null): rb, rt.  state_in
// (batch, dim) fp32 or null for zeros.
extern "C" int fbam_recurrence_fwd(const void* zgo, long long zb, long long zt, long long zk, const float* state_in,
                                   const uint8_t* resets, long long rb, long long rt, void* y, long long yb, long long yt,
                                   float* state_out, float* saved, int batch, int steps, int dim, void* stream) {
  if (batch <= 0 || steps <= 0 || dim <= 0 || batch > 65535 || steps > 0x3fffffff) return GEMM_ERR_SHAPE;
  const Shape s{batch, steps, dim, (steps + kSteps - 1) / kSteps, zb, zt, zk, yb, yt, rb, rt};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool two = pairs(zgo, dim, zb, zt, zk) && pairs(y, dim, yb, yt, 0);
  auto f = s.chunks == 1 ? (two ? launch_fwd<2, 1> : launch_fwd<1, 1>) : (two ? launch_fwd<2, 8> : launch_fwd<1, 8>);
  return f(zgo, state_in, resets, y, state_out, saved, s, st);
}

// dy: strides yb, yt; d_zgo: db, dt and dense (3, dim) steps.  d_state_out and d_state_in (batch, dim) fp32 or null.
extern "C" int fbam_recurrence_bwd(const void* zgo, long long zb, long long zt, long long zk, const uint8_t* resets,
                                   long long rb, long long rt, const float* saved, const void* dy, long long yb, long long yt,
                                   const float* d_state_out, void* d_zgo, long long db, long long dt, float* d_state_in,
                                   int batch, int steps, int dim, void* stream) {
  if (batch <= 0 || steps <= 0 || dim <= 0 || batch > 65535 || steps > 0x3fffffff) return GEMM_ERR_SHAPE;
  const Shape s{batch, steps, dim, (steps + kSteps - 1) / kSteps, zb, zt, zk, yb, yt, rb, rt};
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const bool two = pairs(zgo, dim, zb, zt, zk) && pairs(dy, dim, yb, yt, 0) && pairs(d_zgo, dim, db, dt, 0);
  auto f = s.chunks == 1 ? (two ? launch_bwd<2, 1> : launch_bwd<1, 1>) : (two ? launch_bwd<2, 8> : launch_bwd<1, 8>);
  return f(zgo, resets, saved, dy, d_state_out, d_zgo, d_state_in, s, db, dt, st);
}
