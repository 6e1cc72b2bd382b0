// Gated feed-forward block: h = v * act(g) with (v, g) = x W_inᵀ + b_in, value rows first, and its gradient
//   dv = dh act(g)     dg = dh v act'(g).
#include <cuda_runtime.h>
#include <stdint.h>

#include "elem16.cuh"
#include "gelu_math.cuh"
#include "gemm_tcgen05.h"

namespace {

enum { GATE_GELU = 0, GATE_SILU = 1 };

// act(g) and act'(g) of two values
__device__ __forceinline__ void gate2(float2 g, int act, float2& a, float2& da) {
  if (act == GATE_GELU) {
    a = gelu_math::gelu2(g);
    da = gelu_math::gelu_grad2(g);
  } else {
    const float sx = gelu_math::rcp_approx(1.0f + gelu_math::ex2_approx(-1.4426950408889634f * g.x));
    const float sy = gelu_math::rcp_approx(1.0f + gelu_math::ex2_approx(-1.4426950408889634f * g.y));
    a = make_float2(g.x * sx, g.y * sy);
    da = make_float2(sx * fmaf(g.x, 1.0f - sx, 1.0f), sy * fmaf(g.y, 1.0f - sy, 1.0f));
  }
}

// vg (rows, 2 inner) fp32; h (rows, inner); with dh (rows, inner) fp32: d_vg (rows, 2 inner) instead.  inner % 8 == 0.
__global__ void gated_act_kernel(const float* __restrict__ vg, const float* __restrict__ dh, elem_t* __restrict__ out, long long n,
                                 int inner, int act) {
  for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 2; i < n; i += (long long)gridDim.x * blockDim.x * 2) {
    const long long r = i / inner, c = i % inner;
    const float2 v = *reinterpret_cast<const float2*>(vg + r * 2 * inner + c);
    const float2 g = *reinterpret_cast<const float2*>(vg + r * 2 * inner + inner + c);
    float2 a, da;
    gate2(g, act, a, da);
    if (dh == nullptr) {
      *reinterpret_cast<elem2_t*>(out + i) = ff2e2(v.x * a.x, v.y * a.y);
    } else {
      const float2 d = *reinterpret_cast<const float2*>(dh + i);
      *reinterpret_cast<elem2_t*>(out + r * 2 * inner + c) = ff2e2(d.x * a.x, d.y * a.y);
      *reinterpret_cast<elem2_t*>(out + r * 2 * inner + inner + c) = ff2e2(d.x * v.x * da.x, d.y * v.y * da.y);
    }
  }
}

}  // namespace

extern "C" int fbam_gated_act(const float* vg, const float* dh, void* out, long long rows, int inner, int act, void* stream) {
  if (rows <= 0 || inner <= 0 || inner % 8 != 0 || act < 0 || act > 1) return GEMM_ERR_SHAPE;
  const long long n = rows * inner, blocks = (n + 511) / 512;
  gated_act_kernel<<<(unsigned)(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      vg, dh, (elem_t*)out, n, inner, act);
  return cudaGetLastError() == cudaSuccess ? 0 : GEMM_ERR_LAUNCH;
}
