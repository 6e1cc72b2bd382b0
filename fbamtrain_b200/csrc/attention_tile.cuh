// What the attention kernels share: exponentials, the swizzled operand layout, arrivals of whole warps, a current context for the
// tensor-map encoder.
#pragma once
#include "tc05.cuh"
#include "tensor_map.h"

namespace attn {

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Arrival of a whole warp (one per warp: 32 arrivals on one barrier would be served one after the other): every lane
// has fenced its own accesses before.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) tc05::mbar_arrive(bar);
}

// Descriptors of a [128 x D] operand in 64-wide panels, whose rows are contiguous along K (K-major) or along M or N (MN-major), and the
// steps of 16 along K from their start.  A product is issued by one thread: with a descriptor formed for every instruction, eight
// instructions took that thread as long as the tensor core (520 cycles at 128 x 128 x 128).
__device__ __forceinline__ uint64_t k_major(uint32_t smem_addr) { return tc05::make_smem_desc_sw128(smem_addr, 16, 1024); }
__device__ __forceinline__ uint64_t mn_major(uint32_t smem_addr) { return tc05::make_smem_desc_sw128(smem_addr, 128 * 128, 1024); }
__device__ __forceinline__ constexpr uint64_t k_step(int k) { return uint64_t((k / 4) * 128 * 128 + (k % 4) * 32) >> 4; }
__device__ __forceinline__ constexpr uint64_t mn_step(int k) { return uint64_t(k * 16 * 128) >> 4; }

// Address of element (row, col8 = 8-element group index) in a [rows x 64]-bf16 panel with 128-byte swizzle.
__device__ __forceinline__ uint32_t swz(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) << 4); }

// D[tmem] (+)= A[tmem] * B[smem desc]; single-thread issue.  A: 128 rows, 16-bit elements two to a column.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Thread i of the warp writes 16 consecutive 32-bit columns of row (lane_base + i).
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// The driver entry point needs a context current on this thread (see gemm_tcgen05.h).
inline void bind_context() {
  static thread_local int bound = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess && dev != bound) {
    cudaSetDevice(dev);
    bound = dev;
  }
}

// Map of an (outer, rows, heads, D) view with element strides and inner stride 1: boxes of 64 channels x `box_heads` x `box_rows`.
inline int encode_heads(CUtensorMap* map, const void* base, int D, int heads, int rows, int outer, long long sh, long long sr, long long so,
                        int box_heads, int box_rows) {
  FbamEncodeTiledFn enc = fbam_encode_tiled();
  if (!enc) return 4;
  bind_context();
  if ((reinterpret_cast<uintptr_t>(base) & 15) || sh % 8 || sr % 8 || so % 8) return 2;
  // a dimension of one entry is never stepped over, whatever stride the tensor names; the encoder wants some
  const cuuint64_t step = (cuuint64_t)D * 2;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows, (cuuint64_t)outer};
  cuuint64_t strides[3] = {heads > 1 ? (cuuint64_t)sh * 2 : step, rows > 1 ? (cuuint64_t)sr * 2 : step, outer > 1 ? (cuuint64_t)so * 2 : step};
  cuuint32_t box[4] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, ELEM_TMAP, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 3;
}

template <typename K>
int set_smem(K kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess ? 0 : 5;
}

// The same once for a device and thread, for calls of a few microseconds.
template <auto kernel>
int set_smem_once(int bytes) {
  static thread_local int done = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 5;
  if (dev == done) return 0;
  if (set_smem(kernel, bytes)) return 5;
  done = dev;
  return 0;
}

}  // namespace attn
