// The driver's tensor-map encoder, looked up at run time so that the library links against the runtime only.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

typedef CUresult (*FbamEncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                      const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                      CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Null where the driver has none.
static inline FbamEncodeTiledFn fbam_encode_tiled() {
  static FbamEncodeTiledFn fn = nullptr;
  if (fn == nullptr) {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    fn = reinterpret_cast<FbamEncodeTiledFn>(sym);
  }
  return fn;
}
