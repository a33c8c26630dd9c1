// Host side of tensor maps, for every kernel that copies with them.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <dlfcn.h>

namespace i4mm {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's tensor-map encoder, found at run time so that the library does not link against libcuda.
inline EncodeTiledFn encode_tiled_fn() {
    static const EncodeTiledFn found = [] {
        EncodeTiledFn fn = nullptr;
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess && ptr)
            fn = (EncodeTiledFn)ptr;
        if (!fn) {
            (void)cudaGetLastError();
            void* h = dlopen("libcuda.so.1", RTLD_NOW | RTLD_GLOBAL);
            if (h) fn = (EncodeTiledFn)dlsym(h, "cuTensorMapEncodeTiled");
        }
        return fn;
    }();
    return found;
}

// The encoder needs a context that is current in the calling thread, which the first CUDA call of a new thread may find missing.
template <class Encode>
bool encode_with_context(Encode encode) {
    if (encode() == CUDA_SUCCESS) return true;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) {
        (void)cudaGetLastError();
        return false;
    }
    return encode() == CUDA_SUCCESS;
}

}  // namespace i4mm
