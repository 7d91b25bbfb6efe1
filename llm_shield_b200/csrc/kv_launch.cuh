// How the paged-cache kernels are launched.
#pragma once

#include <cuda_runtime.h>

#include <type_traits>

namespace shield {
namespace kv {

// A launch whose status is its own: cudaGetLastError() would also give an error
// that an earlier call, here or in the caller's code, has left behind.
// early: it may start while the kernel before it in the stream still runs; the
// kernel itself waits (griddepcontrol.wait) where it needs what that one wrote,
// and never ends before it.
template <class... Params>
inline cudaError_t launch(void (*kernel)(Params...), dim3 grid, unsigned threads, int smem, bool early, cudaStream_t s,
                          const std::common_type_t<Params> &...args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = grid;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = (size_t)smem;
    c.stream = s;
    cudaLaunchAttribute a;
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &a;
    c.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&c, kernel, args...);
}

}  // namespace kv
}  // namespace shield
