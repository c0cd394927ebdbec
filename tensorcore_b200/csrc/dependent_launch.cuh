// Launches that may begin while the stream's kernel before them ends.
//
// A kernel launched so begins once every block of the one before has let it (or has returned); it reads and writes nothing until
// wait_for_earlier() returns: the kernel before, and with it all that it waited for, is complete then and its writes are visible.
// Only behind that does it let the next one begin (let_next_begin), so a next kernel that reads something before its own wait
// reads what two kernels back have written.  Without the attribute both are nothing.
//
// Two kernels of attention over pages are not so: the merge of a prompt's chunks lets the next one begin before its wait, and the kernel of
// few rows beside prompts waits at its end.  Each begins when all of the prompts' CTAs have waited, so behind them what was written
// before the prompts' kernel is complete; what the prompts or the merge write is complete behind the next kernel's own wait, as ever.
#pragma once
#include <cuda_runtime.h>

#include <type_traits>

namespace tcb {
namespace dependent {

__device__ __forceinline__ void wait_for_earlier() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, bool early, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<std::decay_t<P>>(args)...);
}

}  // namespace dependent
}  // namespace tcb
