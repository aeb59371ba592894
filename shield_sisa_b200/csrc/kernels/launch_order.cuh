// Kernels that start while the one before them drains.
#pragma once
#include <cuda_runtime.h>

namespace sb {

// A kernel that is launched behind another with programmatic ordering may start when every CTA of that one has said so or left, and
// waits for its end, with its memory, before it reads or writes what an earlier kernel may have to do with.  Every thread waits before it
// returns, so that the end of a kernel is the end of all before it.  A kernel that reads something in front of its wait (where sequences
// lie, slots, the first states) has a kernel of the same call before it that says next_may_start behind its own wait, which holds back
// all that come after it until the call's inputs are there, and no kernel between the two writes what is read early.  (Calls in a graph, one after the other or so: residual and norm of 20,544 x 384 18.2 or
// 17.5 us; a token of one sequence 2.5 or 2.2; a prefill of 321 tokens 34.5 or 32.4, of 37 sequences of up to 1,021 136.2 or 133.8.  Called
// from a host that is slower than the kernels, 20.9 or 18.4 us for the first.)
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void last_is_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... P, typename... A>
inline cudaError_t launch_behind(void (*kernel)(P...), long long ctas, int threads, int smem, cudaStream_t s, A... args) {
    cudaLaunchAttribute order{};
    order.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    order.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(unsigned(ctas));
    c.blockDim = dim3(unsigned(threads));
    c.dynamicSmemBytes = size_t(smem);
    c.stream = s;
    c.attrs = &order;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

}  // namespace sb
