// The kernels of attention_paged_rows.cuh for keys that are split among launches and for lists of pages by K/V head (attention_shared.cu).
#include "attention_paged_rows.cuh"

namespace tcb {

cudaError_t init_attention_split_kernels() {
    const cudaError_t e = init_type<__half, true>();
    return e != cudaSuccess ? e : init_type<__nv_bfloat16, true>();
}
cudaError_t launch_attention_split(const AttnPagedArgs& p, const LaunchEnv& env, cudaStream_t stream, int* launches) { return launch_all<true>(p, env, stream, launches); }

}  // namespace tcb
