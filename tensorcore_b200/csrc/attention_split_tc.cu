// The kernels of attention_paged_prompt.cuh for keys that are split among launches and for lists of pages by K/V head (attention_shared.cu).
#include "attention_paged_prompt.cuh"

namespace tcb {

cudaError_t init_attention_split_prompt_kernels() { return init_all<true>(); }
cudaError_t launch_attention_split_prompts(const AttnPagedArgs& p, int tiles, int chunks, const LaunchEnv& env, cudaStream_t stream) {
    return p.dtype == IO_BF16 ? launch_type<__nv_bfloat16, true>(p, tiles, chunks, env, stream) : launch_type<__half, true>(p, tiles, chunks, env, stream);
}

}  // namespace tcb
