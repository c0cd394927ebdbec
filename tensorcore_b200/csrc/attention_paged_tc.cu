// Prompts over the paged 4-bit cache: the launches of attention_paged_prompt.cuh, and their sizes.
#include "attention_paged_prompt.cuh"

namespace tcb {

cudaError_t init_attention_paged_prompt_kernels() { return init_all<false>(); }

// Rows of a tile, tiles that the sequences can have together, and chunks that a tile's keys are cut into.
void plan_attention_paged_prompts(int tokens, int n_seqs, int max_q, int per_kv, int kv_heads, long long most_keys, int sm_count, AttnPagedPlan* plan) {
    const long long rows = static_cast<long long>(tokens) * per_kv, most = static_cast<long long>(max_q) * per_kv;
    auto tiles_of = [&](int height, int over) {
        const long long one = (most + height - 1) / height, n = rows / height + over;
        return n > one * n_seqs ? one * n_seqs : n;
    };
    // A tile of 256 rows takes 1.6 times as long as one of 128; fewer tiles than SMs take as long as if they were as many.  (Sixteen
    // sequences of 64 tokens, 32 heads on 8: 44.2 us against 50.8; two of them: 52.0 against 35.7, with chunks in both.)
    auto time_of = [&](int height) {
        const long long ctas = tiles_of(height, (n_seqs + 1) / 2) * kv_heads;
        return ctas > sm_count ? ctas : sm_count;
    };
    const bool tall = 8 * time_of(2 * kRows) <= 5 * time_of(kRows);
    plan->tile_rows = tall ? 2 * kRows : kRows;
    const long long n = tiles_of(plan->tile_rows, n_seqs);
    plan->tiles = static_cast<int>(n);
    // Fewer CTAs than SMs: as many chunks as fill the SMs once, of four steps at least (if the sequences fill their pages).
    long long c = sm_count / (n * kv_heads);
    if (c > most_keys / (4 * kKeys)) c = most_keys / (4 * kKeys);
    plan->chunks = static_cast<int>(c < 1 ? 1 : c > 32 ? 32 : c);
}

cudaError_t launch_attention_paged_prompts(const AttnPagedArgs& p, int tiles, int chunks, const LaunchEnv& env, cudaStream_t stream) {
    return p.dtype == IO_BF16 ? launch_type<__nv_bfloat16, false>(p, tiles, chunks, env, stream) : launch_type<__half, false>(p, tiles, chunks, env, stream);
}

}  // namespace tcb
