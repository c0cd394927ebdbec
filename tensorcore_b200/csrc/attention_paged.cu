// Attention over the paged 4-bit cache: which kernel takes which sequences.  Single tokens and few: attention_paged_rows.cuh; prompts: attention_paged_prompt.cuh.
#include "attention_paged_rows.cuh"

namespace tcb {

cudaError_t init_attention_paged_kernels() {
    for (cudaError_t e : {init_type<__half, false>(), init_type<__nv_bfloat16, false>(), init_attention_paged_prompt_kernels(), init_attention_split_kernels(),
                          init_attention_split_prompt_kernels()})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}

// Up to how many (query, head) rows on a K/V head a sequence is taken here, 16 at a time, each reading the keys again.  Eight sequences
// of 3000 keys, 32 heads on 8, fp16: 24 and 32 rows 38.2 and 38.4 us, as prompts 42.7 and 43.2; 40 rows 49.3, as a prompt 43.7.  (Two
// sequences of 48 rows would be faster here, 21.3 against 28.0.)
constexpr int kTokenRows = 32;

int attention_paged_token_rows() { return kTokenRows; }

AttnPagedPlan plan_attention_paged(const AttnPagedArgs& p, int sm_count) {
    AttnPagedPlan plan;
    const int per_kv = p.q_heads / p.kv_heads;
    const bool same = !p.q_start || p.n_seqs == 1;                    // no sequence of few queries beside a prompt
    plan.prompts = static_cast<long long>(p.max_q) * per_kv > kTokenRows;
    plan.tokens = !plan.prompts || !same;
    if (plan.prompts) {
        plan_attention_paged_prompts(p.tokens, p.n_seqs, p.max_q, per_kv, p.kv_heads, static_cast<long long>(p.max_pages) << p.page_shift, sm_count, &plan);
        if (plan.chunks > 1) plan.part_bytes = static_cast<size_t>(p.tokens) * p.q_heads * plan.chunks * (p.head_dim + 2) * sizeof(float);
    }
    if (plan.tokens) {
        const bool one = static_cast<long long>(p.max_q) * per_kv <= 8;
        auto rooms = [&](auto small, auto large) {
            plan.state_bytes = sm_count * (one ? decltype(small)::kStateBytes : decltype(large)::kStateBytes);
            plan.piece_bytes = sm_count * (one ? decltype(small)::kPieceBytes : decltype(large)::kPieceBytes);
        };
        switch (p.head_dim) {
            case 32: rooms(Shape<1, 1, false>(), Shape<1, 2, false>()); break;
            case 64: rooms(Shape<2, 1, false>(), Shape<2, 2, false>()); break;
            case 96: rooms(Shape<3, 1, false>(), Shape<3, 2, false>()); break;
            default: rooms(Shape<4, 1, false>(), Shape<4, 2, false>()); break;
        }
    }
    return plan;
}

void finish_attention_paged_args(AttnPagedArgs* args) {
    AttnPagedArgs& p = *args;
    const uintptr_t q = reinterpret_cast<uintptr_t>(p.Q) | static_cast<uintptr_t>((p.q_token | p.q_head) * 2);
    const uintptr_t o = reinterpret_cast<uintptr_t>(p.O) | static_cast<uintptr_t>((p.o_token | p.o_head) * 2);
    p.q_vec = (q & 15u) == 0;
    p.o_vec = (o & 7u) == 0;
    p.o_vec16 = (o & 15u) == 0;
    p.per_kv = p.q_heads / p.kv_heads;
    p.by_per_kv.set(p.per_kv);
    p.by_kv_heads.set(p.kv_heads);
}

cudaError_t launch_attention_paged(const AttnPagedArgs& args, const AttnPagedPlan& plan, const LaunchEnv& env, cudaStream_t stream, int* launches, const char** name) {
    AttnPagedArgs p = args;
    finish_attention_paged_args(&p);
    if (plan.prompts) p.most_rows = plan.tokens ? kTokenRows : 0;      // (a single sequence is one there whatever its queries: a step may be padded)
    p.tile_rows = plan.tile_rows;
    *launches = 0;
    cudaError_t e = cudaSuccess;
    if (plan.prompts) {
        const int chunks = p.parts ? plan.chunks : 1;                 // nowhere to leave chunks' results: keys in one piece
        e = launch_attention_paged_prompts(p, plan.tiles, chunks, env, stream);
        *launches += chunks > 1 ? 2 : 1;
        *name = "attention_paged_q4_0_prompt_tcgen05_sm100";
    }
    if (!plan.tokens) return e;
    p.beside = plan.prompts;
    *name = p.max_q * p.per_kv <= 8 ? "attention_paged_q4_0_rows8_sm100" : "attention_paged_q4_0_rows16_sm100";
    return e != cudaSuccess ? e : launch_all<false>(p, env, stream, launches);
}

}  // namespace tcb
