// Attention over the paged 4-bit cache for sequences with the same first keys, and for lists of pages by K/V head.
//
// Shared keys: with s_j the score of key j and m, l, o the maximum of a set of keys' scores, the sum of e^(s_j - m) and that of e^(s_j - m) V_j,
// the sets A and B together have m = max(m_A, m_B), l = e^(m_A - m) l_A + e^(m_B - m) l_B, and o likewise.  So a group's shared keys are gone
// through once, with the queries of all of its sequences as the rows of one, and leave a part (m, l, o) for each row and chunk of keys;
// each sequence's own keys follow, and their results are joined with those parts on the way out.  Both are the kernels of
// attention_paged_rows.cuh and attention_paged_prompt.cuh, by the number of rows: what is a sequence to them is worked out by a small kernel first.
#include "dependent_launch.cuh"
#include "kernels.h"

namespace tcb {
namespace {

struct GroupPlan {
    const int* q_start;
    const int* seq_lens;
    const int* group_start;
    const int* shared_lens;
    SplitSeq* groups;
    SplitSeq* own;
    int n_seqs, n_groups, tokens, max_group_q;
    int most_keys;
    uint32_t* err;
};

// The groups' shared keys and queries, and what is left of each sequence: a warp has a group.  Keys that a group shares end before the first
// query of any of its sequences; a group of one sequence with queries, or with more queries than the call declares, shares none.
__global__ void __launch_bounds__(1024) shared_plan_kernel(const GroupPlan p) {
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    auto queries = [&](int s, int* q0) {
        if (!p.q_start) {
            const int n = p.tokens / p.n_seqs;
            *q0 = s * n;
            return n;
        }
        const int a = min(max(p.q_start[s], 0), p.tokens);
        *q0 = a;
        return max(0, min(p.q_start[s + 1], p.tokens) - a);
    };
    for (int s = threadIdx.x; s < p.n_seqs; s += blockDim.x) {
        SplitSeq v;
        v.row = s;
        v.nq = queries(s, &v.q0);
        const int len = p.seq_lens[s];
        v.len = min(max(len, 0), p.most_keys);
        v.begin = 0;
        if (len > p.most_keys && p.err) atomicOr(p.err, ERR_BAD_SHAPE);
        p.own[s] = v;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < p.n_groups; g += blockDim.x >> 5) {
        const int first = p.group_start[g], behind = p.group_start[g + 1];
        if (lane == 0 && p.err && (first < 0 || behind < first || behind > p.n_seqs)) atomicOr(p.err, ERR_BAD_SHAPE);
        const int a = min(max(first, 0), p.n_seqs), b = min(max(behind, a), p.n_seqs);
        int most = max(p.shared_lens[g], 0), row = p.n_seqs, q0 = p.tokens, end = 0, members = 0;
        for (int s = a + lane; s < b; s += 32) {
            const SplitSeq v = p.own[s];
            if (v.nq == 0) continue;
            ++members;
            row = min(row, s);
            q0 = min(q0, v.q0);
            end = max(end, v.q0 + v.nq);
            most = min(most, v.len - v.nq);
        }
        most = __reduce_min_sync(0xffffffffu, most);
        row = __reduce_min_sync(0xffffffffu, row);
        q0 = __reduce_min_sync(0xffffffffu, q0);
        end = __reduce_max_sync(0xffffffffu, end);
        members = __reduce_add_sync(0xffffffffu, members);
        const bool shares = members > 1 && most > 0 && end - q0 <= p.max_group_q;
        if (lane == 0) p.groups[g] = {shares ? row : 0, shares ? q0 : 0, shares ? end - q0 : 0, shares ? most : 0, 0};
        if (shares)
            for (int s = a + lane; s < b; s += 32) p.own[s].begin = most;
    }
}

}  // namespace

AttnSharedPlan plan_attention_shared(const AttnSharedArgs& p, int sm_count) {
    AttnSharedPlan plan;
    plan.own = plan_attention_paged(p.a, sm_count);
    AttnPagedArgs g = p.a;
    g.n_seqs = p.n_groups;
    g.max_q = p.max_group_q;
    static const int some = 0;
    g.q_start = &some;                                                 // groups differ in size
    plan.groups = plan_attention_paged(g, sm_count);
    plan.shares = p.a.n_seqs > 1;
    auto rounded = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t slot = static_cast<size_t>(p.a.tokens) * p.a.q_heads * (p.a.head_dim + 2) * sizeof(float);
    plan.prior_slots = plan.groups.prompts ? plan.groups.chunks : 1;
    plan.prior_at = rounded(sizeof(SplitSeq) * (static_cast<size_t>(p.n_groups) + p.a.n_seqs));
    plan.parts_at = plan.prior_at + rounded(slot * plan.prior_slots);
    plan.bytes = plan.parts_at + (plan.own.prompts ? slot * plan.own.chunks : 0);
    plan.state_bytes = plan.own.state_bytes + plan.groups.state_bytes;
    plan.piece_bytes = plan.own.piece_bytes + plan.groups.piece_bytes;
    return plan;
}

cudaError_t launch_attention_shared(const AttnSharedArgs& args, const AttnSharedPlan& plan, const LaunchEnv& first, cudaStream_t stream, int* launches, const char** name) {
    AttnPagedArgs own = args.a;
    finish_attention_paged_args(&own);
    uint8_t* const room = static_cast<uint8_t*>(args.room);
    SplitSeq* const seqs = reinterpret_cast<SplitSeq*>(room);
    float* const prior = reinterpret_cast<float*>(room + plan.prior_at);
    own.row_pages = own.max_pages;
    *launches = 0;
    *name = "attention_shared_q4_0_sm100";

    const GroupPlan p = {own.q_start, own.seq_lens, args.group_start, args.shared_lens, seqs, seqs + args.n_groups, own.n_seqs, args.n_groups, own.tokens, args.max_group_q,
                         static_cast<int>(static_cast<long long>(own.max_pages) << own.page_shift), own.err};
    const int most = own.n_seqs > 32 * args.n_groups ? own.n_seqs : 32 * args.n_groups;
    cudaError_t e = dependent::launch(shared_plan_kernel, dim3(1), most >= 1024 ? 1024 : (most + 31) / 32 * 32, 0, stream, first.pdl, p);
    ++*launches;
    if (e != cudaSuccess) return e;
    LaunchEnv env = first;
    env.pdl = true;

    AttnPagedArgs g = own;
    g.split = seqs;
    g.n_seqs = args.n_groups;
    g.max_q = args.max_group_q;
    g.causal = 0;
    g.left = g.parts = prior;
    g.left_slots = plan.prior_slots;
    if (plan.groups.prompts) {
        g.most_rows = plan.groups.tokens ? attention_paged_token_rows() : 0;
        g.tile_rows = plan.groups.tile_rows;
        e = launch_attention_split_prompts(g, plan.groups.tiles, plan.groups.chunks, false, env, stream);
        ++*launches;
        g.beside = 1;
    }
    if (plan.groups.tokens && e == cudaSuccess) e = launch_attention_split(g, env, stream, launches);

    own.split = seqs + args.n_groups;
    own.prior = prior;
    own.prior_slots = plan.prior_slots;
    if (own.states) own.states += plan.groups.state_bytes / sizeof(uint32_t);
    if (own.pieces) own.pieces += plan.groups.piece_bytes / sizeof(float);
    own.beside = 1;
    if (plan.own.prompts && e == cudaSuccess) {
        own.most_rows = plan.own.tokens ? attention_paged_token_rows() : 0;
        own.tile_rows = plan.own.tile_rows;
        own.parts = reinterpret_cast<float*>(room + plan.parts_at);
        e = launch_attention_split_prompts(own, plan.own.tiles, plan.own.chunks, true, env, stream);
        *launches += 2;
        own.beside = 0;
    }
    if (plan.own.tokens && e == cudaSuccess) e = launch_attention_split(own, env, stream, launches);
    return e;
}

AttnPagedPlan plan_attention_blocks(const AttnPagedArgs& p, int sm_count) {
    AttnPagedArgs a = p;
    const int per_kv = p.q_heads / p.kv_heads;
    // (planned as few rows whatever their number: a token is never a prompt)
    if (per_kv > 16) { a.q_heads = 16 * p.kv_heads; }
    return plan_attention_paged(a, sm_count);
}

cudaError_t launch_attention_blocks(const AttnPagedArgs& args, const LaunchEnv& env, cudaStream_t stream, int* launches, const char** name) {
    AttnPagedArgs p = args;
    finish_attention_paged_args(&p);
    *launches = 0;
    *name = p.per_kv <= 8 ? "attention_blocks_q4_0_rows8_sm100" : "attention_blocks_q4_0_rows16_sm100";
    return launch_attention_split(p, env, stream, launches);
}

}  // namespace tcb
