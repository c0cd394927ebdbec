// What sequences with the same first keys share, worked out by a block of any size: by every CTA of the kernels that need it, in shared memory, or
// by a kernel of its own where the sequences are too many for that.
#pragma once

#include "kernels.h"

namespace tcb {
namespace groups {

// Clocks of an SM: for 128 keys and a tile of 128 or 256 rows in the kernel of prompts, for 64 keys and an item of 8 or 16 rows in that of few rows (where
// items are short: 430 and 700 in long ones); what the second kernel's start and end take where it runs behind the first; and what two kernels and the
// joining of their results take longer than one.
constexpr int kTileStep = 4100, kTallStep = 6600, kItemUnit = 700, kTallUnit = 1100, kBehind = 14000, kFixed = 24000;

// Of the groups: tiles of rows and most steps of one, units of all sequences' own keys (of one K/V head); what comes of it: chunks that a tile's keys are cut
// into, CTAs of few rows.
struct Totals { int tiles, steps, units, chunks, ctas; };

// Whether `items` of few rows are better `tiles` of rows for that many keys.
__host__ __device__ inline bool worth(int items, int tiles, int keys, bool tall_items, bool tall_tiles, int kv_heads, int sm_count) {
    const long long alone = 2ll * items * (tall_items ? 700 : 430), together = static_cast<long long>(tiles) * (tall_tiles ? kTallStep : kTileStep);
    return (alone - together) * (keys >> 7 < 65536 ? keys >> 7 : 65536) * kv_heads > static_cast<long long>(kFixed) * sm_count;
}

// own [n_seqs] and groups [n_groups] are the block's to write (and so are totals); all threads come here.  Keys that a group shares end before the first query of
// any of its sequences; a group of one sequence with queries, with more queries than the call declares, or without enough to gain, shares none.
__device__ inline void plan(const SharedGroups& p, SplitSeq* own, SplitSeq* groups, Totals* totals, bool tell, uint32_t* err) {
    const int tid = threadIdx.x, lane = tid & 31, threads = blockDim.x;
    int g_first = 0, g_behind = 0, g_keys = 0;    // asked for with the sequences' words
    if (tid < p.n_groups) {
        g_first = p.group_start[tid];
        g_behind = p.group_start[tid + 1];
        g_keys = p.shared_lens[tid];
    }
    for (int s = tid; s < p.n_seqs; s += threads) {
        const int len = p.seq_lens[s], a = p.q_start ? p.q_start[s] : s * p.seq_q, b = p.q_start ? p.q_start[s + 1] : a + p.seq_q;
        const int q0 = min(max(a, 0), p.tokens);
        own[s] = {s, q0, max(0, min(b, p.tokens) - q0), min(max(len, 0), p.most_keys), 0};
        if (len > p.most_keys && tell && err) atomicOr(err, ERR_BAD_SHAPE);
    }
    if (tid < p.n_groups) groups[tid] = {g_first, g_behind, g_keys, 0, 0};
    for (int g = tid + threads; g < p.n_groups; g += threads) groups[g] = {p.group_start[g], p.group_start[g + 1], p.shared_lens[g], 0, 0};
    if (tid == 0) *totals = {0, 0, 0, 0, 0};
    __syncthreads();
    for (int g = tid >> 5; g < p.n_groups; g += threads >> 5) {
        const SplitSeq raw = groups[g];
        const int a = min(max(raw.row, 0), p.n_seqs), b = min(max(raw.q0, a), p.n_seqs);
        if (lane == 0 && tell && err && (a != raw.row || b != raw.q0)) atomicOr(err, ERR_BAD_SHAPE);
        int most = max(raw.nq, 0), row = p.n_seqs, q0 = p.tokens, end = 0, members = 0, items = 0;
        for (int s = a + lane; s < b; s += 32) {
            const SplitSeq v = own[s];
            if (v.nq == 0) continue;
            ++members;
            items += (v.nq * p.per_kv + (1 << p.item_shift) - 1) >> p.item_shift;
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
        items = __reduce_add_sync(0xffffffffu, items);
        const int tiles = ((end - q0) * p.per_kv + (1 << p.tile_shift) - 1) >> p.tile_shift;
        const bool shares = members > 1 && most > 0 && end - q0 <= p.max_group_q && (p.always || worth(items, tiles, most, p.item_shift > 3, p.tile_shift > 7, p.kv_heads, p.sm_count));
        __syncwarp();
        if (lane == 0) {
            groups[g] = {shares ? row : 0, shares ? q0 : 0, shares ? end - q0 : 0, shares ? most : 0, 0};
            if (shares) {
                atomicMax(&totals->steps, (most + 127) >> 7);
                atomicAdd(&totals->tiles, tiles);
            }
        }
        if (shares)
            for (int s = a + lane; s < b; s += 32) own[s].begin = most;
    }
    __syncthreads();
    int units = 0;
    for (int s = tid; s < p.n_seqs; s += threads) {
        const SplitSeq v = own[s];
        units += min((v.nq * p.per_kv + (1 << p.item_shift) - 1 >> p.item_shift) * (1 + (v.len - v.begin + 63 >> 6)), 1 << 20);
    }
    units = __reduce_add_sync(0xffffffffu, units);
    if (lane == 0 && units) atomicAdd(&totals->units, min(units, 1 << 22));
    __syncthreads();
    if (tid < 32) {                               // lane c: c + 1 chunks
        const Totals t = *totals;
        const float shared = static_cast<float>((t.steps + lane) / (lane + 1)) * (p.tile_shift > 7 ? kTallStep : kTileStep);
        const float own_work = static_cast<float>(t.units) * p.kv_heads * (p.item_shift > 3 ? kTallUnit : kItemUnit);
        const int left = p.sm_count - t.tiles * p.kv_heads * (lane + 1);
        const float behind = shared + __fdividef(own_work, p.sm_count) + kBehind, beside = left > 0 ? fmaxf(shared, __fdividef(own_work, left)) : behind;
        uint32_t best = lane < p.chunks ? __float_as_uint(fminf(behind, beside)) & ~31u | lane : 0xFFFFFFFFu;      // (positive: of the same order)
        best = __reduce_min_sync(0xffffffffu, best);
        const int c = best & 31u;
        const bool aside = __shfl_sync(0xffffffffu, left > 0 && beside < behind, c);
        if (lane == 0) {
            totals->chunks = c + 1;
            totals->ctas = t.tiles > 0 && aside ? p.sm_count - t.tiles * p.kv_heads * (c + 1) : p.sm_count;
        }
    }
    __syncthreads();
}

// What the kernels behind need of it.
__device__ inline void hand_over(const SharedGroups& p, const SplitSeq* own, const Totals& totals, uint2* begins, uint4* to, uint32_t mark) {
    if (threadIdx.x == 0) *to = make_uint4(totals.tiles, totals.chunks, mark, totals.ctas);
    __threadfence();
    __syncthreads();
    for (int s = threadIdx.x; s < p.n_seqs; s += blockDim.x) begins[s] = make_uint2(own[s].begin, mark);
    __threadfence();
}

}  // namespace groups
}  // namespace tcb
