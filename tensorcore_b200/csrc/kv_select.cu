// Blocks of the paged 4-bit cache that a token attends to: bounds of each block's keys, a score from them, and the choice.  A block is a page.
//
// Bounds, for a block and K/V head, of 8 bits outwards: with x_td the keys' elements, step = max |x| / 127, hi_d = ceil(max_t x_td / step),
// lo_d = floor(min_t x_td / step).  A block with a scale that is not finite has a NaN for its step and zeros for its codes.
//
// Score of a block for a token's queries q_h of a K/V head: sum over h and d of the larger of q hi and q lo, an upper bound of the sum of q_h . k over
// its keys.  The queries are rounded to 8 bits, one step for all of them (max |q| / 127), and since the larger one is q hi where q is not
// negative, the sum over the heads is taken first: P_d of the queries' codes that are not negative, N_d of the others, and then
//   I = sum_d P_d hi_d + N_d lo_d,   score = (float(I) step) queries' step:
// 2 D whole products a block however many heads, and no order of summation that could change a choice.  NaN is above every number.
#include "dependent_launch.cuh"
#include "io_types.cuh"
#include "kernels.h"
#include "kv_cache.cuh"

namespace tcb {
namespace {

template <int N> __device__ __forceinline__ void words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

constexpr int kBoundsWarps = 8;

// A warp has a block of a K/V head: four lanes a token's keys, eight tokens at a time.
template <int NB>
__global__ void __launch_bounds__(kBoundsWarps * 32) kv_bounds_kernel(const KvBoundsArgs p, int blocks_at_once) {
    constexpr int D = 32 * NB;
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int lane = threadIdx.x & 31, t = lane & 3, sub = lane >> 2, head = blockIdx.y * kBoundsWarps + (threadIdx.x >> 5);
    const int seq = blockIdx.x / blocks_at_once, which = blockIdx.x - seq * blocks_at_once;
    if (head >= p.kv_heads) return;
    const int len = p.seq_lens[seq], first = max(p.first[seq], 0);
    if (len <= first) return;
    const int P = 1 << p.page_shift, tiles = P >> 4;
    const long long most = static_cast<long long>(p.max_pages) << p.page_shift;
    if (len > most && p.err && lane == 0) atomicOr(p.err, ERR_BAD_SHAPE);
    const int end = len > most ? static_cast<int>(most) : len;
    for (int block = (first >> p.page_shift) + which; block < (end + P - 1) >> p.page_shift; block += blocks_at_once) {
        const int page = p.page_table[static_cast<size_t>(seq) * p.max_pages + block], n = min(P, end - (block << p.page_shift));
        if (page < 0 || page >= p.n_pages) {
            if (p.err && lane == 0) atomicOr(p.err, ERR_BAD_SHAPE);
            continue;
        }
        const uint8_t* const keys = p.pages + (static_cast<size_t>(page) * p.kv_heads + head) * tiles * kv::tile_bytes(NB);
        float hi[NB][8], lo[NB][8];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e) { hi[b][e] = -INFINITY; lo[b][e] = INFINITY; }
        bool bad = false;
        for (int base = 0; base < n; base += 8) {
            const int token = base + sub;
            if (token >= n) continue;
            const uint8_t* const tile = keys + (token >> 4) * kv::tile_bytes(NB);
            uint32_t w[NB];
            words<NB>(tile + kv::key_word(NB, token & 15, t, 0), w);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const __half scale = *reinterpret_cast<const __half*>(tile + kv::key_scale(NB, token & 15, b));
                bad = bad || (__half_as_ushort(scale) & 0x7C00u) == 0x7C00u;
                const float d = __half2float(scale);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = (__uint_as_float(0x4B000000u | ((w[b] >> (4 * e)) & 15u)) - 8388616.0f) * d;
                    hi[b][e] = fmaxf(hi[b][e], x);
                    lo[b][e] = fminf(lo[b][e], x);
                }
            }
        }
        float amax = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
#pragma unroll
                for (int x = 4; x < 32; x *= 2) {
                    hi[b][e] = fmaxf(hi[b][e], __shfl_xor_sync(0xffffffffu, hi[b][e], x));
                    lo[b][e] = fminf(lo[b][e], __shfl_xor_sync(0xffffffffu, lo[b][e], x));
                }
                amax = fmaxf(amax, fmaxf(fabsf(hi[b][e]), fabsf(lo[b][e])));
            }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        bad = __any_sync(0xffffffffu, bad);
        const float step = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(amax, 127.0f);
        const bool some = step > 0.f;
        uint8_t* const record = p.bounds + (static_cast<size_t>(page) * p.kv_heads + head) * bounds_bytes(D);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (sub != b) continue;
            uint32_t c[4] = {0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int up = some ? static_cast<int>(fminf(fmaxf(ceilf(__fdiv_rn(hi[b][e], step)), -127.f), 127.f)) : 0;
                const int down = some ? static_cast<int>(fminf(fmaxf(floorf(__fdiv_rn(lo[b][e], step)), -127.f), 127.f)) : 0;
                c[e >> 2] |= (static_cast<uint32_t>(up) & 255u) << (8 * (e & 3));
                c[2 + (e >> 2)] |= (static_cast<uint32_t>(down) & 255u) << (8 * (e & 3));
            }
            *reinterpret_cast<uint2*>(record + 32 * b + 8 * t) = make_uint2(c[0], c[1]);
            *reinterpret_cast<uint2*>(record + D + 32 * b + 8 * t) = make_uint2(c[2], c[3]);
        }
        if (sub == 7 && t == 0) *reinterpret_cast<uint4*>(record + 2 * D) = make_uint4(__float_as_uint(step), 0u, 0u, 0u);
    }
}

// What a token sees: its sequence's list of pages and how many blocks of it; blocks 0: none, the token is passed over.
struct Seen { const int* pages; int blocks, last; };
__device__ __forceinline__ Seen seen_by(const KvPlace& p, int token, bool tell) {
    Seen s = {nullptr, 0, 0};
    const int position = p.positions[token];
    if (position < 0) return s;
    const int seq = p.sequences ? p.sequences[token] : token, blocks = (position >> p.page_shift) + 1;
    if (seq < 0 || seq >= p.n_seqs || blocks > p.max_pages) {
        if (tell && p.err) atomicOr(p.err, ERR_BAD_SHAPE);
        return s;
    }
    s.pages = p.page_table + static_cast<size_t>(seq) * p.max_pages;
    s.blocks = blocks;
    s.last = position & ((1 << p.page_shift) - 1);
    return s;
}

constexpr int kScoreThreads = 128;

// A CTA has a token's K/V head and a part of its blocks; four lanes a block, eight blocks a warp at a time.
template <typename T, int NB>
__global__ void __launch_bounds__(kScoreThreads) kv_score_kernel(const KvSelectArgs p, FastDiv by_heads) {
    constexpr int D = 32 * NB, kWarps = kScoreThreads / 32;
    __shared__ float most_s[kWarps];
    __shared__ __align__(16) int16_t weights[2 * D];
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int token = by_heads(static_cast<int>(blockIdx.x)), head = static_cast<int>(blockIdx.x) - token * p.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Seen seen = seen_by(p.place, token, tid == 0 && head == 0 && blockIdx.y == 0);
    constexpr int kPart = 8 * kWarps;
    if (static_cast<int>(blockIdx.y) * kPart >= seen.blocks) return;

    // the queries' common step, and their codes' sums
    const int G = p.q_heads / p.kv_heads;
    const T* const q = static_cast<const T*>(p.Q) + token * p.q_token + static_cast<long long>(head) * G * p.q_head;
    float most = 0.f;
    bool bad = false;
    for (int u = tid; u < G * D; u += kScoreThreads) {
        const float x = fabsf(io::to_f<T>(q[u / D * p.q_head + u % D]));
        bad = bad || !(x < INFINITY);
        most = fmaxf(most, x);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
    if (lane == 0) most_s[warp] = most;
    bad = __syncthreads_or(bad);
    for (int w = 0; w < kWarps; ++w) most = fmaxf(most, most_s[w]);
    const float step = __fdiv_rn(most, 127.0f);
    const bool some = step > 0.f && !bad;
    for (int d = tid; d < D; d += kScoreThreads) {
        int up = 0, down = 0;
        for (int h = 0; h < G && some; ++h) {
            const int c = static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(io::to_f<T>(q[h * p.q_head + d]), step)), -127.f), 127.f));
            up += max(c, 0);
            down += min(c, 0);
        }
        weights[d] = static_cast<int16_t>(up);
        weights[D + d] = static_cast<int16_t>(down);
    }
    __syncthreads();

    // lane 4 s + part has the 16-byte pieces part, part + 4, .. of block s's codes
    const int part = lane & 3, sub = lane >> 2;
    constexpr int kPieces = 2 * D / 16, kMine = (kPieces + 3) / 4;
    uint32_t w[kMine][8];                         // pairs of weights
#pragma unroll
    for (int i = 0; i < kMine; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int piece = part + 4 * i;
            w[i][k] = piece < kPieces ? reinterpret_cast<const uint32_t*>(weights)[piece * 8 + k] : 0u;
        }
    float* const scores = p.scores + (static_cast<size_t>(token) * p.kv_heads + head) * p.place.max_pages;
    for (int base = blockIdx.y * kPart; base < seen.blocks; base += gridDim.y * kPart) {
        const int block = base + warp * 8 + sub;
        const int page = block < seen.blocks ? seen.pages[block] : -1;
        const bool there = page >= 0 && page < p.place.n_pages;
        const uint8_t* const record = p.bounds + (static_cast<size_t>(there ? page : 0) * p.kv_heads + head) * bounds_bytes(D);
        uint4 x[kMine];
        float s = 0.f;
        if (there) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) x[i] = part + 4 * i < kPieces ? *reinterpret_cast<const uint4*>(record + 16 * (part + 4 * i)) : make_uint4(0, 0, 0, 0);
            s = *reinterpret_cast<const float*>(record + 2 * D);
        }
        int sum = 0;
        if (there) {
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const uint32_t c[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    sum = __dp2a_lo(static_cast<int>(w[i][2 * k]), static_cast<int>(c[k]), sum);
                    sum = __dp2a_hi(static_cast<int>(w[i][2 * k + 1]), static_cast<int>(c[k]), sum);
                }
            }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (part == 0 && block < seen.blocks) {
            scores[block] = there ? __fmul_rn(__fmul_rn(static_cast<float>(sum), s), some ? step : 0.f) : -INFINITY;
            if (!there && p.place.err) atomicOr(p.place.err, ERR_BAD_SHAPE);
        }
    }
}

// Scores as unsigned numbers of the same order; NaN above all.
__device__ __forceinline__ uint32_t order_of(float s) {
    if (!(s == s)) return 0xFFFFFFFFu;
    if (s == 0.f) return 0x80000000u;             // of either sign
    const uint32_t b = __float_as_uint(s);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

constexpr int kPickThreads = 256, kPickKeys = 8192;      // scores that are kept in shared memory

// A CTA has a token's K/V head: the bits of the last score that is taken, eight at a time, then the blocks in their order.
__global__ void __launch_bounds__(kPickThreads) kv_pick_kernel(const KvSelectArgs p, FastDiv by_heads) {
    constexpr int kWarps = kPickThreads / 32;
    __shared__ uint32_t keys[kPickKeys];
    __shared__ int bins[256], warp_sum[2][kWarps], found[2];
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int token = by_heads(static_cast<int>(blockIdx.x)), head = static_cast<int>(blockIdx.x) - token * p.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Seen seen = seen_by(p.place, token, false);
    const int n = seen.blocks, K = p.max_blocks, taken = min(n, K);
    int* const out = p.block_pages + (static_cast<size_t>(token) * p.kv_heads + head) * K;
    if (head == 0 && tid == 0) p.block_lens[token] = n > 0 ? ((taken - 1) << p.place.page_shift) + seen.last + 1 : 0;
    for (int i = taken + tid; i < K; i += kPickThreads) out[i] = -1;
    if (n <= K) {
        for (int i = tid; i < n; i += kPickThreads) out[i] = seen.pages[i];
        return;
    }
    const int from = min(p.first_blocks, n), to = max(n - p.last_blocks, from), wanted = K - from - (n - to);      // of blocks from .. to - 1 (first and last ones are no more than K)
    const float* const scores = p.scores + (static_cast<size_t>(token) * p.kv_heads + head) * p.place.max_pages;
    auto key_at = [&](int i) { return i < kPickKeys ? keys[i] : order_of(scores[i]); };
    for (int i = tid; i < min(n, kPickKeys); i += kPickThreads) keys[i] = order_of(scores[i]);
    __syncthreads();

    uint32_t prefix = 0, mask = 0;                // of the last one taken
    int left = wanted;                            // and how many of those with its bits so far
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += kPickThreads) bins[i] = 0;
        __syncthreads();
        for (int i = from + tid; i < to; i += kPickThreads) {
            const uint32_t k = key_at(i);
            if ((k & mask) == prefix) atomicAdd(&bins[(k >> shift) & 255u], 1);
        }
        __syncthreads();
        if (warp == 0) {                          // from the highest bin down: lane l has bins 255 - 8 l - 7 .. 255 - 8 l
            int mine[8], sum = 0;
#pragma unroll
            for (int b = 0; b < 8; ++b) sum += mine[b] = bins[255 - 8 * lane - b];
            int above = sum;
#pragma unroll
            for (int x = 1; x < 32; x *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, above, x);
                if (lane >= x) above += v;
            }
            above -= sum;
            if (above < left && above + sum >= left) {
#pragma unroll
                for (int b = 0; b < 8; ++b) {
                    if (above < left && above + mine[b] >= left) { found[0] = 255 - 8 * lane - b; found[1] = left - above; }
                    above += mine[b];
                }
            }
        }
        __syncthreads();
        if (wanted > 0) {
            prefix |= static_cast<uint32_t>(found[0]) << shift;
            left = found[1];
        }
        mask |= 255u << shift;
        __syncthreads();
    }

    // In order: a block is taken if it is one of the first or last, above that score, or one of the first `left` with it.
    int at = 0, equal = 0;
    for (int base = 0; base < n; base += kPickThreads) {
        const int i = base + tid;
        const bool middle = i >= from && i < to, live = i < n;
        const uint32_t k = live && middle ? key_at(i) : 0u;
        const bool same = middle && wanted > 0 && k == prefix;
        const uint32_t sames = __ballot_sync(0xffffffffu, same);
        if (lane == 0) warp_sum[0][warp] = __popc(sames);
        __syncthreads();
        int before = equal, all = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += warp_sum[0][w];
            all += warp_sum[0][w];
        }
        equal += all;
        const bool take = live && (!middle || (wanted > 0 && (k > prefix || (same && before + __popc(sames & ((1u << lane) - 1u)) < left))));
        const uint32_t takes = __ballot_sync(0xffffffffu, take);
        if (lane == 0) warp_sum[1][warp] = __popc(takes);
        __syncthreads();
        int place = at;
        all = 0;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) place += warp_sum[1][w];
            all += warp_sum[1][w];
        }
        at += all;
        if (take) out[place + __popc(takes & ((1u << lane) - 1u))] = seen.pages[i];
    }
}

template <typename T>
cudaError_t launch_scores(const KvSelectArgs& p, dim3 grid, FastDiv by_heads, const LaunchEnv& env, cudaStream_t stream) {
    switch (p.head_dim) {
        case 32: return dependent::launch(kv_score_kernel<T, 1>, grid, kScoreThreads, 0, stream, env.pdl, p, by_heads);
        case 64: return dependent::launch(kv_score_kernel<T, 2>, grid, kScoreThreads, 0, stream, env.pdl, p, by_heads);
        case 96: return dependent::launch(kv_score_kernel<T, 3>, grid, kScoreThreads, 0, stream, env.pdl, p, by_heads);
        default: return dependent::launch(kv_score_kernel<T, 4>, grid, kScoreThreads, 0, stream, env.pdl, p, by_heads);
    }
}

}  // namespace

cudaError_t launch_kv_bounds(const KvBoundsArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const int P = 1 << p.page_shift;
    long long blocks = p.max_new > 0 ? (static_cast<long long>(p.max_new) + P - 2) / P + 1 : p.max_pages;      // that as many new tokens can lie in
    if (blocks > p.max_pages) blocks = p.max_pages;
    const long long most = 0x7fffffffLL / p.n_seqs;
    if (blocks > most) blocks = most;
    if (blocks > 4096) blocks = 4096;
    const int y = (p.kv_heads + kBoundsWarps - 1) / kBoundsWarps;
    if (y > 65535) return cudaErrorNotSupported;
    const dim3 grid(static_cast<unsigned>(p.n_seqs * blocks), static_cast<unsigned>(y));
    auto go = [&](auto kernel) { return dependent::launch(kernel, grid, kBoundsWarps * 32, 0, stream, env.pdl, p, static_cast<int>(blocks)); };
    switch (p.head_dim) {
        case 32: return go(kv_bounds_kernel<1>);
        case 64: return go(kv_bounds_kernel<2>);
        case 96: return go(kv_bounds_kernel<3>);
        default: return go(kv_bounds_kernel<4>);
    }
}

cudaError_t launch_kv_select(const KvSelectArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const long long rows = static_cast<long long>(p.tokens) * p.kv_heads;
    if (rows > 0x7fffffffLL) return cudaErrorNotSupported;
    FastDiv by_heads;
    by_heads.set(p.kv_heads);
    constexpr int kPart = kScoreThreads / 4;
    long long parts = (p.place.max_pages + kPart - 1) / kPart, full = (8ll * env.sm_count + rows - 1) / rows;
    if (parts > full) parts = full;
    const dim3 grid(static_cast<unsigned>(rows), static_cast<unsigned>(parts < 1 ? 1 : parts));
    cudaError_t e = p.dtype == IO_BF16 ? launch_scores<__nv_bfloat16>(p, grid, by_heads, env, stream) : launch_scores<__half>(p, grid, by_heads, env, stream);
    if (e != cudaSuccess) return e;
    return dependent::launch(kv_pick_kernel, dim3(static_cast<unsigned>(rows)), kPickThreads, 0, stream, true, p, by_heads);
}

}  // namespace tcb
