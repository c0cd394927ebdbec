// Attention over the paged 4-bit cache (layout: kv_cache.cuh): for every query row
//
//   O = sum_j p_j V_j / sum_j p_j,   p_j = exp(scale Q . K_j),   LSE = log sum_j p_j
//
// over the keys j of the row's sequence that it sees, K and V being (code - 8) * scale.  The last of a sequence's queries is
// at its last key.  A row that sees no key gives zeros and a log-sum-exp of minus infinity.
//
// A CTA per query row and head, a thread per key for the scores, then per element for the output, fp32 throughout.
#include "io_types.cuh"
#include "kernels.h"
#include "kv_cache.cuh"

namespace tcb {
namespace {

using namespace io;

constexpr int kThreads = 128;

template <typename T>
__global__ void __launch_bounds__(kThreads) attention_paged_kernel(const AttnPagedArgs p) {
    __shared__ float q_s[128], p_s[kThreads], red[kThreads / 32];
    __shared__ const uint8_t* at_s[kThreads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, token = blockIdx.x, h = blockIdx.y;
    const int D = p.head_dim, nb = D / 32, hkv = h / (p.q_heads / p.kv_heads);
    int seq, first, n;
    if (p.q_start) {
        int lo = 0, hi = p.n_seqs;                 // the last sequence that starts at or before the token
        while (lo + 1 < hi) {
            const int mid = (lo + hi) / 2;
            (p.q_start[mid] <= token ? lo : hi) = mid;
        }
        seq = lo;
        first = p.q_start[seq];
        n = p.q_start[seq + 1] - first;
        if (token < first || token >= first + n) return;
    } else {
        n = p.tokens / p.n_seqs;
        seq = token / n;
        first = seq * n;
    }
    long long len = p.seq_lens[seq];
    const long long most = static_cast<long long>(p.max_pages) << p.page_shift;
    if (len > most) {
        len = most;
        if (tid == 0 && p.err) atomicOr(p.err, ERR_BAD_SHAPE);
    }
    if (len < 0) len = 0;
    const int pos = static_cast<int>(len) - n + token - first;
    const int k0 = p.window > 0 ? max(0, pos - p.window) : 0, k1 = p.causal ? min(static_cast<int>(len), pos + 1) : static_cast<int>(len);
    if (tid < D) q_s[tid] = to_f<T>(static_cast<const T*>(p.Q)[token * p.q_token + h * p.q_head + tid]);
    float m = -INFINITY, l = 0.f, o = 0.f;
    const int blk = tid >> 5;
    for (int j0 = k0; j0 < k1; j0 += kThreads) {
        __syncthreads();
        const int j = j0 + tid;
        float s = -INFINITY;
        const uint8_t* tile = nullptr;
        if (j < k1) {
            const int page = p.page_table[static_cast<size_t>(seq) * p.max_pages + (j >> p.page_shift)];
            if (page < 0 || page >= p.n_pages) {
                if (p.err) atomicOr(p.err, ERR_BAD_SHAPE);
            } else {
                const int in = j & ((1 << p.page_shift) - 1);
                tile = p.pages + (((static_cast<size_t>(page) * p.kv_heads + hkv) << (p.page_shift - 4)) + (in >> 4)) * kv::tile_bytes(nb);
                s = 0.f;
                for (int b = 0; b < nb; ++b) {
                    float dot = 0.f;
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + kv::key_word(nb, j & 15, t, b));
                        for (int e = 0; e < 8; ++e) dot = fmaf(q_s[32 * b + 8 * t + e], static_cast<float>((w >> (4 * e)) & 15u) - 8.f, dot);
                    }
                    s = fmaf(dot, __half2float(*reinterpret_cast<const __half*>(tile + kv::key_scale(nb, j & 15, b))), s);
                }
                s *= p.scale;                      // a NaN stays one and shows in the result
            }
        }
        at_s[tid] = tile;
        float mx = s;
        for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
        if (lane == 0) red[warp] = mx;
        __syncthreads();
        const float m_new = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float ref = m_new > -INFINITY ? m_new : 0.f, keep = expf(m - ref);
        m = m_new;
        p_s[tid] = expf(s - ref);
        __syncthreads();
        l *= keep;
        o *= keep;
        const int cnt = min(kThreads, k1 - j0);
        for (int u = 0; u < cnt; ++u) {
            l += p_s[u];
            if (tid < D && at_s[u]) {
                const int r = (j0 + u) & 15, g = (tid & 31) >> 2;
                const uint32_t w = *reinterpret_cast<const uint16_t*>(at_s[u] + kv::value_half(nb, r, g, blk));
                const float d = __half2float(*reinterpret_cast<const __half*>(at_s[u] + kv::value_scale(nb, r, blk)));
                o = fmaf(p_s[u], (static_cast<float>((w >> (4 * (tid & 3))) & 15u) - 8.f) * d, o);
            }
        }
    }
    if (tid < D) static_cast<T*>(p.O)[token * p.o_token + h * p.o_head + tid] = from_f<T>(l == 0.f ? 0.f : o / l);
    if (tid == 0 && p.LSE) p.LSE[static_cast<size_t>(token) * p.q_heads + h] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace

cudaError_t launch_attention_paged(const AttnPagedArgs& p, const LaunchEnv&, cudaStream_t stream, int* launches, const char** name) {
    const dim3 grid(static_cast<unsigned>(p.tokens), static_cast<unsigned>(p.q_heads));
    if (p.dtype == IO_BF16) attention_paged_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(p);
    else attention_paged_kernel<__half><<<grid, kThreads, 0, stream>>>(p);
    *launches = 1;
    *name = "attention_paged_q4_0_sm100";
    return cudaGetLastError();
}

}  // namespace tcb
