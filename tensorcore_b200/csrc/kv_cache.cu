// The paged 4-bit key/value cache (layout: kv_cache.cuh): rows appended with the rotation of their positions on the way, and
// rows read back.
//
// A row of head_dim elements is quantised in blocks of 32 with the arithmetic of quantize.cu (Q4_0: d = max|x| / 8 stored as
// fp16, code = round-half-away(x * (8 / max|x|)) + 8 in 0 .. 15, the _rn intrinsics).  A block with a NaN among its
// elements gets a NaN for its scale, so that it shows in what is computed from it (the codes could not say it); an infinity gives an infinite scale.
#include "dependent_launch.cuh"
#include "io_types.cuh"
#include "kernels.h"
#include "kv_cache.cuh"

namespace tcb {
namespace {

using namespace io;

// Where a token's row of the cache is: the tile, and which of its tokens.  False: a token without a position (below zero), or,
// with the error word set, one that the sequence's pages do not hold.
__device__ __forceinline__ bool find_row(const KvPlace& p, int position, int sequence, int kv_heads, int nb, int head, size_t* tile, int* r) {
    if (position < 0) return false;
    const int slot = position >> p.page_shift;
    int page = -1;
    if (sequence >= 0 && sequence < p.n_seqs && slot < p.max_pages) page = p.page_table[static_cast<size_t>(sequence) * p.max_pages + slot];
    if (page < 0 || page >= p.n_pages) {
        if (p.err) atomicOr(p.err, ERR_BAD_SHAPE);
        return false;
    }
    const int in_page = position & ((1 << p.page_shift) - 1);
    *tile = ((static_cast<size_t>(page) * kv_heads + head) << (p.page_shift - 4)) + (in_page >> 4);
    *tile *= kv::tile_bytes(nb);
    *r = in_page & 15;
    return true;
}

// LANES lanes (of eight elements) to a row: queries' rows are turned, keys' turned and written to their page, values'
// written to their page.  WHOLE: rows in 16-byte pieces, and pairs in whole pieces.
template <typename T, int LANES, bool WHOLE>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendArgs p) {
    constexpr int kRows = 32 / LANES;                                    // of a warp
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int lane = threadIdx.x & 31, piece = lane % LANES;
    const int heads = p.q_heads + 2 * p.kv_heads;
    const long long row = (static_cast<long long>(blockIdx.x) * (256 / 32) + (threadIdx.x >> 5)) * kRows + lane / LANES;
    const int D = p.head_dim, nb = D / 32, d0 = piece * 8;
    const bool there = row < static_cast<long long>(p.tokens) * heads && d0 < D;
    const int token = there ? static_cast<int>(row / heads) : 0, slot = there ? static_cast<int>(row - static_cast<long long>(token) * heads) : 0;
    const int kind = slot < p.q_heads ? 0 : slot < p.q_heads + p.kv_heads ? 1 : 2, head = kind == 0 ? slot : kind == 1 ? slot - p.q_heads : slot - p.q_heads - p.kv_heads;
    const T* x = kind == 0 ? static_cast<const T*>(p.Q) + token * p.q_token + head * p.q_head
               : kind == 1 ? static_cast<const T*>(p.K) + token * p.k_token + head * p.k_head
                           : static_cast<const T*>(p.V) + token * p.v_token + head * p.v_head;
    const int position = there ? p.place.positions[token] : -1;
    bool live = there && position >= 0;
    const bool turns = kind < 2 && p.cos_t;
    if (live && p.cos_t && position >= p.table_rows) {                  // values neither: a token is appended whole or not at all
        if (p.place.err) atomicOr(p.place.err, ERR_BAD_SHAPE);
        live = false;
    }
    size_t tile = 0;
    int r = 0;
    // Queries of a token that has no place in the cache are not turned either: what is given back for it is not to be used.
    if (live) live = find_row(p.place, position, p.place.sequences ? p.place.sequences[token] : token, p.kv_heads, nb, kind == 0 ? 0 : head, &tile, &r);

    float a[8];
    Pack8<T> raw = {};
    if (WHOLE) {
        if (live) raw = load8(x + d0);
        unpack8(raw, a);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = live ? to_f<T>(x[d0 + e]) : 0.f;
    }
    if (p.cos_t) {                                                       // all lanes: partners are other lanes' elements
        const int half = p.rot_dim / 2;
        const size_t angles = static_cast<size_t>(live && turns ? position : 0) * half;
        if (WHOLE && p.layout == 0) {
            const int step = half / 8;
            const bool first = piece < step, in = d0 < p.rot_dim;
            const int from = (lane - piece) + (in ? first ? piece + step : piece - step : piece);
            Pack8<T> other;
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
                other.w[i].x = __shfl_sync(0xffffffffu, raw.w[i].x, from);
                other.w[i].y = __shfl_sync(0xffffffffu, raw.w[i].y, from);
                other.w[i].z = __shfl_sync(0xffffffffu, raw.w[i].z, from);
                other.w[i].w = __shfl_sync(0xffffffffu, raw.w[i].w, from);
            }
            if (live && turns && in) {
                float b[8];
                unpack8(other, b);
                const int k = first ? d0 : d0 - half;
#pragma unroll
                for (int e = 0; e < 8; e += 4) {
                    const float4 c = *reinterpret_cast<const float4*>(p.cos_t + angles + k + e), s = *reinterpret_cast<const float4*>(p.sin_t + angles + k + e);
                    const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float own = __fmul_rn(a[e + i], cv[i]), partner = __fmul_rn(b[e + i], sv[i]);
                        a[e + i] = first ? __fsub_rn(own, partner) : __fadd_rn(partner, own);
                    }
                }
            }
        } else if (WHOLE) {
            if (live && turns && d0 < p.rot_dim) {
                const float4 c = *reinterpret_cast<const float4*>(p.cos_t + angles + d0 / 2), s = *reinterpret_cast<const float4*>(p.sin_t + angles + d0 / 2);
                const float cv[4] = {c.x, c.y, c.z, c.w}, sv[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x0 = a[2 * i], x1 = a[2 * i + 1];
                    a[2 * i] = __fsub_rn(__fmul_rn(x0, cv[i]), __fmul_rn(x1, sv[i]));
                    a[2 * i + 1] = __fadd_rn(__fmul_rn(x0, sv[i]), __fmul_rn(x1, cv[i]));
                }
            }
        } else {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = d0 + e;
                y[e] = a[e];
                if (!live || !turns || d >= p.rot_dim) continue;
                const bool first = p.layout == 0 ? d < half : (d & 1) == 0;
                const int k = p.layout == 0 ? first ? d : d - half : d / 2, other = p.layout == 0 ? first ? d + half : d - half : d ^ 1;
                const float own = __fmul_rn(a[e], p.cos_t[angles + k]), partner = __fmul_rn(to_f<T>(x[other]), p.sin_t[angles + k]);
                y[e] = first ? __fsub_rn(own, partner) : __fadd_rn(partner, own);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) a[e] = y[e];
        }
    }
    __syncwarp();                                    // a row that is turned in place has been read by all of its lanes
    if (live && kind == 0) {
        T* y = static_cast<T*>(p.Q_out) + token * p.o_token + head * p.o_head;
        if (WHOLE) {
            store8(y + d0, pack8<T>(a));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[d0 + e] = from_f<T>(a[e]);
        }
    }

    // The block's largest magnitude, as the bits of a float: a NaN is above every number.
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(a[e]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (!live || kind == 0) return;
    const float most = __uint_as_float(top), scale = __fdiv_rn(most, 8.0f), inv = scale > 0.f ? __fdiv_rn(8.0f, most) : 0.f;
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int code = static_cast<int>(roundf(__fmul_rn(a[e], inv))) + 8;
        word |= static_cast<uint32_t>(max(0, min(15, code))) << (4 * e);
    }
    const int block = piece >> 2, t = piece & 3;
    uint8_t* to = p.pages + tile;
    if (kind == 1) {
        *reinterpret_cast<uint32_t*>(to + kv::key_word(nb, r, t, block)) = word;
        if (t == 0) *reinterpret_cast<__half*>(to + kv::key_scale(nb, r, block)) = __float2half_rn(scale);
    } else {
        *reinterpret_cast<uint16_t*>(to + kv::value_half(nb, r, 2 * t, block)) = static_cast<uint16_t>(word);
        *reinterpret_cast<uint16_t*>(to + kv::value_half(nb, r, 2 * t + 1, block)) = static_cast<uint16_t>(word >> 16);
        if (t == 0) *reinterpret_cast<__half*>(to + kv::value_scale(nb, r, block)) = __float2half_rn(scale);
    }
}

// Rows of the cache as numbers, (c - 8) d rounded once: a thread per eight elements of a key and of a value.
template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvReadArgs p) {
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int nb = p.head_dim / 32, pieces = p.head_dim / 8;
    const long long u = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, row = u / pieces;
    if (row >= static_cast<long long>(p.tokens) * p.kv_heads) return;
    const int piece = static_cast<int>(u - row * pieces), token = static_cast<int>(row / p.kv_heads), head = static_cast<int>(row - static_cast<long long>(token) * p.kv_heads);
    size_t tile;
    int r;
    if (!find_row(p.place, p.place.positions[token], p.place.sequences ? p.place.sequences[token] : token, p.kv_heads, nb, head, &tile, &r)) return;
    const uint8_t* from = p.pages + tile;
    const int block = piece >> 2, t = piece & 3;
    const size_t at = row * p.head_dim + piece * 8;
    auto write = [&](T* to, uint32_t word, float d) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (static_cast<float>((word >> (4 * e)) & 15u) - 8.0f) * d;
        if (p.whole) {
            store8(to + at, pack8<T>(f));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) to[at + e] = from_f<T>(f[e]);
        }
    };
    if (p.K) write(static_cast<T*>(p.K), *reinterpret_cast<const uint32_t*>(from + kv::key_word(nb, r, t, block)),
                   __half2float(*reinterpret_cast<const __half*>(from + kv::key_scale(nb, r, block))));
    if (p.V) {
        const uint32_t lo = *reinterpret_cast<const uint16_t*>(from + kv::value_half(nb, r, 2 * t, block));
        const uint32_t hi = *reinterpret_cast<const uint16_t*>(from + kv::value_half(nb, r, 2 * t + 1, block));
        write(static_cast<T*>(p.V), lo | hi << 16, __half2float(*reinterpret_cast<const __half*>(from + kv::value_scale(nb, r, block))));
    }
}

template <typename T>
cudaError_t launch_append_of(const KvAppendArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    auto aligned = [](const void* a, long long token, long long head) {
        return ((reinterpret_cast<uintptr_t>(a) | static_cast<uintptr_t>((token | head) * static_cast<long long>(sizeof(T)))) & 15u) == 0;
    };
    bool whole = aligned(p.K, p.k_token, p.k_head) && aligned(p.V, p.v_token, p.v_head);
    if (p.q_heads) whole = whole && aligned(p.Q, p.q_token, p.q_head) && aligned(p.Q_out, p.o_token, p.o_head);
    if (p.cos_t) whole = whole && p.rot_dim % (p.layout == 0 ? 16 : 8) == 0 && ((reinterpret_cast<uintptr_t>(p.cos_t) | reinterpret_cast<uintptr_t>(p.sin_t)) & 15u) == 0;
    const int lanes = p.head_dim == 32 ? 4 : p.head_dim == 64 ? 8 : 16;
    const long long rows = static_cast<long long>(p.tokens) * (p.q_heads + 2 * p.kv_heads), per_block = 256 / lanes, blocks = (rows + per_block - 1) / per_block;
    if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
    const unsigned grid = static_cast<unsigned>(blocks);
    auto go = [&](auto kernel) { return dependent::launch(kernel, grid, 256, 0, stream, env.pdl, p); };
    if (lanes == 4) return go(whole ? kv_append_kernel<T, 4, true> : kv_append_kernel<T, 4, false>);
    if (lanes == 8) return go(whole ? kv_append_kernel<T, 8, true> : kv_append_kernel<T, 8, false>);
    return go(whole ? kv_append_kernel<T, 16, true> : kv_append_kernel<T, 16, false>);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    switch (p.dtype) {
        case IO_F16: return launch_append_of<__half>(p, env, stream);
        case IO_BF16: return launch_append_of<__nv_bfloat16>(p, env, stream);
        default: return launch_append_of<float>(p, env, stream);
    }
}

cudaError_t launch_kv_read(const KvReadArgs& args, const LaunchEnv& env, cudaStream_t stream) {
    KvReadArgs p = args;
    p.whole = ((reinterpret_cast<uintptr_t>(p.K) | reinterpret_cast<uintptr_t>(p.V)) & 15u) == 0;
    const long long blocks = (static_cast<long long>(p.tokens) * p.kv_heads * (p.head_dim / 8) + 255) / 256;
    if (blocks > 0x7fffffffLL) return cudaErrorNotSupported;
    const unsigned grid = static_cast<unsigned>(blocks);
    switch (p.dtype) {
        case IO_F16: return dependent::launch(kv_read_kernel<__half>, grid, 256, 0, stream, env.pdl, p);
        case IO_BF16: return dependent::launch(kv_read_kernel<__nv_bfloat16>, grid, 256, 0, stream, env.pdl, p);
        default: return dependent::launch(kv_read_kernel<float>, grid, 256, 0, stream, env.pdl, p);
    }
}

}  // namespace tcb
