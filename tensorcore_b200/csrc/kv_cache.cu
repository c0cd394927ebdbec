// The paged 4-bit key/value cache (layout: kv_cache.cuh): rows appended with the rotation of their positions on the way, and
// rows read back.
//
// A row of head_dim elements is quantised in blocks of 32 with the arithmetic of quantize.cu (Q4_0: d = max|x| / 8 stored as
// fp16, code = round-half-away(x * (8 / max|x|)) + 8 in 0 .. 15, the _rn intrinsics).  A block with a NaN among its
// elements gets a NaN for its scale, so that it shows in what is computed from it (the codes could not say it); an infinity gives an infinite scale.
//
// Bound by instructions: 240 for a warp's two rows of 128 elements - turning, a maximum over four lanes, a division, eight codes, stores of
// two and four bytes - in 70% of issue slots, where the rows' bytes would allow 80.  9498 tokens of 8 K/V heads in bf16: append and reading
// back into fp16 35.4 us together; reading is bound by latency, a piece to a thread through position, page and codes.  64 tokens with 32 query heads: 2.4 us each, launch and three dependent loads (position, page, row).
#include <type_traits>

#include "dependent_launch.cuh"
#include "io_types.cuh"
#include "kernels.h"
#include "kv_cache.cuh"

namespace tcb {
namespace {

using namespace io;

// Where a token's rows of the cache are: head 0's tile, and which of its tokens.  False: a token without a position (below zero), or,
// with the error word set, one that the sequence's pages do not hold.
__device__ __forceinline__ bool find_rows(const KvPlace& p, int position, int sequence, int kv_heads, int nb, size_t* tile, int* r) {
    if (position < 0) return false;
    const int slot = position >> p.page_shift;
    int page = -1;
    if (sequence >= 0 && sequence < p.n_seqs && slot < p.max_pages) page = p.page_table[static_cast<size_t>(sequence) * p.max_pages + slot];
    if (page < 0 || page >= p.n_pages) {
        if (p.err) atomicOr(p.err, ERR_BAD_SHAPE);
        return false;
    }
    const int in_page = position & ((1 << p.page_shift) - 1);
    *tile = ((static_cast<size_t>(page) * kv_heads << (p.page_shift - 4)) + (in_page >> 4)) * kv::tile_bytes(nb);
    *r = in_page & 15;
    return true;
}

// The largest magnitude; a NaN is above every number.
__device__ __forceinline__ float most3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
    return d;
}
__device__ __forceinline__ float most2(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)));
    return d;
}

// The codes of eight elements, 32 bits: round-half-away(a inv) + 8 in 0 .. 15, 8 for NaN.  With u = 2 |a inv| cut to an integer, which
// an addition of 2^23 leaves in the lowest bits, that is (17 + u) / 2 or, below zero, (16 - u) / 2 = ((u ^ 31) - 15) / 2 cut to an
// integer: elements e and e + 4 at a time, in halves of a word that never borrow from one another.
__device__ __forceinline__ uint32_t codes_of(const float (&a)[8], float inv) {
    uint32_t word = 0;
    if (inv > 0.f && inv < INFINITY) {               // no product is infinite or NaN, or above 8 by more than a rounding
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = __fmaf_rz(__fmul_rn(fabsf(a[e]), inv), 2.0f, 8388608.0f), y = __fmaf_rz(__fmul_rn(fabsf(a[e + 4]), inv), 2.0f, 8388608.0f);
            const uint32_t u = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x5410);
            uint32_t below;                          // all bits of a half where its sign is set
            asm("prmt.b32 %0, %1, %2, 0xFFBB;" : "=r"(below) : "r"(__float_as_uint(a[e])), "r"(__float_as_uint(a[e + 4])));
            const uint32_t twice = (u ^ (below & 0x001F001Fu)) + 0x00110011u - (below & 0x00200020u);
            word |= ((__vminu2(twice, 0x001F001Fu) >> 1) & 0x000F000Fu) << (4 * e);
        }
    } else {                                         // zeros, a block with an infinity or a NaN, magnitudes below 2^-125
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = __fmul_rn(a[e], inv);
            word |= (x > 0.f ? 15u : x < 0.f ? 0u : 8u) << (4 * e);
        }
    }
    return word;
}

// LANES lanes (of eight elements) to a row, up to N rows - heads of a token's queries, keys or values - to a thread, all asked for before the
// first is used: queries' rows are turned, keys' turned and written to their page, values' written to their page.  WHOLE:
// rows in 16-byte pieces, and pairs in whole pieces.
template <typename T, int LANES, bool WHOLE, int N>
__global__ void __launch_bounds__(256) kv_append_kernel(const KvAppendArgs p, FastDiv by_token, int threads_per_token, int tokens_per_block) {
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int lane = threadIdx.x & 31, piece = lane % LANES, local = by_token(static_cast<int>(threadIdx.x));
    const int token = blockIdx.x * tokens_per_block + local, group = (blockIdx.y * blockDim.x + threadIdx.x - local * threads_per_token) / LANES;
    const int D = p.head_dim, nb = D / 32, d0 = piece * 8, q_groups = (p.q_heads + N - 1) / N, kv_groups = (p.kv_heads + N - 1) / N;
    const int kind = group < q_groups ? 0 : group < q_groups + kv_groups ? 1 : 2;
    const int head0 = (group - (kind == 0 ? 0 : kind == 1 ? q_groups : q_groups + kv_groups)) * N, rows = min(N, (kind == 0 ? p.q_heads : p.kv_heads) - head0);
    const bool there = local < tokens_per_block && token < p.tokens && rows > 0 && d0 < D;
    const int position = there ? p.place.positions[token] : -1;
    bool live = there && position >= 0;
    if (live && p.cos_t && position >= p.table_rows) {                  // values neither: a token is appended whole or not at all
        if (p.place.err) atomicOr(p.place.err, ERR_BAD_SHAPE);
        live = false;
    }
    size_t tile0 = 0;
    int r = 0;
    // Queries of a token that has no place in the cache are not turned either: what is given back for it is not to be used.
    if (live) live = find_rows(p.place, position, p.place.sequences ? p.place.sequences[token] : token, p.kv_heads, nb, &tile0, &r);

    const long long head_stride = kind == 0 ? p.q_head : kind == 1 ? p.k_head : p.v_head;
    const T* const x0 = static_cast<const T*>(kind == 0 ? p.Q : kind == 1 ? p.K : p.V) + token * (kind == 0 ? p.q_token : kind == 1 ? p.k_token : p.v_token) + head0 * head_stride;
    Pack8<T> raw[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        raw[n] = Pack8<T>{};
        if (!live || n >= rows) continue;
        const T* x = x0 + n * head_stride + d0;
        if (WHOLE) {
            raw[n] = load8(x);
        } else {
            T* e = reinterpret_cast<T*>(&raw[n]);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = x[i];
        }
    }

    // The eight elements' angles: pairs are elements of this lane (interleaved) or of a partner lane (half), whose elements the shuffles
    // below bring; where pairs are not whole pieces, the partner is read where it lies.
    const int half = p.rot_dim / 2, step = half / 8;
    const bool turns = p.cos_t && live && d0 < p.rot_dim && kind < 2, first = p.layout != 0 || piece < step;
    const size_t angles = static_cast<size_t>(turns ? position : 0) * half;
    float cv[8], sv[8];
    if (WHOLE && turns) {
        const size_t at = angles + (p.layout != 0 ? d0 / 2 : first ? d0 : d0 - half);
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            if (p.layout != 0 && e > 0) break;
            const float4 c = *reinterpret_cast<const float4*>(p.cos_t + at + e), s = *reinterpret_cast<const float4*>(p.sin_t + at + e);
            cv[e] = c.x; cv[e + 1] = c.y; cv[e + 2] = c.z; cv[e + 3] = c.w;
            sv[e] = s.x; sv[e + 1] = s.y; sv[e + 2] = s.z; sv[e + 3] = s.w;
        }
    }
    const int from = WHOLE && p.cos_t && p.layout == 0 && d0 < p.rot_dim ? first ? lane + step : lane - step : lane;
    const uint32_t row_mask = (LANES == 32 ? 0xffffffffu : (1u << LANES) - 1u) << (lane - piece);      // the lanes of this thread's rows

#pragma unroll
    for (int n = 0; n < N; ++n) {
        float a[8];
        unpack8(raw[n], a);
        if (WHOLE) {
            if (p.cos_t && p.layout == 0) {                              // all lanes: partners are other lanes' elements
                Pack8<T> other;
#pragma unroll
                for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
                    other.w[i].x = __shfl_sync(0xffffffffu, raw[n].w[i].x, from);
                    other.w[i].y = __shfl_sync(0xffffffffu, raw[n].w[i].y, from);
                    other.w[i].z = __shfl_sync(0xffffffffu, raw[n].w[i].z, from);
                    other.w[i].w = __shfl_sync(0xffffffffu, raw[n].w[i].w, from);
                }
                if (turns) {
                    float b[8];
                    unpack8(other, b);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float mine = __fmul_rn(a[e], cv[e]), partner = __fmul_rn(b[e], sv[e]);
                        a[e] = first ? __fsub_rn(mine, partner) : __fadd_rn(partner, mine);
                    }
                }
            } else if (turns) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float left = a[2 * i], right = a[2 * i + 1];
                    a[2 * i] = __fsub_rn(__fmul_rn(left, cv[i]), __fmul_rn(right, sv[i]));
                    a[2 * i + 1] = __fadd_rn(__fmul_rn(left, sv[i]), __fmul_rn(right, cv[i]));
                }
            }
        } else if (turns && n < rows) {
            const T* x = x0 + n * head_stride;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = d0 + e;
                if (d >= p.rot_dim) continue;
                const bool lower = p.layout == 0 ? d < half : (d & 1) == 0;
                const int k = p.layout == 0 ? lower ? d : d - half : d / 2, other = p.layout == 0 ? lower ? d + half : d - half : d ^ 1;
                const float mine = __fmul_rn(a[e], p.cos_t[angles + k]), partner = __fmul_rn(to_f<T>(x[other]), p.sin_t[angles + k]);
                a[e] = lower ? __fsub_rn(mine, partner) : __fadd_rn(partner, mine);
            }
        }
        __syncwarp();                                // a row that is turned in place has been read by all of its lanes
        if (kind == 0) {
            if (!live || n >= rows) continue;
            T* y = static_cast<T*>(p.Q_out) + token * p.o_token + (head0 + n) * p.o_head + d0;
            if (WHOLE) {
                store8(y, pack8<T>(a));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = from_f<T>(a[e]);
            }
            continue;
        }
        float most = most3(most3(most3(a[0], a[1], a[2]), a[3], a[4]), most3(a[5], a[6], a[7]), 0.f);
        most = most2(most, __shfl_xor_sync(row_mask, most, 1));
        most = most2(most, __shfl_xor_sync(row_mask, most, 2));
        if (!live || n >= rows) continue;
        const float scale = __fmul_rn(most, 0.125f), inv = scale > 0.f ? __fdiv_rn(8.0f, most) : 0.f;
        const uint32_t word = codes_of(a, inv);
        const int block = piece >> 2, t = piece & 3;
        uint8_t* to = p.pages + tile0 + (static_cast<size_t>(head0 + n) << (p.place.page_shift - 4)) * kv::tile_bytes(nb);
        if (kind == 1) {
            *reinterpret_cast<uint32_t*>(to + kv::key_word(nb, r, t, block)) = word;
            if (t == 0) *reinterpret_cast<__half*>(to + kv::key_scale(nb, r, block)) = __float2half_rn(scale);
        } else {
            *reinterpret_cast<uint16_t*>(to + kv::value_half(nb, r, 2 * t, block)) = static_cast<uint16_t>(word);
            *reinterpret_cast<uint16_t*>(to + kv::value_half(nb, r, 2 * t + 1, block)) = static_cast<uint16_t>(word >> 16);
            if (t == 0) *reinterpret_cast<__half*>(to + kv::value_scale(nb, r, block)) = __float2half_rn(scale);
        }
    }
}

// A thread has a piece of eight elements of a token's head.
template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvReadArgs p, FastDiv by_token, FastDiv by_pieces, int threads_per_token, int tokens_per_block) {
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int nb = p.head_dim / 32, pieces = p.head_dim / 8, local = by_token(static_cast<int>(threadIdx.x)), token = blockIdx.x * tokens_per_block + local;
    const int u = blockIdx.y * 256 + threadIdx.x - local * threads_per_token, head = by_pieces(u), piece = u - head * pieces;
    if (local >= tokens_per_block || token >= p.tokens || head >= p.kv_heads) return;
    size_t tile;
    int r;
    if (!find_rows(p.place, p.place.positions[token], p.place.sequences ? p.place.sequences[token] : token, p.kv_heads, nb, &tile, &r)) return;
    const uint8_t* from = p.pages + tile + (static_cast<size_t>(head) << (p.place.page_shift - 4)) * kv::tile_bytes(nb);
    const int block = piece >> 2, t = piece & 3;
    const size_t at = (static_cast<size_t>(token) * p.kv_heads + head) * p.head_dim + piece * 8;
    auto write = [&](T* to, uint32_t word, __half scale) {
        Pack8<T> out;
        if constexpr (kIsHalf<T>) {                  // the products are exact but for this one rounding
            const uint32_t d = __half_as_ushort(scale) * 0x10001u;
            uint32_t x[4];
            kv::less8(word, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = kv::hmul2(x[i], d);
            out.w[0] = make_uint4(__byte_perm(x[0], x[1], 0x5410), __byte_perm(x[2], x[3], 0x5410), __byte_perm(x[0], x[1], 0x7632), __byte_perm(x[2], x[3], 0x7632));
        } else {
            const float d = __half2float(scale);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (__uint_as_float(0x4B000000u | ((word >> (4 * e)) & 15u)) - 8388616.0f) * d;      // 2^23 + code: no conversion
            out = pack8<T>(f);
        }
        if (p.whole) {
            store8(to + at, out);
        } else {
            const T* e = reinterpret_cast<const T*>(&out);
#pragma unroll
            for (int i = 0; i < 8; ++i) to[at + i] = e[i];
        }
    };
    if (p.K) write(static_cast<T*>(p.K), *reinterpret_cast<const uint32_t*>(from + kv::key_word(nb, r, t, block)),
                   *reinterpret_cast<const __half*>(from + kv::key_scale(nb, r, block)));
    if (p.V) {
        const uint32_t lo = *reinterpret_cast<const uint16_t*>(from + kv::value_half(nb, r, 2 * t, block));
        const uint32_t hi = *reinterpret_cast<const uint16_t*>(from + kv::value_half(nb, r, 2 * t + 1, block));
        write(static_cast<T*>(p.V), lo | hi << 16, *reinterpret_cast<const __half*>(from + kv::value_scale(nb, r, block)));
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
    const int lanes = p.head_dim == 32 ? 4 : p.head_dim == 64 ? 8 : 16, heads = p.q_heads + 2 * p.kv_heads;
    // Four rows to a thread where they are enough.  Append and read back, four rows and one: 300 tokens of 32 and 8 heads 7.1 and 7.4 us, 1600
    // 18.5 and 22.5, 9498 of 8 heads 38.5 and 50.7 (35.6 since).
    const bool four = static_cast<long long>(p.tokens) * heads * lanes >= 1536ll * env.sm_count;
    const long long units = static_cast<long long>(four ? (p.q_heads + 3) / 4 + 2 * ((p.kv_heads + 3) / 4) : heads) * lanes;
    const int threads_per_token = units < 256 ? static_cast<int>(units) : 256, tokens_per_block = 256 / threads_per_token;
    const long long y = (units + 255) / 256;
    if (y > 65535) return cudaErrorNotSupported;
    FastDiv by_token;
    by_token.set(threads_per_token);
    const dim3 grid(static_cast<unsigned>((p.tokens + tokens_per_block - 1) / tokens_per_block), static_cast<unsigned>(y));
    const unsigned threads = static_cast<unsigned>((threads_per_token * tokens_per_block + 31) / 32 * 32);
    auto go = [&](auto kernel) { return dependent::launch(kernel, grid, threads, 0, stream, env.pdl, p, by_token, threads_per_token, tokens_per_block); };
    auto rows = [&](auto lanes_of) {
        constexpr int L = decltype(lanes_of)::value;
        if (whole) return go(four ? kv_append_kernel<T, L, true, 4> : kv_append_kernel<T, L, true, 1>);
        return go(four ? kv_append_kernel<T, L, false, 4> : kv_append_kernel<T, L, false, 1>);
    };
    if (lanes == 4) return rows(std::integral_constant<int, 4>());
    if (lanes == 8) return rows(std::integral_constant<int, 8>());
    return rows(std::integral_constant<int, 16>());
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
    const long long units = static_cast<long long>(p.kv_heads) * (p.head_dim / 8), y = (units + 255) / 256;
    if (y > 65535) return cudaErrorNotSupported;
    const int threads_per_token = units < 256 ? static_cast<int>(units) : 256, tokens_per_block = 256 / threads_per_token;
    FastDiv by_token, by_pieces;
    by_token.set(threads_per_token);
    by_pieces.set(p.head_dim / 8);
    const dim3 grid(static_cast<unsigned>((p.tokens + tokens_per_block - 1) / tokens_per_block), static_cast<unsigned>(y));
    switch (p.dtype) {
        case IO_F16: return dependent::launch(kv_read_kernel<__half>, grid, 256, 0, stream, env.pdl, p, by_token, by_pieces, threads_per_token, tokens_per_block);
        case IO_BF16: return dependent::launch(kv_read_kernel<__nv_bfloat16>, grid, 256, 0, stream, env.pdl, p, by_token, by_pieces, threads_per_token, tokens_per_block);
        default: return dependent::launch(kv_read_kernel<float>, grid, 256, 0, stream, env.pdl, p, by_token, by_pieces, threads_per_token, tokens_per_block);
    }
}

}  // namespace tcb
