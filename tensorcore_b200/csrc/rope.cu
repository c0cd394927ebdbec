// Rotary positions: rows x [tokens, heads, head_dim] turned in the planes of their pairs (i, j),
//
//   y[i] = x[i] c - x[j] s,   y[j] = x[i] s + x[j] c,   c = cos(angle), s = sin(angle) from fp32 tables [row][pair],
//
// the table row a token's position.  Pairs are (k, k + rot / 2) ("half", what tc_rope_forward and the reference do,
// lib/ops/training_cpu.cpp:541-573) or (2k, 2k + 1) ("interleaved"); elements from rot on are passed through.  Backwards
// is the rotation by the negative angle.  Every product and sum is rounded once in fp32 and the result once to the row's type, in
// the order of tc_rope_forward, so that half pairs of whole heads give its bits.
//
// Bound by the bytes of x and y: 8192 tokens of 32 heads of 128 in bf16 24.8 us, 5.6 TB/s (33.5 while a thread asked for its second head after it
// had written the first); 1531 fp32 rows of 20 heads, 72 of 96 elements turned, 4.8 us (13.4 an element to a thread).
#include <type_traits>

#include "dependent_launch.cuh"
#include "io_types.cuh"
#include "kernels.h"

namespace tcb {
namespace {

using namespace io;

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float x0 = a, x1 = b;
    a = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
    b = __fadd_rn(__fmul_rn(x0, s), __fmul_rn(x1, c));
}

// E elements as they lie in memory, one or two loads of 8 or 16 bytes.
template <typename T, int E> struct PackOf {
    using Word = std::conditional_t<E * sizeof(T) % 16 == 0, uint4, uint2>;
    static constexpr int kWords = E * sizeof(T) / sizeof(Word);
    Word w[kWords];
};
template <typename T, int E> __device__ __forceinline__ PackOf<T, E> load_piece(const T* p) {
    PackOf<T, E> r;
#pragma unroll
    for (int i = 0; i < PackOf<T, E>::kWords; ++i) r.w[i] = reinterpret_cast<const typename PackOf<T, E>::Word*>(p)[i];
    return r;
}
template <typename T, int E> __device__ __forceinline__ void store_piece(T* p, const PackOf<T, E>& r) {
#pragma unroll
    for (int i = 0; i < PackOf<T, E>::kWords; ++i) reinterpret_cast<typename PackOf<T, E>::Word*>(p)[i] = r.w[i];
}
template <typename T, int E> __device__ __forceinline__ void unpack_piece(const PackOf<T, E>& r, float (&f)[E]) {
    const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = to_f<T>(e[i]);
}
template <typename T, int E> __device__ __forceinline__ PackOf<T, E> pack_piece(const float (&f)[E]) {
    PackOf<T, E> r;
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < E; ++i) e[i] = from_f<T>(f[i]);
    return r;
}
template <int N> __device__ __forceinline__ void load_angles(const float* p, float (&f)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + i);
            f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
        }
    } else {
        const float2 v = *reinterpret_cast<const float2*>(p);
        f[0] = v.x; f[1] = v.y;
    }
}

// A token's row of the tables, or -1: a token without a position, or (with the error word set) one past the tables.
__device__ __forceinline__ long long table_row(const int* positions, int token, int rows, uint32_t* err) {
    const int p = positions ? positions[token] : token;
    if (p < 0) return -1;
    if (p >= rows) {
        if (err) atomicOr(err, ERR_BAD_SHAPE);
        return -1;
    }
    return p;
}

// A thread has a piece of E elements (16 bytes where the sizes allow it), in the half layout with its partner piece, of N heads: one
// after the other it asks for all of them, then turns them by angles that it loads once.
template <typename T, bool HALF, int E, int N>
__global__ void __launch_bounds__(256) rope_rows_kernel(const RopeArgs p, int pieces, int turned, FastDiv by_token, FastDiv by_pieces, int threads_per_token, int tokens_per_block) {
    constexpr int kAngles = HALF ? E : E / 2;
    using Piece = PackOf<T, E>;
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int local = by_token(static_cast<int>(threadIdx.x));
    const int token = blockIdx.x * tokens_per_block + local;
    if (local >= tokens_per_block || token >= p.tokens) return;
    const int rest = threadIdx.x - local * threads_per_token;
    const long long row = table_row(p.positions, token, p.table_rows, p.err);
    if (row < 0) return;
    const int groups = (p.heads + N - 1) / N;
    for (int u = rest; u < groups * pieces; u += threads_per_token) {
        const int group = by_pieces(u), k = u - group * pieces, h0 = group * N;
        const bool turns = k < turned;
        const int e0 = HALF && !turns ? p.rot_dim + (k - turned) * E : k * E, e1 = e0 + p.rot_dim / 2;
        const T* x = static_cast<const T*>(p.X) + token * p.x_token + h0 * p.x_head;
        T* y = static_cast<T*>(p.Y) + token * p.y_token + h0 * p.y_head;
        Piece first[N], second[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (h0 + n >= p.heads) break;
            first[n] = load_piece<T, E>(x + n * p.x_head + e0);
            if (HALF && turns) second[n] = load_piece<T, E>(x + n * p.x_head + e1);
        }
        float c[kAngles], s[kAngles];
        if (turns) {
            const float* cr = p.cos_t + row * (p.rot_dim / 2) + k * kAngles;
            const float* sr = p.sin_t + row * (p.rot_dim / 2) + k * kAngles;
            load_angles<kAngles>(cr, c);
            load_angles<kAngles>(sr, s);
            if (p.inverse) {
#pragma unroll
                for (int e = 0; e < kAngles; ++e) s[e] = -s[e];
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (h0 + n >= p.heads) break;
            T* yh = y + n * p.y_head;
            if (!turns) {
                store_piece<T, E>(yh + e0, first[n]);
                continue;
            }
            float a[E];
            unpack_piece<T, E>(first[n], a);
            if constexpr (HALF) {
                float b[E];
                unpack_piece<T, E>(second[n], b);
#pragma unroll
                for (int e = 0; e < E; ++e) turn(a[e], b[e], c[e], s[e]);
                store_piece<T, E>(yh + e1, pack_piece<T, E>(b));
            } else {
#pragma unroll
                for (int e = 0; e < E / 2; ++e) turn(a[2 * e], a[2 * e + 1], c[e], s[e]);
            }
            store_piece<T, E>(yh + e0, pack_piece<T, E>(a));
        }
    }
}

// Any addresses, strides and rot_dim: a thread per pair or element that is passed through.
template <typename T>
__global__ void __launch_bounds__(256) rope_elements_kernel(const RopeArgs p, int half_layout) {
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int half = p.rot_dim / 2, items = half + p.head_dim - p.rot_dim;
    const int token = blockIdx.x;
    const long long row = table_row(p.positions, token, p.table_rows, p.err);
    if (row < 0) return;
    for (long long u = static_cast<long long>(blockIdx.y) * blockDim.x + threadIdx.x; u < static_cast<long long>(p.heads) * items;
         u += static_cast<long long>(gridDim.y) * blockDim.x) {
        const int h = static_cast<int>(u / items), k = static_cast<int>(u - static_cast<long long>(h) * items);
        const T* x = static_cast<const T*>(p.X) + token * p.x_token + h * p.x_head;
        T* y = static_cast<T*>(p.Y) + token * p.y_token + h * p.y_head;
        if (k >= half) {
            y[half + k] = x[half + k];
            continue;
        }
        const int i = half_layout ? k : 2 * k, j = half_layout ? k + half : 2 * k + 1;
        float a = to_f<T>(x[i]), b = to_f<T>(x[j]);
        const float c = p.cos_t[row * half + k], s = p.sin_t[row * half + k];
        turn(a, b, c, p.inverse ? -s : s);
        y[i] = from_f<T>(a);
        y[j] = from_f<T>(b);
    }
}

// Tables: angle = position * frequency in 64 bits, whose rounding is 2^-36 of a turn at position 2^17; one thread per entry.
__global__ void __launch_bounds__(256) rope_table_kernel(const __grid_constant__ RopeTableArgs p) {
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int half = p.rot_dim / 2;
    const long long n = static_cast<long long>(p.rows) * half;
    for (long long u = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; u < n; u += static_cast<long long>(gridDim.x) * blockDim.x) {
        const long long row = u / half;
        double s, c;
        sincos(static_cast<double>(p.first + row) * p.frequency[u - row * half], &s, &c);
        p.cos_t[u] = static_cast<float>(c * p.magnitude);
        p.sin_t[u] = static_cast<float>(s * p.magnitude);
    }
}

template <typename T, int E>
cudaError_t launch_pieces_of(const RopeArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const bool half = p.layout == 0;
    const int turned = p.rot_dim / (half ? 2 * E : E), pieces = turned + (p.head_dim - p.rot_dim) / E;
    // Four heads to a thread - angles loaded once, four loads under way - where they are enough; four heads and one, fp16, 32 heads of 128:
    // 600 tokens 3.2 and 3.1 us, 1200 4.4 and 4.6, 4800 16.3 and 19.7.
    const bool four = static_cast<long long>(p.tokens) * p.heads * pieces >= 1536ll * env.sm_count;
    const long long units = static_cast<long long>(four ? (p.heads + 3) / 4 : p.heads) * pieces;
    const int threads_per_token = units < 256 ? static_cast<int>(units) : 256, tokens_per_block = 256 / threads_per_token;
    FastDiv by_token, by_pieces;
    by_token.set(threads_per_token);
    by_pieces.set(pieces);
    const unsigned grid = static_cast<unsigned>((p.tokens + tokens_per_block - 1) / tokens_per_block);
    const auto kernel = half ? four ? rope_rows_kernel<T, true, E, 4> : rope_rows_kernel<T, true, E, 1> : four ? rope_rows_kernel<T, false, E, 4> : rope_rows_kernel<T, false, E, 1>;
    return dependent::launch(kernel, grid, 256, 0, stream, env.pdl, p, pieces, turned, by_token, by_pieces, threads_per_token, tokens_per_block);
}
template <typename T>
cudaError_t launch_rope_of(const RopeArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const bool half = p.layout == 0;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.X) | reinterpret_cast<uintptr_t>(p.Y);
    const uintptr_t strides = static_cast<uintptr_t>((p.x_token | p.x_head | p.y_token | p.y_head) * static_cast<long long>(sizeof(T)));
    const uintptr_t tables = reinterpret_cast<uintptr_t>(p.cos_t) | reinterpret_cast<uintptr_t>(p.sin_t);
    // Pieces of e elements: heads are whole pieces, and so are the pairs' halves; rows of the tables begin on as many bytes as are loaded.
    auto whole = [&](int e) {
        const int bytes = e * static_cast<int>(sizeof(T)), angles = half ? 16 : 2 * e;      // (pairs of neighbours: e / 2 floats)
        if (static_cast<long long>(p.heads) * (p.head_dim / e) > 0x7fffff00LL) return false;      // a token's pieces are counted in 32 bits
        return ((at | strides) & static_cast<uintptr_t>((bytes < 16 ? bytes : 16) - 1)) == 0 && p.head_dim % e == 0 && p.rot_dim % (half ? 2 * e : e) == 0 &&
               (tables & static_cast<uintptr_t>((angles < 16 ? angles : 16) - 1)) == 0;
    };
    if constexpr (sizeof(T) == 2) {
        if (whole(8)) return launch_pieces_of<T, 8>(p, env, stream);
    }
    if (whole(4)) return launch_pieces_of<T, 4>(p, env, stream);
    const int items = p.rot_dim / 2 + p.head_dim - p.rot_dim;
    const long long blocks = (static_cast<long long>(p.heads) * items + 255) / 256;
    const dim3 grid(p.tokens, static_cast<unsigned>(blocks < 64 ? blocks : 64));
    return dependent::launch(rope_elements_kernel<T>, grid, 256, 0, stream, env.pdl, p, half ? 1 : 0);
}

}  // namespace

cudaError_t launch_rope_rows(const RopeArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    switch (p.dtype) {
        case IO_F16: return launch_rope_of<__half>(p, env, stream);
        case IO_BF16: return launch_rope_of<__nv_bfloat16>(p, env, stream);
        default: return launch_rope_of<float>(p, env, stream);
    }
}

cudaError_t launch_rope_table(const RopeTableArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const long long blocks = (static_cast<long long>(p.rows) * (p.rot_dim / 2) + 255) / 256, most = 16ll * env.sm_count;
    return dependent::launch(rope_table_kernel, static_cast<unsigned>(blocks < most ? blocks : most), 256, 0, stream, env.pdl, p);
}

}  // namespace tcb
