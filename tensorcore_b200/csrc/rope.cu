// Rotary positions: rows x [tokens, heads, head_dim] turned in the planes of their pairs (i, j),
//
//   y[i] = x[i] c - x[j] s,   y[j] = x[i] s + x[j] c,   c = cos(angle), s = sin(angle) from fp32 tables [row][pair],
//
// the table row a token's position.  Pairs are (k, k + rot / 2) ("half", what tc_rope_forward and the reference do,
// lib/ops/training_cpu.cpp:541-573) or (2k, 2k + 1) ("interleaved"); elements from rot on are passed through.  Backwards
// is the rotation by the negative angle.  Every product and sum is rounded once in fp32 and the result once to the row's type, in
// the order of tc_rope_forward, so that half pairs of whole heads give its bits.
//
// Bound by the bytes of x and y.  A thread has a piece of eight elements (with its partner piece in the half layout) of up to
// four heads, whose angles it loads once.
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

// HALF: a thread's piece of pairs is elements [8k, 8k + 8) and [8k + rot / 2, ..); else elements [8k, 8k + 8).
template <typename T, bool HALF>
__global__ void __launch_bounds__(256) rope_rows_kernel(const RopeArgs p, int pieces, int turned, int per_thread, FastDiv by_token, FastDiv by_pieces,
                                                        int threads_per_token, int tokens_per_block) {
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int local = by_token(static_cast<int>(threadIdx.x));
    const int token = blockIdx.x * tokens_per_block + local;
    if (local >= tokens_per_block || token >= p.tokens) return;
    const int rest = threadIdx.x - local * threads_per_token;
    const long long row = table_row(p.positions, token, p.table_rows, p.err);
    if (row < 0) return;
    const int groups = (p.heads + per_thread - 1) / per_thread;
    for (int u = rest; u < groups * pieces; u += threads_per_token) {
        const int group = by_pieces(u), k = u - group * pieces;
        const bool turns = k < turned;
        const int e0 = HALF && !turns ? p.rot_dim + (k - turned) * 8 : k * 8, e1 = e0 + p.rot_dim / 2;
        float c[8], s[8];
        if (turns) {
            constexpr int kAngles = HALF ? 8 : 4;
            const float* cr = p.cos_t + row * (p.rot_dim / 2) + k * kAngles;
            const float* sr = p.sin_t + row * (p.rot_dim / 2) + k * kAngles;
#pragma unroll
            for (int e = 0; e < kAngles; e += 4) {
                const float4 cv = *reinterpret_cast<const float4*>(cr + e), sv = *reinterpret_cast<const float4*>(sr + e);
                c[e] = cv.x; c[e + 1] = cv.y; c[e + 2] = cv.z; c[e + 3] = cv.w;
                s[e] = sv.x; s[e + 1] = sv.y; s[e + 2] = sv.z; s[e + 3] = sv.w;
            }
            if (p.inverse) {
#pragma unroll
                for (int e = 0; e < kAngles; ++e) s[e] = -s[e];
            }
        }
        const T* x = static_cast<const T*>(p.X) + token * p.x_token;
        T* y = static_cast<T*>(p.Y) + token * p.y_token;
        const int h1 = min(p.heads, (group + 1) * per_thread);
        for (int h = group * per_thread; h < h1; ++h) {
            const T* xh = x + h * p.x_head;
            T* yh = y + h * p.y_head;
            const Pack8<T> first = load8(xh + e0);
            if (!turns) {
                store8(yh + e0, first);
                continue;
            }
            float a[8];
            unpack8(first, a);
            if (HALF) {
                float b[8];
                unpack8(load8(xh + e1), b);
#pragma unroll
                for (int e = 0; e < 8; ++e) turn(a[e], b[e], c[e], s[e]);
                store8(yh + e0, pack8<T>(a));
                store8(yh + e1, pack8<T>(b));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) turn(a[2 * e], a[2 * e + 1], c[e], s[e]);
                store8(yh + e0, pack8<T>(a));
            }
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

template <typename T>
cudaError_t launch_rope_of(const RopeArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const bool half = p.layout == 0;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.X) | reinterpret_cast<uintptr_t>(p.Y);
    const uintptr_t tables = reinterpret_cast<uintptr_t>(p.cos_t) | reinterpret_cast<uintptr_t>(p.sin_t);
    const long long strides = (p.x_token | p.x_head | p.y_token | p.y_head) * static_cast<long long>(sizeof(T));
    const bool whole = (at & 15u) == 0 && (tables & 15u) == 0 && (strides & 15) == 0 && p.head_dim % 8 == 0 && p.rot_dim % (half ? 16 : 8) == 0;
    if (!whole) {
        const int items = p.rot_dim / 2 + p.head_dim - p.rot_dim;
        const long long blocks = (static_cast<long long>(p.heads) * items + 255) / 256;
        const dim3 grid(p.tokens, static_cast<unsigned>(blocks < 64 ? blocks : 64));
        return dependent::launch(rope_elements_kernel<T>, grid, 256, 0, stream, env.pdl, p, half ? 1 : 0);
    }
    const int turned = half ? p.rot_dim / 16 : p.rot_dim / 8, pieces = turned + (p.head_dim - p.rot_dim) / 8;
    const int per_thread = static_cast<long long>(p.tokens) * p.heads * pieces >= 4ll * 2048 * env.sm_count ? 4 : 1;
    const long long units = static_cast<long long>((p.heads + per_thread - 1) / per_thread) * pieces;
    const int threads_per_token = units < 256 ? static_cast<int>(units) : 256, tokens_per_block = 256 / threads_per_token;
    FastDiv by_token, by_pieces;
    by_token.set(threads_per_token);
    by_pieces.set(pieces);
    const unsigned grid = static_cast<unsigned>((p.tokens + tokens_per_block - 1) / tokens_per_block);
    return dependent::launch(half ? rope_rows_kernel<T, true> : rope_rows_kernel<T, false>, grid, 256, 0, stream, env.pdl, p, pieces, turned, per_thread, by_token, by_pieces,
                             threads_per_token, tokens_per_block);
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
