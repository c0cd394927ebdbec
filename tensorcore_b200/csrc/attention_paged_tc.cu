// Prompts over the paged 4-bit cache on the tensor cores (tcgen05): sequences with more (query, head) rows on a K/V head than
// attention_paged.cu takes.  Same operation and data (kv_cache.cuh).
//
//   * A CTA owns 256 or 128 rows of a sequence and K/V head (head fastest) and walks the keys it sees 128 at a time; where there are
//     fewer CTAs than SMs the keys are cut into chunks, whose results a second kernel merges.
//   * Eight warps bring the tiles in (bulk copies) and write them as fp16 matrices into shared memory, in 128-byte swizzled rows: keys
//     as rows of K, elements as rows of V^T.  Both in the order that the packed words give without a shuffle: within 32 keys, key
//     16 a + 8 h + 2 t + e is number 8 t + 4 a + 2 h + e, and within eight elements the order is 0 4 1 5 2 6 3 7 for K, and so for Q.
//     K is exact: a scale is taken as its upper eight bits and its lower three, whose products with code - 8 fp16 numbers hold,
//     so S takes two matrices.  (As one, rounded to 11 bits, K was the largest part of O's error, and the log-sum-exp of a row of few keys
//     was off by 1e-5 of itself.)  V is (code - 8) * scale rounded once.
//   * Two groups of eight softmax warps, each with scores, probabilities and an accumulator of its own in tensor memory: while one
//     group works on its scores the tensor cores work for the other.  Of 256 rows a group has 128, at every step; of 128 rows the groups take the
//     steps in turn and their sums meet at the end.  S = Q K^T, then the probabilities in the place of the scores (two fp16 numbers
//     each for fp16 results, 22 bits; one for bf16, whose results have eight bits), then O += P V.  A thread of each group issues;
//     its order - P V of a step, then S of the group's next - keeps the operands apart.
//   * Softmax: two threads per row.  The exponents' reference is the row's maximum when it was last more than 2^8 above
//     the one before, so that O is rescaled rarely; probabilities are carried 2^7 times as large.  Scores are read twice, for the
//     maximum and for the exponentials: 24 warps leave 80 registers.
//   * A key that a row does not see has no part in it: scores are masked, V of keys that are not there is zero, and a V scale that is
//     not finite is left out of the matrix; the rows that do see it have NaN in that block.  Queries are scaled by a power of two to fp16's
//     middle.  A scale of 8192 or more, of K or V, is beyond the matrices (-8 times it is below -65504; caches of fp16 rows have none):
//     V is left out of them, and the rows that see the key are done once more from the pages (rows_again).
//   * What bounds it: the chain of a group's step - scores, maximum, exponentials, products - with the conversions beside it.  128 rows
//     and keys of 128 elements, fp16: 4100 clk a step where the tensor cores need 2050 (K and P twice) and shared memory 3200 of
//     its cycles; without the conversions 3750, without those and the second products 3150, without the second products alone 4100.  256
//     rows share the conversions: 2048 tokens over themselves in bf16 78.4 us (439 Tflop/s), as 128 rows 92.6; four
//     times 1024 in fp16 128.8 and 138.1.  512 tokens over 4608 keys, fp16: 128 CTAs of 128 rows 80.1 us (456 Tflop/s), 64 of 256 rows in two
//     chunks 107.  Warps of their own to issue, to convert K or V only, or twelve to convert: no faster.
#include "attention_math.cuh"
#include "dependent_launch.cuh"
#include "io_types.cuh"
#include "kernels.h"
#include "kv_cache.cuh"
#include "sm100_prims.cuh"

namespace tcb {
namespace {

using namespace sm100;
using attn::pack_h2;
using attn::exp2_of;
using attn::fma2;
using attn::add2;
using kv::hmul2;
using kv::less8;

constexpr int kRows = 128, kKeys = 128;
constexpr int kSoftWarps = 16, kDequantWarps = 8, kThreads = (kSoftWarps + kDequantWarps) * 32;
constexpr int kBarBytes = 8192;
constexpr uint32_t kColS = 0, kColO = 256, kTmemCols = 512;
constexpr float kCarry = 7.0f, kSlack = 8.0f;

// Of a step's four times 32 keys: whether anything follows; keys on pages that do not exist; by block, keys whose V scale is not finite;
// of each warp's blocks, keys with a K or V scale that fp16 matrices do not hold.
struct alignas(16) StepNotes { uint32_t any[8], hidden[4], poison[4][4], large[8]; };
constexpr uint32_t kAgain = 0x80000000u;      // beside a row's NaN blocks: it sees such a key
__device__ __forceinline__ bool too_large(uint32_t scale) { return (scale & 0x7FFFu) >= 0x7000u && (scale & 0x7FFFu) < 0x7C00u; }      // 8192 or more: times -8 below -65504
struct Bars {
    uint64_t q_full, k_full[2], k_empty, v_full[2], v_empty[2], s_full[2], p_full[2], pv_done[2], drain[2], pair[2][4], all;
    uint64_t raw_full[4][2], raw_empty[4][2];
    uint32_t tmem_base;
    int abort_flag, again;             // again: rows are left to rows_again
    float best[2][2][2][kRows];        // [turn][group][half]: maxima that the two threads of a row exchange
    float back[2 * kRows];             // what a row of Q was multiplied by, undone
    uint32_t sick[2][2][kRows];        // [group][half], at the end
    StepNotes notes[4];
};
static_assert(sizeof(Bars) <= kBarBytes, "barrier block too large");

template <int NB> constexpr int kFirstBlocks = (NB + 1) / 2;      // those of the first warp of two that share keys
// BOTH: a group of softmax warps for each half of a tile of 256 rows; else one tile of 128, whose steps the groups take in turn.
template <int NB, bool BOTH> struct TcShape {
    static constexpr int kTileRows = BOTH ? 2 * kRows : kRows, kSlots = BOTH ? 1 : 2, kStride = BOTH ? 1 : 2;      // rows; copies of packed keys; steps of a group
    static constexpr int D = 32 * NB, kSlabs = (NB + 1) / 2;
    static constexpr uint32_t kKSlab = kKeys * 128, kKTile = kSlabs * kKSlab;        // 64 elements of 128 keys; Q likewise
    static constexpr uint32_t kVSlab = D * 128, kVTile = 2 * kVSlab;                 // 64 keys of D elements
    static constexpr int kRawBytes = 2 * kv::tile_bytes(NB);                         // of a warp's 32 keys
    static constexpr uint32_t kQAt = kBarBytes, kKAt = kQAt + (BOTH ? 2 : 1) * kKTile, kVAt = kKAt + 2 * kKTile, kRawAt = kVAt + 2 * kVTile;      // K: its two parts; V: two steps
    static constexpr uint32_t kSmem = kRawAt + 4 * kSlots * kRawBytes;
    static_assert(kSmem <= 227 * 1024, "");
};

__device__ __forceinline__ uint64_t desc128(uint32_t addr) { return smem_desc_kmajor(addr, 16u, 1024u) | (2ull << 61); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <int N> __device__ __forceinline__ void words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N == 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}
// Which of the four times 32 keys' order a key is, and back.
__host__ __device__ constexpr int order_of_key(int a, int r) { return 8 * ((r & 7) >> 1) + 4 * a + 2 * (r >> 3) + (r & 1); }
__host__ __device__ constexpr int key_of_order(int c) { return (c & ~31) + 16 * ((c >> 2) & 1) + 8 * ((c >> 1) & 1) + 2 * ((c & 31) >> 3) + (c & 1); }

// What a CTA works on: a sequence's tile of p.tile_rows rows; false: none is left.
struct Tile { int seq, q0, nq, len, row0; };
__device__ __forceinline__ bool find_tile(const AttnPagedArgs& p, int tile_no, Tile* out) {
    const int lane = threadIdx.x & 31, G = p.per_kv;
    auto tiles_of = [&](int nq) { return nq * G > p.most_rows ? (nq * G + p.tile_rows - 1) / p.tile_rows : 0; };
    int seq = -1, q0 = 0, nq = 0, in = 0;
    if (p.q_start) {
        int before = 0;
        for (int base = 0; base < p.n_seqs && seq < 0; base += 32) {
            const int s = base + lane;
            int a = 0, n = 0;
            if (s < p.n_seqs) {
                a = min(max(p.q_start[s], 0), p.tokens);
                n = max(0, min(p.q_start[s + 1], p.tokens) - a);
            }
            int sum = tiles_of(n);
            const int mine = sum;
#pragma unroll
            for (int x = 1; x < 32; x *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, sum, x);
                if (lane >= x) sum += v;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, tile_no < before + sum);
            if (hit) {
                const int from = __ffs(hit) - 1;
                seq = base + from;
                q0 = __shfl_sync(0xffffffffu, a, from);
                nq = __shfl_sync(0xffffffffu, n, from);
                in = tile_no - before - __shfl_sync(0xffffffffu, sum - mine, from);
            }
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (seq < 0) return false;
    } else {
        nq = p.tokens / p.n_seqs;
        const int n = tiles_of(nq);
        if (n == 0 || tile_no >= n * p.n_seqs) return false;
        seq = tile_no / n;
        q0 = seq * nq;
        in = tile_no - seq * n;
    }
    const long long most = static_cast<long long>(p.max_pages) << p.page_shift;
    const int len = p.seq_lens[seq];
    out->seq = seq;
    out->q0 = q0;
    out->nq = nq;
    out->len = len < 0 ? 0 : len > most ? static_cast<int>(most) : len;
    out->row0 = (tiles_of(nq) - 1 - in) * p.tile_rows;      // long causal tiles first
    if (len > most && lane == 0 && p.err) atomicOr(p.err, ERR_BAD_SHAPE);
    return true;
}

// Keys that any row of the tile sees, from a whole tile of the cache on, and this chunk's steps of them.
__device__ __forceinline__ void steps_of(const AttnPagedArgs& p, const Tile& tile, int rows, int* first_key, int* steps) {
    const int pos0 = tile.len - tile.nq, i_min = p.by_per_kv(tile.row0), i_max = p.by_per_kv(tile.row0 + rows - 1);
    const int k_begin = p.first_seen(pos0 + i_min) & ~15;
    const int k_end = p.causal ? min(tile.len, pos0 + i_max + 1) : tile.len;
    const int all = k_end > k_begin ? (k_end - k_begin + kKeys - 1) / kKeys : 0, chunk = blockIdx.y, chunks = gridDim.y;
    const int step0 = static_cast<int>(static_cast<long long>(all) * chunk / chunks);
    *steps = static_cast<int>(static_cast<long long>(all) * (chunk + 1) / chunks) - step0;
    *first_key = k_begin + step0 * kKeys;
}

// The CTA's rows that see keys whose K or V fp16 matrices do not hold, once more from the pages, in fp32: a warp has a row, a lane an element of
// each block, and the keys go by four at a time.  Nothing is kept for it from before, so that rows of other caches pay nothing; 512 tokens over
// 4608 keys, 32 heads on 8, all of whose rows see such a key: 14 ms, against 82 us without one (one key at a time: 18 ms).
template <typename T, int NB, bool BOTH> __device__ __noinline__ void rows_again(const AttnPagedArgs& p) {
    constexpr int D = 32 * NB;
    extern __shared__ __align__(1024) uint8_t smem[];
    const Bars* const bars = reinterpret_cast<const Bars*>(smem);
    const int lane = threadIdx.x & 31, G = p.per_kv, tile_no = p.by_kv_heads(static_cast<int>(blockIdx.x)), hkv = static_cast<int>(blockIdx.x) - tile_no * p.kv_heads;
    Tile tile;
    if (!find_tile(p, tile_no, &tile)) return;
    const int rows = min(TcShape<NB, BOTH>::kTileRows, tile.nq * G - tile.row0), chunks = gridDim.y, shift = p.page_shift;
    int first_key, steps;
    steps_of(p, tile, rows, &first_key, &steps);
    const int* const own_pages = p.page_table + static_cast<size_t>(tile.seq) * p.max_pages;
    const uint8_t* const head_pages = p.pages + (static_cast<size_t>(hkv * kv::tile_bytes(NB)) << (shift - 4));
    const size_t page_bytes = static_cast<size_t>(p.kv_heads * kv::tile_bytes(NB)) << (shift - 4);
    for (int tr = threadIdx.x >> 5; tr < rows; tr += kThreads / 32) {
        uint32_t ill = bars->sick[BOTH ? tr / kRows : 0][0][tr % kRows] | bars->sick[BOTH ? tr / kRows : 0][1][tr % kRows];
        if (!BOTH) ill |= bars->sick[1][0][tr] | bars->sick[1][1][tr];
        if (!(ill & kAgain)) continue;
        const int r = tile.row0 + tr, i = p.by_per_kv(r), h = hkv * G + (r - i * G), token = tile.q0 + i, pos = tile.len - tile.nq + i;
        const int end = min(first_key + steps * kKeys, p.causal ? min(tile.len, pos + 1) : tile.len), begin = max(first_key, p.first_seen(pos));
        const T* const src = static_cast<const T*>(p.Q) + token * p.q_token + h * p.q_head;
        float q[NB], o[NB], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            q[b] = io::to_f<T>(src[32 * b + lane]);
            o[b] = 0.f;
        }
        constexpr int kAtOnce = 4;                // keys, of one tile
#pragma unroll 1
        for (int key = begin & -kAtOnce; key < end; key += kAtOnce) {
            const int page = own_pages[key >> shift];
            if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.n_pages)) continue;
            const uint8_t* const at = head_pages + page * page_bytes + ((key & ((1 << shift) - 1)) >> 4) * kv::tile_bytes(NB);
            auto number = [&](int byte, int scale) {
                return (static_cast<int>(at[byte + (lane & 3) / 2] >> (4 * (lane & 1)) & 15) - 8) * __half2float(*reinterpret_cast<const __half*>(at + scale));
            };
            float s[kAtOnce], v[kAtOnce][NB];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const int in = (key & 15) + u;
                s[u] = 0.f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    s[u] = fmaf(q[b], number(kv::key_word(NB, in, lane >> 3, b) + (lane & 4) / 2, kv::key_scale(NB, in, b)), s[u]);
                    v[u][b] = number(kv::value_half(NB, in, lane >> 2, b), kv::value_scale(NB, in, b));
                }
            }
            const float was = m;
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], x);
                s[u] *= p.scale * 1.4426950408889634f;
                if (key + u >= begin && key + u < end) m = fmaxf(m, s[u]);
            }
            const float ref = m > -INFINITY ? m : 0.f, keep = was > -INFINITY ? exp2_of(was - ref) : 0.f;
            l *= keep;
#pragma unroll
            for (int b = 0; b < NB; ++b) o[b] *= keep;
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                if (key + u < begin || key + u >= end) continue;
                const float e = exp2_of(s[u] - ref);
                l += e;
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] = fmaf(e, v[u][b], o[b]);
            }
        }
        if (chunks > 1) {
            float* const part = p.parts + ((static_cast<size_t>(token) * p.q_heads + h) * chunks + blockIdx.y) * (D + 2);
#pragma unroll
            for (int b = 0; b < NB; ++b) part[2 + 32 * b + lane] = o[b];
            if (lane < 2) part[lane] = lane == 0 ? m : l;
        } else {
            T* const dst = static_cast<T*>(p.O) + token * p.o_token + h * p.o_head;
#pragma unroll
            for (int b = 0; b < NB; ++b) dst[32 * b + lane] = io::from_f<T>(l == 0.f ? 0.f : o[b] / l);
            if (lane == 0 && p.LSE) p.LSE[static_cast<size_t>(token) * p.q_heads + h] = l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
        }
    }
}

template <typename T, int NB, bool BOTH>
__global__ void __launch_bounds__(kThreads, 1) attention_paged_prompt_kernel(const __grid_constant__ AttnPagedArgs p) {
    using S = TcShape<NB, BOTH>;
    constexpr int D = S::D;
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    constexpr bool kTwo = io::kIsHalf<T>;      // probabilities as two fp16 numbers
    extern __shared__ __align__(1024) uint8_t smem[];
    Bars* bars = reinterpret_cast<Bars*>(smem);
    volatile int* abort_flag = &bars->abort_flag;
    const uint32_t base_s = s_u32(smem);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int G = p.per_kv, tile_no = p.by_kv_heads(static_cast<int>(blockIdx.x)), hkv = static_cast<int>(blockIdx.x) - tile_no * p.kv_heads;
    Tile tile;
    if (!find_tile(p, tile_no, &tile)) return;
    if (p.err && static_cast<unsigned>(blockIdx.x) + 1 == gridDim.x && warp == 0) {      // a tile that nobody has: more queries than declared
        Tile none;
        if (find_tile(p, tile_no + 1, &none) && lane == 0) atomicOr(p.err, ERR_BAD_SHAPE);
    }
    const int R = tile.nq * G, rows_here = min(S::kTileRows, R - tile.row0);
    const int pos0 = tile.len - tile.nq;                          // position of the sequence's first query
    const int chunk = blockIdx.y, chunks = gridDim.y;
    int first_key, steps;
    steps_of(p, tile, rows_here, &first_key, &steps);

    if (tid == 0) {
        bar_init(&bars->q_full, kSoftWarps);
        bar_init(&bars->all, kSoftWarps);
        bar_init(&bars->k_empty, BOTH ? 2 : 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(&bars->k_full[i], kDequantWarps);      // (the steps' parities are the groups' own: a wait sees one phase back only)
            bar_init(&bars->v_full[i], kDequantWarps);
            bar_init(&bars->v_empty[i], BOTH ? 2 : 1);
            bar_init(&bars->s_full[i], 1);
            bar_init(&bars->p_full[i], kSoftWarps / 2);
            bar_init(&bars->pv_done[i], 1);
            bar_init(&bars->drain[i], 1);
            for (int k = 0; k < 4; ++k) bar_init(&bars->pair[i][k], 2);
        }
        for (int i = 0; i < 8; ++i) {
            bar_init(&bars->raw_full[0][0] + i, 1);
            bar_init(&bars->raw_empty[0][0] + i, 2);
        }
        bars->abort_flag = bars->again = 0;
        fence_barrier_init();
    } else if (warp == kSoftWarps) {
        tmem_alloc(&bars->tmem_base, kTmemCols);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = bars->tmem_base;
    bool failed = false;

    if (warp < kSoftWarps) {
        // ---------------- Q: rows scaled by a power of two to 2^13 .. 2^14, as fp16 -----------------------------------
        {
            constexpr int kLanes = NB == 3 ? 16 : 4 * NB, kAtOnce = 32 / kLanes, kTurns = 8 / kAtOnce;
            const int piece = lane % kLanes;
            for (int eight = 0; eight < (BOTH ? 2 : 1); ++eight)
#pragma unroll
            for (int u = 0; u < kTurns; ++u) {
                const int lrow = (BOTH ? 2 * warp + eight : warp) * 8 + u * kAtOnce + lane / kLanes, r = tile.row0 + min(lrow, rows_here - 1);
                const int i = p.by_per_kv(r);
                const T* src = static_cast<const T*>(p.Q) + (tile.q0 + i) * p.q_token + (hkv * G + (r - i * G)) * p.q_head + 8 * piece;
                float v[8], most = 0.f;
                if (8 * piece < D) {
                    if (p.q_vec) {
                        io::unpack8(io::load8(src), v);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = io::to_f<T>(src[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
                }
#pragma unroll
                for (int x = 1; x < kLanes; x *= 2) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, x));
                const int ex = min(max(static_cast<int>(__float_as_uint(most) >> 23), 27), 240);
                const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 + 127 - ex) << 23);
                if (piece == 0) bars->back[lrow] = __uint_as_float(static_cast<uint32_t>(ex - 13) << 23);
                if (8 * piece < D) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] *= up;
                    sts128(base_s + S::kQAt + (lrow / kRows) * S::kKTile + (piece / 8) * S::kKSlab + (lrow % kRows) * 128 + (((piece & 7) ^ (lrow & 7)) * 16),
                           make_uint4(pack_h2(v[0], v[4]), pack_h2(v[1], v[5]), pack_h2(v[2], v[6]), pack_h2(v[3], v[7])));
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars->q_full);
        }
        // ---------------- softmax: two threads per row = TMEM lane, 64 keys of a step each ------------------------------
        const int group = warp >> 3, half = (warp >> 2) & 1, quad = warp & 3, lr = quad * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16), s_at = lanes + kColS + group * 128u;
        if (!wait_all(&bars->q_full, 0, abort_flag)) failed = true;      // the rows' factors are there
        const int row0 = BOTH ? group * kRows : 0, tr = row0 + lr;    // of the tile
        const int i = p.by_per_kv(tile.row0 + min(tr, rows_here - 1)), pos = pos0 + i;
        const float f = fmaxf(bars->back[tr] * p.scale * 1.4426950408889634f, 1.17549435e-38f);      // minus infinity times it is that
        const int hi_key = p.causal ? min(tile.len, pos + 1) : tile.len, lo_key = p.first_seen(pos);
        const int hi_all = p.causal ? min(tile.len, pos0 + p.by_per_kv(tile.row0 + min(row0, rows_here - 1)) + 1) : tile.len;
        const int lo_all = p.first_seen(pos0 + p.by_per_kv(tile.row0 + min(row0 + kRows, rows_here) - 1));
        const int first_step = BOTH ? 0 : group;
        const uint32_t q_at = base_s + S::kQAt + (BOTH ? group * S::kKTile : 0u);
        // The group's first warp issues.
        const bool issues = (warp & 7) == 0;
        auto scores = [&](int t) {
            if (!wait_all(&bars->k_full[t & 1], static_cast<uint32_t>(t >> 1) & 1u, abort_flag)) { failed = true; return; }
            tc_fence_after_sync();
            if (elect_one()) {
                constexpr uint32_t id = idesc_f16_f32(kRows, kKeys);
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    const uint32_t off = (j / 4) * S::kKSlab + (j % 4) * 32;
                    mma_f16_ss(tmem + kColS + group * 128u, desc128(q_at + off), desc128(base_s + S::kKAt + off), id, j > 0 ? 1u : 0u);
                    mma_f16_ss(tmem + kColS + group * 128u, desc128(q_at + off), desc128(base_s + S::kKAt + S::kKTile + off), id, 1u);
                }
                mma_commit(&bars->s_full[group]);
                mma_commit(&bars->k_empty);
            }
            __syncwarp();
        };
        auto product = [&](int t, int turn) {
            if (!wait_all(&bars->v_full[t & 1], static_cast<uint32_t>(t >> 1) & 1u, abort_flag) ||
                !wait_all(&bars->p_full[group], static_cast<uint32_t>(turn) & 1u, abort_flag)) { failed = true; return; }
            tc_fence_after_sync();
            if (elect_one()) {
                constexpr uint32_t id = idesc_f16_f32(kRows, D);
                const uint32_t o_at = tmem + kColO + group * 128u, p_at = tmem + kColS + group * 128u;
#pragma unroll
                for (int j = 0; j < kKeys / 16; ++j) {
                    const uint64_t vd = desc128(base_s + S::kVAt + (t & 1) * S::kVTile + (j / 4) * S::kVSlab + (j % 4) * 32);
                    const uint32_t a = p_at + 64u * (j / 4) + 8u * (j % 4);      // a half's probabilities are where its scores were
                    mma_f16_ts(o_at, a, vd, id, turn > 0 || j > 0 ? 1u : 0u);
                    if constexpr (kTwo) mma_f16_ts(o_at, a + 32u, vd, id, 1u);
                }
                mma_commit(&bars->v_empty[t & 1]);
                if (t + S::kStride >= steps) mma_commit(&bars->pv_done[group]);
            }
            __syncwarp();
        };
        if (issues && !failed && first_step < steps) scores(first_step);
        float ref = -INFINITY, l = 0.f;
        uint32_t sick = 0;                                            // blocks of O that are NaN
        int turn = 0;
        for (int t = first_step; t < steps && !failed; t += S::kStride, ++turn) {
            if (!wait_all(&bars->s_full[group], static_cast<uint32_t>(turn) & 1u, abort_flag)) { failed = true; break; }
            tc_fence_after_sync();
            const int j0 = first_key + t * kKeys;
            const StepNotes& notes = bars->notes[t & 3];
            const uint4 odd4 = *reinterpret_cast<const uint4*>(notes.any), odd5 = *reinterpret_cast<const uint4*>(notes.any + 4);
            const uint32_t odd = odd4.x | odd4.y | odd4.z | odd4.w | odd5.x | odd5.y | odd5.z | odd5.w;
            const bool masked = j0 + kKeys > hi_all || j0 < lo_all || odd;
            const uint32_t mine_at = s_at + 64u * half;
            // 32 of this thread's scores, in the order of the matrix; what the row does not see is minus infinity
            auto read = [&](int c, uint32_t (&raw)[2][16]) {
                tmem_ld16(mine_at + 32u * c, raw[0]);
                tmem_ld16(mine_at + 32u * c + 16u, raw[1]);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) asm volatile("" : "+r"(raw[e / 16][e % 16]));      // read behind the wait
                if (masked) {
                    const int base = j0 + 64 * half + 32 * c, hi_e = hi_key - base, lo_e = lo_key - base;
                    const uint32_t gone = odd ? notes.hidden[2 * half + c] : 0u;
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const int key = key_of_order(e);
                        if (key >= hi_e || key < lo_e || (gone >> e & 1u)) raw[e / 16][e % 16] = 0xff800000u;
                    }
                }
            };
            float mine = -INFINITY;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t raw[2][16];
                read(c, raw);
                float mx[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    mx[k] = __uint_as_float(raw[k][0]);
#pragma unroll
                    for (int e = 1; e < 15; e += 2) mx[k] = max3(mx[k], __uint_as_float(raw[k][e]), __uint_as_float(raw[k][e + 1]));
                }
                mine = max3(mine, fmaxf(mx[0], __uint_as_float(raw[0][15])), fmaxf(mx[1], __uint_as_float(raw[1][15])));
                if (odd) {
                    const int w = 2 * half + c;
                    if ((notes.any[w] | notes.any[w + 4]) & 2u) {
                        const int base = j0 + 32 * w;
                        uint32_t seen = 0;        // by place: a score may be minus infinity
#pragma unroll 1
                        for (int e = 0; e < 32; ++e) seen |= base + key_of_order(e) < hi_key && base + key_of_order(e) >= lo_key ? 1u << e : 0u;
                        seen &= ~notes.hidden[w];
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            if ((notes.any[w + (b < kFirstBlocks<NB> ? 0 : 4)] & 2u) && (notes.poison[w][b] & seen)) sick |= 1u << b;
#pragma unroll
                        for (int k = w; k < 8; k += 4)
                            if ((notes.any[k] & 2u) && (notes.large[k] & seen)) sick |= kAgain;
                    }
                }
            }
            mine *= f;
            // the row's other thread is four warps away; its read of this turn's words is behind it when they are written again
            bars->best[turn & 1][group][half][lr] = mine;
            __syncwarp();
            if (lane == 0) bar_arrive(&bars->pair[group][quad]);
            if (!wait_all(&bars->pair[group][quad], static_cast<uint32_t>(turn) & 1u, abort_flag)) { failed = true; break; }
            const float most = fmaxf(mine, bars->best[turn & 1][group][half ^ 1][lr]);
            const bool grown = most > ref + kSlack || (ref == -INFINITY && most > -INFINITY);
            if (__any_sync(0xffffffffu, grown)) {                     // the product of the group's step before is done: its S came behind it
                const float to = grown ? most : ref, keep = ref > -INFINITY ? exp2_of(ref - to) : to > -INFINITY ? 0.f : 1.f;
                ref = to;
                l *= keep;
                if (turn > 0) {
                    const uint32_t at = lanes + kColO + group * 128u + static_cast<uint32_t>(half * (D / 2));
#pragma unroll
                    for (int c = 0; c < NB; ++c) {
                        uint32_t v[16];
                        tmem_ld16(at + 16u * c, v);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            asm volatile("" : "+r"(v[e]));
                            v[e] = __float_as_uint(__uint_as_float(v[e]) * keep);
                        }
                        tmem_st16(at + 16u * c, v);
                    }
                }
            }
            const float minus = ref > -INFINITY ? kCarry - ref : 0.f;
            float sum[2] = {0.f, 0.f};
            uint32_t low[16];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t raw[2][16], top[16];
                read(c, raw);
                if (kTwo && c == 1) tmem_st16(mine_at + 32u, low);      // into columns that have been read now
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float a = __uint_as_float(raw[e / 8][2 * (e % 8)]), b = __uint_as_float(raw[e / 8][2 * (e % 8) + 1]);
                    fma2(a, b, f, f, minus, minus);
                    a = exp2_of(a);
                    b = exp2_of(b);
                    add2(sum[0], sum[1], a, b);
                    top[e] = pack_h2(a, b);
                    if constexpr (kTwo) {
                        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&top[e]));
                        add2(a, b, -back.x, -back.y);
                        low[e] = pack_h2(a, b);
                    }
                }
                tmem_st16(mine_at + 16u * c, top);
                if (kTwo && c == 1) tmem_st16(mine_at + 48u, low);
            }
            l += sum[0] + sum[1];
            tmem_wait_st();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars->p_full[group]);
            if (issues) {
                product(t, turn);
                if (!failed && t + S::kStride < steps) scores(t + S::kStride);
            }
        }
        // ---------------- results: a row's two threads have its elements' halves, or (steps in turn) its four threads quarters --------
        bars->sick[group][half][lr] = sick;
        if (sick & kAgain) bars->again = 1;
        auto finish = [&](float m, float total, uint32_t ill, int c0, int pieces, auto element) {      // elements c0 .. of eight each, element(c, o) theirs
            const int r = tile.row0 + tr, h = hkv * G + (r - p.by_per_kv(min(r, R - 1)) * G), token = tile.q0 + i;
            const bool live = tr < rows_here;
            const float by = (chunks > 1 ? 1.0f : total == 0.f ? 0.f : 1.0f / total) * (1.0f / 128.0f);
            float* const part = p.parts + ((static_cast<size_t>(token) * p.q_heads + h) * chunks + chunk) * (D + 2);
#pragma unroll
            for (int c = 0; c < 2 * NB; ++c) {
                if (c >= pieces) break;
                float o[8];
                element(c0 + 8 * c, o);
                if (!live) continue;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = (ill >> ((c0 + 8 * c) / 32) & 1u) ? __uint_as_float(0x7fc00000u) : o[e] * by;
                if (chunks > 1) {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) *reinterpret_cast<float2*>(part + 2 + c0 + 8 * c + e) = make_float2(o[e], o[e + 1]);
                } else {
                    T* dst = static_cast<T*>(p.O) + token * p.o_token + h * p.o_head + c0 + 8 * c;
                    if (p.o_vec16) {
                        io::store8(dst, io::pack8<T>(o));
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) dst[e] = io::from_f<T>(o[e]);
                    }
                }
            }
            if (live && c0 == 0) {
                if (chunks > 1) {
                    part[0] = m;
                    part[1] = total;
                } else if (p.LSE) {
                    p.LSE[static_cast<size_t>(token) * p.q_heads + h] = total == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(total);
                }
            }
        };
        auto column = [&](int g, int c, uint32_t (&v)[8]) {
            tmem_ld8(lanes + kColO + 128u * g + static_cast<uint32_t>(c), v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) asm volatile("" : "+r"(v[e]));
        };
        if constexpr (BOTH) {
            if (!failed && steps > 0 && !wait_all(&bars->pv_done[group], 0, abort_flag)) failed = true;
            tc_fence_after_sync();
            if (!failed) {
                bars->best[turn & 1][group][half][lr] = l;
                __syncwarp();
                if (lane == 0) bar_arrive(&bars->pair[group][quad]);
                if (!wait_all(&bars->pair[group][quad], static_cast<uint32_t>(turn) & 1u, abort_flag)) failed = true;
            }
            if (!failed) {
                const float total = (bars->best[turn & 1][group][0][lr] + bars->best[turn & 1][group][1][lr]) * (1.0f / 128.0f);
                finish(ref, total, bars->sick[group][0][lr] | bars->sick[group][1][lr], half * (D / 2), 2 * NB, [&](int c, float (&o)[8]) {
                    uint32_t a[8];
                    if (steps > 0) column(group, c, a);
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = steps > 0 ? __uint_as_float(a[e]) : 0.f;
                });
            }
        } else {
            if (!failed && steps > 0 && !wait_all(&bars->pv_done[0], 0, abort_flag)) failed = true;
            if (!failed && steps > 1 && !wait_all(&bars->pv_done[1], 0, abort_flag)) failed = true;
            tc_fence_after_sync();
            float* const sums = reinterpret_cast<float*>(smem + S::kKAt);      // every MMA is done: [group][half] sums, [group] references
            if (!failed) {
                sums[(2 * group + half) * kRows + lr] = l;
                if (half == 0) sums[(4 + group) * kRows + lr] = ref;
                __syncwarp();
                if (lane == 0) bar_arrive(&bars->all);
                if (!wait_all(&bars->all, 0, abort_flag)) failed = true;
            }
            if (!failed) {
                const float ra = sums[4 * kRows + lr], rb = sums[5 * kRows + lr], m = fmaxf(ra, rb);
                const float wa = ra > -INFINITY ? exp2_of(ra - m) : 0.f, wb = rb > -INFINITY ? exp2_of(rb - m) : 0.f;
                const float total = ((sums[lr] + sums[kRows + lr]) * wa + (sums[2 * kRows + lr] + sums[3 * kRows + lr]) * wb) * (1.0f / 128.0f);
                const uint32_t ill = bars->sick[0][0][lr] | bars->sick[0][1][lr] | bars->sick[1][0][lr] | bars->sick[1][1][lr];
                finish(m, total, ill, (warp >> 2) * (D / 4), NB, [&](int c, float (&o)[8]) {
                    uint32_t a[8], b[8];
                    if (steps > 0) column(0, c, a);
                    if (steps > 1) column(1, c, b);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        o[e] = steps > 0 && wa != 0.f ? __uint_as_float(a[e]) * wa : 0.f;
                        if (steps > 1 && wb != 0.f) o[e] = fmaf(__uint_as_float(b[e]), wb, o[e]);
                    }
                });
            }
        }
        if (issues && (failed || *abort_flag)) {
            // every MMA issued has completed before tensor and shared memory are released
            if (elect_one()) mma_commit(&bars->drain[group]);
            __syncwarp();
            bar_wait(&bars->drain[group], 0, nullptr, 100000000LL);
        }
        tc_fence_before_sync();
    } else {
        // ---------------- 32 keys of every step: from the pages into shared memory, and as fp16 into the matrices -----------
        // Warps w and w + 4 share the keys; each has half of the blocks.
        const int wd = warp - kSoftWarps, w = wd & 3, part = wd >> 2, shift = p.page_shift, in_page = (1 << shift) - 1;
        constexpr int kTileBytes = kv::tile_bytes(NB), kMine = kFirstBlocks<NB>;
        const int b0 = part * kMine;
        uint8_t* const ring = smem + S::kRawAt + w * S::kSlots * S::kRawBytes;
        const int* const own_pages = p.page_table + static_cast<size_t>(tile.seq) * p.max_pages;
        const uint8_t* const head_pages = p.pages + (static_cast<size_t>(hkv * kTileBytes) << (shift - 4));
        const size_t page_bytes = static_cast<size_t>(p.kv_heads * kTileBytes) << (shift - 4);
        // lane 2 i + a: the page of tile a of these 32 keys, in the window's step i
        int page = -1, window = 0;
        auto find_pages = [&](int t) {
            window = t;
            const int key = first_key + (t + (lane >> 1)) * kKeys + 32 * w + 16 * (lane & 1);
            page = key < tile.len && t + (lane >> 1) < steps ? own_pages[key >> shift] : -1;
        };
        uint32_t bad = 0;                                             // two bits a step, the latest loaded lowest
        auto load = [&](int t) {
            bad <<= 2;
            if (t >= steps) return;
            const int slot = t % S::kSlots, key = first_key + t * kKeys + 32 * w;
            const int page_a = __shfl_sync(0xffffffffu, page, 2 * (t - window)), page_b = __shfl_sync(0xffffffffu, page, 2 * (t - window) + 1);
            const bool ask_a = key < tile.len, ask_b = key + 16 < tile.len;
            const bool a = static_cast<unsigned>(page_a) < static_cast<unsigned>(p.n_pages), b = static_cast<unsigned>(page_b) < static_cast<unsigned>(p.n_pages);
            if (ask_a != a || ask_b != b) {
                bad |= (ask_a && !a ? 1u : 0u) | (ask_b && !b ? 2u : 0u);
                if (lane == 0 && p.err) atomicOr(p.err, ERR_BAD_SHAPE);
            }
            if (part == 0) {
                if (!wait_all(&bars->raw_empty[w][slot], (static_cast<uint32_t>(t / S::kSlots) & 1u) ^ 1u, abort_flag)) { failed = true; return; }
                if (elect_one()) {                    // one copy where both tiles are neighbours in a page
                    uint64_t* const full = &bars->raw_full[w][slot];
                    uint8_t* const to = ring + slot * S::kRawBytes;
                    const int in_a = (key & in_page) >> 4, in_b = ((key + 16) & in_page) >> 4;
                    bar_expect_tx(full, (a ? kTileBytes : 0u) + (b ? kTileBytes : 0u));
                    const bool both = a && b && in_b == in_a + 1;
                    if (a) bulk_load(to, head_pages + page_a * page_bytes + in_a * kTileBytes, both ? 2 * kTileBytes : kTileBytes, full);
                    if (b && !both) bulk_load(to + kTileBytes, head_pages + page_b * page_bytes + in_b * kTileBytes, kTileBytes, full);
                }
                __syncwarp();
            }
            if (t + 1 - window == 16) find_pages(t + 1);
        };
        find_pages(0);
        int loaded = 0;
        for (; loaded < S::kSlots && !failed; ++loaded) load(loaded);
        for (int t = 0; t < steps && !failed; ++t) {
            const int slot = t % S::kSlots, buffer = t & 1;
            const uint8_t* const raw = ring + slot * S::kRawBytes;
            if (!wait_all(&bars->raw_full[w][slot], static_cast<uint32_t>(t / S::kSlots) & 1u, abort_flag)) { failed = true; break; }
            const int j0 = first_key + t * kKeys + 32 * w, g = lane >> 2, tq = lane & 3;
            const uint32_t gone = (bad >> (2 * (S::kSlots - 1))) & 3u;
            // K: a lane has a quarter of four keys' elements; the stores of eight lanes fall on banks of their own
            {
                const int a = (lane >> 2) & 1;
                const uint8_t* const from = raw + a * kTileBytes;
                uint32_t code[4][kMine], d[4][kMine];     // all of them first: the stores keep what follows behind them
#pragma unroll
                for (int it = 0; it < 4; ++it)
#pragma unroll
                    for (int b = 0; b < kMine; ++b) {
                        const int r = it * 4 + (lane >> 3), block = min(b0 + b, NB - 1);
                        code[it][b] = *reinterpret_cast<const uint32_t*>(from + kv::key_word(NB, r, tq, block));
                        d[it][b] = *reinterpret_cast<const uint16_t*>(from + kv::key_scale(NB, r, block));
                    }
                if (!wait_all(&bars->k_empty, (static_cast<uint32_t>(t) & 1u) ^ 1u, abort_flag)) { failed = true; break; }
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const int row = 32 * w + order_of_key(a, it * 4 + (lane >> 3));
#pragma unroll
                    for (int b = 0; b < kMine; ++b) {
                        const int block = b0 + b;
                        if (NB % 2 == 1 && block >= NB) continue;
                        const uint32_t two = d[it][b] * 0x10001u, upper = two & 0xFFF8FFF8u, lower = hsub2(two, upper);
                        uint32_t x[4];
                        less8(code[it][b], x);
                        const uint32_t at = base_s + S::kKAt + (block >> 1) * S::kKSlab + row * 128 + ((((block & 1) * 4 + tq) ^ (row & 7)) * 16);
                        sts128(at, make_uint4(hmul2(x[0], upper), hmul2(x[1], upper), hmul2(x[2], upper), hmul2(x[3], upper)));
                        sts128(at + S::kKTile, make_uint4(hmul2(x[0], lower), hmul2(x[1], lower), hmul2(x[2], lower), hmul2(x[3], lower)));
                    }
                }
            }
            // K scales of a lane's key.  (Taken from d above, as a bit more each, 1% slower.)
            uint32_t dk[kMine], all = 0;
#pragma unroll
            for (int b = 0; b < kMine; ++b) all |= dk[b] = *reinterpret_cast<const uint16_t*>(raw + (lane >> 4) * kTileBytes + kv::key_scale(NB, lane & 15, min(b0 + b, NB - 1)));
            // V scales: a lane's words of its blocks (its keys' pairs), none for keys that are not there; those of 8192 and more, or not finite
            uint32_t dv[2][2][kMine];
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int left = (gone >> a & 1u) ? 0 : tile.len - (j0 + 16 * a + 8 * h + 2 * tq);
                    const uint32_t keep = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u;
#pragma unroll
                    for (int b = 0; b < kMine; ++b) {
                        dv[a][h][b] = *reinterpret_cast<const uint32_t*>(raw + a * kTileBytes + kv::value_scales_at(NB) + ((h * 4 + tq) * NB + min(b0 + b, NB - 1)) * 4) & keep;
                        all |= dv[a][h][b];
                    }
                }
            StepNotes& notes = bars->notes[t & 3];
            uint32_t large = 0;                       // keys, in the matrices' order, that are more than fp16 holds
            bool special = false;
            if (__any_sync(0xffffffffu, ((all | all >> 16) & 0x4000u) != 0)) {      // scales of two or more: look at each
                uint32_t beyond = 0;
#pragma unroll
                for (int i = 0; i < 4 * kMine; ++i) beyond |= ((dv[i / (2 * kMine)][i / kMine % 2][i % kMine] & 0x70007000u) + 0x10001000u) & 0x80008000u;
#pragma unroll
                for (int b = 0; b < kMine; ++b)
                    if (too_large(dk[b])) large = 1u << order_of_key(lane >> 4, lane & 15);
                special = __any_sync(0xffffffffu, (beyond | large) != 0);
            }
            if (lane == 0) {
                notes.any[wd] = (gone ? 1u : 0u) | (special ? 2u : 0u);
                if (part == 0) notes.hidden[w] = (gone & 1u ? 0x0F0F0F0Fu : 0u) | (gone & 2u ? 0xF0F0F0F0u : 0u);
            }
            if (special) {
                if (lane < kMine && b0 + lane < NB) notes.poison[w][b0 + lane] = 0;
                if (lane == 0) notes.large[wd] = 0;
                __syncwarp();
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int b = 0; b < kMine; ++b)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                if ((dv[a][h][b] >> (16 * e) & 0x7000u) == 0x7000u) {
                                    const uint32_t key = 1u << (8 * tq + 4 * a + 2 * h + e);
                                    if (too_large(dv[a][h][b] >> (16 * e))) large |= key;
                                    else if (g == 0 && b0 + b < NB) atomicOr(&notes.poison[w][b0 + b], key);
                                    dv[a][h][b] &= e ? 0xFFFFu : 0xFFFF0000u;
                                }
                if (large) atomicOr(&notes.large[wd], large);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) bar_arrive(&bars->k_full[buffer]);

            uint32_t code[2][2][kMine];
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int b = 0; b < kMine; ++b)
                        code[a][h][b] = *reinterpret_cast<const uint32_t*>(raw + a * kTileBytes + kv::values_at(NB) + ((h * 32 + lane) * NB + min(b0 + b, NB - 1)) * 4);
            if (!wait_all(&bars->v_empty[buffer], (static_cast<uint32_t>(t >> 1) & 1u) ^ 1u, abort_flag)) { failed = true; break; }
#pragma unroll
            for (int b = 0; b < kMine; ++b) {
                if (NB % 2 == 1 && b0 + b >= NB) continue;
                uint32_t x[2][2][4];
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        less8(code[a][h][b], x[a][h]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[a][h][e] = hmul2(x[a][h][e], dv[a][h][b]);
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = 32 * (b0 + b) + 4 * g + e;
                    sts128(base_s + S::kVAt + buffer * S::kVTile + (w >> 1) * S::kVSlab + row * 128 + ((((w & 1) * 4 + tq) ^ (row & 7)) * 16),
                           make_uint4(x[0][0][e], x[0][1][e], x[1][0][e], x[1][1][e]));
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                bar_arrive(&bars->v_full[buffer]);
                bar_arrive(&bars->raw_empty[w][slot]);
            }
            load(loaded++);
        }
        if (part == 0 && (failed || *abort_flag)) {        // copies in flight land before the shared memory is released
            for (int t = max(0, loaded - S::kSlots); t < loaded && t < steps; ++t)
                bar_wait(&bars->raw_full[w][t % S::kSlots], static_cast<uint32_t>(t / S::kSlots) & 1u, nullptr, 1000000LL);
        }
    }
    if (failed) {
        *abort_flag = 1;
        if (p.err) atomicOr(p.err, ERR_WAIT_TIMEOUT);
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kSoftWarps) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, kTmemCols);
    }
    if (bars->again && !*abort_flag) rows_again<T, NB, BOTH>(p);
}

// Rows whose keys were cut into chunks: a warp per row.
template <typename T, int NB>
__global__ void __launch_bounds__(256) attention_paged_chunks_kernel(const AttnPagedArgs p, int chunks) {
    constexpr int D = 32 * NB;
    dependent::let_next_begin();                  // (what comes next waits for this one before it touches what is written here)
    dependent::wait_for_earlier();
    const int lane = threadIdx.x & 31, G = p.per_kv, tile_no = p.by_kv_heads(static_cast<int>(blockIdx.x)), hkv = static_cast<int>(blockIdx.x) - tile_no * p.kv_heads;
    Tile tile;
    if (!find_tile(p, tile_no, &tile)) return;
    const int lr = blockIdx.y * 8 + (threadIdx.x >> 5), r = tile.row0 + lr;
    if (r >= tile.nq * G) return;
    const int i = p.by_per_kv(r), h = hkv * G + (r - i * G), token = tile.q0 + i;
    const float* part = p.parts + (static_cast<size_t>(token) * p.q_heads + h) * chunks * (D + 2);
    float m = -INFINITY, l = 0.f, o[NB];
    for (int c = 0; c < chunks; ++c) m = fmaxf(m, part[c * (D + 2)]);
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = 0.f;
    for (int c = 0; c < chunks; ++c, part += D + 2) {
        const float mc = part[0], w = mc > -INFINITY ? exp2_of(mc - m) : 0.f;
        if (part[1] == 0.f) continue;             // no key of it was seen; else its NaN count whatever its weight
        l = fmaf(part[1], w, l);
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] = fmaf(part[2 + 32 * b + lane], w, o[b]);
    }
    T* dst = static_cast<T*>(p.O) + token * p.o_token + h * p.o_head;
#pragma unroll
    for (int b = 0; b < NB; ++b) dst[32 * b + lane] = io::from_f<T>(l == 0.f ? 0.f : o[b] / l);
    if (lane == 0 && p.LSE) p.LSE[static_cast<size_t>(token) * p.q_heads + h] = l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
}

template <typename T, int NB>
cudaError_t launch_as(const AttnPagedArgs& p, int tiles, int chunks, const LaunchEnv& env, cudaStream_t stream) {
    const unsigned x = static_cast<unsigned>(tiles) * p.kv_heads;
    const cudaError_t e = p.tile_rows > kRows ? dependent::launch(attention_paged_prompt_kernel<T, NB, true>, dim3(x, chunks), kThreads, TcShape<NB, true>::kSmem, stream, env.pdl, p)
                                              : dependent::launch(attention_paged_prompt_kernel<T, NB, false>, dim3(x, chunks), kThreads, TcShape<NB, false>::kSmem, stream, env.pdl, p);
    return e != cudaSuccess || chunks == 1 ? e : dependent::launch(attention_paged_chunks_kernel<T, NB>, dim3(x, p.tile_rows / 8), 256, 0, stream, true, p, chunks);
}
template <typename T>
cudaError_t launch_type(const AttnPagedArgs& p, int tiles, int chunks, const LaunchEnv& env, cudaStream_t stream) {
    switch (p.head_dim) {
        case 32: return launch_as<T, 1>(p, tiles, chunks, env, stream);
        case 64: return launch_as<T, 2>(p, tiles, chunks, env, stream);
        case 96: return launch_as<T, 3>(p, tiles, chunks, env, stream);
        default: return launch_as<T, 4>(p, tiles, chunks, env, stream);
    }
}
template <typename T, int NB>
cudaError_t init_as() {
    const cudaError_t e = cudaFuncSetAttribute(attention_paged_prompt_kernel<T, NB, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<NB, false>::kSmem);
    return e != cudaSuccess ? e : cudaFuncSetAttribute(attention_paged_prompt_kernel<T, NB, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<NB, true>::kSmem);
}

}  // namespace

cudaError_t init_attention_paged_prompt_kernels() {
    for (cudaError_t e : {init_as<__half, 1>(), init_as<__half, 2>(), init_as<__half, 3>(), init_as<__half, 4>(), init_as<__nv_bfloat16, 1>(), init_as<__nv_bfloat16, 2>(),
                          init_as<__nv_bfloat16, 3>(), init_as<__nv_bfloat16, 4>()})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}

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
    return p.dtype == IO_BF16 ? launch_type<__nv_bfloat16>(p, tiles, chunks, env, stream) : launch_type<__half>(p, tiles, chunks, env, stream);
}

}  // namespace tcb
