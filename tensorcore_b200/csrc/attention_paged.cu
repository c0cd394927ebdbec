// Attention over the paged 4-bit cache (layout: kv_cache.cuh): for every query row
//
//   O = sum_j p_j V_j / sum_j p_j,   p_j = exp(scale Q . K_j),   LSE = log sum_j p_j
//
// over the keys j of the row's sequence that it sees, K and V being (code - 8) * scale.  The last of a sequence's queries is
// at its last key.  A row that sees no key gives zeros and a log-sum-exp of minus infinity.
//
// attention_paged_kernel: single tokens and few.  The work is a list of items - a sequence, a K/V head, 8 or 16 of its
// (query, head) rows, head fastest - each as many units as it has steps of 32 keys.  One CTA per SM; every warp takes an equal run of the
// units wherever items end (lengths lie on the device, so each CTA adds them up for itself), and goes through it alone, with a ring of bulk
// copies of its own: a tile is one run of bytes in memory.
//
//   * Keys are the rows of the matrices, queries their columns (mma.sync m16n8k16: S^T = K Q^T, O^T = V^T P^T).  A lane's
//     words of a tile are two 16-byte loads for each operand (head_dim 128), without bank conflicts, for codes are stored in fragment order.
//   * Scores are exact products summed in fp32: a code under the mask 0x000F000F or 0x00F000F0 is a subnormal fp16
//     number, c 2^-24 or c 2^-20, as it stands.  The queries carry the factor 2^-4 of the second kind (each row scaled by a power of two, so
//     that neither end of fp16 is near), and minus eight times a block's sum of queries is what its products are added to; then the block's
//     scale of each key, in fp32.
//   * Softmax as usual: running maximum and sum, in base 2.  A probability is carried 2^14 times as large in two fp16 numbers
//     (22 bits), goes from the result's layout to the operand's by movmatrix, and is multiplied by the value's scale there, for each block of 32
//     elements, without error: hi = p d rounded, lo = p d - hi by a fused multiply-add.  Codes of V are (1024 + c) - 1032, or
//     sixteen times that for odd elements, whose sums are divided by 16 at the end.  Scales of two or more (values above 16) are
//     divided by a power of two that a warp keeps for all it has seen, so that products stay below 2^15.
//   * An item's pieces: those of one CTA's warps are merged through shared memory when its warps are done; a CTA that has an item's
//     beginning but not its end hands its sums over through L2 (handover.cuh) to the CTA that has the end, which started later and
//     merges them all.  The order of sums depends on sizes alone.
#include "attention_math.cuh"
#include "handover.cuh"
#include "io_types.cuh"
#include "kernels.h"
#include "kv_cache.cuh"
#include "sm100_prims.cuh"

namespace tcb {
namespace {

using namespace sm100;
using attn::pack_h2;
using io::from_f;
using io::to_f;

constexpr int kStep = 32;                    // keys of a unit: two tiles
constexpr float kCarry = 14.0f;              // probabilities are 2^14 times as large
constexpr int kMaxSeqs = 256;                // of a launch

// Per sequence, worked out by every CTA.
struct SeqInfo { int len, q0, nq; };

template <int NB, int NQ> struct Shape {
    static constexpr int D = 32 * NB, kRows = 8 * NQ;
    static constexpr int kWarps = NQ == 1 ? 12 : 8, kThreads = kWarps * 32;
    static constexpr int kSlots = NQ == 1 ? 3 : 4;
    static constexpr int kSlotBytes = 2 * kv::tile_bytes(NB);
    static constexpr int kStride = D + 4;                                     // floats between rows of a piece
    static constexpr int kPiece = kRows * kStride + 2 * kRows;                // floats: sums, then maximum and sum of each row
    static constexpr int kRingAt = 0;
    static constexpr int kFirstAt = kWarps * kSlots * kSlotBytes;
    static constexpr int kCumAt = kFirstAt + kWarps * kPiece * 4;
    static constexpr int kSeqAt = kCumAt + (kMaxSeqs + 1) * 8;
    static constexpr int kBarAt = (kSeqAt + kMaxSeqs * 12 + 7) / 8 * 8;
    static constexpr int kNoteAt = kBarAt + kWarps * kSlots * 8;              // what each warp's two pieces are
    static constexpr int kSumAt = kNoteAt + 2 * kWarps * 24;
    static constexpr int kAbortAt = kSumAt + kWarps * 8;
    static constexpr int kSmem = kAbortAt + 16;
    static constexpr int kStateWords = kRows * D + 2 * kRows;
    static_assert(kSlots * kSlotBytes >= kPiece * 4, "a warp's last piece goes into its ring");
    static_assert(kSmem <= 227 * 1024, "");
};

struct PieceNote { long long begin, end; int seq, sub; };      // the item's units; begin < 0: no piece

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t hadd2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
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
template <int N> __device__ __forceinline__ void halves(const uint8_t* p, float (&f)[N]) {
    uint16_t h[N];
    if constexpr (N == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        h[0] = static_cast<uint16_t>(v.x); h[1] = static_cast<uint16_t>(v.x >> 16); h[2] = static_cast<uint16_t>(v.y); h[3] = static_cast<uint16_t>(v.y >> 16);
    } else if constexpr (N == 2) {
        const uint32_t v = *reinterpret_cast<const uint32_t*>(p);
        h[0] = static_cast<uint16_t>(v); h[1] = static_cast<uint16_t>(v >> 16);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = reinterpret_cast<const uint16_t*>(p)[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = __half2float(__ushort_as_half(h[i]));
}

template <typename T> __device__ __forceinline__ void store4(T* dst, float a, float b, float c, float d, int vec) {
    T v[4] = {from_f<T>(a), from_f<T>(b), from_f<T>(c), from_f<T>(d)};
    if (vec) {
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[i] = v[i];
    }
}

// What of a sequence the call is asked for, and the first key, in whole steps, that any of its queries sees.
__device__ __forceinline__ SeqInfo seq_info(const AttnPagedArgs& p, int s) {
    SeqInfo q;
    if (p.q_start) {
        const int a = p.q_start[p.seq0 + s], b = p.q_start[p.seq0 + s + 1];
        q.q0 = min(max(a, 0), p.tokens);
        q.nq = max(0, min(b, p.tokens) - q.q0);
    } else {
        q.nq = p.tokens / p.n_seqs;
        q.q0 = (p.seq0 + s) * q.nq;
    }
    const long long most = static_cast<long long>(p.max_pages) << p.page_shift;
    const int len = p.seq_lens[p.seq0 + s];
    q.len = len < 0 ? 0 : len > most ? static_cast<int>(most) : len;
    if (len > most && p.err) atomicOr(p.err, ERR_BAD_SHAPE);
    return q;
}
__device__ __forceinline__ int first_key(const AttnPagedArgs& p, const SeqInfo& q) {
    return p.window > 0 ? max(0, min(q.len - q.nq - p.window, q.len)) & ~(kStep - 1) : 0;
}
__device__ __forceinline__ int steps_of(const AttnPagedArgs& p, const SeqInfo& q) { return max(1, (q.len - first_key(p, q) + kStep - 1) / kStep); }

template <typename T, int NB, int NQ>
__global__ void __launch_bounds__(Shape<NB, NQ>::kThreads, 1) attention_paged_kernel(const AttnPagedArgs p) {
    using S = Shape<NB, NQ>;
    constexpr int D = S::D, kRows = S::kRows, kWarps = S::kWarps, kThreads = S::kThreads, kSlots = S::kSlots, kTileBytes = kv::tile_bytes(NB);
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    long long* const cum = reinterpret_cast<long long*>(smem + S::kCumAt);
    SeqInfo* const seqs = reinterpret_cast<SeqInfo*>(smem + S::kSeqAt);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::kBarAt) + warp * kSlots;
    PieceNote* const notes = reinterpret_cast<PieceNote*>(smem + S::kNoteAt);
    long long* const sums = reinterpret_cast<long long*>(smem + S::kSumAt);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + S::kAbortAt);
    const int G = p.per_kv;

    // ---- the list of all units: a running sum over the sequences -----------------------------------------
    if (lane < kSlots) bar_init(&bars[lane], 1);
    if (lane < 2) notes[2 * warp + lane].begin = -1;
    if (tid == 0) *abort_flag = 0;
    long long units;
    {
        long long carry = 0;
        for (int base = 0; base < p.n_here; base += kThreads) {
            const int s = base + tid;
            long long n = 0;
            if (s < p.n_here) {
                const SeqInfo q = seq_info(p, s);
                seqs[s] = q;
                const int rows = q.nq * G;
                n = static_cast<long long>((rows + kRows - 1) / kRows) * p.kv_heads * steps_of(p, q);
            }
            long long sum = n;
#pragma unroll
            for (int x = 1; x < 32; x *= 2) {
                const long long v = __shfl_up_sync(0xffffffffu, sum, x);
                if (lane >= x) sum += v;
            }
            if (lane == 31) sums[warp] = sum;
            __syncthreads();
            long long before = carry;
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) before += sums[w];
                carry += sums[w];
            }
            if (s < p.n_here) cum[s + 1] = before + sum;
            __syncthreads();
        }
        if (tid == 0) cum[0] = 0;
        units = carry;
    }
    fence_barrier_init();
    __syncthreads();

    // ---- this CTA's run of it, and this warp's ------------------------------------------------------------
    const long long want = (units + p.units_per_cta - 1) / p.units_per_cta;
    const int ctas = static_cast<int>(want < gridDim.x ? want : gridDim.x), cta = blockIdx.x;
    if (cta >= ctas) return;
    auto seq_of = [&](long long u) {              // the sequence that unit u belongs to
        int lo = 0, hi = p.n_here;
        while (lo + 1 < hi) {
            const int mid = (lo + hi) / 2;
            if (cum[mid] <= u) lo = mid; else hi = mid;
        }
        return lo;
    };
    auto cut = [&](int c) {                       // where CTA c's run begins
        const long long u = units * c / ctas;
        if (p.states || c == 0 || c == ctas) return u;
        const int s = seq_of(u);                  // nowhere to hand sums over: runs of whole items
        const int n = steps_of(p, seqs[s]);
        return cum[s] + (u - cum[s]) / n * n;
    };
    const long long c0 = cut(cta), c1 = cut(cta + 1);
    const long long w0 = c0 + (c1 - c0) * warp / kWarps, w1 = c0 + (c1 - c0) * (warp + 1) / kWarps;

    uint8_t* const ring = smem + S::kRingAt + warp * kSlots * S::kSlotBytes;
    bool failed = false;

    // Where a unit is: the loader runs ahead of the arithmetic.
    struct At { long long u; int seq, sub, step, steps; };
    auto place = [&](long long u) {
        At a;
        a.u = u;
        a.seq = seq_of(u);
        a.steps = steps_of(p, seqs[a.seq]);
        const long long in = u - cum[a.seq];
        a.sub = static_cast<int>(in / a.steps);
        a.step = static_cast<int>(in - static_cast<long long>(a.sub) * a.steps);
        return a;
    };
    auto advance = [&](At& a) {
        ++a.u;
        if (++a.step < a.steps) return;
        a.step = 0;
        ++a.sub;
        if (a.u < cum[a.seq + 1] || a.u >= w1) return;
        do ++a.seq; while (cum[a.seq + 1] <= a.u);
        a.sub = 0;
        a.steps = steps_of(p, seqs[a.seq]);
    };
    // Lanes 0 and 1: the page of their tile of a unit; -1: behind the sequence's end.
    auto page_of = [&](const At& a) {
        int page = -1;
        if (lane < 2 && a.u < w1) {
            const SeqInfo q = seqs[a.seq];
            const int key = first_key(p, q) + a.step * kStep + 16 * lane;
            if (key < q.len) page = max(-2, p.page_table[static_cast<size_t>(p.seq0 + a.seq) * p.max_pages + (key >> p.page_shift)]);
            if (page == -1 && key < q.len) page = -2;
        }
        return page;
    };
    uint32_t bad = 0;                             // two bits a unit, the latest loaded lowest: tiles whose page does not exist
    auto load = [&](const At& a, int page, int slot) {
        if (a.u < w1) {
            const bool there = page >= 0 && page < p.n_pages;
            const uint32_t good = __ballot_sync(0xffffffffu, there) & 3u, none = __ballot_sync(0xffffffffu, page != -1 && !there) & 3u;
            bad = bad << 2 | none;
            if (none && lane == 0 && p.err) atomicOr(p.err, ERR_BAD_SHAPE);
            if (lane == 0) bar_expect_tx(&bars[slot], static_cast<uint32_t>(__popc(good)) * kTileBytes);
            __syncwarp();
            if (there) {
                const SeqInfo q = seqs[a.seq];
                const int key = first_key(p, q) + a.step * kStep + 16 * lane, head = a.sub % p.kv_heads;
                const size_t tile = ((static_cast<size_t>(page) * p.kv_heads + head) << (p.page_shift - 4)) + ((key & ((1 << p.page_shift) - 1)) >> 4);
                bulk_load(ring + slot * S::kSlotBytes + lane * kTileBytes, p.pages + tile * kTileBytes, kTileBytes, &bars[slot]);
            }
        } else {
            bad <<= 2;
        }
        __syncwarp();
    };

    if (w0 < w1) {
        At ahead = place(w0);
        At here = ahead;
        int page = page_of(ahead);
#pragma unroll
        for (int i = 0; i < kSlots; ++i) {
            load(ahead, page, i);
            advance(ahead);
            page = page_of(ahead);
        }
        int slot = 0;
        uint32_t parity = 0;

        while (here.u < w1 && !failed) {
            // ---- an item, or the part of it in this warp's run ---------------------------------------------
            const SeqInfo q = seqs[here.seq];
            const int head = here.sub % p.kv_heads, row0 = here.sub / p.kv_heads * kRows, R = q.nq * G;
            const int key0 = first_key(p, q), s_begin = here.step, s_end = static_cast<int>(min(static_cast<long long>(here.steps), here.step + (w1 - here.u)));
            const PieceNote note = {here.u - here.step, here.u - here.step + here.steps, here.seq, here.sub};
            const bool whole = s_begin == 0 && s_end == here.steps, first = here.u == w0;
            uint32_t qf[NQ][NB][4];               // second operand: [block][MMA 0, its halves 2^-4; MMA 1, ..]
            float zero[NQ][NB][2], f[NQ][2];      // what a block's products are added to; score -> base-2 exponent
            int hi[NQ][2], lo[NQ][2];             // keys that the rows of this lane's columns see
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int r = row0 + 8 * n + g, i = p.by_per_kv(min(r, R - 1));
                const T* src = static_cast<const T*>(p.Q) + (q.q0 + i) * p.q_token + (head * G + (min(r, R - 1) - i * G)) * p.q_head + 8 * t;
                float v[NB][8], most = 0.f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (p.q_vec) {
                        io::unpack8(io::load8(src + 32 * b), v[b]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[b][e] = to_f<T>(src[32 * b + e]);
                    }
                    if (r >= R) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[b][e] = 0.f;
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[b][e]));
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // largest element to 2^13 .. 2^14; rows of zeros, infinities as they are
                const int ex = min(max(static_cast<int>(__float_as_uint(most) >> 23), 27), 240);
                const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 + 127 - ex) << 23), down = __uint_as_float(static_cast<uint32_t>(ex - 13) << 23);
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    float sum = 0.f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[b][e] *= up;
                        sum += __half2float(__float2half_rn(v[b][e]));
                    }
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        qf[n][b][2 * m] = pack_h2(v[b][2 * m], v[b][4 + 2 * m]);
                        qf[n][b][2 * m + 1] = pack_h2(v[b][1 + 2 * m] * 0.0625f, v[b][5 + 2 * m] * 0.0625f);
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    sum *= -8.0f / 16777216.0f;
#pragma unroll
                    for (int e = 0; e < 2; ++e) zero[n][b][e] = __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4);
                }
                const float back = down * 16777216.0f * p.scale * 1.4426950408889634f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f[n][e] = __shfl_sync(0xffffffffu, back, (2 * t + e) * 4);
                    const int pos = q.len - q.nq + p.by_per_kv(min(row0 + 8 * n + 2 * t + e, R - 1));
                    hi[n][e] = p.causal ? min(q.len, pos + 1) : q.len;
                    lo[n][e] = p.window > 0 ? pos - p.window : 0;
                }
            }
            const int hi_all = p.causal ? min(q.len, q.len - q.nq + p.by_per_kv(row0) + 1) : q.len;
            const int lo_all = p.window > 0 ? q.len - q.nq + p.by_per_kv(min(row0 + kRows, R) - 1) - p.window : 0;

            float o[NQ][NB][2][4], m[NQ][2], l[NQ][2];
            int shrink = 0;                       // values' scales are divided by 2^shrink
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) { m[n][e] = -INFINITY; l[n][e] = 0.f; }
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][b][0][e] = o[n][b][1][e] = 0.f;
            }

            for (int st = s_begin; st < s_end; ++st) {
                if (!wait_all(&bars[slot], parity, abort_flag)) { failed = true; break; }
                const uint8_t* buf = ring + slot * S::kSlotBytes;
                const int j0 = key0 + st * kStep;
                const uint32_t gone = (bad >> (2 * (kSlots - 1))) & 3u;
                const bool masked = j0 + kStep > hi_all || j0 < lo_all || gone != 0;

                float s[NQ][2][4];                // [tile]: key g + 8 (e / 2), row 2 t + e % 2
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint8_t* tile = buf + k * kTileBytes;
                    uint32_t ka[NB], kb[NB];
                    float da[NB], db[NB];
                    words<NB>(tile + (g * 4 + t) * NB * 4, ka);
                    words<NB>(tile + ((g + 8) * 4 + t) * NB * 4, kb);
                    halves<NB>(tile + kv::key_scales_at(NB) + g * NB * 2, da);
                    halves<NB>(tile + kv::key_scales_at(NB) + (g + 8) * NB * 2, db);
#pragma unroll
                    for (int n = 0; n < NQ; ++n) s[n][k][0] = s[n][k][1] = s[n][k][2] = s[n][k][3] = 0.f;
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint32_t ka8 = ka[b] >> 8, kb8 = kb[b] >> 8;
#pragma unroll
                        for (int n = 0; n < NQ; ++n) {
                            float c[4] = {zero[n][b][0], zero[n][b][1], zero[n][b][0], zero[n][b][1]};
                            mma16816(c, ka[b] & 0x000F000Fu, kb[b] & 0x000F000Fu, ka[b] & 0x00F000F0u, kb[b] & 0x00F000F0u, qf[n][b][0], qf[n][b][1]);
                            mma16816(c, ka8 & 0x000F000Fu, kb8 & 0x000F000Fu, ka8 & 0x00F000F0u, kb8 & 0x00F000F0u, qf[n][b][2], qf[n][b][3]);
                            s[n][k][0] = fmaf(da[b], c[0], s[n][k][0]);
                            s[n][k][1] = fmaf(da[b], c[1], s[n][k][1]);
                            s[n][k][2] = fmaf(db[b], c[2], s[n][k][2]);
                            s[n][k][3] = fmaf(db[b], c[3], s[n][k][3]);
                        }
                    }
                }
                uint32_t ph[NQ][2][2], pl[NQ][2][2];
                bool grown = false;
                float m_new[NQ][2];
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[n][k][e] *= f[n][e & 1];
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < 2; ++k)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int j = j0 + 16 * k + g + 8 * (e >> 1);
                                s[n][k][e] = j < hi[n][e & 1] && j >= lo[n][e & 1] && !(gone >> k & 1u) ? s[n][k][e] : -INFINITY;
                            }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(fmaxf(s[n][0][e], s[n][0][2 + e]), fmaxf(s[n][1][e], s[n][1][2 + e]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        m_new[n][e] = fmaxf(m[n][e], mx);
                        grown = grown || m_new[n][e] > m[n][e];
                    }
                }
                if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float keep = m[n][e] > -INFINITY ? exp2_of(m[n][e] - m_new[n][e]) : 0.f;
                            m[n][e] = m_new[n][e];
                            l[n][e] *= keep;
#pragma unroll
                            for (int b = 0; b < NB; ++b)
#pragma unroll
                                for (int j = 0; j < 2; ++j) { o[n][b][j][e] *= keep; o[n][b][j][2 + e] *= keep; }
                        }
                }
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    float ref[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) ref[e] = m[n][e] > -INFINITY ? m[n][e] - kCarry : 0.f;      // a row that sees no key so far keeps zero sums
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float a = exp2_of(s[n][k][2 * h] - ref[0]), c = exp2_of(s[n][k][2 * h + 1] - ref[1]);
                            l[n][0] += a;
                            l[n][1] += c;
                            const uint32_t top = pack_h2(a, c);
                            const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&top));
                            ph[n][k][h] = transpose_8x8(top);
                            pl[n][k][h] = transpose_8x8(pack_h2(a - back.x, c - back.y));
                        }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint8_t* tile = buf + k * kTileBytes;
                    uint32_t va[NB], vb[NB], da[NB], db[NB];
                    words<NB>(tile + kv::values_at(NB) + lane * NB * 4, va);
                    words<NB>(tile + kv::values_at(NB) + (32 + lane) * NB * 4, vb);
                    words<NB>(tile + kv::value_scales_at(NB) + t * NB * 4, da);
                    words<NB>(tile + kv::value_scales_at(NB) + (4 + t) * NB * 4, db);
                    if (masked) {                 // nothing is behind the end, or on a page that does not exist
                        const int left = (gone >> k & 1u) ? 0 : q.len - (j0 + 16 * k + 2 * t);
                        const uint32_t ma = left >= 2 ? 0xFFFFFFFFu : left == 1 ? 0xFFFFu : 0u, mb = left >= 10 ? 0xFFFFFFFFu : left == 9 ? 0xFFFFu : 0u;
#pragma unroll
                        for (int b = 0; b < NB; ++b) { da[b] &= ma; db[b] &= mb; }
                    }
                    uint32_t large = 0;
#pragma unroll
                    for (int b = 0; b < NB; ++b) large |= da[b] | db[b];
                    if (shrink || __any_sync(0xffffffffu, (large & 0x40004000u) != 0)) {
                        // the largest finite exponent in the tile
                        int top = 15;
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int ex = static_cast<int>(((e < 2 ? da[b] : db[b]) >> (16 * (e & 1) + 10)) & 31u);
                                if (ex < 31) top = max(top, ex);
                            }
                        top = __reduce_max_sync(0xffffffffu, top) - 15;
                        if (top > shrink) {
                            const float less = __uint_as_float(static_cast<uint32_t>(127 - (top - shrink)) << 23);
#pragma unroll
                            for (int n = 0; n < NQ; ++n)
#pragma unroll
                                for (int b = 0; b < NB; ++b)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) { o[n][b][0][e] *= less; o[n][b][1][e] *= less; }
                            shrink = top;
                        }
                        const float by = __uint_as_float(static_cast<uint32_t>(127 - shrink) << 23);
                        const uint32_t by2 = pack_h2(by, by);
#pragma unroll
                        for (int b = 0; b < NB; ++b) { da[b] = hmul2(da[b], by2); db[b] = hmul2(db[b], by2); }
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        uint32_t wh[NQ][2], wl[NQ][2];
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t d = h == 0 ? da[b] : db[b], pr = ph[n][k][h];
                                wh[n][h] = hmul2(pr, d);
                                wl[n][h] = hfma2(pl[n][k][h], d, hfma2(pr, d, wh[n][h] ^ 0x80008000u));
                                if (masked) {     // a key that the row does not see has no part in it, be its scale infinite or NaN
                                    const uint32_t some = (pr & 0xFFFFu ? 0xFFFFu : 0u) | (pr >> 16 ? 0xFFFF0000u : 0u);
                                    wh[n][h] &= some;
                                    wl[n][h] &= some;
                                }
                            }
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t x = va[b] >> (8 * j), y = vb[b] >> (8 * j);
                            const uint32_t a0 = hadd2((x & 0x000F000Fu) | 0x64006400u, 0xE408E408u), a1 = hadd2((x & 0x00F000F0u) | 0x64006400u, 0xE480E480u);
                            const uint32_t a2 = hadd2((y & 0x000F000Fu) | 0x64006400u, 0xE408E408u), a3 = hadd2((y & 0x00F000F0u) | 0x64006400u, 0xE480E480u);
#pragma unroll
                            for (int n = 0; n < NQ; ++n) {
                                mma16816(o[n][b][j], a0, a1, a2, a3, wh[n][0], wh[n][1]);
                                mma16816(o[n][b][j], a0, a1, a2, a3, wl[n][0], wl[n][1]);
                            }
                        }
                    }
                }
                __syncwarp();
                load(ahead, page, slot);
                advance(ahead);
                page = page_of(ahead);
                advance(here);
                if (++slot == kSlots) { slot = 0; parity ^= 1u; }
            }
            if (failed) break;

            // ---- its end: the item's result, or a piece --------------------------------------------------------
            const float grow = __uint_as_float(static_cast<uint32_t>(127 + shrink - 14) << 23);
            float* const piece = reinterpret_cast<float*>(first ? smem + S::kFirstAt + warp * S::kPiece * 4 : ring);      // the last one: the ring is done with
            if (!whole && lane == 0) notes[2 * warp + (first ? 0 : 1)] = note;
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float sum = l[n][e];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    sum *= 1.0f / 16384.0f;
                    const int in = 8 * n + 2 * t + e, r = row0 + in;
                    const float by = whole ? sum == 0.f ? 0.f : grow / sum : grow;
                    if (whole && r >= R) continue;
                    if (whole) {
                        const int i = p.by_per_kv(r), h = head * G + (r - i * G);
                        T* dst = static_cast<T*>(p.O) + (q.q0 + i) * p.o_token + h * p.o_head + 4 * g;
                        if (p.LSE && g == 0) p.LSE[static_cast<size_t>(q.q0 + i) * p.q_heads + h] = sum == 0.f ? -INFINITY : m[n][e] * 0.6931471805599453f + logf(sum);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            store4(dst + 32 * b, o[n][b][0][e] * by, o[n][b][0][2 + e] * (by * 0.0625f), o[n][b][1][e] * by, o[n][b][1][2 + e] * (by * 0.0625f), p.o_vec);
                    } else {
                        if (g == 0) { piece[kRows * S::kStride + 2 * in] = m[n][e]; piece[kRows * S::kStride + 2 * in + 1] = sum; }
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            *reinterpret_cast<float4*>(piece + in * S::kStride + 32 * b + 4 * g) =
                                make_float4(o[n][b][0][e] * by, o[n][b][0][2 + e] * (by * 0.0625f), o[n][b][1][e] * by, o[n][b][1][2 + e] * (by * 0.0625f));
                    }
                }
        }
        if (failed) {                             // copies in flight land before the shared memory is released
            *abort_flag = 1;
            for (int i = 0; i < kSlots && here.u + i < min(ahead.u, w1); ++i) {
                bar_wait(&bars[slot], parity, nullptr, 100000000LL);
                if (++slot == kSlots) { slot = 0; parity ^= 1u; }
            }
        }
    }
    __syncthreads();
    if (*abort_flag) {
        if (tid == 0 && p.err) atomicOr(p.err, ERR_WAIT_TIMEOUT);
        return;
    }

    // ---- pieces of items: a thread has four elements of a row -----------------------------------------------
    constexpr int kQuads = kRows * (D / 4), kTurns = (kQuads + kThreads - 1) / kThreads;
    auto piece_at = [&](int k) {
        return reinterpret_cast<const float*>((k & 1) ? smem + S::kRingAt + (k >> 1) * kSlots * S::kSlotBytes : smem + S::kFirstAt + (k >> 1) * S::kPiece * 4);
    };
    auto weight = [](float m, float all) { return m > -INFINITY ? exp2_of(m - all) : 0.f; };
    auto write = [&](const PieceNote& note, int row, int c, float m, float l, float4 v) {
        const SeqInfo q = seqs[note.seq];
        const int head = note.sub % p.kv_heads, r = note.sub / p.kv_heads * kRows + row;
        if (r >= q.nq * G) return;
        const int i = p.by_per_kv(r), h = head * G + (r - i * G);
        const float by = l == 0.f ? 0.f : 1.0f / l;
        store4(static_cast<T*>(p.O) + (q.q0 + i) * p.o_token + h * p.o_head + c, v.x * by, v.y * by, v.z * by, v.w * by, p.o_vec);
        if (p.LSE && c == 0) p.LSE[static_cast<size_t>(q.q0 + i) * p.q_heads + h] = l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
    };
    bool pending = false;                         // an item that began in a CTA before this one and ends here
    PieceNote late;
    float late_m[kTurns], late_l[kTurns];
    float4 late_v[kTurns];
    for (int k = 0; k < 2 * kWarps;) {
        const PieceNote note = notes[k];
        if (note.begin < 0) { ++k; continue; }
        int end = k + 1;
        while (end < 2 * kWarps && (notes[end].begin < 0 || notes[end].begin == note.begin)) ++end;
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
            const int v = u * kThreads + tid, row = v / (D / 4), c = 4 * (v % (D / 4));
            if (v >= kQuads) break;
            float m = -INFINITY, l = 0.f;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i = k; i < end; ++i)
                if (notes[i].begin >= 0) m = fmaxf(m, piece_at(i)[kRows * S::kStride + 2 * row]);
            for (int i = k; i < end; ++i) {
                if (notes[i].begin < 0) continue;
                const float* piece = piece_at(i);
                const float w = weight(piece[kRows * S::kStride + 2 * row], m);
                const float4 x = *reinterpret_cast<const float4*>(piece + row * S::kStride + c);
                l = fmaf(piece[kRows * S::kStride + 2 * row + 1], w, l);
                sum.x = fmaf(x.x, w, sum.x); sum.y = fmaf(x.y, w, sum.y); sum.z = fmaf(x.z, w, sum.z); sum.w = fmaf(x.w, w, sum.w);
            }
            if (note.end > c1) {
                uint32_t* dst = p.states + static_cast<size_t>(cta) * S::kStateWords;
                if (c == 0) {
                    handover::store(dst + kRows * D + 2 * row, handover::word_of(m));
                    handover::store(dst + kRows * D + 2 * row + 1, handover::word_of(l));
                }
                handover::store4(dst + row * D + c, make_uint4(handover::word_of(sum.x), handover::word_of(sum.y), handover::word_of(sum.z), handover::word_of(sum.w)));
            } else if (note.begin < c0) {
                late_m[u] = m;
                late_l[u] = l;
                late_v[u] = sum;
            } else {
                write(note, row, c, m, l, sum);
            }
        }
        if (note.end <= c1 && note.begin < c0) { pending = true; late = note; }
        k = end;
    }
    if (!pending) return;

    // ---- what earlier CTAs have of it: maxima and sums first, then the rows, eight CTAs' at a time --------------
    int from = static_cast<int>(late.begin * ctas / units);
    while (cut(from + 1) <= late.begin) ++from;
    while (cut(from) > late.begin) --from;
    const int n = cta - from;
    float2* const table = reinterpret_cast<float2*>(smem);
    const uint32_t* const theirs = p.states + static_cast<size_t>(from) * S::kStateWords;
    constexpr uint32_t kNone = handover::kNothing;
    const long long t0 = clock64();
    bool ok = true;
    __syncthreads();                              // the pieces have been read
    for (int i = tid; i < kRows * n && ok; i += kThreads) {
        uint32_t* src = p.states + static_cast<size_t>(from + i / kRows) * S::kStateWords + kRows * D + 2 * (i % kRows);
        uint32_t mw, lw;
        for (;;) {
            mw = handover::load(src);
            lw = handover::load(src + 1);
            ok = handover::there(mw) && handover::there(lw);
            if (ok || clock64() - t0 > 2000000000LL) break;
        }
        handover::store(src, kNone);
        handover::store(src + 1, kNone);
        table[(i % kRows) * n + i / kRows] = make_float2(__uint_as_float(mw), __uint_as_float(lw));
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
        const int v = u * kThreads + tid, row = v / (D / 4), c = 4 * (v % (D / 4));
        if (v >= kQuads) break;
        const float2* mine = table + row * n;
        float m = late_m[u], l = 0.f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i = 0; i < n; ++i) m = fmaxf(m, mine[i].x);
        auto add = [&](float mi, float li, float4 x) {
            const float w = weight(mi, m);
            l = fmaf(li, w, l);
            sum.x = fmaf(x.x, w, sum.x); sum.y = fmaf(x.y, w, sum.y); sum.z = fmaf(x.z, w, sum.z); sum.w = fmaf(x.w, w, sum.w);
        };
        constexpr int kAtOnce = 8;
        for (int base = 0; base < n && ok; base += kAtOnce) {
            uint4 x[kAtOnce];
            for (;;) {
                bool all = true;
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                    if (base + i < n) x[i] = handover::load4(theirs + static_cast<size_t>(base + i) * S::kStateWords + row * D + c);
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                    if (base + i < n) all = all && handover::there(x[i]);
                if (all) break;
                ok = clock64() - t0 <= 2000000000LL;
                if (!ok) break;
            }
            if (!ok) break;
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                if (base + i >= n) continue;
                handover::store4(const_cast<uint32_t*>(theirs) + static_cast<size_t>(base + i) * S::kStateWords + row * D + c, make_uint4(kNone, kNone, kNone, kNone));
                add(mine[base + i].x, mine[base + i].y, make_float4(__uint_as_float(x[i].x), __uint_as_float(x[i].y), __uint_as_float(x[i].z), __uint_as_float(x[i].w)));
            }
        }
        add(late_m[u], late_l[u], late_v[u]);
        if (ok) write(late, row, c, m, l, sum);
    }
    if (!ok && p.err) atomicOr(p.err, ERR_WAIT_TIMEOUT);      // what has not been taken is emptied with the error
}

template <typename T, int NB, int NQ>
cudaError_t launch_as(const AttnPagedArgs& p, int sm_count, cudaStream_t stream) {
    using S = Shape<NB, NQ>;
    attention_paged_kernel<T, NB, NQ><<<sm_count, S::kThreads, S::kSmem, stream>>>(p);
    return cudaGetLastError();
}
template <typename T, int NB>
cudaError_t launch_rows(const AttnPagedArgs& p, int sm_count, cudaStream_t stream) {
    return p.max_q * p.per_kv <= 8 ? launch_as<T, NB, 1>(p, sm_count, stream) : launch_as<T, NB, 2>(p, sm_count, stream);
}
template <typename T, int NB, int NQ>
cudaError_t init_as() {
    return cudaFuncSetAttribute(attention_paged_kernel<T, NB, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<NB, NQ>::kSmem);
}
template <typename T> cudaError_t init_type() {
    for (cudaError_t e : {init_as<T, 1, 1>(), init_as<T, 2, 1>(), init_as<T, 3, 1>(), init_as<T, 4, 1>(), init_as<T, 1, 2>(), init_as<T, 2, 2>(), init_as<T, 3, 2>(), init_as<T, 4, 2>()})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}
template <typename T>
cudaError_t launch_type(const AttnPagedArgs& p, int sm_count, cudaStream_t stream) {
    switch (p.head_dim) {
        case 32: return launch_rows<T, 1>(p, sm_count, stream);
        case 64: return launch_rows<T, 2>(p, sm_count, stream);
        case 96: return launch_rows<T, 3>(p, sm_count, stream);
        default: return launch_rows<T, 4>(p, sm_count, stream);
    }
}

}  // namespace

cudaError_t init_attention_paged_kernels() {
    const cudaError_t e = init_type<__half>();
    return e != cudaSuccess ? e : init_type<__nv_bfloat16>();
}

size_t attention_paged_state_bytes(int max_q, int per_kv, int head_dim, int sm_count) {
    const size_t rows = static_cast<long long>(max_q) * per_kv <= 8 ? 8 : 16;
    return static_cast<size_t>(sm_count) * (rows * head_dim + 2 * rows) * 4;
}

cudaError_t launch_attention_paged(const AttnPagedArgs& args, const LaunchEnv& env, cudaStream_t stream, int* launches, const char** name) {
    AttnPagedArgs p = args;
    const uintptr_t q = reinterpret_cast<uintptr_t>(p.Q) | static_cast<uintptr_t>((p.q_token | p.q_head) * 2);
    const uintptr_t o = reinterpret_cast<uintptr_t>(p.O) | static_cast<uintptr_t>((p.o_token | p.o_head) * 2);
    p.q_vec = (q & 15u) == 0;
    p.o_vec = (o & 7u) == 0;
    p.per_kv = p.q_heads / p.kv_heads;
    p.by_per_kv.set(p.per_kv);
    p.units_per_cta = 8;
    *launches = 0;
    *name = p.max_q * p.per_kv <= 8 ? "attention_paged_q4_0_rows8_sm100" : "attention_paged_q4_0_rows16_sm100";
    cudaError_t e = cudaSuccess;
    for (p.seq0 = 0; p.seq0 < p.n_seqs && e == cudaSuccess; p.seq0 += kMaxSeqs) {
        p.n_here = p.n_seqs - p.seq0 < kMaxSeqs ? p.n_seqs - p.seq0 : kMaxSeqs;
        e = p.dtype == IO_BF16 ? launch_type<__nv_bfloat16>(p, env.sm_count, stream) : launch_type<__half>(p, env.sm_count, stream);
        ++*launches;
    }
    return e;
}

}  // namespace tcb
