// Attention over the paged 4-bit cache (layout: kv_cache.cuh): for every query row
//
//   O = sum_j p_j V_j / sum_j p_j,   p_j = exp(scale Q . K_j),   LSE = log sum_j p_j
//
// over the keys j of the row's sequence that it sees, K and V being (code - 8) * scale.  The last of a sequence's queries is
// at its last key.  A row that sees no key gives zeros and a log-sum-exp of minus infinity.
//
// attention_paged_kernel: single tokens and few.  The work is a list of items - a sequence, a K/V head, 8 or 16 of its
// (query, head) rows, head fastest - each as many units as it has steps of 64 keys, and one more.  One CTA per SM; every warp takes an equal
// run of the units wherever items end (lengths lie on the device, so each CTA adds them up for itself), and goes through it alone, with a
// ring of bulk copies of its own: a tile is one run of bytes in memory.
//
//   * Keys are the rows of the matrices, queries their columns (mma.sync m16n8k16: S^T = K Q^T, O^T = V^T P^T).  A lane's
//     words of a tile are two 16-byte loads for each operand (head_dim 128), without bank conflicts, for codes are stored in fragment order.
//   * Scores are exact products summed in fp32: a code under the mask 0x000F000F or 0x00F000F0 is a subnormal fp16
//     number, c 2^-24 or c 2^-20, as it stands.  The queries carry the factor 2^-4 of the second kind (each row scaled by a power of two, so
//     that neither end of fp16 is near), and minus eight times a block's sum of queries is what its products are added to; then the block's
//     scale of each key, in fp32.
//   * Softmax as usual: running maximum and sum, in base 2.  A probability is carried 2^14 times as large in two fp16 numbers
//     (22 bits), goes from the result's layout to the operand's by movmatrix, and is multiplied by the value's scale there, for each block of 32
//     elements.  The weight p d is rounded once, to fp16: at random 2^-12.8 of a row's result, less than the result's own 2^-12.2 (carrying what
//     is left of it in a second matrix took 9% more time).  For bfloat16 results, rounded to 2^-9.8, a probability is one fp16 number
//     and its weight rounded twice.  Codes of V are (1024 + c) - 1032, or sixteen times that for odd elements, whose sums are divided by 16 at the end.  Scales of two or more (values above 16) are
//     divided by a power of two that a row keeps for all it has seen, so that products stay below 2^15.
//   * An item's pieces: those of one CTA's warps are merged through shared memory when its warps are done; a CTA that has an item's
//     beginning but not its end hands its sums over through L2 (handover.cuh) to the CTA that has the end, which started later and
//     merges them all.  The order of sums depends on sizes alone.
//
// What bounds it: instructions of three warps a scheduler (eight rows: 168 registers, 12 warps a CTA).  64 keys of one head of 128 elements
// cost a scheduler 1700 clk: for every 16 keys 16 matrix products of 8 clk, and about 300 of packing and unpacking beside them; they issue in
// 52% of all cycles.  Measured: 64 sequences of up to 8192 keys, 32 heads on 8, fp16: 77.9 us, 4.3 TB/s of pages;
// 100003 keys, 64 heads on 8: 36.6 us, 3.1 TB/s; 8 sequences of up to 4096, 32 heads on 32, bf16: 26.6 us.  Of the first about 8 us go by
// before the first products (lengths 1.5, the run 1.2, page table 1.2, then 110 KB into each SM) and 5 to 12 after the last (pieces; an
// SM whose items are short has many).  Slower: steps of 32 keys (87.5, 39.2, 29.7 us), the zero point of V as a product with ones
// (1 us), a second matrix for what a weight's rounding leaves (9%), items merged one after the other (4 us).
#include "attention_math.cuh"
#include "dependent_launch.cuh"
#include "handover.cuh"
#include "io_types.cuh"
#include "kernels.h"
#include "kv_cache.cuh"
#include "sm100_prims.cuh"

namespace tcb {
namespace {

using namespace sm100;
using attn::add2;
using attn::exp2_of;
using attn::fma2;
using attn::pack_h2;
using io::from_f;
using io::to_f;

constexpr int kTiles = 4, kStep = 16 * kTiles;      // tiles and keys of a unit
constexpr float kCarry = 14.0f;              // probabilities are 2^14 times as large
constexpr int kMaxSeqs = 256;                // of a launch
constexpr int kItemUnits = 1;                // what an item costs beside its steps
// Fewer CTAs than SMs have work where units are so few.  One sequence of 200 / 611 / 1100 keys, eight K/V heads: 8 units 10.4 / 11.1 / 11.6 us,
// 12 units 11.5 / 10.2 / 13.2, 16 units 14.2 / 14.9 / 16.0.
constexpr int kUnitsPerCta = 8;


// Per sequence, worked out by every CTA.
struct SeqInfo { int len, q0, nq; };

template <int NB, int NQ> struct Shape {
    static constexpr int D = 32 * NB, kRows = 8 * NQ;
    static constexpr int kWarps = NQ == 1 ? 12 : 8, kThreads = kWarps * 32;
    static constexpr int kSlots = 2;
    static constexpr int kSlotBytes = kTiles * kv::tile_bytes(NB);
    static constexpr int kStride = D + 4;                                     // floats between rows of a piece
    static constexpr int kPiece = kRows * kStride;                            // floats of a piece's sums
    static constexpr int kRingAt = 0;
    static constexpr int kCumAt = kWarps * kSlots * kSlotBytes;
    static constexpr int kSeqAt = kCumAt + (kMaxSeqs + 1) * 8;
    static constexpr int kBarAt = (kSeqAt + kMaxSeqs * 12 + 7) / 8 * 8;
    static constexpr int kNoteAt = kBarAt + kWarps * kSlots * 8;              // what each warp's two pieces are
    static constexpr int kSumAt = kNoteAt + 2 * kWarps * 24;
    static constexpr int kStatAt = kSumAt + kWarps * 8;                       // of each piece: maximum and sum of each row
    static constexpr int kAbortAt = kStatAt + 2 * kWarps * kRows * 8;
    static constexpr int kSmem = kAbortAt + 16;
    static constexpr int kStateWords = kRows * D + 2 * kRows;
    static constexpr size_t kStateBytes = kStateWords * 4, kPieceBytes = kWarps * kPiece * 4;      // of a CTA: what it hands over; its warps' pieces
    static_assert(kStateWords % 4 == 0 && kPiece % 4 == 0, "");
    static_assert(kSlots * kSlotBytes >= kPiece * 4, "a warp's last piece goes into its ring");
    static_assert(kSmem <= 227 * 1024, "");
};

template <int N> struct Const { static constexpr int value = N; };
struct PieceNote { long long begin, end; int seq, sub; };      // the item's units; begin < 0: no piece

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same into other registers.
__device__ __forceinline__ void mma16816_to(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
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
// (x & mask) | one, the fp16 number 1024: one instruction (the compiler makes two of it).
__device__ __forceinline__ uint32_t onto_1024(uint32_t x, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(0x64006400u));
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
    if constexpr (N % 2 == 0) {
        uint32_t w[N / 2];
        words<N / 2>(p, w);
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = __half2float(reinterpret_cast<const __half*>(p)[i]);
    }
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
    return p.first_seen(q.len - q.nq) / kStep * kStep;
}
__device__ __forceinline__ int steps_of(const AttnPagedArgs& p, const SeqInfo& q) { return (q.len - first_key(p, q) + kStep - 1) / kStep; }

template <typename T, int NB, int NQ>
__global__ void __launch_bounds__(Shape<NB, NQ>::kThreads, 1) attention_paged_kernel(const AttnPagedArgs p) {
    using S = Shape<NB, NQ>;
    constexpr bool kTwo = !std::is_same<T, __nv_bfloat16>::value;      // weights before they are rounded: 22 bits, or 11
    constexpr int D = S::D, kRows = S::kRows, kWarps = S::kWarps, kThreads = S::kThreads, kSlots = S::kSlots, kTileBytes = kv::tile_bytes(NB);
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, t = lane & 3;
    long long* const cum = reinterpret_cast<long long*>(smem + S::kCumAt);
    SeqInfo* const seqs = reinterpret_cast<SeqInfo*>(smem + S::kSeqAt);
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + S::kBarAt) + warp * kSlots;
    PieceNote* const notes = reinterpret_cast<PieceNote*>(smem + S::kNoteAt);
    long long* const sums = reinterpret_cast<long long*>(smem + S::kSumAt);
    float2* const stats = reinterpret_cast<float2*>(smem + S::kStatAt);
    volatile int* const abort_flag = reinterpret_cast<volatile int*>(smem + S::kAbortAt);
    const int G = p.per_kv;
    // Beside a call's prompts: those have waited for what was before them, and this kernel is not done before they are.
    struct Beside {
        int on;
        __device__ ~Beside() { if (on) dependent::wait_for_earlier(); }
    };
    const Beside beside{p.beside};
    if (!p.beside) dependent::wait_for_earlier();
    dependent::let_next_begin();

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
                if (rows <= p.most_rows) n = static_cast<long long>((rows + kRows - 1) / kRows) * p.kv_heads * (kItemUnits + steps_of(p, q));
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
    const bool few = units < 1ll << 31;           // (a division of 64 bits is several hundred clocks)
    auto divide = [&](long long n, int d) { return few ? static_cast<long long>(static_cast<uint32_t>(n) / static_cast<uint32_t>(d)) : n / d; };
    const long long want = (units + kUnitsPerCta - 1) / kUnitsPerCta;
    const int ctas = static_cast<int>(want < gridDim.x ? want : gridDim.x), cta = blockIdx.x;
    if (cta >= ctas) return;
    const long long share = divide(units, ctas), longer = units - share * ctas;      // the first ones have one more
    auto seq_of = [&](long long u) {              // the sequence that unit u belongs to
        int lo = 0, hi = p.n_here;
        while (lo + 1 < hi) {
            const int mid = (lo + hi) / 2;
            if (cum[mid] <= u) lo = mid; else hi = mid;
        }
        return lo;
    };
    // Nowhere to hand sums over: runs of whole items.
    auto whole_items = [&](long long u) {
        if (p.states || u >= units) return u;
        const int s = seq_of(u), n = kItemUnits + steps_of(p, seqs[s]);
        return cum[s] + divide(u - cum[s], n) * n;
    };
    auto cut = [&](int c) { return whole_items(share * c + min(static_cast<long long>(c), longer)); };      // where CTA c's run begins
    const long long c0 = cut(cta), c1 = cut(cta + 1);
    const long long w0 = whole_items(c0 + divide((c1 - c0) * warp, kWarps)), w1 = whole_items(c0 + divide((c1 - c0) * (warp + 1), kWarps));

    uint8_t* const ring = smem + S::kRingAt + warp * kSlots * S::kSlotBytes;
    float* const my_pieces = p.pieces + static_cast<size_t>(cta) * kWarps * S::kPiece;
    bool failed = false;

    // Items in order, each with the steps of it in this warp's run; the loader runs ahead of the arithmetic.
    struct At { long long begin, end; int seq, sub, from, to; };      // units of its steps, and which of them are ours
    auto set_item = [&](At& a, long long begin) {
        const int steps = steps_of(p, seqs[a.seq]);
        a.begin = begin;
        a.end = begin + steps;
        a.from = w0 > begin ? static_cast<int>(min(w0, a.end) - begin) : 0;
        a.to = w1 < a.end ? static_cast<int>(max(w1, begin) - begin) : steps;
    };
    auto next_item = [&](At& a) {                 // false behind the run
        if (a.end >= w1) return false;
        ++a.sub;
        if (a.end >= cum[a.seq + 1]) {
            do ++a.seq; while (cum[a.seq + 1] <= a.end);
            a.sub = 0;
        }
        set_item(a, a.end + kItemUnits);
        return a.begin - kItemUnits < w1;
    };
    At here;
    here.seq = seq_of(w0 < units ? w0 : 0);
    {
        const int n = kItemUnits + steps_of(p, seqs[here.seq]);
        here.sub = static_cast<int>(divide(max(w0 - cum[here.seq], 0ll), n));
        set_item(here, cum[here.seq] + static_cast<long long>(here.sub) * n + kItemUnits);
    }

    // The loader: the first lanes copy a tile each.  Every lane has the page of one of 32 tiles of the item, asked for a unit before
    // the first of them is needed (-1: behind the sequence's end).
    At ahead = here;
    bool more = w0 < w1;
    int at_step = 0, key = 0, len = 0, page = -1, in_window = 0;
    const int* own_pages = nullptr;
    const uint8_t* head_pages = nullptr;          // the head's part of page 0
    const int shift = p.page_shift, in_page = (1 << shift) - 1;
    const size_t page_bytes = static_cast<size_t>(p.kv_heads * kTileBytes) << (shift - 4);
    uint32_t bad = 0;                             // kTiles bits a unit, the latest loaded lowest: tiles whose page does not exist
    auto find_pages = [&]() {
        in_window = 0;
        page = -1;
        if (key + 16 * lane < len) page = own_pages[(key + 16 * lane) >> shift];
    };
    auto find_item = [&]() {                      // the first from `ahead` on with a step of ours
        while (more && ahead.from >= ahead.to) more = next_item(ahead);
        if (!more) return;
        const SeqInfo q = seqs[ahead.seq];
        at_step = ahead.from;
        len = q.len;
        key = first_key(p, q) + at_step * kStep;
        own_pages = p.page_table + static_cast<size_t>(p.seq0 + ahead.seq) * p.max_pages;
        head_pages = p.pages + (static_cast<size_t>(ahead.sub - p.by_kv_heads(ahead.sub) * p.kv_heads) * kTileBytes << (shift - 4));
        find_pages();
    };
    auto load = [&](int slot) {                   // and on to the next unit
        bad <<= kTiles;
        if (!more) return;
        // (the copies of one lane: those of several lanes are issued one after the other, with the loop around them)
        const int tiles = max(min(kTiles, (len - key + 15) >> 4), 0), run = min(kTiles, 1 << (shift - 4));      // a run of tiles is in one page
        uint32_t good = 0;
        int at[kTiles];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            at[i] = __shfl_sync(0xffffffffu, page, in_window + i);
            if (static_cast<unsigned>(at[i]) < static_cast<unsigned>(p.n_pages)) good |= 1u << i;
        }
        if (good != (1u << tiles) - 1u) {
            bad |= ((1u << tiles) - 1u) & ~good;
            if (tiles > 0 && lane == 0 && p.err) atomicOr(p.err, ERR_BAD_SHAPE);
        }
        if (elect_one()) {
            bar_expect_tx(&bars[slot], static_cast<uint32_t>(__popc(good)) * kTileBytes);
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
                if ((i & (run - 1)) == 0 && (good >> i & 1u))
                    bulk_load(ring + slot * S::kSlotBytes + i * kTileBytes, head_pages + at[i] * page_bytes + (((key >> 4) + i) & (in_page >> 4)) * kTileBytes,
                              min(run, tiles - i) * kTileBytes, &bars[slot]);
        }
        __syncwarp();
        key += kStep;
        in_window += kTiles;
        if (++at_step == ahead.to) {
            more = next_item(ahead);
            find_item();
        } else if (in_window == 32) {
            find_pages();
        }
    };

    if (w0 < w1) {
        io::Pack8<T> raw[NQ][NB];                        // queries as they lie in memory: 8 elements of each block
        auto ask_queries = [&](const At& a) {
            const SeqInfo q = seqs[a.seq];
            const int row_tile = p.by_kv_heads(a.sub), head = a.sub - row_tile * p.kv_heads, R = q.nq * G;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int r = min(row_tile * kRows + 8 * n + g, R - 1), i = p.by_per_kv(r);
                const T* src = static_cast<const T*>(p.Q) + (q.q0 + i) * p.q_token + (head * G + (r - i * G)) * p.q_head + 8 * t;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    if (p.q_vec) {
                        asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(raw[n][b].w[0].x), "=r"(raw[n][b].w[0].y), "=r"(raw[n][b].w[0].z), "=r"(raw[n][b].w[0].w) : "l"(src + 32 * b) : "memory");
                    } else {
                        T v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = src[32 * b + e];
                        raw[n][b].w[0] = *reinterpret_cast<const uint4*>(v);
                    }
                }
            }
        };
        // The first ones are asked for ahead of the copies: what comes behind those comes 4 us later.
        bool asked = here.from < here.to;
        if (asked) ask_queries(here);
        find_item();
        load(0);
        bool filled = false;
        int slot = 0;
        uint32_t parity = 0;

        bool inside = true;
        for (; inside && !failed; inside = next_item(here)) {
            // ---- an item, or the part of it in this warp's run ---------------------------------------------
            const SeqInfo q = seqs[here.seq];
            const int row_tile = p.by_kv_heads(here.sub), head = here.sub - row_tile * p.kv_heads, row0 = row_tile * kRows, R = q.nq * G;
            if (here.begin == here.end && here.begin > w0 && row0 < R) {      // nothing to see; its unit is ours
                for (int u = lane; u < min(kRows, R - row0) * (D / 4); u += 32) {
                    const int r = row0 + u / (D / 4), i = p.by_per_kv(r), h = head * G + (r - i * G);
                    store4(static_cast<T*>(p.O) + (q.q0 + i) * p.o_token + h * p.o_head + u % (D / 4) * 4, 0.f, 0.f, 0.f, 0.f, p.o_vec);
                    if (p.LSE && u % (D / 4) == 0) p.LSE[static_cast<size_t>(q.q0 + i) * p.q_heads + h] = -INFINITY;
                }
            }
            if (here.from >= here.to) continue;
            const int key0 = first_key(p, q), s_begin = here.from, s_end = here.to;
            const PieceNote note = {here.begin, here.end, here.seq, here.sub};
            const bool ends = note.begin + s_end == note.end, whole = s_begin == 0 && ends;
            if (!asked) ask_queries(here);
            asked = false;
            uint32_t qf[NQ][NB][4];               // second operand: [block][MMA 0, its halves 2^-4; MMA 1, ..]
            float zero[NQ][NB][4], f[NQ][2];      // what a block's products are added to; score -> base-2 exponent
            int hi[NQ][2], lo[NQ][2];             // keys that the rows of this lane's columns see
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const int r = row0 + 8 * n + g;
                float v[NB][8], most = 0.f;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    io::unpack8<T>(raw[n][b], v[b]);
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
                    for (int e = 0; e < 4; ++e) zero[n][b][e] = __shfl_sync(0xffffffffu, sum, (2 * t + (e & 1)) * 4 + (e >> 1));      // (from other lanes: registers of their own)
                }
                const float back = down * 16777216.0f * p.scale * 1.4426950408889634f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    f[n][e] = fmaxf(__shfl_sync(0xffffffffu, back, (2 * t + e) * 4), 1.17549435e-38f);      // minus infinity times it is that
                    const int pos = q.len - q.nq + p.by_per_kv(min(row0 + 8 * n + 2 * t + e, R - 1));
                    hi[n][e] = p.causal ? min(q.len, pos + 1) : q.len;
                    lo[n][e] = p.first_seen(pos);
                }
            }
            if (!filled) {                        // the ring's other part is asked for when the first queries are there
                filled = true;
#pragma unroll
                for (int i = 1; i < kSlots; ++i) load(i);
            }
            const int hi_all = p.causal ? min(q.len, q.len - q.nq + p.by_per_kv(row0) + 1) : q.len;
            const int lo_all = p.first_seen(q.len - q.nq + p.by_per_kv(min(row0 + kRows, R) - 1));

            float o[NQ][NB][2][4], m[NQ][2], l[NQ][2];
            uint32_t shrink[NQ];                  // values' scales are divided by 2^shrink for row 8 n + g
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                shrink[n] = 0;
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
                const uint32_t gone = (bad >> (kTiles * (kSlots - 1))) & ((1u << kTiles) - 1u);
                const bool masked = j0 + kStep > hi_all || j0 < lo_all || gone != 0;

                float s[NQ][kTiles][4];           // [tile]: key g + 8 (e / 2), row 2 t + e % 2
#pragma unroll
                for (int k = 0; k < kTiles; ++k) {
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
                            float c[4];
                            mma16816_to(c, ka[b] & 0x000F000Fu, kb[b] & 0x000F000Fu, ka[b] & 0x00F000F0u, kb[b] & 0x00F000F0u, qf[n][b][0], qf[n][b][1], zero[n][b]);
                            mma16816(c, ka8 & 0x000F000Fu, kb8 & 0x000F000Fu, ka8 & 0x00F000F0u, kb8 & 0x00F000F0u, qf[n][b][2], qf[n][b][3]);
                            s[n][k][0] = fmaf(da[b], c[0], s[n][k][0]);
                            s[n][k][1] = fmaf(da[b], c[1], s[n][k][1]);
                            s[n][k][2] = fmaf(db[b], c[2], s[n][k][2]);
                            s[n][k][3] = fmaf(db[b], c[3], s[n][k][3]);
                        }
                    }
                }
                uint32_t ph[NQ][kTiles][2], pl[NQ][kTiles][2];
                bool grown = false;
                float m_new[NQ][2];
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < kTiles; ++k)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int j = j0 + 16 * k + g + 8 * (e >> 1);
                                s[n][k][e] = j < hi[n][e & 1] && j >= lo[n][e & 1] && !(gone >> k & 1u) ? s[n][k][e] : -INFINITY;
                            }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(s[n][0][e], s[n][0][2 + e]);
#pragma unroll
                        for (int k = 1; k < kTiles; ++k) mx = fmaxf(mx, fmaxf(s[n][k][e], s[n][k][2 + e]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        m_new[n][e] = fmaxf(m[n][e], mx * f[n][e]);
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
                    for (int k = 0; k < kTiles; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float a = s[n][k][2 * h], c = s[n][k][2 * h + 1];
                            fma2(a, c, f[n][0], f[n][1], -ref[0], -ref[1]);
                            a = exp2_of(a);
                            c = exp2_of(c);
                            add2(l[n][0], l[n][1], a, c);
                            const uint32_t top = pack_h2(a, c);
                            ph[n][k][h] = transpose_8x8(top);
                            if constexpr (kTwo) {
                                const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&top));
                                add2(a, c, -back.x, -back.y);
                                pl[n][k][h] = transpose_8x8(pack_h2(a, c));
                            }
                        }
                }
#pragma unroll
                for (int k = 0; k < kTiles; ++k) {
                    const uint8_t* tile = buf + k * kTileBytes;
                    uint32_t va[NB], vb[NB], da[NB], db[NB];
                    words<NB>(tile + kv::values_at(NB) + lane * NB * 4, va);
                    words<NB>(tile + kv::values_at(NB) + (32 + lane) * NB * 4, vb);
                    words<NB>(tile + kv::value_scales_at(NB) + t * NB * 4, da);
                    words<NB>(tile + kv::value_scales_at(NB) + (4 + t) * NB * 4, db);
                    auto product = [&](auto first, auto count) {      // of rows' tiles first .. first + count - 1
                        constexpr int n0 = decltype(first)::value, n1 = n0 + decltype(count)::value;
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            uint32_t w[NQ][2];
#pragma unroll
                            for (int n = n0; n < n1; ++n)
#pragma unroll
                                for (int h = 0; h < 2; ++h) {
                                    const uint32_t d = h == 0 ? da[b] : db[b], pr = ph[n][k][h];
                                    if constexpr (kTwo) w[n][h] = hfma2(pr, d, hmul2(pl[n][k][h], d));
                                    else w[n][h] = hmul2(pr, d);
                                }
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const uint32_t x = va[b] >> (8 * j), y = vb[b] >> (8 * j);
                                const uint32_t a0 = hadd2(onto_1024(x, 0x000F000Fu), 0xE408E408u), a1 = hadd2(onto_1024(x, 0x00F000F0u), 0xE480E480u);
                                const uint32_t a2 = hadd2(onto_1024(y, 0x000F000Fu), 0xE408E408u), a3 = hadd2(onto_1024(y, 0x00F000F0u), 0xE480E480u);
#pragma unroll
                                for (int n = n0; n < n1; ++n) mma16816(o[n][b][j], a0, a1, a2, a3, w[n][0], w[n][1]);
                            }
                        }
                    };
                    uint32_t large = 0;
#pragma unroll
                    for (int b = 0; b < NB; ++b) large |= da[b] | db[b];
                    uint32_t shrunk = 0;
#pragma unroll
                    for (int n = 0; n < NQ; ++n) shrunk |= shrink[n];
                    if (!__any_sync(0xffffffffu, ((large & 0x40004000u) | shrunk) != 0)) {
                        product(Const<0>(), Const<NQ>());
                        continue;
                    }
                    // Scales of two or more, infinities and NaN: a lane's scales are for its row (g), of the keys that the row sees.  Another
                    // key has no part in it, be its scale infinite, and one that is seen has, be its weight zero.
                    auto alone = [&](auto first) {
                        constexpr int n = decltype(first)::value;
                        uint32_t ka[NB], kb[NB];
                        const int h0 = __shfl_sync(0xffffffffu, hi[n][0], g >> 1), h1 = __shfl_sync(0xffffffffu, hi[n][1], g >> 1);
                        const int l0 = __shfl_sync(0xffffffffu, lo[n][0], g >> 1), l1 = __shfl_sync(0xffffffffu, lo[n][1], g >> 1);
                        const int row_hi = (gone >> k & 1u) ? 0 : g & 1 ? h1 : h0, row_lo = g & 1 ? l1 : l0, key = j0 + 16 * k + 2 * t;
                        auto seen = [&](int at) {
                            return (at < row_hi && at >= row_lo ? 0xFFFFu : 0u) | (at + 1 < row_hi && at + 1 >= row_lo ? 0xFFFF0000u : 0u);
                        };
                        const uint32_t sa = seen(key), sb = seen(key + 8);
                        uint32_t top = 15;        // the largest finite exponent among them
#pragma unroll
                        for (int b = 0; b < NB; ++b) {
                            ka[b] = da[b];
                            kb[b] = db[b];
                            da[b] &= sa;
                            db[b] &= sb;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint32_t ex = ((e < 2 ? da[b] : db[b]) >> (16 * (e & 1) + 10)) & 31u;
                                if (ex < 31u) top = max(top, ex);
                            }
                        }
                        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        top = max(max(top, __shfl_xor_sync(0xffffffffu, top, 2)) - 15u, shrink[n]);
                        if (__any_sync(0xffffffffu, top > shrink[n])) {
                            const float less = __uint_as_float((127u - (top - shrink[n])) << 23);
                            shrink[n] = top;
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const float of_row = __shfl_sync(0xffffffffu, less, (2 * t + e) * 4);
#pragma unroll
                                for (int b = 0; b < NB; ++b)
#pragma unroll
                                    for (int j = 0; j < 2; ++j) { o[n][b][j][e] *= of_row; o[n][b][j][2 + e] *= of_row; }
                            }
                        }
                        const float by = __uint_as_float((127u - shrink[n]) << 23);
                        const uint32_t by2 = pack_h2(by, by);
#pragma unroll
                        for (int b = 0; b < NB; ++b) { da[b] = hmul2(da[b], by2); db[b] = hmul2(db[b], by2); }
                        product(first, Const<1>());
#pragma unroll
                        for (int b = 0; b < NB; ++b) { da[b] = ka[b]; db[b] = kb[b]; }
                    };
                    alone(Const<0>());
                    if constexpr (NQ == 2) alone(Const<1>());
                }
                __syncwarp();
                load(slot);
                if (++slot == kSlots) { slot = 0; parity ^= 1u; }
            }
            if (failed) break;

            // ---- its end: the item's result, or a piece --------------------------------------------------------
            // An item that goes on in the next warp's run is this one's last: the ring is done with.
            float* const piece = ends ? my_pieces + warp * S::kPiece : reinterpret_cast<float*>(ring);
            if (!whole && lane == 0) notes[2 * warp + (ends ? 0 : 1)] = note;
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float sum = l[n][e];
                    sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                    sum *= 1.0f / 16384.0f;
                    const float grow = __uint_as_float((127u - 14u + __shfl_sync(0xffffffffu, shrink[n], (2 * t + e) * 4)) << 23);
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
                        if (g == 0) stats[(2 * warp + (ends ? 0 : 1)) * kRows + in] = make_float2(m[n][e], sum);
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            *reinterpret_cast<float4*>(piece + in * S::kStride + 32 * b + 4 * g) =
                                make_float4(o[n][b][0][e] * by, o[n][b][0][2 + e] * (by * 0.0625f), o[n][b][1][e] * by, o[n][b][1][2 + e] * (by * 0.0625f));
                    }
                }
        }
        if (failed) {                             // copies in flight land before the shared memory is released
            *abort_flag = 1;
            for (int i = 0; i < kSlots; ++i) {    // (a slot that nothing was loaded into again has completed the phase before)
                bar_wait(&bars[slot], parity, nullptr, 1000000LL);
                if (++slot == kSlots) { slot = 0; parity ^= 1u; }
            }
        }
    }
    __syncthreads();
    if (*abort_flag) {
        if (tid == 0 && p.err) atomicOr(p.err, ERR_WAIT_TIMEOUT);
        return;
    }

    // ---- pieces of items: a warp has a row, a lane four of its elements and the maximum and sum of one piece --------
    constexpr int kTurns = (kRows + kWarps - 1) / kWarps, kPieces = 2 * kWarps;
    static_assert(kPieces <= 32, "");
    auto piece_at = [&](int k) {
        return (k & 1) ? reinterpret_cast<const float*>(smem + S::kRingAt + (k >> 1) * kSlots * S::kSlotBytes) : my_pieces + (k >> 1) * S::kPiece;
    };
    auto weight = [](float m, float all) { return m > -INFINITY ? exp2_of(m - all) : 0.f; };
    auto most_of = [](float m) {
        for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
        return m;
    };
    auto sum_of = [](float v) {
        for (int x = 16; x > 0; x >>= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
        return v;
    };
    auto add = [](float4& sum, float w, float4 x) {
        sum.x = fmaf(x.x, w, sum.x); sum.y = fmaf(x.y, w, sum.y); sum.z = fmaf(x.z, w, sum.z); sum.w = fmaf(x.w, w, sum.w);
    };
    const bool holds = lane < D / 4;
    auto write = [&](const PieceNote& note, int row, float m, float l, float4 v) {
        const SeqInfo q = seqs[note.seq];
        const int row_tile = p.by_kv_heads(note.sub), head = note.sub - row_tile * p.kv_heads, r = row_tile * kRows + row;
        if (r >= q.nq * G || !holds) return;
        const int i = p.by_per_kv(r), h = head * G + (r - i * G);
        const float by = l == 0.f ? 0.f : 1.0f / l;
        store4(static_cast<T*>(p.O) + (q.q0 + i) * p.o_token + h * p.o_head + 4 * lane, v.x * by, v.y * by, v.z * by, v.w * by, p.o_vec);
        if (p.LSE && lane == 0) p.LSE[static_cast<size_t>(q.q0 + i) * p.q_heads + h] = l == 0.f ? -INFINITY : m * 0.6931471805599453f + logf(l);
    };
    const long long my_begin = lane < kPieces ? notes[lane].begin : -1;
    uint32_t left = __ballot_sync(0xffffffffu, my_begin >= 0);
    bool pending = false;                         // an item that began in a CTA before this one and ends here
    PieceNote late;
    int late_first = 0;
    float late_m[kTurns], late_l[kTurns];
    float4 late_v[kTurns];
    // The last item first: the next CTA may wait for it.  Rows are dealt to the warps in turn, across items.
    for (int dealt = 0; left; dealt = (dealt + kRows) % kWarps) {
        const PieceNote note = notes[31 - __clz(left)];
        const bool mine = my_begin == note.begin;
        const uint32_t group = __ballot_sync(0xffffffffu, mine);
        left &= ~group;
        const bool later = note.end <= c1 && note.begin < c0;
        const int first = warp >= dealt ? warp - dealt : warp - dealt + kWarps;
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
            const int row = u * kWarps + first;
            if (row >= kRows) break;
            const float2 ml = mine ? stats[lane * kRows + row] : make_float2(-INFINITY, 0.f);
            constexpr int kAtOnce = 4;            // pieces that are read before their weights are known
            float4 x[kAtOnce];
            uint32_t g = group;
            auto ask = [&](uint32_t from) {       // (the one in L2 is the last)
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    if (from == 0) break;
                    const int k = 31 - __clz(from);
                    from ^= 1u << k;
                    if (holds) x[i] = *reinterpret_cast<const float4*>(piece_at(k) + row * S::kStride + 4 * lane);
                }
            };
            ask(g);
            const float m = most_of(ml.x), w = weight(ml.x, m), l = sum_of(ml.y * w);
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            while (g) {
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    if (g == 0) break;
                    const int k = 31 - __clz(g);
                    g ^= 1u << k;
                    const float wi = __shfl_sync(0xffffffffu, w, k);
                    if (holds) add(sum, wi, x[i]);
                }
                ask(g);
            }
            if (note.end > c1) {
                uint32_t* dst = p.states + static_cast<size_t>(cta) * S::kStateWords;
                if (lane < 2) handover::store(dst + kRows * D + 2 * row + lane, handover::word_of(lane == 0 ? m : l));
                if (holds) handover::store4(dst + row * D + 4 * lane, make_uint4(handover::word_of(sum.x), handover::word_of(sum.y), handover::word_of(sum.z), handover::word_of(sum.w)));
            } else if (later) {
                late_m[u] = m;
                late_l[u] = l;
                late_v[u] = sum;
            } else {
                write(note, row, m, l, sum);
            }
        }
        if (later) { pending = true; late = note; late_first = first; }
    }
    if (!pending) return;

    // ---- what earlier CTAs have of it, 32 of them at a time: their words say that they are there ---------------------
    int from = static_cast<int>(late.begin < (share + 1) * longer ? divide(late.begin, static_cast<int>(share + 1)) : longer + divide(late.begin - (share + 1) * longer, static_cast<int>(share)));
    constexpr uint32_t kNone = handover::kNothing;
    const long long t0 = clock64();
    bool ok = true;
#pragma unroll
    for (int u = 0; u < kTurns; ++u) {
        const int row = u * kWarps + late_first;
        if (row >= kRows) break;
        float m = late_m[u], l = late_l[u];       // all lanes' alike
        float4 sum = late_v[u];
        for (int base = from; base < cta && ok; base += 32) {
            const int n = min(32, cta - base);
            uint32_t* const theirs = p.states + static_cast<size_t>(base) * S::kStateWords;
            uint32_t* const ml_at = theirs + static_cast<size_t>(lane) * S::kStateWords + kRows * D + 2 * row;
            constexpr int kAtOnce = 8;
            uint4 x[kAtOnce];
            auto ask = [&](int at) {
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                    if (at + i < n && holds) x[i] = handover::load4(theirs + static_cast<size_t>(at + i) * S::kStateWords + row * D + 4 * lane);
            };
            ask(0);
            uint32_t mw = 0xff800000u, lw = 0;
            while (lane < n) {
                mw = handover::load(ml_at);
                lw = handover::load(ml_at + 1);
                if (handover::there(mw) && handover::there(lw)) break;
                if (clock64() - t0 > 2000000000LL) { ok = false; break; }
            }
            if (lane < n) {
                handover::store(ml_at, kNone);
                handover::store(ml_at + 1, kNone);
            }
            ok = __all_sync(0xffffffffu, ok) != 0;
            if (!ok) break;
            const float mi = __uint_as_float(mw), m_new = fmaxf(m, most_of(mi)), keep = weight(m, m_new), w = weight(mi, m_new);
            l = l * keep + sum_of(__uint_as_float(lw) * w);
            m = m_new;
            sum = make_float4(sum.x * keep, sum.y * keep, sum.z * keep, sum.w * keep);
            for (int at = 0; at < n && ok; at += kAtOnce) {
                if (at > 0) ask(at);
                for (;;) {
                    bool all = true;
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)
                        if (at + i < n && holds) all = all && handover::there(x[i]);
                    if (__all_sync(0xffffffffu, all)) break;
                    ok = __all_sync(0xffffffffu, clock64() - t0 <= 2000000000LL) != 0;
                    if (!ok) break;
                    ask(at);
                }
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    if (at + i >= n) continue;
                    const float wi = __shfl_sync(0xffffffffu, w, at + i);
                    if (!holds) continue;
                    handover::store4(theirs + static_cast<size_t>(at + i) * S::kStateWords + row * D + 4 * lane, make_uint4(kNone, kNone, kNone, kNone));
                    add(sum, wi, make_float4(__uint_as_float(x[i].x), __uint_as_float(x[i].y), __uint_as_float(x[i].z), __uint_as_float(x[i].w)));
                }
            }
        }
        if (ok) write(late, row, m, l, sum);
    }
    if (!ok && p.err) atomicOr(p.err, ERR_WAIT_TIMEOUT);      // what has not been taken is emptied with the error
}

template <typename T, int NB, int NQ>
cudaError_t launch_as(const AttnPagedArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    using S = Shape<NB, NQ>;
    return dependent::launch(attention_paged_kernel<T, NB, NQ>, env.sm_count, S::kThreads, S::kSmem, stream, env.pdl || p.beside || p.seq0 > 0, p);
}
template <typename T, int NB>
cudaError_t launch_rows(const AttnPagedArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    return p.max_q * p.per_kv <= 8 ? launch_as<T, NB, 1>(p, env, stream) : launch_as<T, NB, 2>(p, env, stream);
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
cudaError_t launch_type(const AttnPagedArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    switch (p.head_dim) {
        case 32: return launch_rows<T, 1>(p, env, stream);
        case 64: return launch_rows<T, 2>(p, env, stream);
        case 96: return launch_rows<T, 3>(p, env, stream);
        default: return launch_rows<T, 4>(p, env, stream);
    }
}

}  // namespace

cudaError_t init_attention_paged_kernels() {
    for (cudaError_t e : {init_type<__half>(), init_type<__nv_bfloat16>(), init_attention_paged_prompt_kernels()})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}

// Up to how many (query, head) rows on a K/V head a sequence is taken here, 16 at a time, each reading the keys again.  Eight sequences
// of 3000 keys, 32 heads on 8, fp16: 24 and 32 rows 38.2 and 38.4 us, as prompts 42.7 and 43.2; 40 rows 49.3, as a prompt 43.7.  (Two
// sequences of 48 rows would be faster here, 21.3 against 28.0.)
constexpr int kTokenRows = 32;

AttnPagedPlan plan_attention_paged(const AttnPagedArgs& p, int sm_count) {
    AttnPagedPlan plan;
    const int per_kv = p.q_heads / p.kv_heads;
    const bool same = !p.q_start || p.n_seqs == 1;                    // no sequence of few queries beside a prompt
    plan.prompts = static_cast<long long>(p.max_q) * per_kv > kTokenRows;
    plan.tokens = !plan.prompts || !same;
    if (plan.prompts) {
        plan_attention_paged_prompts(p.tokens, p.n_seqs, p.max_q, per_kv, p.kv_heads, static_cast<long long>(p.max_pages) << p.page_shift, sm_count, &plan);
        if (plan.chunks > 1) plan.part_bytes = static_cast<size_t>(p.tokens) * p.q_heads * plan.chunks * (p.head_dim + 2) * sizeof(float);
    }
    if (plan.tokens) {
        const bool one = static_cast<long long>(p.max_q) * per_kv <= 8;
        auto rooms = [&](auto small, auto large) {
            plan.state_bytes = sm_count * (one ? decltype(small)::kStateBytes : decltype(large)::kStateBytes);
            plan.piece_bytes = sm_count * (one ? decltype(small)::kPieceBytes : decltype(large)::kPieceBytes);
        };
        switch (p.head_dim) {
            case 32: rooms(Shape<1, 1>(), Shape<1, 2>()); break;
            case 64: rooms(Shape<2, 1>(), Shape<2, 2>()); break;
            case 96: rooms(Shape<3, 1>(), Shape<3, 2>()); break;
            default: rooms(Shape<4, 1>(), Shape<4, 2>()); break;
        }
    }
    return plan;
}

cudaError_t launch_attention_paged(const AttnPagedArgs& args, const AttnPagedPlan& plan, const LaunchEnv& env, cudaStream_t stream, int* launches, const char** name) {
    AttnPagedArgs p = args;
    const uintptr_t q = reinterpret_cast<uintptr_t>(p.Q) | static_cast<uintptr_t>((p.q_token | p.q_head) * 2);
    const uintptr_t o = reinterpret_cast<uintptr_t>(p.O) | static_cast<uintptr_t>((p.o_token | p.o_head) * 2);
    p.q_vec = (q & 15u) == 0;
    p.o_vec = (o & 7u) == 0;
    p.o_vec16 = (o & 15u) == 0;
    p.per_kv = p.q_heads / p.kv_heads;
    p.by_per_kv.set(p.per_kv);
    p.by_kv_heads.set(p.kv_heads);
    if (plan.prompts) p.most_rows = plan.tokens ? kTokenRows : 0;      // (a single sequence is one there whatever its queries: a step may be padded)
    p.tile_rows = plan.tile_rows;
    *launches = 0;
    cudaError_t e = cudaSuccess;
    if (plan.prompts) {
        const int chunks = p.parts ? plan.chunks : 1;                 // nowhere to leave chunks' results: keys in one piece
        e = launch_attention_paged_prompts(p, plan.tiles, chunks, env, stream);
        *launches += chunks > 1 ? 2 : 1;
        *name = "attention_paged_q4_0_prompt_tcgen05_sm100";
    }
    if (!plan.tokens) return e;
    p.beside = plan.prompts;
    *name = p.max_q * p.per_kv <= 8 ? "attention_paged_q4_0_rows8_sm100" : "attention_paged_q4_0_rows16_sm100";
    for (p.seq0 = 0; p.seq0 < p.n_seqs && e == cudaSuccess; p.seq0 += kMaxSeqs) {
        p.n_here = p.n_seqs - p.seq0 < kMaxSeqs ? p.n_seqs - p.seq0 : kMaxSeqs;
        e = p.dtype == IO_BF16 ? launch_type<__nv_bfloat16>(p, env, stream) : launch_type<__half>(p, env, stream);
        ++*launches;
        p.beside = 0;
    }
    return e;
}

}  // namespace tcb
