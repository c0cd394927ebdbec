// Pages and tokens of the paged 4-bit cache moved as they are (layout: kv_cache.cuh), in every layer of a cache at once.
//
// Copies: a head's first tiles of a page are one run of bytes, whole pages are one run altogether.
//
// Compaction: token j of a sequence's list goes from place keep[j] to place to + j <= keep[j].  The list rises, so what chunk c of it is read
// from lies at or above every place that chunks before c are written to: it is enough that a chunk has been read before it is
// written, and one CTA goes through the chunks of a sequence, layer and head in order (a chunk ahead with its reads: those lie above all that is written
// before them).  Keys are runs of a token's own; of the
// values' words a token has every second half (neighbouring tokens share words), so values are moved two places at a time: a
// word's halves from the two tokens that come to lie there.
#include <type_traits>

#include "dependent_launch.cuh"
#include "kernels.h"
#include "kv_cache.cuh"

namespace tcb {
namespace {

constexpr int kCopyThreads = 256, kCopyAtOnce = 4;

__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(const KvCopyArgs p, int tiles, int tile_vecs, int head_vecs) {
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const size_t page_vecs = static_cast<size_t>(head_vecs) * p.kv_heads;
    for (int pair = blockIdx.y; pair < p.pairs; pair += gridDim.y) {
        const int src = p.src[pair], dst = p.dst[pair], count = p.counts ? p.counts[pair] : tiles * 16;
        if (src < 0 || count <= 0) continue;
        if (src >= p.n_pages || dst < 0 || dst >= p.n_pages || count > tiles * 16) {
            if (p.err && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(p.err, ERR_BAD_SHAPE);
            continue;
        }
        if (src == dst) continue;
        const int run = (count + 15) / 16 * tile_vecs;                 // 16-byte pieces of a head
        const bool whole = run == head_vecs;
        const int n = run * p.kv_heads;
        for (int layer = blockIdx.z; layer < p.layers; layer += gridDim.z) {
            uint8_t* const base = p.pages + layer * p.layer_stride;
            const uint4* const from = reinterpret_cast<const uint4*>(base) + src * page_vecs;
            uint4* const to = reinterpret_cast<uint4*>(base) + dst * page_vecs;
            for (int v0 = blockIdx.x * (kCopyThreads * kCopyAtOnce) + threadIdx.x; v0 < n; v0 += gridDim.x * (kCopyThreads * kCopyAtOnce)) {
                uint4 x[kCopyAtOnce];
                int at[kCopyAtOnce];
#pragma unroll
                for (int i = 0; i < kCopyAtOnce; ++i) {
                    const int v = v0 + i * kCopyThreads;
                    at[i] = v;
                    if (!whole && v < n) {
                        const int head = v / run;
                        at[i] = head * head_vecs + (v - head * run);
                    }
                    if (v < n) x[i] = __ldcs(from + at[i]);
                }
#pragma unroll
                for (int i = 0; i < kCopyAtOnce; ++i)
                    if (v0 + i * kCopyThreads < n) to[at[i]] = x[i];
            }
        }
    }
}

// NB words as they lie in memory.
template <int NB> struct alignas(NB == 4 ? 16 : NB == 2 ? 8 : 4) Words { uint32_t w[NB]; };
template <int NB> struct alignas(NB == 4 ? 8 : NB == 2 ? 4 : 2) Halves { uint16_t h[NB]; };

// Where a token is: its tile's number in a layer for head 0, and which of the tile's tokens; tile < 0: nowhere.
struct Spot { int tile, r; };

// Places of some (layer, head)s side by side, `chunk` of each (a multiple of eight), are a chunk.  A thread has quarters of places' key codes, or of the values'
// codes of eight places a run of NB words that two of them share; then the scales.  So eight places' values, and as many keys, are written as runs of 512
// bytes by a warp.  Short lists: a quarter and a run to a thread.  AHEAD, for long ones: keys and values by CTAs of their own (blockIdx.z), two of them an SM, and
// two chunks under way, into a place of their own in shared memory, while the one before them is written.  (8000 tokens of a sequence, 16 layers of 8 heads: a
// thread a place 104 us; one chunk ahead in registers 120; keys and values in one CTA an SM, as here, 86; so 87, and lists of more sequences spread better.)
constexpr int kLongThreads = 384, kShortThreads = 256, kStages = 3, kSpots = 4;
template <int NB> struct Moved { Words<NB> w[2][2], scale[2]; };      // of each unit, and of values of two tokens; of a place's keys in scale[0]'s first half
// Where a thread's are in shared memory.
template <int NB, int THREADS> struct Staged {
    static constexpr int kBytes = (4 * THREADS + THREADS / 2 + THREADS / 4) * 4 * NB;
    Words<NB>* at;
    int tid;
    __device__ __forceinline__ Staged(uint8_t* smem, int stage, int thread) : at(reinterpret_cast<Words<NB>*>(smem + stage * kBytes)), tid(thread) {}
    __device__ __forceinline__ Words<NB>* w(int unit, int which) const { return at + (2 * unit + which) * THREADS + tid; }
    __device__ __forceinline__ Words<NB>* scale(int which) const { return at + 4 * THREADS + which * (THREADS / 2) + tid; }
};
template <int NB> struct InRegisters {
    Moved<NB>& x;
    __device__ __forceinline__ Words<NB>* w(int unit, int which) const { return &x.w[unit][which]; }
    __device__ __forceinline__ Words<NB>* scale(int which) const { return &x.scale[which]; }
};
// An asynchronous copy of 4, 8, 12 or 16 bytes, aligned as Words are (12: in pieces of 4).
template <int BYTES> __device__ __forceinline__ void copy_async(void* to, const void* from) {
    const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(from) : "memory");
    else if constexpr (BYTES == 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(s), "l"(from) : "memory");
    else if constexpr (BYTES == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s), "l"(from) : "memory");
    else {
        static_assert(BYTES % 4 == 0, "");
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) copy_async<4>(static_cast<uint8_t*>(to) + 4 * i, static_cast<const uint8_t*>(from) + 4 * i);
    }
}

template <int NB, int THREADS, bool AHEAD>
__global__ void __launch_bounds__(THREADS) kv_compact_kernel(const KvCompactArgs p, int chunk, int sides, FastDiv by_chunk, FastDiv by_heads) {
    constexpr int kTileBytes = kv::tile_bytes(NB), kPlaces = AHEAD ? THREADS / 2 : THREADS / 4;
    extern __shared__ __align__(16) uint8_t staged[];
    __shared__ Spot from_s[kSpots][kPlaces], to_s[kSpots][kPlaces];      // of the chunk that is written, and those behind it
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int seq = blockIdx.x, tid = threadIdx.x, first = p.to[seq];
    const int k0 = min(max(p.keep_start[seq], 0), p.tokens), k1 = min(max(p.keep_start[seq + 1], k0), p.tokens), n = k1 - k0;
    if (n == 0) return;
    const int tiles = 1 << (p.page_shift - 4), places = static_cast<int>(min(static_cast<long long>(p.max_pages) << p.page_shift, 0x7fffffffll));
    const int combos = p.layers * p.kv_heads, page_tiles = p.kv_heads * tiles;
    auto spot = [&](int place) {
        Spot s = {-1, place & 15};
        if (place < 0 || place >= places) return s;
        const int page = p.page_table[static_cast<size_t>(seq) * p.max_pages + (place >> p.page_shift)];
        if (page >= 0 && page < p.n_pages) s.tile = page * page_tiles + ((place & ((1 << p.page_shift) - 1)) >> 4);
        return s;
    };
    // The first place is rounded down to a multiple of eight.
    const int lead = first & 7, total = static_cast<int>(min(static_cast<long long>(n) + lead, 0x7fffffffll - 16 * kPlaces));
    const bool looks = tid < chunk;
    Spot next_from, next_to;
    int next_place = -1, place_before = -1;       // of the chunk that is looked up next
    auto ask = [&](int base) {
        const int j = base + tid - lead;
        next_place = looks && j >= 0 && j < n ? p.keep[k0 + j] : -1;
        place_before = looks && j > 0 && j < n ? p.keep[k0 + j - 1] : -1;
    };
    auto look = [&](int base) {                   // where the tokens of the chunk from `base` on come from and go to
        next_from = next_to = {-1, 0};
        const int j = base + tid - lead;
        if (!looks || j < 0 || j >= n) return;
        const int place = next_place;
        const long long to = static_cast<long long>(first) + j;
        next_from = spot(place);
        next_to = spot(to < places ? static_cast<int>(to) : -1);
        const bool good = next_from.tile >= 0 && next_to.tile >= 0 && place >= to && place_before < place;
        if (!good && p.err && blockIdx.y + blockIdx.z == 0) atomicOr(p.err, ERR_BAD_SHAPE);
        if (!good || place == to) next_from.tile = -1;
    };
    auto put = [&](int turn) {
        if (!looks) return;
        from_s[turn % kSpots][tid] = next_from;
        to_s[turn % kSpots][tid] = next_to;
    };
    // What of the chunk this thread has: places of it, and the (layer, head).
    struct Of { int place; const uint8_t* base; };
    auto of_slot = [&](int slot) {                // place -1: none
        const int side = by_chunk(slot), combo = blockIdx.y * sides + side;
        Of o = {-1, nullptr};
        if (side >= sides || combo >= combos) return o;
        const int layer = by_heads(combo), head = combo - layer * p.kv_heads;
        o.place = slot - side * chunk;
        o.base = p.pages + layer * p.layer_stride + static_cast<size_t>(head) * tiles * kTileBytes;
        return o;
    };
    auto tile_at = [&](const Of& o, int tile) { return o.base + static_cast<size_t>(tile) * kTileBytes; };
    // Two units: keys and values, or two of what this CTA has.
    const int quarter = tid & 3, run = (tid >> 2) & 7;                 // of a key; of eight places' values
    auto values = [&](int unit) { return AHEAD ? blockIdx.z == 1 : unit == 1; };
    Of of[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = AHEAD ? tid + i * THREADS : tid;
        of[i] = of_slot(values(i) ? (u >> 5) * 8 + 2 * quarter : u >> 2);
    }
    const bool key_scales = AHEAD ? blockIdx.z == 0 && tid < kPlaces : tid < kPlaces;
    const int value_scale = AHEAD ? blockIdx.z == 1 ? tid : -1 : tid - kPlaces;      // which pair of places'
    const bool value_scales = value_scale >= 0 && value_scale < kPlaces / 2;
    Of of_scale = {-1, nullptr};
    if (key_scales || value_scales) of_scale = of_slot(key_scales ? tid : 2 * value_scale);
    auto take = [&](auto* to, const uint8_t* from) {
        using W = std::remove_pointer_t<decltype(to)>;
        if constexpr (AHEAD) copy_async<sizeof(W)>(to, from);
        else *to = *reinterpret_cast<const W*>(from);
    };
    auto load = [&](int turn, const auto& x) {
        const Spot* const from = from_s[turn % kSpots];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Of o = of[i];
            if (o.place < 0) continue;
            const Spot a = from[o.place];
            if (values(i)) {
                const Spot b = from[o.place + 1];
                if (a.tile >= 0) take(x.w(i, 0), tile_at(o, a.tile) + kv::value_half(NB, a.r & ~1, run, 0));
                if (b.tile >= 0) take(x.w(i, 1), tile_at(o, b.tile) + kv::value_half(NB, b.r & ~1, run, 0));
            } else if (a.tile >= 0) {
                take(x.w(i, 0), tile_at(o, a.tile) + kv::key_word(NB, a.r, quarter, 0));
            }
        }
        if (of_scale.place < 0) return;
        const Spot a = from[of_scale.place];
        if (key_scales) {
            if (a.tile < 0) return;
            const uint8_t* const at = tile_at(of_scale, a.tile) + kv::key_scale(NB, a.r, 0);
            if constexpr (AHEAD) {                // whole words: an odd number of halves begins in the middle of one
                const uint8_t* const word = reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(at) & ~static_cast<uintptr_t>(3));
#pragma unroll
                for (int i = 0; i < (NB + 1) / 2; ++i) copy_async<4>(x.scale(0)->w + i, word + 4 * i);
            } else {
                *reinterpret_cast<Halves<NB>*>(x.scale(0)) = *reinterpret_cast<const Halves<NB>*>(at);
            }
        } else {
            const Spot b = from[of_scale.place + 1];
            if (a.tile >= 0) take(x.scale(0), tile_at(of_scale, a.tile) + kv::value_scale(NB, a.r & ~1, 0));
            if (b.tile >= 0) take(x.scale(1), tile_at(of_scale, b.tile) + kv::value_scale(NB, b.r & ~1, 0));
        }
    };
    // A run of words that two places share, from the halves of their tokens.
    auto join = [&](const Of& o, int turn, int g, const Words<NB>& x, const Words<NB>& y) {
        const Spot a = from_s[turn % kSpots][o.place], b = from_s[turn % kSpots][o.place + 1];
        const bool m0 = a.tile >= 0, m1 = b.tile >= 0;
        if (!m0 && !m1) return;
        const Spot there = to_s[turn % kSpots][o.place + (m0 ? 0 : 1)];
        uint8_t* const at = const_cast<uint8_t*>(tile_at(o, there.tile)) + (g < 8 ? kv::value_half(NB, there.r & ~1, g, 0) : kv::value_scale(NB, there.r & ~1, 0));
        const int s0 = 16 * (a.r & 1), s1 = 16 * (b.r & 1);
        if (m0 && m1) {
            Words<NB> z;
#pragma unroll
            for (int k = 0; k < NB; ++k) z.w[k] = ((x.w[k] >> s0) & 0xFFFFu) | (y.w[k] >> s1) << 16;
            *reinterpret_cast<Words<NB>*>(at) = z;
        } else {
#pragma unroll
            for (int k = 0; k < NB; ++k) reinterpret_cast<uint16_t*>(at)[2 * k + (m0 ? 0 : 1)] = static_cast<uint16_t>(m0 ? x.w[k] >> s0 : y.w[k] >> s1);
        }
    };
    auto store = [&](int turn, const auto& x) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Of o = of[i];
            if (o.place < 0) continue;
            if (values(i)) {
                join(o, turn, run, *x.w(i, 0), *x.w(i, 1));
            } else if (from_s[turn % kSpots][o.place].tile >= 0) {
                const Spot b = to_s[turn % kSpots][o.place];
                *reinterpret_cast<Words<NB>*>(const_cast<uint8_t*>(tile_at(o, b.tile)) + kv::key_word(NB, b.r, quarter, 0)) = *x.w(i, 0);
            }
        }
        if (of_scale.place < 0) return;
        if (key_scales) {
            const Spot a = from_s[turn % kSpots][of_scale.place], b = to_s[turn % kSpots][of_scale.place];
            if (a.tile < 0) return;
            const int in_word = AHEAD ? kv::key_scale(NB, a.r, 0) & 2 : 0;
            *reinterpret_cast<Halves<NB>*>(const_cast<uint8_t*>(tile_at(of_scale, b.tile)) + kv::key_scale(NB, b.r, 0)) =
                *reinterpret_cast<const Halves<NB>*>(reinterpret_cast<const uint8_t*>(x.scale(0)) + in_word);
        } else {
            join(of_scale, turn, 8, *x.scale(0), *x.scale(1));
        }
    };
    if constexpr (!AHEAD) {
        for (int base = 0, turn = 0; base < total; base += chunk, ++turn) {
            Moved<NB> moved;
            const InRegisters<NB> x{moved};
            ask(base);
            look(base);
            put(turn);
            __syncthreads();
            load(turn, x);
            __syncthreads();                      // all of it has been read
            store(turn, x);
        }
        return;
    }
    auto load_ahead = [&](int turn) {
        load(turn, Staged<NB, THREADS>(staged, turn % kStages, tid));
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    ask(0);
    look(0);
    put(0);
    ask(chunk);
    look(chunk);
    put(1);
    ask(2 * chunk);
    __syncthreads();
    load_ahead(0);
    load_ahead(1);
    look(2 * chunk);
    ask(3 * chunk);
    for (int base = 0, turn = 0; base < total; base += chunk, ++turn) {
        put(turn + 2);                            // where chunk turn - 2 stood, which all have written by the barrier before
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();                          // all of chunk `turn` has been read
        load_ahead(turn + 2);                     // (a group a chunk, be it empty)
        look(base + 3 * chunk);
        ask(base + 4 * chunk);
        store(turn, Staged<NB, THREADS>(staged, turn % kStages, tid));
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <int NB> constexpr int kLongSmem = kStages * Staged<NB, kLongThreads>::kBytes;

}  // namespace

cudaError_t launch_kv_copy(const KvCopyArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const int tiles = 1 << (p.page_shift - 4), tile_vecs = kv::tile_bytes(p.head_dim / 32) / 16, head_vecs = tiles * tile_vecs;
    const long long page_vecs = static_cast<long long>(head_vecs) * p.kv_heads;
    if (page_vecs > 1 << 30) return cudaErrorNotSupported;
    const long long x = (page_vecs + kCopyThreads * kCopyAtOnce - 1) / (kCopyThreads * kCopyAtOnce);
    const dim3 grid(static_cast<unsigned>(x < 1024 ? x : 1024), static_cast<unsigned>(p.pairs < 65535 ? p.pairs : 65535), static_cast<unsigned>(p.layers < 65535 ? p.layers : 65535));
    return dependent::launch(kv_copy_kernel, grid, kCopyThreads, 0, stream, env.pdl, p, tiles, tile_vecs, head_vecs);
}

cudaError_t init_kv_move_kernels() {
    for (cudaError_t e : {cudaFuncSetAttribute(kv_compact_kernel<1, kLongThreads, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLongSmem<1>),
                          cudaFuncSetAttribute(kv_compact_kernel<2, kLongThreads, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLongSmem<2>),
                          cudaFuncSetAttribute(kv_compact_kernel<3, kLongThreads, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLongSmem<3>),
                          cudaFuncSetAttribute(kv_compact_kernel<4, kLongThreads, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kLongSmem<4>)})
        if (e != cudaSuccess) return e;
    return cudaSuccess;
}

cudaError_t launch_kv_compact(const KvCompactArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const long long combos = static_cast<long long>(p.layers) * p.kv_heads, each = (static_cast<long long>(p.tokens) + p.n_seqs - 1) / p.n_seqs + 1;
    // Lists of up to 64 tokens a sequence in one go or a few.
    const bool shorter = each <= 64;
    const int places = shorter ? kShortThreads / 4 : kLongThreads / 2;
    int chunk = 8;
    if (shorter)
        while (chunk < places && chunk < each) chunk *= 2;
    else
        chunk = each > kLongThreads / 4 ? kLongThreads / 2 : kLongThreads / 4;
    const int sides = places / chunk;
    const long long y = (combos + sides - 1) / sides;
    if (y > 65535 || combos > 0x7fffffffLL) return cudaErrorNotSupported;
    FastDiv by_chunk, by_heads;
    by_chunk.set(chunk);
    by_heads.set(p.kv_heads);
    const dim3 grid(static_cast<unsigned>(p.n_seqs), static_cast<unsigned>(y), shorter ? 1 : 2);
    auto go = [&](auto short_kernel, auto long_kernel) {
        return dependent::launch(shorter ? short_kernel : long_kernel, grid, shorter ? kShortThreads : kLongThreads, shorter ? 0 : kStages * Staged<1, kLongThreads>::kBytes * (p.head_dim / 32), stream, env.pdl, p, chunk, sides, by_chunk, by_heads);
    };
    switch (p.head_dim) {
        case 32: return go(kv_compact_kernel<1, kShortThreads, false>, kv_compact_kernel<1, kLongThreads, true>);
        case 64: return go(kv_compact_kernel<2, kShortThreads, false>, kv_compact_kernel<2, kLongThreads, true>);
        case 96: return go(kv_compact_kernel<3, kShortThreads, false>, kv_compact_kernel<3, kLongThreads, true>);
        default: return go(kv_compact_kernel<4, kShortThreads, false>, kv_compact_kernel<4, kLongThreads, true>);
    }
}

}  // namespace tcb
