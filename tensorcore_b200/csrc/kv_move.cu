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

// Where a token is: its tile's number in a layer, head 0, and which of the tile's tokens; tile < 0: nowhere.
struct Spot { int tile, r; };

// What a thread moves: a quarter of it to a CTA of its own (blockIdx.z), so that a long list of one sequence has four CTAs a layer and head.
//   part 0      keys' codes, and their scales, of a place
//   parts 1 - 3 three of the nine runs of NB words that two places share: eight of values' codes, and their scales
constexpr int kCompactThreads = 256, kParts = 4;
template <int NB> struct Moved {
    Words<NB> w[4];           // keys: quarters of a row; values: a run of each of two tokens, and another
    Halves<NB> scale;
};

// A chunk is `chunk` places, a multiple of 16, of 256 / chunk (layer, head)s side by side.
template <int NB>
__global__ void __launch_bounds__(kCompactThreads) kv_compact_kernel(const KvCompactArgs p, int chunk, int sides, FastDiv by_chunk, FastDiv by_heads) {
    constexpr int kTileBytes = kv::tile_bytes(NB);
    __shared__ Spot from_s[3][kCompactThreads], to_s[3][kCompactThreads];      // of the chunk that is written, the one that is read, the one that is looked up
    dependent::wait_for_earlier();
    dependent::let_next_begin();
    const int seq = blockIdx.x, part = blockIdx.z, tid = threadIdx.x, first = p.to[seq];
    const int k0 = min(max(p.keep_start[seq], 0), p.tokens), k1 = min(max(p.keep_start[seq + 1], k0), p.tokens), n = k1 - k0;
    if (n == 0) return;
    const int tiles = 1 << (p.page_shift - 4), places = static_cast<int>(min(static_cast<long long>(p.max_pages) << p.page_shift, 0x7fffffffll));
    const int combos = p.layers * p.kv_heads;
    auto spot = [&](int place) {
        Spot s = {-1, place & 15};
        if (place < 0 || place >= places) return s;
        const int page = p.page_table[static_cast<size_t>(seq) * p.max_pages + (place >> p.page_shift)];
        if (page >= 0 && page < p.n_pages) s.tile = page * tiles + ((place & ((1 << p.page_shift) - 1)) >> 4);      // (times heads: below)
        return s;
    };
    // The first place is rounded down to an even one, so that the two places of a word are in one chunk.
    const int lead = first & 1, total = n + lead;
    Spot next_from, next_to;
    auto look = [&](int base) {                   // where the tokens of the chunk from `base` on come from and go to
        next_from = next_to = {-1, 0};
        const int j = base + tid - lead;
        if (tid >= chunk || j < 0 || j >= n) return;
        const int place = p.keep[k0 + j], before = j > 0 ? p.keep[k0 + j - 1] : -1, to = first + j;
        next_from = spot(place);
        next_to = spot(to);
        const bool good = next_from.tile >= 0 && next_to.tile >= 0 && place >= to && before < place;
        if (!good && p.err && blockIdx.y + part == 0) atomicOr(p.err, ERR_BAD_SHAPE);
        if (!good || place == to) next_from.tile = -1;
    };
    auto put = [&](int turn) {
        if (tid >= chunk) return;
        from_s[turn % 3][tid] = next_from;
        to_s[turn % 3][tid] = next_to;
    };
    const int side = by_chunk(tid), t = tid - side * chunk, combo = blockIdx.y * sides + side;
    const bool live = side < sides && combo < combos;
    const int layer = live ? by_heads(combo) : 0, head = live ? combo - layer * p.kv_heads : 0;
    uint8_t* const base_at = p.pages + layer * p.layer_stride;
    // tile number of a layer's head: (page, head, tile in page)
    auto tile_at = [&](int tile) {
        const int page = tile >> (p.page_shift - 4), in = tile & (tiles - 1);
        return base_at + ((static_cast<size_t>(page) * p.kv_heads + head) * tiles + in) * kTileBytes;
    };
    auto run_at = [](int r, int g) {              // g 8: the scales
        return g < 8 ? kv::value_half(NB, r & ~1, g, 0) : kv::value_scale(NB, r & ~1, 0);
    };
    // Values: of the two threads of a pair of places the first has its part's first two runs, the other the third.
    const int pair = t >> 1, mine = t & 1;
    auto load = [&](int turn, Moved<NB>& x) {
        const Spot* const from = from_s[turn % 3];
        if (!live) return;
        if (part == 0) {
            const Spot a = from[t];
            if (a.tile < 0) return;
            const uint8_t* const s = tile_at(a.tile);
#pragma unroll
            for (int i = 0; i < 4; ++i) x.w[i] = *reinterpret_cast<const Words<NB>*>(s + kv::key_word(NB, a.r, i, 0));
            x.scale = *reinterpret_cast<const Halves<NB>*>(s + kv::key_scale(NB, a.r, 0));
            return;
        }
        const Spot a = from[2 * pair], b = from[2 * pair + 1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i == 1 && mine) continue;
            const int g = 3 * (part - 1) + (i == 0 ? 2 * mine : 1);
            if (a.tile >= 0) x.w[2 * i] = *reinterpret_cast<const Words<NB>*>(tile_at(a.tile) + run_at(a.r, g));
            if (b.tile >= 0) x.w[2 * i + 1] = *reinterpret_cast<const Words<NB>*>(tile_at(b.tile) + run_at(b.r, g));
        }
    };
    auto store = [&](int turn, const Moved<NB>& x) {
        const Spot* const from = from_s[turn % 3];
        const Spot* const to = to_s[turn % 3];
        if (!live) return;
        if (part == 0) {
            if (from[t].tile < 0) return;
            const Spot b = to[t];
            uint8_t* const d = tile_at(b.tile);
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<Words<NB>*>(d + kv::key_word(NB, b.r, i, 0)) = x.w[i];
            *reinterpret_cast<Halves<NB>*>(d + kv::key_scale(NB, b.r, 0)) = x.scale;
            return;
        }
        const Spot a = from[2 * pair], b = from[2 * pair + 1];
        const bool m0 = a.tile >= 0, m1 = b.tile >= 0;
        if (!m0 && !m1) return;
        const Spot there = to[2 * pair + (m0 ? 0 : 1)];
        uint8_t* const d = tile_at(there.tile);
        const int s0 = 16 * (a.r & 1), s1 = 16 * (b.r & 1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i == 1 && mine) continue;
            uint8_t* const at = d + run_at(there.r, 3 * (part - 1) + (i == 0 ? 2 * mine : 1));
            if (m0 && m1) {
                Words<NB> y;
#pragma unroll
                for (int k = 0; k < NB; ++k) y.w[k] = ((x.w[2 * i].w[k] >> s0) & 0xFFFFu) | (x.w[2 * i + 1].w[k] >> s1) << 16;
                *reinterpret_cast<Words<NB>*>(at) = y;
            } else {
#pragma unroll
                for (int k = 0; k < NB; ++k)
                    reinterpret_cast<uint16_t*>(at)[2 * k + (m0 ? 0 : 1)] = static_cast<uint16_t>(m0 ? x.w[2 * i].w[k] >> s0 : x.w[2 * i + 1].w[k] >> s1);
            }
        }
    };
    // A chunk is read while the one before it waits to be written, and looked up one ahead of that.
    Moved<NB> x[2];
    look(0);
    put(0);
    __syncthreads();
    load(0, x[0]);
    look(chunk);
    for (int base = 0, turn = 0; base < total; base += 2 * chunk, turn += 2) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {             // chunk turn + u is in x[u]
            if (base + u * chunk >= total) break;
            put(turn + u + 1);                    // where chunk turn + u - 2 stood, which all have written by the barrier before
            __syncthreads();                      // all of chunk turn + u has been read
            if (base + (u + 1) * chunk < total) {
                load(turn + u + 1, x[u ^ 1]);
                look(base + (u + 2) * chunk);
            }
            store(turn + u, x[u]);
        }
    }
}

}  // namespace

cudaError_t launch_kv_copy(const KvCopyArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const int tiles = 1 << (p.page_shift - 4), tile_vecs = kv::tile_bytes(p.head_dim / 32) / 16, head_vecs = tiles * tile_vecs;
    const long long page_vecs = static_cast<long long>(head_vecs) * p.kv_heads;
    if (page_vecs > 1 << 30) return cudaErrorNotSupported;
    const long long x = (page_vecs + kCopyThreads * kCopyAtOnce - 1) / (kCopyThreads * kCopyAtOnce);
    const dim3 grid(static_cast<unsigned>(x < 1024 ? x : 1024), static_cast<unsigned>(p.pairs < 65535 ? p.pairs : 65535), static_cast<unsigned>(p.layers < 65535 ? p.layers : 65535));
    return dependent::launch(kv_copy_kernel, grid, kCopyThreads, 0, stream, env.pdl, p, tiles, tile_vecs, head_vecs);
}

cudaError_t launch_kv_compact(const KvCompactArgs& p, const LaunchEnv& env, cudaStream_t stream) {
    const long long combos = static_cast<long long>(p.layers) * p.kv_heads, each = (static_cast<long long>(p.tokens) + p.n_seqs - 1) / p.n_seqs + 1;
    int chunk = 16;
    while (chunk < kCompactThreads && chunk < each) chunk *= 2;
    const int sides = kCompactThreads / chunk;
    const long long y = (combos + sides - 1) / sides;
    if (y > 65535 || combos > 0x7fffffffLL) return cudaErrorNotSupported;
    FastDiv by_chunk, by_heads;
    by_chunk.set(chunk);
    by_heads.set(p.kv_heads);
    const dim3 grid(static_cast<unsigned>(p.n_seqs), static_cast<unsigned>(y), kParts);
    auto go = [&](auto kernel) { return dependent::launch(kernel, grid, kCompactThreads, 0, stream, env.pdl, p, chunk, sides, by_chunk, by_heads); };
    switch (p.head_dim) {
        case 32: return go(kv_compact_kernel<1>);
        case 64: return go(kv_compact_kernel<2>);
        case 96: return go(kv_compact_kernel<3>);
        default: return go(kv_compact_kernel<4>);
    }
}

}  // namespace tcb
