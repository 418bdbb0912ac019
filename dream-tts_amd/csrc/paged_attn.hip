// Attention of each sequence's new tokens over its paged cache, f16 or in 4 bits (q4.hpp): out_i = sum_j softmax_j(scale
// q_i . k_j) v_j over p_i - window < j <= p_i and j < sinks, a ragged batch of chunks and single tokens.
//
// A row is one (new token, query head). The heads / n_kv query heads of a kv head read the same keys,
// so rows are numbered token * gqa + head within (sequence, kv head), and a tile of consecutive rows goes to one
// workgroup: 16 rows where a sequence has few, 128 where it has a chunk. A query's scores, softmax state (running maximum,
// running sum) and output sums are f32; q, k, v are f16 as the cache and the matrix cores hold them;
// the weights e^(s - max) are rounded to f16 for the second product, and the output is rounded once. The weights are
// held times 2^bias (it cancels in the division by their sum), the largest of a tile at 2^bias at least, toward the upper end of
// f16's range: down to 2^(-14 - bias) of the largest each is off by 2^-11 relative at most, as the output's own rounding is,
// and below that by 2^(-25 - bias) of the largest. The bias is kBias = 15 in the 16-row tiles over f16 pages, kChunkBias = 11 in
// those over 4-bit pages and in the 128-row ones, whose maximum may lag. Without it a flat tail far under one leading key would
// leave the numerator and stay in the denominator (65000 keys e^-17.5 below one: all of their 0.16 %). For the same reason a
// tile's weights are summed before they meet the running sum, next to which a single one may be nothing.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "paged.hpp"
#include "q4.hpp"

namespace dtts {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// The fewest keys of a chunk: 128 / 256 / 512, one token over 1024 keys 8.1 / 9.1 / 11.6 us.
constexpr int kMinChunk = 128;

struct AttnArgs {
    PagedBatch batch;
    const half_t *q, *k, *v;  // k and v: of 4-bit pages their bytes, and the batch's page stride counts those
    half_t *out;
    float *part;       // per (row, chunk): D weighted sums, the weight sum, the maximum of q . k
    int64_t q_stride;  // elements between tokens
    int heads, n_kv, gqa, window, sinks;  // sinks: positions that every later token sees, 0 without a window
    float scale2;      // |scale| * log2(e), above 0: the softmax runs in base 2, its maxima are those of q . k
    bool negate;       // scale < 0: the queries change sign
    int chunk, nsplit; // keys per chunk, chunks at most (the last takes what is left)
    int target;        // above 0: the chunk is chosen for this many units (tiles' chunks) of a kv head, see shared_blocks
    float per_target;  // 1 / target
    FastDiv by_kv, by_gqa, by_chunk;
    int64_t few;       // sequences of at most this many rows go to the 16-row tiles
};

// The keys that sequence s's rows see, in chunks: [lo, hi), lo a multiple of 64, `n` chunks. hi stops
// at the table's end, whatever the context says. With sinks the keys are [0, head) and [head + gap, hi), head and gap
// multiples of 64 (no gap where the windows reach the head, which may pass hi), and chunks cut the axis that leaves the gap
// out: a key past the head is `gap` less there.
struct Span {
    int lo, hi, n, head, gap;
    __device__ __forceinline__ Span(const AttnArgs &a, int n_new, int ctx) {
        const int64_t cap = static_cast<int64_t>(a.batch.max_pages) << a.batch.page_shift;
        hi = ctx < 0 ? 0 : ctx < cap ? ctx : static_cast<int>(cap);
        lo = a.window > 0 && ctx - n_new - a.window + 1 > 0 ? (ctx - n_new - a.window + 1) & ~63 : 0;
        if (lo > hi) lo = hi & ~63;
        head = gap = 0;
        if (a.sinks > 0) {
            head = (a.sinks + 63) & ~63;
            gap = lo > head ? lo - head : 0;
            lo = 0;
        }
        cut(a, static_cast<int>(a.by_chunk.div(static_cast<uint32_t>(hi - gap - lo) + a.chunk - 1)));
    }
    __device__ __forceinline__ void cut(const AttnArgs &a, int chunks) { n = chunks < 1 ? 1 : chunks > a.nsplit ? a.nsplit : chunks; }
    __device__ __forceinline__ int blocks() const { return (hi - gap - lo + 63) >> 6; }  // of 64 keys
    __device__ __forceinline__ void chunk_keys(int chunk, int c, int &k0, int &k1) const {
        k0 = lo + c * chunk;
        k1 = c == n - 1 ? hi - gap : k0 + chunk;
    }
};

// A chunk's key tiles of K keys with sinks: those of the head, [k0, mid), then from `next` on up to k1 (all real keys).
// `bottom`: the first key of the tile's rows' windows.
struct SinkTiles {
    int mid, next;
    __device__ __forceinline__ SinkTiles(const Span &span, int bottom, int K, int &k0, int &k1) {
        mid = k0 < span.head ? (k1 < span.head ? k1 : span.head) : k0;
        next = (k0 < span.head ? span.head : k0) + span.gap;
        if (next < (bottom & -K)) next = bottom & -K;
        if (k1 > span.head) k1 += span.gap;
        if (k0 >= span.head) k0 = mid = next;
    }
};

// The keys that the at-th 128-row tile of a sequence sees, in chunks. (Cut by its sequence's, a chunk of 700 tokens of 8 query heads a
// kv head under a window of 1000 has five chunks for each tile's three: 36 and 31 us.)
__device__ __forceinline__ Span tile_span(const AttnArgs &a, int at, int n_new, int ctx) {
    const int rows = n_new * a.gqa, end = (at + 1) * 128 < rows ? (at + 1) * 128 : rows;
    const int first = static_cast<int>(a.by_gqa.div(at * 128)), last = static_cast<int>(a.by_gqa.div(end - 1));
    return Span(a, last - first + 1, ctx - n_new + last + 1);
}

// A tile of rows: its sequence (-1: none), place in it, the sequence's first row and new tokens, context.
struct Tile {
    int s, at, first, n_new, ctx;
};

// The tile-th tile of `rows` rows over the sequences of more than `above` and at most `upto` rows,
// counted in order (every wave for itself; a sequence's last tile first, which under a causal mask is its
// longest). What the lanes have read of the sequence comes along: one memory round trip in all.
__device__ __forceinline__ Tile find_tile(const AttnArgs &a, int rows, int64_t above, int64_t upto, int tile) {
    const int lane = threadIdx.x & 63;
    for (int s0 = 0; s0 < a.batch.b; s0 += 64) {
        int tiles = 0, first = 0, n = 0, ctx = 0;
        if (s0 + lane < a.batch.b) {
            ctx = a.batch.length(s0 + lane);
            a.batch.rows(s0 + lane, first, n);
            const int64_t of = static_cast<int64_t>(n) * a.gqa;
            if (of > above && of <= upto) tiles = static_cast<int>((of + rows - 1) / rows);
        }
        int sum = tiles;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(sum, off, 64);
            if (lane >= off) sum += v;
        }
        const uint64_t past = __ballot(sum > tile);
        if (past) {
            const int l = __ffsll(static_cast<unsigned long long>(past)) - 1;
            const int at = __builtin_amdgcn_readlane(sum, l) - 1 - tile;
            if (at < 0 || at >= __builtin_amdgcn_readlane(tiles, l)) break;  // starts that do not rise can pass any sum
            return Tile{s0 + l, at, __builtin_amdgcn_readlane(first, l), __builtin_amdgcn_readlane(n, l),
                        __builtin_amdgcn_readlane(ctx, l)};
        }
        tile -= __builtin_amdgcn_readlane(sum, 63);
    }
    return Tile{-1, 0, 0, 0, 0};
}

// Inclusive sums and maxima over the wave's lanes, by data-parallel moves: no trip through LDS.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T from_before(T old, T x) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, old), __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
template <typename T>
__device__ __forceinline__ T sums_to_here(T x) {
    x += from_before<0x111, 0xf>(T(0), x);
    x += from_before<0x112, 0xf>(T(0), x);
    x += from_before<0x114, 0xf>(T(0), x);
    x += from_before<0x118, 0xf>(T(0), x);
    x += from_before<0x142, 0xa>(T(0), x);
    return x + from_before<0x143, 0xc>(T(0), x);
}
__device__ __forceinline__ int most_to_here(int x) {
    const auto most = [](int p, int q) { return p > q ? p : q; };
    x = most(x, from_before<0x111, 0xf>(x, x));
    x = most(x, from_before<0x112, 0xf>(x, x));
    x = most(x, from_before<0x114, 0xf>(x, x));
    x = most(x, from_before<0x118, 0xf>(x, x));
    x = most(x, from_before<0x142, 0xa>(x, x));
    return most(x, from_before<0x143, 0xc>(x, x));
}

// Sequence s as a lane of the wave sees it: its first row, new tokens, context, 16-row tiles, and blocks of 64 keys.
struct Lane {
    int first = 0, n = 0, ctx = 0, tiles = 0, blocks = 0;
    __device__ __forceinline__ Lane(const AttnArgs &a, int s) {
        if (s >= a.batch.b) return;
        ctx = a.batch.length(s);
        a.batch.rows(s, first, n);
        if (n == 0) return;
        tiles = static_cast<int>((static_cast<int64_t>(n) * a.gqa + 15) >> 4);
        blocks = Span(a, n, ctx).blocks();
    }
};

// The chunk, in blocks of 64 keys, that cuts what keys there are (not the longest context's, which the host knows) into about
// `target` units of a kv head, all of one size but a tile's last. Every wave finds it for itself from the batch's arrays, in
// the same order of sums.
__device__ __forceinline__ int shared_blocks(const AttnArgs &a, const Lane &first) {
    const int lane = threadIdx.x & 63;
    float total = static_cast<float>(first.tiles) * static_cast<float>(first.blocks);
    int longest = first.blocks;
    for (int s0 = 64; s0 < a.batch.b; s0 += 64) {
        const Lane l(a, s0 + lane);
        total += static_cast<float>(l.tiles) * static_cast<float>(l.blocks);
        longest = l.blocks > longest ? l.blocks : longest;
    }
    const float all = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sums_to_here(total)), 63));
    longest = __builtin_amdgcn_readlane(most_to_here(longest), 63);
    const float even = ceilf(all * a.per_target);
    const int per = static_cast<int>((static_cast<uint32_t>(longest) + a.nsplit - 1) / static_cast<uint32_t>(a.nsplit));  // room for a tile's
    int blocks = even < static_cast<float>(1 << 24) ? static_cast<int>(even) : 1 << 24;
    blocks = blocks < per ? per : blocks;
    blocks = blocks < kMinChunk / 64 ? kMinChunk / 64 : blocks;
    return __builtin_amdgcn_readfirstlane(blocks);
}

__device__ __forceinline__ int chunks_of(int blocks, int per) {
    return static_cast<int>((static_cast<uint32_t>(blocks) + per - 1) / static_cast<uint32_t>(per));
}

// A tile, which of its chunks, and how many it has.
struct Unit {
    Tile tile;
    int c, chunks, chunk;
};

// The unit-th of all sequences' tiles' chunks.
__device__ __forceinline__ Unit find_unit(const AttnArgs &a, int unit) {
    const int lane = threadIdx.x & 63;
    const Lane first(a, lane);
    const int per = shared_blocks(a, first);
    for (int s0 = 0; s0 < a.batch.b; s0 += 64) {
        const Lane l = s0 == 0 ? first : Lane(a, s0 + lane);
        int n = chunks_of(l.blocks, per);
        n = n < 1 ? 1 : n;
        const int units = l.tiles * n, sum = sums_to_here(units);
        const uint64_t past = __ballot(sum > unit);
        if (past) {
            const int at = __ffsll(static_cast<unsigned long long>(past)) - 1;
            const int of = __builtin_amdgcn_readlane(units, at), k = __builtin_amdgcn_readlane(sum, at) - 1 - unit;
            if (k < 0 || k >= of) break;  // starts that do not rise can pass any sum
            const int chunks = __builtin_amdgcn_readlane(n, at);
            const int tile = chunks == 1 ? k : static_cast<int>(static_cast<uint32_t>(k) / static_cast<uint32_t>(chunks));
            return Unit{Tile{s0 + at, tile, __builtin_amdgcn_readlane(l.first, at), __builtin_amdgcn_readlane(l.n, at),
                             __builtin_amdgcn_readlane(l.ctx, at)},
                        k - tile * chunks, chunks, 64 * per};
        }
        unit -= __builtin_amdgcn_readlane(sum, 63);
    }
    return Unit{Tile{-1, 0, 0, 0, 0}, 0, 1, 64 * per};
}

// The largest of the lanes 32 apart (and 16 apart), by exchanging halves of registers: no trip through LDS.
__device__ __forceinline__ float max_32_apart(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_16_32_apart(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return max_32_apart(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// What the exponents of the weights are raised by. The largest weight of the 16-row tiles over f16 pages is 2^kBias; of those over
// 4-bit pages and of the 128-row ones it is 2^kChunkBias to 2^(kChunkBias + kSlack), as their maximum may lag behind by kSlack: all
// under f16's 65504. kSlack 1 / 4 / 8 (and a bias that goes with it): 2048 tokens after 7952 335 / 333 / 335 us.
constexpr float kBias = 15.0f, kSlack = 4.0f, kChunkBias = 11.0f;
// A weight's exponent is fma(q . k, scale2, -m2), m2 the rounded product of the maximum: off by half of m2's last place,
// alike for all keys that a wave takes relative to one maximum, so that it cancels among them as a bias does, but not
// against what was summed relative to another. At 2^12 that is 2^-13, under the weights' own rounding; scores past it are
// taken relative to their maximum first (another instruction a score), which no size of theirs overflows.
constexpr float kFar = 4096.0f;
// m2 for a new maximum m, less the bias; far: sticky, whether any lane's scores are that large.
__device__ __forceinline__ float relative_to(float m, float scale2, float bias, bool &far) {
    const float m2 = m == -INFINITY ? 0.0f : m * scale2;
    far = far || __any(fabsf(m2) >= kFar);
    return (far ? 0.0f : m2) - bias;
}

// A value that is not finite (an overflow of the projection, a slot written over) makes 0 times it a NaN, so in a tile of
// keys that not all of the rows see it may not reach the product: there such values count as 0 (take_out says whether it
// met one), and the rows that see them get them added after the last tile (taken). What all rows see goes through the
// product as it is. Two values at a time and without comparisons, whose masks would fill the scalar registers.
__device__ __forceinline__ uint32_t not_finite(uint32_t pair) {  // ones in the place of each that has the largest exponent
    const uint32_t top = ((pair & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
    return top | (top - (top >> 15));
}
// The same of the groups of 4-bit values of two pairs: ones in the place of each that holds a value with the largest exponent, or could.
__device__ __forceinline__ uint32_t q4_not_finite(half2_t d, half2_t b) {
    const half_t first = static_cast<half_t>(kQ4First), last = static_cast<half_t>(kQ4Last);
    return not_finite(__builtin_bit_cast(uint32_t, __builtin_elementwise_fma(half2_t{first, first}, d, b))) |
           not_finite(__builtin_bit_cast(uint32_t, __builtin_elementwise_fma(half2_t{last, last}, d, b)));
}
__device__ __forceinline__ bool q4_not_finite(uint32_t pair) {
    const half2_t p = __builtin_bit_cast(half2_t, pair);
    return q4_not_finite(half2_t{p[0], p[0]}, half2_t{p[1], p[1]}) != 0;
}
template <int E>
__device__ __forceinline__ uint32_t take_out(half_t __attribute__((ext_vector_type(E))) &v) {
    typedef uint32_t pairs __attribute__((ext_vector_type(E / 2)));
    pairs p = __builtin_bit_cast(pairs, v);
    uint32_t any = 0;
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
        const uint32_t out = not_finite(p[e]);
        any |= out;
        p[e] &= ~out;
    }
    v = __builtin_bit_cast(half_t __attribute__((ext_vector_type(E))), p);
    return any;
}
template <int E>
__device__ __forceinline__ half_t __attribute__((ext_vector_type(E))) taken(half_t __attribute__((ext_vector_type(E))) v) {
    typedef uint32_t pairs __attribute__((ext_vector_type(E / 2)));
    pairs p = __builtin_bit_cast(pairs, v);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) p[e] &= not_finite(p[e]);
    return __builtin_bit_cast(half_t __attribute__((ext_vector_type(E))), p);
}

// ---------------------------------------------------------------- few rows: 16 a tile

// Four waves, each with its own tiles of 32 keys and its own softmax state; the states meet in LDS at
// the end. A score tile is K . Q^T on 16x16x32 MFMAs: a lane holds 4 keys (4g + i of 16, g = lane / 16)
// of one row (lane % 16), two such tiles make 8, and those 8 weights are, as they stand, the lane's
// operand of out^T = V^T . P^T (the k index of a product may name the keys in any order, so long as
// both operands do: 8g + j is key 4g + j for j < 4 and 16 + 4g + j - 4 from there). V^T's operand is
// 8 keys of one dimension; a lane loads those 8 keys' rows 16 bytes wide (dimensions 8h .. 8h + 7, h =
// lane % 16) and the 8 columns of that block are 8 products' operands, product e making the
// dimensions 8h + e. So K, V and the scores go from memory to the matrix cores without LDS.
//
// Bound by memory: 5 tokens of 32 heads over 4 and up to 65000 keys 74 us, 4.9 TB/s; 48 over 16000 each 5.6 TB/s. A few
// hundred keys are a chain of trips to memory (starts, page ids, keys, 32 keys a wave and step): one token over 300
// 7.7 us. Two tiles in flight a wave halve the waves a SIMD holds (74 -> 81); page ids a tile ahead win half a
// microsecond under 1000 keys and lose 1 % of the long ones.
template <bool ONCE, typename T>
__device__ __forceinline__ T fetch(const T *p) {
    if constexpr (ONCE) return __builtin_nontemporal_load(p);
    return *p;
}

template <int D, bool Q4, bool ONCE>
struct KvTile {
    static constexpr int E = D / 16;  // dimensions a lane holds of each of its 8 value rows
    typedef half_t ve __attribute__((ext_vector_type(E)));
    half8_t k[2][D / 32];
    ve v[8];
    int ok;  // bit u: keys 16u .. 16u + 15 have a page

    // Of the score product's step i, a lane of group g has the dimensions from here on.
    __device__ __forceinline__ static int dim(int i, int g) { return 32 * i + 8 * g; }
    struct Lane {
        int l16, g;
        __device__ __forceinline__ Lane(const AttnArgs &, int lane16, int group) : l16(lane16), g(group) {}
    };
    // base: of the page's kv head; slot: keys 16u's place there
    __device__ __forceinline__ void load_keys(const AttnArgs &a, int u, int64_t base, int slot, const Lane &at) {
        base += static_cast<int64_t>(slot) * D;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) k[u][i] = fetch<ONCE>(reinterpret_cast<const half8_t *>(a.k + base + at.l16 * D + dim(i, at.g)));
    }
    __device__ __forceinline__ void load_values(const AttnArgs &a, int u, int64_t base, int slot, const Lane &at) {
        base += static_cast<int64_t>(slot) * D;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * u + j] = fetch<ONCE>(reinterpret_cast<const ve *>(a.v + base + (4 * at.g + j) * D + E * at.l16));
    }
    __device__ __forceinline__ half8_t key(int u, int i, const Q4Bits &) const { return k[u][i]; }
    __device__ __forceinline__ void drop(int j, bool out) { v[j] = out ? ve{} : v[j]; }
    __device__ __forceinline__ void turn(int) {}
    __device__ __forceinline__ void take_out_values(uint32_t &spoilt) {
#pragma unroll
        for (int j = 0; j < 8; ++j) spoilt |= take_out<E>(v[j]);
    }
    __device__ __forceinline__ half8_t value(int e, const Q4Bits &) const {
        half8_t f;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = v[j][e];
        return f;
    }
};

// Of 4-bit pages a lane has 16 or 32 neighbouring dimensions of its key (one load and their pair), and of the values a word
// of four keys at once (one load) with their pairs (another). The words are turned before they become numbers: halves of two
// keys' words make pairs of keys, which is what the product's operand holds. 5 tokens of 32 heads over 4 and up to 65000 keys (132
// MB): 27.4 us, 4.8 TB/s, vector issue 0.63 of the cycles; 48 of 16 over 8 and up to 1536 (49 MB): 15.5, of which one key each takes 6.
template <int D, bool ONCE>
struct KvTile<D, true, ONCE> {
    static constexpr int E = D / 16, W = D / 32;  // W: key words a lane holds
    typedef half_t ve __attribute__((ext_vector_type(E)));
    typedef uint32_t kw __attribute__((ext_vector_type(W)));
    kw k[2];
    uint32_t ks[2];
    u32x4 v[2], vs[2];
    uint32_t lo[4], hi[4];  // of the values' key pairs, after turn
    half2_t d[4], b[4];
    int ok;

    __device__ __forceinline__ static int dim(int i, int g) { return 8 * (W * g + i); }
    // What a lane reads lies at these bytes from what the wave does.
    struct Lane {
        uint32_t k, ks, v, vs;
        __device__ __forceinline__ Lane(const AttnArgs &a, int l16, int g) {
            const int page = 1 << a.batch.page_shift;
            k = Q4Row<D>::key_word(l16, W * g);
            ks = (W * g / 4 * page + l16) * 4;
            v = Q4Row<D>::value_word(4 * g, E * l16 / 8);
            vs = (E * l16 / 32 * page + 4 * g) * 4;
        }
    };
    __device__ __forceinline__ void load_keys(const AttnArgs &a, int u, int64_t base, int slot, const Lane &at) {
        const uint8_t *kp = reinterpret_cast<const uint8_t *>(a.k) + base;
        const uint32_t words = slot * (Q4Row<D>::kWords * 4), pairs = Q4Row<D>::pair(1 << a.batch.page_shift, slot, 0);
        k[u] = fetch<ONCE>(reinterpret_cast<const kw *>(kp + words + at.k));
        ks[u] = fetch<ONCE>(reinterpret_cast<const uint32_t *>(kp + pairs + at.ks));
    }
    __device__ __forceinline__ void load_values(const AttnArgs &a, int u, int64_t base, int slot, const Lane &at) {
        const uint8_t *vp = reinterpret_cast<const uint8_t *>(a.v) + base;
        const uint32_t words = slot * (Q4Row<D>::kWords * 4), pairs = Q4Row<D>::pair(1 << a.batch.page_shift, slot, 0);
        v[u] = fetch<ONCE>(reinterpret_cast<const u32x4 *>(vp + words + at.v));
        vs[u] = fetch<ONCE>(reinterpret_cast<const u32x4 *>(vp + pairs + at.vs));
    }
    __device__ __forceinline__ half8_t key(int u, int i, const Q4Bits &bits) const { return q4_values(k[u][i], ks[u], bits); }
    __device__ __forceinline__ void drop(int j, bool out) { vs[j >> 2][j & 3] = out ? 0 : vs[j >> 2][j & 3]; }  // 64 + n times 0
    __device__ __forceinline__ void turn(int l16) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int u = t >> 1, j = 2 * (t & 1);
            lo[t] = low_halves(v[u][j], v[u][j + 1]);
            hi[t] = high_halves(v[u][j], v[u][j + 1]);
            if (E == 4 && (l16 & 1)) {  // the word's second four dimensions
                lo[t] >>= 8;
                hi[t] >>= 8;
            }
            d[t] = __builtin_bit_cast(half2_t, low_halves(vs[u][j], vs[u][j + 1]));
            b[t] = __builtin_bit_cast(half2_t, high_halves(vs[u][j], vs[u][j + 1]));
        }
    }
    // A group's values lie between those of its first and last code: one of which either is not finite is left out whole.
    __device__ __forceinline__ void take_out_values(uint32_t &spoilt) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint32_t out = q4_not_finite(d[t], b[t]);
            spoilt |= out;
            d[t] = __builtin_bit_cast(half2_t, __builtin_bit_cast(uint32_t, d[t]) & ~out);
            b[t] = __builtin_bit_cast(half2_t, __builtin_bit_cast(uint32_t, b[t]) & ~out);
        }
    }
    __device__ __forceinline__ half8_t value(int e, const Q4Bits &bits) const {
        half8_t f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const half2_t x = __builtin_elementwise_fma(q4_codes(e & 1 ? hi[t] : lo[t], e >> 1, bits), d[t], b[t]);
            f[2 * t] = x[0];
            f[2 * t + 1] = x[1];
        }
        return f;
    }
};

// Four or eight neighbouring dimensions (a multiple of as many) of a key's value row. base: of the page's kv head.
template <int D, bool Q4, int E>
__device__ __forceinline__ half_t __attribute__((ext_vector_type(E))) value_run(const AttnArgs &a, int64_t base, int slot, int dim) {
    typedef half_t ve __attribute__((ext_vector_type(E)));
    if constexpr (Q4) {
        const uint8_t *vp = reinterpret_cast<const uint8_t *>(a.v) + base;
        const uint32_t word = *reinterpret_cast<const uint32_t *>(vp + Q4Row<D>::value_word(slot, dim / 8));
        const half8_t x = q4_values(word, *reinterpret_cast<const uint32_t *>(vp + Q4Row<D>::pair(1 << a.batch.page_shift, slot, dim / 32)), Q4Bits());
        ve y;
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = E == 4 && (dim & 4) ? x[4 + e] : x[e];
        return y;
    } else {
        return *reinterpret_cast<const ve *>(a.v + base + static_cast<int64_t>(slot) * D + dim);
    }
}

// The pair of a key's value group that holds dimension dim.
template <int D>
__device__ __forceinline__ uint32_t value_pair(const AttnArgs &a, int64_t base, int slot, int dim) {
    return *reinterpret_cast<const uint32_t *>(reinterpret_cast<const uint8_t *>(a.v) + base +
                                               Q4Row<D>::pair(1 << a.batch.page_shift, slot, dim / 32));
}

// Where a page's kv head begins in it.
template <int D, bool Q4>
__device__ __forceinline__ int64_t head_offset(const AttnArgs &a, int kh) {
    return (static_cast<int64_t>(kh) << a.batch.page_shift) * (Q4 ? Q4Row<D>::kBytes : D);
}

template <int D>
struct RowsLds {
    float o[4][16][D + 4], m[4][16], l[4][16];
};

template <int D, bool Q4, bool SINKS, bool ONCE>
__device__ __forceinline__ void rows_tile(const AttnArgs &a, RowsLds<D> &lds, int block) {
    constexpr int C = D / 32, E = D / 16, ROWS = 16;
    auto &sm_o = lds.o;
    auto &sm_m = lds.m;
    auto &sm_l = lds.l;
    const bool shared = Q4 && a.target > 0;
    const int tile_no = static_cast<int>(a.by_kv.div(static_cast<uint32_t>(block))), kh = block - tile_no * a.n_kv;
    const Unit unit = shared ? find_unit(a, tile_no) : Unit{find_tile(a, ROWS, 0, a.few, tile_no), static_cast<int>(blockIdx.y), 0, a.chunk};
    const Tile &tile = unit.tile;
    if (tile.s < 0) return;
    const int s = tile.s, at = tile.at, first = tile.first, n_new = tile.n_new, ctx = tile.ctx;
    Span span(a, n_new, ctx);
    if (shared) span.cut(a, unit.chunks);
    const int c = unit.c;
    if (c >= span.n) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int n_rows = n_new * a.gqa - at * ROWS < ROWS ? n_new * a.gqa - at * ROWS : ROWS;
    // the lane's row: token `tok` of the sequence, query head kh * gqa + head
    const int row = at * ROWS + (l16 < n_rows ? l16 : n_rows - 1);
    const auto token_of = [&](int r) { return static_cast<int>(a.by_gqa.div(static_cast<uint32_t>(r))); };
    const int tok = token_of(row), head = kh * a.gqa + row - tok * a.gqa;
    const int pos = ctx - n_new + tok;
    const int first_tok = token_of(at * ROWS), last_tok = token_of(at * ROWS + n_rows - 1);
    int k0, k1;  // the tile's keys in this chunk
    span.chunk_keys(unit.chunk, c, k0, k1);
    const int row_lo = a.window > 0 ? pos - a.window + 1 : 0;
    // one of the tile's rows at least sees the keys [bottom, k1), all of them [from, end)
    const bool one_token = first_tok == last_tok;
    const int bottom = a.window > 0 ? ctx - n_new + first_tok - a.window + 1 : 0;
    const int from = a.window > 0 ? bottom + last_tok - first_tok : 0;
    int end = ctx - n_new + first_tok + 1, mid = 0, next = 0;
    if constexpr (SINKS) {
        const SinkTiles tiles(span, bottom, 32, k0, k1);
        mid = tiles.mid;
        next = tiles.next;
    }
    {
        const int top = ctx - n_new + last_tok + 1;
        if (k1 > top) k1 = top;
        if (!SINKS && k0 < bottom) k0 = bottom & ~31;
        if (end > k1) end = k1;
    }
    const int shown = SINKS ? (a.sinks < end ? a.sinks : end) : 0;  // and all of them [0, shown)
    half8_t qf[C];
    {
        const half_t *qr = a.q + (first + tok) * a.q_stride + static_cast<int64_t>(head) * D;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            qf[i] = *reinterpret_cast<const half8_t *>(qr + KvTile<D, Q4, ONCE>::dim(i, g));
            if (a.negate) qf[i] = -qf[i];
        }
    }
    const int in_page = (1 << a.batch.page_shift) - 1;
    const int64_t head_at = head_offset<D, Q4>(a, kh);
    const typename KvTile<D, Q4, ONCE>::Lane lane_at(a, l16, g);
    // the wave's key tiles are every fourth: the i-th begins at key_of(i)
    const int base = SINKS ? k0 : k0 & ~31;
    const int heads_tiles = SINKS ? (mid - k0 + 31) >> 5 : 0, rest_at = SINKS ? next : base;
    const int n_tiles = heads_tiles + (rest_at < k1 ? (k1 - rest_at + 31) >> 5 : 0);
    auto key_of = [&](int i) { return SINKS && i < heads_tiles ? base + 32 * i : rest_at + 32 * (i - heads_tiles); };
    // The page ids of the wave's next 32 tiles at once, a lane for each 16 keys: a tile's keys wait for no id of their own.
    int id_lane = -1;
    auto ids_from = [&](int i) {
        const int key = key_of(i + 4 * (lane >> 1)) + 16 * (lane & 1);
        id_lane = i + 4 * (lane >> 1) < n_tiles && key < k1 ? a.batch.page(s, key >> a.batch.page_shift) : -1;
    };
    auto page_of = [&](int i, int u) { return __builtin_amdgcn_readlane(id_lane, ((i - w) >> 1 & 62) + u); };  // i: w and every fourth
    auto load_keys = [&](int i, KvTile<D, Q4, ONCE> &t) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int page = page_of(i, u);
            t.load_keys(a, u, (page < 0 ? 0 : page) * a.batch.page_stride + head_at, (key_of(i) + 16 * u) & in_page, lane_at);
        }
    };
    auto load_values = [&](int i, KvTile<D, Q4, ONCE> &t) {
        t.ok = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int page = page_of(i, u);
            if (page >= 0) t.ok |= 1 << u;
            t.load_values(a, u, (page < 0 ? 0 : page) * a.batch.page_stride + head_at, (key_of(i) + 16 * u) & in_page, lane_at);
        }
    };
    float m = -INFINITY, m2 = 0.0f, l = 0.0f;  // m2: what the weights are relative to in log2, anything while there is no m
    bool far = false;
    uint32_t spoilt = 0;
    float4_t o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = float4_t{0.f, 0.f, 0.f, 0.f};
    const Q4Bits bits;
    auto compute = [&](int kb, KvTile<D, Q4, ONCE> &t, auto after_scores) {
        float4_t sc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            sc[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < C; ++i) sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.key(u, i, bits), qf[i], sc[u], 0, 0, 0);
            if (Q4) __builtin_amdgcn_sched_barrier(0);
        }
        after_scores();
        // whether some of the rows do not see some of the keys
        const bool partly = (kb < from && !(SINKS && kb + 32 <= shown)) || kb + 32 > end;
        if (__builtin_expect(partly || t.ok != 3, 0)) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = kb + 16 * u + 4 * g + i;
                const bool seen = key <= pos && (key >= row_lo || (SINKS && key < a.sinks)) && key < k1 && (t.ok >> u & 1);
                sc[u][i] = seen ? sc[u][i] : -INFINITY;
            }
        }
        float mx = Q4 ? sc[0][0] : m;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[u][i]);
        // the row's other keys are 16 and 32 lanes away
        mx = max_16_32_apart(mx);
        // over 4-bit pages, where issue counts, only a maximum that has grown by 2^kSlack moves the sums
        if (Q4 ? __any((mx - m) * a.scale2 > kSlack) : __any(mx > m)) {
            if (Q4) mx = fmaxf(mx, m);
            const float f = exp2_fast(mx == -INFINITY ? 0.0f : (m - mx) * a.scale2);
            l *= f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= f;
            m = mx;
            m2 = relative_to(m, a.scale2, Q4 ? kChunkBias : kBias, far);
        }
        if (far) {
            const float from_m = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int u = 0; u < 2; ++u) sc[u] -= from_m;
        }
        half8_t p;
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = exp2_fast(__builtin_fmaf(sc[u][i], a.scale2, -m2));
                sum += x;
                p[4 * u + i] = static_cast<half_t>(x);
            }
        l += sum;
        // what no row sees holds anything: 0 times it may be NaN. Selected without a branch: of nested ones (k1, window, sinks, page)
        // around a register's part the compiler kept only the first and the zero of a missing page was lost.
        if (__builtin_expect(partly || t.ok != 3, 0)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3);
                const bool sunk = SINKS & (key < a.sinks), there = t.ok >> (j >> 2) & 1;
                t.drop(j, (key >= k1) | ((key < bottom) & !sunk) | !there);
            }
        }
        t.turn(l16);
        if (__builtin_expect(partly && !one_token, 0)) t.take_out_values(spoilt);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.value(e, bits), p, o[e], 0, 0, 0);
            if (Q4 && (e & 1)) __builtin_amdgcn_sched_barrier(0);
        }
    };
    KvTile<D, Q4, ONCE> t;
    if constexpr (Q4) {
        // the next tile's keys are requested as soon as this one's have made their scores, in the same registers; past the last
        // key page 0 is read, for nothing, so that no branch holds a request
        if (w < n_tiles) {
            ids_from(w);
            load_keys(w, t);
        }
        for (int i = w; i < n_tiles; i += 4) {
            load_values(i, t);
            compute(key_of(i), t, [&] {
                if (((i - w) & 124) == 124) ids_from(i + 4);
                load_keys(i + 4, t);
                __builtin_amdgcn_sched_barrier(0);
            });
        }
    } else {
        for (int i = w; i < n_tiles; i += 4) {
            if (((i - w) & 124) == 0) ids_from(i);
            load_keys(i, t);
            load_values(i, t);
            compute(key_of(i), t, [] {});
        }
    }
    // the weight of a key for the lane's row, from the key's row in memory; the four lanes that share the row each take a quarter
    auto weight_again = [&](int64_t at_head, int slot) {
        const uint8_t *kp = reinterpret_cast<const uint8_t *>(a.k) + at_head;
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int d = KvTile<D, Q4, ONCE>::dim(i, g);
            const half8_t k = q4_values(*reinterpret_cast<const uint32_t *>(kp + Q4Row<D>::key_word(slot, d / 8)),
                                        *reinterpret_cast<const uint32_t *>(kp + Q4Row<D>::pair(in_page + 1, slot, d / 32)), bits);
#pragma unroll
            for (int e = 0; e < 8; ++e) x = __builtin_fmaf(static_cast<float>(k[e]), static_cast<float>(qf[i][e]), x);
        }
        x += __shfl_xor(x, 16, 64);
        x += __shfl_xor(x, 32, 64);
        return exp2_fast((x - m) * a.scale2 + kChunkBias);
    };
    if (__builtin_expect(__any(spoilt != 0), 0)) {
        for (int i = w; i < n_tiles; i += 4) {
            const int kb = key_of(i);
            if ((kb >= from || (SINKS && kb + 32 <= shown)) && kb + 32 <= end) continue;
            for (int key = kb; key < kb + 32 && key < k1; ++key) {
                const int page = a.batch.page(s, key >> a.batch.page_shift);
                const bool unseen = page < 0 || key > pos || (key < row_lo && !(SINKS && key < a.sinks));
                if constexpr (Q4) {  // with their weights, taken again; a value that is not finite counts whatever its weight is
                    const int64_t at_head = (page < 0 ? 0 : page) * a.batch.page_stride + head_at;
                    const float x = weight_again(at_head, key & in_page);
                    if (unseen) continue;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int d = 4 * E * g + E * i;
                        const uint32_t pair = value_pair<D>(a, at_head, key & in_page, d);
                        if (!q4_not_finite(pair)) continue;
                        const auto v = value_run<D, Q4, E>(a, at_head, key & in_page, d);
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const float y = static_cast<float>(v[e]);
                            o[e][i] += fabsf(y) < INFINITY ? x * y : y;
                        }
                    }
                    continue;
                }
                if (unseen) continue;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const auto v = taken<E>(value_run<D, Q4, E>(a, page * a.batch.page_stride + head_at, key & in_page, 4 * E * g + E * i));
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e][i] += static_cast<float>(v[e]);
                }
            }
        }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // product e's row r is dimension E r + e: a lane holds 4 runs of E dimensions of its row
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < E; e += 4)
            *reinterpret_cast<float4_t *>(&sm_o[w][l16][E * (4 * g + i) + e]) = float4_t{o[e][i], o[e + 1][i], o[e + 2][i], o[e + 3][i]};
    if (g == 0) {
        sm_m[w][l16] = m;
        sm_l[w][l16] = l;
    }
    __syncthreads();
    // the waves' states: 16 lanes a row, E dimensions each
    const int r = threadIdx.x >> 4;
    float mt = -INFINITY, den = 0.0f, num[E] = {};
#pragma unroll
    for (int u = 0; u < 4; ++u) mt = fmaxf(mt, sm_m[u][r]);
    const float mu = mt == -INFINITY ? 0.0f : mt;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const float f = exp2_fast((sm_m[u][r] - mu) * a.scale2);
        den += sm_l[u][r] * f;
#pragma unroll
        for (int e = 0; e < E; ++e) num[e] += sm_o[u][r][E * l16 + e] * f;
    }
    const int rr = at * ROWS + (r < n_rows ? r : n_rows - 1), rtok = token_of(rr), rhead = kh * a.gqa + rr - rtok * a.gqa;
    const int64_t trow = static_cast<int64_t>(first + rtok) * a.heads + rhead;
    if (r < n_rows) {
        if (span.n > 1) {
            float *pr = a.part + (trow * a.nsplit + c) * (D + 4);
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<float4_t *>(pr + E * l16 + e) = float4_t{num[e], num[e + 1], num[e + 2], num[e + 3]};
            if (l16 == 0) {
                pr[D] = den;
                pr[D + 1] = mt;
            }
        } else {
            const float inv = den == 0.0f ? 0.0f : 1.0f / den;  // a row that sees no key is zero
            typename KvTile<D, Q4, ONCE>::ve y;
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = static_cast<half_t>(num[e] * inv);
            *reinterpret_cast<typename KvTile<D, Q4, ONCE>::ve *>(a.out + trow * D + E * l16) = y;
        }
    }
}

// ---------------------------------------------------------------- chunks: 128 rows a tile

// Four waves of 32 rows each share every 64 keys through LDS. A score block is K . Q^T on 32x32x16
// MFMAs: a lane holds 16 keys (8 (r >> 2) + 4g + (r & 3), g = lane / 32) of one row (lane % 32), and
// registers 8h .. 8h + 7 are, as they stand, its operand of out^T = V^T . P^T for keys 16h .. 16h + 15,
// whose k index 8g + j then names key 4g + j for j < 4 and 8 + 4g + j - 4 from there. V is stored
// transposed in that key order as it is staged (a thread takes 4 keys of E dimensions, so the turn is
// made once for the four waves), and both operands are single 16-byte LDS reads. Neighbouring lanes read different
// banks: key rows are padded by 16 bytes, the 16-byte pieces of V^T's rows XOR-swizzled.
//
// Two buffers: the next keys' rows are requested a tile ahead and stored after the tile's products, one barrier a
// tile. Bound by issue: two waves a SIMD take turns between the matrix cores and the softmax's 32 exponentials,
// products with the scale and conversions a lane (matrix cores busy 49 % of the cycles, vector instructions 46 %,
// LDS 44 %). 2048 tokens after 7952, 32 heads over 8, D = 128: 333 us, 900 TFLOP/s of the unmasked products.
template <int D>
struct ChunkLds {
    static constexpr int KT = 64, KP = D + 8;  // keys a tile; elements from key row to key row
    half_t k[2][KT * KP], v[2][D * KT];
    int ok[2][4], spoilt[4];
};

template <int D, bool Q4, bool SINKS>
__device__ __forceinline__ void chunk_tile(const AttnArgs &a, ChunkLds<D> &lds, int block_no) {
    constexpr int ROWS = 128, KT = 64, E = D / 16, C = D / 16, KL = D / 32;  // C: k steps, KL: 16-byte key loads a thread
    constexpr int KCH = D / 8, KP = ChunkLds<D>::KP;                         // KCH: 16-byte pieces of a key row
    typedef half_t ve __attribute__((ext_vector_type(E)));
    auto &sk = lds.k;
    auto &sv = lds.v;
    auto &s_ok = lds.ok;
    const int tile_no = static_cast<int>(a.by_kv.div(static_cast<uint32_t>(block_no))), kh = block_no - tile_no * a.n_kv;
    const Tile tile = find_tile(a, ROWS, a.few, INT64_MAX, tile_no);
    if (tile.s < 0) return;
    const int s = tile.s, at = tile.at, first = tile.first, n_new = tile.n_new, ctx = tile.ctx, pos0 = ctx - n_new;
    const Span span = Q4 || SINKS ? tile_span(a, at, n_new, ctx) : Span(a, n_new, ctx);
    const int c = blockIdx.y;
    if (c >= span.n) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
    const int r0 = at * ROWS, n_rows = n_new * a.gqa - r0 < ROWS ? n_new * a.gqa - r0 : ROWS;
    int k0, k1;
    span.chunk_keys(a.chunk, c, k0, k1);
    const auto token_of = [&](int r) { return static_cast<int>(a.by_gqa.div(static_cast<uint32_t>(r))); };
    // all of the tile's rows see the keys from `from` to `upto`
    const int upto = pos0 + token_of(r0), from = a.window > 0 ? pos0 + token_of(r0 + n_rows - 1) - a.window + 1 : 0;
    int mid = 0, next = 0;
    {
        const int top = pos0 + token_of(r0 + n_rows - 1) + 1, bottom = a.window > 0 ? upto - a.window + 1 : 0;
        if constexpr (SINKS) {
            const SinkTiles tiles(span, bottom, KT, k0, k1);
            mid = tiles.mid;
            next = tiles.next;
        }
        if (k1 > top) k1 = top;
        if (!SINKS && k0 < bottom) k0 = bottom & ~(KT - 1);
    }
    const int shown = SINKS ? a.sinks : 0;  // and those before `shown`, up to `upto`
    auto after = [&](int kb) {  // the key tile that follows
        kb += KT;
        return SINKS && kb >= mid && kb < next ? next : kb;
    };
    // the wave's rows and the lane's
    const int wrows = n_rows - 32 * w < 32 ? n_rows - 32 * w : 32;
    const int row = r0 + 32 * w + (l32 < wrows ? l32 : wrows > 0 ? wrows - 1 : -32 * w);
    const int tok = token_of(row), head = kh * a.gqa + row - tok * a.gqa, pos = pos0 + tok;
    const int row_lo = a.window > 0 ? pos - a.window + 1 : 0;
    const int wfirst = pos0 + token_of(r0 + 32 * w), wlast = pos0 + token_of(wrows > 0 ? r0 + 32 * w + wrows - 1 : r0);
    half8_t qf[C];
    {
        const half_t *qr = a.q + (first + tok) * a.q_stride + static_cast<int64_t>(head) * D;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            qf[i] = *reinterpret_cast<const half8_t *>(qr + 16 * i + 8 * g);
            if (a.negate) qf[i] = -qf[i];
        }
    }
    const int in_page = (1 << a.batch.page_shift) - 1;
    const int64_t head_at = head_offset<D, Q4>(a, kh);
    // staging: wave w takes keys 16w .. 16w + 15 of a tile, one page; of 4-bit pages as words, a quarter of a key's row and
    // of the values what four keys have of E dimensions
    typedef uint32_t kw __attribute__((ext_vector_type(KL)));
    half8_t gk[KL];
    ve gv[4];
    kw gkw;
    uint32_t gks;
    u32x4 gvw, gvs;
    bool g_ok = false;
    uint32_t spoilt = 0;
    const int krow = lane / KCH, kch = lane % KCH, a4 = lane >> 4, db = lane & 15;
    const int32_t *table = a.batch.table + static_cast<int64_t>(s) * a.batch.max_pages;
    auto id_of = [&](int kb) {
        const int block = (kb + 16 * w) >> a.batch.page_shift;
        return table[block < a.batch.max_pages ? block : a.batch.max_pages - 1];
    };
    int next_id = id_of(k0 & ~(KT - 1));  // of the tile to be requested next
    auto load = [&](int kb) {  // past the last key: somewhere in page 0, for nothing, so that no branch holds a request
        const int key = kb + 16 * w, id = next_id;
        next_id = id_of(after(kb));
        g_ok = key < k1 && id >= 0 && id < a.batch.n_pages;
        if constexpr (Q4) {
            const int64_t base = (g_ok ? id : 0) * a.batch.page_stride + head_at;
            const int page = in_page + 1, slot = key & in_page;
            const uint8_t *kp = reinterpret_cast<const uint8_t *>(a.k) + base, *vp = reinterpret_cast<const uint8_t *>(a.v) + base;
            gkw = *reinterpret_cast<const kw *>(kp + Q4Row<D>::key_word(slot + (lane >> 2), KL * (lane & 3)));
            gks = *reinterpret_cast<const uint32_t *>(kp + Q4Row<D>::pair(page, slot + (lane >> 2), KL * (lane & 3) / 4));
            gvw = *reinterpret_cast<const u32x4 *>(vp + Q4Row<D>::value_word(slot + 4 * a4, E * db / 8));
            gvs = *reinterpret_cast<const u32x4 *>(vp + Q4Row<D>::pair(page, slot + 4 * a4, E * db / 32));
            return;
        }
        const int64_t base = (g_ok ? id : 0) * a.batch.page_stride + head_at + static_cast<int64_t>(key & in_page) * D;
#pragma unroll
        for (int i = 0; i < KL; ++i)
            gk[i] = *reinterpret_cast<const half8_t *>(a.k + base + (krow + i * (64 / KCH)) * D + kch * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) gv[j] = *reinterpret_cast<const ve *>(a.v + base + (4 * a4 + j) * D + E * db);
    };
    const Q4Bits bits;
    auto store = [&](int kb, int buf) {
        // slots that hold no position: 0 times what is there may be NaN
        const bool partly = !g_ok || kb + KT > k1 || (kb < from && !(SINKS && kb + KT <= shown)) || kb + KT - 1 > upto;
        const int kk = 16 * w + ((a4 & 1) << 3 | (a4 >> 1) << 2);
        auto put = [&](int e, half4_t x) {
            const int d = E * db + e;
            *reinterpret_cast<half4_t *>(&sv[buf][d * KT + (((kk >> 3) ^ d ^ (d >> 3)) & 7) * 8 + (kk & 4)]) = x;
        };
        if constexpr (Q4) {
#pragma unroll
            for (int i = 0; i < KL; ++i)
                *reinterpret_cast<half8_t *>(&sk[buf][(16 * w + (lane >> 2)) * KP + 8 * (KL * (lane & 3) + i)]) = q4_values(gkw[i], gks, bits);
            if (partly) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    gvs[j] = (!g_ok | (kb + 16 * w + 4 * a4 + j >= k1)) ? 0 : gvs[j];
            }
            uint32_t lo[2], hi[2];
            half2_t sd[2], sb[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                lo[t] = low_halves(gvw[2 * t], gvw[2 * t + 1]);
                hi[t] = high_halves(gvw[2 * t], gvw[2 * t + 1]);
                if (E == 4 && (db & 1)) {
                    lo[t] >>= 8;
                    hi[t] >>= 8;
                }
                sd[t] = __builtin_bit_cast(half2_t, low_halves(gvs[2 * t], gvs[2 * t + 1]));
                sb[t] = __builtin_bit_cast(half2_t, high_halves(gvs[2 * t], gvs[2 * t + 1]));
            }
            auto value = [&](int e) {
                half4_t x;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const half2_t y = __builtin_elementwise_fma(q4_codes(e & 1 ? hi[t] : lo[t], e >> 1, bits), sd[t], sb[t]);
                    x[2 * t] = y[0];
                    x[2 * t + 1] = y[1];
                }
                return x;
            };
            if (partly) {
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    half4_t x = value(e);
                    spoilt |= take_out<4>(x);
                    put(e, x);
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) put(e, value(e));
            }
        } else {
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                const int r = 16 * w + krow + i * (64 / KCH);
                *reinterpret_cast<half8_t *>(&sk[buf][r * KP + kch * 8]) = gk[i];
            }
            if (partly) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (!g_ok || kb + 16 * w + 4 * a4 + j >= k1) gv[j] = ve{};
#pragma unroll
                for (int j = 0; j < 4; ++j) spoilt |= take_out<E>(gv[j]);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) put(e, half4_t{gv[0][e], gv[1][e], gv[2][e], gv[3][e]});
        }
        if (lane == 0) s_ok[buf][w] = g_ok;
    };
    float m = -INFINITY, m2 = 0.0f, l = 0.0f;  // m2: what the weights are relative to in log2, anything while there is no m
    bool far = false;
    float16_t o[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    auto compute = [&](int kb, auto which) {
        constexpr int buf = decltype(which)::value;
        float16_t sc[2];
        half8_t kf[C][2];
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) kf[i][u] = *reinterpret_cast<const half8_t *>(&sk[buf][(32 * u + l32) * KP + 16 * i + 8 * g]);
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (i == 0)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[u][r] = 0.0f;
                sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[i][u], qf[i], sc[u], 0, 0, 0);
            }
        int ok[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) ok[t] = __builtin_amdgcn_readfirstlane(s_ok[buf][t]);
        // reads run four ahead of the products
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int i = 0; i < 2 * C; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        const bool whole = kb + KT - 1 <= wfirst && kb + KT <= k1 &&
                           (a.window == 0 || kb > wlast - a.window || (SINKS && kb + KT <= a.sinks)) &&
                           (ok[0] & ok[1] & ok[2] & ok[3]);
        if (!whole) {
            const int hi = (pos < k1 ? pos : k1 - 1) - kb - 4 * g, lo = row_lo - kb - 4 * g;  // of the key's place in the tile
            const int sink = a.sinks - kb - 4 * g;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at_key = 32 * u + 8 * (r >> 2) + (r & 3);
                    if (at_key > hi || (at_key < lo && !(SINKS && at_key < sink)) || !ok[2 * u + (r >> 3)]) sc[u][r] = -INFINITY;
                }
        }
        float mx = fmaxf(sc[0][0], sc[1][0]);
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(fmaxf(mx, sc[0][r]), sc[1][r]);
        mx = max_32_apart(mx);
        // weights are taken relative to m, an earlier maximum, until a row outgrows it by 2^kSlack: the sums
        // hold that as well, and few tiles after the first move it
        if (__any((mx - m) * a.scale2 > kSlack)) {
            mx = fmaxf(mx, m);
            const float f = exp2_fast(mx == -INFINITY ? 0.0f : (m - mx) * a.scale2);
            l *= f;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[d][r] *= f;
            m = mx;
            m2 = relative_to(m, a.scale2, kChunkBias, far);
        }
        if (far) {
            const float from_m = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[u][r] -= from_m;
        }
        half8_t pf[4];
        // the other workgroup's wave on this SIMD yields here, so that the two take turns between products and
        // softmax instead of meeting in both (2048 tokens after 7952: 363 -> 353 us)
        __builtin_amdgcn_s_setprio(1);
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = exp2_fast(__builtin_fmaf(sc[t >> 1][8 * (t & 1) + j], a.scale2, -m2));
                sum += x;
                pf[t][j] = static_cast<half_t>(x);
            }
        l += sum;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                const int dd = 32 * d + l32;
                const half8_t vf = *reinterpret_cast<const half8_t *>(&sv[buf][dd * KT + (((2 * t + g) ^ dd ^ (dd >> 3)) & 7) * 8]);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[t], o[d], 0, 0, 0);
            }
        __builtin_amdgcn_s_setprio(0);
    };
    int kb = k0 & ~(KT - 1), then = after(kb);  // the tile, and the one after it
    auto turn = [&](auto which) {
        constexpr int buf = decltype(which)::value;
        if (wrows > 0 && kb <= wlast && (a.window == 0 || kb + KT > wfirst - a.window + 1 || (SINKS && kb < a.sinks))) compute(kb, which);
        store(then, buf ^ 1);
        const int last = after(then);
        load(last);
        __syncthreads();
        kb = then;
        then = last;
    };
    if (kb < k1) {
        load(kb);
        store(kb, 0);
        load(then);
        __syncthreads();
        while (kb < k1) {
            turn(std::integral_constant<int, 0>{});
            if (kb < k1) turn(std::integral_constant<int, 1>{});
        }
    }
    const int met = __any(spoilt != 0);
    if (lane == 0) lds.spoilt[w] = met;
    __syncthreads();
    if (wrows <= 0) return;
    if (__builtin_expect(lds.spoilt[0] | lds.spoilt[1] | lds.spoilt[2] | lds.spoilt[3], 0)) {
        for (int t0 = k0 & ~(KT - 1); t0 < k1; t0 = after(t0)) {
            if (t0 + KT <= k1 && (t0 >= from || (SINKS && t0 + KT <= shown)) && t0 + KT - 1 <= upto) continue;
            for (int key = t0; key < t0 + KT && key < k1; ++key) {
                const int page = a.batch.page(s, key >> a.batch.page_shift);
                if (page < 0 || key > pos || (key < row_lo && !(SINKS && key < a.sinks))) continue;
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const half4_t v = taken<4>(value_run<D, Q4, 4>(a, page * a.batch.page_stride + head_at, key & in_page, 32 * d + 2 * r + 4 * g));
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[d][r + i] += static_cast<float>(v[i]);
                    }
            }
        }
    }
    l += __shfl_xor(l, 32, 64);
    const int64_t trow = static_cast<int64_t>(first + tok) * a.heads + head;
    if (l32 < wrows) {
        if (span.n > 1) {
            float *pr = a.part + (trow * a.nsplit + c) * (D + 4);
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<float4_t *>(pr + 32 * d + 2 * r + 4 * g) = float4_t{o[d][r], o[d][r + 1], o[d][r + 2], o[d][r + 3]};
            if (g == 0) {
                pr[D] = l;
                pr[D + 1] = m;
            }
        } else {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a row that sees no key is zero
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4) {
                    half4_t y;
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[i] = static_cast<half_t>(o[d][r + i] * inv);
                    *reinterpret_cast<half4_t *>(a.out + trow * D + 32 * d + 2 * r + 4 * g) = y;
                }
        }
    }
}

// ---------------------------------------------------------------- the kernels

template <int D, bool Q4, bool SINKS, bool ONCE>
__global__ __launch_bounds__(256, 2) void paged_attn_rows(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) RowsLds<D> lds;
    rows_tile<D, Q4, SINKS, ONCE>(a, lds, blockIdx.x);
}

// Batches with long chunks: the first `large` blocks are 128-row tiles, the rest the short chunks' 16-row
// ones, which fill the CUs that the long ones leave (a launch of its own after them: 37 us for the two chunks
// of 501 and 332 tokens beside 29 single ones, 28 so).
template <int D, bool Q4, bool SINKS>
__global__ __launch_bounds__(256, 2) void paged_attn_mixed(AttnArgs a, int large) {
    __shared__ __attribute__((aligned(16))) union {
        RowsLds<D> rows;
        ChunkLds<D> chunk;
    } lds;
    if (static_cast<int>(blockIdx.x) < large)
        chunk_tile<D, Q4, SINKS>(a, lds.chunk, blockIdx.x);
    else
        rows_tile<D, Q4, SINKS, false>(a, lds.rows, static_cast<int>(blockIdx.x) - large);
}

// ---------------------------------------------------------------- the chunks' states

// Join a row's chunks: out = sum_c num_c w_c / sum_c den_c w_c, w_c = 2^((m_c - M) scale2), M the largest m_c.
constexpr int kFewChunks = 8;

// By what a row's keys were cut into chunks.
enum Cut { kBySequence, kByTile, kShared };

// How many chunks token t's rows of the query heads head .. head + R - 1 were cut into.
template <Cut CUT, int R>
__device__ __forceinline__ void chunks_of_rows(const AttnArgs &a, int s, int t, int head, int first, int n_new, int (&n)[R]) {
    const int ctx = a.batch.length(s);
    if (CUT == kShared)
        n[0] = chunks_of(Span(a, n_new, ctx).blocks(), shared_blocks(a, Lane(a, threadIdx.x & 63)));
    else if (CUT == kBySequence || static_cast<int64_t>(n_new) * a.gqa <= a.few)
        n[0] = Span(a, n_new, ctx).n;
    else {
        int tile = -1;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int h = head + r, row = (t - first) * a.gqa + h - static_cast<int>(a.by_gqa.div(h)) * a.gqa;
            n[r] = r > 0 && row / 128 == tile ? n[r - 1] : tile_span(a, row / 128, n_new, ctx).n;
            tile = row / 128;
        }
        return;
    }
#pragma unroll
    for (int r = 1; r < R; ++r) n[r] = n[0];
}

// Up to kFewChunks: a wave for R heads of a token, which share its lookups, everything requested at once. 862 tokens of
// 16 heads over four chunks with 1 / 2 / 4 heads a wave: 7.3 / 5.6 / 6.5 us; with the chunks requested before it is known
// how many a row has 8.5.
template <int D, int R, Cut CUT>
__global__ __launch_bounds__(256) void paged_attn_merge_few(AttnArgs a) {
    constexpr int PER = D / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t trow = (static_cast<int64_t>(blockIdx.x) * 4 + wave) * R, rows = static_cast<int64_t>(a.batch.tokens) * a.heads;
    if (trow >= rows) return;
    const int t = static_cast<int>(trow / a.heads), s = a.batch.sequence_of(t);
    if (s >= a.batch.b) return;
    int first, n_new;
    a.batch.rows(s, first, n_new);
    if (t < first || t - first >= n_new) return;
    const int head0 = static_cast<int>(trow - static_cast<int64_t>(t) * a.heads);
    int n[R], most = 0;
    chunks_of_rows<CUT, R>(a, s, t, head0, first, n_new, n);
#pragma unroll
    for (int r = 0; r < R; ++r) most = n[r] > most ? n[r] : most;
    if (most <= 1) return;
    const float *pr = a.part + trow * a.nsplit * (D + 4);
    float mc[R][kFewChunks], lc[R][kFewChunks], v[R][kFewChunks][PER];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < kFewChunks; ++c)
            if (c < n[r]) {
                const float *pc = pr + static_cast<int64_t>(r * a.nsplit + c) * (D + 4);
                mc[r][c] = pc[D + 1];
                lc[r][c] = pc[D];
#pragma unroll
                for (int e = 0; e < PER; ++e) v[r][c][e] = pc[lane * PER + e];
            }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (n[r] <= 1) continue;
        float num[PER] = {}, den = 0.0f, m = -INFINITY;
#pragma unroll
        for (int c = 0; c < kFewChunks; ++c)
            if (c < n[r]) m = fmaxf(m, mc[r][c]);
        const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int c = 0; c < kFewChunks; ++c)
            if (c < n[r]) {
                const float f = exp2_fast((mc[r][c] - mu) * a.scale2);
                den += lc[r][c] * f;
#pragma unroll
                for (int e = 0; e < PER; ++e) num[e] += v[r][c][e] * f;
            }
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll
        for (int e = 0; e < PER; ++e) a.out[(trow + r) * D + lane * PER + e] = static_cast<half_t>(num[e] * inv);
    }
}

// More: a workgroup a row, wave w taking chunks w, w + 4, ..; 64 of its chunks at a time have their maxima and sums read
// by a lane each, then their rows follow with U requests in flight (5 tokens of 32 heads, 51 chunks: 19.6 us with a
// loop that carries the maximum along and waits for each, 5.1 so).
template <int D, Cut CUT>
__global__ __launch_bounds__(256) void paged_attn_merge(AttnArgs a) {
    constexpr int PER = D / 64, U = 8, W = 4;
    __shared__ float sm[W][D + 2];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t trow = blockIdx.x;
    const int t = static_cast<int>(trow / a.heads), s = a.batch.sequence_of(t);
    if (s >= a.batch.b) return;
    int first, n_new;
    a.batch.rows(s, first, n_new);
    if (t < first || t - first >= n_new) return;
    int of[1];
    chunks_of_rows<CUT, 1>(a, s, t, static_cast<int>(trow - static_cast<int64_t>(t) * a.heads), first, n_new, of);
    const int n = of[0];
    if (n <= 1) return;
    float num[PER] = {}, den = 0.0f, m = -INFINITY;
    const float *pr = a.part + trow * a.nsplit * (D + 4);
    for (int c0 = w; c0 < n; c0 += 64 * W) {
        const int mine = c0 + lane * W;
        const float mc = mine < n ? pr[static_cast<int64_t>(mine) * (D + 4) + D + 1] : -INFINITY;
        const float lc = mine < n ? pr[static_cast<int64_t>(mine) * (D + 4) + D] : 0.0f;
        float mx = mc;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
        mx = fmaxf(mx, m);
        const float mu = mx == -INFINITY ? 0.0f : mx, back = exp2_fast((m - mu) * a.scale2), f = exp2_fast((mc - mu) * a.scale2);
        float dl = lc * f;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) dl += __shfl_xor(dl, off, 64);
        den = den * back + dl;
        m = mx;
#pragma unroll
        for (int e = 0; e < PER; ++e) num[e] *= back;
        const int left = (n - c0 + W - 1) / W, count = left < 64 ? left : 64;
        const float *pc = pr + static_cast<int64_t>(c0) * (D + 4) + lane * PER;
        for (int i = 0; i < count; i += U) {
            float v[U][PER];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < PER; ++e)
                    v[u][e] = pc[static_cast<int64_t>((i + u < count ? i + u : count - 1) * W) * (D + 4) + e];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float fu = i + u < count ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), i + u)) : 0.0f;
#pragma unroll
                for (int e = 0; e < PER; ++e)
                    if (i + u < count) num[e] += v[u][e] * fu;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) sm[w][lane * PER + e] = num[e];
    if (lane == 0) {
        sm[w][D] = den;
        sm[w][D + 1] = m;
    }
    __syncthreads();
    if (w != 0) return;
    float mx = m;
#pragma unroll
    for (int u = 1; u < W; ++u) mx = fmaxf(mx, sm[u][D + 1]);
    const float mu = mx == -INFINITY ? 0.0f : mx, f0 = exp2_fast((m - mu) * a.scale2);
    den *= f0;
#pragma unroll
    for (int e = 0; e < PER; ++e) num[e] *= f0;
#pragma unroll
    for (int u = 1; u < W; ++u) {
        const float f = exp2_fast((sm[u][D + 1] - mu) * a.scale2);
        den += sm[u][D] * f;
#pragma unroll
        for (int e = 0; e < PER; ++e) num[e] += sm[u][lane * PER + e] * f;
    }
    const float inv = den == 0.0f ? 0.0f : 1.0f / den;
#pragma unroll
    for (int e = 0; e < PER; ++e) a.out[trow * D + lane * PER + e] = static_cast<half_t>(num[e] * inv);
}

// ---------------------------------------------------------------- the launch

struct Plan {
    int64_t small, large;  // tiles of 16 and of 128 rows, at most
    int64_t few;           // rows of a sequence up to which it goes to the small ones
    int chunk, nsplit;
    int target;            // units of a kv head where the device shares the keys out, or 0
    bool once;             // keys and values are read once and not kept
};

// Sequences of up to kFew rows go to the 16-row tiles, the others to the 128-row ones: 64 sequences after 2000 keys
// (32 heads over 8, D = 128) take 107 / 118 us with 16 / 32 rows each in the small tiles and 131 / 124 in the large;
// with 48 rows 151 and 126. A batch without longer chunks has no 128-row tile; one sequence alone goes where its
// chunk does.
constexpr int64_t kFew = 32;
// The keys are cut into chunks until the tiles fill the chip's workgroups, of kMinChunk keys at least. kFillSmall 512 /
// 1024 / 2048 / 4096: 48 tokens over up to 1536 keys each 40 / 35 / 36 / 37 us, 5 over 65000 82 / 79 / 79 / 84;
// kFillLarge 256 / 384 / 512: a batch of two chunks and 30 tokens 28.7 / 28.4 / 29.8. Contexts of up to kWhole keys are not cut, whose second launch costs more than it
// saves. In a captured graph, one token of 8 kv heads over 256 / 384 / 448 / 512 keys: 6.8 / 8.1 / 8.8 / 9.1 us whole,
// 8.0 / 8.2 / 8.2 / 8.3 cut (4 of D = 64: 5.6 / 6.6 / 7.2 / 7.3 and 7.2 / 7.4 / 7.5 / 7.5). From 128 tiles on, twice that
// (16 tokens of 8 kv heads over 512 / 768 / 1024: 10.9 / 15.7 / 19.2 whole, 13.1 / 15.7 / 19.0 cut).
constexpr int64_t kFillSmall = 1024, kFillLarge = 384, kWhole = 384;

// Where the device shares the keys out (a token or a few of each sequence, over 4-bit pages or with sinks):
constexpr int64_t kFillShared = 1024, kShareBytes = int64_t(64) << 20;

// Where one tile of a sequence reads its keys, and all of them are too many for two such calls (two layers) in turn to find them
// in the 256 MB cache before the memory, they are read past it. Over others' data in between, 64 tokens under a window of 2048 (f16,
// D = 64, 134 MB) 32.5 us kept and 28.5 so, 5 over up to 65000 (4 bits, 132 MB) 34.4 and 32.4; again over the same data 27.7 and
// 28.5, 27.1 and 27.8; 48 over up to 1536 (4 bits, 49 MB) 17.6 and 17.9. With two tiles (30 sequences of 6 tokens of 4 heads over 20000,
// f16) 530 and 711. The host knows the longest context alone, which stands for all of them: a batch with one long sequence among short
// ones is read past the caches although its keys would stay there, at those 3 %. f16 pages without sinks are kept: 5 over up to
// 65000 of D = 64 33.0 and 39.4 over the same data.
constexpr double kKeptBytes = 128 << 20;

// How far to cut 128-row tiles over 4-bit pages or with sinks. A tile's time is a fixed part and one for each 64 keys, which
// depend on how many workgroups share its CU (us; 128 and 1152 keys on 2, 256 and 512 workgroups, D = 64 then 128, three
// of D = 64 taken to go on like that): cut, more of them run at once, but each begins anew, and their states are joined. Of the
// cuts that fill the chip once or a few times, the cheapest by that. (Fitted on one card: another one's times would choose other
// cuts, never other results but for their last bits. Batches over f16 pages without sinks keep kFillLarge.) 700 and 615 tokens of 8
// query heads under a window of 1000 (166 tiles): 46 us in two, 38 uncut; 1025 of 4 after 5975 (264 tiles): 202 in two, 179 in three.
inline int64_t cheapest_cut(int64_t wgs, int64_t blocks, int64_t rows, int64_t hd) {
    struct Tile {
        float fixed, block;
    };
    constexpr Tile kNarrow[] = {{7.0f, 1.05f}, {9.0f, 1.57f}, {11.0f, 2.2f}}, kWide[] = {{9.5f, 1.45f}, {13.0f, 2.4f}};
    const int full = hd == 64 ? 3 : 2;  // workgroups a CU holds
    const Tile *of = hd == 64 ? kNarrow : kWide;
    int64_t best = 1;
    float least = 0.0f;
    for (int64_t fill = 0; fill <= 5; ++fill) {
        const int64_t n = fill == 0 ? 1 : kNumCUs * fill / wgs;
        if (n < 1 || (n == 1 && fill > 0)) continue;
        const int64_t all = wgs * n, rounds = all / (kNumCUs * full), left = all - rounds * kNumCUs * full;
        const float keys = static_cast<float>((blocks + n - 1) / n);
        const auto time = [&](int share) { return of[share - 1].fixed + of[share - 1].block * keys; };
        float t = static_cast<float>(rounds) * time(full);
        if (left > 0) t += time(static_cast<int>((left + kNumCUs - 1) / kNumCUs));
        if (n > 1) t += 3.0f + static_cast<float>(rows * n * (hd + 4) * 4) / 5e6f;  // joined at 5 TB/s
        if (fill == 0 || t < least) {
            least = t;
            best = n;
        }
    }
    return best;
}

inline Plan plan_of(int64_t tokens, int64_t b, int64_t gqa, int64_t n_kv, int64_t max_q, int64_t max_context, int64_t window,
                    int64_t sinks, int64_t hd, bool share, bool own) {
    Plan p;
    p.target = 0;
    const int64_t rows = tokens * gqa, live = b < tokens ? b : tokens;
    if (max_q * gqa <= kFew) {
        p.few = INT64_MAX;
        p.small = (rows + 15 * live) / 16;
        p.large = 0;
    } else if (b == 1) {
        p.few = 0;
        p.small = 0;
        p.large = (rows + 127) / 128;
    } else {
        p.few = kFew;
        p.small = (rows + 15 * live) / 16 < live * (kFew / 16) ? (rows + 15 * live) / 16 : live * (kFew / 16);
        const int64_t most = rows / (kFew + 1) < live ? rows / (kFew + 1) : live;  // sequences of that many rows
        p.large = (rows + 127 * most) / 128;
    }
    const int64_t tile = 128 / gqa + 2, q = own && p.large > 0 && tile < max_q ? tile : max_q;  // a 128-row tile's tokens
    const int64_t seen = window + q + 63 + (sinks > 0 ? sinks + 63 : 0);
    int64_t span = window > 0 && seen < max_context ? seen : max_context;
    if (span < 1) span = 1;
    if (span > int64_t(1) << 30) span = int64_t(1) << 30;  // no table holds more
    // the launch is sized for the most tiles there can be; the chunks go by what a batch of long chunks has
    const int64_t wgs = (p.large > 0 ? (own && b == 1 ? p.large : rows / 128 + 1) : p.small) * n_kv, whole = wgs < 128 ? kWhole : 2 * kWhole;
    int64_t n = ((p.large > 0 ? kFillLarge : kFillSmall) + wgs - 1) / wgs;
    const int64_t most = span <= whole ? 1 : (span + kMinChunk - 1) / kMinChunk;
    if (own && p.large > 0) n = cheapest_cut(wgs, (span + 63) / 64, rows * n_kv, hd);
    if (n > most) n = most;
    p.chunk = static_cast<int>(((span + n - 1) / n + 63) / 64 * 64);
    p.nsplit = static_cast<int>((span + p.chunk - 1) / p.chunk);
    const int64_t row_bytes = share ? 5 * hd / 4 : 4 * hd;  // a key's and its value's; share: of 4-bit pages
    p.once = own && p.large == 0 && max_q * gqa <= 16 && static_cast<double>(live * n_kv * row_bytes) * static_cast<double>(span) > kKeptBytes;
    if (share && p.large == 0 && p.nsplit > 1) {
        // room for chunks of kMinChunk keys, as many as a kv head has units or kShareBytes of states hold
        const int64_t left = kFillShared / n_kv - p.small / 2;  // a tile's last chunk is half a one
        p.target = static_cast<int>(left > p.small ? left : p.small);
        int64_t room = kFewChunks;
        if (p.nsplit > kFewChunks / 2) {
            room = kShareBytes / (tokens * gqa * n_kv * (hd + 4) * static_cast<int64_t>(sizeof(float)));
            room = room < p.target ? room : p.target;
        }
        room = room < most ? room : most;
        if (room > p.nsplit) p.nsplit = static_cast<int>(room);
    }
    return p;
}

inline size_t part_bytes(const Plan &p, int64_t tokens, int64_t heads, int64_t hd) {
    return p.nsplit > 1 ? static_cast<size_t>(tokens * heads * p.nsplit * (hd + 4)) * sizeof(float) : 0;
}

template <int D, Cut CUT>
hipError_t merge(const AttnArgs &a, hipStream_t stream) {
    const int64_t rows = static_cast<int64_t>(a.batch.tokens) * a.heads;
    if (a.nsplit <= kFewChunks && a.heads % 2 == 0)
        paged_attn_merge_few<D, 2, CUT><<<static_cast<unsigned>((rows / 2 + 3) / 4), 256, 0, stream>>>(a);
    else if (a.nsplit <= kFewChunks)
        paged_attn_merge_few<D, 1, CUT><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, stream>>>(a);
    else
        paged_attn_merge<D, CUT><<<static_cast<unsigned>(rows), 256, 0, stream>>>(a);
    return hipGetLastError();
}

template <int D, bool Q4, bool SINKS>
hipError_t launch(const AttnArgs &a, const Plan &p, hipStream_t stream) {
    if (p.large > 0)
        paged_attn_mixed<D, Q4, SINKS><<<dim3(static_cast<unsigned>((p.large + p.small) * a.n_kv), a.nsplit), 256, 0, stream>>>(
            a, static_cast<int>(p.large * a.n_kv));
    else {
        const dim3 grid = a.target > 0 ? dim3(static_cast<unsigned>((p.small + a.target + 1) * a.n_kv))
                                       : dim3(static_cast<unsigned>(p.small * a.n_kv), a.nsplit);
        if ((Q4 || SINKS) && p.once)
            paged_attn_rows<D, Q4, SINKS, Q4 || SINKS><<<grid, 256, 0, stream>>>(a);
        else
            paged_attn_rows<D, Q4, SINKS, false><<<grid, 256, 0, stream>>>(a);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1) return e;
    if (Q4 && a.target > 0) return merge<D, Q4 ? kShared : kBySequence>(a, stream);
    return merge<D, Q4 || SINKS ? kByTile : kBySequence>(a, stream);
}

inline bool plannable(int64_t tokens, int64_t b, int64_t heads, int64_t n_kv, int64_t hd, int64_t max_q, int64_t max_context,
                      int64_t window, int64_t sinks) {
    return sinks >= 0 && sinks < (int64_t(1) << 31) && tokens > 0 && b > 0 && n_kv > 0 && heads > 0 && heads % n_kv == 0 && hd > 0 && max_q > 0 && max_context > 0 && window >= 0 &&
           tokens < (int64_t(1) << 24) && b <= kMaxSeqs && heads <= 65536 && hd <= 128 && max_q < (int64_t(1) << 31) &&
           max_context < (int64_t(1) << 31) && window < (int64_t(1) << 31);
}

template <bool Q4, bool SINKS>
hipError_t launch_for(int64_t head_dim, const AttnArgs &a, const Plan &p, hipStream_t stream) {
    return head_dim == 128 ? launch<128, Q4, SINKS>(a, p, stream) : launch<64, Q4, SINKS>(a, p, stream);
}

int attention(const char *name, int bits, const dtts_f16 *q, const void *kpages, const void *vpages, const int32_t *q_start,
              const int32_t *context, const int32_t *page_table, dtts_f16 *out, int64_t tokens, int64_t b, int64_t heads, int64_t n_kv,
              int64_t head_dim, int64_t page, int64_t n_pages, int64_t max_pages, int64_t page_stride, int64_t q_stride, int64_t max_q,
              int64_t max_context, int64_t window, int64_t sinks, float scale, void *workspace, size_t ws_bytes, hipStream_t stream) {
    DTTS_REQUIRE(bits == 16 || bits == 4, "%s: pages of %d bits (16 or 4)", name, bits);
    const int64_t units = bits == 16 ? head_dim : 5 * head_dim / 8;
    DTTS_REQUIRE_PAGED_ROWS(name, tokens, b, n_kv, head_dim, page, n_pages, max_pages, page_stride, units, bits == 16 ? 8 : 16);
    DTTS_REQUIRE(heads > 0 && heads <= 65536 && heads % n_kv == 0, "%s: %lld heads over %lld kv heads", name, (long long)heads,
                 (long long)n_kv);
    DTTS_REQUIRE(q_stride >= heads * head_dim && q_stride % 8 == 0, "%s: q_stride %lld (a multiple of 8, at least heads * head_dim)",
                 name, (long long)q_stride);
    DTTS_REQUIRE(window >= 0 && window < (int64_t(1) << 31), "%s: window %lld", name, (long long)window);
    DTTS_REQUIRE(sinks >= 0 && sinks < (int64_t(1) << 31), "%s: sinks %lld", name, (long long)sinks);
    if (tokens == 0 || b == 0) return DTTS_OK;
    DTTS_REQUIRE(max_q > 0 && max_context > 0 && max_q < (int64_t(1) << 31) && max_context < (int64_t(1) << 31),
                 "%s: max_q %lld, max_context %lld", name, (long long)max_q, (long long)max_context);
    DTTS_REQUIRE(q && kpages && vpages && q_start && context && page_table && out, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(q, 16) && aligned(kpages, 16) && aligned(vpages, 16) && aligned(out, 16) && aligned(q_start, 4) &&
                     aligned(context, 4) && aligned(page_table, 4),
                 "%s: misaligned operand", name);
    DTTS_REQUIRE(std::isfinite(scale * kLog2e), "%s: scale %g", name, static_cast<double>(scale));
    if (window == 0) sinks = 0;  // every token sees them
    const bool share = bits == 4, own = bits == 4 || (sinks > 0 && window < int64_t(1) << 30);
    Plan p = plan_of(tokens, b, heads / n_kv, n_kv, max_q, max_context, window, sinks, head_dim, share, own);
    DTTS_REQUIRE(tokens * heads < (int64_t(1) << 31) && (p.small + p.large + (p.target > 0 ? p.target + 1 : 0)) * n_kv < (int64_t(1) << 24),
                 "%s: too many rows", name);
    const int64_t row = heads * head_dim * static_cast<int64_t>(sizeof(half_t));
    DTTS_REQUIRE(q_stride < (int64_t(1) << 62), "%s: q_stride %lld", name, (long long)q_stride);
    DTTS_REQUIRE(!share_bytes({q, tokens, q_stride * static_cast<int64_t>(sizeof(half_t)), row}, {out, 1, 0, tokens * row}),
                 "%s: the output may not be the queries, nor a part of their memory", name);
    AttnArgs a;
    a.batch = PagedBatch{q_start, context, page_table, static_cast<int>(tokens), static_cast<int>(b), log2_of(page),
                         static_cast<int>(n_pages), static_cast<int>(max_pages), page_stride};
    a.q = reinterpret_cast<const half_t *>(q);
    a.k = static_cast<const half_t *>(kpages);
    a.v = static_cast<const half_t *>(vpages);
    a.out = reinterpret_cast<half_t *>(out);
    a.q_stride = q_stride;
    a.heads = static_cast<int>(heads);
    a.n_kv = static_cast<int>(n_kv);
    a.gqa = static_cast<int>(heads / n_kv);
    // one of 2^30 reaches past every position that a table holds, and the differences below stay ints
    a.window = window >= int64_t(1) << 30 ? 0 : static_cast<int>(window);
    a.sinks = a.window == 0 ? 0 : sinks >= int64_t(1) << 30 ? 1 << 30 : static_cast<int>(sinks);
    // a scale of 0 is the smallest number: every score then is 0, and a masked one still -inf
    a.scale2 = fmaxf(fabsf(scale) * kLog2e, FLT_MIN);
    a.negate = scale < 0.0f;
    a.few = p.few;
    a.part = nullptr;
    if (p.nsplit > 1 && workspace && ws_bytes >= part_bytes(p, tokens, heads, head_dim)) {
        DTTS_REQUIRE(aligned(workspace, 16), "%s: misaligned workspace", name);
        a.part = static_cast<float *>(workspace);
    } else {
        p.nsplit = 1;  // one workgroup takes all of a tile's keys
        p.target = 0;
    }
    a.target = p.target;
    a.per_target = 1.0f / static_cast<float>(p.target > 0 ? p.target : 1);
    a.by_kv = FastDiv(static_cast<uint32_t>(n_kv));
    a.by_gqa = FastDiv(static_cast<uint32_t>(heads / n_kv));
    a.chunk = p.chunk;
    a.by_chunk = FastDiv(static_cast<uint32_t>(p.chunk));
    a.nsplit = p.nsplit;
    const auto fn = bits == 16 ? (a.sinks > 0 ? launch_for<false, true> : launch_for<false, false>)
                               : (a.sinks > 0 ? launch_for<true, true> : launch_for<true, false>);
    DTTS_HIP_CHECK(fn(head_dim, a, p, stream), name);
    return DTTS_OK;
}

}  // namespace
}  // namespace dtts

extern "C" size_t dtts_paged_attention_sinks_workspace_bytes(int32_t bits, int64_t tokens, int64_t b, int64_t heads, int64_t n_kv,
                                                             int64_t head_dim, int64_t max_q, int64_t max_context, int64_t window,
                                                             int64_t sinks) {
    using namespace dtts;
    if ((bits != 16 && bits != 4) || !plannable(tokens, b, heads, n_kv, head_dim, max_q, max_context, window, sinks)) return 0;
    if (window == 0) sinks = 0;
    const bool share = bits == 4, own = bits == 4 || (sinks > 0 && window < int64_t(1) << 30);
    return part_bytes(plan_of(tokens, b, heads / n_kv, n_kv, max_q, max_context, window, sinks, head_dim, share, own), tokens, heads, head_dim);
}

extern "C" size_t dtts_paged_attention_workspace_bytes(int64_t tokens, int64_t b, int64_t heads, int64_t n_kv, int64_t head_dim,
                                                       int64_t max_q, int64_t max_context, int64_t window) {
    return dtts_paged_attention_sinks_workspace_bytes(16, tokens, b, heads, n_kv, head_dim, max_q, max_context, window, 0);
}

extern "C" int dtts_paged_attention(int32_t bits, const dtts_f16 *q, const void *kpages, const void *vpages, const int32_t *q_start,
                                    const int32_t *context, const int32_t *page_table, dtts_f16 *out, int64_t tokens, int64_t b,
                                    int64_t heads, int64_t n_kv, int64_t head_dim, int64_t page, int64_t n_pages, int64_t max_pages,
                                    int64_t page_stride, int64_t q_stride, int64_t max_q, int64_t max_context, int64_t window,
                                    int64_t sinks, float scale, void *workspace, size_t ws_bytes, hipStream_t stream) {
    return dtts::attention("dtts_paged_attention", bits, q, kpages, vpages, q_start, context, page_table, out, tokens, b, heads, n_kv,
                           head_dim, page, n_pages, max_pages, page_stride, q_stride, max_q, max_context, window, sinks, scale, workspace,
                           ws_bytes, stream);
}

extern "C" int dtts_paged_attention_f16(const dtts_f16 *q, const dtts_f16 *kpages, const dtts_f16 *vpages, const int32_t *q_start,
                                        const int32_t *context, const int32_t *page_table, dtts_f16 *out, int64_t tokens,
                                        int64_t b, int64_t heads, int64_t n_kv, int64_t head_dim, int64_t page, int64_t n_pages,
                                        int64_t max_pages, int64_t page_stride, int64_t q_stride, int64_t max_q,
                                        int64_t max_context, int64_t window, float scale, void *workspace, size_t ws_bytes,
                                        hipStream_t stream) {
    return dtts::attention("dtts_paged_attention_f16", 16, q, kpages, vpages, q_start, context, page_table, out, tokens, b, heads, n_kv,
                           head_dim, page, n_pages, max_pages, page_stride, q_stride, max_q, max_context, window, 0, scale, workspace,
                           ws_bytes, stream);
}
