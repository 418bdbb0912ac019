// Attention of each sequence's new tokens over its paged f16 cache: out_i = sum_j softmax_j(scale
// q_i . k_j) v_j over p_i - window < j <= p_i, a ragged batch of chunks and single tokens.
//
// A row is one (new token, query head). The heads / n_kv query heads of a kv head read the same keys,
// so rows are numbered token * gqa + head within (sequence, kv head), and a tile of consecutive rows goes to one
// workgroup: 16 rows where a sequence has few, 128 where it has a chunk. A query's scores, softmax state (running maximum,
// running sum) and output sums are f32; q, k, v are f16 as the cache and the matrix cores hold them;
// the weights e^(s - max) are rounded to f16 for the second product, and the output is rounded once. The weights are
// held times 2^kBias (it cancels in the division by their sum), at the upper end of f16's range: down to 2^(-14 - kBias) of
// the largest each is off by 2^-11 relative at most, as the output's own rounding is, and below that by 2^(-25 - kBias) of
// the largest. Without it a flat tail far under one leading key would leave the numerator and stay in the denominator
// (65000 keys e^-17.5 below one: all of their 0.16 %). For the same reason a tile's weights are summed before they meet
// the running sum, next to which a single one may be nothing.
#include <cfloat>
#include <cmath>
#include <type_traits>

#include "paged.hpp"

namespace dtts {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

struct AttnArgs {
    PagedBatch batch;
    const half_t *q, *k, *v;
    half_t *out;
    float *part;       // per (row, chunk): D weighted sums, the weight sum, the maximum of q . k
    int64_t q_stride;  // elements between tokens
    int heads, n_kv, gqa, window;
    float scale2;      // |scale| * log2(e), above 0: the softmax runs in base 2, its maxima are those of q . k
    bool negate;       // scale < 0: the queries change sign
    int chunk, nsplit; // keys per chunk, chunks at most (the last takes what is left)
    int64_t few;       // sequences of at most this many rows go to the 16-row tiles
};

// The keys that sequence s's rows see, in chunks: [lo, hi), lo a multiple of 64, `n` chunks. hi stops
// at the table's end, whatever the context says.
struct Span {
    int lo, hi, n;
    __device__ __forceinline__ Span(const AttnArgs &a, int s, int n_new, int ctx) {
        const int64_t cap = static_cast<int64_t>(a.batch.max_pages) << a.batch.page_shift;
        hi = ctx < 0 ? 0 : ctx < cap ? ctx : static_cast<int>(cap);
        lo = a.window > 0 && ctx - n_new - a.window + 1 > 0 ? (ctx - n_new - a.window + 1) & ~63 : 0;
        if (lo > hi) lo = hi & ~63;
        n = static_cast<int>((static_cast<int64_t>(hi) - lo + a.chunk - 1) / a.chunk);
        n = n < 1 ? 1 : n > a.nsplit ? a.nsplit : n;
    }
    __device__ __forceinline__ void chunk_keys(const AttnArgs &a, int c, int &k0, int &k1) const {
        k0 = lo + c * a.chunk;
        k1 = c == n - 1 ? hi : k0 + a.chunk;
    }
};

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

// What the exponents of the weights are raised by. The 16-row tiles' largest weight is 2^15, the 128-row ones' up to
// 2^kSlack times 2^kChunkBias (their maximum may lag behind by that): both under f16's 65504. kSlack 1 / 4 / 8 (and a
// bias that goes with it): 2048 tokens after 7952 335 / 333 / 335 us.
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
template <int D>
struct KvTile {
    static constexpr int E = D / 16;  // dimensions a lane holds of each of its 8 value rows
    typedef half_t ve __attribute__((ext_vector_type(E)));
    half8_t k[2][D / 32];
    ve v[8];
    int ok;  // bit u: keys 16u .. 16u + 15 have a page
};

template <int D>
struct RowsLds {
    float o[4][16][D + 4], m[4][16], l[4][16];
};

template <int D>
__device__ __forceinline__ void rows_tile(const AttnArgs &a, RowsLds<D> &lds, int block) {
    constexpr int C = D / 32, E = D / 16, ROWS = 16;
    auto &sm_o = lds.o;
    auto &sm_m = lds.m;
    auto &sm_l = lds.l;
    const int kh = block % a.n_kv;
    const Tile tile = find_tile(a, ROWS, 0, a.few, block / a.n_kv);
    if (tile.s < 0) return;
    const int s = tile.s, at = tile.at, first = tile.first, n_new = tile.n_new, ctx = tile.ctx;
    const Span span(a, s, n_new, ctx);
    const int c = blockIdx.y;
    if (c >= span.n) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int n_rows = n_new * a.gqa - at * ROWS < ROWS ? n_new * a.gqa - at * ROWS : ROWS;
    // the lane's row: token `tok` of the sequence, query head kh * gqa + head
    const int row = at * ROWS + (l16 < n_rows ? l16 : n_rows - 1);
    const int tok = row / a.gqa, head = kh * a.gqa + row - tok * a.gqa;
    const int pos = ctx - n_new + tok;
    const int first_tok = at * ROWS / a.gqa, last_tok = (at * ROWS + n_rows - 1) / a.gqa;
    int k0, k1;  // the tile's keys in this chunk
    span.chunk_keys(a, c, k0, k1);
    const int row_lo = a.window > 0 ? pos - a.window + 1 : 0;
    // one of the tile's rows at least sees the keys [bottom, k1), all of them [from, end)
    const bool one_token = first_tok == last_tok;
    const int bottom = a.window > 0 ? ctx - n_new + first_tok - a.window + 1 : 0;
    const int from = a.window > 0 ? bottom + last_tok - first_tok : 0;
    int end = ctx - n_new + first_tok + 1;
    {
        const int top = ctx - n_new + last_tok + 1;
        if (k1 > top) k1 = top;
        if (k0 < bottom) k0 = bottom & ~31;
        if (end > k1) end = k1;
    }
    half8_t qf[C];
    {
        const half_t *qr = a.q + (first + tok) * a.q_stride + static_cast<int64_t>(head) * D;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            qf[i] = *reinterpret_cast<const half8_t *>(qr + 32 * i + 8 * g);
            if (a.negate) qf[i] = -qf[i];
        }
    }
    const int in_page = (1 << a.batch.page_shift) - 1;
    const int64_t head_at = (static_cast<int64_t>(kh) << a.batch.page_shift) * D;
    auto load = [&](int kb, KvTile<D> &t) {
        t.ok = 0;
        int64_t base[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int key = kb + 16 * u;
            const int page = key < k1 ? a.batch.page(s, key >> a.batch.page_shift) : -1;
            if (page >= 0) t.ok |= 1 << u;
            base[u] = (page < 0 ? 0 : page) * a.batch.page_stride + head_at + static_cast<int64_t>(key & in_page) * D;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < C; ++i)
                t.k[u][i] = *reinterpret_cast<const half8_t *>(a.k + base[u] + l16 * D + 32 * i + 8 * g);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            t.v[j] = *reinterpret_cast<const typename KvTile<D>::ve *>(a.v + base[j >> 2] + (4 * g + (j & 3)) * D + E * l16);
    };
    float m = -INFINITY, m2 = 0.0f, l = 0.0f;  // m2: what the weights are relative to in log2, anything while there is no m
    bool far = false;
    uint32_t spoilt = 0;
    float4_t o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = float4_t{0.f, 0.f, 0.f, 0.f};
    auto compute = [&](int kb, KvTile<D> &t) {
        float4_t sc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            sc[u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < C; ++i) sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(t.k[u][i], qf[i], sc[u], 0, 0, 0);
        }
        float mx = m;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = kb + 16 * u + 4 * g + i;
                const bool seen = key <= pos && key >= row_lo && key < k1 && (t.ok >> u & 1);
                sc[u][i] = seen ? sc[u][i] : -INFINITY;
                mx = fmaxf(mx, sc[u][i]);
            }
        // the row's other keys are 16 and 32 lanes away
        mx = max_16_32_apart(mx);
        if (__any(mx > m)) {
            const float f = exp2_fast(mx == -INFINITY ? 0.0f : (m - mx) * a.scale2);
            l *= f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= f;
            m = mx;
            m2 = relative_to(m, a.scale2, kBias, far);
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
        // what no row sees holds anything: 0 times it may be NaN
        if (kb < from || kb + 32 > end || t.ok != 3) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = kb + 16 * (j >> 2) + 4 * g + (j & 3);
                if (key >= k1 || key < bottom || !(t.ok >> (j >> 2) & 1)) t.v[j] = typename KvTile<D>::ve{};
            }
            if (!one_token && (kb < from || kb + 32 > end)) {
#pragma unroll
                for (int j = 0; j < 8; ++j) spoilt |= take_out<E>(t.v[j]);
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            half8_t f;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = t.v[j][e];
            o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, p, o[e], 0, 0, 0);
        }
    };
    KvTile<D> t;
    for (int kb = (k0 & ~31) + 32 * w; kb < k1; kb += 128) {
        load(kb, t);
        compute(kb, t);
    }
    if (__builtin_expect(__any(spoilt != 0), 0)) {
        for (int kb = (k0 & ~31) + 32 * w; kb < k1; kb += 128) {
            if (kb >= from && kb + 32 <= end) continue;
            for (int key = kb; key < kb + 32 && key < k1; ++key) {
                const int page = a.batch.page(s, key >> a.batch.page_shift);
                if (page < 0 || key > pos || key < row_lo) continue;
                const half_t *vr = a.v + page * a.batch.page_stride + head_at + static_cast<int64_t>(key & in_page) * D + 4 * E * g;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const auto v = taken<E>(*reinterpret_cast<const typename KvTile<D>::ve *>(vr + E * i));
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
    const int rr = at * ROWS + (r < n_rows ? r : n_rows - 1), rtok = rr / a.gqa, rhead = kh * a.gqa + rr - rtok * a.gqa;
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
            typename KvTile<D>::ve y;
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = static_cast<half_t>(num[e] * inv);
            *reinterpret_cast<typename KvTile<D>::ve *>(a.out + trow * D + E * l16) = y;
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

template <int D>
__device__ __forceinline__ void chunk_tile(const AttnArgs &a, ChunkLds<D> &lds, int block_no) {
    constexpr int ROWS = 128, KT = 64, E = D / 16, C = D / 16, KL = D / 32;  // C: k steps, KL: 16-byte key loads a thread
    constexpr int KCH = D / 8, KP = ChunkLds<D>::KP;                         // KCH: 16-byte pieces of a key row
    typedef half_t ve __attribute__((ext_vector_type(E)));
    auto &sk = lds.k;
    auto &sv = lds.v;
    auto &s_ok = lds.ok;
    const int kh = block_no % a.n_kv;
    const Tile tile = find_tile(a, ROWS, a.few, INT64_MAX, block_no / a.n_kv);
    if (tile.s < 0) return;
    const int s = tile.s, at = tile.at, first = tile.first, n_new = tile.n_new, ctx = tile.ctx, pos0 = ctx - n_new;
    const Span span(a, s, n_new, ctx);
    const int c = blockIdx.y;
    if (c >= span.n) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l32 = lane & 31, g = lane >> 5;
    const int r0 = at * ROWS, n_rows = n_new * a.gqa - r0 < ROWS ? n_new * a.gqa - r0 : ROWS;
    int k0, k1;
    span.chunk_keys(a, c, k0, k1);
    // all of the tile's rows see the keys from `from` to `upto`
    const int upto = pos0 + r0 / a.gqa, from = a.window > 0 ? pos0 + (r0 + n_rows - 1) / a.gqa - a.window + 1 : 0;
    {
        const int top = pos0 + (r0 + n_rows - 1) / a.gqa + 1, bottom = a.window > 0 ? upto - a.window + 1 : 0;
        if (k1 > top) k1 = top;
        if (k0 < bottom) k0 = bottom & ~(KT - 1);
    }
    // the wave's rows and the lane's
    const int wrows = n_rows - 32 * w < 32 ? n_rows - 32 * w : 32;
    const int row = r0 + 32 * w + (l32 < wrows ? l32 : wrows > 0 ? wrows - 1 : -32 * w);
    const int tok = row / a.gqa, head = kh * a.gqa + row - tok * a.gqa, pos = pos0 + tok;
    const int row_lo = a.window > 0 ? pos - a.window + 1 : 0;
    const int wfirst = pos0 + (r0 + 32 * w) / a.gqa, wlast = pos0 + (r0 + 32 * w + wrows - 1) / a.gqa;
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
    const int64_t head_at = (static_cast<int64_t>(kh) << a.batch.page_shift) * D;
    // staging: wave w takes keys 16w .. 16w + 15 of a tile, one page
    half8_t gk[KL];
    ve gv[4];
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
        next_id = id_of(kb + KT);
        g_ok = key < k1 && id >= 0 && id < a.batch.n_pages;
        const int64_t base = (g_ok ? id : 0) * a.batch.page_stride + head_at + static_cast<int64_t>(key & in_page) * D;
#pragma unroll
        for (int i = 0; i < KL; ++i)
            gk[i] = *reinterpret_cast<const half8_t *>(a.k + base + (krow + i * (64 / KCH)) * D + kch * 8);
#pragma unroll
        for (int j = 0; j < 4; ++j) gv[j] = *reinterpret_cast<const ve *>(a.v + base + (4 * a4 + j) * D + E * db);
    };
    auto store = [&](int kb, int buf) {
#pragma unroll
        for (int i = 0; i < KL; ++i) {
            const int r = 16 * w + krow + i * (64 / KCH);
            *reinterpret_cast<half8_t *>(&sk[buf][r * KP + kch * 8]) = gk[i];
        }
        if (!g_ok || kb + KT > k1 || kb < from || kb + KT - 1 > upto) {  // slots that hold no position: 0 times what is there may be NaN
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (!g_ok || kb + 16 * w + 4 * a4 + j >= k1) gv[j] = ve{};
#pragma unroll
            for (int j = 0; j < 4; ++j) spoilt |= take_out<E>(gv[j]);
        }
        const int kk = 16 * w + ((a4 & 1) << 3 | (a4 >> 1) << 2);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = E * db + e;
            *reinterpret_cast<half4_t *>(&sv[buf][d * KT + (((kk >> 3) ^ d ^ (d >> 3)) & 7) * 8 + (kk & 4)]) =
                half4_t{gv[0][e], gv[1][e], gv[2][e], gv[3][e]};
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
        const bool whole = kb + KT - 1 <= wfirst && kb + KT <= k1 && (a.window == 0 || kb > wlast - a.window) &&
                           (ok[0] & ok[1] & ok[2] & ok[3]);
        if (!whole) {
            const int hi = (pos < k1 ? pos : k1 - 1) - kb - 4 * g, lo = row_lo - kb - 4 * g;  // of the key's place in the tile
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int at_key = 32 * u + 8 * (r >> 2) + (r & 3);
                    if (at_key > hi || at_key < lo || !ok[2 * u + (r >> 3)]) sc[u][r] = -INFINITY;
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
    int kb = k0 & ~(KT - 1);
    auto turn = [&](auto which) {
        constexpr int buf = decltype(which)::value;
        if (wrows > 0 && kb <= wlast && (a.window == 0 || kb + KT > wfirst - a.window + 1)) compute(kb, which);
        store(kb + KT, buf ^ 1);
        load(kb + 2 * KT);
        __syncthreads();
        kb += KT;
    };
    if (kb < k1) {
        load(kb);
        store(kb, 0);
        load(kb + KT);
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
        for (int t0 = k0 & ~(KT - 1); t0 < k1; t0 += KT) {
            if (t0 + KT <= k1 && t0 >= from && t0 + KT - 1 <= upto) continue;
            for (int key = t0; key < t0 + KT && key < k1; ++key) {
                const int page = a.batch.page(s, key >> a.batch.page_shift);
                if (page < 0 || key > pos || key < row_lo) continue;
                const half_t *vr = a.v + page * a.batch.page_stride + head_at + static_cast<int64_t>(key & in_page) * D + 4 * g;
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
#pragma unroll
                    for (int r = 0; r < 16; r += 4) {
                        const half4_t v = taken<4>(*reinterpret_cast<const half4_t *>(vr + 32 * d + 2 * r));
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

template <int D>
__global__ __launch_bounds__(256, 2) void paged_attn_rows(AttnArgs a) {
    __shared__ __attribute__((aligned(16))) RowsLds<D> lds;
    rows_tile<D>(a, lds, blockIdx.x);
}

// Batches with long chunks: the first `large` blocks are 128-row tiles, the rest the short chunks' 16-row
// ones, which fill the CUs that the long ones leave (a launch of its own after them: 37 us for the two chunks
// of 501 and 332 tokens beside 29 single ones, 28 so).
template <int D>
__global__ __launch_bounds__(256, 2) void paged_attn_mixed(AttnArgs a, int large) {
    __shared__ __attribute__((aligned(16))) union {
        RowsLds<D> rows;
        ChunkLds<D> chunk;
    } lds;
    if (static_cast<int>(blockIdx.x) < large)
        chunk_tile<D>(a, lds.chunk, blockIdx.x);
    else
        rows_tile<D>(a, lds.rows, static_cast<int>(blockIdx.x) - large);
}

// ---------------------------------------------------------------- the chunks' states

// Join a row's chunks: out = sum_c num_c w_c / sum_c den_c w_c, w_c = 2^((m_c - M) scale2), M the largest m_c.
constexpr int kFewChunks = 8;

// Up to kFewChunks: a wave for R heads of a token, which share its lookups, everything requested at once. 862 tokens of
// 16 heads over four chunks with 1 / 2 / 4 heads a wave: 7.3 / 5.6 / 6.5 us; with the chunks requested before it is known
// how many a row has 8.5.
template <int D, int R>
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
    const int n = Span(a, s, n_new, a.batch.length(s)).n;
    if (n <= 1) return;
    const float *pr = a.part + trow * a.nsplit * (D + 4);
    float mc[R][kFewChunks], lc[R][kFewChunks], v[R][kFewChunks][PER];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < kFewChunks; ++c)
            if (c < n) {
                const float *pc = pr + static_cast<int64_t>(r * a.nsplit + c) * (D + 4);
                mc[r][c] = pc[D + 1];
                lc[r][c] = pc[D];
#pragma unroll
                for (int e = 0; e < PER; ++e) v[r][c][e] = pc[lane * PER + e];
            }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float num[PER] = {}, den = 0.0f, m = -INFINITY;
#pragma unroll
        for (int c = 0; c < kFewChunks; ++c)
            if (c < n) m = fmaxf(m, mc[r][c]);
        const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int c = 0; c < kFewChunks; ++c)
            if (c < n) {
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
template <int D>
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
    const int n = Span(a, s, n_new, a.batch.length(s)).n;
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
};

// Sequences of up to kFew rows go to the 16-row tiles, the others to the 128-row ones: 64 sequences after 2000 keys
// (32 heads over 8, D = 128) take 107 / 118 us with 16 / 32 rows each in the small tiles and 131 / 124 in the large;
// with 48 rows 151 and 126. A batch without longer chunks has no 128-row tile; one sequence alone goes where its
// chunk does.
constexpr int64_t kFew = 32;
// The keys are cut into chunks until the tiles fill the chip's workgroups, of kMinChunk keys at least. kFillSmall 512 /
// 1024 / 2048 / 4096: 48 tokens over up to 1536 keys each 40 / 35 / 36 / 37 us, 5 over 65000 82 / 79 / 79 / 84;
// kFillLarge 256 / 384 / 512: a batch of two chunks and 30 tokens 28.7 / 28.4 / 29.8. kMinChunk 128 / 256 / 512: one
// token over 1024 keys 8.1 / 9.1 / 11.6. Contexts of up to kWhole keys are not cut, whose second launch costs more than it
// saves. In a captured graph, one token of 8 kv heads over 256 / 384 / 448 / 512 keys: 6.8 / 8.1 / 8.8 / 9.1 us whole,
// 8.0 / 8.2 / 8.2 / 8.3 cut (4 of D = 64: 5.6 / 6.6 / 7.2 / 7.3 and 7.2 / 7.4 / 7.5 / 7.5). From 128 tiles on, twice that
// (16 tokens of 8 kv heads over 512 / 768 / 1024: 10.9 / 15.7 / 19.2 whole, 13.1 / 15.7 / 19.0 cut).
constexpr int64_t kFillSmall = 1024, kFillLarge = 384, kMinChunk = 128, kWhole = 384;

inline Plan plan_of(int64_t tokens, int64_t b, int64_t gqa, int64_t n_kv, int64_t max_q, int64_t max_context, int64_t window) {
    Plan p;
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
    int64_t span = window > 0 && window + max_q + 63 < max_context ? window + max_q + 63 : max_context;
    if (span < 1) span = 1;
    if (span > int64_t(1) << 30) span = int64_t(1) << 30;  // no table holds more
    // the launch is sized for the most tiles there can be; the chunks go by what a batch of long chunks has
    const int64_t wgs = (p.large > 0 ? rows / 128 + 1 : p.small) * n_kv, whole = wgs < 128 ? kWhole : 2 * kWhole;
    int64_t n = ((p.large > 0 ? kFillLarge : kFillSmall) + wgs - 1) / wgs;
    const int64_t most = span <= whole ? 1 : (span + kMinChunk - 1) / kMinChunk;
    if (n > most) n = most;
    p.chunk = static_cast<int>(((span + n - 1) / n + 63) / 64 * 64);
    p.nsplit = static_cast<int>((span + p.chunk - 1) / p.chunk);
    return p;
}

inline size_t part_bytes(const Plan &p, int64_t tokens, int64_t heads, int64_t hd) {
    return p.nsplit > 1 ? static_cast<size_t>(tokens * heads * p.nsplit * (hd + 4)) * sizeof(float) : 0;
}

template <int D>
hipError_t launch(const AttnArgs &a, const Plan &p, hipStream_t stream) {
    if (p.large > 0)
        paged_attn_mixed<D><<<dim3(static_cast<unsigned>((p.large + p.small) * a.n_kv), a.nsplit), 256, 0, stream>>>(
            a, static_cast<int>(p.large * a.n_kv));
    else
        paged_attn_rows<D><<<dim3(static_cast<unsigned>(p.small * a.n_kv), a.nsplit), 256, 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.nsplit == 1) return e;
    const int64_t rows = static_cast<int64_t>(a.batch.tokens) * a.heads;
    if (a.nsplit <= kFewChunks && a.heads % 2 == 0)
        paged_attn_merge_few<D, 2><<<static_cast<unsigned>((rows / 2 + 3) / 4), 256, 0, stream>>>(a);
    else if (a.nsplit <= kFewChunks)
        paged_attn_merge_few<D, 1><<<static_cast<unsigned>((rows + 3) / 4), 256, 0, stream>>>(a);
    else
        paged_attn_merge<D><<<static_cast<unsigned>(rows), 256, 0, stream>>>(a);
    return hipGetLastError();
}

inline bool plannable(int64_t tokens, int64_t b, int64_t heads, int64_t n_kv, int64_t hd, int64_t max_q, int64_t max_context,
                      int64_t window) {
    return tokens > 0 && b > 0 && n_kv > 0 && heads > 0 && heads % n_kv == 0 && hd > 0 && max_q > 0 && max_context > 0 && window >= 0 &&
           tokens < (int64_t(1) << 24) && b <= kMaxSeqs && heads <= 65536 && hd <= 128 && max_q < (int64_t(1) << 31) &&
           max_context < (int64_t(1) << 31) && window < (int64_t(1) << 31);
}

}  // namespace
}  // namespace dtts

extern "C" size_t dtts_paged_attention_workspace_bytes(int64_t tokens, int64_t b, int64_t heads, int64_t n_kv, int64_t head_dim,
                                                       int64_t max_q, int64_t max_context, int64_t window) {
    using namespace dtts;
    if (!plannable(tokens, b, heads, n_kv, head_dim, max_q, max_context, window)) return 0;
    return part_bytes(plan_of(tokens, b, heads / n_kv, n_kv, max_q, max_context, window), tokens, heads, head_dim);
}

extern "C" int dtts_paged_attention_f16(const dtts_f16 *q, const dtts_f16 *kpages, const dtts_f16 *vpages, const int32_t *q_start,
                                        const int32_t *context, const int32_t *page_table, dtts_f16 *out, int64_t tokens,
                                        int64_t b, int64_t heads, int64_t n_kv, int64_t head_dim, int64_t page, int64_t n_pages,
                                        int64_t max_pages, int64_t page_stride, int64_t q_stride, int64_t max_q,
                                        int64_t max_context, int64_t window, float scale, void *workspace, size_t ws_bytes,
                                        hipStream_t stream) {
    using namespace dtts;
    const char *name = "dtts_paged_attention_f16";
    DTTS_REQUIRE_PAGED(name, tokens, b, n_kv, head_dim, page, n_pages, max_pages, page_stride);
    DTTS_REQUIRE(heads > 0 && heads <= 65536 && heads % n_kv == 0, "%s: %lld heads over %lld kv heads", name, (long long)heads,
                 (long long)n_kv);
    DTTS_REQUIRE(q_stride >= heads * head_dim && q_stride % 8 == 0, "%s: q_stride %lld (a multiple of 8, at least heads * head_dim)",
                 name, (long long)q_stride);
    DTTS_REQUIRE(window >= 0 && window < (int64_t(1) << 31), "%s: window %lld", name, (long long)window);
    if (tokens == 0 || b == 0) return DTTS_OK;
    DTTS_REQUIRE(max_q > 0 && max_context > 0 && max_q < (int64_t(1) << 31) && max_context < (int64_t(1) << 31),
                 "%s: max_q %lld, max_context %lld", name, (long long)max_q, (long long)max_context);
    DTTS_REQUIRE(q && kpages && vpages && q_start && context && page_table && out, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(q, 16) && aligned(kpages, 16) && aligned(vpages, 16) && aligned(out, 16) && aligned(q_start, 4) &&
                     aligned(context, 4) && aligned(page_table, 4),
                 "%s: misaligned operand", name);
    DTTS_REQUIRE(std::isfinite(scale * kLog2e), "%s: scale %g", name, static_cast<double>(scale));
    Plan p = plan_of(tokens, b, heads / n_kv, n_kv, max_q, max_context, window);
    DTTS_REQUIRE(tokens * heads < (int64_t(1) << 31) && (p.small + p.large) * n_kv < (int64_t(1) << 24), "%s: too many rows", name);
    const int64_t row = heads * head_dim * static_cast<int64_t>(sizeof(half_t));
    DTTS_REQUIRE(q_stride < (int64_t(1) << 62), "%s: q_stride %lld", name, (long long)q_stride);
    DTTS_REQUIRE(!share_bytes({q, tokens, q_stride * static_cast<int64_t>(sizeof(half_t)), row}, {out, 1, 0, tokens * row}),
                 "%s: the output may not be the queries, nor a part of their memory", name);
    AttnArgs a;
    a.batch = PagedBatch{q_start, context, page_table, static_cast<int>(tokens), static_cast<int>(b), log2_of(page),
                         static_cast<int>(n_pages), static_cast<int>(max_pages), page_stride};
    a.q = reinterpret_cast<const half_t *>(q);
    a.k = reinterpret_cast<const half_t *>(kpages);
    a.v = reinterpret_cast<const half_t *>(vpages);
    a.out = reinterpret_cast<half_t *>(out);
    a.q_stride = q_stride;
    a.heads = static_cast<int>(heads);
    a.n_kv = static_cast<int>(n_kv);
    a.gqa = static_cast<int>(heads / n_kv);
    // one of 2^30 reaches past every position that a table holds, and the differences below stay ints
    a.window = window >= int64_t(1) << 30 ? 0 : static_cast<int>(window);
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
    }
    a.chunk = p.chunk;
    a.nsplit = p.nsplit;
    DTTS_HIP_CHECK(head_dim == 128 ? launch<128>(a, p, stream) : launch<64>(a, p, stream), name);
    return DTTS_OK;
}
