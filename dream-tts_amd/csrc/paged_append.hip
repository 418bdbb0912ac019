// QK-norm, rotary positions and the write of new keys and values into a paged cache, in one launch
// (dtts_qk_norm_rope_kv_append_* with pages, ragged batches and dtts_rotary_*'s layouts).
//
// Per row of qkv: the first `heads` head rows are queries, then n_kv keys, then n_kv values.
//   x' = x / sqrt(mean(x^2) + eps) * w       (queries and keys, when norms are given)
//   q  = f16(turn(x'))  -> q_out             k = f16(turn(x')), v = f16(v) -> the row's page
// Everything is f32 until the one rounding of the store: the cache is f16, and the queries are f16
// because the attention that reads them multiplies on the f16 matrix cores.
//
// 4-bit pages (q4.hpp) take k = turn(x') and v in groups of 32 instead:
//   d = f16((max - min) / 15), b = f16(min - 64 d), n = rint((x - (64 d + b)) / d) from 0 to 15
// The pair's two roundings are those of the exact numbers, and b is rounded before the codes are chosen, so the steps lie where
// the values read back do. 64 d + b takes two f32 numbers (one where they nearly cancel; a narrow group far from zero needs the
// other). A code is the definition's unless its value lies within 2^-18 of a step of the border between two. A lane needs eight
// neighbours of a row, a group being four lanes: half-split rows, whose lanes hold two groups of four apart, meet in LDS, a wave's
// rows in its own.
//
// HBM-bound: qkv in, q, k and v out, once. D/8 lanes own a head row, two groups of four elements each:
// half-split, four pairs' first and second members; interleaved, eight neighbours (four pairs), so
// both layouts turn in registers and the norm is a shuffle sum over D/8 lanes. At a decode step's
// sizes it is the chain of dependent reads that counts (q_start -> context -> page id and table
// rows): qkv is requested before it, and its ends overlap. Into 4-bit pages: 48 f32 tokens of 32 rows of 128 (2.6 MB) 3.7 us;
// 4436 f16 tokens of 32 rows of 64 (30 MB) 9.9 us (launches one after another of a graph 3.4 and 9.15), half of it vector issue,
// the rest the chain, which a wave a token meets once.
#include <cmath>

#include "norm_rope.hpp"
#include "paged.hpp"
#include "q4.hpp"

#pragma clang fp contract(off)

namespace dtts {
namespace {

typedef half_t h4 __attribute__((ext_vector_type(4)));

struct AppendArgs {
    PagedBatch batch;
    const float *norms, *cos_t, *sin_t;
    half_t *q_out, *kp, *vp;
    int heads, n_kv, half, table_len;
    float eps;
    FastDiv parts;  // waves per token
};

template <typename T>
struct Four;
template <>
struct Four<float> {
    __device__ __forceinline__ static void load(const float *p, float (&o)[4]) {
        const float4_t v = *reinterpret_cast<const float4_t *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = v[i];
    }
};
template <>
struct Four<half_t> {
    __device__ __forceinline__ static void load(const half_t *p, float (&o)[4]) {
        const h4 v = *reinterpret_cast<const h4 *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = static_cast<float>(v[i]);
    }
};

// x / y from per, about 1 / y, with the error taken off once: right to a last place, and where the quotient is a float (half
// way between two codes, as f16 values often are) it is that one.
__device__ __forceinline__ float quotient(float x, float y, float per) {
    const float q = x * per;
    return __builtin_fmaf(__builtin_fmaf(-q, y, x), per, q);
}

// x - y rounded, and what that leaves of it: exact together.
__device__ __forceinline__ float difference(float x, float y, float &rest) {
    const float s = x - y, v = s - x;
    rest = (x - (s - v)) - (y + v);
    return s;
}

// x + rest, less than a last place from x, as the f16 number next to it. Rounded to f32 before, the sum could fall half way between
// two f16 numbers; of x and its neighbours the odd one on the sum's side is on the same side of every such place.
__device__ __forceinline__ half_t half_of(float x, float rest) {
    const uint32_t bits = __float_as_uint(x), away = (bits ^ __float_as_uint(rest)) >> 31;  // 1: the sum is nearer to zero than x
    return static_cast<half_t>(__uint_as_float(rest != 0.0f ? (bits - away) | 1u : bits));
}

// x of the lane OFF (1 or 2) away among four.
template <int OFF>
__device__ __forceinline__ float other_of_four(float x) {
    constexpr int kSwap = OFF == 1 ? 0xb1 : 0x4e;  // quad_perm [1, 0, 3, 2], [2, 3, 0, 1]
    return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(x), kSwap, 0xf, 0xf, false));
}

// Eight neighbours of a row, of a group that four lanes share: their word, and the group's pair. A group with a value that is
// not finite, or whose values pass f16's range, is NaN, all of it.
__device__ __forceinline__ uint32_t quantise(const float (&z)[8], uint32_t &pair) {
    float lo = z[0], hi = z[0], none = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, z[i]);
        hi = fmaxf(hi, z[i]);
        none = __builtin_fmaf(z[i], 0.0f, none);  // NaN from a value that is not finite on
    }
    if (none != 0.0f) hi = INFINITY;
    lo = fminf(lo, other_of_four<1>(lo));
    hi = fmaxf(hi, other_of_four<1>(hi));
    lo = fminf(lo, other_of_four<2>(lo));
    hi = fmaxf(hi, other_of_four<2>(hi));
    constexpr float kPer = 1.0f / 15.0f;
    float rest;
    const float width = difference(hi, lo, rest), about = width * kPer;
    const float fifteenth = __builtin_fmaf(__builtin_fmaf(-about, 15.0f, width) + rest, kPer, about);
    half_t d = half_of(fifteenth, __builtin_fmaf(-fifteenth, 15.0f, width) + rest);
    const float step = static_cast<float>(d), least = difference(lo, kQ4First * step, rest);
    half_t b = half_of(least, rest);
    const float first = difference(kQ4First * step, -static_cast<float>(b), rest);  // code 64 is at first and rest, which few groups have
    const float last = __builtin_fmaf(kQ4Last, step, static_cast<float>(b));
    constexpr float kOver = 65520.0f;  // what f16 rounds to infinity
    if (!(fabsf(first) < kOver && fabsf(last) < kOver)) d = b = static_cast<half_t>(NAN);
    pair = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, d)) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, b)) << 16;
    const float per = step > 0.0f ? __builtin_amdgcn_rcpf(step) : 0.0f;
    float half[2] = {};  // of the word, as numbers
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = z[i] - first;
    if (__any(rest != 0.0f)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] -= rest;
    }
#pragma unroll
    for (int i = 7; i >= 0; --i)
        half[i & 1] = __builtin_fmaf(half[i & 1], 16.0f, __builtin_amdgcn_fmed3f(rintf(quotient(t[i], step, per)), 0.0f, 15.0f));
    return static_cast<uint32_t>(half[0]) | static_cast<uint32_t>(half[1]) << 16;
}

// A wave takes one token, or one of its `parts`: rows part * RW + its lane group's, then parts * RW further.
// What a token's rows share (its sequence, position and page, and a lane's cos and sin, whatever the row) is
// read once for all of them.
template <typename T, int D, bool INTERLEAVED, bool Q4>
__global__ __launch_bounds__(256) void qk_rope_append_paged_kernel(const T *qkv, AppendArgs a) {
    // Lanes per head row, head rows per wave step, steps requested together. Making 4-bit groups takes 150 instructions a step, which
    // are not unrolled (4 / 3 / 2 / 1 steps: 4000 f16 tokens of 32 rows of 64 9.5 / 9.5 / 9.3 / 8.8 us, 400 of 128 5.8 / 5.6 / 5.3 / 5.1,
    // 8000 of 48 rows 36.2 / 36.5 / 37.6 / 35.1).
    constexpr int L = D / 8, RW = 64 / L, U = Q4 ? 1 : 4;
    const uint32_t wid = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    const int t = static_cast<int>(a.parts.div(wid)), part = static_cast<int>(wid - static_cast<uint32_t>(t) * a.parts.d);
    if (t >= a.batch.tokens) return;
    const int lane = threadIdx.x & 63, j = lane % L, per = a.heads + 2 * a.n_kv, stride = static_cast<int>(a.parts.d) * RW;
    // element offsets of the lane's two groups; the dimensions past 2 half pass through
    const bool turns = 4 * j < a.half;
    const int rest = 2 * a.half + 8 * (j - a.half / 4);
    const int o1 = INTERLEAVED ? 8 * j : turns ? 4 * j : rest;
    const int o2 = INTERLEAVED ? 8 * j + 4 : turns ? a.half + 4 * j : rest + 4;
    const T *src = qkv + static_cast<int64_t>(t) * per * D;
    float x[U][4], y[U][4];
    auto load = [&](int r0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * stride < per ? r0 + u * stride : per - 1;
            Four<T>::load(src + static_cast<int64_t>(r) * D + o1, x[u]);
            Four<T>::load(src + static_cast<int64_t>(r) * D + o2, y[u]);
        }
    };
    int r0 = part * RW + lane / L;
    load(r0);
    // Starts and lengths in one trip where a step is long (4-bit rows: 4436 tokens 11.0 -> 9.7 us); with four rows under way the trip
    // that this saves is hidden, and its instructions are not (f16 rows: 800 tokens 5.71 -> 5.96, 300 of as many sequences 4.6 -> 4.73).
    int first, n, len, s;
    if constexpr (Q4) {
        s = a.batch.sequence_of(t, first, n, len);
        if (s >= a.batch.b) return;
    } else {
        s = a.batch.sequence_of(t);
        if (s >= a.batch.b) return;
        a.batch.rows(s, first, n);
        len = a.batch.length(s);
    }
    const int pos = len - n + (t - first);
    if (t < first || t >= first + n || pos < 0 || pos >= a.table_len) return;
    const int page = a.batch.page(s, pos >> a.batch.page_shift);
    if (page < 0) return;
    float c[4] = {}, sn[4] = {};
    if (turns) {
        Four<float>::load(a.cos_t + static_cast<int64_t>(pos) * a.half + 4 * j, c);
        Four<float>::load(a.sin_t + static_cast<int64_t>(pos) * a.half + 4 * j, sn);
    }
    const int in_page = pos & ((1 << a.batch.page_shift) - 1);
    const int64_t slot = page * a.batch.page_stride + static_cast<int64_t>(in_page) * D;
    constexpr bool APART = Q4 && !INTERLEAVED;
    __shared__ __attribute__((aligned(16))) float exchange[APART ? 4 : 1][APART ? RW : 1][APART ? D + 4 : 1];
    for (;;) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = r0 + u * stride;
            if (r >= per) break;
            const bool is_q = r < a.heads, is_v = r >= a.heads + a.n_kv;
            if (!is_v) {
                if (a.norms) {
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) ss += x[u][i] * x[u][i] + y[u][i] * y[u][i];
#pragma unroll
                    for (int off = L / 2; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, 64);
                    const float inv = 1.0f / sqrtf(ss / static_cast<float>(D) + a.eps);
                    float w[4], v[4];
                    const float *wr = a.norms + (is_q ? 0 : D);
                    Four<float>::load(wr + o1, w);
                    Four<float>::load(wr + o2, v);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[u][i] = x[u][i] * inv * w[i];
                        y[u][i] = y[u][i] * inv * v[i];
                    }
                }
                if (turns) {
                    if constexpr (INTERLEAVED) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            rope_pair(x[u][2 * i], x[u][2 * i + 1], c[i], sn[i], x[u][2 * i], x[u][2 * i + 1]);
                            rope_pair(y[u][2 * i], y[u][2 * i + 1], c[2 + i], sn[2 + i], y[u][2 * i], y[u][2 * i + 1]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) rope_pair(x[u][i], y[u][i], c[i], sn[i], x[u][i], y[u][i]);
                    }
                }
            }
            if constexpr (Q4) {
                if (!is_q) {
                    float z[8];
                    if constexpr (INTERLEAVED) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            z[i] = x[u][i];
                            z[4 + i] = y[u][i];
                        }
                    } else {
                        float *row = exchange[threadIdx.x >> 6][lane / L];
                        *reinterpret_cast<float4_t *>(row + o1) = float4_t{x[u][0], x[u][1], x[u][2], x[u][3]};
                        *reinterpret_cast<float4_t *>(row + o2) = float4_t{y[u][0], y[u][1], y[u][2], y[u][3]};
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        __builtin_amdgcn_wave_barrier();
                        Four<float>::load(row + 8 * j, *reinterpret_cast<float (*)[4]>(z));
                        Four<float>::load(row + 8 * j + 4, *reinterpret_cast<float (*)[4]>(z + 4));
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        __builtin_amdgcn_wave_barrier();
                    }
                    uint32_t pair;
                    const uint32_t word = quantise(z, pair);
                    const int kv = r - a.heads - (is_v ? a.n_kv : 0);
                    uint8_t *dst = reinterpret_cast<uint8_t *>(is_v ? a.vp : a.kp) + page * a.batch.page_stride +
                                   (static_cast<int64_t>(kv) << a.batch.page_shift) * Q4Row<D>::kBytes;
                    *reinterpret_cast<uint32_t *>(dst + (is_v ? Q4Row<D>::value_word(in_page, j) : Q4Row<D>::key_word(in_page, j))) = word;
                    if ((j & 3) == 0) *reinterpret_cast<uint32_t *>(dst + Q4Row<D>::pair(1 << a.batch.page_shift, in_page, j >> 2)) = pair;
                    continue;
                }
            }
            half_t *dst;
            if (is_q)
                dst = a.q_out + (static_cast<int64_t>(t) * a.heads + r) * D;
            else
                dst = (is_v ? a.vp : a.kp) + slot +
                      (static_cast<int64_t>(r - a.heads - (is_v ? a.n_kv : 0)) << a.batch.page_shift) * D;
            h4 p, q;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[i] = static_cast<half_t>(x[u][i]);
                q[i] = static_cast<half_t>(y[u][i]);
            }
            *reinterpret_cast<h4 *>(dst + o1) = p;
            *reinterpret_cast<h4 *>(dst + o2) = q;
        }
        r0 += U * stride;
        if (r0 - lane / L >= per) return;
        load(r0);
    }
}

// 5700 tokens, f16, 32 + 2 * 8 rows of 64 (82 MB): 14.3 us with 2048 or 4096, 15.6 with 8192 or more (each
// repeats the token's lookups; a row a lane group and no sharing 18.7); 48 f32 tokens of 32 rows of 128 the same.
constexpr int64_t kFillWaves = 4096;

template <bool Q4, typename T>
int append(const char *name, const T *qkv, const float *norms, const float *cos_t, const float *sin_t,
           const int32_t *q_start, const int32_t *context, const int32_t *page_table, dtts_f16 *q_out, void *kp,
           void *vp, int64_t tokens, int64_t b, int64_t heads, int64_t n_kv, int64_t hd, int64_t rot, int32_t layout,
           int64_t page, int64_t n_pages, int64_t max_pages, int64_t page_stride, int64_t table_len, float eps,
           hipStream_t stream) {
    const int64_t row_units = Q4 ? 5 * hd / 8 : hd, unit = Q4 ? 1 : sizeof(half_t);
    DTTS_REQUIRE_PAGED_ROWS(name, tokens, b, n_kv, hd, page, n_pages, max_pages, page_stride, row_units, Q4 ? 16 : 8);
    DTTS_REQUIRE(heads > 0 && heads <= 65536, "%s: %lld heads", name, (long long)heads);
    DTTS_REQUIRE(rot > 0 && rot % 8 == 0 && rot <= hd, "%s: %lld rotated dimensions of %lld (a multiple of 8)", name,
                 (long long)rot, (long long)hd);
    DTTS_REQUIRE(layout == DTTS_ROPE_HALF || layout == DTTS_ROPE_INTERLEAVED, "%s: unknown layout %d", name, layout);
    DTTS_REQUIRE(table_len > 0 && table_len < (int64_t(1) << 31), "%s: a table of %lld positions", name, (long long)table_len);
    if (tokens == 0 || b == 0) return DTTS_OK;
    DTTS_REQUIRE(qkv && cos_t && sin_t && q_start && context && page_table && q_out && kp && vp, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(qkv, 4 * sizeof(T)) && aligned(cos_t, 16) && aligned(sin_t, 16) && aligned(q_out, 8) && aligned(kp, Q4 ? 16 : 8) &&
                     aligned(vp, Q4 ? 16 : 8) && aligned(norms, 16) && aligned(q_start, 4) && aligned(context, 4) && aligned(page_table, 4),
                 "%s: misaligned operand", name);
    const int64_t per = heads + 2 * n_kv, f16 = sizeof(half_t), page_bytes = n_kv * page * row_units * unit;
    DTTS_REQUIRE(!share_bytes({qkv, 1, 0, tokens * per * hd * static_cast<int64_t>(sizeof(T))}, {q_out, 1, 0, tokens * heads * hd * f16}),
                 "%s: the queries may not replace qkv, nor a part of it", name);
    DTTS_REQUIRE(!share_bytes({kp, n_pages, page_stride * unit, page_bytes}, {vp, n_pages, page_stride * unit, page_bytes}),
                 "%s: pages of keys and of values share memory", name);
    // Steps of RW head rows a token has, shared by enough waves to fill the chip (kFillWaves, 16 a CU): few tokens
    // spread over many, each with one step; many tokens have a wave each.
    const int64_t rw = 64 / (hd / 8), steps = (per + rw - 1) / rw;
    int64_t parts = (kFillWaves + tokens - 1) / tokens;
    if (parts > steps) parts = steps;
    DTTS_REQUIRE(tokens * parts < (int64_t(1) << 31), "%s: too many rows", name);
    AppendArgs a;
    a.batch = PagedBatch{q_start, context, page_table, static_cast<int>(tokens), static_cast<int>(b), log2_of(page),
                         static_cast<int>(n_pages), static_cast<int>(max_pages), page_stride};
    a.norms = norms;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.q_out = reinterpret_cast<half_t *>(q_out);
    a.kp = static_cast<half_t *>(kp);
    a.vp = static_cast<half_t *>(vp);
    a.heads = static_cast<int>(heads);
    a.n_kv = static_cast<int>(n_kv);
    a.half = static_cast<int>(rot / 2);
    a.table_len = static_cast<int>(table_len);
    a.eps = eps;
    a.parts = FastDiv(static_cast<uint32_t>(parts));
    const unsigned blocks = static_cast<unsigned>((tokens * parts + 3) / 4);
    const bool inter = layout == DTTS_ROPE_INTERLEAVED;
    if (hd == 128 && inter)
        qk_rope_append_paged_kernel<T, 128, true, Q4><<<blocks, 256, 0, stream>>>(qkv, a);
    else if (hd == 128)
        qk_rope_append_paged_kernel<T, 128, false, Q4><<<blocks, 256, 0, stream>>>(qkv, a);
    else if (inter)
        qk_rope_append_paged_kernel<T, 64, true, Q4><<<blocks, 256, 0, stream>>>(qkv, a);
    else
        qk_rope_append_paged_kernel<T, 64, false, Q4><<<blocks, 256, 0, stream>>>(qkv, a);
    DTTS_LAUNCH_CHECK(name);
    return DTTS_OK;
}

}  // namespace
}  // namespace dtts

extern "C" int dtts_qk_rope_append_paged_f32(const float *qkv, const float *norms, const float *cos_t, const float *sin_t,
                                             const int32_t *q_start, const int32_t *context, const int32_t *page_table,
                                             dtts_f16 *q_out, dtts_f16 *kpages, dtts_f16 *vpages, int64_t tokens, int64_t b,
                                             int64_t heads, int64_t n_kv, int64_t head_dim, int64_t rot_dim, int32_t layout,
                                             int64_t page, int64_t n_pages, int64_t max_pages, int64_t page_stride,
                                             int64_t table_len, float eps, hipStream_t stream) {
    return dtts::append<false>("dtts_qk_rope_append_paged_f32", qkv, norms, cos_t, sin_t, q_start, context, page_table, q_out,
                               kpages, vpages, tokens, b, heads, n_kv, head_dim, rot_dim, layout, page, n_pages, max_pages,
                               page_stride, table_len, eps, stream);
}

extern "C" int dtts_qk_rope_append_paged_f16(const dtts_f16 *qkv, const float *norms, const float *cos_t, const float *sin_t,
                                             const int32_t *q_start, const int32_t *context, const int32_t *page_table,
                                             dtts_f16 *q_out, dtts_f16 *kpages, dtts_f16 *vpages, int64_t tokens, int64_t b,
                                             int64_t heads, int64_t n_kv, int64_t head_dim, int64_t rot_dim, int32_t layout,
                                             int64_t page, int64_t n_pages, int64_t max_pages, int64_t page_stride,
                                             int64_t table_len, float eps, hipStream_t stream) {
    return dtts::append<false>("dtts_qk_rope_append_paged_f16", reinterpret_cast<const dtts::half_t *>(qkv), norms,
                                      cos_t, sin_t, q_start, context, page_table, q_out, kpages, vpages, tokens, b, heads,
                                      n_kv, head_dim, rot_dim, layout, page, n_pages, max_pages, page_stride, table_len, eps,
                                      stream);
}

extern "C" int dtts_qk_rope_append_paged_q4_f32(const float *qkv, const float *norms, const float *cos_t, const float *sin_t,
                                             const int32_t *q_start, const int32_t *context, const int32_t *page_table,
                                             dtts_f16 *q_out, void *kpages, void *vpages, int64_t tokens, int64_t b,
                                             int64_t heads, int64_t n_kv, int64_t head_dim, int64_t rot_dim, int32_t layout,
                                             int64_t page, int64_t n_pages, int64_t max_pages, int64_t page_stride,
                                             int64_t table_len, float eps, hipStream_t stream) {
    return dtts::append<true>("dtts_qk_rope_append_paged_q4_f32", qkv, norms, cos_t, sin_t, q_start, context, page_table, q_out,
                               kpages, vpages, tokens, b, heads, n_kv, head_dim, rot_dim, layout, page, n_pages, max_pages,
                               page_stride, table_len, eps, stream);
}

extern "C" int dtts_qk_rope_append_paged_q4_f16(const dtts_f16 *qkv, const float *norms, const float *cos_t, const float *sin_t,
                                             const int32_t *q_start, const int32_t *context, const int32_t *page_table,
                                             dtts_f16 *q_out, void *kpages, void *vpages, int64_t tokens, int64_t b,
                                             int64_t heads, int64_t n_kv, int64_t head_dim, int64_t rot_dim, int32_t layout,
                                             int64_t page, int64_t n_pages, int64_t max_pages, int64_t page_stride,
                                             int64_t table_len, float eps, hipStream_t stream) {
    return dtts::append<true>("dtts_qk_rope_append_paged_q4_f16", reinterpret_cast<const dtts::half_t *>(qkv), norms,
                                      cos_t, sin_t, q_start, context, page_table, q_out, kpages, vpages, tokens, b, heads,
                                      n_kv, head_dim, rot_dim, layout, page, n_pages, max_pages, page_stride, table_len, eps,
                                      stream);
}
