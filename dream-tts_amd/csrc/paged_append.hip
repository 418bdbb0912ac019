// QK-norm, rotary positions and the write of new keys and values into a paged cache, in one launch
// (dtts_qk_norm_rope_kv_append_* with pages, ragged batches and dtts_rotary_*'s layouts).
//
// Per row of qkv: the first `heads` head rows are queries, then n_kv keys, then n_kv values.
//   x' = x / sqrt(mean(x^2) + eps) * w       (queries and keys, when norms are given)
//   q  = f16(turn(x'))  -> q_out             k = f16(turn(x')), v = f16(v) -> the row's page
// Everything is f32 until the one rounding of the store: the cache is f16, and the queries are f16
// because the attention that reads them multiplies on the f16 matrix cores.
//
// HBM-bound: qkv in, q, k and v out, once. D/8 lanes own a head row, two groups of four elements each:
// half-split, four pairs' first and second members; interleaved, eight neighbours (four pairs), so
// both layouts turn in registers and the norm is a shuffle sum over D/8 lanes. At a decode step's
// sizes it is the chain of dependent reads that counts (q_start -> context -> page id and table
// rows): qkv is requested before it, and its ends overlap.
#include <cmath>

#include "norm_rope.hpp"
#include "paged.hpp"

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

// A wave takes one token, or one of its `parts`: rows part * RW + its lane group's, then parts * RW further.
// What a token's rows share (its sequence, position and page, and a lane's cos and sin, whatever the row) is
// read once for all of them.
template <typename T, int D, bool INTERLEAVED>
__global__ __launch_bounds__(256) void qk_rope_append_paged_kernel(const T *qkv, AppendArgs a) {
    constexpr int L = D / 8, RW = 64 / L, U = 4;  // lanes per head row, head rows per wave step, steps requested together
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
    const int s = a.batch.sequence_of(t);
    if (s >= a.batch.b) return;
    int first, n;
    a.batch.rows(s, first, n);
    const int pos = a.batch.length(s) - n + (t - first);
    if (t < first || t >= first + n || pos < 0 || pos >= a.table_len) return;
    const int page = a.batch.page(s, pos >> a.batch.page_shift);
    if (page < 0) return;
    float c[4] = {}, sn[4] = {};
    if (turns) {
        Four<float>::load(a.cos_t + static_cast<int64_t>(pos) * a.half + 4 * j, c);
        Four<float>::load(a.sin_t + static_cast<int64_t>(pos) * a.half + 4 * j, sn);
    }
    const int64_t slot = page * a.batch.page_stride + static_cast<int64_t>(pos & ((1 << a.batch.page_shift) - 1)) * D;
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

template <typename T>
int append(const char *name, const T *qkv, const float *norms, const float *cos_t, const float *sin_t,
           const int32_t *q_start, const int32_t *context, const int32_t *page_table, dtts_f16 *q_out, dtts_f16 *kp,
           dtts_f16 *vp, int64_t tokens, int64_t b, int64_t heads, int64_t n_kv, int64_t hd, int64_t rot, int32_t layout,
           int64_t page, int64_t n_pages, int64_t max_pages, int64_t page_stride, int64_t table_len, float eps,
           hipStream_t stream) {
    DTTS_REQUIRE_PAGED(name, tokens, b, n_kv, hd, page, n_pages, max_pages, page_stride);
    DTTS_REQUIRE(heads > 0 && heads <= 65536, "%s: %lld heads", name, (long long)heads);
    DTTS_REQUIRE(rot > 0 && rot % 8 == 0 && rot <= hd, "%s: %lld rotated dimensions of %lld (a multiple of 8)", name,
                 (long long)rot, (long long)hd);
    DTTS_REQUIRE(layout == DTTS_ROPE_HALF || layout == DTTS_ROPE_INTERLEAVED, "%s: unknown layout %d", name, layout);
    DTTS_REQUIRE(table_len > 0 && table_len < (int64_t(1) << 31), "%s: a table of %lld positions", name, (long long)table_len);
    if (tokens == 0 || b == 0) return DTTS_OK;
    DTTS_REQUIRE(qkv && cos_t && sin_t && q_start && context && page_table && q_out && kp && vp, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(qkv, 4 * sizeof(T)) && aligned(cos_t, 16) && aligned(sin_t, 16) && aligned(q_out, 8) && aligned(kp, 8) &&
                     aligned(vp, 8) && aligned(norms, 16) && aligned(q_start, 4) && aligned(context, 4) && aligned(page_table, 4),
                 "%s: misaligned operand", name);
    const int64_t per = heads + 2 * n_kv, f16 = sizeof(half_t), page_bytes = n_kv * page * hd * f16;
    DTTS_REQUIRE(!share_bytes({qkv, 1, 0, tokens * per * hd * static_cast<int64_t>(sizeof(T))}, {q_out, 1, 0, tokens * heads * hd * f16}),
                 "%s: the queries may not replace qkv, nor a part of it", name);
    DTTS_REQUIRE(!share_bytes({kp, n_pages, page_stride * f16, page_bytes}, {vp, n_pages, page_stride * f16, page_bytes}),
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
    a.kp = reinterpret_cast<half_t *>(kp);
    a.vp = reinterpret_cast<half_t *>(vp);
    a.heads = static_cast<int>(heads);
    a.n_kv = static_cast<int>(n_kv);
    a.half = static_cast<int>(rot / 2);
    a.table_len = static_cast<int>(table_len);
    a.eps = eps;
    a.parts = FastDiv(static_cast<uint32_t>(parts));
    const unsigned blocks = static_cast<unsigned>((tokens * parts + 3) / 4);
    const bool inter = layout == DTTS_ROPE_INTERLEAVED;
    if (hd == 128 && inter)
        qk_rope_append_paged_kernel<T, 128, true><<<blocks, 256, 0, stream>>>(qkv, a);
    else if (hd == 128)
        qk_rope_append_paged_kernel<T, 128, false><<<blocks, 256, 0, stream>>>(qkv, a);
    else if (inter)
        qk_rope_append_paged_kernel<T, 64, true><<<blocks, 256, 0, stream>>>(qkv, a);
    else
        qk_rope_append_paged_kernel<T, 64, false><<<blocks, 256, 0, stream>>>(qkv, a);
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
    return dtts::append<float>("dtts_qk_rope_append_paged_f32", qkv, norms, cos_t, sin_t, q_start, context, page_table, q_out,
                               kpages, vpages, tokens, b, heads, n_kv, head_dim, rot_dim, layout, page, n_pages, max_pages,
                               page_stride, table_len, eps, stream);
}

extern "C" int dtts_qk_rope_append_paged_f16(const dtts_f16 *qkv, const float *norms, const float *cos_t, const float *sin_t,
                                             const int32_t *q_start, const int32_t *context, const int32_t *page_table,
                                             dtts_f16 *q_out, dtts_f16 *kpages, dtts_f16 *vpages, int64_t tokens, int64_t b,
                                             int64_t heads, int64_t n_kv, int64_t head_dim, int64_t rot_dim, int32_t layout,
                                             int64_t page, int64_t n_pages, int64_t max_pages, int64_t page_stride,
                                             int64_t table_len, float eps, hipStream_t stream) {
    return dtts::append<dtts::half_t>("dtts_qk_rope_append_paged_f16", reinterpret_cast<const dtts::half_t *>(qkv), norms,
                                      cos_t, sin_t, q_start, context, page_table, q_out, kpages, vpages, tokens, b, heads,
                                      n_kv, head_dim, rot_dim, layout, page, n_pages, max_pages, page_stride, table_len, eps,
                                      stream);
}
