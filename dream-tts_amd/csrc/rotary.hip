// Rotary positions for callers that keep their own layout: half-split or interleaved pairs, part of
// the head, any number of rows at device-resident positions, and tables scaled for contexts longer
// than the trained one. (dtts_rope_halfsplit_* is the reference's form: whole heads, host positions.)
//
//   o1 = x1 c - x2 s, o2 = x2 c + x1 s over pairs (i, i + rot/2) or (2i, 2i + 1), i < rot/2;
//   dimensions rot .. D - 1 pass through.
//
// HBM-bound: x in and y out once (a row's table entries are read by all its heads, from L2). A lane
// takes 16 bytes of each half of its pairs (interleaved: 16 bytes, whole pairs), so every wave access
// is full segments; rows, heads and offsets come from one flat index by multiplications (FastDiv). 8192 f16 rows of
// 32 heads of 128 and their table rows, 138 MB: 22.8 us, 6.05 TB/s (a large copy: 6.2).
// Products are rounded separately (no FMA), f32 arithmetic, one rounding on the store.
#include <cmath>

#include "common.hpp"
#include "norm_rope.hpp"

#pragma clang fp contract(off)

namespace dtts {
namespace {

struct RotaryArgs {
    const float *cos_t, *sin_t;
    const int32_t *pos;
    int64_t xs, ys;  // elements between rows
    uint32_t units;  // work items in all
    int hd, half, table_len;
    FastDiv per_row, per_head;
};

template <typename T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
};

// V elements a lane and access. Per head, half/V items of two vectors each (interleaved: 2 half/V of
// one) turn pairs, then (D - 2 half)/V copy a vector (none in place: per_head counts them or not).
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(const T *x, T *y, RotaryArgs a) {
    typedef typename Vec<T, V>::type vec;
    const uint32_t e = blockIdx.x * 256u + threadIdx.x;
    if (e >= a.units) return;
    const uint32_t row = a.per_row.div(e), in_row = e - row * a.per_row.d;
    const uint32_t head = a.per_head.div(in_row);
    const int j = static_cast<int>(in_row - head * a.per_head.d);
    const int turning = (INTERLEAVED ? 2 * a.half : a.half) / V;
    const T *xr = x + row * a.xs + static_cast<int64_t>(head) * a.hd;
    T *yr = y + row * a.ys + static_cast<int64_t>(head) * a.hd;
    const int p = a.pos[row];
    if (p < 0 || p >= a.table_len) return;  // padding: the row stays as it was
    if (j >= turning) {
        const int o = 2 * a.half + (j - turning) * V;
        *reinterpret_cast<vec *>(yr + o) = *reinterpret_cast<const vec *>(xr + o);
        return;
    }
    const float *cr = a.cos_t + static_cast<int64_t>(p) * a.half, *sr = a.sin_t + static_cast<int64_t>(p) * a.half;
    if constexpr (INTERLEAVED) {
        const vec v = *reinterpret_cast<const vec *>(xr + j * V);
        vec o;
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            float o1, o2;
            rope_pair(static_cast<float>(v[i]), static_cast<float>(v[i + 1]), cr[(j * V + i) / 2], sr[(j * V + i) / 2], o1, o2);
            o[i] = static_cast<T>(o1);
            o[i + 1] = static_cast<T>(o2);
        }
        *reinterpret_cast<vec *>(yr + j * V) = o;
    } else {
        const vec v1 = *reinterpret_cast<const vec *>(xr + j * V), v2 = *reinterpret_cast<const vec *>(xr + a.half + j * V);
        vec w1, w2;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float o1, o2;
            rope_pair(static_cast<float>(v1[i]), static_cast<float>(v2[i]), cr[j * V + i], sr[j * V + i], o1, o2);
            w1[i] = static_cast<T>(o1);
            w2[i] = static_cast<T>(o2);
        }
        *reinterpret_cast<vec *>(yr + j * V) = w1;
        *reinterpret_cast<vec *>(yr + a.half + j * V) = w2;
    }
}

// One element a lane (V = 1 half-split) or one pair (V = 2 interleaved) where a size or an address is
// no multiple of 16 bytes.
template <typename T>
int rotary(const char *name, const T *x, const float *cos_t, const float *sin_t, const int32_t *pos, T *y, int64_t rows,
           int64_t heads, int64_t hd, int64_t rot, int32_t layout, int64_t xs, int64_t ys, int64_t table_len,
           hipStream_t stream) {
    DTTS_REQUIRE(rows >= 0 && heads > 0 && hd > 0 && table_len > 0 && table_len < (int64_t(1) << 31) && heads < (1 << 20) &&
                     hd < (1 << 20),
                 "%s: bad shape (rows %lld, heads %lld, head_dim %lld, table_len %lld)", name, (long long)rows,
                 (long long)heads, (long long)hd, (long long)table_len);
    DTTS_REQUIRE(rot > 0 && rot % 2 == 0 && rot <= hd, "%s: %lld rotated dimensions of %lld (even, 2 to head_dim)", name,
                 (long long)rot, (long long)hd);
    DTTS_REQUIRE(layout == DTTS_ROPE_HALF || layout == DTTS_ROPE_INTERLEAVED, "%s: unknown layout %d", name, layout);
    DTTS_REQUIRE(xs >= heads * hd && ys >= heads * hd, "%s: row strides %lld, %lld under heads * head_dim", name,
                 (long long)xs, (long long)ys);
    if (rows == 0) return DTTS_OK;
    DTTS_REQUIRE(x && y && cos_t && sin_t && pos, "%s: null pointer", name);
    DTTS_REQUIRE(x != y || xs == ys, "%s: in place needs equal row strides", name);
    DTTS_REQUIRE(aligned(x, sizeof(T)) && aligned(y, sizeof(T)) && aligned(cos_t, 4) && aligned(sin_t, 4) && aligned(pos, 4),
                 "%s: misaligned operand", name);
    constexpr int V = 16 / sizeof(T);
    const bool inter = layout == DTTS_ROPE_INTERLEAVED;
    const int64_t half = rot / 2;
    const bool wide = aligned(x, 16) && aligned(y, 16) && hd % V == 0 && rot % (inter ? V : 2 * V) == 0 && xs % V == 0 &&
                      ys % V == 0;
    // one pair at least, and the copied tail in its own width: odd head sizes have an odd tail
    DTTS_REQUIRE(wide || !inter || (hd % 2 == 0 && xs % 2 == 0 && ys % 2 == 0 && aligned(x, 2 * sizeof(T)) && aligned(y, 2 * sizeof(T))),
                 "%s: interleaved pairs need even sizes, strides and addresses", name);
    const int64_t v = wide ? V : inter ? 2 : 1;
    const int64_t per_head = (inter ? rot : half) / v + (x == y ? 0 : (hd - rot) / v);
    DTTS_REQUIRE(rows < (int64_t(1) << 31) && heads * per_head < (int64_t(1) << 31), "%s: too many rows", name);
    const int64_t units = rows * heads * per_head;
    DTTS_REQUIRE(units < (int64_t(1) << 31), "%s: too many rows", name);
    DTTS_REQUIRE(xs < (int64_t(1) << 60) && ys < (int64_t(1) << 60), "%s: row strides %lld, %lld", name, (long long)xs, (long long)ys);
    const int64_t of = sizeof(T);
    DTTS_REQUIRE(x == y || !share_bytes({x, rows, xs * of, heads * hd * of}, {y, rows, ys * of, heads * hd * of}),
                 "%s: the output shares memory with x without being x", name);
    RotaryArgs a;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.pos = pos;
    a.xs = xs;
    a.ys = ys;
    a.units = static_cast<uint32_t>(units);
    a.hd = static_cast<int>(hd);
    a.half = static_cast<int>(half);
    a.table_len = static_cast<int>(table_len);
    a.per_row = FastDiv(static_cast<uint32_t>(heads * per_head));
    a.per_head = FastDiv(static_cast<uint32_t>(per_head));
    const unsigned blocks = static_cast<unsigned>((units + 255) / 256);
    if (inter && wide)
        rotary_kernel<T, V, true><<<blocks, 256, 0, stream>>>(x, y, a);
    else if (inter)
        rotary_kernel<T, 2, true><<<blocks, 256, 0, stream>>>(x, y, a);
    else if (wide)
        rotary_kernel<T, V, false><<<blocks, 256, 0, stream>>>(x, y, a);
    else
        rotary_kernel<T, 1, false><<<blocks, 256, 0, stream>>>(x, y, a);
    DTTS_LAUNCH_CHECK(name);
    return DTTS_OK;
}

}  // namespace
}  // namespace dtts

using dtts::half_t;

extern "C" int dtts_rope_table_scaled_f32(int64_t len, int64_t rot_dim, double base, int32_t scaling, double factor,
                                          int64_t original_len, double beta_fast, double beta_slow, double attn_factor,
                                          float *cos_out, float *sin_out) {
    const char *name = "dtts_rope_table_scaled_f32";
    DTTS_REQUIRE(len >= 0 && rot_dim > 0 && rot_dim % 2 == 0 && base > 1.0 && std::isfinite(base), "%s: bad arguments", name);
    DTTS_REQUIRE(scaling >= DTTS_ROPE_SCALE_NONE && scaling <= DTTS_ROPE_SCALE_YARN, "%s: unknown scaling %d", name, scaling);
    DTTS_REQUIRE(scaling == DTTS_ROPE_SCALE_NONE || (factor >= 1.0 && std::isfinite(factor)), "%s: factor %g under 1", name, factor);
    DTTS_REQUIRE(scaling != DTTS_ROPE_SCALE_NTK || rot_dim > 2, "%s: NTK scaling needs more than one pair", name);
    DTTS_REQUIRE(scaling != DTTS_ROPE_SCALE_YARN || (original_len > 0 && beta_fast > beta_slow && beta_slow > 0.0 &&
                                                     std::isfinite(beta_fast) && attn_factor >= 0.0 && std::isfinite(attn_factor)),
                 "%s: YaRN needs original_len > 0, beta_fast > beta_slow > 0 and attn_factor >= 0", name);
    DTTS_REQUIRE(len == 0 || (cos_out && sin_out), "%s: null output", name);
    const int64_t half = rot_dim / 2;
    const double d = static_cast<double>(rot_dim);
    double b = base, m = 1.0, low = 0.0, high = 0.0;
    if (scaling == DTTS_ROPE_SCALE_NTK) b = base * std::pow(factor, d / (d - 2.0));
    if (scaling == DTTS_ROPE_SCALE_YARN) {
        // the pair that makes `turns` turns over the trained length, as a real index
        auto at = [&](double turns) {
            return d * std::log(static_cast<double>(original_len) / (turns * 2.0 * M_PI)) / (2.0 * std::log(base));
        };
        low = std::fmax(std::floor(at(beta_fast)), 0.0);
        high = std::fmin(std::ceil(at(beta_slow)), d - 1.0);
        m = attn_factor > 0.0 ? attn_factor : 0.1 * std::log(factor) + 1.0;
    }
    for (int64_t i = 0; i < half; ++i) {
        double freq = 1.0 / std::pow(b, 2.0 * static_cast<double>(i) / d);
        if (scaling == DTTS_ROPE_SCALE_LINEAR) freq /= factor;
        if (scaling == DTTS_ROPE_SCALE_YARN) {
            const double ramp = std::fmin(std::fmax((static_cast<double>(i) - low) / std::fmax(high - low, 1e-3), 0.0), 1.0);
            freq = freq / factor * ramp + freq * (1.0 - ramp);
        }
        for (int64_t t = 0; t < len; ++t) {
            const double phase = static_cast<double>(t) * freq;
            cos_out[t * half + i] = static_cast<float>(std::cos(phase) * m);
            sin_out[t * half + i] = static_cast<float>(std::sin(phase) * m);
        }
    }
    return DTTS_OK;
}

extern "C" int dtts_rotary_f32(const float *x, const float *cos_t, const float *sin_t, const int32_t *pos, float *y,
                               int64_t rows, int64_t heads, int64_t head_dim, int64_t rot_dim, int32_t layout,
                               int64_t x_stride, int64_t y_stride, int64_t table_len, hipStream_t stream) {
    return dtts::rotary<float>("dtts_rotary_f32", x, cos_t, sin_t, pos, y, rows, heads, head_dim, rot_dim, layout, x_stride,
                               y_stride, table_len, stream);
}

extern "C" int dtts_rotary_f16(const dtts_f16 *x, const float *cos_t, const float *sin_t, const int32_t *pos, dtts_f16 *y,
                               int64_t rows, int64_t heads, int64_t head_dim, int64_t rot_dim, int32_t layout,
                               int64_t x_stride, int64_t y_stride, int64_t table_len, hipStream_t stream) {
    return dtts::rotary<half_t>("dtts_rotary_f16", reinterpret_cast<const half_t *>(x), cos_t, sin_t, pos,
                                reinterpret_cast<half_t *>(y), rows, heads, head_dim, rot_dim, layout, x_stride, y_stride,
                                table_len, stream);
}
