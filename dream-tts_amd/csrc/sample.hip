// Sampling: one token per row of logits, by temperature, top-k, top-p and min-p, from a given uniform
// random number.
//
//   w_i   = e^((l_i - max) / T), the largest weight 1
//   order = logits descending, equal ones by index ascending
//   kept  = the longest prefix of that order that top-k (count), top-p (weight before the token under
//           p of the top-k's sum) and min-p (w_i >= min_p) all allow, one token at least
//   token = the first index whose kept weight up to and including it, in index order, exceeds u Z
//
// No sort: the kept set is a prefix, so it is one threshold on (logit, index), packed into 64 bits
// (an order-preserving image of the logit, then the index reversed). The threshold is where a
// histogram over the logits crosses k or the weight sought, settled inside the crossing bin by
// sorting its few members, or bit by bit where they are many.
//
// Which token comes out is decided by comparing sums of weights, so the weights are taken in f64 and
// summed as integers (units of 2^-42 of the largest: 2^20 of them stay under 2^62). Integer sums have
// no order, so the atomics and the split over threads cannot change a result.
//
// A short row is one workgroup with its logits and weights in registers. A long one is shared by
// workgroups in four launches (its largest logit; the histogram; the crossing bins' members; the token),
// every pass over the logits after the first from L2 or the MALL. What bounds them: a short row the chain
// of block-wide steps, a long one the f64 exponentials and the launches.
#include <cmath>

#include "common.hpp"

namespace dtts {
namespace {

typedef unsigned long long u64;

constexpr int64_t kMaxVocab = 1 << 20;
constexpr double kUnit = 4398046511104.0;  // 2^42
constexpr int kBins = 2048;
// Bins are 1/51 wide in units of max(T, 1): 40 of those units below the maximum a weight is under
// 2^-57 of it, below what the sums hold, and the last bin takes all that is left.
constexpr float kRange = 40.0f;
constexpr int kCand = 1024;  // members of the crossing bins that are sorted

template <typename T>
struct SampleArgs {
    const T *logits;
    int64_t stride;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t *top_k;
    int32_t *token;
    float *logprob;
    int rows, vocab;
};

struct Row {  // one row's settings, made safe
    float p, m, per_unit;  // per_unit: bins per logit
    int k;
    double u, inv_t;
    bool greedy;
    __device__ __forceinline__ bool filters() const { return k > 0 || (p < 1.0f && p > 0.0f); }
};

template <typename T>
__device__ __forceinline__ Row row_of(const SampleArgs<T> &a, int r) {
    Row s;
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    const int k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.0f, m = a.min_p ? a.min_p[r] : 0.0f, u = a.u[r];
    s.greedy = !(t > 0.0f);
    s.inv_t = 1.0 / static_cast<double>(s.greedy ? 1.0f : t);
    s.per_unit = kBins / (kRange * fmaxf(t, 1.0f));
    s.k = k <= 0 || k >= a.vocab ? 0 : k;  // 0: all
    s.p = p < 1.0f ? p : 1.0f;             // 1 (or not a number): all
    s.m = m > 0.0f ? m : 0.0f;
    s.u = u > 0.0f ? static_cast<double>(fminf(u, 1.0f)) : 0.0;
    return s;
}

// The logit as f32; what is not a number counts as masked. -0 becomes +0, its equal.
template <typename T>
__device__ __forceinline__ float logit(T v) {
    const float f = static_cast<float>(v);
    return f == f ? f + 0.0f : -INFINITY;
}

__device__ __forceinline__ u64 pack(float l, int index) {
    const uint32_t b = __float_as_uint(l);
    const uint32_t key = b & 0x80000000u ? ~b : b | 0x80000000u;
    return static_cast<u64>(key) << 32 | (0xffffffffu - static_cast<uint32_t>(index));
}
__device__ __forceinline__ int index_of(u64 k) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(k)); }
__device__ __forceinline__ float logit_of(u64 k) {
    const uint32_t key = static_cast<uint32_t>(k >> 32);
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// e^((l - top) / T) for l <= top: 2^n 2^f with n the nearest integer to the exponent and 2^f by its Taylor
// series, whose remainder at |f| <= 1/2 is (ln 2 / 2)^11 / 11! = 2.2e-13, the sums' own unit. (The
// library's exp carries 53 bits, at twice the instructions.)
__device__ __forceinline__ double weight(float l, float top, double inv_t) {
    if (l == top) return 1.0;
    if (top == INFINITY) return 0.0;
    const double y = (static_cast<double>(l) - static_cast<double>(top)) * inv_t * 1.4426950408889634074;
    if (!(y > -64.0)) return 0.0;  // under half a unit
    const double n = rint(y), f = (y - n) * 0.69314718055994530942;
    double r = 1.0 / 3628800;
    r = fma(r, f, 1.0 / 362880);
    r = fma(r, f, 1.0 / 40320);
    r = fma(r, f, 1.0 / 5040);
    r = fma(r, f, 1.0 / 720);
    r = fma(r, f, 1.0 / 120);
    r = fma(r, f, 1.0 / 24);
    r = fma(r, f, 1.0 / 6);
    r = fma(r, f, 0.5);
    r = fma(r, f, 1.0);
    r = fma(r, f, 1.0);
    return ldexp(r, static_cast<int>(n));
}
// The nearest number of units: added to 2^52, an f64's last place is one unit.
__device__ __forceinline__ u64 mass(double w) {
    return static_cast<u64>(__double_as_longlong(fma(w, kUnit, 4503599627370496.0))) & 0xfffffffffffffull;
}

__device__ __forceinline__ int bin_of(float l, float top, float per_unit) {
    const float d = l == top ? 0.0f : (top - l) * per_unit;
    return d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
}

// ---------------------------------------------------------------- sums over a wave and a workgroup

// A step of a wave-wide scan: v of the lane `CTRL` says (0x111 .. 0x118: 1 .. 8 lanes before in the
// row of 16; 0x142, 0x143: the last lane of the row, of the half, before), 0 where there is none.
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_before(u64 v) {
    const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
    return static_cast<u64>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo);
}
// The sum over the wave's lanes up to and including this one.
__device__ __forceinline__ u64 wave_scan(u64 v) {
    v += dpp_before<0x111, 0xf>(v);
    v += dpp_before<0x112, 0xf>(v);
    v += dpp_before<0x114, 0xf>(v);
    v += dpp_before<0x118, 0xf>(v);
    v += dpp_before<0x142, 0xa>(v);
    v += dpp_before<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ u64 last_lane(u64 v) {
    return static_cast<u64>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), 63))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
__device__ __forceinline__ u64 wave_max(u64 v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const u64 o = __shfl_xor(v, off, 64);
        v = o > v ? o : v;
    }
    return v;
}

constexpr int kSegs = 4096;  // runs of 256 logits: vocabularies of up to 2^20

template <int NT>
struct Shared {
    static constexpr int NW = NT / 64;
    union {
        struct {
            u64 mass[kBins];
            uint32_t count[kBins];
        } h;
        u64 seg[kSegs];
    };
    u64 cand[kCand];
    u64 digit_mass[256];
    uint32_t digit_count[256];
    u64 red[2][NW];
    u64 out0, out1;
    int n, bin;
};

template <int NT>
__device__ __forceinline__ u64 block_max(Shared<NT> &sh, u64 v) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) sh.red[0][threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Shared<NT>::NW; ++i) v = sh.red[0][i] > v ? sh.red[0][i] : v;
    __syncthreads();
    return v;
}

// The workgroup's sums of a and b, and each thread's sum over the threads before it.
template <int NT>
__device__ __forceinline__ void block_scan(Shared<NT> &sh, u64 a, u64 b, u64 &a_before, u64 &b_before, u64 &a_all, u64 &b_all) {
    const int w = threadIdx.x >> 6;
    const u64 au = wave_scan(a), bu = wave_scan(b);
    if ((threadIdx.x & 63) == 63) {
        sh.red[0][w] = au;
        sh.red[1][w] = bu;
    }
    __syncthreads();
    a_before = au - a;
    b_before = bu - b;
    a_all = b_all = 0;
#pragma unroll
    for (int i = 0; i < Shared<NT>::NW; ++i) {
        const u64 x = sh.red[0][i], y = sh.red[1][i];
        if (i < w) {
            a_before += x;
            b_before += y;
        }
        a_all += x;
        b_all += y;
    }
    __syncthreads();
}

// ---------------------------------------------------------------- a row as a workgroup sees it

// Calls f(logit, index, slot) for the logits [i0, i1) of a row, four neighbours a thread and step, so a
// wave covers 256 consecutive ones in index order. vec: the row is aligned to four of them.
template <typename T, int NT, typename F>
__device__ __forceinline__ void each(const T *row, int i0, int i1, bool vec, F f) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    for (int i = i0 + threadIdx.x * 4; i < i1; i += NT * 4) {
        if (vec && i + 4 <= i1) {
            const v4 v = *reinterpret_cast<const v4 *>(row + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) f(logit(v[e]), i + e);
        } else {
            for (int e = 0; e < 4 && i + e < i1; ++e) f(logit(row[i + e]), i + e);
        }
    }
}

// A row of up to NT * E logits in registers (E > 0), masked past its end; or in memory (E = 0).
template <typename T, int NT, int E>
struct Held {
    const T *row;
    int vocab;
    bool vec;
    float l[E > 0 ? E : 1];
    u64 m[E > 0 ? E : 1];

    __device__ __forceinline__ Held(const T *r, int n) : row(r), vocab(n), vec(reinterpret_cast<uintptr_t>(r) % (4 * sizeof(T)) == 0) {
        if constexpr (E > 0) {
            typedef T v4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int s = 0; s < E / 4; ++s) {
                const int i = (s * NT + threadIdx.x) * 4;
                if (vec && i + 4 <= vocab) {
                    const v4 v = *reinterpret_cast<const v4 *>(row + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) l[4 * s + e] = logit(v[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) l[4 * s + e] = i + e < vocab ? logit(row[i + e]) : -INFINITY;
                }
            }
        }
    }
    __device__ __forceinline__ void weigh(float top, double inv_t) {
        if constexpr (E > 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) m[e] = l[e] == -INFINITY ? 0 : mass(weight(l[e], top, inv_t));
        }
    }
    // f(logit, index, mass()) for every logit that is not masked
    template <typename F>
    __device__ __forceinline__ void all(float top, double inv_t, F f) const {
        if constexpr (E > 0) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (l[e] != -INFINITY) f(l[e], (e / 4 * NT + static_cast<int>(threadIdx.x)) * 4 + e % 4, [&] { return m[e]; });
        } else {
            each<T, NT>(row, 0, vocab, vec, [&](float v, int i) {
                if (v != -INFINITY) f(v, i, [&] { return mass(weight(v, top, inv_t)); });
            });
        }
    }
};

// Descending, in place; the first n of a power of two at least n are given, the rest are filled. Up to 64:
// the first wave's lanes hold them.
template <int NT>
__device__ __forceinline__ void sort_desc(u64 *c, int n) {
    int size = 1;
    while (size < n) size <<= 1;
    if (size <= 64) {
        if (threadIdx.x < 64) {
            const int i = threadIdx.x;
            u64 v = i < n ? c[i] : 0;
            for (int k = 2; k <= size; k <<= 1)
                for (int j = k >> 1; j > 0; j >>= 1) {
                    const u64 o = __shfl_xor(v, j, 64);
                    const bool keep_max = ((i & j) == 0) == ((i & k) == 0);
                    v = keep_max == (o > v) ? o : v;
                }
            if (i < n) c[i] = v;
        }
        __syncthreads();
        return;
    }
    for (int i = n + threadIdx.x; i < size; i += NT) c[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            for (int i = threadIdx.x; i < size; i += NT) {
                const int o = i ^ j;
                if (o > i) {
                    const u64 x = c[i], y = c[o];
                    if ((x < y) == ((i & k) == 0)) {
                        c[i] = y;
                        c[o] = x;
                    }
                }
            }
            __syncthreads();
        }
}

// The member of the sorted cand[0 .. n) where the running count (from above_c) or weight (from above_m)
// reaches `want`; upto: the weight up to and including it.
template <int NT>
__device__ __forceinline__ u64 cut_in(Shared<NT> &sh, int n, bool by_mass, u64 above_c, u64 above_m, double want, float top,
                                      double inv_t, u64 &upto) {
    constexpr int CP = (kCand + NT - 1) / NT;
    u64 v[CP], t = 0, before, all, x, y;
#pragma unroll
    for (int i = 0; i < CP; ++i) {
        const int at = threadIdx.x * CP + i;
        t += v[i] = at < n ? mass(weight(logit_of(sh.cand[at]), top, inv_t)) : 0;
    }
    block_scan<NT>(sh, t, 0, before, x, all, y);
    u64 run = above_m + before;
#pragma unroll
    for (int i = 0; i < CP; ++i) {
        const int at = threadIdx.x * CP + i;
        const u64 prev = run;
        run += v[i];
        if (at < n) {
            const double lo = static_cast<double>(by_mass ? prev : above_c + at);
            const double hi = static_cast<double>(by_mass ? run : above_c + at + 1);
            if ((lo < want && hi >= want) || (at == n - 1 && hi < want)) {
                sh.n = at;
                sh.out1 = run;
            }
        }
    }
    __syncthreads();
    const u64 cut = sh.cand[sh.n];
    upto = sh.out1;
    __syncthreads();
    return cut;
}

// The same among the many members of a bin that are `floor` or more: eight bits of the packed token at a
// time, keeping the digit where the running sum crosses. Many members: equal logits, or a narrow spread.
template <typename T, int NT>
__device__ __noinline__ u64 cut_by_digits(Shared<NT> &sh, const T *row, int vocab, int bin, u64 floor, bool by_mass, u64 above_c,
                                          u64 above_m, double want, float top, float per_unit, double inv_t) {
    const bool vec = reinterpret_cast<uintptr_t>(row) % (4 * sizeof(T)) == 0;
    u64 prefix = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += NT) {
            sh.digit_mass[i] = 0;
            sh.digit_count[i] = 0;
        }
        __syncthreads();
        each<T, NT>(row, 0, vocab, vec, [&](float l, int i) {
            if (l == -INFINITY || bin_of(l, top, per_unit) != bin) return;
            const u64 k = pack(l, i);
            if (k < floor || (shift < 56 && k >> (shift + 8) != prefix)) return;
            const int d = 255 - static_cast<int>(k >> shift & 255);
            atomicAdd(&sh.digit_count[d], 1u);
            atomicAdd(&sh.digit_mass[d], mass(weight(l, top, inv_t)));
        });
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 cc = above_c, mm = above_m;
            int last = -1;
            sh.out0 = cc;
            sh.out1 = mm;
            for (int d = 0; d < 256; ++d) {
                if (!sh.digit_count[d]) continue;
                last = d;
                sh.out0 = cc;
                sh.out1 = mm;
                cc += sh.digit_count[d];
                mm += sh.digit_mass[d];
                if (static_cast<double>(by_mass ? mm : cc) >= want) break;
            }
            sh.n = last < 0 ? 255 : last;
        }
        __syncthreads();
        prefix = prefix << 8 | static_cast<u64>(255 - sh.n);
        above_c = sh.out0;
        above_m = sh.out1;
        __syncthreads();
        if (threadIdx.x == 0) sh.out1 = above_m + sh.digit_mass[sh.n];
        __syncthreads();
    }
    return prefix;  // sh.out1: the weight up to and including it
}

// A thread's bins of the histogram and the sums over the bins before them.
template <int NT>
struct Bins {
    static constexpr int PER = kBins / NT;
    u64 c[PER], m[PER], c_before, m_before, c_all, m_all;
    __device__ __forceinline__ void scan(Shared<NT> &sh, const u64 *mass_of, const uint32_t *count_of) {
        u64 ct = 0, mt = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            ct += c[i] = count_of[threadIdx.x * PER + i];
            mt += m[i] = mass_of[threadIdx.x * PER + i];
        }
        block_scan<NT>(sh, ct, mt, c_before, m_before, c_all, m_all);
    }
    // The bin whose running count or weight reaches `want` (-1: none does), and the sums before it. Bins
    // past `last` hold nothing, and that one `last_mass` (~0: what it has).
    __device__ __forceinline__ int cross(Shared<NT> &sh, bool by_mass, double want, int last, u64 last_mass, u64 &above_c,
                                         u64 &above_m) const {
        if (threadIdx.x == 0) sh.bin = -1;
        __syncthreads();
        u64 cc = c_before, mm = m_before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int b = threadIdx.x * PER + i;
            const u64 more = b == last && last_mass != ~0ull ? last_mass : m[i];
            const double lo = static_cast<double>(by_mass ? mm : cc), hi = static_cast<double>(by_mass ? mm + more : cc + c[i]);
            if (b <= last && lo < want && hi >= want) {  // one bin at most: the sums only rise
                sh.bin = b;
                sh.out0 = cc;
                sh.out1 = mm;
            }
            cc += c[i];
            mm += m[i];
        }
        __syncthreads();
        above_c = sh.out0;
        above_m = sh.out1;
        const int bin = sh.bin;
        __syncthreads();
        return bin;
    }
};

// The threshold of a row's kept tokens by top-k and top-p: a packed token is kept when it is >= the result.
// The histogram is in sh.h.
template <typename T, int NT, int E>
__device__ u64 threshold(Shared<NT> &sh, const Held<T, NT, E> &row, float top, const Row &s) {
    Bins<NT> bins;
    bins.scan(sh, sh.h.mass, sh.h.count);
    u64 cut = 0, sum = bins.m_all, above_c, above_m;
    int k_bin = kBins - 1, n = 0, held = -1;  // held: the bin whose members are in sh.cand, sorted
    u64 k_bin_mass = ~0ull;
    auto cut_of = [&](int bin, bool by_mass, double want, u64 floor, u64 &upto) {
        if (held != bin) {
            if (threadIdx.x == 0) sh.n = 0;
            __syncthreads();
            row.all(top, s.inv_t, [&](float l, int i, auto) {
                if (bin_of(l, top, s.per_unit) != bin) return;
                const int at = atomicAdd(&sh.n, 1);
                if (at < kCand) sh.cand[at] = pack(l, i);
            });
            __syncthreads();
            n = sh.n;
            __syncthreads();
            if (n <= kCand) {
                sort_desc<NT>(sh.cand, n);
                held = bin;
            }
        }
        if (n <= kCand) return cut_in<NT>(sh, n, by_mass, above_c, above_m, want, top, s.inv_t, upto);
        const u64 c = cut_by_digits<T, NT>(sh, row.row, row.vocab, bin, floor, by_mass, above_c, above_m, want, top, s.per_unit, s.inv_t);
        upto = sh.out1;
        __syncthreads();
        return c;
    };
    if (s.k) {
        const double want = static_cast<double>(s.k);
        const int bin = bins.cross(sh, false, want, kBins - 1, ~0ull, above_c, above_m);
        if (bin >= 0) {
            cut = cut_of(bin, false, want, 0, sum);
            k_bin = bin;
            k_bin_mass = sum - above_m;
        }
    }
    if (s.p < 1.0f) {
        const double want = static_cast<double>(s.p) * static_cast<double>(sum);
        const int bin = bins.cross(sh, true, want, k_bin, k_bin_mass, above_c, above_m);
        if (bin >= 0) {
            u64 upto;
            const u64 c = cut_of(bin, true, want, cut, upto);
            cut = c > cut ? c : cut;
        }
    }
    return cut;
}

// ---------------------------------------------------------------- one workgroup a row

// The row's token from its kept tokens' weights: in runs of 256 logits, then inside the run that u falls into.
template <typename T, int NT, int E>
__device__ __forceinline__ void choose(Shared<NT> &sh, const SampleArgs<T> &a, const Held<T, NT, E> &row, int r, const Row &s, u64 best,
                                       u64 cut) {
    constexpr int NW = NT / 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, vocab = a.vocab;
    const float top = logit_of(best);
    const double min_p = static_cast<double>(s.m);
    auto kept = [&](float l, int i) -> u64 {
        if (l == -INFINITY) return 0;
        const u64 k = pack(l, i);
        if (k < cut) return 0;
        const double x = weight(l, top, s.inv_t);
        return x >= min_p || k == best ? mass(x) : 0;
    };
    const int segs = (vocab + 255) / 256;
    if constexpr (E > 0) {
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
            u64 m = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = (q * NT + static_cast<int>(threadIdx.x)) * 4 + e;
                const float l = row.l[4 * q + e];
                if (l == -INFINITY) continue;
                const u64 k = pack(l, i);
                if (k >= cut && (s.m == 0.0f || k == best || weight(l, top, s.inv_t) >= min_p)) m += row.m[4 * q + e];
            }
            m = last_lane(wave_scan(m));
            if (lane == 0 && q * NW + w < kSegs) sh.seg[q * NW + w] = m;
        }
    } else {
        for (int seg = w; seg < segs; seg += NW) {
            u64 m = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = seg * 256 + lane * 4 + e;
                if (i < vocab) m += kept(logit(row.row[i]), i);
            }
            m = last_lane(wave_scan(m));
            if (lane == 0) sh.seg[seg] = m;
        }
    }
    __syncthreads();
    constexpr int SP = E > 0 ? (E / 4 * NW + NT - 1) / NT : kSegs / NT;
    u64 t = 0, before, z, x, y;
#pragma unroll
    for (int i = 0; i < SP; ++i)
        if (static_cast<int>(threadIdx.x) * SP + i < segs) t += sh.seg[threadIdx.x * SP + i];
    block_scan<NT>(sh, t, 0, before, x, z, y);
    u64 target = static_cast<u64>(s.u * static_cast<double>(z));
    if (target >= z) target = z - 1;
    if (before <= target && target < before + t) {  // one thread
        u64 upto = before;
        for (int i = 0; i < SP; ++i) {
            const u64 m = sh.seg[threadIdx.x * SP + i];
            if (target < upto + m) {
                sh.n = threadIdx.x * SP + i;
                sh.out0 = upto;
                break;
            }
            upto += m;
        }
    }
    __syncthreads();
    if (w != 0) return;
    const int i0 = sh.n * 256 + lane * 4;
    u64 m[4], mine = 0;
    float l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        l[e] = i0 + e < vocab ? logit(row.row[i0 + e]) : -INFINITY;
        mine += m[e] = kept(l[e], i0 + e);
    }
    u64 upto = sh.out0 + wave_scan(mine) - mine;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (upto <= target && target < upto + m[e]) {
            a.token[r] = i0 + e;
            if (a.logprob) {
                const double d = l[e] == top ? 0.0 : (static_cast<double>(l[e]) - static_cast<double>(top)) * s.inv_t;
                a.logprob[r] = static_cast<float>(d - log(static_cast<double>(z) / kUnit));
            }
        }
        upto += m[e];
    }
}

// Nothing to choose from, or no choice. True when that was so.
template <typename T>
__device__ __forceinline__ bool settled(const SampleArgs<T> &a, int r, const Row &s, u64 best) {
    const float top = logit_of(best);
    if (top != -INFINITY && !s.greedy) return false;
    if (threadIdx.x == 0) {
        a.token[r] = top == -INFINITY ? -1 : index_of(best);
        if (a.logprob) a.logprob[r] = top == -INFINITY ? -INFINITY : 0.0f;
    }
    return true;
}

template <typename T, int NT, int E>
__device__ __forceinline__ void sample_whole(Shared<NT> &sh, const SampleArgs<T> &a, int r) {
    Held<T, NT, E> row(a.logits + r * a.stride, a.vocab);
    const Row s = row_of(a, r);
    if (s.filters()) {
        for (int i = threadIdx.x; i < kBins; i += NT) {
            sh.h.mass[i] = 0;
            sh.h.count[i] = 0;
        }
    }
    u64 best = 0;
    row.all(0.0f, 1.0, [&](float l, int i, auto) {
        const u64 k = pack(l, i);
        best = k > best ? k : best;
    });
    best = block_max<NT>(sh, best);
    if (best == 0) best = pack(-INFINITY, 0);
    if (settled(a, r, s, best)) return;
    const float top = logit_of(best);
    row.weigh(top, s.inv_t);
    u64 cut = 0;
    if (s.p <= 0.0f) {
        cut = best;
    } else if (s.filters()) {
        row.all(top, s.inv_t, [&](float l, int, auto m) {
            const int b = bin_of(l, top, s.per_unit);
            atomicAdd(&sh.h.count[b], 1u);
            atomicAdd(&sh.h.mass[b], m());
        });
        __syncthreads();
        cut = threshold<T, NT, E>(sh, row, top, s);
        __syncthreads();
    }
    choose<T, NT, E>(sh, a, row, r, s, best, cut);
}

template <typename T, int NT, int E>
__global__ __launch_bounds__(NT) void sample_row(SampleArgs<T> a) {
    __shared__ Shared<NT> sh;
    sample_whole<T, NT, E>(sh, a, blockIdx.x);
}

template <typename T>
int sample(const char *name, const T *logits, const float *temperature, const int32_t *top_k, const float *top_p,
           const float *min_p, const float *u, int32_t *token, float *logprob, int64_t rows, int64_t vocab, int64_t stride,
           void *workspace, size_t ws_bytes, hipStream_t stream) {
    DTTS_REQUIRE(rows >= 0 && rows < (int64_t(1) << 24) && vocab > 0, "%s: bad shape (%lld, %lld)", name, (long long)rows,
                 (long long)vocab);
    DTTS_REQUIRE(vocab <= kMaxVocab, "%s: a vocabulary of %lld (2^20 at most)", name, (long long)vocab);
    DTTS_REQUIRE(stride >= vocab, "%s: row stride %lld under the vocabulary's %lld", name, (long long)stride, (long long)vocab);
    if (rows == 0) return DTTS_OK;
    DTTS_REQUIRE(logits && u && token, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(logits, sizeof(T)) && aligned(temperature, 4) && aligned(top_k, 4) && aligned(top_p, 4) &&
                     aligned(min_p, 4) && aligned(u, 4) && aligned(token, 4) && aligned(logprob, 4),
                 "%s: misaligned operand", name);
    (void)workspace;
    (void)ws_bytes;
    SampleArgs<T> a{logits, stride, temperature, top_p, min_p, u, top_k, token, logprob, static_cast<int>(rows),
                    static_cast<int>(vocab)};
    const unsigned grid = static_cast<unsigned>(rows);
    if (vocab <= 1024)
        sample_row<T, 256, 4><<<grid, 256, 0, stream>>>(a);
    else if (vocab <= 2048)
        sample_row<T, 256, 8><<<grid, 256, 0, stream>>>(a);
    else if (vocab <= 4096)
        sample_row<T, 512, 8><<<grid, 512, 0, stream>>>(a);
    else if (vocab <= 16384)
        sample_row<T, 1024, 16><<<grid, 1024, 0, stream>>>(a);
    else
        sample_row<T, 1024, 0><<<grid, 1024, 0, stream>>>(a);
    DTTS_LAUNCH_CHECK(name);
    return DTTS_OK;
}

}  // namespace
}  // namespace dtts

extern "C" size_t dtts_sample_workspace_bytes(int64_t rows, int64_t vocab) {
    (void)rows;
    (void)vocab;
    return 0;
}

extern "C" int dtts_sample_f32(const float *logits, const float *temperature, const int32_t *top_k, const float *top_p,
                               const float *min_p, const float *u, int32_t *token, float *logprob, int64_t rows, int64_t vocab,
                               int64_t row_stride, void *workspace, size_t ws_bytes, hipStream_t stream) {
    return dtts::sample<float>("dtts_sample_f32", logits, temperature, top_k, top_p, min_p, u, token, logprob, rows, vocab,
                               row_stride, workspace, ws_bytes, stream);
}

extern "C" int dtts_sample_f16(const dtts_f16 *logits, const float *temperature, const int32_t *top_k, const float *top_p,
                               const float *min_p, const float *u, int32_t *token, float *logprob, int64_t rows, int64_t vocab,
                               int64_t row_stride, void *workspace, size_t ws_bytes, hipStream_t stream) {
    return dtts::sample<dtts::half_t>("dtts_sample_f16", reinterpret_cast<const dtts::half_t *>(logits), temperature, top_k, top_p,
                                      min_p, u, token, logprob, rows, vocab, row_stride, workspace, ws_bytes, stream);
}
