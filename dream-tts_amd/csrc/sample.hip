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
// of block-wide steps (48 rows of 2048: 10 us, of which the bytes are 0.1), a long one the f64 exponentials (two
// passes of 8.4M at 64 x 131072; vector instructions 0.5 and 0.65 of those launches' cycles) and the launches' chains of
// small steps. 64 x 131072 with all rows by top-p 0.9: 62 us; with rows of every kind (about a seventh each greedy,
// unfiltered, by top-k, top-p or min-p alone, by two and by all three): 51, the launches 8.5 + 15 + 15.4 + 13.6. One row by
// top-p: 30.
//
// A row whose crossing bins have more than 1024 members (equal logits, a narrow spread, a wide vocabulary at a high
// temperature) falls to one workgroup and eight passes. 131072 logits by top-p: all equal 1.9 ms, within 1e-3 0.8, spread by
// 2.5 at a temperature of 5 0.5; 64 such rows take as long as one; 2^20 equal ones 14 ms.
#include <cmath>
#include <type_traits>

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
    double u, inv_t, least;  // log2(e) / T; min-p's weight in units
    bool greedy;
    __device__ __forceinline__ bool filters() const { return k > 0 || p < 1.0f; }
};

template <typename T>
__device__ __forceinline__ Row row_of(const SampleArgs<T> &a, int r) {
    Row s;
    const float t = a.temperature ? a.temperature[r] : 1.0f;
    const int k = a.top_k ? a.top_k[r] : 0;
    const float p = a.top_p ? a.top_p[r] : 1.0f, m = a.min_p ? a.min_p[r] : 0.0f, u = a.u[r];
    s.greedy = !(t > 0.0f) || p <= 0.0f || m > 1.0f;  // such a top-p or min-p keeps the first token alone
    // at least 1e-290, so that an infinite T leaves +inf above the rest
    s.inv_t = fmax(1.4426950408889634074 / static_cast<double>(t > 0.0f ? t : 1.0f), 1e-290);
    s.per_unit = kBins / (kRange * fmaxf(t, 1.0f));
    s.k = k <= 0 || k >= a.vocab ? 0 : k;  // 0: all
    s.p = p < 1.0f ? p : 1.0f;             // 1 (or not a number): all
    s.m = m > 0.0f ? m : 0.0f;
    s.least = static_cast<double>(s.m) * kUnit;
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

// a b + c with c in scalar registers (the two-operand form that the compiler picks copies c first: 10 moves of 57
// instructions a weight; with it, and four weights side by side, the histogram of 64 x 131072 takes 17 us for 21.5).
__device__ __forceinline__ double fma_const(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// e^((l - top) / T) for l <= top in units of 2^-42, inv_t = log2(e) / T: 2^(n + 42) 2^f with n the exponent's nearest
// integer, 2^f - 1 = f P(f) by the P of degree 8 that meets (2^f - 1) / f at the nine Chebyshev nodes of |f| <= 1/2: off
// by 4e-14 of the weight, a sixth of a unit at most. (The library's exp carries 53 bits.) Adding 1.5 * 2^52 + 42 leaves
// n + 42 in the low word, which goes straight into the result's exponent. Exponents stop at -64, under half a unit, and
// +inf counts as 1e300, so that no weight needs a branch: the largest is 1 and a masked one rounds to nothing.
__device__ __forceinline__ double weight(float l, float top, double inv_t) {
    constexpr double kRound = 6755399441055744.0 + 42.0;
    const double d = fmin(static_cast<double>(l), 1e300) - fmin(static_cast<double>(top), 1e300);
    const double y = fmax(d * inv_t, -64.0), t = y + kRound, f = y - (t - kRound);
    double r = fma_const(1.0203121063391729e-07, f, 1.3255224878668817e-06);
    r = fma_const(r, f, 1.525268684626772e-05);
    r = fma_const(r, f, 0.00015403455852453838);
    r = fma_const(r, f, 0.0013333558179043112);
    r = fma_const(r, f, 0.009618129159402558);
    r = fma_const(r, f, 0.055504108664760424);
    r = fma_const(r, f, 0.2402265069581299);
    r = fma_const(r, f, 0.6931471805599453);
    r = fma(r, f, 1.0);
    return __hiloint2double(__double2hiint(r) + (__double2loint(t) << 20), __double2loint(r));
}
// The nearest number of units: added to 2^52, an f64's last place is one unit.
__device__ __forceinline__ u64 mass(double w) {
    return static_cast<u64>(__double_as_longlong(w + 4503599627370496.0)) & 0xfffffffffffffull;
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

// One barrier a sum: the waves' parts go to the two halves of `red` in turn, and every other value that one
// thread leaves the rest has a place of its own (k: [0], p: [1]).
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
    u64 red[2][2][NW];
    u64 above_c[2], above_m[2], cut[2], upto[2];  // of a threshold: the sums before its bin, itself, the sum with it
    int bin[2], n[2];                             // its bin (-1: none), the bin's members
    u64 run_before;                               // the run that u falls into
    int run, digit;

    // By any thread before the first barrier.
    __device__ __forceinline__ void clear() {
        if (threadIdx.x < 2) {
            bin[threadIdx.x] = -1;
            n[threadIdx.x] = 0;
        }
    }
};

template <int NT>
__device__ __forceinline__ u64 block_max(Shared<NT> &sh, int &half, u64 v) {
    v = wave_max(v);
    if ((threadIdx.x & 63) == 0) sh.red[half][0][threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Shared<NT>::NW; ++i) v = sh.red[half][0][i] > v ? sh.red[half][0][i] : v;
    half ^= 1;
    return v;
}

// The workgroup's sums of a and b, and each thread's sum over the threads before it.
template <int NT>
__device__ __forceinline__ void block_scan(Shared<NT> &sh, int &half, u64 a, u64 b, u64 &a_before, u64 &b_before, u64 &a_all, u64 &b_all) {
    const int w = threadIdx.x >> 6;
    const u64 au = wave_scan(a), bu = wave_scan(b);
    if ((threadIdx.x & 63) == 63) {
        sh.red[half][0][w] = au;
        sh.red[half][1][w] = bu;
    }
    __syncthreads();
    a_before = au - a;
    b_before = bu - b;
    a_all = b_all = 0;
#pragma unroll
    for (int i = 0; i < Shared<NT>::NW; ++i) {
        const u64 x = sh.red[half][0][i], y = sh.red[half][1][i];
        if (i < w) {
            a_before += x;
            b_before += y;
        }
        a_all += x;
        b_all += y;
    }
    half ^= 1;
}
template <int NT>
__device__ __forceinline__ u64 block_scan(Shared<NT> &sh, int &half, u64 a, u64 &before) {
    u64 x, all, y;
    block_scan<NT>(sh, half, a, 0, before, x, all, y);
    return all;
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
            for (int e = 0; e < E; ++e) m[e] = mass(weight(l[e], top, inv_t));
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

// The first wave's lanes' values, descending; the others' are 0. All 64 lanes of it call.
__device__ __forceinline__ u64 wave_sort_desc(u64 v, int size) {
    const int i = threadIdx.x & 63;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            const u64 o = __shfl_xor(v, j, 64);
            const bool keep_max = ((i & j) == 0) == ((i & k) == 0);
            v = keep_max == (o > v) ? o : v;
        }
    return v;
}

// c[0 .. n), n > 64, descending, in place (bitonic). With a thread for each, steps inside a wave are lane
// exchanges.
template <int NT>
__device__ __forceinline__ void sort_desc(u64 *c, int n) {
    int size = 128;
    while (size < n) size <<= 1;
    if (size <= NT) {
        const int i = threadIdx.x;
        u64 v = i < n ? c[i] : 0;
        for (int k = 2; k <= size; k <<= 1)
            for (int j = k >> 1; j > 0; j >>= 1) {
                u64 o;
                if (j >= 64) {
                    __syncthreads();
                    if (i < size) c[i] = v;
                    __syncthreads();
                    o = i < size ? c[i ^ j] : 0;
                } else {
                    o = __shfl_xor(v, j, 64);
                }
                const bool keep_max = ((i & j) == 0) == ((i & k) == 0);
                v = keep_max == (o > v) ? o : v;
            }
        __syncthreads();
        if (i < n) c[i] = v;
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

// Sorts cand[0 .. n) (given unsorted when `sort`) and leaves in cut[WHICH] and upto[WHICH] the member where
// the running count (WHICH 0, from above_c) or weight (1, from above_m) reaches `want`, and the weight up to
// and including it.
template <int NT, int WHICH>
__device__ __forceinline__ void cut_in(Shared<NT> &sh, int &half, int n, bool sort, u64 above_c, u64 above_m, double want, float top,
                                       double inv_t) {
    if (n <= 64) {  // the first wave does it alone
        if (threadIdx.x < 64) {
            const int i = threadIdx.x;
            u64 k = i < n ? sh.cand[i] : 0;
            if (sort) {
                int size = 1;
                while (size < n) size <<= 1;
                k = wave_sort_desc(k, size);
                if (i < n) sh.cand[i] = k;
            }
            const u64 v = i < n ? mass(weight(logit_of(k), top, inv_t)) : 0, run = above_m + wave_scan(v);
            const double lo = static_cast<double>(WHICH ? run - v : above_c + i), hi = static_cast<double>(WHICH ? run : above_c + i + 1);
            if (i < n && ((lo < want && hi >= want) || (i == n - 1 && hi < want))) {
                sh.cut[WHICH] = k;
                sh.upto[WHICH] = run;
            }
        }
        __syncthreads();
        return;
    }
    if (sort) sort_desc<NT>(sh.cand, n);
    constexpr int CP = (kCand + NT - 1) / NT;
    u64 v[CP], t = 0, before;
#pragma unroll
    for (int i = 0; i < CP; ++i) {
        const int at = threadIdx.x * CP + i;
        t += v[i] = at < n ? mass(weight(logit_of(sh.cand[at]), top, inv_t)) : 0;
    }
    block_scan<NT>(sh, half, t, before);
    u64 run = above_m + before;
#pragma unroll
    for (int i = 0; i < CP; ++i) {
        const int at = threadIdx.x * CP + i;
        const u64 prev = run;
        run += v[i];
        const double lo = static_cast<double>(WHICH ? prev : above_c + at), hi = static_cast<double>(WHICH ? run : above_c + at + 1);
        if (at < n && ((lo < want && hi >= want) || (at == n - 1 && hi < want))) {
            sh.cut[WHICH] = sh.cand[at];
            sh.upto[WHICH] = run;
        }
    }
    __syncthreads();
}

// The same among the many members of a bin that are `floor` or more, from memory: eight bits of the packed
// token at a time, keeping the digit where the running sum crosses. Many members: equal logits, or a narrow
// spread.
template <typename T, int NT, int WHICH>
__device__ __noinline__ void cut_by_digits(Shared<NT> &sh, const T *row, int vocab, int bin, u64 floor, u64 above_c, u64 above_m,
                                           double want, float top, float per_unit, double inv_t) {
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
            int last = 255;
            for (int d = 0; d < 256; ++d) {
                if (!sh.digit_count[d]) continue;
                last = d;
                sh.above_c[WHICH] = cc;
                sh.above_m[WHICH] = mm;
                cc += sh.digit_count[d];
                mm += sh.digit_mass[d];
                if (static_cast<double>(WHICH ? mm : cc) >= want) break;
            }
            sh.digit = last;
            sh.upto[WHICH] = mm;
        }
        __syncthreads();
        prefix = prefix << 8 | static_cast<u64>(255 - sh.digit);
        above_c = sh.above_c[WHICH];
        above_m = sh.above_m[WHICH];
    }
    if (threadIdx.x == 0) sh.cut[WHICH] = prefix;
    __syncthreads();
}

// A thread's bins of the histogram and the sums over the bins before them.
template <int NT>
struct Bins {
    static constexpr int PER = kBins / NT;
    u64 c[PER], m[PER], c_before, m_before, c_all, m_all;
    __device__ __forceinline__ void scan(Shared<NT> &sh, int &half, const u64 *mass_of, const uint32_t *count_of) {
        u64 ct = 0, mt = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            ct += c[i] = count_of[threadIdx.x * PER + i];
            mt += m[i] = mass_of[threadIdx.x * PER + i];
        }
        block_scan<NT>(sh, half, ct, mt, c_before, m_before, c_all, m_all);
    }
    // bin[WHICH]: the one whose running count (BY_MASS false) or weight reaches `want` (it stays -1 where none
    // does), above_c and above_m the sums before it. Bins past `last` hold nothing, and that one `last_mass`
    // (~0: what it has). The caller's next barrier shows them.
    template <int WHICH, bool BY_MASS>
    __device__ __forceinline__ void cross(Shared<NT> &sh, double want, int last, u64 last_mass) const {
        u64 cc = c_before, mm = m_before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int b = threadIdx.x * PER + i;
            const u64 more = b == last && last_mass != ~0ull ? last_mass : m[i];
            const double lo = static_cast<double>(BY_MASS ? mm : cc), hi = static_cast<double>(BY_MASS ? mm + more : cc + c[i]);
            if (b <= last && lo < want && hi >= want) {  // one bin at most: the sums only rise
                sh.bin[WHICH] = b;
                sh.above_c[WHICH] = cc;
                sh.above_m[WHICH] = mm;
            }
            cc += c[i];
            mm += m[i];
        }
    }
};

// The threshold of a row's kept tokens by top-k and top-p: a packed token is kept when it is >= the result.
// The histogram is in sh.h.
template <typename T, int NT, int E>
__device__ __forceinline__ u64 threshold(Shared<NT> &sh, int &half, const Held<T, NT, E> &row, float top, const Row &s) {
    Bins<NT> bins;
    bins.scan(sh, half, sh.h.mass, sh.h.count);
    u64 cut = 0, sum = bins.m_all, k_bin_mass = ~0ull;
    int k_bin = kBins - 1, n = 0, held = -1;  // held: the bin whose members are in sh.cand, sorted
    auto settle = [&](auto which, double want, u64 floor) {
        constexpr int W = decltype(which)::value;
        const int bin = sh.bin[W];
        const bool fresh = held != bin;
        if (fresh) {
            row.all(top, s.inv_t, [&](float l, int i, auto) {
                if (bin_of(l, top, s.per_unit) != bin) return;
                const int at = atomicAdd(&sh.n[W], 1);
                if (at < kCand) sh.cand[at] = pack(l, i);
            });
            __syncthreads();
            n = sh.n[W];
            if (n <= kCand) held = bin;
        }
        if (n <= kCand)
            cut_in<NT, W>(sh, half, n, fresh, sh.above_c[W], sh.above_m[W], want, top, s.inv_t);
        else
            cut_by_digits<T, NT, W>(sh, row.row, row.vocab, bin, floor, sh.above_c[W], sh.above_m[W], want, top, s.per_unit, s.inv_t);
    };
    if (s.k) {
        const double want = static_cast<double>(s.k);
        bins.template cross<0, false>(sh, want, kBins - 1, ~0ull);
        __syncthreads();
        if (sh.bin[0] >= 0) {
            k_bin = sh.bin[0];
            const u64 above = sh.above_m[0];
            settle(std::integral_constant<int, 0>{}, want, 0);
            cut = sh.cut[0];
            sum = sh.upto[0];
            k_bin_mass = sum - above;
        }
    }
    if (s.p < 1.0f) {
        const double want = static_cast<double>(s.p) * static_cast<double>(sum);
        bins.template cross<1, true>(sh, want, k_bin, k_bin_mass);
        __syncthreads();
        if (sh.bin[1] >= 0) {
            settle(std::integral_constant<int, 1>{}, want, cut);
            cut = sh.cut[1] > cut ? sh.cut[1] : cut;
        }
    }
    return cut;
}

// ---------------------------------------------------------------- one workgroup a row

// A logit's weight if min-p keeps it (the largest's is 1, and min-p at most 1 here); and if the threshold does too.
__device__ __forceinline__ u64 min_p_mass(float l, float top, const Row &s) {
    const double x = weight(l, top, s.inv_t);
    return x >= s.least ? mass(x) : 0;
}
__device__ __forceinline__ u64 kept_mass(float l, int i, float top, const Row &s, u64 cut) {
    return pack(l, i) >= cut ? min_p_mass(l, top, s) : 0;
}

// The kept weights of a row's runs of 256 logits, to sh.seg.
template <typename T, int NT>
__device__ __forceinline__ void sum_runs(Shared<NT> &sh, const T *row, int i1, float top, const Row &s, u64 cut) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, segs = (i1 + 255) / 256;
    const bool vec = reinterpret_cast<uintptr_t>(row) % (4 * sizeof(T)) == 0;
    for (int seg = w; seg < segs; seg += NT / 64) {
        const int i = seg * 256 + lane * 4;
        u64 m = 0;
        if (vec && i + 4 <= i1) {
            const v4 v = *reinterpret_cast<const v4 *>(row + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) m += kept_mass(logit(v[e]), i + e, top, s, cut);
        } else {
            for (int e = 0; e < 4 && i + e < i1; ++e) m += kept_mass(logit(row[i + e]), i + e, top, s, cut);
        }
        m = last_lane(wave_scan(m));
        if (lane == 0) sh.seg[seg] = m;
    }
}

// The token where the kept weight passes `target`, inside the run of 256 logits of [.., i1) from i on, `before`
// the kept weight before it; by one wave. z: the whole row's.
template <typename T>
__device__ __forceinline__ void find_token(const SampleArgs<T> &a, const T *row, int r, const Row &s, u64 best, u64 cut, int i, int i1,
                                           u64 before, u64 target, u64 z) {
    const float top = logit_of(best);
    i += (threadIdx.x & 63) * 4;
    u64 m[4], mine = 0;
    float l[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        l[e] = i + e < i1 ? logit(row[i + e]) : -INFINITY;
        mine += m[e] = kept_mass(l[e], i + e, top, s, cut);
    }
    u64 run = before + wave_scan(mine) - mine;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (run <= target && target < run + m[e]) {
            a.token[r] = i + e;
            if (a.logprob) {
                const double d = l[e] == top ? 0.0 : (static_cast<double>(l[e]) - static_cast<double>(top)) * s.inv_t;
                a.logprob[r] = static_cast<float>(d * 0.69314718055994530942 - log(static_cast<double>(z) / kUnit));
            }
        }
        run += m[e];
    }
}

__device__ __forceinline__ u64 target_of(const Row &s, u64 z) {
    const u64 t = static_cast<u64>(s.u * static_cast<double>(z));
    return t >= z ? z - 1 : t;
}

// The row's token from its kept tokens' weights: in runs of 256 logits, then inside the run that u falls into.
template <typename T, int NT, int E>
__device__ __forceinline__ void choose(Shared<NT> &sh, int &half, const SampleArgs<T> &a, const Held<T, NT, E> &row, int r, const Row &s,
                                       u64 best, u64 cut) {
    constexpr int NW = NT / 64, MOST = E > 0 ? E / 4 * NW : kSegs, SP = (MOST + NT - 1) / NT;
    const float top = logit_of(best);
    const int segs = (a.vocab + 255) / 256;
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
                if (k >= cut && (s.m == 0.0f || weight(l, top, s.inv_t) >= s.least)) m += row.m[4 * q + e];
            }
            m = last_lane(wave_scan(m));
            if ((threadIdx.x & 63) == 0) sh.seg[q * NW + (threadIdx.x >> 6)] = m;
        }
    } else {
        sum_runs<T, NT>(sh, row.row, a.vocab, top, s, cut);
    }
    __syncthreads();
    if constexpr (MOST <= 64) {  // the first wave has a run a lane
        if (threadIdx.x >= 64) return;
        const u64 m = static_cast<int>(threadIdx.x) < segs ? sh.seg[threadIdx.x] : 0, upto = wave_scan(m), z = last_lane(upto);
        const u64 target = target_of(s, z);
        const int at = __ffsll(static_cast<unsigned long long>(__ballot(target < upto))) - 1;
        const u64 before = upto - m;
        const u64 b = static_cast<u64>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(before >> 32), at))) << 32 |
                      static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(before), at));
        find_token<T>(a, row.row, r, s, best, cut, at * 256, a.vocab, b, target, z);
    } else {
        u64 t = 0, before;
#pragma unroll
        for (int i = 0; i < SP; ++i)
            if (static_cast<int>(threadIdx.x) * SP + i < segs) t += sh.seg[threadIdx.x * SP + i];
        const u64 z = block_scan<NT>(sh, half, t, before), target = target_of(s, z);
        if (before <= target && target < before + t) {  // one thread
            for (int i = 0; i < SP; ++i) {
                const u64 m = sh.seg[threadIdx.x * SP + i];
                if (target < before + m) {
                    sh.run = threadIdx.x * SP + i;
                    sh.run_before = before;
                    break;
                }
                before += m;
            }
        }
        __syncthreads();
        if (threadIdx.x < 64) find_token<T>(a, row.row, r, s, best, cut, sh.run * 256, a.vocab, sh.run_before, target, z);
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

// Calls follow a barrier or start the kernel.
template <typename T, int NT, int E>
__device__ __forceinline__ void sample_whole(Shared<NT> &sh, const SampleArgs<T> &a, int r) {
    Held<T, NT, E> row(a.logits + r * a.stride, a.vocab);
    const Row s = row_of(a, r);
    int half = 0;
    sh.clear();
    if (s.filters()) {
        for (int i = threadIdx.x; i < kBins; i += NT) {
            sh.h.mass[i] = 0;
            sh.h.count[i] = 0;
        }
    }
    u64 best = pack(-INFINITY, 0);
    row.all(0.0f, 1.0, [&](float l, int i, auto) {
        const u64 k = pack(l, i);
        best = k > best ? k : best;
    });
    best = block_max<NT>(sh, half, best);
    if (settled(a, r, s, best)) return;
    const float top = logit_of(best);
    row.weigh(top, s.inv_t);
    u64 cut = 0;
    if (s.filters()) {
        row.all(top, s.inv_t, [&](float l, int, auto m) {
            const int b = bin_of(l, top, s.per_unit);
            atomicAdd(&sh.h.count[b], 1u);
            atomicAdd(&sh.h.mass[b], m());
        });
        __syncthreads();
        cut = threshold<T, NT, E>(sh, half, row, top, s);
    }
    choose<T, NT, E>(sh, half, a, row, r, s, best, cut);
}

template <typename T, int NT, int E>
__global__ __launch_bounds__(NT) void sample_row(SampleArgs<T> a) {
    __shared__ Shared<NT> sh;
    sample_whole<T, NT, E>(sh, a, blockIdx.x);
}

// ---------------------------------------------------------------- several workgroups a row

// Threads of the workgroups that share a row, and of the one that ends it, whose barriers cost more the more waves
// meet (64 x 131072, 3 x 50021 f16: 512 and 512 threads 57 and 24 us; 256 and 512 68 and 26; 1024 and 512 69 and
// 26; 512 and 256 65 and 25; 512 and 1024 60 and 25).
constexpr int kPartNT = 512, kFinishNT = 512;
constexpr int kMostParts = 256;  // of a row

// What the workgroups of a row leave each other. All but the candidates beyond n_cand is written by one
// launch before the next reads it.
struct RowState {
    u64 hist_mass[kBins];
    u64 run_mass[kSegs];  // the kept weight of each run of 256 logits
    u64 best[kMostParts];
    u64 cand[kCand];
    uint32_t hist_count[kBins];
    uint32_t n_cand;
    // the bins that hold the top-k threshold (-1: none) and may hold the top-p one (lo .. hi), the sums
    // above them, the members of the first
    int32_t k_bin, lo, hi;
    u64 k_above_c, k_above_m, lo_above_m;
    uint32_t k_count, pad;
};

template <typename T>
struct PartArgs {
    SampleArgs<T> a;
    RowState *rows;
    int part, parts;  // logits of a part (a multiple of 1024), parts of a row
};

template <int NT>
__device__ __forceinline__ u64 best_of(Shared<NT> &sh, int &half, const RowState &st, int parts) {
    return block_max<NT>(sh, half, static_cast<int>(threadIdx.x) < parts ? st.best[threadIdx.x] : 0);
}

// A part of a row, in steps of four logits a thread (a wave's are a run of 256). Eight steps are requested
// together, the first eight before anything else: a launch's chain of small reads runs under them.
template <typename T>
struct Part {
    static constexpr int STEP = kPartNT * 4, BATCH = 8;
    typedef T v4 __attribute__((ext_vector_type(4)));
    const T *row;
    int i0, i1;
    bool vec;
    float l[BATCH][4];

    __device__ __forceinline__ Part(const PartArgs<T> &p, int g, int r) : row(p.a.logits + r * p.a.stride), i0(g * p.part) {
        i1 = i0 + p.part < p.a.vocab ? i0 + p.part : p.a.vocab;
        vec = reinterpret_cast<uintptr_t>(row) % (4 * sizeof(T)) == 0;
        load(i0);
    }
    __device__ __forceinline__ void load(int from) {
#pragma unroll
        for (int q = 0; q < BATCH; ++q) {
            const int i = from + q * STEP + static_cast<int>(threadIdx.x) * 4;
            if (vec && i + 4 <= i1) {
                const v4 v = *reinterpret_cast<const v4 *>(row + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) l[q][e] = static_cast<float>(v[e]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) l[q][e] = i + e < i1 ? static_cast<float>(row[i + e]) : -INFINITY;
            }
        }
    }
    // f(four logits, the first's index) for every logit of the part and, past its end, some masked ones; after every
    // step, end(index of the wave's run) by whole waves.
    template <typename F, typename G>
    __device__ __forceinline__ void all(F f, G end) {
        for (int from = i0; from < i1; from += BATCH * STEP) {
            if (from != i0) load(from);
#pragma unroll
            for (int q = 0; q < BATCH; ++q) {
                const int run = from + q * STEP + (static_cast<int>(threadIdx.x) & ~63) * 4;
                if (run >= i1) break;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = logit(l[q][e]);
                f(v, from + q * STEP + static_cast<int>(threadIdx.x) * 4);
                end(run / 256);
            }
        }
    }
};

// First launch: each part's largest; the histogram is cleared.
template <typename T>
__global__ __launch_bounds__(kPartNT) void sample_part_max(PartArgs<T> p) {
    __shared__ Shared<kPartNT> sh;
    const int g = blockIdx.x, r = blockIdx.y;
    const int i0 = g * p.part, i1 = i0 + p.part < p.a.vocab ? i0 + p.part : p.a.vocab;
    RowState &st = p.rows[r];
    for (int i = g * kPartNT + threadIdx.x; i < kBins; i += p.parts * kPartNT) {
        st.hist_mass[i] = 0;
        st.hist_count[i] = 0;
    }
    if (g == 0 && threadIdx.x == 0) st.n_cand = 0;
    const T *row = p.a.logits + r * p.a.stride;
    const bool vec = reinterpret_cast<uintptr_t>(row) % (4 * sizeof(T)) == 0;
    u64 best = pack(-INFINITY, i0);
    each<T, kPartNT>(row, i0, i1, vec, [&](float l, int i) {
        const u64 k = pack(l, i);
        best = k > best ? k : best;
    });
    int half = 0;
    best = block_max<kPartNT>(sh, half, best);
    if (threadIdx.x == 0) st.best[g] = best;
}

// Second: the histogram of a row that filters by rank or weight, the runs' kept weights of one that does not.
template <typename T>
__global__ __launch_bounds__(kPartNT) void sample_part_hist(PartArgs<T> p) {
    __shared__ Shared<kPartNT> sh;
    const int r = blockIdx.y;
    Part<T> part(p, blockIdx.x, r);
    RowState &st = p.rows[r];
    const Row s = row_of(p.a, r);
    if (s.filters())
        for (int i = threadIdx.x; i < kBins; i += kPartNT) {
            sh.h.mass[i] = 0;
            sh.h.count[i] = 0;
        }
    int half = 0;
    const u64 best = best_of<kPartNT>(sh, half, st, p.parts);
    const float top = logit_of(best);
    if (top == -INFINITY || s.greedy) return;
    if (!s.filters()) {
        u64 m = 0;
        part.all(
            [&](const float(&l)[4], int) {
#pragma unroll
                for (int e = 0; e < 4; ++e) m += min_p_mass(l[e], top, s);
            },
                 [&](int run) {
                     if (__any(m != 0)) m = last_lane(wave_scan(m));
                     if ((threadIdx.x & 63) == 0) st.run_mass[run] = m;
                     m = 0;
                 });
        return;
    }
    const bool by_count = s.k > 0, by_mass = s.p < 1.0f;
    part.all(
        [&](const float(&l)[4], int) {
            int b[4];
            u64 m[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) b[e] = bin_of(l[e], top, s.per_unit);
            if (by_mass) {  // four chains of dependent f64 instructions side by side
#pragma unroll
                for (int e = 0; e < 4; ++e) m[e] = mass(weight(l[e], top, s.inv_t));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (m[e]) atomicAdd(&sh.h.mass[b[e]], m[e]);
            }
            if (by_count)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (l[e] != -INFINITY) atomicAdd(&sh.h.count[b[e]], 1u);
        },
        [](int) {});
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kPartNT) {
        if (sh.h.count[i]) atomicAdd(&st.hist_count[i], sh.h.count[i]);
        if (sh.h.mass[i]) atomicAdd(&st.hist_mass[i], sh.h.mass[i]);
    }
}

// Third: where the thresholds lie (every workgroup for itself, from the histogram), the members of those bins,
// and the runs' kept weights above them.
template <typename T>
__global__ __launch_bounds__(kPartNT) void sample_part_collect(PartArgs<T> p) {
    __shared__ Shared<kPartNT> sh;
    const int r = blockIdx.y;
    RowState &st = p.rows[r];
    const Row s = row_of(p.a, r);
    if (s.greedy || !s.filters()) return;
    Part<T> part(p, blockIdx.x, r);
    int half = 0;
    sh.clear();
    if (threadIdx.x == 0) sh.digit = 0;
    const u64 best = best_of<kPartNT>(sh, half, st, p.parts);
    const float top = logit_of(best);
    if (top == -INFINITY) return;
    Bins<kPartNT> bins;
    bins.scan(sh, half, st.hist_mass, st.hist_count);
    int k_bin = -1, lo = kBins, hi = -1;
    u64 k_above_c = 0, k_above_m = 0, lo_above_m = 0;
    if (s.k) {
        bins.template cross<0, false>(sh, static_cast<double>(s.k), kBins - 1, ~0ull);
        __syncthreads();
        k_bin = sh.bin[0];
        k_above_c = sh.above_c[0];
        k_above_m = sh.above_m[0];
        __syncthreads();
    }
    if (s.p < 1.0f) {
        // the top-k's weight is between those of the bins above its threshold's and with it
        const u64 least = k_bin >= 0 ? k_above_m : bins.m_all;
        const u64 most = k_bin >= 0 ? k_above_m + st.hist_mass[k_bin] : bins.m_all;
        const int last = k_bin >= 0 ? k_bin : kBins - 1;
        const double p64 = static_cast<double>(s.p);
        if (threadIdx.x == 0) sh.bin[0] = -1;
        __syncthreads();
        bins.template cross<0, true>(sh, p64 * static_cast<double>(least), last, ~0ull);
        bins.template cross<1, true>(sh, p64 * static_cast<double>(most), last, ~0ull);
        __syncthreads();
        lo = sh.bin[0];
        hi = sh.bin[1];
        lo_above_m = sh.above_m[0];
        if (lo < 0) {  // least is 0
            lo = 0;
            lo_above_m = 0;
        }
        if (hi < 0) lo = kBins;  // no threshold: all of the top-k
    } else {
        lo = hi = k_bin;
        if (k_bin < 0) lo = kBins;
        lo_above_m = k_above_m;
    }
    const int sure = k_bin >= 0 && k_bin < lo ? k_bin : lo;  // the bins before it are kept
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        st.k_bin = k_bin;
        st.lo = lo;
        st.hi = hi;
        st.k_above_c = k_above_c;
        st.k_above_m = k_above_m;
        st.lo_above_m = lo_above_m;
        st.k_count = k_bin >= 0 ? st.hist_count[k_bin] : 0;
    }
    u64 m = 0;
    part.all(
        [&](const float(&l)[4], int i) {
            int b[4];
            bool above = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                b[e] = bin_of(l[e], top, s.per_unit);
                above |= b[e] < sure;
            }
            if (__any(above)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const u64 x = min_p_mass(l[e], top, s);
                    m += b[e] < sure ? x : 0;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (l[e] != -INFINITY && b[e] >= sure && ((b[e] >= lo && b[e] <= hi) || b[e] == k_bin)) {
                    const int at = atomicAdd(&sh.digit, 1);
                    if (at < kCand) sh.cand[at] = pack(l[e], i + e);
                }
        },
        [&](int run) {
            if (__any(m != 0)) m = last_lane(wave_scan(m));
            if ((threadIdx.x & 63) == 0) st.run_mass[run] = m;
            m = 0;
        });
    __syncthreads();
    const int n = sh.digit;  // the part's members: a place for all of them at once
    if (threadIdx.x == 0) sh.run = n ? static_cast<int>(atomicAdd(&st.n_cand, static_cast<uint32_t>(n))) : 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n && i < kCand; i += kPartNT)
        if (sh.run + i < kCand) st.cand[sh.run + i] = sh.cand[i];
}

// Fourth, a workgroup a row: the thresholds among the members, the run that u falls into, the token.
template <typename T>
__global__ __launch_bounds__(kFinishNT) void sample_finish(PartArgs<T> p) {
    constexpr int NT = kFinishNT, SP = kSegs / NT, CP = kCand / NT;
    __shared__ Shared<NT> sh;
    const int r = blockIdx.x, i = threadIdx.x, runs = (p.a.vocab + 255) / 256;
    RowState &st = p.rows[r];
    const Row s = row_of(p.a, r);
    int half = 0;
    const u64 best = best_of<NT>(sh, half, st, p.parts);
    if (settled(p.a, r, s, best)) return;
    const float top = logit_of(best);
    for (int q = i; q < runs; q += NT) sh.seg[q] = st.run_mass[q];
    u64 cut = 0, before;
    if (s.filters()) {
        const int n = static_cast<int>(st.n_cand);
        if (n > kCand) {  // many members: equal logits, or a narrow spread
            __syncthreads();
            sample_whole<T, NT, 0>(sh, p.a, r);
            return;
        }
        if (n > 64) {
            for (int q = i; q < n; q += NT) sh.cand[q] = st.cand[q];
            __syncthreads();
            sort_desc<NT>(sh.cand, n);
        } else {
            if (i < 64) {
                const u64 v = wave_sort_desc(i < n ? st.cand[i] : 0, 64);
                if (i < n) sh.cand[i] = v;
            }
            __syncthreads();
        }
        // the top-k bin's members are the last of the list
        u64 sum = 0;
        if (st.k_bin >= 0) {
            const int from = n - static_cast<int>(st.k_count), at = from + s.k - static_cast<int>(st.k_above_c) - 1;
            cut = sh.cand[at];
            if (s.p < 1.0f) {
                u64 t = 0;
#pragma unroll
                for (int c = 0; c < CP; ++c) {
                    const int q = c * NT + i;
                    if (q >= from && q <= at) t += mass(weight(logit_of(sh.cand[q]), top, s.inv_t));
                }
                sum = st.k_above_m + block_scan<NT>(sh, half, t, before);
            }
        } else if (s.p < 1.0f) {
            u64 t = 0;
#pragma unroll
            for (int c = 0; c < kBins / NT; ++c) t += st.hist_mass[c * NT + i];
            sum = block_scan<NT>(sh, half, t, before);
        }
        if (s.p < 1.0f && st.hi >= 0) {
            cut_in<NT, 1>(sh, half, n, false, 0, st.lo_above_m, static_cast<double>(s.p) * static_cast<double>(sum), top, s.inv_t);
            cut = sh.cut[1] > cut ? sh.cut[1] : cut;
        }
        // their weights to their runs
#pragma unroll
        for (int c = 0; c < CP; ++c) {
            const u64 mine = c * NT + i < n ? sh.cand[c * NT + i] : 0;
            if (c * NT + i < n && mine >= cut) {
                const u64 m = min_p_mass(logit_of(mine), top, s);
                if (m) atomicAdd(&sh.seg[index_of(mine) / 256], m);
            }
        }
    }
    __syncthreads();
    u64 t = 0;
#pragma unroll
    for (int q = 0; q < SP; ++q)
        if (i * SP + q < runs) t += sh.seg[i * SP + q];
    const u64 z = block_scan<NT>(sh, half, t, before), target = target_of(s, z);
    if (before <= target && target < before + t) {  // one thread
        for (int q = 0; q < SP; ++q) {
            const u64 m = sh.seg[i * SP + q];
            if (target < before + m) {
                sh.run = i * SP + q;
                sh.run_before = before;
                break;
            }
            before += m;
        }
    }
    __syncthreads();
    if (i < 64) find_token<T>(p.a, p.a.logits + r * p.a.stride, r, s, best, cut, sh.run * 256, p.a.vocab, sh.run_before, target, z);
}

struct Parts {
    int part, parts;
};

// Rows of up to kWholeVocab logits are one workgroup each: 1024 threads hold them in registers, past 8192 (16 a thread)
// with 84 registers a lane in scratch. 16384 logits by top-p, 1 / 16 / 64 / 256 rows: 27 / 28 / 30 / 43 us, shared 24 / 27
// / 33 / 43; 10240: 24 / 25 / 27 / 35, shared 24 / 26 / 30 / 38; 32 a thread spill more (58 us for a row of 32768, shared
// 23). Longer ones are shared by as many as the chip runs at once (kPartFill: two a CU of 512 threads and 104 registers; 64
// x 131072 with 512 / 768: 62 / 69) and none has under 2048 logits; from 257 rows on that is one (400 rows of 131072: 298
// us, in two parts 336).
constexpr int64_t kWholeVocab = 16384, kPartFill = 512;

inline Parts parts_of(int64_t rows, int64_t vocab) {
    int64_t parts = kPartFill / rows;
    if (parts > vocab / 2048) parts = vocab / 2048;
    if (parts > kMostParts) parts = kMostParts;
    if (parts < 1 || vocab <= kWholeVocab) parts = 1;
    const int64_t part = ((vocab + parts - 1) / parts + 1023) / 1024 * 1024;
    return Parts{static_cast<int>(part), static_cast<int>((vocab + part - 1) / part)};
}

inline size_t sample_bytes(int64_t rows, int64_t vocab) {
    return parts_of(rows, vocab).parts > 1 ? static_cast<size_t>(rows) * sizeof(RowState) : 0;
}

template <typename T>
int sample(const char *name, const T *logits, const float *temperature, const int32_t *top_k, const float *top_p,
           const float *min_p, const float *u, int32_t *token, float *logprob, int64_t rows, int64_t vocab, int64_t stride,
           void *workspace, size_t ws_bytes, hipStream_t stream) {
    DTTS_REQUIRE(rows >= 0 && rows < (int64_t(1) << 20) && vocab > 0, "%s: bad shape (%lld, %lld)", name, (long long)rows,
                 (long long)vocab);
    DTTS_REQUIRE(vocab <= kMaxVocab, "%s: a vocabulary of %lld (2^20 at most)", name, (long long)vocab);
    DTTS_REQUIRE(stride >= vocab, "%s: row stride %lld under the vocabulary's %lld", name, (long long)stride, (long long)vocab);
    if (rows == 0) return DTTS_OK;
    DTTS_REQUIRE(logits && u && token, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(logits, sizeof(T)) && aligned(temperature, 4) && aligned(top_k, 4) && aligned(top_p, 4) &&
                     aligned(min_p, 4) && aligned(u, 4) && aligned(token, 4) && aligned(logprob, 4),
                 "%s: misaligned operand", name);
    SampleArgs<T> a{logits, stride, temperature, top_p, min_p, u, top_k, token, logprob, static_cast<int>(rows),
                    static_cast<int>(vocab)};
    const unsigned grid = static_cast<unsigned>(rows);
    const Parts parts = parts_of(rows, vocab);
    if (parts.parts > 1 && workspace && ws_bytes >= sample_bytes(rows, vocab)) {
        DTTS_REQUIRE(aligned(workspace, 16), "%s: misaligned workspace", name);
        const PartArgs<T> p{a, static_cast<RowState *>(workspace), parts.part, parts.parts};
        const dim3 each_part(static_cast<unsigned>(parts.parts), grid);
        sample_part_max<T><<<each_part, kPartNT, 0, stream>>>(p);
        DTTS_LAUNCH_CHECK(name);
        sample_part_hist<T><<<each_part, kPartNT, 0, stream>>>(p);
        DTTS_LAUNCH_CHECK(name);
        sample_part_collect<T><<<each_part, kPartNT, 0, stream>>>(p);
        DTTS_LAUNCH_CHECK(name);
        sample_finish<T><<<grid, kFinishNT, 0, stream>>>(p);
        DTTS_LAUNCH_CHECK(name);
        return DTTS_OK;
    }
    if (vocab <= 1024)
        sample_row<T, 256, 4><<<grid, 256, 0, stream>>>(a);
    else if (vocab <= 2048)
        sample_row<T, 512, 4><<<grid, 512, 0, stream>>>(a);
    else if (vocab <= 4096)
        sample_row<T, 1024, 4><<<grid, 1024, 0, stream>>>(a);
    else if (vocab <= 8192)
        sample_row<T, 1024, 8><<<grid, 1024, 0, stream>>>(a);
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
    return rows > 0 && vocab > 0 && rows < (int64_t(1) << 20) && vocab <= dtts::kMaxVocab ? dtts::sample_bytes(rows, vocab) : 0;
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
