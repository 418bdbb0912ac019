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
constexpr int kCand = 1024;  // members of the crossing bin that are sorted

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
    float t, p, m;
    int k;
    double u, inv_t;
    bool greedy;
};

template <typename T>
__device__ __forceinline__ Row row_of(const SampleArgs<T> &a, int r) {
    Row s;
    s.t = a.temperature ? a.temperature[r] : 1.0f;
    s.greedy = !(s.t > 0.0f);
    s.inv_t = 1.0 / static_cast<double>(s.greedy ? 1.0f : s.t);
    const int k = a.top_k ? a.top_k[r] : 0;
    s.k = k <= 0 || k >= a.vocab ? 0 : k;  // 0: all
    const float p = a.top_p ? a.top_p[r] : 1.0f;
    s.p = p < 1.0f ? p : 1.0f;  // 1 (or not a number): all
    const float m = a.min_p ? a.min_p[r] : 0.0f;
    s.m = m > 0.0f ? m : 0.0f;
    const float u = a.u[r];
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

__device__ __forceinline__ double weight(float l, float top, double inv_t) {
    if (l == top) return 1.0;
    if (top == INFINITY) return 0.0;
    return exp((static_cast<double>(l) - static_cast<double>(top)) * inv_t);
}
__device__ __forceinline__ u64 mass(double w) { return static_cast<u64>(w * kUnit + 0.5); }

__device__ __forceinline__ int bin_of(float l, float top, float per_unit) {
    const float d = l == top ? 0.0f : (top - l) * per_unit;
    return d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
}

__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
__device__ __forceinline__ u64 wave_max_u64(u64 v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const u64 o = __shfl_xor(v, off, 64);
        v = o > v ? o : v;
    }
    return v;
}
// The sum over the wave's lanes up to and including this one.
__device__ __forceinline__ u64 wave_scan_u64(u64 v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const u64 o = __shfl_up(v, off, 64);
        if (lane >= off) v += o;
    }
    return v;
}

constexpr int kSegs = 4096;  // 256 logits each: vocabularies of up to 2^20

template <int NT>
struct Shared {
    static constexpr int NW = NT / 64;
    union {
        struct {
            u64 mass[kBins];
            uint32_t count[kBins];
            u64 cand[kCand];
        } h;
        u64 seg[kSegs];
    };
    u64 red[NW];
    u64 out0, out1;
    int n;
};

// The workgroup's sum of v, and the sum over the threads before this one.
template <int NT>
__device__ __forceinline__ u64 block_scan(Shared<NT> &sh, u64 v, u64 &before) {
    const int w = threadIdx.x >> 6;
    const u64 upto = wave_scan_u64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.red[w] = upto;
    __syncthreads();
    u64 all = 0, base = 0;
#pragma unroll
    for (int i = 0; i < Shared<NT>::NW; ++i) {
        if (i < w) base += sh.red[i];
        all += sh.red[i];
    }
    before = base + upto - v;
    return all;
}

// Calls f(logit, index) for every logit of the row, four neighbours a thread and step: with 16-byte
// aligned rows one load, and every wave covers 256 consecutive ones in index order.
template <typename T, int NT, typename F>
__device__ __forceinline__ void each(const T *row, int vocab, bool vec, F f) {
    typedef T v4 __attribute__((ext_vector_type(4)));
    for (int i = threadIdx.x * 4; i < vocab; i += NT * 4) {
        if (vec && i + 4 <= vocab) {
            const v4 v = *reinterpret_cast<const v4 *>(row + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) f(logit(v[e]), i + e);
        } else {
            for (int e = 0; e < 4 && i + e < vocab; ++e) f(logit(row[i + e]), i + e);
        }
    }
}

// The threshold of the kept prefix (a packed token is kept when it is >= the result) for `want`
// tokens (BY_MASS false) or for the shortest prefix of weight `want` or more, among tokens >= floor.
// top: the largest logit; per_unit: bins per logit; sh.h.mass and sh.h.count hold the row's histogram.
// sum: the weight of the prefix.
template <typename T, int NT, bool BY_MASS>
__device__ u64 threshold(Shared<NT> &sh, const T *row, int vocab, bool vec, float top, double inv_t, float per_unit, u64 floor,
                         double want, u64 &sum) {
    constexpr int PER = kBins / NT;
    // the bin where the running count or weight, from the top, reaches `want`
    u64 c[PER], m[PER], ct = 0, mt = 0, cb, mb;
    const int b0 = threadIdx.x * PER;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        ct += c[i] = sh.h.count[b0 + i];
        mt += m[i] = sh.h.mass[b0 + i];
    }
    const u64 call = block_scan<NT>(sh, ct, cb), mall = block_scan<NT>(sh, mt, mb);
    if (threadIdx.x == 0) sh.n = -1;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const double lo = static_cast<double>(BY_MASS ? mb : cb), hi = static_cast<double>(BY_MASS ? mb + m[i] : cb + c[i]);
        if (lo < want && hi >= want) {  // one bin at most: the sums only rise
            sh.n = b0 + i;
            sh.out0 = cb;
            sh.out1 = mb;
        }
        cb += c[i];
        mb += m[i];
    }
    __syncthreads();
    const int bin = sh.n;
    u64 above_c = sh.out0, above_m = sh.out1;
    __syncthreads();
    if (bin < 0) {  // everything
        sum = mall;
        return floor;
    }
    (void)call;
    // its members
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    each<T, NT>(row, vocab, vec, [&](float l, int i) {
        if (l == -INFINITY || bin_of(l, top, per_unit) != bin) return;
        const u64 k = pack(l, i);
        if (k < floor) return;
        const int at = atomicAdd(&sh.n, 1);
        if (at < kCand) sh.h.cand[at] = k;
    });
    __syncthreads();
    const int n = sh.n;
    if (n <= kCand) {
        int size = 1;
        while (size < n) size <<= 1;
        for (int i = n + threadIdx.x; i < size; i += NT) sh.h.cand[i] = 0;
        __syncthreads();
        for (int k = 2; k <= size; k <<= 1)  // bitonic, descending
            for (int j = k >> 1; j > 0; j >>= 1) {
                for (int i = threadIdx.x; i < size; i += NT) {
                    const int o = i ^ j;
                    if (o > i) {
                        const u64 x = sh.h.cand[i], y = sh.h.cand[o];
                        if ((x < y) == ((i & k) == 0)) {
                            sh.h.cand[i] = y;
                            sh.h.cand[o] = x;
                        }
                    }
                }
                __syncthreads();
            }
        // the member that reaches `want`
        constexpr int CP = kCand / NT;
        u64 v[CP], t = 0, before;
#pragma unroll
        for (int i = 0; i < CP; ++i) {
            const int at = threadIdx.x * CP + i;
            t += v[i] = at < n ? mass(weight(logit_of(sh.h.cand[at]), top, inv_t)) : 0;
        }
        block_scan<NT>(sh, t, before);
        if (threadIdx.x == 0) sh.n = n - 1;
        __syncthreads();
        u64 upto = above_m + before;
#pragma unroll
        for (int i = 0; i < CP; ++i) {
            const int at = threadIdx.x * CP + i;
            const u64 prev = upto;
            upto += v[i];
            if (at < n) {
                const double lo = BY_MASS ? static_cast<double>(prev) : static_cast<double>(above_c + at);
                const double hi = BY_MASS ? static_cast<double>(upto) : static_cast<double>(above_c + at + 1);
                if ((lo < want && hi >= want) || (at == n - 1 && hi < want)) {
                    sh.n = at;
                    sh.out1 = upto;
                }
            }
        }
        __syncthreads();
        const u64 cut = sh.h.cand[sh.n];
        sum = sh.out1;
        __syncthreads();
        return cut;
    }
    // many members (equal logits, or a narrow spread): eight bits of the packed token at a time, keeping
    // the digit where the running sum crosses
    u64 prefix = 0;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += NT) {
            sh.h.mass[i] = 0;
            sh.h.count[i] = 0;
        }
        __syncthreads();
        each<T, NT>(row, vocab, vec, [&](float l, int i) {
            if (l == -INFINITY || bin_of(l, top, per_unit) != bin) return;
            const u64 k = pack(l, i);
            if (k < floor || (shift < 56 && k >> (shift + 8) != prefix)) return;
            const int d = 255 - static_cast<int>(k >> shift & 255);
            atomicAdd(&sh.h.count[d], 1u);
            atomicAdd(&sh.h.mass[d], mass(weight(l, top, inv_t)));
        });
        __syncthreads();
        if (threadIdx.x == 0) {
            u64 cc = above_c, mm = above_m, last_c = cc, last_m = mm;
            int d = 0, last = -1;
            for (; d < 256; ++d) {
                if (!sh.h.count[d]) continue;
                last = d;
                last_c = cc;
                last_m = mm;
                const double hi = BY_MASS ? static_cast<double>(mm + sh.h.mass[d]) : static_cast<double>(cc + sh.h.count[d]);
                if (hi >= want) break;
                cc += sh.h.count[d];
                mm += sh.h.mass[d];
            }
            sh.n = last;
            sh.out0 = last_c;
            sh.out1 = last_m;
        }
        __syncthreads();
        prefix = prefix << 8 | static_cast<u64>(255 - sh.n);
        above_c = sh.out0;
        above_m = sh.out1;
        sum = above_m + sh.h.mass[sh.n];
        __syncthreads();
    }
    return prefix;
}

template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_row(SampleArgs<T> a) {
    __shared__ Shared<NT> sh;
    constexpr int NW = NT / 64;
    const int r = blockIdx.x, vocab = a.vocab, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const T *row = a.logits + r * a.stride;
    const bool vec = reinterpret_cast<uintptr_t>(row) % (4 * sizeof(T)) == 0;
    const Row s = row_of(a, r);
    u64 best = 0;
    each<T, NT>(row, vocab, vec, [&](float l, int i) {
        const u64 k = pack(l, i);
        best = k > best ? k : best;
    });
    best = wave_max_u64(best);
    if (lane == 0) sh.red[w] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) best = sh.red[i] > best ? sh.red[i] : best;
    __syncthreads();
    const float top = logit_of(best);
    if (top == -INFINITY || s.greedy) {  // nothing to choose from, or no choice
        if (threadIdx.x == 0) {
            a.token[r] = top == -INFINITY ? -1 : index_of(best);
            if (a.logprob) a.logprob[r] = top == -INFINITY ? -INFINITY : 0.0f;
        }
        return;
    }
    u64 cut = 0;
    if (s.p <= 0.0f) {
        cut = best;
    } else if (s.k || s.p < 1.0f) {
        const float per_unit = kBins / (kRange * fmaxf(s.t, 1.0f));
        for (int i = threadIdx.x; i < kBins; i += NT) {
            sh.h.mass[i] = 0;
            sh.h.count[i] = 0;
        }
        __syncthreads();
        u64 all = 0, before;
        each<T, NT>(row, vocab, vec, [&](float l, int i) {
            if (l == -INFINITY) return;
            const int b = bin_of(l, top, per_unit);
            const u64 m = mass(weight(l, top, s.inv_t));
            atomicAdd(&sh.h.count[b], 1u);
            atomicAdd(&sh.h.mass[b], m);
            all += m;
        });
        __syncthreads();
        all = block_scan<NT>(sh, all, before);
        u64 sum = all;
        if (s.k) {
            cut = threshold<T, NT, false>(sh, row, vocab, vec, top, s.inv_t, per_unit, 0, static_cast<double>(s.k), sum);
            // a crossing bin of many members was settled in the histogram's place
            if (s.p < 1.0f) {
                __syncthreads();
                for (int i = threadIdx.x; i < kBins; i += NT) {
                    sh.h.mass[i] = 0;
                    sh.h.count[i] = 0;
                }
                __syncthreads();
                each<T, NT>(row, vocab, vec, [&](float l, int i) {
                    if (l == -INFINITY || pack(l, i) < cut) return;
                    const int b = bin_of(l, top, per_unit);
                    atomicAdd(&sh.h.count[b], 1u);
                    atomicAdd(&sh.h.mass[b], mass(weight(l, top, s.inv_t)));
                });
                __syncthreads();
            }
        }
        if (s.p < 1.0f) {
            u64 kept;
            const u64 c = threshold<T, NT, true>(sh, row, vocab, vec, top, s.inv_t, per_unit, cut,
                                                 static_cast<double>(s.p) * static_cast<double>(sum), kept);
            cut = c > cut ? c : cut;
        }
        __syncthreads();
    }
    // the kept weight of every run of 256 logits, then the run that u falls into, then the token
    auto kept_mass = [&](float l, int i) -> u64 {
        if (l == -INFINITY) return 0;
        const u64 k = pack(l, i);
        if (k < cut) return 0;
        const double x = weight(l, top, s.inv_t);
        return x >= static_cast<double>(s.m) || k == best ? mass(x) : 0;
    };
    const int segs = (vocab + 255) / 256;
    for (int seg = w; seg < segs; seg += NW) {
        u64 m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = seg * 256 + lane * 4 + e;
            if (i < vocab) m += kept_mass(logit(row[i]), i);
        }
        m = wave_sum_u64(m);
        if (lane == 0) sh.seg[seg] = m;
    }
    __syncthreads();
    constexpr int SP = kSegs / NT;
    u64 t = 0, before;
#pragma unroll
    for (int i = 0; i < SP; ++i)
        if (threadIdx.x * SP + i < segs) t += sh.seg[threadIdx.x * SP + i];
    const u64 z = block_scan<NT>(sh, t, before);
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
    u64 m[4], own = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) own += m[e] = i0 + e < vocab ? kept_mass(logit(row[i0 + e]), i0 + e) : 0;
    u64 upto = sh.out0 + wave_scan_u64(own) - own;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (upto <= target && target < upto + m[e]) {
            a.token[r] = i0 + e;
            if (a.logprob) {
                const float l = logit(row[i0 + e]);
                const double x = l == top ? 0.0 : (static_cast<double>(l) - static_cast<double>(top)) * s.inv_t;
                a.logprob[r] = static_cast<float>(x - log(static_cast<double>(z) / kUnit));
            }
        }
        upto += m[e];
    }
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
    if (vocab <= 4096)
        sample_row<T, 256><<<static_cast<unsigned>(rows), 256, 0, stream>>>(a);
    else
        sample_row<T, 1024><<<static_cast<unsigned>(rows), 1024, 0, stream>>>(a);
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
