// The pages of a paged cache between steps: fork (reorder, free), claim, trim, compact, copy.
//
//   pages  [b, max_pages] int32: a sequence's page of each block of positions, an id outside [0, n_pages) for none
//   refs   [n_pages] int32: how many entries hold each page; under 1 is free
//
// Everything is decided on the device, by order and not by whose atomic comes first: a page's count is the same whatever
// the order of its additions, free pages go out from the lowest id on, sequences are served in order. So a result depends
// on nothing but the arguments, and the calls of a step can be captured.
//
// All but the copy are a few dependent trips to memory over some hundred kilobytes at most.
#include <algorithm>
#include <memory>
#include <new>

#include "paged.hpp"

namespace dtts {
namespace {

constexpr int64_t kMostPages = 1 << 24;

#define DTTS_REQUIRE_TABLE(name, b, max_pages, n_pages)                                                                  \
    DTTS_REQUIRE((b) >= 0 && (b) <= kMaxSeqs && (max_pages) > 0 && (b) * (max_pages) < (int64_t(1) << 31) &&              \
                     (max_pages) <= (int64_t(1) << 30) && (n_pages) > 0 && (n_pages) <= kMostPages,                       \
                 "%s: a table of %lld x %lld over %lld pages", name, (long long)(b), (long long)(max_pages),              \
                 (long long)(n_pages))

__device__ __forceinline__ bool holds(int e, int n_pages) { return e >= 0 && e < n_pages; }

// ---------------------------------------------------------------- fork

// An entry that stays what it was changes no count: rows that keep their sequence, and what beams share.
__global__ __launch_bounds__(256) void fork_kernel(const int32_t *old, int b, const int32_t *parent, int n, int32_t *out,
                                                   int32_t *refs, int n_pages, FastDiv m, int64_t most) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= most) return;
    const int row = static_cast<int>(m.div(static_cast<uint32_t>(i))), col = static_cast<int>(i - static_cast<int64_t>(row) * m.d);
    const int was = row < b ? old[i] : -1;
    int is = -1;
    if (row < n) {
        const int p = parent[row];
        if (p >= 0 && p < b) is = old[static_cast<int64_t>(p) * m.d + col];
        out[i] = is;
    }
    if (is == was) return;
    if (holds(is, n_pages)) atomicAdd(refs + is, 1);
    if (holds(was, n_pages)) atomicSub(refs + was, 1);
}

__global__ __launch_bounds__(256) void snapshot_kernel(const int32_t *x, int32_t *y, int64_t n) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i < n) y[i] = x[i];
}

// ---------------------------------------------------------------- trim

__global__ __launch_bounds__(256) void trim_kernel(int32_t *pages, int32_t *refs, const int32_t *context, int n_pages, FastDiv m,
                                                   int64_t entries, int page_shift, int window, int sinks) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= entries) return;
    const int row = static_cast<int>(m.div(static_cast<uint32_t>(i))), col = static_cast<int>(i - static_cast<int64_t>(row) * m.d);
    const int64_t start = static_cast<int64_t>(col) << page_shift, end = start + (int64_t(1) << page_shift);
    if (start < sinks || end > static_cast<int64_t>(context[row]) - window + 1) return;
    const int e = pages[i];
    if (e == -1) return;
    pages[i] = -1;
    if (holds(e, n_pages)) atomicSub(refs + e, 1);
}

// ---------------------------------------------------------------- one workgroup's sums in order

constexpr int kNT = 1024, kWaves = kNT / 64;

// Inclusive sums over the wave's lanes, by data-parallel moves: no trip through LDS.
template <int CTRL, int ROWS>
__device__ __forceinline__ int from_before(int x) {
    return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int sums_to_here(int x) {
    x += from_before<0x111, 0xf>(x);
    x += from_before<0x112, 0xf>(x);
    x += from_before<0x114, 0xf>(x);
    x += from_before<0x118, 0xf>(x);
    x += from_before<0x142, 0xa>(x);
    return x + from_before<0x143, 0xc>(x);
}

// The exclusive prefix of x over the workgroup, and the total. `sums` holds 2 * kWaves, used in turn by calls of changing
// `which`, so that one barrier is enough; every thread calls it.
__device__ __forceinline__ int block_prefix(int x, int *sums, int which, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, inc = sums_to_here(x);
    sums += which * kWaves;
    if (lane == 63) sums[w] = inc;
    __syncthreads();
    const int of = sums_to_here(lane < kWaves ? sums[lane] : 0);
    total = __builtin_amdgcn_readlane(of, kWaves - 1);
    return (w > 0 ? __shfl(of, w - 1, 64) : 0) + inc - x;
}

// ---------------------------------------------------------------- claim

struct ClaimArgs {
    int32_t *pages, *refs;
    const int32_t *q_start, *context;
    int32_t *src, *dst, *lacking;
    int32_t *items, *free_pages;  // workspace: a word an item, the free pages that are given out
    int b, m, n_pages, page_shift;
};

// Items are the (sequence, block) pairs that a step writes to, in order. Their words:
constexpr int kOwned = -2, kMissing = -1;  // else the id of a page that others hold too, with kKept where it stays
constexpr int kKept = 1 << 30;

// The blocks that sequence s writes to.
__device__ __forceinline__ void blocks_of(const ClaimArgs &a, int s, int &first, int &count, bool &partial) {
    constexpr int kMost = (1 << 30) + (1 << 24);
    int64_t n = static_cast<int64_t>(a.q_start[s + 1]) - a.q_start[s];
    n = n < 0 ? 0 : n > (1 << 24) ? (1 << 24) : n;
    int c = a.context[s];
    c = c < 0 ? 0 : c > kMost ? kMost : c;
    const int at = c - static_cast<int>(n) < 0 ? 0 : c - static_cast<int>(n);
    const int64_t cap = static_cast<int64_t>(a.m) << a.page_shift;
    const int end = c < cap ? c : static_cast<int>(cap);
    first = at >> a.page_shift;
    count = n == 0 || end <= at ? 0 : ((end - 1) >> a.page_shift) - first + 1;
    partial = (at & ((1 << a.page_shift) - 1)) != 0;
}

constexpr int kSlots = 2 * kNT;   // of a hash table over the shared pages of up to kNT items
constexpr int kItemsHere = 4096;  // items whose words, and free pages that, stay in LDS; the workspace has those past them

struct ClaimLds {
    int start[kNT], first[kNT];  // of kNT sequences: the items before theirs, their first block (and a bit: partly filled)
    int sums[2 * kWaves];
    __attribute__((aligned(16))) int items[kItemsHere];
    int free_pages[kItemsHere];
    int key[kSlots], writers[kSlots], last[kSlots];  // of a shared page: how many items write to it, and the last of them
};

// f(item, sequence, block, whether the block holds earlier positions) for all items in order, a workgroup's worth at a
// time; threads past the last get item -1. Returns the number of items.
template <typename F>
__device__ __forceinline__ int for_items(const ClaimArgs &a, ClaimLds &lds, F f) {
    int base = 0;
    for (int s0 = 0; s0 < a.b; s0 += kNT) {
        int total, first = 0, count = 0;
        bool partial = false;
        if (s0 + static_cast<int>(threadIdx.x) < a.b) blocks_of(a, s0 + threadIdx.x, first, count, partial);
        __syncthreads();
        lds.start[threadIdx.x] = block_prefix(count, lds.sums, 0, total);
        lds.first[threadIdx.x] = first << 1 | partial;
        __syncthreads();
        for (int i0 = 0; i0 < total; i0 += kNT) {
            const int i = i0 + threadIdx.x;
            int s = -1, j = 0;
            bool old = false;
            if (i < total) {  // the last sequence that starts at or before i (those without blocks start where the next does)
                int lo = 0;
#pragma unroll
                for (int half = kNT / 2; half >= 1; half >>= 1)
                    if (lds.start[lo + half] <= i) lo += half;
                const int first = lds.first[lo], k = i - lds.start[lo];
                s = s0 + lo;
                j = (first >> 1) + k;
                old = (first & 1) && k == 0;
            }
            f(i < total ? base + i : -1, s, j, old);
        }
        base += total;
        __syncthreads();
    }
    return base;
}

// How many of four words name page w, those from `end` on (counted from the first of them) left out.
__device__ __forceinline__ int named(const int *words, int w, int end) {
    typedef int four __attribute__((ext_vector_type(4)));
    const four x = *reinterpret_cast<const four *>(words);
    int n = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) n += ((x[k] ^ w) & ~kKept) == 0 && k < end;  // no page's word differs from it in the sign
    return n;
}

// One workgroup. A page of r owners to which c of them write is copied by the first min(c, r - 1), as if they came one
// after another: by all of them where c < r, by all but the last where c = r. Where a table has more entries of a page than its
// count says (c > r), and for items past the first kNT, a writer's rank is counted over the earlier items' words.
//
// Bound by its trips to memory, one after another (the starts, the entries, their counts, the free pages' counts, the answers), and
// by its instructions, each of which the 16 waves of one CU take turns for. 160 sequences that share pages, over 20011: 23.3
// us with a barrier for every kNT counts; 18.1 with all ranks counted over words in LDS, of which those took 8; 11.1 with the
// hash, while the compiler compared the counts (and so waited for them) where they were requested; 6.7 so.
__global__ __launch_bounds__(kNT) void claim_kernel(ClaimArgs a) {
    __shared__ ClaimLds lds;
    typedef int four __attribute__((ext_vector_type(4), aligned(4)));
    constexpr int U = 4, kWaveCounts = 4 * 64 * U;  // a thread requests U times four counts together, a wave as many neighbours
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    four count[U];
    auto first_of = [&](int p0, int k) { return p0 + w * kWaveCounts + (k * 64 + lane) * 4; };
    auto load_counts = [&](int p0) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int p = first_of(p0, k);
            count[k] = four{1, 1, 1, 1};
            if (p + 3 < a.n_pages) {
                count[k] = *reinterpret_cast<const four *>(a.refs + p);
            } else {
#pragma unroll
                for (int c = 0; c < 3; ++c)
                    if (p + c < a.n_pages) count[k][c] = a.refs[p + c];
            }
        }
    };
    for (int s = threadIdx.x; s < a.b; s += kNT) a.src[s] = a.dst[s] = -1;
    for (int s = threadIdx.x; s < kSlots; s += kNT) {
        lds.key[s] = lds.last[s] = -1;
        lds.writers[s] = 0;
    }
    int my_s = -1, my_j = 0, my_owners = 0;  // of item threadIdx.x, where there is one round of sequences and of items
    bool my_old = false;
    const int items = for_items(a, lds, [&](int i, int s, int j, bool old) {
        if (i < 0) return;
        const int e = a.pages[static_cast<int64_t>(s) * a.m + j];
        const int r = holds(e, a.n_pages) ? a.refs[e] : 0;
        const int word = r < 1 ? kMissing : r == 1 ? kOwned : e;
        if (i == static_cast<int>(threadIdx.x)) {
            my_s = s;
            my_j = j;
            my_old = old;
            my_owners = r;
        }
        if (i < kItemsHere) lds.items[i] = word;
        else a.items[i] = word;
    });
    const bool single = items <= kNT && a.b <= kNT;  // item i was thread i's
    if (items > kItemsHere) __threadfence_block();
    __syncthreads();
    load_counts(0);
    int need = 0, turn = 0, slot = 0;
    if (items <= kNT) {
        const int x = static_cast<int>(threadIdx.x) < items ? lds.items[threadIdx.x] : kOwned;
        if (x >= 0) {
            slot = static_cast<uint32_t>(x) * 2654435769u >> (32 - 11);
            static_assert(kSlots == 1 << 11, "the hash takes as many bits");
            for (;;) {  // at most kNT of the 2 kNT slots are taken, so it meets its key or a free one
                const int met = atomicCAS(&lds.key[slot], -1, x);
                if (met == -1 || met == x) break;
                slot = (slot + 1) & (kSlots - 1);
            }
            atomicAdd(&lds.writers[slot], 1);
            atomicMax(&lds.last[slot], static_cast<int>(threadIdx.x));
        }
        __syncthreads();
    }
    for (int i0 = 0; i0 < items; i0 += kNT) {
        const int i = i0 + threadIdx.x;
        int wants = 0, total;
        if (i < items) {
            const int x = i < kItemsHere ? lds.items[i] : a.items[i];
            if (x == kMissing) wants = 1;
            if (x >= 0) {
                const int r = single ? my_owners : a.refs[x], here = i < kItemsHere ? i : kItemsHere;
                if (items <= kNT && lds.writers[slot] <= r) {
                    wants = lds.writers[slot] < r || lds.last[slot] != i;
                } else {
                    int rank = 0;
                    for (int k = 0; k < here && rank < r - 1; k += 4) rank += named(lds.items + k, x, here - k);
                    for (int k = kItemsHere; k < i && rank < r - 1; ++k) rank += ((a.items[k] ^ x) & ~kKept) == 0;
                    wants = rank < r - 1;
                }
                if (!wants) {
                    if (i < kItemsHere) lds.items[i] = x | kKept;
                    else a.items[i] = x | kKept;
                }
            }
        }
        block_prefix(wants, lds.sums, turn ^= 1, total);
        need += total;
    }
    // the lowest free pages: a wave's, in order, after those of the waves before
    int found = 0;
    for (int p0 = 0; p0 < a.n_pages && found < need; p0 += kWaves * kWaveCounts) {
        if (p0 > 0) load_counts(p0);
        uint64_t is_free[U][4];
        int mine = 0, total;
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                int x = count[k][c];
                asm volatile("" : "+v"(x));  // not looked at before here, while the counts are under way
                is_free[k][c] = __ballot(x < 1);
                mine += __popcll(is_free[k][c]);
            }
        const int before = block_prefix(lane == 0 ? mine : 0, lds.sums, turn ^= 1, total);
        int at = found + __builtin_amdgcn_readfirstlane(before);
        if (at < need && mine > 0)
#pragma unroll
            for (int k = 0; k < U; ++k) {
                int to = at;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    to += __popcll(is_free[k][c] & ((uint64_t(1) << lane) - 1));
                    at += __popcll(is_free[k][c]);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (!(is_free[k][c] >> lane & 1)) continue;
                    if (to < need) {
                        if (to < kItemsHere) lds.free_pages[to] = first_of(p0, k) + c;
                        else a.free_pages[to] = first_of(p0, k) + c;
                    }
                    ++to;
                }
            }
        found += total;
    }
    if (threadIdx.x == 0) a.lacking[0] = need > found ? need - found : 0;
    if (need > found || need == 0) return;
    if (items > kItemsHere || need > kItemsHere) __threadfence_block();
    __syncthreads();
    int given = 0;
    auto give = [&](int i, int s, int j, bool old) {
        const int x = i < 0 ? kOwned : i < kItemsHere ? lds.items[i] : a.items[i];
        const bool wants = x == kMissing || (x >= 0 && !(x & kKept));
        int total;
        const int at = given + block_prefix(wants, lds.sums, turn ^= 1, total);
        given += total;
        if (!wants) return;
        const int p = at < kItemsHere ? lds.free_pages[at] : a.free_pages[at];
        a.pages[static_cast<int64_t>(s) * a.m + j] = p;
        a.refs[p] = 1;
        if (x >= 0) {
            atomicSub(a.refs + x, 1);
            if (old) {
                a.src[s] = x;
                a.dst[s] = p;
            }
        }
    };
    if (single)
        give(static_cast<int>(threadIdx.x) < items ? static_cast<int>(threadIdx.x) : -1, my_s, my_j, my_old);
    else
        for_items(a, lds, give);
}

// ---------------------------------------------------------------- compact

struct CompactArgs {
    int32_t *pages, *refs, *src, *dst, *used;
    int32_t *rank;    // workspace [n_pages]: of a used page the used ones before it, of a free one -1 - the free ones before it
    int32_t *counts;  // workspace: used pages of each kSpan
    int64_t entries;
    int n_pages, spans;
};

constexpr int kSpan = 4096;  // pages a workgroup of 1024 threads counts
// Spans up to which every workgroup counts all of them for itself, which saves the launch before (6001 pages: 12.0 -> 9.6 us a call).
constexpr int kFewSpans = 4;

// Thread's share of span `span`'s pages that are used.
__device__ __forceinline__ int used_of_span(const CompactArgs &a, int span) {
    int used = 0;
#pragma unroll
    for (int k = 0; k < kSpan / kNT; ++k) {
        const int p = span * kSpan + k * kNT + threadIdx.x;
        used += p < a.n_pages && a.refs[p] > 0;
    }
    return used;
}

// The first launch: how many pages of each span are used.
__global__ __launch_bounds__(kNT) void compact_count_kernel(CompactArgs a) {
    __shared__ int sums[2 * kWaves];
    int total;
    block_prefix(used_of_span(a, blockIdx.x), sums, 0, total);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = total;
}

// The second: every workgroup sums the spans' counts for itself (and the used pages before the first one past all of them, in
// whose span it looks), ranks its span's pages and writes the moves down.
__global__ __launch_bounds__(kNT) void compact_rank_kernel(CompactArgs a) {
    __shared__ int sums[2 * kWaves];
    int used, before, total, mine[kSpan / kNT];
#pragma unroll
    for (int k = 0; k < kSpan / kNT; ++k) {
        const int p = blockIdx.x * kSpan + k * kNT + threadIdx.x;
        mine[k] = p < a.n_pages && a.refs[p] > 0;
    }
    int all = 0, here = 0, of[kFewSpans] = {};
    const bool few = a.spans <= kFewSpans;
    if (few) {
#pragma unroll
        for (int i = 0; i < kFewSpans; ++i) {
            of[i] = used_of_span(a, i);
            all += of[i];
            here += i < static_cast<int>(blockIdx.x) ? of[i] : 0;
        }
    } else {
        for (int i = threadIdx.x; i < a.spans; i += kNT) {
            const int c = a.counts[i];
            all += c;
            here += i < static_cast<int>(blockIdx.x) ? c : 0;
        }
    }
    block_prefix(all, sums, 0, used);
    block_prefix(here, sums, 1, before);
    const int at = used / kSpan;  // the span that page `used` is in (or past the last)
    int low = 0, below;
    if (few) {
#pragma unroll
        for (int i = 0; i < kFewSpans; ++i) low += i < at ? of[i] : 0;
    } else {
        for (int i = threadIdx.x; i < a.spans; i += kNT) low += i < at ? a.counts[i] : 0;
    }
#pragma unroll
    for (int k = 0; k < kSpan / kNT; ++k) {
        const int p = at * kSpan + k * kNT + threadIdx.x;
        low += p < used && p < a.n_pages && a.refs[p] > 0;
    }
    block_prefix(low, sums, 0, below);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.used[0] = used;
        a.counts[a.spans] = below;
    }
    const int moves = used - below;
#pragma unroll
    for (int k = 0; k < kSpan / kNT; ++k) {
        const int p = blockIdx.x * kSpan + k * kNT + threadIdx.x;
        const int r = before + block_prefix(mine[k], sums, (k & 1) ^ 1, total);
        before += total;
        if (p >= a.n_pages) continue;
        a.rank[p] = mine[k] ? r : -1 - (p - r);
        if (mine[k] && p >= used) a.src[r - below] = p;
        if (!mine[k] && p < used) a.dst[p - r] = p;
        if (p >= moves) a.src[p] = a.dst[p] = -1;
    }
}

// The third: counts and entries.
__global__ __launch_bounds__(256) void compact_apply_kernel(CompactArgs a) {
    const int used = a.used[0], below = a.counts[a.spans];
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i < used - below) {
        const int s = a.src[i];
        a.refs[a.dst[i]] = a.refs[s];
        a.refs[s] = 0;
    } else if (i >= used && i < a.n_pages && a.rank[i] < 0) {
        a.refs[i] = 0;
    }
    if (i < a.entries) {
        const int e = a.pages[i], r = holds(e, a.n_pages) ? a.rank[e] : -1;
        const int to = r < 0 ? -1 : e < used ? e : a.dst[r - below];
        if (to != e) a.pages[i] = to;
    }
}

// ---------------------------------------------------------------- copy

constexpr int kMostCaches = 64;

// MOST: caches there is room for (a launch copies the arguments, and one layer's keys and values need no kilobytes of them).
template <int MOST>
struct CopyArgs {
    uint8_t *cache[MOST];
    int64_t stride[MOST];   // bytes from page to page
    uint32_t units[MOST];   // of 16 bytes in a page
    uint32_t slices[MOST];  // the caches' pages are cut into slices of at most kSlice units: those before the next cache's
    FastDiv by_last[MOST];  // by the units of a cache's last slice
    FastDiv by_slice;
    const int32_t *src, *dst;
    int n, n_pages;
};

// Units a thread requests together, and a workgroup's at a time.
constexpr int kRequests = 2, kSlice = 256 * kRequests;
constexpr int64_t kMostSlices = 65535, kMostPageBytes = kMostSlices * kSlice * 16;  // of a launch, a slice a row of its grid
constexpr int64_t kCopyFill = 8192;  // workgroups: 866 pages of 64 KB and 18980 of 2.5 KB 24.2 and 21.9 us with 4 requests and 4096, 23.6 and 21.1 so; each 4 us less with stores past the caches, which a list of pages fills

// HBM-bound: every byte read once and written once. A workgroup takes one slice of every gridDim.x-th pair's pages, 256 pairs at
// a time: those that copy something are put together first, so that a list with few of them, or with all of them in front, is
// shared out as evenly as a full one, and small pages fill a workgroup.
template <int MOST>
__global__ __launch_bounds__(256) void copy_kernel(CopyArgs<MOST> a) {
    __shared__ int from[256], to[256], waves[4];
    uint32_t c = 0, slice = blockIdx.y;
    while (slice >= a.slices[c]) ++c;
    if (c > 0) slice -= a.slices[c - 1];
    const uint32_t u0 = slice * kSlice, units = a.units[c] - u0 < kSlice ? a.units[c] - u0 : kSlice;
    const FastDiv by_units = units == kSlice ? a.by_slice : a.by_last[c];
    uint8_t *base = a.cache[c] + static_cast<int64_t>(u0) * 16;
    const int64_t stride = a.stride[c];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int64_t i0 = blockIdx.x; i0 < a.n; i0 += 256 * static_cast<int64_t>(gridDim.x)) {
        const int64_t i = i0 + static_cast<int64_t>(threadIdx.x) * gridDim.x;
        const int s = i < a.n ? a.src[i] : -1, d = i < a.n ? a.dst[i] : -1;
        const bool copies = holds(s, a.n_pages) && holds(d, a.n_pages);
        const uint64_t mask = __ballot(copies);
        __syncthreads();
        if (lane == 0) waves[w] = __popcll(mask);
        __syncthreads();
        int at = __popcll(mask & ((uint64_t(1) << lane) - 1)), pairs = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (k < w) at += waves[k];
            pairs += waves[k];
        }
        if (copies) {
            from[at] = s;
            to[at] = d;
        }
        __syncthreads();
        const uint32_t all = static_cast<uint32_t>(pairs) * units;
        for (uint32_t t0 = threadIdx.x; t0 < all; t0 += kSlice) {
            float4_t x[kRequests];
#pragma unroll
            for (int k = 0; k < kRequests; ++k) {
                const uint32_t t = t0 + k * 256, p = by_units.div(t);
                if (t < all) x[k] = *reinterpret_cast<const float4_t *>(base + from[p] * stride + static_cast<int64_t>(t - p * units) * 16);
            }
#pragma unroll
            for (int k = 0; k < kRequests; ++k) {
                const uint32_t t = t0 + k * 256, p = by_units.div(t);
                if (t < all) __builtin_nontemporal_store(x[k], reinterpret_cast<float4_t *>(base + to[p] * stride + static_cast<int64_t>(t - p * units) * 16));
            }
        }
    }
}

// One launch for the first of the caches, as many as it has room for: how many.
template <int MOST>
int64_t copy_some(void **caches, const int64_t *page_bytes, const int64_t *page_strides, int64_t n_caches, const int32_t *src,
                  const int32_t *dst, int64_t n, int64_t n_pages, hipStream_t stream) {
    CopyArgs<MOST> a;
    int64_t slices = 0, c = 0;
    for (; c < MOST && c < n_caches; ++c) {
        const int64_t units = page_bytes[c] / 16, more = (units + kSlice - 1) / kSlice;
        if (c > 0 && slices + more > kMostSlices) break;
        slices += more;
        a.cache[c] = static_cast<uint8_t *>(caches[c]);
        a.stride[c] = page_strides[c];
        a.units[c] = static_cast<uint32_t>(units);
        a.slices[c] = static_cast<uint32_t>(slices);
        a.by_last[c] = FastDiv(static_cast<uint32_t>(units - (more - 1) * kSlice));
    }
    a.by_slice = FastDiv(kSlice);
    a.src = src;
    a.dst = dst;
    a.n = static_cast<int>(n);
    a.n_pages = static_cast<int>(n_pages);
    // enough workgroups that the pairs which copy something, few or many, keep the chip busy
    int64_t x = (kCopyFill + slices - 1) / slices;
    x = x < n ? x : n;
    copy_kernel<MOST><<<dim3(static_cast<unsigned>(x), static_cast<unsigned>(slices)), 256, 0, stream>>>(a);
    return c;
}

// Two pools that share memory without being one and the same (which is then copied twice, to the same end), or false. In order
// of address each meets those alone that begin before its end: none where every pool is an allocation, all where the layers'
// pages lie side by side in one, and there strides that are equal tell.
inline bool pools_meet(const ByteRows *pools, int32_t *order, int64_t n, int32_t &one, int32_t &other) {
    const auto from = [&](int64_t i) { return reinterpret_cast<uintptr_t>(pools[order[i]].p); };
    for (int64_t i = 0; i < n; ++i) order[i] = static_cast<int32_t>(i);
    std::sort(order, order + n, [&](int32_t i, int32_t j) { return pools[i].p < pools[j].p; });
    for (int64_t i = 0; i + 1 < n; ++i) {
        const ByteRows &x = pools[order[i]];
        const __int128 end = static_cast<__int128>(from(i)) + static_cast<__int128>(x.n - 1) * x.stride + x.width;
        for (int64_t j = i + 1; j < n && static_cast<__int128>(from(j)) < end; ++j) {
            const ByteRows &y = pools[order[j]];
            const uintptr_t apart = from(j) - from(i);
            const bool alike = x.stride == y.stride;
            if (alike && apart >= static_cast<uintptr_t>(x.width) && apart + static_cast<uintptr_t>(y.width) <= static_cast<uintptr_t>(x.stride)) continue;
            if (apart == 0 && alike && x.width == y.width) continue;
            if (!share_bytes(x, y)) continue;
            one = order[i];
            other = order[j];
            return true;
        }
    }
    return false;
}

inline unsigned blocks_for(int64_t n) { return static_cast<unsigned>((n + 255) / 256); }

}  // namespace
}  // namespace dtts

extern "C" int dtts_fork_pages(const int32_t *pages, int32_t *refs, const int32_t *parent, int32_t *out, int64_t b, int64_t n,
                               int64_t max_pages, int64_t n_pages, void *workspace, size_t ws_bytes, hipStream_t stream) {
    using namespace dtts;
    const char *name = "dtts_fork_pages";
    DTTS_REQUIRE_TABLE(name, b, max_pages, n_pages);
    DTTS_REQUIRE_TABLE(name, n, max_pages, n_pages);
    const int64_t most = (b > n ? b : n) * max_pages;
    if (most == 0) return DTTS_OK;
    DTTS_REQUIRE(refs && (b == 0 || pages) && (n == 0 || (parent && out)), "%s: null pointer", name);
    DTTS_REQUIRE(aligned(pages, 4) && aligned(refs, 4) && aligned(parent, 4) && aligned(out, 4), "%s: misaligned operand", name);
    const int64_t was = b * max_pages * 4, is = n * max_pages * 4;
    const bool in_place = pages == out && b == n;
    DTTS_REQUIRE(in_place || !share_bytes({pages, 1, 0, was}, {out, 1, 0, is}), "%s: the new table is the old one or no part of it", name);
    DTTS_REQUIRE(!share_bytes({refs, 1, 0, n_pages * 4}, {pages, 1, 0, was}) && !share_bytes({refs, 1, 0, n_pages * 4}, {out, 1, 0, is}) &&
                     !share_bytes({refs, 1, 0, n_pages * 4}, {parent, 1, 0, n * 4}) && !share_bytes({parent, 1, 0, n * 4}, {out, 1, 0, is}),
                 "%s: operands share memory", name);
    const int32_t *old = pages;
    if (in_place) {
        DTTS_REQUIRE(workspace && ws_bytes >= static_cast<size_t>(was) && aligned(workspace, 4),
                     "%s: a table in its own place needs a workspace of %lld bytes", name, (long long)was);
        DTTS_REQUIRE(!share_bytes({workspace, 1, 0, was}, {pages, 1, 0, was}) && !share_bytes({workspace, 1, 0, was}, {refs, 1, 0, n_pages * 4}) &&
                         !share_bytes({workspace, 1, 0, was}, {parent, 1, 0, n * 4}),
                     "%s: operands share memory", name);
        snapshot_kernel<<<blocks_for(b * max_pages), 256, 0, stream>>>(pages, static_cast<int32_t *>(workspace), b * max_pages);
        DTTS_LAUNCH_CHECK(name);
        old = static_cast<int32_t *>(workspace);
    }
    fork_kernel<<<blocks_for(most), 256, 0, stream>>>(old, static_cast<int>(b), parent, static_cast<int>(n), out, refs,
                                                      static_cast<int>(n_pages), FastDiv(static_cast<uint32_t>(max_pages)), most);
    DTTS_LAUNCH_CHECK(name);
    return DTTS_OK;
}

extern "C" int dtts_trim_pages(int32_t *pages, int32_t *refs, const int32_t *context, int64_t b, int64_t page, int64_t max_pages,
                               int64_t n_pages, int64_t window, int64_t sinks, hipStream_t stream) {
    using namespace dtts;
    const char *name = "dtts_trim_pages";
    DTTS_REQUIRE_TABLE(name, b, max_pages, n_pages);
    DTTS_REQUIRE_PAGE(name, page, max_pages);
    DTTS_REQUIRE(window > 0 && window < (int64_t(1) << 31) && sinks >= 0 && sinks < (int64_t(1) << 31), "%s: window %lld, sinks %lld", name,
                 (long long)window, (long long)sinks);
    if (b == 0) return DTTS_OK;
    DTTS_REQUIRE(pages && refs && context, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(pages, 4) && aligned(refs, 4) && aligned(context, 4), "%s: misaligned operand", name);
    const ByteRows t{pages, 1, 0, b * max_pages * 4}, r{refs, 1, 0, n_pages * 4}, c{context, 1, 0, b * 4};
    DTTS_REQUIRE(!share_bytes(t, r) && !share_bytes(t, c) && !share_bytes(r, c), "%s: operands share memory", name);
    trim_kernel<<<blocks_for(b * max_pages), 256, 0, stream>>>(pages, refs, context, static_cast<int>(n_pages),
                                                               FastDiv(static_cast<uint32_t>(max_pages)), b * max_pages, log2_of(page),
                                                               static_cast<int>(window), static_cast<int>(sinks));
    DTTS_LAUNCH_CHECK(name);
    return DTTS_OK;
}

extern "C" size_t dtts_claim_pages_workspace_bytes(int64_t b, int64_t max_pages, int64_t n_pages) {
    using namespace dtts;
    if (b < 1 || b > kMaxSeqs || max_pages < 1 || max_pages > (int64_t(1) << 30) || b * max_pages >= (int64_t(1) << 31) || n_pages < 1 ||
        n_pages > kMostPages)
        return 0;
    return static_cast<size_t>(b * max_pages + n_pages) * 4;
}

extern "C" int dtts_claim_pages(int32_t *pages, int32_t *refs, const int32_t *q_start, const int32_t *context, int32_t *src, int32_t *dst,
                                int32_t *lacking, int64_t b, int64_t page, int64_t max_pages, int64_t n_pages, void *workspace,
                                size_t ws_bytes, hipStream_t stream) {
    using namespace dtts;
    const char *name = "dtts_claim_pages";
    DTTS_REQUIRE_TABLE(name, b, max_pages, n_pages);
    DTTS_REQUIRE_PAGE(name, page, max_pages);
    DTTS_REQUIRE(b * max_pages <= (int64_t(1) << 31) - kNT, "%s: a table of %lld x %lld has items past an int in its last round", name,
                 (long long)b, (long long)max_pages);
    // counts and `lacking` are read and written without sequences too
    DTTS_REQUIRE(lacking && refs && aligned(lacking, 4) && aligned(refs, 4), "%s: counts or lacking null or misaligned", name);
    const size_t need = b > 0 ? dtts_claim_pages_workspace_bytes(b, max_pages, n_pages) : 0;
    if (b > 0) {
        DTTS_REQUIRE(pages && q_start && context && src && dst, "%s: null pointer", name);
        DTTS_REQUIRE(aligned(pages, 4) && aligned(q_start, 4) && aligned(context, 4) && aligned(src, 4) && aligned(dst, 4),
                     "%s: misaligned operand", name);
        DTTS_REQUIRE(workspace && ws_bytes >= need && aligned(workspace, 4), "%s: a workspace of %zu bytes is needed", name, need);
    }
    const int64_t rows = b > 0 ? 1 : 0;  // arrays of a batch without sequences are not looked at
    const ByteRows of[] = {{refs, 1, 0, n_pages * 4}, {lacking, 1, 0, 4}, {pages, rows, 0, b * max_pages * 4}, {src, rows, 0, b * 4},
                           {dst, rows, 0, b * 4}, {workspace, rows, 0, static_cast<int64_t>(need)}, {q_start, rows, 0, (b + 1) * 4},
                           {context, rows, 0, b * 4}};
    for (int i = 0; i < 6; ++i)
        for (int j = i + 1; j < 8; ++j) DTTS_REQUIRE(!share_bytes(of[i], of[j]), "%s: operands share memory", name);
    ClaimArgs a;
    a.pages = pages;
    a.refs = refs;
    a.q_start = q_start;
    a.context = context;
    a.src = src;
    a.dst = dst;
    a.lacking = lacking;
    a.items = static_cast<int32_t *>(workspace);
    a.free_pages = a.items + b * max_pages;
    a.b = static_cast<int>(b);
    a.m = static_cast<int>(max_pages);
    a.n_pages = static_cast<int>(n_pages);
    a.page_shift = log2_of(page);
    claim_kernel<<<1, kNT, 0, stream>>>(a);
    DTTS_LAUNCH_CHECK(name);
    return DTTS_OK;
}

extern "C" size_t dtts_compact_pages_workspace_bytes(int64_t n_pages) {
    using namespace dtts;
    return n_pages < 1 || n_pages > kMostPages ? 0 : static_cast<size_t>(n_pages + (n_pages + kSpan - 1) / kSpan + 1) * 4;
}

extern "C" int dtts_compact_pages(int32_t *pages, int32_t *refs, int32_t *src, int32_t *dst, int32_t *used, int64_t b, int64_t max_pages,
                                  int64_t n_pages, void *workspace, size_t ws_bytes, hipStream_t stream) {
    using namespace dtts;
    const char *name = "dtts_compact_pages";
    DTTS_REQUIRE_TABLE(name, b, max_pages, n_pages);
    DTTS_REQUIRE((b == 0 || pages) && refs && src && dst && used, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(pages, 4) && aligned(refs, 4) && aligned(src, 4) && aligned(dst, 4) && aligned(used, 4), "%s: misaligned operand",
                 name);
    const size_t need = dtts_compact_pages_workspace_bytes(n_pages);
    DTTS_REQUIRE(workspace && ws_bytes >= need && aligned(workspace, 4), "%s: a workspace of %zu bytes is needed", name, need);
    const ByteRows of[] = {{pages, 1, 0, b * max_pages * 4}, {refs, 1, 0, n_pages * 4}, {src, 1, 0, n_pages * 4}, {dst, 1, 0, n_pages * 4},
                           {used, 1, 0, 4}, {workspace, 1, 0, static_cast<int64_t>(need)}};
    for (int i = 0; i < 6; ++i)
        for (int j = i + 1; j < 6; ++j)
            DTTS_REQUIRE(of[i].width == 0 || of[j].width == 0 || !share_bytes(of[i], of[j]), "%s: operands share memory", name);
    CompactArgs a;
    a.pages = pages;
    a.refs = refs;
    a.src = src;
    a.dst = dst;
    a.used = used;
    a.rank = static_cast<int32_t *>(workspace);
    a.counts = a.rank + n_pages;
    a.entries = b * max_pages;
    a.n_pages = static_cast<int>(n_pages);
    a.spans = static_cast<int>((n_pages + kSpan - 1) / kSpan);
    if (a.spans > kFewSpans) {
        compact_count_kernel<<<a.spans, kNT, 0, stream>>>(a);
        DTTS_LAUNCH_CHECK(name);
    }
    compact_rank_kernel<<<a.spans, kNT, 0, stream>>>(a);
    DTTS_LAUNCH_CHECK(name);
    compact_apply_kernel<<<blocks_for(a.entries > n_pages ? a.entries : n_pages), 256, 0, stream>>>(a);
    DTTS_LAUNCH_CHECK(name);
    return DTTS_OK;
}

extern "C" int dtts_copy_pages(void **caches, const int64_t *page_bytes, const int64_t *page_strides, int64_t n_caches,
                               const int32_t *src, const int32_t *dst, int64_t n, int64_t n_pages, hipStream_t stream) {
    using namespace dtts;
    const char *name = "dtts_copy_pages";
    DTTS_REQUIRE(n_caches >= 0 && n_caches <= 65536 && n >= 0 && n < (int64_t(1) << 31) && n_pages > 0 && n_pages < (int64_t(1) << 31),
                 "%s: %lld pairs in %lld caches of %lld pages", name, (long long)n, (long long)n_caches, (long long)n_pages);
    if (n == 0 || n_caches == 0) return DTTS_OK;
    DTTS_REQUIRE(caches && page_bytes && page_strides && src && dst, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(src, 4) && aligned(dst, 4), "%s: misaligned operand", name);
    for (int64_t c = 0; c < n_caches; ++c) {
        DTTS_REQUIRE(caches[c] && aligned(caches[c], 16), "%s: cache %lld is null or not 16-byte aligned", name, (long long)c);
        DTTS_REQUIRE(page_bytes[c] > 0 && page_bytes[c] % 16 == 0 && page_bytes[c] <= kMostPageBytes && page_strides[c] % 16 == 0 &&
                         page_strides[c] >= page_bytes[c] && page_strides[c] < (int64_t(1) << 34),
                     "%s: pages of %lld bytes, %lld apart (multiples of 16, up to %lld and under 2^34)", name, (long long)page_bytes[c],
                     (long long)page_strides[c], (long long)kMostPageBytes);
    }
    const std::unique_ptr<ByteRows[]> pools(new (std::nothrow) ByteRows[n_caches]);
    const std::unique_ptr<int32_t[]> order(new (std::nothrow) int32_t[n_caches]);
    DTTS_REQUIRE(pools && order, "%s: no host memory for %lld caches", name, (long long)n_caches);
    for (int64_t c = 0; c < n_caches; ++c) {
        pools[c] = {caches[c], n_pages, page_strides[c], page_bytes[c]};
        DTTS_REQUIRE(!share_bytes(pools[c], {src, 1, 0, n * 4}) && !share_bytes(pools[c], {dst, 1, 0, n * 4}),
                     "%s: cache %lld and the pairs share memory", name, (long long)c);
    }
    int32_t one, other;
    DTTS_REQUIRE(!pools_meet(pools.get(), order.get(), n_caches, one, other), "%s: caches %d and %d share memory", name, one, other);
    for (int64_t c0 = 0; c0 < n_caches;) {
        const int64_t done = n_caches - c0 <= 2 ? copy_some<2>(caches + c0, page_bytes + c0, page_strides + c0, n_caches - c0, src, dst, n, n_pages, stream)
                                                : copy_some<kMostCaches>(caches + c0, page_bytes + c0, page_strides + c0, n_caches - c0, src, dst,
                                                                         n, n_pages, stream);
        DTTS_LAUNCH_CHECK(name);
        c0 += done;
    }
    return DTTS_OK;
}
