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

// The exclusive prefix of x over the workgroup, and the total. `sums` holds kWaves + 1; every thread calls it.
__device__ __forceinline__ int block_prefix(int x, int *sums, int &total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int inc = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int v = __shfl_up(inc, off, 64);
        if (lane >= off) inc += v;
    }
    if (lane == 63) sums[w] = inc;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const int v = sums[i];
        if (i < w) before += v;
        total += v;
    }
    __syncthreads();
    return before + inc - x;
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

// f(item, sequence, block, whether the block holds earlier positions) for all items in order, a workgroup's worth at a
// time; threads past the last get item -1. Returns the number of items.
template <typename F>
__device__ __forceinline__ int for_items(const ClaimArgs &a, int *starts, int *sums, F f) {
    int base = 0;
    for (int s0 = 0; s0 < a.b; s0 += kNT) {
        int first = 0, count = 0, total;
        bool partial = false;
        if (s0 + static_cast<int>(threadIdx.x) < a.b) blocks_of(a, s0 + threadIdx.x, first, count, partial);
        starts[threadIdx.x] = block_prefix(count, sums, total);
        __syncthreads();
        for (int i0 = 0; i0 < total; i0 += kNT) {
            const int i = i0 + threadIdx.x;
            int s = -1, j = 0;
            bool old = false;
            if (i < total) {  // the last sequence that starts at or before i (those without blocks start where the next does)
                int lo = 0, hi = kNT - 1;
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (starts[mid] <= i) lo = mid; else hi = mid - 1;
                }
                s = s0 + lo;
                int c;
                blocks_of(a, s, first, c, partial);
                j = first + i - starts[lo];
                old = partial && i == starts[lo];
            }
            f(i < total ? base + i : -1, s, j, old);
        }
        base += total;
        __syncthreads();
    }
    return base;
}

// One workgroup. A page of r owners to which c of them write is copied by the first min(c, r - 1), as if they came one
// after another; a writer's rank among them is counted over the earlier items' words.
__global__ __launch_bounds__(kNT) void claim_kernel(ClaimArgs a) {
    __shared__ int starts[kNT], sums[kWaves];
    for (int s = threadIdx.x; s < a.b; s += kNT) a.src[s] = a.dst[s] = -1;
    const int items = for_items(a, starts, sums, [&](int i, int s, int j, bool) {
        if (i < 0) return;
        const int e = a.pages[static_cast<int64_t>(s) * a.m + j];
        const int r = holds(e, a.n_pages) ? a.refs[e] : 0;
        a.items[i] = r < 1 ? kMissing : r == 1 ? kOwned : e;
    });
    __threadfence_block();
    __syncthreads();
    int need = 0;
    for (int i0 = 0; i0 < items; i0 += kNT) {
        const int i = i0 + threadIdx.x;
        int wants = 0, total;
        if (i < items) {
            const int w = a.items[i];
            if (w == kMissing) wants = 1;
            if (w >= 0) {
                const int r = a.refs[w];
                int rank = 0;
                for (int k = 0; k < i && rank < r - 1; ++k) {
                    const int x = a.items[k];
                    rank += x >= 0 && (x & ~kKept) == w;
                }
                wants = rank < r - 1;
                if (!wants) a.items[i] = w | kKept;
            }
        }
        block_prefix(wants, sums, total);
        need += total;
    }
    // the lowest free pages
    int found = 0;
    for (int p0 = 0; p0 < a.n_pages && found < need; p0 += kNT) {
        const int p = p0 + threadIdx.x;
        const int is_free = p < a.n_pages && a.refs[p] < 1;
        int total;
        const int at = found + block_prefix(is_free, sums, total);
        if (is_free && at < need) a.free_pages[at] = p;
        found += total;
    }
    if (threadIdx.x == 0) a.lacking[0] = need > found ? need - found : 0;
    if (need > found || need == 0) return;
    __threadfence_block();
    __syncthreads();
    int given = 0;
    for_items(a, starts, sums, [&](int i, int s, int j, bool old) {
        const int w = i < 0 ? kOwned : a.items[i];
        const bool wants = w == kMissing || (w >= 0 && !(w & kKept));
        int total;
        const int at = given + block_prefix(wants, sums, total);
        given += total;
        if (!wants) return;
        const int p = a.free_pages[at];
        a.pages[static_cast<int64_t>(s) * a.m + j] = p;
        a.refs[p] = 1;
        if (w >= 0) {
            atomicSub(a.refs + w, 1);
            if (old) {
                a.src[s] = w;
                a.dst[s] = p;
            }
        }
    });
}

// ---------------------------------------------------------------- compact

struct CompactArgs {
    int32_t *pages, *refs, *src, *dst, *used;
    int32_t *rank;  // workspace [n_pages]: of a used page the used ones before it, of a free one -1 - the free ones before it
    int32_t *below; // workspace: the used pages under the count of all used ones
    int64_t entries;
    int n_pages;
};

__global__ __launch_bounds__(kNT) void compact_rank_kernel(CompactArgs a) {
    __shared__ int sums[kWaves];
    int count = 0;
    for (int p0 = 0; p0 < a.n_pages; p0 += kNT) {
        const int p = p0 + threadIdx.x, is_used = p < a.n_pages && a.refs[p] > 0;
        int total;
        const int at = count + block_prefix(is_used, sums, total);
        if (p < a.n_pages) a.rank[p] = is_used ? at : -1 - (p - at);
        count += total;
    }
    if (threadIdx.x == 0) {
        a.used[0] = count;
        a.below[0] = count;
    }
    __threadfence_block();
    __syncthreads();
    // the rank of the first page past them, whichever kind it is
    if (threadIdx.x == 0 && count < a.n_pages) a.below[0] = a.rank[count] >= 0 ? a.rank[count] : count - (-1 - a.rank[count]);
}

__global__ __launch_bounds__(256) void compact_pairs_kernel(CompactArgs a) {
    const int p = blockIdx.x * 256 + threadIdx.x;
    if (p >= a.n_pages) return;
    const int used = a.used[0], below = a.below[0], r = a.rank[p];
    if (r >= 0 && p >= used) a.src[r - below] = p;
    if (r < 0 && p < used) a.dst[-1 - r] = p;
    if (p >= used - below) a.src[p] = a.dst[p] = -1;
}

__global__ __launch_bounds__(256) void compact_apply_kernel(CompactArgs a) {
    const int used = a.used[0], below = a.below[0];
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

struct CopyArgs {
    uint8_t *cache[kMostCaches];
    int64_t stride[kMostCaches];  // bytes from page to page
    int parts[kMostCaches];       // 16-byte parts of a page
    const int32_t *src, *dst;
    int n, n_pages;
};

__global__ __launch_bounds__(256) void copy_kernel(CopyArgs a) {
    const int i = blockIdx.x, c = blockIdx.y;
    const int s = a.src[i], d = a.dst[i];
    if (!holds(s, a.n_pages) || !holds(d, a.n_pages)) return;
    const float4_t *x = reinterpret_cast<const float4_t *>(a.cache[c] + s * a.stride[c]);
    float4_t *y = reinterpret_cast<float4_t *>(a.cache[c] + d * a.stride[c]);
    for (int k = threadIdx.x; k < a.parts[c]; k += 256) y[k] = x[k];
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
    DTTS_REQUIRE(lacking && aligned(lacking, 4), "%s: null or misaligned pointer", name);
    const size_t need = dtts_claim_pages_workspace_bytes(b, max_pages, n_pages);
    if (b > 0) {
        DTTS_REQUIRE(pages && refs && q_start && context && src && dst, "%s: null pointer", name);
        DTTS_REQUIRE(aligned(pages, 4) && aligned(refs, 4) && aligned(q_start, 4) && aligned(context, 4) && aligned(src, 4) && aligned(dst, 4),
                     "%s: misaligned operand", name);
        DTTS_REQUIRE(workspace && ws_bytes >= need && aligned(workspace, 4), "%s: a workspace of %zu bytes is needed", name, need);
        const ByteRows of[] = {{pages, 1, 0, b * max_pages * 4}, {refs, 1, 0, n_pages * 4}, {src, 1, 0, b * 4}, {dst, 1, 0, b * 4},
                               {lacking, 1, 0, 4}, {workspace, 1, 0, static_cast<int64_t>(need)}, {q_start, 1, 0, (b + 1) * 4},
                               {context, 1, 0, b * 4}};
        for (int i = 0; i < 6; ++i)
            for (int j = i + 1; j < 8; ++j) DTTS_REQUIRE(!share_bytes(of[i], of[j]), "%s: operands share memory", name);
    }
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
    return n_pages < 1 || n_pages > dtts::kMostPages ? 0 : static_cast<size_t>(n_pages + 1) * 4;
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
    a.below = static_cast<int32_t *>(workspace);
    a.rank = a.below + 1;
    a.entries = b * max_pages;
    a.n_pages = static_cast<int>(n_pages);
    compact_rank_kernel<<<1, kNT, 0, stream>>>(a);
    DTTS_LAUNCH_CHECK(name);
    compact_pairs_kernel<<<blocks_for(n_pages), 256, 0, stream>>>(a);
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
        DTTS_REQUIRE(page_bytes[c] > 0 && page_bytes[c] % 16 == 0 && page_bytes[c] < (int64_t(1) << 34) && page_strides[c] % 16 == 0 &&
                         page_strides[c] >= page_bytes[c] && page_strides[c] < (int64_t(1) << 34),
                     "%s: pages of %lld bytes, %lld apart (multiples of 16 under 2^34)", name, (long long)page_bytes[c],
                     (long long)page_strides[c]);
    }
    for (int64_t c0 = 0; c0 < n_caches; c0 += kMostCaches) {
        CopyArgs a;
        const int64_t left = n_caches - c0, some = left < kMostCaches ? left : kMostCaches;
        for (int64_t c = 0; c < some; ++c) {
            a.cache[c] = static_cast<uint8_t *>(caches[c0 + c]);
            a.stride[c] = page_strides[c0 + c];
            a.parts[c] = static_cast<int>(page_bytes[c0 + c] / 16);
        }
        a.src = src;
        a.dst = dst;
        a.n = static_cast<int>(n);
        a.n_pages = static_cast<int>(n_pages);
        copy_kernel<<<dim3(static_cast<unsigned>(n), static_cast<unsigned>(some)), 256, 0, stream>>>(a);
        DTTS_LAUNCH_CHECK(name);
    }
    return DTTS_OK;
}
