// A ragged batch over a paged f16 KV cache, as the append and the attention see it.
//
//   pages       k and v, [n_pages, n_kv, page, D] with page_stride elements between pages
//   page_table  [b, max_pages]: sequence s's position p lives in page page_table[s, p / page]
//   q_start     [b + 1]: sequence s's new tokens are rows q_start[s] .. q_start[s + 1] - 1 of the batch
//   context     [b]: its positions so far, the new ones included, so row q_start[s] + i is at
//               position context[s] - n + i
//
// All of them are device arrays, so a captured graph stays valid from step to step; the host cannot
// check them, so every value is checked where it is used and an impossible one selects nothing: rows
// past q_start[b] belong to no sequence, and a page id outside [0, n_pages) holds no position.
#pragma once

#include "common.hpp"

namespace dtts {
namespace {

constexpr int64_t kMaxSeqs = 1 << 16;

struct PagedBatch {
    const int32_t *q_start, *context, *table;
    int tokens, b;
    int page_shift, n_pages, max_pages;
    int64_t page_stride;

    // Sequence s's first row and row count: clipped to the batch, so that no value of q_start reaches
    // outside it.
    __device__ __forceinline__ void rows(int s, int &first, int &n) const { clip(q_start[s], q_start[s + 1], first, n); }
    __device__ __forceinline__ void clip(int lo, int hi, int &first, int &n) const {
        first = lo < 0 ? 0 : lo > tokens ? tokens : lo;
        const int end = hi > tokens ? tokens : hi;
        n = end > first ? end - first : 0;
    }

    // Sequence s's length. A table holds 2^30 positions at most and a batch 2^24 tokens: clipped so that positions,
    // and a kernel's look ahead of them, stay ints, and none of an impossible length's is in a table.
    __device__ __forceinline__ int length(int s) const { return clip(context[s]); }
    __device__ __forceinline__ static int clip(int c) {
        constexpr int kMost = (1 << 30) + (1 << 24);
        return c < 0 ? 0 : c > kMost ? kMost : c;
    }

    // The page of position-block `at` (position >> page_shift) of sequence s, or -1.
    __device__ __forceinline__ int page(int s, int at) const {
        if (at < 0 || at >= max_pages) return -1;
        const int id = table[static_cast<int64_t>(s) * max_pages + at];
        return id >= 0 && id < n_pages ? id : -1;
    }

    // The sequence that the wave's row t belongs to: how many of them end at or before it (b: all of
    // them). The wave reads 64 ends at a time and counts with ballots, one memory round trip for any b
    // up to 64 and b / 64 overlapping ones past it (a binary search takes log2 b dependent ones). Every
    // lane of the wave calls it.
    __device__ __forceinline__ int sequence_of(int t) const {
        const int lane = threadIdx.x & 63;
        int ended = 0;
        for (int s0 = 0; s0 < b; s0 += 64) {
            const int end = s0 + lane < b ? q_start[s0 + lane + 1] : 0x7fffffff;
            ended += __popcll(__ballot(end <= t));
        }
        return ended;
    }

    // The same with the sequence's rows and length (nothing for b). Of up to 64 sequences a lane each has read all of them along
    // with their ends, which saves a trip to memory.
    __device__ __forceinline__ int sequence_of(int t, int &first, int &n, int &len) const {
        first = n = len = 0;
        if (b > 64) {
            const int s = sequence_of(t);
            if (s >= b) return s;
            rows(s, first, n);
            len = length(s);
            return s;
        }
        const int lane = threadIdx.x & 63;
        int lo = 0, hi = 0x7fffffff, c = 0;
        if (lane < b) {
            lo = q_start[lane];
            hi = q_start[lane + 1];
            c = context[lane];
        }
        const int s = __popcll(__ballot(hi <= t));
        if (s >= b) return s;
        clip(__builtin_amdgcn_readlane(lo, s), __builtin_amdgcn_readlane(hi, s), first, n);
        len = clip(__builtin_amdgcn_readlane(c, s));
        return s;
    }
};

// row_units: elements of a row of f16 pages, bytes of a row of 4-bit ones; page_stride and its multiple are in the same.
#define DTTS_REQUIRE_PAGED_ROWS(name, tokens, b, n_kv, head_dim, page, n_pages, max_pages, page_stride, row_units, multiple)      \
    do {                                                                                                                          \
        DTTS_REQUIRE((tokens) >= 0 && (b) >= 0 && (n_kv) > 0 && (n_pages) > 0 && (max_pages) > 0,                                 \
                     "%s: bad shape (tokens %lld, b %lld, n_kv %lld, n_pages %lld, max_pages %lld)", name, (long long)(tokens),   \
                     (long long)(b), (long long)(n_kv), (long long)(n_pages), (long long)(max_pages));                            \
        DTTS_REQUIRE((head_dim) == 64 || (head_dim) == 128, "%s: head_dim %lld (64 or 128 supported)", name,                      \
                     (long long)(head_dim));                                                                                      \
        DTTS_REQUIRE((page) >= 16 && (page) <= 65536 && ((page) & ((page) - 1)) == 0,                                             \
                     "%s: page of %lld positions (a power of two from 16 to 65536)", name, (long long)(page));                    \
        DTTS_REQUIRE((tokens) < (int64_t(1) << 24) && (b) <= kMaxSeqs && (n_kv) <= 4096 && (n_pages) < (int64_t(1) << 31) &&      \
                         (max_pages) <= (int64_t(1) << 30) / (page),                                                              \
                     "%s: too many rows, sequences, heads or positions", name);                                                   \
        DTTS_REQUIRE((page_stride) >= (n_kv) * (page) * (row_units) && (page_stride) % (multiple) == 0 &&                         \
                         (page_stride) < (int64_t(1) << 32),                                                                      \
                     "%s: page_stride %lld (a multiple of %d under 2^32, at least a page)", name, (long long)(page_stride),       \
                     static_cast<int>(multiple));                                                                                 \
    } while (0)

#define DTTS_REQUIRE_PAGED(name, tokens, b, n_kv, head_dim, page, n_pages, max_pages, page_stride)                               \
    DTTS_REQUIRE_PAGED_ROWS(name, tokens, b, n_kv, head_dim, page, n_pages, max_pages, page_stride, head_dim, 8)

#define DTTS_REQUIRE_PAGE(name, page, max_pages)                                                                                 \
    DTTS_REQUIRE((page) >= 16 && (page) <= 65536 && ((page) & ((page) - 1)) == 0 && (max_pages) <= (int64_t(1) << 30) / (page),  \
                 "%s: pages of %lld positions, %lld a sequence (a power of two from 16 to 65536, 2^30 positions at most)", name, \
                 (long long)(page), (long long)(max_pages))

inline int log2_of(int64_t page) {
    int s = 0;
    while ((int64_t(1) << s) < page) ++s;
    return s;
}

}  // namespace
}  // namespace dtts
