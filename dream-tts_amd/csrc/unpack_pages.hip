// The f16 pages that 4-bit pages stand for: HBM-bound, each word read once, its eight values written with one store. 650 pages of
// 16 rows of 8 kv heads of 128 (13 MB read, 43 written): 9.6 us, 5.8 TB/s.
#include "paged.hpp"
#include "q4.hpp"

namespace dtts {
namespace {

struct UnpackArgs {
    const uint8_t *k, *v;
    const int32_t *ids;  // or NULL: all pages in order
    half_t *k_out, *v_out;
    int64_t page_stride;
    int n_pages, page_shift;
};

// blockIdx.y: keys or values; blockIdx.x walks (page, kv head, 16-byte piece of its codes). A wave's stores are runs of whole
// rows either way: of values a thread takes eight dimensions of four rows, one load; of keys words 64 apart, so that each
// store of the wave is 64 neighbouring words' values (with 16 bytes a thread, stores of 64 bytes apart: 13.9 us for 57 MB).
// Values are stored past the caches, keys are not: both kept / keys past / values past / both 13.0 / 12.9 / 12.6 / 13.2 us (with the append of
// 48 tokens before, 43 MB) and 14.2 / 13.9 / 13.85 / 13.65 (4436 tokens, 16 MB).
template <int D>
__global__ __launch_bounds__(256) void unpack_kernel(UnpackArgs a, FastDiv pieces, FastDiv heads, uint32_t most) {
    constexpr int W = Q4Row<D>::kWords;
    const int page = 1 << a.page_shift;
    const Q4Bits bits;
    auto at = [&](uint32_t head, const uint8_t *pages, const uint8_t *&x) {  // whether there is a page
        const uint32_t n = heads.div(head), kv = head - n * heads.d;
        const int id = a.ids ? a.ids[n] : static_cast<int>(n);
        x = pages + id * a.page_stride + static_cast<int64_t>(kv) * page * Q4Row<D>::kBytes;
        return id >= 0 && id < a.n_pages;
    };
    const uint8_t *x;
    if (blockIdx.y) {
        const uint32_t i = blockIdx.x * 256 + threadIdx.x;
        if (i >= most) return;
        const uint32_t head = pieces.div(i), piece = i - head * pieces.d;
        if (!at(head, a.v, x)) return;
        const int row = piece / W * 4, w = piece % W;
        const u32x4 words = *reinterpret_cast<const u32x4 *>(x + piece * 16);
        const u32x4 pairs = *reinterpret_cast<const u32x4 *>(x + Q4Row<D>::pair(page, row, w / 4));
        half_t *y = a.v_out + (static_cast<int64_t>(head) << a.page_shift) * D + row * D + 8 * w;
#pragma unroll
        for (int k = 0; k < 4; ++k) __builtin_nontemporal_store(q4_values(words[k], pairs[k], bits), reinterpret_cast<half8_t *>(y + k * D));
    } else {
        const uint32_t first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 64;  // the wave's pieces; its words are four times as many
        uint32_t word[4], pair[4];
        bool there[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t i = first + 16 * k + (threadIdx.x & 63) / 4;  // the word's piece
            const uint32_t head = pieces.div(i), w = (i - head * pieces.d) * 4 + (threadIdx.x & 3);
            there[k] = i < most && at(head, a.k, x);
            if (!there[k]) continue;
            word[k] = *reinterpret_cast<const uint32_t *>(x + w * 4);
            pair[k] = *reinterpret_cast<const uint32_t *>(x + Q4Row<D>::pair(page, w / W, w % W / 4));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t i = first + 16 * k + (threadIdx.x & 63) / 4;
            if (there[k])
                *reinterpret_cast<half8_t *>(a.k_out + (static_cast<int64_t>(i) * 4 + (threadIdx.x & 3)) * 8) = q4_values(word[k], pair[k], bits);
        }
    }
}

}  // namespace
}  // namespace dtts

extern "C" int dtts_unpack_pages_q4(const void *kpages, const void *vpages, const int32_t *ids, dtts_f16 *k_out, dtts_f16 *v_out, int64_t n,
                                    int64_t n_kv, int64_t head_dim, int64_t page, int64_t n_pages, int64_t page_stride,
                                    hipStream_t stream) {
    using namespace dtts;
    const char *name = "dtts_unpack_pages_q4";
    DTTS_REQUIRE_PAGED_ROWS(name, 0, 0, n_kv, head_dim, page, n_pages, 1, page_stride, 5 * head_dim / 8, 16);
    DTTS_REQUIRE(n >= 0 && n < (int64_t(1) << 31) && (ids || n <= n_pages), "%s: %lld of %lld pages", name, (long long)n, (long long)n_pages);
    if (n == 0) return DTTS_OK;
    DTTS_REQUIRE(kpages && vpages && k_out && v_out, "%s: null pointer", name);
    DTTS_REQUIRE(aligned(kpages, 16) && aligned(vpages, 16) && aligned(k_out, 16) && aligned(v_out, 16) && aligned(ids, 4),
                 "%s: misaligned operand", name);
    const int64_t bytes = n_kv * page * 5 * head_dim / 8, out = n * n_kv * page * head_dim * static_cast<int64_t>(sizeof(half_t));
    const ByteRows k{kpages, n_pages, page_stride, bytes}, v{vpages, n_pages, page_stride, bytes}, ko{k_out, 1, 0, out}, vo{v_out, 1, 0, out};
    DTTS_REQUIRE(!share_bytes(k, ko) && !share_bytes(k, vo) && !share_bytes(v, ko) && !share_bytes(v, vo) && !share_bytes(ko, vo),
                 "%s: the values share memory with one another or with the pages", name);
    const int64_t pieces = page * head_dim / 32, most = n * n_kv * pieces;
    DTTS_REQUIRE((most + 255) / 256 < (int64_t(1) << 24), "%s: too many pages", name);  // a launch has under 2^32 threads
    const UnpackArgs a{static_cast<const uint8_t *>(kpages), static_cast<const uint8_t *>(vpages), ids, reinterpret_cast<half_t *>(k_out),
                       reinterpret_cast<half_t *>(v_out), page_stride, static_cast<int>(n_pages), log2_of(page)};
    const dim3 grid(static_cast<unsigned>((most + 255) / 256), 2);
    if (head_dim == 128)
        unpack_kernel<128><<<grid, 256, 0, stream>>>(a, FastDiv(static_cast<uint32_t>(pieces)), FastDiv(static_cast<uint32_t>(n_kv)), static_cast<uint32_t>(most));
    else
        unpack_kernel<64><<<grid, 256, 0, stream>>>(a, FastDiv(static_cast<uint32_t>(pieces)), FastDiv(static_cast<uint32_t>(n_kv)), static_cast<uint32_t>(most));
    DTTS_LAUNCH_CHECK(name);
    return DTTS_OK;
}
