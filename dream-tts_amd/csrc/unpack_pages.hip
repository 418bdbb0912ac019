// The f16 pages that 4-bit pages stand for: HBM-bound, each word read once, its eight values written with one store.
#include "paged.hpp"
#include "q4.hpp"

namespace dtts {
namespace {

struct UnpackArgs {
    const uint8_t *k, *v;
    const int32_t *ids;  // or NULL: all pages in order
    half_t *k_out, *v_out;
    int64_t page_stride;
    int n_pages, n_kv, page_shift;
};

// blockIdx.y: keys or values; blockIdx.x walks (page, kv head, 256 pieces of 16 bytes). Of keys that is 32 dimensions of a
// row, of values eight dimensions of four rows.
template <int D>
__global__ __launch_bounds__(256) void unpack_kernel(UnpackArgs a, FastDiv pieces, int64_t most) {
    const bool values = blockIdx.y != 0;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i >= most) return;
    const int page = 1 << a.page_shift;
    const int64_t head = pieces.div(static_cast<uint32_t>(i));
    const int piece = static_cast<int>(i - head * pieces.d), at = static_cast<int>(head / a.n_kv), kv = static_cast<int>(head - static_cast<int64_t>(at) * a.n_kv);
    const int id = a.ids ? a.ids[at] : at;
    if (id < 0 || id >= a.n_pages) return;
    const uint8_t *x = (values ? a.v : a.k) + id * a.page_stride + static_cast<int64_t>(kv) * page * Q4Row<D>::kBytes;
    half_t *y = (values ? a.v_out : a.k_out) + (head << a.page_shift) * D;
    const Q4Bits bits;
    const u32x4 words = *reinterpret_cast<const u32x4 *>(x + piece * 16);
    if (values) {
        constexpr int W = Q4Row<D>::kWords;
        const int row = piece / W * 4, w = piece % W;
        const u32x4 pairs = *reinterpret_cast<const u32x4 *>(x + Q4Row<D>::pair(page, row, w / 4));
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<half8_t *>(y + (row + k) * D + 8 * w) = q4_values(words[k], pairs[k], bits);
    } else {
        constexpr int G = D / 32;
        const int row = piece / G, group = piece % G;
        const uint32_t pair = *reinterpret_cast<const uint32_t *>(x + Q4Row<D>::pair(page, row, group));
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<half8_t *>(y + row * D + 32 * group + 8 * k) = q4_values(words[k], pair, bits);
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
                       reinterpret_cast<half_t *>(v_out), page_stride, static_cast<int>(n_pages), static_cast<int>(n_kv), log2_of(page)};
    const dim3 grid(static_cast<unsigned>((most + 255) / 256), 2);
    if (head_dim == 128)
        unpack_kernel<128><<<grid, 256, 0, stream>>>(a, FastDiv(static_cast<uint32_t>(pieces)), most);
    else
        unpack_kernel<64><<<grid, 256, 0, stream>>>(a, FastDiv(static_cast<uint32_t>(pieces)), most);
    DTTS_LAUNCH_CHECK(name);
    return DTTS_OK;
}
