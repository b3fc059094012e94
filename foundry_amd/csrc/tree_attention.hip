// Attention of a tree of drafted tokens over a paged cache
// (fh_paged_tree_attention).
#include <algorithm>
#include <tuple>

#include "paged_cache.hpp"

namespace fh {

constexpr uint32_t kMaxTree = 1024;

struct TreeArgs {
    const uint16_t *q, *k_pages, *v_pages;
    const uint32_t *page_table, *lengths, *counts, *masks;
    uint32_t batch, width, n_heads, n_kv, n_pages, page_size, max_pages;
    float scale;
    uint16_t *out;
};

// The nodes of sequence b, 0 where they do not fit its table.
__device__ __forceinline__ uint32_t nodes_of(const TreeArgs &a, uint32_t b) {
    const uint32_t count = a.counts ? min(a.counts[b], a.width) : a.width;
    const uint32_t capacity = a.max_pages * a.page_size, len = a.lengths[b];
    return len <= capacity && count <= capacity - len ? count : 0;
}

// One pass over the keys with the running maximum m, sum l and weighted values o:
//   m' = max(m, s), l' = l e^(m - m') + e^(s - m'), o' = o e^(m - m') + e^(s - m') v.
// One wavefront per row (head, node, sequence): a lane scores one of 64 keys, then
// adds up HD / 64 of the values' dims.
template <int HD>
__global__ __launch_bounds__(64) void tree_row_kernel(const TreeArgs a) {
    constexpr int DL = HD / 64;
    __shared__ float qs[HD], ps[64];
    __shared__ uint64_t at[64];
    const uint32_t h = blockIdx.x, node = blockIdx.y, b = blockIdx.z, lane = threadIdx.x;
    const uint64_t row = ((static_cast<uint64_t>(b) * a.width + node) * a.n_heads + h) * HD;
    const uint32_t kv = h / (a.n_heads / a.n_kv), count = nodes_of(a, b);
    float o[DL] = {}, m = -INFINITY, l = 0.0f;
    bool any = false;
    if (node < count) {
        for (int d = lane; d < HD; d += 64) qs[d] = bf(a.q[row + d]);
        __syncthreads();
        const uint32_t len = a.lengths[b], keys = len + count, words = (a.width + 31) / 32;
        for (uint32_t j0 = 0; j0 < keys; j0 += 64) {
            const uint32_t j = j0 + lane;
            bool seen = j < keys;
            if (seen && j >= len) {
                const uint32_t i = j - len;
                seen = a.masks ? a.masks[(static_cast<uint64_t>(b) * a.width + node) * words + i / 32] >> (i % 32) & 1u
                               : i <= node;
            }
            float s = -INFINITY;
            if (seen) {
                const uint32_t page = a.page_table[static_cast<uint64_t>(b) * a.max_pages + j / a.page_size];
                seen = page < a.n_pages;
                if (seen) {
                    const uint64_t region = (static_cast<uint64_t>(page) * a.n_kv + kv) * a.page_size * HD;
                    const uint16_t *k = a.k_pages + region;
                    at[lane] = region + static_cast<uint64_t>(j % a.page_size) * HD;
                    float dot = 0.0f;
                    for (uint32_t d = 0; d < HD; d += 8) {
                        float x[8];
                        unpack8(*reinterpret_cast<const uint4 *>(k + k_offset(j % a.page_size, d, a.page_size, HD)), x);
#pragma unroll
                        for (int e = 0; e < 8; ++e) dot = fmaf(qs[d + e], x[e], dot);
                    }
                    s = dot * a.scale;
                }
            }
            const float next = fmaxf(m, wave_max(s)), ref = next == -INFINITY ? 0.0f : next;
            const float keep = __expf(m - ref), p = seen ? __expf(s - ref) : 0.0f;
            m = next;
            l = l * keep + wave_sum(p);
            ps[lane] = p;
            __syncthreads();
#pragma unroll
            for (int d = 0; d < DL; ++d) o[d] *= keep;
            uint64_t left = __ballot(seen);
            any = any || left != 0;
            while (left) {
                const int i = __builtin_ctzll(left);
                left &= left - 1;
#pragma unroll
                for (int d = 0; d < DL; ++d) o[d] = fmaf(ps[i], bf(a.v_pages[at[i] + lane * DL + d]), o[d]);
            }
            __syncthreads();
        }
    }
    for (int d = 0; d < DL; ++d) a.out[row + lane * DL + d] = any ? rne(o[d] / l) : 0;
}

}  // namespace fh

using namespace fh;

namespace {

int check_shape(const char *fn, int64_t batch, int64_t width, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                int64_t page_size, int64_t max_pages) {
    if (int rc = fh_check_dims(fn, {batch, width, n_heads, n_kv, head_dim, page_size, max_pages})) return rc;
    if (int rc = check_pages(fn, 1, page_size, max_pages)) return rc;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(FH_ERR_UNSUPPORTED, "%s: head_dim %lld must be 64, 128 or 256", fn, (long long)head_dim);
    if (n_kv < 1 || n_heads < 1 || n_heads % n_kv != 0 || n_heads > 65535)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: %lld heads do not share %lld KV heads", fn, (long long)n_heads,
                    (long long)n_kv);
    if (width < 1 || width > kMaxTree)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: width %lld must be 1 to %u", fn, (long long)width, kMaxTree);
    if (batch > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: batch %lld exceeds 65535", fn, (long long)batch);
    if (batch * width * n_heads > 0x3FFFFFF)
        return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld sequences of %lld nodes and %lld heads", fn, (long long)batch,
                    (long long)width, (long long)n_heads);
    return FH_OK;
}

}  // namespace

extern "C" int fh_paged_tree_attention_workspace(int64_t batch, int64_t width, int64_t n_heads, int64_t n_kv,
                                                 int64_t head_dim, int64_t page_size, int64_t max_pages,
                                                 uint64_t *bytes) {
    const char *fn = "fh_paged_tree_attention_workspace";
    if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: bytes is null", fn);
    if (int rc = check_shape(fn, batch, width, n_heads, n_kv, head_dim, page_size, max_pages)) return rc;
    *bytes = 16;
    return FH_OK;
}

extern "C" int fh_paged_tree_attention(fh_device *dev, const uint16_t *q, int64_t batch, int64_t width, int64_t n_heads,
                                       int64_t n_kv, int64_t head_dim, const uint16_t *k_pages,
                                       const uint16_t *v_pages, int64_t n_pages, int64_t page_size,
                                       const uint32_t *page_table, int64_t max_pages, const uint32_t *lengths,
                                       const uint32_t *counts, const uint32_t *masks, float scale, void *workspace,
                                       uint64_t workspace_bytes, uint16_t *out) {
    const char *fn = "fh_paged_tree_attention";
    if (int rc = check_usable(dev, fn)) return rc;
    if (int rc = check_shape(fn, batch, width, n_heads, n_kv, head_dim, page_size, max_pages)) return rc;
    if (int rc = fh_check_dims(fn, {n_pages})) return rc;
    if (int rc = check_pages(fn, n_pages, page_size, max_pages)) return rc;
    if (!(scale > 0.0f && scale < INFINITY))
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: scale %g must be finite and above 0", fn, static_cast<double>(scale));
    if (batch == 0) return FH_OK;
    uint64_t need = 0;
    if (int rc = fh_paged_tree_attention_workspace(batch, width, n_heads, n_kv, head_dim, page_size, max_pages, &need))
        return rc;
    if (workspace_bytes < need)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: workspace of %llu bytes, %llu needed", fn,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) &
        15u)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: q, out and workspace must be 16-byte aligned", fn);
    const uint64_t nodes = static_cast<uint64_t>(batch) * width, each = static_cast<uint64_t>(batch) * 4;
    const uint64_t rows = nodes * n_heads * head_dim * 2, bits = nodes * ((width + 31) / 32) * 4;
    uint64_t pool;
    if (int rc = check_pools(dev, fn, k_pages, v_pages, n_pages, n_kv, page_size, head_dim, page_table, batch,
                             max_pages, &pool))
        return rc;
    if (int rc = check_range(dev, workspace, need, fn, "workspace")) return rc;
    if (int rc = check_range(dev, q, rows, fn, "q")) return rc;
    if (int rc = check_range(dev, lengths, each, fn, "lengths")) return rc;
    if (counts)
        if (int rc = check_range(dev, counts, each, fn, "counts")) return rc;
    if (masks)
        if (int rc = check_range(dev, masks, bits, fn, "masks")) return rc;
    if (int rc = check_range(dev, out, rows, fn, "out")) return rc;
    for (const auto &[what, ptr, size] : {std::tuple{"out", static_cast<const void *>(out), rows},
                                          std::tuple{"workspace", static_cast<const void *>(workspace), need}})
        for (const auto &[with, p, n] :
             {std::tuple{"q", static_cast<const void *>(q), rows},
              std::tuple{"k_pages", static_cast<const void *>(k_pages), pool},
              std::tuple{"v_pages", static_cast<const void *>(v_pages), pool},
              std::tuple{"page_table", static_cast<const void *>(page_table), each * max_pages},
              std::tuple{"lengths", static_cast<const void *>(lengths), each},
              std::tuple{"counts", static_cast<const void *>(counts), each},
              std::tuple{"masks", static_cast<const void *>(masks), bits}})
            if (p)
                if (int rc = refuse_overlap(fn, what, ptr, size, with, p, n)) return rc;
    if (int rc = refuse_overlap(fn, "workspace", workspace, need, "out", out, rows)) return rc;
    if (int rc = set_current(dev, fn)) return rc;
    const TreeArgs a{q,
                     k_pages,
                     v_pages,
                     page_table,
                     lengths,
                     counts,
                     masks,
                     static_cast<uint32_t>(batch),
                     static_cast<uint32_t>(width),
                     static_cast<uint32_t>(n_heads),
                     static_cast<uint32_t>(n_kv),
                     static_cast<uint32_t>(n_pages),
                     static_cast<uint32_t>(page_size),
                     static_cast<uint32_t>(max_pages),
                     scale,
                     out};
    const dim3 grid(static_cast<uint32_t>(n_heads), static_cast<uint32_t>(width), static_cast<uint32_t>(batch));
    return dispatch(dev, fn, [&] {
        if (head_dim == 64)
            hipLaunchKernelGGL(tree_row_kernel<64>, grid, dim3(64), 0, dev->stream, a);
        else if (head_dim == 128)
            hipLaunchKernelGGL(tree_row_kernel<128>, grid, dim3(64), 0, dev->stream, a);
        else
            hipLaunchKernelGGL(tree_row_kernel<256>, grid, dim3(64), 0, dev->stream, a);
    });
}
