// Attention of one new token per sequence over a paged cache
// (fh_paged_attention).
#include <tuple>

#include "paged_cache.hpp"

namespace fh {

constexpr uint32_t kPagedThreads = 256;

// One block per (query head, sequence). A pass takes 256 keys: each thread
// scores one key, then (the running maximum and sum updated) each thread of a
// dim adds the pass's 256 weighted values.
__global__ __launch_bounds__(kPagedThreads) void paged_attention_kernel(
    const uint16_t *__restrict__ q, uint32_t n_heads, uint32_t n_kv, uint32_t head_dim,
    const uint16_t *__restrict__ k_pages, const uint16_t *__restrict__ v_pages, uint32_t n_pages, uint32_t page_size,
    const uint32_t *__restrict__ page_table, uint32_t max_pages, const uint32_t *__restrict__ positions, float scale,
    uint16_t *__restrict__ out) {
    __shared__ float qs[256], ps[kPagedThreads], red[4];
    __shared__ uint64_t where[kPagedThreads];
    const uint32_t h = blockIdx.x, b = blockIdx.y, kv = h / (n_heads / n_kv), t = threadIdx.x;
    const uint32_t pos = positions[b], keys = pos < max_pages * page_size ? pos + 1 : 0;
    const uint64_t row = (static_cast<uint64_t>(b) * n_heads + h) * head_dim;
    if (t < head_dim) qs[t] = bf(q[row + t]);
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    bool any = false;
    for (uint32_t k0 = 0; k0 < keys; k0 += kPagedThreads) {
        const uint32_t j = k0 + t;
        const uint32_t page = j < keys ? page_table[static_cast<uint64_t>(b) * max_pages + j / page_size] : n_pages;
        const bool live = page < n_pages;
        const uint64_t at = (static_cast<uint64_t>(live ? page : 0) * n_kv + kv) * page_size * head_dim;
        __syncthreads();
        float s = -INFINITY;
        if (live) {
            s = 0.0f;
            for (uint32_t d = 0; d < head_dim; ++d)
                s = fmaf(qs[d], bf(k_pages[at + k_offset(j % page_size, d, page_size, head_dim)]), s);
            s *= scale;
        }
        float top = s;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        if (t % 64 == 0) red[t / 64] = top;
        where[t] = live ? at + static_cast<uint64_t>(j % page_size) * head_dim : ~0ull;
        __syncthreads();
        const float next = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        const float ref = next == -INFINITY ? 0.0f : next;
        const float keep = expf(m - ref);
        ps[t] = live ? expf(s - ref) : 0.0f;
        m = next;
        __syncthreads();
        acc *= keep;
        l *= keep;
        for (uint32_t i = 0; i < kPagedThreads && k0 + i < keys; ++i)
            if (where[i] != ~0ull) {
                any = true;
                l += ps[i];
                if (t < head_dim) acc = fmaf(ps[i], bf(v_pages[where[i] + t]), acc);
            }
    }
    if (t < head_dim) out[row + t] = any ? rne(acc / l) : 0;
}

}  // namespace fh

using namespace fh;

namespace {

int check_shape(const char *fn, int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t page_size,
                int64_t max_pages) {
    if (int rc = fh_check_dims(fn, {batch, n_heads, n_kv, head_dim, page_size, max_pages})) return rc;
    if (int rc = check_pages(fn, 1, page_size, max_pages)) return rc;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(FH_ERR_UNSUPPORTED, "%s: head_dim %lld must be 64, 128 or 256", fn, (long long)head_dim);
    if (n_kv < 1 || n_heads < 1 || n_heads % n_kv != 0 || n_heads > 65535)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: %lld heads do not share %lld KV heads", fn, (long long)n_heads,
                    (long long)n_kv);
    if (batch > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: batch %lld exceeds 65535", fn, (long long)batch);
    return FH_OK;
}

}  // namespace

extern "C" int fh_paged_attention_workspace(int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                                            int64_t page_size, int64_t max_pages, uint64_t *bytes) {
    const char *fn = "fh_paged_attention_workspace";
    if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: bytes is null", fn);
    if (int rc = check_shape(fn, batch, n_heads, n_kv, head_dim, page_size, max_pages)) return rc;
    *bytes = 16;
    return FH_OK;
}

extern "C" int fh_paged_attention(fh_device *dev, const uint16_t *q, int64_t batch, int64_t n_heads, int64_t n_kv,
                                  int64_t head_dim, const uint16_t *k_pages, const uint16_t *v_pages, int64_t n_pages,
                                  int64_t page_size, const uint32_t *page_table, int64_t max_pages,
                                  const uint32_t *positions, float scale, void *workspace, uint64_t workspace_bytes,
                                  uint16_t *out) {
    const char *fn = "fh_paged_attention";
    if (int rc = check_usable(dev, fn)) return rc;
    if (int rc = check_shape(fn, batch, n_heads, n_kv, head_dim, page_size, max_pages)) return rc;
    if (int rc = fh_check_dims(fn, {n_pages})) return rc;
    if (int rc = check_pages(fn, n_pages, page_size, max_pages)) return rc;
    if (batch == 0) return FH_OK;
    uint64_t need = 0;
    if (int rc = fh_paged_attention_workspace(batch, n_heads, n_kv, head_dim, page_size, max_pages, &need)) return rc;
    if (workspace_bytes < need)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: workspace of %llu bytes, %llu needed", fn,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) &
        15u)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: q, out and workspace must be 16-byte aligned", fn);
    const uint64_t rows = static_cast<uint64_t>(batch) * n_heads * head_dim * 2;
    uint64_t pool;
    if (int rc = check_pools(dev, fn, k_pages, v_pages, n_pages, n_kv, page_size, head_dim, page_table, batch,
                             max_pages, &pool))
        return rc;
    if (int rc = check_range(dev, workspace, need, fn, "workspace")) return rc;
    if (int rc = check_range(dev, q, rows, fn, "q")) return rc;
    if (int rc = check_range(dev, positions, static_cast<uint64_t>(batch) * 4, fn, "positions")) return rc;
    if (int rc = check_range(dev, out, rows, fn, "out")) return rc;
    for (const auto &[what, ptr, size] : {std::tuple{"out", static_cast<const void *>(out), rows},
                                          std::tuple{"workspace", static_cast<const void *>(workspace), need}}) {
        if (int rc = refuse_overlap(fn, what, ptr, size, "q", q, rows)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "k_pages", k_pages, pool)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "v_pages", v_pages, pool)) return rc;
    }
    if (int rc = refuse_overlap(fn, "workspace", workspace, need, "out", out, rows)) return rc;
    if (int rc = set_current(dev, fn)) return rc;
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(paged_attention_kernel, dim3(static_cast<uint32_t>(n_heads), static_cast<uint32_t>(batch)),
                           dim3(kPagedThreads), 0, dev->stream, q, static_cast<uint32_t>(n_heads),
                           static_cast<uint32_t>(n_kv), static_cast<uint32_t>(head_dim), k_pages, v_pages,
                           static_cast<uint32_t>(n_pages), static_cast<uint32_t>(page_size), page_table,
                           static_cast<uint32_t>(max_pages), positions, scale, out);
    });
}
