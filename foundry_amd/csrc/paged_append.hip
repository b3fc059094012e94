// Appending to a paged cache with the rotation on the way (fh_paged_rope_kv).
#include <tuple>

#include "paged_cache.hpp"

namespace fh {

// 8 dims of each half of a head, rotated: a' = RNE(a cos - b sin), b' = RNE(b
// cos + a sin), each half with its own table rows, in fp32 with one rounding.
__device__ __forceinline__ void rotate_pair(uint4 &a4, uint4 &b4, const uint4 ca4, const uint4 cb4, const uint4 sa4,
                                            const uint4 sb4) {
    float a[8], b[8], ca[8], cb[8], sa[8], sb[8];
    unpack8(a4, a);
    unpack8(b4, b);
    unpack8(ca4, ca);
    unpack8(cb4, cb);
    unpack8(sa4, sa);
    unpack8(sb4, sb);
    uint32_t x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = f32x2_to_bf16x2_rne(fmaf(a[2 * e], ca[2 * e], -b[2 * e] * sa[2 * e]),
                                   fmaf(a[2 * e + 1], ca[2 * e + 1], -b[2 * e + 1] * sa[2 * e + 1]));
        y[e] = f32x2_to_bf16x2_rne(fmaf(b[2 * e], cb[2 * e], a[2 * e] * sb[2 * e]),
                                   fmaf(b[2 * e + 1], cb[2 * e + 1], a[2 * e + 1] * sb[2 * e + 1]));
    }
    a4 = make_uint4(x[0], x[1], x[2], x[3]);
    b4 = make_uint4(y[0], y[1], y[2], y[3]);
}

constexpr uint64_t kStreamBytes = 32ull << 20;

// STREAM: past the caches, for more than they hold.
template <bool STREAM>
__device__ __forceinline__ void put16(uint16_t *p, uint4 v) {
    if constexpr (STREAM)
        __builtin_nontemporal_store(__builtin_bit_cast(stream_u32x4_t, v), reinterpret_cast<stream_u32x4_t *>(p));
    else
        *reinterpret_cast<uint4 *>(p) = v;
}

// Bound by memory: every value is read and written once. One block per token;
// a thread takes 8 dims and the 8 that the rotation pairs them with, so that
// each is loaded once.
template <bool STREAM>
__global__ __launch_bounds__(256) void paged_rope_kv_kernel(
    const uint16_t *__restrict__ qkv, uint32_t n_heads, uint32_t n_kv, uint32_t head_dim,
    const uint16_t *__restrict__ cos_tab, const uint16_t *__restrict__ sin_tab, uint32_t table_len,
    const uint32_t *__restrict__ sequences, const uint32_t *__restrict__ positions,
    const uint32_t *__restrict__ page_table, uint32_t n_seqs, uint32_t max_pages, uint16_t *__restrict__ k_pages,
    uint16_t *__restrict__ v_pages, uint32_t n_pages, uint32_t page_size, uint16_t *__restrict__ q_out) {
    const uint32_t t = blockIdx.x;
    const uint32_t pos = positions[t], seq = sequences ? sequences[t] : t;
    // device data the host cannot check: such a token writes nothing
    if (pos >= max_pages * page_size || pos >= table_len || seq >= n_seqs) return;
    const uint32_t page = page_table[static_cast<uint64_t>(seq) * max_pages + pos / page_size];
    if (page >= n_pages) return;
    const uint32_t slot = pos % page_size, heads = n_heads + 2 * n_kv, half = head_dim / 2, pairs = head_dim / 16;
    const uint16_t *row = qkv + static_cast<uint64_t>(t) * heads * head_dim;
    const uint16_t *c = cos_tab + static_cast<uint64_t>(pos) * head_dim;
    const uint16_t *s = sin_tab + static_cast<uint64_t>(pos) * head_dim;
    const uint64_t region = static_cast<uint64_t>(page_size) * head_dim;
    const uint64_t base = static_cast<uint64_t>(page) * n_kv * region;
    auto get = [](const uint16_t *p) { return *reinterpret_cast<const uint4 *>(p); };
    for (uint32_t i = threadIdx.x; i < heads * pairs; i += blockDim.x) {
        const uint32_t h = i / pairs, d = i % pairs * 8;
        const uint16_t *head = row + h * head_dim + d;
        uint4 x = get(head), y = get(head + half);
        if (h < n_heads + n_kv) rotate_pair(x, y, get(c + d), get(c + half + d), get(s + d), get(s + half + d));
        uint16_t *to, *to2;
        if (h < n_heads) {
            to = q_out + (static_cast<uint64_t>(t) * n_heads + h) * head_dim + d;
            to2 = to + half;
        } else if (h < n_heads + n_kv) {
            uint16_t *keys = k_pages + base + (h - n_heads) * region;
            to = keys + k_offset(slot, d, page_size, head_dim);
            to2 = keys + k_offset(slot, half + d, page_size, head_dim);
        } else {
            to = v_pages + base + (h - n_heads - n_kv) * region + static_cast<uint64_t>(slot) * head_dim + d;
            to2 = to + half;
        }
        put16<STREAM>(to, x);
        put16<STREAM>(to2, y);
    }
}

}  // namespace fh

using namespace fh;

extern "C" int fh_paged_rope_kv(fh_device *dev, const uint16_t *qkv, int64_t tokens, int64_t n_heads, int64_t n_kv,
                                int64_t head_dim, const uint16_t *cos_tab, const uint16_t *sin_tab, int64_t table_len,
                                const uint32_t *sequences, const uint32_t *positions, const uint32_t *page_table,
                                int64_t n_seqs, int64_t max_pages, uint16_t *k_pages, uint16_t *v_pages,
                                int64_t n_pages, int64_t page_size, uint16_t *q_out) {
    const char *fn = "fh_paged_rope_kv";
    if (int rc = check_usable(dev, fn)) return rc;
    if (int rc = fh_check_dims(fn, {tokens, n_heads, n_kv, head_dim, table_len, n_seqs, max_pages, n_pages, page_size}))
        return rc;
    if (tokens == 0) return FH_OK;
    if (int rc = check_pages(fn, n_pages, page_size, max_pages)) return rc;
    if (head_dim < 32 || head_dim > 256 || head_dim % 32 != 0)
        return fail(FH_ERR_UNSUPPORTED, "%s: head_dim %lld must be a multiple of 32, at most 256", fn,
                    (long long)head_dim);
    if (n_heads < 1 || n_kv < 1 || (n_heads + 2 * n_kv) * head_dim > 0x7FFFFFFFll)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: %lld heads and %lld KV heads", fn, (long long)n_heads,
                    (long long)n_kv);
    if (n_seqs < 1 || table_len < 1)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: n_seqs and table_len must be at least 1", fn);
    // a launch has fewer than 2^32 threads
    if (tokens > 0xFFFFFF) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld tokens exceed 2^24 - 1", fn, (long long)tokens);
    if (sequences == nullptr && tokens > n_seqs)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: %lld tokens of %lld sequences need their sequences named", fn,
                    (long long)tokens, (long long)n_seqs);
    for (const void *p : {static_cast<const void *>(qkv), static_cast<const void *>(cos_tab),
                          static_cast<const void *>(sin_tab), static_cast<const void *>(q_out)})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0)
            return fail(FH_ERR_INVALID_ARGUMENT, "%s: operands must be 16-byte aligned", fn);
    const uint64_t width = static_cast<uint64_t>(n_heads + 2 * n_kv) * head_dim, t = static_cast<uint64_t>(tokens);
    const uint64_t table = static_cast<uint64_t>(table_len) * head_dim * 2;
    uint64_t pool;
    if (int rc = check_pools(dev, fn, k_pages, v_pages, n_pages, n_kv, page_size, head_dim, page_table, n_seqs,
                             max_pages, &pool))
        return rc;
    if (int rc = check_range(dev, qkv, t * width * 2, fn, "qkv")) return rc;
    if (int rc = check_range(dev, cos_tab, table, fn, "cos_tab")) return rc;
    if (int rc = check_range(dev, sin_tab, table, fn, "sin_tab")) return rc;
    if (sequences)
        if (int rc = check_range(dev, sequences, t * 4, fn, "sequences")) return rc;
    if (int rc = check_range(dev, positions, t * 4, fn, "positions")) return rc;
    if (int rc = check_range(dev, q_out, t * n_heads * head_dim * 2, fn, "q_out")) return rc;
    const uint64_t q_bytes = t * n_heads * head_dim * 2;
    if (int rc = refuse_overlap(fn, "v_pages", v_pages, pool, "k_pages", k_pages, pool)) return rc;
    if (int rc = refuse_overlap(fn, "q_out", q_out, q_bytes, "k_pages", k_pages, pool)) return rc;
    if (int rc = refuse_overlap(fn, "q_out", q_out, q_bytes, "v_pages", v_pages, pool)) return rc;
    const uint64_t entries = static_cast<uint64_t>(n_seqs) * max_pages * 4;
    for (const auto &[what, ptr, size] : {std::tuple{"q_out", static_cast<const void *>(q_out), q_bytes},
                                          std::tuple{"k_pages", static_cast<const void *>(k_pages), pool},
                                          std::tuple{"v_pages", static_cast<const void *>(v_pages), pool}}) {
        if (int rc = refuse_overlap(fn, what, ptr, size, "qkv", qkv, t * width * 2)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "cos_tab", cos_tab, table)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "sin_tab", sin_tab, table)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "positions", positions, t * 4)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "page_table", page_table, entries)) return rc;
        if (sequences)
            if (int rc = refuse_overlap(fn, what, ptr, size, "sequences", sequences, t * 4)) return rc;
    }
    if (int rc = set_current(dev, fn)) return rc;
    // what 8 XCDs' L2s do not hold anyway goes past them: 8192 tokens of 32 and 8
    // heads of 128 (100 MB) 40.3 -> 35.1 us (5.8 TB/s); no difference at 61 tokens
    const bool stream = t * width * 2 > kStreamBytes;
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(stream ? paged_rope_kv_kernel<true> : paged_rope_kv_kernel<false>,
                           dim3(static_cast<uint32_t>(tokens)), dim3(256), 0, dev->stream, qkv,
                           static_cast<uint32_t>(n_heads), static_cast<uint32_t>(n_kv),
                           static_cast<uint32_t>(head_dim), cos_tab, sin_tab, static_cast<uint32_t>(table_len),
                           sequences, positions, page_table, static_cast<uint32_t>(n_seqs),
                           static_cast<uint32_t>(max_pages), k_pages, v_pages, static_cast<uint32_t>(n_pages),
                           static_cast<uint32_t>(page_size), q_out);
    });
}
