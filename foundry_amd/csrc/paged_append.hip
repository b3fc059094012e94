// Appending to a paged cache with the rotation on the way, and the norm before it
// (fh_paged_rope_kv, fh_paged_norm_rope_kv).
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

// 8 dims of each half of a head: a' = RNE(a cos - b sin), b' = RNE(b cos + a sin).
__device__ __forceinline__ void rotate_pair_f32(const float (&a)[8], const float (&b)[8], uint4 &a4, uint4 &b4,
                                                const uint4 ca4, const uint4 cb4, const uint4 sa4, const uint4 sb4) {
    float ca[8], cb[8], sa[8], sb[8];
    unpack8(ca4, ca);
    unpack8(cb4, cb);
    unpack8(sa4, sa);
    unpack8(sb4, sb);
    uint32_t x[4], y[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        x[e / 2] = f32x2_to_bf16x2_rne(fmaf(a[e], ca[e], -b[e] * sa[e]), fmaf(a[e + 1], ca[e + 1], -b[e + 1] * sa[e + 1]));
        y[e / 2] = f32x2_to_bf16x2_rne(fmaf(b[e], cb[e], a[e] * sb[e]), fmaf(b[e + 1], cb[e + 1], a[e + 1] * sb[e + 1]));
    }
    a4 = make_uint4(x[0], x[1], x[2], x[3]);
    b4 = make_uint4(y[0], y[1], y[2], y[3]);
}

struct NormArgs {
    const uint16_t *q_norm, *k_norm;  // null: no norm
    float eps;
    const uint32_t *slots;  // null: the positions
    uint32_t lane_bits;     // a head takes 2^lane_bits lanes, at least head_dim / 16
};

// The same with each head's norm before the rotation, and places apart from the
// positions. A head's threads are lanes of one wavefront, which add their squares
// among themselves; for a head_dim that is no power of two some of them idle. Bound by
// memory: 8192 tokens of 32 + 2 x 8 heads of 128 take 38 us (5.3 TB/s), 512 nodes 5.5 us, the launch.
template <bool STREAM>
__global__ __launch_bounds__(256) void paged_norm_rope_kv_kernel(
    const uint16_t *__restrict__ qkv, uint32_t n_heads, uint32_t n_kv, uint32_t head_dim, const NormArgs norm,
    const uint16_t *__restrict__ cos_tab, const uint16_t *__restrict__ sin_tab, uint32_t table_len,
    const uint32_t *__restrict__ sequences, const uint32_t *__restrict__ positions,
    const uint32_t *__restrict__ page_table, uint32_t n_seqs, uint32_t max_pages, uint16_t *__restrict__ k_pages,
    uint16_t *__restrict__ v_pages, uint32_t n_pages, uint32_t page_size, uint16_t *__restrict__ q_out) {
    const uint32_t t = blockIdx.x;
    const uint32_t pos = positions[t], seq = sequences ? sequences[t] : t, place = norm.slots ? norm.slots[t] : pos;
    // device data the host cannot check: such a token writes nothing
    if (place >= max_pages * page_size || pos >= table_len || seq >= n_seqs) return;
    const uint32_t page = page_table[static_cast<uint64_t>(seq) * max_pages + place / page_size];
    if (page >= n_pages) return;
    const uint32_t slot = place % page_size, heads = n_heads + 2 * n_kv, half = head_dim / 2, pairs = head_dim / 16;
    const uint16_t *row = qkv + static_cast<uint64_t>(t) * heads * head_dim;
    const uint16_t *c = cos_tab + static_cast<uint64_t>(pos) * head_dim;
    const uint16_t *s = sin_tab + static_cast<uint64_t>(pos) * head_dim;
    const uint64_t region = static_cast<uint64_t>(page_size) * head_dim;
    const uint64_t base = static_cast<uint64_t>(page) * n_kv * region;
    auto get = [](const uint16_t *p) { return *reinterpret_cast<const uint4 *>(p); };
    for (uint32_t i = threadIdx.x; i < heads << norm.lane_bits; i += blockDim.x) {
        const uint32_t h = i >> norm.lane_bits, p = i & ((1u << norm.lane_bits) - 1);
        const bool mine = p < pairs;
        const uint32_t d = mine ? p * 8 : 0;
        const uint16_t *head = row + h * head_dim + d;
        uint4 x = get(head), y = get(head + half);
        if (h < n_heads + n_kv) {
            float a[8], b[8];
            unpack8(x, a);
            unpack8(y, b);
            const uint16_t *w = h < n_heads ? norm.q_norm : norm.k_norm;
            if (w) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(a[e], a[e], fmaf(b[e], b[e], sum));
                if (!mine) sum = 0.0f;
                for (uint32_t off = 1; off >> norm.lane_bits == 0; off <<= 1) sum += __shfl_xor(sum, off, 64);
                const float inv = 1.0f / sqrtf(sum / static_cast<float>(head_dim) + norm.eps);
                float wa[8], wb[8];
                unpack8(get(w + d), wa);
                unpack8(get(w + half + d), wb);
#pragma unroll
                for (int e = 0; e < 8; ++e) a[e] = a[e] * inv * wa[e], b[e] = b[e] * inv * wb[e];
            }
            rotate_pair_f32(a, b, x, y, get(c + d), get(c + half + d), get(s + d), get(s + half + d));
        }
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
        if (mine) {
            put16<STREAM>(to, x);
            put16<STREAM>(to2, y);
        }
    }
}

}  // namespace fh

using namespace fh;

namespace {

// The checks of both appends (fh_paged_rope_kv has no norm and no slots).
int check_append(fh_device *dev, const char *fn, const uint16_t *qkv, int64_t tokens, int64_t n_heads, int64_t n_kv,
                 int64_t head_dim, const uint16_t *cos_tab, const uint16_t *sin_tab, int64_t table_len,
                 const uint32_t *sequences, const uint32_t *positions, const NormArgs &norm,
                 const uint32_t *page_table, int64_t n_seqs, int64_t max_pages, uint16_t *k_pages, uint16_t *v_pages,
                 int64_t n_pages, int64_t page_size, uint16_t *q_out) {
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
                          static_cast<const void *>(sin_tab), static_cast<const void *>(q_out),
                          static_cast<const void *>(norm.q_norm), static_cast<const void *>(norm.k_norm)})
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0)
            return fail(FH_ERR_INVALID_ARGUMENT, "%s: operands must be 16-byte aligned", fn);
    if (int rc = check_words(fn, {{"sequences", sequences},
                                  {"positions", positions},
                                  {"slots", norm.slots},
                                  {"page_table", page_table}}))
        return rc;
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
    if (norm.slots)
        if (int rc = check_range(dev, norm.slots, t * 4, fn, "slots")) return rc;
    if (norm.q_norm)
        if (int rc = check_range(dev, norm.q_norm, head_dim * 2, fn, "q_norm")) return rc;
    if (norm.k_norm)
        if (int rc = check_range(dev, norm.k_norm, head_dim * 2, fn, "k_norm")) return rc;
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
        if (norm.slots)
            if (int rc = refuse_overlap(fn, what, ptr, size, "slots", norm.slots, t * 4)) return rc;
        for (const uint16_t *w : {norm.q_norm, norm.k_norm})
            if (w)
                if (int rc = refuse_overlap(fn, what, ptr, size, "a norm's weights", w, head_dim * 2)) return rc;
    }
    return FH_OK;
}

// Bytes of qkv, for the choice of stores.
uint64_t append_bytes(int64_t tokens, int64_t n_heads, int64_t n_kv, int64_t head_dim) {
    return static_cast<uint64_t>(tokens) * static_cast<uint64_t>(n_heads + 2 * n_kv) * head_dim * 2;
}

}  // namespace

extern "C" int fh_paged_rope_kv(fh_device *dev, const uint16_t *qkv, int64_t tokens, int64_t n_heads, int64_t n_kv,
                                int64_t head_dim, const uint16_t *cos_tab, const uint16_t *sin_tab, int64_t table_len,
                                const uint32_t *sequences, const uint32_t *positions, const uint32_t *page_table,
                                int64_t n_seqs, int64_t max_pages, uint16_t *k_pages, uint16_t *v_pages,
                                int64_t n_pages, int64_t page_size, uint16_t *q_out) {
    const char *fn = "fh_paged_rope_kv";
    if (int rc = check_append(dev, fn, qkv, tokens, n_heads, n_kv, head_dim, cos_tab, sin_tab, table_len, sequences,
                              positions, NormArgs{}, page_table, n_seqs, max_pages, k_pages, v_pages, n_pages,
                              page_size, q_out))
        return rc;
    if (tokens == 0) return FH_OK;
    if (int rc = set_current(dev, fn)) return rc;
    // what 8 XCDs' L2s do not hold anyway goes past them: 8192 tokens of 32 and 8
    // heads of 128 (100 MB) 40.3 -> 35.1 us (5.8 TB/s); no difference at 61 tokens
    const bool stream = append_bytes(tokens, n_heads, n_kv, head_dim) > kStreamBytes;
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

extern "C" int fh_paged_norm_rope_kv(fh_device *dev, const uint16_t *qkv, int64_t tokens, int64_t n_heads, int64_t n_kv,
                                     int64_t head_dim, const uint16_t *q_norm, const uint16_t *k_norm, float eps,
                                     const uint16_t *cos_tab, const uint16_t *sin_tab, int64_t table_len,
                                     const uint32_t *sequences, const uint32_t *positions, const uint32_t *slots,
                                     const uint32_t *page_table, int64_t n_seqs, int64_t max_pages, uint16_t *k_pages,
                                     uint16_t *v_pages, int64_t n_pages, int64_t page_size, uint16_t *q_out) {
    const char *fn = "fh_paged_norm_rope_kv";
    NormArgs norm{q_norm, k_norm, eps, slots, 0};
    if (int rc = check_append(dev, fn, qkv, tokens, n_heads, n_kv, head_dim, cos_tab, sin_tab, table_len, sequences,
                              positions, norm, page_table, n_seqs, max_pages, k_pages, v_pages, n_pages, page_size,
                              q_out))
        return rc;
    if (!(eps >= 0.0f && eps < INFINITY))
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: eps %g must be finite and not negative", fn, static_cast<double>(eps));
    if (tokens == 0) return FH_OK;
    while ((16 << norm.lane_bits) < head_dim) ++norm.lane_bits;
    if (int rc = set_current(dev, fn)) return rc;
    const bool stream = append_bytes(tokens, n_heads, n_kv, head_dim) > kStreamBytes;
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(stream ? paged_norm_rope_kv_kernel<true> : paged_norm_rope_kv_kernel<false>,
                           dim3(static_cast<uint32_t>(tokens)), dim3(256), 0, dev->stream, qkv,
                           static_cast<uint32_t>(n_heads), static_cast<uint32_t>(n_kv),
                           static_cast<uint32_t>(head_dim), norm, cos_tab, sin_tab, static_cast<uint32_t>(table_len),
                           sequences, positions, page_table, static_cast<uint32_t>(n_seqs),
                           static_cast<uint32_t>(max_pages), k_pages, v_pages, static_cast<uint32_t>(n_pages),
                           static_cast<uint32_t>(page_size), q_out);
    });
}
