// The pages of a cache of all layers: handed out, shared, freed, and an accepted
// path's tokens moved together (fh_paged_reserve, fh_paged_fork, fh_paged_free,
// fh_paged_compact). Page counts stay on the device, so that none of these waits
// for the host; the lowest free page goes to the first that asks, so that results
// do not depend on the order in which threads run. The tables' kernels are bound by
// dependent loads: 4 to 5 us each for tens of sequences, a few entries of each and pools of hundreds of pages.
// fh_paged_reserve fills a sequence's entries one after another in one thread and looks for free pages from page 0
// on, so that it grows with both: 2048 entries of one sequence (32768 tokens) take 0.57 ms, 8192 2.2 ms, one of
// each of 64 sequences 51 us where the first 90000 of 100000 pages are in use. The copies are bound by memory: 16
// forks of 28 layers' pages take 21.2 us (4.8 TB/s), 24 sequences' paths over 28 layers 8 to 9 us (2.4 to 2.8
// TB/s behind five dependent loads).
#include <algorithm>
#include <vector>

#include "paged_cache.hpp"

namespace fh {

constexpr uint32_t kMaxLayers = 128, kMaxSeqs = 16384, kMaxForks = 1024, kMaxNew = 16384;
constexpr uint32_t kTableThreads = 1024;
constexpr uint32_t kNoPage = 0xFFFFFFFFu;

struct PageArgs {
    uint32_t *table, *lengths, *refs;
    uint32_t n_seqs, max_pages, n_pages, page_size;
};

struct PoolArgs {
    fh_paged_pool pools[kMaxLayers];
    uint32_t n_kv, head_dim;
};

// The block's exclusive prefix sums of v, and their total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *waves, uint32_t &total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t upto = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_up(upto, off, 64);
        if (lane >= static_cast<uint32_t>(off)) upto += o;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
    for (uint32_t w = 0; w < blockDim.x / 64; ++w) {
        if (w < wave) before += waves[w];
        total += waves[w];
    }
    return before + upto - v;
}

// The lowest `want` free pages (or as many as there are) into list; returns their number.
__device__ __forceinline__ uint32_t free_pages(const PageArgs &a, uint32_t want, uint32_t *list, uint32_t *waves) {
    constexpr uint32_t kEach = 4;
    uint32_t got = 0;
    for (uint32_t p0 = 0; p0 < a.n_pages && got < want; p0 += kTableThreads * kEach) {
        const uint32_t p = p0 + threadIdx.x * kEach;
        uint32_t bits = 0;
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e)
            if (p + e < a.n_pages && a.refs[p + e] == 0) bits |= 1u << e;
        uint32_t total, at = got + block_scan(__popc(bits), waves, total);
#pragma unroll
        for (uint32_t e = 0; e < kEach; ++e)
            if (bits >> e & 1u) {
                if (at < want) list[at] = p + e;
                ++at;
            }
        got += total;
    }
    __syncthreads();
    return min(got, want);
}

// One block. A thread takes a run of sequences: their empty entries are counted,
// the counts scanned, and entry i of all gets the i-th free page.
__global__ __launch_bounds__(kTableThreads) void reserve_kernel(const PageArgs a, const uint32_t *extra,
                                                                uint32_t *missing) {
    __shared__ uint32_t list[kMaxNew];
    __shared__ uint32_t waves[kTableThreads / 64];
    const uint32_t each = (a.n_seqs + kTableThreads - 1) / kTableThreads;
    const uint32_t s0 = min(threadIdx.x * each, a.n_seqs), s1 = min(s0 + each, a.n_seqs);
    const uint64_t capacity = static_cast<uint64_t>(a.max_pages) * a.page_size;
    // entries first .. last - 1 of sequence s; what lies past the table in `over`
    auto entries = [&](uint32_t s, uint32_t &first, uint32_t &last) {
        const uint64_t len = a.lengths[s], end = len + extra[s];
        first = static_cast<uint32_t>(min(len, capacity) / a.page_size);
        last = static_cast<uint32_t>((min(end, capacity) + a.page_size - 1) / a.page_size);
        if (extra[s] == 0) last = first;
        const uint64_t pages = (end + a.page_size - 1) / a.page_size;
        const uint64_t from = max(len / a.page_size, static_cast<uint64_t>(a.max_pages));
        return extra[s] && pages > from ? static_cast<uint32_t>(pages - from) : 0u;
    };
    uint32_t need = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        uint32_t first, last;
        entries(s, first, last);
        for (uint32_t e = first; e < last; ++e) need += a.table[static_cast<uint64_t>(s) * a.max_pages + e] >= a.n_pages;
    }
    // (a thread's entries are below 2^31: need does not wrap, but the sum over threads might)
    uint32_t total, at = block_scan(min(need, kMaxNew), waves, total);
    const uint32_t got = free_pages(a, min(total, kMaxNew), list, waves);
    for (uint32_t s = s0; s < s1; ++s) {
        uint32_t first, last;
        uint32_t lost = entries(s, first, last);
        for (uint32_t e = first; e < last; ++e) {
            uint32_t &entry = a.table[static_cast<uint64_t>(s) * a.max_pages + e];
            if (entry < a.n_pages) continue;
            if (at < got) {
                entry = list[at++];
                a.refs[entry] = 1;
            } else {
                ++lost;
            }
        }
        if (missing) missing[s] = lost;
    }
}

__global__ __launch_bounds__(256) void free_kernel(const PageArgs a, const uint32_t *seqs) {
    const uint32_t s = seqs[blockIdx.x];
    if (s >= a.n_seqs) return;
    uint32_t *row = a.table + static_cast<uint64_t>(s) * a.max_pages;
    // the exchange gives an entry to one block where a sequence is named twice
    for (uint32_t e = threadIdx.x; e < a.max_pages; e += blockDim.x) {
        const uint32_t page = atomicExch(&row[e], kNoPage);
        if (page < a.n_pages) atomicSub(&a.refs[page], 1u);
    }
    if (threadIdx.x == 0) a.lengths[s] = 0;
}

struct ForkArgs {
    const uint32_t *from, *to;
    uint32_t n;
    uint32_t *lost;
};

// Whether fork i stands, for the whole block (which calls it together).
__device__ __forceinline__ bool fork_stands(const PageArgs &a, const ForkArgs &f, uint32_t i) {
    const uint32_t s = f.from[i], d = f.to[i];
    bool bad = s >= a.n_seqs || d >= a.n_seqs || a.lengths[min(s, a.n_seqs - 1)] > a.max_pages * a.page_size;
    for (uint32_t j = threadIdx.x; j < f.n; j += blockDim.x) bad = bad || f.from[j] == d || (j < i && f.to[j] == d);
    return !__syncthreads_or(bad);
}

// Block i: the table row of fork i, but for the page that is copied.
__global__ __launch_bounds__(256) void fork_share_kernel(const PageArgs a, const ForkArgs f) {
    const uint32_t i = blockIdx.x;
    if (!fork_stands(a, f, i)) {
        if (threadIdx.x == 0) f.lost[i] = 1;
        return;
    }
    const uint32_t *src = a.table + static_cast<uint64_t>(f.from[i]) * a.max_pages;
    uint32_t *dst = a.table + static_cast<uint64_t>(f.to[i]) * a.max_pages;
    const uint32_t whole = a.lengths[f.from[i]] / a.page_size;
    for (uint32_t e = threadIdx.x; e < a.max_pages; e += blockDim.x) {
        const uint32_t old = dst[e];
        if (old < a.n_pages) atomicSub(&a.refs[old], 1u);
        const uint32_t page = e < whole ? src[e] : kNoPage;
        if (page < a.n_pages) atomicAdd(&a.refs[page], 1u);
        dst[e] = page < a.n_pages ? page : kNoPage;
    }
    if (threadIdx.x == 0) f.lost[i] = 0;
}

// One block: thread i hands fork i the page for its copy, or empties it.
__global__ __launch_bounds__(kTableThreads) void fork_take_kernel(const PageArgs a, const ForkArgs f) {
    __shared__ uint32_t list[kMaxForks];
    __shared__ uint32_t waves[kTableThreads / 64];
    const uint32_t i = threadIdx.x;
    const bool stands = i < f.n && f.lost[i] == 0;
    const uint32_t len = stands ? a.lengths[f.from[i]] : 0, whole = len / a.page_size;
    const bool part = len % a.page_size != 0;
    uint32_t total;
    const uint32_t at = block_scan(part, waves, total);
    const uint32_t got = free_pages(a, total, list, waves);
    if (!stands) return;
    uint32_t *dst = a.table + static_cast<uint64_t>(f.to[i]) * a.max_pages;
    if (!part || at < got) {
        if (part) {
            dst[whole] = list[at];
            a.refs[list[at]] = 1;
        }
        a.lengths[f.to[i]] = len;
        return;
    }
    for (uint32_t e = 0; e < whole; ++e) {
        if (dst[e] < a.n_pages) atomicSub(&a.refs[dst[e]], 1u);
        dst[e] = kNoPage;
    }
    a.lengths[f.to[i]] = 0;
    f.lost[i] = 1;
}

// Block (fork, layer, K or V): the tokens of the last page that is not full.
__global__ __launch_bounds__(256) void fork_copy_kernel(const PageArgs a, const ForkArgs f, const PoolArgs p) {
    const uint32_t i = blockIdx.x;
    if (f.lost[i]) return;
    const uint32_t len = a.lengths[f.from[i]], whole = len / a.page_size, used = len % a.page_size;
    if (used == 0) return;
    const uint32_t from = a.table[static_cast<uint64_t>(f.from[i]) * a.max_pages + whole];
    const uint32_t to = a.table[static_cast<uint64_t>(f.to[i]) * a.max_pages + whole];
    if (from >= a.n_pages || to >= a.n_pages) return;
    const bool keys = blockIdx.z == 0;
    uint16_t *pool = keys ? p.pools[blockIdx.y].k_pages : p.pools[blockIdx.y].v_pages;
    const uint64_t region = static_cast<uint64_t>(a.page_size) * p.head_dim, page = region * p.n_kv;
    const uint32_t pieces = p.head_dim / 8;
    for (uint32_t x = threadIdx.x; x < p.n_kv * used * pieces; x += blockDim.x) {
        const uint32_t d = x % pieces * 8, slot = x / pieces % used, kv = x / pieces / used;
        const uint64_t at = kv * region + (keys ? k_offset(slot, d, a.page_size, p.head_dim)
                                                : static_cast<uint64_t>(slot) * p.head_dim + d);
        *reinterpret_cast<uint4 *>(pool + to * page + at) = *reinterpret_cast<const uint4 *>(pool + from * page + at);
    }
}

struct CompactArgs {
    const uint32_t *path, *accepted;
    uint32_t width;
    uint32_t *new_lengths;  // null where they are the lengths themselves
};

constexpr uint32_t kMoves = 8;

// Block (sequence, layer, K or V). A thread moves its pieces of heads for one path
// entry after the other, kMoves of them loaded before any is stored: no entry's
// source is a place that an earlier entry's goes to, since path[i] >= i rises.
__global__ __launch_bounds__(256) void compact_kernel(const PageArgs a, const CompactArgs c, const PoolArgs p) {
    __shared__ uint64_t rows[2][kMoves];  // where a source and its place begin in the pool, ~0 for none
    const uint32_t s = blockIdx.x, tid = threadIdx.x;
    const bool keys = blockIdx.z == 0;
    uint16_t *pool = keys ? p.pools[blockIdx.y].k_pages : p.pools[blockIdx.y].v_pages;
    const uint64_t capacity = static_cast<uint64_t>(a.max_pages) * a.page_size;
    const uint64_t region = static_cast<uint64_t>(a.page_size) * p.head_dim;
    const uint32_t pieces = p.head_dim / 8;
    const uint32_t *path = c.path + static_cast<uint64_t>(s) * c.width;
    // threads 2 u and 2 u + 1 look up move u; its node is read before the count is known
    const uint32_t u = tid / 2, to = tid % 2;
    uint32_t node = u < min(kMoves, c.width) ? path[u] : 0;
    const uint32_t len = a.lengths[s], count = min(c.accepted[s], c.width);
    if (c.new_lengths && blockIdx.y == 0 && keys && tid == 0) c.new_lengths[s] = len + count;
    for (uint32_t i0 = 0; i0 < count; i0 += kMoves) {
        if (u < kMoves) {
            const uint32_t i = i0 + u;
            if (i0) node = i < count ? path[i] : i;
            const uint64_t j = static_cast<uint64_t>(len) + (to ? i : node);
            uint32_t page = kNoPage;
            if (i < count && node != i && j < capacity)
                page = a.table[static_cast<uint64_t>(s) * a.max_pages + j / a.page_size];
            const uint32_t other = __shfl_xor(page, 1, 64);
            const bool there = page < a.n_pages && other < a.n_pages;
            const uint32_t slot = j % a.page_size;
            rows[to][u] = there ? page * p.n_kv * region + (keys ? k_offset(slot, 0, a.page_size, p.head_dim)
                                                                 : static_cast<uint64_t>(slot) * p.head_dim)
                                : ~0ull;
        }
        __syncthreads();
        for (uint32_t x = tid; x < p.n_kv * pieces; x += blockDim.x) {
            const uint32_t d = x % pieces * 8;
            // a group's keys lie 32 dims apart: dim d of a K row is (d / 32) * 512 + d % 32 further on
            uint16_t *mine = pool + x / pieces * region + (keys ? (d / 32) * 512 + d % 32 : d);
            stream_u32x4_t v[kMoves];
#pragma unroll
            for (uint32_t m = 0; m < kMoves; ++m)
                if (rows[0][m] != ~0ull) v[m] = *reinterpret_cast<const stream_u32x4_t *>(mine + rows[0][m]);
#pragma unroll
            for (uint32_t m = 0; m < kMoves; ++m)
                if (rows[1][m] != ~0ull) *reinterpret_cast<stream_u32x4_t *>(mine + rows[1][m]) = v[m];
        }
        __syncthreads();
    }
}

__global__ __launch_bounds__(256) void advance_kernel(uint32_t *lengths, const uint32_t *accepted, uint32_t width,
                                                      uint32_t n) {
    const uint32_t s = blockIdx.x * blockDim.x + threadIdx.x;
    if (s < n) lengths[s] += min(accepted[s], width);
}

}  // namespace fh

using namespace fh;

namespace {

struct Operand {
    const char *what;
    const void *ptr;
    uint64_t bytes;
};

// The checks of a cache's tables and (with_pools) its pools; `with` are the call's
// other operands, written or not. Nothing overlaps anything here.
int check_cache(fh_device *dev, const char *fn, const fh_paged_cache *cache, bool with_refs, bool with_pools,
                std::initializer_list<Operand> with, PageArgs *pages, PoolArgs *pools) {
    if (int rc = check_usable(dev, fn)) return rc;
    if (cache == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: cache is null", fn);
    const fh_paged_cache &c = *cache;
    if (int rc = fh_check_dims(fn, {c.n_layers, c.n_kv, c.head_dim, c.n_pages, c.page_size, c.n_seqs, c.max_pages}))
        return rc;
    if (int rc = check_pages(fn, c.n_pages, c.page_size, c.max_pages)) return rc;
    if (c.n_seqs > kMaxSeqs)
        return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld sequences exceed %u", fn, (long long)c.n_seqs, kMaxSeqs);
    const uint64_t seqs = static_cast<uint64_t>(c.n_seqs) * 4;
    std::vector<Operand> all = {{"page_table", c.page_table, seqs * c.max_pages}, {"lengths", c.lengths, seqs}};
    if (with_refs) all.push_back({"refs", c.refs, static_cast<uint64_t>(c.n_pages) * 4});
    for (const Operand &o : with)
        if (o.ptr) all.push_back(o);
    for (const Operand &o : all)
        if (reinterpret_cast<uintptr_t>(o.ptr) % 4 != 0)
            return fail(FH_ERR_INVALID_ARGUMENT, "%s: %s must be 4-byte aligned", fn, o.what);
    if (with_pools) {
        if (c.head_dim < 32 || c.head_dim > 256 || c.head_dim % 32 != 0)
            return fail(FH_ERR_UNSUPPORTED, "%s: head_dim %lld must be a multiple of 32, at most 256", fn,
                        (long long)c.head_dim);
        if (c.n_kv < 1 || c.n_kv * c.head_dim > 0xFFFFFFll || c.page_size * c.n_kv * c.head_dim > 0x7FFFFFFFll)
            return fail(FH_ERR_INVALID_ARGUMENT, "%s: %lld KV heads", fn, (long long)c.n_kv);
        if (c.n_layers < 1 || c.n_layers > kMaxLayers || c.pools == nullptr)
            return fail(FH_ERR_INVALID_ARGUMENT, "%s: %lld layers (1 to %u, with their pools)", fn,
                        (long long)c.n_layers, kMaxLayers);
        uint64_t pool;
        if (int rc = size_product(fn, "a pool",
                                  {static_cast<uint64_t>(c.n_pages), static_cast<uint64_t>(c.n_kv),
                                   static_cast<uint64_t>(c.page_size), static_cast<uint64_t>(c.head_dim) * 2},
                                  &pool))
            return rc;
        for (int64_t l = 0; l < c.n_layers; ++l) {
            const fh_paged_pool &p = c.pools[l];
            if ((reinterpret_cast<uintptr_t>(p.k_pages) | reinterpret_cast<uintptr_t>(p.v_pages)) & 15u)
                return fail(FH_ERR_INVALID_ARGUMENT, "%s: pools must be 16-byte aligned", fn);
            all.push_back({"k_pages", p.k_pages, pool});
            all.push_back({"v_pages", p.v_pages, pool});
            pools->pools[l] = p;
        }
        pools->n_kv = static_cast<uint32_t>(c.n_kv);
        pools->head_dim = static_cast<uint32_t>(c.head_dim);
    }
    for (const Operand &o : all)
        if (int rc = check_range(dev, o.ptr, o.bytes, fn, o.what)) return rc;
    // by address, each may reach up to the next at most
    std::sort(all.begin(), all.end(), [](const Operand &x, const Operand &y) { return x.ptr < y.ptr; });
    for (size_t i = 0; i + 1 < all.size(); ++i)
        if (int rc = refuse_overlap(fn, all[i].what, all[i].ptr, all[i].bytes, all[i + 1].what, all[i + 1].ptr,
                                    all[i + 1].bytes))
            return rc;
    *pages = PageArgs{c.page_table,
                      c.lengths,
                      c.refs,
                      static_cast<uint32_t>(c.n_seqs),
                      static_cast<uint32_t>(c.max_pages),
                      static_cast<uint32_t>(c.n_pages),
                      static_cast<uint32_t>(c.page_size)};
    return set_current(dev, fn);
}

}  // namespace

extern "C" int fh_paged_reserve(fh_device *dev, const fh_paged_cache *cache, const uint32_t *extra, uint32_t *missing) {
    const char *fn = "fh_paged_reserve";
    if (int rc = check_usable(dev, fn)) return rc;
    if (cache == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: cache is null", fn);
    if (cache->n_seqs == 0) return FH_OK;
    if (extra == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: extra is null", fn);
    const uint64_t seqs = static_cast<uint64_t>(cache->n_seqs) * 4;
    PageArgs a;
    if (int rc = check_cache(dev, fn, cache, true, false, {{"extra", extra, seqs}, {"missing", missing, seqs}}, &a,
                             nullptr))
        return rc;
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kTableThreads), 0, dev->stream, a, extra, missing);
    });
}

extern "C" int fh_paged_free(fh_device *dev, const fh_paged_cache *cache, const uint32_t *seqs, int64_t n) {
    const char *fn = "fh_paged_free";
    if (int rc = check_usable(dev, fn)) return rc;
    if (int rc = fh_check_dims(fn, {n})) return rc;
    if (n > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld sequences exceed 65535", fn, (long long)n);
    if (n == 0) return FH_OK;
    if (seqs == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: seqs is null", fn);
    PageArgs a;
    if (int rc = check_cache(dev, fn, cache, true, false, {{"seqs", seqs, static_cast<uint64_t>(n) * 4}}, &a, nullptr))
        return rc;
    if (cache->n_seqs == 0) return FH_OK;
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(free_kernel, dim3(static_cast<uint32_t>(n)), dim3(256), 0, dev->stream, a, seqs);
    });
}

extern "C" int fh_paged_fork(fh_device *dev, const fh_paged_cache *cache, const uint32_t *from, const uint32_t *to,
                             int64_t n, uint32_t *lost) {
    const char *fn = "fh_paged_fork";
    if (int rc = check_usable(dev, fn)) return rc;
    if (int rc = fh_check_dims(fn, {n})) return rc;
    if (n > kMaxForks) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld forks exceed %u", fn, (long long)n, kMaxForks);
    if (n == 0) return FH_OK;
    if (from == nullptr || to == nullptr || lost == nullptr)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: from, to and lost must not be null", fn);
    if (cache != nullptr && cache->n_seqs == 0)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: a cache of no sequences", fn);
    const uint64_t each = static_cast<uint64_t>(n) * 4;
    PageArgs a;
    PoolArgs p;
    if (int rc = check_cache(dev, fn, cache, true, true, {{"from", from, each}, {"to", to, each}, {"lost", lost, each}},
                             &a, &p))
        return rc;
    const ForkArgs f{from, to, static_cast<uint32_t>(n), lost};
    if (int rc = dispatch(dev, fn, [&] {
            hipLaunchKernelGGL(fork_share_kernel, dim3(f.n), dim3(256), 0, dev->stream, a, f);
        }))
        return rc;
    if (int rc = dispatch(dev, fn, [&] {
            hipLaunchKernelGGL(fork_take_kernel, dim3(1), dim3(kTableThreads), 0, dev->stream, a, f);
        }))
        return rc;
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(fork_copy_kernel, dim3(f.n, static_cast<uint32_t>(cache->n_layers), 2), dim3(256), 0,
                           dev->stream, a, f, p);
    });
}

extern "C" int fh_paged_compact(fh_device *dev, const fh_paged_cache *cache, const uint32_t *path,
                                const uint32_t *accepted, int64_t width, uint32_t *new_lengths) {
    const char *fn = "fh_paged_compact";
    if (int rc = check_usable(dev, fn)) return rc;
    if (int rc = fh_check_dims(fn, {width})) return rc;
    if (width < 1 || width > 0xFFFF)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: width %lld must be 1 to 65535", fn, (long long)width);
    if (cache == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: cache is null", fn);
    if (cache->n_seqs == 0) return FH_OK;
    if (path == nullptr || accepted == nullptr || new_lengths == nullptr)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: path, accepted and new_lengths must not be null", fn);
    const uint64_t seqs = static_cast<uint64_t>(cache->n_seqs) * 4;
    const bool in_place = new_lengths == cache->lengths;
    PageArgs a;
    PoolArgs p;
    if (int rc = check_cache(dev, fn, cache, false, true,
                             {{"path", path, seqs * width},
                              {"accepted", accepted, seqs},
                              {"new_lengths", in_place ? nullptr : new_lengths, seqs}},
                             &a, &p))
        return rc;
    const CompactArgs c{path, accepted, static_cast<uint32_t>(width), in_place ? nullptr : new_lengths};
    // a thread for each piece of a token's heads
    const uint32_t threads = std::min(256u, (p.n_kv * (p.head_dim / 8) + 63) / 64 * 64);
    if (int rc = dispatch(dev, fn, [&] {
            hipLaunchKernelGGL(compact_kernel, dim3(a.n_seqs, static_cast<uint32_t>(cache->n_layers), 2), dim3(threads), 0,
                               dev->stream, a, c, p);
        }))
        return rc;
    if (!in_place) return FH_OK;
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(advance_kernel, dim3((a.n_seqs + 255) / 256), dim3(256), 0, dev->stream, a.lengths, accepted,
                           c.width, a.n_seqs);
    });
}
