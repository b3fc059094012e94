// Distributions of logits at a temperature (fh_logits_probs).
#include <algorithm>
#include <tuple>
#include <type_traits>

#include "serving_checks.hpp"

namespace fh {

// p_j = 2^((z_j - max z) k) / sum, k = log2 e / t. Bound by memory: the logits are
// read, the probabilities written. A row is cut into runs of tokens: one launch
// takes each run's maximum and its sum relative to that (and a greedy row's first
// largest token), the next joins a row's runs, reads the logits again, from the
// caches where they hold them, and writes. Runs are as long as a filled GPU allows.
// 512 bf16 rows of 128256 take 83 us (4.75 TB/s; 23 and 59 of the launches), 384 f32 rows 102 (3.9 TB/s), one
// bf16 row 7.1 us.
constexpr uint32_t kProbTokens = 8192;
constexpr uint32_t kProbThreads = 256;
// The shortest run, and the blocks that a launch aims for before runs get longer: each block of the
// second launch joins all runs of its row, so fewer are better (rows of 128256, one call over and over, with runs
// of 1024 and 2048 blocks beside these: 16 rows 14.1 and 9.1 us, 64 rows 16.3 and 14.0, 1 row 8.0 and 7.4).
constexpr uint32_t kProbLeast = 2048;
constexpr uint32_t kProbBlocks = 512;

struct RunStats {
    float m, sum;
    uint32_t first;  // the first token of logit m
};

template <typename T>
struct ProbArgs {
    const T *z;
    uint32_t n, run;
    const float *temperatures;
    RunStats *stats;  // [rows][runs]
    float *probs;
};

__device__ __forceinline__ uint32_t word_of(const uint4 raw, uint32_t i) {
    return i == 0 ? raw.x : i == 1 ? raw.y : i == 2 ? raw.z : raw.w;
}
__device__ __forceinline__ uint32_t word_of(const uint2 raw, uint32_t i) { return i == 0 ? raw.x : raw.y; }

// A piece's logits, NaN as -inf.
template <typename T, uint32_t E, typename Raw>
__device__ __forceinline__ void logits_of(const Raw raw, float (&v)[E]) {
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        const uint32_t word = word_of(raw, e * sizeof(T) / 4);
        v[e] = __uint_as_float(sizeof(T) == 4 ? word : e % 2 ? word & 0xFFFF0000u : word << 16);
        v[e] = fmaxf(v[e], -INFINITY);
    }
}

template <typename T>
__device__ __forceinline__ float logit_of(T z) {
    if constexpr (sizeof(T) == 2)
        return fmaxf(bf(z), -INFINITY);
    else
        return fmaxf(z, -INFINITY);
}

__device__ __forceinline__ float factor_of(float t) { return 1.4426950408889634f / fminf(fmaxf(t, 1e-30f), 1e30f); }

// The weight of v beside a largest logit m > -inf; infinite logits all weigh 1.
__device__ __forceinline__ float weight_of(float v, float m, float k) {
    return v == m ? 1.0f : __builtin_amdgcn_exp2f((v - m) * k);
}

// What a block has of its run: whole pieces of E tokens (a row's first may begin before it), the
// row's ends left to single tokens.
template <typename T, uint32_t Tokens>
struct Run {
    static constexpr uint32_t E = Tokens, kPieces = kProbTokens / (kProbThreads * E);
    typedef std::conditional_t<E * sizeof(T) == 16, uint4, uint2> Raw;
    __device__ __forceinline__ Raw load(uint32_t p) const { return *reinterpret_cast<const Raw *>(from + token(p)); }
    const T *from;
    int32_t lo;  // the run's first token (below 0 where the first piece begins before the row)
    uint32_t n, run;
    __device__ __forceinline__ Run(const ProbArgs<T> &a, uint32_t x, uint32_t row) : n(a.n), run(a.run) {
        from = a.z + static_cast<uint64_t>(row) * n;
        lo = static_cast<int32_t>(x * run) - static_cast<int32_t>((reinterpret_cast<uintptr_t>(from) & 15u) / sizeof(T));
    }
    // token of the thread's piece p, and whether it is whole
    __device__ __forceinline__ int32_t token(uint32_t p) const {
        return lo + static_cast<int32_t>((p * kProbThreads + threadIdx.x) * E);
    }
    __device__ __forceinline__ bool inside(uint32_t p) const {
        return (p * kProbThreads + threadIdx.x) * E < run && token(p) < static_cast<int32_t>(n);
    }
    __device__ __forceinline__ bool whole(uint32_t p) const {
        return inside(p) && token(p) >= 0 && token(p) + E <= n;
    }
    // the logits of piece p, -inf outside the row
    __device__ __forceinline__ void get(uint32_t p, const Raw raw, float (&v)[E]) const {
        if (whole(p)) {
            logits_of<T, E>(raw, v);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < E; ++e) {
                const int32_t j = token(p) + static_cast<int32_t>(e);
                v[e] = inside(p) && j >= 0 && j < static_cast<int32_t>(n) ? logit_of<T>(from[j]) : -INFINITY;
            }
        }
    }
};

// Block (run, row).
template <typename T>
__global__ __launch_bounds__(kProbThreads) void prob_stats_kernel(const ProbArgs<T> a) {
    using R = Run<T, 16 / sizeof(T)>;  // loads of 16 bytes
    __shared__ float part[kProbThreads / 64];
    __shared__ uint32_t first;
    const R r(a, blockIdx.x, blockIdx.y);
    typename R::Raw raw[R::kPieces];
#pragma unroll
    for (uint32_t p = 0; p < R::kPieces; ++p)
        if (r.whole(p)) raw[p] = r.load(p);
    const float t = a.temperatures ? a.temperatures[blockIdx.y] : 1.0f;
    const uint32_t wave = threadIdx.x / 64;
    float m = -INFINITY;
    float v[R::kPieces][R::E];
#pragma unroll
    for (uint32_t p = 0; p < R::kPieces; ++p) {
        r.get(p, raw[p], v[p]);
#pragma unroll
        for (uint32_t e = 0; e < R::E; ++e) m = fmaxf(m, v[p][e]);
    }
    m = wave_max(m);
    if (threadIdx.x % 64 == 0) part[wave] = m;
    if (threadIdx.x == 0) first = a.n;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kProbThreads / 64; ++w) m = fmaxf(m, part[w]);
    __syncthreads();
    float sum = 0.0f;
    if (!(t > 0.0f)) {  // greedy
#pragma unroll
        for (uint32_t p = 0; p < R::kPieces; ++p)
#pragma unroll
            for (uint32_t e = 0; e < R::E; ++e) {
                const int32_t j = r.token(p) + static_cast<int32_t>(e);
                if (v[p][e] == m && r.inside(p) && j >= 0 && j < static_cast<int32_t>(a.n))
                    atomicMin(&first, static_cast<uint32_t>(j));
            }
    } else if (m > -INFINITY) {
        const float k = factor_of(t);
#pragma unroll
        for (uint32_t p = 0; p < R::kPieces; ++p) {
            float s = 0.0f;
#pragma unroll
            for (uint32_t e = 0; e < R::E; ++e) s += weight_of(v[p][e], m, k);
            sum += s;
        }
        sum = wave_sum(sum);
        if (threadIdx.x % 64 == 0) part[wave] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0f;
        if (t > 0.0f && m > -INFINITY)
            for (uint32_t w = 0; w < kProbThreads / 64; ++w) sum += part[w];
        a.stats[static_cast<uint64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = {m, sum, first};
    }
}

// Block (run, row): every wavefront joins the row's runs, 64 at a time.
template <typename T>
__global__ __launch_bounds__(kProbThreads) void prob_write_kernel(const ProbArgs<T> a) {
    using R = Run<T, 4>;  // stores of 16 bytes, next to each other
    const R r(a, blockIdx.x, blockIdx.y);
    if (r.lo >= static_cast<int32_t>(a.n)) return;
    typename R::Raw raw[R::kPieces];
#pragma unroll
    for (uint32_t p = 0; p < R::kPieces; ++p)
        if (r.whole(p)) raw[p] = r.load(p);
    const float t = a.temperatures ? a.temperatures[blockIdx.y] : 1.0f;
    const float k = factor_of(t);
    const RunStats *stats = a.stats + static_cast<uint64_t>(blockIdx.y) * gridDim.x;
    const uint32_t lane = threadIdx.x % 64;
    float m = -INFINITY, sum = 0.0f;
    uint32_t first = a.n;
    for (uint32_t i = lane; i < gridDim.x; i += 64) {
        const RunStats x = stats[i];
        if (x.m > m) {  // the first run of the largest maximum
            sum = x.sum + sum * weight_of(m, x.m, k);
            m = x.m, first = x.first;
        } else if (x.m > -INFINITY) {
            sum += x.sum * weight_of(x.m, m, k);
        }
    }
    const float top = wave_max(m);
    sum = wave_sum(m > -INFINITY ? sum * weight_of(m, top, k) : 0.0f);
    if (m != top) first = a.n;
#pragma unroll
    for (int off = 32; off; off >>= 1) first = min(first, static_cast<uint32_t>(__shfl_xor(first, off, 64)));
    const bool greedy = !(t > 0.0f), none = top == -INFINITY;
    const float inv = 1.0f / sum;
    float *to = a.probs + static_cast<uint64_t>(blockIdx.y) * a.n;
    const bool aligned = (reinterpret_cast<uintptr_t>(to + r.lo) & 15u) == 0;
#pragma unroll
    for (uint32_t p = 0; p < R::kPieces; ++p) {
        if (!r.inside(p)) break;
        const int32_t j0 = r.token(p);
        float v[R::E];
        r.get(p, raw[p], v);
#pragma unroll
        for (uint32_t e = 0; e < R::E; ++e) {
            const float w = greedy ? (j0 + static_cast<int32_t>(e) == static_cast<int32_t>(first) ? 1.0f : 0.0f)
                                   : weight_of(v[e], top, k) * inv;
            v[e] = none ? 0.0f : w;
        }
        if (aligned && r.whole(p)) {
            __builtin_nontemporal_store(__builtin_bit_cast(stream_u32x4_t, make_float4(v[0], v[1], v[2], v[3])),
                                        reinterpret_cast<stream_u32x4_t *>(to + j0));
        } else {
#pragma unroll
            for (uint32_t e = 0; e < R::E; ++e) {
                const int32_t j = j0 + static_cast<int32_t>(e);
                if (j >= 0 && j < static_cast<int32_t>(a.n)) to[j] = v[e];
            }
        }
    }
}

}  // namespace fh

using namespace fh;

namespace {

// Tokens of a run for these sizes, and runs of a row (one may begin up to a piece before it).
uint32_t run_of(int64_t rows, int64_t n) {
    uint32_t run = kProbLeast;
    while (run < kProbTokens && rows * ((n + run - 1) / run) > kProbBlocks) run *= 2;
    return run;
}

uint64_t runs_of(int64_t n, uint32_t run) { return (static_cast<uint64_t>(n) + 7 + run - 1) / run; }

template <typename T>
int launch(fh_device *dev, const char *fn, const dim3 grid, const ProbArgs<T> &a) {
    if (int rc = dispatch(dev, fn, [&] {
            hipLaunchKernelGGL(prob_stats_kernel<T>, grid, dim3(kProbThreads), 0, dev->stream, a);
        }))
        return rc;
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(prob_write_kernel<T>, grid, dim3(kProbThreads), 0, dev->stream, a);
    });
}

}  // namespace

extern "C" int fh_logits_probs_workspace(int64_t rows, int64_t n, uint64_t *bytes) {
    const char *fn = "fh_logits_probs_workspace";
    if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: bytes is null", fn);
    if (int rc = fh_check_dims(fn, {rows, n})) return rc;
    if (rows > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld rows exceed 65535", fn, (long long)rows);
    if (n > 0x7FFFFFFFll - 2 * kProbTokens) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: n %lld", fn, (long long)n);
    // runs get longer where there are more than kProbBlocks of them, not counting a row's last piece
    *bytes = std::max<uint64_t>(kProbBlocks + rows, rows * runs_of(n, kProbTokens)) * sizeof(RunStats) + 16;
    return FH_OK;
}

extern "C" int fh_logits_probs(fh_device *dev, const void *logits, int dtype, int64_t rows, int64_t n,
                               const float *temperatures, void *workspace, uint64_t workspace_bytes, float *probs) {
    const char *fn = "fh_logits_probs";
    if (int rc = check_usable(dev, fn)) return rc;
    if (dtype != FH_BF16 && dtype != FH_F32)
        return fail(FH_ERR_DTYPE, "%s: dtype %d is neither F32 nor BF16", fn, dtype);
    uint64_t need = 0;
    if (int rc = fh_logits_probs_workspace(rows, n, &need)) return rc;
    if (rows == 0 || n == 0) return FH_OK;
    if (workspace_bytes < need)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: workspace of %llu bytes, %llu needed", fn,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
    const uint64_t elem = dtype == FH_F32 ? 4 : 2, count = static_cast<uint64_t>(rows) * n;
    if (reinterpret_cast<uintptr_t>(logits) % elem != 0 || reinterpret_cast<uintptr_t>(probs) % 4 != 0)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: logits and probs must be aligned to their types", fn);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", fn);
    if (int rc = check_words(fn, {{"temperatures", temperatures}})) return rc;
    const uint64_t each = static_cast<uint64_t>(rows) * 4;
    if (int rc = check_range(dev, logits, count * elem, fn, "logits")) return rc;
    if (int rc = check_range(dev, probs, count * 4, fn, "probs")) return rc;
    if (int rc = check_range(dev, workspace, need, fn, "workspace")) return rc;
    if (temperatures)
        if (int rc = check_range(dev, temperatures, each, fn, "temperatures")) return rc;
    for (const auto &[what, ptr, size] : {std::tuple{"probs", static_cast<const void *>(probs), count * 4},
                                          std::tuple{"workspace", static_cast<const void *>(workspace), need}}) {
        if (int rc = refuse_overlap(fn, what, ptr, size, "logits", logits, count * elem)) return rc;
        if (temperatures)
            if (int rc = refuse_overlap(fn, what, ptr, size, "temperatures", temperatures, each)) return rc;
    }
    if (int rc = refuse_overlap(fn, "workspace", workspace, need, "probs", probs, count * 4)) return rc;
    if (int rc = set_current(dev, fn)) return rc;
    const uint32_t run = run_of(rows, n);
    const dim3 grid(static_cast<uint32_t>(runs_of(n, run)), static_cast<uint32_t>(rows));
    RunStats *stats = static_cast<RunStats *>(workspace);
    if (dtype == FH_F32)
        return launch(dev, fn, grid,
                      ProbArgs<float>{static_cast<const float *>(logits), static_cast<uint32_t>(n), run, temperatures,
                                      stats, probs});
    return launch(dev, fn, grid,
                  ProbArgs<uint16_t>{static_cast<const uint16_t *>(logits), static_cast<uint32_t>(n), run, temperatures,
                                     stats, probs});
}
