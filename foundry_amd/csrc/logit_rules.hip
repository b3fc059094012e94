// Penalties, biases and grammar masks on logits (fh_logits_process).
#include <tuple>
#include <type_traits>

#include "serving_checks.hpp"

namespace fh {

// Bound by memory: the logits go through once, in pieces of 16 bytes where
// their rows are so aligned (a row's first piece may begin before it). What a
// token needs to know of the row's lists stands in LDS: a block takes a run of
// tokens, enters the bias list into a table of them and counts the whole history
// there too. Every block of a row reads its lists, from the L2: runs are as long
// as the LDS and a filled GPU allow. 64 rows of 128256 bf16 take 6.7 us with no
// rule (4.9 TB/s), 10.1 with histories to 500, 12.7 with histories to 8192, 13.5
// with a mask and 300 biases a row as well: the lists' latency and the tables.
// (256 threads with runs of 4096: 14.5; 512 with 4096: 15.5; 1024 with 8192:
// 16.0, with 16384: 13.8.)
constexpr uint32_t kRuleTokens = 8192;
constexpr uint32_t kRuleThreads = 512;
// The shortest run, and the blocks that a launch aims for before runs get longer.
constexpr uint32_t kRuleLeast = 512;
constexpr uint32_t kRuleBlocks = 1024;
// A token's word: its count among the generated, then a bit for an id of the
// prompt, then a bias entry's index + 1, for lists up to these lengths.
constexpr uint32_t kCountBits = 20, kMaxCounted = (1u << kCountBits) - 1, kMaxBiases = (1u << (31 - kCountBits)) - 1;

// Calls take(i, list[i]) for i < n: 16-byte loads where the list is aligned,
// several requested together (the list's last words again past its end).
template <typename Take>
__device__ __forceinline__ void for_list(const uint32_t *list, uint32_t n, Take take) {
    constexpr uint32_t kLoads = 4;
    if (n == 0) return;
    if ((reinterpret_cast<uintptr_t>(list) & 15u) == 0) {
        const uint32_t quads = n / 4;
        for (uint32_t q0 = threadIdx.x; q0 < quads; q0 += kRuleThreads * kLoads) {
            uint4 v[kLoads];
#pragma unroll
            for (uint32_t u = 0; u < kLoads; ++u)
                v[u] = reinterpret_cast<const uint4 *>(list)[min(q0 + u * kRuleThreads, quads - 1)];
#pragma unroll
            for (uint32_t u = 0; u < kLoads; ++u) {
                const uint32_t i = (q0 + u * kRuleThreads) * 4;
                if (q0 + u * kRuleThreads < quads) {
                    take(i, v[u].x);
                    take(i + 1, v[u].y);
                    take(i + 2, v[u].z);
                    take(i + 3, v[u].w);
                }
            }
        }
        if (threadIdx.x < n % 4) take(quads * 4 + threadIdx.x, list[quads * 4 + threadIdx.x]);
        return;
    }
    for (uint32_t i0 = threadIdx.x; i0 < n; i0 += kRuleThreads * kLoads) {
        uint32_t v[kLoads];
#pragma unroll
        for (uint32_t u = 0; u < kLoads; ++u) v[u] = list[min(i0 + u * kRuleThreads, n - 1)];
#pragma unroll
        for (uint32_t u = 0; u < kLoads; ++u)
            if (i0 + u * kRuleThreads < n) take(i0 + u * kRuleThreads, v[u]);
    }
}

// Block (run, row). Of a bias id listed twice the last entry stays. TWO: lists
// too long for one word: a table of counts (bit 31: an id of the prompt) and one
// of bias entries. Whole-number LDS atomics: their order does not matter.
// Contraction is off, so that each step is one fp32 rounding.
template <typename T, bool TWO>
__global__ __launch_bounds__(kRuleThreads) void logit_rules_kernel(const T *z, uint32_t n, uint32_t run,
                                                                   const fh_logit_rules rules, T *out) {
#pragma clang fp contract(off)
    constexpr uint32_t E = 16 / sizeof(T);  // logits of a piece
    constexpr uint32_t kPieces = kRuleTokens / (kRuleThreads * E);
    constexpr uint32_t kSaid = TWO ? 0x80000000u : 1u << kCountBits, kShift = TWO ? 0 : kCountBits + 1;
    __shared__ __attribute__((aligned(16))) uint32_t said[TWO ? 2 * kRuleTokens : kRuleTokens];
    uint32_t *entry = TWO ? said + kRuleTokens : said;
    const uint32_t r = blockIdx.y;
    const T *from = z + static_cast<uint64_t>(r) * n;
    T *to = out + static_cast<uint64_t>(r) * n;
    // tokens before the row that its first piece begins with
    const uint32_t before = (reinterpret_cast<uintptr_t>(from) & 15u) / sizeof(T);
    const bool same = ((reinterpret_cast<uintptr_t>(from) ^ reinterpret_cast<uintptr_t>(to)) & 15u) == 0;
    // this run: tokens lo .. lo + run - 1 (lo < 0 where the first piece begins before the row)
    const int32_t lo = static_cast<int32_t>(blockIdx.x * run) - static_cast<int32_t>(before);
    if (lo >= static_cast<int32_t>(n)) return;
    const bool history = rules.history != nullptr, bias = rules.bias_ids != nullptr;
    const float rep = rules.repetition ? rules.repetition[r] : 1.0f;
    const float freq = rules.frequency ? rules.frequency[r] : 0.0f;
    const float pres = rules.presence ? rules.presence[r] : 0.0f;
    const uint32_t said_len = history ? min(rules.history_len[r], static_cast<uint32_t>(rules.history_ld)) : 0;
    const uint32_t prompt = history && rules.prompt_len ? rules.prompt_len[r] : 0;
    const uint32_t bias_ld = static_cast<uint32_t>(rules.bias_ld);
    const uint32_t bias_used = bias && rules.bias_len ? min(bias_ld, rules.bias_len[r]) : bias_ld;
    const float *values = bias ? rules.bias_values + static_cast<uint64_t>(r) * rules.bias_ld : nullptr;
    const uint32_t *mask = rules.mask ? rules.mask + static_cast<uint64_t>(r) * ((n + 31) / 32) : nullptr;
    // the thread's whole pieces and their mask bits are requested before the lists are gone through
    uint4 raw[kPieces];
    uint32_t bits[kPieces][2];
#pragma unroll
    for (uint32_t p = 0; p < kPieces; ++p) {
        const uint32_t at = (p * kRuleThreads + threadIdx.x) * E;
        const int32_t j0 = lo + static_cast<int32_t>(at);
        if (at < run && j0 >= 0 && j0 + E <= n) {
            raw[p] = *reinterpret_cast<const uint4 *>(from + j0);
            bits[p][0] = mask ? mask[j0 / 32] : ~0u;
            bits[p][1] = mask ? mask[(j0 + E - 1) / 32] : ~0u;
        }
    }
    for (uint32_t i = threadIdx.x * 4; i < run; i += kRuleThreads * 4) {
        if (history || (bias && !TWO)) *reinterpret_cast<uint4 *>(said + i) = make_uint4(0, 0, 0, 0);
        if (bias && TWO) *reinterpret_cast<uint4 *>(entry + i) = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    if (bias) {
        for_list(rules.bias_ids + static_cast<uint64_t>(r) * rules.bias_ld, bias_used, [&](uint32_t i, uint32_t id) {
            const uint32_t at = id - static_cast<uint32_t>(lo);
            if (id < n && at < run) atomicMax(&entry[at], (i + 1) << kShift);
        });
        if (!TWO) __syncthreads();  // the entries are the words' largest part: before the counts
    }
    if (history)
        for_list(rules.history + static_cast<uint64_t>(r) * rules.history_ld, said_len, [&](uint32_t i, uint32_t id) {
            const uint32_t at = id - static_cast<uint32_t>(lo);
            if (id >= n || at >= run) return;
            if (i < prompt)
                atomicOr(&said[at], kSaid);
            else
                atomicAdd(&said[at], 1u);
        });
    __syncthreads();
    const bool words = history || (bias && !TWO);
    // one logit: s its word, e its entry's where that is another
    auto apply = [&](float v, uint32_t s, uint32_t e) {
        if (!TWO) e = s >> kShift, s &= 2 * kSaid - 1;
        const uint32_t times = s & (kSaid - 1);
        if (rules.repetition && s) v = v > 0.0f ? v / rep : v * rep;
        if (times) {
            if (rules.frequency) v = v - freq * static_cast<float>(times);
            if (rules.presence) v = v - pres;
        }
        if (e) v = v + values[e - 1];
        return v;
    };
#pragma unroll
    for (uint32_t p = 0; p < kPieces; ++p) {
        const uint32_t at = (p * kRuleThreads + threadIdx.x) * E;
        const int32_t j0 = lo + static_cast<int32_t>(at);
        if (at >= run || j0 >= static_cast<int32_t>(n)) break;
        if (j0 >= 0 && j0 + E <= n) {
            const uint32_t allow = (static_cast<uint64_t>(bits[p][1]) << 32 | bits[p][0]) >> (j0 % 32);
            float v[E];
            if constexpr (sizeof(T) == 2) {
                unpack8(raw[p], v);
            } else {
                v[0] = __uint_as_float(raw[p].x), v[1] = __uint_as_float(raw[p].y);
                v[2] = __uint_as_float(raw[p].z), v[3] = __uint_as_float(raw[p].w);
            }
            uint32_t s[E], e[E], any = 0;
#pragma unroll
            for (uint32_t i = 0; i < E; i += 4) {
                const uint4 a = words ? *reinterpret_cast<const uint4 *>(said + at + i) : make_uint4(0, 0, 0, 0);
                const uint4 b = bias && TWO ? *reinterpret_cast<const uint4 *>(entry + at + i) : make_uint4(0, 0, 0, 0);
                s[i] = a.x, s[i + 1] = a.y, s[i + 2] = a.z, s[i + 3] = a.w;
                e[i] = b.x, e[i + 1] = b.y, e[i + 2] = b.z, e[i + 3] = b.w;
                any |= a.x | a.y | a.z | a.w | b.x | b.y | b.z | b.w;
            }
            if (any)
#pragma unroll
                for (uint32_t i = 0; i < E; ++i) v[i] = apply(v[i], s[i], e[i]);
#pragma unroll
            for (uint32_t i = 0; i < E; ++i)
                if (!(allow >> i & 1)) v[i] = -INFINITY;
            uint4 o;
            if constexpr (sizeof(T) == 2)
                o = make_uint4(f32x2_to_bf16x2_rne(v[0], v[1]), f32x2_to_bf16x2_rne(v[2], v[3]),
                               f32x2_to_bf16x2_rne(v[4], v[5]), f32x2_to_bf16x2_rne(v[6], v[7]));
            else
                o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                               __float_as_uint(v[3]));
            if (same) {
                *reinterpret_cast<uint4 *>(to + j0) = o;
            } else {
                const T *x = reinterpret_cast<const T *>(&o);
#pragma unroll
                for (uint32_t i = 0; i < E; ++i) to[j0 + i] = x[i];
            }
            continue;
        }
        // the row's ends
        for (int32_t j = max(j0, 0); j < min(j0 + static_cast<int32_t>(E), static_cast<int32_t>(n)); ++j) {
            const uint32_t i = j - lo;
            float v;
            if constexpr (sizeof(T) == 2)
                v = bf(from[j]);
            else
                v = from[j];
            v = apply(v, words ? said[i] : 0, bias && TWO ? entry[i] : 0);
            if (mask && !(mask[j / 32] >> (j % 32) & 1u)) v = -INFINITY;
            if constexpr (sizeof(T) == 2)
                to[j] = rne(v);
            else
                to[j] = v;
        }
    }
}

}  // namespace fh

using namespace fh;

extern "C" int fh_logits_process(fh_device *dev, const void *logits, int dtype, int64_t rows, int64_t n,
                                 const fh_logit_rules *rules, void *out) {
    const char *fn = "fh_logits_process";
    if (int rc = check_usable(dev, fn)) return rc;
    if (rules == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: rules is null", fn);
    const fh_logit_rules &u = *rules;
    if (int rc = fh_check_dims(fn, {rows, n, u.history_ld, u.bias_ld})) return rc;
    if (dtype != FH_BF16 && dtype != FH_F32)
        return fail(FH_ERR_DTYPE, "%s: dtype %d is neither F32 nor BF16", fn, dtype);
    if (n > 0x7FFFFFFFll - 2 * kRuleTokens) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: n %lld", fn, (long long)n);
    if (rows > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld rows exceed 65535", fn, (long long)rows);
    if ((u.history == nullptr) != (u.history_len == nullptr))
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: history and history_len go together", fn);
    if (u.history == nullptr && (u.repetition || u.frequency || u.presence))
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: penalties need the history", fn);
    if ((u.bias_ids == nullptr) != (u.bias_values == nullptr))
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: bias_ids and bias_values go together", fn);
    if (rows == 0 || n == 0) return FH_OK;
    const uint64_t elem = dtype == FH_F32 ? 4 : 2, r = static_cast<uint64_t>(rows);
    const uint64_t bytes = r * n * elem;
    for (const void *p : {logits, static_cast<const void *>(out)})
        if (reinterpret_cast<uintptr_t>(p) % elem != 0)
            return fail(FH_ERR_INVALID_ARGUMENT, "%s: logits and out must be aligned to their dtype", fn);
    if (int rc = check_range(dev, logits, bytes, fn, "logits")) return rc;
    if (int rc = check_range(dev, out, bytes, fn, "out")) return rc;
    if (logits != out)
        if (int rc = refuse_overlap(fn, "out", out, bytes, "logits", logits, bytes)) return rc;
    const uint64_t each = r * 4;
    for (const auto &[what, ptr, size] :
         {std::tuple{"history", static_cast<const void *>(u.history), each * u.history_ld},
          std::tuple{"history_len", static_cast<const void *>(u.history_len), each},
          std::tuple{"prompt_len", static_cast<const void *>(u.prompt_len), each},
          std::tuple{"repetition", static_cast<const void *>(u.repetition), each},
          std::tuple{"frequency", static_cast<const void *>(u.frequency), each},
          std::tuple{"presence", static_cast<const void *>(u.presence), each},
          std::tuple{"bias_ids", static_cast<const void *>(u.bias_ids), each * u.bias_ld},
          std::tuple{"bias_values", static_cast<const void *>(u.bias_values), each * u.bias_ld},
          std::tuple{"bias_len", static_cast<const void *>(u.bias_ids ? u.bias_len : nullptr), each},
          std::tuple{"mask", static_cast<const void *>(u.mask), each * ((n + 31) / 32)}}) {
        if (ptr == nullptr) continue;
        if (int rc = check_range(dev, ptr, size, fn, what)) return rc;
        if (int rc = refuse_overlap(fn, "out", out, bytes, what, ptr, size)) return rc;
    }
    if (int rc = set_current(dev, fn)) return rc;
    const bool two = (u.history && u.history_ld > kMaxCounted) || (u.bias_ids && u.bias_ld >= kMaxBiases);
    uint32_t run = kRuleLeast;
    while (run < kRuleTokens && r * ((n + run - 1) / run) > kRuleBlocks) run *= 2;
    // a run may begin up to a piece before its row
    const dim3 grid(static_cast<uint32_t>((n + 16 / elem - 1 + run - 1) / run), static_cast<uint32_t>(rows));
    auto launch = [&](auto kernel, auto *of) {
        using T = std::remove_pointer_t<decltype(of)>;
        return dispatch(dev, fn, [&] {
            hipLaunchKernelGGL(kernel, grid, dim3(kRuleThreads), 0, dev->stream, static_cast<const T *>(logits),
                               static_cast<uint32_t>(n), run, u, static_cast<T *>(out));
        });
    };
    float *const f32 = nullptr;
    uint16_t *const bf16 = nullptr;
    if (dtype == FH_F32)
        return two ? launch(logit_rules_kernel<float, true>, f32) : launch(logit_rules_kernel<float, false>, f32);
    return two ? launch(logit_rules_kernel<uint16_t, true>, bf16) : launch(logit_rules_kernel<uint16_t, false>, bf16);
}
