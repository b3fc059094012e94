// Penalties, biases and grammar masks on logits (fh_logits_process).
#include "serving_checks.hpp"

namespace fh {

// Tokens of one block: their counts and bias entries are a table in LDS.
constexpr uint32_t kRuleChunk = 4096;

// Block (chunk of tokens, row): the row's history is counted into the chunk's
// table (bit 31: said at all; bits 0..30: times generated) and the row's bias
// list entered into another (entry index + 1, the last of one id staying),
// then each logit of the chunk goes through the rules. Whole-number LDS
// atomics: the result does not depend on their order. Contraction is off, so
// that each step is one fp32 rounding.
template <typename T>
__global__ __launch_bounds__(256) void logit_rules_kernel(const T *z, uint32_t n, fh_logit_rules rules, T *out) {
#pragma clang fp contract(off)
    __shared__ uint32_t said[kRuleChunk], entry[kRuleChunk];
    const uint32_t r = blockIdx.y, lo = blockIdx.x * kRuleChunk, count = min(kRuleChunk, n - lo);
    for (uint32_t i = threadIdx.x; i < kRuleChunk; i += 256) said[i] = entry[i] = 0;
    __syncthreads();
    if (rules.history) {
        const uint32_t *ids = rules.history + static_cast<uint64_t>(r) * rules.history_ld;
        const uint32_t used = min(rules.history_len[r], static_cast<uint32_t>(rules.history_ld));
        const uint32_t prompt = rules.prompt_len ? rules.prompt_len[r] : 0;
        for (uint32_t i = threadIdx.x; i < used; i += 256) {
            const uint32_t at = ids[i] - lo;
            if (ids[i] >= lo && at < count) {
                atomicOr(&said[at], 0x80000000u);
                if (i >= prompt) atomicAdd(&said[at], 1u);
            }
        }
    }
    if (rules.bias_ids) {
        const uint32_t *ids = rules.bias_ids + static_cast<uint64_t>(r) * rules.bias_ld;
        uint32_t used = static_cast<uint32_t>(rules.bias_ld);
        if (rules.bias_len) used = min(used, rules.bias_len[r]);
        for (uint32_t i = threadIdx.x; i < used; i += 256) {
            const uint32_t at = ids[i] - lo;
            if (ids[i] >= lo && at < count) atomicMax(&entry[at], i + 1);
        }
    }
    __syncthreads();
    const float rep = rules.repetition ? rules.repetition[r] : 1.0f;
    const float freq = rules.frequency ? rules.frequency[r] : 0.0f;
    const float pres = rules.presence ? rules.presence[r] : 0.0f;
    const uint32_t words = (n + 31) / 32;
    for (uint32_t i = threadIdx.x; i < count; i += 256) {
        const uint64_t at = static_cast<uint64_t>(r) * n + lo + i;
        float v;
        if constexpr (sizeof(T) == 2)
            v = bf(z[at]);
        else
            v = z[at];
        const uint32_t s = said[i], times = s & 0x7FFFFFFFu;
        if (rules.repetition && s) v = v > 0.0f ? v / rep : v * rep;
        if (times) {
            if (rules.frequency) v = v - freq * static_cast<float>(times);
            if (rules.presence) v = v - pres;
        }
        if (entry[i]) v = v + rules.bias_values[static_cast<uint64_t>(r) * rules.bias_ld + entry[i] - 1];
        if (rules.mask) {
            const uint32_t j = lo + i;
            if (!(rules.mask[static_cast<uint64_t>(r) * words + j / 32] >> (j % 32) & 1u)) v = -INFINITY;
        }
        if constexpr (sizeof(T) == 2)
            out[at] = rne(v);
        else
            out[at] = v;
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
    if (u.history) {
        if (int rc = check_range(dev, u.history, r * u.history_ld * 4, fn, "history")) return rc;
        if (int rc = check_range(dev, u.history_len, r * 4, fn, "history_len")) return rc;
    }
    if (u.bias_ids) {
        if (int rc = check_range(dev, u.bias_ids, r * u.bias_ld * 4, fn, "bias_ids")) return rc;
        if (int rc = check_range(dev, u.bias_values, r * u.bias_ld * 4, fn, "bias_values")) return rc;
        if (u.bias_len)
            if (int rc = check_range(dev, u.bias_len, r * 4, fn, "bias_len")) return rc;
    }
    if (u.prompt_len)
        if (int rc = check_range(dev, u.prompt_len, r * 4, fn, "prompt_len")) return rc;
    if (u.repetition)
        if (int rc = check_range(dev, u.repetition, r * 4, fn, "repetition")) return rc;
    if (u.frequency)
        if (int rc = check_range(dev, u.frequency, r * 4, fn, "frequency")) return rc;
    if (u.presence)
        if (int rc = check_range(dev, u.presence, r * 4, fn, "presence")) return rc;
    if (u.mask)
        if (int rc = check_range(dev, u.mask, r * ((n + 31) / 32) * 4, fn, "mask")) return rc;
    if (int rc = set_current(dev, fn)) return rc;
    const dim3 grid(static_cast<uint32_t>((n + kRuleChunk - 1) / kRuleChunk), static_cast<uint32_t>(rows));
    return dispatch(dev, fn, [&] {
        if (dtype == FH_F32)
            hipLaunchKernelGGL(logit_rules_kernel<float>, grid, dim3(256), 0, dev->stream,
                               static_cast<const float *>(logits), static_cast<uint32_t>(n), u,
                               static_cast<float *>(out));
        else
            hipLaunchKernelGGL(logit_rules_kernel<uint16_t>, grid, dim3(256), 0, dev->stream,
                               static_cast<const uint16_t *>(logits), static_cast<uint32_t>(n), u,
                               static_cast<uint16_t *>(out));
    });
}
