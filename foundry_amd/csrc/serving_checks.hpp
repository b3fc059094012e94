// Host checks shared by the entry points of a serving step (paged cache,
// adapters, logit rules).
#pragma once

#include "decoder_common.hpp"

namespace fh {

// Product of sizes in bytes, refused where it does not fit 64 bits.
inline int size_product(const char *fn, const char *what, std::initializer_list<uint64_t> factors, uint64_t *out) {
    uint64_t n = 1;
    for (uint64_t f : factors)
        if (__builtin_mul_overflow(n, f, &n))
            return fail(FH_ERR_INVALID_ARGUMENT, "%s: the size of %s does not fit 64 bits", fn, what);
    *out = n;
    return FH_OK;
}

// Refuses an output that shares memory with an operand.
inline int refuse_overlap(const char *fn, const char *what, const void *p, uint64_t pn, const char *with, const void *q,
                          uint64_t qn) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    if (pn != 0 && qn != 0 && a < b + qn && b < a + pn)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: %s must not overlap %s", fn, what, with);
    return FH_OK;
}

}  // namespace fh
