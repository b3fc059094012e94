// Distributions of logits at a temperature (fh_logits_probs).
#include <tuple>
#include <type_traits>

#include "serving_checks.hpp"

namespace fh {

// p_j = 2^((z_j - max z) log2 e / t) / sum. One block per row, which it reads three
// times: for the maximum (and, for a greedy row, its first place), the sum, and p.
constexpr uint32_t kProbThreads = 1024;

template <typename T>
__device__ __forceinline__ float logit(const T *z, uint32_t j) {
    float v;
    if constexpr (sizeof(T) == 2)
        v = bf(z[j]);
    else
        v = z[j];
    return fmaxf(v, -INFINITY);  // a NaN counts as -inf
}

template <typename T>
__global__ __launch_bounds__(kProbThreads) void probs_kernel(const T *__restrict__ z, uint32_t n,
                                                             const float *__restrict__ temperatures,
                                                             float *__restrict__ probs) {
    __shared__ float part[kProbThreads / 64];
    __shared__ uint32_t first;
    const T *row = z + static_cast<uint64_t>(blockIdx.x) * n;
    float *to = probs + static_cast<uint64_t>(blockIdx.x) * n;
    const uint32_t wave = threadIdx.x / 64;
    float m = -INFINITY;
    for (uint32_t j = threadIdx.x; j < n; j += kProbThreads) m = fmaxf(m, logit(row, j));
    m = wave_max(m);
    if (threadIdx.x % 64 == 0) part[wave] = m;
    if (threadIdx.x == 0) first = n;
    __syncthreads();
    for (uint32_t w = 0; w < kProbThreads / 64; ++w) m = fmaxf(m, part[w]);
    __syncthreads();
    const float t = temperatures ? temperatures[blockIdx.x] : 1.0f;
    if (m == -INFINITY) {
        for (uint32_t j = threadIdx.x; j < n; j += kProbThreads) to[j] = 0.0f;
        return;
    }
    if (!(t > 0.0f)) {
        for (uint32_t j = threadIdx.x; j < n; j += kProbThreads)
            if (logit(row, j) == m) {
                atomicMin(&first, j);
                break;
            }
        __syncthreads();
        for (uint32_t j = threadIdx.x; j < n; j += kProbThreads) to[j] = j == first ? 1.0f : 0.0f;
        return;
    }
    const float k = 1.4426950408889634f / fminf(fmaxf(t, 1e-30f), 1e30f);
    auto weight = [&](uint32_t j) {
        const float v = logit(row, j);
        return v == m ? 1.0f : __builtin_amdgcn_exp2f((v - m) * k);
    };
    float sum = 0.0f;
    for (uint32_t j = threadIdx.x; j < n; j += kProbThreads) sum += weight(j);
    sum = wave_sum(sum);
    if (threadIdx.x % 64 == 0) part[wave] = sum;
    __syncthreads();
    sum = 0.0f;
    for (uint32_t w = 0; w < kProbThreads / 64; ++w) sum += part[w];
    for (uint32_t j = threadIdx.x; j < n; j += kProbThreads) to[j] = weight(j) / sum;
}

}  // namespace fh

using namespace fh;

extern "C" int fh_logits_probs_workspace(int64_t rows, int64_t n, uint64_t *bytes) {
    const char *fn = "fh_logits_probs_workspace";
    if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: bytes is null", fn);
    if (int rc = fh_check_dims(fn, {rows, n})) return rc;
    if (rows > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld rows exceed 65535", fn, (long long)rows);
    *bytes = 16;
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
    const dim3 grid(static_cast<uint32_t>(rows)), threads(kProbThreads);
    return dispatch(dev, fn, [&] {
        if (dtype == FH_F32)
            hipLaunchKernelGGL(probs_kernel<float>, grid, threads, 0, dev->stream, static_cast<const float *>(logits),
                               static_cast<uint32_t>(n), temperatures, probs);
        else
            hipLaunchKernelGGL(probs_kernel<uint16_t>, grid, threads, 0, dev->stream,
                               static_cast<const uint16_t *>(logits), static_cast<uint32_t>(n), temperatures, probs);
    });
}
