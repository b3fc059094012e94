// Low-rank adapters of many requests beside a shared projection (fh_lora_add).
#include <tuple>

#include "serving_checks.hpp"

namespace fh {

// v[i, r] = scales[a] * sum_j x[i, j] A_a[r, j]: one block per row, a
// wavefront per rank at a time.
__global__ __launch_bounds__(256) void lora_down_kernel(const uint16_t *__restrict__ x, uint32_t k, uint64_t x_ld,
                                                        const uint16_t *__restrict__ a,
                                                        const float *__restrict__ scales, uint32_t n_adapters,
                                                        uint32_t rank, const uint32_t *__restrict__ adapters,
                                                        float *__restrict__ v) {
    const uint32_t i = blockIdx.x, id = adapters[i], lane = threadIdx.x & 63u;
    if (id >= n_adapters) return;
    for (uint32_t r = threadIdx.x >> 6; r < rank; r += 4) {
        const uint16_t *ar = a + (static_cast<uint64_t>(id) * rank + r) * k;
        float sum = 0.0f;
        for (uint32_t j = lane; j < k; j += 64) sum = fmaf(bf(x[i * x_ld + j]), bf(ar[j]), sum);
        sum = wave_sum(sum);
        if (lane == 0) v[static_cast<uint64_t>(i) * rank + r] = sum * scales[id];
    }
}

// y[i, c] = base[i, c] + sum_r v[i, r] B_a[c, r]: a thread per column.
template <typename T>
__global__ __launch_bounds__(256) void lora_up_kernel(const float *__restrict__ v, const uint16_t *__restrict__ b,
                                                      uint32_t n_adapters, uint32_t rank, uint32_t n,
                                                      const uint32_t *__restrict__ adapters, const T *base,
                                                      uint64_t base_ld, T *y, uint64_t y_ld) {
    const uint32_t i = blockIdx.x, c = blockIdx.y * 256 + threadIdx.x, id = adapters[i];
    if (c >= n) return;
    constexpr bool kBf16 = sizeof(T) == 2;
    if (id >= n_adapters) {
        y[i * y_ld + c] = base[i * base_ld + c];
        return;
    }
    float sum = 0.0f;
    for (uint32_t r = 0; r < rank; ++r)
        sum = fmaf(v[static_cast<uint64_t>(i) * rank + r], bf(b[(static_cast<uint64_t>(id) * n + c) * rank + r]), sum);
    if constexpr (kBf16)
        y[i * y_ld + c] = rne(bf(base[i * base_ld + c]) + sum);
    else
        y[i * y_ld + c] = base[i * base_ld + c] + sum;
}

}  // namespace fh

using namespace fh;

extern "C" int fh_lora_workspace(int64_t m, int64_t k, int64_t rank, uint64_t *bytes) {
    const char *fn = "fh_lora_workspace";
    if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: bytes is null", fn);
    if (int rc = fh_check_dims(fn, {m, k, rank})) return rc;
    if (rank < 8 || rank > 128 || rank % 8 != 0)
        return fail(FH_ERR_UNSUPPORTED, "%s: rank %lld must be a multiple of 8, at most 128", fn, (long long)rank);
    if (k < 8 || k % 8 != 0)
        return fail(FH_ERR_UNSUPPORTED, "%s: k %lld must be a multiple of 8", fn, (long long)k);
    *bytes = static_cast<uint64_t>(m) * rank * 4 + 16;
    return FH_OK;
}

extern "C" int fh_lora_add(fh_device *dev, const uint16_t *x, int64_t m, int64_t k, int64_t x_ld, const uint16_t *a,
                           const uint16_t *b, const float *scales, int64_t n_adapters, int64_t rank, int64_t n,
                           const uint32_t *adapters, const void *base, int64_t base_ld, void *y, int64_t y_ld,
                           int dtype, void *workspace, uint64_t workspace_bytes) {
    const char *fn = "fh_lora_add";
    if (int rc = check_usable(dev, fn)) return rc;
    if (int rc = fh_check_dims(fn, {m, k, x_ld, n_adapters, rank, n, base_ld, y_ld})) return rc;
    uint64_t need = 0;
    if (int rc = fh_lora_workspace(m, k, rank, &need)) return rc;
    if (dtype != FH_BF16 && dtype != FH_F32)
        return fail(FH_ERR_DTYPE, "%s: dtype %d is neither F32 nor BF16", fn, dtype);
    if (m == 0 || n == 0) return FH_OK;
    if (x_ld < k || x_ld % 8 != 0)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: x_ld %lld must be a multiple of 8 and at least k", fn,
                    (long long)x_ld);
    if (base_ld < n || y_ld < n)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: base_ld %lld and y_ld %lld must be at least n", fn,
                    (long long)base_ld, (long long)y_ld);
    if (n_adapters < 1) return fail(FH_ERR_INVALID_ARGUMENT, "%s: n_adapters must be at least 1", fn);
    if (base == y && base_ld != y_ld)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: y in base's place needs base's stride", fn);
    if (workspace_bytes < need)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: workspace of %llu bytes, %llu needed", fn,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
    const uint64_t elem = dtype == FH_F32 ? 4 : 2, rows = static_cast<uint64_t>(m);
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) |
         reinterpret_cast<uintptr_t>(workspace)) &
        15u)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: x, a, b and workspace must be 16-byte aligned", fn);
    if ((reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(y)) & (elem - 1))
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: base and y must be aligned to their dtype", fn);
    const uint64_t u = static_cast<uint64_t>(n_adapters) * rank * 2;
    const uint64_t x_bytes = ((rows - 1) * x_ld + k) * 2, y_bytes = ((rows - 1) * y_ld + n) * elem;
    const uint64_t base_bytes = ((rows - 1) * base_ld + n) * elem;
    uint64_t a_bytes, b_bytes;
    if (int rc = size_product(fn, "a", {u, static_cast<uint64_t>(k)}, &a_bytes)) return rc;
    if (int rc = size_product(fn, "b", {u, static_cast<uint64_t>(n)}, &b_bytes)) return rc;
    if (int rc = check_range(dev, x, x_bytes, fn, "x")) return rc;
    if (int rc = check_range(dev, a, a_bytes, fn, "a")) return rc;
    if (int rc = check_range(dev, b, b_bytes, fn, "b")) return rc;
    if (int rc = check_range(dev, scales, static_cast<uint64_t>(n_adapters) * 4, fn, "scales")) return rc;
    if (int rc = check_range(dev, adapters, rows * 4, fn, "adapters")) return rc;
    if (int rc = check_range(dev, base, base_bytes, fn, "base")) return rc;
    if (int rc = check_range(dev, y, y_bytes, fn, "y")) return rc;
    if (int rc = check_range(dev, workspace, need, fn, "workspace")) return rc;
    if (base != y)
        if (int rc = refuse_overlap(fn, "y", y, y_bytes, "base", base, base_bytes)) return rc;
    for (const auto &[what, ptr, size] :
         {std::tuple{"y", static_cast<const void *>(y), y_bytes},
          std::tuple{"workspace", static_cast<const void *>(workspace), need}}) {
        if (int rc = refuse_overlap(fn, what, ptr, size, "x", x, x_bytes)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "a", a, a_bytes)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "b", b, b_bytes)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "adapters", adapters, rows * 4)) return rc;
    }
    if (int rc = refuse_overlap(fn, "workspace", workspace, need, "y", y, y_bytes)) return rc;
    if (int rc = refuse_overlap(fn, "workspace", workspace, need, "base", base, base_bytes)) return rc;
    if ((n + 255) / 256 > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: n %lld", fn, (long long)n);
    if (int rc = set_current(dev, fn)) return rc;
    float *v = static_cast<float *>(workspace);
    if (int rc = dispatch(dev, fn, [&] {
            hipLaunchKernelGGL(lora_down_kernel, dim3(static_cast<uint32_t>(m)), dim3(256), 0, dev->stream, x,
                               static_cast<uint32_t>(k), static_cast<uint64_t>(x_ld), a, scales,
                               static_cast<uint32_t>(n_adapters), static_cast<uint32_t>(rank), adapters, v);
        }))
        return rc;
    const dim3 grid(static_cast<uint32_t>(m), static_cast<uint32_t>((n + 255) / 256));
    return dispatch(dev, fn, [&] {
        if (dtype == FH_F32)
            hipLaunchKernelGGL(lora_up_kernel<float>, grid, dim3(256), 0, dev->stream, v, b,
                               static_cast<uint32_t>(n_adapters), static_cast<uint32_t>(rank),
                               static_cast<uint32_t>(n), adapters, static_cast<const float *>(base),
                               static_cast<uint64_t>(base_ld), static_cast<float *>(y), static_cast<uint64_t>(y_ld));
        else
            hipLaunchKernelGGL(lora_up_kernel<uint16_t>, grid, dim3(256), 0, dev->stream, v, b,
                               static_cast<uint32_t>(n_adapters), static_cast<uint32_t>(rank),
                               static_cast<uint32_t>(n), adapters, static_cast<const uint16_t *>(base),
                               static_cast<uint64_t>(base_ld), static_cast<uint16_t *>(y),
                               static_cast<uint64_t>(y_ld));
    });
}
