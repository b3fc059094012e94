// Which drafted tokens the target's distributions accept (fh_verify_draft).
#include "serving_checks.hpp"

namespace fh {

// The mathematics. At node a a child's token x, drawn from q, is accepted with
// probability min(1, w(x) / (Z q(x))), w being what is left of p = probs[a] and Z
// its sum; else w' = max(w - Z q, 0), Z' = sum w'. Starting from w = p, Z = 1, all of
// these are w = max(p - c q, 0) for one number c: c = 0 at first and c' = c + Z, since
// max(max(p - c q, 0) - Z q, 0) = max(p - (c + Z) q, 0) for q >= 0. So a refusal costs
// one sum over the two rows, and nothing is stored. Without the draft's
// distribution w is p without the refused tokens, and Z one subtraction.
constexpr uint32_t kVerifyThreads = 1024;
constexpr uint32_t kMaxWidth = 1024;
constexpr uint32_t kNone = 0xFFFFFFFFu;
// Tokens that a block goes over at a time.
constexpr uint32_t kVerifyTokens = 4096;

struct VerifyArgs {
    const float *probs, *draft_probs;
    const uint32_t *tokens, *parents, *counts;
    const float *uniforms;
    uint32_t batch, width, n;
    uint32_t *path, *out_tokens, *accepted;
};

// The drafted nodes of one sequence, in LDS: parent (kNone for what is passed
// over), token, and the token's p and q at the parent.
struct Nodes {
    uint32_t parent[kMaxWidth], token[kMaxWidth], path[kMaxWidth];
    float p[kMaxWidth], q[kMaxWidth], u[kMaxWidth];
};

// Where a walk stands: at node `at`, its children up to `last` asked.
struct Walk {
    uint32_t at, last, took;
    double cut, mass;
};

__device__ __forceinline__ uint32_t load_nodes(const VerifyArgs &a, uint32_t b, Nodes &nodes) {
    const uint32_t count = a.counts ? min(a.counts[b], a.width) : a.width;
    const uint64_t first = static_cast<uint64_t>(b) * a.width;
    for (uint32_t i = threadIdx.x; i < count; i += blockDim.x) {
        uint32_t parent = i == 0 ? kNone : a.parents ? a.parents[first + i] : i - 1;
        const uint32_t x = a.tokens[first + i];
        if (parent >= i || x >= a.n) parent = kNone;
        nodes.parent[i] = parent;
        nodes.token[i] = x;
        nodes.u[i] = a.uniforms[first + i];
        nodes.p[i] = parent == kNone ? 0.0f : a.probs[(first + parent) * a.n + x];
        nodes.q[i] = parent == kNone || !a.draft_probs ? 1.0f : a.draft_probs[(first + parent) * a.n + x];
    }
    __syncthreads();
    return count;
}

// Goes on until a refusal needs the sum of what it leaves (true), or no child is
// left to ask. Every wavefront of a block does the same.
__device__ __forceinline__ bool walk(const VerifyArgs &a, Nodes &nodes, uint32_t count, Walk &w) {
#pragma clang fp contract(off)
    const uint32_t lane = threadIdx.x & 63u;
    for (;;) {
        // the next child of w.at
        uint32_t i = kNone;
        for (uint32_t base = (w.last + 1) & ~63u; base < count; base += 64) {
            const uint32_t k = base + lane;
            const uint64_t hit = __ballot(k > w.last && k < count && nodes.parent[min(k, count - 1)] == w.at);
            if (hit) {
                i = base + __builtin_ctzll(hit);
                break;
            }
        }
        if (i == kNone) return false;
        w.last = i;
        const double q = nodes.q[i], p = nodes.p[i];
        double left;
        if (a.draft_probs) {
            left = p - w.cut * q;
            left = left > 0 ? left : 0;
        } else {
            // a token that was refused here already has nothing left
            left = p > 0 ? p : 0;
            for (uint32_t base = 0; base < i; base += 64) {
                const uint32_t k = min(base + lane, i - 1);
                if (__ballot(nodes.parent[k] == w.at && nodes.token[k] == nodes.token[i])) left = 0;
            }
        }
        if (static_cast<double>(nodes.u[i]) * q * w.mass < left) {
            if (threadIdx.x == 0) nodes.path[w.took] = i;
            ++w.took;
            w.at = i;
            w.cut = 0, w.mass = 1;
        } else if (a.draft_probs) {
            w.cut += w.mass;
            return true;
        } else {
            w.mass -= left;
        }
    }
}

// What is left of token j: w's weight, or p's own (plain).
struct Weights {
    const float *p, *q;  // the node's rows; q null without the draft's distribution
    double cut;
    const uint32_t *gone;  // bits of the refused tokens from `base` on, null for none
    uint32_t base;
    __device__ __forceinline__ double operator()(uint32_t j) const {
#pragma clang fp contract(off)
        double v = p[j];
        if (q) v = v - cut * static_cast<double>(q[j]);
        if (gone && gone[(j - base) / 32] >> ((j - base) % 32) & 1u) v = 0;
        return v > 0 ? v : 0;
    }
};

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// One block per sequence: the walk, and each sum over the rows by the whole block.
__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(const VerifyArgs a) {
    __shared__ Nodes nodes;
    __shared__ uint32_t gone[kVerifyTokens / 32];
    __shared__ double part[kVerifyThreads / 64];
    __shared__ uint32_t best, lastpos;
    const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t count = load_nodes(a, b, nodes);
    const uint64_t first = static_cast<uint64_t>(b) * a.width;
    if (count == 0) {
        for (uint32_t i = tid; i < a.width; i += kVerifyThreads) a.path[first + i] = a.out_tokens[first + i] = kNone;
        if (tid == 0) a.accepted[b] = 0;
        return;
    }
    if (tid == 0) nodes.path[0] = 0;
    Walk w{0, 0, 1, 0.0, 1.0};
    Weights weight{};
    // marks the refused tokens among the next ones
    auto mark = [&](uint32_t base) {
        weight.base = base;
        if (!weight.gone) return;
        __syncthreads();
        for (uint32_t i = tid; i < kVerifyTokens / 32; i += kVerifyThreads) gone[i] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < count; i += kVerifyThreads)
            if (nodes.parent[i] == w.at && nodes.token[i] - base < kVerifyTokens)
                atomicOr(&gone[(nodes.token[i] - base) / 32], 1u << ((nodes.token[i] - base) % 32));
        __syncthreads();
    };
    auto rows = [&] {
        weight.p = a.probs + (first + w.at) * a.n;
        weight.q = a.draft_probs ? a.draft_probs + (first + w.at) * a.n : nullptr;
        weight.cut = w.cut;
    };
    auto total = [&] {
        double sum = 0;
        for (uint32_t base = 0; base < a.n; base += kVerifyTokens) {
            mark(base);
            for (uint32_t j = base + tid; j < min(base + kVerifyTokens, a.n); j += kVerifyThreads) sum += weight(j);
        }
        sum = wave_sum_f64(sum);
        __syncthreads();
        if (lane == 0) part[wave] = sum;
        __syncthreads();
        sum = 0;
        for (uint32_t i = 0; i < kVerifyThreads / 64; ++i) sum += part[i];
        return sum;
    };
    while (walk(a, nodes, count, w)) {
        rows();
        w.mass = total();
    }
    rows();
    if (!a.draft_probs) weight.gone = gone;
    double sum = total();
    if (!(sum > 0)) {
        weight.q = nullptr, weight.gone = nullptr, weight.cut = 0;
        sum = total();
    }
    const double target = static_cast<double>(nodes.u[0]) * sum;
    if (tid == 0) best = kNone, lastpos = 0;
    double before = 0;
    for (uint32_t base = 0; base < a.n; base += kVerifyTokens) {
        mark(base);
        constexpr uint32_t E = kVerifyTokens / kVerifyThreads;
        double v[E], own = 0;
        uint32_t any = 0;
        for (uint32_t e = 0; e < E; ++e) {
            const uint32_t j = base + tid * E + e;
            v[e] = j < a.n ? weight(j) : 0;
            own += v[e];
            if (v[e] > 0) any = j + 1;
        }
        double upto = own;
        for (int off = 1; off < 64; off <<= 1) {
            const double o = __shfl_up(upto, off, 64);
            if (lane >= static_cast<uint32_t>(off)) upto += o;
        }
        __syncthreads();
        if (lane == 63) part[wave] = upto;
        if (any) atomicMax(&lastpos, any);
        __syncthreads();
        double at = before + (upto - own);
        for (uint32_t i = 0; i < kVerifyThreads / 64; ++i) {
            if (i < wave) at += part[i];
            before += part[i];
        }
        for (uint32_t e = 0; e < E; ++e) {
            at += v[e];
            if (v[e] > 0 && at > target) {
                atomicMin(&best, base + tid * E + e);
                break;
            }
        }
        __syncthreads();
        if (best != kNone) break;
    }
    // rounding may leave the last running sum at the target
    const uint32_t next = best != kNone ? best : lastpos - 1;
    for (uint32_t i = tid; i < a.width; i += kVerifyThreads) {
        a.path[first + i] = i < w.took ? nodes.path[i] : kNone;
        a.out_tokens[first + i] = i + 1 < w.took ? nodes.token[nodes.path[i + 1]] : i + 1 == w.took ? next : kNone;
    }
    if (tid == 0) a.accepted[b] = w.took;
}

}  // namespace fh

using namespace fh;

extern "C" int fh_verify_draft_workspace(int64_t batch, int64_t width, int64_t n, uint64_t *bytes) {
    const char *fn = "fh_verify_draft_workspace";
    if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: bytes is null", fn);
    if (int rc = fh_check_dims(fn, {batch, width, n})) return rc;
    if (width < 1 || width > kMaxWidth)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: width %lld must be 1 to %u", fn, (long long)width, kMaxWidth);
    if (batch > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: batch %lld exceeds 65535", fn, (long long)batch);
    if (n < 1 || n > 0x7FFFFFFFll - kVerifyTokens)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: n %lld", fn, (long long)n);
    *bytes = 16;
    return FH_OK;
}

extern "C" int fh_verify_draft(fh_device *dev, const float *probs, const float *draft_probs, int64_t batch,
                               int64_t width, int64_t n, const uint32_t *tokens, const uint32_t *parents,
                               const uint32_t *counts, const float *uniforms, void *workspace, uint64_t workspace_bytes,
                               uint32_t *path, uint32_t *out_tokens, uint32_t *accepted) {
    const char *fn = "fh_verify_draft";
    if (int rc = check_usable(dev, fn)) return rc;
    uint64_t need = 0;
    if (int rc = fh_verify_draft_workspace(batch, width, n, &need)) return rc;
    if (batch == 0) return FH_OK;
    if (workspace_bytes < need)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: workspace of %llu bytes, %llu needed", fn,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", fn);
    const uint64_t nodes = static_cast<uint64_t>(batch) * width * 4, each = static_cast<uint64_t>(batch) * 4;
    uint64_t rows;
    if (int rc = size_product(fn, "probs", {nodes, static_cast<uint64_t>(n)}, &rows)) return rc;
    struct Operand {
        const char *what;
        const void *ptr;
        uint64_t bytes;
        bool optional;
    };
    const Operand in[] = {{"probs", probs, rows, false},     {"draft_probs", draft_probs, rows, true},
                          {"tokens", tokens, nodes, false},  {"parents", parents, nodes, true},
                          {"counts", counts, each, true},    {"uniforms", uniforms, nodes, false}};
    const Operand out[] = {{"path", path, nodes, false},
                           {"out_tokens", out_tokens, nodes, false},
                           {"accepted", accepted, each, false},
                           {"workspace", workspace, need, false}};
    auto check = [&](const Operand &o) {
        if (o.ptr == nullptr && o.optional) return static_cast<int>(FH_OK);
        if (reinterpret_cast<uintptr_t>(o.ptr) % 4 != 0)
            return fail(FH_ERR_INVALID_ARGUMENT, "%s: %s must be 4-byte aligned", fn, o.what);
        return check_range(dev, o.ptr, o.bytes, fn, o.what);
    };
    for (const Operand &o : in)
        if (int rc = check(o)) return rc;
    for (const Operand &o : out) {
        if (int rc = check(o)) return rc;
        for (const Operand &i : in)
            if (i.ptr)
                if (int rc = refuse_overlap(fn, o.what, o.ptr, o.bytes, i.what, i.ptr, i.bytes)) return rc;
        for (const Operand &i : out)
            if (&i != &o)
                if (int rc = refuse_overlap(fn, o.what, o.ptr, o.bytes, i.what, i.ptr, i.bytes)) return rc;
    }
    if (int rc = set_current(dev, fn)) return rc;
    const VerifyArgs a{probs,
                       draft_probs,
                       tokens,
                       parents,
                       counts,
                       uniforms,
                       static_cast<uint32_t>(batch),
                       static_cast<uint32_t>(width),
                       static_cast<uint32_t>(n),
                       path,
                       out_tokens,
                       accepted};
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(verify_kernel, dim3(static_cast<uint32_t>(batch)), dim3(kVerifyThreads), 0, dev->stream, a);
    });
}
