// Which drafted tokens the target's distributions accept (fh_verify_draft).
#include <algorithm>

#include "serving_checks.hpp"

namespace fh {

// The mathematics. At node a a child's token x, drawn from q, is accepted with
// probability min(1, w(x) / (Z q(x))), w being what is left of p = probs[a] and Z
// its sum; else w' = max(w - Z q, 0), Z' = sum w'. Starting from w = p, Z = 1, all of
// these are w = max(p - c q, 0) for one number c: c = 0 at first and c' = c + Z, since
// max(max(p - c q, 0) - Z q, 0) = max(p - (c + Z) q, 0) for q >= 0. So a refusal costs
// one sum over the two rows, and nothing is stored. Without the draft's
// distribution w is p without the refused tokens, and Z one subtraction.
//
// The walk down the tree needs single entries of the rows, which are loaded for all
// nodes at once, up to the first refusal that has to be summed up: at the only
// child of its parent (a chain), that sum is of what the next token is drawn
// from. So every block of a first launch walks that far for itself and adds up one
// piece of the rows that count then, and only those rows are read; a second
// launch's block per sequence goes on from there, finds the piece that the
// token lies in and reads that. Further refusals (trees with the draft's
// distributions) are summed by that block alone, those behind the last one twice. Bound by memory: 64 chains of 6
// over 128256 tokens take 21.8 us (15.0, at 4.4 TB/s, and 6.8 of the launches; 20.0 without the draft's
// distributions), one 10.5 us. Trees with the draft's distributions are bound by that one block's reads: 8 of 32
// nodes 62 us, one of 64 33, by the refusals; without them 8 of 32 13.5 us.
constexpr uint32_t kVerifyThreads = 256;
constexpr uint32_t kWavesMost = 16;  // of a block that goes on with a walk
constexpr uint32_t kMaxWidth = 1024;
constexpr uint32_t kNone = 0xFFFFFFFFu;
// Tokens that a block goes over at a time, and the shortest piece
// of a row and the blocks that the first launch aims for before pieces get longer.
constexpr uint32_t kVerifyTokens = 4096;
constexpr uint32_t kLeastPiece = 1024;
// (16 chains with 2048 blocks 14.0 us, 12.8 with these; 1 or 64 the same.)
constexpr uint32_t kVerifyBlocks = 1024;
// Pieces of a row at most.
constexpr uint32_t kMaxPieces = 1024;

struct VerifyArgs {
    const float *probs, *draft_probs;
    const uint32_t *tokens, *parents, *counts;
    const float *uniforms;
    uint32_t batch, width, n, piece, pieces;
    uint32_t *path, *out_tokens, *accepted;
    double *sums;        // [batch][pieces] of the rows that the first launch stopped at
    struct Walk *walks;  // [batch]
};

// The drafted nodes of one sequence, in LDS: parent (kNone for what is passed
// over), token, and the token's p and q at the parent.
// The launch gives it room for `width` of them: 64 take 1.5 KB, the most 24 KB, which
// let only six blocks onto a CU.
struct Nodes {
    uint32_t *parent, *token, *path;
    float *p, *q, *u;
    __device__ __forceinline__ explicit Nodes(uint32_t width) {
        extern __shared__ uint32_t room[];
        parent = room, token = room + width, path = room + 2 * width;
        p = reinterpret_cast<float *>(room + 3 * width), q = p + width, u = q + width;
    }
    static uint32_t bytes(uint32_t width) { return 24 * width; }
};

// Where a walk stands: at node `at`, its children up to `last` asked.
struct Walk {
    uint32_t at, last, took;
    uint32_t open;  // a child is left to ask, once the sum is known
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

// The next child of w.at to ask, kNone for none.
__device__ __forceinline__ uint32_t next_child(const Nodes &nodes, uint32_t count, const Walk &w) {
    for (uint32_t base = (w.last + 1) & ~63u; base < count; base += 64) {
        const uint32_t k = base + (threadIdx.x & 63u);
        const uint64_t hit = __ballot(k > w.last && k < count && nodes.parent[min(k, count - 1)] == w.at);
        if (hit) return base + __builtin_ctzll(hit);
    }
    return kNone;
}

// Goes on until a refusal needs the sum of what it leaves (true), or no child is
// left to ask. Every wavefront of a block does the same.
__device__ __forceinline__ bool walk(const VerifyArgs &a, Nodes &nodes, uint32_t count, Walk &w) {
#pragma clang fp contract(off)
    const uint32_t lane = threadIdx.x & 63u;
    for (;;) {
        const uint32_t i = next_child(nodes, count, w);
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

// What is left of the tokens behind a node.
struct Weights {
    const float *p, *q;  // the node's rows; q null without the draft's distribution
    double cut;
    const uint32_t *gone;  // bits of the refused tokens from `base` on, null for none
    uint32_t n, base;
    bool wide;  // rows begin at 16-byte boundaries less `before` tokens, p's and q's the same
    uint32_t before;

    __device__ __forceinline__ double of(float pj, float qj, uint32_t j) const {
#pragma clang fp contract(off)
        double v = pj;
        if (q) v = v - cut * static_cast<double>(qj);
        if (gone && gone[(j - base) / 32] >> ((j - base) % 32) & 1u) v = 0;
        return v > 0 ? v : 0;
    }
    // The weights of tokens j0 .. j0 + 3 (0 outside the row); j0 + before is a multiple of 4.
    __device__ __forceinline__ void four(int32_t j0, double (&w)[4]) const {
        float x[4], y[4] = {0, 0, 0, 0};
        if (wide && j0 >= 0 && j0 + 4 <= static_cast<int32_t>(n)) {
            const float4 a = *reinterpret_cast<const float4 *>(p + j0);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
            if (q) {
                const float4 b = *reinterpret_cast<const float4 *>(q + j0);
                y[0] = b.x, y[1] = b.y, y[2] = b.z, y[3] = b.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = j0 + e >= 0 && j0 + e < static_cast<int32_t>(n);
                x[e] = in ? p[j0 + e] : 0.0f;
                if (q) y[e] = in ? q[j0 + e] : 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = j0 + e >= 0 && j0 + e < static_cast<int32_t>(n) ? of(x[e], y[e], j0 + e) : 0;
    }
    // The sum of K times four tokens' weights, j0 + 256 k on, up to token hi. Where the
    // wavefront's are all whole, with every load on its way before the first is used.
    template <uint32_t K>
    __device__ __forceinline__ double sum(int32_t j0, int32_t hi, bool all_whole) const {
        double all = 0;
        if (wide && all_whole) {
            float4 x[K], y[K];
#pragma unroll
            for (uint32_t k = 0; k < K; ++k) {
                x[k] = *reinterpret_cast<const float4 *>(p + j0 + k * 256);
                y[k] = q ? *reinterpret_cast<const float4 *>(q + j0 + k * 256) : make_float4(0, 0, 0, 0);
            }
#pragma unroll
            for (uint32_t k = 0; k < K; ++k) {
                const uint32_t j = j0 + k * 256;
                all += (of(x[k].x, y[k].x, j) + of(x[k].y, y[k].y, j + 1)) +
                       (of(x[k].z, y[k].z, j + 2) + of(x[k].w, y[k].w, j + 3));
            }
        } else {
            for (uint32_t k = 0; k < K; ++k) {
                const int32_t j = j0 + static_cast<int32_t>(k) * 256;
                double w[4] = {0, 0, 0, 0};
                if (j < hi) four(j, w);
                all += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }
        return all;
    }
};

// The rows behind w.at.
__device__ __forceinline__ Weights weights_of(const VerifyArgs &a, uint32_t b, const Walk &w) {
    const uint64_t row = (static_cast<uint64_t>(b) * a.width + w.at) * a.n;
    Weights x{};
    x.p = a.probs + row;
    x.q = a.draft_probs ? a.draft_probs + row : nullptr;
    x.cut = w.cut;
    x.n = a.n;
    x.before = (reinterpret_cast<uintptr_t>(x.p) & 15u) / 4;
    x.wide = !x.q || (reinterpret_cast<uintptr_t>(x.q) & 15u) / 4 == x.before;
    return x;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int off = 32; off; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

struct Scratch {
    static constexpr uint32_t kWaves = kVerifyThreads / 64;
    double part[kWavesMost];
    uint32_t gone[kVerifyTokens / 32];
    // of each wavefront: its first value past the target, the running sum before that
    // value's thread, and its last positive value
    uint32_t first[kWaves], last[kWaves];
    double from[kWaves];
};

// The block's sum, the same in every thread.
__device__ __forceinline__ double block_sum(double v, Scratch &s, uint32_t waves) {
    v = wave_sum_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0) s.part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (uint32_t i = 0; i < waves; ++i) v += s.part[i];
    return v;
}

// Marks the refused children's tokens among kVerifyTokens from lo - x.before on.
__device__ __forceinline__ void mark(Weights &x, uint32_t lo, const Nodes &nodes, uint32_t count, uint32_t at,
                                     Scratch &s) {
    if (!x.gone) return;
    x.base = lo - x.before;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kVerifyTokens / 32; i += kVerifyThreads) s.gone[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < count; i += kVerifyThreads) {
        const uint32_t bit = nodes.token[i] - x.base;
        if (nodes.parent[i] == at && bit < kVerifyTokens) atomicOr(&s.gone[bit / 32], 1u << (bit % 32));
    }
    __syncthreads();
}

// The sum of the weights of tokens lo - x.before .. hi - x.before - 1 of a row by a wavefront, where
// none is marked. hi is at most n + x.before.
__device__ __forceinline__ double wave_sum_of(const Weights &x, uint64_t lo, uint64_t hi) {
    constexpr uint32_t K = 4;
    double sum = 0;
    for (uint64_t base = lo; base < hi; base += K * 256) {
        const int32_t j0 = static_cast<int32_t>(base) - static_cast<int32_t>(x.before);
        sum += x.sum<K>(j0 + static_cast<int32_t>(threadIdx.x & 63u) * 4,
                        static_cast<int32_t>(hi) - static_cast<int32_t>(x.before), j0 >= 0 && base + K * 256 <= hi);
    }
    return wave_sum_f64(sum);
}

// Block (piece, sequence): the walk to the first sum, and this piece of it.
__global__ __launch_bounds__(kVerifyThreads) void verify_walk_kernel(const VerifyArgs a) {
    Nodes nodes(a.width);
    __shared__ Scratch scratch;
    const uint32_t b = blockIdx.y, tid = threadIdx.x;
    const uint32_t count = load_nodes(a, b, nodes);
    const uint64_t first = static_cast<uint64_t>(b) * a.width;
    if (count == 0) {
        if (blockIdx.x) return;
        for (uint32_t i = tid; i < a.width; i += kVerifyThreads) a.path[first + i] = a.out_tokens[first + i] = kNone;
        if (tid == 0) a.accepted[b] = 0, a.walks[b] = Walk{0, 0, 0, 0, 0.0, 0.0};
        return;
    }
    if (tid == 0) nodes.path[0] = 0;
    Walk w{0, 0, 1, 0, 0.0, 1.0};
    w.open = walk(a, nodes, count, w) && next_child(nodes, count, w) != kNone;
    Weights x = weights_of(a, b, w);
    if (!a.draft_probs) x.gone = scratch.gone;
    const uint64_t lo = static_cast<uint64_t>(blockIdx.x) * a.piece;
    const uint64_t hi = min(lo + a.piece, static_cast<uint64_t>(a.n) + x.before);
    double sum = 0;
    for (uint64_t base = lo; base < hi; base += kVerifyTokens) {
        mark(x, static_cast<uint32_t>(base), nodes, count, w.at, scratch);
        constexpr uint32_t K = kVerifyTokens / (4 * kVerifyThreads);
        double v[K][4];
#pragma unroll
        for (uint32_t k = 0; k < K; ++k) {
            const uint64_t j = base + (k * kVerifyThreads + tid) * 4;
            v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0;
            if (j < hi) x.four(static_cast<int32_t>(j) - static_cast<int32_t>(x.before), v[k]);
        }
#pragma unroll
        for (uint32_t k = 0; k < K; ++k) sum += (v[k][0] + v[k][1]) + (v[k][2] + v[k][3]);
    }
    sum = block_sum(sum, scratch, Scratch::kWaves);
    if (tid == 0) a.sums[static_cast<uint64_t>(b) * a.pieces + blockIdx.x] = sum;
    if (blockIdx.x) return;
    __syncthreads();
    if (tid == 0) a.walks[b] = w, a.accepted[b] = w.took;
    for (uint32_t i = tid; i < a.width; i += kVerifyThreads) {
        a.path[first + i] = i < w.took ? nodes.path[i] : kNone;
        a.out_tokens[first + i] = i + 1 < w.took ? nodes.token[nodes.path[i + 1]] : kNone;
    }
}

// Block (sequence): what is left of the walk, by all its wavefronts, and the token behind
// it, by four of them (more only wait for each other there: 5.4 us with four, 9.0 with
// sixteen; 8 sequences' trees of 32 nodes, the same ones, took 476 us with four, 81 with sixteen).
__global__ __launch_bounds__(64 * kWavesMost) void verify_draw_kernel(const VerifyArgs a) {
    Nodes nodes(a.width);
    __shared__ Scratch scratch;
    __shared__ double sums[kMaxPieces];
    const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint64_t first = static_cast<uint64_t>(b) * a.width;
    Walk w = a.walks[b];
    const double u = a.uniforms[first];
    uint32_t waves = w.open ? blockDim.x / 64 : Scratch::kWaves;
    if (w.took == 0 || wave >= waves) return;  // no node, or nothing for this wavefront
    for (uint32_t i = tid; i < a.pieces; i += 64 * waves) sums[i] = a.sums[static_cast<uint64_t>(b) * a.pieces + i];
    const uint32_t before_took = w.took;
    // nodes: where children are left to ask, or refused tokens to leave out
    uint32_t count = 0;
    if (w.open || !a.draft_probs) count = load_nodes(a, b, nodes);
    Weights x = weights_of(a, b, w);
    auto total = [&] {
        double sum = 0;
        __syncthreads();
        for (uint32_t i = tid; i < a.pieces; i += 64 * waves) sum += sums[i];
        return block_sum(sum, scratch, waves);
    };
    // the pieces' sums anew, a wavefront's after one another
    auto pieces = [&] {
        __syncthreads();
        for (uint32_t i = wave; i < a.pieces; i += waves) {
            const uint64_t lo = static_cast<uint64_t>(i) * a.piece;
            const uint64_t hi = min(lo + a.piece, static_cast<uint64_t>(a.n) + x.before);
            const double sum = lo < hi ? wave_sum_of(x, lo, hi) : 0;
            if (lane == 0) sums[i] = sum;
        }
        __syncthreads();
    };
    if (!a.draft_probs) x.gone = scratch.gone;
    double sum = total();
    if (w.open) {
        do {
            w.mass = sum;
            // a refusal (or no child left) has the rows at hand summed up again
            const bool more = walk(a, nodes, count, w);
            x = weights_of(a, b, w);
            pieces();
            sum = total();
            w.open = more;
        } while (w.open);
        for (uint32_t i = before_took + tid; i < w.took; i += 64 * waves) {
            a.path[first + i] = nodes.path[i];
            a.out_tokens[first + i - 1] = nodes.token[nodes.path[i]];
        }
        if (tid == 0) a.accepted[b] = w.took;
        waves = Scratch::kWaves;
        __syncthreads();  // the sum is read
        if (wave >= waves) return;
    }
    if (!(sum > 0)) {  // nothing is left: p itself
        x.q = nullptr, x.gone = nullptr, x.cut = 0;
        pieces();
        sum = total();
    }
    // the piece whose running sum passes the target, then the token in it
    const double target = u * sum;
    // best: the first of the block's values (thread by thread, E of each) whose running sum from
    // `from` passes the target, kNone if none does; last: one more than the last that is positive.
    // `from` moves on, to the running sum before best's thread once there is one. The wavefronts'
    // results are picked by ballots: atomics of all threads on one place took 4 us.
    uint32_t best = kNone, last = 0;
    double from = 0;
    auto find = [&](auto &v, uint32_t base) {
        constexpr uint32_t E = sizeof(v) / sizeof(double);
        double own = 0;
        uint32_t any = 0;
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
            own += v[e];
            if (v[e] > 0) any = base + tid * E + e + 1;
        }
        double upto = own;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const double o = __shfl_up(upto, off, 64);
            if (lane >= static_cast<uint32_t>(off)) upto += o;
        }
        __syncthreads();
        if (lane == 63) scratch.part[wave] = upto;
        if (lane == 0) scratch.first[wave] = kNone, scratch.last[wave] = 0;
        __syncthreads();
        double at = from + (upto - own);
        for (uint32_t i = 0; i < kVerifyThreads / 64; ++i) {
            if (i < wave) at += scratch.part[i];
            from += scratch.part[i];
        }
        const double start = at;
        uint32_t mine = kNone;
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) {
            at += v[e];
            if (v[e] > 0 && at > target && mine == kNone) mine = base + tid * E + e;
        }
        const uint64_t past = __ballot(mine != kNone), some = __ballot(any != 0);
        if (past && lane == __builtin_ctzll(past)) scratch.first[wave] = mine, scratch.from[wave] = start;
        if (some && lane == 63u - __builtin_clzll(some)) scratch.last[wave] = any;
        __syncthreads();
        for (uint32_t i = kVerifyThreads / 64; i-- > 0;) {
            if (scratch.first[i] != kNone) best = scratch.first[i], from = scratch.from[i];
            last = max(last, scratch.last[i]);
        }
    };
    for (uint32_t base = 0; base < a.pieces && best == kNone; base += kVerifyThreads) {
        double v[1] = {base + tid < a.pieces ? sums[base + tid] : 0.0};
        find(v, base);
    }
    // (rounding may leave the last running sum at the target: the last piece and token with a weight)
    const uint32_t piece = best != kNone ? best : last - 1;
    uint32_t next = kNone;
    if (piece != kNone) {
        if (best == kNone) from -= sums[piece];
        best = kNone, last = 0;
        const uint64_t lo = static_cast<uint64_t>(piece) * a.piece;
        const uint64_t hi = min(lo + a.piece, static_cast<uint64_t>(a.n) + x.before);
        for (uint64_t base = lo; base < hi && best == kNone; base += kVerifyTokens) {
            mark(x, static_cast<uint32_t>(base), nodes, count, w.at, scratch);
            static_assert(kVerifyTokens == 16 * kVerifyThreads);
            double v[16];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {  // 16 tokens in a row
                double w4[4] = {0, 0, 0, 0};
                const uint64_t j = base + tid * 16 + k * 4;
                if (j < hi) x.four(static_cast<int32_t>(j) - static_cast<int32_t>(x.before), w4);
                v[k * 4] = w4[0], v[k * 4 + 1] = w4[1], v[k * 4 + 2] = w4[2], v[k * 4 + 3] = w4[3];
            }
            find(v, static_cast<uint32_t>(base));
        }
        if (best != kNone || last) next = (best != kNone ? best : last - 1) - x.before;
    }
    if (tid == 0) a.out_tokens[first + w.took - 1] = next;
}

}  // namespace fh

using namespace fh;

namespace {

// Tokens of a row's piece for these sizes, and pieces of a row (which may begin up to three tokens before it).
uint32_t piece_of(int64_t batch, int64_t n) {
    uint64_t piece = kLeastPiece;
    while (piece < kVerifyTokens && batch * ((n + piece - 1) / piece) > kVerifyBlocks) piece *= 2;
    while ((n + 3 + piece - 1) / piece > kMaxPieces) piece *= 2;
    return static_cast<uint32_t>(piece);
}

uint64_t pieces_of(int64_t n, uint32_t piece) { return (static_cast<uint64_t>(n) + 3 + piece - 1) / piece; }

}  // namespace

extern "C" int fh_verify_draft_workspace(int64_t batch, int64_t width, int64_t n, uint64_t *bytes) {
    const char *fn = "fh_verify_draft_workspace";
    if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: bytes is null", fn);
    if (int rc = fh_check_dims(fn, {batch, width, n})) return rc;
    if (width < 1 || width > kMaxWidth)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: width %lld must be 1 to %u", fn, (long long)width, kMaxWidth);
    if (batch > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: batch %lld exceeds 65535", fn, (long long)batch);
    if (n < 1 || n > 0x7FFFFFFFll - kVerifyTokens)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: n %lld", fn, (long long)n);
    // pieces get longer where there are more than kVerifyBlocks of them, not counting a row's last four tokens
    *bytes = static_cast<uint64_t>(batch) * sizeof(Walk) + 16 +
             std::max<uint64_t>(kVerifyBlocks + kMaxPieces + batch, batch * pieces_of(n, piece_of(65535, n))) * 8;
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
    const uint32_t piece = piece_of(batch, n);
    const VerifyArgs a{probs,
                       draft_probs,
                       tokens,
                       parents,
                       counts,
                       uniforms,
                       static_cast<uint32_t>(batch),
                       static_cast<uint32_t>(width),
                       static_cast<uint32_t>(n),
                       piece,
                       static_cast<uint32_t>(pieces_of(n, piece)),
                       path,
                       out_tokens,
                       accepted,
                       reinterpret_cast<double *>(static_cast<char *>(workspace) + batch * sizeof(Walk)),
                       static_cast<Walk *>(workspace)};
    const dim3 grid(a.pieces, a.batch);
    if (int rc = dispatch(dev, fn, [&] {
            hipLaunchKernelGGL(verify_walk_kernel, grid, dim3(kVerifyThreads), Nodes::bytes(a.width), dev->stream, a);
        }))
        return rc;
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL(verify_draw_kernel, dim3(a.batch), dim3(a.draft_probs ? 64 * kWavesMost : kVerifyThreads), Nodes::bytes(a.width), dev->stream, a);
    });
}
