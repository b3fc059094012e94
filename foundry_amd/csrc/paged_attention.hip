// Attention of one new token per sequence over a paged cache
// (fh_paged_attention).
#include <algorithm>
#include <tuple>

#include "paged_cache.hpp"

namespace fh {

// The mathematics: one pass over a sequence's keys with the running maximum m,
// sum l and weighted values o of each query head,
//   m' = max(m, s), l' = l e^(m - m') + e^(s - m'), o' = o e^(m - m') + e^(s - m') v,
// joined over disjoint key ranges by the same rule. Exponentials are taken as
// powers of two, their exponents scaled by log2 e after the maximum is taken off:
// any finite score has a finite weight.
//
// The split: a block of four wavefronts takes a part of the batch's keys (whole
// steps of kStepKeys) for one KV head and up to 8 of the query heads that share
// it; of each sequence in its part every wavefront streams a quarter of the
// keys, 32 at a time, and the four join in LDS. The parts are laid out from
// the positions on the device (see Layout), so the same launch serves one long
// context and a ragged batch, and may be captured.
//
// Per 32 keys the scores are S^T = K Q^T on the matrix cores
// (v_mfma_f32_16x16x32_bf16, 16 keys x 16 columns): a lane ends up with its
// column's scores of keys 4 q .. 4 q + 3 (q = lane / 16) of both 16-key groups.
// Those eight probabilities are the fragment that O^T = V^T P^T needs of that
// lane if its keys are numbered so, so P never leaves its lane; V's rows, read
// as they lie, become V^T fragments by byte permutes within a lane. The 16
// columns are 8 heads twice: columns 0..7 hold the probabilities rounded to
// bf16, columns 8..15 what that rounding lost, so that P V has 16 bits of P at
// the cost of none (the columns would idle). What 16 bits lose, 2^-16 of a term,
// is far below the half step of 2^-8 that bf16 V is off by itself; p's sum, the
// maximum and all sums of values are fp32.
//
// Bound by memory: K and V come once, with the nontemporal hint (131077 keys of
// 8 KV heads of 128: 104 us without, 90 with), the next tile's K in flight behind
// a tile's softmax, its V behind the next one's. 131077 keys (537 MB) take 92 us
// with the join (5.9 TB/s; the parts alone 89, 6.0 TB/s), 96 ragged sequences of
// 17 to 16384 keys (949 MB) 161 (5.9 TB/s; the parts 152), 8 of 1900 to 4111 (97
// MB) 24 (the parts 20, 4.8 TB/s). 8 KV heads of 64: 48 us (268 MB, 5.6 TB/s), 89
// (480 MB, 5.4), 16.4 (48 MB); one of 256 with 8 heads: 53 (134 MB, 2.5 TB/s; the
// parts 38, the join's 8 blocks 15), 63 (241 MB, 3.8), 15.6 (24 MB).
constexpr uint32_t kPagedThreads = 256;
constexpr uint32_t kStepKeys = 128;
constexpr uint32_t kHeadTile = 8;
// Blocks of a launch: with heads of 128 what the GPU holds at once, 2 per CU (of
// 64 it holds 4, of 256 one; their number was not measured apart). 8 sequences, 96,
// one of 131077 keys of 128: 24.0, 161, 91.9 us with 512; 29.0, 169, 92.3 with 768.
constexpr uint32_t kPartBlocks = 512;
// Tables of so few positions (times head_dim) take one block per sequence, of 8
// wavefronts (4 at head_dim 256), and no join: one launch. One sequence of 500
// keys of 128: 8.5 us against 10.1 split, of 1000: 14.2 against 10.7; of 1000
// keys of 64: 9.1 against 9.2, of 1500: 11.3 against 9.2; of 300 of 256: 11.2
// against 12.3, of 500: 13.3 against 12.6. 48 sequences: even up to 4000 keys. The
// table's width decides, not the positions, which the host does not know: 300 keys
// of 128 take 8.0 us, behind a table of 8000 pages 12.3.
constexpr uint32_t kWholeElements = 65536;
// Larger batches take one part per sequence, as every block would lay them all out:
// for 1024 sequences (one of 131077 keys, the others of 100) that makes 0.2 of the
// two launches' 0.42 ms. Unsplit, as with 1025, they take 1.23 ms.
constexpr uint32_t kPlanBatch = 1024;

typedef __attribute__((ext_vector_type(8))) __bf16 pa_bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float pa_f32x4_t;

__device__ __forceinline__ pa_f32x4_t pa_mfma(uint4 a, uint4 b, pa_f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8_t, a),
                                                   __builtin_bit_cast(pa_bf16x8_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ float pa_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }

struct PagedArgs {
    const uint16_t *q, *k_pages, *v_pages;
    const uint32_t *page_table, *positions;
    uint32_t batch, n_heads, n_kv, n_pages, page_size, max_pages;
    uint32_t want_parts;  // parts of one (KV head, head tile); 0: a block per sequence
    float scale;
    float *records;
    uint16_t *out;
};

__device__ __forceinline__ uint32_t steps_of(const PagedArgs &a, uint32_t b) {
    const uint32_t pos = a.positions[b];
    return pos < a.max_pages * a.page_size ? pos / kStepKeys + 1 : 0;
}

__device__ __forceinline__ uint32_t scan_wave(uint32_t v, uint32_t lane) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_up(v, off, 64);
        if (lane >= static_cast<uint32_t>(off)) v += o;
    }
    return v;
}

// The steps of all sequences, in order, are cut into equal parts, one per
// block of a (KV head, head tile): part x takes steps x * size .. of them,
// which may be the end of one sequence, whole ones, and the start of another.
// Such a piece of sequence b in part x leaves record x + b: no two pieces
// share one (a later piece has a larger x or b), and those of one sequence
// follow each other. Every wavefront works the layout out for itself from the
// positions, 64 sequences at a time.
struct Layout {
    uint32_t size;   // steps of a part
    uint32_t b0;     // first sequence of the 64 at hand
    uint32_t mine;   // lane's sequence's steps
    uint32_t upto;   // and the batch's steps up to its end
};

__device__ __forceinline__ void layout_at(const PagedArgs &a, Layout &y, uint32_t b0, uint32_t before, uint32_t lane) {
    y.b0 = b0;
    y.mine = b0 + lane < a.batch ? steps_of(a, b0 + lane) : 0;
    y.upto = before + scan_wave(y.mine, lane);
}

__device__ __forceinline__ Layout layout_of(const PagedArgs &a, uint32_t lane) {
    Layout y;
    uint32_t total = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
        layout_at(a, y, b0, total, lane);
        total = __builtin_amdgcn_readlane(y.upto, 63);
    }
    y.size = max(1u, (total + a.want_parts - 1) / a.want_parts);
    if (a.batch > 64) layout_at(a, y, 0, 0, lane);
    return y;
}

// Moves to the sequence that holds step `at` of the batch and returns it, its
// steps in n and the steps before it in `start`; ~0 behind the last one.
__device__ __forceinline__ uint32_t sequence_of(const PagedArgs &a, Layout &y, uint32_t at, uint32_t lane, uint32_t &n,
                                                uint32_t &start) {
    for (;;) {
        const uint64_t hit = __ballot(at < y.upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            n = __builtin_amdgcn_readlane(y.mine, l);
            start = __builtin_amdgcn_readlane(y.upto, l) - n;
            return y.b0 + l;
        }
        if (y.b0 + 64 >= a.batch) return ~0u;
        layout_at(a, y, y.b0 + 64, __builtin_amdgcn_readlane(y.upto, 63), lane);
    }
}

// A record: what a part leaves to be joined, [8 heads][HD] weighted values,
// then m, l and (in the third row) whether any key was there, of each head.
template <int HD>
constexpr uint32_t record_floats() { return kHeadTile * HD + 3 * kHeadTile; }

template <int HD, int W>
__global__ __launch_bounds__(64 * W, HD == 256 ? 1 : 2) void paged_part_kernel(const PagedArgs a) {
    constexpr int KC = HD / 32;                    // score products per 16 keys
    constexpr int VP = HD == 64 ? 1 : HD / 128;    // pieces of a lane's V row
    constexpr int PD = HD == 64 ? 4 : 8;           // dims of a piece
    constexpr int VT = VP * PD;                    // products per 32 keys
    __shared__ float part_o[W][kHeadTile][HD + 4];
    __shared__ float part_ml[W][3][kHeadTile];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, c = lane & 15u, q = lane >> 4;
    const uint32_t group = a.n_heads / a.n_kv, tiles = (group + kHeadTile - 1) / kHeadTile;
    const uint32_t kv = blockIdx.y / tiles, head0 = (blockIdx.y % tiles) * kHeadTile;
    const uint32_t heads = min(kHeadTile, group - head0);  // this block's, from kv * group + head0
    const uint32_t groups_pp = a.page_size / 16;
    Layout y;
    uint32_t at = 0, end = 1;
    if (a.want_parts) {
        y = layout_of(a, lane);
        at = blockIdx.x * y.size;
        end = at + y.size;
    }
    while (at < end) {
        // the next piece: `count` steps from `first` of sequence seq
        uint32_t seq = blockIdx.x, first = 0, count, whole = 1;
        if (a.want_parts) {
            uint32_t n, start;
            seq = sequence_of(a, y, at, lane, n, start);
            if (seq == ~0u) break;
            first = at - start;
            count = min(n - first, end - at);
            whole = count == n;
            at += count;
        } else {
            count = steps_of(a, seq);
            at = end;
        }
        const uint64_t row0 = (static_cast<uint64_t>(seq) * a.n_heads + kv * group + head0) * HD;
        const uint32_t keys = count ? a.positions[seq] + 1 : 0;
        // this wavefront's keys: from .. to, in tiles of 32
        const uint32_t share = (count * (kStepKeys / 32) + W - 1) / W * 32;
        const uint32_t from = first * kStepKeys + wave * share;
        const uint32_t to = min(from + share, min(keys, (first + count) * kStepKeys));
        const uint32_t n_tiles = from < to ? (to - from + 31) / 32 : 0;

        uint4 qf[KC];
        const uint16_t *qrow = a.q + row0 + min(c & 7u, heads - 1) * HD + q * 8;
#pragma unroll
        for (int s = 0; s < KC; ++s) qf[s] = *reinterpret_cast<const uint4 *>(qrow + s * 32);

        pa_f32x4_t acc[VT];
#pragma unroll
        for (int t = 0; t < VT; ++t) acc[t] = pa_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        bool any = false;

        for (uint32_t t0 = 0; t0 < n_tiles; t0 += 32) {
            // lane i: where the i-th 16-key group of the next 32 tiles lies, in
            // groups from the pools' start; ~0 for none (past the keys, no page)
            const uint32_t g = from / 16 + t0 * 2 + lane;
            uint32_t where = ~0u;
            if (g * 16 < to) {
                const uint32_t pi = g / groups_pp;
                const uint32_t page = a.page_table[static_cast<uint64_t>(seq) * a.max_pages + pi];
                if (page < a.n_pages) where = (page * a.n_kv + kv) * groups_pp + (g - pi * groups_pp);
            }
            const uint32_t batch_tiles = min(32u, n_tiles - t0);
            uint4 kf[2][KC];
            uint4 vf[8][VP];
            // a missing group reads the pool's first group, whose scores are left out
            auto group_at = [&](uint32_t t, int half) {
                const uint32_t w = __builtin_amdgcn_readlane(where, t * 2 + half);
                return static_cast<uint64_t>(w == ~0u ? 0u : w) * (16 * HD);
            };
            auto load_k = [&](uint32_t t) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint16_t *src = a.k_pages + group_at(t, h) + c * 32 + q * 8;
#pragma unroll
                    for (int s = 0; s < KC; ++s)
                        kf[h][s] = load_stream16(reinterpret_cast<const uint4 *>(src + s * 512));
                }
            };
            auto load_v = [&](uint32_t t) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint16_t *src = a.v_pages + group_at(t, i / 4) + (q * 4 + i % 4) * HD + c * PD;
#pragma unroll
                    for (int u = 0; u < VP; ++u) {
                        if constexpr (HD == 64) {
                            const uint2 v = load_stream8(reinterpret_cast<const uint2 *>(src));
                            vf[i][u] = make_uint4(v.x, v.y, 0, 0);
                        } else {
                            vf[i][u] = load_stream16(reinterpret_cast<const uint4 *>(src + u * 128));
                        }
                    }
                }
            };
            pa_f32x4_t s0, s1;
            auto scores = [&] {
                s0 = s1 = pa_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < KC; ++s) {
                    s0 = pa_mfma(kf[0][s], qf[s], s0);
                    s1 = pa_mfma(kf[1][s], qf[s], s1);
                }
            };
            uint4 pf;
            auto weigh = [&](uint32_t t) {
                float s[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = s0[i] * a.scale, s[4 + i] = s1[i] * a.scale;
                const uint32_t w0 = __builtin_amdgcn_readlane(where, t * 2);
                const uint32_t w1 = __builtin_amdgcn_readlane(where, t * 2 + 1);
                const uint32_t key0 = from + (t0 + t) * 32;
                if (w0 == ~0u || w1 == ~0u || key0 + 32 > to) {
                    // keys past the position or of no page: no score, and no value, whatever lies there
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t key = key0 + (i / 4) * 16 + q * 4 + i % 4;
                        if (key >= to || (i < 4 ? w0 : w1) == ~0u) {
                            s[i] = -INFINITY;
#pragma unroll
                            for (int u = 0; u < VP; ++u) vf[i][u] = make_uint4(0, 0, 0, 0);
                        }
                    }
                    any = any || w0 != ~0u || w1 != ~0u;
                } else {
                    any = true;
                }
                float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                                  fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float next = fmaxf(m, top);
                const float ref = next == -INFINITY ? 0.0f : next;
                if (__any(next != m)) {
                    const float keep = pa_exp(m - ref);
                    l *= keep;
#pragma unroll
                    for (int t = 0; t < VT; ++t) acc[t] *= keep;
                }
                m = next;
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p0 = pa_exp(s[2 * i] - ref);
                    const float p1 = pa_exp(s[2 * i + 1] - ref);
                    l += p0 + p1;
                    const uint32_t hi = f32x2_to_bf16x2_rne(p0, p1);
                    // what the rounding lost; nothing of an inf or NaN
                    const uint32_t lo = f32x2_to_bf16x2_rne(p0 - bf(hi & 0xFFFFu), p1 - bf(hi >> 16));
                    w[i] = c < 8 ? hi : lo;
                }
                pf = make_uint4(w[0], w[1], w[2], w[3]);
            };
            auto values = [&] {
#pragma unroll
                for (int t = 0; t < VT; ++t) {
                    const int u = t / PD, d = t % PD;
                    auto word = [&](int i) {
                        const uint4 v = vf[i][u];
                        return d / 2 == 0 ? v.x : d / 2 == 1 ? v.y : d / 2 == 2 ? v.z : v.w;
                    };
                    const uint32_t sel = d % 2 ? 0x07060302u : 0x05040100u;
                    auto pair = [&](int i) { return __builtin_amdgcn_perm(word(i + 1), word(i), sel); };
                    const uint4 f = make_uint4(pair(0), pair(2), pair(4), pair(6));
                    acc[t] = pa_mfma(f, pf, acc[t]);
                }
            };
            // each tile's keys are in flight behind the values before them
            load_k(0);
            load_v(0);
            for (uint32_t t = 0; t + 1 < batch_tiles; ++t) {
                scores();
                load_k(t + 1);
                weigh(t);
                values();
                load_v(t + 1);
            }
            scores();
            weigh(batch_tiles - 1);
            values();
        }

        // the wavefront's result: l over its four key quarters, the two parts of P
        // together (a sum that is inf or NaN already stays as it is)
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
#pragma unroll
        for (int t = 0; t < VT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float lo = __shfl_xor(acc[t][r], 8, 64), hi = acc[t][r];
                const int d = (t / PD) * 128 + (q * 4 + r) * PD + t % PD;
                if (c < 8) part_o[wave][c][d] = fabsf(hi) < INFINITY ? hi + lo : hi;
            }
        if (lane < 8) {
            part_ml[wave][0][c] = m;
            part_ml[wave][1][c] = l;
            part_ml[wave][2][c] = any ? 1.0f : 0.0f;
        }
        __syncthreads();

        // the four joined: thread (head, dims)
        constexpr int DT = std::max<int>(2, kHeadTile * HD / (64 * W));  // dims of a thread
        const uint32_t own = threadIdx.x / (HD / DT), h = min(own, kHeadTile - 1);
        const uint32_t d0 = threadIdx.x % (HD / DT) * DT;
        float top = -INFINITY;
        bool some = false;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            top = fmaxf(top, part_ml[w][0][h]);
            some = some || part_ml[w][2][h] != 0.0f;
        }
        const float ref = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f, o[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < W; ++w) {
            const float f = pa_exp(part_ml[w][0][h] - ref);
            sum = fmaf(f, part_ml[w][1][h], sum);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] = fmaf(f, part_o[w][h][d0 + d], o[d]);
        }
        if (whole) {
            if (own < heads) {
                uint16_t *to = a.out + row0 + h * HD + d0;
#pragma unroll
                for (int d = 0; d < DT; d += 2)
                    *reinterpret_cast<uint32_t *>(to + d) = some ? f32x2_to_bf16x2_rne(o[d] / sum, o[d + 1] / sum) : 0u;
            }
        } else if (own < kHeadTile) {
            float *rec =
                a.records + (static_cast<uint64_t>(blockIdx.x + seq) * gridDim.y + blockIdx.y) * record_floats<HD>();
#pragma unroll
            for (int d = 0; d < DT; ++d) rec[h * HD + d0 + d] = o[d];
            if (d0 == 0) {
                rec[kHeadTile * HD + h] = top;
                rec[kHeadTile * HD + kHeadTile + h] = sum;
                rec[kHeadTile * HD + 2 * kHeadTile + h] = some ? 1.0f : 0.0f;
            }
        }
        __syncthreads();  // the LDS is read: the next piece may write it
    }
}

// Joins the pieces of one sequence's query head: block (sequence, head). Rows
// of HD / 4 threads each take every (256 / that)-th piece, kJoinLoads of them
// requested together, then join in LDS in order.
constexpr int kJoinLoads = 8;

template <int HD>
__global__ __launch_bounds__(kPagedThreads) void paged_join_kernel(const PagedArgs a) {
    constexpr uint32_t kRow = HD / 4, kRows = kPagedThreads / kRow;
    __shared__ float rows_o[kRows][HD + 4];
    __shared__ float rows_ml[kRows][3];
    const uint32_t h = blockIdx.y, row = threadIdx.x / kRow, d = threadIdx.x % kRow * 4, lane = threadIdx.x & 63u;
    Layout y = layout_of(a, lane);
    // this sequence among the 64 at hand, and the pieces that it was cut into
    const uint32_t seq = blockIdx.x;
    while (y.b0 + 64 <= seq) layout_at(a, y, y.b0 + 64, __builtin_amdgcn_readlane(y.upto, 63), lane);
    const uint32_t n = __builtin_amdgcn_readlane(y.mine, seq - y.b0);
    uint16_t *to = a.out + (static_cast<uint64_t>(seq) * a.n_heads + h) * HD;
    if (n == 0) {  // idle
        if (row == 0) *reinterpret_cast<uint2 *>(to + d) = make_uint2(0, 0);
        return;
    }
    const uint32_t start = __builtin_amdgcn_readlane(y.upto, seq - y.b0) - n;
    const uint32_t first = start / y.size, pieces = (start + n - 1) / y.size - first + 1;
    if (pieces == 1) return;  // written by its block
    const uint32_t group = a.n_heads / a.n_kv, tiles = (group + kHeadTile - 1) / kHeadTile;
    const uint32_t slot = h % group % kHeadTile;
    const uint64_t stride = static_cast<uint64_t>(a.n_kv) * tiles * record_floats<HD>();
    const float *rec = a.records + (first + seq) * stride +
                       static_cast<uint64_t>(h / group * tiles + h % group / kHeadTile) * record_floats<HD>();
    float m = -INFINITY, l = 0.0f, some = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    for (uint32_t i0 = row; i0 < pieces; i0 += kRows * kJoinLoads) {
        float pm[kJoinLoads], pl[kJoinLoads], ps[kJoinLoads];
        float4 v[kJoinLoads];
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u) {
            const float *x = rec + min(i0 + u * kRows, pieces - 1) * stride;
            pm[u] = x[kHeadTile * HD + slot];
            pl[u] = x[kHeadTile * HD + kHeadTile + slot];
            ps[u] = x[kHeadTile * HD + 2 * kHeadTile + slot];
            v[u] = *reinterpret_cast<const float4 *>(x + slot * HD + d);
        }
        float next = m;
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u) {
            if (i0 + u * kRows >= pieces) pm[u] = -INFINITY;
            next = fmaxf(next, pm[u]);
        }
        const float ref = next == -INFINITY ? 0.0f : next, f = pa_exp(m - ref);
        m = next;
        l *= f, o.x *= f, o.y *= f, o.z *= f, o.w *= f;
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u)
            if (i0 + u * kRows < pieces) {
                const float g = pa_exp(pm[u] - ref);
                some = fmaxf(some, ps[u]);
                l = fmaf(pl[u], g, l);
                o.x = fmaf(v[u].x, g, o.x), o.y = fmaf(v[u].y, g, o.y);
                o.z = fmaf(v[u].z, g, o.z), o.w = fmaf(v[u].w, g, o.w);
            }
    }
    *reinterpret_cast<float4 *>(&rows_o[row][d]) = o;
    if (d == 0) rows_ml[row][0] = m, rows_ml[row][1] = l, rows_ml[row][2] = some;
    __syncthreads();
    if (row != 0) return;
    for (uint32_t r = 0; r < kRows; ++r) m = fmaxf(m, rows_ml[r][0]);
    const float ref = m == -INFINITY ? 0.0f : m;
    l = 0.0f, some = 0.0f;
    o = make_float4(0, 0, 0, 0);
#pragma unroll
    for (uint32_t r = 0; r < kRows; ++r) {
        const float f = pa_exp(rows_ml[r][0] - ref);
        const float4 v = *reinterpret_cast<const float4 *>(&rows_o[r][d]);
        l = fmaf(f, rows_ml[r][1], l);
        some = fmaxf(some, rows_ml[r][2]);
        o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
    }
    *reinterpret_cast<uint2 *>(to + d) = some != 0.0f ? make_uint2(f32x2_to_bf16x2_rne(o.x / l, o.y / l),
                                                                  f32x2_to_bf16x2_rne(o.z / l, o.w / l))
                                                      : make_uint2(0, 0);
}

}  // namespace fh

using namespace fh;

namespace {

int check_shape(const char *fn, int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t page_size,
                int64_t max_pages) {
    if (int rc = fh_check_dims(fn, {batch, n_heads, n_kv, head_dim, page_size, max_pages})) return rc;
    if (int rc = check_pages(fn, 1, page_size, max_pages)) return rc;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(FH_ERR_UNSUPPORTED, "%s: head_dim %lld must be 64, 128 or 256", fn, (long long)head_dim);
    if (n_kv < 1 || n_heads < 1 || n_heads % n_kv != 0 || n_heads > 65535)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: %lld heads do not share %lld KV heads", fn, (long long)n_heads,
                    (long long)n_kv);
    if (batch > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: batch %lld exceeds 65535", fn, (long long)batch);
    // the steps of all sequences are counted in 32 bits (pages may be shared, so their number bounds nothing)
    if (batch * (max_pages * page_size / kStepKeys + 1) > 0x7FFFFFFFll)
        return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld sequences of %lld positions", fn, (long long)batch,
                    (long long)(max_pages * page_size));
    return FH_OK;
}

// The launch for these sizes: parts per (KV head, head tile), or 0 for a block
// per sequence, the grid, and the bytes of the pieces' records.
struct Plan {
    uint32_t want_parts, grid_parts, grid_heads;
    uint64_t bytes;
    bool wide;  // 8 wavefronts to a block, where each takes a whole sequence
};

Plan plan(int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t page_size, int64_t max_pages) {
    const uint64_t tiles = n_kv * ((n_heads / n_kv + kHeadTile - 1) / kHeadTile);
    const uint64_t capacity = static_cast<uint64_t>(max_pages) * page_size;
    const bool whole = capacity * head_dim <= kWholeElements;
    if (whole) return {0, static_cast<uint32_t>(batch), static_cast<uint32_t>(tiles), 16, true};
    if (batch > kPlanBatch)  // what serves the largest batch serves smaller ones: the bytes of those that are split
        return {0, static_cast<uint32_t>(batch), static_cast<uint32_t>(tiles),
                plan(kPlanBatch, n_heads, n_kv, head_dim, page_size, max_pages).bytes, false};
    // a table of few steps has no use for more parts than steps
    const uint64_t steps = (capacity + kStepKeys - 1) / kStepKeys;
    const uint64_t parts = std::max<uint64_t>(1, std::min<uint64_t>(kPartBlocks / tiles, batch * steps));
    const uint64_t record = (kHeadTile * head_dim + 3 * kHeadTile) * 4;
    return {static_cast<uint32_t>(parts), static_cast<uint32_t>(parts), static_cast<uint32_t>(tiles),
            (parts + batch) * tiles * record + 16, false};
}

}  // namespace

extern "C" int fh_paged_attention_workspace(int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                                            int64_t page_size, int64_t max_pages, uint64_t *bytes) {
    const char *fn = "fh_paged_attention_workspace";
    if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: bytes is null", fn);
    if (int rc = check_shape(fn, batch, n_heads, n_kv, head_dim, page_size, max_pages)) return rc;
    *bytes = plan(batch, n_heads, n_kv, head_dim, page_size, max_pages).bytes;
    return FH_OK;
}

extern "C" int fh_paged_attention(fh_device *dev, const uint16_t *q, int64_t batch, int64_t n_heads, int64_t n_kv,
                                  int64_t head_dim, const uint16_t *k_pages, const uint16_t *v_pages, int64_t n_pages,
                                  int64_t page_size, const uint32_t *page_table, int64_t max_pages,
                                  const uint32_t *positions, float scale, void *workspace, uint64_t workspace_bytes,
                                  uint16_t *out) {
    const char *fn = "fh_paged_attention";
    if (int rc = check_usable(dev, fn)) return rc;
    if (int rc = check_shape(fn, batch, n_heads, n_kv, head_dim, page_size, max_pages)) return rc;
    if (int rc = fh_check_dims(fn, {n_pages})) return rc;
    if (int rc = check_pages(fn, n_pages, page_size, max_pages)) return rc;
    if (batch == 0) return FH_OK;
    uint64_t need = 0;
    if (int rc = fh_paged_attention_workspace(batch, n_heads, n_kv, head_dim, page_size, max_pages, &need)) return rc;
    if (workspace_bytes < need)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: workspace of %llu bytes, %llu needed", fn,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) &
        15u)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: q, out and workspace must be 16-byte aligned", fn);
    const uint64_t rows = static_cast<uint64_t>(batch) * n_heads * head_dim * 2;
    uint64_t pool;
    if (int rc = check_pools(dev, fn, k_pages, v_pages, n_pages, n_kv, page_size, head_dim, page_table, batch,
                             max_pages, &pool))
        return rc;
    if (int rc = check_range(dev, workspace, need, fn, "workspace")) return rc;
    if (int rc = check_range(dev, q, rows, fn, "q")) return rc;
    if (int rc = check_range(dev, positions, static_cast<uint64_t>(batch) * 4, fn, "positions")) return rc;
    if (int rc = check_range(dev, out, rows, fn, "out")) return rc;
    for (const auto &[what, ptr, size] : {std::tuple{"out", static_cast<const void *>(out), rows},
                                          std::tuple{"workspace", static_cast<const void *>(workspace), need}}) {
        if (int rc = refuse_overlap(fn, what, ptr, size, "q", q, rows)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "k_pages", k_pages, pool)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "v_pages", v_pages, pool)) return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "page_table", page_table,
                                    static_cast<uint64_t>(batch) * max_pages * 4))
            return rc;
        if (int rc = refuse_overlap(fn, what, ptr, size, "positions", positions, static_cast<uint64_t>(batch) * 4))
            return rc;
    }
    if (int rc = refuse_overlap(fn, "workspace", workspace, need, "out", out, rows)) return rc;
    if (int rc = set_current(dev, fn)) return rc;
    const Plan w = plan(batch, n_heads, n_kv, head_dim, page_size, max_pages);
    const PagedArgs a{q,
                      k_pages,
                      v_pages,
                      page_table,
                      positions,
                      static_cast<uint32_t>(batch),
                      static_cast<uint32_t>(n_heads),
                      static_cast<uint32_t>(n_kv),
                      static_cast<uint32_t>(n_pages),
                      static_cast<uint32_t>(page_size),
                      static_cast<uint32_t>(max_pages),
                      w.want_parts,
                      scale,
                      static_cast<float *>(workspace),
                      out};
    const dim3 grid(w.grid_parts, w.grid_heads), threads(kPagedThreads), wide(2 * kPagedThreads);
    if (int rc = dispatch(dev, fn, [&] {
            if (head_dim == 256)
                hipLaunchKernelGGL((paged_part_kernel<256, 4>), grid, threads, 0, dev->stream, a);
            else if (head_dim == 128 && w.wide)
                hipLaunchKernelGGL((paged_part_kernel<128, 8>), grid, wide, 0, dev->stream, a);
            else if (head_dim == 128)
                hipLaunchKernelGGL((paged_part_kernel<128, 4>), grid, threads, 0, dev->stream, a);
            else if (w.wide)
                hipLaunchKernelGGL((paged_part_kernel<64, 8>), grid, wide, 0, dev->stream, a);
            else
                hipLaunchKernelGGL((paged_part_kernel<64, 4>), grid, threads, 0, dev->stream, a);
        }))
        return rc;
    if (w.want_parts == 0) return FH_OK;
    const dim3 join(static_cast<uint32_t>(batch), static_cast<uint32_t>(n_heads));
    return dispatch(dev, fn, [&] {
        if (head_dim == 64)
            hipLaunchKernelGGL(paged_join_kernel<64>, join, threads, 0, dev->stream, a);
        else if (head_dim == 128)
            hipLaunchKernelGGL(paged_join_kernel<128>, join, threads, 0, dev->stream, a);
        else
            hipLaunchKernelGGL(paged_join_kernel<256>, join, threads, 0, dev->stream, a);
    });
}
