// Attention of a tree of drafted tokens over a paged cache
// (fh_paged_tree_attention).
#include <algorithm>
#include <limits>
#include <tuple>

#include "paged_cache.hpp"

namespace fh {

// The mathematics: one pass over the keys with the running reference m, sum l and
// weighted values o of each row (a node's query head),
//   l' = l 2^(m k - m' k) + 2^(s k - m' k), o' = o 2^(m k - m' k) + 2^(s k - m' k) v,
// k = scale log2 e, joined over disjoint key ranges by the same rule. m k is rounded
// once, the same way wherever it stands, so that its rounding is no weight's. m follows
// the largest score only where that has grown by more than kSlack in the exponent, so
// that o is seldom multiplied; the weights are then up to 2^kSlack, which fp32 sums
// and 16-bit factors hold as well as those up to 1.
//
// The split: the rows of one KV head (nodes x the query heads that share it) are
// cut into tiles of 16 NT. A block of four wavefronts takes a tile and a part of
// the batch's keys (whole steps of kStepKeys), with the tile's q in LDS; every
// wavefront has o in registers and streams a quarter of the part's keys, 32 at a time, and
// the four join in LDS. So K and V are read once per tile, straight into the fragments that
// the matrix cores take. The parts are laid out from lengths and counts on the
// device (see Layout): the same launch serves one long context and a ragged batch,
// and may be captured.
//
// Per 32 keys the scores are S^T = K Q^T (v_mfma_f32_16x16x32_bf16, 16 keys x 16
// rows): a lane ends up with its row's scores of keys 4 q .. 4 q + 3 (q = lane / 16)
// of both 16-key groups. Those eight weights are the fragment that O^T = V^T P^T
// needs of that lane if its keys are numbered so, so P never leaves its lane; V's rows,
// read as they lie, become V^T fragments by byte permutes within a lane, once for all
// NT row groups. P goes in twice, as what rounding to bf16 leaves and as what it
// loses, for 16 bits of P: what those lose, 2^-16 of a term, is far below the half
// step of 2^-8 that bf16 V is off by itself. m, l and o are fp32.
//
// Measured among calls on other data, 32 heads of 128 over 8 KV heads: 64 nodes of 8 sequences of 1900 to 4111
// tokens 74 us (291 TFLOP/s), 32 nodes behind 131077 tokens 167 us (3.2 TB/s, 412 TFLOP/s), 8 nodes 107 us
// (5.0 TB/s), 6 nodes behind 700 tokens 12.8 us. Many nodes are bound by K and V on
// their way through the L1, once per 32 rows (45 of its 64 bytes a cycle), and by the vector instructions around
// the products (about 190 of 4 cycles for 48 products of 16, per 32 keys and rows), few nodes by memory,
// short contexts by two launches of dependent loads. Figures of settings side by side below are of one call over
// and over, which finds its keys in the caches as far as they hold them (64 nodes of the 8 sequences 66 us).
constexpr uint32_t kMaxTree = 1024;
constexpr uint32_t kTreeThreads = 256;
constexpr uint32_t kWaves = kTreeThreads / 64;
constexpr uint32_t kStepKeys = 128;
constexpr float kSlack = 8.0f;
// Tables of so few positions (times head_dim) take one block per sequence and tile,
// and no join: one launch (512 positions of head_dim 128, 24 rows: 10.9 us, 12.7 in parts; 850:
// 13.2 and 12.9; 1506: 18.8 and 14.8).
constexpr uint32_t kWholeElements = 65536;
// Batches of more steps take at least two to a part.
constexpr uint32_t kFewSteps = 16;
// What a sequence's start and join count beside its steps where parts of several sequences are
// cut (with 0, 2, 4, 6, 9: 12 nodes of 64 sequences of 17 to 16384 tokens 107, 95, 97, 100, 105 us,
// 64 nodes of 8 of 1900 to 4111 72, 69, 66, 66, 67, 8 nodes of 32 over one KV head of 256 50, 43, 36, 37, 36).
constexpr uint32_t kStart = 4;
// Larger batches take one part per sequence, as every block would lay them all out.
constexpr uint32_t kPlanBatch = 1024;
// Where a sum of values passes 2^64 (or is not finite) and finite ones from 2^40 on are among them, they are taken
// 2^-48 times as large: 2^31 keys of weights up to 2^16 and values up to the type's largest then stay below
// fp32's. What is multiplied so is exact down to 2^-78. Sums that are not stay so far below fp32's largest (2^64, or
// 2^31 keys of 2^16 times 2^40) that joining them cannot pass it.
constexpr float kShrink = 0x1p-48f, kGrow = 0x1p48f;
constexpr uint16_t kLarge = (127 + 40) << 7, kInfinite = 0x7F80;  // bf16 2^40 and infinity

typedef __attribute__((ext_vector_type(8))) __bf16 ta_bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float ta_f32x4_t;
// whole registers of a fragment: a struct of words would be carried around loops word by word
typedef __attribute__((ext_vector_type(4))) uint32_t ta_u32x4_t;

__device__ __forceinline__ ta_f32x4_t ta_mfma(ta_u32x4_t a, ta_u32x4_t b, ta_f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(ta_bf16x8_t, a),
                                                   __builtin_bit_cast(ta_bf16x8_t, b), c, 0, 0, 0);
}

// n / by for n below 2^27, by up to 2^27, as one product: with m = ceil(2^k / by), k = 27
// + ceil(log2 by), the quotient is off by n (m by - 2^k) / (by 2^k) < 1 / by.
struct Divider {
    uint32_t by, m, k;
    explicit Divider(uint32_t d) : by(d), k(27) {
        while ((1u << (k - 27)) < d) ++k;
        m = static_cast<uint32_t>(((1ull << k) + d - 1) / d);
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        return static_cast<uint32_t>(static_cast<uint64_t>(n) * m >> k);
    }
};

struct TreeArgs {
    const uint16_t *q, *k_pages, *v_pages;
    const uint32_t *page_table, *lengths, *counts, *masks;
    uint32_t batch, width, n_heads, n_kv, n_pages, max_pages, capacity;
    Divider group;        // query heads of a KV head
    Divider page_groups;  // 16-key groups of a page
    uint32_t tiles;       // row tiles of a KV head
    uint32_t want_parts;  // parts of one (KV head, tile); 0: a block per sequence
    float k, slack;       // scale log2 e; kSlack in scores
    float *records;
    uint16_t *out;
};

// The nodes of sequence b, 0 where they do not fit its table.
__device__ __forceinline__ uint32_t nodes_of(const TreeArgs &a, uint32_t b) {
    const uint32_t count = a.counts ? min(a.counts[b], a.width) : a.width;
    const uint32_t len = a.lengths[b];
    return len <= a.capacity && count <= a.capacity - len ? count : 0;
}

// The steps of a sequence of `len` tokens and `count` nodes for rows from row0 on.
__device__ __forceinline__ uint32_t steps_of(const TreeArgs &a, uint32_t len, uint32_t count, uint32_t row0) {
    return count * a.group.by > row0 ? (len + count + kStepKeys - 1) / kStepKeys : 0;
}

__device__ __forceinline__ uint32_t scan_wave(uint32_t v, uint32_t lane) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t o = __shfl_up(v, off, 64);
        if (lane >= static_cast<uint32_t>(off)) v += o;
    }
    return v;
}

// The steps of all sequences that have rows in a tile, in order and (of more than one)
// kStart blank ones before each sequence's, are cut into equal parts: part x takes steps x * size .. of
// them, which may be the end of one sequence, whole ones, and the start of another. Of
// a part's pieces only two can be less than a sequence: what began before it leaves record
// 2 x, and what goes on behind it, from its sequence's first step, 2 x + 1. Every
// wavefront works the layout out for itself, 64 sequences at a time.
struct Layout {
    uint32_t size;   // steps of a part, blank ones among them
    uint32_t row0;   // the tile's first row
    uint32_t b0;     // first sequence of the 64 at hand
    uint32_t len, count;  // lane's sequence's tokens and nodes
    uint32_t mine;   // its steps, without the blank ones
    uint32_t upto;   // and all steps up to its end
};

__device__ __forceinline__ void layout_at(const TreeArgs &a, Layout &y, uint32_t b0, uint32_t before, uint32_t lane) {
    y.b0 = b0;
    y.count = b0 + lane < a.batch ? nodes_of(a, b0 + lane) : 0;
    y.len = y.count ? a.lengths[b0 + lane] : 0;
    y.mine = steps_of(a, y.len, y.count, y.row0);
    y.upto = before + scan_wave(y.mine && a.batch > 1 ? y.mine + kStart : y.mine, lane);
}

__device__ __forceinline__ Layout layout_of(const TreeArgs &a, uint32_t row0, uint32_t lane) {
    Layout y;
    y.row0 = row0;
    uint32_t total = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
        layout_at(a, y, b0, total, lane);
        total = __builtin_amdgcn_readlane(y.upto, 63);
    }
    // (a part of one step is mostly its start and join: 32 steps of 32 rows take 19.2 us by one
    // and 15.6 by two; 12 steps 14.7 and 14.4, 7 steps 12.9 and 13.1)
    y.size = max(total > kFewSteps ? 2u : 1u, (total + a.want_parts - 1) / a.want_parts);
    if (a.batch > 64) layout_at(a, y, 0, 0, lane);
    return y;
}

// Moves to the sequence that holds step `at` of the batch and returns it, its
// steps in n and all before its first in `start`; ~0 behind the last one.
__device__ __forceinline__ uint32_t sequence_of(const TreeArgs &a, Layout &y, uint32_t at, uint32_t lane, uint32_t &n,
                                                uint32_t &start, uint32_t &len, uint32_t &count) {
    for (;;) {
        const uint64_t hit = __ballot(at < y.upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            len = __builtin_amdgcn_readlane(y.len, l);
            count = __builtin_amdgcn_readlane(y.count, l);
            n = __builtin_amdgcn_readlane(y.mine, l);
            start = __builtin_amdgcn_readlane(y.upto, l) - n;  // behind the blank ones
            return y.b0 + l;
        }
        if (y.b0 + 64 >= a.batch) return ~0u;
        layout_at(a, y, y.b0 + 64, __builtin_amdgcn_readlane(y.upto, 63), lane);
    }
}

// A record: what a piece leaves to be joined, [16 NT rows][HD] weighted values,
// then m, l and whether any key was there (0: none, 1: yes, 2: yes, and the values are kShrink times as large), of
// each row.
template <int HD, int NT>
constexpr uint32_t record_floats() { return 16 * NT * (HD + 3); }

// p less one half of a word of two bf16, as a product of the word with (-1, 0) or (0, -1). Exact where
// the half is p's rounding.
template <int H>
__device__ __forceinline__ float less_half(float p, uint32_t two) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
    uint32_t unit = H ? 0xBF800000u : 0x0000BF80u;
    asm("" : "+s"(unit));  // in a register: written as the constant -1.0 it would stand in the upper half
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, two), __builtin_bit_cast(bf16x2_t, unit), p,
                                           false);
}

// The exponent of reference a's weights beside reference b > -inf, for products too large for fp32 too.
__device__ __forceinline__ float apart(float a, float b, float k) {
#pragma clang fp contract(off)
    const float x = a * k, y = b * k;
    return fabsf(y) < INFINITY && x < INFINITY ? x - y : (a - b) * k;
}

// Which of the 32 keys from key0 on a node of these mask words sees, as far as
// lengths and masks go.
__device__ __forceinline__ uint32_t window(const uint32_t *mask, uint32_t words, uint32_t key0, uint32_t len,
                                           uint32_t count) {
    const int32_t past = static_cast<int32_t>(key0 - len);           // places below 2^31
    const uint32_t before = min(max(-past, 0), 32);                  // tokens among them
    const uint32_t j0 = min(max(past, 0), static_cast<int>(count));  // the first node among them
    const uint32_t left = min(count - j0, 32u), w = min(j0 / 32, words - 1);
    const uint64_t two = mask[w] | static_cast<uint64_t>(mask[min(w + 1, words - 1)]) << 32;
    const uint64_t nodes = (two >> (j0 % 32)) & ((1ull << left) - 1);
    return static_cast<uint32_t>(nodes << before | ((1ull << before) - 1));
}

// v, worked out again from here on: what depends on it alone is not kept in registers
// over the loop around.
__device__ __forceinline__ uint32_t anew(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}

// The maximum over the lanes that share lane % 16.
__device__ __forceinline__ float max_over_quarters(float v) {
    typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
    const u32x2_t a = __builtin_bit_cast(
        u32x2_t, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const u32x2_t b = __builtin_bit_cast(
        u32x2_t, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <int HD, int NT>
__global__ __launch_bounds__(kTreeThreads, HD == 256 ? 1 : 2) void tree_part_kernel(const TreeArgs a) {
    constexpr int KC = HD / 32;                  // score products per 16 keys
    constexpr int VP = HD == 64 ? 1 : HD / 128;  // pieces of a lane's V row
    constexpr int PD = HD == 64 ? 4 : 8;         // dims of a piece
    constexpr int VT = VP * PD;                  // products per 32 keys
    struct Results {  // of the wavefronts
        float o[kWaves][16 * NT][HD + 4];
        float ml[kWaves][3][16 * NT];
    };
    // The tile's q as fragments [KC][NT][64 lanes], read for every 32 keys (registers are short), and
    // after them the wavefronts' results.
    __shared__ union {
        ta_u32x4_t q[KC * NT * 64];
        Results results;
    } shared;
    Results &part = shared.results;
    constexpr uint32_t kWords = kMaxTree / 32;
    __shared__ uint32_t bits[(16 * NT + 1) * kWords];  // the mask words of the tile's nodes
    // (the wavefront's number as a scalar: its loops then count in scalars too)
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t c = lane & 15u, q = lane >> 4;
    const uint32_t group = a.group.by, kv = blockIdx.z, row0 = blockIdx.y * (16 * NT);
    const uint32_t unit = kv * a.tiles + blockIdx.y;  // of the records
    const uint32_t words = (a.width + 31) / 32, node0 = a.group(row0);
    // where row `row` of sequence seq lies in q and out
    auto place = [&](uint32_t seq, uint32_t row) {
        const uint32_t node = a.group(row);
        return ((static_cast<uint64_t>(seq) * a.width + node) * a.n_heads + kv * group + (row - node * group)) * HD;
    };
    // zeros to the tile's rows past the nodes of sequence b
    auto clear = [&](uint32_t b, uint32_t count) {
        const uint32_t lo = max(row0, count * group), hi = min(row0 + 16 * NT, a.width * group);
        for (uint32_t i = anew(threadIdx.x); lo < hi && i < (hi - lo) * (HD / 8); i += kTreeThreads)
            *reinterpret_cast<uint4 *>(a.out + place(b, lo + i / (HD / 8)) + i % (HD / 8) * 8) = make_uint4(0, 0, 0, 0);
    };
    Layout y;
    uint32_t at = 0, end = 1;
    if (a.want_parts) {
        y = layout_of(a, row0, lane);
        at = blockIdx.x * y.size;
        end = at + y.size;
        for (uint32_t b = blockIdx.x; b < a.batch; b += gridDim.x)
            clear(b, b < 64 ? __builtin_amdgcn_readlane(y.count, b) : nodes_of(a, b));
    }
    while (at < end) {
        // the next piece: `steps` from `first` of sequence seq
        uint32_t seq = blockIdx.x, first = 0, steps, whole = 1, len, count;
        if (a.want_parts) {
            uint32_t n, start;
            seq = sequence_of(a, y, at, lane, n, start, len, count);
            if (seq == ~0u) break;
            first = max(at, start) - start;
            at = min(end, start + n);
            if (at <= start + first) continue;  // blank steps alone
            steps = at - start - first;
            whole = steps == n;
        } else {
            count = nodes_of(a, seq);
            len = a.lengths[seq];
            steps = steps_of(a, len, count, row0);
            at = end;
            clear(seq, count);
            if (steps == 0) break;
        }
        const uint32_t keys = len + count, rows = count * group;
        // this wavefront's keys: from .. to, in tiles of 32
        const uint32_t share = (steps * (kStepKeys / 32) + kWaves - 1) / kWaves * 32;
        const uint32_t from = first * kStepKeys + wave * share;
        const uint32_t to = min(from + share, min(keys, (first + steps) * kStepKeys));
        const uint32_t n_tiles = from < to ? (to - from + 31) / 32 : 0;
        // lane i: where the i-th 16-key group from tile t0 on lies, in groups from the
        // pools' start; ~0 for none (past the keys, no page)
        auto places = [&](uint32_t t0) {
            const uint32_t g = from / 16 + t0 * 2 + lane;
            uint32_t w = ~0u;
            if (t0 < n_tiles && g * 16 < to) {
                const uint32_t pi = a.page_groups(g);
                const uint32_t page = a.page_table[static_cast<uint64_t>(seq) * a.max_pages + pi];
                if (page < a.n_pages) w = (page * a.n_kv + kv) * a.page_groups.by + (g - pi * a.page_groups.by);
            }
            return w;
        };
        uint32_t first_where = places(0);
        // the tile's rows (behind the last one: that again, left out at the end)
        for (uint32_t i = anew(threadIdx.x); i < KC * NT * 64; i += kTreeThreads) {
            const uint32_t row = min(row0 + i / 64 % NT * 16 + i % 16, rows - 1);
            shared.q[i] = *reinterpret_cast<const ta_u32x4_t *>(a.q + place(seq, row) + i / (64 * NT) * 32 + i / 16 % 4 * 8);
        }
        uint32_t node[NT];
#pragma unroll
        for (int r = 0; r < NT; ++r) node[r] = a.group(min(row0 + r * 16 + c, rows - 1)) - node0;
        if ((first + steps) * kStepKeys > len) {
            const uint32_t tid = anew(threadIdx.x), w = tid % kWords;
            const uint32_t nodes = a.group(min(row0 + 16 * NT, rows) - 1) - node0 + 1;
            const uint32_t *mask = a.masks + (static_cast<uint64_t>(seq) * a.width + node0) * words + w;
            for (uint32_t i = tid / kWords; i < nodes && w < words; i += kTreeThreads / kWords) {
                const uint32_t upto = node0 + i + 1;  // of a chain
                bits[i * kWords + w] = a.masks           ? mask[i * words]
                                       : upto <= w * 32       ? 0u
                                       : upto - w * 32 >= 32 ? ~0u
                                                             : (1u << (upto - w * 32)) - 1;
            }
        }
        auto seen_by = [&](int r, uint32_t key0) {
            return window(bits + node[r] * kWords, words, key0, len, count);
        };
        __syncthreads();
        ta_f32x4_t acc[NT][VT];
        float m[NT], ref[NT], l[NT];  // ref: m k, as far as there is one
        uint32_t any[NT];
        // Once as above. Where that leaves a sum whose square is not finite, or m k is not, again with care: scores
        // whose products with k are too large are taken relative to m first, and keys that have an inf or NaN
        // among their values stay out of the products, where weights of 0 (a row that does not see the key, a P
        // that lost nothing) would make NaN of them, and are added row by row. Where large finite values were
        // among the keys, once more with all values kShrink times as large.
        bool careful = false, large = false, shrunk = false;
#pragma unroll 1
        for (;;) {
#pragma unroll
            for (int r = 0; r < NT; ++r) {
#pragma unroll
                for (int t = 0; t < VT; ++t) acc[r][t] = ta_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                m[r] = -INFINITY, ref[r] = 0.0f, l[r] = 0.0f, any[r] = 0;
            }
            if (n_tiles) {
                uint32_t even = first_where, odd = 0;  // the places of 32 tiles each, in turn
                // a tile's two groups; a missing one reads the pool's first group, whose scores are left out
                uint32_t g0 = __builtin_amdgcn_readlane(even, 0), g1 = __builtin_amdgcn_readlane(even, 1);
                ta_u32x4_t kf[2][KC];
                ta_u32x4_t vf[8][VP];
                auto start_of = [&](uint32_t g) { return static_cast<uint64_t>(g == ~0u ? 0u : g) * (16 * HD); };
                // (a scalar address and the lane's bytes from there)
                auto load_k = [&](uint32_t g0, uint32_t g1) {
                    const uint32_t mine = anew(c * 64 + q * 16);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const char *src = reinterpret_cast<const char *>(a.k_pages + start_of(h ? g1 : g0));
#pragma unroll
                        for (int s = 0; s < KC; ++s)
                            kf[h][s] = *reinterpret_cast<const ta_u32x4_t *>(src + mine + s * 1024);
                    }
                };
                auto load_v = [&](uint32_t g0, uint32_t g1) {
                    const uint32_t mine = anew(q * (8 * HD) + c * (2 * PD));
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const char *src = reinterpret_cast<const char *>(a.v_pages + start_of(i / 4 ? g1 : g0));
#pragma unroll
                        for (int u = 0; u < VP; ++u) {
                            if constexpr (HD == 64) {
                                const uint2 v = *reinterpret_cast<const uint2 *>(src + mine + i % 4 * (2 * HD));
                                vf[i][u] = ta_u32x4_t{v.x, v.y, 0, 0};
                            } else {
                                vf[i][u] =
                                    *reinterpret_cast<const ta_u32x4_t *>(src + mine + i % 4 * (2 * HD) + u * 256);
                            }
                        }
                    }
                };
                ta_f32x4_t s0[NT], s1[NT];
                // half of the tile's q: requested before the weights are formed, and the other half while
                // the products of the first are
                ta_u32x4_t qf[KC / 2 * NT];
                auto load_q = [&](int s) {
                    const ta_u32x4_t *src = shared.q + anew(lane);
#pragma unroll
                    for (int i = 0; i < NT; ++i) qf[s % (KC / 2) * NT + i] = src[(s * NT + i) * 64];
                };
                auto load_first_q = [&] {
#pragma unroll
                    for (int s = 0; s < KC / 2; ++s) load_q(s);
                    __builtin_amdgcn_sched_barrier(0);
                };
                auto scores = [&](ta_f32x4_t(&x0)[NT], ta_f32x4_t(&x1)[NT]) {
#pragma unroll
                    for (int r = 0; r < NT; ++r) x0[r] = x1[r] = ta_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int s = 0; s < KC; ++s) {
#pragma unroll
                        for (int r = 0; r < NT; ++r) {
                            const ta_u32x4_t f = qf[s % (KC / 2) * NT + r];
                            x0[r] = ta_mfma(kf[0][s], f, x0[r]);
                            x1[r] = ta_mfma(kf[1][s], f, x1[r]);
                        }
                        if (s < KC / 2) load_q(s + KC / 2);
                    }
                };
                ta_u32x4_t hi[NT], lo[NT];
                // the scores at hand: what no row sees goes, and the references follow
                auto limit = [&](uint32_t key0) {
                    if (key0 + 32 > len || g0 == ~0u || g1 == ~0u) {
                        const uint32_t there = (g0 != ~0u ? 0xFFFFu : 0u) | (g1 != ~0u ? 0xFFFF0000u : 0u), q = anew(lane) >> 4;
                        // keys behind the last or of no page: no value, whatever lies there
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint32_t at = (i / 4) * 16 + q * 4 + i % 4;
                            if (key0 + at >= keys || !(there >> at & 1u))
#pragma unroll
                                for (int u = 0; u < VP; ++u) vf[i][u] = ta_u32x4_t{0, 0, 0, 0};
                        }
#pragma unroll
                        for (int r = 0; r < NT; ++r) {
                            const uint32_t seen = seen_by(r, key0) & there;
                            any[r] |= seen;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (!(seen >> (q * 4 + i) & 1u)) s0[r][i] = -INFINITY;
                                if (!(seen >> (16 + q * 4 + i) & 1u)) s1[r][i] = -INFINITY;
                            }
                        }
                    } else {
#pragma unroll
                        for (int r = 0; r < NT; ++r) any[r] = 1;
                    }
                    float top[NT];
                    bool grown = false;
#pragma unroll
                    for (int r = 0; r < NT; ++r) {
                        const ta_f32x4_t x = s0[r], z = s1[r];
                        top[r] = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                       fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3])));
                        grown = grown || top[r] > m[r] + a.slack;  // m = -inf: any score at all
                    }
                    if (__any(grown)) {
#pragma unroll
                        for (int r = 0; r < NT; ++r) {
                            top[r] = max_over_quarters(top[r]);
                            top[r] = top[r] > m[r] + a.slack ? top[r] : m[r];
                            const float keep = top[r] == m[r] ? 1.0f : __builtin_amdgcn_exp2f(apart(m[r], top[r], a.k));
                            l[r] *= keep;
#pragma unroll
                            for (int t = 0; t < VT; ++t) acc[r][t] *= keep;
                            m[r] = top[r];
                            ref[r] = m[r] == -INFINITY ? 0.0f : m[r] * a.k;
                        }
                    }
                    if (careful) {
#pragma unroll
                        for (int r = 0; r < NT; ++r) {
                            const bool big = m[r] > -INFINITY && !(fabsf(m[r] * a.k) < INFINITY);
#pragma unroll
                            for (int i = 0; i < 4; ++i) s0[r][i] -= big ? m[r] : 0.0f, s1[r][i] -= big ? m[r] : 0.0f;
                            if (big) ref[r] = 0.0f;
                        }
                    }
                };
                auto weigh = [&] {
#pragma unroll
                    for (int r = 0; r < NT; ++r) {
                        float p[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            p[i] = __builtin_amdgcn_exp2f(fmaf(s0[r][i], a.k, -ref[r]));
                            p[4 + i] = __builtin_amdgcn_exp2f(fmaf(s1[r][i], a.k, -ref[r]));
                        }
                        l[r] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                        uint32_t wh[4], wl[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            wh[i] = f32x2_to_bf16x2_rne(p[2 * i], p[2 * i + 1]);
                            asm("" : "+v"(wh[i]));  // both halves from this one conversion
                            wl[i] = f32x2_to_bf16x2_rne(less_half<0>(p[2 * i], wh[i]), less_half<1>(p[2 * i + 1], wh[i]));
                        }
                        hi[r] = ta_u32x4_t{wh[0], wh[1], wh[2], wh[3]};
                        lo[r] = ta_u32x4_t{wl[0], wl[1], wl[2], wl[3]};
                    }
                };
                // keys with an inf or NaN among their values: added to the rows that see them, and taken out of vf;
                // large finite values are noted, or all made smaller
                auto special = [&](uint32_t key0) {
                    typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;
                    const float unit = shrunk ? kShrink : 1.0f;
                    u16x2_t least = {0xFFFF, 0xFFFF};
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int u = 0; u < VP; ++u)
#pragma unroll
                            for (int x = 0; x < PD / 2; ++x)
                                least = __builtin_elementwise_min(
                                    least, __builtin_bit_cast(u16x2_t, vf[i][u][x] & 0x7FFF7FFFu) - u16x2_t{kLarge, kLarge});
                    large = large || __any(min(least[0], least[1]) < kInfinite - kLarge);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint32_t found = 0;
#pragma unroll
                        for (int u = 0; u < VP; ++u)
                            found |= bf16_specials(vf[i][u].x) | bf16_specials(vf[i][u].y) |
                                     bf16_specials(vf[i][u].z) | bf16_specials(vf[i][u].w);
                        const uint64_t lanes = __ballot(found != 0);
                        if (lanes == 0) continue;
                        for (uint32_t of = 0; of < 4; ++of) {
                            if (!(lanes >> (of * 16) & 0xFFFFu)) continue;
                            const uint32_t at = (i / 4) * 16 + of * 4 + i % 4;
                            if (q == of)
#pragma unroll
                                for (int u = 0; u < VP; ++u) vf[i][u] = ta_u32x4_t{0, 0, 0, 0};
                            const uint16_t *v = a.v_pages + start_of(i / 4 ? g1 : g0) + (of * 4 + i % 4) * HD;
#pragma unroll
                            for (int r = 0; r < NT; ++r) {
                                // the row's weight of this key, from the lane that has it
                                auto half = [&](const ta_u32x4_t p) {
                                    const uint32_t two = i / 4 ? (i % 4 / 2 ? p.w : p.z) : (i % 4 / 2 ? p.y : p.x);
                                    return bf(i % 2 ? two >> 16 : two & 0xFFFFu);
                                };
                                const float w = __shfl(half(hi[r]) + half(lo[r]), of * 16 + c, 64);
                                const uint16_t *mine = v + anew(q * (4 * PD));
                                if (seen_by(r, key0) >> at & 1u)
#pragma unroll
                                    for (int t = 0; t < VT; ++t) {
                                        asm volatile("" ::: "memory");  // four loads at a time
#pragma unroll
                                        for (int x = 0; x < 4; ++x)
                                            acc[r][t][x] = fmaf(w, bf(mine[(t / PD) * 128 + x * PD + t % PD]) * unit,
                                                                acc[r][t][x]);
                                    }
                            }
                        }
                    }
                    if (!shrunk) return;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
#pragma unroll
                        for (int u = 0; u < VP; ++u)
#pragma unroll
                            for (int x = 0; x < PD / 2; ++x)
                                vf[i][u][x] = f32x2_to_bf16x2_rne(bf(vf[i][u][x] & 0xFFFFu) * kShrink,
                                                                  bf(vf[i][u][x] >> 16) * kShrink);
                };
                auto values = [&] {
#pragma unroll
                    for (int t = 0; t < VT; ++t) {
                        const int u = t / PD, d = t % PD;
                        auto word = [&](int i) { return vf[i][u][d / 2]; };
                        const uint32_t sel = d % 2 ? 0x07060302u : 0x05040100u;
                        auto pair = [&](int i) { return __builtin_amdgcn_perm(word(i + 1), word(i), sel); };
                        const ta_u32x4_t f = {pair(0), pair(2), pair(4), pair(6)};
#pragma unroll
                        for (int r = 0; r < NT; ++r) acc[r][t] = ta_mfma(f, hi[r], acc[r][t]);
#pragma unroll
                        for (int r = 0; r < NT; ++r) acc[r][t] = ta_mfma(f, lo[r], acc[r][t]);
                    }
                };
                // The next tile's scores are formed on the matrix cores while this one's weights are; its
                // keys are two tiles ahead, its values one. (Behind the last: that tile again; a load that
                // may not be there would have the values wait for all of them.)
                auto groups = [&](uint32_t t, uint32_t &x0, uint32_t &x1) {
                    t = min(t, n_tiles - 1);
                    x0 = __builtin_amdgcn_readlane(t / 32 % 2 ? odd : even, t % 32 * 2);
                    x1 = __builtin_amdgcn_readlane(t / 32 % 2 ? odd : even, t % 32 * 2 + 1);
                };
                uint32_t n0, n1;
                groups(1, n0, n1);
                load_k(g0, g1);
                load_first_q();
                scores(s0, s1);
                load_k(n0, n1);
                load_v(g0, g1);
#pragma unroll 1
                for (uint32_t t = 0; t < n_tiles; ++t) {
                    limit(from + t * 32);
                    if (t % 32 == 8) (t / 32 % 2 ? even : odd) = places((t / 32 + 1) * 32);
                    load_first_q();
                    weigh();
                    ta_f32x4_t x0[NT], x1[NT];
                    scores(x0, x1);
                    uint32_t f0, f1;
                    groups(t + 2, f0, f1);
                    load_k(f0, f1);
                    if (__builtin_expect(careful, false)) special(from + t * 32);
                    values();
                    load_v(n0, n1);
#pragma unroll
                    for (int r = 0; r < NT; ++r) s0[r] = x0[r], s1[r] = x1[r];
                    g0 = n0, g1 = n1, n0 = f0, n1 = f1;
                }
            }
            ta_f32x4_t size = {0.0f, 0.0f, 0.0f, 0.0f};  // not finite if a sum's square is not
#pragma unroll
            for (int r = 0; r < NT; ++r) {
                size[0] = fmaf(m[r] == -INFINITY ? 0.0f : m[r] * a.k, 0.0f, size[0]);
#pragma unroll
                for (int t = 0; t < VT; ++t)
#pragma unroll
                    for (int x = 0; x < 4; ++x) size[x] = fmaf(acc[r][t][x], acc[r][t][x], size[x]);
            }
            if (careful ? shrunk || !large : !__any(!((size[0] + size[1]) + (size[2] + size[3]) < INFINITY))) break;
            shrunk = careful;
            careful = true;
        }

        // the four wavefronts joined: thread (row, dims), 16 rows at a time
        __syncthreads();  // q is read
#pragma unroll
        for (int r = 0; r < NT; ++r) {
            l[r] += __shfl_xor(l[r], 16, 64);
            l[r] += __shfl_xor(l[r], 32, 64);
            const uint32_t at = anew(lane), i = r * 16 + at % 16, q = at >> 4;
#pragma unroll
            for (int t = 0; t < VT; t += 4)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    *reinterpret_cast<float4 *>(&part.o[wave][i][(t / PD) * 128 + (q * 4 + x) * PD + t % PD]) =
                        make_float4(acc[r][t][x], acc[r][t + 1][x], acc[r][t + 2][x], acc[r][t + 3][x]);
            if (lane < 16) {
                part.ml[wave][0][i] = m[r];
                part.ml[wave][1][i] = l[r];
                part.ml[wave][2][i] = !any[r] ? 0.0f : shrunk ? 2.0f : 1.0f;
            }
        }
        __syncthreads();
        constexpr uint32_t DT = 16 * HD / kTreeThreads;  // dims of a thread
        const uint32_t tid = anew(threadIdx.x), d0 = tid % (HD / DT) * DT;
        float *rec = a.records + (static_cast<uint64_t>(blockIdx.x * 2 + (first == 0)) * (a.n_kv * a.tiles) + unit) *
                                     record_floats<HD, NT>();
#pragma unroll 1
        for (uint32_t i = tid / (HD / DT); i < 16 * NT && row0 + i < rows; i += 16) {
            float top = -INFINITY, some = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kWaves; ++w) {
                top = fmaxf(top, part.ml[w][0][i]);
                some = fmaxf(some, part.ml[w][2][i]);
            }
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f, o[DT];
#pragma unroll
            for (uint32_t d = 0; d < DT; ++d) o[d] = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(apart(part.ml[w][0][i], ref, a.k));
                const float g = f * (part.ml[w][2][i] < some ? kShrink : 1.0f);  // (0 for none: its sums are 0)
                sum = fmaf(f, part.ml[w][1][i], sum);
#pragma unroll
                for (uint32_t d = 0; d < DT; ++d) o[d] = fmaf(g, part.o[w][i][d0 + d], o[d]);
            }
            if (whole) {
                uint16_t *to = a.out + place(seq, row0 + i) + d0;
                const float inv = (some > 1.0f ? kGrow : 1.0f) / sum;
#pragma unroll
                for (uint32_t d = 0; d < DT; d += 2)
                    *reinterpret_cast<uint32_t *>(to + d) =
                        some != 0.0f ? f32x2_to_bf16x2_rne(o[d] * inv, o[d + 1] * inv) : 0u;
            } else {
#pragma unroll
                for (uint32_t d = 0; d < DT; d += 4)
                    *reinterpret_cast<float4 *>(rec + i * HD + d0 + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
                if (d0 == 0) {
                    rec[16 * NT * HD + i] = top;
                    rec[16 * NT * (HD + 1) + i] = sum;
                    rec[16 * NT * (HD + 2) + i] = some;
                }
            }
        }
        __syncthreads();  // the LDS is read: the next piece may write it
    }
}

// Joins the pieces of rows of one sequence: block (sequence, KV head and rows), a
// row by HD / 4 threads, kJoinLoads pieces requested together.
constexpr int kJoinLoads = 8;

template <int HD, int NT>
__global__ __launch_bounds__(kTreeThreads) void tree_join_kernel(const TreeArgs a) {
    constexpr uint32_t kRow = HD / 4, kRows = kTreeThreads / kRow, kBlocks = (16 * NT + kRows - 1) / kRows;
    const uint32_t seq = blockIdx.x, lane = threadIdx.x & 63u, d = threadIdx.x % kRow * 4;
    const uint32_t tile = blockIdx.y / kBlocks, kv = blockIdx.z, unit = kv * a.tiles + tile;
    const uint32_t i = blockIdx.y % kBlocks * kRows + threadIdx.x / kRow;  // the row in its tile
    const uint32_t row0 = tile * (16 * NT), row = row0 + i;
    Layout y = layout_of(a, row0, lane);
    while (y.b0 + 64 <= seq) layout_at(a, y, y.b0 + 64, __builtin_amdgcn_readlane(y.upto, 63), lane);
    const uint32_t n = __builtin_amdgcn_readlane(y.mine, seq - y.b0);
    if (n == 0) return;  // no row here
    const uint32_t rows = __builtin_amdgcn_readlane(y.count, seq - y.b0) * a.group.by;
    const uint32_t start = __builtin_amdgcn_readlane(y.upto, seq - y.b0) - n;
    const uint32_t first = start / y.size, pieces = (start + n - 1) / y.size - first + 1;
    if (pieces == 1 || row >= rows || i >= 16 * NT) return;  // written by its block, or no row
    const uint64_t stride = static_cast<uint64_t>(a.n_kv) * a.tiles * record_floats<HD, NT>();
    const float *rec = a.records + static_cast<uint64_t>(unit) * record_floats<HD, NT>();
    auto piece = [&](uint32_t p) {
        return rec + (static_cast<uint64_t>(first + p) * 2 + (p == 0)) * stride;
    };
    float m = -INFINITY, l = 0.0f, some = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    for (uint32_t p0 = 0; p0 < pieces; p0 += kJoinLoads) {
        float pm[kJoinLoads], pl[kJoinLoads], ps[kJoinLoads];
        float4 v[kJoinLoads];
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u) {
            const float *x = piece(min(p0 + u, pieces - 1));
            pm[u] = x[16 * NT * HD + i];
            pl[u] = x[16 * NT * (HD + 1) + i];
            ps[u] = x[16 * NT * (HD + 2) + i];
            v[u] = *reinterpret_cast<const float4 *>(x + i * HD + d);
        }
        float next = m;
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u) {
            if (p0 + u >= pieces) pm[u] = -INFINITY;
            next = fmaxf(next, pm[u]);
        }
        const float ref = next == -INFINITY ? 0.0f : next, f = __builtin_amdgcn_exp2f(apart(m, ref, a.k));
        m = next;
        const float before = some;
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u)
            if (p0 + u < pieces) some = fmaxf(some, ps[u]);
        const float h = f * (before < some ? kShrink : 1.0f);
        l *= f, o.x *= h, o.y *= h, o.z *= h, o.w *= h;
#pragma unroll
        for (int u = 0; u < kJoinLoads; ++u)
            if (p0 + u < pieces) {
                const float g = __builtin_amdgcn_exp2f(apart(pm[u], ref, a.k));
                const float e = g * (ps[u] < some ? kShrink : 1.0f);
                l = fmaf(pl[u], g, l);
                o.x = fmaf(v[u].x, e, o.x), o.y = fmaf(v[u].y, e, o.y);
                o.z = fmaf(v[u].z, e, o.z), o.w = fmaf(v[u].w, e, o.w);
            }
    }
    const uint32_t node = a.group(row);
    uint16_t *to = a.out +
                   ((static_cast<uint64_t>(seq) * a.width + node) * a.n_heads + kv * a.group.by +
                    (row - node * a.group.by)) * HD + d;
    const float inv = (some > 1.0f ? kGrow : 1.0f) / l;
    *reinterpret_cast<uint2 *>(to) = some != 0.0f ? make_uint2(f32x2_to_bf16x2_rne(o.x * inv, o.y * inv),
                                                              f32x2_to_bf16x2_rne(o.z * inv, o.w * inv))
                                                  : make_uint2(0, 0);
}

}  // namespace fh

using namespace fh;

namespace {

int check_shape(const char *fn, int64_t batch, int64_t width, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                int64_t page_size, int64_t max_pages) {
    if (int rc = fh_check_dims(fn, {batch, width, n_heads, n_kv, head_dim, page_size, max_pages})) return rc;
    if (int rc = check_pages(fn, 1, page_size, max_pages)) return rc;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256)
        return fail(FH_ERR_UNSUPPORTED, "%s: head_dim %lld must be 64, 128 or 256", fn, (long long)head_dim);
    if (n_kv < 1 || n_heads < 1 || n_heads % n_kv != 0 || n_heads > 65535)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: %lld heads do not share %lld KV heads", fn, (long long)n_heads,
                    (long long)n_kv);
    if (width < 1 || width > kMaxTree)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: width %lld must be 1 to %u", fn, (long long)width, kMaxTree);
    if (batch > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: batch %lld exceeds 65535", fn, (long long)batch);
    // rows of a KV head (below 2^27, and the joining launch's blocks of at least 4), and KV heads
    if (width * (n_heads / n_kv) > 4 * 65535 - 64 || n_kv > 65535)
        return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld nodes of %lld heads", fn, (long long)width, (long long)n_heads);
    // the steps of all sequences are counted in 32 bits (pages may be shared, so their number bounds nothing)
    if (batch * (max_pages * page_size / kStepKeys + 1 + kStart) > 0x7FFFFFFFll)
        return fail(FH_ERR_INDEX_TOO_LARGE, "%s: %lld sequences of %lld positions", fn, (long long)batch,
                    (long long)(max_pages * page_size));
    return FH_OK;
}

// The launch for these sizes: 16-row groups per block, tiles of a KV head, parts per
// (KV head, tile), or 0 for a block per sequence, and the bytes of the pieces' records.
struct Plan {
    uint32_t groups, tiles, want_parts;
    uint64_t bytes;
};

Plan plan(int64_t batch, int64_t width, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t page_size,
          int64_t max_pages) {
    const uint64_t rows = width * (n_heads / n_kv), capacity = static_cast<uint64_t>(max_pages) * page_size;
    // 4 nodes of 4 heads over 30000 tokens: 32.4 us as one group, 33.8 as two; four groups (64 rows,
    // registers for one block to a CU) took 80 where two then took 63, 64 nodes over 8 x 3000
    const uint32_t groups = rows <= 16 ? 1 : 2;
    const uint64_t tiles = (rows + 16 * groups - 1) / (16 * groups), units = tiles * n_kv;
    Plan w{groups, static_cast<uint32_t>(tiles), 0, 16};
    if (capacity * head_dim <= kWholeElements) return w;
    // what serves the largest batch serves smaller ones: the bytes of those that are split
    const uint64_t split = std::min<uint64_t>(batch, kPlanBatch);
    // A block's registers leave room for two on a CU, or for one with head_dim 256 (8 x 3000 tokens, 32
    // nodes of 8 heads: 32 us, 44 with 512 blocks). Where a KV head has one tile, memory is the bound, which
    // one block per CU draws on as well, and there are half as many pieces to join (8 nodes over 131000
    // tokens 106 us, 116 with 512; over 30000 34.8 and 41.1; 64 x 600, 37.4 and 33.5, pays for it);
    // with more tiles two keep the matrix cores busier (64 nodes over 30000: 68 us, 74 with 256).
    // Parts are whole for each (KV head, tile), so that up to half of the blocks may be missing where these do not
    // divide their number: 8 x 3000 tokens, 256 nodes 222 us (512 blocks), 260 373 us (264).
    const uint64_t blocks = head_dim == 256 || tiles == 1 ? 256 : 512;
    // a table of few steps has no use for more parts than steps
    const uint64_t steps = (capacity + kStepKeys - 1) / kStepKeys;
    const uint64_t parts = std::max<uint64_t>(1, std::min<uint64_t>(blocks / units, split * steps));
    w.bytes = parts * 2 * units * (16 * groups * (head_dim + 3) * 4) + 16;
    if (batch <= kPlanBatch) w.want_parts = static_cast<uint32_t>(parts);
    return w;
}

template <int HD, int NT>
int launch(fh_device *dev, const char *fn, const TreeArgs &a) {
    const dim3 grid(a.want_parts ? a.want_parts : a.batch, a.tiles, a.n_kv), threads(kTreeThreads);
    if (int rc = dispatch(dev, fn, [&] {
            hipLaunchKernelGGL((tree_part_kernel<HD, NT>), grid, threads, 0, dev->stream, a);
        }))
        return rc;
    if (a.want_parts <= 1) return FH_OK;
    constexpr uint32_t kRows = kTreeThreads / (HD / 4), kBlocks = (16 * NT + kRows - 1) / kRows;
    const dim3 join(a.batch, a.tiles * kBlocks, a.n_kv);
    return dispatch(dev, fn, [&] {
        hipLaunchKernelGGL((tree_join_kernel<HD, NT>), join, threads, 0, dev->stream, a);
    });
}

}  // namespace

extern "C" int fh_paged_tree_attention_workspace(int64_t batch, int64_t width, int64_t n_heads, int64_t n_kv,
                                                 int64_t head_dim, int64_t page_size, int64_t max_pages,
                                                 uint64_t *bytes) {
    const char *fn = "fh_paged_tree_attention_workspace";
    if (bytes == nullptr) return fail(FH_ERR_INVALID_ARGUMENT, "%s: bytes is null", fn);
    if (int rc = check_shape(fn, batch, width, n_heads, n_kv, head_dim, page_size, max_pages)) return rc;
    *bytes = plan(batch, width, n_heads, n_kv, head_dim, page_size, max_pages).bytes;
    return FH_OK;
}

extern "C" int fh_paged_tree_attention(fh_device *dev, const uint16_t *q, int64_t batch, int64_t width, int64_t n_heads,
                                       int64_t n_kv, int64_t head_dim, const uint16_t *k_pages,
                                       const uint16_t *v_pages, int64_t n_pages, int64_t page_size,
                                       const uint32_t *page_table, int64_t max_pages, const uint32_t *lengths,
                                       const uint32_t *counts, const uint32_t *masks, float scale, void *workspace,
                                       uint64_t workspace_bytes, uint16_t *out) {
    const char *fn = "fh_paged_tree_attention";
    if (int rc = check_usable(dev, fn)) return rc;
    if (int rc = check_shape(fn, batch, width, n_heads, n_kv, head_dim, page_size, max_pages)) return rc;
    if (int rc = fh_check_dims(fn, {n_pages})) return rc;
    if (int rc = check_pages(fn, n_pages, page_size, max_pages)) return rc;
    const float k = scale * 1.4426950408889634f;
    if (!(scale > 0.0f && k < INFINITY))
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: scale %g must be above 0 and at most 2e38", fn,
                    static_cast<double>(scale));
    if (batch == 0) return FH_OK;
    uint64_t need = 0;
    if (int rc = fh_paged_tree_attention_workspace(batch, width, n_heads, n_kv, head_dim, page_size, max_pages, &need))
        return rc;
    if (workspace_bytes < need)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: workspace of %llu bytes, %llu needed", fn,
                    (unsigned long long)workspace_bytes, (unsigned long long)need);
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) &
        15u)
        return fail(FH_ERR_INVALID_ARGUMENT, "%s: q, out and workspace must be 16-byte aligned", fn);
    if (int rc = check_words(
            fn, {{"page_table", page_table}, {"lengths", lengths}, {"counts", counts}, {"masks", masks}}))
        return rc;
    const uint64_t nodes = static_cast<uint64_t>(batch) * width, each = static_cast<uint64_t>(batch) * 4;
    const uint64_t rows = nodes * n_heads * head_dim * 2, bits = nodes * ((width + 31) / 32) * 4;
    uint64_t pool;
    if (int rc = check_pools(dev, fn, k_pages, v_pages, n_pages, n_kv, page_size, head_dim, page_table, batch,
                             max_pages, &pool))
        return rc;
    if (int rc = check_range(dev, workspace, need, fn, "workspace")) return rc;
    if (int rc = check_range(dev, q, rows, fn, "q")) return rc;
    if (int rc = check_range(dev, lengths, each, fn, "lengths")) return rc;
    if (counts)
        if (int rc = check_range(dev, counts, each, fn, "counts")) return rc;
    if (masks)
        if (int rc = check_range(dev, masks, bits, fn, "masks")) return rc;
    if (int rc = check_range(dev, out, rows, fn, "out")) return rc;
    for (const auto &[what, ptr, size] : {std::tuple{"out", static_cast<const void *>(out), rows},
                                          std::tuple{"workspace", static_cast<const void *>(workspace), need}})
        for (const auto &[with, p, n] :
             {std::tuple{"q", static_cast<const void *>(q), rows},
              std::tuple{"k_pages", static_cast<const void *>(k_pages), pool},
              std::tuple{"v_pages", static_cast<const void *>(v_pages), pool},
              std::tuple{"page_table", static_cast<const void *>(page_table), each * max_pages},
              std::tuple{"lengths", static_cast<const void *>(lengths), each},
              std::tuple{"counts", static_cast<const void *>(counts), each},
              std::tuple{"masks", static_cast<const void *>(masks), bits}})
            if (p)
                if (int rc = refuse_overlap(fn, what, ptr, size, with, p, n)) return rc;
    if (int rc = refuse_overlap(fn, "workspace", workspace, need, "out", out, rows)) return rc;
    if (int rc = set_current(dev, fn)) return rc;
    const Plan w = plan(batch, width, n_heads, n_kv, head_dim, page_size, max_pages);
    const TreeArgs a{q,
                     k_pages,
                     v_pages,
                     page_table,
                     lengths,
                     counts,
                     masks,
                     static_cast<uint32_t>(batch),
                     static_cast<uint32_t>(width),
                     static_cast<uint32_t>(n_heads),
                     static_cast<uint32_t>(n_kv),
                     static_cast<uint32_t>(n_pages),
                     static_cast<uint32_t>(max_pages),
                     static_cast<uint32_t>(max_pages * page_size),
                     Divider(static_cast<uint32_t>(n_heads / n_kv)),
                     Divider(static_cast<uint32_t>(page_size / 16)),
                     w.tiles,
                     w.want_parts,
                     k,
                     std::min(kSlack / k, std::numeric_limits<float>::max()),
                     static_cast<float *>(workspace),
                     out};
    if (head_dim == 64)
        return w.groups == 1 ? launch<64, 1>(dev, fn, a) : launch<64, 2>(dev, fn, a);
    if (head_dim == 128)
        return w.groups == 1 ? launch<128, 1>(dev, fn, a) : launch<128, 2>(dev, fn, a);
    return w.groups == 1 ? launch<256, 1>(dev, fn, a) : launch<256, 2>(dev, fn, a);
}
