// Low-rank adapters of many requests beside a shared projection (fh_lora_add).
#include <algorithm>
#include <tuple>
#include <type_traits>

#include "serving_checks.hpp"

namespace fh {

// The mathematics: y = base + (scale x A^T) B^T per row, with A, B and scale of
// the row's adapter. Two launches, since every column of y needs all of v =
// scale x A^T: lora_down_kernel leaves v's sums over ranges of k in the
// workspace, lora_up_kernel adds them in order and goes on to y. Both are bound
// by memory: x, base and y go through once, an adapter's A and B once per
// window of rows that uses it.
//
// Grouping: rows come with their adapters in any order, so a block takes a
// window of rows (64, or 256) and finds in it the groups of rows that share an
// adapter, by ballots over the adapter ids; each group is cut into chunks of up
// to 64 rows. Whatever the order, the products run on the matrix cores with the
// adapter's rows read once for up to 64 rows (four tiles of 16).
//
// Measured (down + up): 8 rows of 8 adapters, k 4096, n 6144, rank 16: 9.1 us,
// of which each launch has 4 at least; 200 rows of 48 adapters, n 28672, rank
// 16, f32 (98 MB): 28 us, 3.5 TB/s, a wavefront's few loads per 64 columns in
// flight; 4096 packed rows, n 4096, rank 32 (103 MB): 37 us, 2.8 TB/s, the
// latencies from ids to chunk to x or v before the stream begins; 754 packed
// rows, n 16384, rank 128, f32 (121 MB): 89 us (down 22, up 70), 1.4 TB/s, one
// wavefront per SIMD; 2000 rows of 40 adapters of rank 16, n 4096: 32 us by
// request, 84 in no order, as past kWideRows rows each 64 read their own.
typedef __attribute__((ext_vector_type(8))) __bf16 lo_bf16x8_t;
typedef __attribute__((ext_vector_type(4))) float lo_f32x4_t;

__device__ __forceinline__ lo_f32x4_t lo_mfma(uint4 a, uint4 b, lo_f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lo_bf16x8_t, a),
                                                   __builtin_bit_cast(lo_bf16x8_t, b), c, 0, 0, 0);
}

constexpr uint32_t kLoraThreads = 256;
constexpr uint32_t kLoraWaves = kLoraThreads / 64;
// Rows up to which a window is 256 rows (and an adapter that they share is
// read once for all of them).
constexpr uint32_t kWideRows = 1024;
// Blocks that the windows share, down and up. How many chunks a window has is
// known on the device alone: there its blocks divide the chunks among
// themselves, and each chunk's k (down) or columns (up) as far as they go round.
// With estimates of the host 1024 packed rows of rank 16 were left to 40 blocks:
// 36 us against 24. k is cut into kMaxSplits ranges at most, of kDownSteps steps
// of 32 per wavefront at least, a long one of up to kWideRows rows into more, of
// kLongSteps: k 14336, 71 rows of 5 adapters of rank 128: 51 -> 38 us, 8 rows of 8
// of rank 16: 11.7 -> 10.0; 1820 rows of 3 of rank 32: 39.2 -> 41.8, so not there.
constexpr uint32_t kDownBlocks = 512, kMaxSplits = 4, kDownSteps = 2, kLongSplits = 8, kLongSteps = 8;
// Up: 200 rows of 48 adapters of rank 16, of which the GPU holds 3 blocks per CU,
// take 28 us at 768 blocks, 31.8 at 512, 32.7 at 1024; 4096 packed rows of rank 32
// (2 per CU) 36.8 at 512, 40.1 at 768. Higher ranks take the same numbers: 1 per CU
// is held of most forms past rank 32, which run in up to three rounds.
constexpr uint32_t kUpBlocks = 768, kUpPacked = 512;

// The ranges of k of a window with `chunks` chunks and `blocks` blocks: `splits`
// of them, of kLoraWaves x `steps` x 32.
struct Ranges {
    uint32_t splits, steps;
};

__host__ __device__ __forceinline__ uint32_t most_splits(uint32_t k, uint32_t m) {
    const uint32_t all = (k + 31) / 32;
    const uint32_t n = (all + kLoraWaves * kDownSteps - 1) / (kLoraWaves * kDownSteps);
    const uint32_t more = m > kWideRows ? 0 : all / (kLoraWaves * kLongSteps);
    if (more > kMaxSplits) return more < kLongSplits ? more : kLongSplits;
    return n < kMaxSplits ? n : kMaxSplits;
}

__device__ __forceinline__ Ranges ranges_of(uint32_t k, uint32_t m, uint32_t chunks, uint32_t blocks) {
    const uint32_t all = (k + 31) / 32, want = min(max(blocks / max(chunks, 1u), 1u), most_splits(k, m));
    const uint32_t steps = (all + want * kLoraWaves - 1) / (want * kLoraWaves);
    return {(all + steps * kLoraWaves - 1) / (steps * kLoraWaves), steps};
}

// The rows of a window and its chunks. A row's rank is the number of rows
// before it with its adapter; rows of rank 0, 64, .. lead a chunk, and the
// chunks are numbered by their leaders' order. Ranks come from match masks,
// formed bit by bit of the ids: a ballot per bit and 64 rows, instead of a
// round per adapter (200 rows of 48 adapters: 181 -> 55 us, with the splits'
// sums requested together).
template <int Q>
struct Window {
    uint32_t id[Q];     // lane's rows' adapters
    uint64_t live[Q];   // rows that have one
    uint64_t leads[Q];  // chunk leaders
    uint32_t chunks;
};

// shared: Q words that the block's wavefronts exchange leaders through (Q > 1,
// when wavefront w works out those of rows 64 w .. 64 w + 63).
template <int Q>
__device__ __forceinline__ Window<Q> window_of(const uint32_t *adapters, uint32_t row0, uint32_t m, uint32_t n_adapters,
                                               uint32_t lane, uint32_t wave, uint64_t *shared) {
    Window<Q> o;
    uint64_t match[Q];
    uint32_t own = 0;
    bool alive = false;
    const int word = wave % Q;
#pragma unroll
    for (int w = 0; w < Q; ++w) {
        const uint32_t row = row0 + w * 64 + lane;
        o.id[w] = row < m ? adapters[row] : ~0u;
        match[w] = o.live[w] = __ballot(o.id[w] < n_adapters);
        if (Q == 1 || w == word) own = o.id[w], alive = o.id[w] < n_adapters;
    }
    for (uint32_t bit = 0; (n_adapters - 1) >> bit; ++bit) {
        const bool set = own >> bit & 1;
#pragma unroll
        for (int w = 0; w < Q; ++w) {
            const uint64_t have = __ballot(o.id[w] >> bit & 1);
            match[w] &= set ? have : ~have;
        }
    }
    uint32_t rank = 0;
#pragma unroll
    for (int w = 0; w < Q; ++w) {
        const uint64_t before = Q == 1 || w == word ? (1ull << lane) - 1 : w < word ? ~0ull : 0ull;
        rank += __builtin_popcountll(match[w] & before);
    }
    const uint64_t lead = __ballot(alive && rank % 64 == 0);
    o.chunks = 0;
    if constexpr (Q == 1) {
        o.leads[0] = lead;
        o.chunks = __builtin_popcountll(lead);
    } else {
        if (lane == 0 && wave < Q) shared[wave] = lead;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < Q; ++w) {
            const uint64_t v = shared[w];
            o.leads[w] = static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32))) << 32 |
                         static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v)));
            o.chunks += __builtin_popcountll(o.leads[w]);
        }
    }
    return o;
}

// Chunk `item` of the window: its adapter, its rows (in the window) in list[0
// .. rows), this wavefront's 64 bytes of LDS.
template <int Q>
__device__ __forceinline__ uint32_t chunk_of(const Window<Q> &o, uint32_t item, uint32_t lane, uint8_t *list,
                                             uint32_t &rows) {
    uint32_t id = 0, lead = 0, skip = item;
    bool found = false;
#pragma unroll
    for (int w = 0; w < Q; ++w) {
        const uint32_t here = __builtin_popcountll(o.leads[w]);
        if (!found && skip < here) {
            uint64_t bits = o.leads[w];
            for (uint32_t i = 0; i < skip; ++i) bits &= bits - 1;
            lead = __builtin_ctzll(bits);
            id = __builtin_amdgcn_readlane(o.id[w], lead);
            lead += w * 64;
            found = true;
        }
        if (!found) skip -= here;
    }
    // the leader's rank, then the rows of ranks from there on
    uint64_t mask[Q];
    uint32_t all = 0, first = 0;
#pragma unroll
    for (int w = 0; w < Q; ++w) {
        mask[w] = __ballot(o.id[w] == id);
        all += __builtin_popcountll(mask[w]);
        const uint64_t before = lead >= w * 64u + 64u ? ~0ull : lead > w * 64u ? (1ull << (lead - w * 64u)) - 1 : 0ull;
        first += __builtin_popcountll(mask[w] & before);
    }
    uint32_t before = 0;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int w = 0; w < Q; ++w) {
        const uint32_t at = before + __builtin_popcountll(mask[w] & ((1ull << lane) - 1)) - first;
        if ((mask[w] >> lane & 1) && at < 64) list[at] = static_cast<uint8_t>(w * 64 + lane);
        before += __builtin_popcountll(mask[w]);
    }
    __builtin_amdgcn_wave_barrier();
    rows = min(all - first, 64u);
    return id;
}

// v[split][row][r] = sum over the split's k of x[row, k] A[r, k], for a chunk of
// up to 16 RT rows. Each wavefront takes a quarter of the split's k for all the
// rows, so that A's rows come once per chunk; they add up in LDS in their order.
// A product has the ranks along its rows, so that a lane ends up with 4 ranks of
// a row. (With 16 rows and all the k to a wavefront A comes four times: 16.9 us
// against 15.5 for 4096 packed rows of k 4096, rank 32.)
template <int RT, int NR>
__device__ __forceinline__ void lora_down_chunk(const uint16_t *x, uint32_t k, uint64_t x_ld, const uint16_t *a,
                                                uint32_t rank, uint32_t k0, uint32_t k1, uint32_t row0, uint32_t rows,
                                                const uint8_t *list, float4 *sums, float *v, uint32_t lane,
                                                uint32_t wave) {
    constexpr int U = RT + NR <= 2 ? 8 : RT + NR <= 6 ? 4 : RT + NR <= 9 ? 2 : 1;  // steps of 32 requested together
    const uint32_t c = lane & 15u, q = lane >> 4;
    const uint16_t *xr[RT], *ar[NR];
#pragma unroll
    for (int t = 0; t < RT; ++t) xr[t] = x + (row0 + list[min(t * 16 + c, rows - 1)]) * x_ld;
#pragma unroll
    for (int t = 0; t < NR; ++t) ar[t] = a + static_cast<uint64_t>(min(t * 16 + c, rank - 1)) * k;
    lo_f32x4_t acc[RT][NR];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[t][r] = lo_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t s = k0; s < k1; s += 32 * U) {
        uint4 xf[U][RT], af[U][NR];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t at = min(s + u * 32 + q * 8, k - 8);  // clamped: the pieces past k1 are zeroed below
#pragma unroll
            for (int t = 0; t < RT; ++t) xf[u][t] = *reinterpret_cast<const uint4 *>(xr[t] + at);
#pragma unroll
            for (int t = 0; t < NR; ++t) af[u][t] = *reinterpret_cast<const uint4 *>(ar[t] + at);
        }
        if (s + 32 * U > k1) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (s + u * 32 + q * 8 >= k1) {
#pragma unroll
                    for (int t = 0; t < RT; ++t) xf[u][t] = make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int t = 0; t < NR; ++t) af[u][t] = make_uint4(0, 0, 0, 0);
                }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int r = 0; r < NR; ++r) acc[t][r] = lo_mfma(af[u][r], xf[u][t], acc[t][r]);
    }
    // wavefront w adds to what those before it left; the last one's sums go out
    for (uint32_t w = 0; w < kLoraWaves; ++w) {
        if (w == wave) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    float4 f = make_float4(acc[t][r][0], acc[t][r][1], acc[t][r][2], acc[t][r][3]);
                    if (w) {
                        const float4 o = sums[(t * NR + r) * 64 + lane];
                        f = make_float4(o.x + f.x, o.y + f.y, o.z + f.z, o.w + f.w);
                    }
                    if (w + 1 < kLoraWaves)
                        sums[(t * NR + r) * 64 + lane] = f;
                    else if (t * 16 + c < rows && r * 16 + q * 4 < rank)
                        *reinterpret_cast<float4 *>(v + static_cast<uint64_t>(row0 + list[t * 16 + c]) * rank + r * 16 +
                                                    q * 4) = f;
                }
        }
        __syncthreads();
    }
}

// Grid (windows, blocks of a window): neighbouring blocks run on different XCDs,
// and a window may have fewer units than blocks (the other way round 4096 packed
// rows' down products ran on 4 of 8).
template <int Q, int NR>
__global__ __launch_bounds__(kLoraThreads) void lora_down_kernel(const uint16_t *__restrict__ x, uint32_t m, uint32_t k,
                                                                 uint64_t x_ld, const uint16_t *__restrict__ a,
                                                                 uint32_t n_adapters, uint32_t rank,
                                                                 const uint32_t *__restrict__ adapters,
                                                                 float *__restrict__ v) {
    __shared__ uint8_t lists[kLoraWaves][64];
    __shared__ uint64_t leads[Q];
    __shared__ float4 sums[4 * NR * 64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row0 = blockIdx.x * 64 * Q;
    const Window<Q> o = window_of<Q>(adapters, row0, m, n_adapters, lane, wave, leads);
    const Ranges g = ranges_of(k, m, o.chunks, gridDim.y);
    for (uint32_t unit = blockIdx.y; unit < o.chunks * g.splits; unit += gridDim.y) {
        const uint32_t split = unit % g.splits;
        const uint32_t k0 = min((split * kLoraWaves + wave) * g.steps * 32, k), k1 = min(k0 + g.steps * 32, k);
        float *to = v + static_cast<uint64_t>(split) * m * rank;
        uint32_t rows;
        const uint32_t id = chunk_of<Q>(o, unit / g.splits, lane, lists[wave], rows);
        const uint16_t *au = a + static_cast<uint64_t>(id) * rank * k;
        if (rows <= 16)
            lora_down_chunk<1, NR>(x, k, x_ld, au, rank, k0, k1, row0, rows, lists[wave], sums, to, lane, wave);
        else
            lora_down_chunk<4, NR>(x, k, x_ld, au, rank, k0, k1, row0, rows, lists[wave], sums, to, lane, wave);
    }
}

// 16 neighbouring values of a row of base, as they lie in memory.
template <typename T>
struct Raw16 {
    uint4 w[sizeof(T)];
};

// Requests them from an aligned row.
template <typename T>
__device__ __forceinline__ Raw16<T> request16(const T *p) {
    Raw16<T> r;
#pragma unroll
    for (uint32_t i = 0; i < sizeof(T); ++i) r.w[i] = reinterpret_cast<const uint4 *>(p)[i];
    return r;
}

template <typename T>
__device__ __forceinline__ void floats16(const Raw16<T> &raw, float (&f)[16]) {
#pragma unroll
    for (uint32_t i = 0; i < sizeof(T); ++i) {
        if constexpr (sizeof(T) == 2) {
            float h[8];
            unpack8(raw.w[i], h);
#pragma unroll
            for (int e = 0; e < 8; ++e) f[i * 8 + e] = h[e];
        } else {
            f[i * 4] = __uint_as_float(raw.w[i].x), f[i * 4 + 1] = __uint_as_float(raw.w[i].y);
            f[i * 4 + 2] = __uint_as_float(raw.w[i].z), f[i * 4 + 3] = __uint_as_float(raw.w[i].w);
        }
    }
}

template <typename T>
__device__ __forceinline__ void store16(T *p, const float (&f)[16]) {
    if constexpr (sizeof(T) == 2) {
        uint32_t w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = f32x2_to_bf16x2_rne(f[2 * e], f[2 * e + 1]);
        reinterpret_cast<uint4 *>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4 *>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            reinterpret_cast<float4 *>(p)[i] = make_float4(f[i * 4], f[i * 4 + 1], f[i * 4 + 2], f[i * 4 + 3]);
    }
}

// Parts of two values in bf16: 0 the values rounded, 1 and 2 what the parts before
// have lost, rounded (nothing of an inf or NaN). A finite value past the largest bf16
// begins with that one, as its rounding would be inf.
__device__ __forceinline__ uint32_t parts_of(float x, float y, uint32_t part) {
    constexpr float kLargest = 0x1.FEp127f;
    auto first = [](float v) { return fabsf(v) < INFINITY ? fminf(fmaxf(v, -kLargest), kLargest) : v; };
    uint32_t p = f32x2_to_bf16x2_rne(first(x), first(y));
#pragma unroll
    for (uint32_t i = 1; i <= 2; ++i) {
        if (i > part) break;
        const float x0 = bf(p & 0xFFFFu), y0 = bf(p >> 16);
        x = fabsf(x0) < INFINITY ? x - x0 : 0.0f;
        y = fabsf(y0) < INFINITY ? y - y0 : 0.0f;
        p = f32x2_to_bf16x2_rne(x, y);
    }
    return p;
}

// A lane's terms of v: of each 16 ranks its 8 as part 0 or 1 (q & 1), and for
// f32 results part 2 (as the second product of the same B; zero where q & 1).
// f32 results take 24 bits of v. bf16 ones take 16: what those lose, 2^-16 of a
// term, is far below the half step of 2^-8 that B's own entry is off by, and with
// 24 2000 packed rows of rank 64 took 42 us instead of 32, others 5% less to 14% more.
template <typename T, int NJ>
struct Terms {
    uint4 v[NJ];
    uint4 low[sizeof(T) == 4 ? NJ : 1];
};

template <typename T>
constexpr uint32_t kParts = sizeof(T) == 4 ? 3 : 2;

// v B^T of 16 rows and 64 columns. A product has 16 of the columns along its
// rows and the rows along its columns, so that a lane holds 4 columns of row c
// per product; along its 32 terms lie 16 ranks, 8 at a time as (first part,
// second part) of v. WIDE: the columns of the
// four products are taken so that a lane's 16 are neighbours (from q * 16 on),
// else product t has columns 16 t .. 16 t + 15 and a lane 4 from t * 16 + q * 4.
template <int NJ, bool WIDE>
__device__ __forceinline__ void request_b(const uint16_t *b, uint32_t rank, uint32_t n, uint32_t col0, uint32_t c,
                                          uint32_t q, uint4 (&f)[4][NJ]) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const uint32_t col = min(col0 + (WIDE ? c / 4 * 16 + t * 4 + c % 4 : t * 16 + c), n - 1);
        const uint16_t *br = b + static_cast<uint64_t>(col) * rank;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
            f[t][j] = *reinterpret_cast<const uint4 *>(br + min((2 * j + q / 2) * 8, rank - 8));
    }
}

// APART: infs and NaNs of B meet v's first part alone (a rest has the other sign,
// or is 0, as it falls: with it an infinite sum would be NaN), and none that lies
// past the ranks, where v is 0 and what stands for B need not be.
template <bool APART, typename T, int NJ>
__device__ __forceinline__ void sum_products(const uint4 (&bfr)[4][NJ], const Terms<T, NJ> &vf, uint32_t rank,
                                             uint32_t q, lo_f32x4_t (&acc)[4]) {
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[u] = lo_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            uint4 f = bfr[u][j], rest = f;
            if constexpr (APART) {
                // here and now, one after the other: ahead of the loops around it would take twice B's registers
                asm volatile("" : "+v"(rest.x), "+v"(rest.y), "+v"(rest.z), "+v"(rest.w));
                __builtin_amdgcn_sched_barrier(0);
                clear_specials(rest);
                if ((q & 1) || (2 * j + q / 2) * 8 >= rank) f = rest;
            }
            if constexpr (sizeof(T) == 4) acc[u] = lo_mfma(rest, vf.low[j], acc[u]);
            acc[u] = lo_mfma(f, vf.v[j], acc[u]);
        }
}

// Infs and NaNs of B are looked for in the sums, fewer than its entries: an inf or
// NaN among a wavefront's, or sums that large, and they are formed again, apart
// (finite ones are the same again).
template <typename T, int NJ>
__device__ __forceinline__ void products(const uint4 (&bfr)[4][NJ], const Terms<T, NJ> &vf, uint32_t rank, uint32_t q,
                                         lo_f32x4_t (&acc)[4]) {
    sum_products<false>(bfr, vf, rank, q, acc);
    float all = 0.0f;
#pragma unroll
    for (int u = 0; u < 4; ++u) all += (fabsf(acc[u][0]) + fabsf(acc[u][1])) + (fabsf(acc[u][2]) + fabsf(acc[u][3]));
    if (__any(!(all < INFINITY))) sum_products<true>(bfr, vf, rank, q, acc);
}

template <typename T>
__device__ __forceinline__ T plus(T base, float d) {
    if constexpr (sizeof(T) == 2)
        return rne(bf(base) + d);
    else
        return base + d;
}

// Up to R rows of a chunk through LDS (tile: this wavefront's), `tiles` times 64
// columns: a lane has one column of each row, so that rows are read and written
// in whole lines whatever their alignment and however few they are. The first 64
// columns are requested before terms() forms the lane's terms of v, with AHEAD
// the next 64 before a tile's products.
template <typename T, int NJ, int R>
struct RowsTile {
    uint4 b[4][NJ];
    T base[R];
};

template <typename T, int NJ, int R, bool AHEAD, typename Form>
__device__ __forceinline__ void lora_up_rows(const uint16_t *b, uint32_t rank, uint32_t n, const T *base,
                                             uint64_t base_ld, T *y, uint64_t y_ld, uint32_t mine, uint32_t rows,
                                             uint32_t col0, uint32_t tiles, float (*tile)[68], uint32_t lane,
                                             Form terms) {
    const uint32_t c = lane & 15u, q = lane >> 4;
    Terms<T, NJ> vf;
    auto row = [&](int i) {
        return static_cast<uint64_t>(__builtin_amdgcn_readlane(mine, min(i, static_cast<int>(rows) - 1)));
    };
    auto request = [&](RowsTile<T, NJ, R> &x, uint32_t u) {
        const uint32_t at = col0 + min(u, tiles - 1) * kLoraWaves * 64;
        request_b<NJ, false>(b, rank, n, at, c, q, x.b);
#pragma unroll
        for (int i = 0; i < R; ++i) x.base[i] = (base + row(i) * base_ld)[min(at + lane, n - 1)];
    };
    auto finish = [&](const RowsTile<T, NJ, R> &x, uint32_t u) {
        const uint32_t col = col0 + u * kLoraWaves * 64 + lane;
        lo_f32x4_t acc[4];
        products(x.b, vf, rank, q, acc);
        // 8 rows at a time
#pragma unroll
        for (int h = 0; h < R; h += 8) {
            if (h >= static_cast<int>(rows)) break;
            if (c / 8 == h / 8)
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    *reinterpret_cast<lo_f32x4_t *>(&tile[c % 8][t * 16 + q * 4]) = acc[t];
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = h; i < h + 8 && i < R; ++i)
                if (i < static_cast<int>(rows) && col < n)
                    (y + row(i) * y_ld)[col] = plus(x.base[i], tile[i - h][lane]);
            __builtin_amdgcn_wave_barrier();
        }
    };
    RowsTile<T, NJ, R> one, two;
    request(one, 0);
    terms(vf);
    if constexpr (!AHEAD) {
        for (uint32_t u = 0; u < tiles; ++u) {
            if (u) request(one, u);
            finish(one, u);
        }
        return;
    }
    for (uint32_t u = 0; u < tiles; u += 2) {
        request(two, u + 1);
        finish(one, u);
        if (u + 1 >= tiles) break;
        request(one, u + 2);
        finish(two, u + 1);
    }
}

// Grid (windows, blocks of a window): neighbouring blocks run on different XCDs,
// and a window may have fewer units than blocks (the other way round 4096 packed
// rows' down products ran on 4 of 8). v is formed in LDS from the splits' sums:
// for a chunk of up to 16 rows by each wavefront for itself, with no barrier,
// else once for the block. wide: there a lane reads and writes 16 neighbouring
// columns of a row (n a multiple of 16, rows 16-byte aligned). SPLITS: as many
// as k has at most, whose sums are requested together.
template <typename T, int Q, int NJ, bool PACKED, uint32_t SPLITS>
__global__ __launch_bounds__(kLoraThreads) void lora_up_kernel(const float *__restrict__ v, uint32_t down_blocks,
                                                               uint32_t m, uint32_t k, const uint16_t *__restrict__ b,
                                                               const float *__restrict__ scales, uint32_t n_adapters,
                                                               uint32_t rank, uint32_t n,
                                                               const uint32_t *__restrict__ adapters, const T *base,
                                                               uint64_t base_ld, T *y, uint64_t y_ld, bool wide) {
    constexpr int P = sizeof(T) == 2 ? 4 : 2;       // row tiles requested together
    constexpr bool kAhead = !PACKED && NJ <= 2;     // the registers hold two tiles of B
    __shared__ uint8_t lists[kLoraWaves][64];
    __shared__ uint64_t leads[Q];
    __shared__ __attribute__((aligned(16))) uint16_t vs[64 * (kParts<T> * 16 * NJ + 8)];
    __shared__ __attribute__((aligned(16))) float tile[kLoraWaves][8][68];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, row0 = blockIdx.x * 64 * Q;
    const uint32_t c = lane & 15u, q = lane >> 4, vs_ld = kParts<T> * rank + 8, quads = rank / 4;
    const uint64_t split = static_cast<uint64_t>(m) * rank;
    const Window<Q> o = window_of<Q>(adapters, row0, m, n_adapters, lane, wave, leads);
    const uint32_t splits = ranges_of(k, m, o.chunks, down_blocks).splits;
    // a chunk's columns in `parts` parts of `tiles` times 64 per wavefront
    const uint32_t all = (n + kLoraWaves * 64 - 1) / (kLoraWaves * 64);
    const uint32_t tiles = (all + min(max(gridDim.y / max(o.chunks, 1u), 1u), all) - 1) /
                           min(max(gridDim.y / max(o.chunks, 1u), 1u), all);
    const uint32_t parts = (all + tiles - 1) / tiles;
    for (uint32_t unit = blockIdx.y; unit < o.chunks * parts; unit += gridDim.y) {
        const uint32_t col0 = (unit % parts * tiles * kLoraWaves + wave) * 64;  // then every kLoraWaves-th tile
        uint32_t rows;
        const uint8_t *list = lists[wave];
        const uint32_t id = chunk_of<Q>(o, unit / parts, lane, lists[wave], rows);
        const float scale = scales[id];
        const uint16_t *bu = b + static_cast<uint64_t>(id) * n * rank;
        const bool few = rows <= 16;
        uint16_t *terms_of = few ? vs + wave * 16 * vs_ld : vs;
        if (!few) __syncthreads();  // other wavefronts may still read theirs, of a chunk before
        auto fill = [&](uint32_t from, uint32_t by) {
            for (uint32_t i = from; i < rows * quads; i += by) {
                const uint32_t member = i / quads, r = i % quads * 4;
                const float *p = v + static_cast<uint64_t>(row0 + list[member]) * rank + r;
                float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                float4 part[SPLITS];
#pragma unroll
                for (uint32_t u = 0; u < SPLITS; ++u)
                    part[u] = *reinterpret_cast<const float4 *>(p + min(u, splits - 1) * split);
#pragma unroll
                for (uint32_t u = 0; u < SPLITS; ++u)
                    if (u < splits) f[0] += part[u].x, f[1] += part[u].y, f[2] += part[u].z, f[3] += part[u].w;
#pragma unroll
                for (uint32_t h = 0; h < kParts<T>; ++h)
                    *reinterpret_cast<uint2 *>(terms_of + member * vs_ld + h * rank + r) =
                        make_uint2(parts_of(f[0] * scale, f[1] * scale, h), parts_of(f[2] * scale, f[3] * scale, h));
            }
        };
        auto terms = [&](uint32_t member, Terms<T, NJ> &vf) {
            const uint16_t *of = terms_of + min(member, rows - 1) * vs_ld;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const uint32_t r = (2 * j + q / 2) * 8, at = min(r, rank - 8);
                vf.v[j] = *reinterpret_cast<const uint4 *>(of + (q & 1) * rank + at);
                if (r >= rank) vf.v[j] = make_uint4(0, 0, 0, 0);
                if constexpr (sizeof(T) == 4) {
                    vf.low[j] = *reinterpret_cast<const uint4 *>(of + 2 * rank + at);
                    if (r >= rank || (q & 1)) vf.low[j] = make_uint4(0, 0, 0, 0);
                }
            }
        };
        if (few) {
            if (col0 >= n) continue;
            const uint32_t mine = row0 + list[min(c, rows - 1)];
            auto form = [&](Terms<T, NJ> &vf) {
                fill(lane, 64);
                __builtin_amdgcn_wave_barrier();
                terms(c, vf);
                __builtin_amdgcn_wave_barrier();
            };
            if (!PACKED && rows <= 4)
                lora_up_rows<T, NJ, 4, kAhead>(bu, rank, n, base, base_ld, y, y_ld, mine, rows, col0, tiles, tile[wave],
                                               lane, form);
            else if (!PACKED && rows <= 8)
                lora_up_rows<T, NJ, 8, kAhead>(bu, rank, n, base, base_ld, y, y_ld, mine, rows, col0, tiles, tile[wave],
                                               lane, form);
            else
                lora_up_rows<T, NJ, 16, false>(bu, rank, n, base, base_ld, y, y_ld, mine, rows, col0, tiles, tile[wave],
                                               lane, form);
            continue;
        }
        fill(threadIdx.x, kLoraThreads);
        __syncthreads();
        if (!wide || (!PACKED && NJ == 1)) {
            for (uint32_t t = 0; t * 16 < rows && col0 < n; ++t)
                lora_up_rows<T, NJ, 16, false>(bu, rank, n, base, base_ld, y, y_ld,
                                               row0 + list[min(t * 16 + c, rows - 1)], min(rows - t * 16, 16u), col0,
                                               tiles, tile[wave], lane,
                                               [&](Terms<T, NJ> &vf) { terms(t * 16 + c, vf); });
        } else {
            for (uint32_t u = 0; u < tiles; ++u) {
                const uint32_t first = col0 + u * kLoraWaves * 64;
                if (first >= n) break;
                uint4 bfr[4][NJ];
                request_b<NJ, true>(bu, rank, n, first, c, q, bfr);
                const uint32_t col = min(first + q * 16, n - 16);  // the last ones twice where n ends before
                for (uint32_t t0 = 0; t0 * 16 < rows; t0 += P) {
                    Raw16<T> raw[P];
#pragma unroll
                    for (int t = 0; t < P; ++t) {
                        const uint64_t row = row0 + list[min((t0 + t) * 16 + c, rows - 1)];
                        raw[t] = request16(base + row * base_ld + col);
                    }
#pragma unroll
                    for (int t = 0; t < P; ++t) {
                        const uint32_t member = (t0 + t) * 16 + c;
                        Terms<T, NJ> vf;
                        terms(member, vf);
                        lo_f32x4_t acc[4];
                        products(bfr, vf, rank, q, acc);
                        float f[16];
                        floats16(raw[t], f);
#pragma unroll
                        for (int e = 0; e < 16; ++e) f[e] += acc[e / 4][e % 4];
                        if (member < rows && first + q * 16 < n)
                            store16(y + static_cast<uint64_t>(row0 + list[member]) * y_ld + col, f);
                    }
                }
            }
        }
        __syncthreads();  // vs is read
    }
    // rows without an adapter are base, where y is not: in runs of kBareCols columns, to the blocks in turn
    // from the last one on, which have the fewest units
    if (y == base) return;
    constexpr uint32_t kBareLoads = 8, kBareCols = kBareLoads * kLoraThreads;
    const uint32_t runs = (n + kBareCols - 1) / kBareCols;
    uint32_t turn = gridDim.y - 1 - blockIdx.y;  // this block's next run
#pragma unroll
    for (int w = 0; w < Q; ++w) {
        const uint32_t here = m - row0 > w * 64u ? min(m - row0 - w * 64u, 64u) : 0;
        const uint64_t bare = ~o.live[w] & (here < 64 ? (1ull << here) - 1 : ~0ull);
        const uint32_t turns = __builtin_popcountll(bare) * runs;
        for (; turn < turns; turn += gridDim.y) {
            uint64_t left = bare;
            for (uint32_t i = 0; i < turn / runs; ++i) left &= left - 1;
            const uint64_t row = row0 + w * 64 + __builtin_ctzll(left);
            const uint32_t at = turn % runs * kBareCols + threadIdx.x;
            T held[kBareLoads];
#pragma unroll
            for (uint32_t i = 0; i < kBareLoads; ++i) held[i] = base[row * base_ld + min(at + i * kLoraThreads, n - 1)];
#pragma unroll
            for (uint32_t i = 0; i < kBareLoads; ++i)
                if (at + i * kLoraThreads < n) y[row * y_ld + at + i * kLoraThreads] = held[i];
        }
        turn -= turns;
    }
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
    // fewer rows never need more: what serves the largest batch serves them all
    const uint32_t m32 = static_cast<uint32_t>(m), k32 = static_cast<uint32_t>(k), wide = std::min(m32, kWideRows);
    const uint64_t rows = std::max<uint64_t>(static_cast<uint64_t>(most_splits(k32, m32)) * m32,
                                             static_cast<uint64_t>(most_splits(k32, wide)) * wide);
    *bytes = rows * rank * 4 + 16;
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
        if (int rc = refuse_overlap(fn, what, ptr, size, "scales", scales, static_cast<uint64_t>(n_adapters) * 4))
            return rc;
    }
    if (int rc = refuse_overlap(fn, "workspace", workspace, need, "y", y, y_bytes)) return rc;
    if (int rc = refuse_overlap(fn, "workspace", workspace, need, "base", base, base_bytes)) return rc;
    const uint32_t quads = m > 64 && m <= kWideRows ? 4 : 1, rows_of = 64 * quads;
    const uint64_t windows = (rows + rows_of - 1) / rows_of, cols = (n + kLoraWaves * 64 - 1) / (kLoraWaves * 64);
    if (windows > 65535) return fail(FH_ERR_INDEX_TOO_LARGE, "%s: m %lld", fn, (long long)m);
    if (int rc = set_current(dev, fn)) return rc;
    const uint32_t m32 = static_cast<uint32_t>(m), k32 = static_cast<uint32_t>(k);
    // a window has at most as many chunks as rows
    const uint64_t most = std::min<uint64_t>(rows, rows_of);
    const uint32_t down_blocks = static_cast<uint32_t>(
        std::clamp<uint64_t>(kDownBlocks / windows, 1, most * most_splits(k32, m32)));
    const uint64_t up_all = m > kWideRows ? kUpPacked : kUpBlocks;
    const uint32_t up_blocks = static_cast<uint32_t>(std::clamp<uint64_t>(up_all / windows, 1, most * cols));
    const dim3 down(static_cast<uint32_t>(windows), down_blocks), up(static_cast<uint32_t>(windows), up_blocks);
    const dim3 threads(kLoraThreads);
    float *v = static_cast<float *>(workspace);
    const uint32_t n32 = static_cast<uint32_t>(n);
    const uint32_t rank32 = static_cast<uint32_t>(rank), u32 = static_cast<uint32_t>(n_adapters);
    const bool wide = ((reinterpret_cast<uintptr_t>(base) | reinterpret_cast<uintptr_t>(y)) & 15u) == 0 &&
                     base_ld * elem % 16 == 0 && y_ld * elem % 16 == 0 && n % 16 == 0;
    auto run_down = [&](auto kernel) {
        return dispatch(dev, fn, [&] {
            hipLaunchKernelGGL(kernel, down, threads, 0, dev->stream, x, m32, k32, static_cast<uint64_t>(x_ld), a, u32,
                               rank32, adapters, v);
        });
    };
    auto run_up = [&](auto kernel, auto *of) {
        using T = std::remove_pointer_t<decltype(of)>;
        return dispatch(dev, fn, [&] {
            hipLaunchKernelGGL(kernel, up, threads, 0, dev->stream, v, down_blocks, m32, k32, b, scales, u32, rank32,
                               n32, adapters, static_cast<const T *>(base), static_cast<uint64_t>(base_ld),
                               static_cast<T *>(y), static_cast<uint64_t>(y_ld), wide);
        });
    };
    // rank tiles of 16: 1, 2, 4 or 8
    auto run = [&](auto q, auto tiles) {
        constexpr int Q = decltype(q)::value, N = decltype(tiles)::value;
        if (int rc = run_down(lora_down_kernel<Q, N>)) return rc;
        auto run_as = [&](auto packed, auto splits) {
            constexpr bool P = decltype(packed)::value;
            constexpr uint32_t S = decltype(splits)::value;
            return dtype == FH_F32 ? run_up(lora_up_kernel<float, Q, N, P, S>, static_cast<float *>(nullptr))
                                   : run_up(lora_up_kernel<uint16_t, Q, N, P, S>, static_cast<uint16_t *>(nullptr));
        };
        constexpr std::integral_constant<uint32_t, kMaxSplits> few{};
        constexpr std::integral_constant<uint32_t, kLongSplits> many{};
        // windows of 64 rows past kWideRows rows: mostly whole chunks of 64
        if constexpr (Q == 1)
            if (m > kWideRows) return run_as(std::true_type{}, few);
        return most_splits(k32, m32) > kMaxSplits ? run_as(std::false_type{}, many) : run_as(std::false_type{}, few);
    };
    auto by_rank = [&](auto q) {
        if (rank <= 16) return run(q, std::integral_constant<int, 1>{});
        if (rank <= 32) return run(q, std::integral_constant<int, 2>{});
        if (rank <= 64) return run(q, std::integral_constant<int, 4>{});
        return run(q, std::integral_constant<int, 8>{});
    };
    return quads == 4 ? by_rank(std::integral_constant<int, 4>{}) : by_rank(std::integral_constant<int, 1>{});
}
