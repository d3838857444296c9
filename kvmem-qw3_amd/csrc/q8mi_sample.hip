// Sampling of one token per row of logits by temperature, top-k, top-p and min-p from a given uniform number.
//
// The three cuts keep a prefix of the row's ranks (logit descending, index ascending), so what is kept is known from its
// last rank: a key (the logit's bits in an order-preserving form) and the index of the last element with that key.
// Weights are p = exp((logit - max) / temperature) rounded to multiples of 2^-42: sums are 64-bit integers, exact and
// free of their order, so that neither the split of a row nor the arrival of atomics moves a border.
//
// No sort of the row.  Four launches, the first three over (spans of chunks of 1024 logits) x rows:
//   1  largest logit of each quarter of a chunk; clears the row's counters
//   2  where top_k is no more than the chunks (or, up to 128, half of their quarters): the top_k-th largest of the maxima is no
//      larger than the top_k-th logit, so the few logits from it up are collected.  Otherwise the weights: where nothing is cut but by min-p, their sum per
//      chunk, else a histogram of count and weight over 1024 steps of 1/32 in (max - logit) / temperature (what lies 31.9
//      and more below the maximum weighs nothing)
//   3  the histogram says in which steps the cuts fall: the few logits of those steps are collected, what lies above them
//      is kept for certain and summed per chunk
//   4  one workgroup a row ranks the collected logits, takes the cuts in them, finds the chunk that holds the drawn element
//      and walks it
// Bound by the launches' latency for one row (248320 logits, top_k 20 and top_p: 2.8 + 5.2 + 2.1 + 6.8 us; top_p alone 23 us in
// all, at temperature 1), for many by the 64-bit weights and the histograms (64 rows: 26 us by top_k 40 of 151936, 33 us by
// temperature alone, 71 us by top_p of 248320 at temperature 1; reading those once takes 11).
// A row with more than 4096 logits to collect (thousands of equal ones, a temperature that levels all) is searched by the
// fourth launch's workgroup alone, digit by digit of the ranks.
#include "q8mi_device.hpp"
#include "q8mi_internal.hpp"

namespace q8mi {
namespace {

constexpr uint32_t kMaxVocab = 1u << 20;
constexpr uint32_t kChunk = 1024;                     // logits
constexpr uint32_t kMaxChunks = kMaxVocab / kChunk;
// Chunks of a workgroup: one while that leaves CUs idle, up to these where rows are many.  In launches 2 and 3 a span clears a
// histogram and sends it off, or adds one up, once for all its chunks, while long spans leave the chip unevenly loaded by rows
// of unlike settings (64 rows of 248320 by top_p, spans of 4, 8, 12: 81, 77, 81 us); launch 1 holds nothing (spans of 2, 4: 1 us
// apart).
constexpr uint32_t kMostSpan = 8, kMostSpanOfBest = 2;
constexpr uint32_t kGridWanted = 512;                 // spans above one begin at twice this many workgroups
constexpr uint32_t kAhead = 4;                        // chunks that a workgroup of launches 1 to 3 loads at a time
constexpr uint32_t kChunkThreads = kChunk / 4;
constexpr uint32_t kRowThreads = 256;                 // launch 4
constexpr uint32_t kBins = 1024;
constexpr double kBinsPerUnit = 32.0;
constexpr double kReach = 31.875;                     // exp(-31.875) * 2^42 rounds to 0
constexpr uint32_t kMaxCandidates = 4096;             // of a row
constexpr uint32_t kChunkCandidates = 64;             // of a chunk
constexpr uint32_t kFewRanks = 128;                   // up to this top_k, quarters of chunks bound it as well
constexpr double kOne = 4398046511104.0;              // 2^42: the weight of the largest logit; 2^20 of them sum below 2^63
constexpr double kBottom = 64.0;                      // the depth of everything that is deeper, or never drawn
constexpr uint32_t kRoots = 32;                       // 2^(i / 32): 256 bytes, so that no two of them share a bank of LDS

typedef unsigned long long u64;
typedef float v4f __attribute__((ext_vector_type(4)));

// Where the cuts fall: steps below `sure` are kept, steps sure .. last hold the last rank, steps k_first .. k_last the
// top_k-th (kBins: top_k cuts nothing); the weight of the steps below `sure`, below k_first, and of all; the count below
// k_first.
struct Cut {
    uint32_t sure, last, k_first, k_last, k_count;
    u64 sure_mass, k_mass, all_mass;
};

struct Row;
struct SampleParams {
    const float *logits;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    q8mi_argmax_pair *out;
    u64 *chunk_mass;    // [row][chunk]: weight kept for certain
    u64 *bin_mass;      // [row][copy][kBins]
    u64 *candidates;    // [row][chunk][kChunkCandidates]: key << 32 | ~index, in any order
    Cut *cut;           // [row] (launch 2 or 3)
    Row *rows;          // [row]
    uint32_t *best;     // [row][chunk][quarter]: largest key
    uint32_t *top;      // [row]: largest key (launch 2)
    uint32_t *listed;   // [row]: launch 2 has collected everything from rank 0 to the cuts
    uint32_t *bin_count;     // [row][copy][kBins]
    uint32_t *n_candidates;  // [row][chunk]: may be beyond kChunkCandidates
    uint32_t vocab, stride, chunks;
    uint32_t span;           // chunks of a workgroup (launches 1 to 3)
    uint32_t copies;         // of a row's histogram
    int vec;
};

// Order-preserving bits of a logit; NaN and -inf (never drawn) come below every number as 0.
__device__ __forceinline__ uint32_t key_of(float v) {
    if (!(v > -INFINITY)) return 0;
    const uint32_t u = __builtin_bit_cast(uint32_t, v == 0.0f ? 0.0f : v);   // -0 ties with +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7fffffffu : ~key);
}
__device__ __forceinline__ u64 rank_of(uint32_t key, uint32_t index) {   // larger comes first
    return static_cast<u64>(key) << 32 | (0xffffffffu - index);
}

// A row's settings as the launches use them; worked out once, by launch 1.
struct Row {
    double max;        // launches 2 to 4
    double per_unit;   // 1 / temperature, above zero
    double deepest;    // what min_p keeps lies no deeper: p >= min_p <=> depth <= -log(min_p)
    double top_p;      // 1: off
    double far;        // a cut by weight alone lies above this depth
    uint32_t top_k;    // 0: off
    uint32_t greedy;
};
__device__ __forceinline__ Row settings_of(const SampleParams &p, uint32_t row) {
    Row r{};
    const float t = p.temperature ? p.temperature[row] : 1.0f;
    r.greedy = !(t > 0.0f);
    // an infinite temperature: depths below 1e-250, which no other one gives, where p is 1 and -inf still lies at the bottom
    r.per_unit = r.greedy ? 1.0 : fmax(1.0 / static_cast<double>(t), 1e-300);
    const float min_p = p.min_p ? p.min_p[row] : 0.0f;
    r.deepest = min_p > 0.0f ? (min_p < 1.0f ? -log(static_cast<double>(min_p)) : 1e-250) : INFINITY;
    const int32_t k = p.top_k ? p.top_k[row] : 0;
    r.top_k = k > 0 && static_cast<uint32_t>(k) < p.vocab ? k : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f;
    r.top_p = top_p < 1.0f ? top_p : 1.0;
    // the largest weighs 1, so 1 - top_p may always be dropped, and `vocab` logits below a depth whose weight is
    // (1 - top_p) / vocab, less the half step that rounding may add to it, cannot hold the cut
    const double spare = (1.0 - r.top_p) / p.vocab - 0.5 / kOne;
    r.far = spare > 0.0 ? fmin(kReach, 0.1 - log(spare)) : kReach;
    return r;
}
__device__ __forceinline__ Row row_of(const SampleParams &p, uint32_t row, uint32_t top_key) {
    Row r = p.rows[row];
    r.max = logit_of(top_key);
    return r;
}
// How far below the maximum, in temperatures, 0 .. kBottom.  NaN and -inf lie at the bottom; below +inf, it itself is the only
// number that does not (inf - inf is no number, whose larger with 0 is 0).
__device__ __forceinline__ double depth_at(float v, const Row &r) {
    return fmin(fmax((r.max - static_cast<double>(fmaxf(v, -INFINITY))) * r.per_unit, 0.0), kBottom);
}
__device__ __forceinline__ double depth_of(uint32_t key, const Row &r) { return depth_at(key ? logit_of(key) : -INFINITY, r); }

// The table of weight_at, worked out anew from the series of the exponential (0 gives 1 exactly): 16 dependent steps, where
// fetching it from memory cost each launch 2 us.  A barrier follows before the first weight.
__device__ __forceinline__ void make_roots(double *roots) {
    if (threadIdx.x >= kRoots) return;
    const double x = threadIdx.x * (0.693147180559945309417 / kRoots);
    double e = 1.0;
#pragma unroll
    for (int k = 16; k > 0; --k) e = fma(x * (1.0 / k), e, 1.0);
    roots[threadIdx.x] = e;
}

// exp(-depth) * 2^42 rounded to an integer: 2^(y / 32), y = 32 * (42 - depth * log2(e)) = 32 n + i + f with -1/2 <= f <= 1/2,
// is 2^n from the exponent, 2^(i / 32) from the table and 2^(f / 32) from its series (terms up to the 5th power: 2e-15).
// Adding 1.5 * 2^52 leaves 32 n + i in the sum's low bits, adding 2^52 the rounded integer.  Off by 1e-14 of itself and the
// last rounding; depth 0 gives 2^42.  About 25 instructions, less than half of a series over a whole binade (64 rows of 151936
// by temperature alone: 41 -> 34 us).
__device__ __forceinline__ u64 weight_at(double depth, const double *roots) {
    constexpr double kHead = 6755399441055744.0, kLn = 0.693147180559945309417 / kRoots;
    const double y = fma(depth, -1.44269504088896340736 * kRoots, 42.0 * kRoots), head = y + kHead, f = y - (head - kHead);
    const int k = static_cast<int>(__builtin_bit_cast(u64, head));
    double e = kLn * kLn * kLn * kLn * kLn / 120.0;
    e = fma(e, f, kLn * kLn * kLn * kLn / 24.0);
    e = fma(e, f, kLn * kLn * kLn / 6.0);
    e = fma(e, f, kLn * kLn / 2.0);
    e = fma(e, f, kLn);
    e = fma(e, f, 1.0) * roots[k & (kRoots - 1)];
    const u64 scaled = __builtin_bit_cast(u64, e) + (static_cast<u64>(static_cast<uint32_t>(k >> 5) << 20) << 32);
    return __builtin_bit_cast(u64, __builtin_bit_cast(double, scaled) + 4503599627370496.0) - 0x4330000000000000ull;
}
__device__ __forceinline__ u64 kept_weight_at(double depth, const Row &r, const double *roots) {
    return depth <= r.deepest ? weight_at(depth, roots) : 0;
}
__device__ __forceinline__ uint32_t bin_at(double depth) { return static_cast<uint32_t>(depth * kBinsPerUnit); }

// v + what a cross-lane move brings to the rows of 16 lanes in ROWS (0 where nothing comes).
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp_add(u64 v) {
    const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), CTRL, ROWS, 0xf, false);
    return v + (static_cast<u64>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo));
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
    v = dpp_add<kDppXor1, 0xf>(v);
    v = dpp_add<kDppXor2, 0xf>(v);
    v = dpp_add<kDppRowHalfMirror, 0xf>(v);
    v = dpp_add<kDppRowMirror, 0xf>(v);
    u64 all = 0;
#pragma unroll
    for (int row = 0; row < 64; row += 16)
        all += static_cast<u64>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), row))) << 32 |
               static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), row));
    return all;
}
__device__ __forceinline__ u64 wave_max_u64(u64 v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u64 o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}
// Sum of v over the threads below this one, and of all (`part`: one u64 a wave of LDS).
template <uint32_t THREADS>
__device__ __forceinline__ u64 sum_below(u64 v, u64 *part, u64 &all) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    u64 upto = v;
    upto = dpp_add<0x111, 0xf>(upto);   // one lane below, two, four, eight, within rows of 16 lanes
    upto = dpp_add<0x112, 0xf>(upto);
    upto = dpp_add<0x114, 0xf>(upto);
    upto = dpp_add<0x118, 0xf>(upto);
    upto = dpp_add<0x142, 0xa>(upto);   // the last lane of rows 0 and 2 to the rows behind them
    upto = dpp_add<0x143, 0xc>(upto);   // lane 31 to rows 2 and 3
    __syncthreads();
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    u64 before = 0;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < THREADS / kWave; ++w) {
        before += w < wave ? part[w] : 0;
        all += part[w];
    }
    return before + upto - v;
}

// Four logits from element i (a multiple of 4) of a row; those past its end are -inf.
__device__ __forceinline__ v4f load4(const SampleParams &p, const float *x, uint32_t i) {
    if (p.vec && i + 4 <= p.vocab) return *reinterpret_cast<const v4f *>(x + i);
    auto one = [&](uint32_t k) {
        const float v = x[k < p.vocab ? k : p.vocab - 1];
        return k < p.vocab ? v : -INFINITY;
    };
    return v4f{one(i), one(i + 1), one(i + 2), one(i + 3)};
}
// Register u of four by selection: what works on them is written once in a loop and not four times in a row.  Code is
// fetched, too: the four launches fit the 64 KiB instruction cache together, so that a call finds what the last one left
// (108 KB unrolled: the last launch alone took 10.9 us of one row, now 6.9).
__device__ __forceinline__ v4f pick(const v4f (&v)[4], uint32_t u) {
    const v4f a = v[0], b = v[1], c = v[2], d = v[3];   // selected as values, so that they stay in registers
    return u == 0 ? a : u == 1 ? b : u == 2 ? c : d;
}
__device__ __forceinline__ void unpack(v4f t, float (&v)[4]) { v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w; }

// A workgroup's span of chunks, kAhead chunks in registers and the next ones asked for before those in hand are looked at.
// `early`: the first are asked for when the object is made, before it is known what the row wants of them.
struct Span {
    const SampleParams &p;
    const float *x;
    uint32_t first, end;
    bool early;
    v4f v[kAhead];

    __device__ __forceinline__ Span(const SampleParams &params, const float *row, bool at_once) : p(params), x(row), early(at_once) {
        first = blockIdx.x * p.span;
        end = first + p.span < p.chunks ? first + p.span : p.chunks;
#pragma unroll
        for (uint32_t u = 0; u < kAhead; ++u) {
            v[u] = v4f{0, 0, 0, 0};
            if (early && first + u < end) v[u] = load4(p, x, (first + u) * kChunk + threadIdx.x * 4);
        }
    }
    // f(v, i, c) for every four logits v, from element i, that this thread has of the span's chunk c (counted from 0), of
    // the chunks that want(c); no others are read from here on
    template <typename F, typename W>
    __device__ __forceinline__ void walk(F f, W want) {
        if (!early) {   // uniform
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u)
                if (first + u < end && want(u)) v[u] = load4(p, x, (first + u) * kChunk + threadIdx.x * 4);
        }
#pragma unroll 1
        for (uint32_t c = first; c < end; c += kAhead) {
            v4f next[kAhead] = {};
            if (c + kAhead < end) {
#pragma unroll
                for (uint32_t u = 0; u < kAhead; ++u) {
                    const uint32_t n = c + kAhead + u;
                    if (n < end && want(n - first)) next[u] = load4(p, x, n * kChunk + threadIdx.x * 4);   // uniform
                }
            }
#pragma unroll 1
            for (uint32_t u = 0; u < kAhead && c + u < end; ++u) {
                if (!want(c + u - first)) continue;   // uniform
                float four[4];
                unpack(pick(v, u), four);
                f(four, (c + u) * kChunk + threadIdx.x * 4, c + u - first);
            }
#pragma unroll
            for (uint32_t u = 0; u < kAhead; ++u) v[u] = next[u];
        }
    }
    template <typename F>
    __device__ __forceinline__ void walk(F f) { walk(f, [](uint32_t) { return true; }); }
};
static_assert(kAhead == 4, "pick() takes one of four");

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto larger = [](uint32_t a, int b) { return a > static_cast<uint32_t>(b) ? a : static_cast<uint32_t>(b); };
    v = larger(v, dpp_i32<kDppXor1>(static_cast<int>(v)));
    v = larger(v, dpp_i32<kDppXor2>(static_cast<int>(v)));
    v = larger(v, dpp_i32<kDppRowHalfMirror>(static_cast<int>(v)));
    v = larger(v, dpp_i32<kDppRowMirror>(static_cast<int>(v)));
    const uint32_t a = larger(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16));
    return larger(larger(a, __builtin_amdgcn_readlane(v, 32)), __builtin_amdgcn_readlane(v, 48));
}

// ---- 1 ----------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(kChunkThreads) void sample_best_kernel(const SampleParams p) {
    const uint32_t t = threadIdx.x, row = blockIdx.y;
    Span span(p, p.logits + static_cast<uint64_t>(row) * p.stride, true);
    if (blockIdx.x < p.copies) {
        const uint64_t first = (static_cast<uint64_t>(row) * p.copies + blockIdx.x) * kBins;
        for (uint32_t b = t; b < kBins; b += kChunkThreads) {
            p.bin_mass[first + b] = 0;
            p.bin_count[first + b] = 0;
        }
        if (blockIdx.x == 0 && t == 0) {
            p.listed[row] = 0;
            p.rows[row] = settings_of(p, row);
        }
    }
    span.walk([&](const float (&v)[4], uint32_t, uint32_t c) {
        const uint32_t key = wave_max_u32(key_of(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]))));   // of a number and NaN, the number
        if (t % kWave == 0) p.best[(static_cast<uint64_t>(row) * p.chunks + span.first + c) * 4 + t / kWave] = key;
    });
}

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
// The largest key of a row's chunk c.
__device__ __forceinline__ uint32_t best_of(const SampleParams &p, uint32_t row, uint32_t c) {
    const v4u q = *reinterpret_cast<const v4u *>(p.best + (static_cast<uint64_t>(row) * p.chunks + c) * 4);
    const uint32_t a = q.x > q.y ? q.x : q.y, b = q.z > q.w ? q.z : q.w;
    return a > b ? a : b;
}

// Sums and candidates of a span's chunks on their way out of a workgroup.
struct ChunkSpace {   // LDS
    u64 mass[kMostSpan][kChunkThreads / kWave];
    double roots[kRoots];
    uint32_t n[kMostSpan], best[kMostSpan];
};
// Clears it and fetches the chunks' maxima; a barrier follows.
__device__ __forceinline__ void open_space(ChunkSpace &s, const Span &span, const SampleParams &p, uint32_t row) {
    const uint32_t t = threadIdx.x;
    if (t >= kMostSpan) return;
    s.n[t] = 0;
    s.best[t] = span.first + t < span.end ? best_of(p, row, span.first + t) : 0;
#pragma unroll
    for (uint32_t w = 0; w < kChunkThreads / kWave; ++w) s.mass[t][w] = 0;
}
// The elements (bits of `mine`) of the four logits v from element i on go to their chunk's list, c-th of the span.
__device__ __forceinline__ void collect(const SampleParams &p, uint32_t row, ChunkSpace &s, const float (&v)[4], uint32_t i, uint32_t c,
                                        uint32_t mine) {
    if (mine == 0) return;
    uint32_t at = atomicAdd(&s.n[c], static_cast<uint32_t>(__popc(mine)));
    u64 *list = p.candidates + (static_cast<uint64_t>(row) * p.chunks + i / kChunk) * kChunkCandidates;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
        if (mine >> k & 1) {
            if (at < kChunkCandidates) list[at] = rank_of(key_of(v[k]), i + k);
            ++at;
        }
}

// The largest key, in its upper 20 bits, that k of the maxima which at(0 .. count - 1) gives reach (0: none): bit by bit, from
// the first in which they differ.  One wave finds it for the workgroup.
template <uint32_t N, typename F>
__device__ __forceinline__ uint32_t reached_by(F at, uint32_t count, uint32_t k, uint32_t &shared) {
    if (threadIdx.x < kWave) {
        uint32_t keys[N], most = 0, inverse = 0;
#pragma unroll
        for (uint32_t u = 0; u < N; ++u) {
            const uint32_t c = u * kWave + threadIdx.x;
            keys[u] = c < count ? at(c) : 0;
            most = keys[u] > most ? keys[u] : most;
            inverse = c < count && ~keys[u] > inverse ? ~keys[u] : inverse;
        }
        most = wave_max_u32(most);
        inverse = wave_max_u32(inverse);
        const uint32_t differ = (most ^ ~inverse) | 1u << 11;
        uint32_t bit = 0x80000000u >> __clz(differ), least = most & ~(2 * bit - 1);
#pragma unroll 1
        for (; bit >= 1u << 12; bit >>= 1) {
            uint32_t reach = 0;
#pragma unroll
            for (uint32_t u = 0; u < N; ++u) reach += __popcll(__builtin_amdgcn_ballot_w64(keys[u] >= (least | bit)));
            if (reach >= k) least |= bit;
        }
        if (threadIdx.x == 0) shared = least;
    }
    __syncthreads();
    return shared;
}

// ---- 2 ----------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(kChunkThreads) void sample_weigh_kernel(const SampleParams p) {
    __shared__ u64 mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ u64 part[kChunkThreads / kWave];
    __shared__ ChunkSpace out;
    __shared__ uint32_t found, tops[kChunkThreads / kWave];
    const uint32_t t = threadIdx.x, row = blockIdx.y;
    Row r = p.rows[row];
    Span span(p, p.logits + static_cast<uint64_t>(row) * p.stride, p.span == 1);
    open_space(out, span, p, row);
    // the row's largest key
    uint32_t top = 0;
    for (uint32_t c = t; c < p.chunks; c += kChunkThreads) {
        const uint32_t key = best_of(p, row, c);
        top = key > top ? key : top;
    }
    top = wave_max_u32(top);
    if (t % kWave == 0) tops[t / kWave] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kChunkThreads / kWave; ++w) top = tops[w] > top ? tops[w] : top;
    if (blockIdx.x == 0 && t == 0) p.top[row] = top;
    r.max = logit_of(top);
    if ((top == 0) | (r.greedy != 0)) return;
    // quarters: of fewer than kFewRanks chunks then; half as many ranks as quarters make few candidates (1000 rows of
    // 32000, top_k 40: 125 -> 86 us; one row 23.7 -> 18.2)
    const bool by_chunks = r.top_k <= p.chunks, by_quarters = r.top_k <= 2 * p.chunks && r.top_k <= kFewRanks;
    if (r.top_k != 0 && (by_chunks || by_quarters)) {
        auto chunk = [&](uint32_t c) { return best_of(p, row, c); };
        auto quarter = [&](uint32_t c) { return p.best[static_cast<uint64_t>(row) * p.chunks * 4 + c]; };
        const uint32_t least = !by_chunks ? reached_by<4 * kFewRanks / kWave>(quarter, 4 * p.chunks, r.top_k, found)
                               : p.chunks <= 4 * kWave ? reached_by<4>(chunk, p.chunks, r.top_k, found)
                                                       : reached_by<kMaxChunks / kWave>(chunk, p.chunks, r.top_k, found);
        if (least != 0) {
            if (blockIdx.x == 0 && t == 0) {
                Cut cut{};
                cut.last = cut.k_last = kBins - 1;
                p.cut[row] = cut;
                p.listed[row] = 1;
            }
            const float least_logit = logit_of(least);
            span.walk([&](const float (&v)[4], uint32_t i, uint32_t c) {
                uint32_t mine = 0;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) mine |= v[k] >= least_logit ? 1u << k : 0;
                collect(p, row, out, v, i, c, mine);
            }, [&](uint32_t c) { return out.best[c] >= least; });
            __syncthreads();
            if (span.first + t < span.end) p.n_candidates[static_cast<uint64_t>(row) * p.chunks + span.first + t] = out.n[t];
            return;
        }
    }
    const bool by_count = r.top_k != 0, by_mass = r.top_p < 1.0;   // each needs its half of the histogram
    if (by_count || by_mass) {
        for (uint32_t b = t; b < kBins; b += kChunkThreads) { mass[b] = 0; count[b] = 0; }
        make_roots(out.roots);
        __syncthreads();
        // The row's steps are added up by atomics, so few are sent.  Where this span alone has top_k above a step, the cut
        // lies above it, too.  Without top_k, it does not lie below r.far: from there on only the sum counts, in the last
        // step, which no logit reaches.
        const double far = by_count ? kReach : r.far;
        // The top_k-th largest of the maxima of quarters of chunks, where they are that many, is a bound as well: what lies
        // below it is not looked at (64 rows of 248320, top_k 400: 80 -> 72 us).
        uint32_t least = 0;
        if (by_count && r.top_k <= 4 * p.chunks && 4 * p.chunks <= 16 * kWave)
            least = reached_by<16>([&](uint32_t c) { return p.best[static_cast<uint64_t>(row) * p.chunks * 4 + c]; }, 4 * p.chunks, r.top_k, found);
        const float least_logit = least ? logit_of(least) : -INFINITY;
        u64 rest = 0;
        span.walk([&](const float (&v)[4], uint32_t, uint32_t) {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                if (!(v[k] >= least_logit)) continue;
                const double depth = depth_at(v[k], r);
                if (!(depth < kReach)) continue;
                const uint32_t b = bin_at(depth);
                if (by_count) atomicAdd(&count[b], 1u);
                if (!by_mass) continue;
                const u64 w = weight_at(depth, out.roots);
                if (depth < far) atomicAdd(&mass[b], w);
                else rest += w;
            }
        }, [&](uint32_t c) { return out.best[c] >= least; });
        rest = wave_sum_u64(rest);
        if (t % kWave == 0 && rest != 0) atomicAdd(&mass[kBins - 1], rest);
        __syncthreads();
        uint32_t mine[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) mine[k] = count[4 * t + k];
        u64 all, before = by_count ? sum_below<kChunkThreads>((mine[0] + mine[1]) + (mine[2] + mine[3]), part, all) : 0;
        const uint64_t first = (static_cast<uint64_t>(row) * p.copies + blockIdx.x % p.copies) * kBins;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const uint32_t b = 4 * t + k;
            if (by_count && before >= r.top_k) break;
            if (mine[k] != 0) atomicAdd(&p.bin_count[first + b], mine[k]);
            if (mass[b] != 0) atomicAdd(&p.bin_mass[first + b], mass[b]);
            before += mine[k];
        }
        return;
    }
    make_roots(out.roots);
    __syncthreads();
    span.walk([&](const float (&v)[4], uint32_t, uint32_t c) {
        u64 sum = 0;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) sum += kept_weight_at(depth_at(v[k], r), r, out.roots);
        sum = wave_sum_u64(sum);
        if (t % kWave == 0) out.mass[c][t / kWave] = sum;
    });
    __syncthreads();
    if (span.first + t < span.end)
        p.chunk_mass[static_cast<uint64_t>(row) * p.chunks + span.first + t] = (out.mass[t][0] + out.mass[t][1]) + (out.mass[t][2] + out.mass[t][3]);
}

struct CutSpace {   // LDS
    u64 mass_upto[kBins];
    u64 part[kRowThreads / kWave];
    uint32_t found[3], k_count;
};
// Every thread of the workgroup calls it; the first kBins / 4 hold four steps each.
template <uint32_t THREADS>
__device__ __forceinline__ Cut find_cut(const SampleParams &p, uint32_t row, const Row &r, CutSpace &s) {
    constexpr uint32_t kHolders = kBins / 4;
    static_assert(THREADS >= kHolders, "four steps a thread");
    const uint32_t t = threadIdx.x;
    const bool holds = t < kHolders;
    u64 m[4] = {}, c[4] = {}, all_mass, all_count;
    if (holds) {
        const uint64_t first = static_cast<uint64_t>(row) * p.copies * kBins + 4 * t;
#pragma unroll 4
        for (uint32_t i = 0; i < p.copies; ++i) {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                m[k] += p.bin_mass[first + i * kBins + k];
                c[k] += p.bin_count[first + i * kBins + k];
            }
        }
    }
    if (t == 0) { s.found[0] = s.found[1] = s.found[2] = kBins; s.k_count = 0; }
    u64 m_before = r.top_p < 1.0 ? sum_below<THREADS>((m[0] + m[1]) + (m[2] + m[3]), s.part, all_mass) : 0;
    u64 c_before = r.top_k != 0 ? sum_below<THREADS>((c[0] + c[1]) + (c[2] + c[3]), s.part, all_count) : 0;
    const u64 m_first = m_before;
    __syncthreads();
    if (holds) {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            if (r.top_k != 0 && c_before < r.top_k && c_before + c[k] >= r.top_k) {   // one thread's one step
                s.found[0] = 4 * t + k;
                s.k_count = static_cast<uint32_t>(c_before);
            }
            c_before += c[k];
            m_before += m[k];
            s.mass_upto[4 * t + k] = m_before;
        }
    }
    __syncthreads();
    Cut cut{};
    cut.k_first = cut.k_last = cut.sure = cut.last = s.found[0];
    cut.k_count = s.k_count;
    if (r.top_p < 1.0) {
        // the weight that top_k keeps lies between these two; so does the last rank that top_p keeps
        const u64 hi = s.mass_upto[cut.k_first < kBins ? cut.k_first : kBins - 1];
        const u64 lo = cut.k_first == kBins ? hi : cut.k_first ? s.mass_upto[cut.k_first - 1] : 0;
        const double limit_lo = r.top_p * static_cast<double>(lo), limit_hi = r.top_p * static_cast<double>(hi);
        if (holds) {
            u64 b = m_first;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {   // the step that reaches a limit: one thread's
                const u64 e = b + m[k];
                const bool first = 4 * t + k == 0;   // rank 0 lies in step 0 and always stays
                if ((first || static_cast<double>(b) < limit_lo) && static_cast<double>(e) >= limit_lo) s.found[1] = 4 * t + k;
                if ((first || static_cast<double>(b) < limit_hi) && static_cast<double>(e) >= limit_hi) s.found[2] = 4 * t + k;
                b = e;
            }
        }
        __syncthreads();
        cut.sure = s.found[1] < cut.k_first ? s.found[1] : cut.k_first;
        cut.last = s.found[2] < cut.k_first ? s.found[2] : cut.k_first;
        cut.sure_mass = cut.sure ? s.mass_upto[cut.sure - 1] : 0;
        cut.k_mass = lo;
        cut.all_mass = s.mass_upto[kBins - 1];
    }
    return cut;
}

// ---- 3 ----------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(kChunkThreads) void sample_collect_kernel(const SampleParams p) {
    __shared__ CutSpace space;
    __shared__ ChunkSpace out;
    const uint32_t t = threadIdx.x, row = blockIdx.y;
    Span span(p, p.logits + static_cast<uint64_t>(row) * p.stride, p.span == 1);
    open_space(out, span, p, row);   // find_cut's barriers follow
    const uint32_t top = p.top[row];
    const Row r = row_of(p, row, top);
    if (top == 0 || r.greedy || !(r.top_k != 0 || r.top_p < 1.0)) return;
    if (p.listed[row]) return;
    make_roots(out.roots);
    const Cut cut = find_cut<kChunkThreads>(p, row, r, space);
    if (blockIdx.x == 0 && t == 0) p.cut[row] = cut;
    // logits well below the last step of interest need no 64-bit depth
    const uint32_t deep = cut.k_first < kBins ? cut.k_first : cut.last;
    const double reach = (deep + 1) / kBinsPerUnit / r.per_unit;
    const float least = r.max < INFINITY && reach < 1e30 ? static_cast<float>(r.max - reach - (fabs(r.max) + reach) * 1e-6) : -INFINITY;
    span.walk([&](const float (&v)[4], uint32_t i, uint32_t c) {
        u64 sum = 0;
        uint32_t mine = 0;   // elements to collect
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            if (!(v[k] >= least)) continue;
            const double depth = depth_at(v[k], r);
            if (!(depth < kReach)) continue;
            const uint32_t b = bin_at(depth);
            if (b < cut.sure) sum += kept_weight_at(depth, r, out.roots);
            else if (b <= cut.last || b == cut.k_first) mine |= 1u << k;
        }
        collect(p, row, out, v, i, c, mine);
        if (__builtin_amdgcn_ballot_w64(sum != 0) != 0) sum = wave_sum_u64(sum);   // uniform
        if (t % kWave == 0) out.mass[c][t / kWave] = sum;
    }, [&](uint32_t c) { return out.best[c] != 0 && logit_of(out.best[c]) >= least; });
    __syncthreads();
    if (span.first + t < span.end) {
        const uint64_t at = static_cast<uint64_t>(row) * p.chunks + span.first + t;
        p.chunk_mass[at] = (out.mass[t][0] + out.mass[t][1]) + (out.mass[t][2] + out.mass[t][3]);
        p.n_candidates[at] = out.n[t];
    }
}

// ---- 4 ----------------------------------------------------------------------------------------------------------------
struct DrawSpace {   // LDS
    u64 cand[kMaxCandidates];
    u64 part[kRowThreads / kWave];
    u64 chunk_mass[kMaxChunks];
    u64 mass[256], result[2];
    uint32_t count[256];
    u64 target;
    uint32_t at, bounds[2];
    double roots[kRoots];
};

// Sorts the first n of x, larger first: a bitonic network over 1024 numbers, four neighbouring ones a thread.  Partners meet in
// registers, by lane exchange (33 of the 55 steps), or, 256 and 512 apart, through x.  About 4 us; the search by digits that
// takes over beyond 1024 needs about 12.
constexpr uint32_t kSorted = 4 * kRowThreads;
__device__ __forceinline__ void sort_down(u64 *x, uint32_t n) {
    const uint32_t t = threadIdx.x;
    u64 v[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) v[i] = 4 * t + i < n ? x[4 * t + i] : 0;
    auto order = [](u64 &a, u64 &b, bool down) {
        const u64 more = a > b ? a : b, less = a > b ? b : a;
        a = down ? more : less;
        b = down ? less : more;
    };
    order(v[0], v[1], true);
    order(v[2], v[3], false);
#pragma unroll 1
    for (uint32_t k = 4; k <= kSorted; k *= 2) {
        const bool down = (4 * t & k) == 0;
        uint32_t j = k / 2;
#pragma unroll 1
        for (; j >= 4; j /= 2) {
            const bool take_more = ((4 * t & j) == 0) == down;
            u64 other[4];
            if (j >= 4 * kWave) {   // uniform
                __syncthreads();
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) x[4 * t + i] = v[i];
                __syncthreads();
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) other[i] = x[(4 * t ^ j) + i];
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) other[i] = __shfl_xor(v[i], static_cast<int>(j / 4));
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) v[i] = (v[i] > other[i]) == take_more ? v[i] : other[i];
        }
        order(v[0], v[2], down);
        order(v[1], v[3], down);
        order(v[0], v[1], down);
        order(v[2], v[3], down);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) x[4 * t + i] = v[i];
}

__global__ __launch_bounds__(kRowThreads) void sample_draw_kernel(const SampleParams p) {
    __shared__ DrawSpace s;
    const uint32_t t = threadIdx.x, row = blockIdx.x;
    const float *x = p.logits + static_cast<uint64_t>(row) * p.stride;
    // Everything the earlier launches left, asked for at once: the counts and the first two candidates of this thread's four
    // chunks (most have no more), and the chunks' sums.  What a row's settings did not write is not looked at.
    const uint32_t top = p.top[row];
    const bool may_cut = p.top_k != nullptr || p.top_p != nullptr;
    uint32_t of[4] = {};
    u64 two[4][2] = {}, left[4] = {};
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        const uint64_t c = static_cast<uint64_t>(row) * p.chunks + 4 * t + k;
        if (4 * t + k >= p.chunks) continue;
        left[k] = p.chunk_mass[c];
        if (!may_cut) continue;   // uniform
        of[k] = p.n_candidates[c];
        two[k][0] = p.candidates[c * kChunkCandidates];
        two[k][1] = p.candidates[c * kChunkCandidates + 1];
    }
    const Cut cut = p.cut[row];
    float u = p.uniform[row];
    const Row r = row_of(p, row, top);
    const uint32_t is_listed = p.listed[row];
    if ((top == 0) | (r.greedy != 0)) {   // both are asked for before either is looked at
        if (top == 0) {
            if (t == 0) p.out[row] = q8mi_argmax_pair{-INFINITY, -1};
            return;
        }
        // the first chunk with that key, its first such element
        if (t == 0) s.at = kMaxChunks;
        __syncthreads();
        for (uint32_t c = t; c < p.chunks; c += kRowThreads)
            if (best_of(p, row, c) == top) atomicMin(&s.at, c);
        if (t == 0) s.bounds[0] = 0xffffffffu;
        __syncthreads();
        const uint32_t i = s.at * kChunk + 4 * t;
        float v[4];
        unpack(load4(p, x, i), v);
        uint32_t k = 0;
        while (k < 4 && key_of(v[k]) != top) ++k;
        if (k < 4) atomicMin(&s.bounds[0], i + k);
        __syncthreads();
        if (k < 4 && s.bounds[0] == i + k) p.out[row] = q8mi_argmax_pair{x[i + k], static_cast<int32_t>(i + k)};
        return;
    }
    make_roots(s.roots);   // sum_below's barriers follow
    const bool cuts = r.top_k != 0 || r.top_p < 1.0;
    const bool listed = cuts && is_listed != 0;
    // the candidates of the chunks, one list after the other; `whole`: more than their places hold
    uint32_t n = 0;
    bool whole = false;
    if (cuts) {
        u64 sum = 0, all;   // candidates; from bit 32 on, chunks with more than two; from bit 48 on, with more than their list holds
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) sum += of[k] + (of[k] > 2 ? 1ull << 32 : 0) + (of[k] > kChunkCandidates ? 1ull << 48 : 0);
        uint32_t at = static_cast<uint32_t>(sum_below<kRowThreads>(sum, s.part, all));
        n = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(all));   // loops to it are scalar
        const uint32_t flags = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(all >> 32));
        whole = flags >> 16 != 0 || n > kMaxCandidates;
        if (!whole) {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                s.chunk_mass[4 * t + k] = static_cast<u64>(of[k]) << 32 | at;   // for what follows here alone
                if (of[k] > 0) s.cand[at] = two[k][0];
                if (of[k] > 1) s.cand[at + 1] = two[k][1];
                at += of[k];
            }
            if (flags != 0) {   // the others: sixteen lanes a chunk, four chunks of theirs asked for at once
                __syncthreads();
                const uint32_t lane = threadIdx.x % 16;
#pragma unroll 1
                for (uint32_t c0 = t / 16; c0 < p.chunks; c0 += 4 * (kRowThreads / 16)) {
                    u64 place[4], got[4];
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u) {
                        const uint32_t c = c0 + u * (kRowThreads / 16);
                        place[u] = c < p.chunks ? s.chunk_mass[c] : 0;
                        if (2 + lane < place[u] >> 32)
                            got[u] = p.candidates[(static_cast<uint64_t>(row) * p.chunks + c) * kChunkCandidates + 2 + lane];
                    }
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u) {
                        const uint32_t c = c0 + u * (kRowThreads / 16), count = place[u] >> 32, to = static_cast<uint32_t>(place[u]);
                        if (2 + lane < count) s.cand[to + 2 + lane] = got[u];
                        for (uint32_t i = 18 + lane; i < count; i += 16)
                            s.cand[to + i] = p.candidates[(static_cast<uint64_t>(row) * p.chunks + c) * kChunkCandidates + i];
                    }
                }
            }
        }
        __syncthreads();
    }
    const bool summed = !listed && !whole;   // the earlier launches have left the chunks' sums
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) s.chunk_mass[4 * t + k] = summed ? left[k] : 0;
    u64 last = 0;   // rank of the last kept element: everything from it up is kept
    if (cuts && (whole || n > kSorted)) {
        // Many candidates, or more than the lists hold: then all logits of the row are.  The last rank that a cut keeps, of
        // the steps lo .. hi and from `after` up, is the one before which fewer than `limit` (by count or weight) come: eight
        // bits of the 64-bit ranks a walk, with counts and weights of the 256 values in LDS.  One loop around one walk, since
        // the code of a walk is long.
        uint32_t width = 64;   // digits are of rank - low: among the candidates, no more than their range has
        u64 low = 0;
        if (!whole) {
            u64 high = 0, inverse = 0;
            for (uint32_t c = t; c < n; c += kRowThreads) {
                high = s.cand[c] > high ? s.cand[c] : high;
                inverse = ~s.cand[c] > inverse ? ~s.cand[c] : inverse;
            }
            high = wave_max_u64(high);
            inverse = wave_max_u64(inverse);
            if (t % kWave == 0) { s.part[t / kWave] = high; s.mass[t / kWave] = inverse; }
            __syncthreads();
#pragma unroll
            for (uint32_t w = 0; w < kRowThreads / kWave; ++w) {
                high = s.part[w] > high ? s.part[w] : high;
                inverse = s.mass[w] > inverse ? s.mass[w] : inverse;
            }
            low = ~inverse;
            width = 64 - __clzll(high - low);   // candidates are more than one, and differ
            __syncthreads();
        }
        enum { kByCount, kSum, kByMass, kKeep };
        uint32_t stage = cut.k_first < kBins ? kByCount : r.top_p < 1.0 ? kByMass : kKeep;
        bool alone = false;        // one rank has the digits found so far: the rest of it at once
        uint32_t shift = width;    // found: the bits of rank - low from `shift` on
        u64 found = 0, before = 0, after = 0, sum = 0;
        u64 limit = r.top_k - cut.k_count;
        auto mass_limit = [&](u64 kept) {   // of a cut by weight, when top_k keeps `kept`
            const double limit_f = ceil(r.top_p * static_cast<double>(kept));
            return (limit_f > 1.0 ? static_cast<u64>(limit_f) : 1ull) - cut.sure_mass;   // rank 0 always stays
        };
        if (stage == kByMass) limit = mass_limit(cut.all_mass);
        for (;;) {   // everything that steers it is uniform
            const bool digits = stage == kByCount || stage == kByMass;
            const uint32_t lo = stage == kByCount ? cut.k_first : cut.sure, hi = stage == kByCount ? cut.k_last : cut.last;
            const uint32_t bits = shift < 8 ? shift : 8, next = shift - bits;
            if (digits && !alone) {
                s.mass[t] = 0;
                s.count[t] = 0;
                if (t == 0) { s.at = 0; s.result[0] = ~0ull; }
                __syncthreads();
            }
            auto visit = [&](u64 rank) {
                const double depth = depth_of(static_cast<uint32_t>(rank >> 32), r);
                const uint32_t b = depth < kReach ? bin_at(depth) : kBins - 1;
                if (digits) {
                    const u64 v = rank - low;
                    if (rank < after || (shift < 64 && v >> shift != found) || b < lo || b > hi) return;
                    if (alone) {
                        s.result[0] = v;
                        return;
                    }
                    const uint32_t digit = static_cast<uint32_t>(v >> next) & ((1u << bits) - 1);
                    atomicAdd(&s.count[digit], 1u);
                    if (stage == kByMass) atomicAdd(&s.mass[digit], weight_at(depth, s.roots));
                } else if (rank >= last) {
                    const u64 w = weight_at(depth, s.roots);
                    if (stage == kSum) sum += b >= cut.k_first ? w : 0;
                    else if (w != 0 && depth <= r.deepest) atomicAdd(&s.chunk_mass[(0xffffffffu - static_cast<uint32_t>(rank)) / kChunk], w);
                }
            };
            if (!whole) {
#pragma unroll 1
                for (uint32_t c = t; c < n; c += 4 * kRowThreads) {   // one wave a SIMD: four at a time hide each other's latency
                    u64 rank[4];
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u) rank[u] = c + u * kRowThreads < n ? s.cand[c + u * kRowThreads] : 0;
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u)
                        if (rank[u] != 0) visit(rank[u]);
                }
            } else {
#pragma unroll 1
                for (uint32_t i0 = 4 * t; i0 < p.vocab; i0 += 16 * kRowThreads) {
                    v4f v[4];
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u) {
                        const uint32_t i = i0 + u * 4 * kRowThreads;
                        v[u] = load4(p, x, i);
                    }
#pragma unroll 1
                    for (uint32_t u = 0; u < 4; ++u) {
                        float four[4];
                        unpack(pick(v, u), four);
                        const uint32_t i = i0 + u * 4 * kRowThreads;
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k)
                            if (key_of(four[k]) != 0) visit(rank_of(key_of(four[k]), i + k));
                    }
                }
            }
            __syncthreads();
            if (digits) {
                if (!alone) {
                    const uint32_t mine = 255 - t;   // larger digits come first
                    const uint32_t of = s.count[mine];
                    const u64 v = stage == kByMass ? s.mass[mine] : of;
                    u64 all;
                    const u64 upto = before + sum_below<kRowThreads>(v, s.part, all);
                    // where the limit is beyond all: the last value that occurs (atomics of a whole wave on one address would
                    // take 40 cycles a lane)
                    const u64 occurs = __builtin_amdgcn_ballot_w64(of != 0);
                    if (t % kWave == 0 && occurs != 0) atomicMax(&s.at, t + 63u - static_cast<uint32_t>(__builtin_clzll(occurs)));
                    if (upto < limit && upto + v >= limit) { s.result[0] = mine; s.result[1] = upto; }
                    __syncthreads();
                    if (s.result[0] == ~0ull && t == s.at) { s.result[0] = mine; s.result[1] = upto; }
                    __syncthreads();
                    alone = s.count[s.result[0]] == 1 && next != 0;
                    found = (shift < 64 ? found << bits : 0) | s.result[0];
                    before = s.result[1];
                    shift = next;
                    __syncthreads();
                    if (shift != 0) continue;
                } else {
                    found = s.result[0];
                    __syncthreads();
                }
                last = after = found + low;
                stage = stage == kByCount && r.top_p < 1.0 ? kSum : kKeep;
            } else if (stage == kSum) {
                u64 kept;
                (void)sum_below<kRowThreads>(sum, s.part, kept);
                limit = mass_limit(kept + cut.k_mass);
                stage = kByMass;
                alone = false;
                shift = width;
                found = 0;
                before = 0;
            } else {
                break;
            }
        }
    } else if (cuts) {
        if (n <= kRowThreads) {   // ranked by counting
            const u64 own = t < n ? s.cand[t] : 0;
            s.cand[kRowThreads + t] = own;
            __syncthreads();
            uint32_t above = 0;
#pragma unroll 8
            for (uint32_t i = 0; i < n; ++i) above += s.cand[kRowThreads + i] > own;
            if (t < n) s.cand[above] = own;   // ranks differ
        } else {
            sort_down(s.cand, n);
        }
        __syncthreads();
        // four neighbouring ranks a thread
        double depth[4];
        uint32_t step[4];
        u64 w[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const u64 own = 4 * t + k < n ? s.cand[4 * t + k] : 0;
            depth[k] = depth_of(static_cast<uint32_t>(own >> 32), r);
            step[k] = depth[k] < kReach ? bin_at(depth[k]) : kBins - 1;
            w[k] = weight_at(depth[k], s.roots);   // of no rank: 0
        }
        uint32_t kept = n;   // candidates that stay: a prefix of their ranks
        u64 mass_k = cut.all_mass, all;
        if (cut.k_first < kBins) {
            uint32_t first = 0;   // the first candidate of top_k's step
            if (!listed) {
                uint32_t above = 0;   // steps never fall along the ranks
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) above += 4 * t + k < n && step[k] < cut.k_first;
                (void)sum_below<kRowThreads>(above, s.part, all);
                first = static_cast<uint32_t>(all);
            }
            kept = first + (r.top_k - cut.k_count);
            if (r.top_p < 1.0) {
                u64 sum = 0;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) sum += 4 * t + k >= first && 4 * t + k < kept ? w[k] : 0;
                (void)sum_below<kRowThreads>(sum, s.part, mass_k);
                mass_k += cut.k_mass;
            }
        }
        if (r.top_p < 1.0) {
            const double limit_f = ceil(r.top_p * static_cast<double>(mass_k));
            const u64 limit = limit_f > 1.0 ? static_cast<u64>(limit_f) : 1ull;   // rank 0 always stays
            u64 run = cut.sure_mass + sum_below<kRowThreads>((w[0] + w[1]) + (w[2] + w[3]), s.part, all);
            uint32_t within = 0;   // nor do sums
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                within += 4 * t + k < n && step[k] <= cut.last && run < limit;
                run += w[k];
            }
            (void)sum_below<kRowThreads>(within, s.part, all);
            kept = all < kept ? static_cast<uint32_t>(all) : kept;
        }
        // Each cut that falls within reach keeps a candidate: the step before which it falls short holds it.  There are none where
        // top_k wants more logits than lie within reach, and nothing else cuts: all of those stay.
        last = kept != 0 ? s.cand[kept - 1] : 0;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (4 * t + k < kept && w[k] != 0 && depth[k] <= r.deepest)
                atomicAdd(&s.chunk_mass[(0xffffffffu - static_cast<uint32_t>(s.cand[4 * t + k])) / kChunk], w[k]);
    }
    __syncthreads();

    // the chunk, then the element, at which the sum exceeds uniform * all
    u64 share[4], sum = 0, all;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) sum += share[k] = s.chunk_mass[4 * t + k];
    u64 before = sum_below<kRowThreads>(sum, s.part, all);
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    u64 target = static_cast<u64>(static_cast<double>(u) * static_cast<double>(all));
    if (target >= all) target = all - 1;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        if (before <= target && target < before + share[k]) { s.at = 4 * t + k; s.target = target - before; }
        before += share[k];
    }
    __syncthreads();
    const uint32_t i = s.at * kChunk + 4 * t;
    target = s.target;
    float v[4];
    unpack(load4(p, x, i), v);
    sum = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        const uint32_t key = key_of(v[k]);
        sum += share[k] = rank_of(key, i + k) >= last ? kept_weight_at(depth_of(key, r), r, s.roots) : 0;
    }
    u64 run = sum_below<kRowThreads>(sum, s.part, all);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        if (run <= target && target < run + share[k]) p.out[row] = q8mi_argmax_pair{v[k], static_cast<int32_t>(i + k)};
        run += share[k];
    }
}

// A workgroup's histogram is added to one of a row's copies, one for kSpansOfCopy workgroups: atomics on the same few hundred
// numbers wait for each other (one row of 248320 by top_p, 1, 4 and 8 copies: 38, 25 and 27 us).
constexpr uint32_t kSpansOfCopy = 15, kMostCopies = 4;

uint32_t chunks_of(uint32_t vocab) { return (vocab + kChunk - 1) / kChunk; }
uint32_t span_of(uint32_t batch, uint32_t vocab, uint32_t most) {
    const uint64_t crowd = static_cast<uint64_t>(batch) * chunks_of(vocab) / kGridWanted;
    return crowd < 1 ? 1 : crowd > most ? most : static_cast<uint32_t>(crowd);
}
uint32_t copies_of(uint32_t batch, uint32_t vocab) {
    const uint32_t spans = chunks_of(vocab) / span_of(batch, vocab, kMostSpan), copies = spans / kSpansOfCopy;
    return copies < 1 ? 1 : copies > kMostCopies ? kMostCopies : copies;
}
// Bytes of a row: best, chunk_mass, bin_mass, candidates, cut, rows, bin_count, n_candidates, top, listed.  With the most copies
// that a row of such a vocabulary can have, those of a single row: fewer rows may have more copies than many, and a scratch for
// many must serve them.
uint64_t row_bytes(uint32_t vocab) {
    const uint64_t chunks = chunks_of(vocab), bins = kBins * copies_of(1, vocab);
    return 16 * chunks + 8 * (chunks + bins + chunks * kChunkCandidates) + sizeof(Cut) + sizeof(Row) + 4 * (bins + chunks + 2);
}

}  // namespace
}  // namespace q8mi

using namespace q8mi;

extern "C" size_t q8mi_sample_scratch_bytes(uint32_t batch, uint32_t vocab) {
    return 16 + batch * row_bytes(vocab);
}

extern "C" int q8mi_sample(const float *logits, uint32_t batch, uint32_t vocab, uint32_t stride, const float *temperature,
                           const int32_t *top_k, const float *top_p, const float *min_p, const float *uniform,
                           q8mi_argmax_pair *out, void *scratch, void *stream) {
    if (batch == 0) return Q8MI_OK;
    if (logits == nullptr || uniform == nullptr || out == nullptr || scratch == nullptr) return fail(Q8MI_REJECTED, "sample: null pointer");
    if (vocab == 0 || vocab > kMaxVocab) return fail(Q8MI_REJECTED, "sample: vocabulary of %u (1..%u)", vocab, kMaxVocab);
    if (batch > 1 && stride < vocab) return fail(Q8MI_REJECTED, "sample: rows overlap");
    if (batch > 65535) return fail(Q8MI_REJECTED, "sample: batch %u too large for one launch", batch);
    if (reinterpret_cast<uintptr_t>(scratch) % 16 != 0) return fail(Q8MI_REJECTED, "sample: scratch is not 16-byte aligned");
    SampleParams p{};
    p.logits = logits; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
    p.uniform = uniform; p.out = out; p.vocab = vocab; p.stride = stride;
    p.chunks = chunks_of(vocab);
    p.copies = copies_of(batch, vocab);
    p.vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (batch == 1 || stride % 4 == 0);
    uint8_t *at = static_cast<uint8_t *>(scratch);
    auto take = [&](uint64_t bytes) { uint8_t *a = at; at += batch * bytes; return a; };
    p.best = reinterpret_cast<uint32_t *>(take(16ull * p.chunks));   // read by 16 bytes
    p.chunk_mass = reinterpret_cast<u64 *>(take(8ull * p.chunks));
    p.bin_mass = reinterpret_cast<u64 *>(take(8ull * p.copies * kBins));
    p.candidates = reinterpret_cast<u64 *>(take(8ull * p.chunks * kChunkCandidates));
    p.cut = reinterpret_cast<Cut *>(take(sizeof(Cut)));
    p.rows = reinterpret_cast<Row *>(take(sizeof(Row)));
    p.bin_count = reinterpret_cast<uint32_t *>(take(4ull * p.copies * kBins));
    p.n_candidates = reinterpret_cast<uint32_t *>(take(4ull * p.chunks));
    p.top = reinterpret_cast<uint32_t *>(take(4));
    p.listed = reinterpret_cast<uint32_t *>(take(4));
    hipStream_t s = as_stream(stream);
    p.span = span_of(batch, vocab, kMostSpanOfBest);
    sample_best_kernel<<<dim3((p.chunks + p.span - 1) / p.span, batch), kChunkThreads, 0, s>>>(p);
    p.span = span_of(batch, vocab, kMostSpan);
    const dim3 grid((p.chunks + p.span - 1) / p.span, batch);
    sample_weigh_kernel<<<grid, kChunkThreads, 0, s>>>(p);
    if (top_k != nullptr || top_p != nullptr) sample_collect_kernel<<<grid, kChunkThreads, 0, s>>>(p);
    sample_draw_kernel<<<batch, kRowThreads, 0, s>>>(p);
    return check_launch("sample");
}
