// Sampling of one token per row of logits by temperature, top-k, top-p and min-p from a given uniform number.
//
// The three cuts keep a prefix of the row's ranks (logit descending, index ascending), so what is kept is known from its
// last rank: a key (the logit's bits in an order-preserving form) and the index of the last element with that key.
// Weights are p = exp((logit - max) / temperature) rounded to multiples of 2^-42: sums are 64-bit integers, exact and
// free of their order, so that neither the split of a row nor the arrival of atomics moves a border.
//
// No sort of the row.  Four launches, the first three over (chunks of 4096 logits) x rows:
//   1  largest (logit, lowest index) of each chunk; clears the row's counters
//   2  weights; where nothing is cut but by min-p, their sum per chunk, else a histogram of count and weight over 256
//      steps of 1/8 in (max - logit) / temperature (what lies 31.9 and more below the maximum weighs nothing)
//   3  the histogram says in which steps the cuts fall: the few logits of those steps are collected, what lies above them
//      is kept for certain and summed per chunk
//   4  one workgroup a row sorts the collected logits, takes the cuts in them, finds the chunk that holds the drawn element
//      and walks it
// A row with more than 4096 logits in the steps of its cuts (thousands of equal ones) is instead searched digit by digit
// of the keys, by the fourth launch's workgroup alone.
#include "q8mi_device.hpp"
#include "q8mi_internal.hpp"

namespace q8mi {
namespace {

constexpr uint32_t kMaxVocab = 1u << 20;
constexpr uint32_t kChunk = 4096;                     // logits of a workgroup of launches 1 to 3
constexpr uint32_t kMaxChunks = kMaxVocab / kChunk;
constexpr uint32_t kChunkThreads = 256;
constexpr uint32_t kRowThreads = 1024;                // launch 4
constexpr uint32_t kBins = 256;
constexpr double kBinsPerUnit = 8.0;
constexpr double kReach = 31.875;                     // exp(-31.875) * 2^42 rounds to 0
constexpr uint32_t kMaxCandidates = 4096;
constexpr double kOne = 4398046511104.0;              // 2^42: the weight of the largest logit; 2^20 of them sum below 2^63

typedef unsigned long long u64;

struct SampleParams {
    const float *logits;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    q8mi_argmax_pair *out;
    u64 *best;          // [row][chunk]: key << 32 | ~index of the chunk's rank 0
    u64 *chunk_mass;    // [row][chunk]: weight kept for certain
    u64 *bin_mass;      // [row][kBins]
    u64 *candidates;    // [row][kMaxCandidates]: key << 32 | ~index
    uint32_t *bin_count;     // [row][kBins]
    uint32_t *n_candidates;  // [row]
    uint32_t vocab, stride, chunks;
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

struct Row {
    float max;
    double per_unit;   // 1 / temperature
    double min_p;      // 0: off
    uint32_t top_k;    // 0: off
    double top_p;      // 1: off
    bool greedy;
};
__device__ __forceinline__ Row row_of(const SampleParams &p, uint32_t row, uint32_t top_key) {
    Row r;
    r.max = logit_of(top_key);
    const float t = p.temperature ? p.temperature[row] : 1.0f;
    r.greedy = !(t > 0.0f);
    r.per_unit = r.greedy ? 1.0 : 1.0 / static_cast<double>(t);
    const float min_p = p.min_p ? p.min_p[row] : 0.0f;
    r.min_p = min_p > 0.0f ? (min_p < 1.0f ? min_p : 1.0) : 0.0;
    const int32_t k = p.top_k ? p.top_k[row] : 0;
    r.top_k = k > 0 && static_cast<uint32_t>(k) < p.vocab ? k : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f;
    r.top_p = top_p < 1.0f ? top_p : 1.0;
    return r;
}
// How far below the maximum, in temperatures; not below kReach (or NaN): weighs nothing.
__device__ __forceinline__ double depth_of(uint32_t key, const Row &r) {
    if (key == 0) return INFINITY;
    const float v = logit_of(key);
    return v == r.max ? 0.0 : (static_cast<double>(r.max) - static_cast<double>(v)) * r.per_unit;
}
__device__ __forceinline__ u64 weight_at(double depth, double min_p) {
    if (!(depth < kReach)) return 0;
    const double s = exp(-depth);
    return s >= min_p ? static_cast<u64>(rint(s * kOne)) : 0;
}
__device__ __forceinline__ uint32_t bin_at(double depth) { return static_cast<uint32_t>(depth * kBinsPerUnit); }

__device__ __forceinline__ u64 xor_u64(u64 v, int d) { return __shfl_xor(v, d); }
__device__ __forceinline__ u64 wave_max_u64(u64 v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) { const u64 o = xor_u64(v, d); v = o > v ? o : v; }
    return v;
}
__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += xor_u64(v, d);
    return v;
}
// Sum of v over the threads below this one, and of all (`part`: one u64 a wave of LDS).
template <uint32_t THREADS>
__device__ __forceinline__ u64 sum_below(u64 v, u64 *part, u64 &all) {
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    u64 upto = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u64 o = __shfl_up(upto, d);
        upto += lane >= static_cast<uint32_t>(d) ? o : 0;
    }
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
__device__ __forceinline__ void load4(const SampleParams &p, const float *x, uint32_t i, float (&v)[4]) {
    if (p.vec && i + 4 <= p.vocab) {
        const float4 t = *reinterpret_cast<const float4 *>(x + i);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        return;
    }
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) v[k] = i + k < p.vocab ? x[i + k] : -INFINITY;
}

// ---- 1 ----------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(kChunkThreads) void sample_best_kernel(const SampleParams p) {
    __shared__ u64 part[kChunkThreads / kWave];
    const uint32_t t = threadIdx.x, chunk = blockIdx.x, row = blockIdx.y;
    const float *x = p.logits + static_cast<uint64_t>(row) * p.stride;
    float v[4][4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) load4(p, x, chunk * kChunk + u * 1024 + t * 4, v[u]);
    if (chunk == 0) {
        p.bin_mass[row * kBins + t] = 0;
        p.bin_count[row * kBins + t] = 0;
        if (t == 0) p.n_candidates[row] = 0;
    }
    u64 best = 0;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const u64 r = rank_of(key_of(v[u][k]), chunk * kChunk + u * 1024 + t * 4 + k);
            best = r > best ? r : best;
        }
    best = wave_max_u64(best);
    if (t % kWave == 0) part[t / kWave] = best;
    __syncthreads();
    if (t == 0) {
#pragma unroll
        for (uint32_t w = 1; w < kChunkThreads / kWave; ++w) best = part[w] > best ? part[w] : best;
        p.best[row * p.chunks + chunk] = best;
    }
}

// The row's rank 0, by every wave for itself.
__device__ __forceinline__ u64 row_best(const SampleParams &p, uint32_t row) {
    u64 best = 0;
    for (uint32_t c = threadIdx.x % kWave; c < p.chunks; c += kWave) {
        const u64 b = p.best[row * p.chunks + c];
        best = b > best ? b : best;
    }
    return wave_max_u64(best);
}

// ---- 2 ----------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(kChunkThreads) void sample_weigh_kernel(const SampleParams p) {
    __shared__ u64 mass[kBins];
    __shared__ uint32_t count[kBins];
    __shared__ u64 part[kChunkThreads / kWave];
    const uint32_t t = threadIdx.x, chunk = blockIdx.x, row = blockIdx.y;
    const float *x = p.logits + static_cast<uint64_t>(row) * p.stride;
    float v[4][4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) load4(p, x, chunk * kChunk + u * 1024 + t * 4, v[u]);
    const uint32_t top = static_cast<uint32_t>(row_best(p, row) >> 32);
    const Row r = row_of(p, row, top);
    if (top == 0 || r.greedy) return;
    const bool cuts = r.top_k != 0 || r.top_p < 1.0;
    if (cuts) {
        mass[t] = 0;
        count[t] = 0;
        __syncthreads();
    }
    u64 sum = 0;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const double depth = depth_of(key_of(v[u][k]), r);
            if (!(depth < kReach)) continue;
            if (cuts) {
                const uint32_t b = bin_at(depth);
                atomicAdd(&mass[b], weight_at(depth, 0.0));
                atomicAdd(&count[b], 1u);
            } else {
                sum += weight_at(depth, r.min_p);
            }
        }
    if (cuts) {
        __syncthreads();
        if (count[t] != 0) {
            atomicAdd(&p.bin_count[row * kBins + t], count[t]);
            atomicAdd(&p.bin_mass[row * kBins + t], mass[t]);
        }
        return;
    }
    sum = wave_sum_u64(sum);
    if (t % kWave == 0) part[t / kWave] = sum;
    __syncthreads();
    if (t == 0) p.chunk_mass[row * p.chunks + chunk] = (part[0] + part[1]) + (part[2] + part[3]);
}

// Where the cuts fall: steps below `sure` are kept, steps first .. last hold the last rank, step `k_bin` the top_k-th.
struct Cut {
    uint32_t sure, last, k_bin;   // kBins: nothing is cut there
};
// Every thread of at least kBins calls it; `low`: kBins of LDS for counts and masses up to and with a step.
__device__ __forceinline__ Cut find_cut(const SampleParams &p, uint32_t row, const Row &r, u64 *mass_upto, uint32_t *count_upto,
                                        uint32_t *found) {
    const uint32_t t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    u64 m = 0;
    uint32_t c = 0;
    if (t < kBins) {
        m = p.bin_mass[row * kBins + t];
        c = p.bin_count[row * kBins + t];
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const u64 om = __shfl_up(m, d);
            const uint32_t oc = __shfl_up(c, d);
            if (lane >= static_cast<uint32_t>(d)) { m += om; c += oc; }
        }
        mass_upto[t] = m;
        count_upto[t] = c;
    }
    if (t == 0) { found[0] = found[1] = found[2] = kBins; }
    __syncthreads();
    if (t < kBins) {
        for (uint32_t w = 0; w < wave; ++w) { m += mass_upto[w * kWave + 63]; c += count_upto[w * kWave + 63]; }
    }
    __syncthreads();
    if (t < kBins) { mass_upto[t] = m; count_upto[t] = c; }
    __syncthreads();
    const uint32_t c_before = t == 0 || t >= kBins ? 0 : count_upto[t - 1];
    if (t < kBins && r.top_k != 0 && c_before < r.top_k && c >= r.top_k) found[0] = t;   // one thread
    __syncthreads();
    Cut cut;
    cut.k_bin = found[0];
    cut.sure = cut.last = cut.k_bin;
    if (r.top_p < 1.0) {
        // the mass that top_k keeps lies between these; so does the last rank that top_p keeps
        const uint32_t kb = cut.k_bin < kBins ? cut.k_bin : kBins - 1;
        const u64 hi = mass_upto[kb], lo = cut.k_bin < kBins ? (kb ? mass_upto[kb - 1] : 0) : hi;
        const double limit_lo = r.top_p * static_cast<double>(lo), limit_hi = r.top_p * static_cast<double>(hi);
        const u64 m_before = t == 0 || t >= kBins ? 0 : mass_upto[t - 1];
        // the first step that reaches the limit: the mass before it falls short
        if (t < kBins && m != m_before) {
            if ((t == 0 || m_before == 0 || static_cast<double>(m_before) < limit_lo) && static_cast<double>(m) >= limit_lo) atomicMin(&found[1], t);
            if ((t == 0 || m_before == 0 || static_cast<double>(m_before) < limit_hi) && static_cast<double>(m) >= limit_hi) atomicMin(&found[2], t);
        }
        __syncthreads();
        cut.sure = found[1] < cut.k_bin ? found[1] : cut.k_bin;
        cut.last = found[2] < cut.k_bin ? found[2] : cut.k_bin;
    }
    return cut;
}

// ---- 3 ----------------------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(kChunkThreads) void sample_collect_kernel(const SampleParams p) {
    __shared__ u64 mass_upto[kBins];
    __shared__ uint32_t count_upto[kBins], found[3], n_here, base;
    __shared__ u64 part[kChunkThreads / kWave];
    const uint32_t t = threadIdx.x, chunk = blockIdx.x, row = blockIdx.y;
    const float *x = p.logits + static_cast<uint64_t>(row) * p.stride;
    float v[4][4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) load4(p, x, chunk * kChunk + u * 1024 + t * 4, v[u]);
    const uint32_t top = static_cast<uint32_t>(row_best(p, row) >> 32);
    const Row r = row_of(p, row, top);
    if (top == 0 || r.greedy || !(r.top_k != 0 || r.top_p < 1.0)) return;
    if (t == 0) n_here = 0;
    const Cut cut = find_cut(p, row, r, mass_upto, count_upto, found);
    // the elements to collect, and their places among this chunk's
    uint32_t mine = 0;   // bit per element
    u64 sum = 0;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            const double depth = depth_of(key_of(v[u][k]), r);
            if (!(depth < kReach)) continue;
            const uint32_t b = bin_at(depth);
            if (b < cut.sure) sum += weight_at(depth, r.min_p);
            else if (b <= cut.last || b == cut.k_bin) mine |= 1u << (u * 4 + k);
        }
    uint32_t at = mine ? atomicAdd(&n_here, static_cast<uint32_t>(__popc(mine))) : 0;
    sum = wave_sum_u64(sum);
    if (t % kWave == 0) part[t / kWave] = sum;
    __syncthreads();
    if (t == 0) {
        p.chunk_mass[row * p.chunks + chunk] = (part[0] + part[1]) + (part[2] + part[3]);
        base = n_here ? atomicAdd(&p.n_candidates[row], n_here) : 0;
    }
    __syncthreads();
    at += base;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (mine >> (u * 4 + k) & 1) {
                if (at < kMaxCandidates)
                    p.candidates[static_cast<uint64_t>(row) * kMaxCandidates + at] = rank_of(key_of(v[u][k]), chunk * kChunk + u * 1024 + t * 4 + k);
                ++at;
            }
}

// ---- 4 ----------------------------------------------------------------------------------------------------------------
// The last kept rank of a row by its keys' digits: eight bits a pass over the whole row, counts and weights of the 256
// values in LDS, first for top_k, then for top_p among what that keeps.  The workgroup's scratch is the candidates' LDS.
__device__ u64 cut_by_digits(const SampleParams &p, const float *x, const Row &r, u64 *lds) {
    u64 *mass = lds, *part = lds + 256, *sh = lds + 256 + kRowThreads;
    uint32_t *count = reinterpret_cast<uint32_t *>(sh + 8);
    const uint32_t t = threadIdx.x;
    uint32_t last_key = 1, last_ties = 0xffffffffu;   // elements above last_key, and the first last_ties of those equal to it
    // The last rank that stays when ranks are taken in order: while fewer than `limit` (count or mass) came before it.
    auto cut = [&](bool by_mass, u64 limit) {
        uint32_t prefix = 0;
        u64 before = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (t < 256) { mass[t] = 0; count[t] = 0; }
            __syncthreads();
            for (uint32_t i = t; i < p.vocab; i += kRowThreads) {
                const uint32_t key = key_of(x[i]);
                if (key < last_key || (shift != 24 && (key >> (shift + 8)) != prefix)) continue;
                const double depth = depth_of(key, r);
                if (!(depth < kReach)) continue;
                atomicAdd(&count[(key >> shift) & 255], 1u);
                if (by_mass) atomicAdd(&mass[(key >> shift) & 255], weight_at(depth, 0.0));
            }
            __syncthreads();
            if (t == 0) {
                int digit = -1;
                u64 upto = 0;
                for (int d = 255; d >= 0; --d) {
                    if (count[d] == 0) continue;
                    if (digit >= 0) before = upto;
                    digit = d;
                    upto = before + (by_mass ? mass[d] : count[d]);
                    if (upto >= limit) break;
                }
                sh[0] = static_cast<u64>(prefix << 8 | static_cast<uint32_t>(digit));
                sh[1] = before;
                sh[2] = count[digit];
            }
            __syncthreads();
            prefix = static_cast<uint32_t>(sh[0]);
            before = sh[1];
            __syncthreads();
        }
        uint32_t ties = static_cast<uint32_t>(sh[2]);
        const u64 left = limit > before ? limit - before : 1;
        const u64 each = by_mass ? weight_at(depth_of(prefix, r), 0.0) : 1;
        if (each != 0) {
            const u64 need = (left + each - 1) / each;
            if (need < ties) ties = static_cast<uint32_t>(need);
        }
        if (prefix != last_key || ties < last_ties) last_ties = ties;
        last_key = prefix;
        __syncthreads();
    };
    const uint32_t per = (p.vocab + kRowThreads - 1) / kRowThreads;
    const uint32_t lo = t * per < p.vocab ? t * per : p.vocab, hi = lo + per < p.vocab ? lo + per : p.vocab;
    auto ties_below = [&]() {   // elements equal to last_key before this thread's range
        u64 mine = 0, all;
        for (uint32_t i = lo; i < hi; ++i) mine += key_of(x[i]) == last_key;
        return static_cast<uint32_t>(sum_below<kRowThreads>(mine, part, all));
    };
    if (r.top_k != 0) cut(false, r.top_k);
    if (r.top_p < 1.0) {
        uint32_t seen = ties_below();
        u64 sum = 0, all;
        for (uint32_t i = lo; i < hi; ++i) {
            const uint32_t key = key_of(x[i]);
            if (key < last_key || (key == last_key && seen++ >= last_ties)) continue;
            sum += weight_at(depth_of(key, r), 0.0);
        }
        (void)sum_below<kRowThreads>(sum, part, all);
        const double limit = ceil(r.top_p * static_cast<double>(all));
        cut(true, limit > 1.0 ? static_cast<u64>(limit) : 1ull);   // rank 0 always stays
    }
    // the index of the last tie that stays
    uint32_t seen = ties_below();
    __syncthreads();
    if (t == 0) sh[3] = 0xffffffffu;
    __syncthreads();
    for (uint32_t i = lo; i < hi; ++i)
        if (key_of(x[i]) == last_key && ++seen == last_ties) sh[3] = i;
    __syncthreads();
    return rank_of(last_key, static_cast<uint32_t>(sh[3]));
}

__global__ __launch_bounds__(kRowThreads) void sample_draw_kernel(const SampleParams p) {
    __shared__ u64 cand[kMaxCandidates];
    __shared__ u64 mass_upto[kBins];
    __shared__ uint32_t count_upto[kBins], found[3];
    __shared__ u64 part[kRowThreads / kWave];
    __shared__ u64 chunk_mass[kMaxChunks];
    __shared__ u64 shared_last, shared_target;
    __shared__ uint32_t shared_at, bounds[2];
    const uint32_t t = threadIdx.x, row = blockIdx.x;
    const float *x = p.logits + static_cast<uint64_t>(row) * p.stride;
    const u64 best = row_best(p, row);
    const uint32_t top = static_cast<uint32_t>(best >> 32);
    if (top == 0) {
        if (t == 0) p.out[row] = q8mi_argmax_pair{-INFINITY, -1};
        return;
    }
    const Row r = row_of(p, row, top);
    if (r.greedy) {
        const uint32_t i = 0xffffffffu - static_cast<uint32_t>(best);
        if (t == 0) p.out[row] = q8mi_argmax_pair{x[i], static_cast<int32_t>(i)};
        return;
    }
    u64 last = 0;   // rank of the last kept element: everything from it up is kept
    for (uint32_t c = t; c < p.chunks; c += kRowThreads) chunk_mass[c] = 0;
    bool from_chunks = true;   // launches 2 and 3 have left the chunks' sums
    if (r.top_k != 0 || r.top_p < 1.0) {
        const uint32_t n = p.n_candidates[row];
        if (n > kMaxCandidates) {
            last = cut_by_digits(p, x, r, cand);
            from_chunks = false;
        } else {
            const Cut cut = find_cut(p, row, r, mass_upto, count_upto, found);
            uint32_t size = 2;
            while (size < n) size *= 2;
            for (uint32_t i = t; i < size; i += kRowThreads) cand[i] = i < n ? p.candidates[static_cast<uint64_t>(row) * kMaxCandidates + i] : 0;
            __syncthreads();
            for (uint32_t k = 2; k <= size; k *= 2)           // bitonic, descending
                for (uint32_t j = k / 2; j > 0; j /= 2) {
                    for (uint32_t i = t; i < size; i += kRowThreads) {
                        const uint32_t o = i ^ j;
                        if (o > i) {
                            const u64 a = cand[i], b = cand[o];
                            if ((a < b) == ((i & k) == 0)) { cand[i] = b; cand[o] = a; }
                        }
                    }
                    __syncthreads();
                }
            // this thread's candidates, neighbours in rank: 4 * t ..
            u64 w[4], sum = 0, all;
            uint32_t bin[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t c = 4 * t + i;
                const double depth = c < n ? depth_of(static_cast<uint32_t>(cand[c] >> 32), r) : INFINITY;
                w[i] = weight_at(depth, 0.0);
                bin[i] = c < n ? bin_at(depth) : kBins;
                sum += w[i];
            }
            // k: candidates of the steps up to cut.last begin at 0; those of a separate k_bin behind them
            if (t == 0) { bounds[0] = bounds[1] = n; shared_last = 0; }
            const u64 before_me = sum_below<kRowThreads>(sum, part, all);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (4 * t + i < n && bin[i] == cut.k_bin) atomicMin(&bounds[0], 4 * t + i);   // the first candidate of the k step
            __syncthreads();
            uint32_t kept = n;          // candidates in rank order that stay
            u64 mass_k = mass_upto[kBins - 1];
            if (cut.k_bin < kBins) {
                const uint32_t first = bounds[0], count0 = cut.k_bin ? count_upto[cut.k_bin - 1] : 0;
                kept = first + (r.top_k - count0);
                // the k step's kept weight: sum over [first, kept)
                u64 in_step = 0;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    if (4 * t + i >= first && 4 * t + i < kept) in_step += w[i];
                u64 step_all;
                (void)sum_below<kRowThreads>(in_step, part, step_all);
                mass_k = (cut.k_bin ? mass_upto[cut.k_bin - 1] : 0) + step_all;
            }
            if (r.top_p < 1.0) {
                const double limit_f = ceil(r.top_p * static_cast<double>(mass_k));
                const u64 limit = limit_f > 1.0 ? static_cast<u64>(limit_f) : 1ull;   // rank 0 always stays
                const u64 sure = cut.sure ? mass_upto[cut.sure - 1] : 0;
                // candidates of the steps first .. last follow one another in rank from the mass `sure` on
                u64 run = sure + before_me;
                uint32_t stay = 0;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (4 * t + i < n && bin[i] <= cut.last && run < limit) stay = 4 * t + i + 1;
                    run += w[i];
                }
                if (t == 0) bounds[1] = 0;
                __syncthreads();
                if (stay) atomicMax(&bounds[1], stay);
                __syncthreads();
                kept = bounds[1] < kept ? bounds[1] : kept;
            }
            if (kept > 0 && t == 0) shared_last = cand[kept - 1];
            __syncthreads();
            last = shared_last;
            if (kept == 0) last = 0;   // everything above the candidates: handled by the sums below
            for (uint32_t c = t; c < p.chunks; c += kRowThreads) chunk_mass[c] = p.chunk_mass[row * p.chunks + c];
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t c = 4 * t + i;
                if (c < kept && w[i] != 0) {
                    const uint32_t index = 0xffffffffu - static_cast<uint32_t>(cand[c]);
                    const u64 kept_w = weight_at(depth_of(static_cast<uint32_t>(cand[c] >> 32), r), r.min_p);
                    atomicAdd(&chunk_mass[index / kChunk], kept_w);
                }
            }
            __syncthreads();
        }
    } else {
        for (uint32_t c = t; c < p.chunks; c += kRowThreads) chunk_mass[c] = p.chunk_mass[row * p.chunks + c];
        __syncthreads();
    }
    auto kept_weight = [&](float v, uint32_t i) -> u64 {
        const uint32_t key = key_of(v);
        return rank_of(key, i) >= last ? weight_at(depth_of(key, r), r.min_p) : 0;
    };
    if (!from_chunks) {
        __syncthreads();
        for (uint32_t c = 0; c < p.chunks; ++c) {
            float v[4];
            load4(p, x, c * kChunk + 4 * t, v);
            u64 sum = 0, all;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) sum += kept_weight(v[k], c * kChunk + 4 * t + k);
            (void)sum_below<kRowThreads>(sum, part, all);
            if (t == 0) chunk_mass[c] = all;
        }
        __syncthreads();
    }

    // the chunk, then the element, at which the sum exceeds uniform * all
    u64 all;
    const u64 mine = t < p.chunks ? chunk_mass[t] : 0;
    const u64 before = sum_below<kRowThreads>(mine, part, all);
    float u = p.uniform[row];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    u64 target = static_cast<u64>(static_cast<double>(u) * static_cast<double>(all));
    if (target >= all) target = all - 1;
    if (before <= target && target < before + mine) { shared_at = t; shared_target = target - before; }
    __syncthreads();
    const uint32_t chunk = shared_at;
    target = shared_target;
    float v[4];
    u64 w[4], sum = 0;
    load4(p, x, chunk * kChunk + 4 * t, v);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
        w[k] = kept_weight(v[k], chunk * kChunk + 4 * t + k);
        sum += w[k];
    }
    u64 run = sum_below<kRowThreads>(sum, part, all);
    if (run <= target && target < run + sum) {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            if (run <= target && target < run + w[k]) p.out[row] = q8mi_argmax_pair{v[k], static_cast<int32_t>(chunk * kChunk + 4 * t + k)};
            run += w[k];
        }
    }
}

uint32_t chunks_of(uint32_t vocab) { return (vocab + kChunk - 1) / kChunk; }
// u64 words of a row: best and chunk_mass, bin_mass, candidates, bin_count; n_candidates behind all rows
uint64_t row_words(uint32_t vocab) { return 2ull * chunks_of(vocab) + kBins + kMaxCandidates + kBins / 2; }

}  // namespace
}  // namespace q8mi

using namespace q8mi;

extern "C" size_t q8mi_sample_scratch_bytes(uint32_t batch, uint32_t vocab) {
    return 16 + batch * (row_words(vocab) * 8 + 4);
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
    p.vec = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (batch == 1 || stride % 4 == 0);
    u64 *words = static_cast<u64 *>(scratch);
    auto take = [&](uint64_t n) { u64 *at = words; words += n; return at; };
    p.best = take(static_cast<uint64_t>(batch) * p.chunks);
    p.chunk_mass = take(static_cast<uint64_t>(batch) * p.chunks);
    p.bin_mass = take(static_cast<uint64_t>(batch) * kBins);
    p.candidates = take(static_cast<uint64_t>(batch) * kMaxCandidates);
    p.bin_count = reinterpret_cast<uint32_t *>(take(static_cast<uint64_t>(batch) * kBins / 2));
    p.n_candidates = reinterpret_cast<uint32_t *>(words);
    hipStream_t s = as_stream(stream);
    const dim3 grid(p.chunks, batch);
    sample_best_kernel<<<grid, kChunkThreads, 0, s>>>(p);
    sample_weigh_kernel<<<grid, kChunkThreads, 0, s>>>(p);
    if (top_k != nullptr || top_p != nullptr) sample_collect_kernel<<<grid, kChunkThreads, 0, s>>>(p);
    sample_draw_kernel<<<batch, kRowThreads, 0, s>>>(p);
    return check_launch("sample");
}
