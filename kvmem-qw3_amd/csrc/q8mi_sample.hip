// Sampling of one token per row of logits by temperature, top-k, top-p and min-p from a given uniform number.
//
// The three cuts keep a prefix of the row's ranks (logit descending, index ascending), so what is kept is known from its
// last rank: a key (the logit's bits in an order-preserving form) and how many of the elements that equal it stay.
// Weights are p = exp((logit - max) / temperature) rounded to multiples of 2^-42: sums are 64-bit integers, exact and
// free of their order, so that neither the split of a row nor the arrival of atomics moves a border.
//
// One workgroup per row: it finds the last key of each cut digit by digit (8 bits a pass: counts and weights of the 256
// values in LDS), sums the kept weights, and walks the row in index order to the drawn element.
#include "q8mi_device.hpp"
#include "q8mi_internal.hpp"

namespace q8mi {
namespace {

constexpr uint32_t kSampleThreads = 1024;
constexpr uint32_t kMaxVocab = 1u << 20;
constexpr double kOne = 4398046511104.0;   // 2^42: the weight of the largest logit; 2^20 of them sum below 2^63

struct SampleParams {
    const float *logits;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    q8mi_argmax_pair *out;
    uint32_t vocab, stride;
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

struct Row {
    float max;
    double temperature;
    double min_p;
};

__device__ __forceinline__ double share_of(uint32_t key, const Row &r) {
    if (key == 0) return 0.0;
    const float v = logit_of(key);
    if (v == r.max) return 1.0;   // also +inf
    return exp((static_cast<double>(v) - static_cast<double>(r.max)) / r.temperature);
}
__device__ __forceinline__ uint64_t weight_of(uint32_t key, const Row &r) {
    const double s = share_of(key, r);
    return s >= r.min_p ? static_cast<uint64_t>(rint(s * kOne)) : 0;
}

__global__ __launch_bounds__(kSampleThreads) void sample_kernel(const SampleParams p) {
    __shared__ unsigned long long mass[256];
    __shared__ uint32_t count[256];
    __shared__ unsigned long long part[kSampleThreads];
    __shared__ uint32_t sh_key, sh_prefix, sh_ties;
    __shared__ unsigned long long sh_mass;
    __shared__ int sh_found;
    const uint32_t t = threadIdx.x, row = blockIdx.x;
    const float *x = p.logits + static_cast<uint64_t>(row) * p.stride;

    if (t == 0) { sh_key = 0; sh_found = 0; }
    __syncthreads();
    uint32_t top = 0;
    for (uint32_t i = t; i < p.vocab; i += kSampleThreads) top = max(top, key_of(x[i]));
    atomicMax(&sh_key, top);
    __syncthreads();
    top = sh_key;
    __syncthreads();
    if (top == 0) {
        if (t == 0) p.out[row] = q8mi_argmax_pair{-INFINITY, -1};
        return;
    }
    Row r;
    r.max = logit_of(top);
    const float temperature = p.temperature ? p.temperature[row] : 1.0f;
    const bool greedy = !(temperature > 0.0f);
    r.temperature = greedy ? 1.0 : temperature;
    r.min_p = 0.0;
    const float min_p = p.min_p ? p.min_p[row] : 0.0f;

    // the cut: elements above last_key, and the first last_ties (by index) of those that equal it
    uint32_t last_key = 1, last_ties = 0xffffffffu;
    // Finds the last rank that `stays` when ranks are taken in order: by count (rank < limit) or by mass (the mass before
    // it is below the limit).  Eight bits a pass.
    auto cut = [&](bool by_mass, unsigned long long limit) {
        uint32_t prefix = 0;
        unsigned long long before = 0;   // count or mass above the prefix
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (t < 256) { mass[t] = 0; count[t] = 0; }
            __syncthreads();
            for (uint32_t i = t; i < p.vocab; i += kSampleThreads) {
                const uint32_t key = key_of(x[i]);
                if (key < last_key || (shift != 24 && (key >> (shift + 8)) != prefix)) continue;
                atomicAdd(&count[(key >> shift) & 255], 1u);
                if (by_mass) atomicAdd(&mass[(key >> shift) & 255], weight_of(key, r));
            }
            __syncthreads();
            if (t == 0) {
                int digit = -1;
                for (int d = 255; d >= 0; --d) {
                    if (count[d] == 0) continue;
                    if (before >= limit) break;
                    if (digit >= 0) before = sh_mass;
                    digit = d;
                    sh_mass = before + (by_mass ? mass[d] : count[d]);
                    if (sh_mass >= limit) break;
                }
                sh_prefix = prefix << 8 | static_cast<uint32_t>(digit);
                sh_mass = before;
                sh_ties = count[digit];
            }
            __syncthreads();
            prefix = sh_prefix;
            before = sh_mass;
            __syncthreads();
        }
        uint32_t ties = sh_ties;
        const unsigned long long left = limit > before ? limit - before : 1;
        const unsigned long long each = by_mass ? weight_of(prefix, r) : 1;
        if (each != 0) {
            const unsigned long long need = (left + each - 1) / each;
            if (need < ties) ties = static_cast<uint32_t>(need);
        }
        if (prefix != last_key || ties < last_ties) last_ties = ties;
        last_key = prefix;
        __syncthreads();
    };
    // Walks the kept elements in index order; the mass of all, or (target given) the element at which the sum exceeds it.
    auto walk = [&](bool find, unsigned long long target, int &index) -> unsigned long long {
        unsigned long long sum = 0;
        uint32_t ties = 0;
        const uint32_t per = (p.vocab + kSampleThreads - 1) / kSampleThreads;
        const uint32_t lo = min(p.vocab, t * per), hi = min(p.vocab, lo + per);
        uint32_t mine = 0;
        for (uint32_t i = lo; i < hi; ++i) mine += key_of(x[i]) == last_key;
        part[t] = mine;
        __syncthreads();
        for (uint32_t u = 0; u < t; ++u) ties += static_cast<uint32_t>(part[u]);
        __syncthreads();
        auto each = [&](uint32_t i, uint32_t &seen) -> unsigned long long {
            const uint32_t key = key_of(x[i]);
            if (key < last_key || (key == last_key && seen++ >= last_ties)) return 0;
            return weight_of(key, r);
        };
        uint32_t seen = ties;
        for (uint32_t i = lo; i < hi; ++i) sum += each(i, seen);
        part[t] = sum;
        __syncthreads();
        unsigned long long before = 0, all = 0;
        for (uint32_t u = 0; u < kSampleThreads; ++u) {
            if (u == t) before = all;
            all += part[u];
        }
        if (find && before <= target && target < before + sum) {
            seen = ties;
            for (uint32_t i = lo; i < hi; ++i) {
                before += each(i, seen);
                if (before > target) { sh_found = static_cast<int>(i); break; }
            }
        }
        __syncthreads();
        index = sh_found;
        return all;
    };

    int index = 0;
    if (greedy) {
        last_key = top;
        last_ties = 1;
    } else {
        const int32_t k = p.top_k ? p.top_k[row] : 0;
        if (k > 0) cut(false, static_cast<unsigned long long>(k));
        const float top_p = p.top_p ? p.top_p[row] : 1.0f;
        if (top_p < 1.0f) {
            const unsigned long long all = walk(false, 0, index);
            const double limit = ceil(static_cast<double>(top_p) * static_cast<double>(all));
            cut(true, limit > 1.0 ? static_cast<unsigned long long>(limit) : 1ull);   // rank 0 always stays
        }
        if (min_p > 0.0f) r.min_p = min_p < 1.0f ? min_p : 1.0;
    }
    const unsigned long long all = walk(false, 0, index);
    float u = p.uniform[row];
    u = u > 0.0f ? fminf(u, 1.0f) : 0.0f;
    unsigned long long at = static_cast<unsigned long long>(static_cast<double>(u) * static_cast<double>(all));
    if (at >= all) at = all - 1;
    walk(true, at, index);
    if (t == 0) p.out[row] = q8mi_argmax_pair{x[index], index};
}

}  // namespace
}  // namespace q8mi

using namespace q8mi;

extern "C" size_t q8mi_sample_scratch_bytes(uint32_t, uint32_t) { return 16; }

extern "C" int q8mi_sample(const float *logits, uint32_t batch, uint32_t vocab, uint32_t stride, const float *temperature,
                           const int32_t *top_k, const float *top_p, const float *min_p, const float *uniform,
                           q8mi_argmax_pair *out, void *scratch, void *stream) {
    if (batch == 0) return Q8MI_OK;
    if (logits == nullptr || uniform == nullptr || out == nullptr || scratch == nullptr) return fail(Q8MI_REJECTED, "sample: null pointer");
    if (vocab == 0 || vocab > kMaxVocab) return fail(Q8MI_REJECTED, "sample: vocabulary of %u (1..%u)", vocab, kMaxVocab);
    if (batch > 1 && stride < vocab) return fail(Q8MI_REJECTED, "sample: rows overlap");
    if (batch > 65535) return fail(Q8MI_REJECTED, "sample: batch %u too large for one launch", batch);
    SampleParams p{};
    p.logits = logits; p.temperature = temperature; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p;
    p.uniform = uniform; p.out = out; p.vocab = vocab; p.stride = stride;
    sample_kernel<<<batch, kSampleThreads, 0, as_stream(stream)>>>(p);
    return check_launch("sample");
}
