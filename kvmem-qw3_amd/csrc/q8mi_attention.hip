// Attention of each sequence's newest rows over a paged key / value cache (decode, speculative verification).
//
//   out = sum_t p_t v_t,  p = softmax_t(scale * q . k_t),  t <= kv_len - rows + i
//
// One workgroup per query row and head.  Its four waves take every fourth token, a lane holds head_dim / 64 elements of
// the query and of the output; each wave keeps a running maximum, sum and output, which meet in LDS at the end.
#include "q8mi_kv.hpp"

namespace q8mi {
namespace {

constexpr uint32_t kMaxRows = 16;     // new rows of a sequence
constexpr uint32_t kAttnThreads = 256;

struct AttnParams {
    const void *q;
    void *out;
    const int32_t *page_table, *kv_lens, *q_starts;
    q8mi_kv_cache cache;
    uint32_t q_rows, stride_q, stride_out, stride_page_table;
    uint32_t n_seqs, max_q_len, q_heads, group, max_kv_len;
    float scale;
    int q_is_bf16, out_is_bf16;
};

__device__ __forceinline__ float load_kv(const void *pool, uint64_t at, int dtype) {
    if (dtype == Q8MI_KV_E4M3) return __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t *>(pool)[at], 0);
    const uint16_t h = static_cast<const uint16_t *>(pool)[at];
    return dtype == Q8MI_KV_BF16 ? bf16_bits_to_float(h) : half_bits_to_float(h);
}

template <uint32_t D>
__global__ __launch_bounds__(kAttnThreads) void attention_kernel(const AttnParams p) {
    constexpr uint32_t E = D / kWave;
    const uint32_t lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const uint32_t seq = blockIdx.x / p.max_q_len, i = blockIdx.x % p.max_q_len, head = blockIdx.y;
    int64_t start = static_cast<int64_t>(seq) * p.max_q_len, rows = p.max_q_len;
    if (p.q_starts != nullptr) {
        start = p.q_starts[seq];
        rows = p.q_starts[seq + 1] - start;
    }
    const int64_t row = start + i;
    if (i >= rows || row < 0 || row >= p.q_rows) return;
    const int64_t kv_len = p.kv_lens[seq];
    int64_t seen = kv_len - rows + i + 1;
    seen = seen > p.max_kv_len ? p.max_kv_len : seen;
    const uint32_t kv_head = head / p.group;

    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) {
        const uint64_t at = static_cast<uint64_t>(row) * p.stride_q + head * D + e * kWave + lane;
        q[e] = p.q_is_bf16 ? bf16_bits_to_float(static_cast<const uint16_t *>(p.q)[at]) : static_cast<const float *>(p.q)[at];
        o[e] = 0.0f;
    }
    const bool e4m3 = p.cache.dtype == Q8MI_KV_E4M3;
    const float scale = p.scale * (e4m3 ? p.cache.k_scale : 1.0f);
    for (int64_t t = wave; t < seen; t += kAttnThreads / kWave) {
        const int32_t page = p.page_table[static_cast<uint64_t>(seq) * p.stride_page_table + t / p.cache.page_size];
        if (page < 0 || static_cast<uint32_t>(page) >= p.cache.pages) continue;
        const uint64_t at = page * p.cache.stride_page + kv_head * p.cache.stride_head + (t % p.cache.page_size) * p.cache.stride_token;
        float dot = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < E; ++e) dot += q[e] * load_kv(p.cache.k, at + e * kWave + lane, p.cache.dtype);
        const float score = wave_sum(dot) * scale;
        const float top = fmaxf(m, score);
        const float keep = m == top ? 1.0f : expf(m - top), w = expf(score - top);
        l = l * keep + w;
#pragma unroll
        for (uint32_t e = 0; e < E; ++e)
            o[e] = o[e] * keep + w * load_kv(p.cache.v, at + e * kWave + lane, p.cache.dtype);
        m = top;
    }
    __shared__ float om[4][D], mm[4], ll[4];
#pragma unroll
    for (uint32_t e = 0; e < E; ++e) om[wave][e * kWave + lane] = o[e];
    if (lane == 0) { mm[wave] = m; ll[wave] = l; }
    __syncthreads();
    const float top = fmaxf(fmaxf(mm[0], mm[1]), fmaxf(mm[2], mm[3]));
    for (uint32_t d = threadIdx.x; d < D; d += kAttnThreads) {
        float sum = 0.0f, total = 0.0f;
        for (int w = 0; w < 4; ++w) {
            const float f = ll[w] == 0.0f ? 0.0f : expf(mm[w] - top);
            sum += f * om[w][d];
            total += f * ll[w];
        }
        const float r = total == 0.0f ? 0.0f : sum / total * (e4m3 ? p.cache.v_scale : 1.0f);
        const uint64_t at = static_cast<uint64_t>(row) * p.stride_out + head * D + d;
        if (p.out_is_bf16) static_cast<uint16_t *>(p.out)[at] = float_to_bf16_bits(r);
        else static_cast<float *>(p.out)[at] = r;
    }
}

}  // namespace
}  // namespace q8mi

using namespace q8mi;

extern "C" size_t q8mi_paged_attention_scratch_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 16; }

extern "C" int q8mi_paged_attention(const void *q, int q_is_bf16, uint32_t q_rows, uint32_t stride_q_row,
                                    const q8mi_kv_cache *cache, const int32_t *page_table, uint32_t stride_page_table,
                                    const int32_t *kv_lens, const int32_t *q_starts, uint32_t n_seqs, uint32_t max_q_len,
                                    uint32_t q_heads, uint32_t max_kv_len, float scale, void *out, int out_is_bf16,
                                    uint32_t stride_out_row, void *scratch, void *stream) {
    const char *what = "paged_attention";
    if (const int rc = check_kv_cache(what, cache); rc != Q8MI_OK) return rc;
    if (n_seqs == 0 || q_rows == 0) return Q8MI_OK;
    if (q == nullptr || out == nullptr || page_table == nullptr || kv_lens == nullptr || scratch == nullptr)
        return fail(Q8MI_REJECTED, "%s: null pointer", what);
    if (q_heads == 0 || q_heads > 65536 || q_heads % cache->kv_heads != 0)
        return fail(Q8MI_REJECTED, "%s: %u query heads over %u", what, q_heads, cache->kv_heads);
    if (max_q_len == 0 || max_q_len > kMaxRows) return fail(Q8MI_REJECTED, "%s: %u rows a sequence (1..%u)", what, max_q_len, kMaxRows);
    if (max_kv_len > static_cast<uint64_t>(stride_page_table) * cache->page_size)
        return fail(Q8MI_REJECTED, "%s: max_kv_len %u is beyond a page table row of %u", what, max_kv_len, stride_page_table);
    if (!isfinite(scale)) return fail(Q8MI_REJECTED, "%s: scale is not finite", what);
    const uint64_t q_es = q_is_bf16 ? 2 : 4, o_es = out_is_bf16 ? 2 : 4, width = static_cast<uint64_t>(q_heads) * cache->head_dim;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(scratch)) % 16 != 0 ||
        stride_q_row * q_es % 16 != 0 || stride_out_row * o_es % 16 != 0)
        return fail(Q8MI_REJECTED, "%s: rows of q and out must begin on 16-byte boundaries", what);
    if (q_rows > 1 && (stride_q_row < width || stride_out_row < width)) return fail(Q8MI_REJECTED, "%s: rows overlap", what);
    if (static_cast<uint64_t>(n_seqs) * max_q_len > 0x7fffffffull) return fail(Q8MI_REJECTED, "%s: too many sequences", what);

    AttnParams p{};
    p.q = q; p.out = out; p.page_table = page_table; p.kv_lens = kv_lens; p.q_starts = q_starts; p.cache = *cache;
    p.q_rows = q_rows; p.stride_q = stride_q_row; p.stride_out = stride_out_row; p.stride_page_table = stride_page_table;
    p.n_seqs = n_seqs; p.max_q_len = max_q_len; p.q_heads = q_heads; p.group = q_heads / cache->kv_heads;
    p.max_kv_len = max_kv_len; p.scale = scale; p.q_is_bf16 = q_is_bf16; p.out_is_bf16 = out_is_bf16;
    const dim3 grid(n_seqs * max_q_len, q_heads);
    hipStream_t s = as_stream(stream);
    if (cache->head_dim == 64) attention_kernel<64><<<grid, kAttnThreads, 0, s>>>(p);
    else if (cache->head_dim == 128) attention_kernel<128><<<grid, kAttnThreads, 0, s>>>(p);
    else attention_kernel<256><<<grid, kAttnThreads, 0, s>>>(p);
    return check_launch(what);
}
