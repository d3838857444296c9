// Per-head RMS norm of queries and keys, position rotation, and the append of keys and values to a paged cache: the
// step between the Q/K/V projections and the attention, in one launch.
//
//   y = x / sqrt(mean(x^2) + eps) * w            over the head_dim elements of a head
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),   t = position * freq
//
// A head is held by head_dim / 4 neighbouring lanes, four elements each: the sum of squares is a butterfly among them,
// the rotation's partner element comes from another lane (or lies in the same one for neighbouring pairs).  The angle is
// taken in revolutions in 64 bits and only its fraction, at most half a turn, goes to the 32-bit sine and cosine: an
// fp32 product of position 200 000 and a frequency is off by up to 0.008 radians, the fraction by 2e-7.
#include "q8mi_kv.hpp"
#include "q8mi_quantize_core.hpp"

namespace q8mi {
namespace {

constexpr uint32_t kAppendThreads = 256;
constexpr uint32_t kAppendWaves = kAppendThreads / kWave;
// Few tokens: a wave per head (or two, or four, that fit its lanes), so that one token occupies several CUs.  From kManyWaves
// such waves on, a workgroup per token, kManyHeads times as many heads a wave at a time: the angles of a token are worked out
// once for all of them (32 heads of 256: 128 tokens 5.7 and not 6.8 us, 192 both 8.2, 256 8.5 and not 9.7, 512 8.9 and not
// 13.9).  Many tokens run at the rate of a copy (2048 of 32 heads of 256 in fp32, 126 MB: 27.7 us) or, in bf16, three quarters
// of it (8191 of 48 heads of 128, 201 MB: 53.6 us; four heads at a time 59, the next ones already on their way 54.5, 16 bytes
// a lane 82: waves in flight count for more than bytes of each).
constexpr uint32_t kManyHeads = 2, kManyWaves = 6144;

struct AppendParams {
    const void *q, *k, *v;
    void *q_out;
    const float *q_weight, *k_weight;
    const double *freqs;
    const int32_t *positions;
    const int64_t *slots;
    q8mi_kv_cache cache;
    uint32_t tokens, q_heads, kv_heads;
    uint32_t stride_q_row, stride_q_head, stride_k_row, stride_v_row, stride_q_out_row;
    uint32_t rotary_dim;
    uint32_t waves_per_token;
    int interleaved;
    int small;            // slots are below 2^32: a 32-bit division finds the page
    uint64_t slots_end;   // pages * page_size
    float eps;
};

template <bool BF16, bool VEC>
__device__ __forceinline__ void load_act4(const void *base, uint64_t at, float (&v)[4]) {
    if constexpr (BF16) {
        const uint16_t *p = static_cast<const uint16_t *>(base) + at;
        if (VEC) {
            const uint2 t = *reinterpret_cast<const uint2 *>(p);
            v[0] = bf16_bits_to_float(static_cast<uint16_t>(t.x & 0xffffu));
            v[1] = bf16_bits_to_float(static_cast<uint16_t>(t.x >> 16));
            v[2] = bf16_bits_to_float(static_cast<uint16_t>(t.y & 0xffffu));
            v[3] = bf16_bits_to_float(static_cast<uint16_t>(t.y >> 16));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = bf16_bits_to_float(p[i]);
        }
    } else {
        const Float4 t = load4<VEC>(static_cast<const float *>(base) + at);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    }
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void store_act4(void *base, uint64_t at, const float (&v)[4]) {
    if constexpr (BF16) {
        uint16_t *p = static_cast<uint16_t *>(base) + at;
        const uint2 h = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
        if (VEC) {
            *reinterpret_cast<uint2 *>(p) = h;
        } else {
            p[0] = static_cast<uint16_t>(h.x); p[1] = static_cast<uint16_t>(h.x >> 16);
            p[2] = static_cast<uint16_t>(h.y); p[3] = static_cast<uint16_t>(h.y >> 16);
        }
    } else {
        float *p = static_cast<float *>(base) + at;
        if (VEC) {
            *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = v[i];
        }
    }
}

// Sum over the LANES neighbouring lanes that hold a head.
template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
    v += lane_xor<1>(v);
    v += lane_xor<2>(v);
    v += lane_xor<4>(v);
    v += lane_xor<8>(v);
    if constexpr (LANES >= 32) v += lane_xor<16>(v);
    if constexpr (LANES >= 64) v += lane_xor<32>(v);
    return v;
}

// Sine and cosine of a token's pair.
__device__ __forceinline__ float2 angle_of(const AppendParams &p, double position_turns, uint32_t pair) {
    const double turn = position_turns * p.freqs[pair];
    float2 r;
    sincospif(2.0f * static_cast<float>(turn - rint(turn)), &r.x, &r.y);
    return r;
}

// A wave takes kBatch x kAtOnce neighbouring heads of one token at a time, kAtOnce = 64 / (D / 4) of them side by side on its
// lanes, all asked for before the first is looked at.  Heads are numbered queries, keys, values.
//   kBatch = 1: every wave has heads of its own and works its angles out itself
//   kBatch > 1: a workgroup has a token, whose angles it works out once, in LDS
template <bool BF16, uint32_t D, bool VEC, uint32_t kBatch>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(const AppendParams p) {
    constexpr uint32_t kLanes = D / 4, kAtOnce = kWave / kLanes;
    constexpr bool kTokenPerGroup = kBatch > 1;
    __shared__ float2 angles[kTokenPerGroup ? D / 2 : 1];
    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane((kTokenPerGroup ? 0 : blockIdx.x * kAppendWaves) + threadIdx.x / kWave);
    const uint32_t token = kTokenPerGroup ? blockIdx.x : wave / p.waves_per_token;
    if (token >= p.tokens) return;
    const uint32_t heads = p.q_heads + 2 * p.kv_heads;
    const uint32_t e0 = (lane % kLanes) * 4;
    const uint32_t half = p.rotary_dim / 2;
    const bool turns = e0 < p.rotary_dim;
    const uint32_t first_pair = !turns ? 0 : p.interleaved ? e0 / 2 : e0 < half ? e0 : e0 - half;
    const uint32_t pairs = !turns ? 0 : p.interleaved ? 2 : 4;

    float x[kBatch][4];
    auto load = [&](uint32_t first) {   // heads from `first` on
#pragma unroll
        for (uint32_t u = 0; u < kBatch; ++u) {
            const uint32_t h = first + u * kAtOnce + lane / kLanes;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[u][i] = 0.0f;
            if (h < p.q_heads)
                load_act4<BF16, VEC>(p.q, static_cast<uint64_t>(token) * p.stride_q_row + static_cast<uint64_t>(h) * p.stride_q_head + e0, x[u]);
            else if (h < p.q_heads + p.kv_heads)
                load_act4<BF16, VEC>(p.k, static_cast<uint64_t>(token) * p.stride_k_row + (h - p.q_heads) * D + e0, x[u]);
            else if (h < heads)
                load_act4<BF16, VEC>(p.v, static_cast<uint64_t>(token) * p.stride_v_row + (h - p.q_heads - p.kv_heads) * D + e0, x[u]);
        }
    };
    uint32_t first = (kTokenPerGroup ? wave : wave - token * p.waves_per_token) * kBatch * kAtOnce;
    load(first);
    float qw[4], kw[4];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        qw[i] = p.q_weight != nullptr ? p.q_weight[e0 + i] : 1.0f;
        kw[i] = p.k_weight != nullptr ? p.k_weight[e0 + i] : 1.0f;
    }
    const int64_t slot = p.slots[token];

    float c[4] = {1.0f, 1.0f, 1.0f, 1.0f}, s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.rotary_dim != 0) {   // uniform
        const double position = p.positions[token] * 0.15915494309189533577;   // 1 / (2 pi): angles in revolutions
        if constexpr (kTokenPerGroup) {
            if (threadIdx.x < half) angles[threadIdx.x] = angle_of(p, position, threadIdx.x);
            __syncthreads();
        }
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (i < pairs) {
                const float2 a = kTokenPerGroup ? angles[first_pair + i] : angle_of(p, position, first_pair + i);
                s[i] = a.x;
                c[i] = a.y;
            }
    }
    const bool held = slot >= 0 && static_cast<uint64_t>(slot) < p.slots_end;
    const uint32_t slot32 = static_cast<uint32_t>(slot);
    const uint64_t page = p.small ? slot32 / p.cache.page_size : static_cast<uint64_t>(slot) / p.cache.page_size;
    const uint64_t row0 = page * p.cache.stride_page + (static_cast<uint64_t>(slot) - page * p.cache.page_size) * p.cache.stride_token;
    const uint64_t element = kv_element_bytes(p.cache.dtype);

    for (;;) {
#pragma unroll
    for (uint32_t u = 0; u < kBatch; ++u) {
        const uint32_t h = first + u * kAtOnce + lane / kLanes;
        const bool is_q = h < p.q_heads, is_k = !is_q && h < p.q_heads + p.kv_heads;
        const uint32_t hk = is_q ? 0 : is_k ? h - p.q_heads : h - p.q_heads - p.kv_heads;
        float y[4] = {x[u][0], x[u][1], x[u][2], x[u][3]};
        const float squares = head_sum<kLanes>((y[0] * y[0] + y[1] * y[1]) + (y[2] * y[2] + y[3] * y[3]));
        if (is_q ? p.q_weight != nullptr : is_k && p.k_weight != nullptr) {
            // the hardware's reciprocal root is good to one step of fp32; every lane of a head has the same sum
            const float scale = __builtin_amdgcn_rsqf(squares * (1.0f / D) + p.eps);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) y[i] = (y[i] * scale) * (is_q ? qw[i] : kw[i]);
        }
        if (p.rotary_dim != 0) {   // uniform: the exchange needs every lane
            float r[4];
            if (p.interleaved) {
                r[0] = y[0] * c[0] - y[1] * s[0];
                r[1] = y[1] * c[0] + y[0] * s[0];
                r[2] = y[2] * c[1] - y[3] * s[1];
                r[3] = y[3] * c[1] + y[2] * s[1];
            } else {
                const bool low = e0 < half;
                const uint32_t from = turns ? (low ? lane + half / 4 : lane - half / 4) : lane;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float other = as_f32(__builtin_amdgcn_ds_bpermute(static_cast<int>(from * 4), as_i32(y[i])));
                    r[i] = low ? y[i] * c[i] - other * s[i] : y[i] * c[i] + other * s[i];
                }
            }
            if (turns && (is_q || is_k)) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) y[i] = r[i];
            }
        }
        if (is_q) {
            store_act4<BF16, VEC>(p.q_out, static_cast<uint64_t>(token) * p.stride_q_out_row + h * D + e0, y);
        } else if (held && h < heads) {
            uint8_t *pool = static_cast<uint8_t *>(is_k ? p.cache.k : p.cache.v);
            store_kv4(pool + (row0 + hk * p.cache.stride_head) * element, e0, p.cache.dtype,
                      is_k ? p.cache.k_scale : p.cache.v_scale, y);
        }
    }
        if constexpr (!kTokenPerGroup) break;
        first += kAppendWaves * kBatch * kAtOnce;
        if (first >= heads) break;
        load(first);
    }
}

template <bool BF16, uint32_t D>
void launch_append(const AppendParams &p, uint32_t batch, bool vec, uint32_t grid, hipStream_t s) {
    if (batch == 1 && vec) append_kernel<BF16, D, true, 1><<<grid, kAppendThreads, 0, s>>>(p);
    else if (batch == 1) append_kernel<BF16, D, false, 1><<<grid, kAppendThreads, 0, s>>>(p);
    else if (vec) append_kernel<BF16, D, true, kManyHeads><<<grid, kAppendThreads, 0, s>>>(p);
    else append_kernel<BF16, D, false, kManyHeads><<<grid, kAppendThreads, 0, s>>>(p);
}

}  // namespace
}  // namespace q8mi

using namespace q8mi;

extern "C" int q8mi_qk_norm_rope_append(const void *q, const void *k, const void *v, void *q_out, int is_bf16,
                                        uint32_t tokens, uint32_t q_heads, uint32_t stride_q_row, uint32_t stride_q_head,
                                        uint32_t stride_k_row, uint32_t stride_v_row, uint32_t stride_q_out_row,
                                        const float *q_norm_weight, const float *k_norm_weight, float eps,
                                        const double *freqs, uint32_t rotary_dim, int interleaved,
                                        const int32_t *positions, const int64_t *slots, const q8mi_kv_cache *cache,
                                        void *stream) {
    const char *what = "qk_norm_rope_append";
    if (const int rc = check_kv_cache(what, cache); rc != Q8MI_OK) return rc;
    if (tokens == 0) return Q8MI_OK;
    if (q == nullptr || k == nullptr || v == nullptr || q_out == nullptr || slots == nullptr)
        return fail(Q8MI_REJECTED, "%s: null pointer", what);
    if (rotary_dim % 8 != 0 || rotary_dim > cache->head_dim)
        return fail(Q8MI_REJECTED, "%s: rotary_dim %u is not a multiple of 8 up to head_dim", what, rotary_dim);
    if (rotary_dim != 0 && (freqs == nullptr || positions == nullptr))
        return fail(Q8MI_REJECTED, "%s: rotation without frequencies or positions", what);
    const uint64_t D = cache->head_dim;
    if (q_heads == 0 || q_heads > 65536 || cache->kv_heads > 65536) return fail(Q8MI_REJECTED, "%s: %u query heads", what, q_heads);
    if (stride_q_head < D || (tokens > 1 && (stride_q_row < (q_heads - 1) * static_cast<uint64_t>(stride_q_head) + D ||
                                            stride_k_row < cache->kv_heads * D || stride_v_row < cache->kv_heads * D ||
                                            stride_q_out_row < q_heads * D)))
        return fail(Q8MI_REJECTED, "%s: rows overlap", what);
    if (q_out == q && (stride_q_head != D || (tokens > 1 && stride_q_row != stride_q_out_row)))
        return fail(Q8MI_REJECTED, "%s: in place needs dense heads and one row stride", what);
    {
        const uint64_t es = is_bf16 ? 2 : 4;
        auto rows_at = [&](const void *base, uint64_t first, uint64_t stride, uint64_t width) {
            return RowSet{reinterpret_cast<uintptr_t>(base) + first * es, tokens, stride * es, width * es};
        };
        const RowSet to = rows_at(q_out, 0, stride_q_out_row, q_heads * D);
        if (rows_meet(rows_at(k, 0, stride_k_row, cache->kv_heads * D), to) || rows_meet(rows_at(v, 0, stride_v_row, cache->kv_heads * D), to))
            return fail(Q8MI_REJECTED, "%s: q_out overlaps k or v", what);
        if (q_out != q && rows_meet(rows_at(q, 0, stride_q_row, (q_heads - 1) * static_cast<uint64_t>(stride_q_head) + D), to))
            for (uint32_t h = 0; h < q_heads; ++h)   // it may still lie in what is between the heads
                if (rows_meet(rows_at(q, static_cast<uint64_t>(h) * stride_q_head, stride_q_row, D), to))
                    return fail(Q8MI_REJECTED, "%s: q_out overlaps q", what);
    }

    AppendParams p{};
    p.q = q; p.k = k; p.v = v; p.q_out = q_out;
    p.q_weight = q_norm_weight; p.k_weight = k_norm_weight;
    p.freqs = freqs; p.positions = positions; p.slots = slots; p.cache = *cache;
    p.tokens = tokens; p.q_heads = q_heads; p.kv_heads = cache->kv_heads;
    p.stride_q_row = stride_q_row; p.stride_q_head = stride_q_head; p.stride_k_row = stride_k_row;
    p.stride_v_row = stride_v_row; p.stride_q_out_row = stride_q_out_row;
    p.rotary_dim = rotary_dim; p.interleaved = interleaved; p.eps = eps;
    const uint32_t at_once = kWave / (cache->head_dim / 4);
    const uint32_t heads = q_heads + 2 * cache->kv_heads;
    const uint32_t groups = (heads + at_once - 1) / at_once;
    const uint32_t batch = static_cast<uint64_t>(tokens) * groups >= kManyWaves ? kManyHeads : 1;
    p.waves_per_token = groups;
    p.slots_end = static_cast<uint64_t>(cache->pages) * cache->page_size;
    p.small = p.slots_end <= 0xffffffffull;
    const uint64_t grid = batch > 1 ? tokens : (static_cast<uint64_t>(tokens) * groups + kAppendWaves - 1) / kAppendWaves;
    if (grid > 0xffffffull) return fail(Q8MI_REJECTED, "%s: %u tokens are too many for one launch", what, tokens);

    const uintptr_t bases = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                            reinterpret_cast<uintptr_t>(q_out);
    const uint32_t unit = is_bf16 ? 8 : 4;   // elements of 16 bytes
    const bool vec = bases % 16 == 0 && (stride_q_row | stride_q_head | stride_k_row | stride_v_row | stride_q_out_row) % unit == 0;
    hipStream_t s = as_stream(stream);
    auto by_dim = [&](auto bf16) {
        constexpr bool B = decltype(bf16)::value;
        if (cache->head_dim == 64) launch_append<B, 64>(p, batch, vec, static_cast<uint32_t>(grid), s);
        else if (cache->head_dim == 128) launch_append<B, 128>(p, batch, vec, static_cast<uint32_t>(grid), s);
        else launch_append<B, 256>(p, batch, vec, static_cast<uint32_t>(grid), s);
    };
    if (is_bf16) by_dim(std::true_type{});
    else by_dim(std::false_type{});
    return check_launch(what);
}
