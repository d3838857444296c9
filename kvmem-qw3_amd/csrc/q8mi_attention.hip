// Attention of each sequence's newest rows over a paged key / value cache (decode, speculative verification).
//
//   out = sum_t p_t v_t,  p = softmax_t(scale * q . k_t),  t <= kv_len - rows + i
//
// One pass over the cache with a running maximum and sum per query row.  An item is one key head of a sequence and a tile of the
// query rows that read it (rows of the sequence x query heads of the group, 16 a wave); every workgroup takes an equal run of
// all items' tokens, and the pieces' (maximum, sum, output) of an item that several share meet in a second small launch, in
// order, so results repeat.
//
// A step is a tile of 32 tokens, held in LDS exactly as in memory, each row's 16-byte pieces permuted by an exclusive or
// with the token so that the reads below meet different banks.  Tiles travel global -> LDS without passing through
// registers, one page lookup per 16 bytes and lane, so a page may end anywhere inside a tile.  Both products run on the
// matrix cores with the tokens' side as the first operand:
//   scores   S^T = K Q^T     a lane gets 8 tokens (2 x 4) of ONE query row, row lane % 16
//   output   O^T += V^T P^T  V^T from the transposing LDS read; the order of the 32 tokens inside the product is the one
//            the lane's 8 weights already have, so P needs no exchange between lanes, and a lane's outputs belong to the
//            same row as its weights: rescaling by a new maximum is one factor per lane.
// Precision: cache elements are exact operands (bf16, or fp16 for fp16 and e4m3).  The fp32 side, q and the weights, is
// split into operands that add up to it: three bf16 terms (all 24 bits), or two fp16 terms (22 bits) after scaling by a
// power of two that keeps the second term clear of fp16's subnormals (of those from 2^-17 of the row's largest on; smaller ones are
// off by up to 2^-39 of it).  Sums are fp32 throughout.
// Bound by HBM where a key head has few query rows (128 x 4096 tokens of fp16, 8 heads of 128: 2.1 GB in 324 us, 6.6 TB/s; one
// sequence of 131072 tokens of bf16, 4 heads of 256: 537 MB in 92 us), by the matrix cores and VALUs in turn where it has many
// (48 rows, 298 MB: 71 us; the call's largest number of rows arranges the waves of all its sequences, and waves that a sequence has
// no rows for only load), by latency where there is little to read (2000 tokens: 14 us for the two launches).
#include <atomic>

#include "q8mi_kv.hpp"

namespace q8mi {
namespace {

constexpr uint32_t kMaxRows = 16;      // new rows of a sequence
constexpr uint32_t kAttnThreads = 256;
constexpr uint32_t kTile = 32;         // tokens of a step and wave
constexpr uint32_t kMaxChunk = 2048;   // tokens of a workgroup: their page ids are held in LDS
constexpr uint32_t kRowTile = 16;      // query rows of a wave

typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

// Division of numbers below 2^31 by one that the host knows: mulhi(t, magic) >> shift; magic 0: by 1.
struct Divisor {
    uint32_t magic, shift;
};
__device__ __forceinline__ uint32_t operator/(uint32_t t, Divisor d) { return d.magic ? __umulhi(t, d.magic) >> d.shift : t; }
Divisor divisor(uint32_t by) {   // the error of magic, below 2^-31 relative, stays below 1 for every such t
    if (by == 1) return {0, 0};
    uint32_t bits = 1;
    while ((1u << bits) < by) ++bits;
    return {static_cast<uint32_t>((1ull << (31 + bits)) / by + 1), bits - 1};
}

struct AttnParams {
    const void *q;
    void *out;
    float *part;       // [workgroup][its first, its last piece][row of the tile][D]: outputs, not yet divided by their sum
    float2 *part_ml;   // [workgroup][first, last][row of the tile]: maximum (log2 units) and sum
    const int32_t *page_table, *kv_lens, *q_starts;
    q8mi_kv_cache cache;
    uint32_t q_rows, stride_q, stride_out, stride_page_table;
    uint32_t n_seqs, max_q_len, q_heads, group, max_kv_len;
    uint32_t groups;   // workgroups
    Divisor by_page, by_group, by_groups;   // page_size, group, groups
    uint32_t unit_page, unit_token;    // cache strides in units of 16 bytes
    uint32_t waves_log2;               // waves side by side on rows: tiles of 16 << waves_log2 rows, units of 128 >> it tokens
    int whole_loads;                   // the tokens of one transfer instruction never straddle pages
    float scale_log2;  // scale * log2(e) * k_scale
    int q_is_bf16, out_is_bf16;
};

// What a sequence's rows are and see.
struct Rows {
    int64_t start, count, kv_len;
    uint32_t used;     // rows that are computed, 0 .. max_q_len
    uint32_t tokens;   // tokens that some row sees, 0 .. max_kv_len
};
__device__ __forceinline__ Rows rows_of(const AttnParams &p, uint32_t seq) {
    Rows r;
    r.start = static_cast<int64_t>(seq) * p.max_q_len;
    r.count = p.max_q_len;
    if (p.q_starts != nullptr) {
        r.start = p.q_starts[seq];
        r.count = p.q_starts[seq + 1] - r.start;
    }
    r.kv_len = p.kv_lens[seq];
    r.used = r.count < 0 ? 0u : r.count > p.max_q_len ? p.max_q_len : static_cast<uint32_t>(r.count);
    const int64_t seen = r.kv_len - (r.count > r.used ? r.count - r.used : 0);   // by the last computed row
    r.tokens = seen < 0 ? 0u : seen > p.max_kv_len ? p.max_kv_len : static_cast<uint32_t>(seen);
    return r;
}

// The work is counted in units: 128 >> waves_log2 tokens of one key head and one tile of query rows, in the order sequence, head, row
// tile, token.  Every workgroup takes an equal run of them, whatever the lengths of the sequences: the end of one item, whole
// items, the beginning of one.  An item that several workgroups share is joined by a second kernel.
__device__ __forceinline__ uint32_t units_of_item(uint32_t waves_log2, const Rows &r) {
    return r.tokens ? (r.tokens + (128u >> waves_log2) - 1) >> (7 - waves_log2) : 1;   // without tokens: zeros to write
}
__device__ __forceinline__ uint32_t units_of_seq(const AttnParams &p, uint32_t waves_log2, const Rows &r) {
    const uint32_t tiles = (r.used * p.group + (16u << waves_log2) - 1) >> (4 + waves_log2);
    return tiles * p.cache.kv_heads * units_of_item(waves_log2, r);
}
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ uint32_t page_of(const AttnParams &p, uint32_t t) {
    return t / p.by_page;
}

__device__ __forceinline__ void store_out(const AttnParams &p, uint64_t at, float v) {
    if (p.out_is_bf16) static_cast<uint16_t *>(p.out)[at] = float_to_bf16_bits(v);
    else static_cast<float *>(p.out)[at] = v;
}

// 16 bytes per lane, each lane from its own address, to LDS at lds_off + lane * 16.  Inline assembly, so that the
// compiler does not make every later LDS read wait for it; the counts are waited for by hand.  A cache is read once a step:
// the streaming hint (nt) leaves the L2 to others and is 10 % faster (128 x 4096 tokens of fp16: 367 -> 326 us).
__device__ __forceinline__ void dma16_lanes(const void *lane_ptr, uint32_t lds_off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(lds_off), "v"(lane_ptr)
                 : "memory", "m0");
}
// The same from a scalar base plus a 32-bit offset per lane.
__device__ __forceinline__ void dma16_base(const void *uniform_base, uint32_t lane_off, uint32_t lds_off) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds_off), "v"(lane_off), "s"(uniform_base)
                 : "memory", "m0");
}
__device__ __forceinline__ const uint8_t *uniform_ptr(const uint8_t *p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
    return reinterpret_cast<const uint8_t *>((static_cast<uint64_t>(hi) << 32) | lo);
}
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

using lds_ptr = __attribute__((address_space(3))) void *;
__device__ __forceinline__ uint32_t lds_offset(const void *p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_ptr)p));
}

template <int KV>
struct Operand;   // how eight elements become a matrix operand, and fp32 values a sum of operands
template <>
struct Operand<Q8MI_KV_BF16> {
    using Raw = v8s;
    static __device__ __forceinline__ v8s operand(Raw x) { return x; }
    static constexpr int kTerms = 3;
    static constexpr float kWeightScale = 1.0f;
    static __device__ __forceinline__ v4f mma(v8s a, v8s b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
    }
    // the upper 16 bits are a bf16: each term takes eight of the 24 bits, the last one is exact
    static __device__ __forceinline__ void split(const float (&x)[8], v8s (&t)[kTerms]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float r = x[i];
#pragma unroll
            for (int k = 0; k < kTerms; ++k) {
                const uint32_t hi = __builtin_bit_cast(uint32_t, r) & 0xffff0000u;
                t[k][i] = static_cast<short>(hi >> 16);
                r -= __builtin_bit_cast(float, hi);
            }
        }
    }
};
template <>
struct Operand<Q8MI_KV_F16> {
    using Raw = v8s;
    static __device__ __forceinline__ v8s operand(Raw x) { return x; }
    static constexpr int kTerms = 2;
    static constexpr float kWeightScale = 16384.0f;   // weights are at most 1: the terms' last step is 2^-24 / 2^14
    static __device__ __forceinline__ v4f mma(v8s a, v8s b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ void split(const float (&x)[8], v8s (&t)[kTerms]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const _Float16 hi = static_cast<_Float16>(x[i]);
            const _Float16 lo = static_cast<_Float16>(x[i] - static_cast<float>(hi));
            t[0][i] = __builtin_bit_cast(short, hi);
            t[1][i] = __builtin_bit_cast(short, lo);
        }
    }
};
template <>
struct Operand<Q8MI_KV_E4M3> : Operand<Q8MI_KV_F16> {
    using Raw = v2i;
    static __device__ __forceinline__ v8s operand(Raw w) {   // exact: every e4m3 value is an fp16
        union { v2h h[4]; v8s s; } u;
        u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, 1.0f, false);
        u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.x, 1.0f, true);
        u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, 1.0f, false);
        u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w.y, 1.0f, true);
        return u.s;
    }
};

// Whether one of the elements in a word is an infinity or NaN.
template <int KV>
__device__ __forceinline__ bool not_finite(int w) {
    if constexpr (KV == Q8MI_KV_E4M3)   // 0x7f / 0xff, the type's only ones: a byte whose lower seven bits carry into the eighth
        return (((w & 0x7f7f7f7f) + 0x01010101) & static_cast<int>(0x80808080u)) != 0;
    constexpr int kTop = KV == Q8MI_KV_BF16 ? 0x7f80 : 0x7c00;
    return (w & kTop) == kTop || (w >> 16 & kTop) == kTop;
}

// The word with such elements cleared.
template <int KV>
__device__ __forceinline__ int finite_part(int w) {
    const uint32_t u = static_cast<uint32_t>(w);
    if constexpr (KV == Q8MI_KV_E4M3) {
        const uint32_t odd = ((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;   // bit 7 of every such byte
        return static_cast<int>(u & ~(odd | (odd - (odd >> 7))));
    }
    constexpr uint32_t kTop = KV == Q8MI_KV_BF16 ? 0x7f80 : 0x7c00;
    return static_cast<int>(((u & kTop) == kTop ? 0 : u & 0xffffu) | ((u >> 16 & kTop) == kTop ? 0 : u & 0xffff0000u));
}

__device__ __forceinline__ float rows_max(float v) {   // over the four lanes that hold a query row
    v = fmaxf(v, lane_xor<16>(v));
    return fmaxf(v, lane_xor<32>(v));
}
__device__ __forceinline__ float rows_sum(float v) {
    v += lane_xor<16>(v);
    return v + lane_xor<32>(v);
}

// WR waves side by side on the query rows (16 each), 4 / WR of these groups on alternating tiles of tokens.
template <uint32_t D, int KV, uint32_t WR>
struct Layout {
    static constexpr uint32_t kRowBytes = D * (KV == Q8MI_KV_E4M3 ? 1 : 2);
    static constexpr uint32_t kLanesPerRow = kRowBytes / 16;
    static constexpr uint32_t kRowsPerLoad = kWave / kLanesPerRow;    // tokens that one transfer instruction of a wave brings
    static constexpr uint32_t kLoads = kTile / kRowsPerLoad;          // transfers of a tile
    static constexpr uint32_t kLoadsPerWave = kLoads >= WR ? kLoads / WR : 1;
    static constexpr uint32_t kSwizzle = (kLanesPerRow < 16 ? kLanesPerRow : 16) - 1;
    static constexpr uint32_t kTileBytes = kTile * kRowBytes;
    static constexpr uint32_t kGroups = 4 / WR;
    static constexpr uint32_t kUnit = kGroups * kTile;                 // tokens of a step
    // Waves that share a tile meet at barriers, of which two stages need one a step instead of four (16 sequences of 8 rows, heads
    // of 256: 91 -> 78 us, together with waves that only load).  Waves on tiles of their own are hidden by each other and by the
    // other workgroups of the CU, for which a second stage leaves less room (heads of 64, 64 sequences of 4096 tokens: 90 and 85 us,
    // one of 6000: 12.8 and 14.6).
    static constexpr uint32_t kStages = WR > 1 && kGroups * 4 * kTileBytes <= 64 * 1024 ? 2 : 1;
    static_assert(WR < 4 || kStages == 2, "a wave without rows passes no barrier but the first of a step");
    static constexpr uint32_t kTiles = 0;                              // [group][stage][K, V][tile]
    static constexpr uint32_t kPages = kGroups * kStages * 2 * kTileBytes;   // page ids of the chunk
    static constexpr uint32_t kMergeBytes = kGroups > 1 ? 4 * kRowTile * (D + 4) * 4 + 4 * kRowTile * 8 : 0;
    static constexpr uint32_t kScores = kPages + (kMaxChunk + 2) * 4;  // [wave][new row's token][row of the wave]
    static constexpr uint32_t kEnd = kScores + 4 * kMaxRows * kRowTile * 4;
    static constexpr uint32_t kBytes = kEnd > kMergeBytes ? kEnd : kMergeBytes;
    static constexpr uint32_t kByLds = 160 * 1024 / kBytes, kByRegisters = D == 64 ? 3 : 2;
    static constexpr uint32_t kResident = kByLds < kByRegisters ? kByLds : kByRegisters;   // workgroups of a CU
};

template <uint32_t D, int KV, uint32_t WR>
__global__ __launch_bounds__(kAttnThreads, (Layout<D, KV, WR>::kResident)) void attention_kernel(const AttnParams p) {
    using L = Layout<D, KV, WR>;
    using Op = Operand<KV>;
    constexpr uint32_t kSteps = D / 32, kOuts = D / 16;
    // steps that LDS reads run ahead of the products: fewer where registers are short
    constexpr uint32_t kKeysAhead = D == 256 && KV == Q8MI_KV_BF16 && WR > 1 ? 1 : 2;
    constexpr uint32_t kBlock = D == 256 && KV == Q8MI_KV_BF16 && WR > 1 ? 2 : 4;   // tiles of outputs worked on in turn
    extern __shared__ __align__(16) uint8_t lds[];
    int32_t *pages = reinterpret_cast<int32_t *>(lds + L::kPages);
    float *kept_scores = reinterpret_cast<float *>(lds + L::kScores);
    __shared__ uint32_t bad_pages[kAttnThreads / kWave];

    const uint32_t lane = threadIdx.x % kWave;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t wr = wave % WR, wg = wave / WR;
    const uint32_t g = lane / 16;

    // this workgroup's units: begin .. end - 1, the first of them in sequence seq, whose own begin at seq_begin
    constexpr uint32_t kLog = WR == 1 ? 0 : WR == 2 ? 1 : 2;
    auto units_at = [&](uint32_t s) { return s < p.n_seqs ? units_of_seq(p, kLog, rows_of(p, s)) : 0; };
    auto upto_lane = [&](uint32_t v) {   // sum over this lane and those below it
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t other = __shfl_up(v, d);
            v += lane >= static_cast<uint32_t>(d) ? other : 0;
        }
        return v;
    };
    uint32_t total = 0, mine = 0, upto = 0;
    if (p.n_seqs == 1) {
        total = units_at(0);
    } else {
        for (uint32_t at = (p.n_seqs - 1) / kWave * kWave;; at -= kWave) {   // ends with the first 64 in `mine` and `upto`
            mine = units_at(at + lane);
            upto = upto_lane(mine);
            total += __builtin_amdgcn_readlane(upto, 63);
            if (at == 0) break;
        }
    }
    const uint32_t share = __builtin_amdgcn_readfirstlane((total + p.groups - 1) / p.by_groups);
    uint32_t begin = blockIdx.x * share;
    if (begin >= total) return;
    const uint32_t end = __builtin_amdgcn_readfirstlane(begin + share < total ? begin + share : total);
    uint32_t seq = 0, seq_begin = 0;
    if (p.n_seqs > 1) {
        for (;;) {
            const uint64_t beyond = __builtin_amdgcn_ballot_w64(seq_begin + upto > begin);
            if (beyond != 0) {   // begin < total: some lane's
                const int who = __builtin_ctzll(beyond);
                seq += who;
                seq_begin += __builtin_amdgcn_readlane(upto, who) - __builtin_amdgcn_readlane(mine, who);
                break;
            }
            seq += kWave;
            seq_begin += __builtin_amdgcn_readlane(upto, 63);
            mine = units_at(seq + lane);
            upto = upto_lane(mine);
        }
        seq = __builtin_amdgcn_readfirstlane(seq);
        seq_begin = __builtin_amdgcn_readfirstlane(seq_begin);
    }

    for (uint32_t piece = 0; begin < end;) {
    const Rows rows = rows_of(p, seq);
    const uint32_t item_units = units_of_item(kLog, rows), seq_units = units_of_seq(p, kLog, rows);
    if (begin >= seq_begin + seq_units) {   // on to the next sequence
        seq_begin += seq_units;
        ++seq;
        continue;
    }
    const uint32_t n_rows = rows.used * p.group, tiles = (n_rows + WR * kRowTile - 1) / (WR * kRowTile);
    const uint32_t item = __builtin_amdgcn_readfirstlane((begin - seq_begin) / item_units);
    const uint32_t unit0 = __builtin_amdgcn_readfirstlane((begin - seq_begin) % item_units);
    const uint32_t units = item_units - unit0 < end - begin ? item_units - unit0 : end - begin;
    const uint32_t kv_head = __builtin_amdgcn_readfirstlane(item / tiles);
    const uint32_t row0 = (item - kv_head * tiles) * (WR * kRowTile);
    const bool whole_item = units == item_units;
    const uint32_t slot_of_piece = blockIdx.x * 2 + (piece ? 1 : 0);   // only a first or last piece is not whole
    ++piece;
    begin += units;

    const int32_t *table = p.page_table + static_cast<uint64_t>(seq) * p.stride_page_table;
    uint32_t t0 = unit0 * L::kUnit;                                           // tokens of this piece: t0 .. t_end - 1,
    const uint32_t t_end = t0 + units * L::kUnit < rows.tokens ? t0 + units * L::kUnit : rows.tokens;
    uint32_t t1 = t0 + kMaxChunk < t_end ? t0 + kMaxChunk : t_end;            // by chunks t0 .. t1 - 1 with their page ids in LDS
    uint32_t page0 = page_of(p, t0);

    // this lane's query row
    const uint32_t row = row0 + wr * kRowTile + lane % 16;
    const uint32_t token = row / p.by_group, head = kv_head * p.group + row - token * p.group;
    const int64_t q_row = rows.start + token;
    const bool live = row < n_rows && q_row >= 0 && q_row < p.q_rows;
    const int64_t last64 = rows.kv_len - rows.count + token;                   // the last token it sees
    const int32_t last = !live || last64 < 0 ? -1 : last64 >= p.max_kv_len ? static_cast<int32_t>(p.max_kv_len) - 1
                                                                           : static_cast<int32_t>(last64);

    // the queries' bits (lanes without a row read row 0: what they compute goes nowhere)
    v4i raw[kSteps][2] = {};
    if (p.q_is_bf16) {
        const uint16_t *src = static_cast<const uint16_t *>(p.q) + (live ? static_cast<uint64_t>(q_row) * p.stride_q : 0) + head * D + g * 8;
#pragma unroll
        for (uint32_t j = 0; j < kSteps; ++j) raw[j][0] = *reinterpret_cast<const v4i *>(src + j * 32);
    } else {
        const float *src = static_cast<const float *>(p.q) + (live ? static_cast<uint64_t>(q_row) * p.stride_q : 0) + head * D + g * 8;
#pragma unroll
        for (uint32_t j = 0; j < kSteps; ++j) {
            raw[j][0] = *reinterpret_cast<const v4i *>(src + j * 32);
            raw[j][1] = *reinterpret_cast<const v4i *>(src + j * 32 + 4);
        }
    }
    bool any_bad = false;
    auto load_pages = [&]() {
        const uint32_t n_pages = t1 > t0 ? page_of(p, t1 - 1) - page0 + 1 : 0;
        bool bad = false;
        for (uint32_t i = threadIdx.x; i < n_pages; i += kAttnThreads) {
            const int32_t id = table[page0 + i];
            const bool ok = id >= 0 && static_cast<uint32_t>(id) < p.cache.pages;
            pages[i] = ok ? id : -1;
            bad |= !ok;
        }
        // Everything requested so far is here before the first tile is asked for: a later wait for it would wait for the tile.
        __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
        const bool wave_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
        if (lane == 0) bad_pages[wave] = wave_bad;
        __syncthreads();
        any_bad = false;
#pragma unroll
        for (uint32_t w = 0; w < kAttnThreads / kWave; ++w) any_bad |= bad_pages[w] != 0;
        any_bad = __builtin_amdgcn_readfirstlane(any_bad);
    };
    if (piece > 1) __syncthreads();   // the piece before has left LDS
    load_pages();

    // ---- the tiles' way into LDS ----
    uint32_t k_tile = L::kTiles + wg * L::kStages * 2 * L::kTileBytes, v_tile = k_tile + L::kTileBytes;   // of this step
    const uint32_t lds0 = lds_offset(lds);
    const uint64_t head_bytes = kv_head * p.cache.stride_head * kv_element_bytes(p.cache.dtype);
    const uint8_t *k_pool = uniform_ptr(static_cast<const uint8_t *>(p.cache.k) + head_bytes);
    const uint8_t *v_pool = uniform_ptr(static_cast<const uint8_t *>(p.cache.v) + head_bytes);
    auto page_id = [&](uint32_t t) { return pages[page_of(p, t) - page0]; };   // t0 <= t < t1
    auto visible = [&](uint32_t t) { return t < t1 && page_id(t) >= 0; };
    // Where token first + lane % 32 lies, in units of 16 bytes; tokens that do not exist read the pool's first row.
    auto locate = [&](uint32_t first) -> uint32_t {
        const uint32_t t = first + lane % kTile;
        if (t >= t1) return 0;
        const uint32_t pg = page_of(p, t);
        const int32_t id = pages[pg - page0];
        return id < 0 ? 0 : static_cast<uint32_t>(id) * p.unit_page + (t - pg * p.cache.page_size) * p.unit_token;
    };
    uint32_t piece0 = lane % L::kLanesPerRow ^ (lane / L::kLanesPerRow & L::kSwizzle);
    const uint32_t rows_off = lane / L::kLanesPerRow * p.unit_token * 16;   // used where p.whole_loads: below 4 GiB
    auto load_tile = [&](const uint8_t *pool, uint32_t tile, uint32_t where) {
        asm volatile("" : "+v"(piece0));   // its variants are made anew, not held in registers
        constexpr uint32_t kUnroll = L::kLoadsPerWave < 4 ? L::kLoadsPerWave : 4;   // of up to 16: code has to be fetched, too
        if (p.whole_loads) {
            // a transfer's tokens are neighbours in one page: a scalar base, and what the lanes add never changes
#pragma unroll kUnroll
            for (uint32_t u = 0; u < L::kLoadsPerWave; ++u) {
                const uint32_t r = u * WR + wr;
                if (L::kLoads < WR && r >= L::kLoads) break;   // uniform
                const uint32_t slot0 = r * L::kRowsPerLoad;
                const uint64_t at = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(where), static_cast<int>(slot0)));
                dma16_base(pool + at * 16, rows_off + (piece0 ^ (slot0 & L::kSwizzle)) * 16, lds0 + tile + r * 1024);
            }
            return;
        }
#pragma unroll kUnroll
        for (uint32_t u = 0; u < L::kLoadsPerWave; ++u) {
            const uint32_t r = u * WR + wr;
            if (L::kLoads < WR && r >= L::kLoads) break;   // uniform
            const uint32_t slot0 = r * L::kRowsPerLoad;
            const uint32_t at = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(
                static_cast<int>((lane / L::kLanesPerRow + slot0) * 4), static_cast<int>(where)));
            const uint64_t off = static_cast<uint64_t>(at) + (piece0 ^ (slot0 & L::kSwizzle));
            dma16_lanes(pool + off * 16, lds0 + tile + r * 1024);
        }
    };

    // Where this lane reads its operands: piece c of a row lies at c ^ (token & kSwizzle), and c = (step or tile of
    // outputs) * 4, 2 or 1 | (lane part), so that one exclusive or with the first part gives every address.
    uint32_t k_at, v_at;
    {
        const uint32_t i = lane % 16;
        const uint32_t k_piece = (KV == Q8MI_KV_E4M3 ? g / 2 : g) ^ (i & L::kSwizzle);
        k_at = k_tile + i * L::kRowBytes + k_piece * 16 + (KV == Q8MI_KV_E4M3 ? g % 2 * 8 : 0);
        const uint32_t v_token = KV == Q8MI_KV_E4M3 ? (i / 2 < 4 ? 0 : 12) + g * 4 + i / 2 : g * 4 + i / 4;
        const uint32_t v_piece = (KV == Q8MI_KV_E4M3 ? 0 : i % 4 / 2) ^ (v_token & L::kSwizzle);
        v_at = v_tile + v_token * L::kRowBytes + v_piece * 16 + i % 2 * 8;
    }

    // ---- the walk over the chunk ----
    float m = -INFINITY, l = 0.0f;
    v4f o[kOuts];
#pragma unroll
    for (uint32_t d = 0; d < kOuts; ++d) o[d] = v4f{0, 0, 0, 0};
    const int64_t first_last = rows.kv_len - rows.count;   // what row 0 of the sequence sees last
    uint32_t odd_tokens = 0;                               // bit i: token first_last + 1 + i holds values that are not finite
    uint32_t n_steps = (t1 - t0 + L::kUnit - 1) / L::kUnit;
    auto load_first = [&]() {
    if (n_steps == 0) return;   // uniform
    const uint32_t where = locate(t0 + wg * kTile);
    load_tile(k_pool, k_tile, where);
    load_tile(v_pool, v_tile, where);
    };
    load_first();
    __builtin_amdgcn_sched_barrier(0);

    // the queries as operands, while the first tiles travel
    float qv[kSteps][8];
#pragma unroll
    for (uint32_t j = 0; j < kSteps; ++j) {
        const int ws[8] = {raw[j][0].x, raw[j][0].y, raw[j][0].z, raw[j][0].w, raw[j][1].x, raw[j][1].y, raw[j][1].z, raw[j][1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            qv[j][i] = as_f32(!p.q_is_bf16 ? ws[i] : i % 2 ? ws[i / 2] & static_cast<int>(0xffff0000u) : ws[i / 2] << 16);
    }
    int row_shift = 0;   // fp16 operands: the row's largest |q| goes to 2^14 .. 2^15, so that the second term's last step is 2^-38 of it
    if constexpr (KV != Q8MI_KV_BF16) {
        float top = 0.0f;
#pragma unroll
        for (uint32_t j = 0; j < kSteps; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(qv[j][i]));
        top = rows_max(top);
        if (top > 0.0f && top < INFINITY) {
            (void)frexpf(top, &row_shift);
            row_shift = 15 - row_shift;   // up to 163: applied by ldexp, since as a factor it would leave fp32
        }
    }
    v8s qf[kSteps][Op::kTerms];
#pragma unroll
    for (uint32_t j = 0; j < kSteps; ++j) {
        if constexpr (KV != Q8MI_KV_BF16) {
#pragma unroll
            for (int i = 0; i < 8; ++i) qv[j][i] = ldexpf(qv[j][i], row_shift);
        }
        Op::split(qv[j], qf[j]);
    }
    const float to_log2 = KV == Q8MI_KV_BF16 ? p.scale_log2 : ldexpf(p.scale_log2, -row_shift);

    auto turn = [&]() {   // to the other stage
        k_tile ^= 2 * L::kTileBytes; v_tile ^= 2 * L::kTileBytes;
        k_at ^= 2 * L::kTileBytes; v_at ^= 2 * L::kTileBytes;
    };
    // a wave of the tile's end without a query row only loads: its LDS reads and products would slow the others (48 rows in
    // tiles of 64: 86 -> 78 us)
    const bool idle = row0 + wr * kRowTile >= n_rows;   // uniform
    for (uint32_t step = 0; n_steps != 0; ++step) {
        if (step == n_steps) {   // the next chunk of the piece
            if (t1 == t_end) break;
            t0 = t1;
            t1 = t0 + kMaxChunk < t_end ? t0 + kMaxChunk : t_end;
            page0 = page_of(p, t0);
            n_steps = (t1 - t0 + L::kUnit - 1) / L::kUnit;
            step = 0;
            __syncthreads();   // every wave has read the page ids it needed
            load_pages();
            load_first();
        }
        const uint32_t first = t0 + (step * L::kGroups + wg) * kTile;
        const uint32_t next = locate(first + L::kGroups * kTile);
        const bool more = step + 1 < n_steps;
        if constexpr (L::kStages == 2) {   // this step's tile is here, and every wave has left the one before: its place takes the next
            wait_loads<0>();
            __syncthreads();
            if (more) {
                load_tile(k_pool, k_tile ^ 2 * L::kTileBytes, next);
                load_tile(v_pool, v_tile ^ 2 * L::kTileBytes, next);
            }
        } else {   // the keys are here; the values may still travel
            wait_loads<L::kLoadsPerWave>();
            if constexpr (WR > 1) __syncthreads();
        }
        // whole: every row sees the whole tile (with several waves on a tile: all tiles of the step, so that the barriers below
        // are met by all)
        const uint32_t behind = WR > 1 ? t0 + (step + 1) * L::kGroups * kTile : first + kTile;
        const bool whole = !any_bad && behind <= t1 && static_cast<int64_t>(behind) - 1 <= first_last;   // uniform
        if constexpr (WR == 4) {   // two stages: no barrier before the next step's
            if (idle && whole) {
                turn();
                continue;
            }
        }
        asm volatile("" : "+v"(k_at), "+v"(v_at));   // their variants are made anew each step: held, they cost 32 registers
        v4f s[2][Op::kTerms];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < Op::kTerms; ++k) s[h][k] = v4f{0, 0, 0, 0};
        // The operands of a step are read while the products of the step before run; the barriers keep the compiler from
        // reading all of them ahead into registers that it does not have.
        auto keys = [&](uint32_t j, uint32_t h) {
            return *reinterpret_cast<const typename Op::Raw *>(lds + (k_at ^ j * (KV == Q8MI_KV_E4M3 ? 32 : 64)) + h * 16 * L::kRowBytes);
        };
        typename Op::Raw kf[kKeysAhead + 1][2];
#pragma unroll
        for (uint32_t j = 0; j < kKeysAhead; ++j) {
            kf[j][0] = keys(j, 0);
            kf[j][1] = keys(j, 1);
        }
#pragma unroll
        for (uint32_t j = 0; j < kSteps; ++j) {
            if (j + kKeysAhead < kSteps) {
                kf[(j + kKeysAhead) % (kKeysAhead + 1)][0] = keys(j + kKeysAhead, 0);
                kf[(j + kKeysAhead) % (kKeysAhead + 1)][1] = keys(j + kKeysAhead, 1);
            }
            const v8s a[2] = {Op::operand(kf[j % (kKeysAhead + 1)][0]), Op::operand(kf[j % (kKeysAhead + 1)][1])};
#pragma unroll
            for (int k = 0; k < Op::kTerms; ++k)
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) s[h][k] = Op::mma(a[h], qf[j][k], s[h][k]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (L::kStages == 1) {
            wait_lds_reads();
            if constexpr (WR > 1) __syncthreads();
            if (more) load_tile(k_pool, k_tile, next);
        }

        float w[8];   // of a lane's eight tokens: first + h * 16 + g * 4 + i
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float dot = s[h][Op::kTerms - 1][i];
#pragma unroll
                for (int k = Op::kTerms - 2; k >= 0; --k) dot += s[h][k][i];
                w[h * 4 + i] = dot * to_log2;
            }
        uint32_t there = 0;   // not whole: bit i, token first + i exists
        if (!whole) {
            there = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(visible(first + lane % kTile)));
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                const uint32_t slot = i / 4 * 16 + g * 4 + i % 4;
                w[i] = (there >> slot & 1) && static_cast<int32_t>(first + slot) <= last ? w[i] : -INFINITY;
            }
        }
        float top = fmaxf(fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3])), fmaxf(fmaxf(w[4], w[5]), fmaxf(w[6], w[7])));
        if (__builtin_amdgcn_ballot_w64(top > m) != 0) {   // uniform, and rare after the first tiles; NaN changes no maximum
            top = fmaxf(rows_max(top), m);
            const float keep = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
            l *= keep;
#pragma unroll
            for (uint32_t d = 0; d < kOuts; ++d) o[d] *= keep;
            m = top;
        }
        const float base = m == -INFINITY ? 0.0f : m;
        float scores[8];   // dead but for the rare tokens kept below
#pragma unroll
        for (int i = 0; i < 8; ++i) scores[i] = w[i];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = __builtin_amdgcn_exp2f(w[i] - base);
            l += w[i];
            w[i] *= Op::kWeightScale;
        }
        v8s pf[Op::kTerms];
        Op::split(w, pf);

        // the values are here; what was asked for after them may still travel
        if constexpr (L::kStages == 1) {
            if (more) wait_loads<L::kLoadsPerWave>();
            else wait_loads<0>();
            if constexpr (WR > 1) __syncthreads();
        }
        // V^T operand of 16 outputs: the transposing read gives lane i of a group of 16 column i of the rows that the
        // group's lanes point to, here its tokens g * 4 .. + 3 and 16 + g * 4 .. + 3
        auto values = [&](uint32_t d) -> typename Op::Raw {
            if constexpr (KV == Q8MI_KV_E4M3) {
                using tp = __attribute__((address_space(3))) v2i *;
                return __builtin_amdgcn_ds_read_tr8_b64_v2i32((tp)(lds + (v_at ^ d * 16)));
            } else {
                using tp = __attribute__((address_space(3))) v4s *;
                uint8_t *at = lds + (v_at ^ d * 32);
                const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tp)at);
                const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((tp)(at + 16 * L::kRowBytes));
                return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
            }
        };
        if (!whole) {
            // A weight of 0 does not silence an infinity or NaN.  What no row sees (rows behind the last token, tokens of a
            // bad page) is cleared; of a token that some rows see and others not, a new row's own, such elements are cleared
            // here and added behind the loop to the rows that see them.
            const uint32_t slot = lane % kTile;
            v4i *mine = reinterpret_cast<v4i *>(lds + v_tile + slot * L::kRowBytes + lane / kTile * (L::kRowBytes / 2));
            const bool partly = static_cast<int64_t>(first) + slot > first_last;
            bool odd = false;
            if (!(there >> slot & 1)) {
                for (uint32_t i = 0; i < L::kRowBytes / 32; ++i) mine[i] = v4i{0, 0, 0, 0};
            } else if (partly) {
                for (uint32_t i = 0; i < L::kRowBytes / 32; ++i) {
                    const v4i x = mine[i];
                    odd |= not_finite<KV>(x.x) || not_finite<KV>(x.y) || not_finite<KV>(x.z) || not_finite<KV>(x.w);
                }
            }
            const uint64_t odd_lanes = __builtin_amdgcn_ballot_w64(odd);
            for (uint32_t slots = static_cast<uint32_t>(odd_lanes) | static_cast<uint32_t>(odd_lanes >> 32); slots != 0; slots &= slots - 1) {
                const uint32_t at = __builtin_ctz(slots);   // token first + at, new row number
                const uint32_t number = static_cast<uint32_t>(static_cast<int64_t>(first) + at - first_last) - 1;
                if (g == at / 4 % 4) {
                    float score = -INFINITY;   // register i of these lanes
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) score = i == at / 16 * 4 + at % 4 ? scores[i] : score;
                    kept_scores[(wave * kMaxRows + number) * kRowTile + lane % 16] = score;
                }
                odd_tokens |= 1u << number;
            }
            if constexpr (WR > 1) __syncthreads();   // every wave has read what is cleared now
            if (odd) {
                for (uint32_t i = 0; i < L::kRowBytes / 32; ++i) {
                    const v4i x = mine[i];
                    mine[i] = v4i{finite_part<KV>(x.x), finite_part<KV>(x.y), finite_part<KV>(x.z), finite_part<KV>(x.w)};
                }
            }
            if constexpr (WR > 1) __syncthreads();
            wait_lds_reads();
        }
        // kBlock accumulators in turn, so that a product does not wait for the one before it
        typename Op::Raw vf[2][kBlock];
#pragma unroll
        for (uint32_t d = 0; d < kBlock; ++d) vf[0][d] = values(d);
#pragma unroll
        for (uint32_t b = 0; b < kOuts / kBlock; ++b) {
            if ((b + 1) * kBlock < kOuts) {
#pragma unroll
                for (uint32_t d = 0; d < kBlock; ++d) vf[(b + 1) % 2][d] = values((b + 1) * kBlock + d);
            }
            v8s a[kBlock];
#pragma unroll
            for (uint32_t d = 0; d < kBlock; ++d) a[d] = Op::operand(vf[b % 2][d]);
#pragma unroll
            for (int k = Op::kTerms - 1; k >= 0; --k)
#pragma unroll
                for (uint32_t d = 0; d < kBlock; ++d) o[b * kBlock + d] = Op::mma(a[d], pf[k], o[b * kBlock + d]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (L::kStages == 1) {
            wait_lds_reads();
            if constexpr (WR > 1) __syncthreads();
            if (more) load_tile(v_pool, v_tile, next);
        } else {
            turn();
        }
    }
    l = rows_sum(l);
    while (odd_tokens != 0) {   // uniform; see above
        const uint32_t number = __builtin_ctz(odd_tokens);
        odd_tokens &= odd_tokens - 1;
        const uint32_t t = static_cast<uint32_t>(first_last + 1 + number);
        const float weight = Op::kWeightScale * __builtin_amdgcn_exp2f(kept_scores[(wave * kMaxRows + number) * kRowTile + lane % 16] - m);
        const bool sees = static_cast<int32_t>(t) <= last;
        const uint32_t pg = page_of(p, t);
        const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(table[pg])) * p.unit_page + static_cast<uint64_t>(t - pg * p.cache.page_size) * p.unit_token;
#pragma unroll
        for (uint32_t d = 0; d < kOuts; ++d) {
            const uint8_t *src = v_pool + at * 16 + (d * 16 + g * 4) * (KV == Q8MI_KV_E4M3 ? 1 : 2);
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const int bits = KV == Q8MI_KV_E4M3 ? src[i] : reinterpret_cast<const uint16_t *>(src)[i];
                const float v = KV == Q8MI_KV_BF16 ? as_f32(bits << 16) : KV == Q8MI_KV_F16 ? half_bits_to_float(static_cast<uint16_t>(bits)) : NAN;
                o[d][i] = sees && not_finite<KV>(bits) ? o[d][i] + weight * v : o[d][i];
            }
        }
    }

    // ---- the groups of a workgroup meet ----
    if constexpr (L::kGroups > 1) {
        // per wave [16 rows][D + 4] outputs, then [16 rows] maxima and sums; the pad spreads the rows over the banks
        float *mo = reinterpret_cast<float *>(lds);
        float2 *ml = reinterpret_cast<float2 *>(lds + 4 * kRowTile * (D + 4) * 4);
        __syncthreads();
        if (g == 0) ml[wave * kRowTile + lane % 16] = make_float2(m, l);
        __syncthreads();
        float all = -INFINITY;
#pragma unroll
        for (uint32_t k = 0; k < L::kGroups; ++k) all = fmaxf(all, ml[(k * WR + wr) * kRowTile + lane % 16].x);
        float sum = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < L::kGroups; ++k) {
            const float2 x = ml[(k * WR + wr) * kRowTile + lane % 16];
            sum += x.x == all ? x.y : x.y * __builtin_amdgcn_exp2f(x.x - all);
        }
        const float f = m == all ? 1.0f : __builtin_amdgcn_exp2f(m - all);
        m = all;
        l = sum;
        if (live) {   // few of the tile's rows may be
#pragma unroll
            for (uint32_t d = 0; d < kOuts; ++d) {
                const v4f x = o[d] * f;
                *reinterpret_cast<v4f *>(mo + (wave * kRowTile + lane % 16) * (D + 4) + d * 16 + g * 4) = x;
            }
        }
        __syncthreads();
        // every wave adds a share of the columns of its rows
        constexpr uint32_t kShare = kOuts / L::kGroups;
        if (live) {
#pragma unroll
        for (uint32_t u = 0; u < kShare; ++u) {
            const uint32_t d = wg * kShare + u;
            v4f x = v4f{0, 0, 0, 0};
#pragma unroll
            for (uint32_t k = 0; k < L::kGroups; ++k)
                x += *reinterpret_cast<const v4f *>(mo + ((k * WR + wr) * kRowTile + lane % 16) * (D + 4) + d * 16 + g * 4);
            o[u] = x;
        }
        }
    }
    constexpr uint32_t kOwn = kOuts / L::kGroups;
    const uint32_t d0 = wg * kOwn;
    const float v_scale = KV == Q8MI_KV_E4M3 ? p.cache.v_scale : 1.0f;
    if (live && whole_item) {
        // the cache's scale comes last: it may be so small that its quotient by the sum would be a subnormal
        const float norm = l > 0.0f || l != l ? 1.0f / Op::kWeightScale / l : 0.0f;
        const uint64_t at = static_cast<uint64_t>(q_row) * p.stride_out + head * D + g * 4;
#pragma unroll
        for (uint32_t u = 0; u < kOwn; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) store_out(p, at + (d0 + u) * 16 + i, norm == 0.0f ? 0.0f : o[u][i] * norm * v_scale);
    } else if (live) {
        const uint64_t at = static_cast<uint64_t>(slot_of_piece) * (WR * kRowTile) + wr * kRowTile + lane % 16;
#pragma unroll
        for (uint32_t u = 0; u < kOwn; ++u) *reinterpret_cast<v4f *>(p.part + at * D + (d0 + u) * 16 + g * 4) = o[u];
        if (g == 0 && wg == 0) p.part_ml[at] = make_float2(m, l);
    }
    }
}

// Joins the pieces of one query row and head, in their order: kGroups threads share a column and meet in LDS.
template <uint32_t D, int KV, uint32_t kJoinThreads>
__global__ __launch_bounds__(kJoinThreads) void attention_join_kernel(const AttnParams p) {
    constexpr uint32_t kGroups = kJoinThreads / (D / 4);
    __shared__ float2 sums[kGroups];
    __shared__ uint32_t units[kJoinThreads / kWave][2];
    __shared__ v4f parts[kGroups][D / 4];
    const uint32_t seq = blockIdx.x / p.max_q_len, token = blockIdx.x % p.max_q_len, head = blockIdx.y;
    const uint32_t group = threadIdx.x / (D / 4), d = threadIdx.x % (D / 4);
    const Rows rows = rows_of(p, seq);
    const int64_t q_row = rows.start + token;
    if (token >= rows.used || q_row < 0 || q_row >= p.q_rows) return;
    uint32_t total = 0, before = 0;   // units of all sequences, and of those before this one
    for (uint32_t s = p.n_seqs == 1 ? 1 : threadIdx.x; s < p.n_seqs; s += kJoinThreads) {
        const uint32_t u = units_of_seq(p, p.waves_log2, rows_of(p, s));
        total += u;
        before += s < seq ? u : 0;
    }
    if (p.n_seqs == 1) {
        total = units_of_seq(p, p.waves_log2, rows);
    } else {
        total = wave_sum_u32(total);
        before = wave_sum_u32(before);
        if (threadIdx.x % kWave == 0) { units[threadIdx.x / kWave][0] = total; units[threadIdx.x / kWave][1] = before; }
        __syncthreads();
        total = before = 0;
#pragma unroll
        for (uint32_t i = 0; i < kJoinThreads / kWave; ++i) { total += units[i][0]; before += units[i][1]; }
    }
    const uint32_t share = (total + p.groups - 1) / p.by_groups, kv_head = head / p.by_group;
    const uint32_t tile_log2 = 4 + p.waves_log2, row = token * p.group + head - kv_head * p.group, tile = row >> tile_log2;
    const uint32_t tiles = (rows.used * p.group + (1u << tile_log2) - 1) >> tile_log2, item_units = units_of_item(p.waves_log2, rows);
    const uint32_t begin = before + (kv_head * tiles + tile) * item_units, end = begin + item_units;
    const uint32_t w0 = begin / share, n = (end - 1) / share - w0 + 1;   // the workgroups that share the item
    if (n == 1) return;
    auto place = [&](uint32_t s) -> uint64_t {   // of the row in piece s
        const uint64_t slot = static_cast<uint64_t>(w0 + s) * 2 + (s == 0 && begin > w0 * share ? 1 : 0);
        return (slot << tile_log2) + (row & ((1u << tile_log2) - 1));
    };
    // one pass: a piece's maximum and sum are asked for together with its outputs
    float top = -INFINITY, sum = 0.0f;
    v4f out = v4f{0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t s = group; s < n; s += kGroups) {
        const uint64_t at = place(s);
        const float2 ml = p.part_ml[at];
        const v4f x = *reinterpret_cast<const v4f *>(p.part + at * D + d * 4);
        const float all = fmaxf(top, ml.x);
        const float keep = top == all ? 1.0f : __builtin_amdgcn_exp2f(top - all), f = ml.x == all ? 1.0f : __builtin_amdgcn_exp2f(ml.x - all);
        sum = sum * keep + f * ml.y;
        out = out * keep + f * x;
        top = all;
    }
    if constexpr (kGroups > 1) {
        parts[group][d] = out;
        if (d == 0) sums[group] = make_float2(top, sum);
        __syncthreads();
        if (group != 0) return;
        float all = top;
#pragma unroll
        for (uint32_t i = 1; i < kGroups; ++i) all = fmaxf(all, sums[i].x);
        const float keep = top == all ? 1.0f : __builtin_amdgcn_exp2f(top - all);
        sum *= keep;
        out *= keep;
#pragma unroll
        for (uint32_t i = 1; i < kGroups; ++i) {
            const float f = sums[i].x == all ? 1.0f : __builtin_amdgcn_exp2f(sums[i].x - all);
            sum += f * sums[i].y;
            out += f * parts[i][d];
        }
    }
    constexpr float kNorm = 1.0f / Operand<KV>::kWeightScale;
    const float v_scale = KV == Q8MI_KV_E4M3 ? p.cache.v_scale : 1.0f;   // last, as above
#pragma unroll
    for (int i = 0; i < 4; ++i)
        store_out(p, static_cast<uint64_t>(q_row) * p.stride_out + head * D + d * 4 + i, sum == 0.0f ? 0.0f : out[i] / sum * kNorm * v_scale);
}

constexpr uint32_t kChipCus = 256;
// Where units of fewer tokens still leave CUs idle, waves without rows help to load: a workgroup then takes 32 tokens instead of
// 128 through its one CU's path to memory (4 key heads of 256, 500 tokens: 14.6 -> 13.6 us; with 250 units, 2000 tokens, the
// join of so many pieces takes more than that: 14.8 and 15.8 us).
constexpr uint32_t kFewUnits = 192;
// How a call is cut: waves side by side on rows, and workgroups: as many as a chip of 256 CUs holds at once (one to three a CU,
// by registers and LDS), so that equal runs of the work end together, or one a unit.  Sizes alone decide, for every device.
struct Plan {
    uint32_t waves_on_rows, groups;
};
uint32_t resident_groups(uint32_t head_dim) { return kChipCus * (head_dim == 64 ? 3 : 2); }
uint64_t row_tiles(uint64_t rows, uint32_t waves) { return (rows + kRowTile * waves - 1) / (kRowTile * waves); }
uint64_t token_units(uint32_t max_kv_len, uint32_t waves) {
    const uint64_t unit = kTile * 4 / waves;
    return max_kv_len ? (max_kv_len + unit - 1) / unit : 1;
}
Plan plan_of(uint32_t n_seqs, uint32_t max_q_len, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_kv_len,
             uint64_t *units = nullptr) {
    Plan r;
    const uint32_t rows = max_q_len * (kv_heads ? q_heads / kv_heads : 0);
    r.waves_on_rows = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    auto units_by = [&](uint32_t waves) {
        return n_seqs * static_cast<uint64_t>(kv_heads) * row_tiles(rows, waves) * token_units(max_kv_len, waves);
    };
    if (units_by(4) <= kFewUnits) r.waves_on_rows = 4;
    const uint64_t most = units_by(r.waves_on_rows);
    const uint32_t resident = resident_groups(head_dim);
    r.groups = static_cast<uint32_t>(most < resident ? most : resident);
    if (units) *units = most;
    return r;
}

// Rows of queries and heads from which a wave, and not four, joins the pieces of one: they fill the chip, each has few pieces, and
// four waves would mostly meet (128 x 32 rows: 9.2 -> 5.2 us; below, 24 rows of 128 pieces: 5.4 and not 9.8 us).
constexpr uint32_t kManyJoined = 1024;

// More LDS than the default grant is asked for once per head_dim, cache type and device, for every arrangement of waves: which of
// them a call takes depends on all its sizes, and a later one may be under capture.
template <uint32_t D, int KV, uint32_t WR>
bool grant() {
    constexpr uint32_t kBytes = Layout<D, KV, WR>::kBytes;
    return kBytes <= 64 * 1024 || hipFuncSetAttribute(reinterpret_cast<const void *>(attention_kernel<D, KV, WR>),
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, kBytes) == hipSuccess;
}
template <uint32_t D, int KV>
int grant_lds() {
    static std::atomic<uint64_t> granted{0};   // a bit a device; two threads may both get here first: the grant is idempotent
    int dev = 0;
    if (const hipError_t e = hipGetDevice(&dev); e != hipSuccess) return fail(Q8MI_LAUNCH_ERROR, "paged_attention: %s", hipGetErrorString(e));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;   // devices beyond are asked for every time
    if (granted & bit) return Q8MI_OK;
    if (!grant<D, KV, 1>() || !grant<D, KV, 2>() || !grant<D, KV, 4>()) {
        (void)hipGetLastError();
        return fail(Q8MI_LAUNCH_ERROR, "paged_attention: cannot reserve LDS");
    }
    granted |= bit;
    return Q8MI_OK;
}

template <uint32_t D, int KV, uint32_t WR>
int launch_waves(AttnParams &p, hipStream_t s) {
    using L = Layout<D, KV, WR>;
    p.whole_loads = p.cache.page_size % L::kRowsPerLoad == 0 && static_cast<uint64_t>(L::kRowsPerLoad) * p.unit_token < 1u << 28;
    p.waves_log2 = WR == 1 ? 0 : WR == 2 ? 1 : 2;
    const uint32_t resident = kChipCus * L::kResident;
    if (p.groups > resident) p.groups = resident;
    p.by_groups = divisor(p.groups);
    attention_kernel<D, KV, WR><<<p.groups, kAttnThreads, L::kBytes, s>>>(p);
    if (p.max_kv_len > L::kUnit) {
        const dim3 rows(p.n_seqs * p.max_q_len, p.q_heads);
        if (static_cast<uint64_t>(rows.x) * rows.y >= kManyJoined) attention_join_kernel<D, KV, 64><<<rows, 64, 0, s>>>(p);
        else attention_join_kernel<D, KV, 256><<<rows, 256, 0, s>>>(p);
    }
    return check_launch("paged_attention");
}
template <uint32_t D, int KV>
int launch_dim(AttnParams &p, uint32_t waves_on_rows, hipStream_t s) {
    if (const int rc = grant_lds<D, KV>(); rc != Q8MI_OK) return rc;
    if (waves_on_rows == 1) return launch_waves<D, KV, 1>(p, s);
    if (waves_on_rows == 2) return launch_waves<D, KV, 2>(p, s);
    return launch_waves<D, KV, 4>(p, s);
}
template <int KV>
int launch_type(AttnParams &p, uint32_t waves_on_rows, hipStream_t s) {
    if (p.cache.head_dim == 64) return launch_dim<64, KV>(p, waves_on_rows, s);
    if (p.cache.head_dim == 128) return launch_dim<128, KV>(p, waves_on_rows, s);
    return launch_dim<256, KV>(p, waves_on_rows, s);
}

uint64_t partial_rows(const Plan &plan) { return 2ull * plan.groups * plan.waves_on_rows * kRowTile; }

// No call of these heads with no more sequences, rows and tokens takes more partial rows.  A smaller call may take more than the
// largest one does: up to kFewUnits a workgroup's tile has the rows of four waves, above it, with as few query rows, those of one.
// So every arrangement that a smaller call can get counts, with the most units that it can have.
uint64_t most_partial_rows(uint32_t n_seqs, uint32_t max_q_len, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_kv_len) {
    const uint64_t rows = static_cast<uint64_t>(max_q_len) * (kv_heads ? q_heads / kv_heads : 0);
    const uint64_t resident = resident_groups(head_dim), items = static_cast<uint64_t>(n_seqs) * kv_heads;
    auto partial = [&](uint32_t waves, uint64_t most_rows, uint64_t most_groups) {
        const uint64_t units = items * row_tiles(most_rows < rows ? most_rows : rows, waves) * token_units(max_kv_len, waves);
        return 2 * (units < most_groups ? units : most_groups) * waves * kRowTile;
    };
    uint64_t most = partial(4, rows, rows > 32 ? resident : kFewUnits);
    if (const uint64_t one = partial(1, 16, resident); one > most) most = one;
    if (const uint64_t two = rows > 16 ? partial(2, 32, resident) : 0; two > most) most = two;
    return most;
}

}  // namespace
}  // namespace q8mi

using namespace q8mi;

extern "C" size_t q8mi_paged_attention_scratch_bytes(uint32_t n_seqs, uint32_t max_q_len, uint32_t q_heads, uint32_t kv_heads,
                                                     uint32_t head_dim, uint32_t max_kv_len) {
    return 16 + most_partial_rows(n_seqs, max_q_len, q_heads, kv_heads, head_dim, max_kv_len) * (head_dim + 2) * sizeof(float);
}

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
    if (out == q) return fail(Q8MI_REJECTED, "%s: out is q", what);   // a row's outputs are stored while others still read it
    if (q_heads == 0 || q_heads > 65535 || q_heads % cache->kv_heads != 0)
        return fail(Q8MI_REJECTED, "%s: %u query heads over %u", what, q_heads, cache->kv_heads);
    if (max_q_len == 0 || max_q_len > kMaxRows) return fail(Q8MI_REJECTED, "%s: %u rows a sequence (1..%u)", what, max_q_len, kMaxRows);
    if (max_kv_len > 0x7fffffffu || max_kv_len > static_cast<uint64_t>(stride_page_table) * cache->page_size)
        return fail(Q8MI_REJECTED, "%s: max_kv_len %u is beyond a page table row of %u", what, max_kv_len, stride_page_table);
    const float scale_log2 = scale * 1.44269504088896340736f * (cache->dtype == Q8MI_KV_E4M3 ? cache->k_scale : 1.0f);
    if (!isfinite(scale_log2)) return fail(Q8MI_REJECTED, "%s: scale %g is not finite, or too large", what, static_cast<double>(scale));
    const uint64_t q_es = q_is_bf16 ? 2 : 4, o_es = out_is_bf16 ? 2 : 4, width = static_cast<uint64_t>(q_heads) * cache->head_dim;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(scratch)) % 16 != 0 ||
        stride_q_row * q_es % 16 != 0 || stride_out_row * o_es % 16 != 0)
        return fail(Q8MI_REJECTED, "%s: rows of q and out must begin on 16-byte boundaries", what);
    if (q_rows > 1 && (stride_q_row < width || stride_out_row < width)) return fail(Q8MI_REJECTED, "%s: rows overlap", what);
    if (rows_meet({reinterpret_cast<uintptr_t>(q), q_rows, stride_q_row * q_es, width * q_es},
                  {reinterpret_cast<uintptr_t>(out), q_rows, stride_out_row * o_es, width * o_es}))
        return fail(Q8MI_REJECTED, "%s: out overlaps q", what);

    uint64_t units = 0;
    const Plan plan = plan_of(n_seqs, max_q_len, q_heads, cache->kv_heads, cache->head_dim, max_kv_len, &units);
    if (units > 0x3fffffffull || static_cast<uint64_t>(n_seqs) * max_q_len > 0x3fffffull)
        return fail(Q8MI_REJECTED, "%s: %u sequences of %u tokens are too many for one launch", what, n_seqs, max_kv_len);
    const uint64_t es = kv_element_bytes(cache->dtype);
    const uint64_t unit_page = cache->stride_page * es / 16, unit_token = cache->stride_token * es / 16;
    if (unit_page > 0xffffffffull || unit_token > 0xffffffffull ||
        (cache->pages - 1) * unit_page + (cache->page_size - 1) * unit_token > 0xffffffffull)
        return fail(Q8MI_REJECTED, "%s: a pool of 64 GiB and more", what);
    AttnParams p{};
    p.unit_page = static_cast<uint32_t>(unit_page); p.unit_token = static_cast<uint32_t>(unit_token);
    p.by_page = divisor(cache->page_size);
    p.q = q; p.out = out; p.page_table = page_table; p.kv_lens = kv_lens; p.q_starts = q_starts; p.cache = *cache;
    p.part = static_cast<float *>(scratch);
    p.part_ml = reinterpret_cast<float2 *>(p.part + partial_rows(plan) * cache->head_dim);
    p.q_rows = q_rows; p.stride_q = stride_q_row; p.stride_out = stride_out_row; p.stride_page_table = stride_page_table;
    p.n_seqs = n_seqs; p.max_q_len = max_q_len; p.q_heads = q_heads; p.group = q_heads / cache->kv_heads;
    p.by_group = divisor(p.group);
    p.max_kv_len = max_kv_len; p.groups = plan.groups;
    p.scale_log2 = scale_log2;
    p.q_is_bf16 = q_is_bf16; p.out_is_bf16 = out_is_bf16;
    hipStream_t s = as_stream(stream);
    if (cache->dtype == Q8MI_KV_BF16) return launch_type<Q8MI_KV_BF16>(p, plan.waves_on_rows, s);
    if (cache->dtype == Q8MI_KV_F16) return launch_type<Q8MI_KV_F16>(p, plan.waves_on_rows, s);
    return launch_type<Q8MI_KV_E4M3>(p, plan.waves_on_rows, s);
}
