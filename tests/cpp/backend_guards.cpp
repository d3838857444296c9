// What HipQ8Backend answers to handles of the wrong kind and to caches that no operator would take, and what one eager call with a
// program's largest bounds prepares.
//   frequencies  64-bit rotation frequencies are no norm weight, and 32-bit ones no frequencies
//   caches       what the cache operators would refuse is not made, nor a pool whose size leaves 64 bits
//   captured     after the largest attention and sampling have run once, smaller ones are captured without growing a scratch, and
//                replays give the eager calls' bits
// Prints one line per case; exit code 0 only if all pass.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <vector>

#include <unistd.h>

#include "../../kvmem-qw3_amd/host/hip_q8_backend.hpp"

namespace {

int g_failed = 0;

void report(const char *name, bool ok) {
    if (!ok) ++g_failed;
    std::printf("%s %s\n", ok ? "PASS" : "FAIL", name);
    std::fflush(stdout);
}
bool refused(const qw3::DeviceStatus &st) { return !st.ok && st.message && *st.message; }

void frequencies(qw3::HipQ8Backend &b) {
    constexpr uint32_t n = 64;
    auto x = b.tensor_f32(9 * n, "x"), y = b.tensor_f32(9 * n, "y"), z = b.tensor_f32(9 * n, "z");
    auto freqs = b.rope_frequencies(std::vector<double>(n, 1.0).data(), n, "freqs");
    auto norm = b.weight_f32(std::vector<float>(n, 1.0f).data(), n, "norm");
    auto w = b.weight_q8_0(std::vector<uint8_t>(n * (n / 32) * 34, 0).data(), n, n, "w");
    qw3::DeviceTensor *outs[1] = {z.get()};
    const qw3::DeviceWeight *ws[1] = {w.get()};
    const uint32_t strides[1] = {n};
    bool ok = b.copy_bytes_from_host(*x, 0, std::vector<float>(9 * n, 1.0f).data(), 9 * n * 4).ok;
    for (uint32_t batch : {1u, 4u, 9u}) {
        ok = ok && refused(b.rms_norm_batch(*y, *x, *freqs, batch, n, 1e-6f)) &&
             refused(b.rms_norm_q8_0_matmul_fanout(*y, outs, ws, strides, 1, *x, *freqs, batch, n, 1e-6f));
        ok = ok && b.rms_norm_batch(*y, *x, *norm, batch, n, 1e-6f).ok &&
             b.rms_norm_q8_0_matmul_fanout(*y, outs, ws, strides, 1, *x, *norm, batch, n, 1e-6f).ok;
    }
    auto one = b.tensor_f32(n, "one row");
    ok = ok && b.copy_bytes_from_host(*one, 0, std::vector<float>(n, 1.0f).data(), n * 4).ok && refused(b.rms_norm(*y, *one, *freqs, 1e-6f)) &&
         b.rms_norm(*y, *one, *norm, 1e-6f).ok && b.synchronize().ok;
    report("frequencies", ok);
}

void caches(qw3::HipQ8Backend &b) {
    using D = qw3::DeviceTensorDType;
    auto made = [&](D t, uint32_t pages, uint32_t page_size, uint32_t heads, uint32_t dim, float ks = 1.0f, float vs = 1.0f) {
        return b.kv_cache(t, pages, page_size, heads, dim, ks, vs, "kv") != nullptr;
    };
    const float nan = std::nanf(""), inf = INFINITY;
    bool ok = made(D::BF16, 1, 65536, 1, 64) && !made(D::BF16, 1, 65537, 1, 64) && !made(D::BF16, 0, 16, 1, 64) && !made(D::BF16, 1, 0, 1, 64) &&
              !made(D::BF16, 1, 16, 0, 64);
    for (float bad : {0.0f, -1.0f, nan, inf})
        ok = ok && !made(D::FP8_E4M3, 2, 16, 1, 64, bad, 1.0f) && !made(D::FP8_E4M3, 2, 16, 1, 64, 1.0f, bad) && made(D::F16, 2, 16, 1, 64, bad, bad);
    ok = ok && made(D::FP8_E4M3, 2, 16, 1, 64, 1e-30f, 1e30f);
    // 2^64 bytes and a little more: their low bits alone are a pool of moderate size
    ok = ok && !made(D::F16, 1u << 30, 65536, 1u << 9, 256) && !made(D::FP8_E4M3, 1u << 31, 65536, 1u << 9, 256) &&
         !made(D::F16, 1u << 30, 65536, (1u << 9) + (1u << 11), 256) && !made(D::BF16, 0x80000001u, 65536, 1u << 16, 64);
    report("caches", ok && b.synchronize().ok);
}

void captured(qw3::HipQ8Backend &b) {
    constexpr uint32_t heads = 24, kv_heads = 4, dim = 256, seqs = 3, wide = 1250, page = 16, width = heads * dim, rows = 32, vocab = 32000;
    auto cache = b.kv_cache(qw3::DeviceTensorDType::F16, 4, page, kv_heads, dim, 1.0f, 1.0f, "kv");
    auto q = b.tensor_f32(seqs * width, "q"), out = b.tensor_f32(seqs * width, "out"), logits = b.tensor_f32(rows * vocab, "logits"),
         u = b.tensor_f32(rows, "u"), top_p = b.tensor_f32(rows, "top_p"), k = b.tensor_f32(40 * kv_heads * dim, "k"),
         v = b.tensor_f32(40 * kv_heads * dim, "v"), unused = b.tensor_f32(40 * width, "q_out"), queries = b.tensor_f32(40 * width, "queries");
    auto table = b.tensor_i32(seqs * wide, "table"), lens = b.tensor_i32(seqs, "lens"), positions = b.tensor_i32(40, "positions");
    auto slots = b.tensor_i64(40, "slots");
    auto tokens = b.argmax_buffer(rows);
    bool ok = true;
    auto put = [&](qw3::DeviceTensor &t, const auto &x) { ok = ok && b.copy_bytes_from_host(t, 0, x.data(), x.size() * sizeof(x[0])).ok; };
    auto noise = [](size_t n, uint32_t seed) {
        std::vector<float> x(n);
        for (auto &f : x) f = static_cast<float>((seed = seed * 1664525u + 1013904223u) >> 8) / 8388608.0f - 1.0f;
        return x;
    };
    std::vector<int32_t> pages(seqs * wide, 0), at(40);
    std::vector<int64_t> slot(40);
    for (uint32_t i = 0; i < 40; ++i) { at[i] = static_cast<int32_t>(i); slot[i] = i; }
    for (uint32_t s = 0; s < seqs; ++s)
        for (uint32_t i = 0; i < 3; ++i) pages[s * wide + i] = static_cast<int32_t>(i);
    put(*table, pages); put(*lens, std::vector<int32_t>{40, 17, 33}); put(*positions, at); put(*slots, slot);
    put(*q, noise(seqs * width, 1)); put(*k, noise(40 * kv_heads * dim, 2)); put(*v, noise(40 * kv_heads * dim, 3));
    put(*queries, noise(40 * width, 4)); put(*logits, noise(rows * vocab, 5)); put(*u, std::vector<float>(rows, 0.4f));
    put(*top_p, std::vector<float>(rows, 0.9f));
    ok = ok && b.qk_norm_rope_append(*unused, *queries, *k, *v, nullptr, nullptr, 1e-6f, nullptr, 0, false, *positions, *slots, 40, heads, width, dim,
                                     kv_heads * dim, kv_heads * dim, width, *cache).ok;
    auto attend = [&](uint32_t n, uint32_t max_kv) {
        const auto st = b.paged_attention(*out, *q, *cache, *table, wide, *lens, nullptr, n, n, 1, heads, max_kv, 0.0625f, width, width);
        if (!st.ok) std::printf("  attention of %u, %u: %s\n", n, max_kv, st.message);
        return st.ok;
    };
    auto sample = [&](uint32_t n) {
        const auto st = b.sample_rows(*logits, n, vocab, vocab, nullptr, nullptr, top_p.get(), nullptr, *u, *tokens);
        if (!st.ok) std::printf("  sampling of %u: %s\n", n, st.message);
        return st.ok;
    };
    auto outputs = [&](uint32_t n) {
        std::vector<float> x(n * width);
        ok = ok && b.copy_to_host(*out, x.data(), 0, x.size()).ok;
        return x;
    };
    auto drawn = [&](uint32_t n) {
        std::vector<qw3::DeviceArgmax> x(n);
        std::vector<int> t;
        ok = ok && b.copy_argmax_buffer_to_host(*tokens, x.data(), n).ok;
        for (auto &a : x) t.push_back(a.token);
        return t;
    };
    ok = ok && attend(seqs, wide * page) && sample(rows);   // the largest, once
    const uint32_t n_seqs[] = {1, 2, 3, 1, 3}, max_kv[] = {1536, 700, 700, 64, 20000}, batch[] = {31, 16, 1, 20, 32};
    for (int i = 0; ok && i < 5; ++i) {
        ok = b.begin_capture();
        if (!ok) break;
        const bool served = attend(n_seqs[i], max_kv[i]) && sample(batch[i]);
        ok = b.end_capture().ok && served;
        ok = ok && attend(n_seqs[i], max_kv[i]) && sample(batch[i]);
        const auto want = outputs(n_seqs[i]);
        const auto want_tokens = drawn(batch[i]);
        for (int replay = 0; ok && replay < 3; ++replay) {
            ok = b.zero_tensor(*out).ok && b.replay_graph().ok;
            ok = ok && outputs(n_seqs[i]) == want && drawn(batch[i]) == want_tokens;
        }
        for (float f : want) ok = ok && std::isfinite(f);
    }
    report("captured", ok);
}

}  // namespace

int main() {
    {
        qw3::HipQ8Backend b;
        frequencies(b);
        caches(b);
        captured(b);
    }
    std::printf("%d failed\n", g_failed);
    std::fflush(stdout);
    _exit(g_failed ? 1 : 0);
}
