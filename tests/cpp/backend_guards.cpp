// What HipQ8Backend answers to handles of the wrong kind and to caches that no operator would take.
//   frequencies  64-bit rotation frequencies are no norm weight, and 32-bit ones no frequencies
//   caches       what the cache operators would refuse is not made, nor a pool whose size leaves 64 bits
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

}  // namespace

int main() {
    {
        qw3::HipQ8Backend b;
        frequencies(b);
        caches(b);
    }
    std::printf("%d failed\n", g_failed);
    std::fflush(stdout);
    _exit(g_failed ? 1 : 0);
}
