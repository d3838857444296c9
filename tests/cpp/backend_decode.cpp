// A decode loop through HipQ8Backend's operators, the way an executor drives them: a prompt of five tokens in one pass (rows
// of one sequence, as in verification), then single tokens chained on the device -- embedding row of the sampled token, norm,
// Q/K/V projections, head norms + rotation + cache append, attention over the paged cache, O, FFN, logits, sampling.
//   attention  every attention output against a CPU double computation from the projections the device made
//   tokens     every sampled token against a CPU sampler on the device's logits
//   graph      the same loop with the step captured once and replayed: the same tokens, also after larger calls have outgrown the
//              scratch that the graph names
//   refusals   what the operators answer to tensors that are too small or of another type
// Prints one line per case; exit code 0 only if all pass.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <numeric>
#include <string>
#include <vector>

#include <unistd.h>

#include "../../kvmem-qw3_amd/host/hip_q8_backend.hpp"
#include "../../oracle/q8_oracle.h"

namespace {

int g_failed = 0;

void report(const char *name, bool ok, const std::string &detail = "") {
    if (!ok) ++g_failed;
    std::printf("%s %s%s%s\n", ok ? "PASS" : "FAIL", name, detail.empty() ? "" : ": ", detail.c_str());
    std::fflush(stdout);
}

struct Rng {   // splitmix64
    uint64_t s;
    uint64_t next() {
        uint64_t z = (s += 0x9E3779B97F4A7C15ull);
        z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
        z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
        return z ^ (z >> 31);
    }
    float uniform() { return static_cast<float>(next() >> 40) * (1.0f / 16777216.0f); }
    float normal() { return std::sqrt(-2.0f * std::log(uniform() + 1e-7f)) * std::cos(6.2831853f * uniform()); }
};

constexpr uint32_t kHidden = 256, kHeads = 6, kKvHeads = 2, kDim = 64, kFfn = 512, kVocab = 3000, kRot = 32, kPage = 8, kPages = 12;
constexpr uint32_t kQ = kHeads * kDim, kKv = kKvHeads * kDim, kPrompt = 5, kSteps = 14, kMaxKv = 64, kWide = kMaxKv / kPage;
constexpr float kEps = 1e-6f;

struct Model {
    qw3::HipQ8Backend backend;
    std::unique_ptr<qw3::DeviceWeight> embed, wq, wk, wv, wo, gate, up, down, head, norm_w, qn, kn, freqs;
    std::vector<float> qn_host, kn_host;
    std::vector<double> freqs_host;

    std::unique_ptr<qw3::DeviceWeight> q8(uint32_t rows, uint32_t cols, uint64_t seed, float scale) {
        Rng r{seed};
        std::vector<float> v(static_cast<size_t>(rows) * cols);
        for (auto &f : v) f = r.normal() * scale;
        std::vector<uint8_t> g(static_cast<size_t>(rows) * (cols / 32) * 34);
        q8o_quantize_q8_0(v.data(), rows, cols, g.data());
        return backend.weight_q8_0(g.data(), rows, cols, "w");
    }
    std::unique_ptr<qw3::DeviceWeight> ones(uint32_t n, uint64_t seed, std::vector<float> *host = nullptr) {
        Rng r{seed};
        std::vector<float> v(n);
        for (auto &f : v) f = 1.0f + 0.1f * r.normal();
        if (host) *host = v;
        return backend.weight_f32(v.data(), n, "norm");
    }
    Model() {
        embed = q8(kVocab, kHidden, 1, 1.0f);
        wq = q8(kQ, kHidden, 2, 0.08f); wk = q8(kKv, kHidden, 3, 0.08f); wv = q8(kKv, kHidden, 4, 0.08f);
        wo = q8(kHidden, kQ, 5, 0.05f);
        gate = q8(kFfn, kHidden, 6, 0.06f); up = q8(kFfn, kHidden, 7, 0.06f); down = q8(kHidden, kFfn, 8, 0.05f);
        head = q8(kVocab, kHidden, 9, 0.15f);
        norm_w = ones(kHidden, 10); qn = ones(kDim, 11, &qn_host); kn = ones(kDim, 12, &kn_host);
        for (uint32_t i = 0; i < kRot / 2; ++i) freqs_host.push_back(std::pow(1e4, -double(i) / (kRot / 2)));
        freqs = backend.rope_frequencies(freqs_host.data(), freqs_host.size(), "freqs");
    }
};

struct Run {
    Model &m;
    qw3::HipQ8Backend &b;
    std::unique_ptr<qw3::DeviceKvCache> cache;
    std::unique_ptr<qw3::DeviceTensor> h, norm, q, k, v, qr, attn, mid, tmp, logits, pos, slots, table, lens, temp, top_k, top_p, min_p, u;
    std::unique_ptr<qw3::DeviceArgmaxBuffer> tok;
    std::vector<int32_t> table_host;
    std::string error;

    explicit Run(Model &model) : m(model), b(model.backend) {
        cache = b.kv_cache(qw3::DeviceTensorDType::F16, kPages, kPage, kKvHeads, kDim, 1.0f, 1.0f, "kv");
        auto f = [&](uint64_t n) { return b.tensor_f32(n, "t"); };
        h = f(kPrompt * kHidden); norm = f(kPrompt * kHidden); q = f(kPrompt * kQ); k = f(kPrompt * kKv); v = f(kPrompt * kKv);
        qr = f(kPrompt * kQ); attn = f(kPrompt * kQ); mid = f(kPrompt * kFfn); tmp = f(kPrompt * kHidden); logits = f(kVocab);
        pos = b.tensor_i32(kPrompt, "pos"); slots = b.tensor_i64(kPrompt, "slots");
        table = b.tensor_i32(kWide, "table"); lens = b.tensor_i32(1, "lens");
        temp = f(1); top_p = f(1); min_p = f(1); u = f(1); top_k = b.tensor_i32(1, "k");
        tok = b.argmax_buffer(1);
        for (uint32_t i = 0; i < kWide; ++i) table_host.push_back((i * 5 + 3) % kPages);   // pages in no order
        put(*table, table_host);
        put(*temp, std::vector<float>{0.8f}); put(*top_k, std::vector<int32_t>{40}); put(*top_p, std::vector<float>{0.95f});
        put(*min_p, std::vector<float>{0.01f});
    }
    bool ok(const qw3::DeviceStatus &st, const char *what) {
        if (!st.ok && error.empty()) error = std::string(what) + ": " + st.message;
        return st.ok;
    }
    template <typename V> void put(qw3::DeviceTensor &t, const V &x) { ok(b.copy_bytes_from_host(t, 0, x.data(), x.size() * sizeof(x[0])), "upload"); }
    std::vector<float> get(const qw3::DeviceTensor &t, uint64_t n) {
        std::vector<float> x(n);
        ok(b.copy_to_host(t, x.data(), 0, n), "download");
        return x;
    }
    void place(uint32_t first, uint32_t n) {   // tokens first .. first + n - 1: positions, slots, length
        std::vector<int32_t> p(n);
        std::vector<int64_t> s(n);
        for (uint32_t i = 0; i < n; ++i) {
            p[i] = static_cast<int32_t>(first + i);
            s[i] = static_cast<int64_t>(table_host[(first + i) / kPage]) * kPage + (first + i) % kPage;
        }
        put(*pos, p); put(*slots, s); put(*lens, std::vector<int32_t>{static_cast<int32_t>(first + n)});
    }
    // the layer on n rows of h, logits of the last row, a token
    bool layer(uint32_t n) {
        qw3::DeviceTensor *outs[3] = {q.get(), k.get(), v.get()};
        const qw3::DeviceWeight *ws[3] = {m.wq.get(), m.wk.get(), m.wv.get()};
        const uint32_t strides[3] = {kQ, kKv, kKv};
        bool good = ok(b.rms_norm_batch(*norm, *h, *m.norm_w, n, kHidden, kEps), "norm") &&
                    ok(b.q8_0_matmul_fanout(outs, ws, strides, 3, *norm, n, kHidden), "qkv") &&
                    ok(b.qk_norm_rope_append(*qr, *q, *k, *v, m.qn.get(), m.kn.get(), kEps, m.freqs.get(), kRot, false, *pos, *slots, n,
                                             kHeads, kQ, kDim, kKv, kKv, kQ, *cache), "append") &&
                    ok(b.paged_attention(*attn, *qr, *cache, *table, kWide, *lens, nullptr, 1, n, n, kHeads, kMaxKv,
                                         1.0f / std::sqrt(float(kDim)), kQ, kQ), "attention") &&
                    ok(b.q8_0_matmul_add(*h, *h, *tmp, *m.wo, *attn, n, kQ, kHidden), "o") &&
                    ok(b.rms_norm_batch(*norm, *h, *m.norm_w, n, kHidden, kEps), "norm") &&
                    ok(b.q8_0_matmul_silu_mul(*mid, *m.gate, *m.up, *norm, n, kHidden, kFfn), "ffn") &&
                    ok(b.q8_0_matmul_add(*h, *h, *tmp, *m.down, *mid, n, kFfn, kHidden), "down") &&
                    ok(b.rms_norm_batch(*norm, *h, *m.norm_w, n, kHidden, kEps), "norm");
        return good;
    }
    bool sample() {   // from the first row of norm
        return ok(b.q8_0_matmul(*logits, *m.head, *norm, 1, kHidden, kVocab), "head") &&
               ok(b.sample_rows(*logits, 1, kVocab, kVocab, temp.get(), top_k.get(), top_p.get(), min_p.get(), *u, *tok), "sample");
    }
    bool step() { return ok(b.q8_0_get_row_from_argmax(*h, *m.embed, *tok, 0), "embed") && layer(1) && sample(); }
    int32_t token() {
        qw3::DeviceArgmax t;
        ok(b.copy_argmax_buffer_to_host(*tok, &t, 1), "token");
        return t.token;
    }
    bool prompt(float uniform) {
        const uint64_t ids[kPrompt] = {17, 2999, 5, 5, 1234};
        place(0, kPrompt);
        put(*u, std::vector<float>{uniform});
        if (!ok(b.q8_0_get_rows_batch(*h, *m.embed, ids, kPrompt), "embed") || !layer(kPrompt)) return false;
        // the last row's norm to the front, where the head reads it
        auto rows = get(*norm, kPrompt * kHidden);
        rows.erase(rows.begin(), rows.begin() + (kPrompt - 1) * kHidden);
        put(*norm, rows);
        return sample();
    }
};

// CPU doubles: what the cache and the attention hold, from the projections that the device made.
struct Check {
    const Model &m;
    std::vector<std::vector<double>> keys, values;   // per token [kv_heads * dim]
    static double half(double x) { return static_cast<double>(static_cast<_Float16>(static_cast<float>(x))); }
    std::vector<double> head(const float *x, const std::vector<float> &w, uint32_t position) const {
        double s = 0.0;
        for (uint32_t i = 0; i < kDim; ++i) s += double(x[i]) * x[i];
        std::vector<double> y(kDim);
        for (uint32_t i = 0; i < kDim; ++i) y[i] = x[i] / std::sqrt(s / kDim + kEps) * w[i];
        for (uint32_t i = 0; i < kRot / 2; ++i) {
            const double a = y[i], c = y[i + kRot / 2], t = position * m.freqs_host[i];
            y[i] = a * std::cos(t) - c * std::sin(t);
            y[i + kRot / 2] = c * std::cos(t) + a * std::sin(t);
        }
        return y;
    }
    void append(const std::vector<float> &k, const std::vector<float> &v, uint32_t n) {
        for (uint32_t t = 0; t < n; ++t) {
            std::vector<double> kr, vr;
            for (uint32_t h = 0; h < kKvHeads; ++h) {
                for (double x : head(&k[t * kKv + h * kDim], m.kn_host, static_cast<uint32_t>(keys.size()))) kr.push_back(half(x));
                for (uint32_t i = 0; i < kDim; ++i) vr.push_back(half(v[t * kKv + h * kDim + i]));
            }
            keys.push_back(kr);
            values.push_back(vr);
        }
    }
    // largest error of the device's attention outputs of the newest n tokens, relative to the values' size
    double worst(const std::vector<float> &q, const std::vector<float> &out, uint32_t n) const {
        double bad = 0.0;
        for (uint32_t t = 0; t < n; ++t) {
            const uint32_t seen = static_cast<uint32_t>(keys.size()) - n + t + 1;
            for (uint32_t h = 0; h < kHeads; ++h) {
                const auto qr = head(&q[t * kQ + h * kDim], m.qn_host, seen - 1);
                const uint32_t kv = h / (kHeads / kKvHeads) * kDim;
                std::vector<double> s(seen);
                for (uint32_t j = 0; j < seen; ++j) {
                    for (uint32_t i = 0; i < kDim; ++i) s[j] += qr[i] * keys[j][kv + i];
                    s[j] = s[j] / std::sqrt(double(kDim));
                }
                const double top = *std::max_element(s.begin(), s.end());
                double sum = 0.0;
                for (auto &x : s) sum += x = std::exp(x - top);
                for (uint32_t i = 0; i < kDim; ++i) {
                    double o = 0.0;
                    for (uint32_t j = 0; j < seen; ++j) o += s[j] / sum * values[j][kv + i];
                    bad = std::max(bad, std::fabs(o - out[t * kQ + h * kDim + i]));
                }
            }
        }
        return bad;
    }
};

int32_t cpu_sample(const std::vector<float> &z, double t, uint32_t k, double top_p, double min_p, double u) {
    std::vector<uint32_t> order(z.size());
    std::iota(order.begin(), order.end(), 0u);
    std::stable_sort(order.begin(), order.end(), [&](uint32_t a, uint32_t b) { return z[a] > z[b]; });
    std::vector<double> p;
    for (uint32_t i = 0; i < k; ++i) p.push_back(std::exp((double(z[order[i]]) - z[order[0]]) / t));
    const double total = std::accumulate(p.begin(), p.end(), 0.0);
    uint32_t kept = 0;
    for (double before = 0.0; kept < k && (kept == 0 || before < top_p * total) && p[kept] >= min_p; ++kept) before += p[kept];
    std::vector<uint32_t> ids(kept);
    std::iota(ids.begin(), ids.end(), 0u);
    std::sort(ids.begin(), ids.end(), [&](uint32_t a, uint32_t b) { return order[a] < order[b]; });
    double all = 0.0, run = 0.0;
    for (uint32_t i : ids) all += p[i];
    for (uint32_t i : ids)
        if ((run += p[i]) > u * all) return static_cast<int32_t>(order[i]);
    return -2;
}

}  // namespace

int main(int argc, char **argv) {
    (void)argc; (void)argv;
    Model m;
    std::vector<float> us;
    Rng r{99};
    for (uint32_t i = 0; i <= kSteps; ++i) us.push_back(r.uniform());
    std::vector<int32_t> eager;
    {
        Run run(m);
        Check c{m, {}, {}};
        double worst = 0.0;
        bool good = run.prompt(us[0]), tokens = true;
        auto look = [&](uint32_t n, float u) {
            c.append(run.get(*run.k, n * kKv), run.get(*run.v, n * kKv), n);
            worst = std::max(worst, c.worst(run.get(*run.q, n * kQ), run.get(*run.attn, n * kQ), n));
            eager.push_back(run.token());
            const int32_t want = cpu_sample(run.get(*run.logits, kVocab), 0.8f, 40, 0.95f, 0.01f, u);
            if (want != eager.back()) { tokens = false; std::printf("  token %zu: got %d want %d\n", eager.size(), eager.back(), want); }
        };
        if (good) look(kPrompt, us[0]);
        for (uint32_t i = 0; good && i < kSteps; ++i) {
            run.place(kPrompt + i, 1);
            run.put(*run.u, std::vector<float>{us[i + 1]});
            good = run.step();
            if (good) look(1, us[i + 1]);
        }
        // a value near the middle of two fp16 numbers may be rounded to the other one on the device: a step is at most
        // 2^-8 = 3.9e-3 below 8, six standard deviations of what wv makes
        report("attention", good && worst < 4e-3, run.error.empty() ? "largest error " + std::to_string(worst) : run.error);
        report("tokens", good && tokens, run.error);
    }
    {
        Run run(m);
        std::vector<int32_t> got;
        bool good = run.prompt(us[0]);
        if (good) got.push_back(run.token());
        for (uint32_t i = 0; good && i < kSteps; ++i) {
            run.place(kPrompt + i, 1);
            run.put(*run.u, std::vector<float>{us[i + 1]});
            if (i == 0) {
                good = run.step();              // eager: every scratch has its size, every kernel its grants
            } else if (i == 1) {
                good = run.b.begin_capture() && run.step() && run.ok(run.b.end_capture(), "end capture") &&
                       run.ok(run.b.replay_graph(), "replay");
            } else {
                good = run.ok(run.b.replay_graph(), "replay");
            }
            if (good) got.push_back(run.token());
            if (good && i == 4) {   // larger calls: their scratch takes the place of the one that the graph names
                auto many = m.backend.tensor_f32(9 * kVocab, "logits"), us9 = m.backend.tensor_f32(9, "u");
                auto toks = m.backend.argmax_buffer(9);
                auto lens = m.backend.tensor_i32(40, "lens"), pages = m.backend.tensor_i32(40 * kWide, "pages");
                auto rows = m.backend.tensor_f32(40 * kQ, "q"), out = m.backend.tensor_f32(40 * kQ, "out");
                run.put(*many, std::vector<float>(9 * kVocab, 0.5f));
                run.put(*us9, std::vector<float>(9, 0.5f));
                run.put(*lens, std::vector<int32_t>(40, 9));
                run.put(*pages, std::vector<int32_t>(40 * kWide, 1));
                run.put(*rows, std::vector<float>(40 * kQ, 1.0f));
                good = run.ok(m.backend.sample_rows(*many, 9, kVocab, kVocab, nullptr, nullptr, nullptr, nullptr, *us9, *toks), "large sample") &&
                       run.ok(m.backend.paged_attention(*out, *rows, *run.cache, *pages, kWide, *lens, nullptr, 40, 40, 1, kHeads, kMaxKv, 0.1f, kQ, kQ),
                              "large attention") &&
                       run.ok(m.backend.synchronize(), "synchronize");
            }
        }
        report("graph", good && got == eager, run.error);
    }
    {
        Run run(m);
        auto refused = [&](const qw3::DeviceStatus &st) { return !st.ok && st.message && *st.message; };
        auto half = m.backend.tensor_bf16(kPrompt * kQ, "bf16");
        auto append = [&](const qw3::DeviceTensor &q, const qw3::DeviceTensor &k, const qw3::DeviceWeight *n, const qw3::DeviceWeight *f,
                          uint32_t rot, const qw3::DeviceTensor &slots, uint32_t tokens) {
            return m.backend.qk_norm_rope_append(*run.qr, q, k, *run.v, n, m.kn.get(), kEps, f, rot, false, *run.pos, slots, tokens, kHeads,
                                                 kQ, kDim, kKv, kKv, kQ, *run.cache);
        };
        auto attend = [&](const qw3::DeviceTensor &q, const qw3::DeviceTensor &table, const qw3::DeviceTensor &lens, uint32_t rows, uint32_t max_kv) {
            return m.backend.paged_attention(*run.attn, q, *run.cache, table, kWide, lens, nullptr, 1, rows, 1, kHeads, max_kv, 1.0f, kQ, kQ);
        };
        auto sample = [&](const qw3::DeviceTensor &x, uint32_t batch, const qw3::DeviceTensor *k) {
            return m.backend.sample_rows(x, batch, kVocab, kVocab, run.temp.get(), k, nullptr, nullptr, *run.u, *run.tok);
        };
        auto &q = *run.q, &k = *run.k;
        const bool good =
            refused(append(*half, k, nullptr, m.freqs.get(), kRot, *run.slots, 1)) && refused(append(q, *run.u, nullptr, m.freqs.get(), kRot, *run.slots, 1)) &&
            refused(append(q, k, m.freqs.get(), m.freqs.get(), kRot, *run.slots, 1)) && refused(append(q, k, nullptr, m.qn.get(), kRot, *run.slots, 1)) &&
            refused(append(q, k, nullptr, m.freqs.get(), 2 * kRot, *run.slots, 1)) && refused(append(q, k, nullptr, m.freqs.get(), kRot, *run.pos, 1)) &&
            refused(append(q, k, nullptr, m.freqs.get(), kRot, *run.slots, kPrompt + 1)) && refused(append(q, k, nullptr, m.freqs.get(), kRot - 4, *run.slots, 1)) &&
            refused(attend(*run.u, *run.table, *run.lens, 1, kMaxKv)) && refused(attend(q, *run.lens, *run.lens, 1, kMaxKv)) &&
            refused(attend(q, *run.table, *run.u, 1, kMaxKv)) && refused(attend(q, *run.table, *run.lens, kPrompt + 1, kMaxKv)) &&
            refused(attend(q, *run.table, *run.lens, 1, kMaxKv + 1)) && refused(sample(*run.u, 1, nullptr)) && refused(sample(*half, 1, nullptr)) &&
            refused(sample(*run.logits, 2, nullptr)) && refused(sample(*run.logits, 1, run.u.get())) &&
            !m.backend.kv_cache(qw3::DeviceTensorDType::F32, 4, 8, 2, 64, 1.0f, 1.0f, "x") &&
            !m.backend.kv_cache(qw3::DeviceTensorDType::F16, 4, 8, 2, 96, 1.0f, 1.0f, "x");
        report("refusals", good);
    }
    std::printf("%d failed\n", g_failed);
    std::fflush(stdout);
    _exit(g_failed ? 1 : 0);
}
