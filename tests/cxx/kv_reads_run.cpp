// The 4-bit cache's and the page selection's calls of include/reef_hip/attention.hpp on a device,
// each against its formula on the host. Prints each step before it runs.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <stdexcept>
#include <type_traits>
#include <vector>

#include "reef_hip/attention.hpp"

static int failures = 0;

static void need(hipError_t e) {
    if (e != hipSuccess) throw std::runtime_error(hipGetErrorString(e));
}

template <typename T>
struct Device {
    T *p = nullptr;
    size_t n;
    explicit Device(const std::vector<T> &v) : n(v.size()) {
        need(hipMalloc(reinterpret_cast<void **>(&p), n * sizeof(T)));
        need(hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice));
    }
    Device(const Device &) = delete;
    ~Device() { (void)hipFree(p); }
    std::vector<T> host() const {
        std::vector<T> v(n);
        need(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
        return v;
    }
};

static void step(const char *name) {
    std::printf("[step] %s\n", name);
    std::fflush(stdout);
}

static void check(const char *name, bool ok) {
    std::printf("%s %s\n", ok ? "ok  " : "FAIL", name);
    failures += !ok;
}

static std::vector<float> uniform(size_t n, uint32_t seed) {
    std::vector<float> v(n);
    for (auto &x : v) {
        seed = seed * 1664525u + 1013904223u;
        x = (float)(seed >> 8) * 0x1p-23f - 1.0f;
    }
    return v;
}

// One sequence of T tokens in pages {3, 1, 4}, two query heads of one key head.
static const int64_t T = 40, D = 64, P = 6, G = 2, blocks = 3;
static const std::vector<int32_t> table{3, 1, 4};

// Attention of codes q (scale qs[head]) over the rows of some tokens, in 64 bits.
static double attention(const std::vector<float> &k, const std::vector<float> &v, const int8_t *q, float qs,
                        const std::vector<int64_t> &tokens, int64_t channel) {
    double sum = 0, out = 0, top = -1e300;
    std::vector<double> s;
    for (int64_t t : tokens) {
        double x = 0;
        for (int64_t d = 0; d < D; ++d) x += (double)q[d] * k[t * D + d];
        s.push_back(x * qs / 8);
        top = std::max(top, s.back());
    }
    for (size_t i = 0; i < s.size(); ++i) {
        const double p = std::exp(s[i] - top);
        sum += p;
        out += p * v[tokens[i] * D + channel];
    }
    return out / sum;
}

// Rows as the cache holds them: quantized with `most` steps, times their scale.
static std::vector<float> held(const std::vector<float> &x, float most) {
    std::vector<float> y(x.size());
    for (int64_t t = 0; t < T; ++t) {
        float top = 0;
        for (int64_t d = 0; d < D; ++d) top = std::max(top, std::fabs(x[t * D + d]));
        volatile float scale = top / most;
        for (int64_t d = 0; d < D; ++d) y[t * D + d] = std::nearbyint(x[t * D + d] / scale) * scale;
    }
    return y;
}

template <typename Code>
static void run(const std::vector<float> &k, const std::vector<float> &v) {
    const bool int4 = std::is_same<Code, uint8_t>::value;
    const int64_t row = int4 ? D / 2 : D;
    const auto hk = held(k, int4 ? 7.0f : 127.0f), hv = held(v, int4 ? 7.0f : 127.0f);
    Device<float> dk(k), dv(v), ks(std::vector<float>(P * 16)), vs(std::vector<float>(P * 16));
    Device<Code> kc(std::vector<Code>(P * 16 * row)), vc(std::vector<Code>(P * 16 * row));
    Device<int32_t> dt(table), start({0}), lens({0});
    Device<uint32_t> status({0});
    const reef_kv_append_params rows{1, 1, D, T, blocks * 16};
    step(int4 ? "append, 4 bits" : "append, 8 bits");
    if constexpr (std::is_same<Code, uint8_t>::value) {
        reef_hip::append_kv_cache_int4(rows, dk.p, nullptr, dv.p, nullptr, start.p, dt.p, blocks, P, kc.p,
                                       vc.p, ks.p, vs.p, lens.p, status.p, nullptr);
        Device<float> fk(std::vector<float>(P * 16 * D)), fv(std::vector<float>(P * 16 * D));
        step("unpack");
        reef_hip::kv_unpack_int4(kc.p, vc.p, ks.p, vs.p, P, D, fk.p, fv.p, nullptr);
        const auto gk = fk.host(), gv = fv.host();
        bool ok = true;
        for (int64_t t = 0; t < T; ++t)
            for (int64_t d = 0; d < D; ++d) {
                const int64_t i = (table[t / 16] * 16 + t % 16) * D + d;
                ok &= gk[i] == hk[t * D + d] && gv[i] == hv[t * D + d];
            }
        check("rows", ok);
        step("copy of a page");
        Device<int32_t> src({3}), dst({0});
        reef_hip::kv_copy_pages(src.p, dst.p, 1, 1, D, kc.p, vc.p, ks.p, vs.p, P, status.p, nullptr);
        const auto c = kc.host();
        check("page", std::equal(c.begin(), c.begin() + 16 * row, c.begin() + 3 * 16 * row));
    } else {
        reef_hip::check(reef_kv_append_int8_paged(&rows, dk.p, nullptr, dv.p, nullptr, start.p, dt.p,
                                                  blocks, P, kc.p, vc.p, ks.p, vs.p, lens.p, status.p,
                                                  nullptr),
                        "append");
    }
    check("length", lens.host()[0] == T);

    Device<int8_t> bounds(std::vector<int8_t>(P * 2 * D));
    Device<float> bs{std::vector<float>(P)};
    step("bounds");
    reef_hip::kv_page_bounds(rows, start.p, kc.p, ks.p, dt.p, blocks, P, bounds.p, bs.p, status.p, nullptr);
    const auto gb = bounds.host();
    const auto gs = bs.host();
    bool ok = true;
    for (int64_t pg = 0; pg < blocks; ++pg) {
        float top = 0;
        for (int64_t t = pg * 16; t < std::min(T, pg * 16 + 16); ++t)
            for (int64_t d = 0; d < D; ++d) top = std::max(top, std::fabs(hk[t * D + d]));
        volatile float scale = top / 127.0f;
        ok &= gs[table[pg]] == scale;
        for (int64_t d = 0; d < D; ++d) {
            float hi = -1e30f, lo = 1e30f;
            for (int64_t t = pg * 16; t < std::min(T, pg * 16 + 16); ++t) {
                hi = std::max(hi, hk[t * D + d]);
                lo = std::min(lo, hk[t * D + d]);
            }
            const int8_t *b = &gb[table[pg] * 2 * D];
            ok &= b[d] == std::min(127.0f, std::ceil(hi / scale));
            ok &= b[D + d] == std::max(-127.0f, std::floor(lo / scale));
        }
    }
    check("bounds", ok);

    std::vector<int8_t> q(G * D);
    const auto qf = uniform(G * D, 11);
    for (size_t i = 0; i < q.size(); ++i) q[i] = (int8_t)(qf[i] * 127);
    const std::vector<float> qs{0.02f, 0.03f};
    Device<int8_t> dq(q);
    Device<float> dqs(qs), out(std::vector<float>(G * D));
    Device<int32_t> pages({9, 9}), counts({9});
    const reef_decode_params p{1, G, 1, D, blocks * 16, 0, 0.125f, REEF_SCALE_PER_TOKEN, 0, 0};
    Device<int8_t> words(std::vector<int8_t>(reef_hip::select_workspace_bytes(p)));
    Device<int8_t> work(std::vector<int8_t>(reef_hip::decode_workspace_bytes(p)));
    step("selection");
    reef_hip::kv_select_pages(p, dq.p, dqs.p, bounds.p, bs.p, dt.p, blocks, P, lens.p, 2, 0, 1, pages.p,
                              counts.p, words.p, words.n, status.p, nullptr);
    float score[2] = {-1e30f, -1e30f};
    for (int64_t pg = 0; pg < 2; ++pg)
        for (int64_t h = 0; h < G; ++h) {
            int64_t sum = 0;
            for (int64_t d = 0; d < D; ++d) {
                const int x = q[h * D + d];
                sum += x * gb[table[pg] * 2 * D + (x > 0 ? d : D + d)];
            }
            volatile float unit = qs[h] * gs[table[pg]];
            score[pg] = std::max(score[pg], (float)sum * unit);
        }
    const int32_t best = score[1] > score[0] ? 1 : 0;
    const auto gp = pages.host();
    check("pages", counts.host()[0] == 2 && gp[0] == best && gp[1] == 2);

    step("decode over the selected pages");
    const reef_page_selection chosen{pages.p, counts.p, 2};
    std::vector<int64_t> tokens;
    for (int64_t t = 0; t < T; ++t)
        if (t / 16 == best || t / 16 == 2) tokens.push_back(t);
    if constexpr (std::is_same<Code, uint8_t>::value)
        reef_hip::decode_int4(p, dq.p, dqs.p, kc.p, vc.p, ks.p, vs.p, dt.p, blocks, P, lens.p, &chosen,
                              out.p, work.p, work.n, status.p, nullptr);
    else
        reef_hip::decode_selected(p, dq.p, dqs.p, kc.p, vc.p, ks.p, vs.p, dt.p, blocks, P, lens.p, chosen,
                                  out.p, work.p, work.n, status.p, nullptr);
    const auto go = out.host();
    ok = true;
    for (int64_t h = 0; h < G; ++h)
        for (int64_t d = 0; d < D; ++d)
            ok &= std::fabs(go[h * D + d] - attention(hk, hv, &q[h * D], qs[h], tokens, d)) < 1e-5;
    check("outputs", ok);

    if constexpr (std::is_same<Code, uint8_t>::value) {
        step("prefill over the cache");
        const reef_attention_params a{1, G, 1, 1, T, D, T - 1, 0, 0.125f, REEF_SCALE_PER_HEAD,
                                      REEF_SCALE_PER_TOKEN, 0};
        Device<int8_t> chunk(std::vector<int8_t>(reef_hip::prefill_cache_workspace_bytes(a)));
        reef_hip::context_cache(a, dq.p, nullptr, dqs.p, kc.p, vc.p, ks.p, vs.p, 0, dt.p, blocks, P, out.p,
                                nullptr, chunk.p, chunk.n, status.p, nullptr);
        tokens.resize(T);
        for (int64_t t = 0; t < T; ++t) tokens[t] = t;
        const auto gc = out.host();
        ok = true;
        for (int64_t h = 0; h < G; ++h)
            for (int64_t d = 0; d < D; ++d)
                ok &= std::fabs(gc[h * D + d] - attention(hk, hv, &q[h * D], qs[h], tokens, d)) < 1e-3;
        check("outputs", ok);
    }
    check("no status", status.host()[0] == 0);
}

int main() {
    try {
        const auto k = uniform(T * D, 3), v = uniform(T * D, 5);
        run<uint8_t>(k, v);
        run<int8_t>(k, v);
    } catch (const std::exception &e) {
        std::printf("FAIL exception: %s\n", e.what());
        ++failures;
    }
    std::printf("%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
