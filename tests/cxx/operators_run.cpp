// The drafted-token, page, norm and epilogue calls of include/reef_hip/attention.hpp on a device,
// each against its formula on the host. Prints each step before it runs.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <stdexcept>
#include <string>
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

// A pseudorandom sequence of codes in [-127, 127].
static std::vector<int8_t> codes(size_t n, uint32_t seed) {
    std::vector<int8_t> v(n);
    for (auto &x : v) {
        seed = seed * 1664525u + 1013904223u;
        x = (int8_t)((int)(seed >> 16) % 255 - 127);
    }
    return v;
}

static void pages() {
    const int64_t B = 2, blocks = 3, P = 8, H = 1, D = 64;
    Device<int32_t> table(std::vector<int32_t>(B * blocks, -1)), lens({0, 0}),
        refs(std::vector<int32_t>(P, 0)), src({5, 5}), dst({5, 5}), msrc(std::vector<int32_t>(P / 2)),
        mdst(std::vector<int32_t>(P / 2)), live({-1}), zero({0}), one({1});
    Device<uint32_t> status({0});
    Device<int8_t> k(codes(P * H * 16 * D, 1)), v(codes(P * H * 16 * D, 2));
    Device<float> ks(std::vector<float>(P * H * 16, 0.5f)), vs(std::vector<float>(P * H * 16, 0.25f));
    const reef_hip::page_table t{table.p, B, blocks, lens.p, refs.p, P};
    Device<int8_t> ws(std::vector<int8_t>(t.reserve_workspace_bytes(20) + t.compact_workspace_bytes()));

    step("reserve");
    t.reserve(20, src.p, dst.p, ws.p, ws.n, status.p, nullptr);
    check("two pages a sequence", table.host() == std::vector<int32_t>{0, 1, -1, 2, 3, -1});
    const std::vector<int32_t> lengths{20, 0};
    need(hipMemcpy(lens.p, lengths.data(), 8, hipMemcpyHostToDevice));
    step("fork");
    t.fork(zero.p, one.p, 1, status.p, nullptr);
    check("the child shares", table.host() == std::vector<int32_t>{0, 1, -1, 0, 1, -1});
    check("counts", refs.host() == std::vector<int32_t>{2, 2, 0, 0, 0, 0, 0, 0});
    check("lengths", lens.host() == std::vector<int32_t>{20, 20});
    step("reserve with copy on write");
    t.reserve(3, src.p, dst.p, ws.p, ws.n, status.p, nullptr);
    check("pages of their own", table.host() == std::vector<int32_t>{0, 2, -1, 0, 3, -1});
    check("copies", src.host() == std::vector<int32_t>{1, 1} && dst.host() == std::vector<int32_t>{2, 3});
    const auto before = k.host();
    step("copy pages");
    reef_hip::kv_copy_pages(src.p, dst.p, B, H, D, k.p, v.p, ks.p, vs.p, P, status.p, nullptr);
    auto want = before;
    for (int64_t i = 0; i < 16 * D; ++i) want[2 * 16 * D + i] = want[3 * 16 * D + i] = before[16 * D + i];
    check("keys copied", k.host() == want);
    step("free, compact");
    t.free(zero.p, 1, status.p, nullptr);
    t.compact(msrc.p, mdst.p, live.p, ws.p, ws.n, status.p, nullptr);
    check("two live pages", live.host() == std::vector<int32_t>{2});
    check("at the front", table.host() == std::vector<int32_t>{-1, -1, -1, 0, 1, -1});
    check("moves", msrc.host() == std::vector<int32_t>{3, -1, -1, -1} &&
                       mdst.host() == std::vector<int32_t>{1, -1, -1, -1});
    check("no status", status.host()[0] == 0);
}

static void tree(bool paged) {
    const int64_t B = 1, Hq = 2, H = 1, D = 64, T = 3, L = 32, n = 21;
    const auto q = codes(B * Hq * T * D, 3), k = codes(B * H * L * D, 4), v = codes(B * H * L * D, 5);
    std::vector<int8_t> vp(v.size());  // [L / 16, D, 16]
    for (int64_t j = 0; j < L; ++j)
        for (int64_t d = 0; d < D; ++d) vp[(j / 16 * D + d) * 16 + j % 16] = v[j * D + d];
    const float qs = 0.01f, ksc = 0.02f, vsc = 0.03f;
    const std::vector<uint64_t> mask{1, 3, 5};  // two branches after the first token
    Device<int8_t> dq(q), dk(k), dv(vp);
    Device<float> dqs(std::vector<float>(B * Hq * T, qs)), dks(std::vector<float>(L, ksc)),
        dvs(std::vector<float>(L, vsc)), out(std::vector<float>(B * Hq * T * D, -1.0f));
    Device<int32_t> lens({(int32_t)n}), table({0, 1}), kept({0, 2, 0}), kept_n({2}), new_lens({0});
    Device<uint64_t> dm(mask);
    Device<uint32_t> status({0});
    const reef_tree_params p{B, Hq, H, D, T, L, 0, 0.125f, REEF_SCALE_PER_TOKEN, 0, 0};
    Device<int8_t> ws(std::vector<int8_t>(reef_hip::tree_workspace_bytes(p), 0));
    step(paged ? "tree, paged" : "tree");
    if (paged)
        reef_hip::decode_tree_paged(p, dq.p, nullptr, dqs.p, dk.p, dv.p, dks.p, dvs.p, table.p, L / 16,
                                    L / 16, lens.p, dm.p, out.p, nullptr, ws.p, ws.n, status.p, nullptr);
    else
        reef_hip::decode_tree(p, dq.p, nullptr, dqs.p, dk.p, dv.p, dks.p, dvs.p, lens.p, dm.p, out.p,
                              nullptr, ws.p, ws.n, status.p, nullptr);
    const auto got = out.host();
    // Of the largest value: an exponent of X log2 units in four roundings, and 40 units for exp2, the
    // weights' parts and the merges, 2^-24 (5.6 X + 40).
    double worst = 0.0, top = 0.0;
    for (int64_t h = 0; h < Hq; ++h)
        for (int64_t i = 0; i < T; ++i) {
            std::vector<double> w(n, 0.0);
            double sum = 0.0, m = -1e300;
            for (int64_t j = 0; j < n; ++j) {
                double s = 0.0;
                for (int64_t d = 0; d < D; ++d) s += q[(h * T + i) * D + d] * k[j * D + d];
                w[j] = s * (double)qs * (double)ksc * 0.125;
                if (j >= n - T && !(mask[i] >> (j - (n - T)) & 1)) w[j] = -1e300;
                m = std::fmax(m, w[j]);
                if (w[j] > -1e299) top = std::fmax(top, std::fabs(w[j]) / std::log(2.0));
            }
            for (auto &x : w) sum += x = x < -1e299 ? 0.0 : std::exp(x - m);
            for (int64_t d = 0; d < D; ++d) {
                double o = 0.0;
                for (int64_t j = 0; j < n; ++j) o += w[j] * v[j * D + d] * (double)vsc / sum;
                worst = std::fmax(worst, std::fabs(o - got[(h * T + i) * D + d]));
            }
        }
    std::printf("     worst %.3g, exponents up to %.3g\n", worst, top);
    check("rows", worst <= 127 * vsc * (2 * 2.8 * top + 40) * std::ldexp(1.0, -24));

    step(paged ? "keep, paged" : "keep");
    const reef_kv_append_params rows{B, H, D, T, L};
    if (paged)
        reef_hip::kv_keep_paged(rows, kept.p, kept_n.p, lens.p, table.p, L / 16, L / 16, dk.p, dv.p, dks.p,
                                dvs.p, new_lens.p, status.p, nullptr);
    else
        reef_hip::kv_keep(rows, kept.p, kept_n.p, lens.p, dk.p, dv.p, dks.p, dvs.p, new_lens.p, status.p,
                          nullptr);
    auto want = k;
    for (int64_t d = 0; d < D; ++d) want[(n - T + 1) * D + d] = k[(n - T + 2) * D + d];
    check("kept keys", dk.host() == want);
    check("new length", new_lens.host()[0] == n - T + 2);
    check("no status", status.host()[0] == 0);
}

static void norm_and_product() {
    const int64_t rows = 3, width = 16, out = 5;
    std::vector<float> x(rows * width), r(rows * width), w(width);
    const auto a = codes(x.size(), 6), b = codes(x.size(), 7), c = codes(width, 8);
    for (size_t i = 0; i < x.size(); ++i) x[i] = a[i] / 32.0f, r[i] = b[i] / 64.0f;
    for (size_t i = 0; i < w.size(); ++i) w[i] = 1.0f + c[i] / 256.0f;
    Device<float> dx(x), dr(r), dw(w), scales(std::vector<float>(rows, 0.0f)), sum(std::vector<float>(x.size()));
    Device<int8_t> q(std::vector<int8_t>(x.size()));
    Device<uint32_t> status({0});
    step("norm");
    reef_hip::rmsnorm_quantize(dx.p, rows, width, width, dr.p, width, dw.p, 1e-6, q.p, scales.p, sum.p, width,
                               status.p, nullptr);
    const auto gq = q.host();
    const auto gs = scales.host(), gsum = sum.host();
    bool ok = true;
    for (int64_t i = 0; i < rows; ++i) {
        double ms = 0.0, top = 0.0;
        std::vector<double> y(width);
        for (int64_t j = 0; j < width; ++j) {
            const float h = x[i * width + j] + r[i * width + j];
            ok &= gsum[i * width + j] == h;
            ms += (double)h * h / width;
            y[j] = (double)h * w[j];
        }
        for (auto &e : y) top = std::fmax(top, std::fabs(e /= std::sqrt(ms + 1e-6)));
        ok &= std::fabs(gs[i] - top / 127) <= std::ldexp(top / 127, -23);
        for (int64_t j = 0; j < width; ++j) ok &= std::fabs(y[j] / gs[i] - gq[i * width + j]) <= 0.5 + 1e-9;
    }
    check("sum, scales, codes", ok);

    const auto weight = codes(out * width, 9);
    std::vector<float> ws(out, 0.01f), bias(out, 0.5f), res(rows * out, 2.0f);
    Device<int8_t> dweight(weight);
    Device<float> dws(ws), dbias(bias), y(res), z(std::vector<float>(rows * out));
    Device<int8_t> work(std::vector<int8_t>(reef_linear_w8a8_workspace_bytes(rows, width)));
    step("product with its epilogue");
    const reef_epilogue relu{y.p, out, REEF_ACT_RELU};  // in place: the residual is the output
    reef_hip::gemm_w8a8(q.p, scales.p, rows, width, dweight.p, dws.p, dbias.p, relu, out, y.p, out, status.p,
                        nullptr);
    const reef_epilogue none{nullptr, 0, REEF_ACT_NONE};
    reef_hip::linear_w8a8(sum.p, rows, width, width, dweight.p, dws.p, dbias.p, none, out, z.p, out, work.p,
                          work.n, status.p, nullptr);
    const auto gy = y.host(), gz = z.host();
    ok = true;
    for (int64_t i = 0; i < rows; ++i) {
        float top = 0.0f;
        for (int64_t j = 0; j < width; ++j) top = std::fmax(top, std::fabs(gsum[i * width + j]));
        const float scale = top / 127.0f;
        for (int64_t o = 0; o < out; ++o) {
            int64_t s = 0, t = 0;
            for (int64_t j = 0; j < width; ++j) {
                s += gq[i * width + j] * weight[o * width + j];
                t += (int)std::nearbyint(gsum[i * width + j] / scale) * weight[o * width + j];
            }
            // (no contraction: each step rounded on its own)
            volatile float e = gs[i] * ws[o], f = (float)s * e, g = f + bias[o];
            ok &= gy[i * out + o] == std::fmax((float)g, 0.0f) + 2.0f;
            volatile float l = scale * ws[o], m = (float)t * l;
            ok &= gz[i * out + o] == m + bias[o];
        }
    }
    check("products", ok);
    check("no status", status.host()[0] == 0);
}

int main() {
    try {
        pages();
        tree(false);
        tree(true);
        norm_and_product();
    } catch (const std::exception &e) {
        std::printf("FAIL exception: %s\n", e.what());
        ++failures;
    }
    std::printf("%d failures\n", failures);
    return failures == 0 ? 0 : 1;
}
