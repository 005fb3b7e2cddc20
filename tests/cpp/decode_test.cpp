// GPU check of the C++ host adapter's answering path (include/te_b200.hpp): rotary positions of q and k head views inside a
// projections' buffer, keys and values kept in pages, attention of each new token, against plain loops in double on the host.
// Exit code 0 on success.
#include <cmath>
#include <cstdio>
#include <iostream>
#include <vector>

#include "te_b200.hpp"

using te::IndexArray;
using te::KvCache;
using te::Rotary;
using te::Tensor;

static int failures = 0;

static void expect(const char* what, bool ok) {
    std::cout << (ok ? "ok   " : "FAIL ") << what << "\n";
    if (!ok) ++failures;
}
template <typename F>
static void expect_throw(const char* what, F&& f, const std::string& part) {
    bool ok = false;
    try {
        f();
    } catch (const std::runtime_error& e) {
        ok = std::string(e.what()).find(part) != std::string::npos;
        if (!ok) std::cout << "     got message: " << e.what() << "\n";
    }
    expect(what, ok);
}

static uint64_t state = 88172645463325252ull;
static float uniform() {
    state ^= state << 13; state ^= state >> 7; state ^= state << 17;
    return (float)((double)(state >> 11) / 9007199254740992.0 * 2.0 - 1.0);
}

int main() {
    try {
        const int64_t B = 2, T = 21, HQ = 4, HK = 2, D = 32, page = 8, max_pages = 3;
        // [B, T, (HQ + 2 HK) D] as the projections leave it, and its head view [B, H, T, D]
        std::vector<float> host((size_t)(B * T * (HQ + 2 * HK) * D));
        for (float& x : host) x = uniform();
        Tensor qkv = Tensor::from_host(host, {B, T, HQ + 2 * HK, D});
        Tensor heads = qkv.transpose_view(1, 2);
        std::vector<int64_t> pos((size_t)(B * T)), table = {4, 0, 2, 5, 1, 3};
        for (int64_t b = 0; b < B; ++b)
            for (int64_t t = 0; t < T; ++t) pos[(size_t)(b * T + t)] = t;
        IndexArray positions(pos), page_table(table);
        Rotary rotary(D);
        Tensor turned = rotary.forward(heads, positions);           // v heads too; only q and k heads are used
        std::vector<float> got = turned.to_host();
        std::vector<double> want(got.size());
        double worst = 0.0;
        for (int64_t b = 0; b < B; ++b)
            for (int64_t h = 0; h < HQ + 2 * HK; ++h)
                for (int64_t t = 0; t < T; ++t) {
                    const float* x = &host[(size_t)(((b * T + t) * (HQ + 2 * HK) + h) * D)];
                    double* y = &want[(size_t)(((b * (HQ + 2 * HK) + h) * T + t) * D)];
                    for (int64_t j = 0; j < D / 2; ++j) {
                        const double a = (double)t * std::pow(10000.0, -2.0 * (double)j / (double)D), c = std::cos(a), s = std::sin(a);
                        y[j] = x[j] * c - x[j + D / 2] * s;
                        y[j + D / 2] = x[j] * s + x[j + D / 2] * c;
                    }
                    for (int64_t j = 0; j < D; ++j) worst = std::fmax(worst, std::fabs(y[j] - got[(size_t)(y - want.data() + j)]));
                }
        expect("rotary positions of head views", worst <= 2.0 * 12.0 * std::ldexp(1.0, -24));      // 12 * 2^-24 of |x0| + |x1| <= 2
        worst = 0.0;
        std::vector<float> back = rotary.backward(turned, positions).to_host(), original = heads.to_host();
        for (size_t i = 0; i < back.size(); ++i) worst = std::fmax(worst, std::fabs((double)back[i] - original[i]));
        expect("turned back", worst <= 2.0 * 2.0 * std::sqrt(2.0) * 12.0 * std::ldexp(1.0, -24));  // two turns

        // the first HK heads behind the queries are keys; values are taken untouched
        auto part = [&](const std::vector<float>& all, int64_t first, int64_t count) {     // of [B, H, T, D]
            std::vector<float> r;
            for (int64_t b = 0; b < B; ++b)
                r.insert(r.end(), all.begin() + (b * (HQ + 2 * HK) + first) * T * D, all.begin() + (b * (HQ + 2 * HK) + first + count) * T * D);
            return r;
        };
        const std::vector<float> kh = part(got, HQ, HK), vh = part(original, HQ + HK, HK);
        Tensor k = Tensor::from_host(kh, {B, HK, T, D}), v = Tensor::from_host(vh, {B, HK, T, D});
        for (int dtype : {TE_KV_F32, TE_KV_BF16, TE_KV_E4M3}) {
            KvCache cache(6, HK, page, D, dtype);
            cache.append(k, v, page_table, max_pages, positions);
            std::vector<Tensor> kept = cache.read(page_table, max_pages, positions, B, T);
            const std::vector<float> kk = kept[0].to_host(), vv = kept[1].to_host();
            const double half_step = dtype == TE_KV_F32 ? 0.0 : dtype == TE_KV_BF16 ? std::ldexp(1.0, -8) : std::ldexp(1.0, -4);
            // an 8-bit value below the grid's normal range is off by 2^-10 of the row's scale, which is at most 2 / 224
            const double floor_step = dtype == TE_KV_E4M3 ? std::ldexp(1.0, -10) * 4.0 / 224.0 : 0.0;
            bool near = true;
            for (size_t i = 0; i < kk.size(); ++i)
                near = near && std::fabs((double)kk[i] - kh[i]) <= half_step * std::fabs(kh[i]) + floor_step && std::fabs((double)vv[i] - vh[i]) <= half_step * std::fabs(vh[i]) + floor_step;
            expect("cache keeps what went in", near);
            for (int64_t n : {(int64_t)0, (int64_t)1, (int64_t)8, (int64_t)13, T}) {
                std::vector<float> q((size_t)(B * HQ * D));
                for (float& x : q) x = uniform();
                Tensor lse;
                Tensor o = te::paged_attention(Tensor::from_host(q, {B, HQ, D}), cache, page_table, max_pages, IndexArray({n, T - n}), 0, &lse);
                const std::vector<float> oh = o.to_host();
                double off = 0.0;
                for (int64_t b = 0; b < B; ++b)
                    for (int64_t h = 0; h < HQ; ++h) {
                        const int64_t len = b == 0 ? n : T - n, g = h / (HQ / HK);
                        std::vector<double> acc((size_t)D, 0.0);
                        double total = 0.0;
                        for (int64_t t = 0; t < len; ++t) {
                            double s = 0.0;
                            for (int64_t i = 0; i < D; ++i) s += (double)q[(size_t)((b * HQ + h) * D + i)] * kk[(size_t)(((b * HK + g) * T + t) * D + i)];
                            const double w = std::exp(s / std::sqrt((double)D));
                            total += w;
                            for (int64_t i = 0; i < D; ++i) acc[(size_t)i] += w * vv[(size_t)(((b * HK + g) * T + t) * D + i)];
                        }
                        for (int64_t i = 0; i < D; ++i)
                            off = std::fmax(off, std::fabs((total > 0.0 ? acc[(size_t)i] / total : 0.0) - oh[(size_t)((b * HQ + h) * D + i)]));
                    }
                // |v| <= 1; scores of 32 products of magnitudes up to sqrt(2), scaled, sum |q||k| / sqrt(32) <= 8: 4 sqrt(32) 2^-24 * 8, twice, and
                // 2 * 2^-22 for exp2, sums of 21 and a few roundings
                expect("attention of a new token", off <= (2.0 * 4.0 * 5.7 * 8.0 + 8.0 + 8.0 * 4.6 + 8.0) * std::ldexp(1.0, -24));
            }
        }
        expect_throw("wrong page table", [&] { KvCache c(6, HK, page, D); c.append(k, v, page_table, 2, positions); }, "row of max_pages");
        expect_throw("d not a multiple of 16", [&] { KvCache c(6, HK, page, 24); c.read(page_table, max_pages, positions, B, T); }, "multiple of 16");
        expect_throw("odd rotated width", [&] { Rotary r(7); }, "even");
        expect_throw("cache dtype", [&] { KvCache c(6, HK, page, D, 9); }, "TE_KV_");
        te::check(te_b200_check_device_status(te::Backend::instance().ctx()));
    } catch (const std::exception& e) {
        std::cout << "FAIL exception: " << e.what() << "\n";
        return 1;
    }
    if (failures) {
        std::cout << failures << " checks failed.\n";
        return 1;
    }
    std::cout << "All decode checks passed.\n";
    return 0;
}
