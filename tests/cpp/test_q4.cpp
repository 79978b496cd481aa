// test_q4.cpp -- the C++ API of the appends that rotate and of caches held in 4 bits
// (serving-engine_amd/engine/kernels.h, PagedKVCache with Format::kQ4): a prompt, a
// chunk behind a shared prefix and decode steps through one PagedKVCache, against
// attention in double over what its pages hold.
//
//   test_q4 --cpu   refusals
//   test_q4 --gpu   every case
// Exit status 0 when every check passed.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <stdexcept>
#include <string>
#include <vector>

#include "half.h"
#include "hip_utils.h"
#include "kernels.h"
#include "kv_cache.h"

using namespace engine;

namespace {

int g_checks = 0;
int g_failures = 0;

#define EXPECT(cond, ...)                                                  \
    do {                                                                   \
        ++g_checks;                                                        \
        if (!(cond)) {                                                     \
            if (++g_failures < 40) {                                       \
                std::printf("  FAIL %s:%d: %s -- ", __FILE__, __LINE__, #cond); \
                std::printf(__VA_ARGS__);                                  \
                std::printf("\n");                                         \
            }                                                              \
        }                                                                  \
    } while (0)

constexpr int kHq = 8, kHkv = 2, kD = 64, kG = kHq / kHkv, kH = kHq + 2 * kHkv;
constexpr int kLayers = 2, kLayer = 1, kSlots = 3;
constexpr float kTheta = 10000.f;
constexpr double kU16 = 1.0 / 2048, kU32 = 1.0 / (1 << 24), kTiny = 1.0 / (1 << 25);

std::vector<half> random_half(std::mt19937& rng, size_t n) {
    std::uniform_real_distribution<float> dist(-1.f, 1.f);
    std::vector<half> v(n);
    for (auto& x : v) x = float_to_half(dist(rng));
    return v;
}

template <typename T>
DeviceBuffer<T> upload(const std::vector<T>& v) {
    DeviceBuffer<T> d(v.size());
    d.copy_from_host(v.data(), v.size());
    return d;
}

template <typename T>
std::vector<T> download(const T* d, size_t n) {
    std::vector<T> v(n);
    HIP_CHECK(hipMemcpy(v.data(), d, n * sizeof(T), hipMemcpyDeviceToHost));
    return v;
}

template <typename F>
std::string refusal(F&& f) {
    try {
        f();
    } catch (const std::exception& e) {
        return e.what();
    }
    return "";
}

void case_refusals() {
    // addresses that no call reaches: each is refused before any device work
    alignas(16) static half data[64] = {};
    alignas(16) static uint8_t bytes[64] = {};
    alignas(16) static int32_t ints[64] = {};
    EXPECT(!refusal([&] {
               hip::rope_append(data, data, data, kHq * kD, kHkv * kD - 1, kHkv * kD, ints, nullptr,
                                nullptr, kTheta, data, data, data, ints, 2, 4, 1, 1, kHq, kHkv, kD);
           }).empty(), "rope_append took rows that overlap");
    EXPECT(!refusal([&] {
               hip::q4_rope_append(data, data, data, kHq * 60, kHkv * 60, kHkv * 60, ints, nullptr,
                                   nullptr, kTheta, data, bytes, ints, 2, 4, 1, 1, kHq, kHkv, 60);
           }).empty(), "q4_rope_append took head_dim 60");
    EXPECT(!refusal([&] {
               hip::q4_gather(bytes, ints, 2, 4, nullptr, nullptr, data, data, 1, kHkv, kD, 8);
           }).empty(), "q4_gather took no lengths");
    EXPECT(refusal([&] {
               hip::q4_decode(data, bytes, ints, 2, 4, ints, data, 1, 6, 4, kD, 16, nullptr, 0);
           }).find("num_q_heads") != std::string::npos, "q4_decode took Hq = 6, Hkv = 4");
    EXPECT(!refusal([&] {
               hip::q4_decode(data, bytes, ints, 512, 4, ints, data, 1, kHq, kHkv, kD, 8192, nullptr, 0);
           }).empty(), "q4_decode took no workspace for 8192 keys");
    EXPECT(!refusal([&] {
               hip::q4_prefill(data, bytes + 1, ints, 2, 4, nullptr, ints, data, nullptr, 1, 4, kHq,
                               kHkv, kD, 16, nullptr, 0);
           }).empty(), "q4_prefill took a pool off its alignment");
    EXPECT(hip::q4_page_bytes(kD) == 16 * (kD + 8) && hip::q4_page_bytes(60) == 0, "page sizes");
    const size_t fp16 = (size_t)kLayers * 2 * kHkv * 16 * kD * sizeof(half);
    using Format = PagedKVCache::Format;
    EXPECT(PagedKVCache::pages_for_bytes(9 * fp16, kLayers, kHkv, kD) == 9, "fp16 pages");
    EXPECT(PagedKVCache::pages_for_bytes(9 * fp16, kLayers, kHkv, kD, Format::kQ4) == 32, "4-bit pages");
    EXPECT(!refusal([&] { PagedKVCache(1, 1, 60, 1, 1, 1, Format::kQ4); }).empty(), "head_dim 60 in 4 bits");
    // nothing to do is done at once
    EXPECT(refusal([&] {
               hip::q4_decode(data, bytes, ints, 2, 4, ints, data, 0, kHq, kHkv, kD, 16, nullptr, 0);
           }).empty(), "an empty batch threw");
}

// What slot j of KV head h of a sequence stands for: K's and V's rows.
struct Rows {
    double k[kD], v[kD];
};
Rows stands(const std::vector<half>& pool, const PagedKVCache& cache, int slot, int h, int j) {
    const size_t pb = hip::q4_page_bytes(kD);
    const uint8_t* pg = reinterpret_cast<const uint8_t*>(pool.data()) +
                        (((size_t)kLayer * kHkv + h) * cache.num_pages() + cache.host_block_table(slot)[j / 16]) * pb;
    Rows r;
    for (int is_v = 0; is_v < 2; ++is_v) {
        half p[2];
        std::memcpy(p, pg + 16 * kD + 64 * is_v + 4 * (j % 16), 4);
        const double s = half_to_float(p[0]), o = half_to_float(p[1]);
        for (int i = 0; i < kD; ++i) {
            const int code = pg[8 * kD * is_v + j % 16 * (kD / 2) + i / 2] >> 4 * (i % 2) & 15;
            (is_v ? r.v : r.k)[i] = s * (code + o);
        }
    }
    return r;
}
// A row rotated to `pos`.
void rotated(const half* x, int pos, double* y) {
    for (int i = 0; i < kD / 2; ++i) {
        const double a = pos * std::pow((double)kTheta, -2.0 * i / kD), c = std::cos(a), s = std::sin(a);
        const double u = half_to_float(x[i]), w = half_to_float(x[i + kD / 2]);
        y[i] = u * c - w * s;
        y[i + kD / 2] = w * c + u * s;
    }
}
// A row against what its four bits may be off by: half a step, the steps' rounding up to
// fp16, fp16's rounding before and the offset's (at most half a unit of n + r, 2^-6).
void check_codes(const double* want, const double* got, const char* what, int j) {
    const double lo = *std::min_element(want, want + kD), hi = *std::max_element(want, want + kD);
    const double big = std::max(std::abs(lo), std::abs(hi)), s = std::max((hi - lo) / 15, big / 1984) * 1.002;
    double worst = 0;
    for (int i = 0; i < kD; ++i) worst = std::max(worst, std::abs(got[i] - want[i]));
    EXPECT(worst <= s * (0.5 + 1.0 / 64) + 2 * kU16 * big, "%s token %d: off by %g of %g", what, j, worst, s);
}
// Attention of q over the first n slots; the tolerance of each output.
void check_attention(const half* q, const half* got, float lse, bool has_lse, const std::vector<Rows>& rows, int n,
                     const char* what) {
    std::vector<double> s(n);
    double top = -INFINITY, size = 0, vmax = 0;
    for (int j = 0; j < n; ++j) {
        double a = 0, b = 0;
        for (int i = 0; i < kD; ++i) {
            const double x = half_to_float(q[i]) * rows[j].k[i];
            a += x;
            b += std::abs(x);
            vmax = std::max(vmax, std::abs(rows[j].v[i]));
        }
        s[j] = a / std::sqrt((double)kD);
        top = std::max(top, s[j]);
        size = std::max(size, b / std::sqrt((double)kD));
    }
    double l = 0;
    for (auto& x : s) l += x = std::exp(x - top);
    // scores of kD exact products, the weight's rounding to fp16 (2^-25 below the smallest
    // normal one), sums of n terms, the result's rounding
    const double ds = (kD + 8) * kU32 * size;
    for (int i = 0; i < kD; ++i) {
        double o = 0, spread = 0;
        for (int j = 0; j < n; ++j) {
            o += s[j] / l * rows[j].v[i];
            spread += s[j] / l * std::abs(rows[j].v[i]);
        }
        const double tol = kU16 * std::abs(o) + (2 * kU16 + 2 * ds + 2 * n * kU32) * spread + n * kTiny * vmax / l + kTiny;
        EXPECT(std::abs(half_to_float(got[i]) - o) <= tol, "%s of %d keys, dim %d: %g, not %g (+- %g)", what, n, i,
               half_to_float(got[i]), o, tol);
    }
    if (has_lse)
        EXPECT(std::abs(lse - (top + std::log(l))) <= ds + (n + 12) * kU32 + 4 * kU32 * std::abs(top + std::log(l)),
               "%s lse %g, not %g", what, lse, top + std::log(l));
}

void case_served() {
    std::mt19937 rng(4);
    using Format = PagedKVCache::Format;
    PagedKVCache cache(kLayers, kHkv, kD, 24, kSlots, 10, Format::kQ4);
    EXPECT(cache.pool_bytes() == (size_t)kLayers * kHkv * 24 * hip::q4_page_bytes(kD), "pool");
    EXPECT(cache.add_sequence() == 0 && cache.add_sequence() == 1, "slots");   // the third stays idle
    const int cap = cache.max_pages_per_seq() * PagedKVCache::kPage;
    const size_t nd = hip::q4_decode_workspace_bytes(kSlots, kHq, kHkv, kD, cap);
    const size_t np = hip::q4_prefill_workspace_bytes(kSlots, 70, kHq, kHkv, kD, cap);
    DeviceBuffer<char> ws(std::max<size_t>({nd, np, 16}));
    std::vector<std::vector<half>> text(kSlots);   // each token's projection [kH][kD], by slot
    const size_t token = (size_t)kH * kD;

    // One step of R rows for every slot: append, attend, and check against the pages.
    auto step = [&](int R, bool decode, const char* what) {
        auto x = random_half(rng, (size_t)kSlots * R * token);
        int at[kSlots];
        for (int b = 0; b < kSlots; ++b) at[b] = cache.seq_len(b) - R;
        for (int b = 0; b < 2; ++b) {
            text[b].resize(at[b] * token);
            text[b].insert(text[b].end(), x.begin() + b * R * token, x.begin() + (b + 1) * R * token);
        }
        cache.sync();
        auto dx = upload(x);
        const half seven = float_to_half(7.f);
        auto q = upload(std::vector<half>((size_t)kSlots * R * kHq * kD, seven));
        auto out = upload(std::vector<half>(q.size(), seven));
        auto lse = upload(std::vector<float>((size_t)kSlots * kHq * R, 7.f));
        cache.rope_append(kLayer, dx.data(), dx.data() + kHq * kD, dx.data() + (kHq + kHkv) * kD, token, token,
                          token, kTheta, q.data(), kSlots, R, kHq);
        if (decode)
            cache.q4_decode(kLayer, q.data(), out.data(), kSlots, kHq, cap, ws.data(), nd);
        else
            cache.q4_prefill(kLayer, q.data(), out.data(), lse.data(), kSlots, R, kHq, cap, ws.data(), np);
        HIP_CHECK(hipDeviceSynchronize());
        const auto hq = download(q.data(), q.size()), ho = download(out.data(), out.size());
        const auto hl = download(lse.data(), lse.size());
        const auto pool = download(cache.raw_data(), cache.pool_bytes() / sizeof(half));
        double y[kD];
        for (int b = 0; b < 2; ++b)
            for (int h = 0; h < kHkv; ++h) {
                std::vector<Rows> rows(cache.seq_len(b));
                for (int j = 0; j < cache.seq_len(b); ++j) {
                    rows[j] = stands(pool, cache, b, h, j);
                    const half* t = &text[b][j * token];
                    rotated(t + (kHq + h) * kD, j, y);
                    check_codes(y, rows[j].k, "K of", j);
                    for (int i = 0; i < kD; ++i) y[i] = half_to_float(t[(kHq + kHkv + h) * kD + i]);
                    check_codes(y, rows[j].v, "V of", j);
                }
                for (int r = 0; r < R; ++r)
                    for (int g = h * kG; g < (h + 1) * kG; ++g) {
                        const size_t i = (((size_t)b * R + r) * kHq + g) * kD;
                        rotated(&x[(b * R + r) * token + g * kD], at[b] + r, y);
                        for (int e = 0; e < kD; ++e)
                            EXPECT(std::abs(half_to_float(hq[i + e]) - y[e]) <= 1.01 * kU16 * std::abs(y[e]) + 1e-6,
                                   "%s: q of row %d", what, r);
                        check_attention(&hq[i], &ho[i], hl[((size_t)b * kHq + g) * R + r], !decode, rows, at[b] + r + 1,
                                        what);
                    }
            }
        // the idle slot's rows
        for (size_t i = (size_t)2 * R * kHq * kD; i < ho.size(); ++i) {
            const float o = half_to_float(ho[i]), p = half_to_float(hq[i]);
            EXPECT(p == 7.f && o == (decode ? 0.f : 7.f), "%s: the idle slot", what);
        }
    };
    cache.begin_prefill(kSlots, 70);
    step(70, false, "prompt");
    // another sequence takes the first one's prefix; both go on by a chunk
    cache.release(1);
    EXPECT(cache.add_sequence() == 1 && cache.share_prefix(1, 0, 40) == 32, "a shared prefix");
    text[1].assign(text[0].begin(), text[0].begin() + 32 * token);
    cache.begin_prefill(kSlots, 20);
    step(20, false, "chunk");
    for (int i = 0; i < 4; ++i) {
        cache.begin_decode_step(kSlots);
        step(1, true, "step");
    }
    // what is for fp16 pages refuses, before any work
    const half* none = nullptr;
    EXPECT(!refusal([&] { cache.get_layer_ptr(0, 0); }).empty(), "get_layer_ptr");
    EXPECT(!refusal([&] { cache.k_view(0); }).empty(), "k_view");
    EXPECT(!refusal([&] { cache.append(0, none, none, 1, 1); }).empty(), "append");
    EXPECT(!refusal([&] { cache.decode(0, none, nullptr, 1, kHq, 16); }).empty(), "decode");
    EXPECT(!refusal([&] { cache.append_decode(0, none, none, none, nullptr, 1, kHq, 16); }).empty(), "append_decode");
    EXPECT(!refusal([&] { cache.drop_hidden(0, 16, 0); }).empty(), "drop_hidden");
    EXPECT(!refusal([&] { cache.get_q4_layer_ptr(kLayers); }).empty(), "a layer past the last");
}

// The same append into fp16 pages, and the fp16 members next to it.
void case_half() {
    std::mt19937 rng(8);
    PagedKVCache cache(1, kHkv, kD, 8, 1, 8);
    EXPECT(cache.add_sequence() == 0 && cache.format() == PagedKVCache::Format::kHalf, "a cache of fp16");
    const int S = 37;
    auto x = random_half(rng, (size_t)S * kH * kD);
    cache.begin_prefill(1, S);
    cache.sync();
    auto dx = upload(x);
    DeviceBuffer<half> q((size_t)S * kHq * kD);
    const int token = kH * kD;
    cache.rope_append(0, dx.data(), dx.data() + kHq * kD, dx.data() + (kHq + kHkv) * kD, token, token, token, kTheta,
                      q.data(), 1, S, kHq);
    HIP_CHECK(hipDeviceSynchronize());
    const auto pk = download(cache.get_layer_ptr(0, 0), (size_t)kHkv * 8 * 16 * kD);
    const auto pv = download(cache.get_layer_ptr(0, 1), pk.size());
    double y[kD];
    for (int j = 0; j < S; ++j)
        for (int h = 0; h < kHkv; ++h) {
            const size_t at = (((size_t)h * 8 + cache.host_block_table(0)[j / 16]) * 16 + j % 16) * kD;
            const half* t = &x[(size_t)j * token];
            rotated(t + (kHq + h) * kD, j, y);
            for (int i = 0; i < kD; ++i) {
                EXPECT(std::abs(half_to_float(pk[at + i]) - y[i]) <= 1.01 * kU16 * std::abs(y[i]) + 1e-6, "K of %d", j);
                EXPECT(half_to_float(pv[at + i]) == half_to_float(t[(kHq + kHkv + h) * kD + i]), "V of %d", j);
            }
        }
    EXPECT(!refusal([&] { cache.get_q4_layer_ptr(0); }).empty(), "4-bit pages of a cache of fp16");
    EXPECT(!refusal([&] { cache.q4_decode(0, nullptr, nullptr, 1, kHq, 16, nullptr, 0); }).empty(), "q4_decode");
    EXPECT(!refusal([&] { cache.rope_append(1, nullptr, nullptr, nullptr, 0, 0, 0, 0.f, nullptr, 1, 1, kHq); }).empty(),
           "a layer past the last");
}

}  // namespace

int main(int argc, char** argv) {
    const bool gpu = argc > 1 && std::strcmp(argv[1], "--gpu") == 0;
    const bool cpu = argc > 1 && std::strcmp(argv[1], "--cpu") == 0;
    if (!gpu && !cpu) {
        std::fprintf(stderr, "usage: %s --cpu | --gpu\n", argv[0]);
        return 2;
    }
    struct {
        const char* name;
        bool gpu;
        void (*fn)();
    } cases[] = {{"refusals", false, case_refusals}, {"half", true, case_half}, {"served", true, case_served}};
    for (const auto& c : cases) {
        if (c.gpu && !gpu) continue;
        std::printf("case %s ...\n", c.name);
        std::fflush(stdout);
        try {
            c.fn();
        } catch (const std::exception& e) {
            ++g_failures;
            std::printf("  FAIL [%s] exception: %s\n", c.name, e.what());
        }
    }
    std::printf("%d checks, %d failures\n", g_checks, g_failures);
    return g_failures ? 1 : 0;
}
