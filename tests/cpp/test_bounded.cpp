// test_bounded.cpp -- the C++ API of the caches of bounded length
// (serving-engine_amd/engine/kernels.h, PagedKVCache::shrink, require_private and
// drop_hidden): a prompt with its weights, decode steps that add theirs, an
// eviction and steps over what it left, and windowed steps that give hidden
// pages away, through one PagedKVCache, against definitions in double.
//
//   test_bounded --cpu   refusals
//   test_bounded --gpu   every case
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
#include "kv_view.h"

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

constexpr int kB = 2, kHq = 8, kHkv = 2, kD = 64, kG = kHq / kHkv;

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
std::vector<T> download(const DeviceBuffer<T>& d) {
    std::vector<T> v(d.size());
    d.copy_to_host(v.data(), v.size());
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
    alignas(16) static float sums[64] = {};
    alignas(16) static int ints[64] = {};
    const hip::KVView flat{data, 0, 0, 8, 1};
    const hip::KVView paged = hip::paged_view(data, 4, kD, ints, 2);
    EXPECT(refusal([&] {
               hip::window_decode(data, flat, flat, ints, data, 1, 6, 4, kD, 16, 8, 0, nullptr, 0);
           }).find("num_q_heads") != std::string::npos, "window_decode took Hq = 6, Hkv = 4");
    EXPECT(!refusal([&] {
               hip::window_prefill(data, flat, flat, nullptr, nullptr, data, nullptr, 1, 4, kHq,
                                   kHkv, kD, 16, -1, 0, nullptr, 0);
           }).empty(), "window_prefill took window -1");
    EXPECT(!refusal([&] {
               hip::weighted_decode(data, flat, flat, ints, nullptr, data, sums, nullptr, 1, kHq,
                                    kHkv, kD, 16, 1, nullptr, 0);
           }).empty(), "weighted_decode took strided views");
    EXPECT(!refusal([&] {
               hip::prompt_weights(data, paged, nullptr, nullptr, ints, nullptr, sums, nullptr, 1,
                                   4, kHq, kHkv, kD, 16, 0, 0, 1, nullptr, 0);
           }).empty(), "prompt_weights took no lse");
    EXPECT(!refusal([&] {
               hip::evict_plan(sums, ints, ints, 2, ints, nullptr, ints + 8, ints + 4, ints + 6, 1,
                               kHkv, 4, 32, 8, 5, 4, 8);
           }).empty(), "evict_plan protected more slots than the budget");
    EXPECT(!refusal([&] {
               hip::evict_apply(data, data, sums, ints, ints, 2, ints + 1, ints, 1, kHkv, kD, 4, 8);
           }).empty(), "evict_apply took moves off their alignment");
    // nothing to do is done at once
    EXPECT(refusal([&] {
               hip::window_decode(data, flat, flat, ints, data, 0, kHq, kHkv, kD, 16, 8, 0,
                                  nullptr, 0);
           }).empty(), "an empty batch threw");
}

// The tokens of one KV head of one sequence, in slot order.
struct Head {
    std::vector<std::vector<double>> k, v;
    std::vector<double> sum, err;   // weight received, and the bound on its error
    std::vector<int> age;
};

// One row of one query head over the visible keys: its output, its bound, and
// (add) its weights into the sums.
void row(const half* q, Head& c, int p, int window, int sinks, bool add, double* out,
         double* spread) {
    const int n = (int)c.k.size();
    std::vector<double> s(n, -INFINITY);
    double m = -INFINITY, l = 0;
    for (int j = 0; j < n && j <= p; ++j) {
        if (window > 0 && j >= sinks && p - j >= window) continue;
        double dot = 0;
        for (int i = 0; i < kD; ++i) dot += (double)half_to_float(q[i]) * c.k[j][i];
        s[j] = dot / std::sqrt((double)kD);
        m = std::max(m, s[j]);
    }
    for (double& x : s) l += (x = std::exp(x - m));
    for (int i = 0; i < kD; ++i) out[i] = spread[i] = 0;
    for (int j = 0; j < n; ++j) {
        const double w = s[j] / l;
        for (int i = 0; i < kD; ++i) {
            out[i] += w * c.v[j][i];
            spread[i] += w * std::fabs(c.v[j][i]);
        }
        // Score: at most 64 terms of magnitude 1 over 8, D + 4 roundings of
        // 2^-24 of 8, in the weight and in the row's sum, and n + 16 roundings
        // of the sums themselves.
        if (add) {
            c.sum[j] += w;
            c.err[j] += w * (2 * (kD + 8) * 8 + 2 * (n + 16)) * std::ldexp(1.0, -24);
        }
    }
}

// Against got: the result's rounding to fp16 (2^-11 of it), the weights' (2^-11
// each, above and below the line), the scores' fp32 errors as above, and the
// absolute roundings of weights below fp16's normal range, at most 2^-25 for
// each of n keys with values up to 1, over a sum of at least 2^-8.
void check_row(const half* got, const double* want, const double* spread, int n, const char* what) {
    for (int i = 0; i < kD; ++i) {
        const double u = std::ldexp(1.0, -11);
        const double tol = u * std::fabs(want[i]) +
                           (2 * u + (2 * (kD + 8) * 8 + 2 * n) * std::ldexp(1.0, -24)) * spread[i] +
                           n * std::ldexp(1.0, -25) * 256 + std::ldexp(1.0, -25);
        EXPECT(std::fabs(half_to_float(got[i]) - want[i]) <= tol, "%s: got %g want %g tol %g", what,
               half_to_float(got[i]), want[i], tol);
    }
}

void case_served() {
    std::mt19937 rng(66);
    const int S = 70, steps = 3, budget = 48, sinks = 4, recent = 20;
    PagedKVCache cache(1, kHkv, kD, 16, kB, 8);
    EXPECT(cache.add_sequence() == 0 && cache.add_sequence() == 1, "slots");
    const int num_pages = cache.num_pages(), cap = cache.max_pages_per_seq() * PagedKVCache::kPage;
    DeviceBuffer<float> weights((size_t)kHkv * num_pages * 16);
    DeviceBuffer<int32_t> ages(weights.size());
    {   // what an earlier owner left
        std::vector<float> w(weights.size(), NAN);
        std::vector<int32_t> a(ages.size(), 12345);
        weights.copy_from_host(w.data(), w.size());
        ages.copy_from_host(a.data(), a.size());
    }
    Head head[kB][kHkv];
    std::vector<int> text(kB, 0);   // tokens of the text so far
    auto extend = [&](const std::vector<half>& k, const std::vector<half>& v, int T) {
        for (int b = 0; b < kB; ++b)
            for (int t = 0; t < T; ++t, ++text[b])
                for (int h = 0; h < kHkv; ++h) {
                    const size_t at = (((size_t)b * T + t) * kHkv + h) * kD;
                    std::vector<double> kr(kD), vr(kD);
                    for (int i = 0; i < kD; ++i) {
                        kr[i] = half_to_float(k[at + i]);
                        vr[i] = half_to_float(v[at + i]);
                    }
                    Head& c = head[b][h];
                    c.k.push_back(kr);
                    c.v.push_back(vr);
                    c.sum.push_back(0);
                    c.err.push_back(0);
                    c.age.push_back(text[b]);
                }
    };
    double want[kD], spread[kD];

    // the prompt: attention, and the weights of its last rows
    {
        auto q = random_half(rng, (size_t)kB * S * kHq * kD);
        auto k = random_half(rng, (size_t)kB * S * kHkv * kD);
        auto v = random_half(rng, k.size());
        cache.begin_prefill(kB, S);
        cache.sync();
        auto dq = upload(q), dk = upload(k), dv = upload(v);
        cache.append(0, dk.data(), dv.data(), kB, S);
        extend(k, v, S);
        DeviceBuffer<half> out(q.size());
        DeviceBuffer<float> lse((size_t)kB * kHq * S);
        const size_t nb = hip::window_prefill_workspace_bytes(kB, S, kHq, kHkv, kD, cap, 0, 0);
        const size_t nw = hip::prompt_weights_workspace_bytes(kB, S, kHq, kHkv, kD, cap);
        DeviceBuffer<char> ws(std::max(nb, nw));
        hip::window_prefill(dq.data(), cache.k_view(0), cache.v_view(0), nullptr, cache.seq_lens(),
                            out.data(), lse.data(), kB, S, kHq, kHkv, kD, cap, 0, 0, ws.data(), nb);
        hip::prompt_weights(dq.data(), cache.k_view(0), lse.data(), nullptr, cache.seq_lens(),
                            nullptr, weights.data(), ages.data(), kB, S, kHq, kHkv, kD, cap, 0, 0,
                            S, ws.data(), nw);
        HIP_CHECK(hipDeviceSynchronize());
        const auto got = download(out);
        for (int b = 0; b < kB; ++b)
            for (int r = 0; r < S; ++r)
                for (int h = 0; h < kHq; ++h) {
                    const size_t at = (((size_t)b * S + r) * kHq + h) * kD;
                    row(&q[at], head[b][h / kG], r, 0, 0, true, want, spread);
                    check_row(&got[at], want, spread, S, "prompt");
                }
    }
    auto check_sums = [&](const char* what) {
        const auto w = download(weights);
        const auto a = download(ages);
        for (int b = 0; b < kB; ++b)
            for (int h = 0; h < kHkv; ++h)
                for (size_t j = 0; j < head[b][h].k.size(); ++j) {
                    const size_t at = ((size_t)h * num_pages + cache.host_block_table(b)[j / 16]) * 16 + j % 16;
                    const Head& c = head[b][h];
                    EXPECT(std::fabs(w[at] - c.sum[j]) <= c.err[j] + 1e-30, "%s: sum of slot %zu", what, j);
                    EXPECT(a[at] == c.age[j], "%s: age of slot %zu: %d, not %d", what, j, a[at], c.age[j]);
                }
    };
    check_sums("prompt");

    auto step = [&](bool weighted, int window, int first, const char* what) {
        auto q = random_half(rng, (size_t)kB * kHq * kD);
        auto k = random_half(rng, (size_t)kB * kHkv * kD);
        auto v = random_half(rng, k.size());
        cache.begin_decode_step(kB);
        cache.sync();
        auto dq = upload(q), dk = upload(k), dv = upload(v);
        cache.append(0, dk.data(), dv.data(), kB, 1);
        auto newest = upload(text);
        extend(k, v, 1);
        DeviceBuffer<half> out(q.size());
        const size_t nb =
            weighted ? hip::weighted_decode_workspace_bytes(kB, kHq, kHkv, kD, cap)
                     : hip::window_decode_workspace_bytes(kB, kHq, kHkv, kD, cap, window, first);
        DeviceBuffer<char> ws(std::max(nb, (size_t)16));
        if (weighted)
            hip::weighted_decode(dq.data(), cache.k_view(0), cache.v_view(0), cache.seq_lens(),
                                 newest.data(), out.data(), weights.data(), ages.data(), kB, kHq,
                                 kHkv, kD, cap, 1, ws.data(), nb);
        else
            hip::window_decode(dq.data(), cache.k_view(0), cache.v_view(0), cache.seq_lens(),
                               out.data(), kB, kHq, kHkv, kD, cap, window, first, ws.data(), nb);
        HIP_CHECK(hipDeviceSynchronize());
        const auto got = download(out);
        for (int b = 0; b < kB; ++b)
            for (int h = 0; h < kHq; ++h) {
                Head& c = head[b][h / kG];
                const int n = (int)c.k.size();
                EXPECT(n == cache.seq_len(b), "%s: length", what);
                row(&q[((size_t)b * kHq + h) * kD], c, n - 1, window, first, weighted, want, spread);
                check_row(&got[((size_t)b * kHq + h) * kD], want, spread, n, what);
            }
    };
    for (int i = 0; i < steps; ++i) step(true, 0, 0, "weighted step");
    check_sums("steps");
    for (int b = 0; b < kB; ++b) cache.require_private(b);

    // the eviction, by the sums as the device holds them
    const int n = S + steps, used = cache.pages_used(0);
    auto newest = upload(std::vector<int>(kB, n - 1));
    const int max_moves = std::min(budget, cap - budget);
    DeviceBuffer<int32_t> moves((size_t)kB * kHkv * max_moves * 2), counts(kB * kHkv), new_lens(kB);
    hip::evict_plan(weights.data(), ages.data(), cache.block_tables(), cache.max_pages_per_seq(),
                    cache.seq_lens(), newest.data(), moves.data(), counts.data(), new_lens.data(),
                    kB, kHkv, num_pages, cap, budget, sinks, recent, max_moves);
    hip::evict_apply(cache.get_layer_ptr(0, 0), cache.get_layer_ptr(0, 1), weights.data(),
                     ages.data(), cache.block_tables(), cache.max_pages_per_seq(), moves.data(),
                     counts.data(), kB, kHkv, kD, num_pages, max_moves);
    const auto mv = download(moves);
    const auto cnt = download(counts);
    for (int b = 0; b < kB; ++b)
        for (int h = 0; h < kHkv; ++h) {
            Head& c = head[b][h];
            const int m = cnt[b * kHkv + h];
            EXPECT(m >= 0 && m <= max_moves, "count %d", m);
            std::vector<bool> kept(n, false);
            for (int j = 0; j < budget; ++j) kept[j] = true;
            int last_from = budget - 1, last_to = -1;
            for (int i = 0; i < m; ++i) {
                const int from = mv[((size_t)(b * kHkv + h) * max_moves + i) * 2];
                const int to = mv[((size_t)(b * kHkv + h) * max_moves + i) * 2 + 1];
                EXPECT(from > last_from && from < n && to > last_to && to < budget, "move %d -> %d", from, to);
                last_from = from;
                last_to = to;
                kept[from] = true;
                kept[to] = false;
            }
            // every slot kept for its weight has at least an evicted one's,
            // up to the bounds on both; the protected ones are all kept
            for (int j = 0; j < n; ++j) {
                const bool guard = c.age[j] < sinks || c.age[j] > n - 1 - recent;
                EXPECT(!guard || kept[j], "slot %d was protected", j);
                for (int i = 0; i < n; ++i)
                    if (kept[j] && !guard && !kept[i])
                        EXPECT(c.sum[j] + c.err[j] >= c.sum[i] - c.err[i], "kept %d, not %d", j, i);
            }
            for (int i = 0; i < m; ++i) {
                const int from = mv[((size_t)(b * kHkv + h) * max_moves + i) * 2];
                const int to = mv[((size_t)(b * kHkv + h) * max_moves + i) * 2 + 1];
                c.k[to] = c.k[from];
                c.v[to] = c.v[from];
                c.sum[to] = c.sum[from];
                c.err[to] = c.err[from];
                c.age[to] = c.age[from];
            }
            c.k.resize(budget);
            c.v.resize(budget);
            c.sum.resize(budget);
            c.err.resize(budget);
            c.age.resize(budget);
        }
    for (int x : download(new_lens)) EXPECT(x == budget, "new length %d", x);
    const int free_before = cache.free_page_count();
    for (int b = 0; b < kB; ++b) cache.shrink(b, budget);
    EXPECT(cache.pages_used(0) == budget / 16 && cache.seq_len(0) == budget &&
               cache.free_page_count() == free_before + kB * (used - budget / 16),
           "pages after shrink");
    EXPECT(cache.host_block_table(0)[budget / 16] == -1, "a page given back is still named");
    check_sums("cut");
    step(true, 0, 0, "step over the cut cache");
    step(false, 20, 4, "windowed step over the cut cache");
    step(true, 0, 0, "another step");
}

// What an eviction must not write into is refused before one is enqueued.
void case_private() {
    PagedKVCache cache(1, 1, 8, 8, 3, 4);
    const int a = cache.add_sequence(), b = cache.add_sequence();
    cache.require_private(a);   // nothing held
    cache.set_seq_len(a, 40);
    cache.require_private(a);
    cache.share_prefix(b, a, 16);
    EXPECT(refusal([&] { cache.require_private(a); }).find("slot 0 shares") != std::string::npos,
           "a page lent");
    EXPECT(refusal([&] { cache.require_private(b); }).find("slot 1 shares") != std::string::npos,
           "a page borrowed");
    EXPECT(!refusal([&] { cache.require_private(3); }).empty(), "no such slot");
    EXPECT(!refusal([&] { cache.require_private(-1); }).empty(), "no such slot");
    cache.release(b);
    cache.require_private(a);
}

void case_drop_hidden() {
    PagedKVCache cache(1, 1, 8, 12, 3, 8);
    const int a = cache.add_sequence(), b = cache.add_sequence();
    EXPECT(cache.drop_hidden(a, 5, 0) == 0, "nothing held");
    cache.set_seq_len(a, 100);   // pages 0 .. 6
    EXPECT(!refusal([&] { cache.drop_hidden(a, 0, 4); }).empty(), "no window");
    EXPECT(!refusal([&] { cache.drop_hidden(a, 10, -1); }).empty(), "negative first tokens");
    EXPECT(!refusal([&] { cache.drop_hidden(3, 10, 4); }).empty(), "no such slot");
    EXPECT(cache.drop_hidden(a, INT32_MAX, 0) == 0 && cache.drop_hidden(a, 10, INT32_MAX) == 0 &&
               cache.drop_hidden(a, 85, 0) == 0 && cache.drop_hidden(a, 20, 80) == 0,
           "no page is hidden");
    cache.share_prefix(b, a, 48);
    // position 99 sees keys 60 .. 99 and 0 .. 16: page 2 is hidden
    EXPECT(cache.drop_hidden(a, 40, 17) == 1 && cache.host_block_table(a)[2] == -1 &&
               cache.host_block_table(a)[1] >= 0 && cache.host_block_table(a)[3] >= 0,
           "page 2 alone");
    EXPECT(cache.page_refs(cache.host_block_table(b)[2]) == 1 && cache.free_page_count() == 5,
           "the other sequence's page");
    EXPECT(cache.drop_hidden(a, 40, 17) == 0 && cache.drop_hidden(a, 36, 17) == 1 &&
               cache.free_page_count() == 6, "page 3 too, keys 48 .. 63");
    EXPECT(!refusal([&] { cache.require_private(a); }).empty() &&
               !refusal([&] { cache.shrink(a, 20); }).empty(), "an eviction needs every page");
    EXPECT(!refusal([&] { cache.set_seq_len(a, 99); }).empty(), "shorter");
    const int c = cache.add_sequence();
    EXPECT(!refusal([&] { cache.share_prefix(c, a, 48); }).empty() && cache.pages_used(c) == 0 &&
               cache.free_page_count() == 6, "a prefix with pages missing");
    EXPECT(cache.share_prefix(c, a, 32) == 32, "one without");
    cache.release(c);
    EXPECT(cache.cached_tokens(b) == 48 && cache.drop_hidden(b, 1, 1) == 1 &&
               cache.cached_tokens(b) == 16, "cached tokens end in front of the first page given up");
    cache.set_seq_len(a, 112);
    cache.sync();
    cache.release(b);
    cache.begin_decode_step(2);
    EXPECT(cache.seq_len(a) == 113 && cache.pages_used(a) == 8, "the sequence goes on");
    cache.release(a);
    EXPECT(cache.free_page_count() == 12, "every page came back once");
}

// Windowed steps over a cache that keeps the window's pages and the first tokens' only; what
// was given up goes to another sequence, which fills it with NaN.
void case_windowed() {
    std::mt19937 rng(5);
    const int S = 90, steps = 60, window = 37, sinks = 4;
    // two sequences of at most 1 + 4 pages, one of which grows before the other is cut
    PagedKVCache cache(1, kHkv, kD, 14, kB + 1, 12);
    EXPECT(cache.add_sequence() == 0 && cache.add_sequence() == 1, "slots");
    Head head[kB][kHkv];
    const int cap = cache.max_pages_per_seq() * PagedKVCache::kPage;
    auto extend = [&](const std::vector<half>& k, const std::vector<half>& v) {
        for (int b = 0; b < kB; ++b)
            for (int h = 0; h < kHkv; ++h) {
                const size_t at = ((size_t)b * kHkv + h) * kD;
                std::vector<double> kr(kD), vr(kD);
                for (int i = 0; i < kD; ++i) {
                    kr[i] = half_to_float(k[at + i]);
                    vr[i] = half_to_float(v[at + i]);
                }
                head[b][h].k.push_back(kr);
                head[b][h].v.push_back(vr);
            }
    };
    DeviceBuffer<char> ws(std::max<size_t>(
        hip::window_decode_workspace_bytes(kB, kHq, kHkv, kD, cap, window, sinks), 16));
    double want[kD], spread[kD];
    for (int t = 0; t < S + steps; ++t) {
        auto q = random_half(rng, (size_t)kB * kHq * kD);
        auto k = random_half(rng, (size_t)kB * kHkv * kD);
        auto v = random_half(rng, k.size());
        cache.begin_decode_step(kB);
        if (t % 5 == 4)
            for (int b = 0; b < kB; ++b) cache.drop_hidden(b, window, sinks);
        cache.sync();
        auto dq = upload(q), dk = upload(k), dv = upload(v);
        cache.append(0, dk.data(), dv.data(), kB, 1);
        extend(k, v);
        DeviceBuffer<half> out(q.size());
        hip::window_decode(dq.data(), cache.k_view(0), cache.v_view(0), cache.seq_lens(), out.data(),
                           kB, kHq, kHkv, kD, cap, window, sinks, ws.data(), ws.size());
        HIP_CHECK(hipDeviceSynchronize());
        if (t < S) continue;
        const auto got = download(out);
        for (int b = 0; b < kB; ++b)
            for (int h = 0; h < kHq; ++h) {
                row(&q[((size_t)b * kHq + h) * kD], head[b][h / kG], t, window, sinks, false, want, spread);
                check_row(&got[((size_t)b * kHq + h) * kD], want, spread, window + sinks, "windowed step");
            }
        if (t % 20 == 0) {   // the pages given up, as their next owner leaves them
            const int c = cache.add_sequence(), n = cache.free_page_count() * PagedKVCache::kPage;
            cache.reserve(c, n);
            std::vector<half> nan((size_t)n * kHkv * kD, float_to_half(NAN));
            auto dn = upload(nan);
            DeviceBuffer<int32_t> table = upload(std::vector<int32_t>(
                cache.host_block_table(c), cache.host_block_table(c) + cache.pages_used(c)));
            auto zero = upload(std::vector<int32_t>(1, 0));
            hip::paged_append_kv(dn.data(), dn.data(), cache.get_layer_ptr(0, 0),
                                 cache.get_layer_ptr(0, 1), table.data(), cache.pages_used(c),
                                 zero.data(), 1, n, kHkv, kD, cache.num_pages());
            HIP_CHECK(hipDeviceSynchronize());
            cache.release(c);
        }
    }
    EXPECT(cache.free_page_count() >= 14 - kB * 5, "pages held: %d", 14 - cache.free_page_count());
}

void case_shrink() {
    PagedKVCache cache(1, 1, 8, 8, 2, 4);
    const int a = cache.add_sequence(), b = cache.add_sequence();
    cache.set_seq_len(a, 40);
    EXPECT(cache.pages_used(a) == 3 && cache.free_page_count() == 5, "three pages");
    EXPECT(!refusal([&] { cache.shrink(a, 41); }).empty(), "longer than it is");
    EXPECT(!refusal([&] { cache.shrink(a, -1); }).empty(), "a negative length");
    EXPECT(!refusal([&] { cache.shrink(2, 0); }).empty(), "no such slot");
    EXPECT(cache.seq_len(a) == 40 && cache.pages_used(a) == 3, "a refusal changed the sequence");
    cache.share_prefix(b, a, 32);
    EXPECT(!refusal([&] { cache.shrink(a, 8); }).empty(), "its pages are shared");
    EXPECT(!refusal([&] { cache.shrink(b, 8); }).empty(), "its pages are another's");
    EXPECT(cache.free_page_count() == 5 && cache.page_refs(cache.host_block_table(a)[0]) == 2,
           "a refusal changed the pages");
    cache.release(b);
    cache.shrink(a, 17);
    EXPECT(cache.pages_used(a) == 2 && cache.seq_len(a) == 17 && cache.free_page_count() == 6, "cut to 17");
    cache.shrink(a, 16);
    EXPECT(cache.pages_used(a) == 1 && cache.free_page_count() == 7, "cut to 16");
    cache.reserve(a, 64);   // pages ahead of the text go too
    cache.shrink(a, 16);
    EXPECT(cache.pages_used(a) == 1 && cache.free_page_count() == 7, "reserved pages");
    cache.shrink(a, 0);
    EXPECT(cache.pages_used(a) == 0 && cache.free_page_count() == 8, "cut to nothing");
    cache.begin_decode_step(2);
    EXPECT(cache.seq_len(a) == 1 && cache.pages_used(a) == 1, "goes on from there");
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
    } cases[] = {{"refusals", false, case_refusals},
                 {"private", true, case_private},
                 {"drop_hidden", true, case_drop_hidden},
                 {"windowed", true, case_windowed},
                 {"shrink", true, case_shrink},
                 {"served", true, case_served}};
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
