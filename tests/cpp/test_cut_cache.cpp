// test_cut_cache.cpp -- PagedKVCache::rope_append into caches that were cut
// (serving-engine_amd/engine/kv_cache.h): slots fall behind the text's positions, to which
// q and k are rotated all the same, in fp16 and in 4 bits.
//
//   test_cut_cache --gpu
// Exit status 0 when every check passed.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <stdexcept>
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

constexpr int kHq = 4, kHkv = 2, kD = 64, kH = kHq + 2 * kHkv, kSlots = 3, kToken = kH * kD;
constexpr float kTheta = 10000.f;
constexpr double kU16 = 1.0 / 2048;
using Format = PagedKVCache::Format;

// A row rotated to `pos`.
void rotated(const half* x, int pos, double* y) {
    for (int i = 0; i < kD / 2; ++i) {
        const double a = pos * std::pow((double)kTheta, -2.0 * i / kD), c = std::cos(a), s = std::sin(a);
        const double u = half_to_float(x[i]), w = half_to_float(x[i + kD / 2]);
        y[i] = u * c - w * s;
        y[i + kD / 2] = w * c + u * s;
    }
}

// K of KV head h at a sequence's slot j, as the pool holds it.
void key_at(const PagedKVCache& cache, const std::vector<half>& pool, int slot, int h, int j, double* y) {
    const size_t page = (size_t)h * cache.num_pages() + cache.host_block_table(slot)[j / 16];
    if (cache.format() == Format::kHalf) {   // K's pool is the first half
        for (int i = 0; i < kD; ++i) y[i] = half_to_float(pool[(page * 16 + j % 16) * kD + i]);
        return;
    }
    const uint8_t* pg = reinterpret_cast<const uint8_t*>(pool.data()) + page * hip::q4_page_bytes(kD);
    half p[2];
    std::memcpy(p, pg + 16 * kD + 4 * (j % 16), 4);
    for (int i = 0; i < kD; ++i)
        y[i] = half_to_float(p[0]) * ((pg[j % 16 * (kD / 2) + i / 2] >> 4 * (i % 2) & 15) + half_to_float(p[1]));
}

class Served {
public:
    explicit Served(Format format) : cache(1, kHkv, kD, 40, kSlots, 12, format) {}

    // One step of R rows a slot; sequence b's first row has to stand at text position at[b]
    // (-1: an idle slot).
    void step(int R, bool decode, const std::vector<int>& at, const char* what) {
        decode ? cache.begin_decode_step(kSlots) : cache.begin_prefill(kSlots, R);
        cache.sync();
        std::uniform_real_distribution<float> dist(-1.f, 1.f);
        std::vector<half> x((size_t)kSlots * R * kToken);
        for (auto& e : x) e = float_to_half(dist(rng));
        DeviceBuffer<half> dx(x.size()), q((size_t)kSlots * R * kHq * kD);
        dx.copy_from_host(x.data(), x.size());
        std::vector<half> hq(q.size(), float_to_half(7.f));
        q.copy_from_host(hq.data(), hq.size());
        cache.rope_append(0, dx.data(), dx.data() + kHq * kD, dx.data() + (kHq + kHkv) * kD, kToken, kToken, kToken,
                          kTheta, q.data(), kSlots, R, kHq);
        HIP_CHECK(hipDeviceSynchronize());
        HIP_CHECK(hipMemcpy(hq.data(), q.data(), hq.size() * sizeof(half), hipMemcpyDeviceToHost));
        std::vector<half> pool(cache.pool_bytes() / sizeof(half));
        HIP_CHECK(hipMemcpy(pool.data(), cache.raw_data(), cache.pool_bytes(), hipMemcpyDeviceToHost));
        double want[kD], got[kD];
        for (int b = 0; b < kSlots; ++b)
            for (int r = 0; r < R; ++r) {
                const half* t = &x[((size_t)b * R + r) * kToken];
                for (int h = 0; h < kHq; ++h) {
                    const half* to = &hq[(((size_t)b * R + r) * kHq + h) * kD];
                    if (at[b] >= 0) rotated(t + h * kD, at[b] + r, want);
                    for (int i = 0; i < kD; ++i)
                        EXPECT(at[b] < 0 ? half_to_float(to[i]) == 7.f
                                         : std::abs(half_to_float(to[i]) - want[i]) <=
                                               1.01 * kU16 * std::abs(want[i]) + 1e-6,
                               "%s: q of sequence %d row %d", what, b, r);
                }
                if (at[b] < 0) continue;
                const int slot = cache.seq_len(b) - R + r;
                for (int h = 0; h < kHkv; ++h) {
                    rotated(t + (kHq + h) * kD, at[b] + r, want);
                    key_at(cache, pool, b, h, slot, got);
                    const double lo = *std::min_element(want, want + kD), hi = *std::max_element(want, want + kD);
                    // 4 bits: half a step, its rounding up to fp16, the offset's (2^-6 of a step at most)
                    const double q4 = cache.format() == Format::kQ4 ? (hi - lo) / 15 * 1.002 * (0.5 + 1.0 / 64) : 0;
                    for (int i = 0; i < kD; ++i)
                        EXPECT(std::abs(got[i] - want[i]) <= 2.02 * kU16 * std::max(-lo, hi) + q4 + 1e-6,
                               "%s: K of sequence %d slot %d is not at position %d", what, b, slot, at[b] + r);
                }
            }
    }

    PagedKVCache cache;

private:
    std::mt19937 rng{11};
};

void case_cut(Format format) {
    Served s(format);
    PagedKVCache& cache = s.cache;
    EXPECT(cache.add_sequence() == 0 && cache.add_sequence() == 1, "slots");   // the third stays idle
    s.step(60, false, {0, 0, -1}, "prompt");
    // an eviction kept 40 of the first one's tokens
    cache.shrink(0, 40);
    s.step(1, true, {60, 60, -1}, "step after the cut");
    EXPECT(cache.seq_len(0) == 41 && cache.seq_len(1) == 61, "lengths");
    s.step(5, false, {61, 61, -1}, "chunk after the cut");
    cache.shrink(0, 20);   // once more
    cache.shrink(1, cache.seq_len(1));   // nothing of this one
    s.step(3, false, {66, 66, -1}, "chunk after the second cut");
    // tokens taken back: the text is shorter by as many
    cache.set_seq_len(0, 21);
    s.step(1, true, {67, 69, -1}, "step after two tokens were taken back");
    // a sequence that takes the cut one's first page goes on behind it, as the cut one would
    EXPECT(cache.add_sequence() == 2 && cache.share_prefix(2, 0, 18) == 16, "a shared prefix");
    s.step(2, false, {68, 70, 62}, "a sharer");
    // a new sequence in the cut one's place begins a text of its own
    cache.release(0);
    EXPECT(cache.add_sequence() == 0, "the slot again");
    s.step(4, false, {0, 72, 64}, "a new sequence");
    cache.set_seq_len(1, 0);
    s.step(2, false, {4, 0, 68}, "a text begun anew");
}

void case_half() { case_cut(Format::kHalf); }
void case_q4() { case_cut(Format::kQ4); }

}  // namespace

int main(int argc, char** argv) {
    if (argc < 2 || std::strcmp(argv[1], "--gpu") != 0) {
        std::fprintf(stderr, "usage: %s --gpu\n", argv[0]);
        return 2;
    }
    struct {
        const char* name;
        void (*fn)();
    } cases[] = {{"fp16", case_half}, {"4 bits", case_q4}};
    for (const auto& c : cases) {
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
