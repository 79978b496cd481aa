// rope_append.hip -- rows of q, k and v as the projections leave them: q and k rotated to
// their place in the text, K and V written into the cache's pages, fp16 or 4 bits.
//
// The rotation's angle is counted in turns in 64 bits, p theta^(-2i/D) / 2 pi, and its sine
// and cosine are rounded to fp32 once, so that far positions lose nothing: in fp32 the angle
// itself is off by up to 2^-11 at position 2^13 and 2^-10 at 2^14, more than fp16 rounds.
//
// head_dim 64 and 128, 16-byte aligned tensors: a workgroup takes 1 to 16 tokens and some of
// their heads, computes the tokens' rotations once, into LDS, and moves rows by 16-byte chunks,
// a lane both halves' chunks of 8 pairs, two rows' loads in flight.  In 4 bits the 4 or 8
// lanes of a row find its range among themselves and write a word of codes per chunk.
// 8192 tokens of 32/8 heads of 128: 43.3 us, 201 MB at 4.65 TB/s, where a copy of 1 GiB reaches
// 5.04; into 4 bits 41.3 (177 MB).  The same with the rotation computed per row took 134 and
// 163: 64-bit sines and cosines, 40 times a token instead of once.  A step's tokens are bound by
// their dependent waits: 32 of them 4.0 us, one 2.2.
// Other shapes: one wave per token and up to 8 of its heads, a lane per pair of dims (2048 tokens of 32/8
// heads of 96: 19.2 us; a head a wave, each with its own rotation, 38).
#include "q4.h"

#include <algorithm>
#include <type_traits>

namespace kvhp {
namespace {

constexpr int kMostVecTokens = 1 << 27;   // 16 tokens a workgroup, 2^31 threads along a grid's axis

struct AppendArgs {
    const f16 *q, *k, *v;
    int64_t sq, sk, sv;       // between tokens
    const int32_t* positions; // NULL: 0
    const int32_t* slots;     // NULL: the positions
    const int32_t* seq_lens;  // NULL: no limit
    f16* q_out;
    f16 *pool_k, *pool_v;     // fp16 pages, or
    uint8_t* pool;            // 4-bit pages
    const int32_t* bt;
    int max_pages, num_pages;
    int batch, rows, Hq, Hkv, D;   // Hq 0: no q
    double log2_theta;        // theta > 0
    int rotate;
};

// cos and sin of position p times theta^(-2i/D), each rounded once to fp32.  The turns are
// reduced to an eighth in 64 bits; there the Taylor series to x^13 and x^14 leave 2^-46.
__device__ __forceinline__ float2 rotation(int64_t p, int i, int D, double log2_theta) {
    const double freq = exp2(-log2_theta * (2 * i) / D);
    double t = static_cast<double>(p) * (freq * 0.15915494309189533577);   // 1 / 2 pi
    t -= rint(t);
    const double k = rint(4 * t);
    const double x = (t - 0.25 * k) * 6.283185307179586477;
    const double y = x * x;
    double s = 1.0 / 6227020800, c = -1.0 / 87178291200;
    s = fma(s, y, -1.0 / 39916800);
    c = fma(c, y, 1.0 / 479001600);
    s = fma(s, y, 1.0 / 362880);
    c = fma(c, y, -1.0 / 3628800);
    s = fma(s, y, -1.0 / 5040);
    c = fma(c, y, 1.0 / 40320);
    s = fma(s, y, 1.0 / 120);
    c = fma(c, y, -1.0 / 720);
    s = fma(s, y, -1.0 / 6);
    c = fma(c, y, 1.0 / 24);
    s = fma(s * y, x, x);
    c = fma(c, y, -0.5);
    c = fma(c, y, 1.0);
    const int quarter = static_cast<int>(k) & 3;   // k in -2 .. 2
    const float fs = static_cast<float>(quarter & 1 ? c : s);
    const float fc = static_cast<float>(quarter & 1 ? s : c);
    return float2{quarter == 1 || quarter == 2 ? -fc : fc, quarter >= 2 ? -fs : fs};
}

// The rotation's two products and their sum are rounded to fp32 one after the other (no fused
// multiply-add, whose choice would be the compiler's, kernel by kernel), the result once to fp16.
__device__ __forceinline__ void rotate(float a, float b, float2 cs, f16& x, f16& y) {
#pragma clang fp contract(off)
    const float ac = a * cs.x, bs = b * cs.y, bc = b * cs.x, as = a * cs.y;
    const float u = ac - bs, v = bc + as;
    x = static_cast<f16>(u);
    y = static_cast<f16>(v);
}

// One wave per token and `per` of its heads, whose rotation it computes once; the next head's row is on
// its way meanwhile.
template <bool Q4>
__global__ void __launch_bounds__(kWave) append_row_kernel(const AppendArgs a, int per) {
    const int lane = threadIdx.x, D = a.D, half = D / 2;
    const int H = a.Hq + 2 * a.Hkv, parts = (H + per - 1) / per;
    const int64_t token = blockIdx.x / parts;
    const int h0 = static_cast<int>(blockIdx.x % parts) * per, h1 = min(h0 + per, H);
    const int b = static_cast<int>(token / a.rows), row = static_cast<int>(token % a.rows);
    const int64_t pos = (a.positions ? a.positions[b] : 0) + (int64_t)row;
    const int64_t slot = a.slots ? a.slots[b] + (int64_t)row : pos;
    if (slot < 0 || (a.seq_lens && slot >= a.seq_lens[b])) return;
    int pid = -1;   // -1: K and V are dropped
    if (h1 > a.Hq && slot < (int64_t)a.max_pages * kPage) {
        pid = a.bt[(int64_t)b * a.max_pages + (slot >> 4)];
        if (pid >= a.num_pages) pid = -1;
    }
    const int o = static_cast<int>(slot & 15);
    f16 next[2][2] = {};   // pairs lane, lane + 64: dims i, i + half
    auto load = [&](int h) {
        const f16* src = h < a.Hq ? a.q + token * a.sq + (int64_t)h * D
                         : h < a.Hq + a.Hkv ? a.k + token * a.sk + (int64_t)(h - a.Hq) * D
                                            : a.v + token * a.sv + (int64_t)(h - a.Hq - a.Hkv) * D;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = lane + kWave * u;
            if (i >= half) continue;
            next[u][0] = src[i];
            next[u][1] = src[i + half];
        }
    };
    load(h0);
    float2 cs[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        cs[u] = float2{1.f, 0.f};
        if (a.rotate && h0 < a.Hq + a.Hkv && lane + kWave * u < half)
            cs[u] = rotation(pos, lane + kWave * u, D, a.log2_theta);
    }
    for (int h = h0; h < h1; ++h) {
        const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
        const int kvh = is_v ? h - a.Hq - a.Hkv : h - a.Hq;
        f16 x[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            x[u][0] = next[u][0];
            x[u][1] = next[u][1];
        }
        if (h + 1 < h1) load(h + 1);
        if (!is_q && pid < 0) continue;
        if (a.rotate && !is_v)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                rotate(static_cast<float>(x[u][0]), static_cast<float>(x[u][1]), cs[u], x[u][0], x[u][1]);
        if (is_q || !Q4) {
            f16* dst = is_q ? a.q_out + (token * a.Hq + h) * D
                            : (is_v ? a.pool_v : a.pool_k) +
                                  (((int64_t)kvh * a.num_pages + pid) * kPage + o) * D;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int i = lane + kWave * u;
                if (i >= half) continue;
                dst[i] = x[u][0];
                dst[i + half] = x[u][1];
            }
            continue;
        }
        float lo = INFINITY, hi = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int u = 0; u < 2; ++u)
            if (lane + kWave * u < half)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float f = static_cast<float>(x[u][e]);
                    lo = fminf(lo, f);
                    hi = fmaxf(hi, f);
                    bad |= !(fabsf(f) < INFINITY);
                }
        lo = -wave_max(-lo);
        hi = wave_max(hi);
        bad = __ballot(bad) != 0;
        Q4Quant z = q4_quant(bad ? 0.f : lo, bad ? 0.f : hi);
        if (bad) z.bits = kQ4NanRow;
        uint8_t* pg = a.pool + ((int64_t)kvh * a.num_pages + pid) * q4_page_bytes(D);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = lane + kWave * u;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const uint32_t n = bad || z.flat ? 0 : q4_code(z, static_cast<float>(x[u][e]));
                const uint32_t odd = __shfl_down(n, 1);   // half is even: the pair's other dim
                if (i < half && !(i & 1))
                    pg[q4_codes_at(D, is_v, o) + (i + e * half) / 2] = static_cast<uint8_t>(n | odd << 4);
            }
        }
        if (lane == 0) *reinterpret_cast<uint32_t*>(pg + q4_params_at(D, is_v, o)) = z.bits;
    }
}

// The same by 16-byte chunks, D = 64 and 128.  Grid (groups of TB tokens, pieces of HP heads).
template <int D, bool Q4>
__global__ void __launch_bounds__(256) append_vec_kernel(const AppendArgs a, int TB, int HP, uint32_t inv_hp) {
    constexpr int half = D / 2, CPH = half / 8, RPI = 256 / CPH, U = 2, kMostTokens = 16;
    __shared__ float2 cs[kMostTokens * half];
    __shared__ int slot_of[kMostTokens], pid_of[kMostTokens];   // slot -1: padding; page -1: dropped
    const int tid = threadIdx.x, H = a.Hq + 2 * a.Hkv;
    const int64_t token0 = (int64_t)blockIdx.x * TB;
    const int nt = static_cast<int>(min((int64_t)TB, (int64_t)a.batch * a.rows - token0));
    const int h0 = blockIdx.y * HP, nh = min(HP, H - h0);
    const int nrows = nt * HP, c = tid % CPH;
    half8 x[U], y[U];
    auto head_of = [&](int rr, int& tt) {
        tt = inv_hp ? static_cast<int>(__umulhi(static_cast<uint32_t>(rr), inv_hp)) : rr;
        return h0 + rr - tt * HP;
    };
    auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int rr = base + RPI * u + tid / CPH;
            int tt;
            const int h = head_of(rr, tt);
            if (rr >= nrows || h >= h0 + nh) continue;
            const int64_t token = token0 + tt;
            const f16* src = h < a.Hq ? a.q + token * a.sq + (int64_t)h * D
                             : h < a.Hq + a.Hkv ? a.k + token * a.sk + (int64_t)(h - a.Hq) * D
                                                : a.v + token * a.sv + (int64_t)(h - a.Hq - a.Hkv) * D;
            x[u] = load_half8(src + 8 * c);
            y[u] = load_half8(src + half + 8 * c);
        }
    };
    load(0);
    // where the tokens go, by the last wave; their rotations meanwhile, by the first ones at least
    if (tid >= 256 - kMostTokens && tid - (256 - kMostTokens) < nt) {
        const int t = tid - (256 - kMostTokens);
        const uint32_t token = static_cast<uint32_t>(token0) + t, b = token / a.rows;   // tokens fit an int
        const int64_t row = token - b * a.rows;
        const int64_t slot = (a.slots ? a.slots[b] : a.positions ? a.positions[b] : 0) + row;
        const bool live = slot >= 0 && !(a.seq_lens && slot >= a.seq_lens[b]);
        int pid = -1;
        if (live && slot < (int64_t)a.max_pages * kPage) {
            pid = a.bt[(int64_t)b * a.max_pages + (slot >> 4)];
            if (pid >= a.num_pages) pid = -1;
        }
        slot_of[t] = live ? static_cast<int>(slot & 15) : -1;
        pid_of[t] = pid;
    }
    if (a.rotate)
        for (int i = tid; i < nt * half; i += 256) {
            const uint32_t token = static_cast<uint32_t>(token0) + i / half, b = token / a.rows;
            const int64_t pos = (a.positions ? a.positions[b] : 0) + static_cast<int64_t>(token - b * a.rows);
            cs[i] = rotation(pos, i % half, D, a.log2_theta);
        }
    __syncthreads();
    for (int base = 0; base < nrows; base += U * RPI) {
        if (base > 0) load(base);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int rr = base + RPI * u + tid / CPH;
            int tt;
            const int h = head_of(rr, tt);
            // the lanes of a row all go on or none
            if (rr >= nrows || h >= h0 + nh || slot_of[tt] < 0) continue;
            const int64_t token = token0 + tt;
            const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
            half8 lo8 = x[u], hi8 = y[u];
            if (a.rotate && !is_v) {
                const float2* r = cs + tt * half + 8 * c;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f16 f, g;
                    rotate(static_cast<float>(x[u][e]), static_cast<float>(y[u][e]), r[e], f, g);
                    lo8[e] = f;
                    hi8[e] = g;
                }
            }
            if (is_q) {
                f16* dst = a.q_out + (token * a.Hq + h) * D + 8 * c;
                store_half8(dst, lo8);
                store_half8(dst + half, hi8);
                continue;
            }
            const int kvh = is_v ? h - a.Hq - a.Hkv : h - a.Hq, pid = pid_of[tt], o = slot_of[tt];
            if (pid < 0) continue;
            const int64_t page = (int64_t)kvh * a.num_pages + pid;
            if constexpr (!Q4) {
                f16* dst = (is_v ? a.pool_v : a.pool_k) + (page * kPage + o) * D + 8 * c;
                store_half8(dst, lo8);
                store_half8(dst + half, hi8);
            } else {
                float lo = INFINITY, hi = -INFINITY;
                uint32_t bad = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float f = static_cast<float>(lo8[e]), g = static_cast<float>(hi8[e]);
                    lo = fminf(lo, fminf(f, g));
                    hi = fmaxf(hi, fmaxf(f, g));
                    bad |= fabsf(f) < INFINITY && fabsf(g) < INFINITY ? 0u : 1u;
                }
                auto across = [&](auto ctrl) {
                    constexpr int CTRL = decltype(ctrl)::value;
                    lo = fminf(lo, dpp_f32<CTRL>(lo));
                    hi = fmaxf(hi, dpp_f32<CTRL>(hi));
                    bad |= __float_as_uint(dpp_f32<CTRL>(__uint_as_float(bad)));
                };
                across(std::integral_constant<int, 0xB1>{});
                across(std::integral_constant<int, 0x4E>{});
                if constexpr (CPH == 8) across(std::integral_constant<int, 0x141>{});
                Q4Quant z = q4_quant(bad ? 0.f : lo, bad ? 0.f : hi);
                if (bad) z.bits = kQ4NanRow;
                uint32_t n0 = 0, n1 = 0;
                if (!bad && !z.flat) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        n0 |= q4_code(z, static_cast<float>(lo8[e])) << 4 * e;
                        n1 |= q4_code(z, static_cast<float>(hi8[e])) << 4 * e;
                    }
                }
                uint8_t* pg = a.pool + page * q4_page_bytes(D);
                uint8_t* codes = pg + q4_codes_at(D, is_v, o) + 4 * c;
                *reinterpret_cast<uint32_t*>(codes) = n0;
                *reinterpret_cast<uint32_t*>(codes + D / 4) = n1;
                if (c == 0) *reinterpret_cast<uint32_t*>(pg + q4_params_at(D, is_v, o)) = z.bits;
            }
        }
    }
}

int append(AppendArgs& a, const char* what, bool q4, int batch, int rows, int hq, int hkv, int d,
           float theta, hipStream_t s) {
    KVHP_REQUIRE(a.k && a.v && a.bt && (q4 ? a.pool != nullptr : a.pool_k && a.pool_v) &&
                     (a.q == nullptr) == (a.q_out == nullptr),
                 KVHP_ERR_INVALID, "%s: null pointer", what);
    KVHP_REQUIRE(a.max_pages > 0 && a.num_pages > 0, KVHP_ERR_INVALID,
                 "%s: max_pages=%d and num_pages=%d must be positive", what, a.max_pages,
                 a.num_pages);
    KVHP_REQUIRE(hkv > 0 && (hq > 0 || !a.q), KVHP_ERR_INVALID,
                 "%s: num_q_heads=%d and num_kv_heads=%d must be positive", what, hq, hkv);
    KVHP_REQUIRE(theta >= 0.f && theta < INFINITY, KVHP_ERR_INVALID,
                 "%s: rope_theta=%g must be 0 (no rotation) or positive", what, (double)theta);
    if (q4)
        KVHP_REQUIRE(d > 0 && d <= 256 && d % 8 == 0, KVHP_ERR_UNSUPPORTED,
                     "%s: head_dim=%d is no multiple of 8 up to 256", what, d);
    else
        KVHP_REQUIRE(d > 0 && d <= 256 && d % 2 == 0, KVHP_ERR_UNSUPPORTED,
                     "%s: head_dim=%d is no even number up to 256", what, d);
    KVHP_REQUIRE(!q4 || aligned16(a.pool), KVHP_ERR_INVALID, "%s: pool not 16-byte aligned", what);
    a.Hq = a.q ? hq : 0;
    a.Hkv = hkv;
    a.D = d;
    a.batch = batch;
    a.rows = rows;
    KVHP_REQUIRE(hkv <= kMaxKvHeads && a.Hq <= kMaxHeads, KVHP_ERR_UNSUPPORTED,
                 "%s: %d query heads, %d KV heads", what, a.Hq, hkv);
    KVHP_REQUIRE((!a.q || a.sq >= (int64_t)hq * d) && a.sk >= (int64_t)hkv * d &&
                     a.sv >= (int64_t)hkv * d,
                 KVHP_ERR_INVALID, "%s: a token's rows overlap the next one's", what);
    a.rotate = theta > 0.f;
    a.log2_theta = a.rotate ? std::log2(static_cast<double>(theta)) : 0.0;
    const int64_t tokens = (int64_t)batch * rows;
    const int H = a.Hq + 2 * hkv;
    auto whole = [](const void* x, int64_t stride) { return !x || (aligned16(x) && stride % 8 == 0); };
    if ((d == 64 || d == 128) && tokens <= kMostVecTokens && H <= 1 << 14 && whole(a.q, a.sq) &&
        whole(a.k, a.sk) && whole(a.v, a.sv) && aligned16(a.q_out) && aligned16(a.pool_k) &&
        aligned16(a.pool_v)) {
        // (16 H rows of a workgroup, part by part: __umulhi is exact to 2^32 of row x heads.)
        // Four workgroups a CU where there are tokens for them, of up to 16 tokens (a page); fewer
        // where a workgroup's threads would not have a row each; where tokens are few, the heads of
        // one are parted too.  (8192 tokens of 32/8 heads of 128: two a CU 52.4 us, four 44.2,
        // eight 44.5; 3108 of 14/2 heads of 64: 4 tokens 5.4, 2 6.3, 1 7.9.)
        const int per = 256 / (d / 16);   // rows of a workgroup at once
        int TB = 1;
        while (TB < 16 && (tokens >= 2 * TB * 1024 || (H * TB < per && tokens >= 2 * TB * 256))) TB *= 2;
        const int64_t groups = (tokens + TB - 1) / TB;
        const int64_t most = ((int64_t)H * TB + per - 1) / per;
        const int64_t pieces = std::max<int64_t>(1, std::min<int64_t>(most, 512 / groups));
        const int HP = static_cast<int>((H + pieces - 1) / pieces);
        const uint32_t inv = HP == 1 ? 0 : static_cast<uint32_t>(((uint64_t(1) << 32) + HP - 1) / HP);
        const dim3 grid(static_cast<unsigned>(groups), (H + HP - 1) / HP);
        if (d == 64 && q4)
            hipLaunchKernelGGL((append_vec_kernel<64, true>), grid, dim3(256), 0, s, a, TB, HP, inv);
        else if (d == 64)
            hipLaunchKernelGGL((append_vec_kernel<64, false>), grid, dim3(256), 0, s, a, TB, HP, inv);
        else if (q4)
            hipLaunchKernelGGL((append_vec_kernel<128, true>), grid, dim3(256), 0, s, a, TB, HP, inv);
        else
            hipLaunchKernelGGL((append_vec_kernel<128, false>), grid, dim3(256), 0, s, a, TB, HP, inv);
        return check_launch(what);
    }
    KVHP_REQUIRE(tokens <= 1 << 25 && tokens * H <= 1 << 25, KVHP_ERR_UNSUPPORTED,
                 "%s: %d x %d rows of %d heads", what, batch, rows, H);
    int per = 1;   // heads of a wave, once there are some 8 waves a SIMD
    while (per < 8 && tokens * H >= 16384 * per) per *= 2;
    const dim3 grid(static_cast<unsigned>(tokens * ((H + per - 1) / per)));
    if (q4)
        hipLaunchKernelGGL(append_row_kernel<true>, grid, dim3(kWave), 0, s, a, per);
    else
        hipLaunchKernelGGL(append_row_kernel<false>, grid, dim3(kWave), 0, s, a, per);
    return check_launch(what);
}

}  // namespace
}  // namespace kvhp

using namespace kvhp;

extern "C" int kvhp_rope_append(const void* q, const void* k, const void* v, int64_t q_stride,
                                int64_t k_stride, int64_t v_stride, const int32_t* positions,
                                const int32_t* slots, const int32_t* seq_lens, float rope_theta,
                                void* q_out, void* pool_k, void* pool_v,
                                const int32_t* block_tables, int max_pages, int num_pages,
                                int batch, int rows, int num_q_heads, int num_kv_heads,
                                int head_dim, void* stream) {
    clear_error();
    if (batch <= 0 || rows <= 0) return KVHP_OK;
    AppendArgs a{};
    a.q = static_cast<const f16*>(q);
    a.k = static_cast<const f16*>(k);
    a.v = static_cast<const f16*>(v);
    a.sq = q_stride;
    a.sk = k_stride;
    a.sv = v_stride;
    a.positions = positions;
    a.slots = slots;
    a.seq_lens = seq_lens;
    a.q_out = static_cast<f16*>(q_out);
    a.pool_k = static_cast<f16*>(pool_k);
    a.pool_v = static_cast<f16*>(pool_v);
    a.bt = block_tables;
    a.max_pages = max_pages;
    a.num_pages = num_pages;
    return append(a, "rope_append", false, batch, rows, num_q_heads, num_kv_heads, head_dim,
                  rope_theta, static_cast<hipStream_t>(stream));
}

extern "C" int kvhp_q4_rope_append(const void* q, const void* k, const void* v, int64_t q_stride,
                                   int64_t k_stride, int64_t v_stride, const int32_t* positions,
                                   const int32_t* slots, const int32_t* seq_lens,
                                   float rope_theta, void* q_out, void* pool,
                                   const int32_t* block_tables, int max_pages, int num_pages,
                                   int batch, int rows, int num_q_heads, int num_kv_heads,
                                   int head_dim, void* stream) {
    clear_error();
    if (batch <= 0 || rows <= 0) return KVHP_OK;
    AppendArgs a{};
    a.q = static_cast<const f16*>(q);
    a.k = static_cast<const f16*>(k);
    a.v = static_cast<const f16*>(v);
    a.sq = q_stride;
    a.sk = k_stride;
    a.sv = v_stride;
    a.positions = positions;
    a.slots = slots;
    a.seq_lens = seq_lens;
    a.q_out = static_cast<f16*>(q_out);
    a.pool = static_cast<uint8_t*>(pool);
    a.bt = block_tables;
    a.max_pages = max_pages;
    a.num_pages = num_pages;
    return append(a, "q4_rope_append", true, batch, rows, num_q_heads, num_kv_heads, head_dim,
                  rope_theta, static_cast<hipStream_t>(stream));
}
