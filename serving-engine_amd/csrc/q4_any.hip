// q4_any.hip -- attention over a paged cache held in 4 bits for any head_dim (a multiple of 8 up to
// 256) and any alignment of the rows (gfx950): what q4_decode.hip and q4_prefill.hip do not take, and
// few rows (q4.hip).
//
// One wave takes one KV head of one sequence, 16 of its (row, query head) pairs and a range of
// keys, in tiles of 64, four whole pages:
//   S^T = K Q^T       v_mfma_f32_16x16x32_f16: a lane's operand is eight dims of a row, one dword
//                     of codes where it lies; its scores are four keys of a page and one pair
//   O^T += V^T P^T    those keys' weights are its operand as they are, beside the codes of eight
//                     keys for one dim, gathered by bytes from the pages' codes in LDS
// Both operands are (n + r) 2^-9, exact (q4.h), from the denormal that a code is in a half's low
// bits.  s multiplies the fp32 scores, and the weight before its one rounding to fp16, by a power
// of two per tile that brings the tile's largest s up to 8 to 2^14; keys of larger ones, rows with
// values past 60 or so, have no weight then, and their tile is gone through once more for them
// alone, so that the others' weights keep their bits.  dims past head_dim and keys past the
// last are operands of 0; a key that holds NaN has those too, and a scale of NaN for the pairs
// that see it.
//
// Ranges of keys until the card has 4096 waves, down to one tile (one sequence of 2048 keys, 32/8 heads
// of 96: 10.6 us; of two tiles 14.2, of four 20.8); a second launch joins them.  Nothing is loaded
// ahead but a tile's V: what bounds it is the waits for page ids, then for codes, which the waves of
// a SIMD hide from each other (32 sequences of up to 8192 keys, 32/8 heads of 96, 117 MB: 82 us with
// three, 136 with the two that the compiler takes by itself, 131 with four, which spill; 2048 rows
// of them 166, 175 and 228).  A wave per (row, query head) and a key per trip took 4300 and 6444.
#include "q4.h"

#include <algorithm>
#include <type_traits>

namespace kvhp {
namespace {

constexpr int kTile = 64;       // keys
constexpr int kCols = 16;       // pairs of a wave
constexpr int kWaves = 4096;    // wanted
constexpr float kMostScale = 8.f;   // of keys whose weights share a power of two
constexpr int64_t kMostRowHeads = 1 << 29;

struct AnyPlan {
    int blocks;            // of pairs, per sequence and KV head
    int range, nsplit;     // tiles of a range, ranges
    bool aligned;          // q and out to 16 bytes
    float* ws_o;           // [batch * rows * Hq][nsplit][D]
    float* ws_ml;          // [batch * rows * Hq][nsplit][2]
};

__device__ __forceinline__ half2v as_half2(uint32_t x) { return __builtin_bit_cast(half2v, x); }
__device__ __forceinline__ half8 cat4(half2v a, half2v b, half2v c, half2v d) {
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// r 2^-9 of a row's two numbers, 0 where they are not finite or the key is none.
__device__ __forceinline__ f16 offset_of(uint32_t sr, bool key) {
    const bool ok = key && (sr & 0x7c00u) != 0x7c00u && (sr & 0x7c000000u) != 0x7c000000u;
    return ok ? as_half2(sr)[1] * f16(0x1p-9f) : f16(0);
}

// NC: chunks of 32 dims.
template <int NC>
__global__ void __launch_bounds__(kWave) __attribute__((amdgpu_waves_per_eu(NC <= 4 ? 3 : 2))) q4_any_kernel(const Q4Args a, const AnyPlan p) {
    constexpr int NB = 2 * NC;
    __shared__ __attribute__((aligned(16))) uint8_t vs[4 * kPage * 16 * NC + 16];
    const int lane = threadIdx.x, g = lane >> 4, c = lane & 15, D = a.D, RB = D / 2;
    const int kvh = blockIdx.x % a.Hkv, b = blockIdx.y, split = blockIdx.z;
    const int blk = p.blocks - 1 - static_cast<int>(blockIdx.x / a.Hkv);   // longest first
    const int n = q4_len(a, b);
    // a start outside +-2^30 leaves no row among at most 2^30 keys
    const int first = static_cast<int>(min(max(q4_first(a, b, n), -(int64_t)(1 << 30)), (int64_t)(1 << 30)));
    const int pair = blk * kCols + c, row = pair / a.G, qh = kvh * a.G + pair - row * a.G;
    const int r0 = blk * kCols / a.G, r1 = min((blk * kCols + kCols - 1) / a.G, a.rows - 1);
    const int p_lo = max(first + r0, 0), p_hi = min(first + r1, n - 1), pos = first + row;
    const int64_t at = ((int64_t)b * a.rows + row) * a.Hq + qh;
    if (p_lo > p_hi) {
        if (a.last_row && split == 0 && row < a.rows)   // no keys
            for (int d = g; d < D; d += 4) a.out[at * D + d] = f16(0);
        return;
    }
    const bool live = row < a.rows && pos >= p_lo && pos <= p_hi;
    const int tiles = p_hi / kTile + 1, t0 = split * p.range, t1 = min(tiles, t0 + p.range);
    if (t0 >= t1) return;

    half8 q[NC];   // dims 32 ch + 8 g .., in the codes' order
#pragma unroll
    for (int ch = 0; ch < NC; ++ch) {
        const int d0 = 32 * ch + 8 * g;
        half8 x{};
        if (live && d0 < D) {
            if (p.aligned) {
                x = load_half8(a.q + at * D + d0);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = a.q[at * D + d0 + e];
            }
        }
        q[ch] = __builtin_shufflevector(x, x, 0, 4, 1, 5, 2, 6, 3, 7);
    }
    floatx4 o[NB];
#pragma unroll
    for (int db = 0; db < NB; ++db) o[db] = floatx4{0.f, 0.f, 0.f, 0.f};
    float m = -1e30f, l = 0.f;
    const half2v lo15 = {f16(32768), f16(32768)}, hi15 = {f16(2048), f16(2048)};
    const float sc = 512.f * a.scale_log2;

    bool again = false;   // the tile's keys of large scales
    for (int t = t0; t < t1; t += again ? 0 : 1) {
        const uint8_t* pg[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pi = min(4 * t + i, p_hi >> 4);
            pg[i] = q4_page(a.pool, a.num_pages, D, kvh, a.bt[(int64_t)b * a.max_pages + pi]);
        }
        // V's codes, to LDS once K is done with: D / 2 chunks of 16 bytes a page
        constexpr int VL = (16 * NC + kWave - 1) / kWave;
        u32x4 v[4][VL];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < VL; ++u) {
                const int ch = lane + kWave * u;
                v[i][u] = ch < RB ? *reinterpret_cast<const u32x4*>(pg[i] + kPage * RB + 16 * ch) : u32x4{};
            }
        float s[4][4], mx = -INFINITY, big = 0.f;
        // V's scales; as they lie in the page where floats would spill (4 rows of 1024 keys of 32/8 heads
        // of 128: 12.4 us, as floats 12.8; 32 sequences of up to 8192 of 96: 82.4, as they lie 85.5)
        std::conditional_t<NC == 4, uint32_t, float> vnum[4][4];
        auto vscale = [&](int i, int e) {
            if constexpr (NC == 4)
                return static_cast<float>(as_half2(vnum[i][e])[0]);
            else
                return vnum[i][e];
        };
        f16 voff[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = kTile * t + kPage * i;
            const uint32_t kp = *reinterpret_cast<const uint32_t*>(pg[i] + kPage * D + 4 * c);
            const u32x4 ks = *reinterpret_cast<const u32x4*>(pg[i] + kPage * D + 16 * g);
            const u32x4 vp = *reinterpret_cast<const u32x4*>(pg[i] + kPage * D + 64 + 16 * g);
            const f16 r = offset_of(kp, key + c <= p_hi);
            floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ch = 0; ch < NC; ++ch) {
                const bool in = 32 * ch + 8 * g < D;
                const uint32_t x = in ? *reinterpret_cast<const uint32_t*>(pg[i] + c * RB + 16 * ch + 4 * g) : 0u;
                const half2v f = {in ? r : f16(0), in ? r : f16(0)};
                const uint32_t y = x >> 8;
                const half8 k = cat4(__builtin_elementwise_fma(as_half2(x & 0x000f000fu), lo15, f),
                                     __builtin_elementwise_fma(as_half2(x & 0x00f000f0u), hi15, f),
                                     __builtin_elementwise_fma(as_half2(y & 0x000f000fu), lo15, f),
                                     __builtin_elementwise_fma(as_half2(y & 0x00f000f0u), hi15, f));
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[ch], acc, 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = key + 4 * g + e;
                s[i][e] = live && j <= pos ? acc[e] * (static_cast<float>(as_half2(ks[e])[0]) * sc) : -INFINITY;
                mx = fmaxf(mx, s[i][e]);
                voff[i][e] = offset_of(vp[e], j <= p_hi);
                if constexpr (NC == 4)
                    vnum[i][e] = vp[e];
                else
                    vnum[i][e] = static_cast<float>(as_half2(vp[e])[0]);
                // a NaN is none of the largest, an infinity is only behind the last key
                big = fmaxf(big, j <= p_hi ? fabsf(vscale(i, e)) : 0.f);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        const bool large = __ballot(big > kMostScale) != 0;
        if (large) big = again ? 65504.f : kMostScale;   // for all that the pass may have
        const float mn = fmaxf(m, mx), alpha = fast_exp2(m - mn);
        m = mn;
        // 2^14 over big's power of two, and its inverse; big is 0 or at least 2^-24
        const int e2 = big > 0.f ? min(static_cast<int>(__float_as_uint(big) >> 23), 127 + 15) : 127;
        const float up = __uint_as_float(static_cast<uint32_t>(127 + 14 + 127 - e2) << 23);
        const float down = __uint_as_float(static_cast<uint32_t>(e2 - 14 + 9) << 23);
        l *= alpha;
        half8 w[2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = fast_exp2(s[i][e] - mn);
                l = fmaf(x, again ? 0.f : 1.f, l);
                // of keys not seen nothing, whatever their scale
                w[i / 2][4 * (i & 1) + e] = s[i][e] == -INFINITY ? f16(0) : static_cast<f16>(x * (vscale(i, e) * up));
            }
        if (large) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if ((fabsf(vscale(i, e)) > kMostScale) != again) w[i / 2][4 * (i & 1) + e] = f16(0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < VL; ++u) {
                const int ch = lane + kWave * u;
                if (ch < RB) *reinterpret_cast<u32x4*>(vs + kPage * RB * i + 16 * ch) = v[i][u];
            }
        __syncthreads();   // one wave: the order of its writes and reads
        const int sh = 4 * (c & 1);
#pragma unroll
        for (int db = 0; db < NB; ++db) {
            if (16 * db >= D) break;
            floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                half2v x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {   // keys 4 g + e, + 1 of page 2 u or 2 u + 1
                    const int i = 2 * u + k / 2, e = 2 * (k & 1);
                    const uint8_t* at_v = vs + (kPage * i + 4 * g + e) * RB + (16 * db + c) / 2;
                    const uint32_t y = at_v[0] | static_cast<uint32_t>(at_v[RB]) << 16;
                    x[k] = __builtin_elementwise_fma(as_half2(y >> sh & 0x000f000fu), lo15,
                                                     half2v{voff[i][e], voff[i][e + 1]});
                }
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(cat4(x[0], x[1], x[2], x[3]), w[u], acc, 0, 0, 0);
            }
            o[db] = o[db] * alpha + acc * down;
        }
        __syncthreads();
        again = large && !again;
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (!live) return;
    const bool cut = tiles > p.range;
    if (cut && g == 0) {
        p.ws_ml[(at * p.nsplit + split) * 2] = m;
        p.ws_ml[(at * p.nsplit + split) * 2 + 1] = l;
    }
    if (!cut && a.lse && g == 0)
        a.lse[((int64_t)b * a.Hq + qh) * a.rows + row] = (m + __builtin_amdgcn_logf(l)) * kLn2;
    const float inv = 1.f / l;
#pragma unroll
    for (int db = 0; db < NB; ++db) {   // dims 16 db + 4 g .. of the pair
        const int d0 = 16 * db + 4 * g;
        if (d0 >= D) continue;
        if (cut) {
            *reinterpret_cast<floatx4*>(p.ws_o + (at * p.nsplit + split) * D + d0) = o[db];
            continue;
        }
        half4 h;
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = static_cast<f16>(o[db][e] * inv);
        h = q4_finite(h);
        f16* to = a.out + at * D + d0;
        if (p.aligned) {
            *reinterpret_cast<half4*>(to) = h;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e] = h[e];
        }
    }
}

// Joins the ranges of a (row, head), D / 4 threads side by side, each four dims and four ranges' loads
// in flight.  ALL: a whole workgroup takes one (row, head), the threads past the first D / 4 the next
// ranges; else a workgroup takes 256 / (D / 4) of them (512 rows of 32/8 heads of 96, four ranges: 26.3
// us with both launches, 29.3 where four threads of every (row, head) part the ranges).
template <bool ALL>
__global__ void __launch_bounds__(256) q4_any_join_kernel(const Q4Args a, const AnyPlan p) {
    const int cpr = a.D / 4, most = 256 / cpr, b = blockIdx.y;
    const int group = threadIdx.x / cpr, c = threadIdx.x % cpr;
    if (!ALL && group >= most) return;
    const int lanes = ALL ? most : 1, r = ALL ? group : 0;
    const int rh = ALL ? blockIdx.x : blockIdx.x * most + group;   // at most 2^29
    const int row = rh / a.Hq, qh = rh - row * a.Hq;
    const int n = q4_len(a, b);
    const int64_t first = q4_first(a, b, n), pos = first + row, at = (int64_t)b * a.rows * a.Hq + rh;
    // the block's tiles, as the first launch has them
    const int pair = row * a.G + qh % a.G, r1 = min((pair / kCols * kCols + kCols - 1) / a.G, a.rows - 1);
    const int64_t last = min(first + r1, (int64_t)n - 1);
    int ranges = 0;
    if (row < a.rows && pos >= 0 && pos < n) ranges = (static_cast<int>(last) / kTile + p.range) / p.range;
    if (ranges < 2) ranges = 0;   // no row, or written by its one range
    float m = -3.0e38f, l = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
    auto fold = [&](float2 ml, floatx4 x) {
        const float mn = fmaxf(m, ml.x), al = fast_exp2(m - mn), be = fast_exp2(ml.x - mn);
        o = o * al + x * be;
        l = fmaf(l, al, ml.y * be);
        m = mn;
    };
    constexpr int U = 4;
    if (r < lanes)
        for (int j0 = r; j0 < ranges; j0 += U * lanes) {
            float2 ml[U];
            floatx4 x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t j = at * p.nsplit + min(j0 + u * lanes, ranges - 1);
                ml[u] = reinterpret_cast<const float2*>(p.ws_ml)[j];
                x[u] = *reinterpret_cast<const floatx4*>(p.ws_o + j * a.D + 4 * c);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j0 + u * lanes < ranges) fold(ml[u], x[u]);
        }
    if constexpr (ALL) {
        __shared__ __attribute__((aligned(16))) floatx4 part[256];
        __shared__ float2 state[256];
        part[threadIdx.x] = o;
        state[threadIdx.x] = float2{m, l};
        __syncthreads();
        if (r > 0) return;
        for (int k = 1; k < min(lanes, ranges); ++k) fold(state[threadIdx.x + k * cpr], part[threadIdx.x + k * cpr]);
    }
    if (ranges == 0) return;
    const float inv = 1.f / l;
    f16* to = a.out + at * a.D + 4 * c;
#pragma unroll
    for (int e = 0; e < 4; ++e) to[e] = q4_finite(static_cast<f16>(o[e] * inv));
    if (a.lse && c == 0) a.lse[((int64_t)b * a.Hq + qh) * a.rows + row] = (m + __builtin_amdgcn_logf(l)) * kLn2;
}

int64_t bytes(int64_t nsplit, int batch, int rows, int hq, int d) {
    return nsplit * (int64_t)sizeof(float) * batch * rows * hq * (d + 2);
}
// room: bytes of workspace (at head_dim 64 and 128 off 16 bytes what the other kernels asked for).
AnyPlan plan_of(int batch, int rows, int hq, int hkv, int d, int max_len, int64_t room) {
    AnyPlan p{};
    const int64_t pairs = (int64_t)rows * (hq / hkv), tiles = ((int64_t)max_len + kTile - 1) / kTile;
    p.blocks = static_cast<int>((pairs + kCols - 1) / kCols);
    int64_t n = std::min(std::max<int64_t>(kWaves / ((int64_t)p.blocks * hkv * batch), 1), tiles);
    n = std::min(n, std::max<int64_t>(room / bytes(1, batch, rows, hq, d), 1));
    p.range = static_cast<int>((tiles + n - 1) / n);
    p.nsplit = static_cast<int>((tiles + p.range - 1) / p.range);
    return p;
}

}  // namespace

size_t q4_any_workspace(int batch, int rows, int hq, int hkv, int d, int max_len) {
    if (rows <= 0 || !bound_sizes(batch, hq, hkv, max_len, 0, 0) || (int64_t)rows * hq > kMostRowHeads || d <= 0 ||
        d > 256 || d % 8)
        return 0;
    const AnyPlan p = plan_of(batch, rows, hq, hkv, d, max_len, INT64_MAX);
    return p.nsplit == 1 ? 0 : bytes(p.nsplit, batch, rows, hq, d);
}

// The workspace holds `room` bytes.
int q4_any(const Q4Args& a, int batch, const char* what, void* ws, size_t room, hipStream_t s) {
    KVHP_REQUIRE((int64_t)a.rows * a.Hq <= kMostRowHeads, KVHP_ERR_UNSUPPORTED, "%s: %d rows of %d heads", what,
                 a.rows, a.Hq);
    AnyPlan p = plan_of(batch, a.rows, a.Hq, a.Hkv, a.D, a.max_len, static_cast<int64_t>(room));
    const size_t rh = (size_t)batch * a.rows * a.Hq;
    p.aligned = aligned16(a.q) && aligned16(a.out);
    p.ws_o = static_cast<float*>(ws);
    p.ws_ml = p.ws_o + rh * p.nsplit * a.D;
    const dim3 grid(static_cast<unsigned>(p.blocks) * a.Hkv, batch, p.nsplit);
    auto go = [&](auto nc) {
        hipLaunchKernelGGL((q4_any_kernel<decltype(nc)::value>), grid, dim3(kWave), 0, s, a, p);
    };
    if (a.D <= 64)
        go(std::integral_constant<int, 2>{});
    else if (a.D <= 96)
        go(std::integral_constant<int, 3>{});
    else if (a.D <= 128)
        go(std::integral_constant<int, 4>{});
    else
        go(std::integral_constant<int, 8>{});
    const int rc = check_launch(what);
    if (rc || p.nsplit == 1) return rc;
    const unsigned heads = static_cast<unsigned>(a.rows) * a.Hq, per = 256 / (a.D / 4);
    if (p.nsplit > 8)
        hipLaunchKernelGGL(q4_any_join_kernel<true>, dim3(heads, batch), dim3(256), 0, s, a, p);
    else
        hipLaunchKernelGGL(q4_any_join_kernel<false>, dim3((heads + per - 1) / per, batch), dim3(256), 0, s, a, p);
    return check_launch(what);
}

}  // namespace kvhp
