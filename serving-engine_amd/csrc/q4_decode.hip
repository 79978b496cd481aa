// q4_decode.hip -- one new token per sequence over a paged cache held in 4 bits (gfx950,
// head_dim 64 and 128).
//
// Split-K decode: a workgroup takes a range of a sequence's keys for one KV head and up to 16
// of its query heads, its waves the range's tiles of 64 keys, four whole pages, round robin.
// A tile's pages go to the wave's own LDS stages as they are (global_load_lds), the next
// tile's on their way while this one is worked on; codes become operands in registers:
//   S^T = K Q^T       v_mfma_f32_16x16x32_f16, A = n + r of K, rows of the tile so dealt out
//                     that lane group g receives the scores of page g's 16 keys
//   O^T += V^T W^T    A = V's codes by ds_read_b64_tr_b4: a lane gets all 16 keys' codes of a
//                     page for one dim, which are the 16 keys whose weights its group holds
// so no score or weight crosses a lane.  A code becomes fp16 by its place: with its four bits
// in mantissa bits 6..9 below the exponent of 16 it is 16 + n, and + (r - 16) gives n + r
// without rounding (q4.h).  K's scale s multiplies the fp32 score.  V's is split into a power
// of two E, which goes with the codes, (16 + n) E + (r - 16) E, exact again, and s / E, of 4
// to 8 for all but the smallest, which multiplies the weight before its one rounding to fp16.
// Weights are biased by 2^10, so that 2^-11 of each holds down to 2^-24 of the largest.
#include "q4.h"

#include <algorithm>

namespace kvhp {
namespace {

constexpr int kTok = 64;          // keys per tile: one page per 16 lanes
constexpr int kMaxChunk = 1024;   // keys per split: 64 page ids, one per lane
constexpr int kHeads = 16;        // query heads per workgroup
constexpr float kBias = 10.f;

struct DecodePlan {
    int chunk;        // keys per split, a multiple of kTok
    int nsplit;
    int groups;       // workgroups per KV head and split, of up to kHeads query heads
    float* ws_o;      // [B * Hq][nsplit][D]
    float* ws_ml;     // [B * Hq][nsplit][2], the maximum in log2 units
};

// global_load_lds_dwordx4 from an address per lane.
__device__ __forceinline__ void dma16(const void* src, const void* lds_base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(lds_at(lds_base)), "v"(src) : "memory", "m0");
}

// A stage of a wave.  Operand reads touch a page's rows in all four pages at once, so the
// pages lie apart by what keeps them on distinct banks.
template <int D>
struct Stage {
    static constexpr int RB = D / 2;             // bytes of a row's codes
    static constexpr int kpage(int p) { return D == 128 ? p * 1040 : p * 1024 + (p & 1) * 16 + (p >> 1) * 128; }
    static constexpr int vpage(int p) { return D == 128 ? 4 * 1040 + p * 1024 : kpage(p) + 512; }
    static constexpr int PAR = D == 128 ? 4 * 1040 + 4096 : kpage(3) + 1024;   // (s, r): [page][K, V][16]
    static constexpr int BYTES = PAR + 512;
    static constexpr int LOADS = D == 128 ? 9 : 5;
    // V's 16-byte chunk c of row t lies at c ^ vswz(t): a transposing read's 16 rows on 16 banks
    __device__ __forceinline__ static int vswz(int t) { return D == 128 ? t >> 2 : t >> 3; }
};

// Eight codes as n + r times a power of two: E (16 + n) + F in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ half2v code_pair(uint32_t x) {
    return __builtin_bit_cast(half2v, (x & 0x03c003c0u) | 0x4c004c00u);
}
__device__ __forceinline__ half8 cat4(half2v a, half2v b, half2v c, half2v d) {
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ half8 k_operand(uint32_t x, half2v f) {
    return cat4(code_pair(x << 6) + f, code_pair(x << 2) + f, code_pair(x >> 2) + f, code_pair(x >> 6) + f);
}
__device__ __forceinline__ half8 v_operand(uint32_t x, const half2v (&e)[4], const half2v (&f)[4]) {
    return cat4(__builtin_elementwise_fma(code_pair(x << 6), e[0], f[0]),
                __builtin_elementwise_fma(code_pair(x << 2), e[1], f[1]),
                __builtin_elementwise_fma(code_pair(x >> 2), e[2], f[2]),
                __builtin_elementwise_fma(code_pair(x >> 6), e[3], f[3]));
}
// Scales of two rows as m E: E a power of two of at least 2^-14, m of 4 to 8 above that.
struct Scales {
    half2v e, f, m;
};
__device__ __forceinline__ Scales scales(uint32_t a, uint32_t b) {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    const uint32_t s = __builtin_amdgcn_perm(b, a, 0x05040100u), r = __builtin_amdgcn_perm(b, a, 0x07060302u);
    u16x2 e = __builtin_bit_cast(u16x2, s & 0x7c007c00u);
    e = __builtin_elementwise_max(__builtin_elementwise_sub_sat(e, u16x2{0x0800, 0x0800}), u16x2{0x0400, 0x0400});
    Scales x;
    x.e = __builtin_bit_cast(half2v, e);
    x.m = __builtin_bit_cast(half2v, s) * __builtin_bit_cast(half2v, u16x2{0x7800, 0x7800} - e);   // by 1 / E
    x.f = (__builtin_bit_cast(half2v, r) + half2v{f16(-16), f16(-16)}) * x.e;
    return x;
}
typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i lds_v2i;
// Within each 16 lanes, whose addresses name 16 rows of 16 codes: all rows' codes of column i
// to lane i, row k in bits 4k ...
__device__ __forceinline__ v2i lds_read_tr4(const uint8_t* p) {
    return __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_v2i*)(__attribute__((address_space(3))) uint8_t*)p);
}

template <int D, int W>
__global__ void __launch_bounds__(W * kWave) __attribute__((amdgpu_waves_per_eu(2)))
q4_decode_kernel(const Q4Args a, const DecodePlan p) {
    using St = Stage<D>;
    constexpr int NS = D / 32, ND = D / 16, PB = q4_page_bytes(D), RB = St::RB;
    __shared__ __attribute__((aligned(16))) uint8_t ring[W][2][St::BYTES];

    const int lane = threadIdx.x & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, col = lane & 15;
    const int kvh = blockIdx.x / p.groups, h0 = blockIdx.x % p.groups * kHeads;
    const int split = blockIdx.y, b = blockIdx.z;
    const int L = q4_len(a, b);
    const int nh = min(a.G - h0, kHeads);
    const int64_t row0 = (int64_t)b * a.Hq + (int64_t)kvh * a.G + h0;
    if (L <= 0) {
        if (split == 0)
            for (int i = threadIdx.x; i < nh * (D / 8); i += W * kWave)
                store_half8(a.out + row0 * D + 8 * i, half8{});
        return;
    }
    const int nsb = (L + p.chunk - 1) / p.chunk;
    if (split >= nsb) return;
    const int t_begin = split * p.chunk, t_end = min(L, t_begin + p.chunk);
    const int n_iter = (t_end - t_begin + kTok - 1) / kTok;
    const bool hvalid = col < nh;

    const uint8_t* head = a.pool + (int64_t)kvh * a.num_pages * PB;
    const int last = (t_end - 1 - t_begin) >> 4;   // page of the split's last key
    const int pidv = min(max(a.bt[(int64_t)b * a.max_pages + (t_begin >> 4) + min(lane, last)], 0),
                         a.num_pages - 1);
    half8 qb[NS];   // lane (g, col): head col, dims (D/4) g + 8 s .., in the codes' order
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const half8 x = hvalid ? load_half8(a.q + (row0 + col) * D + RB / 2 * g + 8 * s) : half8{};
        qb[s] = __builtin_shufflevector(x, x, 0, 4, 1, 5, 2, 6, 3, 7);
    }

    // The lane's place in a page of codes: D = 128 1 KB of K and 1 KB of V; D = 64 both in one
    uint32_t ko, vo = 0;
    if constexpr (D == 128) {
        ko = 16 * lane;
        vo = 1024 + 64 * (lane >> 2) + 16 * ((lane & 3) ^ St::vswz(lane >> 2));
    } else {
        const int t = (lane & 31) >> 1;
        ko = lane < 32 ? 16 * lane : 512 + 32 * t + 16 * ((lane & 1) ^ St::vswz(t));
    }
    auto issue = [&](int it, uint8_t* st) {
        const int pg = 4 * it;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int pid = __builtin_amdgcn_readlane(pidv, min(pg + i, last));
            const uint8_t* src = head + (int64_t)pid * PB;
            dma16s(src, ko, st + St::kpage(i));
            if constexpr (D == 128) dma16s(src, vo, st + St::vpage(i));
        }
        const int pid = __shfl(pidv, min(pg + (lane >> 3 & 3), last));
        if (lane < 32) dma16(head + (int64_t)pid * PB + kPage * D + 16 * (lane & 7), st + St::PAR);
    };

    float m_run = -1e30f, l_part = 0.f;
    floatx4 o[ND];   // lane (g, col): dims 16 db + 4 g + e of head col
#pragma unroll
    for (int db = 0; db < ND; ++db) o[db] = floatx4{0.f, 0.f, 0.f, 0.f};
    const float sc = a.scale_log2;

    auto step = [&](int it, const uint8_t* st) {
        const int T0 = t_begin + kTok * it;
        // scores: tile i's row m is page m / 4, key 4 i + m % 4
        const uint8_t* kr = st + St::kpage(0) + (col >> 2) * 1024 +
                            (D == 128 ? (col >> 2) * 16 : (col >> 2 & 1) * 16 + (col >> 3) * 128) +
                            (col & 3) * RB + g * (RB / 4);
        const uint8_t* kpar = st + St::PAR + (col >> 2) * 128 + (col & 3) * 4;
        floatx4 C[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f16 r = __builtin_bit_cast(half2v, *reinterpret_cast<const uint32_t*>(kpar + 16 * i))[1] - f16(16);
            const half2v f = {r, r};
            uint32_t x[NS];
            if constexpr (D == 128) {
                const u32x4 y = *reinterpret_cast<const u32x4*>(kr + 4 * i * RB);
#pragma unroll
                for (int s = 0; s < NS; ++s) x[s] = y[s];
            } else {
                const uint2 y = *reinterpret_cast<const uint2*>(kr + 4 * i * RB);
                x[0] = y.x;
                x[1] = y.y;
            }
            C[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < NS; ++s)
                C[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k_operand(x[s], f), qb[s], C[i], 0, 0, 0);
        }
        // page g's (s, r) of K and V
        const uint8_t* par = st + St::PAR + g * 128;
        u32x4 vp[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u32x4 kp = *reinterpret_cast<const u32x4*>(par + 16 * i);
            vp[i] = *reinterpret_cast<const u32x4*>(par + 64 + 16 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) C[i][e] *= q4_row(kp[e]).s;
        }
        if (T0 + kTok > t_end) {   // behind the last key: no weight, and nothing of the row
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (T0 + 16 * g + 4 * i + e >= t_end) {
                        C[i][e] = -INFINITY;
                        vp[i][e] = 0;
                    }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            mx = fmaxf(mx, fmaxf(fmaxf(C[i][0], C[i][1]), fmaxf(C[i][2], C[i][3])));
        mx = rows4_max(mx);
        const float mn = fmaxf(m_run, mx);
        const float alpha = fast_exp2((m_run - mn) * sc);
        m_run = mn;
        const float nm = hvalid ? kBias - mn * sc : -INFINITY;
        float ps = 0.f;
        half2v e[2][4], f[2][4];
        half8 pt[2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) {   // keys 8 u + j and 8 u + j + 4
                const Scales z = scales(vp[2 * u][j], vp[2 * u + 1][j]);
                e[u][j] = z.e;
                f[u][j] = z.f;
                const float x = fast_exp2(fmaf(C[2 * u][j], sc, nm));
                const float y = fast_exp2(fmaf(C[2 * u + 1][j], sc, nm));
                pt[u][2 * j] = static_cast<f16>(x * static_cast<float>(z.m[0]));
                pt[u][2 * j + 1] = static_cast<f16>(y * static_cast<float>(z.m[1]));
                ps += x + y;
            }
        l_part = fmaf(l_part, alpha, ps);
        if (__builtin_amdgcn_read_exec() & __ballot(alpha != 1.f)) {
#pragma unroll
            for (int db = 0; db < ND; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[db][i] *= alpha;
        }
        const uint8_t* vr = st + St::vpage(0) + (D == 128 ? g * 1024 : g * 1024 + (g & 1) * 16 + (g >> 1) * 128) +
                            col * RB;
#pragma unroll
        for (int db = 0; db < ND; ++db) {
            const v2i x = lds_read_tr4(vr + 16 * (db / 2 ^ St::vswz(col)) + 8 * (db & 1));
            o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v_operand(x[0], e[0], f[0]), pt[0], o[db], 0, 0, 0);
            o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v_operand(x[1], e[1], f[1]), pt[1], o[db], 0, 0, 0);
        }
    };

    const int n_w = n_iter > wv ? (n_iter - wv + W - 1) / W : 0;   // this wave's tiles
    if (n_w > 0) {
        asm volatile("" ::: "memory");
        wait_ring<0>();
        issue(wv, ring[wv][0]);
        for (int j = 0; j < n_w; ++j) {
            __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): the other stage's reads have returned
            if (j + 1 < n_w) {
                issue(wv + W * (j + 1), ring[wv][(j + 1) & 1]);
                wait_ring<St::LOADS>();
            } else {
                wait_ring<0>();
            }
            asm volatile("" ::: "memory");
            step(wv + W * j, ring[wv][j & 1]);
            asm volatile("" ::: "memory");
        }
    }

    // The waves leave (O, m, l) in their rings; each joins every W-th 16 dims.
    static_assert((ND * kWave * 4 + 2 * kWave) * 4 <= 2 * St::BYTES, "a wave's state in its ring");
    float* xs = reinterpret_cast<float*>(ring[wv][0]);
#pragma unroll
    for (int db = 0; db < ND; ++db)
        *reinterpret_cast<floatx4*>(&xs[(db * kWave + lane) * 4]) = o[db];
    *reinterpret_cast<float2*>(&xs[ND * kWave * 4 + 2 * lane]) = float2{m_run, l_part};
    __syncthreads();
    if (wv >= ND) return;
    float2 ml[W];
    float m = -1e30f, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        ml[w] = *reinterpret_cast<const float2*>(&reinterpret_cast<const float*>(ring[w][0])[ND * kWave * 4 + 2 * lane]);
        m = fmaxf(m, ml[w].x);
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
        ml[w].x = fast_exp2((ml[w].x - m) * sc);
        l = fmaf(ml[w].y, ml[w].x, l);
    }
    l = rows4_sum(l);
    if (!hvalid) return;
    const int64_t prow = (row0 + col) * p.nsplit + split;
    if (nsb > 1 && g == 0 && wv == 0) {
        p.ws_ml[prow * 2] = m * sc;
        p.ws_ml[prow * 2 + 1] = l;
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int d0 = 0; d0 < ND; d0 += W) {
        const int db = d0 + wv;
        if (db >= ND) break;
        floatx4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w)
            r += *reinterpret_cast<const floatx4*>(&reinterpret_cast<const float*>(ring[w][0])[(db * kWave + lane) * 4]) * ml[w].x;
        if (nsb == 1) {
            half4 h;
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = static_cast<f16>(r[i] * inv);
            *reinterpret_cast<half4*>(a.out + (row0 + col) * D + 16 * db + 4 * g) = h;
        } else {
            *reinterpret_cast<floatx4*>(p.ws_o + prow * D + 16 * db + 4 * g) = r;
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kJoinWaves * kWave)
q4_join_kernel(const Q4Args a, const DecodePlan p) {
    const int b = blockIdx.y, L = q4_len(a, b);
    const int nsb = (L + p.chunk - 1) / p.chunk;
    if (nsb > 1) join_head<D>(a.out, p.ws_o, p.ws_ml, p.nsplit, (int64_t)b * a.Hq + blockIdx.x, nsb);
}

DecodePlan plan_of(int batch, int hkv, int G, int64_t max_len) {
    DecodePlan p{};
    p.groups = (G + kHeads - 1) / kHeads;
    const int64_t units = (int64_t)batch * hkv * p.groups;
    int64_t s = std::max<int64_t>(1, 1024 / units);          // splits wanted
    int64_t chunk = (max_len + s - 1) / s;
    chunk = std::min<int64_t>(std::max<int64_t>((chunk + 255) / 256 * 256, 256), kMaxChunk);
    p.chunk = static_cast<int>(chunk);
    p.nsplit = static_cast<int>((max_len + chunk - 1) / chunk);
    return p;
}

}  // namespace

size_t q4_decode_workspace(int batch, int hq, int hkv, int d, int max_len) {
    if (!bound_sizes(batch, hq, hkv, max_len, 0, 0) || (d != 64 && d != 128)) return 0;
    const DecodePlan p = plan_of(batch, hkv, hq / hkv, max_len);
    return p.nsplit == 1 ? 0 : sizeof(float) * (size_t)batch * hq * p.nsplit * (d + 2);
}

bool q4_decode_fits(const Q4Args& a, int batch) {
    const DecodePlan p = plan_of(batch, a.Hkv, a.G, a.max_len);
    return (a.D == 64 || a.D == 128) && aligned16(a.q) && aligned16(a.out) && p.nsplit <= 65535 &&
           (int64_t)a.Hkv * p.groups <= INT32_MAX;
}

// The workspace holds q4_decode_workspace bytes.
int q4_decode(const Q4Args& a, int batch, void* ws, hipStream_t s) {
    DecodePlan p = plan_of(batch, a.Hkv, a.G, a.max_len);
    p.ws_o = static_cast<float*>(ws);
    p.ws_ml = p.ws_o + (size_t)batch * a.Hq * p.nsplit * a.D;
    const dim3 grid(a.Hkv * p.groups, p.nsplit, batch);
    auto go = [&](auto kernel, auto join) {
        hipLaunchKernelGGL(kernel, grid, dim3(4 * kWave), 0, s, a, p);
        if (p.nsplit > 1)
            hipLaunchKernelGGL(join, dim3(a.Hq, batch), dim3(kJoinWaves * kWave), 0, s, a, p);
    };
    if (a.D == 64)
        go(q4_decode_kernel<64, 4>, q4_join_kernel<64>);
    else
        go(q4_decode_kernel<128, 4>, q4_join_kernel<128>);
    return check_launch("q4_decode");
}

}  // namespace kvhp
