// q4_decode.hip -- one new token per sequence over a paged cache held in 4 bits (gfx950,
// head_dim 64 and 128).
//
// Split-K decode: a workgroup takes a range of a sequence's keys for one KV head and up to 16
// of its query heads, its waves the range's tiles of 64 keys, four whole pages, round robin.
// A tile's pages go to the wave's own LDS stage as they are (global_load_lds), the next tile's
// K as soon as this one's is read and V after it; codes become operands in registers:
//   S^T = K Q^T       v_mfma_f32_16x16x32_f16, A = n + r of K, rows of the tile so dealt out
//                     that lane group g receives the scores of page g's 16 keys
//   O^T += V^T W^T    A = V's codes by ds_read_b64_tr_b4: a lane gets all 16 keys' codes of a
//                     page for one dim, which are the 16 keys whose weights its group holds
// A code becomes an operand as the denormal it is: four bits at the bottom of a half are n 2^-24
// (n 2^-20 at bits 4..7), which a packed multiply-add takes to (n + r) 2^-9, or to (n + r) E
// for V, without rounding (q4.h): a shift, four ands and four multiply-adds for eight codes.
// K's scale s multiplies the fp32 score.  V's is split into a power of two E of 2^-14 to 2^-9,
// which goes with the codes, and s / E, of 4 to 4096, which multiplies the weight before its
// one rounding to fp16.  A weight's 2^-11 holds down to 2^-16 of the largest; below it is an
// absolute 2^-25 of at most a quarter of that.  (Keys of scales past 8, rows with values past 60
// or so, would take it past fp16: their weights are 2^-13 of it, in products of their own that are
// multiplied back, so that the other keys' keep their bits.  Theirs hold 2^-11 down to 2^-13.)
//
// What bounds it: 32 sequences of up to 8192 keys, 32/8 heads of 128 (152 MB): 34.2 us, 4.5 TB/s, of
// which reading the pages alone takes 31 (a probe that reads pages of 2176 bytes in a random order
// 28.6 for as much); the vector unit is busy for 44 % of it, the matrix cores for 12.
// Then the join, 4.8.  Short contexts take a chain of waits, length, page id, page, 4.4 us, and the
// join's launch, 3.4.
//
// With up to 4 query heads (8), three (one) of four lanes of a 16-column product are idle: the
// scores of the four row tiles are dealt out to them, so that a lane has 4 (8) exponentials a
// tile instead of 16.
#include "q4.h"

#include <algorithm>
#include <type_traits>

namespace kvhp {
namespace {

constexpr int kTok = 64;          // keys per tile: one page per 16 lanes
constexpr int kMaxTiles = 16;     // per wave and split: 64 page ids, one per lane
constexpr int kMinTiles = 4;      // per balanced split
constexpr int kHeads = 16;        // query heads per workgroup
constexpr float kLazyLog2 = 3.f;  // a row's reference moves when a score passes it by this
constexpr float kMostM = 4096.f;  // s / E: weights up to 2^15 in fp16,
constexpr float kLarge = 8192.f;  // and this part of larger ones, which are up to 2^25

struct DecodePlan {
    int chunk;        // keys per split, a multiple of kTok
    int nsplit;       // split slots in the workspace
    int batch;
    int waves;        // per workgroup
    int balance;      // > 0: about this many splits per KV head over the batch
    int groups;       // workgroups per KV head and split, of up to kHeads query heads
    float* ws_o;      // [B * Hq][nsplit][D]
    float* ws_ml;     // [B * Hq][nsplit][2], the maximum in log2 units
    int32_t* ws_n;    // [B] splits
};

__device__ __forceinline__ int tiles_of(int L) { return (L + kTok - 1) / kTok; }
// Tiles of a sequence's splits where the batch has `tiles`.
__device__ __forceinline__ uint32_t share_tiles(const DecodePlan& p, uint32_t t, uint32_t target) {
    const uint32_t n = min((t + target - 1) / target, (uint32_t)p.nsplit);
    return t > 0 ? (t + n - 1) / n : 1;   // at most kMaxTiles: nsplit of them hold the longest
}
// The i-th split of the batch, counted in sequence order (sequences without keys keep one,
// which writes their zeros).
__device__ __forceinline__ bool share_of(const Q4Args& a, const DecodePlan& p, uint32_t i, int lane, int& b,
                                         int& split, int& L, int& chunk) {
    uint32_t tiles = 0;
    int li = lane < p.batch ? q4_len(a, lane) : 0;
    for (int g0 = 0; g0 < p.batch; g0 += kWave) {
        // at most 2^24 a sequence and 65535 of them: what 32 bits lose is only a balance
        const int l = g0 == 0 ? li : g0 + lane < p.batch ? q4_len(a, g0 + lane) : 0;
        tiles = min(tiles + (uint32_t)__builtin_amdgcn_readlane(prefix_sum(tiles_of(l)), kWave - 1), 1u << 30);
    }
    const uint32_t target = min(max((tiles + p.balance - 1) / p.balance, (uint32_t)kMinTiles), (uint32_t)kMaxTiles);
    uint32_t base = 0;
    for (int g0 = 0; g0 < p.batch; g0 += kWave) {
        const bool in = g0 + lane < p.batch;
        if (g0 > 0) li = in ? q4_len(a, g0 + lane) : 0;
        const uint32_t t = tiles_of(li), ti = share_tiles(p, t, target);
        const uint32_t ni = in ? max((t + ti - 1) / ti, 1u) : 0;
        const uint32_t inc = prefix_sum(ni), tot = __builtin_amdgcn_readlane(inc, kWave - 1);
        if (i < base + tot) {
            const int owner = __builtin_ctzll(__ballot(base + inc > i));
            b = g0 + owner;
            split = i - base - (__builtin_amdgcn_readlane(inc, owner) - __builtin_amdgcn_readlane(ni, owner));
            L = __builtin_amdgcn_readlane(li, owner);
            chunk = __builtin_amdgcn_readlane(ti, owner) * kTok;
            return true;
        }
        base += tot;
    }
    return false;
}

// global_load_lds_dwordx4 to LDS offset `to`, from a wave-uniform base and the lane's offset,
// or from an address per lane.
__device__ __forceinline__ void dma16(const void* base, uint32_t voff, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(to), "v"(voff), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void dma16(const void* src, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :: "s"(to), "v"(src) : "memory", "m0");
}

// A wave's tile in LDS.  Operand reads touch a page's rows in all four pages at once, so K's
// pages lie apart by what keeps them on distinct banks (D = 64, where a load brings two: by
// the chunks' order in every other page, and by pairs).
template <int D>
struct Stage {
    static constexpr int RB = D / 2;             // bytes of a row's codes
    static constexpr int PAGE = kPage * RB;
    static constexpr int PPL = 1024 / PAGE;      // pages per load
    static constexpr int kpage(int p) { return D == 128 ? p * 1040 : p * 512 + (p >> 1) * 128; }
    static constexpr int VOFF = kpage(3) + PAGE;
    static constexpr int PAR = VOFF + 4 * PAGE;  // (s, r): [page][K, V][16]
    static constexpr int BYTES = PAR + 512;
    static constexpr int LOADS = 4 / PPL;        // of K's codes, or of V's
    // 16-byte chunk c of V's row t lies at c ^ vswz(t): a transposing read's 16 rows on 16 banks
    __device__ __forceinline__ static int vswz(int t) { return D == 128 ? t >> 2 : t >> 3; }
};

// Eight codes of K as 2^-9 (n + r), in the order 0 4 1 5 2 6 3 7: four bits at the bottom of a
// half are the denormal n 2^-24 (at bits 4..7 n 2^-20), a multiply-add away from it, exact;
// f = 2^-9 r.
__device__ __forceinline__ half2v as_half2(uint32_t x) { return __builtin_bit_cast(half2v, x); }
__device__ __forceinline__ half8 cat4(half2v a, half2v b, half2v c, half2v d) {
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ half8 k_operand(uint32_t x, half2v f) {
    const half2v lo = {f16(32768), f16(32768)}, hi = {f16(2048), f16(2048)};
    const uint32_t y = x >> 8;
    return cat4(__builtin_elementwise_fma(as_half2(x & 0x000f000fu), lo, f),
                __builtin_elementwise_fma(as_half2(x & 0x00f000f0u), hi, f),
                __builtin_elementwise_fma(as_half2(y & 0x000f000fu), lo, f),
                __builtin_elementwise_fma(as_half2(y & 0x00f000f0u), hi, f));
}
// Eight codes of V, of eight rows, as (n + r) E: e = E 2^24, or E 2^20 for those that lie in
// bits 4..7, f = E r.
__device__ __forceinline__ half8 v_operand(uint32_t x, const u32x4& e, const u32x4& f) {
    auto pair = [&](uint32_t y, int i) {
        return __builtin_elementwise_fma(as_half2(y), as_half2(e[i]), as_half2(f[i]));
    };
    const uint32_t y = x >> 8;
    return cat4(pair(x & 0x000f000fu, 0), pair(x & 0x00f000f0u, 1), pair(y & 0x000f000fu, 2),
                pair(y & 0x00f000f0u, 3));
}
// The scale of row t as m E, E a power of two.
struct Scale {
    uint16_t e;
    f16 f;
    float m;
};
__device__ __forceinline__ Scale scale_of(uint32_t sr, int t) {
    const int e = min(max((int)(sr & 0x7c00u) - 0x0800, 0x0400), 0x1800);   // 2^-14 .. 2^-9
    const half2v h = as_half2(sr);
    Scale x;
    x.e = static_cast<uint16_t>(e + (t & 1 ? 0x5000 : 0x6000));
    x.f = h[1] * __builtin_bit_cast(f16, static_cast<uint16_t>(e));
    x.m = static_cast<float>(h[0]) * static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(0x7800 - e)));
    return x;
}
// Moves within 16 lanes: lane n gets lane n - S (or n + S: ROW_SHL) of x, in the quads of MASK;
// others keep `old`.
template <int CTRL, int MASK>
__device__ __forceinline__ uint32_t row_move(uint32_t old, uint32_t x) {
    return __builtin_amdgcn_update_dpp(old, x, CTRL, 0xf, MASK, false);
}
constexpr int kShl = 0x100, kShr = 0x110, kRor = 0x120;   // + the distance
template <int CTRL, int MASK>
__device__ __forceinline__ float row_move(float old, float x) {
    return __uint_as_float(row_move<CTRL, MASK>(__float_as_uint(old), __float_as_uint(x)));
}
typedef int v2i __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) v2i lds_v2i;
// Within each 16 lanes, whose addresses name 16 rows of 16 codes: all rows' codes of column i
// to lane i, row k in bits 4k ...
__device__ __forceinline__ v2i lds_read_tr4(const uint8_t* p) {
    return __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_v2i*)(__attribute__((address_space(3))) uint8_t*)p);
}

// What the lanes of a tile's keys leave for the others: lane group g reads page g's, 16 keys in
// the order 0 4 1 5 2 6 3 7, 8 12 .. of the codes' pairs.
struct __attribute__((aligned(16))) Prepared {
    float2 sm[kTok];        // K's s and V's m
    uint16_t e[kTok];       // V's E 2^24 or E 2^20 ...
    f16 f[kTok];            // ... and E r
    float large[kTok];      // m / kLarge where it is past kMostM (and 0 in sm)
};

// W waves per workgroup take the tiles of one split round robin and meet in LDS.
// PK: parts that a tile's scores are dealt out to, 16 / PK query heads or fewer.  Four waves a SIMD
// where their registers allow it without spills.
template <int D, int W, int PK>
__global__ void __launch_bounds__(W * kWave) __attribute__((amdgpu_waves_per_eu(D == 128 || PK < 4 ? 3 : 4)))
q4_decode_kernel(const Q4Args a, const DecodePlan p) {
    using St = Stage<D>;
    constexpr int NS = D / 32, ND = D / 16, PB = q4_page_bytes(D), RB = St::RB;
    __shared__ __attribute__((aligned(16))) uint8_t stage[W][St::BYTES];
    __shared__ Prepared prep_all[W];

    const int lane = threadIdx.x & (kWave - 1);
    const int wv = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int g = lane >> 4, col = lane & 15;
    const int kvh = blockIdx.x / p.groups, h0 = blockIdx.x % p.groups * kHeads;
    int b, split, L, chunk;
    if constexpr (W == 1) {
        if (!share_of(a, p, blockIdx.y, lane, b, split, L, chunk)) return;
    } else {
        split = blockIdx.y;
        b = blockIdx.z;
        L = q4_len(a, b);
        chunk = p.chunk;
    }
    const int nh = min(a.G - h0, kHeads);
    const int64_t row0 = (int64_t)b * a.Hq + (int64_t)kvh * a.G + h0;
    const int nsb = L > 0 ? (L + chunk - 1) / chunk : 0;
    if (p.nsplit > 1 && split == 0 && blockIdx.x == 0 && threadIdx.x == 0) p.ws_n[b] = nsb;
    if (L <= 0) {
        if (split == 0)
            for (int i = threadIdx.x; i < nh * (D / 8); i += W * kWave)
                store_half8(a.out + row0 * D + 8 * i, half8{});
        return;
    }
    if (split >= nsb) return;
    const int t_begin = split * chunk, t_end = min(L, t_begin + chunk);
    const int n_iter = (t_end - t_begin + kTok - 1) / kTok;
    const int n_w = n_iter > wv ? (n_iter - wv + W - 1) / W : 0;   // this wave's tiles
    const int hcol = col % (kHeads / PK), part = col / (kHeads / PK);   // of the scores dealt out
    const bool hvalid = hcol < nh;

    // Page ids of this wave's tiles, four to a tile; past the split's last key: its page.
    const uint8_t* head = a.pool + (int64_t)kvh * a.num_pages * PB;
    const int last = (t_end - 1) >> 4;
    const int pi = min((t_begin >> 4) + 4 * (wv + W * (lane >> 2)) + (lane & 3), last);
    const int pidv = min(max(a.bt[(int64_t)b * a.max_pages + pi], 0), a.num_pages - 1);
    half8 qb[NS];   // lane (g, col): head col, dims (D/4) g + 8 s .., in the codes' order
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const half8 x = col < nh ? load_half8(a.q + (row0 + col) * D + RB / 2 * g + 8 * s) : half8{};
        qb[s] = __builtin_shufflevector(x, x, 0, 4, 1, 5, 2, 6, 3, 7);
    }

    // The lane's place in a page's codes of K and of V
    const int lt = lane / (RB / 16) % kPage, lc = lane % (RB / 16);
    const int kt = (lt & 9) | (lt & 2) << 1 | (lt & 4) >> 1;   // K's rows in the order of the tiles' reads
    const uint32_t ko = RB * kt + 16 * (D == 128 ? lc : lc ^ (lane >> 5));
    const uint32_t vo = St::PAGE + RB * lt + 16 * (lc ^ St::vswz(lt));
    uint8_t* const st = stage[wv];
    const uint32_t st0 = lds_at(st);
    auto issue = [&](int j, uint32_t off, uint32_t to, auto kpage) {   // one matrix of this wave's j-th tile
#pragma unroll
        for (int i = 0; i < St::LOADS; ++i) {
            if constexpr (D == 128) {
                const int pid = __builtin_amdgcn_readlane(pidv, 4 * j + i);
                dma16(head + (int64_t)pid * PB, off, to + kpage(i));
            } else {
                const int pid = __shfl(pidv, 4 * j + 2 * i + (lane >> 5));
                dma16(head + (int64_t)pid * PB + off, to + kpage(2 * i));
            }
        }
    };
    auto issue_k = [&](int j) {   // and both matrices' (s, r)
        issue(j, ko, st0, [](int i) { return St::kpage(i); });
        const int pid = __shfl(pidv, 4 * j + (lane >> 3 & 3));
        if (lane < 32) dma16(head + (int64_t)pid * PB + kPage * D + 16 * (lane & 7), st0 + St::PAR);
    };
    auto issue_v = [&](int j) {
        issue(j, vo, st0 + St::VOFF, [](int i) { return i * St::PAGE; });
    };

    float m_run = -1e30f, l_part = 0.f;
    floatx4 o[ND];   // lane (g, col): dims 16 db + 4 g + e of head col
#pragma unroll
    for (int db = 0; db < ND; ++db) o[db] = floatx4{0.f, 0.f, 0.f, 0.f};
    auto scale_o = [&](float x) {
#pragma unroll
        for (int db = 0; db < ND; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[db][i] *= x;
    };
    const float sc = a.scale_log2 * 512.f;   // K's operands are 2^-9 (n + r)
    const float lazy = kLazyLog2 / sc;
    Prepared& prep = prep_all[wv];
    const int at = 16 * g + 8 * (col >> 3) + 2 * (col & 3) + (col >> 2 & 1);   // of key `col` of page g
    constexpr int X = 16 / PK;   // scores of a lane

    // LAST: only a wave's last tile may reach past the split's last key
    auto step = [&](auto LAST_, int j) {
        constexpr bool LAST = decltype(LAST_)::value;
        const int T0 = t_begin + kTok * (wv + W * j);
        wait_ring<St::LOADS>();   // K and the numbers have landed, V may be on its way
        asm volatile("" ::: "memory");
        bool large;   // some key's scale is past 8
        {   // this lane's key, for all
            const uint32_t kp = *reinterpret_cast<const uint32_t*>(st + St::PAR + g * 128 + 4 * col);
            uint32_t vp = *reinterpret_cast<const uint32_t*>(st + St::PAR + g * 128 + 64 + 4 * col);
            if (LAST && T0 + lane >= t_end) vp = 0;   // nothing of a row behind the last key
            Scale z = scale_of(vp, col);
            large = __ballot(fabsf(z.m) > kMostM) != 0;
            if (large) {
                const bool mine = fabsf(z.m) > kMostM;
                prep.large[at] = mine ? z.m * (1 / kLarge) : 0.f;
                z.m = mine ? 0.f : z.m;
            }
            prep.sm[at] = float2{q4_row(kp).s, z.m};
            prep.e[at] = z.e;
            prep.f[at] = z.f;
        }
        // scores: row 4 p + e of tile i is page p's key 0 2 8 10 (i) + 0 4 1 5 (e)
        const uint8_t* kr = st + (col >> 2) * St::PAGE + (D == 128 ? (col >> 2) * 16 : (col >> 3) * 128) +
                            (2 * (col & 1) + (col >> 1 & 1)) * RB + (D == 128 ? 16 * g : 8 * g ^ (col & 4) * 4);
        const uint8_t* kpar = st + St::PAR + (col >> 2) * 128 + ((col >> 1 & 1) + 4 * (col & 1)) * 4;
        floatx4 C[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t sr = *reinterpret_cast<const uint32_t*>(kpar + 4 * (8 * (i >> 1) + 2 * (i & 1)));
            const f16 r = as_half2(sr)[1] * f16(1.f / 512);
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
        if constexpr (!LAST) {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): all of it has been read
            issue_k(j + 1);
        }
        // this lane's scores, of keys X part .. in the prepared order, of head hcol
        float x[X], m[X];
#pragma unroll
        for (int t = 0; t < X; ++t) {
            x[t] = C[t / 4][t % 4];
            if constexpr (PK == 2) x[t] = row_move<kShr + 8, 0xc>(x[t], C[2 + t / 4][t % 4]);
            if constexpr (PK == 4) {
                x[t] = row_move<kShr + 4, 0x2>(x[t], C[1][t]);
                x[t] = row_move<kShr + 8, 0x4>(x[t], C[2][t]);
                x[t] = row_move<kShr + 12, 0x8>(x[t], C[3][t]);
            }
        }
        const floatx4* sm = reinterpret_cast<const floatx4*>(&prep.sm[16 * g + X * part]);
#pragma unroll
        for (int t = 0; t < X; t += 2) {
            const floatx4 z = sm[t / 2];
            x[t] *= z[0];
            x[t + 1] *= z[2];
            m[t] = z[1];
            m[t + 1] = z[3];
        }
        if constexpr (LAST) {
#pragma unroll
            for (int t = 0; t < X; ++t) {
                const int pos = X * part + t;
                const int key = (pos & 8) + (pos >> 1 & 3) + 4 * (pos & 1);
                if (T0 + 16 * g + key >= t_end) x[t] = -INFINITY;
            }
        }
        float mx = x[0];
#pragma unroll
        for (int t = 1; t < X; ++t) mx = fmaxf(mx, x[t]);
        if constexpr (PK == 4) mx = fmaxf(mx, row_move<kRor + 4, 0xf>(mx, mx));
        if constexpr (PK >= 2) mx = fmaxf(mx, row_move<kRor + 8, 0xf>(mx, mx));
        mx = rows4_max(mx);
        if (__builtin_amdgcn_read_exec() & __ballot(mx > m_run + lazy)) {
            const float mn = fmaxf(m_run, mx);
            const float alpha = fast_exp2((m_run - mn) * sc);
            m_run = mn;
            l_part *= alpha;
            scale_o(alpha);
        }
        const float nm = hvalid ? -m_run * sc : -INFINITY;
        uint32_t w[X / 2];
#pragma unroll
        for (int t = 0; t < X; t += 2) {
            const float y = fast_exp2(fmaf(x[t], sc, nm)), z = fast_exp2(fmaf(x[t + 1], sc, nm));
            l_part += y + z;
            w[t / 2] = __builtin_bit_cast(uint32_t, half2v{static_cast<f16>(y * m[t]), static_cast<f16>(z * m[t + 1])});
        }
        // the weights of page g's keys, of head col
        auto deal = [&](const uint32_t (&w)[X / 2], u32x4 (&pt)[2]) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (PK == 1) pt[u][i] = w[4 * u + i];
                    if constexpr (PK == 2) pt[u][i] = u == 0 ? w[i] : row_move<kShl + 8, 0xf>(w[i], w[i]);
                    if constexpr (PK == 4) {
                        const uint32_t v = w[i % 2];
                        pt[u][i] = u == 0 ? (i < 2 ? v : row_move<kShl + 4, 0xf>(v, v))
                                          : (i < 2 ? row_move<kShl + 8, 0xf>(v, v) : row_move<kShl + 12, 0xf>(v, v));
                    }
                }
        };
        const uint8_t* vr = st + St::VOFF + g * St::PAGE + col * RB;
        auto codes = [&](int db) { return lds_read_tr4(vr + 16 * (db / 2 ^ St::vswz(col)) + 8 * (db & 1)); };
        u32x4 pt[2], e[2], f[2];
        auto scales = [&]() {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                e[u] = *reinterpret_cast<const u32x4*>(&prep.e[16 * g + 8 * u]);
                f[u] = *reinterpret_cast<const u32x4*>(&prep.f[16 * g + 8 * u]);
            }
        };
        if (large) {   // seldom: what those keys add, before the others
            uint32_t wl[X / 2];
#pragma unroll
            for (int t = 0; t < X; t += 2) {
                const float2 z = *reinterpret_cast<const float2*>(&prep.large[16 * g + X * part + t]);
                wl[t / 2] = __builtin_bit_cast(uint32_t, half2v{static_cast<f16>(fast_exp2(fmaf(x[t], sc, nm)) * z.x),
                                                                static_cast<f16>(fast_exp2(fmaf(x[t + 1], sc, nm)) * z.y)});
            }
            deal(wl, pt);
            scales();
            wait_ring<0>();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int db = 0; db < ND; ++db) {
                const v2i y = codes(db);
                floatx4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < 2; ++u)
                    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(v_operand(y[u], e[u], f[u]),
                                                               __builtin_bit_cast(half8, pt[u]), c, 0, 0, 0);
                o[db] += c * kLarge;
                __builtin_amdgcn_sched_barrier(0);   // registers count here, not waits
            }
        }
        deal(w, pt);
        scales();
        if constexpr (LAST)
            wait_ring<0>();
        else
            wait_ring<St::LOADS + 1>();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int db = 0; db < ND; ++db) {
            const v2i y = codes(db);
#pragma unroll
            for (int u = 0; u < 2; ++u)
                o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v_operand(y[u], e[u], f[u]),
                                                               __builtin_bit_cast(half8, pt[u]), o[db], 0, 0, 0);
        }
        if constexpr (!LAST) {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xC07F);
            issue_v(j + 1);
        }
    };

    if (n_w > 0) {
        asm volatile("" ::: "memory");
        wait_ring<0>();
        issue_k(0);
        issue_v(0);
        for (int j = 0; j + 1 < n_w; ++j) step(std::false_type{}, j);
        step(std::true_type{}, n_w - 1);
        asm volatile("" ::: "memory");
    }
    if constexpr (PK == 4) l_part += row_move<kRor + 4, 0xf>(l_part, l_part);
    if constexpr (PK >= 2) l_part += row_move<kRor + 8, 0xf>(l_part, l_part);

    // Dims 16 db + 4 g + e of head col: all of them, or every W-th 16 of the waves' sum.
    constexpr int NB = (ND + W - 1) / W;
    floatx4 r[NB];
    float m = m_run, l = l_part;
    if constexpr (W == 1) {
#pragma unroll
        for (int db = 0; db < ND; ++db) r[db] = o[db];
    } else {
        // the waves leave (O, m, l) in their stages
        static_assert((ND * kWave * 4 + 2 * kWave) * 4 <= St::BYTES, "a wave's state in its stage");
        float* xs = reinterpret_cast<float*>(stage[wv]);
#pragma unroll
        for (int db = 0; db < ND; ++db)
            *reinterpret_cast<floatx4*>(&xs[(db * kWave + lane) * 4]) = o[db];
        *reinterpret_cast<float2*>(&xs[ND * kWave * 4 + 2 * lane]) = float2{m_run, l_part};
        __syncthreads();
        if (wv >= ND) return;
        float2 ml[W];
        l = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            ml[w] = *reinterpret_cast<const float2*>(
                &reinterpret_cast<const float*>(stage[w])[ND * kWave * 4 + 2 * lane]);
            m = fmaxf(m, ml[w].x);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) r[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float al = fast_exp2((ml[w].x - m) * sc);
            l = fmaf(ml[w].y, al, l);
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (W * i + wv < ND)
                    r[i] += al * *reinterpret_cast<const floatx4*>(
                        &reinterpret_cast<const float*>(stage[w])[((W * i + wv) * kWave + lane) * 4]);
        }
    }
    l = rows4_sum(l);
    if (col >= nh) return;
    const int64_t prow = (row0 + col) * p.nsplit + split;
    if (nsb > 1 && g == 0 && wv == 0) {
        p.ws_ml[prow * 2] = m * sc;
        p.ws_ml[prow * 2 + 1] = l;
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int db = W * i + wv;
        if (db >= ND) break;
        if (nsb == 1) {
            half4 h;
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = static_cast<f16>(r[i][e] * inv);
            *reinterpret_cast<half4*>(a.out + (row0 + col) * D + 16 * db + 4 * g) = q4_finite(h);
        } else {
            *reinterpret_cast<floatx4*>(p.ws_o + prow * D + 16 * db + 4 * g) = r[i];
        }
    }
}

// Joins the splits of a row (a query head of a sequence), a wave per row: lane (r, c) takes
// dims 8c .. of every (64 / (D/8))-th split, U of them at once.  The first are on their way
// before it is known how many there are (the workspace holds nsplit).
constexpr int kJoinRows = 4;   // waves per workgroup
template <int D, int U>
__global__ void __launch_bounds__(kJoinRows * kWave) q4_join_kernel(const Q4Args a, const DecodePlan p) {
    constexpr int LPR = D / 8, R = kWave / LPR;
    const int lane = threadIdx.x & (kWave - 1), c = lane % LPR, r = lane / LPR;
    const int head = blockIdx.x * kJoinRows + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), b = blockIdx.y;
    if (head >= a.Hq) return;
    const int64_t row = (int64_t)b * a.Hq + head;
    const float* po = p.ws_o + row * p.nsplit * D + 8 * c;
    const float2* pml = reinterpret_cast<const float2*>(p.ws_ml) + row * p.nsplit;
    float M = -3.0e38f, S = 0.f;
    floatx4 x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0;
    auto fold = [&](float m, float s, floatx4 y0, floatx4 y1) {
        const float mn = fmaxf(M, m);
        const float al = fast_exp2(M - mn), be = fast_exp2(m - mn);
        x0 = x0 * al + y0 * be;
        x1 = x1 * al + y1 * be;
        S = S * al + s * be;
        M = mn;
    };
    float2 ml[U];
    floatx4 y[U][2];
    auto load = [&](int j0, int n) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = min(j0 + R * u + r, n - 1);
            ml[u] = pml[j];
            y[u][0] = *reinterpret_cast<const floatx4*>(po + (int64_t)j * D);
            y[u][1] = *reinterpret_cast<const floatx4*>(po + (int64_t)j * D + 4);
        }
    };
    load(0, p.nsplit);
    const int nsb = p.ws_n[b];
    if (nsb <= 1) return;   // no keys, or written by its one split
    for (int j0 = 0;;) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + R * u + r < nsb) fold(ml[u].x, ml[u].y, y[u][0], y[u][1]);
        if ((j0 += R * U) >= nsb) break;
        load(j0, nsb);
    }
#pragma unroll
    for (int o = LPR; o < kWave; o <<= 1) {
        floatx4 y0, y1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y0[e] = __shfl_xor(x0[e], o);
            y1[e] = __shfl_xor(x1[e], o);
        }
        const float m = __shfl_xor(M, o), s = __shfl_xor(S, o);
        fold(m, s, y0, y1);
    }
    if (r > 0) return;
    const float inv = 1.f / S;
    half8 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = static_cast<f16>(x0[e] * inv);
        h[4 + e] = static_cast<f16>(x1[e] * inv);
    }
    store_half8(a.out + row * D + 8 * c, q4_finite(h));
}

// Where one split of eight waves holds a sequence, it saves the join's launch: 5 to 7 us against
// 7 to 8 for splits up to 1024 keys at D = 64 and 768 at D = 128, of one to four sequences; past
// that its waves' own tiles take longer (1024 keys at D = 128: 8.1 against 7.5).  Batches fill the
// card with one split each up to 2048 keys (32 sequences of 8 heads, D = 128: 13.7 against 14.9;
// of 4 heads, D = 64: 9.3 against 11.0; 64 of 8 heads are level, 4096 keys are not better).
constexpr int kBalanced = 16;      // sequences from which the splits are the whole batch's
constexpr int kWaveSlots = 2048;   // one wave per split, two per SIMD of 256 CUs
constexpr int kWaves = 4;          // per workgroup in fixed splits
constexpr int kShortWaves = 8;     // and where a sequence is one split

// Most splits that a batch may have: along a grid's second axis.
int64_t most_splits(int64_t batch, int64_t tiles, int balance) {
    return std::max<int64_t>(balance, (batch * tiles + kMaxTiles - 1) / kMaxTiles) + batch;
}

DecodePlan plan_of(int batch, int hkv, int G, int d, int64_t max_len) {
    DecodePlan p{};
    p.batch = batch;
    p.groups = (G + kHeads - 1) / kHeads;
    const int64_t heads = (int64_t)hkv * p.groups, tiles = (max_len + kTok - 1) / kTok;
    if (tiles <= (batch >= kBalanced ? 32 : d == 64 ? 16 : 12)) {
        p.waves = kShortWaves;
        p.chunk = static_cast<int>(tiles * kTok);
        p.nsplit = 1;
        return p;
    }
    const int64_t balance = std::max<int64_t>(1, kWaveSlots / heads - batch / 2);
    if (batch >= kBalanced && most_splits(batch, tiles, balance) <= 65535) {
        p.waves = 1;
        p.balance = static_cast<int>(balance);
        // splits of a sequence: of the target, which is the least where it alone has keys
        const int64_t target =
            std::min<int64_t>(std::max<int64_t>((tiles + p.balance - 1) / p.balance, kMinTiles), kMaxTiles);
        p.nsplit = static_cast<int>((tiles + target - 1) / target);
        return p;
    }
    p.waves = kWaves;
    const int64_t want = std::max<int64_t>(1, 512 / (heads * batch));   // workgroups per head
    const int64_t per = std::min<int64_t>(std::max<int64_t>((tiles + want - 1) / want, kWaves), kWaves * kMaxTiles);
    p.chunk = static_cast<int>(per * kTok);
    p.nsplit = static_cast<int>((tiles + per - 1) / per);
    return p;
}
}  // namespace

size_t q4_decode_workspace(int batch, int hq, int hkv, int d, int max_len) {
    if (!bound_sizes(batch, hq, hkv, max_len, 0, 0) || (d != 64 && d != 128)) return 0;
    const DecodePlan p = plan_of(batch, hkv, hq / hkv, d, max_len);
    return p.nsplit == 1 ? 0 : sizeof(float) * ((size_t)batch * hq * p.nsplit * (d + 2) + batch);
}

bool q4_decode_fits(const Q4Args& a, int batch) {
    const DecodePlan p = plan_of(batch, a.Hkv, a.G, a.D, a.max_len);
    return (a.D == 64 || a.D == 128) && aligned16(a.q) && aligned16(a.out) &&
           p.nsplit <= 65535 && (int64_t)a.Hkv * p.groups <= INT32_MAX;
}

// The workspace holds q4_decode_workspace bytes.
int q4_decode(const Q4Args& a, int batch, void* ws, hipStream_t s) {
    DecodePlan p = plan_of(batch, a.Hkv, a.G, a.D, a.max_len);
    p.ws_o = static_cast<float*>(ws);
    p.ws_ml = p.ws_o + (size_t)batch * a.Hq * p.nsplit * a.D;
    p.ws_n = reinterpret_cast<int32_t*>(p.ws_ml + (size_t)batch * a.Hq * p.nsplit * 2);
    const int64_t tiles = ((int64_t)a.max_len + kTok - 1) / kTok;
    const int64_t splits = p.balance ? most_splits(batch, tiles, p.balance) : p.nsplit;
    const dim3 grid(a.Hkv * p.groups, static_cast<unsigned>(splits), p.balance ? 1 : batch);
    auto go = [&](auto d, auto pk) {
        constexpr int D = decltype(d)::value, PK = decltype(pk)::value;
        const dim3 threads(p.waves * kWave);
        if (p.waves == 1)
            hipLaunchKernelGGL((q4_decode_kernel<D, 1, PK>), grid, threads, 0, s, a, p);
        else if (p.waves == kWaves)
            hipLaunchKernelGGL((q4_decode_kernel<D, kWaves, PK>), grid, threads, 0, s, a, p);
        else
            hipLaunchKernelGGL((q4_decode_kernel<D, kShortWaves, PK>), grid, threads, 0, s, a, p);
    };
    auto parts = [&](auto d) {
        if (a.G <= 4)
            go(d, std::integral_constant<int, 4>{});
        else if (a.G <= 8)
            go(d, std::integral_constant<int, 2>{});
        else
            go(d, std::integral_constant<int, 1>{});
    };
    a.D == 64 ? parts(std::integral_constant<int, 64>{}) : parts(std::integral_constant<int, 128>{});
    if (p.nsplit > 1) {
        const dim3 rows((a.Hq + kJoinRows - 1) / kJoinRows, batch), threads(kJoinRows * kWave);
        auto join = [&](auto d) {
            constexpr int D = decltype(d)::value;
            const int u = (p.nsplit * (D / 8) + kWave - 1) / kWave;   // splits of a lane
            if (u == 1)
                hipLaunchKernelGGL((q4_join_kernel<D, 1>), rows, threads, 0, s, a, p);
            else
                hipLaunchKernelGGL((q4_join_kernel<D, 2>), rows, threads, 0, s, a, p);
        };
        a.D == 64 ? join(std::integral_constant<int, 64>{}) : join(std::integral_constant<int, 128>{});
    }
    return check_launch("q4_decode");
}

}  // namespace kvhp
