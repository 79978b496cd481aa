// window_prefill.hip -- rows of prompts and chunks attending a sliding window
// and the first tokens of their sequence, over a cache view (gfx950, head_dim
// 64 and 128).
//
// A workgroup of four waves takes one KV head of one sequence and 128 of its (row, query
// head) pairs, query head fastest: 32 pairs a wave, whatever the group size, so the heads
// of a group share the K/V tiles and a chunk of a few rows still fills a wave.  Two
// workgroups share a CU.
//
// Keys: those that some row of the block sees, numbered through without the pages
// between the first tokens' and the earliest window's: `nv` keys, 64 to a tile.  (The
// gap is whole pages so that the rows of a load share a page, whose id is then
// scalar; the rest of the two pages at its edges is masked.)  A block of a long prompt
// walks (window + sinks + its rows) / 64 tiles, all blocks alike, where causal attention
// would walk up to S / 64.  Only tiles at the window's two edges and those that hold
// first tokens need a mask.
//
// Per tile, on v_mfma_f32_32x32x16_f16 with one lane per pair: S^T = K Q^T; an fp32 online
// softmax in the log2 domain whose reference lies 2^7 to 2^15 below a row's largest weight
// (it moves when a row passes it by 2^15).  Weights are rounded to fp16 for the product: 2^-11
// each down to 2^-14 of the reference, an absolute 2^-25 of it below, so that 10^5 keys of
// little weight beside a first token of much still count; O^T += V^T P^T.  K and V rows go
// from memory to two LDS stages per matrix without registers (global_load_lds, a scalar base
// and the lane's fixed offset; page ids from LDS), with their 16-byte chunks XOR-swizzled so
// that both operand reads touch all banks.
//
// At 8192 rows, window 2048, 32/8 heads of 128: 255-273 us by box, 0.89-0.95 PFLOP/s; a chunk
// of 128 rows of each of four sequences of 1062 to 8192 keys, window 4096, 47-49, of which the
// join 7 (the ranges go by the window, so 96 of their 512 workgroups have no keys and the
// others up to 17 tiles).  Without a window, with lse, 512 / 2048 / 8192 rows take 18.3 / 48.7 /
// 512 us where the causal prefill without lse takes 14.7 / 45.7 / 508.  Counters: matrix cores 55 %,
// vector unit 50 %, LDS reads 28 % of the cycles, at the 1.6 GHz that the card holds under
// this load (a large library product: 1.18 PFLOP/s).  The MFMAs alone take 172 us of 262;
// without the exponentials the kernel takes 228, without LDS operand reads 234, without
// loads 225.  More waves do not help (tiles of 32 keys, three workgroups a CU: 280); more
// pairs a wave, half the LDS reads, need more registers than the 256 a lane of two waves
// per SIMD has (64 pairs on one wave per SIMD, O and Q in accumulation registers: 625, the
// compiler moves O between the register files at every branch).
//
// A masked key's weight is 0, but 0 times an infinite or NaN V is NaN: in the
// tiles that some row sees only in part such elements are set to 0 in LDS, noted,
// and added as they are at the end to the rows that see their key.
//
// Few rows over a long cache are cut into ranges of keys (blockIdx.z) whose
// partials a second launch joins.
#include "bounded.h"

#include <algorithm>
#include <type_traits>

namespace kvhp {
namespace {

constexpr int kBN = 64;               // keys per tile
constexpr int kWaves = 4;
constexpr int kPairs = 32 * kWaves;   // (row, head) pairs per workgroup
constexpr int kRing = 512;            // tiles whose page ids LDS holds, read in halves of it
constexpr int kPages = kRing * (kBN / kPage);
constexpr int kMaxStride = 1 << 24;   // halfs between rows: 15 rows stay below 2^31 bytes
constexpr int kEdge = 6;              // tiles at either edge of the window in a block
constexpr int kBadWords = 4 * kEdge;  // a bit per key of those
constexpr int kMaxRowHeads = 1 << 29; // (row, query head) pairs of a sequence: a grid of 2^22
constexpr int kCUs = 256;
constexpr float kRefLog2 = 7.f;       // a row's reference below its maximum where it is set,
constexpr float kLazyLog2 = 15.f;     // and where it moves: weights up to 2^15 in fp16

struct PrefillPlan {
    uint32_t inv_g;        // ceil(2^32 / G), 0 for G = 1
    int blocks;            // of pairs, per sequence and KV head
    int tiles_per_split, nsplit;
    float* ws_o;           // [batch * rows * Hq][nsplit][D]
    float* ws_ml;          // [batch * rows * Hq][nsplit][2], the reference in log2 units
};

// Row of a pair: pair / G, exact for pair * G below 2^32.
__device__ __forceinline__ int row_of(const PrefillPlan& p, uint32_t pair) {
    return static_cast<int>(p.inv_g ? __umulhi(pair, p.inv_g) : pair);
}
// The rows of a block that lie in their sequence, and the keys they see.
struct Block {
    int first;       // position of row 0
    int p_lo, p_hi;  // positions of the block's first and last live row; none: p_lo > p_hi
    int sinks;       // first tokens that every row sees
    int head;        // keys in front of the gap: up to the end of their page
    int shift;       // the gap, whole pages; 0: none (head is 0 then)
    int nv;          // keys, numbered through: v < head is key v, others key v + shift
};
__device__ __forceinline__ Block block_of(const BoundArgs& a, const PrefillPlan& p, int b, int blk,
                                          int pairs) {
    Block k;
    const int n = bound_len(a, b);
    // a start outside +-2^30 leaves no row among at most 2^30 keys
    const int64_t first = min(max(bound_first(a, b, n), -(int64_t)(1 << 30)), (int64_t)(1 << 30));
    const int r0 = row_of(p, blk * pairs), r1 = min(row_of(p, (blk + 1) * pairs - 1), a.rows - 1);
    k.first = static_cast<int>(first);
    k.p_lo = static_cast<int>(max(first + r0, (int64_t)0));
    k.p_hi = static_cast<int>(min(first + r1, (int64_t)n - 1));
    const int low = bound_low(k.p_lo, a.window);
    k.sinks = a.window > 0 ? min(a.sinks, k.p_hi + 1) : 0;
    k.head = (k.sinks + kPage - 1) & ~(kPage - 1);
    k.shift = max((low & ~(kPage - 1)) - k.head, 0);
    if (k.shift == 0) k.head = 0;
    k.nv = k.p_hi + 1 - k.shift;
    return k;
}

// A block's keys: page ids, loads into LDS stages, and the V
// elements of masked keys that are not finite.
template <int D, bool PAGED>
struct Keys {
    static constexpr int CPR = D / 8, RPI = kWave / CPR;
    static constexpr int IPW = kBN / RPI / kWaves;   // loads per wave, matrix and tile
    static constexpr int NDB = D / 32;
    // chunk c of row r lies at position c ^ swizzle: the 16 rows of an operand read of K,
    // and the four rows x four chunks of a transposing read of V, on distinct banks
    __device__ __forceinline__ static int kswz(int r) { return CPR == 16 ? r & 15 : r >> 1 & 7; }
    __device__ __forceinline__ static int vswz(int r) { return CPR == 16 ? 4 * (r & 3) : (r & 3) << 1; }

    const BoundArgs& a;
    const Block& k;
    int32_t* ptab;
    uint32_t* bad;
    int wave, lane, t_lo, last_tile, window;
    const char *kb, *vb;
    const int32_t* table;
    uint32_t ssk, ssv;
    uint32_t ko[IPW], vo[IPW];   // the lane's offsets from the wave's first row of a tile
    int edge_hi, edge_lo, edge_end;

    __device__ __forceinline__ Keys(const BoundArgs& a_, const Block& k_, int32_t* ptab_,
                                    uint32_t* bad_, int b, int kvh, int t_lo_, int n_tiles)
        : a(a_), k(k_), ptab(ptab_), bad(bad_) {
        static_assert(kPage % (IPW * RPI) == 0, "a wave's rows of a tile lie in one page");
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        lane = threadIdx.x & 63;
        t_lo = t_lo_;
        last_tile = n_tiles - 1;
        window = a.window > 0 ? a.window : INT32_MAX;
        kb = reinterpret_cast<const char*>(a.k.data + (PAGED ? 0 : b * a.k.stride_b) + kvh * a.k.stride_h);
        vb = reinterpret_cast<const char*>(a.v.data + (PAGED ? 0 : b * a.v.stride_b) + kvh * a.v.stride_h);
        ssk = 2 * static_cast<uint32_t>(a.k.stride_s);
        ssv = 2 * static_cast<uint32_t>(a.v.stride_s);
#pragma unroll
        for (int i = 0; i < IPW; ++i) {
            const int r = (wave * IPW + i) * RPI + lane / CPR;
            ko[i] = (i * RPI + lane / CPR) * ssk + 16 * ((lane % CPR) ^ kswz(r));
            vo[i] = (i * RPI + lane / CPR) * ssv + 16 * ((lane % CPR) ^ vswz(r));
        }
        // Tiles that some row of the block sees in part: from `edge_hi` on (keys past the
        // first row), and from `edge_lo`, the first behind the first tokens, to `edge_end`,
        // that of the last key that the last row's window has left.
        edge_hi = max(k.p_lo - k.shift + 1, 0) / kBN;
        edge_lo = k.sinks / kBN;
        const int64_t left = (int64_t)k.p_hi - window - k.shift;
        edge_end = left < 0 ? -1 : static_cast<int>(left / kBN);
        if constexpr (PAGED) {
            table = a.k.bt + (int64_t)b * a.k.max_pages;
            pages_of(0, kRing);
        }
        if (threadIdx.x < kBadWords) bad[threadIdx.x] = 0;
    }
    __device__ __forceinline__ int key_of(int v) const { return v < k.head ? v : v + k.shift; }
    __device__ __forceinline__ int page_of(int key) const {
        return min(max(table[key >> 4], 0), a.k.num_pages - 1);
    }
    // Page ids of tiles [t0, t1) of the split's, 16 keys to a page, into their places in LDS.
    __device__ __forceinline__ void pages_of(int t0, int t1) const {
        const int v0 = t_lo * kBN, v1 = min((t_lo + min(t1, last_tile + 1)) * kBN, k.nv);
        for (int i = t0 * (kBN / kPage) + threadIdx.x; v0 + i * kPage < v1; i += kWaves * kWave)
            ptab[i & (kPages - 1)] = page_of(key_of(v0 + i * kPage));
    }
    // In front of iteration j: all waves have begun j - 1 and ask for pages from tile j + 2 on
    // (issue), so the half ring before tile j is free for the tiles behind the next half.
    __device__ __forceinline__ void more_pages(int j) const {
        if constexpr (PAGED)
            if (j % (kRing / 2) == 0 && j > 0) pages_of(j + kRing / 2, j + kRing);
    }
    // First row of this wave in a tile.  Tiles past the last re-load it, so every wave
    // issues the same loads.
    __device__ __forceinline__ int first_row(int tt) const {
        return min((t_lo + min(tt, last_tile)) * kBN + wave * IPW * RPI, k.nv - 1);
    }
    // The page of this wave's rows of a tile, read one issue ahead.
    __device__ __forceinline__ int page(int tt) const {
        return PAGED ? ptab[((first_row(tt) >> 4) - t_lo * (kBN / kPage)) & (kPages - 1)] : 0;
    }
    // One tile of a matrix to a stage; rows past the last key re-read it.
    __device__ __forceinline__ void issue(int tt, int pid, const char* base, uint32_t ss,
                                          const uint32_t (&off)[IPW], f16* stage) const {
        const int v = first_row(tt);
        const int key = key_of(v);
        const uint32_t row = PAGED ? __builtin_amdgcn_readfirstlane(pid) * kPage + (key & 15) : key;
        const char* src = base + (uint64_t)row * ss;
        f16* dst = stage + wave * IPW * RPI * D;
        if ((t_lo + min(tt, last_tile)) * kBN + (wave + 1) * IPW * RPI <= k.nv) {
#pragma unroll
            for (int i = 0; i < IPW; ++i) dma16s(src, off[i], dst + i * RPI * D);
        } else {
#pragma unroll
            for (int i = 0; i < IPW; ++i) {
                const int r = i * RPI + lane / CPR;
                dma16s(src, off[i] + (min(r, k.nv - 1 - v) - r) * ss, dst + i * RPI * D);
            }
        }
    }
    __device__ __forceinline__ void issue_k(int tt, int pid, f16* stage) const {
        issue(tt, pid, kb, ssk, ko, stage);
    }
    __device__ __forceinline__ void issue_v(int tt, int pid, f16* stage) const {
        issue(tt, pid, vb, ssv, vo, stage);
    }
    // This wave's rows of a V tile, just landed: where some row of the block does not see
    // all of it, elements that are not finite become 0 and their keys are noted.
    __device__ __forceinline__ void clean(int j, f16* stage) const {
        const int t = t_lo + j;
        if (t < edge_hi && (t < edge_lo || t > edge_end)) return;
        const int word = t >= edge_hi ? 2 * (kEdge + t - edge_hi) : 2 * (t - edge_lo);
        f16* Vt = stage + wave * IPW * RPI * D + 8 * lane;
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < IPW; ++i) {
            u32x4 x = *reinterpret_cast<const u32x4*>(Vt + i * RPI * D);
            uint32_t m[4], any = 0;   // bits 15 / 31: an exponent of all ones
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m[e] = ((x[e] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
                any |= m[e];
            }
            if (any == 0) continue;
            const int r = (wave * IPW + i) * RPI + lane / CPR;
            atomicOr(&bad[word + (r >> 5)], 1u << (r & 31));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] &= ~(m[e] | (m[e] - (m[e] >> 15)));
            *reinterpret_cast<u32x4*>(Vt + i * RPI * D) = x;
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): written before the barrier
    }
    // Those elements to a row that sees their keys (all waves are past their last clean).
    __device__ __forceinline__ void add_back(floatx16 (&o)[NDB], bool live, int pos) const {
        const int h = lane >> 5;
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < kBadWords; ++i) any |= bad[i];
        if (!__builtin_amdgcn_readfirstlane(any)) return;
#pragma unroll 1
        for (int i = 0; i < 32 * kBadWords; ++i) {
            if (!(bad[i >> 5] >> (i & 31) & 1)) continue;
            const int v = (i < kEdge * kBN ? edge_lo : edge_hi) * kBN + i % (kEdge * kBN);
            if (v >= k.nv) continue;   // a repeated row
            const int key = key_of(v);
            int64_t s = key;
            if constexpr (PAGED) s = (int64_t)page_of(key) * kPage + (key & 15);
            const f16* src = reinterpret_cast<const f16*>(vb + s * (int64_t)ssv) + 4 * h;
            const bool sees = live && key <= pos && (key < a.sinks || pos - key < window);
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    half4 x4 = *reinterpret_cast<const half4*>(src + 32 * db + 8 * q4);
                    if (!sees) x4 = half4{};
#pragma unroll
                    for (int e4 = 0; e4 < 4; ++e4) {
                        const float x = static_cast<float>(x4[e4]);
                        o[db][4 * q4 + e4] += fabsf(x) < INFINITY ? 0.f : x;
                    }
                }
        }
    }
};

// 32 pairs of a wave, one per lane of either half.
struct Pairs {
    int row, qh, pos;
    bool live;
    int64_t at;           // (sequence, row, head)
    // Tiles (of the block's) that need a mask: from `past` on (keys past some pair's row),
    // and from gone_lo to gone_hi (keys that a pair's window has left).
    int past, gone_lo, gone_hi;
};
__device__ __forceinline__ Pairs pairs_at(const BoundArgs& a, const PrefillPlan& p, const Block& k,
                                          int b, int kvh, int pair0, int c32) {
    Pairs x;
    const int pair = pair0 + c32;
    x.row = row_of(p, pair);
    x.qh = kvh * a.G + pair - x.row * a.G;
    x.pos = k.first + x.row;
    x.live = x.row < a.rows && x.pos >= k.p_lo && x.pos <= k.p_hi;
    x.at = ((int64_t)b * a.rows + x.row) * a.Hq + x.qh;
    const int lo = k.first + row_of(p, pair0), hi = k.first + row_of(p, pair0 + 31);
    const int whole = lo - k.shift - (kBN - 1);   // last key a wholly seen tile may begin with
    x.past = lo < k.p_lo || hi > k.p_hi || whole < 0 ? 0 : whole / kBN + 1;
    x.gone_lo = k.sinks / kBN;
    x.gone_hi = a.window > 0 && hi - k.shift >= a.window ? (hi - k.shift - a.window) / kBN : -1;
    return x;
}
// Masks the scores of N 32-key blocks of tile t; element (n, i) is key v0 + 32 n +
// 8 (i / 4) + i % 4.  Returns whether there was anything to mask.
template <int N>
__device__ __forceinline__ bool mask(const Block& k, const Pairs& x, int window, int t, int v0,
                                     floatx16 (&sc)[N]) {
    const bool gone = t >= x.gone_lo && t <= x.gone_hi;
    if (t < x.past && !gone) return false;
    if (t >= x.past) {
        const int hi = x.live ? x.pos - k.shift - v0 : -1;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                sc[n][i] = 32 * n + 8 * (i / 4) + (i % 4) > hi ? -INFINITY : sc[n][i];
    }
    if (gone) {   // from the first tokens' end to `left`
        const int64_t left = (int64_t)x.pos - window - k.shift - v0;
        const int head = k.sinks - v0;
        const uint32_t span = static_cast<uint32_t>(max(left - head + 1, (int64_t)0));
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                sc[n][i] = static_cast<uint32_t>(32 * n + 8 * (i / 4) + (i % 4) - head) < span
                               ? -INFINITY : sc[n][i];
    }
    return true;
}
template <int N>
__device__ __forceinline__ float max_of(const floatx16 (&sc)[N]) {
    float t = -INFINITY;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) t = fmaxf(t, sc[n][i]);
    return t;
}
// Weights of N 32-key blocks as the operands of O^T's product; returns their sum before
// the rounding (the log-sum-exp is an fp32 output).
template <int N>
__device__ __forceinline__ float weights_of(const floatx16 (&sc)[N], float scale, float nm,
                                            half8 (&pop)[2 * N]) {
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < 2 * N; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = fast_exp2(fmaf(sc[t / 2][8 * (t % 2) + e], scale, nm));
            pop[t][e] = static_cast<f16>(x);
            ps[e % 4] += x;
        }
    return (ps[0] + ps[1]) + (ps[2] + ps[3]);
}
// Stores a lane's dims 32 db + 8 q + 4 h + e of its pair: the output, or the partial.
template <int D>
__device__ __forceinline__ void store_pair(const BoundArgs& a, const PrefillPlan& p, const Pairs& x,
                                           int b, int h, int all_tiles, const floatx16 (&o)[D / 32],
                                           float m, float l) {
    if (!x.live) return;
    if (all_tiles > p.tiles_per_split) {   // joined by window_join_kernel
        const int64_t prow = x.at * p.nsplit + blockIdx.z;
        float* po = p.ws_o + prow * D + 4 * h;
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<floatx4*>(po + 32 * db + 8 * q4) =
                    floatx4{o[db][4 * q4], o[db][4 * q4 + 1], o[db][4 * q4 + 2], o[db][4 * q4 + 3]};
        if (h == 0) {
            p.ws_ml[prow * 2] = m * a.scale_log2;
            p.ws_ml[prow * 2 + 1] = l;
        }
        return;
    }
    const float inv = 1.f / l;
    f16* orow = a.out + x.at * D + 4 * h;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            half4 hv;
#pragma unroll
            for (int e = 0; e < 4; ++e) hv[e] = static_cast<f16>(o[db][4 * q4 + e] * inv);
            *reinterpret_cast<half4*>(orow + 32 * db + 8 * q4) = hv;
        }
    if (a.lse && h == 0)
        a.lse[((int64_t)b * a.Hq + x.qh) * a.rows + x.row] =
            fmaf(m, a.scale_log2, __builtin_amdgcn_logf(l)) * kLn2;
}
// LDS read offsets (halfs) inside a stage: K operand chunk c (+ 32 D per 32 keys), and V^T
// operand of 32-dim block db (+ 16 D per 16 keys, + 8 D for the second read).
template <int D, bool PAGED>
__device__ __forceinline__ void read_offsets(int lane, int (&kro)[D / 16], int (&vro)[D / 32]) {
    using K = Keys<D, PAGED>;
    const int h = lane >> 5, c32 = lane & 31, j16 = lane & 15, blk2 = (lane >> 4) & 1;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
        const int r = c32;
        kro[c] = r * D + 8 * ((2 * c + h) ^ K::kswz(r));
    }
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
        const int r = 4 * h + j16 / 4;
        const int ch = 4 * db + 2 * blk2 + ((j16 & 3) >> 1);
        vro[db] = r * D + 8 * (ch ^ K::vswz(r)) + 4 * (j16 & 1);
    }
}

// 128 pairs a workgroup of four waves, 32 a wave, two LDS stages per matrix: two workgroups
// share a CU, and each wave overlaps its own MFMAs and exponentials: iteration j runs S^T
// of tile j + 1 between the exponentials of tile j's first 32 keys, O^T of these between the
// other exponentials, and the rest of O^T beside the maxima of tile j + 1.
template <int D, bool PAGED>
__global__ void __launch_bounds__(kWaves * kWave) __attribute__((amdgpu_waves_per_eu(2)))
window_prefill_kernel(const BoundArgs a, const PrefillPlan p) {
    constexpr int NC = D / 16, NDB = D / 32, TB = kBN * D;
    using K = Keys<D, PAGED>;
    __shared__ __attribute__((aligned(16))) f16 kring[2 * TB];
    __shared__ __attribute__((aligned(16))) f16 vring[2 * TB];
    __shared__ int32_t ptab[PAGED ? kPages : 1];
    __shared__ uint32_t bad[kBadWords];

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int h = lane >> 5;
    const int kvh = blockIdx.x % a.Hkv;
    const int blk = p.blocks - 1 - static_cast<int>(blockIdx.x / a.Hkv);   // longest first
    const int b = blockIdx.y;
    const Block k = block_of(a, p, b, blk, kPairs);
    if (k.p_lo > k.p_hi) return;
    const int t_lo = static_cast<int>(blockIdx.z) * p.tiles_per_split;
    const int all_tiles = (k.nv + kBN - 1) / kBN;
    const int n = min(all_tiles - t_lo, p.tiles_per_split);
    if (n <= 0) return;
    const K keys(a, k, ptab, bad, b, kvh, t_lo, n);

    const Pairs x = pairs_at(a, p, k, b, kvh, blk * kPairs + 32 * wave, lane & 31);
    half8 qop[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
        qop[c] = x.live ? load_half8(a.q + x.at * D + 16 * c + 8 * h) : half8{};
    int kro[NC], vro[NDB];
    read_offsets<D, PAGED>(lane, kro, vro);
    floatx16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m_run = -1e30f, l_part = 0.f;
    const float lazy_thr = kLazyLog2 / a.scale_log2, ref = kRefLog2 / a.scale_log2;

    // Group g: K of tile g + 2 and V of tile g + 1, issued by iteration g into the stages
    // that iteration g - 1 was the last to read, and waited for by iteration g + 1.
    int pid_k, pid_v;
    auto issue = [&](int g) {
        keys.issue_k(g + 2, pid_k, kring + (g & 1) * TB);
        if (g >= -1) keys.issue_v(g + 1, pid_v, vring + (~g & 1) * TB);
        pid_v = pid_k;
        pid_k = keys.page(g + 3);
    };
    auto begin = [&](int j) {
        wait_ring<0>();
        if (j >= 0) keys.clean(j, vring + (j & 1) * TB);
        ring_barrier();
        issue(j);
    };
    auto qk = [&](int j, floatx16 (&s)[2]) {
        const f16* Kt = kring + (j & 1) * TB;
#pragma unroll
        for (int n2 = 0; n2 < 2; ++n2)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[n2][e] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int n2 = 0; n2 < 2; ++n2)
                s[n2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    *reinterpret_cast<const half8*>(&Kt[kro[c] + 32 * n2 * D]), qop[c], s[n2], 0, 0, 0);
    };
    auto exps = [&](const floatx16& s, half8 (&pop)[2]) {
        const floatx16 one[1] = {s};
        l_part += weights_of(one, a.scale_log2, -m_run * a.scale_log2, pop);
    };
    auto pv = [&](int j, int n2, const half8 (&pop)[2]) {
        const f16* Vt = vring + (j & 1) * TB + 32 * n2 * D;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int db = 0; db < NDB; ++db) {
                const f16* q = &Vt[vro[db] + 16 * t * D];
                o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    cat_half8(lds_read_tr16(q), lds_read_tr16(q + 8 * D)), pop[t], o[db], 0, 0, 0);
            }
    };
    // Masks tile j's scores; moves the reference where a row passes it by 2^15.
    float tmax;
    auto refer = [&](int j, floatx16 (&s)[2]) {
        if (mask(k, x, keys.window, t_lo + j, (t_lo + j) * kBN + 4 * h, s)) tmax = max_of(s);
        tmax = halves_max(tmax);
        if (__builtin_amdgcn_read_exec() & __ballot(tmax > m_run + lazy_thr)) {
            const float mn = fmaxf(m_run, tmax - ref);
            const float alpha = fast_exp2((m_run - mn) * a.scale_log2);
            l_part *= alpha;
#pragma unroll
            for (int db = 0; db < NDB; ++db) o[db] *= alpha;
            m_run = mn;
        }
    };
    // Iteration j < n - 1: tile j's scores in s, tile j + 1's go to sn.
    auto iterate = [&](int j, floatx16 (&s)[2], floatx16 (&sn)[2]) {
        half8 pa[2], pb[2];
        begin(j);
        refer(j, s);
        qk(j + 1, sn);
        exps(s[0], pa);
        pv(j, 0, pa);
        exps(s[1], pb);
        pv(j, 1, pb);
        tmax = max_of(sn);
        // One MFMA, the LDS reads of one four ahead, and its share of the 112 and then 56 + 22
        // exponentials, sums and maxima (262 us instead of 267 as the compiler orders them).
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int i = 0; i < 2 * NC; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x402, 4, 0);
        }
#pragma unroll
        for (int i = 0; i < 2 * NDB; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x402, 8, 0);
        }
#pragma unroll
        for (int i = 0; i < 2 * NDB; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x402, 3, 0);
        }
    };

    wait_ring<0>();   // q in registers before the ring: no other waits inside it
    __syncthreads();   // ptab, bad
    pid_k = pid_v = keys.page(0);
    issue(-2);
    floatx16 s0[2], s1[2];
    begin(-1);
    qk(0, s0);
    tmax = max_of(s0);
    int j = 0;
    for (; j + 2 < n; j += 2) {
        keys.more_pages(j);
        iterate(j, s0, s1);
        iterate(j + 1, s1, s0);
    }
    if (j + 1 < n) {
        iterate(j, s0, s1);
        ++j;
        s0[0] = s1[0];
        s0[1] = s1[1];
    }
    begin(j);   // j == n - 1
    refer(j, s0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        half8 pa[2];
        exps(s0[t], pa);
        pv(j, t, pa);
    }
    wait_ring<0>();   // the ring's trailing re-loads
    keys.add_back(o, x.live, x.pos);
    store_pair<D>(a, p, x, b, h, all_tiles, o, m_run, halves_sum(l_part));
}

// Joins the partials of the blocks that were cut into ranges of keys: R times D / 8 lanes
// per (row, head), lane (r, c) taking dims 8c .. of every R-th range.
template <int D, int R>
__global__ void __launch_bounds__(256) window_join_kernel(const BoundArgs a, const PrefillPlan p) {
    constexpr int LPR = D / 8;
    const int c = threadIdx.x % LPR, r = threadIdx.x / LPR % R;
    const int b = blockIdx.y;
    const uint32_t i = blockIdx.x * (256 / LPR / R) + threadIdx.x / (LPR * R);
    const int row = static_cast<int>(i / a.Hq), qh = static_cast<int>(i % a.Hq);
    if (row >= a.rows) return;
    const Block k = block_of(a, p, b, (row * a.G + qh - row_of(p, qh) * a.G) / kPairs, kPairs);
    const int64_t pos = (int64_t)k.first + row;
    if (pos < k.p_lo || pos > k.p_hi) return;
    const int tiles = (k.nv + kBN - 1) / kBN;
    if (tiles <= p.tiles_per_split) return;
    const int n = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
    const int64_t at = ((int64_t)b * a.rows + row) * a.Hq + qh;
    const float* po = p.ws_o + at * p.nsplit * D + 8 * c;
    const float2* pml = reinterpret_cast<const float2*>(p.ws_ml) + at * p.nsplit;
    float M = -3.0e38f, L = 0.f;
    floatx4 o0 = {0.f, 0.f, 0.f, 0.f}, o1 = o0;
    auto fold = [&](float m, float l, floatx4 x0, floatx4 x1) {
        const float mn = fmaxf(M, m);
        const float al = fast_exp2(M - mn), be = fast_exp2(m - mn);
        o0 = o0 * al + x0 * be;
        o1 = o1 * al + x1 * be;
        L = fmaf(L, al, l * be);
        M = mn;
    };
    auto some = [&](auto U_, int j0) {   // U ranges in flight
        constexpr int U = decltype(U_)::value;
        float2 ml[U];
        floatx4 x[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = min(j0 + R * u, n - 1);
            ml[u] = pml[j];
            x[u][0] = *reinterpret_cast<const floatx4*>(po + (int64_t)j * D);
            x[u][1] = *reinterpret_cast<const floatx4*>(po + (int64_t)j * D + 4);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + R * u < n) fold(ml[u].x, ml[u].y, x[u][0], x[u][1]);
    };
    if (n <= R)
        some(std::integral_constant<int, 1>{}, r);
    else
        for (int j0 = r; j0 < n; j0 += 4 * R) some(std::integral_constant<int, 4>{}, j0);
#pragma unroll
    for (int s = LPR; s < LPR * R; s <<= 1) {
        floatx4 x0, x1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x0[e] = __shfl_xor(o0[e], s);
            x1[e] = __shfl_xor(o1[e], s);
        }
        const float m = __shfl_xor(M, s), l = __shfl_xor(L, s);
        fold(m, l, x0, x1);
    }
    if (r > 0) return;
    const float inv = 1.f / L;
    half8 hv;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hv[e] = static_cast<f16>(o0[e] * inv);
        hv[4 + e] = static_cast<f16>(o1[e] * inv);
    }
    store_half8(a.out + at * D + 8 * c, hv);
    if (a.lse && c == 0)
        a.lse[((int64_t)b * a.Hq + qh) * a.rows + row] = (M + __builtin_amdgcn_logf(L)) * kLn2;
}

// Ranges of keys until every CU has two workgroups, each of at least 3 tiles.  (One sequence, us with at least 4 / 3 / 2 tiles: 16 rows of
// 32/8 heads of 64, window 500, 13.1 / 11.0 / 10.9, 4000 13.8 / 11.9 / 11.8; of 128 15.1 /
// 14.4 / 14.0; but 700 rows, window 200, 9.7 / 9.7 / 15.8: what the second launch costs.)
PrefillPlan plan_of(int batch, int rows, int hkv, int G, int max_len, int window, int sinks) {
    PrefillPlan p{};
    const int64_t pairs = (int64_t)rows * G;
    const int64_t wgs = (pairs + kPairs - 1) / kPairs * hkv * batch, per = kPairs;
    p.inv_g = G == 1 ? 0 : static_cast<uint32_t>(((uint64_t(1) << 32) + G - 1) / G);
    p.blocks = static_cast<int>((pairs + per - 1) / per);
    // the most keys that a block's rows see
    const int64_t block_rows = std::min<int64_t>((per + G - 1) / G + 1, rows);
    const int64_t keys = window > 0 ? std::min<int64_t>(max_len, (int64_t)window + sinks + block_rows + 2 * kPage)
                                    : max_len;
    const int64_t tiles = (keys + kBN - 1) / kBN;
    int64_t n = std::min<int64_t>(2 * kCUs / wgs, tiles / 3);
    n = std::max<int64_t>(n, 1);
    p.tiles_per_split = static_cast<int>((tiles + n - 1) / n);
    p.nsplit = static_cast<int>((tiles + p.tiles_per_split - 1) / p.tiles_per_split);
    return p;
}

}  // namespace

size_t window_prefill_workspace(int batch, int rows, int hq, int hkv, int d, int max_len,
                                int window, int sinks) {
    if (rows <= 0 || !bound_sizes(batch, hq, hkv, max_len, window, sinks) ||
        (int64_t)rows * hq > kMaxRowHeads || (d != 64 && d != 128))
        return 0;
    const PrefillPlan p = plan_of(batch, rows, hkv, hq / hkv, max_len, window, sinks);
    return p.nsplit == 1 ? 0 : sizeof(float) * (size_t)batch * rows * hq * p.nsplit * (d + 2);
}

bool window_prefill_fits(const BoundArgs& a, int batch) {
    if ((int64_t)a.rows * a.Hq > kMaxRowHeads) return false;   // the plan counts them in an int
    const PrefillPlan p = plan_of(batch, a.rows, a.Hkv, a.G, a.max_len, a.window, a.sinks);
    return (a.D == 64 || a.D == 128) && p.nsplit <= 65535 &&
           (int64_t)p.blocks * a.Hkv <= kMaxRowHeads / kPairs && a.k.stride_s < kMaxStride &&
           (int64_t)a.rows * a.G * a.G < (int64_t)1 << 31 &&   // row_of, and pairs in an int
           a.v.stride_s < kMaxStride;
}

int window_prefill(const BoundArgs& a, int batch, bool paged, void* ws, hipStream_t s) {
    PrefillPlan p = plan_of(batch, a.rows, a.Hkv, a.G, a.max_len, a.window, a.sinks);
    const size_t rh = (size_t)batch * a.rows * a.Hq;
    p.ws_o = static_cast<float*>(ws);
    p.ws_ml = p.ws_o + rh * p.nsplit * a.D;
    const dim3 grid(p.blocks * a.Hkv, batch, p.nsplit);
    auto flag = [](bool x, auto f) { x ? f(std::true_type{}) : f(std::false_type{}); };
    flag(a.D == 64, [&](auto d64) {
        flag(paged, [&](auto pg) {
            hipLaunchKernelGGL((window_prefill_kernel<decltype(d64)::value ? 64 : 128,
                                                      decltype(pg)::value>),
                               grid, dim3(kWaves * kWave), 0, s, a, p);
        });
    });
    const int rc = check_launch("window_prefill");
    if (rc || p.nsplit == 1) return rc;
    // A wave per (row, head) while they all run at once (16 rows of 32 heads over 16 ranges
    // 13 us instead of 17), D / 8 lanes above (512 rows of 32 heads over 4: 48.8 instead of
    // 52.4, rounds of waves that wait for their first loads).
    const int64_t heads = (int64_t)batch * a.rows * a.Hq;   // rows Hq <= 2^29
    auto join = [&](auto kernel, int lanes) {
        const unsigned per = 256 / lanes;
        hipLaunchKernelGGL(kernel, dim3((static_cast<unsigned>(a.rows) * a.Hq + per - 1) / per, batch),
                           dim3(256), 0, s, a, p);
    };
    if (a.D == 64)
        heads <= 32 * kCUs ? join(window_join_kernel<64, 8>, 64) : join(window_join_kernel<64, 1>, 8);
    else
        heads <= 32 * kCUs ? join(window_join_kernel<128, 4>, 64) : join(window_join_kernel<128, 1>, 16);
    return check_launch("window_prefill (join)");
}

}  // namespace kvhp
