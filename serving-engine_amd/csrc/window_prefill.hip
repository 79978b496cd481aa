// window_prefill.hip -- rows of prompts and chunks attending a sliding window
// and the first tokens of their sequence, over a cache view (gfx950, head_dim
// 64 and 128).
//
// A workgroup of 8 waves takes one KV head of one sequence and 256 (KG = 1) or
// 128 (KG = 2) of its (row, query head) pairs, query head fastest: 32 pairs a
// wave, whatever the group size, so the heads of a group share the K/V tiles and
// a chunk of a few rows still fills a wave.  With KG = 2 two wave groups take
// the same pairs and half the keys of every tile, and join at the end.
//
// Keys: those that some row of the block sees, numbered through without the pages
// between the first tokens' and the earliest window's: `nv` keys, 64 to a tile.  (The
// gap is whole pages so that the rows of a load share a page, whose id is then
// scalar; the rest of the two pages at its edges is masked.)
// A block of a long prompt walks (window + sinks + its rows) / 64 tiles, all
// blocks alike, where causal attention would walk up to S / 64.  Only tiles at the
// window's two edges and those that hold first tokens need a mask.
//
// Per tile, on v_mfma_f32_32x32x16_f16 with one lane per pair:
//   S^T = K Q^T; fp32 online softmax in the log2 domain whose reference maximum
//   moves when a row passes it by 2^8 (weights up to 2^8 stay far inside fp16's
//   range, to which they are rounded for the product: 2^-11 each, over a sum of
//   many); O^T += V^T P^T.
// K and V rows go from memory to a ring of four LDS stages without registers
// (global_load_lds, a scalar base and the lane's fixed offset; page ids from LDS), two
// tiles ahead; rows are stored with their 16-byte chunks XOR-swizzled so that
// both operand reads touch all banks.  Waves 0-3 and 4-7, one of each per SIMD,
// alternate a step of MFMAs and a step of exponentials.
//
// A masked key's weight is 0, but 0 times an infinite or NaN V is NaN: in the
// tiles that some row sees only in part such elements are set to 0 in LDS, noted,
// and added as they are at the end to the rows that see their key.
//
// Few rows over a long cache are cut into ranges of keys (blockIdx.z) whose
// partials a second launch joins.
//
// Bound by the MFMA and exponential units: 4 D flops per visible (key, pair).
#include "bounded.h"

#include <algorithm>
#include <type_traits>

namespace kvhp {
namespace {

constexpr int kBN = 64;               // keys per tile
constexpr int kPages = 4088;          // page ids of a split held in LDS
constexpr int kMaxStride = 1 << 24;   // halfs between rows: 15 rows stay below 2^31 bytes
constexpr int kEdge = 6;              // tiles at either edge of the window in a block
constexpr int kBadWords = 4 * kEdge;  // a bit per key of those
constexpr int kCUs = 256;
constexpr float kLazyLog2 = 8.f;

typedef short short4v __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) short4v lds_short4v;
typedef __attribute__((address_space(3))) f16 lds_f16;
typedef __attribute__((address_space(3))) void lds_void;

__device__ __forceinline__ short4v lds_read_tr16(const f16* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4v*)(lds_f16*)p);
}
__device__ __forceinline__ half8 cat_half8(short4v lo, short4v hi) {
    return __builtin_bit_cast(half8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// 16 bytes from a scalar base and lane l's byte offset to lds_base + 16 l; only the
// ring's own waits order it.
__device__ __forceinline__ void dma16s(const char* base, uint32_t voff, f16* lds_base) {
    const uint32_t m0v = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((lds_void*)(lds_f16*)lds_base));
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(m0v), "v"(voff), "s"(base) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}
// A workgroup barrier that leaves the ring's loads in flight.
__device__ __forceinline__ void ring_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ float halves_max(float x) {
    auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
    auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(t[0]) + __uint_as_float(t[1]);
}

struct PrefillPlan {
    int kg;
    int blocks;            // of pairs, per sequence and KV head
    int tiles_per_split, nsplit;
    float* ws_o;           // [batch * rows * Hq][nsplit][D]
    float* ws_ml;          // [batch * rows * Hq][nsplit][2], the maximum in log2 units
};

// The rows of a block that lie in their sequence, and the keys they see.
struct Block {
    int first;       // position of row 0
    int p_lo, p_hi;  // positions of the block's first and last live row; none: p_lo > p_hi
    int sinks;       // first tokens that every row sees
    int head;        // keys in front of the gap: up to the end of their page
    int shift;       // the gap, whole pages; 0: none (head is 0 then)
    int nv;          // keys, numbered through: v < head is key v, others key v + shift
};
__device__ __forceinline__ Block block_of(const BoundArgs& a, int b, int blk, int pairs) {
    Block k;
    const int n = bound_len(a, b);
    // a start outside +-2^30 leaves no row among at most 2^30 keys
    const int64_t first = min(max(bound_first(a, b, n), -(int64_t)(1 << 30)), (int64_t)(1 << 30));
    const int64_t r0 = (int64_t)blk * pairs / a.G;
    const int64_t r1 = min(((int64_t)(blk + 1) * pairs - 1) / a.G, (int64_t)a.rows - 1);
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

template <int D, int KG, bool PAGED>
__global__ void __launch_bounds__(8 * kWave)
window_prefill_kernel(const BoundArgs a, const PrefillPlan p) {
    constexpr int WAVES = 8, UPG = WAVES / KG, NTH = WAVES * kWave;
    constexpr int NC = D / 16, NDB = D / 32, CPR = D / 8, RPI = kWave / CPR;
    constexpr int IPW = kBN / RPI / WAVES;   // loads per wave per matrix
    constexpr int LPT = 2 * IPW;
    constexpr int TB = kBN * D, NSTAGE = 4;
    constexpr int NKB = 2 / KG;              // this wave's 32-key blocks per tile
    auto kswz = [](int r) { return CPR == 16 ? r & 15 : r >> 1 & 7; };
    auto vswz = [](int r) { return CPR == 16 ? 4 * (r & 3) : (r & 3) << 1; };

    __shared__ __attribute__((aligned(16))) f16 ring[NSTAGE * 2 * TB];
    __shared__ int32_t ptab[PAGED ? kPages : 1];
    __shared__ uint32_t bad_keys[kBadWords];

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int h = lane >> 5, c32 = lane & 31, j16 = lane & 15, blk2 = (lane >> 4) & 1;
    const int kvh = blockIdx.x % a.Hkv;
    const int blk = p.blocks - 1 - static_cast<int>(blockIdx.x / a.Hkv);   // longest first
    const int b = blockIdx.y;
    const Block k = block_of(a, b, blk, 32 * UPG);
    if (k.p_lo > k.p_hi) return;
    const int t_lo = static_cast<int>(blockIdx.z) * p.tiles_per_split;
    const int all_tiles = (k.nv + kBN - 1) / kBN;
    const int n_tiles = min(all_tiles - t_lo, p.tiles_per_split);
    if (n_tiles <= 0) return;
    const int last_tile = n_tiles - 1;
    const int window = a.window > 0 ? a.window : INT32_MAX;

    const char* kb = reinterpret_cast<const char*>(
        a.k.data + (PAGED ? 0 : b * a.k.stride_b) + kvh * a.k.stride_h);
    const char* vb = reinterpret_cast<const char*>(
        a.v.data + (PAGED ? 0 : b * a.v.stride_b) + kvh * a.v.stride_h);
    const uint64_t ssk = 2 * (uint64_t)a.k.stride_s, ssv = 2 * (uint64_t)a.v.stride_s;

    // ---- page ids of this split's keys, 16 to a page
    if constexpr (PAGED) {
        const int v0 = t_lo * kBN, v1 = min((t_lo + n_tiles) * kBN, k.nv);
        for (int i = tid; i < (v1 - v0 + kPage - 1) / kPage; i += NTH) {
            const int v = v0 + i * kPage;
            const int pid = a.k.bt[(int64_t)b * a.k.max_pages + ((v < k.head ? v : v + k.shift) >> 4)];
            ptab[i] = min(max(pid, 0), a.k.num_pages - 1);
        }
    }
    if (tid < kBadWords) bad_keys[tid] = 0;

    // ---- this wave's pairs; its half of every tile's keys with KG = 2
    const int u = wave % UPG, kgrp = wave / UPG;
    const int64_t pair = ((int64_t)blk * UPG + u) * 32 + c32;
    const int row = static_cast<int>(pair / a.G), qh = kvh * a.G + static_cast<int>(pair % a.G);
    const int pos = k.first + row;
    const bool live = row < a.rows && pos >= k.p_lo && pos <= k.p_hi;
    const int64_t at = ((int64_t)b * a.rows + row) * a.Hq + qh;
    half8 qop[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c)
        qop[c] = live ? load_half8(a.q + at * D + 16 * c + 8 * h) : half8{};
    // positions of the wave's first and last pair's rows, and whether all are live
    const int u_lo = k.first + static_cast<int>((((int64_t)blk * UPG + u) * 32) / a.G);
    const int u_hi = k.first + static_cast<int>((((int64_t)blk * UPG + u) * 32 + 31) / a.G);
    const bool u_live = u_lo >= k.p_lo && u_hi <= k.p_hi;

    // ---- DMA: this wave's rows (wave * IPW + i) * RPI + lane / CPR of a tile, those of a
    //      load in one page.  Tiles past the last re-load it, so every wave issues the
    //      same loads; rows past the last key re-read it.
    const uint32_t ssk32 = static_cast<uint32_t>(ssk), ssv32 = static_cast<uint32_t>(ssv);
    uint32_t ko[IPW], vo[IPW];   // the lane's offsets inside the load's rows
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
        const int r0 = (wave * IPW + i) * RPI, r = r0 + lane / CPR;
        ko[i] = (r - r0) * ssk32 + 16 * ((lane % CPR) ^ kswz(r));
        vo[i] = (r - r0) * ssv32 + 16 * ((lane % CPR) ^ vswz(r));
    }
    int pid_next[IPW];   // pages of the next issue, read one ahead
    auto pages_of = [&](int tt) {
        if constexpr (PAGED)
#pragma unroll
            for (int i = 0; i < IPW; ++i) {
                const int v = min((t_lo + min(tt, last_tile)) * kBN + (wave * IPW + i) * RPI, k.nv - 1);
                pid_next[i] = ptab[(v >> 4) - t_lo * (kBN / kPage)];
            }
    };
    auto issue = [&](int tt) {
        f16* stg = ring + (tt % NSTAGE) * 2 * TB;
        const int k0 = (t_lo + min(tt, last_tile)) * kBN;
#pragma unroll
        for (int i = 0; i < IPW; ++i) {
            const int r0 = (wave * IPW + i) * RPI;
            const int v = min(k0 + r0, k.nv - 1);   // the load's first row
            const int key = v < k.head ? v : v + k.shift;
            int64_t row = key;
            if constexpr (PAGED)
                row = (int64_t)__builtin_amdgcn_readfirstlane(pid_next[i]) * kPage + (key & 15);
            uint32_t x = ko[i], y = vo[i];
            if (k0 + r0 + RPI > k.nv) {   // some of them lie past the last key
                const int r = min(lane / CPR, k.nv - 1 - v);
                x += (r - lane / CPR) * ssk32;
                y += (r - lane / CPR) * ssv32;
            }
            dma16s(kb + row * (int64_t)ssk, x, stg + r0 * D);
            dma16s(vb + row * (int64_t)ssv, y, stg + TB + r0 * D);
        }
        pages_of(tt + 1);
    };
    int kro[NC], vro[NDB];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int r = 32 * kgrp + c32;
        kro[c] = r * D + 8 * ((2 * c + h) ^ kswz(r));
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
        const int r = 32 * kgrp + 4 * h + j16 / 4;
        const int ch = 4 * db + 2 * blk2 + ((j16 & 3) >> 1);
        vro[db] = r * D + 8 * (ch ^ vswz(r)) + 4 * (j16 & 1);
    }
    floatx16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m_run = -1e30f, l_part = 0.f;
    const float lazy_thr = kLazyLog2 / a.scale_log2;

    wait_vmcnt<0>();   // q in registers before the ring: no other waits inside it
    __syncthreads();   // ptab, bad_keys
    pages_of(0);
    issue(0);
    issue(1);

    auto qk = [&](const f16* Kt, floatx16 (&sc)[NKB]) {
#pragma unroll
        for (int kb2 = 0; kb2 < NKB; ++kb2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kb2][i] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const half8 kop = *reinterpret_cast<const half8*>(&Kt[kro[c] + 32 * kb2 * D]);
                sc[kb2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kop, qop[c], sc[kb2], 0, 0, 0);
            }
        }
    };
    floatx16 sc[NKB];
    half8 pop[2 * NKB];
#pragma unroll
    for (int t = 0; t < 2 * NKB; ++t) pop[t] = half8{};
    auto pv = [&](int j) {
        const f16* Vt = ring + (j % NSTAGE) * 2 * TB + TB;
#pragma unroll
        for (int t = 0; t < 2 * NKB; ++t)
#pragma unroll
            for (int db = 0; db < NDB; ++db) {
                const f16* p1 = &Vt[vro[db] + 16 * t * D];
                const half8 vop = cat_half8(lds_read_tr16(p1), lds_read_tr16(p1 + 8 * D));
                o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vop, pop[t], o[db], 0, 0, 0);
            }
    };
    constexpr int NQK = NKB * NC, NPV = 2 * NKB * NDB, PF = 8;
    auto mstep = [&](int j) {   // S^T of tile j, O^T of tile j - 1, operand reads PF ahead
        __builtin_amdgcn_s_setprio(1);
        qk(ring + (j % NSTAGE) * 2 * TB, sc);
        pv(j - 1);
        __builtin_amdgcn_sched_group_barrier(0x100, PF, 0);
#pragma unroll
        for (int i = 0; i < NQK - PF; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
#pragma unroll
        for (int i = 0; i < NPV; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, PF, 0);
        __builtin_amdgcn_s_setprio(0);
    };
    auto sstep = [&](int j) {
        const int k0 = (t_lo + j) * kBN;
        // element (kb2, i) is key k0 + 32 (kb2 + kgrp) + 4h + 8 (i / 4) + i % 4
        const int v0 = k0 + 32 * kgrp + 4 * h;
        if (k0 + kBN - 1 + k.shift > u_lo || !u_live) {   // keys past some pair's row
            const int hi = live ? pos - k.shift - v0 : -1;
#pragma unroll
            for (int kb2 = 0; kb2 < NKB; ++kb2)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    sc[kb2][i] = 32 * kb2 + 8 * (i / 4) + (i % 4) > hi ? -INFINITY : sc[kb2][i];
        }
        if (u_hi - (k0 + k.shift) >= window && k0 + kBN > k.sinks) {   // keys that a window left
            const int64_t left = (int64_t)pos - window - k.shift - v0;
            const int head = k.sinks - v0;   // from it on and up to `left`
            const uint32_t span = static_cast<uint32_t>(max(left - head + 1, (int64_t)0));
#pragma unroll
            for (int kb2 = 0; kb2 < NKB; ++kb2)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    sc[kb2][i] = static_cast<uint32_t>(32 * kb2 + 8 * (i / 4) + (i % 4) - head) < span
                                     ? -INFINITY : sc[kb2][i];
        }
        float tmax = -INFINITY;
#pragma unroll
        for (int kb2 = 0; kb2 < NKB; ++kb2)
#pragma unroll
            for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, sc[kb2][i]);
        tmax = halves_max(tmax);
        if (__builtin_amdgcn_read_exec() & __ballot(tmax > m_run + lazy_thr)) {
            const float mn = fmaxf(m_run, tmax);
            const float alpha = fast_exp2((m_run - mn) * a.scale_log2);
            l_part *= alpha;
#pragma unroll
            for (int db = 0; db < NDB; ++db) o[db] *= alpha;
            m_run = mn;
        }
        const float nmc = -m_run * a.scale_log2;
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < 2 * NKB; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = fast_exp2(fmaf(sc[t / 2][8 * (t % 2) + e], a.scale_log2, nmc));
                pop[t][e] = static_cast<f16>(x);
                ps[e % 4] += x;
            }
        // of the unrounded weights: the log-sum-exp is an fp32 output
        l_part += (ps[0] + ps[1]) + (ps[2] + ps[3]);
    };
    // Tiles that some row of the block sees in part: from `edge_hi` on (keys past the
    // first row), and from `edge_lo`, the first behind the first tokens, to the last key
    // that the last row's window has left.
    const int edge_hi = max(k.p_lo - k.shift + 1, 0) / kBN;
    const int edge_lo = k.sinks / kBN;
    const int64_t left = (int64_t)k.p_hi - window - k.shift;   // that key
    auto edge_word = [&](int t) {   // first word of tile t's bits, or -1
        if (t >= edge_hi) return 2 * kEdge + 2 * (t - edge_hi);
        return t >= edge_lo && (int64_t)t * kBN <= left ? 2 * (t - edge_lo) : -1;
    };
    auto clean = [&](int j) {   // this wave's rows of the tile, just landed
        const int word = edge_word(t_lo + j);
        if (word < 0) return;
        f16* Vt = ring + (j % NSTAGE) * 2 * TB + TB + wave * IPW * RPI * D + 8 * lane;
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
            atomicOr(&bad_keys[word + (r >> 5)], 1u << (r & 31));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] &= ~(m[e] | (m[e] - (m[e] >> 15)));
            *reinterpret_cast<u32x4*>(Vt + i * RPI * D) = x;
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): written before the barrier
    };
    // Phase 2j: waves 0-3 MFMAs of tile j, waves 4-7 exponentials of tile j - 1;
    // phase 2j + 1 the other way round.  Tile j + 2 is issued when phase 2j begins,
    // into the stage of tile j - 2, whose last reader ran in phase 2j - 1.
    auto phase_start = [&](int j) {
        wait_vmcnt<LPT>();
        if (j < n_tiles) clean(j);
        ring_barrier();
        issue(j + 2);
    };
    if ((wave >> 2) == 0) {
        phase_start(0);
        qk(ring, sc);
        ring_barrier();
        sstep(0);
        for (int j = 1; j < n_tiles; ++j) {
            phase_start(j);
            mstep(j);
            ring_barrier();
            sstep(j);
        }
        phase_start(n_tiles);
        pv(n_tiles - 1);
        ring_barrier();
    } else {
        phase_start(0);
        ring_barrier();
        qk(ring, sc);
        for (int j = 1; j < n_tiles; ++j) {
            phase_start(j);
            sstep(j - 1);
            ring_barrier();
            mstep(j);
        }
        phase_start(n_tiles);
        sstep(n_tiles - 1);
        ring_barrier();
        pv(n_tiles - 1);
    }
    wait_vmcnt<0>();   // the ring's trailing re-loads

    if constexpr (KG == 2) {
        float* xo = reinterpret_cast<float*>(ring);
        float* xml = xo + UPG * NDB * 16 * kWave;
        ring_barrier();
        if (kgrp == 1) {
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4)
                    *reinterpret_cast<floatx4*>(&xo[(((u * NDB + db) * 4 + q4) * kWave + lane) * 4]) =
                        floatx4{o[db][4 * q4], o[db][4 * q4 + 1], o[db][4 * q4 + 2],
                                o[db][4 * q4 + 3]};
            xml[(u * kWave + lane) * 2] = m_run;
            xml[(u * kWave + lane) * 2 + 1] = l_part;
        }
        __syncthreads();
        if (kgrp == 1) return;
        const float m1 = xml[(u * kWave + lane) * 2];
        const float l1 = xml[(u * kWave + lane) * 2 + 1];
        const float mn = fmaxf(m_run, m1);
        const float a0 = fast_exp2((m_run - mn) * a.scale_log2);
        const float a1 = fast_exp2((m1 - mn) * a.scale_log2);
        m_run = mn;
        l_part = l_part * a0 + l1 * a1;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const floatx4 v4 = *reinterpret_cast<const floatx4*>(
                    &xo[(((u * NDB + db) * 4 + q4) * kWave + lane) * 4]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    o[db][4 * q4 + e] = o[db][4 * q4 + e] * a0 + v4[e] * a1;
            }
    }

    // ---- the V elements left out, to the rows that see their keys
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < kBadWords; ++i) any |= bad_keys[i];
    if (__builtin_amdgcn_readfirstlane(any)) {
#pragma unroll 1
        for (int i = 0; i < 32 * kBadWords; ++i) {
            if (!(bad_keys[i >> 5] >> (i & 31) & 1)) continue;
            const int e = i % (kEdge * kBN);
            const int v = (i < kEdge * kBN ? edge_lo : edge_hi) * kBN + e;
            if (v >= k.nv) continue;   // a repeated row
            const int key = v < k.head ? v : v + k.shift;
            uint64_t s = key;
            if constexpr (PAGED)
                s = (uint64_t)ptab[(v >> 4) - t_lo * (kBN / kPage)] * kPage + (v & 15);
            const f16* src = reinterpret_cast<const f16*>(vb + s * ssv) + 4 * h;
            const bool sees = live && key <= pos && (key < a.sinks || pos - key < window);
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
                for (int q4 = 0; q4 < 4; ++q4) {
                    const half4 x4 = *reinterpret_cast<const half4*>(src + 32 * db + 8 * q4);
#pragma unroll
                    for (int e4 = 0; e4 < 4; ++e4) {
                        const float x = static_cast<float>(x4[e4]);
                        if (sees && !(fabsf(x) < INFINITY)) o[db][4 * q4 + e4] += x;
                    }
                }
        }
    }

    const float lt = halves_sum(l_part);
    if (!live) return;
    if (all_tiles > p.tiles_per_split) {   // joined by window_join_kernel
        const int64_t prow = at * p.nsplit + blockIdx.z;
        float* po = p.ws_o + prow * D + 4 * h;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *reinterpret_cast<floatx4*>(po + 32 * db + 8 * q4) =
                    floatx4{o[db][4 * q4], o[db][4 * q4 + 1], o[db][4 * q4 + 2], o[db][4 * q4 + 3]};
        if (h == 0) {
            p.ws_ml[prow * 2] = m_run * a.scale_log2;
            p.ws_ml[prow * 2 + 1] = lt;
        }
        return;
    }
    const float inv = 1.f / lt;
    f16* orow = a.out + at * D + 4 * h;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) {
            half4 hv;
#pragma unroll
            for (int e = 0; e < 4; ++e) hv[e] = static_cast<f16>(o[db][4 * q4 + e] * inv);
            *reinterpret_cast<half4*>(orow + 32 * db + 8 * q4) = hv;
        }
    if (a.lse && h == 0)
        a.lse[((int64_t)b * a.Hq + qh) * a.rows + row] =
            fmaf(m_run, a.scale_log2, __builtin_amdgcn_logf(lt)) * kLn2;
}

// Joins the partials of the blocks that were cut into ranges of keys, 8 dims of a
// (row, head) a thread.
__global__ void __launch_bounds__(256)
window_join_kernel(const BoundArgs a, const PrefillPlan p, int pairs, int64_t threads) {
    const int64_t t = blockIdx.x * (int64_t)256 + threadIdx.x;
    if (t >= threads) return;
    const int cpr = a.D / 8, c = static_cast<int>(t % cpr);
    const int64_t at = t / cpr;   // (sequence, row, head)
    const int qh = static_cast<int>(at % a.Hq);
    const int row = static_cast<int>(at / a.Hq % a.rows), b = static_cast<int>(at / a.Hq / a.rows);
    const int blk = static_cast<int>(((int64_t)row * a.G + qh % a.G) / pairs);
    const Block k = block_of(a, b, blk, pairs);
    const int64_t pos = (int64_t)k.first + row;
    if (pos < k.p_lo || pos > k.p_hi) return;
    const int tiles = (k.nv + kBN - 1) / kBN;
    if (tiles <= p.tiles_per_split) return;
    const int n = (tiles + p.tiles_per_split - 1) / p.tiles_per_split;
    const float* po = p.ws_o + at * p.nsplit * a.D + 8 * c;
    const float2* pml = reinterpret_cast<const float2*>(p.ws_ml) + at * p.nsplit;
    float M = -3.0e38f, L = 0.f;
    floatx4 o0 = {0.f, 0.f, 0.f, 0.f}, o1 = o0;
    constexpr int U = 4;
    for (int j0 = 0; j0 < n; j0 += U) {
        float2 ml[U];
        floatx4 x[U][2];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int j = min(j0 + i, n - 1);
            ml[i] = pml[j];
            x[i][0] = *reinterpret_cast<const floatx4*>(po + (int64_t)j * a.D);
            x[i][1] = *reinterpret_cast<const floatx4*>(po + (int64_t)j * a.D + 4);
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (j0 + i >= n) continue;
            const float mn = fmaxf(M, ml[i].x);
            const float al = fast_exp2(M - mn), be = fast_exp2(ml[i].x - mn);
            o0 = o0 * al + x[i][0] * be;
            o1 = o1 * al + x[i][1] * be;
            L = fmaf(L, al, ml[i].y * be);
            M = mn;
        }
    }
    const float inv = 1.f / L;
    half8 hv;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hv[e] = static_cast<f16>(o0[e] * inv);
        hv[4 + e] = static_cast<f16>(o1[e] * inv);
    }
    store_half8(a.out + at * a.D + 8 * c, hv);
    if (a.lse && c == 0)
        a.lse[((int64_t)b * a.Hq + qh) * a.rows + row] = (M + __builtin_amdgcn_logf(L)) * kLn2;
}

// A KG = 2 workgroup takes about 0.57 of a KG = 1 one's time over half the pairs, so
// it pays where it adds less than that to the rounds of CUs.  Key ranges where the
// workgroups still leave CUs idle: of at least 4 tiles, and as many as keep a
// range's page ids in LDS.
PrefillPlan plan_of(int batch, int rows, int hkv, int G, int max_len, int window, int sinks) {
    PrefillPlan p{};
    const int64_t pairs = (int64_t)rows * G;
    const int64_t wg1 = (pairs + 255) / 256 * hkv * batch, wg2 = (pairs + 127) / 128 * hkv * batch;
    const auto rounds = [](int64_t n) { return (n + kCUs - 1) / kCUs; };
    p.kg = 57 * rounds(wg2) < 100 * rounds(wg1) ? 2 : 1;
    const int64_t per = p.kg == 2 ? 128 : 256, wgs = p.kg == 2 ? wg2 : wg1;
    p.blocks = static_cast<int>((pairs + per - 1) / per);
    // the most keys that a block's rows see
    const int64_t block_rows = std::min<int64_t>((per + G - 1) / G + 1, rows);
    const int64_t keys = window > 0 ? std::min<int64_t>(max_len, (int64_t)window + sinks + block_rows + 2 * kPage)
                                    : max_len;
    const int64_t tiles = (keys + kBN - 1) / kBN;
    int64_t n = std::min<int64_t>(kCUs / wgs, tiles / 4);
    n = std::max<int64_t>(n, (tiles * (kBN / kPage) + kPages - 5) / (kPages - 4));
    n = std::max<int64_t>(n, 1);
    p.tiles_per_split = static_cast<int>((tiles + n - 1) / n);
    p.nsplit = static_cast<int>((tiles + p.tiles_per_split - 1) / p.tiles_per_split);
    return p;
}

}  // namespace

size_t window_prefill_workspace(int batch, int rows, int hq, int hkv, int d, int max_len,
                                int window, int sinks) {
    if (batch <= 0 || rows <= 0 || hkv <= 0 || hq < hkv || hq % hkv || max_len <= 0 || window < 0 ||
        sinks < 0 || (d != 64 && d != 128))
        return 0;
    const PrefillPlan p = plan_of(batch, rows, hkv, hq / hkv, max_len, window, sinks);
    return p.nsplit == 1 ? 0 : sizeof(float) * (size_t)batch * rows * hq * p.nsplit * (d + 2);
}

bool window_prefill_fits(const BoundArgs& a, int batch) {
    const PrefillPlan p = plan_of(batch, a.rows, a.Hkv, a.G, a.max_len, a.window, a.sinks);
    return (a.D == 64 || a.D == 128) && p.nsplit <= 65535 &&
           (int64_t)p.blocks * a.Hkv <= 1 << 22 && a.k.stride_s < kMaxStride &&
           a.v.stride_s < kMaxStride;
}

int window_prefill(const BoundArgs& a, int batch, bool paged, void* ws, hipStream_t s) {
    PrefillPlan p = plan_of(batch, a.rows, a.Hkv, a.G, a.max_len, a.window, a.sinks);
    const size_t rh = (size_t)batch * a.rows * a.Hq;
    p.ws_o = static_cast<float*>(ws);
    p.ws_ml = p.ws_o + rh * p.nsplit * a.D;
    const dim3 grid(p.blocks * a.Hkv, batch, p.nsplit), blk(8 * kWave);
    auto flag = [](bool x, auto f) { x ? f(std::true_type{}) : f(std::false_type{}); };
    flag(a.D == 64, [&](auto d64) {
        flag(p.kg == 2, [&](auto two) {
            flag(paged, [&](auto pg) {
                hipLaunchKernelGGL((window_prefill_kernel<decltype(d64)::value ? 64 : 128,
                                                          decltype(two)::value ? 2 : 1,
                                                          decltype(pg)::value>),
                                   grid, blk, 0, s, a, p);
            });
        });
    });
    const int rc = check_launch("window_prefill");
    if (rc || p.nsplit == 1) return rc;
    const int64_t threads = (int64_t)rh * (a.D / 8);
    hipLaunchKernelGGL(window_join_kernel, dim3(static_cast<unsigned>((threads + 255) / 256)),
                       dim3(256), 0, s, a, p, p.kg == 2 ? 128 : 256, threads);
    return check_launch("window_prefill (join)");
}

}  // namespace kvhp
