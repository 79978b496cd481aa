// prompt_weights.hip -- the attention weights that rows of a prompt gave each cached
// key, summed over the rows and the query heads of its KV head (gfx950, head_dim 64
// and 128):  w_j = sum over rows i that see j, heads g, of exp(q_ig . k_j / sqrt(D) - lse_ig).
//
// The log-sum-exps are known, so this is one product and one pass.  A workgroup of
// four waves holds 32 keys a wave as MFMA operands in registers and walks
// the (row, head) pairs, head fastest, in tiles of 64 that go from memory to a ring
// of three LDS stages without registers:  S^T = K Q^T on v_mfma_f32_32x32x16_f16
// gives a lane one pair and 16 keys per block, so the sum over pairs stays in the
// lane until the end, where 32 lanes are added once.  Keys are the operand that
// stays because their sums do; walking keys instead would add lanes per tile.
//
// A wave runs the MFMAs of the next 32 pairs between the exponentials of the present
// ones.  Tiles whose pairs see none of its keys are passed over; pairs that see some are
// masked by a select (a NaN score of an unseen pair must not count).  Long prompts
// are cut into ranges of pairs whose sums a second launch adds in order, so the
// result does not depend on timing.
//
// Per 32 x 32 scores at D = 128 a wave runs 8 MFMAs of 32 cycles and 16 times (fma, exp,
// add) of 24: over a prompt of 4096 rows of 32/8 heads (69 GFLOP) 28 us and 41, and the
// LDS reads of the pairs some 30; the call takes 109 (0.63 PFLOP/s).  Three workgroups share a CU; with 64 keys a
// wave, which would halve the reads of the pairs from LDS, registers spill (136 to 300 us).
#include "bounded.h"

#include <algorithm>

namespace kvhp {
namespace {

constexpr int kWaves = 4;
constexpr int kTile = 64;        // pairs per tile
constexpr int kStages = 3;
constexpr int KB = 32 * kWaves;  // keys per workgroup
constexpr int kMaxPairs = 1024;  // pairs per range, whose log-sum-exps LDS holds

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) f16 lds_f16;
typedef __attribute__((address_space(3))) void lds_void;

struct SumPlan {
    int range;        // pairs per range, a multiple of kTile
    int nrange;
    int keys_pitch;
    uint32_t inv_g;   // ceil(2^32 / G), 0 for G = 1
    float* ws;        // [nrange][batch][Hkv][keys_pitch], nrange > 1
};

// Row of a pair: pair / G, exact for pair * G below 2^32.
__device__ __forceinline__ uint32_t row_of(const SumPlan& p, uint32_t pair) {
    return p.inv_g ? __umulhi(pair, p.inv_g) : pair;
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
__device__ __forceinline__ void ring_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The live rows' positions [p0, p1] of a sequence (p0 > p1: none).
struct Rows {
    int64_t first;
    int p0, p1;
};
__device__ __forceinline__ Rows rows_of(const BoundArgs& a, int b, int n) {
    Rows r;
    r.first = bound_first(a, b, n);
    r.p0 = static_cast<int>(min(max(r.first, (int64_t)0), (int64_t)n));
    r.p1 = static_cast<int>(max(min(r.first + a.rows, (int64_t)n) - 1, (int64_t)-1));
    return r;
}
// Pairs [lo, hi) of a range that may see a key of [j0, j1].
__device__ __forceinline__ void pairs_of(const BoundArgs& a, const SumPlan& p, const Rows& r,
                                         int j0, int j1, int range, int& lo, int& hi) {
    const int q0 = max(r.p0, j0);
    int64_t q1 = r.p1;
    if (a.window > 0 && j0 >= a.sinks) q1 = min(q1, (int64_t)j1 + a.window - 1);
    lo = hi = 0;
    if (q1 < q0) return;
    const int64_t at = (int64_t)range * p.range;
    lo = static_cast<int>(max((q0 - r.first) * a.G, at));
    hi = static_cast<int>(min((q1 - r.first + 1) * a.G, at + p.range));
    if (hi < lo) hi = lo;
}
// Whether a live row sees key j.
__device__ __forceinline__ bool key_seen(const BoundArgs& a, const Rows& r, int j) {
    int64_t q1 = r.p1;
    if (a.window > 0 && j >= a.sinks) q1 = min(q1, (int64_t)j + a.window - 1);
    return max(r.p0, j) <= q1;
}

template <int D>
__global__ void __launch_bounds__(kWaves * kWave) __attribute__((amdgpu_waves_per_eu(3)))
prompt_weights_kernel(const BoundArgs a, const SumPlan p) {
    constexpr int NC = D / 16, CPR = D / 8, RPI = kWave / CPR;
    constexpr int IPW = kTile / RPI / kWaves;   // loads per wave and tile
    __shared__ __attribute__((aligned(16))) f16 ring[kStages][kTile * D];
    __shared__ float lse2[kMaxPairs + kTile];   // log2 units; the last tile may end past them
    auto swz = [](int r) { return CPR == 16 ? r & 15 : r >> 1 & 7; };

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, c32 = lane & 31;
    const int kvh = blockIdx.x % a.Hkv, j0 = static_cast<int>(blockIdx.x / a.Hkv) * KB;
    const int range = blockIdx.y, b = blockIdx.z;
    const int n = bound_len(a, b);
    if (j0 >= n) return;
    const Rows rr = rows_of(a, b, n);
    int lo, hi;
    pairs_of(a, p, rr, j0, min(j0 + KB, n) - 1, range, lo, hi);
    if (lo >= hi && p.nrange > 1) return;   // the adding launch knows

    floatx16 w;
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 0.f;
    const int jw = j0 + 32 * wave;   // this wave's first key

    if (lo < hi) {
        const int t0 = lo & ~(kTile - 1);   // tiles are aligned within the sequence's pairs
        const int n_tiles = (hi - t0 + kTile - 1) / kTile;
        const char* qb = reinterpret_cast<const char*>(
            a.q + ((int64_t)b * a.rows * a.Hq + kvh * a.G) * D);
        auto issue = [&](int t) {   // tiles past the last re-load it
            f16* stg = ring[t % kStages];
            const int base = t0 + min(t, n_tiles - 1) * kTile;
            const uint32_t row0 = row_of(p, max(base, lo));
            const char* src = qb + (uint64_t)row0 * a.Hq * (2 * D);
#pragma unroll
            for (int i = 0; i < IPW; ++i) {
                const int r0 = (wave * IPW + i) * RPI, r = r0 + lane / CPR;
                const uint32_t pr = min(max(base + r, lo), hi - 1);
                const uint32_t row = row_of(p, pr);   // at most 64 behind row0
                const uint32_t at = ((row - row0) * a.Hq + (pr - row * a.G)) * (2 * D);
                dma16s(src, at + 16 * ((lane % CPR) ^ swz(r)), stg + r0 * D);
            }
        };
        issue(0);
        issue(1);
        // ---- log-sum-exps of the range; pairs outside [lo, hi) get +inf: no weight
        for (int i = tid; i < n_tiles * kTile; i += kWaves * kWave) {
            const int pr = t0 + i;
            float x = INFINITY;
            if (pr >= lo && pr < hi) {
                const int row = static_cast<int>(row_of(p, pr));
                const int qh = kvh * a.G + pr - row * a.G;
                x = a.lse[((int64_t)b * a.Hq + qh) * a.rows + row] * kLog2e;
            }
            lse2[i] = x;
        }
        // ---- keys: lane (h, c32) holds dims 16c + 8h .. of key jw + c32
        half8 kop[NC];
        {
            const int j = min(jw + c32, n - 1);
            const f16* kr = a.k.data + kvh * a.k.stride_h + bound_row<true>(a.k, b, j) * a.k.stride_s;
#pragma unroll
            for (int c = 0; c < NC; ++c) kop[c] = load_half8(kr + 16 * c + 8 * h);
        }
        int qro[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) qro[c] = c32 * D + 8 * ((2 * c + h) ^ swz(c32));

        // Pairs that see some key of the wave, and those that see all of them.
        const int window = a.window > 0 ? a.window : INT32_MAX;
        const int jl = jw + 31;
        auto pair_of = [&](int64_t pos) {   // first pair of the row at pos, within [lo, hi]
            return static_cast<int>(min(max((pos - rr.first) * a.G, (int64_t)lo), (int64_t)hi));
        };
        const int some0 = pair_of(jw), some1 = jw < a.sinks ? hi : pair_of((int64_t)jl + window);
        const int all0 = pair_of(jl), all1 = jl < a.sinks ? hi : pair_of((int64_t)jw + window);
        const bool any = some0 < some1;
        const int ta = any ? (some0 - t0) / kTile : n_tiles;
        const int tb = any ? (some1 - 1 - t0) / kTile + 1 : n_tiles;

        auto begin = [&](int t) {
            wait_vmcnt<IPW>();
            ring_barrier();
            issue(t + 2);
        };
        // Scores of 32 pairs of tile t, and the weights they add.
        auto scores = [&](int t, int half, floatx16& s) {
            const f16* stg = ring[t % kStages] + 32 * half * D;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    kop[c], *reinterpret_cast<const half8*>(&stg[qro[c]]), s, 0, 0, 0);
        };
        auto whole = [&](int t, int half) {
            const int pr0 = t0 + t * kTile + 32 * half;
            return pr0 >= all0 && pr0 + 32 <= all1;
        };
        auto add = [&](int t, int half, const floatx16& s) {
            const float nl = -lse2[t * kTile + 32 * half + c32];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] += fast_exp2(fmaf(s[i], a.scale_log2, nl));
        };
        auto add_masked = [&](int t, int half, const floatx16& s) {
            const float nl = -lse2[t * kTile + 32 * half + c32];
            const int pr = t0 + t * kTile + 32 * half + c32;
            const int pos = static_cast<int>(rr.first + row_of(p, min(max(pr, lo), hi - 1)));
            // element i is key jw + 4h + 8 (i / 4) + i % 4: counted up to the
            // row's own, but not from the first tokens' end to the last that its window left
            int v0 = jw + 4 * h;
            asm volatile("" : "+v"(v0));   // (or its 16 sums with constants are kept over the loop)
            const int last = pr >= lo && pr < hi ? pos - v0 : -1;
            const int head = a.sinks - v0;
            const uint32_t span = static_cast<uint32_t>(
                max((int64_t)pos - window - v0 - head + 1, (int64_t)0));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int e = 8 * (i / 4) + (i % 4);
                float x = fast_exp2(fmaf(s[i], a.scale_log2, nl));
                x = e > last ? 0.f : x;
                w[i] += static_cast<uint32_t>(e - head) < span ? 0.f : x;
            }
        };
        // The MFMAs of the next 32 pairs run between the exponentials of these.
        auto overlap = [&](int t, int half, int tn, int hn, const floatx16& s, floatx16& sn) {
            if (!whole(t, half)) {
                scores(tn, hn, sn);
                add_masked(t, half, s);
                return;
            }
            scores(tn, hn, sn);
            add(t, half, s);
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x402, 48 / NC, 0);
            }
        };

        wait_vmcnt<0>();   // the keys, before the ring
        __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0): lse2 is written before the barrier
        begin(0);
        int t = 0;
        for (; t < ta; ++t) begin(t + 1);
        if (any) {
            floatx16 s0, s1;
            scores(t, 0, s0);
            for (; t + 1 < tb; ++t) {
                overlap(t, 0, t, 1, s0, s1);
                begin(t + 1);   // every wave has read tile t
                overlap(t, 1, t + 1, 0, s1, s0);
            }
            overlap(t, 0, t, 1, s0, s1);
            begin(t + 1);
            if (whole(t, 1))
                add(t, 1, s1);
            else
                add_masked(t, 1, s1);
            ++t;
        }
        for (; t < n_tiles; ++t) begin(t + 1);
        wait_vmcnt<0>();   // the ring's trailing re-loads
    }

    // ---- over the 32 lanes of a half; lane c32 < 16 keeps element c32
    float mine = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float x = row16_sum(w[i]);
        auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(t[0]) + __uint_as_float(t[1]);
        mine = c32 == i ? x : mine;
    }
    const int j = jw + 8 * (c32 / 4) + 4 * h + c32 % 4;
    if (c32 >= 16 || j >= n) return;
    if (p.nrange > 1)
        p.ws[(((int64_t)range * gridDim.z + b) * a.Hkv + kvh) * p.keys_pitch + j] = mine;
    else if (key_seen(a, rr, j) || (int64_t)j + a.new_keys >= n)
        bound_add(a, b, kvh, j, n, mine);
}

// Adds the ranges' sums in order and updates the slots.
__global__ void __launch_bounds__(256)
prompt_weights_add_kernel(const BoundArgs a, const SumPlan p) {
    const int j = blockIdx.x * 256 + threadIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const int n = bound_len(a, b);
    if (j >= n) return;
    const Rows rr = rows_of(a, b, n);
    const int j0 = j / KB * KB, j1 = min(j0 + KB, n) - 1;
    const float* ws = p.ws + ((int64_t)b * a.Hkv + kvh) * p.keys_pitch + j;
    const int64_t step = (int64_t)gridDim.z * a.Hkv * p.keys_pitch;
    float sum = 0.f;
    for (int r = 0; r < p.nrange; ++r) {
        int lo, hi;
        pairs_of(a, p, rr, j0, j1, r, lo, hi);
        if (lo < hi) sum += ws[r * step];
    }
    if (key_seen(a, rr, j) || (int64_t)j + a.new_keys >= n) bound_add(a, b, kvh, j, n, sum);
}

// Ranges of at least 4 tiles, for about 8 workgroups per CU (half of them see nothing in a
// whole prompt).
SumPlan plan_of(int batch, int rows, int hkv, int G, int max_len) {
    SumPlan p{};
    const int64_t pairs = (int64_t)rows * G;
    const int64_t blocks = ((int64_t)max_len + KB - 1) / KB * hkv * batch;
    int64_t nr = std::min((2048 + blocks - 1) / blocks, (pairs + 255) / 256);
    nr = std::max(nr, (pairs + kMaxPairs - 1) / kMaxPairs);
    p.range = static_cast<int>(((pairs + nr - 1) / nr + kTile - 1) / kTile * kTile);
    p.nrange = static_cast<int>((pairs + p.range - 1) / p.range);
    p.keys_pitch = (max_len + 255) / 256 * 256;
    p.inv_g = G == 1 ? 0 : static_cast<uint32_t>(((uint64_t(1) << 32) + G - 1) / G);
    return p;
}

}  // namespace

size_t prompt_weights_workspace(int batch, int rows, int hq, int hkv, int d, int max_len) {
    if (batch <= 0 || rows <= 0 || hkv <= 0 || hq < hkv || hq % hkv || max_len <= 0 ||
        max_len > 1 << 30 || (d != 64 && d != 128))
        return 0;
    const SumPlan p = plan_of(batch, rows, hkv, hq / hkv, max_len);
    return p.nrange == 1 ? 0 : sizeof(float) * (size_t)p.nrange * batch * hkv * p.keys_pitch;
}

bool prompt_weights_fits(const BoundArgs& a, int batch) {
    const SumPlan p = plan_of(batch, a.rows, a.Hkv, a.G, a.max_len);
    // (pairs times G below 2^31: row_of)
    return (a.D == 64 || a.D == 128) && p.nrange <= 65535 &&
           (int64_t)a.rows * a.G * a.G < (int64_t(1) << 31) &&
           (int64_t)p.keys_pitch / KB * a.Hkv <= 1 << 22 &&
           (int64_t)65 * a.Hq * 2 * a.D < (int64_t)1 << 32;   // a tile's offsets
}

int prompt_weights(const BoundArgs& a, int batch, void* ws, hipStream_t s) {
    SumPlan p = plan_of(batch, a.rows, a.Hkv, a.G, a.max_len);
    p.ws = static_cast<float*>(ws);
    const dim3 grid((a.max_len + KB - 1) / KB * a.Hkv, p.nrange, batch), blk(kWaves * kWave);
    if (a.D == 64)
        hipLaunchKernelGGL((prompt_weights_kernel<64>), grid, blk, 0, s, a, p);
    else
        hipLaunchKernelGGL((prompt_weights_kernel<128>), grid, blk, 0, s, a, p);
    const int rc = check_launch("prompt_weights");
    if (rc || p.nrange == 1) return rc;
    const dim3 grid2((a.max_len + 255) / 256, a.Hkv, batch);
    hipLaunchKernelGGL(prompt_weights_add_kernel, grid2, dim3(256), 0, s, a, p);
    return check_launch("prompt_weights (add)");
}

}  // namespace kvhp
