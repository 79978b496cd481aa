// prompt_weights.hip -- the attention weights that rows of a prompt gave each cached
// key, summed over the rows and the query heads of its KV head (gfx950, head_dim 64
// and 128):  w_j = sum over rows i that see j, heads g, of exp(q_ig . k_j / sqrt(D) - lse_ig).
//
// The log-sum-exps are known, so this is one product and one pass.  A workgroup of
// four waves holds 32 keys a wave as MFMA operands in registers and walks the (row, head)
// pairs in tiles of 64, which go from memory to two LDS stages without registers, with
// their log-sum-exps:  S^T = K Q^T on v_mfma_f32_32x32x16_f16 gives a lane one pair and 16
// keys per block, so the sum over pairs stays in the lane until the end, where 32 lanes
// are added once.  Keys are the operand that stays because their sums do; walking keys
// instead would add lanes per tile.
//
// A tile is 64 rows of one head (or all rows, where they are fewer, of several): no row
// is found by a division, and a lane's offsets stay the same from tile to tile.  Tiles
// whose pairs see none of a wave's keys are passed over; pairs that see some get a weight
// of 2^-inf by a select (a NaN score of an unseen pair must not count).  Long prompts are
// cut into ranges of tiles whose sums a second launch adds in order, so the result does
// not depend on timing.
//
// 4096 rows of 32/8 heads of 128 (69 GFLOP) take 88 us, 0.78 PFLOP/s, 32 rows of four
// sequences of 3001 keys at 32/4 heads of 64 9.1.  Bound by the vector unit, per 32 x 32
// scores 16 times (fma, exp, add) of 24 cycles, 47 us over the prompt if it never waited;
// the 8 MFMAs of 32 cycles run beside it in other waves, four workgroups a CU.  The second
// launch takes 4; waves wait for a quarter of their cycles (counters: vector unit 65 % busy,
// matrix cores 45 %, LDS 24 %), at what is not known: it is not whole rounds of workgroups, see
// the ranges below.  One wave running the next pairs' MFMAs between the exponentials of
// these was no faster (three workgroups a CU, 104 us); 64 keys a wave, half the LDS reads,
// spill registers (136 to 300).
#include "bounded.h"

#include <algorithm>

namespace kvhp {
namespace {

constexpr int kWaves = 4;
constexpr int kTile = 64;        // pairs per tile
constexpr int KB = 32 * kWaves;  // keys per workgroup
constexpr int kMaxRowHeads = 1 << 30;   // (row, query head) pairs of a KV head

// A tile is 2^lr rows of `gc` heads, 64 pairs, row fastest; tile f is row tile f / nh and
// heads (f % nh) * gc on.
struct SumPlan {
    int lr, gc, nh;
    int range;        // tiles per range
    int nrange;
    int keys_pitch;
    float* ws;        // [nrange][batch][Hkv][keys_pitch], nrange > 1
};

// dma16s with 4 bytes a lane.
__device__ __forceinline__ void dma4s(const char* base, uint32_t voff, float* lds_base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
                 :: "s"(lds_at(lds_base)), "v"(voff), "s"(base) : "memory", "m0");
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
// Tiles [lo, hi) with rows that see a key of [j0, j1].
__device__ __forceinline__ void tiles_of(const BoundArgs& a, const SumPlan& p, const Rows& r,
                                         int j0, int j1, int& lo, int& hi) {
    const int q0 = max(r.p0, j0);
    int64_t q1 = r.p1;
    if (a.window > 0 && j0 >= a.sinks) q1 = min(q1, (int64_t)j1 + a.window - 1);
    lo = hi = 0;
    if (q1 < q0) return;
    lo = (static_cast<int>(q0 - r.first) >> p.lr) * p.nh;
    hi = ((static_cast<int>(q1 - r.first) >> p.lr) + 1) * p.nh;
}
// Whether a live row sees key j.
__device__ __forceinline__ bool key_seen(const BoundArgs& a, const Rows& r, int j) {
    int64_t q1 = r.p1;
    if (a.window > 0 && j >= a.sinks) q1 = min(q1, (int64_t)j + a.window - 1);
    return max(r.p0, j) <= q1;
}

template <int D>
__global__ void __launch_bounds__(kWaves * kWave) __attribute__((amdgpu_waves_per_eu(4)))
prompt_weights_kernel(const BoundArgs a, const SumPlan p) {
    constexpr int NC = D / 16, CPR = D / 8, RPI = kWave / CPR;
    constexpr int IPW = kTile / RPI / kWaves;   // loads per wave and tile
    __shared__ __attribute__((aligned(16))) f16 ring[2][kTile * D];
    __shared__ float lse[2][kTile];
    auto swz = [](int r) { return CPR == 16 ? r & 15 : r >> 1 & 7; };

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = lane >> 5, c32 = lane & 31;
    const int kvh = blockIdx.x % a.Hkv, j0 = static_cast<int>(blockIdx.x / a.Hkv) * KB;
    const int range = blockIdx.y, b = blockIdx.z;
    const int n = bound_len(a, b);
    if (j0 >= n) return;
    const Rows rr = rows_of(a, b, n);
    int f0, f1;
    tiles_of(a, p, rr, j0, min(j0 + KB, n) - 1, f0, f1);
    f0 = max(f0, range * p.range);
    f1 = static_cast<int>(min((int64_t)f1, ((int64_t)range + 1) * p.range));
    const int n_tiles = f1 - f0;
    const int jw = j0 + 32 * wave;   // this wave's first key
    // the key whose sum this lane ends up with (lanes c32 < 16)
    const int j = jw + 8 * (c32 / 4) + 4 * h + c32 % 4;
    const bool mine = c32 < 16 && j < n;
    if (n_tiles <= 0) {   // (of more ranges, the adding launch knows)
        if (p.nrange == 1 && mine && (int64_t)j + a.new_keys >= n) bound_add(a, b, kvh, j, n, 0.f);
        return;
    }

    floatx16 w;
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = 0.f;
    const int R = 1 << p.lr;
    // ---- loads: tile t goes to stage t % 2; tiles past the last re-load it
    const char* qb = reinterpret_cast<const char*>(
        a.q + ((int64_t)b * a.rows * a.Hq + kvh * a.G) * D);
    const char* lb = reinterpret_cast<const char*>(
        a.lse + ((int64_t)b * a.Hq + kvh * a.G) * a.rows);
    // offsets of a slot from its tile's first row and head; rows and heads past the last
    // (of a tile that has some) are read as the last
    auto q_off = [&](int i, int l, int rows, int heads) {
        const int slot = (wave * IPW + i) * RPI + l / CPR;
        const int row = min(slot & (R - 1), rows - 1), head = min(slot >> p.lr, heads - 1);
        return static_cast<uint32_t>(row * a.Hq + head) * (2 * D) +
               16 * ((l % CPR) ^ swz(slot));
    };
    auto l_off = [&](int l, int rows, int heads) {
        const int row = min(l & (R - 1), rows - 1), head = min(l >> p.lr, heads - 1);
        return static_cast<uint32_t>(head * a.rows + row) * 4;
    };
    uint32_t qo[IPW];
#pragma unroll
    for (int i = 0; i < IPW; ++i) qo[i] = q_off(i, lane, R, p.gc);
    const uint32_t lo = l_off(lane, R, p.gc);
    int ld = 0, ld_r = f0 / p.nh << p.lr, ld_h = f0 % p.nh * p.gc;   // the next tile to load
    const char* qs = qb + ((int64_t)ld_r * a.Hq + ld_h) * (2 * D);
    const char* ls = lb + ((int64_t)ld_h * a.rows + ld_r) * 4;
    auto issue = [&](int t) {
        f16* stage = ring[t & 1] + wave * IPW * RPI * D;
        if (ld_r + R <= a.rows && ld_h + p.gc <= a.G) {
#pragma unroll
            for (int i = 0; i < IPW; ++i) dma16s(qs, qo[i], stage + i * RPI * D);
            dma4s(ls, lo, lse[t & 1]);
        } else {
            int l = lane;
            asm volatile("" : "+v"(l));   // (or the parts of these are kept over the loop)
#pragma unroll
            for (int i = 0; i < IPW; ++i)
                dma16s(qs, q_off(i, l, a.rows - ld_r, a.G - ld_h), stage + i * RPI * D);
            dma4s(ls, l_off(l, a.rows - ld_r, a.G - ld_h), lse[t & 1]);
        }
        if (++ld >= n_tiles) return;
        ld_h += p.gc;
        qs += 2 * D * p.gc;
        ls += (int64_t)4 * a.rows * p.gc;
        if (ld_h < a.G) return;
        qs += ((int64_t)R * a.Hq - ld_h) * (2 * D);
        ls += (R - (int64_t)ld_h * a.rows) * 4;
        ld_h = 0;
        ld_r += R;
    };
    issue(0);
    // ---- keys: lane (h, c32) holds dims 16c + 8h .. of key jw + c32
    half8 kop[NC];
    {
        const f16* kr = a.k.data + kvh * a.k.stride_h +
                        bound_row<true>(a.k, b, min(jw + c32, n - 1)) * a.k.stride_s;
#pragma unroll
        for (int c = 0; c < NC; ++c) kop[c] = load_half8(kr + 16 * c + 8 * h);
    }
    int qro[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) qro[c] = c32 * D + 8 * ((2 * c + h) ^ swz(c32));

    // Rows that see some key of the wave, and those that see all of them.
    const int window = a.window > 0 ? a.window : INT32_MAX;
    const int jl = jw + 31;
    auto row_at = [&](int64_t pos) {   // of a position, within the live rows
        return static_cast<int>(min(max(pos, (int64_t)rr.p0), (int64_t)rr.p1 + 1) - rr.first);
    };
    const int some0 = row_at(jw), some1 = row_at(jw < a.sinks ? INT32_MAX : (int64_t)jl + window);
    const int all0 = row_at(jl), all1 = row_at(jl < a.sinks ? INT32_MAX : (int64_t)jw + window);
    int ta = n_tiles, tb = n_tiles;   // tiles with such rows
    if (some0 < some1) {
        ta = min(max((some0 >> p.lr) * p.nh - f0, 0), n_tiles);
        tb = static_cast<int>(min(((int64_t)((some1 - 1) >> p.lr) + 1) * p.nh - f0, (int64_t)n_tiles));
        if (tb <= ta) ta = tb = n_tiles;
    }
    int at_r = (f0 + ta) / p.nh, at_h = f0 + ta - at_r * p.nh;   // the tile at hand

    // Tile t has landed everywhere, and every wave is past tile t - 1.
    auto begin = [&](int t) {
        wait_ring<0>();
        ring_barrier();
        issue(t + 1);
    };
    begin(0);
    int t = 0;
    for (; t < ta; ++t) begin(t + 1);
    for (; t < tb; ++t) {
        // ---- scores of both halves
        const f16* stg = ring[t & 1];
        floatx16 s[2];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[half][i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                s[half] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    kop[c], *reinterpret_cast<const half8*>(&stg[qro[c] + 32 * half * D]),
                    s[half], 0, 0, 0);
        // six operands ahead (93 us instead of 96 in the order the compiler takes)
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 0);
#pragma unroll
        for (int i = 0; i < 2 * NC; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        // ---- the weights' logarithms, those of unseen pairs -inf (whatever their
        //      row's log-sum-exp holds)
        const int r0 = at_r << p.lr;
        const bool whole = r0 >= all0 && r0 + R <= all1 && (at_h + 1) * p.gc <= a.G;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float nl = -kLog2e * lse[t & 1][32 * half + c32];
#pragma unroll
            for (int i = 0; i < 16; ++i) s[half][i] = fmaf(s[half][i], a.scale_log2, nl);
        }
        if (!whole) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                int slot = 32 * half + c32, v0 = jw + 4 * h;
                asm volatile("" : "+v"(slot), "+v"(v0));   // (or sums with them are kept over the loop)
                const int row = r0 + (slot & (R - 1));
                const int pos = static_cast<int>(rr.first + row);
                const bool live = row < a.rows && pos <= rr.p1 && at_h * p.gc + (slot >> p.lr) < a.G;
                // element i is key jw + 4h + 8 (i / 4) + i % 4: counted up to the row's
                // own, but not from the first tokens' end to the last that its window left
                const int last = live ? pos - v0 : -1;
                const int head = a.sinks - v0;
                const uint32_t span = static_cast<uint32_t>(
                    max((int64_t)pos - window - v0 - head + 1, (int64_t)0));
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[half][i] = 8 * (i / 4) + (i % 4) > last ? -INFINITY : s[half][i];
                if (__builtin_amdgcn_read_exec() & __ballot(span > 0)) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        s[half][i] = static_cast<uint32_t>(8 * (i / 4) + (i % 4) - head) < span
                                         ? -INFINITY : s[half][i];
                }
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] += fast_exp2(s[half][i]);
        if (++at_h == p.nh) {
            at_h = 0;
            ++at_r;
        }
        begin(t + 1);
    }
    for (; t < n_tiles; ++t) begin(t + 1);
    wait_ring<0>();   // the ring's trailing re-loads

    // ---- over the 32 lanes of a half; lane c32 < 16 keeps element c32
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float x = row16_sum(w[i]);
        auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(t[0]) + __uint_as_float(t[1]);
        sum = c32 == i ? x : sum;
    }
    if (!mine) return;
    if (p.nrange > 1)
        p.ws[(((int64_t)range * gridDim.z + b) * a.Hkv + kvh) * p.keys_pitch + j] = sum;
    else if (key_seen(a, rr, j) || (int64_t)j + a.new_keys >= n)
        bound_add(a, b, kvh, j, n, sum);
}

// Adds the ranges' sums in order and updates the slots.  (One load after the other the sums
// of 56 ranges took 15 us, eight at a time 3.)
__global__ void __launch_bounds__(256)
prompt_weights_add_kernel(const BoundArgs a, const SumPlan p) {
    const int j = blockIdx.x * 256 + threadIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const int n = bound_len(a, b);
    if (j >= n) return;
    const Rows rr = rows_of(a, b, n);
    const int j0 = j / KB * KB, j1 = min(j0 + KB, n) - 1;
    const float* ws = p.ws + ((int64_t)b * a.Hkv + kvh) * p.keys_pitch + j;
    const int64_t step = (int64_t)gridDim.z * a.Hkv * p.keys_pitch;
    int f0, f1;
    tiles_of(a, p, rr, j0, j1, f0, f1);
    float sum = 0.f;
    if (f0 < f1) {
        constexpr int U = 8;   // ranges in flight
        const int last = (f1 - 1) / p.range;
        for (int r = f0 / p.range; r <= last; r += U) {
            float x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) x[u] = ws[min(r + u, last) * step];
#pragma unroll
            for (int u = 0; u < U; ++u) sum += r + u <= last ? x[u] : 0.f;
        }
    }
    if (key_seen(a, rr, j) || (int64_t)j + a.new_keys >= n) bound_add(a, b, kvh, j, n, sum);
}

// Tiles of one head's 64 rows, or of all rows where they are fewer, of as many heads as fit.
// Ranges of at least 6 tiles, for about 12 workgroups per CU, of which half see nothing in a
// whole prompt (4096 rows of 32/8 heads of 128, for 7 / 8 / 10 / 12 / 14 / 16 / 20: 91.4 / 94.5 /
// 88.0 / 86.2 / 87.8 / 89.7 / 87.2 us; 2048 34.4 / 33.8 / 32.7 / 32.7 / 32.9 / 32.6 / 32.7); of at least 2 while all run at once (512
// rows 10.6 us, 4 tiles 11.6, 8 15.4; but 1000 rows 18.2 / 16.8 / 17.6).  Up to 5 tiles
// are not worth a second launch (64 rows of 4 heads 8.0 us whole, 10.4 in two; of 7 11.1 and
// 9.6 in four).
SumPlan plan_of(int batch, int rows, int hkv, int G, int max_len) {
    SumPlan p{};
    while (p.lr < 6 && (1 << p.lr) < rows) ++p.lr;
    p.gc = kTile >> p.lr;
    p.nh = (G + p.gc - 1) / p.gc;
    const int64_t tiles = (((int64_t)rows + (1 << p.lr) - 1) >> p.lr) * p.nh;
    const int64_t blocks = ((int64_t)max_len + KB - 1) / KB * hkv * batch;
    const int64_t most = (3000 + blocks - 1) / blocks, once = 1024 / blocks;
    const int64_t nr = tiles <= 5 ? 1
        : std::min(most, std::max((tiles + 5) / 6, std::min((tiles + 1) / 2, once)));
    p.range = static_cast<int>(std::min<int64_t>((tiles + nr - 1) / nr, INT32_MAX));
    p.nrange = static_cast<int>((tiles + p.range - 1) / p.range);
    p.keys_pitch = (max_len + 255) / 256 * 256;
    return p;
}

}  // namespace

size_t prompt_weights_workspace(int batch, int rows, int hq, int hkv, int d, int max_len) {
    if (rows <= 0 || !bound_sizes(batch, hq, hkv, max_len, 0, 0) ||
        (int64_t)rows * (hq / hkv) > kMaxRowHeads || (d != 64 && d != 128))
        return 0;
    const SumPlan p = plan_of(batch, rows, hkv, hq / hkv, max_len);
    return p.nrange == 1 ? 0 : sizeof(float) * (size_t)p.nrange * batch * hkv * p.keys_pitch;
}

bool prompt_weights_fits(const BoundArgs& a, int batch) {
    if ((int64_t)a.rows * a.G > kMaxRowHeads) return false;   // tiles in an int
    const SumPlan p = plan_of(batch, a.rows, a.Hkv, a.G, a.max_len);
    return (a.D == 64 || a.D == 128) && p.nrange <= 65535 &&
           (int64_t)p.keys_pitch / KB * a.Hkv <= 1 << 22 &&
           (int64_t)kTile * a.Hq * 2 * a.D < (int64_t)1 << 32;   // a tile's offsets
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
