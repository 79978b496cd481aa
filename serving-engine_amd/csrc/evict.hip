// evict.hip -- cutting a paged cache to a budget of slots per sequence and KV
// head by the attention weight that the slots' keys have received.
//
// Plan: slots rank by (protected by age, weight, lowest slot); the `budget`
// first stay.  One workgroup of 1024 threads per (KV head, sequence).  Every
// slot's rank is a 32-bit key whose order is that of the weights (protected:
// all ones; NaN: zero); the budget-th largest key is found by a radix select
// of 12 + 10 + 10 bits on histograms in LDS, ties going to the lowest slots.
// Evicted slots below the budget ("holes") and kept ones at or past it
// ("movers") are paired in ascending order, from two prefix sums: moving only
// those costs min(evicted, kept past the budget) rows, where closing the gaps
// in order would move nearly every kept row.  The order of the tokens changes,
// which attention over all of them does not see; the ages say which is which.
//
// A thread owns consecutive slots, four to a load: up to 16 quads (65536
// slots) are held in registers between the passes, longer caches are read
// again.  12 bits come first because the weights of a cache span a few binary
// orders: sign, exponent and three bits of mantissa spread a wave's 64 keys
// over many histogram counters, while an 8-bit digit has nearly all of them
// in the same two, and counts on one address go one by one.
#include "kvhp_internal.h"

#include <algorithm>

namespace kvhp {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / kWave;
constexpr int kBins = 4096;

struct PlanArgs {
    const float* weights;     // [Hkv][num_pages][16]
    const int32_t* ages;
    const int32_t* bt;
    const int32_t* seq_lens;
    const int32_t* newest;
    int32_t* moves;           // [B][Hkv][max_moves][2]
    int32_t* counts;          // [B][Hkv]
    int32_t* new_lens;        // [B]
    int max_pages, num_pages, Hkv;
    int cap, budget, sinks, recent, max_moves;
    int quads;                // quads of slots per thread
};

// Rank of a weight: order-preserving, 0 for NaN, below 0xFFFFFFFF; -0 counts as 0.
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w + 0.f);
    return u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}

// Exclusive prefix sum over the workgroup's threads; `total` gets the sum.
// red: kPlanWaves ints of LDS, free again after the caller's next barrier.
__device__ __forceinline__ int block_scan(int x, int* red, int& total) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    int inc = x;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int t = __shfl_up(inc, o);
        if (lane >= o) inc += t;
    }
    if (lane == kWave - 1) red[wave] = inc;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        const int t = red[w];
        before += w < wave ? t : 0;
        total += t;
    }
    __syncthreads();
    return before + inc - x;
}

// Q > 0: Q quads per thread in registers; 0: a.quads of them, read in each pass.
template <int Q>
__global__ void __launch_bounds__(kPlanThreads) evict_plan_kernel(const PlanArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ int red[kPlanWaves];
    __shared__ int found[2];
    const int tid = threadIdx.x, kvh = blockIdx.x, b = blockIdx.y;
    const int n = min(max(a.seq_lens[b], 0), a.cap);
    if (tid == 0 && kvh == 0) a.new_lens[b] = min(n, a.budget);
    int32_t* const count = a.counts + (int64_t)b * a.Hkv + kvh;
    if (n <= a.budget) {
        if (tid == 0) *count = 0;
        return;
    }
    const int nq = Q > 0 ? Q : a.quads;
    const int newest = a.newest ? a.newest[b] : n - 1;
    const int64_t old = (int64_t)newest - a.recent;   // ages above it are recent
    const int32_t* table = a.bt + (int64_t)b * a.max_pages;
    const int s0 = tid * nq * 4;                      // this thread's first slot

    auto load = [&](int q, uint32_t (&k)[4]) {
        const int j = s0 + 4 * q;
        if (j >= n) return;
        const int pid = min(max(table[j >> 4], 0), a.num_pages - 1);
        const int64_t at = ((int64_t)kvh * a.num_pages + pid) * kPage + (j & 15);
        const floatx4 w = *reinterpret_cast<const floatx4*>(a.weights + at);
        int32_t age[4] = {j, j + 1, j + 2, j + 3};
        if (a.ages) {
            const int4 t = *reinterpret_cast<const int4*>(a.ages + at);
            age[0] = t.x, age[1] = t.y, age[2] = t.z, age[3] = t.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            k[e] = age[e] < a.sinks || age[e] > old ? 0xFFFFFFFFu : rank_of(w[e]);
    };
    uint32_t held[Q > 0 ? Q : 1][4];
    if constexpr (Q > 0) {
#pragma unroll
        for (int q = 0; q < Q; ++q) load(q, held[q]);
    }
    // f(slot, key) for this thread's live slots in order
    auto each = [&](auto f) {
        if constexpr (Q > 0) {
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (s0 + 4 * q + e < n) f(s0 + 4 * q + e, held[q][e]);
        } else {
            for (int q = 0; q < nq; ++q) {
                uint32_t k[4];
                load(q, k);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (s0 + 4 * q + e < n) f(s0 + 4 * q + e, k[e]);
            }
        }
    };

    // ---- the budget-th largest key, digit by digit from the top
    uint32_t prefix = 0;       // its digits so far
    int want = a.budget;       // its rank among the keys with that prefix
    int shift = 32;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass == 0 ? 12 : 10;
        shift -= bits;
        for (int i = tid; i < kBins; i += kPlanThreads) hist[i] = 0;
        __syncthreads();
        each([&](int, uint32_t k) {
            if (pass > 0 && (k >> (shift + bits)) != prefix) return;
            const uint32_t digit = k >> shift & ((1u << bits) - 1);
            // lanes that all count the same digit (protected slots, weights of
            // zero) do it at once
            const uint32_t lead = __builtin_amdgcn_readfirstlane(digit);
            const uint64_t in = __builtin_amdgcn_read_exec();
            if (__ballot(digit == lead) == in) {
                if ((threadIdx.x & (kWave - 1)) == (unsigned)__builtin_ctzll(in))
                    atomicAdd(&hist[lead], (uint32_t)__builtin_popcountll(in));
            } else {
                atomicAdd(&hist[digit], 1u);
            }
        });
        __syncthreads();
        // thread t holds the bins kBins - 1 - 4t .. - 3, largest first
        uint32_t c[4];
        int sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = hist[kBins - 1 - 4 * tid - i];
            sum += c[i];
        }
        int total;
        int above = block_scan(sum, red, total);
        if (above < want && above + sum >= want) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (above < want && above + (int)c[i] >= want) {
                    found[0] = kBins - 1 - 4 * tid - i;
                    found[1] = want - above;
                }
                above += c[i];
            }
        }
        __syncthreads();
        prefix = prefix << bits | found[0];
        want = found[1];
    }
    // keys above `prefix` stay, and the first `want` that equal it

    int ties = 0, total;
    each([&](int, uint32_t k) { ties += k == prefix; });
    int tie = block_scan(ties, red, total);
    const int tie0 = tie;
    int holes = 0, movers = 0;
    auto kept = [&](uint32_t k) { return k > prefix || (k == prefix && tie++ < want); };
    each([&](int j, uint32_t k) {
        const bool stay = kept(k);
        holes += j < a.budget && !stay;
        movers += j >= a.budget && stay;
    });
    int hole = block_scan(holes, red, total);
    int mover = block_scan(movers, red, total);
    if (tid == 0) *count = total;
    tie = tie0;
    int32_t* const mv = a.moves + ((int64_t)b * a.Hkv + kvh) * a.max_moves * 2;
    each([&](int j, uint32_t k) {
        const bool stay = kept(k);
        if (j < a.budget && !stay) mv[2 * hole++ + 1] = j;
        if (j >= a.budget && stay) mv[2 * mover++] = j;
    });
}

struct MoveArgs {
    f16 *pool_k, *pool_v;
    float* weights;
    int32_t* ages;
    const int32_t* bt;
    const int32_t* moves;
    const int32_t* counts;
    int max_pages, num_pages, Hkv, D, max_moves;
};

__device__ __forceinline__ void store_half8_stream(f16* p, half8 v) {
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), reinterpret_cast<u32x4*>(p));
}

// A group of `lanes` lanes takes kMoves moves (VEC: 16 bytes a lane, D / 8 lanes rounded
// up to a power of two).  Every row is read and written once and not again soon, so both
// go past the caches: 32 x 8192 slots cut to 4096 at 8 heads of 128, 204 k moves, in us:
// 62 with plain accesses, 57 with such loads, 53 with such stores, 52 with both, and
// with both 51 / 54 / 93 for 2 / 4 / 8 moves a group; 213 MB, 4.2 TB/s, where a copy of
// long runs reaches 4.7.
constexpr int kMoves = 2;

template <bool VEC>
__global__ void __launch_bounds__(256) evict_apply_kernel(const MoveArgs a, int lanes) {
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int count = min(a.counts[(int64_t)b * a.Hkv + kvh], a.max_moves);
    const int lane = threadIdx.x % lanes;
    const int i0 = (blockIdx.x * (256 / lanes) + threadIdx.x / lanes) * kMoves;
    if (i0 >= count) return;
    const int32_t* table = a.bt + (int64_t)b * a.max_pages;
    const int2* mv = reinterpret_cast<const int2*>(a.moves) + ((int64_t)b * a.Hkv + kvh) * a.max_moves;
    int64_t f[kMoves], t[kMoves];   // slots in the head's pools; t < 0: no move
#pragma unroll
    for (int u = 0; u < kMoves; ++u) {
        const int2 m = mv[min(i0 + u, count - 1)];
        const bool ok = i0 + u < count && m.x >= 0 && m.y >= 0 && (m.x >> 4) < a.max_pages &&
                        (m.y >> 4) < a.max_pages;
        const int pf = ok ? table[m.x >> 4] : -1, pt = ok ? table[m.y >> 4] : -1;
        const bool in = pf >= 0 && pt >= 0 && pf < a.num_pages && pt < a.num_pages;
        const int64_t head = (int64_t)kvh * a.num_pages;
        f[u] = in ? (head + pf) * kPage + (m.x & 15) : 0;
        t[u] = in ? (head + pt) * kPage + (m.y & 15) : -1;
    }
    if constexpr (VEC) {
        if (8 * lane < a.D) {
            half8 k[kMoves], v[kMoves];
#pragma unroll
            for (int u = 0; u < kMoves; ++u) {
                k[u] = load_half8_stream(a.pool_k + f[u] * a.D + 8 * lane);
                v[u] = load_half8_stream(a.pool_v + f[u] * a.D + 8 * lane);
            }
#pragma unroll
            for (int u = 0; u < kMoves; ++u)
                if (t[u] >= 0) {
                    store_half8_stream(a.pool_k + t[u] * a.D + 8 * lane, k[u]);
                    store_half8_stream(a.pool_v + t[u] * a.D + 8 * lane, v[u]);
                }
        }
    } else {
#pragma unroll
        for (int u = 0; u < kMoves; ++u)
            if (t[u] >= 0)
                for (int d = lane; d < a.D; d += lanes) {
                    a.pool_k[t[u] * a.D + d] = a.pool_k[f[u] * a.D + d];
                    a.pool_v[t[u] * a.D + d] = a.pool_v[f[u] * a.D + d];
                }
    }
#pragma unroll
    for (int u = 0; u < kMoves; ++u) {
        if (t[u] < 0) continue;
        if (lane == u % lanes && a.weights) a.weights[t[u]] = a.weights[f[u]];
        if (lane == (u + kMoves) % lanes && a.ages) a.ages[t[u]] = a.ages[f[u]];
    }
}

}  // namespace
}  // namespace kvhp

using namespace kvhp;

extern "C" int kvhp_evict_plan(const float* weights, const int32_t* ages,
                               const int32_t* block_tables, int max_pages,
                               const int32_t* seq_lens, const int32_t* newest, int32_t* moves,
                               int32_t* counts, int32_t* new_lens, int batch, int num_kv_heads,
                               int num_pages, int max_seq_len, int budget, int sinks, int recent,
                               int max_moves, void* stream) {
    clear_error();
    if (batch <= 0) return KVHP_OK;
    const char* what = "evict_plan";
    KVHP_REQUIRE(weights && block_tables && seq_lens && counts && new_lens, KVHP_ERR_INVALID,
                 "%s: null pointer", what);
    KVHP_REQUIRE(num_kv_heads > 0 && max_pages > 0 && num_pages > 0, KVHP_ERR_INVALID,
                 "%s: num_kv_heads, max_pages and num_pages must be positive", what);
    KVHP_REQUIRE(batch <= 65535, KVHP_ERR_UNSUPPORTED, "%s: more than 65535 sequences", what);
    KVHP_REQUIRE(max_seq_len <= 1 << 30, KVHP_ERR_UNSUPPORTED, "%s: max_seq_len=%d above 2^30",
                 what, max_seq_len);
    KVHP_REQUIRE(budget > 0 && sinks >= 0 && recent >= 0 && (int64_t)sinks + recent <= budget,
                 KVHP_ERR_INVALID,
                 "%s: budget=%d must be positive and hold sinks=%d and recent=%d", what, budget,
                 sinks, recent);
    KVHP_REQUIRE(new_lens != seq_lens, KVHP_ERR_INVALID, "%s: new_lens aliases seq_lens", what);
    KVHP_REQUIRE(aligned16(weights) && aligned16(ages), KVHP_ERR_INVALID,
                 "%s: weights and ages must be 16-byte aligned", what);
    const int cap = static_cast<int>(
        std::min<int64_t>(std::max(max_seq_len, 0), (int64_t)max_pages * kPage));
    const int need = std::min(budget, std::max(cap - budget, 0));
    KVHP_REQUIRE(max_moves >= need && (need == 0 || moves), KVHP_ERR_INVALID,
                 "%s: room for %d moves, %d needed", what, moves ? max_moves : 0, need);
    PlanArgs a{weights, ages, block_tables, seq_lens, newest, moves, counts, new_lens,
               max_pages, num_pages, num_kv_heads, cap, budget, sinks, recent, max_moves, 0};
    a.quads = (cap + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
    const dim3 grid(num_kv_heads, batch), blk(kPlanThreads);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.quads <= 1)
        hipLaunchKernelGGL(evict_plan_kernel<1>, grid, blk, 0, s, a);
    else if (a.quads <= 4)
        hipLaunchKernelGGL(evict_plan_kernel<4>, grid, blk, 0, s, a);
    else if (a.quads <= 16)
        hipLaunchKernelGGL(evict_plan_kernel<16>, grid, blk, 0, s, a);
    else
        hipLaunchKernelGGL(evict_plan_kernel<0>, grid, blk, 0, s, a);
    return check_launch(what);
}

extern "C" int kvhp_evict_apply(void* pool_k, void* pool_v, float* weights, int32_t* ages,
                                const int32_t* block_tables, int max_pages, const int32_t* moves,
                                const int32_t* counts, int batch, int num_kv_heads, int head_dim,
                                int num_pages, int max_moves, void* stream) {
    clear_error();
    if (batch <= 0 || max_moves <= 0) return KVHP_OK;
    const char* what = "evict_apply";
    KVHP_REQUIRE(pool_k && pool_v && block_tables && moves && counts, KVHP_ERR_INVALID,
                 "%s: null pointer", what);
    KVHP_REQUIRE(num_kv_heads > 0 && max_pages > 0 && num_pages > 0, KVHP_ERR_INVALID,
                 "%s: num_kv_heads, max_pages and num_pages must be positive", what);
    KVHP_REQUIRE(head_dim > 0 && head_dim <= 256, KVHP_ERR_UNSUPPORTED,
                 "%s: head_dim=%d outside 1..256", what, head_dim);
    KVHP_REQUIRE((reinterpret_cast<uintptr_t>(moves) & 7u) == 0, KVHP_ERR_INVALID,
                 "%s: moves must be 8-byte aligned", what);
    KVHP_REQUIRE(batch <= 65535 && num_kv_heads <= 65535, KVHP_ERR_UNSUPPORTED,
                 "%s: more than 65535 sequences or KV heads", what);
    MoveArgs a{static_cast<f16*>(pool_k), static_cast<f16*>(pool_v), weights, ages, block_tables,
               moves, counts, max_pages, num_pages, num_kv_heads, head_dim, max_moves};
    const bool vec = head_dim % 8 == 0 && aligned16(pool_k) && aligned16(pool_v);
    int lanes = 1;
    while (lanes * (vec ? 8 : 1) < head_dim && lanes < kWave) lanes *= 2;
    const int per = 256 / lanes * kMoves;
    const dim3 grid((max_moves + per - 1) / per, num_kv_heads, batch);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (vec)
        hipLaunchKernelGGL(evict_apply_kernel<true>, grid, dim3(256), 0, s, a, lanes);
    else
        hipLaunchKernelGGL(evict_apply_kernel<false>, grid, dim3(256), 0, s, a, lanes);
    return check_launch(what);
}
