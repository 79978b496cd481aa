// evict.hip -- cutting a paged cache to a budget of slots per sequence and KV
// head by the attention weight that the slots' keys have received.
//
// Plan: slots rank by (protected by age, weight, lowest slot); the `budget`
// first stay.  One workgroup of 1024 threads per (KV head, sequence).  Every
// slot has a 32-bit key in the order of the ranks; the budget-th largest is
// found by a radix select of 12 + 10 + 10 bits on histograms in LDS, which
// ends once all keys that share the digits so far are wanted, ties going to the
// lowest slots.  12 bits come first because the weights of a cache span a few
// binary orders: sign, exponent and three bits of mantissa spread a wave's 64
// keys over many counters, while an 8-bit digit has nearly all of them in the
// same two, and counts on one address go one by one.
//
// Evicted slots below the budget ("holes") and kept ones at or past it
// ("movers") are as many as each other and are paired in ascending order, from
// one prefix sum over both: moving only those costs min(evicted, kept past the
// budget) rows, where closing the gaps in order would move nearly every kept
// row.  The order of the tokens changes, which attention over all of them does
// not see; the ages say which is which.
//
// A thread owns consecutive slots, whose keys stay in registers between the
// passes (up to 8192 slots), in LDS (32768), or are read again.  Bound by the
// chain of 13 barriers (5 a digit, two digits nearly always) and, in longer
// caches, by one CU's instructions per slot: 8.6 us for one sequence of 2064 slots
// cut to 2048, 7.3 for 4096 to half, 10.3 for 8192, 12.5 for 32 of up to 8192, 21
// for 16384, 33 for 32768, 131 for 65536 read again (their 8 bytes a slot are 4 us
// or less at the card's rate).
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

// Keys: of a slot behind the sequence, of a NaN, of a weight of zero, of a protected slot.
constexpr uint32_t kDead = 0, kNaN = 1, kZero = 0x80000000u, kGuard = 0xFFFFFFFFu;

// Key of a weight, in the weights' order (-0 as 0), between kNaN and kGuard.
__device__ __forceinline__ uint32_t key_of(float w) {
    const uint32_t u = __float_as_uint(w + 0.f);
    const uint32_t k = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
    return w != w ? kNaN : k;
}

// Inclusive prefix sum over the wave: shifts by 1, 2, 4, 8 lanes within rows of 16, then
// the rows' last lanes broadcast to the rows behind (no LDS round trips).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) {
    return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int x) {
    x = dpp_add<0x111, 0xF>(x);
    x = dpp_add<0x112, 0xF>(x);
    x = dpp_add<0x114, 0xF>(x);
    x = dpp_add<0x118, 0xF>(x);
    x = dpp_add<0x142, 0xA>(x);   // lane 15 of rows 0, 2 to rows 1, 3
    return dpp_add<0x143, 0xC>(x);   // lane 31 to rows 2, 3
}

// Exclusive prefix sum over the workgroup's threads; `total` gets the sum.
// red: kPlanWaves ints of LDS, free again after the caller's next barrier.
__device__ __forceinline__ int block_scan(int x, int* red, int& total) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    const int inc = wave_scan(x);
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

// A thread's quads of keys between the passes: Q in registers (Q > 0), a.quads of them in
// LDS (kInLds), or nowhere, read and made again in each pass (kAgain).
constexpr int kInLds = 0, kAgain = -1;
constexpr int kLdsQuads = 8;

template <int Q>
__global__ void __launch_bounds__(kPlanThreads) evict_plan_kernel(const PlanArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ int red[kPlanWaves];
    __shared__ int found[3];
    __shared__ int special[2];
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
        const int jc = min(j, n - 1) & ~3;   // behind the sequence: its last quad's, then dead
        const int pid = min(max(table[jc >> 4], 0), a.num_pages - 1);
        const int64_t at = ((int64_t)kvh * a.num_pages + pid) * kPage + (jc & 15);
        const floatx4 w = *reinterpret_cast<const floatx4*>(a.weights + at);
        int32_t age[4] = {j, j + 1, j + 2, j + 3};
        if (a.ages) {
            const int4 t = *reinterpret_cast<const int4*>(a.ages + at);
            age[0] = t.x, age[1] = t.y, age[2] = t.z, age[3] = t.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            k[e] = j + e >= n                              ? kDead
                   : age[e] < a.sinks || age[e] > old ? kGuard
                                                      : key_of(w[e]);
    };
    uint32_t held[Q > 0 ? Q : 1][4];
    __shared__ u32x4 lds_keys[Q == kInLds ? kLdsQuads : 1][Q == kInLds ? kPlanThreads : 1];
    if constexpr (Q > 0) {
#pragma unroll
        for (int q = 0; q < Q; ++q) load(q, held[q]);
    } else if constexpr (Q == kInLds) {
        for (int q0 = 0; q0 < nq; q0 += 4) {   // read back by this thread only
            uint32_t k[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) load(min(q0 + i, nq - 1), k[i]);   // four under way
#pragma unroll
            for (int i = 0; i < 4; ++i)
                lds_keys[min(q0 + i, nq - 1)][tid] = u32x4{k[i][0], k[i][1], k[i][2], k[i][3]};
        }
    }
    // f(slot, key) for this thread's slots in order
    auto each = [&](auto f) {
        if constexpr (Q > 0) {
#pragma unroll
            for (int q = 0; q < Q; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t k = held[q][e];
                    asm volatile("" : "+v"(k));   // (or every comparison's outcome is kept)
                    f(s0 + 4 * q + e, k);
                }
        } else {
            for (int q = 0; q < nq; ++q) {
                uint32_t k[4];
                if constexpr (Q == kInLds) {
                    const u32x4 x = lds_keys[q][tid];
                    k[0] = x[0], k[1] = x[1], k[2] = x[2], k[3] = x[3];
                } else {
                    load(q, k);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) f(s0 + 4 * q + e, k[e]);
            }
        }
    };
    // Two keys that many slots have, protected and never attended, are counted apart:
    // counts on one address go one by one.
    int guards = 0, zeros = 0;
    each([&](int, uint32_t k) {
        guards += k == kGuard;
        zeros += k == kZero;
    });
    if (tid < 2) special[tid] = 0;
    __syncthreads();
    guards = wave_scan(guards);
    zeros = wave_scan(zeros);
    if ((tid & (kWave - 1)) == kWave - 1) {
        atomicAdd(&special[0], guards);
        atomicAdd(&special[1], zeros);
    }

    // ---- the budget-th largest key, digit by digit from the top, until those that share its
    //      digits so far are all wanted (after two digits nearly always)
    uint32_t prefix = 0;       // its digits so far
    int want = a.budget;       // its rank among the keys with that prefix
    int shift = 32;
    bool all = false;          // every key with that prefix is wanted
#pragma unroll 1
    for (int pass = 0; pass < 3 && !all; ++pass) {
        const int bits = pass == 0 ? 12 : 10;
        const int per = pass == 0 ? kBins / kPlanThreads : 1;   // counters per thread
        const int from = shift;                                 // digits above it are `prefix`
        shift -= bits;
        const uint32_t mask = (1u << bits) - 1;
        for (int i = tid; i < per * kPlanThreads; i += kPlanThreads) hist[i] = 0;
        __syncthreads();
        auto mine = [&](uint32_t k) { return pass == 0 || k >> from == prefix; };
        if (tid < 2 && mine(tid ? kZero : kGuard))
            atomicAdd(&hist[(tid ? kZero : kGuard) >> shift & mask], (uint32_t)special[tid]);
        each([&](int, uint32_t k) {
            if (k != kGuard && k != kZero && k != kDead && mine(k)) atomicAdd(&hist[k >> shift & mask], 1u);
        });
        __syncthreads();
        // thread t holds `per` counters, the largest digits first
        const int top = per * (kPlanThreads - tid) - 1;
        int c[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[i] = i < per ? hist[top - i] : 0;
            sum += c[i];
        }
        int total;
        int above = block_scan(sum, red, total);
        if (above < want && above + sum >= want) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (above < want && above + c[i] >= want) {
                    found[0] = top - i;
                    found[1] = want - above;
                    found[2] = c[i] == want - above;
                }
                above += c[i];
            }
        }
        __syncthreads();
        prefix = prefix << bits | found[0];
        want = found[1];
        all = found[2];
    }
    // Keys whose digits are above `prefix` stay, and the first `want` whose digits equal it.
    int total, tie = 0;
    if (!all) {
        int ties = 0;
        each([&](int, uint32_t k) { ties += k != kDead && (k >> shift) == prefix; });
        tie = block_scan(ties, red, total);
    }
    const int tie0 = tie;
    auto kept = [&](uint32_t k) {
        const uint32_t d = k >> shift;
        if (all) return k != kDead && d >= prefix;
        const bool equal = k != kDead && d == prefix;
        tie += equal;
        return d > prefix || (equal && tie <= want);
    };
    // Holes below the budget and movers from it on are as many as each other: one prefix
    // sum over both counts the holes, then the movers.
    int here = 0;
    each([&](int j, uint32_t k) { here += kept(k) == (j >= a.budget); });
    int at = block_scan(here, red, total);
    const int half = total / 2;
    if (tid == 0) *count = half;
    tie = tie0;
    int32_t* const mv = a.moves + ((int64_t)b * a.Hkv + kvh) * a.max_moves * 2;
    each([&](int j, uint32_t k) {
        if (kept(k) != (j >= a.budget)) return;
        if (j < a.budget)
            mv[2 * at + 1] = j;
        else
            mv[2 * (at - half)] = j;
        ++at;
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
    else if (a.quads <= 2)
        hipLaunchKernelGGL(evict_plan_kernel<2>, grid, blk, 0, s, a);
    else if (a.quads <= kLdsQuads)
        hipLaunchKernelGGL(evict_plan_kernel<kInLds>, grid, blk, 0, s, a);
    else
        hipLaunchKernelGGL(evict_plan_kernel<kAgain>, grid, blk, 0, s, a);
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
    KVHP_REQUIRE(max_moves <= 1 << 30, KVHP_ERR_UNSUPPORTED, "%s: max_moves=%d above 2^30", what,
                 max_moves);
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
