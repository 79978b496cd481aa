// q4_prefill.hip -- rows of prompts and chunks over a paged cache held in 4 bits (gfx950,
// head_dim 64 and 128).
//
// A workgroup of four waves takes one KV head of one sequence and 128 of its (row, query head)
// pairs, query head fastest, 32 pairs a wave, and walks the keys up to its last row in tiles of
// 64.  Each tile's codes are turned into operands once for all its waves: a wave brings its page
// of the tile into LDS as it is, one tile ahead (global_load_lds), and writes it out again as
// fp16 while the matrix cores are at the tile before.  The operands are exact (q4.h).  K's are
// (n + r) 2^-9 from the denormals that the codes are in a half's low bits (q4_decode.hip has the
// same); V's are (n + r) E: four bits in mantissa bits 6..9 below the exponent of 16 are 16 + n,
// and times E plus (r - 16) E that is it; E is the power of two that leaves s / E = m between 4
// and 8 (less for scales below 2^-12, up to 16 for those from 2^15 on, which rows of equal values
// have: a higher E would take their (r - 16) E past fp16).  K's s multiplies the scores inside
// the exponent's multiply-add, V's m a weight before its one rounding to fp16.
//
// Per tile, on v_mfma_f32_32x32x16_f16 with one lane per pair, in halves of 32 keys: S^T = K Q^T
// and O^T += V^T W^T beside the exponentials and the next codes' conversion, each operand read
// from LDS a phase before its product.
// Weights are taken against a reference that moves when a sum of 16 of a row's passes 2^12 (to
// 2^4 for the largest), seen from the weights themselves, so that no maximum of the scores is
// needed: 2^-11 of each holds down to 2^-16 of the reference, below it is an absolute 2^-27 of it.
//
// A key that holds NaN has operands of 0.  K's scale is NaN, which a row that does not see the
// key drops with its weight; of V's the first is kept, and the rows at or past it are NaN.
//
// Few rows over a long cache are cut into ranges of keys whose partials a second launch joins.
//
// What bounds it: the vector unit.  8192 rows of 32/8 heads of 128 take 619 to 660 us (550 GFLOP,
// 833 to 889 TFLOP/s, a third of the matrix cores' peak): it is busy for 62 % of the SIMDs' cycles
// (a tile's 32 exponentials of 16 cycles each, their multiply-adds, sums and conversions: some 960
// of 2600; the codes: 340), the matrix cores for 43 %, LDS for 55 % (each wave reads all of a
// tile's operands, 32 KB).  Two waves a SIMD is what 240 registers leave; more pairs a wave would
// halve the operand reads but not fit beside O.  Of what was tried: eight waves
// a workgroup (fewer conversions a pair, longer waits at its barriers) and hints to the scheduler
// were slower; pages through registers spilled (930 us); the row maxima in place of the check of
// the sums cost 11 us, sixteens in place of denormals for K 8.
#include "q4.h"

#include <algorithm>
#include <type_traits>

namespace kvhp {
namespace {

constexpr int kBN = 64;               // keys per tile
constexpr int kMaxRowHeads = 1 << 29; // (row, query head) pairs of a sequence: a grid of 2^22
constexpr int kCUs = 256;
constexpr int kLeastTiles = 3;        // of a range of keys
constexpr float kRefLog2 = 4.f;       // weights where a row's reference is set,
constexpr float kMostWeight = 4096.f; // and where it moves: times m, below 16, no more than 65504

struct PrefillPlan {
    uint32_t inv_g;        // ceil(2^32 / G), 0 for G = 1
    int blocks;            // of pairs, per sequence and KV head
    int batch;
    int tiles;             // of the longest sequence there may be
    int nsplit;            // ranges of keys a sequence may have
    // > 0: ranges over the batch, shared out by its lengths, where a CU has one workgroup, and
    // where it has as many as it holds
    int slots, slots_full;
    float* ws_o;           // [batch * rows * Hq][nsplit][D]
    float* ws_ml;          // [batch * rows * Hq][nsplit][2], the reference in log2 units
    int32_t* ws_range;     // tiles of a range
};

// Row of a pair: pair / G, exact for pair * G below 2^32.
__device__ __forceinline__ int row_of(const PrefillPlan& p, uint32_t pair) {
    return static_cast<int>(p.inv_g ? __umulhi(pair, p.inv_g) : pair);
}
// The rows of a block that lie in their sequence.
struct Block {
    int first;       // position of row 0
    int p_lo, p_hi;  // positions of the block's first and last live row; none: p_lo > p_hi
    __device__ __forceinline__ int tiles() const { return p_hi / kBN + 1; }
};
__device__ __forceinline__ Block block_of(const Q4Args& a, const PrefillPlan& p, int b, int blk, int pairs) {
    Block k;
    const int n = q4_len(a, b);
    // a start outside +-2^30 leaves no row among at most 2^30 keys
    const int64_t first = min(max(q4_first(a, b, n), -(int64_t)(1 << 30)), (int64_t)(1 << 30));
    const int r0 = row_of(p, blk * pairs), r1 = min(row_of(p, (blk + 1) * pairs - 1), a.rows - 1);
    k.first = static_cast<int>(first);
    k.p_lo = static_cast<int>(max(first + r0, (int64_t)0));
    k.p_hi = static_cast<int>(min(first + r1, (int64_t)n - 1));
    return k;
}

// What ranges cost in tiles of a workgroup that has its CU to itself (1.4 to 1.65 us at D = 128, 1.1 to
// 1.3 at 64): a tile of one of two (three; 2.7 us), and what they are written and joined in, the more
// ranges the longer.  (Chunks of 128 rows in four sequences of 1062 to 8192 keys, 32/8 heads of 128:
// 256 ranges of 47 tiles 86.6 us, 488 of 23 80.1; of 200 rows and up to 4096 keys, 32/4 of 64: 208 of
// 64 87.9, 724 of 13 53.0.  Without a regard to lengths 94.9 and 66.9.)
__host__ __device__ constexpr float full_tiles(int d, float tiles) { return (d == 128 ? 1.65f : 2.1f) * tiles + 4.f; }
constexpr int kJoinTiles = 5;

// Tiles of a range of keys where the batch's are shared out: the least with which there are no
// more ranges than slots, either way, and of the two the cheaper.  Each lane tries its own.
template <int D>
__device__ __forceinline__ int range_tiles(const Q4Args& a, const PrefillPlan& p, int lane, int& t) {
    t = 0;
    if (lane < p.batch) {
        const int n = q4_len(a, lane);
        const int64_t first = q4_first(a, lane, n), hi = min(first + a.rows - 1, (int64_t)n - 1);
        t = hi >= max(first, (int64_t)0) ? static_cast<int>(hi) / kBN + 1 : 0;
    }
    const int most = wave_max(t);
    const int total = __builtin_amdgcn_readlane(prefix_sum(t), kWave - 1);
    const int slots = lane < kWave / 2 ? p.slots : p.slots_full;
    const int least = max(max((total + slots - 1) / slots, kLeastTiles), (most + p.nsplit - 1) / p.nsplit);
    const int mine = least + (lane & (kWave / 2 - 1)) * (1 + least / 16);
    int count = 0;
    for (int b = 0; b < p.batch; ++b) count += (__builtin_amdgcn_readlane(t, b) + mine - 1) / mine;
    const uint64_t fit = __ballot(count <= slots);
    const uint32_t one = static_cast<uint32_t>(fit), full = static_cast<uint32_t>(fit >> 32);
    const int x = one ? __builtin_amdgcn_readlane(mine, __builtin_ctz(one)) : p.tiles;
    const int y = full ? __builtin_amdgcn_readlane(mine, kWave / 2 + __builtin_ctz(full)) : p.tiles;
    return full_tiles(D, y) < x ? y : x;
}

// The 16-byte chunks of LDS rows lie at c ^ swizzle(row): the 16 rows of an operand read of K,
// the four rows x four chunks of a transposing read of V, and the conversion's writes each on
// distinct banks.  V's is the same for rows 8 apart.
template <int D>
__device__ __forceinline__ int kswz(int r) { return D == 128 ? r & 15 : r >> 1 & 7; }
template <int D>
__device__ __forceinline__ int vswz(int r) {
    return D == 128 ? 5 * (r & 3) : 2 * (r & 3) + (r >> 1 & 1);
}

__device__ __forceinline__ half2v as_half2(uint32_t x) { return __builtin_bit_cast(half2v, x); }
struct CodeBits {
    uint32_t mask = 0x03c003c0u, sixteen = 0x4c004c00u, low = 0x000f000fu, high = 0x00f000f0u;
    // in registers: as literals they would keep v_and_or_b32 from taking both
    __device__ __forceinline__ CodeBits() { asm("" : "+s"(mask), "+v"(sixteen), "+s"(low), "+s"(high)); }
};
// Eight codes as (n + r) E, in the order 0 4 1 5 2 6 3 7.
__device__ __forceinline__ half8 operand(uint32_t x, half2v e, half2v f, const CodeBits& c) {
    auto pair = [&](uint32_t y) {
        return __builtin_elementwise_fma(as_half2((y & c.mask) | c.sixteen), e, f);
    };
    const half2v p0 = pair(x << 6), p1 = pair(x << 2), p2 = pair(x >> 2), p3 = pair(x >> 6);
    return half8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// Eight codes as (n + r) 2^-9, in the same order, given r 2^-9: four bits at the bottom of a half are
// n 2^-24, at bits 4..7 n 2^-20.
__device__ __forceinline__ half8 small_operand(uint32_t x, half2v f, const CodeBits& c) {
    auto pair = [&](uint32_t y, f16 e) {
        return __builtin_elementwise_fma(as_half2(y), half2v{e, e}, f);
    };
    const f16 e0 = 32768.f, e4 = 2048.f;
    const uint32_t y = x >> 8;
    const half2v p0 = pair(x & c.low, e0), p1 = pair(x & c.high, e4), p2 = pair(y & c.low, e0), p3 = pair(y & c.high, e4);
    return half8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

template <typename T>
__device__ __forceinline__ T lds_read(uint32_t at) {
    return *reinterpret_cast<const __attribute__((address_space(3))) T*>(at);
}
__device__ __forceinline__ short4v lds_tr16(uint32_t at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_short4v*>(at));
}

// global_load_lds_dwordx4 to LDS offset `to`, from a wave-uniform base and the lane's offset.
__device__ __forceinline__ void dma16(const void* base, uint32_t voff, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :: "s"(to), "v"(voff), "s"(base) : "memory", "m0");
}
// The same for the first 8 lanes of a whole wave (a branch would part the block that the
// products and the conversion share).
__device__ __forceinline__ void dma16_8(const void* base, uint32_t voff, uint32_t to) {
    uint64_t all;
    asm volatile("s_mov_b64 %0, exec\n\ts_mov_b64 exec, 0xff\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\t"
                 "global_load_lds_dwordx4 %2, %3\n\ts_mov_b64 exec, %0"
                 : "=&s"(all) : "s"(to), "v"(voff), "s"(base) : "memory", "m0");
}
template <int N>
__device__ __forceinline__ void wait_raw() {   // all but N loads have landed, and reads of LDS returned
    wait_ring<N>();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void reads_done() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
}

constexpr int kWaves = 4;             // each converts one page of a tile
constexpr int kPairs = 32 * kWaves;   // (row, head) pairs per workgroup
static_assert(kBN == kWaves * kPage, "a page per wave");

template <int D>
__global__ void __launch_bounds__(kWaves * kWave) __attribute__((amdgpu_waves_per_eu(D == 128 ? 2 : 3)))
q4_prefill_kernel(const Q4Args a, const PrefillPlan p) {
    constexpr int NC = D / 16, NDB = D / 32, RB = D / 2, PB = q4_page_bytes(D);
    constexpr uint32_t TB = 2 * kBN * D;   // bytes of a stage of operands
    constexpr int RAW = 2 * kPage * RB + 128;   // a page as it is in the pool, per wave
    constexpr int RST = D == 128 ? 1 : 2;       // stages of those
    // K's operands in two stages, then V's: multiples of 8 KB in LDS, so that an operand's place in
    // its row is an exclusive or with its address
    __shared__ __attribute__((aligned(8192))) f16 tiles[4 * kBN * D];
    __shared__ __attribute__((aligned(16))) uint8_t raw[kWaves][RST][RAW];
    // a tile's s log2(e) / sqrt(D) and m in the order a lane of half h takes them: [h][32 keys]
    __shared__ __attribute__((aligned(16))) float scale_s[2][kBN];
    __shared__ __attribute__((aligned(16))) f16 scale_m[2][kBN];
    __shared__ int bad[kWaves];            // each wave's first key whose V is NaN

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int h = lane >> 5, c32 = lane & 31;
    const int kvh = blockIdx.x % a.Hkv;
    const int blk = p.blocks - 1 - static_cast<int>(blockIdx.x / a.Hkv);   // longest first
    int b = blockIdx.y, split = blockIdx.z, range = (p.tiles + p.nsplit - 1) / p.nsplit;
    if (p.slots) {   // the blockIdx.y-th range of the batch
        int t;
        range = range_tiles<D>(a, p, lane, t);
        const uint32_t mine = (t + range - 1) / range, upto = prefix_sum(mine);
        const uint64_t past = __ballot(upto > blockIdx.y);
        if (past == 0) return;
        b = __builtin_ctzll(past);
        split = blockIdx.y - (__builtin_amdgcn_readlane(upto, b) - __builtin_amdgcn_readlane(mine, b));
    }
    if (p.nsplit > 1 && (blockIdx.x | blockIdx.y | blockIdx.z | threadIdx.x) == 0) *p.ws_range = range;
    const Block k = block_of(a, p, b, blk, kPairs);
    if (k.p_lo > k.p_hi) return;
    const int t_lo = split * range;
    const int all_tiles = k.tiles();
    const int n = min(all_tiles - t_lo, range);
    if (n <= 0) return;

    // This lane's pair.
    const int pair0 = blk * kPairs + 32 * wave, pair = pair0 + c32;
    const int row = row_of(p, pair), qh = kvh * a.G + pair - row * a.G, pos = k.first + row;
    const bool live = row < a.rows && pos >= k.p_lo && pos <= k.p_hi;
    const int64_t at = ((int64_t)b * a.rows + row) * a.Hq + qh;
    // tiles from `past` on (of the range's) hold keys that some pair of the wave does not see
    const int lo = k.first + row_of(p, pair0), hi = k.first + row_of(p, pair0 + 31);
    const int past = (lo < k.p_lo || hi > k.p_hi || lo < kBN - 1 ? 0 : (lo - (kBN - 1)) / kBN + 1) - t_lo;
    const int seen0 = live ? pos - t_lo * kBN - 4 * h : -1;
    half8 qop[NC];   // in the codes' order
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const half8 x = live ? load_half8(a.q + at * D + 16 * c + 8 * h) : half8{};
        qop[c] = __builtin_shufflevector(x, x, 0, 4, 1, 5, 2, 6, 3, 7);
    }

    // ---- codes: a wave loads its page of each tile and converts it, a lane D / 4 dims of a row
    const int crow = lane >> 2, cc = lane & 3;
    const int key0 = t_lo * kBN + kPage * wave + crow;   // in the range's first tile
    const int32_t* bt = a.bt + (int64_t)b * a.max_pages;
    const uint8_t* head = a.pool + (int64_t)kvh * a.num_pages * PB;
    const int last_page = k.p_hi >> 4;
    // Page ids of 64 tiles, a lane each (clamped into the pool): loaded tile by tile, each would be
    // waited for with the next reads of LDS.
    int ids = 0;
    auto page_of = [&](int t) {
        if (t % kWave == 0 && t < n) {
            const int pi = min((t_lo + min(t + lane, n - 1)) * kWaves + wave, last_page);
            ids = min(max(bt[pi], 0), a.num_pages - 1);
        }
        return __builtin_amdgcn_readlane(ids, t % kWave);
    };
    const uint8_t* const raw0 = raw[wave][0];
    const uint32_t raw_at = __builtin_amdgcn_readfirstlane(lds_at(raw0));
    // D = 128: K's codes and the numbers, then V's codes; D = 64: all at once, to a stage of its own
    auto ask_k = [&](int t, int pid) {
        const uint8_t* pg = head + (int64_t)pid * PB;
        const uint32_t to = raw_at + (RST == 2 ? (t & 1) * RAW : 0);
        dma16(pg, 16 * lane, to);
        dma16_8(pg, kPage * D + 16 * lane, to + 2 * kPage * RB);
    };
    auto ask_v = [&](int pid) {
        if constexpr (D == 128) dma16(head + (int64_t)pid * PB, 1024 + 16 * lane, raw_at + 1024);
    };
    const CodeBits bits;
    const uint32_t lds0 = lds_at(tiles);
    const uint32_t kput = 2 * ((kPage * wave + crow) * D) + 16 * ((D / 32 * cc) ^ kswz<D>(kPage * wave + crow));
    const uint32_t vput = 2 * ((kPage * wave + crow) * D) + 16 * ((D / 32 * cc) ^ vswz<D>(kPage * wave + crow));
    auto convert = [&](const uint8_t* codes, auto&& operand_of, uint32_t to) {
        uint32_t x[D / 32];
        if constexpr (D == 128) {
            const u32x4 y = *reinterpret_cast<const u32x4*>(codes);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = y[i];
        } else {
            const uint2 y = *reinterpret_cast<const uint2*>(codes);
            x[0] = y.x;
            x[1] = y.y;
        }
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            *reinterpret_cast<__attribute__((address_space(3))) half8*>(to ^ 16 * i) = operand_of(x[i]);
    };
    // This lane's row of a tile's V: E and (r - 16) E, kept from the numbers' read to the codes'.
    half2v v_e, v_f;
    int nan_at = INT32_MAX;   // the wave's first key whose V is NaN
    // A row's s and m: key 32 n + 8 q + 4 h + e to [h][16 n + 4 q + e].
    const int srow = kPage * wave + crow;
    const int sat = 32 * (srow >> 2 & 1) + 16 * (srow >> 5) + 4 * (srow >> 3 & 3) + (srow & 3);
    auto put_k = [&](int t) {
        const uint8_t* r0 = raw0 + (RST == 2 ? (t & 1) * RAW : 0);
        const uint8_t* num = r0 + 2 * kPage * RB + 4 * crow;
        uint32_t ks = *reinterpret_cast<const uint32_t*>(num), vs = *reinterpret_cast<const uint32_t*>(num + 64);
        const bool behind = key0 + t * kBN > k.p_hi;   // the last key
        scale_s[t & 1][sat] = static_cast<float>(as_half2(ks)[0]) * (512.f * a.scale_log2);   // by four lanes alike
        // of NaN and of what is behind the last key: operands of 0
        ks = behind || (ks & 0x7c00u) == 0x7c00u ? 0u : ks;
        const bool nan = !behind && (vs & 0x7c00u) == 0x7c00u;
        vs = behind || nan ? 0u : vs;
        const int e = min(max((int)(vs & 0x7c00u) - 0x0800, 0x0400), 0x6c00);   // 2^-14 .. 2^12
        scale_m[t & 1][sat] = as_half2(vs)[0] * __builtin_bit_cast(f16, static_cast<uint16_t>(0x7800 - e));   // exact
        const uint64_t nans = __ballot(nan);
        nan_at = nans && nan_at == INT32_MAX ? t_lo * kBN + t * kBN + kPage * wave + (__builtin_ctzll(nans) >> 2) : nan_at;
        const f16 eh = __builtin_bit_cast(f16, static_cast<uint16_t>(e));
        v_e = half2v{eh, eh};
        v_f = (half2v{as_half2(vs)[1], as_half2(vs)[1]} + half2v{f16(-16), f16(-16)}) * v_e;
        const half2v k_f = half2v{as_half2(ks)[1], as_half2(ks)[1]} * half2v{f16(0x1p-9f), f16(0x1p-9f)};
        convert(r0 + RB / 4 * lane, [&](uint32_t x) { return small_operand(x, k_f, bits); },
                lds0 + (t & 1) * TB + kput);
    };
    auto put_v = [&](int t) {
        convert(raw0 + (RST == 2 ? (t & 1) * RAW : 0) + kPage * RB + RB / 4 * lane,
                [&](uint32_t x) { return operand(x, v_e, v_f, bits); }, lds0 + (2 + (t & 1)) * TB + vput);
    };

    // ---- operand reads: K's chunk 2 c + h of row c32 (and 32), V's of 32-dim block db
    const uint32_t kat = lds0 + 2 * c32 * D + 16 * (h ^ kswz<D>(c32));
    uint32_t vat;
    {
        const int j16 = lane & 15, r = 4 * h + j16 / 4;
        vat = lds0 + 2 * TB + 2 * r * D + 16 * ((2 * (lane >> 4 & 1) + ((j16 & 3) >> 1)) ^ vswz<D>(r)) + 8 * (j16 & 1);
    }
    floatx16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m_run = -1e30f, l_part = 0.f;

    // Operands are read a phase ahead of their products: left to itself the compiler reads one
    // and waits for it, product by product.
    struct KOps {
        half8 x[NC];
    };
    struct VOps {
        half8 x[2][NDB];
    };
    auto read_k = [&](int j, int u) {
        const uint32_t Kt = kat + (j & 1) * TB;
        KOps k8;
#pragma unroll
        for (int c = 0; c < NC; ++c) k8.x[c] = lds_read<half8>((Kt ^ 32 * c) + 64 * u * D);
        return k8;
    };
    auto read_v = [&](int j, int u) {
        const uint32_t Vt = vat + (j & 1) * TB + 64 * u * D;
        VOps v8;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int db = 0; db < NDB; ++db) {
                const uint32_t q = (Vt ^ 64 * db) + 32 * t * D;
                v8.x[t][db] = cat_half8(lds_tr16(q), lds_tr16(q + 16 * D));
            }
        return v8;
    };
    auto fence = []() { asm volatile("" ::: "memory"); };
    // Scores of half u of tile j: element i is key 32 u + 8 (i / 4) + 4 h + i % 4.
    auto qk = [&](const KOps& k8) {
        floatx16 s = {};
#pragma unroll
        for (int c = 0; c < NC; ++c) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k8.x[c], qop[c], s, 0, 0, 0);
        return s;
    };
    // Weights as the operands of O^T's product; returns their sum before the rounding.
    auto weights = [&](auto MASKED_, int j, int u, const floatx16& s, half8 (&w)[2]) {
        constexpr bool MASKED = decltype(MASKED_)::value;
        float ps[2] = {0.f, 0.f};
        int seen = seen0 - j * kBN - 32 * u;
        asm volatile("" : "+v"(seen));   // compared where it is used: kept masks would spill
        const float* ks = &scale_s[j & 1][32 * h + 16 * u];
        const f16* vm = &scale_m[j & 1][32 * h + 16 * u];
        // in fp16, where it is exact, and multiplied from there (v_fma_mix_f32; a product gets no such)
        const half8 m8[2] = {*reinterpret_cast<const half8*>(vm), *reinterpret_cast<const half8*>(vm + 8)};
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const floatx4 k4 = *reinterpret_cast<const floatx4*>(ks + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = fast_exp2(fmaf(s[i + e], k4[e], -m_run));
                if (MASKED && 2 * i + e > seen) x = 0.f;
                w[i / 8][i % 8 + e] = static_cast<f16>(fmaf(x, static_cast<float>(m8[i / 8][i % 8 + e]), 0.f));
                ps[e & 1] += x;
            }
        }
        return ps[0] + ps[1];
    };
    // Moves the reference of rows with a weight past 2^12 to 2^4 below their largest score.
    auto refer = [&](int j, int u, const floatx16& s) {
        float t = -INFINITY;
        int seen = seen0 - j * kBN - 32 * u;
        asm volatile("" : "+v"(seen));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = s[i] * scale_s[j & 1][32 * h + 16 * u + i];
            if (8 * (i / 4) + i % 4 <= seen) t = fmaxf(t, x);
        }
        t = halves_max(t);
        const float mn = fmaxf(m_run, t - kRefLog2);
        const float alpha = fast_exp2(m_run - mn);
        l_part *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db] *= alpha;
        m_run = mn;
    };
    auto pv = [&](const VOps& v8, const half8 (&w)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int db = 0; db < NDB; ++db)
                o[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8.x[t][db], w[t], o[db], 0, 0, 0);
    };
    // A weight past 2^12 shows in the sum (which passes it with none that large only where the
    // reference would have moved before long).
    auto checked = [&](int j, int u, float sum, const floatx16& s, half8 (&w)[2]) {
        if (__builtin_amdgcn_read_exec() & __ballot(sum > kMostWeight)) {
            refer(j, u, s);   // now none is past 2^4
            sum = weights(std::true_type{}, j, u, s, w);
        }
        l_part += sum;
    };

    // ---- the pipeline: iteration j works on tile j, converts the codes of tile j + 1 and asks
    // for those of j + 2: S of the first half beside K's conversion, S of the second beside the
    // first's weights, O of the first beside the second's weights, O of the second beside V's
    // conversion
    int pid = page_of(0);
    wait_raw<0>();
    ask_k(0, pid);
    ask_v(pid);
    pid = page_of(1);
    wait_raw<0>();
    put_k(0);
    put_v(0);
    reads_done();
    ask_k(1, pid);
    ask_v(pid);
    pid = page_of(2);
    // MASKED: some row of the wave does not see all of the tile
    auto iterate = [&](auto LAST_, auto MASKED_, int j) {
        constexpr bool LAST = decltype(LAST_)::value;
        reads_done();   // and this wave's writes are in LDS
        ring_barrier();
        if constexpr (!LAST && RST == 2) ask_k(j + 2, pid);
        const KOps k0 = read_k(j, 0), k1 = read_k(j, 1);
        fence();
        const floatx16 s0 = qk(k0);
        if constexpr (!LAST) {
            wait_raw<RST == 2 ? 2 : 1>();
            put_k(j + 1);
            if constexpr (RST == 1) {
                reads_done();
                ask_k(j + 2, pid);
            }
        }
        const VOps v0 = read_v(j, 0);
        fence();
        const floatx16 s1 = qk(k1);
        half8 w0[2], w1[2];
        checked(j, 0, weights(MASKED_, j, 0, s0, w0), s0, w0);
        const VOps v1 = read_v(j, 1);
        fence();
        pv(v0, w0);
        checked(j, 1, weights(MASKED_, j, 1, s1, w1), s1, w1);
        pv(v1, w1);
        if constexpr (!LAST) {
            if constexpr (RST == 1) wait_raw<2>();
            put_v(j + 1);
            reads_done();
            ask_v(pid);
            pid = page_of(j + 3);
        }
    };
    int j = 0;
    for (const int whole = min(past, n - 1); j < whole; ++j) iterate(std::false_type{}, std::false_type{}, j);
    for (; j + 1 < n; ++j) iterate(std::false_type{}, std::true_type{}, j);
    wait_raw<0>();   // the trailing loads
    bad[wave] = nan_at;
    iterate(std::true_type{}, std::true_type{}, j);
    ring_barrier();   // the operands' place takes the results
    int first_bad = bad[0];   // written before the last tile's barrier
#pragma unroll
    for (int w = 1; w < kWaves; ++w) first_bad = min(first_bad, bad[w]);
    const bool cut = all_tiles > range;   // joined by q4_prefill_join_kernel
    const float l = halves_sum(l_part);
    if (live && h == 0) {
        if (cut) {
            const int64_t prow = at * p.nsplit + split;
            p.ws_ml[prow * 2] = m_run;
            p.ws_ml[prow * 2 + 1] = l;
        } else if (a.lse) {
            a.lse[((int64_t)b * a.Hq + qh) * a.rows + row] = (m_run + __builtin_amdgcn_logf(l)) * kLn2;
        }
    }
    // Rows of D floats in LDS, 16-byte chunk c of row r at c ^ r: a lane has dims 32 db + 8 q +
    // 2 h + (0 4 1 5) of its pair and writes whole rows out.
    constexpr int CPR = D / 4;
    const float scale = pos >= first_bad ? NAN : cut ? 1.f : 1.f / l;
    float* const mine = reinterpret_cast<float*>(tiles) + 32 * D * wave;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                *reinterpret_cast<float2*>(mine + D * c32 + 4 * ((8 * db + 2 * q4 + e) ^ (c32 & (CPR - 1))) + 2 * h) =
                    float2{o[db][4 * q4 + e] * scale, o[db][4 * q4 + 2 + e] * scale};
    auto row_at = [&](int r, int64_t& to) {   // where the wave's r-th pair goes, if anywhere
        const int pr = pair0 + r, rw = row_of(p, pr);
        to = ((int64_t)b * a.rows + rw) * a.Hq + kvh * a.G + pr - rw * a.G;
        return rw < a.rows && k.first + rw >= k.p_lo && k.first + rw <= k.p_hi;
    };
    auto chunk = [&](int r, int c) {
        return *reinterpret_cast<const floatx4*>(mine + D * r + 4 * (c ^ (r & (CPR - 1))));
    };
    int64_t to;
    if (cut) {
        for (int i = lane; i < 32 * CPR; i += kWave) {
            const int r = i / CPR, c = i % CPR;
            if (row_at(r, to)) *reinterpret_cast<floatx4*>(p.ws_o + (to * p.nsplit + split) * D + 4 * c) = chunk(r, c);
        }
        return;
    }
    for (int i = lane; i < 32 * (CPR / 2); i += kWave) {
        const int r = i / (CPR / 2), c = i % (CPR / 2);
        if (!row_at(r, to)) continue;
        const floatx4 x = chunk(r, 2 * c), y = chunk(r, 2 * c + 1);
        half8 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[e] = static_cast<f16>(x[e]);
            v[4 + e] = static_cast<f16>(y[e]);
        }
        store_half8(a.out + to * D + 8 * c, q4_finite(v));
    }
}

// Joins the partials of the blocks that were cut into ranges of keys: R times D / 8 lanes per
// (row, head), lane (r, c) taking dims 8c .. of every R-th range.
template <int D, int R>
__global__ void __launch_bounds__(256) q4_prefill_join_kernel(const Q4Args a, const PrefillPlan p, int pairs) {
    constexpr int LPR = D / 8;
    const int c = threadIdx.x % LPR, r = threadIdx.x / LPR % R;
    const int b = blockIdx.y;
    const uint32_t i = blockIdx.x * (256 / LPR / R) + threadIdx.x / (LPR * R);
    const int row = static_cast<int>(i / a.Hq), qh = static_cast<int>(i % a.Hq);
    if (row >= a.rows) return;
    const Block k = block_of(a, p, b, (row * a.G + qh - row_of(p, qh) * a.G) / pairs, pairs);
    const int64_t pos = (int64_t)k.first + row;
    if (pos < k.p_lo || pos > k.p_hi) return;
    const int tiles = k.tiles();
    const int range = *p.ws_range;
    if (tiles <= range) return;
    const int n = (tiles + range - 1) / range;
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
    constexpr int U = 4;   // ranges in flight
    for (int j0 = r; j0 < n; j0 += U * R) {
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
    }
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
    store_half8(a.out + at * D + 8 * c, q4_finite(hv));
    if (a.lse && c == 0)
        a.lse[((int64_t)b * a.Hq + qh) * a.rows + row] = (M + __builtin_amdgcn_logf(L)) * kLn2;
}

// Blocks of few rows are cut into ranges of keys, one a CU or as many as it holds, where that
// saves more than it costs.  Up to 64 sequences' ranges are shared out by their lengths as they are.
PrefillPlan plan_of(int batch, int rows, int hkv, int G, int d, int max_len) {
    PrefillPlan p{};
    const int64_t pairs = (int64_t)rows * G;
    const int64_t per = (pairs + kPairs - 1) / kPairs * hkv;   // workgroups of a sequence
    p.inv_g = G == 1 ? 0 : static_cast<uint32_t>(((uint64_t(1) << 32) + G - 1) / G);
    p.blocks = static_cast<int>((pairs + kPairs - 1) / kPairs);
    p.batch = batch;
    p.tiles = static_cast<int>(((int64_t)max_len + kBN - 1) / kBN);
    p.nsplit = 1;
    const int64_t one = kCUs / per, full = (d == 64 ? 3 : 2) * kCUs / per;
    const auto range = [&](int64_t slots) {   // of equal sequences
        const int64_t n = slots / batch;
        return n > 1 ? std::max<int64_t>((p.tiles + n - 1) / n, kLeastTiles) : p.tiles;
    };
    if (kJoinTiles + std::min<float>(range(one), full_tiles(d, range(full))) >= p.tiles) return p;
    const int64_t most = p.tiles / kLeastTiles;
    if (batch > kWave) {
        p.nsplit = static_cast<int>(std::min(full / batch, most));
    } else {
        p.slots = static_cast<int>(std::max<int64_t>(one, batch));
        p.slots_full = static_cast<int>(full);
        // a sequence's at most twice its share
        p.nsplit = static_cast<int>(std::min(batch == 1 ? full : 2 * ((full + batch - 1) / batch), most));
    }
    return p;
}

}  // namespace

size_t q4_prefill_workspace(int batch, int rows, int hq, int hkv, int d, int max_len) {
    if (rows <= 0 || !bound_sizes(batch, hq, hkv, max_len, 0, 0) ||
        (int64_t)rows * hq > kMaxRowHeads || (d != 64 && d != 128))
        return 0;
    const PrefillPlan p = plan_of(batch, rows, hkv, hq / hkv, d, max_len);
    return p.nsplit == 1 ? 0 : sizeof(float) * ((size_t)batch * rows * hq * p.nsplit * (d + 2) + 1);
}

bool q4_prefill_fits(const Q4Args& a, int batch) {
    if ((int64_t)a.rows * a.Hq > kMaxRowHeads) return false;   // the plan counts them in an int
    const PrefillPlan p = plan_of(batch, a.rows, a.Hkv, a.G, a.D, a.max_len);
    return (a.D == 64 || a.D == 128) && aligned16(a.q) && aligned16(a.out) && p.nsplit <= 65535 &&
           (int64_t)p.blocks * a.Hkv <= kMaxRowHeads / kPairs &&
           (int64_t)a.rows * a.G * a.G < (int64_t)1 << 31;   // row_of, and pairs in an int
}

// The workspace holds q4_prefill_workspace bytes.
int q4_prefill(const Q4Args& a, int batch, void* ws, hipStream_t s) {
    PrefillPlan p = plan_of(batch, a.rows, a.Hkv, a.G, a.D, a.max_len);
    const size_t rh = (size_t)batch * a.rows * a.Hq;
    p.ws_o = static_cast<float*>(ws);
    p.ws_ml = p.ws_o + rh * p.nsplit * a.D;
    p.ws_range = reinterpret_cast<int32_t*>(p.ws_ml + rh * p.nsplit * 2);
    const dim3 threads(kWaves * kWave);
    const dim3 grid = p.slots ? dim3(p.blocks * a.Hkv, p.slots_full) : dim3(p.blocks * a.Hkv, batch, p.nsplit);
    if (a.D == 64)
        hipLaunchKernelGGL((q4_prefill_kernel<64>), grid, threads, 0, s, a, p);
    else
        hipLaunchKernelGGL((q4_prefill_kernel<128>), grid, threads, 0, s, a, p);
    const int rc = check_launch("q4_prefill");
    if (rc || p.nsplit == 1) return rc;
    // A wave per (row, head) while they all run at once, D / 8 lanes above.
    const int64_t heads = (int64_t)batch * a.rows * a.Hq;   // rows Hq <= 2^29
    auto join = [&](auto kernel, int lanes) {
        const unsigned per = 256 / lanes;
        hipLaunchKernelGGL(kernel, dim3((static_cast<unsigned>(a.rows) * a.Hq + per - 1) / per, batch),
                           dim3(256), 0, s, a, p, kPairs);
    };
    if (a.D == 64)
        heads <= 32 * kCUs ? join(q4_prefill_join_kernel<64, 8>, 64) : join(q4_prefill_join_kernel<64, 1>, 8);
    else
        heads <= 32 * kCUs ? join(q4_prefill_join_kernel<128, 4>, 64) : join(q4_prefill_join_kernel<128, 1>, 16);
    return check_launch("q4_prefill (join)");
}

}  // namespace kvhp
