// bounded_decode.hip -- one new token per sequence over a cache of bounded
// length: sliding window and first tokens, or every key with its attention
// weight summed per slot (gfx950, head_dim 64 and 128).
//
// The visible keys of a sequence, its first `sinks` and its last `window`, are
// numbered through without the gap between them, so a sequence is
// min(n, sinks + window) keys long and nothing hidden is loaded or masked.
// From there on it is split-K decode: a wave takes a chunk of keys in steps of
// 32, both contractions on v_mfma_f32_16x16x32_f16 in transposed form so that
// a lane owns one query head through the online softmax,
//   S^T = K Q^T      A = K rows through LDS, B = Q^T in registers
//   O^T += V^T P^T   A = V^T by transposing LDS reads, B = P^T from S^T's
//                    accumulators, rounded to fp16 (2^-11 of each down to 2^-14 of
//                    the split's largest, an absolute 2^-25 of it below, less than
//                    2^-14 over a split; the softmax's sum takes them unrounded)
// K is fetched two steps ahead and V one, as whole rows.  A key's row is found
// through the chunk's page ids, one per lane, by an exchange between lanes:
// with a window the chunks start anywhere in a page.  Up to 16 query heads of
// a KV head go together; larger groups read the keys once per 16.
//
// Sums: the scores go to the workspace in fp32, 32 keys of each head side by side;
// once the maximum and the sum of every head are known from the chunks' partials,
// the launch that joins the partials also turns the scores into weights, adds them
// over the heads of a KV head and updates the slots; a workgroup that holds all heads and
// keys of a KV head does so itself, without a second launch.  (16 bytes a key and four
// heads, written and read, beside 512 of K and V at D = 128.  Written past the
// caches they cost 132 us instead of 125 below.)
//
// Bound by HBM, 4 D bytes per visible key and KV head, where there is much of it.  32
// sequences of up to 8192 keys, 32/8 heads of 128: windows of 4096 73.5 us, 412 MB at
// 5.6 TB/s (shuffled pages alone read at 5.9-6.3); every key with its sums 122-125 us, of
// which 114 are the first launch's, 579 MB at 5.1 TB/s, and 11 the second's.  One
// sequence of 1028 visible keys at D = 64 takes 6.9 us and 500 5.1, in one launch, 2048 with
// sums 8.7: launches, and the latency of their loads.  Where several waves share a split,
// each joins the dims of one MFMA block for all of them (one wave joining everything cost
// 0.7 us more at D = 64 and 2 at D = 128).
#include "bounded.h"

#include <type_traits>

namespace kvhp {
namespace {

constexpr int kMaxChunk = 960;    // keys per split: at most 64 pages, three of them cut
constexpr int kMinChunk = 64;     // (of a batch's own splits)
constexpr int kMaxOne = 1152;     // and where one split takes all, at D = 64 (75 pages)
constexpr int kHeads = 16;        // query heads per workgroup
constexpr int kBalanced = 16;     // sequences from which the splits are the whole batch's

struct DecodePlan {
    int chunk;        // keys per split (fixed mode), a multiple of 32
    int nsplit;       // split slots in the workspace
    int batch;
    int balance;      // > 0: about this many splits per KV head over the batch
    int groups;       // workgroups per KV head and split, of up to kHeads query heads
    int fused;        // 1: one split and one workgroup per KV head, which adds its sums itself
    int scap;         // keys that the scores have room for, a multiple of 32
    float* ws_o;      // [B * Hq][nsplit][D]
    float* ws_ml;     // [B * Hq][nsplit][2], the maximum in log2 units
    float* ws_s;      // [B][Hkv][scap / 32][G][32] raw scores
};

// Where the scores of the 32 keys from j (a multiple of 32) on lie: [head of the group][32].
__device__ __forceinline__ int64_t score_at(const BoundArgs& a, const DecodePlan& p, int b,
                                            int kvh, int j) {
    return (((int64_t)b * a.Hkv + kvh) * p.scap + j) * a.G;
}
// Visible keys of sequence b.
__device__ __forceinline__ int vis_len(const BoundArgs& a, int b) {
    const int n = bound_len(a, b);
    return a.window > 0 ? static_cast<int>(min((int64_t)n, (int64_t)a.sinks + a.window)) : n;
}

__device__ __forceinline__ long long batch_keys(const BoundArgs& a, int batch, int lane) {
    long long t = 0;
    for (int i = lane; i < batch; i += kWave) t += vis_len(a, i);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) t += __shfl_xor(t, o);
    return t;
}

// Keys per split of a sequence of L visible keys; split and join agree on it.
__device__ __forceinline__ int chunk_of(const DecodePlan& p, int L, long long keys) {
    if (p.balance <= 0 || L <= 0) return p.chunk;
    const int target = static_cast<int>(
        min(max((keys + p.balance - 1) / p.balance, (long long)kMinChunk), (long long)kMaxChunk));
    const int n = min((L + target - 1) / target, p.nsplit);
    return ((L + n - 1) / n + 31) / 32 * 32;   // at most kMaxChunk; whole steps
}

// Four keys of a KV head from j (a multiple of 4) on: their slot (-1: none) and sums.
struct Quad {
    int64_t slot;
    floatx4 old;
};
__device__ __forceinline__ Quad quad_at(const BoundArgs& a, int b, int kvh, int j) {
    Quad q{bound_slot(a.k, b, kvh, j), {0.f, 0.f, 0.f, 0.f}};   // four in one page
    if (q.slot >= 0) q.old = *reinterpret_cast<const floatx4*>(a.weights + q.slot);
    return q;
}
// Adds the weights w of keys j .. j + 3 to their sums, or starts them, with their ages.
__device__ __forceinline__ void put_quad(const BoundArgs& a, const Quad& q, int b, int j, int n,
                                         const floatx4& w) {
    if (j >= n || q.slot < 0) return;
    const int64_t fresh = (int64_t)n - a.new_keys;     // keys from here on start anew
    floatx4 x = q.old;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (j + e < n) x[e] = j + e >= fresh ? w[e] : x[e] + w[e];
    *reinterpret_cast<floatx4*>(a.weights + q.slot) = x;   // slots behind the sequence as they were
    if (a.ages && j + 3 >= fresh) {
        const int newest = a.newest ? a.newest[b] : n - 1;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < n && j + e >= fresh) a.ages[q.slot + e] = newest - (n - 1 - j - e);
    }
}

// W waves per workgroup take the steps of one split round robin and meet in LDS.
// WIDE: rows may lie 2^32 bytes and more behind their head's first.
template <int D, bool PAGED, bool SUMS, int W, bool WIDE = false>
__global__ void __launch_bounds__(W * kWave) __attribute__((amdgpu_waves_per_eu(2)))
bound_decode_kernel(const BoundArgs a, const DecodePlan p) {
    constexpr int TOK = 32, NC = D / 32, ND = D / 16;
    constexpr int LPR = D / 8, RPL = kWave / LPR, NVL = TOK / RPL;
    constexpr int VP = D + 16, KP = D + 8;   // row pitches in LDS (bank skew)
    __shared__ __attribute__((aligned(16))) f16 v_lds_all[W][TOK * VP];
    __shared__ __attribute__((aligned(16))) f16 k_lds_all[W][TOK * KP];

    const int lane = threadIdx.x & (kWave - 1);
    const int wv = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    f16* const v_lds = v_lds_all[wv];
    f16* const k_lds = k_lds_all[wv];
    const int g = lane >> 4, col = lane & 15;
    const int kvh = blockIdx.x / p.groups, h0 = blockIdx.x % p.groups * kHeads;
    int b, split, L, chunk;
    if (W == 1 && p.balance > 0) {
        // The work list: blockIdx.y counts the splits of the batch in sequence
        // order (sequences without keys keep one, which writes their zeros).
        const long long keys = batch_keys(a, p.batch, lane);
        const int i = blockIdx.y;
        int base = 0;
        b = -1, split = 0, L = 0, chunk = p.chunk;
        for (int g0 = 0; g0 < p.batch; g0 += kWave) {
            const bool in = g0 + lane < p.batch;
            const int li = in ? vis_len(a, g0 + lane) : 0;
            const int ci = chunk_of(p, li, keys);
            const int ni = in ? (li > 0 ? (li + ci - 1) / ci : 1) : 0;
            int inc = ni;
#pragma unroll
            for (int o = 1; o < kWave; o <<= 1) {
                const int t = __shfl_up(inc, o);
                if (lane >= o) inc += t;
            }
            const int tot = __shfl(inc, kWave - 1);
            if (i < base + tot) {
                const int owner = __builtin_ctzll(__ballot(base + inc > i));
                b = g0 + owner;
                split = i - base - (__shfl(inc, owner) - __shfl(ni, owner));
                L = __shfl(li, owner);
                chunk = __shfl(ci, owner);
                break;
            }
            base += tot;
        }
        if (b < 0) return;
        b = __builtin_amdgcn_readfirstlane(b);
        split = __builtin_amdgcn_readfirstlane(split);
        L = __builtin_amdgcn_readfirstlane(L);
        chunk = __builtin_amdgcn_readfirstlane(chunk);
    } else {
        split = blockIdx.y;
        b = blockIdx.z;
        L = vis_len(a, b);
        chunk = p.chunk;
    }
    const int nh = min(a.G - h0, kHeads);   // query heads of this workgroup
    const int64_t row0 = (int64_t)b * a.Hq + (int64_t)kvh * a.G + h0;
    if (L <= 0) {
        if (split == 0)
            for (int i = threadIdx.x; i < nh * LPR; i += W * kWave)
                store_half8(a.out + row0 * D + 8 * i, half8{});
        return;
    }
    const int nsb = (L + chunk - 1) / chunk;
    if (split >= nsb) return;
    const int t_begin = split * chunk;
    const int t_end = min(L, t_begin + chunk);
    const int n_iter = (t_end - t_begin + TOK - 1) / TOK;
    const bool hvalid = col < nh;

    // Visible key v is position v + (v >= sinks ? shift : 0).
    const int shift = a.window > 0 ? bound_len(a, b) - L : 0;
    const int sinks = shift > 0 ? a.sinks : 0;
    // Page ids of the chunk, one per lane (two where one split takes all, up to 75 pages):
    // those of its first tokens, then the others.
    constexpr bool kTwo = (W == 8 || WIDE) && D == 64 && !SUMS;
    int pidv = 0, pid2 = 0, n_a = 0, p_a = 0, p_b = 0;
    if constexpr (PAGED) {
        p_a = t_begin >> 4;
        n_a = t_begin < sinks ? ((min(t_end, sinks) - 1) >> 4) - p_a + 1 : 0;
        p_b = (max(t_begin, sinks) + shift) >> 4;
        const int last = t_end > sinks ? (t_end - 1 + shift) >> 4 : (t_end - 1) >> 4;
        auto page = [&](int i) {
            const int pi = min(i < n_a ? p_a + i : p_b + i - n_a, last);
            return min(max(a.k.bt[(int64_t)b * a.k.max_pages + pi], 0), a.k.num_pages - 1);
        };
        pidv = page(lane);
        if constexpr (kTwo) pid2 = page(lane + kWave);
    }
    const char* kbase = reinterpret_cast<const char*>(
        a.k.data + (PAGED ? 0 : b * a.k.stride_b) + kvh * a.k.stride_h);
    const char* vbase = reinterpret_cast<const char*>(
        a.v.data + (PAGED ? 0 : b * a.v.stride_b) + kvh * a.v.stride_h);

    half8 qb[NC];   // lane (g, col): head col, dims 32c + 8g ..
#pragma unroll
    for (int c = 0; c < NC; ++c)
        qb[c] = hvalid ? load_half8(a.q + (row0 + col) * D + 32 * c + 8 * g) : half8{};

    const int vrow = lane / LPR, vdim = 8 * (lane % LPR);
    using offset = std::conditional_t<WIDE, uint64_t, uint32_t>;
    const offset ssk = 2 * (offset)a.k.stride_s, ssv = 2 * (offset)a.v.stride_s;

    // This lane's row of load j of the step at T0; past the split's last key: that one.
    auto rows = [&](int T0, uint32_t (&r)[NVL]) {
#pragma unroll
        for (int j = 0; j < NVL; ++j) {
            const int v = min(T0 + RPL * j + vrow, t_end - 1);
            const bool first = v < sinks;
            const int real = first ? v : v + shift;
            if constexpr (PAGED) {
                const int at = first ? (real >> 4) - p_a : (real >> 4) - p_b + n_a;
                int pid = __builtin_amdgcn_ds_bpermute(at << 2, pidv);
                if constexpr (kTwo) {
                    const int other = __builtin_amdgcn_ds_bpermute(at << 2, pid2);
                    pid = at < kWave ? pid : other;
                }
                r[j] = (uint32_t)pid * kPage + (real & 15);
            } else {
                r[j] = real;
            }
        }
    };
    half8 kbuf[2][NVL], vbuf[NVL];
    auto load_k = [&](auto S_, int T0) {
        constexpr int S = decltype(S_)::value;
        uint32_t r[NVL];
        rows(T0, r);
#pragma unroll
        for (int j = 0; j < NVL; ++j)
            kbuf[S][j] = load_half8_stream(
                reinterpret_cast<const f16*>(kbase + ((offset)r[j] * ssk + 2u * vdim)));
    };
    auto load_v = [&](int T0) {
        uint32_t r[NVL];
        rows(T0, r);
#pragma unroll
        for (int j = 0; j < NVL; ++j)
            vbuf[j] = load_half8_stream(reinterpret_cast<const f16*>(vbase + ((offset)r[j] * ssv + 2u * vdim)));
    };

    float m_run = -1e30f, l_part = 0.f;
    floatx4 o[ND];   // lane (g, col): dims 16db + 4g + e of head col
#pragma unroll
    for (int db = 0; db < ND; ++db) o[db] = floatx4{0.f, 0.f, 0.f, 0.f};
    const float sc = a.scale_log2;
    const f16* vrd = &v_lds[(4 * g + col / 4) * VP + 4 * (col % 4)];

    auto step = [&](auto S_, auto PFK_, auto PFV_, int it) {
        constexpr int S = decltype(S_)::value;
        const int T0 = t_begin + TOK * it;
#pragma unroll
        for (int j = 0; j < NVL; ++j)
            *reinterpret_cast<half8*>(&k_lds[(RPL * j + vrow) * KP + vdim]) = kbuf[S][j];
        if constexpr (decltype(PFK_)::value) load_k(S_, T0 + 2 * W * TOK);
        floatx4 C[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            C[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const half8 ka = *reinterpret_cast<const half8*>(
                    &k_lds[(16 * t + col) * KP + 32 * c + 8 * g]);
                C[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, qb[c], C[t], 0, 0, 0);
            }
        }
        if constexpr (SUMS) {
            // the step's scores of a head, 128 bytes; the heads of a KV head side by side
            float* ss = p.ws_s + score_at(a, p, b, kvh, T0) + 32 * (h0 + col) + 4 * g;
            if (hvalid) {
                *reinterpret_cast<floatx4*>(ss) = C[0];
                *reinterpret_cast<floatx4*>(ss + 16) = C[1];
            }
        }
        const bool tail = T0 + TOK > t_end;
        if (tail) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (T0 + 16 * t + 4 * g + e >= t_end) C[t][e] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(C[0][0], C[0][1]), fmaxf(C[0][2], C[0][3])),
                         fmaxf(fmaxf(C[1][0], C[1][1]), fmaxf(C[1][2], C[1][3])));
        mx = rows4_max(mx);
        const float mn = fmaxf(m_run, mx);
        const float alpha = fast_exp2((m_run - mn) * sc);
        m_run = mn;
        const float nm = hvalid ? -mn * sc : -INFINITY;
        half8 pt;
        float ps = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = fast_exp2(fmaf(C[t][e], sc, nm));
                pt[4 * t + e] = static_cast<f16>(x);
                ps += x;
            }
        l_part = fmaf(l_part, alpha, ps);
        if (tail) {   // the repeated rows: 0 times an infinite V is no zero
#pragma unroll
            for (int j = 0; j < NVL; ++j)
                if (T0 + RPL * j + vrow >= t_end) vbuf[j] = half8{};
        }
#pragma unroll
        for (int j = 0; j < NVL; ++j)
            *reinterpret_cast<half8*>(&v_lds[(RPL * j + vrow) * VP + vdim]) = vbuf[j];
        if constexpr (decltype(PFV_)::value) load_v(T0 + W * TOK);
        if (__builtin_amdgcn_read_exec() & __ballot(alpha != 1.f)) {
#pragma unroll
            for (int db = 0; db < ND; ++db)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[db][e] *= alpha;
        }
#pragma unroll
        for (int db = 0; db < ND; ++db) {
            const half8 va = cat_half8(lds_read_tr16(vrd + 16 * db),
                                       lds_read_tr16(vrd + 16 * VP + 16 * db));
            o[db] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pt, o[db], 0, 0, 0);
        }
    };

    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using Pf = std::true_type;
    using NoPf = std::false_type;
    const int n_w = n_iter > wv ? (n_iter - wv + W - 1) / W : 0;   // this wave's steps
    if (n_w > 0) {
        const int s0 = t_begin + TOK * wv;
        load_k(I0{}, s0);
        load_v(s0);
        load_k(I1{}, s0 + W * TOK);
        int j = 0;
        for (; j + 3 < n_w; j += 2) {
            step(I0{}, Pf{}, Pf{}, wv + W * j);
            step(I1{}, Pf{}, Pf{}, wv + W * (j + 1));
        }
        if (j + 2 < n_w) {
            step(I0{}, Pf{}, Pf{}, wv + W * j);
            step(I1{}, NoPf{}, Pf{}, wv + W * (j + 1));
            step(I0{}, NoPf{}, NoPf{}, wv + W * (j + 2));
        } else if (j + 1 < n_w) {
            step(I0{}, NoPf{}, Pf{}, wv + W * j);
            step(I1{}, NoPf{}, NoPf{}, wv + W * (j + 1));
        } else {
            step(I0{}, NoPf{}, NoPf{}, wv + W * j);
        }
    }

    // One workgroup holds every head of its KV head and all keys: its thread t adds the sums of
    // keys 4t .. 4t + 3, whose slots' loads start here.
    constexpr bool kSums = SUMS && W == 8;
    static_assert(!kSums || kMaxChunk <= 4 * W * kWave, "a quad of keys per thread");
    __shared__ float head[kSums ? kHeads : 1][2];   // -M in log2 units, 1 / sum
    const int j4 = 4 * threadIdx.x;
    Quad quad{};
    if constexpr (kSums)
        if (p.fused) quad = quad_at(a, b, kvh, min(j4, L - 1) & ~3);
    auto sums = [&]() {
        __syncthreads();   // the heads, and every wave's scores
        if (j4 >= L) return;
        const float* sj = p.ws_s + score_at(a, p, b, kvh, j4 & ~31) + (j4 & 31);
        floatx4 w = {0.f, 0.f, 0.f, 0.f};
        for (int h = 0; h < nh; ++h) {
            const floatx4 x = *reinterpret_cast<const floatx4*>(sj + 32 * h);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = fmaf(fast_exp2(fmaf(x[e], sc, head[h][0])), head[h][1], w[e]);
        }
        put_quad(a, quad, b, j4, L, w);
    };

    // Dims 16 (d0 + i) + 4g + e of head col: all of them, or wave d0's share of the waves' sum.
    constexpr int NB = W > 1 ? 1 : ND;
    floatx4 r[NB];
    int d0 = 0;
    if constexpr (W == 1) {
#pragma unroll
        for (int db = 0; db < ND; ++db) r[db] = o[db];
    } else {
        // every wave leaves (O, m, l) in its own K tile, 64 (D + 8) bytes of it
        static_assert(W >= ND, "a wave for every 16 dims");
        float* xs = reinterpret_cast<float*>(k_lds);
#pragma unroll
        for (int db = 0; db < ND; ++db)
            *reinterpret_cast<floatx4*>(&xs[(db * kWave + lane) * 4]) = o[db];
        *reinterpret_cast<float2*>(&xs[ND * kWave * 4 + 2 * lane]) = float2{m_run, l_part};
        __syncthreads();
        if (wv >= ND) {
            if constexpr (kSums)
                if (p.fused) sums();
            return;
        }
        d0 = wv;
        float2 ml[W];
        floatx4 x[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float* xw = reinterpret_cast<const float*>(k_lds_all[w]);
            ml[w] = *reinterpret_cast<const float2*>(&xw[ND * kWave * 4 + 2 * lane]);
            x[w] = *reinterpret_cast<const floatx4*>(&xw[(d0 * kWave + lane) * 4]);
            m_run = fmaxf(m_run, ml[w].x);
        }
        l_part = 0.f;
        r[0] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float al = fast_exp2((ml[w].x - m_run) * sc);
            l_part = fmaf(ml[w].y, al, l_part);
            r[0] += x[w] * al;
        }
    }

    const float l_tot = rows4_sum(l_part);
    if constexpr (kSums) {
        if (p.fused) {
            if (hvalid && g == 0 && d0 == 0) {
                head[col][0] = -m_run * sc;
                head[col][1] = 1.f / l_tot;
            }
            sums();
        }
    }
    if (!hvalid) return;
    const int64_t prow = (row0 + col) * p.nsplit + split;
    if ((SUMS || nsb > 1) && g == 0 && d0 == 0) {
        p.ws_ml[prow * 2] = m_run * sc;
        p.ws_ml[prow * 2 + 1] = l_tot;
    }
    if (nsb == 1) {
        const float inv = 1.f / l_tot;
        f16* orow = a.out + (row0 + col) * D + 16 * d0 + 4 * g;
#pragma unroll
        for (int db = 0; db < NB; ++db) {
            half4 h;
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = static_cast<f16>(r[db][e] * inv);
            *reinterpret_cast<half4*>(orow + 16 * db) = h;
        }
        return;
    }
    float* po = p.ws_o + prow * D + 16 * d0 + 4 * g;
#pragma unroll
    for (int db = 0; db < NB; ++db) *reinterpret_cast<floatx4*>(po + 16 * db) = r[db];
}

// ------------------------------------------------------------------ join --
constexpr int kJoinWaves = 4;

// Joins the partials of one query head of one sequence: lane (r, c) owns dims
// 8c .. of every (4R)-th split, U of them in flight.
template <int D>
__device__ __forceinline__ void join_head(const BoundArgs& a, const DecodePlan& p, int64_t row,
                                          int nsb) {
    constexpr int LPR = D / 8, R = kWave / LPR, STRIDE = kJoinWaves * R, U = 4;
    __shared__ __attribute__((aligned(16))) float red[kJoinWaves - 1][LPR][12];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane % LPR, r = lane / LPR;
    const float* po = p.ws_o + row * p.nsplit * D + 8 * c;
    const float* pml = p.ws_ml + row * p.nsplit * 2;
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
    for (int j0 = wave * R + r; j0 < nsb; j0 += STRIDE * U) {
        float2 ml[U];
        floatx4 y[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = min(j0 + STRIDE * u, nsb - 1);
            ml[u] = *reinterpret_cast<const float2*>(pml + 2 * j);
            y[u][0] = *reinterpret_cast<const floatx4*>(po + (int64_t)j * D);
            y[u][1] = *reinterpret_cast<const floatx4*>(po + (int64_t)j * D + 4);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + STRIDE * u < nsb) fold(ml[u].x, ml[u].y, y[u][0], y[u][1]);
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
    if (wave > 0 && r == 0) {
        float* q = red[wave - 1][c];
        *reinterpret_cast<floatx4*>(q) = x0;
        *reinterpret_cast<floatx4*>(q + 4) = x1;
        q[8] = M;
        q[9] = S;
    }
    __syncthreads();
    if (wave != 0 || r != 0) return;
#pragma unroll
    for (int w = 0; w < kJoinWaves - 1; ++w) {
        const float* q = red[w][c];
        fold(q[8], q[9], *reinterpret_cast<const floatx4*>(q),
             *reinterpret_cast<const floatx4*>(q + 4));
    }
    const float inv = 1.f / S;
    half8 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        h[e] = static_cast<f16>(x0[e] * inv);
        h[4 + e] = static_cast<f16>(x1[e] * inv);
    }
    store_half8(a.out + row * D + 8 * c, h);
}

template <int D>
__global__ void __launch_bounds__(kJoinWaves * kWave)
bound_join_kernel(const BoundArgs a, const DecodePlan p) {
    const int b = blockIdx.y, lane = threadIdx.x & (kWave - 1);
    const int L = vis_len(a, b);
    if (L <= 0) return;
    const int chunk = chunk_of(p, L, p.balance > 0 ? batch_keys(a, p.batch, lane) : 0);
    const int nsb = (L + chunk - 1) / chunk;
    if (nsb > 1) join_head<D>(a, p, (int64_t)b * a.Hq + blockIdx.x, nsb);
}

// The join with the sums.  Grid (key blocks of kSumKeys, then G query heads to
// join; KV head; sequence).
constexpr int kSumKeys = 4 * kJoinWaves * kWave;

template <int D>
__global__ void __launch_bounds__(kJoinWaves * kWave)
bound_sums_kernel(const BoundArgs a, const DecodePlan p, int key_blocks) {
    const int kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int lane = tid & (kWave - 1), wave = tid >> 6;
    const int n = bound_len(a, b);
    if (n <= 0) return;
    const int64_t row0 = (int64_t)b * a.Hq + (int64_t)kvh * a.G;
    const int at = blockIdx.x;
    if (at < key_blocks && at * kSumKeys >= n) return;
    const int chunk = chunk_of(p, n, p.balance > 0 ? batch_keys(a, p.batch, lane) : 0);
    const int nsb = (n + chunk - 1) / chunk;
    if (at >= key_blocks) {
        if (nsb > 1) join_head<D>(a, p, row0 + at - key_blocks, nsb);
        return;
    }
    // Four keys a thread.  Their scores, page id and sums are on their way before the
    // heads' maxima and sums are folded (one memory round trip instead of three: 5.7 to
    // 4.7 us at 2048 keys).
    const int j = at * kSumKeys + 4 * tid;
    const int jc = min(j, n - 1) & ~3;
    const float* sj = p.ws_s + score_at(a, p, b, kvh, jc & ~31) + (jc & 31);
    const Quad quad = quad_at(a, b, kvh, jc);
    floatx4 w = {0.f, 0.f, 0.f, 0.f};
    constexpr int H = 8, HW = H / kJoinWaves;   // heads at a time, and per wave
    __shared__ float head[H][2];                // -M in log2 units, 1 / sum
    for (int g0 = 0; g0 < a.G; g0 += H) {
        const int gn = min(a.G - g0, H);
        floatx4 s[H];
#pragma unroll
        for (int g = 0; g < H; ++g)
            s[g] = *reinterpret_cast<const floatx4*>(sj + 32 * (g0 + min(g, gn - 1)));
        float2 x[HW];
        const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + (row0 + g0) * p.nsplit;
#pragma unroll
        for (int i = 0; i < HW; ++i)
            x[i] = ml[(int64_t)min(wave + i * kJoinWaves, gn - 1) * p.nsplit + min(lane, nsb - 1)];
#pragma unroll
        for (int i = 0; i < HW; ++i) {
            const int g = wave + i * kJoinWaves;
            if (g >= gn) continue;
            float M = lane < nsb ? x[i].x : -3.0e38f, S = lane < nsb ? x[i].y : 0.f;
            for (int t = lane + kWave; t < nsb; t += kWave) {
                const float2 y = ml[(int64_t)g * p.nsplit + t];
                const float mn = fmaxf(M, y.x);
                S = S * fast_exp2(M - mn) + y.y * fast_exp2(y.x - mn);
                M = mn;
            }
            const float mx = wave_max_fast(M);
            S = wave_sum_fast(S * fast_exp2(M - mx));
            if (lane == 0) {
                head[g][0] = -mx;
                head[g][1] = 1.f / S;
            }
        }
        __syncthreads();
#pragma unroll
        for (int g = 0; g < H; ++g) {
            if (g >= gn) break;
            const float nm = head[g][0], inv = head[g][1];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = fmaf(fast_exp2(fmaf(s[g][e], a.scale_log2, nm)), inv, w[e]);
        }
        __syncthreads();
    }
    put_quad(a, quad, b, j, n, w);
}

// ------------------------------------------------------------------ plan --
// Up to so many keys a sequence takes one split: eight waves share its steps, and no second
// launch joins.  `units` is the workgroups of that launch.  us as one split / as splits, at as
// many keys in every sequence, replayed from a graph (called among other work the second launch
// costs up to 0.8 more, so the limits there lie higher):
//   D = 64             1 to 16 units 768 keys 6.5 / 6.6, 896 6.8 / 6.5, 1088 7.7 / 6.7; 24 to 40
//                      896 6.9 / 7.3, 1088 7.8 / 7.6; 48 and more 1088 7.8 / 9.1, of 256 11.8 / 18.4
//   D = 128            to 16 512 7.5 / 7.6, 576 7.8 / 7.6, 900 11.0 / 7.7; 32 576 8.0 / 8.1, 640
//                      8.2 / 8.2; 64 640 9.0 / 8.9, 768 10.0 / 9.4; 96 768 11.2 / 11.7, 900 13.8 /
//                      12.9; 112 900 14.5 / 14.6
//   with sums, which the workgroup then adds itself
//     D = 64           to 16 704 7.3 / 7.3, 896 7.6 / 7.3; 32 896 7.8 / 7.9, 960 8.4 / 8.0; 48 960
//                      8.6 / 8.9
//     D = 128          to 16 384 7.6 / 8.3, 448 8.6 / 8.4; 40 512 9.0 / 9.0; 64 576 9.8 / 9.9, 640
//                      10.6 / 10.0; 96 640 11.3 / 11.9, 900 15.6 / 14.3
// Batches of 16 and more, whose splits go by a list of lengths: 16 units of 64 1088 7.7 / 9.8; of
// 128 768 9.6 / 10.7, 900 11.4 / 10.8; 64 900 13.0 / 13.8, 256 21.8 / 28.3.  Strided views have
// no page ids to wait for: D = 64, 8 units 800 5.7 / 6.3, 1152 6.6 / 6.3, but called among other
// work 7.0 / 7.4, which is worth more; 32 1152 7.0 / 7.2.  Of more than 16 heads a KV head a
// second launch adds the workgroups' sums either way (among other work 128 8.2 / 8.4, 350 9.1 / 8.4).
int one_split_keys(int batch, int64_t units, int d, int groups, bool sums, bool paged) {
    if (sums && groups > 1) return 128;
    if (d == 64) {
        if (!paged || batch >= kBalanced || units >= 48) return sums ? kMaxChunk : kMaxOne;
        return units >= 24 ? 896 : sums ? 768 : 832;
    }
    if (batch >= kBalanced) return units < 64 ? 832 : kMaxChunk;
    const int64_t keys = sums ? std::max<int64_t>(416, 352 + 4 * units)
                              : std::max<int64_t>(units < 24 ? 544 : 608, 256 + 6 * units);
    return static_cast<int>(std::min<int64_t>(kMaxChunk, keys));
}

DecodePlan plan_of(int batch, int hkv, int G, int d, int64_t maxv, bool sums, bool paged) {
    DecodePlan p{};
    p.batch = batch;
    p.groups = (G + kHeads - 1) / kHeads;
    const int64_t units = (int64_t)batch * hkv * p.groups;
    const int64_t per = std::max<int64_t>(64, ((maxv + 63) / 64 + 63) / 64 * 64);
    int64_t s = std::min((maxv + per - 1) / per, units >= 6144 ? 1 : 6144 / units);
    int64_t chunk = std::min<int64_t>(((maxv + s - 1) / s + 63) / 64 * 64, kMaxChunk);
    const int one = one_split_keys(batch, units, d, p.groups, sums, paged);
    if (maxv <= one) chunk = (maxv + 31) / 32 * 32;
    p.chunk = static_cast<int>(chunk);
    p.nsplit = static_cast<int>((maxv + chunk - 1) / chunk);
    return p;
}

int64_t most_visible(int cap, int window, int sinks) {
    return window > 0 ? std::min<int64_t>(cap, (int64_t)window + sinks) : cap;
}

// One wave per split, two per SIMD of 256 CUs.
constexpr int kWaveSlots = 2048;

}  // namespace

size_t bound_decode_workspace(int batch, int hq, int hkv, int d, int cap, int window, int sinks,
                              bool sums) {
    if (!bound_sizes(batch, hq, hkv, cap, window, sinks) || (d != 64 && d != 128)) return 0;
    // paged views: the lower limits of one split, so never less than strided ones need
    const DecodePlan p = plan_of(batch, hkv, hq / hkv, d, most_visible(cap, window, sinks), sums, true);
    const size_t rows = (size_t)batch * hq;
    size_t n = p.nsplit > 1 || sums ? rows * p.nsplit * 2 : 0;
    if (p.nsplit > 1) n += rows * p.nsplit * d;
    if (sums) n += rows * ((cap + 31) / 32 * 32);
    return sizeof(float) * n;
}

bool bound_decode_fits(const BoundArgs& a, int batch) {
    const DecodePlan p = plan_of(batch, a.Hkv, a.G, a.D, most_visible(a.max_len, a.window, a.sinks),
                                 a.weights != nullptr, a.k.bt != nullptr);
    return (a.D == 64 || a.D == 128) && p.nsplit <= 65535 && (int64_t)a.Hkv * p.groups <= INT32_MAX;
}

template <int D, bool PAGED, bool SUMS>
static int launch(const BoundArgs& a, DecodePlan p, int64_t maxv, hipStream_t s) {
    const int heads = a.Hkv * p.groups;
    const int64_t reach = PAGED ? (int64_t)a.k.num_pages * kPage : a.cap;   // rows of a head
    const bool wide = reach * std::max(a.k.stride_s, a.v.stride_s) >= (int64_t)1 << 31;
    dim3 grid(heads, p.nsplit, p.batch);
    // Batches of 16 and more cut each sequence by what the whole batch has (8 of up to 1200
    // keys, 32/8 heads of 128, 11.8 us so and 8.8 in fixed splits, 8000 34 and 29; 24 of up to
    // 8000 keys of 64 42.3 and 45.6).
    if (p.batch >= kBalanced && p.nsplit > 1) {
        p.balance = std::max(1, kWaveSlots / heads - p.batch / 2);
        const int64_t worst = (p.batch * maxv + kMaxChunk - 1) / kMaxChunk;
        const int64_t units = std::max<int64_t>(p.balance, worst) + p.batch;
        if (units <= 65535)
            grid = dim3(heads, static_cast<unsigned>(units), 1);
        else
            p.balance = 0;
    }
    p.fused = SUMS && !wide && p.balance == 0 && p.nsplit == 1 && p.groups == 1;
    // one split: eight waves take its steps round robin; fixed splits at D = 64: four
    // (at D = 128 four are no faster on one sequence and 26-52 % slower on four of 1024
    // to 4000 keys)
    auto go = [&](auto kernel, int waves) {
        hipLaunchKernelGGL(kernel, grid, dim3(waves * kWave), 0, s, a, p);
    };
    if (wide)
        go(bound_decode_kernel<D, PAGED, SUMS, 1, true>, 1);
    else if (p.balance == 0 && p.nsplit == 1)
        go(bound_decode_kernel<D, PAGED, SUMS, 8>, 8);
    else if (D == 64 && p.balance == 0)
        go(bound_decode_kernel<D, PAGED, SUMS, D == 64 ? 4 : 1>, 4);
    else
        go(bound_decode_kernel<D, PAGED, SUMS, 1>, 1);
    if (SUMS && !p.fused) {
        const int kb = (a.cap + kSumKeys - 1) / kSumKeys;
        hipLaunchKernelGGL((bound_sums_kernel<D>), dim3(kb + (p.nsplit > 1 ? a.G : 0), a.Hkv, p.batch),
                           dim3(kJoinWaves * kWave), 0, s, a, p, kb);
    } else if (!SUMS && p.nsplit > 1) {
        hipLaunchKernelGGL((bound_join_kernel<D>), dim3(a.Hq, p.batch), dim3(kJoinWaves * kWave), 0,
                           s, a, p);
    }
    return check_launch(SUMS ? "weighted_decode" : "window_decode");
}

// The workspace holds bound_decode_workspace bytes; views of one kind with one
// block table, 16-byte aligned.
int bound_decode(const BoundArgs& a, int batch, bool paged, bool sums, void* ws, hipStream_t s) {
    const int64_t maxv = most_visible(a.max_len, a.window, a.sinks);
    DecodePlan p = plan_of(batch, a.Hkv, a.G, a.D, maxv, sums, paged);
    const size_t rows = (size_t)batch * a.Hq;
    p.scap = (a.max_len + 31) / 32 * 32;
    float* w = static_cast<float*>(ws);
    if (sums) {
        p.ws_s = w;
        w += rows * p.scap;
    }
    p.ws_o = w;
    p.ws_ml = w + (p.nsplit > 1 ? rows * p.nsplit * a.D : 0);
    if (a.D == 64)
        return sums ? launch<64, true, true>(a, p, maxv, s)
                    : paged ? launch<64, true, false>(a, p, maxv, s)
                            : launch<64, false, false>(a, p, maxv, s);
    return sums ? launch<128, true, true>(a, p, maxv, s)
                : paged ? launch<128, true, false>(a, p, maxv, s)
                        : launch<128, false, false>(a, p, maxv, s);
}

}  // namespace kvhp
