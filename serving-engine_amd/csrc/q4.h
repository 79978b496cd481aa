// q4.h -- the paged KV cache held in 4 bits: page layout, quantiser, arguments, shared by
// its append, gather and attention kernels (rope_append.hip, q4.hip, q4_decode.hip,
// q4_prefill.hip, q4_any.hip).
//
// A row x of D values (one token's K or V of one KV head) is held as D codes n of 0..15 and
// two fp16 numbers s and r, and stands for s (n + r):
//   s = max((max x - min x) / 15, max |x| / 1984), rounded up to fp16,
//   r = min x / s to the nearest multiple of 2^(floor(log2(|min x / s| + 16)) - 10),
//   n = x / s - r to the nearest, in 0..15,
// in fp32, the first two quotients as products with 1 / 15 and 1 / 1984 in fp32 (1 / 15 is
// rounded up, so that a quotient that fp16 holds may go up by one of its steps).
// That multiple, and |r| <= 1984, make n + r and r - 16 exact in fp16 for every n (rows about
// 0 have multiples of 2^-6: the range is off by s/128 at most; the second bound on s costs
// 2^-12 of a row's largest, as much as fp16 itself).  So n + r is an operand of the matrix
// cores as it is, and a row's scale meets the fp32 scores or the weights: neither K nor V is
// rounded a second time.  (Scale and minimum, the usual pair, need either a rounded operand
// or a term of their own per key and head.)  A row of equal values c: s = c, r = 1, n = 0.  A
// row with a value that is not finite: s = r = NaN, n = 0, all NaN as its product would be.
// s and r are rounded, so that a row with values past 65400 or so may stand for up to 65700 (s is
// up by 2^-10 of its 15 steps, at most 128, and s r by s 2^-7): what is written in fp16, values
// read back and weighted means, then is +-65504 (q4_finite), never infinite.
//
// A page of a KV head is 16 (D + 8) bytes in a row, whole 128-byte lines at any D that is a
// multiple of 8: K codes [16][D/2] (the even dim in the low half of a byte), V codes, K's
// (s, r) [16], V's.  4.25 bits a value at D = 128, 4.5 at 64.
#pragma once

#include "bounded.h"

namespace kvhp {

__host__ __device__ constexpr int q4_page_bytes(int d) { return kPage * (d + 8); }
// Byte offsets inside a page.
__host__ __device__ constexpr int q4_codes_at(int d, int is_v, int row) {
    return (is_v * kPage + row) * (d / 2);
}
__host__ __device__ constexpr int q4_params_at(int d, int is_v, int row) {
    return kPage * d + 4 * (is_v * kPage + row);
}

// A row's two numbers as they lie in a page: s in the low half.
struct Q4Row {
    float s, r;
};
__device__ __forceinline__ Q4Row q4_row(uint32_t p) {
    const half2v h = __builtin_bit_cast(half2v, p);
    return Q4Row{static_cast<float>(h[0]), static_cast<float>(h[1])};
}
// s and r of a row with values from lo to hi, all finite, and what turns values into codes.
struct Q4Quant {
    uint32_t bits;   // (s, r) as stored
    float s, sr, inv;
    bool flat;
};
__device__ __forceinline__ Q4Quant q4_quant(float lo, float hi) {
    Q4Quant z;
    lo += 0.f;   // no -0, whichever of the two zeros a minimum took
    z.flat = lo == hi;
    z.s = lo;
    float r = 1.f;
    if (!z.flat) {
        const float t = fmaxf((hi - lo) * (1.f / 15.f), fmaxf(fabsf(lo), fabsf(hi)) * (1.f / 1984.f));
        f16 s16 = static_cast<f16>(t);
        if (static_cast<float>(s16) < t)   // positive: the next one up
            s16 = __builtin_bit_cast(f16, static_cast<uint16_t>(__builtin_bit_cast(uint16_t, s16) + 1));
        z.s = static_cast<float>(s16);
        const float r0 = lo / z.s;
        // 2^(floor(log2(|r0| + 16)) - 10), by the exponent's bits
        const float step = __uint_as_float(
            (__float_as_uint(fabsf(r0) + 16.f) & 0x7f800000u) - (10u << 23));
        r = rintf(r0 / step) * step;
    }
    z.sr = z.s * r;   // exact: 11 bits each
    z.inv = z.flat ? 0.f : 1.f / z.s;   // s is at least 2^-24
    z.bits = __builtin_bit_cast(uint32_t, half2v{static_cast<f16>(z.s), static_cast<f16>(r)});
    return z;
}
// The code of x: (x - s r) / s to the nearest, even where it lies between two.  The quotient
// is rounded as a division would be (one Newton step from the rounded reciprocal).
__device__ __forceinline__ uint32_t q4_code(const Q4Quant& z, float x) {
    const float d = x - z.sr;
    const float q0 = d * z.inv;
    const float q = fmaf(fmaf(-q0, z.s, d), z.inv, q0);
    return static_cast<uint32_t>(fminf(fmaxf(rintf(q), 0.f), 15.f));
}
constexpr uint32_t kQ4NanRow = 0x7e007e00u;
// Values rounded to fp16, where infinite its largest (NaN stays: the minimum and maximum that keep
// it, packed, an instruction a value).
template <typename T>
__device__ __forceinline__ T q4_finite(T h) {
    const T most = static_cast<f16>(65504.f);
    return __builtin_elementwise_maximum(__builtin_elementwise_minimum(h, most), -most);
}

// What the attention over a 4-bit cache reads and writes.  Rows: q, out [batch][rows][Hq][D],
// row r of sequence b at position first(b) + r.
struct Q4Args {
    const f16* q;
    const uint8_t* pool;      // [Hkv][num_pages][16 (D + 8)]
    const int32_t* bt;        // [batch][max_pages]
    int max_pages, num_pages;
    const int32_t* q_start;   // NULL: 0
    const int32_t* seq_lens;  // NULL: cap
    f16* out;
    float* lse;               // [batch][Hq][rows] or NULL
    int rows, Hq, Hkv, G, D;
    int cap;                  // keys addressable per sequence ...
    int max_len;              // ... and the call's limit, which plans and workspaces go by
    int last_row;             // 1: decode, the one row is the last key's
    float scale_log2;         // log2(e) / sqrt(D)
};

__device__ __forceinline__ int q4_len(const Q4Args& a, int b) {
    return a.seq_lens ? min(max(a.seq_lens[b], 0), a.cap) : a.cap;
}
__device__ __forceinline__ int64_t q4_first(const Q4Args& a, int b, int n) {
    return a.last_row ? (int64_t)n - 1 : (a.q_start ? a.q_start[b] : 0);
}
// A head's page of the pool (ids clamped into it).
__device__ __forceinline__ const uint8_t* q4_page(const uint8_t* pool, int num_pages, int d,
                                                  int kvh, int pid) {
    return pool + ((int64_t)kvh * num_pages + min(max(pid, 0), num_pages - 1)) * q4_page_bytes(d);
}

// Sums over lanes 0 .. this one, by row shifts and row broadcasts.
__device__ __forceinline__ uint32_t prefix_sum(uint32_t x) {
    x += __builtin_amdgcn_update_dpp(0u, x, 0x111, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x142, 0xa, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x143, 0xc, 0xf, false);
    return x;
}
// The largest of all lanes' x, which are not negative.
__device__ __forceinline__ int wave_max(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(x, kWave - 1);
}

// q4_decode.hip: one token per sequence at D = 64 and 128.
size_t q4_decode_workspace(int batch, int hq, int hkv, int d, int max_len);
bool q4_decode_fits(const Q4Args& a, int batch);
int q4_decode(const Q4Args& a, int batch, void* ws, hipStream_t s);
// q4_prefill.hip: rows at D = 64 and 128.
size_t q4_prefill_workspace(int batch, int rows, int hq, int hkv, int d, int max_len);
bool q4_prefill_fits(const Q4Args& a, int batch);
int q4_prefill(const Q4Args& a, int batch, void* ws, hipStream_t s);
// q4_any.hip: either at any shape.
size_t q4_any_workspace(int batch, int rows, int hq, int hkv, int d, int max_len);
int q4_any(const Q4Args& a, int batch, const char* what, void* ws, size_t room, hipStream_t s);

}  // namespace kvhp
