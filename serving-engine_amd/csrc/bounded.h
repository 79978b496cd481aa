// bounded.h -- shared by the attention kernels of caches of bounded length (bounded.hip,
// bounded_decode.hip, window_prefill.hip, prompt_weights.hip): views, visibility,
// argument checks.
#pragma once

#include "kvhp_internal.h"

#include <algorithm>
#include <cmath>

namespace kvhp {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// A K or V view as the kernels take it.
struct BoundView {
    const f16* data;
    int64_t stride_b, stride_h, stride_s, stride_d;
    const int32_t* bt;
    int32_t max_pages;
    int32_t num_pages;
};

inline BoundView bound_view(const kvhp_kv_view& v) {
    return BoundView{static_cast<const f16*>(v.data), v.stride_b, v.stride_h, v.stride_s,
                     v.stride_d, v.block_table, v.max_pages, v.num_pages};
}

// What the attention and the sums of a bounded cache read and write.  Rows: q,
// out [batch][rows][Hq][D], row r of sequence b at position first(b) + r.
struct BoundArgs {
    const f16* q;
    BoundView k, v;
    const int32_t* q_start;   // NULL: 0
    const int32_t* seq_lens;  // NULL: cap
    f16* out;
    float* lse;               // [batch][Hq][rows] or NULL
    float* weights;           // [Hkv][num_pages][16]
    int32_t* ages;            // [Hkv][num_pages][16] or NULL
    const int32_t* newest;    // NULL: the length - 1
    int rows, Hq, Hkv, G, D;
    int cap;                  // keys addressable per sequence ...
    int max_len;              // ... and the call's limit, which plans and workspaces go by
    int window, sinks;        // window 0: none
    int new_keys;
    int last_row;             // 1: decode, the one row is the last key's
    float scale_log2;         // log2(e) / sqrt(D)
};

__device__ __forceinline__ int bound_len(const BoundArgs& a, int b) {
    return a.seq_lens ? min(max(a.seq_lens[b], 0), a.cap) : a.cap;
}
// Position of row 0 (64 bits: a start far below zero only makes padding rows).
__device__ __forceinline__ int64_t bound_first(const BoundArgs& a, int b, int n) {
    return a.last_row ? (int64_t)n - 1 : (a.q_start ? a.q_start[b] : 0);
}
// First key of position p's window.
__device__ __forceinline__ int bound_low(int p, int window) {
    return window > 0 ? max(p - window + 1, 0) : 0;
}
// Row of position j in a head's pool or view (page ids clamped into the pool).
template <bool PAGED>
__device__ __forceinline__ int64_t bound_row(const BoundView& v, int b, int j) {
    if constexpr (PAGED) {
        const int pid = v.bt[(int64_t)b * v.max_pages + (j >> 4)];
        return (int64_t)min(max(pid, 0), v.num_pages - 1) * kPage + (j & 15);
    }
    return j;
}
// Slot of position j in a pool of sums, or -1 where the page id is outside it.
__device__ __forceinline__ int64_t bound_slot(const BoundView& k, int b, int kvh, int j) {
    const int pid = k.bt[(int64_t)b * k.max_pages + (j >> 4)];
    if (pid < 0 || pid >= k.num_pages) return -1;
    return ((int64_t)kvh * k.num_pages + pid) * kPage + (j & 15);
}
// Adds w to key j's slot, or starts it there for the last new_keys of n keys.
__device__ __forceinline__ void bound_add(const BoundArgs& a, int b, int kvh, int j, int n,
                                          float w) {
    const int64_t at = bound_slot(a.k, b, kvh, j);
    if (at < 0) return;
    const bool fresh = (int64_t)j + a.new_keys >= n;
    a.weights[at] = fresh ? w : a.weights[at] + w;
    if (fresh && a.ages) a.ages[at] = (a.newest ? a.newest[b] : n - 1) - (n - 1 - j);
}

// ---------------------------------------------------------------- host ----
int bound_check_view(const kvhp_kv_view* v, const char* what, const char* name);
constexpr int kMaxBatch = 65535, kMaxKvHeads = 65535;   // grid dimensions
constexpr int kMaxHeads = 1 << 25, kMaxLen = 1 << 30;
// What bound_shapes takes: the size queries, which a caller asks first, plan for nothing else.
inline bool bound_sizes(int batch, int hq, int hkv, int max_len, int window, int sinks) {
    return batch > 0 && batch <= kMaxBatch && hkv > 0 && hkv <= kMaxKvHeads && hq > 0 &&
           hq <= kMaxHeads && hq % hkv == 0 && max_len > 0 && max_len <= kMaxLen && window >= 0 &&
           sinks >= 0;
}
// Shapes every call checks; fills the fields of `a` that they give.
int bound_shapes(BoundArgs& a, const char* what, int batch, int hq, int hkv, int d,
                 int max_seq_len, int window, int sinks);
// Views for the fast kernels: rows of contiguous dims, 16-byte aligned, 32-bit
// byte offsets inside a page.
inline bool bound_fast_view(const kvhp_kv_view& v) {
    return v.stride_d == 1 && v.stride_s % 8 == 0 && v.stride_s > 0 && v.stride_s < (1 << 26) &&
           aligned16(v.data) && v.stride_h % 8 == 0 && (v.block_table || v.stride_b % 8 == 0);
}
inline bool bound_one_table(const kvhp_kv_view& k, const kvhp_kv_view& v) {
    return k.block_table == v.block_table &&
           (!k.block_table || (k.max_pages == v.max_pages && k.num_pages == v.num_pages));
}

// bounded_decode.hip: one token per sequence at D = 64 and 128, with the sums
// (paged views) or with a window.
size_t bound_decode_workspace(int batch, int hq, int hkv, int d, int cap, int window, int sinks,
                              bool sums);
bool bound_decode_fits(const BoundArgs& a, int batch);
int bound_decode(const BoundArgs& a, int batch, bool paged, bool sums, void* ws, hipStream_t s);
// window_prefill.hip: rows at D = 64 and 128.
size_t window_prefill_workspace(int batch, int rows, int hq, int hkv, int d, int max_len,
                                int window, int sinks);
bool window_prefill_fits(const BoundArgs& a, int batch);
int window_prefill(const BoundArgs& a, int batch, bool paged, void* ws, hipStream_t s);
// prompt_weights.hip: the sums of rows at D = 64 and 128 (paged K).
size_t prompt_weights_workspace(int batch, int rows, int hq, int hkv, int d, int max_len);
bool prompt_weights_fits(const BoundArgs& a, int batch);
int prompt_weights(const BoundArgs& a, int batch, void* ws, hipStream_t s);

}  // namespace kvhp
