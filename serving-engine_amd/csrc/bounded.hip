// bounded.hip -- attention over a cache of bounded length (sliding window and
// first tokens) and the sums of attention weight that an eviction goes by:
// entry points, and the kernels that take any shape.
//
// Any head_dim <= 256, any strides, any group: one wave per (query head, row),
// one pass over its visible keys with an online softmax, fp32 throughout; and
// one wave per (key, KV head) for the weights that rows gave a key.  These are for
// rare shapes and no more: one key per trip behind a six-step sum over the wave, K
// and V read again for every query head, no split over the keys.  At D = 96, 32/8
// heads, windows of 4096 in 32 sequences take 5.9 ms where memory would need 65 us,
// a 2048-row prompt with window 512 2.9 ms, its sums 7.7 ms (D = 256 13, 4.5 and 14
// ms): 2 to 8 times the elementary torch operations.  What bounds them is latency,
// a wave's loads one after the other.
#include "bounded.h"

namespace kvhp {

int bound_check_view(const kvhp_kv_view* v, const char* what, const char* name) {
    KVHP_REQUIRE(v && v->data, KVHP_ERR_INVALID, "%s: %s view is null", what, name);
    if (v->block_table)
        KVHP_REQUIRE(v->max_pages > 0 && v->num_pages > 0 && v->page_size == kPage,
                     KVHP_ERR_INVALID,
                     "%s: %s paged view needs max_pages, num_pages > 0 and page_size %d", what,
                     name, kPage);
    return KVHP_OK;
}

int bound_shapes(BoundArgs& a, const char* what, int batch, int hq, int hkv, int d,
                 int max_seq_len, int window, int sinks) {
    KVHP_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, KVHP_ERR_INVALID,
                 "%s: num_q_heads=%d must be a positive multiple of num_kv_heads=%d", what, hq,
                 hkv);
    KVHP_REQUIRE(d > 0 && d <= 256, KVHP_ERR_UNSUPPORTED, "%s: head_dim=%d outside 1..256", what,
                 d);
    KVHP_REQUIRE(window >= 0 && sinks >= 0, KVHP_ERR_INVALID,
                 "%s: window=%d and sinks=%d must not be negative", what, window, sinks);
    KVHP_REQUIRE(batch <= kMaxBatch && hkv <= kMaxKvHeads, KVHP_ERR_UNSUPPORTED,
                 "%s: more than 65535 sequences or KV heads", what);
    KVHP_REQUIRE(hq <= kMaxHeads, KVHP_ERR_UNSUPPORTED, "%s: num_q_heads=%d above 2^25", what, hq);
    KVHP_REQUIRE(max_seq_len <= kMaxLen, KVHP_ERR_UNSUPPORTED, "%s: max_seq_len=%d above 2^30",
                 what, max_seq_len);
    a.Hq = hq;
    a.Hkv = hkv;
    a.G = hq / hkv;
    a.D = d;
    a.cap = a.max_len = max_seq_len;
    a.window = window;
    a.sinks = window > 0 ? sinks : 0;   // without a window every key is visible anyway
    a.scale_log2 = kLog2e / std::sqrt(static_cast<float>(d));
    return KVHP_OK;
}

namespace {

__device__ __forceinline__ float dot_row(const float (&qv)[4], const f16* row, int64_t stride,
                                         int lane, int D) {
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + kWave * i;
        if (d < D) dot = fmaf(qv[i], static_cast<float>(row[d * stride]), dot);
    }
    return wave_sum(dot);
}

// One wave per (row, query head) of a sequence.
template <bool PAGED>
__global__ void __launch_bounds__(kWave) bound_rows_kernel(const BoundArgs a) {
    const int lane = threadIdx.x;
    const int row = blockIdx.x / a.Hq, qh = blockIdx.x % a.Hq, b = blockIdx.y;
    const int kvh = qh / a.G, D = a.D;
    const int64_t at = ((int64_t)b * a.rows + row) * a.Hq + qh;
    const int n = bound_len(a, b);
    const int64_t p64 = bound_first(a, b, n) + row;
    if (p64 < 0 || p64 >= n) {
        if (a.last_row)   // no keys
            for (int d = lane; d < D; d += kWave) a.out[at * D + d] = f16(0);
        return;
    }
    const int p = static_cast<int>(p64);
    float qv[4], acc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + kWave * i;
        qv[i] = d < D ? static_cast<float>(a.q[at * D + d]) : 0.f;
        acc[i] = 0.f;
    }
    const int64_t hk = kvh * a.k.stride_h + (PAGED ? 0 : b * a.k.stride_b);
    const int64_t hv = kvh * a.v.stride_h + (PAGED ? 0 : b * a.v.stride_b);
    const int low = bound_low(p, a.window);
    float m = -1e30f, l = 0.f;
    for (int j = a.sinks > 0 ? 0 : low; j <= p; ++j) {
        if (j >= a.sinks && j < low) j = low;
        const f16* kr = a.k.data + hk + bound_row<PAGED>(a.k, b, j) * a.k.stride_s;
        const f16* vr = a.v.data + hv + bound_row<PAGED>(a.v, b, j) * a.v.stride_s;
        const float s = dot_row(qv, kr, a.k.stride_d, lane, D) * a.scale_log2;
        const float mn = fmaxf(m, s);
        const float al = fast_exp2(m - mn), w = fast_exp2(s - mn);
        l = l * al + w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + kWave * i;
            const float vv = d < D ? static_cast<float>(vr[d * a.v.stride_d]) : 0.f;
            acc[i] = fmaf(w, vv, acc[i] * al);
        }
        m = mn;
    }
    const float inv = 1.f / l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + kWave * i;
        if (d < D) a.out[at * D + d] = static_cast<f16>(acc[i] * inv);
    }
    if (a.lse && lane == 0)
        a.lse[((int64_t)b * a.Hq + qh) * a.rows + row] = (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// One wave per (key, KV head) of a sequence: the weights that its rows gave it.
__global__ void __launch_bounds__(kWave) bound_weights_kernel(const BoundArgs a) {
    const int lane = threadIdx.x;
    const int j = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, D = a.D;
    const int n = bound_len(a, b);
    if (j >= n) return;
    const int64_t first = bound_first(a, b, n);
    // rows at positions j .. last that see key j
    int64_t last = min(first + a.rows, (int64_t)n) - 1;
    if (a.window > 0 && j >= a.sinks) last = min(last, (int64_t)j + a.window - 1);
    // a key that none sees is not touched (its page may be another's by now), a new one
    // starts at zero
    if (max(max(first, (int64_t)0), (int64_t)j) > last) {
        if (lane == 0 && (int64_t)j + a.new_keys >= n) bound_add(a, b, kvh, j, n, 0.f);
        return;
    }
    const f16* kr = a.k.data + kvh * a.k.stride_h + bound_row<true>(a.k, b, j) * a.k.stride_s;
    float kv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + kWave * i;
        kv[i] = d < D ? static_cast<float>(kr[d * a.k.stride_d]) : 0.f;
    }
    float w = 0.f;
    for (int64_t p = max(first, (int64_t)j); p <= last; ++p) {
        const int64_t r = p - first;
        for (int g = 0; g < a.G; ++g) {
            const int qh = kvh * a.G + g;
            const f16* qr = a.q + (((int64_t)b * a.rows + r) * a.Hq + qh) * D;
            const float s = dot_row(kv, qr, 1, lane, D) * a.scale_log2;
            w += fast_exp2(s - a.lse[((int64_t)b * a.Hq + qh) * a.rows + r] * kLog2e);
        }
    }
    if (lane == 0) bound_add(a, b, kvh, j, n, w);
}

int launch_rows(const BoundArgs& a, int batch, bool paged, const char* what, hipStream_t s) {
    KVHP_REQUIRE((int64_t)a.rows * a.Hq <= 1 << 25, KVHP_ERR_UNSUPPORTED,   // 2^31 threads
                 "%s: %d rows of %d heads", what, a.rows, a.Hq);
    const dim3 grid(static_cast<unsigned>(a.rows) * a.Hq, batch);
    if (paged)
        hipLaunchKernelGGL(bound_rows_kernel<true>, grid, dim3(kWave), 0, s, a);
    else
        hipLaunchKernelGGL(bound_rows_kernel<false>, grid, dim3(kWave), 0, s, a);
    return check_launch(what);
}

int launch_weights(const BoundArgs& a, int batch, const char* what, hipStream_t s) {
    KVHP_REQUIRE(a.cap <= 1 << 25, KVHP_ERR_UNSUPPORTED, "%s: %d keys", what, a.cap);
    hipLaunchKernelGGL(bound_weights_kernel, dim3(a.cap, a.Hkv, batch), dim3(kWave), 0, s, a);
    return check_launch(what);
}

int k_view_of(BoundArgs& a, const kvhp_kv_view* kv, const char* what) {
    const int rc = bound_check_view(kv, what, "K");
    if (rc) return rc;
    a.k = bound_view(*kv);
    if (kv->block_table) a.cap = static_cast<int>(std::min<int64_t>(a.cap, (int64_t)kv->max_pages * kPage));
    return KVHP_OK;
}

int views(BoundArgs& a, const kvhp_kv_view* kv, const kvhp_kv_view* vv, const char* what) {
    int rc = k_view_of(a, kv, what);
    if (rc || (rc = bound_check_view(vv, what, "V"))) return rc;
    KVHP_REQUIRE((kv->block_table == nullptr) == (vv->block_table == nullptr), KVHP_ERR_INVALID,
                 "%s: K and V views must both be paged or both strided", what);
    a.v = bound_view(*vv);
    if (vv->block_table) a.cap = static_cast<int>(std::min<int64_t>(a.cap, (int64_t)vv->max_pages * kPage));
    return KVHP_OK;
}

int workspace_check(const char* what, const void* ws, size_t bytes, size_t need) {
    if (need == 0) return KVHP_OK;
    KVHP_REQUIRE(ws && bytes >= need, KVHP_ERR_WORKSPACE,
                 "%s: workspace of %zu bytes, %zu needed", what, ws ? bytes : 0, need);
    KVHP_REQUIRE(aligned16(ws), KVHP_ERR_INVALID, "%s: workspace not 16-byte aligned", what);
    return KVHP_OK;
}

int sums_check(const BoundArgs& a, const kvhp_kv_view* kv, const char* what) {
    KVHP_REQUIRE(kv->block_table, KVHP_ERR_UNSUPPORTED, "%s: paged views required", what);
    KVHP_REQUIRE(a.weights && a.new_keys >= 0, KVHP_ERR_INVALID,
                 "%s: null weights or negative new_keys", what);
    KVHP_REQUIRE(aligned16(a.weights) && aligned16(a.ages), KVHP_ERR_INVALID,
                 "%s: weights and ages must be 16-byte aligned", what);
    return KVHP_OK;
}

}  // namespace
}  // namespace kvhp

using namespace kvhp;

extern "C" size_t kvhp_window_decode_workspace_bytes(int batch, int num_q_heads, int num_kv_heads,
                                                     int head_dim, int max_seq_len, int window,
                                                     int sinks) {
    return bound_decode_workspace(batch, num_q_heads, num_kv_heads, head_dim, max_seq_len, window,
                                  sinks, false);
}

extern "C" int kvhp_window_decode(const void* q, const kvhp_kv_view* k_view,
                                  const kvhp_kv_view* v_view, const int32_t* seq_lens, void* out,
                                  int batch, int num_q_heads, int num_kv_heads, int head_dim,
                                  int max_seq_len, int window, int sinks, void* workspace,
                                  size_t workspace_bytes, void* stream) {
    clear_error();
    if (batch <= 0 || max_seq_len <= 0) return KVHP_OK;
    const char* what = "window_decode";
    KVHP_REQUIRE(q && out && seq_lens, KVHP_ERR_INVALID, "%s: null pointer", what);
    BoundArgs a{};
    int rc = bound_shapes(a, what, batch, num_q_heads, num_kv_heads, head_dim, max_seq_len,
                          window, sinks);
    if (rc || (rc = views(a, k_view, v_view, what))) return rc;
    a.q = static_cast<const f16*>(q);
    a.out = static_cast<f16*>(out);
    a.seq_lens = seq_lens;
    a.rows = 1;
    a.last_row = 1;
    rc = workspace_check(what, workspace, workspace_bytes,
                         kvhp_window_decode_workspace_bytes(batch, num_q_heads, num_kv_heads,
                                                            head_dim, max_seq_len, window, sinks));
    if (rc) return rc;
    const bool paged = k_view->block_table != nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (aligned16(q) && aligned16(out) && bound_fast_view(*k_view) && bound_fast_view(*v_view) &&
        bound_one_table(*k_view, *v_view) && bound_decode_fits(a, batch))
        return bound_decode(a, batch, paged, false, workspace, s);
    return launch_rows(a, batch, paged, what, s);
}

extern "C" size_t kvhp_weighted_decode_workspace_bytes(int batch, int num_q_heads,
                                                       int num_kv_heads, int head_dim,
                                                       int max_seq_len) {
    if (batch <= 0 || num_q_heads <= 0 || max_seq_len <= 0) return 0;
    // other shapes leave each head's log-sum-exp
    return std::max(sizeof(float) * (size_t)batch * num_q_heads,
                    bound_decode_workspace(batch, num_q_heads, num_kv_heads, head_dim,
                                           max_seq_len, 0, 0, true));
}

extern "C" int kvhp_weighted_decode(const void* q, const kvhp_kv_view* k_view,
                                    const kvhp_kv_view* v_view, const int32_t* seq_lens,
                                    const int32_t* newest, void* out, float* weights,
                                    int32_t* ages, int batch, int num_q_heads, int num_kv_heads,
                                    int head_dim, int max_seq_len, int new_keys, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    clear_error();
    if (batch <= 0 || max_seq_len <= 0) return KVHP_OK;
    const char* what = "weighted_decode";
    KVHP_REQUIRE(q && out && seq_lens, KVHP_ERR_INVALID, "%s: null pointer", what);
    BoundArgs a{};
    int rc = bound_shapes(a, what, batch, num_q_heads, num_kv_heads, head_dim, max_seq_len, 0, 0);
    if (rc || (rc = views(a, k_view, v_view, what))) return rc;
    a.q = static_cast<const f16*>(q);
    a.out = static_cast<f16*>(out);
    a.seq_lens = seq_lens;
    a.newest = newest;
    a.weights = weights;
    a.ages = ages;
    a.new_keys = new_keys;
    a.rows = 1;
    a.last_row = 1;
    if ((rc = sums_check(a, k_view, what))) return rc;
    rc = workspace_check(what, workspace, workspace_bytes,
                         kvhp_weighted_decode_workspace_bytes(batch, num_q_heads, num_kv_heads,
                                                              head_dim, max_seq_len));
    if (rc) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (aligned16(q) && aligned16(out) && bound_fast_view(*k_view) && bound_fast_view(*v_view) &&
        bound_one_table(*k_view, *v_view) && bound_decode_fits(a, batch))
        return bound_decode(a, batch, true, true, workspace, s);
    a.lse = static_cast<float*>(workspace);
    rc = launch_rows(a, batch, true, what, s);
    return rc ? rc : launch_weights(a, batch, what, s);
}

extern "C" size_t kvhp_window_prefill_workspace_bytes(int batch, int rows, int num_q_heads,
                                                      int num_kv_heads, int head_dim,
                                                      int max_seq_len, int window, int sinks) {
    return window_prefill_workspace(batch, rows, num_q_heads, num_kv_heads, head_dim, max_seq_len,
                                    window, sinks);
}

extern "C" int kvhp_window_prefill(const void* q, const kvhp_kv_view* k_view,
                                   const kvhp_kv_view* v_view, const int32_t* q_start,
                                   const int32_t* seq_lens, void* out, float* lse, int batch,
                                   int rows, int num_q_heads, int num_kv_heads, int head_dim,
                                   int max_seq_len, int window, int sinks, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    clear_error();
    if (batch <= 0 || rows <= 0 || max_seq_len <= 0) return KVHP_OK;
    const char* what = "window_prefill";
    KVHP_REQUIRE(q && out, KVHP_ERR_INVALID, "%s: null pointer", what);
    BoundArgs a{};
    int rc = bound_shapes(a, what, batch, num_q_heads, num_kv_heads, head_dim, max_seq_len,
                          window, sinks);
    if (rc || (rc = views(a, k_view, v_view, what))) return rc;
    a.q = static_cast<const f16*>(q);
    a.out = static_cast<f16*>(out);
    a.lse = lse;
    a.q_start = q_start;
    a.seq_lens = seq_lens;
    a.rows = rows;
    rc = workspace_check(what, workspace, workspace_bytes,
                         kvhp_window_prefill_workspace_bytes(batch, rows, num_q_heads,
                                                             num_kv_heads, head_dim, max_seq_len,
                                                             window, sinks));
    if (rc) return rc;
    const bool paged = k_view->block_table != nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (aligned16(q) && aligned16(out) && bound_fast_view(*k_view) && bound_fast_view(*v_view) &&
        bound_one_table(*k_view, *v_view) && window_prefill_fits(a, batch))
        return window_prefill(a, batch, paged, workspace, s);
    return launch_rows(a, batch, paged, what, s);
}

extern "C" size_t kvhp_prompt_weights_workspace_bytes(int batch, int rows, int num_q_heads,
                                                      int num_kv_heads, int head_dim,
                                                      int max_seq_len) {
    return prompt_weights_workspace(batch, rows, num_q_heads, num_kv_heads, head_dim, max_seq_len);
}

extern "C" int kvhp_prompt_weights(const void* q, const kvhp_kv_view* k_view, const float* lse,
                                   const int32_t* q_start, const int32_t* seq_lens,
                                   const int32_t* newest, float* weights, int32_t* ages,
                                   int batch, int rows, int num_q_heads, int num_kv_heads,
                                   int head_dim, int max_seq_len, int window, int sinks,
                                   int new_keys, void* workspace, size_t workspace_bytes,
                                   void* stream) {
    clear_error();
    if (batch <= 0 || rows <= 0 || max_seq_len <= 0) return KVHP_OK;
    const char* what = "prompt_weights";
    KVHP_REQUIRE(q && lse, KVHP_ERR_INVALID, "%s: null pointer", what);
    BoundArgs a{};
    int rc = bound_shapes(a, what, batch, num_q_heads, num_kv_heads, head_dim, max_seq_len,
                          window, sinks);
    if (rc || (rc = k_view_of(a, k_view, what))) return rc;
    a.q = static_cast<const f16*>(q);
    a.lse = const_cast<float*>(lse);
    a.q_start = q_start;
    a.seq_lens = seq_lens;
    a.newest = newest;
    a.weights = weights;
    a.ages = ages;
    a.new_keys = new_keys;
    a.rows = rows;
    if ((rc = sums_check(a, k_view, what))) return rc;
    rc = workspace_check(what, workspace, workspace_bytes,
                         kvhp_prompt_weights_workspace_bytes(batch, rows, num_q_heads,
                                                             num_kv_heads, head_dim, max_seq_len));
    if (rc) return rc;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (aligned16(q) && bound_fast_view(*k_view) && prompt_weights_fits(a, batch))
        return prompt_weights(a, batch, workspace, s);
    return launch_weights(a, batch, what, s);
}
