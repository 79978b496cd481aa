// q4.hip -- attention over a paged cache held in 4 bits, and its rows read back: entry
// points, and the kernel that reads back.
#include "q4.h"

#include <algorithm>

namespace kvhp {
namespace {

// Rows read back: a thread takes 8 dims of K and V of two positions, the loads of both in
// flight together (8192 positions of 8 heads of 128: 9.2 us, 4.6 TB/s; one position 11.4).
// Grid (positions; KV head; sequence).  DT: head_dim, 0 for any.
template <int DT>
__global__ void __launch_bounds__(256)
q4_gather_kernel(const uint8_t* pool, const int32_t* bt, int max_pages, int num_pages,
                 const int32_t* start, const int32_t* seq_lens, f16* out_k, f16* out_v, int Hkv,
                 int any_d, int max_len) {
    const int D = DT ? DT : any_d;
    const uint32_t cpr = D / 8;
    const int h = blockIdx.y, b = blockIdx.z;
    const int n = static_cast<int>(min((int64_t)max(seq_lens[b], 0), (int64_t)max_pages * kPage));
    const int64_t first = start ? start[b] : 0;
    constexpr int U = 2;
    uint32_t x[U][2], sr[U][2];
    int t[U], c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint64_t i = (uint64_t)blockIdx.x * (256 * U) + 256 * u + threadIdx.x;
        t[u] = static_cast<int>(min(i / cpr, (uint64_t)INT32_MAX));
        c[u] = static_cast<int>(i % cpr);
        const int64_t pos = first + t[u];
        x[u][0] = x[u][1] = sr[u][0] = sr[u][1] = 0;   // zeros stand for zeros
        if (t[u] >= max_len || pos < 0 || pos >= n) continue;
        const uint8_t* pg = q4_page(pool, num_pages, D, h, bt[(int64_t)b * max_pages + (pos >> 4)]);
        const int o = static_cast<int>(pos & 15);
#pragma unroll
        for (int is_v = 0; is_v < 2; ++is_v) {
            sr[u][is_v] = *reinterpret_cast<const uint32_t*>(pg + q4_params_at(D, is_v, o));
            x[u][is_v] = *reinterpret_cast<const uint32_t*>(pg + q4_codes_at(D, is_v, o) + 4 * c[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (t[u] >= max_len) continue;
        const int64_t at = (((int64_t)b * Hkv + h) * max_len + t[u]) * D + 8 * c[u];
#pragma unroll
        for (int is_v = 0; is_v < 2; ++is_v) {
            f16* out = is_v ? out_v : out_k;
            if (!out) continue;
            const Q4Row p = q4_row(sr[u][is_v]);
            half8 y;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[e] = static_cast<f16>(p.s * (static_cast<float>(x[u][is_v] >> 4 * e & 15) + p.r));
            store_half8(out + at, q4_finite(y));
        }
    }
}

// Shapes, pool and tables that every attention call checks; fills what they give.
int q4_shapes(Q4Args& a, const char* what, const void* pool, const int32_t* bt, int max_pages,
              int num_pages, int batch, int hq, int hkv, int d, int max_seq_len) {
    KVHP_REQUIRE(pool && bt, KVHP_ERR_INVALID, "%s: null pool or block tables", what);
    KVHP_REQUIRE(aligned16(pool), KVHP_ERR_INVALID, "%s: pool not 16-byte aligned", what);
    KVHP_REQUIRE(max_pages > 0 && num_pages > 0, KVHP_ERR_INVALID,
                 "%s: max_pages=%d and num_pages=%d must be positive", what, max_pages, num_pages);
    KVHP_REQUIRE(hq > 0 && hkv > 0 && hq % hkv == 0, KVHP_ERR_INVALID,
                 "%s: num_q_heads=%d must be a positive multiple of num_kv_heads=%d", what, hq,
                 hkv);
    KVHP_REQUIRE(d > 0 && d <= 256 && d % 8 == 0, KVHP_ERR_UNSUPPORTED,
                 "%s: head_dim=%d is no multiple of 8 up to 256", what, d);
    KVHP_REQUIRE(batch <= kMaxBatch && hkv <= kMaxKvHeads, KVHP_ERR_UNSUPPORTED,
                 "%s: more than 65535 sequences or KV heads", what);
    KVHP_REQUIRE(hq <= kMaxHeads, KVHP_ERR_UNSUPPORTED, "%s: num_q_heads=%d above 2^25", what, hq);
    KVHP_REQUIRE(max_seq_len <= kMaxLen, KVHP_ERR_UNSUPPORTED, "%s: max_seq_len=%d above 2^30",
                 what, max_seq_len);
    a.pool = static_cast<const uint8_t*>(pool);
    a.bt = bt;
    a.max_pages = max_pages;
    a.num_pages = num_pages;
    a.Hq = hq;
    a.Hkv = hkv;
    a.G = hq / hkv;
    a.D = d;
    a.max_len = max_seq_len;
    a.cap = static_cast<int>(std::min<int64_t>(max_seq_len, (int64_t)max_pages * kPage));
    a.scale_log2 = kLog2e / std::sqrt(static_cast<float>(d));
    return KVHP_OK;
}

// Rows that the kernel for any head_dim, which works on 16 (row, query head) pairs a wave, takes before
// the one that works on 128 a workgroup: up to 64 pairs of a KV head, contexts of four tiles of 64 keys
// and more, up to 1024 of a wave's tiles in all.  (32/8 heads of 128: 4 rows of 1024 keys 12.6 us
// against 17.4, of 4096 15.8 and 18.0, of 8 times 1024 17.8 and 18.5; past it, 8 rows of 8192 keys 25.0
// and 22.0; below, 4 of 128 11.6 and 9.4.  32/4 heads of 64: 2, 4 and 8 rows of 4096 keys 10.9, 11.5 and
// 13.3 against 15.0 to 15.6; 8 of 8192 17.2 and 16.4.)
bool few_pairs(int batch, int rows, int hq, int hkv, int max_len) {
    if (batch <= 0 || rows <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || max_len <= 0) return false;
    const int64_t pairs = (int64_t)rows * (hq / hkv), tiles = ((int64_t)max_len + 63) / 64;
    return pairs <= 64 && tiles >= 4 && tiles <= 1024 && (pairs + 15) / 16 * hkv * batch * tiles <= 1024;
}

int workspace_check(const char* what, const void* ws, size_t bytes, size_t need) {
    if (need == 0) return KVHP_OK;
    KVHP_REQUIRE(ws && bytes >= need, KVHP_ERR_WORKSPACE,
                 "%s: workspace of %zu bytes, %zu needed", what, ws ? bytes : 0, need);
    KVHP_REQUIRE(aligned16(ws), KVHP_ERR_INVALID, "%s: workspace not 16-byte aligned", what);
    return KVHP_OK;
}

}  // namespace
}  // namespace kvhp

using namespace kvhp;

extern "C" size_t kvhp_q4_page_bytes(int head_dim) {
    return head_dim > 0 && head_dim <= 256 && head_dim % 8 == 0 ? q4_page_bytes(head_dim) : 0;
}

extern "C" int kvhp_q4_gather(const void* pool, const int32_t* block_tables, int max_pages,
                              int num_pages, const int32_t* start, const int32_t* seq_lens,
                              void* out_k, void* out_v, int batch, int num_kv_heads, int head_dim,
                              int max_len, void* stream) {
    clear_error();
    if (batch <= 0 || max_len <= 0) return KVHP_OK;
    const char* what = "q4_gather";
    KVHP_REQUIRE(seq_lens && (out_k || out_v), KVHP_ERR_INVALID, "%s: null pointer", what);
    Q4Args a{};
    int rc = q4_shapes(a, what, pool, block_tables, max_pages, num_pages, batch, num_kv_heads,
                       num_kv_heads, head_dim, max_len);
    if (rc) return rc;
    KVHP_REQUIRE(aligned16(out_k) && aligned16(out_v), KVHP_ERR_INVALID,
                 "%s: outputs not 16-byte aligned", what);
    const dim3 grid(static_cast<unsigned>(((int64_t)max_len * (head_dim / 8) + 511) / 512),
                    num_kv_heads, batch);
    auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, static_cast<hipStream_t>(stream), a.pool,
                           block_tables, max_pages, num_pages, start, seq_lens,
                           static_cast<f16*>(out_k), static_cast<f16*>(out_v), num_kv_heads,
                           head_dim, max_len);
    };
    if (head_dim == 64)
        go(q4_gather_kernel<64>);
    else if (head_dim == 128)
        go(q4_gather_kernel<128>);
    else
        go(q4_gather_kernel<0>);
    return check_launch(what);
}

extern "C" size_t kvhp_q4_decode_workspace_bytes(int batch, int num_q_heads, int num_kv_heads,
                                                 int head_dim, int max_seq_len) {
    // at 64 and 128 the same rows off their alignment make do with it
    return head_dim == 64 || head_dim == 128
               ? q4_decode_workspace(batch, num_q_heads, num_kv_heads, head_dim, max_seq_len)
               : q4_any_workspace(batch, 1, num_q_heads, num_kv_heads, head_dim, max_seq_len);
}

extern "C" int kvhp_q4_decode(const void* q, const void* pool, const int32_t* block_tables,
                              int max_pages, int num_pages, const int32_t* seq_lens, void* out,
                              int batch, int num_q_heads, int num_kv_heads, int head_dim,
                              int max_seq_len, void* workspace, size_t workspace_bytes,
                              void* stream) {
    clear_error();
    if (batch <= 0 || max_seq_len <= 0) return KVHP_OK;
    const char* what = "q4_decode";
    KVHP_REQUIRE(q && out && seq_lens, KVHP_ERR_INVALID, "%s: null pointer", what);
    Q4Args a{};
    int rc = q4_shapes(a, what, pool, block_tables, max_pages, num_pages, batch, num_q_heads,
                       num_kv_heads, head_dim, max_seq_len);
    if (rc) return rc;
    a.q = static_cast<const f16*>(q);
    a.out = static_cast<f16*>(out);
    a.seq_lens = seq_lens;
    a.rows = 1;
    a.last_row = 1;
    const size_t need =
        kvhp_q4_decode_workspace_bytes(batch, num_q_heads, num_kv_heads, head_dim, max_seq_len);
    rc = workspace_check(what, workspace, workspace_bytes, need);
    if (rc) return rc;
    if (q4_decode_fits(a, batch))
        return q4_decode(a, batch, workspace, static_cast<hipStream_t>(stream));
    return q4_any(a, batch, what, workspace, need, static_cast<hipStream_t>(stream));
}

extern "C" size_t kvhp_q4_prefill_workspace_bytes(int batch, int rows, int num_q_heads,
                                                  int num_kv_heads, int head_dim,
                                                  int max_seq_len) {
    return (head_dim == 64 || head_dim == 128) && !few_pairs(batch, rows, num_q_heads, num_kv_heads, max_seq_len)
               ? q4_prefill_workspace(batch, rows, num_q_heads, num_kv_heads, head_dim, max_seq_len)
               : q4_any_workspace(batch, rows, num_q_heads, num_kv_heads, head_dim, max_seq_len);
}

extern "C" int kvhp_q4_prefill(const void* q, const void* pool, const int32_t* block_tables,
                               int max_pages, int num_pages, const int32_t* q_start,
                               const int32_t* seq_lens, void* out, float* lse, int batch, int rows,
                               int num_q_heads, int num_kv_heads, int head_dim, int max_seq_len,
                               void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    if (batch <= 0 || rows <= 0 || max_seq_len <= 0) return KVHP_OK;
    const char* what = "q4_prefill";
    KVHP_REQUIRE(q && out, KVHP_ERR_INVALID, "%s: null pointer", what);
    Q4Args a{};
    int rc = q4_shapes(a, what, pool, block_tables, max_pages, num_pages, batch, num_q_heads,
                       num_kv_heads, head_dim, max_seq_len);
    if (rc) return rc;
    a.q = static_cast<const f16*>(q);
    a.out = static_cast<f16*>(out);
    a.lse = lse;
    a.q_start = q_start;
    a.seq_lens = seq_lens;
    a.rows = rows;
    const size_t need = kvhp_q4_prefill_workspace_bytes(batch, rows, num_q_heads, num_kv_heads,
                                                        head_dim, max_seq_len);
    rc = workspace_check(what, workspace, workspace_bytes, need);
    if (rc) return rc;
    if (q4_prefill_fits(a, batch) && !few_pairs(batch, rows, num_q_heads, num_kv_heads, max_seq_len))
        return q4_prefill(a, batch, workspace, static_cast<hipStream_t>(stream));
    return q4_any(a, batch, what, workspace, need, static_cast<hipStream_t>(stream));
}
