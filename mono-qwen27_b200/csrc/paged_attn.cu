// paged_attn.cu — attention of new tokens over a paged cache
// (include/m27b_paged.h).
//
// Row (token t, query head h) of sequence b at position p, kv head j = h / (n_q
// / n_kv):  s_i = scale * q . k_i,  lo <= i <= p,  lo = window > 0 ? max(0, p -
// window + 1) : 0;  out = sum_i exp(s_i - m) v_i / sum_i exp(s_i - m), lse = m +
// log of that sum, with the running maximum m of one pass over the positions.
//
// One warp per row, the head's values over the lanes.
#include "paged_common.cuh"

namespace m27b {

struct AttnArgs {
    M27BPagedKV kv;
    M27BPagedBatch bt;
    const void *q;
    void *out;
    float *lse;
    long long q_stride, out_stride;
    int n_q, window;
    float scale;
    int *status;
};

template <bool BF, int V>
__global__ void __launch_bounds__(256) k_paged_attn_rows(const AttnArgs a) {
    constexpr int HD = 32 * V;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const long long t64 = w / a.n_q;
    if (t64 >= a.bt.n_tok) return;
    const int t = (int)t64, h = (int)(w - t64 * a.n_q), j = h / (a.n_q / a.kv.n_kv);
    int b = 0;
    while (b < a.bt.n_seq && __ldg(a.bt.cu_q + b + 1) <= t) ++b;
    if (b >= a.bt.n_seq || t < __ldg(a.bt.cu_q + b)) return;
    const int row = seq_row(a.bt, b, a.kv.n_rows);
    const int len = row < 0 ? 0 : __ldg(a.bt.lens + row), cap = a.kv.n_cols * a.kv.page_size;
    if (len > cap && lane == 0) paged_bad(a.status);
    const int p = row < 0 ? -1 : min(len, cap) - __ldg(a.bt.cu_q + b + 1) + t;
    const int lo = a.window > 0 ? max(0, p - a.window + 1) : 0;
    float q[V], o[V], m = -INFINITY, l = 0.0f;
    const uint16_t *qp = (const uint16_t *)a.q + t * a.q_stride + h * HD + lane * V;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
        const float2 f = Half16<BF>::up(((const uint32_t *)qp)[i]);
        q[2 * i] = f.x, q[2 * i + 1] = f.y;
        o[2 * i] = o[2 * i + 1] = 0.0f;
    }
    if (row < 0 && lane == 0) paged_bad(a.status);
    for (int i = lo; i <= p; ++i) {
        const int c = i / a.kv.page_size;
        const int page = c < a.kv.n_cols ? __ldg(a.kv.table + (long long)row * a.kv.n_cols + c) : -1;
        if (page < 0 || page >= a.kv.n_pages) {
            if (lane == 0) paged_bad(a.status);
            continue;
        }
        const long long at = page * a.kv.page_stride + ((long long)(i - c * a.kv.page_size) * a.kv.n_kv + j) * HD + lane * V;
        const uint32_t *kp = (const uint32_t *)((const uint16_t *)a.kv.k + at);
        const uint32_t *vp = (const uint32_t *)((const uint16_t *)a.kv.v + at);
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            const float2 f = Half16<BF>::up(__ldg(kp + e));
            s = fmaf(q[2 * e], f.x, s);
            s = fmaf(q[2 * e + 1], f.y, s);
        }
        s = warp_sum(s) * a.scale;
        const float mn = fmaxf(m, s), c0 = expf(m - mn), w0 = expf(s - mn);
        l = l * c0 + w0;
        m = mn;
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            const float2 f = Half16<BF>::up(__ldg(vp + e));
            o[2 * e] = o[2 * e] * c0 + w0 * f.x;
            o[2 * e + 1] = o[2 * e + 1] * c0 + w0 * f.y;
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    uint32_t *op = (uint32_t *)((uint16_t *)a.out + t * a.out_stride + h * HD + lane * V);
#pragma unroll
    for (int e = 0; e < V / 2; ++e) op[e] = Half16<BF>::down(o[2 * e] * inv, o[2 * e + 1] * inv);
    if (a.lse && lane == 0) a.lse[(long long)t * a.n_q + h] = l > 0.0f ? m + logf(l) : -INFINITY;
}

template <bool BF>
cudaError_t attn_rows_launch(const AttnArgs &a, cudaStream_t st) {
    const dim3 grid((unsigned)(((long long)a.bt.n_tok * a.n_q + 7) / 8)), block(256);
    switch (a.kv.head_dim) {
    case 64: return launch_pdl(k_paged_attn_rows<BF, 2>, grid, block, 0, st, a);
    case 128: return launch_pdl(k_paged_attn_rows<BF, 4>, grid, block, 0, st, a);
    default: return launch_pdl(k_paged_attn_rows<BF, 8>, grid, block, 0, st, a);
    }
}

}  // namespace m27b

using namespace m27b;

extern "C" {

size_t m27b_paged_attn_scratch_bytes(int n_q, int n_kv, int head_dim) {
    if (n_kv < 1 || n_kv > 1024 || n_q < n_kv || n_q % n_kv || n_q / n_kv > 128) return 0;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    return 4096;
}

bool m27b_paged_attn(const M27BPagedKV *kv, const M27BPagedBatch *batch, const void *q, long long q_stride, int n_q,
                     float scale, int window, void *out, long long out_stride, float *lse, void *scratch,
                     cudaStream_t stream, char *err, size_t err_cap) {
    const char *what = "m27b_paged_attn";
    if (!paged_check_kv(kv, what, err, err_cap) || !paged_check_batch(batch, kv, what, err, err_cap)) return false;
    if (!batch->n_seq || !batch->n_tok) return paged_ok(cudaSuccess, what, err, err_cap);
    if (!q || !out || !scratch) return paged_fail(err, err_cap, "%s: null q, out or scratch", what);
    if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)scratch) & 15u)
        return paged_fail(err, err_cap, "%s: q, out and scratch must be 16-byte aligned", what);
    if (n_q < kv->n_kv || n_q % kv->n_kv || n_q / kv->n_kv > 128)
        return paged_fail(err, err_cap, "%s: n_q (%d) must be a multiple of n_kv (%d), at most 128 per kv head", what, n_q,
                          kv->n_kv);
    if (q_stride < (long long)n_q * kv->head_dim || out_stride < (long long)n_q * kv->head_dim || q_stride % 8 || out_stride % 8)
        return paged_fail(err, err_cap, "%s: token strides must be multiples of 8, at least n_q x head_dim", what);
    if (!(scale > 0.0f) || scale > 1e30f) return paged_fail(err, err_cap, "%s: scale must be positive and finite", what);
    if ((long long)batch->n_tok * n_q > 0x7fffffffll * 8) return paged_fail(err, err_cap, "%s: too many rows", what);
    const AttnArgs a = {*kv, *batch, q, out, lse, q_stride, out_stride, n_q, window > 0 ? window : 0, scale,
                        status_ptr_current()};
    return paged_ok(kv->type == M27B_TYPE_BF16 ? attn_rows_launch<true>(a, stream) : attn_rows_launch<false>(a, stream), what,
                    err, err_cap);
}

}  // extern "C"
