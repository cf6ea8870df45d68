// paged_common.cuh — what the kernels of the paged key/value cache share:
// 16-bit types, the batch's sequences, and the C entries' error helpers.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdarg>
#include <cstdio>

#include "m27b_device.cuh"
#include "m27b_launch.cuh"
#include "m27b_paged.h"

namespace m27b {

constexpr int PAGED_BAD = 6;  // status word: a table row, page id or position out of range

// The 16-bit type of a cache.
template <bool BF> struct Half16;
template <> struct Half16<true> {
    using T = __nv_bfloat16;
    using T2 = __nv_bfloat162;
    static M27B_DI float2 up(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const T2 *>(&v)); }
    static M27B_DI uint32_t down(float a, float b) {
        const T2 t = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&t);
    }
};
template <> struct Half16<false> {
    using T = __half;
    using T2 = __half2;
    static M27B_DI float2 up(uint32_t v) { return __half22float2(*reinterpret_cast<const T2 *>(&v)); }
    static M27B_DI uint32_t down(float a, float b) {
        const T2 t = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&t);
    }
};

M27B_DI void paged_bad(int *status) {
    if (status) atomicCAS(status, 0, PAGED_BAD);
}

// Offsets, lengths, rows, tables and tokens may come from the launch before, whose
// end pdl_wait() awaits while this kernel already runs: they are read by ordinary
// loads, not by the read-only path (__ldg), which wants data that no one writes
// during the kernel.

// Rows [lo, hi) of sequence b in the token buffers, held to [0, n_tok).
M27B_DI int2 seq_tokens(const M27BPagedBatch &bt, int b) {
    const int lo = max(0, bt.cu_q[b]), hi = min(bt.n_tok, bt.cu_q[b + 1]);
    return make_int2(lo, max(lo, hi));
}

// Table row of sequence b, -1 if it is out of range.
M27B_DI int seq_row(const M27BPagedBatch &bt, int b, int n_rows) {
    const int r = bt.rows ? bt.rows[b] : b;
    return r >= 0 && r < n_rows ? r : -1;
}

inline bool paged_fail(char *err, size_t cap, const char *fmt, ...) {
    if (err && cap) {
        va_list ap;
        va_start(ap, fmt);
        std::vsnprintf(err, cap, fmt, ap);
        va_end(ap);
    }
    return false;
}
inline bool paged_ok(cudaError_t e, const char *what, char *err, size_t cap) {
    if (e != cudaSuccess) return paged_fail(err, cap, "%s: %s", what, cudaGetErrorString(e));
    if (err && cap) err[0] = '\0';
    return true;
}

// Checks of the cache and the batch that every entry makes (paged_rope.cu).
bool paged_check_kv(const M27BPagedKV *kv, const char *what, char *err, size_t cap);
bool paged_check_batch(const M27BPagedBatch *b, const M27BPagedKV *kv, const char *what, char *err, size_t cap);

}  // namespace m27b
