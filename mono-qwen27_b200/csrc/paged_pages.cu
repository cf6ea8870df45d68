// paged_pages.cu — upkeep of a paged cache's pages (include/m27b_paged.h):
// resize, fork, free, compact, copy.
//
// Which pages are free is what the counts say (ref <= 0), and a page is always
// taken lowest id first, in request order, so the outcome depends on the
// arguments alone: not on the order in which CTAs run or rows were freed.
//
// resize, fork and compact are two launches: k_*_plan, one CTA, reads counts
// and lengths, checks every request and decides all pages; k_*_apply, a CTA
// or more per SM, writes tables and counts and moves the data.  A refused call
// leaves hdr.go = 0, and the second launch returns at once.
#include "paged_common.cuh"

namespace m27b {

constexpr int PLAN_THREADS = 1024;
constexpr int COPY_THREADS = 256;
constexpr int COPY_UNROLL = 8;
constexpr unsigned COPY_CHUNK = COPY_THREADS * COPY_UNROLL * 16;  // bytes a CTA moves at once: 32 KB

// Scratch: the header, then four int arrays.
struct PagesHdr {
    int go;       // fork, resize: the request stands
    int n_moves;  // compact
};
struct PagesScratch {
    PagesHdr *hdr;
    int *fresh;  // [n_pages] pages taken, in order; compact: the move list's targets
    int *from;   // [max(n_pages, n)] sources of the moves (compact: by rank; fork, resize: by request)
    int *at;     // [max(n_pages, n)] first index into fresh of request i; compact: new id of page p
    int *claim;  // [n_rows] the request that names a row, -1 for none (only rows that are named)
};
inline size_t pages_scratch(int n_pages, int n_rows, int n, void *base, PagesScratch *s) {
    const size_t m = (size_t)(n_pages > n ? n_pages : n);
    size_t off = (sizeof(PagesHdr) + 15) & ~(size_t)15;
    if (s) {
        s->hdr = (PagesHdr *)base;
        s->fresh = (int *)((char *)base + off);
        s->from = s->fresh + n_pages;
        s->at = s->from + m;
        s->claim = s->at + m;
    }
    return off + ((size_t)n_pages + 2 * m + (size_t)n_rows) * sizeof(int);
}

struct Pools {
    M27BPagePool p[M27B_MAX_POOLS];
    int n;
};

struct PagesArgs {
    M27BPages pg;
    Pools pools;
    PagesScratch s;
    const int *a, *b;  // rows and new lengths, or sources and targets
    int n;
    int *out;  // status, or n_live
    int *bad;  // the library's status word
};

M27B_DI int held_pages(int len, int ps) { return len / ps + (len % ps != 0); }

// Sums of non-negative counts stop at a value no pool reaches.
M27B_DI int sat_add(int a, int b) { return min(a + b, 0x3fffffff); }

// Sum of v (at most 0x3fffffff) over the threads before this one, and over the CTA; `red`: 32 ints.
M27B_DI int block_exclusive(int v, int *red, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc = sat_add(inc, u);
    }
    __syncthreads();  // red may still be read from the call before
    if (lane == 31) red[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        int x = red[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x = sat_add(x, u);
        }
        red[lane] = x;
    }
    __syncthreads();
    *total = red[31];
    return sat_add(warp ? red[warp - 1] : 0, inc - v);
}

// The lowest `want` free pages into fresh[]; false if there are fewer.  Four
// pages a thread between two scans of the CTA.
M27B_DI bool take_free(const int *ref, int n_pages, int want, int *fresh, int *red) {
    int got = 0;
    for (int p0 = 0; p0 < n_pages && got < want; p0 += 4 * PLAN_THREADS) {
        const int p = p0 + 4 * threadIdx.x;
        bool free[4];
        int n = 0, total;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            free[i] = p + i < n_pages && ref[p + i] <= 0;
            n += free[i];
        }
        int k = got + block_exclusive(n, red, &total);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (free[i] && k < want) fresh[k++] = p + i;
        got += total;
    }
    return got >= want;
}

// Does any thread say so?  (Also a barrier.)
M27B_DI bool any_bad(bool bad) { return __syncthreads_or(bad) != 0; }

M27B_DI void end_plan(const PagesArgs &a, int why) {
    if (threadIdx.x == 0) {
        a.s.hdr->go = !why;
        if (why && a.out) *a.out = why;
    }
}

__global__ void __launch_bounds__(PLAN_THREADS) k_fork_plan(const PagesArgs a) {
    __shared__ int red[32];
    pdl_wait();
    pdl_trigger();
    const M27BPages &pg = a.pg;
    const int ps = pg.page_size;
    bool bad = false;
    for (int i = threadIdx.x; i < a.n; i += PLAN_THREADS) {
        const int s = a.a[i], d = a.b[i];
        if (s < 0 || s >= pg.n_rows || d < 0 || d >= pg.n_rows || pg.lens[d] != 0) bad = true;
        else a.s.claim[s] = a.s.claim[d] = -1;
    }
    if (any_bad(bad)) return end_plan(a, M27B_PAGES_BAD);
    for (int i = threadIdx.x; i < a.n; i += PLAN_THREADS)
        if (atomicCAS(a.s.claim + a.b[i], -1, i) != -1) bad = true;  // a target named twice
    if (any_bad(bad)) return end_plan(a, M27B_PAGES_BAD);
    int want = 0;
    for (int i0 = 0; i0 < a.n; i0 += PLAN_THREADS) {
        const int i = i0 + threadIdx.x;
        int part = 0;
        if (i < a.n) {
            const int s = a.a[i], len = pg.lens[s], h = len >= 0 ? held_pages(len, ps) : 0;
            if (len < 0 || h > pg.n_cols || a.s.claim[s] != -1) bad = true;  // a broken length, or a target as source
            else if (len % ps) {
                part = 1;
                const int p = pg.table[(size_t)s * pg.n_cols + h - 1];
                if (p < 0 || p >= pg.n_pages) bad = true;
                a.s.from[i] = p;
            }
        }
        int total;
        const int k = block_exclusive(part, red, &total);
        if (i < a.n) a.s.at[i] = part ? want + k : -1;
        want = sat_add(want, total);
    }
    if (any_bad(bad)) return end_plan(a, M27B_PAGES_BAD);
    end_plan(a, take_free(pg.ref, pg.n_pages, want, a.s.fresh, red) ? 0 : M27B_PAGES_FULL);
}

__global__ void __launch_bounds__(PLAN_THREADS) k_resize_plan(const PagesArgs a) {
    __shared__ int red[32];
    pdl_wait();
    pdl_trigger();
    const M27BPages &pg = a.pg;
    const int ps = pg.page_size;
    bool bad = false;
    for (int i = threadIdx.x; i < a.n; i += PLAN_THREADS) {
        const int r = a.a[i];
        if (r < 0 || r >= pg.n_rows) bad = true;
        else a.s.claim[r] = -1;
    }
    if (any_bad(bad)) return end_plan(a, M27B_PAGES_BAD);
    for (int i = threadIdx.x; i < a.n; i += PLAN_THREADS)
        if (atomicCAS(a.s.claim + a.a[i], -1, i) != -1) bad = true;  // a row named twice
    if (any_bad(bad)) return end_plan(a, M27B_PAGES_BAD);
    int want = 0;
    for (int i0 = 0; i0 < a.n; i0 += PLAN_THREADS) {
        const int i = i0 + threadIdx.x;
        int need = 0;
        if (i < a.n) {
            const int r = a.a[i], old = pg.lens[r], len = a.b[i], h = old >= 0 ? held_pages(old, ps) : 0;
            int src = -1;
            if (old < 0 || h > pg.n_cols || len < 0 || held_pages(len, ps) > pg.n_cols) bad = true;
            else {
                need = max(0, held_pages(len, ps) - h);
                if (len > old && old % ps) {
                    const int p = pg.table[(size_t)r * pg.n_cols + h - 1];
                    if (p < 0 || p >= pg.n_pages) bad = true;
                    else if (pg.ref[p] > 1) src = p, ++need;  // others hold it too: a copy of its own
                }
            }
            a.s.from[i] = src;
        }
        int total;
        const int k = block_exclusive(need, red, &total);
        if (i < a.n) a.s.at[i] = sat_add(want, k);
        want = sat_add(want, total);
    }
    if (any_bad(bad)) return end_plan(a, M27B_PAGES_BAD);
    end_plan(a, want <= pg.n_pages && take_free(pg.ref, pg.n_pages, want, a.s.fresh, red) ? 0 : M27B_PAGES_FULL);
}

__global__ void __launch_bounds__(PLAN_THREADS) k_compact_plan(const PagesArgs a) {
    __shared__ int red[32];
    pdl_wait();
    pdl_trigger();
    const M27BPages &pg = a.pg;
    int live = 0;
    for (int p = threadIdx.x; p < pg.n_pages; p += PLAN_THREADS) live += pg.ref[p] > 0;
    int total, holes = 0, movers = 0;
    block_exclusive(live, red, &total);
    live = total;
    for (int p0 = 0; p0 < pg.n_pages; p0 += PLAN_THREADS) {
        const int p = p0 + threadIdx.x;
        const bool used = p < pg.n_pages && pg.ref[p] > 0;
        const bool hole = p < live && !used, mover = p >= live && used;
        int nh, nm;
        const int kh = holes + block_exclusive(hole, red, &nh), km = movers + block_exclusive(mover, red, &nm);
        if (hole) a.s.fresh[kh] = p;
        if (mover) a.s.from[km] = p;
        else if (p < pg.n_pages) a.s.at[p] = -1;  // stays
        holes += nh;
        movers += nm;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += PLAN_THREADS) a.s.at[a.s.from[k]] = a.s.fresh[k];
    if (threadIdx.x == 0) {
        a.s.hdr->n_moves = movers;
        if (a.out) *a.out = live;
    }
}

// `bytes` bytes (a multiple of 16) by one CTA, COPY_UNROLL loads in flight per thread.
M27B_DI void copy_chunk(char *dst, const char *src, unsigned bytes) {
    uint4 v[COPY_UNROLL];
#pragma unroll
    for (int u = 0; u < COPY_UNROLL; ++u) {
        const unsigned o = (u * COPY_THREADS + threadIdx.x) * 16u;
        if (o < bytes) v[u] = __ldcs((const uint4 *)(src + o));
    }
#pragma unroll
    for (int u = 0; u < COPY_UNROLL; ++u) {
        const unsigned o = (u * COPY_THREADS + threadIdx.x) * 16u;
        if (o < bytes) __stcs((uint4 *)(dst + o), v[u]);
    }
}

// The moves pair(i) -> (source, target), i < n, over every plane of the pools,
// dealt to the CTAs in chunks.
template <class Pair>
M27B_DI void move_pages(const Pools &pools, int n, Pair pair) {
    for (int q = 0; q < pools.n; ++q) {
        const M27BPagePool &p = pools.p[q];
        const long long chunks = (long long)((p.page_bytes + COPY_CHUNK - 1) / COPY_CHUNK);
        const long long units = chunks * p.n_planes * n;
        for (long long u = blockIdx.x; u < units; u += gridDim.x) {
            const long long i = u / (chunks * p.n_planes), rest = u - i * chunks * p.n_planes;
            const long long plane = rest / chunks, c = rest - plane * chunks;
            const int2 m = pair((int)i);
            if (m.x < 0) continue;
            const size_t off = (size_t)c * COPY_CHUNK;
            const size_t left = p.page_bytes - off;
            char *base = (char *)p.base + plane * p.plane_stride + off;
            copy_chunk(base + (size_t)m.y * p.page_stride, base + (size_t)m.x * p.page_stride,
                       (unsigned)(left < COPY_CHUNK ? left : COPY_CHUNK));
        }
    }
}

__global__ void __launch_bounds__(COPY_THREADS) k_fork_apply(const PagesArgs a) {
    pdl_wait();
    pdl_trigger();
    if (!a.s.hdr->go) return;
    const M27BPages &pg = a.pg;
    for (int i = blockIdx.x; i < a.n; i += gridDim.x) {
        const int len = pg.lens[a.a[i]], h = held_pages(len, pg.page_size), k = a.s.at[i];
        const int *src = pg.table + (size_t)a.a[i] * pg.n_cols;
        int *dst = pg.table + (size_t)a.b[i] * pg.n_cols;
        for (int c = threadIdx.x; c < h; c += COPY_THREADS) {
            const int p = k >= 0 && c == h - 1 ? a.s.fresh[k] : src[c];
            dst[c] = p;
            if (p >= 0 && p < pg.n_pages) {
                if (k >= 0 && c == h - 1) pg.ref[p] = 1;
                else atomicAdd(pg.ref + p, 1);
            } else paged_bad(a.bad);
        }
        if (threadIdx.x == 0) pg.lens[a.b[i]] = len;
    }
    move_pages(a.pools, a.n, [&](int i) {
        const int k = a.s.at[i];
        return k >= 0 ? make_int2(a.s.from[i], a.s.fresh[k]) : make_int2(-1, -1);
    });
}

__global__ void __launch_bounds__(COPY_THREADS) k_resize_apply(const PagesArgs a) {
    pdl_wait();
    pdl_trigger();
    if (!a.s.hdr->go) return;
    const M27BPages &pg = a.pg;
    const int ps = pg.page_size;
    for (int i = blockIdx.x; i < a.n; i += gridDim.x) {
        const int r = a.a[i], old = pg.lens[r], len = a.b[i], ho = held_pages(old, ps), hn = held_pages(len, ps);
        int *row = pg.table + (size_t)r * pg.n_cols;
        int k = a.s.at[i];
        if (a.s.from[i] >= 0) {
            if (threadIdx.x == 0) {
                atomicSub(pg.ref + a.s.from[i], 1);
                row[ho - 1] = a.s.fresh[k];
                pg.ref[a.s.fresh[k]] = 1;
            }
            ++k;
        }
        for (int c = ho + threadIdx.x; c < hn; c += COPY_THREADS) {
            const int p = a.s.fresh[k + c - ho];
            row[c] = p;
            pg.ref[p] = 1;
        }
        for (int c = hn + threadIdx.x; c < ho; c += COPY_THREADS) {
            const int p = row[c];
            row[c] = -1;
            if (p >= 0 && p < pg.n_pages) atomicSub(pg.ref + p, 1);
            else paged_bad(a.bad);
        }
        __syncthreads();
        if (threadIdx.x == 0) pg.lens[r] = len;
    }
    move_pages(a.pools, a.n, [&](int i) {
        return a.s.from[i] >= 0 ? make_int2(a.s.from[i], a.s.fresh[a.s.at[i]]) : make_int2(-1, -1);
    });
}

__global__ void __launch_bounds__(COPY_THREADS) k_compact_apply(const PagesArgs a) {
    pdl_wait();
    pdl_trigger();
    const M27BPages &pg = a.pg;
    const int n = a.s.hdr->n_moves;
    if (n == 0) return;
    for (int r = blockIdx.x; r < pg.n_rows; r += gridDim.x) {
        const int h = min(held_pages(max(0, pg.lens[r]), pg.page_size), pg.n_cols);
        for (int c = threadIdx.x; c < h; c += COPY_THREADS) {
            int *e = pg.table + (size_t)r * pg.n_cols + c;
            const int p = *e;
            if (p >= 0 && p < pg.n_pages && a.s.at[p] >= 0) *e = a.s.at[p];
        }
    }
    // nothing here reads the counts: at[] says which pages move
    for (int k = blockIdx.x * COPY_THREADS + threadIdx.x; k < n; k += gridDim.x * COPY_THREADS) {
        pg.ref[a.s.fresh[k]] = pg.ref[a.s.from[k]];
        pg.ref[a.s.from[k]] = 0;
    }
    move_pages(a.pools, n, [&](int i) { return make_int2(a.s.from[i], a.s.fresh[i]); });
}

__global__ void __launch_bounds__(COPY_THREADS) k_pages_free(const PagesArgs a) {
    pdl_wait();
    pdl_trigger();
    const M27BPages &pg = a.pg;
    for (int i = blockIdx.x; i < a.n; i += gridDim.x) {
        const int r = a.a[i];
        if (r < 0 || r >= pg.n_rows) {
            if (threadIdx.x == 0) paged_bad(a.bad);
            continue;
        }
        const int h = min(held_pages(max(0, *(volatile int *)(pg.lens + r)), pg.page_size), pg.n_cols);
        // an entry is taken by exchange: a row named twice gives each page back once
        for (int c = threadIdx.x; c < h; c += COPY_THREADS) {
            const int p = atomicExch(pg.table + (size_t)r * pg.n_cols + c, -1);
            if (p >= 0 && p < pg.n_pages) atomicSub(pg.ref + p, 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) *(volatile int *)(pg.lens + r) = 0;
    }
}

__global__ void __launch_bounds__(COPY_THREADS) k_pages_copy(const PagesArgs a) {
    pdl_wait();
    pdl_trigger();
    move_pages(a.pools, a.n, [&](int i) {
        const int s = a.a[i], d = a.b[i];
        if (s < 0 || s >= a.pg.n_pages || d < 0 || d >= a.pg.n_pages) {
            if (threadIdx.x == 0) paged_bad(a.bad);
            return make_int2(-1, -1);
        }
        return make_int2(s, d);
    });
}

namespace {

bool check_pages(const M27BPages *p, const char *what, char *err, size_t cap) {
    if (!p || !p->ref || !p->table || !p->lens) return paged_fail(err, cap, "%s: null ref, table or lens", what);
    if (p->n_pages < 1 || p->n_rows < 1 || p->n_cols < 1)
        return paged_fail(err, cap, "%s: empty cache (%d pages, %d rows of %d)", what, p->n_pages, p->n_rows, p->n_cols);
    if (p->page_size < 1 || p->page_size > 65536)
        return paged_fail(err, cap, "%s: bad page_size (%d)", what, p->page_size);
    if (p->n_pages > 0x3ffffff || p->n_cols > 0x3ffffff)
        return paged_fail(err, cap, "%s: at most 2^26 - 1 pages and columns", what);
    return true;
}

bool check_pools(const M27BPagePool *p, int n, Pools *out, const char *what, char *err, size_t cap) {
    if (n < 1 || n > M27B_MAX_POOLS || !p) return paged_fail(err, cap, "%s: 1 to %d pools (got %d)", what, M27B_MAX_POOLS, n);
    for (int i = 0; i < n; ++i) {
        if (!p[i].base || p[i].n_planes < 1) return paged_fail(err, cap, "%s: pool %d is empty", what, i);
        if (((uintptr_t)p[i].base | p[i].plane_stride | p[i].page_stride | p[i].page_bytes) & 15u)
            return paged_fail(err, cap, "%s: pool %d: base, strides and page bytes must be multiples of 16", what, i);
        if (!p[i].page_bytes || p[i].page_stride < p[i].page_bytes)
            return paged_fail(err, cap, "%s: pool %d: page_stride is shorter than a page", what, i);
        out->p[i] = p[i];
    }
    out->n = n;
    return true;
}

// Four CTAs for each of the 148 SMs, each with up to 32 KB of reads in flight.
unsigned copy_grid() { return 148 * 4; }

bool requests(const void *a, const void *b, const void *scratch, int n, const char *what, char *err, size_t cap) {
    if (n < 0 || n > 0x3fffffff) return paged_fail(err, cap, "%s: bad n (%d)", what, n);
    if (n && (!a || !b)) return paged_fail(err, cap, "%s: null requests", what);
    if (!scratch || ((uintptr_t)scratch & 15u)) return paged_fail(err, cap, "%s: scratch must be 16-byte aligned", what);
    return true;
}

}  // namespace
}  // namespace m27b

using namespace m27b;

extern "C" {

size_t m27b_pages_scratch_bytes(int n_pages, int n_rows, int n) {
    return n_pages < 1 || n_rows < 1 || n < 0 ? 0 : pages_scratch(n_pages, n_rows, n, nullptr, nullptr);
}

bool m27b_pages_resize(const M27BPages *pages, const M27BPagePool *pools, int n_pools, const int *rows,
                       const int *new_lens, int n, void *scratch, int *status, cudaStream_t stream, char *err,
                       size_t err_cap) {
    const char *what = "m27b_pages_resize";
    PagesArgs a = {};
    if (!check_pages(pages, what, err, err_cap) || !check_pools(pools, n_pools, &a.pools, what, err, err_cap) ||
        !requests(rows, new_lens, scratch, n, what, err, err_cap))
        return false;
    if (n == 0) return paged_ok(cudaSuccess, what, err, err_cap);
    a.pg = *pages, a.a = rows, a.b = new_lens, a.n = n, a.out = status, a.bad = status_ptr_current();
    pages_scratch(pages->n_pages, pages->n_rows, n, scratch, &a.s);
    cudaError_t e = launch_pdl(k_resize_plan, dim3(1), dim3(PLAN_THREADS), 0, stream, a);
    if (e == cudaSuccess) e = launch_pdl(k_resize_apply, dim3(copy_grid()), dim3(COPY_THREADS), 0, stream, a);
    return paged_ok(e, what, err, err_cap);
}

bool m27b_pages_fork(const M27BPages *pages, const M27BPagePool *pools, int n_pools, const int *src, const int *dst,
                     int n, void *scratch, int *status, cudaStream_t stream, char *err, size_t err_cap) {
    const char *what = "m27b_pages_fork";
    PagesArgs a = {};
    if (!check_pages(pages, what, err, err_cap) || !check_pools(pools, n_pools, &a.pools, what, err, err_cap) ||
        !requests(src, dst, scratch, n, what, err, err_cap))
        return false;
    if (n == 0) return paged_ok(cudaSuccess, what, err, err_cap);
    a.pg = *pages, a.a = src, a.b = dst, a.n = n, a.out = status, a.bad = status_ptr_current();
    pages_scratch(pages->n_pages, pages->n_rows, n, scratch, &a.s);
    cudaError_t e = launch_pdl(k_fork_plan, dim3(1), dim3(PLAN_THREADS), 0, stream, a);
    if (e == cudaSuccess) e = launch_pdl(k_fork_apply, dim3(copy_grid()), dim3(COPY_THREADS), 0, stream, a);
    return paged_ok(e, what, err, err_cap);
}

bool m27b_pages_free(const M27BPages *pages, const int *rows, int n, cudaStream_t stream, char *err, size_t err_cap) {
    const char *what = "m27b_pages_free";
    if (!check_pages(pages, what, err, err_cap)) return false;
    if (n < 0 || (n && !rows)) return paged_fail(err, err_cap, "%s: bad n (%d) or null rows", what, n);
    if (n == 0) return paged_ok(cudaSuccess, what, err, err_cap);
    PagesArgs a = {};
    a.pg = *pages, a.a = rows, a.n = n, a.bad = status_ptr_current();
    return paged_ok(launch_pdl(k_pages_free, dim3(n < 1184 ? n : 1184), dim3(COPY_THREADS), 0, stream, a), what, err, err_cap);
}

bool m27b_pages_compact(const M27BPages *pages, const M27BPagePool *pools, int n_pools, int *n_live, void *scratch,
                        cudaStream_t stream, char *err, size_t err_cap) {
    const char *what = "m27b_pages_compact";
    PagesArgs a = {};
    if (!check_pages(pages, what, err, err_cap) || !check_pools(pools, n_pools, &a.pools, what, err, err_cap) ||
        !requests(scratch, scratch, scratch, 0, what, err, err_cap))
        return false;
    a.pg = *pages, a.out = n_live;
    pages_scratch(pages->n_pages, pages->n_rows, 0, scratch, &a.s);
    cudaError_t e = launch_pdl(k_compact_plan, dim3(1), dim3(PLAN_THREADS), 0, stream, a);
    if (e == cudaSuccess) e = launch_pdl(k_compact_apply, dim3(copy_grid()), dim3(COPY_THREADS), 0, stream, a);
    return paged_ok(e, what, err, err_cap);
}

bool m27b_pages_copy(const M27BPagePool *pools, int n_pools, int n_pages, const int *src, const int *dst, int n,
                     cudaStream_t stream, char *err, size_t err_cap) {
    const char *what = "m27b_pages_copy";
    PagesArgs a = {};
    if (!check_pools(pools, n_pools, &a.pools, what, err, err_cap)) return false;
    if (n_pages < 1 || n < 0 || (n && (!src || !dst))) return paged_fail(err, err_cap, "%s: bad n (%d) or null pages", what, n);
    if (n == 0) return paged_ok(cudaSuccess, what, err, err_cap);
    a.pg.n_pages = n_pages, a.a = src, a.b = dst, a.n = n, a.bad = status_ptr_current();
    return paged_ok(launch_pdl(k_pages_copy, dim3(copy_grid()), dim3(COPY_THREADS), 0, stream, a), what, err, err_cap);
}

}  // extern "C"
