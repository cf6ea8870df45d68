// paged_attn.cu — attention of new tokens over a paged cache
// (include/m27b_paged.h) on the 5th-generation tensor cores.
//
// Row (token i of sequence b, query head h) at position p, kv head j = h / G,
// G = n_q / n_kv:
//   s_x = scale * q . k_x,  lo <= x <= p,  lo = window > 0 ? max(0, p - window + 1) : 0
//   out = sum_x 2^(c s_x - m) v_x / l,  l = sum_x 2^(c s_x - m),  c = log2 e,
// with a reference value m that follows the running maximum of c s (any m
// gives the same quotient); lse = ln 2 * (m + log2 l).
//
// Work.  An item is 128 rows (128 / G tokens x the G heads of a kv head, so
// that a key tile is read once for the group) of one sequence and kv head,
// over the key tiles its rows see; a unit is one item's work on one key tile.
// All items' units in a row are cut into one even run per CTA (one CTA per
// SM), whatever the batch: a decode step of one long sequence is split over
// its positions, a batch of prompts over its rows, and no CTA gets more than a
// unit above the mean.  An item that several CTAs share leaves one partial
// record (O, m, l of the rows it has) per CTA in the scratch, and the last of
// them to arrive adds the records in CTA order, so that the result does not
// depend on who was last.  Every CTA finds its run itself from cu_q and lens.
//
// A CTA's roles (10 warps):
//   * warp 8 streams the key tiles: TMA boxes of 64 values x the positions of
//     a page (or of the tile, if a page is longer), 128-byte swizzle, each lane
//     one box; a page outside the item's positions is a box past the end of the
//     pool, which reads zeros;
//   * warp 9 issues the MMAs: S = Q K^T with Q in TMEM and K (K-major) in shared
//     memory, O += P V with P in TMEM and V (N-major) in shared memory;
//   * warps 0-7 have half a row per thread, warps w and w + 4 the halves of the
//     same rows: Q into TMEM, the softmax of S (the two halves tell each other
//     their maximum), P back into TMEM, and at the item's end O / l to global
//     memory.  A warp none of whose rows is live (decode: G rows of 128) only
//     passes the barriers.
// TMEM (512 columns): O | Q | S | P, P.  S is free again once the warps
// have loaded it, so the next product runs while they compute; P has two
// buffers.  Steady state of the tensor pipe: P V of tile t, Q K of tile t + 2,
// P V of tile t + 1, ...
//
// m moves only when the running maximum has grown by more than 2^8 since it
// was set: weights then stay below 2^8 (fp32 sums, and far from the 16-bit
// types' limits), and O in TMEM is rescaled on few tiles.
//
// Rows of a V tile that the item does not see may hold anything: their weights
// are 0, but 0 * NaN is not, so the softmax warps overwrite them with zeros in
// shared memory before the product (the first and last tile of an item only).
#include <cudaTypedefs.h>

#include "paged_common.cuh"
#include "tc05.cuh"

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
    unsigned *count;  // arrivals at an item, by the CTA that has its first unit
    float *part;      // two records per CTA
    int *status;
};

constexpr int PA_ROWS = 128;
constexpr int PA_SOFTMAX = 8;  // softmax warps: two for each 32 rows, each with half of a tile's positions
constexpr int PA_PRODUCER = PA_SOFTMAX, PA_ISSUER = PA_SOFTMAX + 1;
constexpr int PA_THREADS = (PA_SOFTMAX + 2) * 32;
constexpr int PA_JOIN = 1024;  // (row, part) pairs whose factors are held at once when records are joined
constexpr int PA_MAX_CTAS = 1024;  // counters in the scratch's first 4096 bytes
constexpr float PA_SLACK = 8.0f;   // growth of the maximum (log2) before m follows

template <int HD> struct PaPlan {
    static constexpr int KT = HD == 256 ? 64 : 128;  // positions per key tile
    static constexpr int STAGES = HD == 64 ? 6 : 3;
    static constexpr int TILE = KT * HD * 2;         // bytes of K (or V) of a tile
    static constexpr int O = 0, Q = HD, S = Q + HD / 2, P = S + KT;  // TMEM columns
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * 2 * TILE + 512;
    static_assert(P + KT <= 512, "TMEM plan");
    static_assert(SMEM > MMA_SMEM_MIN && SMEM <= MMA_SMEM_LIMIT, "one CTA per SM");
};

// floats of a partial record: O[d / 4][row][4], then (m, l) of the rows
__host__ __device__ constexpr size_t pa_record(int hd) { return (size_t)PA_ROWS * (hd + 2); }

// ---- tensor core helpers ----

// D[tmem] (+)= A[tmem] B[smem], 16-bit operands, fp32 sums, one thread.
M27B_DI void umma_f16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0)
        : "memory");
}
// Matrix descriptor, 128-byte swizzle: 1024 bytes between groups of 8
// 128-byte rows; `lead` bytes between 64-value columns (N-major operands).
M27B_DI uint64_t umma_desc128(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// fp32 accumulator, f16 or bf16 operands, A K-major, B K-major or N-major, M = 128.
template <bool BF, int N, bool BMN>
constexpr uint32_t umma_idesc_f16() {
    return (1u << 4) | ((BF ? 1u : 0u) << 7) | ((BF ? 1u : 0u) << 10) | ((BMN ? 1u : 0u) << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
M27B_DI void tmem_ld32(uint32_t taddr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
          "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
          "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
M27B_DI void tmem_st32(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
        "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
        "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
M27B_DI void tmem_st16(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
M27B_DI void tma_load_4d(uint32_t dst, const CUtensorMap *tm, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"((unsigned long long)tm), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
M27B_DI float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---- the list of items ----

// One sequence as the kernel sees it: q_n tokens from row q_lo of q, the first
// at position `base` (negative: before the first position), nrt row tiles.
struct PaSeq {
    int q_lo, q_n, base, nrt, row;
};

M27B_DI PaSeq pa_seq(const AttnArgs &a, int b, int tq, bool report) {
    PaSeq s;
    const int2 t = seq_tokens(a.bt, b);
    s.q_lo = t.x, s.q_n = t.y - t.x;
    s.row = seq_row(a.bt, b, a.kv.n_rows);
    const int cap = a.kv.n_cols * a.kv.page_size;
    int len = s.row < 0 ? 0 : __ldg(a.bt.lens + s.row);
    if (report && s.q_n > 0 && (s.row < 0 || len > cap)) paged_bad(a.status);
    len = max(0, min(len, cap));
    s.row = max(0, s.row);
    s.base = (int)max((long long)-(1 << 30), (long long)len - __ldg(a.bt.cu_q + b + 1) + t.x);
    s.nrt = (s.q_n + tq - 1) / tq;
    return s;
}

// Positions [lo, hi) that row tile r sees, and its key tiles [kt0, kt1).
struct PaSpan {
    int lo, hi, kt0, kt1;
    M27B_DI int units() const { return max(1, kt1 - kt0); }
};
template <int KT>
M27B_DI PaSpan pa_span(const PaSeq &s, int r, int tq, int window) {
    const int i0 = r * tq, i1 = min(s.q_n, i0 + tq);
    PaSpan p;
    p.hi = max(0, s.base + i1);
    p.lo = window > 0 ? min(p.hi, max(0, s.base + i0 - window + 1)) : 0;
    p.kt0 = p.lo / KT;
    p.kt1 = p.hi > p.lo ? (p.hi + KT - 1) / KT : p.kt0;
    return p;
}

// Units of one kv head of a sequence, for each lane its own; sequences of many
// row tiles are summed by the whole warp.
template <int KT>
M27B_DI long long pa_head_units(const PaSeq &s, int tq, int window) {
    const int lane = threadIdx.x & 31;
    long long u = 0;
    if (s.nrt <= 4)
        for (int r = 0; r < s.nrt; ++r) u += pa_span<KT>(s, r, tq, window).units();
    for (unsigned big = __ballot_sync(0xffffffffu, s.nrt > 4); big; big &= big - 1) {
        const int src = __ffs(big) - 1;
        PaSeq o;
        o.q_n = __shfl_sync(0xffffffffu, s.q_n, src);
        o.base = __shfl_sync(0xffffffffu, s.base, src);
        o.nrt = __shfl_sync(0xffffffffu, s.nrt, src);
        long long v = 0;
        for (int r = lane; r < o.nrt; r += 32) v += pa_span<KT>(o, r, tq, window).units();
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (lane == src) u = v;
    }
    return u;
}

// A CTA's run of units, and where it begins.
struct PaRun {
    long long total, begin, end;
    int ctas;             // CTAs that have a run
    int b, j, r, off;     // first item, and units of it that belong to the CTAs before
    long long seq_off, head_units;  // the run's begin within sequence b; units of a kv head of it
    PaSeq seq;                      // sequence b
};

// x / y for counts that nearly always fit 32 bits (a 64-bit division is a
// routine of some hundred cycles, and the prologue has several in a row).
M27B_DI long long div_count(long long x, long long y) {
    return (x | y) >> 32 ? x / y : (long long)((unsigned)x / (unsigned)y);
}

// The item at hand and its neighbours, walked alike by every role.
template <int KT>
struct PaWalk {
    const AttnArgs &a;
    int tq;
    long long u, end;
    int b, j, r, off;
    PaSeq s;
    PaSpan sp;
    int take;  // units of this item in this run

    M27B_DI PaWalk(const AttnArgs &a_, const PaRun &run, int tq_) : a(a_), tq(tq_) {
        u = run.begin, end = run.end, b = run.b, j = run.j, r = run.r, off = run.off;
        s = run.seq;
        if (more()) span();
    }
    M27B_DI bool more() const { return u < end; }
    M27B_DI void seq() { s = pa_seq(a, b, tq, false); }
    M27B_DI void span() {
        sp = pa_span<KT>(s, r, tq, a.window);
        take = (int)min((long long)(sp.units() - off), end - u);
    }
    // key tiles of this item in this run
    M27B_DI int tiles() const { return sp.kt1 > sp.kt0 ? take : 0; }
    M27B_DI int first() const { return sp.kt0 + off; }
    M27B_DI bool whole() const { return off == 0 && take == sp.units(); }
    M27B_DI void next() {
        u += take;
        off = 0;
        if (!more()) return;
        if (++r == s.nrt) {
            r = 0;
            if (++j == a.kv.n_kv) {
                j = 0;
                do {
                    ++b;
                    seq();
                } while (s.nrt == 0);  // units are left, so a sequence with tokens follows
            }
        }
        span();
    }
};

// Sum over the CTA and of the threads before this one.
M27B_DI long long pa_scan(long long v, long long *red, long long *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    __syncthreads();
    if (lane == 31) red[warp] = inc;
    __syncthreads();
    long long before = 0, all = 0;
    for (int w = 0; w < PA_THREADS / 32; ++w) {
        if (w < warp) before += red[w];
        all += red[w];
    }
    *total = all;
    return before + inc - v;
}

// All threads: fill `run` (shared memory) with this CTA's run.
template <int KT>
M27B_DI void pa_find_run(const AttnArgs &a, int tq, PaRun *run, long long *red) {
    const int n = a.bt.n_seq;
    long long total = 0, head = 0, u = 0, before = 0, sum;
    PaSeq s;
    for (int b0 = 0; b0 < n; b0 += PA_THREADS) {
        const int b = b0 + threadIdx.x;
        s = {0, 0, 0, 0, 0};
        if (b < n) s = pa_seq(a, b, tq, blockIdx.x == 0);
        head = pa_head_units<KT>(s, tq, a.window);
        u = head * a.kv.n_kv;
        before = pa_scan(u, red, &sum);
        total += sum;
    }
    const long long ctas = min((long long)gridDim.x, total), c = blockIdx.x;
    const long long begin = c < ctas ? div_count(c * total, ctas) : 0,
                    end = c < ctas ? div_count((c + 1) * total, ctas) : 0;
    if (threadIdx.x == 0) {
        run->total = total, run->ctas = (int)ctas, run->begin = begin, run->end = end;
        run->b = n;
    }
    __syncthreads();
    if (begin >= end) return;
    long long at = 0;
    for (int b0 = 0; b0 < n && at <= begin; b0 += PA_THREADS) {
        const int b = b0 + threadIdx.x;
        if (n > PA_THREADS) {
            s = {0, 0, 0, 0, 0};
            if (b < n) s = pa_seq(a, b, tq, false);
            head = pa_head_units<KT>(s, tq, a.window);
            u = head * a.kv.n_kv;
            before = pa_scan(u, red, &sum);
        }
        if (begin >= at + before && begin < at + before + u) {
            run->b = b;
            run->seq_off = begin - at - before;
            run->head_units = head;
            run->seq = s;
        }
        at += sum;
        __syncthreads();
    }
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        s = run->seq;
        const long long j = div_count(run->seq_off, run->head_units);
        long long off = run->seq_off - j * run->head_units;
        int r0 = 0;
        for (;; r0 += 32) {
            const int v = r0 + lane < s.nrt ? pa_span<KT>(s, r0 + lane, tq, a.window).units() : 0;
            long long inc = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long x = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += x;
            }
            const unsigned past = __ballot_sync(0xffffffffu, inc > off);
            if (past) {
                const int l = __ffs(past) - 1;
                if (lane == l) run->j = (int)j, run->r = r0 + l, run->off = (int)(off - (inc - v));
                break;
            }
            off -= __shfl_sync(0xffffffffu, inc, 31);
            if (r0 + 32 >= s.nrt) break;  // not reached: the units add up
        }
    }
    __syncthreads();
}

struct PaShared {
    PaRun run;
    long long red[PA_THREADS / 32];
    float half[2][2][PA_ROWS];  // what the two warps of a row tell each other, by turns
    float2 join[PA_JOIN];
    uint32_t tmem;
    int abort;
    int last;
};

// Add up the np records of an item of CTAs c0, c0 + 1, ... and write its rows;
// the softmax warps of the CTA that arrived last.  Rows are taken so many at a
// time that their parts' m and l fit `join`, fetched in one round trip; a
// part's factor is 2^(m - max) / sum.  Then four quadruples of values x four
// parts a thread are in flight.
template <int HD, bool BF, class Walk, class Sync>
M27B_DI bool pa_join(const AttnArgs &a, const Walk &w, int c0, int np, int rows, int G, int tq, float2 *join, int tid,
                     Sync all_here) {
    constexpr int NT = 32 * PA_SOFTMAX;
    auto record = [&](int x) { return a.part + (size_t)(2 * (c0 + x) + (x == 0 ? 1 : 0)) * pa_record(HD); };
    const int at_once = min(rows, PA_JOIN / np);
    for (int r0 = 0; r0 < rows; r0 += at_once) {
        const int nr = min(at_once, rows - r0);
        for (int e = tid; e < nr * np; e += NT) {
            const int x = e / nr;
            join[e] = __ldcg((const float2 *)(record(x) + (size_t)PA_ROWS * HD) + r0 + e - x * nr);
        }
        if (!all_here()) return false;
        for (int r = tid; r < nr; r += NT) {
            float mx = -INFINITY, ls = 0.0f;
            for (int x = 0; x < np; ++x) mx = fmaxf(mx, join[x * nr + r].x);
            const float ref = mx == -INFINITY ? 0.0f : mx;
            for (int x = 0; x < np; ++x) {
                const float2 ml = join[x * nr + r];
                const float f = ex2(ml.x - ref);
                join[x * nr + r].x = f;
                ls = fmaf(f, ml.y, ls);
            }
            const float inv = ls > 0.0f ? 1.0f / ls : 0.0f;
            for (int x = 0; x < np; ++x) join[x * nr + r].x *= inv;
            if (a.lse)
                a.lse[(w.s.q_lo + w.r * tq + (r0 + r) / G) * (long long)a.n_q + w.j * G + (r0 + r) % G] =
                    ls > 0.0f ? 0.69314718055994530942f * (mx + log2f(ls)) : -INFINITY;
        }
        if (!all_here()) return false;
        for (int e0 = tid; e0 < nr * (HD / 4); e0 += 4 * NT) {
            float4 o[4] = {};
            int rr[4], dd[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) dd[g] = (e0 + NT * g) / nr, rr[g] = e0 + NT * g - dd[g] * nr;
            for (int x0 = 0; x0 < np; x0 += 4) {
                float4 y[4][4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float4 *rx = (const float4 *)record(x0 + x) + r0;
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        y[g][x] = x0 + x < np && dd[g] < HD / 4 ? __ldcg(rx + (size_t)dd[g] * PA_ROWS + rr[g])
                                                               : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float f = x0 + x < np ? join[(x0 + x) * nr + rr[g]].x : 0.0f;
                        o[g].x = fmaf(f, y[g][x].x, o[g].x), o[g].y = fmaf(f, y[g][x].y, o[g].y);
                        o[g].z = fmaf(f, y[g][x].z, o[g].z), o[g].w = fmaf(f, y[g][x].w, o[g].w);
                    }
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (dd[g] >= HD / 4) continue;
                const long long tk = w.s.q_lo + w.r * tq + (r0 + rr[g]) / G;
                *(uint2 *)((uint16_t *)a.out + tk * a.out_stride + (long long)(w.j * G + (r0 + rr[g]) % G) * HD + 4 * dd[g]) =
                    make_uint2(Half16<BF>::down(o[g].x, o[g].y), Half16<BF>::down(o[g].z, o[g].w));
            }
        }
        if (r0 + at_once < rows && !all_here()) return false;  // the factors are about to be replaced
    }
    return true;
}

template <int HD, bool BF>
__global__ void __launch_bounds__(PA_THREADS, 1)
    k_paged_attn(const AttnArgs a, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
    using L = PaPlan<HD>;
    constexpr int KT = L::KT, ST = L::STAGES, TILE = L::TILE, NCH = HD / 64;
    extern __shared__ uint8_t pa_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)pa_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = (uint64_t *)(smem + (size_t)ST * 2 * TILE);
    uint64_t *kfull = bars, *vfull = kfull + ST, *empty = vfull + ST, *qfull = empty + ST, *sfull = qfull + 1,
             *sfree = sfull + 1, *pfull = sfree + 1, *pdone = pfull + 2, *drain = pdone + 2, *meet = drain + 1, *pair = meet + 1;
    __shared__ PaShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = a.n_q / a.kv.n_kv, tq = PA_ROWS / G;
    volatile int *abort = &sh.abort;

    if (tid == 0) {
        for (int s = 0; s < ST; ++s) {
            mbar_init(&kfull[s], 1);
            mbar_init(&vfull[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(qfull, PA_SOFTMAX);
        mbar_init(sfull, 1);
        mbar_init(sfree, PA_SOFTMAX);
        for (int i = 0; i < 4; ++i) mbar_init(&pair[i], 2);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&pfull[i], PA_SOFTMAX);
            mbar_init(&pdone[i], 1);
        }
        mbar_init(drain, 1);
        mbar_init(meet, PA_SOFTMAX);
        sh.abort = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    }
    pdl_wait();
    pdl_trigger();
    tc_fence_before();
    pa_find_run<KT>(a, tq, &sh.run, sh.red);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    PaWalk<KT> w(a, sh.run, tq);

    if (warp == PA_PRODUCER) {
        // lane = box: K or V, 64-value column, page of the tile
        const int ps = a.kv.page_size, rows = min(ps, KT), npp = KT / rows;
        const int pg = lane % npp, ch = (lane / npp) % NCH, isv = lane / (npp * NCH);
        const uint32_t dst0 = smem_u32(smem) + isv * TILE + ch * (KT * 128) + pg * rows * 128;
        const int shift = 31 - __clz(ps);
        int t = 0;
        bool ok = true;
        for (; ok && w.more(); w.next()) {
            const int n = w.tiles();
            const int *ids = a.kv.table + (long long)w.s.row * a.kv.n_cols;
            int have = -1, cur = 0;  // lane's page id of pages have + lane
            for (int i = 0; i < n; ++i, ++t) {
                const int s = t % ST, x0 = (w.first() + i) * KT, p0 = x0 >> shift;
                if (have < 0 || p0 < have || p0 + npp > have + 32) {
                    have = p0;
                    const int p = have + lane;
                    const bool in = p < a.kv.n_cols && (p << shift) < w.sp.hi && (p + 1) << shift > w.sp.lo;
                    cur = in ? __ldg(ids + p) : a.kv.n_pages;
                    if (cur < 0 || cur > a.kv.n_pages || (in && cur == a.kv.n_pages)) {
                        paged_bad(a.status);
                        cur = a.kv.n_pages;
                    }
                }
                const int page = __shfl_sync(0xffffffffu, cur, p0 + pg - have);
                if (t >= ST && !warp_wait_or_abort(&empty[s], (uint32_t)((t / ST - 1) & 1), abort, a.status)) {
                    ok = false;
                    break;
                }
                if (lane == 0) {
                    mbar_arrive_expect_tx(&kfull[s], TILE);
                    mbar_arrive_expect_tx(&vfull[s], TILE);
                }
                __syncwarp();
                if (isv < 2)
                    tma_load_4d(dst0 + s * 2 * TILE, isv ? &tmv : &tmk, ch * 64, x0 & (ps - 1), w.j,
                                page, isv ? &vfull[s] : &kfull[s]);
            }
        }
        // every copy lands before the CTA's shared memory is released (bounded)
        for (int i = max(0, t - ST); i < t; ++i) {
            mbar_wait_bounded(&kfull[i % ST], (uint32_t)((i / ST) & 1), a.status, 5);
            mbar_wait_bounded(&vfull[i % ST], (uint32_t)((i / ST) & 1), a.status, 5);
        }
    } else if (warp == PA_ISSUER) {
        if (lane == 0) {
            constexpr uint32_t id_s = umma_idesc_f16<BF, KT, false>(), id_o = umma_idesc_f16<BF, HD, true>();
            const uint32_t base = smem_u32(smem);
            int t0 = 0, item = 0;
            bool ok = true;
            for (; ok && w.more(); w.next()) {
                const int n = w.tiles();
                if (n == 0) continue;
                // S of tile t = Q K^T, once S has been read and the keys are there
                auto scores = [&](int t) {
                    if (t > 0 && !wait_or_abort(sfree, (uint32_t)((t - 1) & 1), abort, a.status)) return false;
                    if (!wait_or_abort(&kfull[t % ST], (uint32_t)((t / ST) & 1), abort, a.status)) return false;
                    tc_fence_after();
                    const uint32_t k = base + (t % ST) * 2 * TILE;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk)
                        umma_f16_ts(tmem + L::S, tmem + L::Q + kk * 8,
                                    umma_desc128(k + (kk / 4) * (KT * 128) + (kk % 4) * 32, 16), id_s, kk > 0);
                    umma_commit(sfull);
                    return true;
                };
                ok = wait_or_abort(qfull, (uint32_t)(item & 1), abort, a.status);
                tc_fence_after();
                ok = ok && scores(t0) && (n < 2 || scores(t0 + 1));
                for (int i = 0; ok && i < n; ++i) {
                    const int t = t0 + i;
                    if (!wait_or_abort(&pfull[t & 1], (uint32_t)((t >> 1) & 1), abort, a.status) ||
                        !wait_or_abort(&vfull[t % ST], (uint32_t)((t / ST) & 1), abort, a.status)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t v = base + (t % ST) * 2 * TILE + TILE;
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        umma_f16_ts(tmem + L::O, tmem + L::P + (t & 1) * (KT / 2) + kk * 8,
                                    umma_desc128(v + kk * 2048, KT * 128), id_o, i > 0 || kk > 0);
                    umma_commit(&empty[t % ST]);
                    umma_commit(&pdone[t & 1]);
                    if (i + 2 < n) ok = scores(t + 2);
                }
                t0 += n;
                ++item;
            }
            // every MMA issued above (bounded, even after an abort)
            umma_commit(drain);
            mbar_wait_bounded(drain, 0u, a.status, 5);
        }
        __syncwarp();
    } else {
        // row = TMEM lane; this thread has positions [half KH, half KH + KH) of
        // each tile, and columns [half HD / 2, ..) of O
        constexpr int KH = KT / 2;
        const int quarter = warp & 3, half = warp >> 2, row = 32 * quarter + lane;
        const uint32_t lane_base = tmem + ((uint32_t)(32 * quarter) << 16);
        const float c = a.scale * 1.44269504088896340736f;  // log2 e
        int t = 0, met = 0, told = 0;
        bool ok = true;
        // the softmax warps wait for one another (bounded: a warp that gave up never comes)
        auto all_here = [&] {
            __syncwarp();
            if (lane == 0) mbar_arrive(meet);
            return warp_wait_or_abort(meet, (uint32_t)(met++ & 1), abort, a.status);
        };
        // this row's value of the other half
        auto other = [&](float mine, float &theirs) {
            const int turn = told++ & 1;
            sh.half[turn][half][row] = mine;
            __syncwarp();
            if (lane == 0) mbar_arrive(&pair[quarter]);
            const bool here = warp_wait_or_abort(&pair[quarter], (uint32_t)turn, abort, a.status);
            theirs = *(volatile float *)&sh.half[turn][half ^ 1][row];
            return here;
        };
        for (; ok && w.more(); w.next()) {
            const int n = w.tiles(), i = w.r * tq + row / G, h = w.j * G + row % G;
            const int rows = min(tq, w.s.q_n - w.r * tq) * G;
            const bool live = row < rows, idle = 32 * quarter >= rows;  // idle: no row of this warp is live
            // a dead row's scores are garbage that no one reads
            const int hi = live ? w.s.base + i + 1 : 0x7fffffff;
            const int lo = live && a.window > 0 ? max(0, hi - a.window) : 0;
            float m = -INFINITY, l = 0.0f;  // m in units of c s
            if (n > 0) {
                // half of this row's Q into TMEM (its last product has been read as S)
                const uint16_t *qp = (const uint16_t *)a.q + (long long)(w.s.q_lo + i) * a.q_stride + (long long)h * HD + half * (HD / 2);
#pragma unroll
                for (int x = 0; x < HD / 64; ++x) {
                    uint32_t v[16];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint4 y = live ? __ldg((const uint4 *)(qp + 32 * x) + e) : make_uint4(0, 0, 0, 0);
                        v[4 * e] = y.x, v[4 * e + 1] = y.y, v[4 * e + 2] = y.z, v[4 * e + 3] = y.w;
                    }
                    tmem_st16(lane_base + L::Q + half * (HD / 4) + 16 * x, v);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(qfull);
            }
            for (int k = 0; k < n; ++k, ++t) {
                const int x0 = (w.first() + k) * KT;
                if (!(ok = warp_wait_or_abort(sfull, (uint32_t)(t & 1), abort, a.status))) break;
                if (idle) {
                    if (lane == 0) mbar_arrive(sfree);
                } else {
                    tc_fence_after();
                    float s[KH];
#pragma unroll
                    for (int x = 0; x < KH / 32; ++x) tmem_ld32(lane_base + L::S + half * KH + 32 * x, (uint32_t *)s + 32 * x);
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sfree);
                    const int xh = x0 + half * KH;
                    if (__any_sync(0xffffffffu, xh < lo || xh + KH > hi)) {
#pragma unroll
                        for (int x = 0; x < KH; ++x)
                            if (xh + x < lo || xh + x >= hi) s[x] = -INFINITY;
                    }
                    float tops[4] = {s[0], s[1], s[2], s[3]}, theirs;
#pragma unroll
                    for (int x = 4; x < KH; ++x) tops[x & 3] = fmaxf(tops[x & 3], s[x]);
                    const float mine = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    if (!(ok = other(mine, theirs))) break;
                    const float top = c * fmaxf(mine, theirs);
                    if (__any_sync(0xffffffffu, top > m + PA_SLACK)) {
                        const float to = top > m + PA_SLACK ? top : m;
                        const float f = m == -INFINITY ? 1.0f : ex2(m - to);
                        m = to;
                        l *= f;
                        if (k > 0) {
                            // this half's columns of O, once the products so far are done
                            if (!(ok = warp_wait_or_abort(&pdone[(t - 1) & 1], (uint32_t)(((t - 1) >> 1) & 1), abort, a.status)))
                                break;
                            tc_fence_after();
#pragma unroll 1
                            for (int x = 0; x < HD / 64; ++x) {
                                uint32_t v[32];
                                tmem_ld32(lane_base + L::O + half * (HD / 2) + 32 * x, v);
                                tmem_wait_ld();
#pragma unroll
                                for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                                tmem_st32(lane_base + L::O + half * (HD / 2) + 32 * x, v);
                            }
                            tmem_wait_st();
                        }
                    }
                    const float mm = m == -INFINITY ? 0.0f : m;
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    uint32_t p[KH / 2];
#pragma unroll
                    for (int e = 0; e < KH / 2; ++e) {
                        const float p0 = ex2(fmaf(s[2 * e], c, -mm)), p1 = ex2(fmaf(s[2 * e + 1], c, -mm));
                        sum[e & 3] += p0 + p1;
                        p[e] = Half16<BF>::down(p0, p1);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    // P's buffer is free once the product of two tiles ago is done
                    if (t >= 2 && !(ok = warp_wait_or_abort(&pdone[t & 1], (uint32_t)(((t - 2) >> 1) & 1), abort, a.status))) break;
                    const uint32_t pc = lane_base + L::P + (t & 1) * (KT / 2) + half * (KH / 2);
                    if constexpr (KH == 64) tmem_st32(pc, p);
                    else tmem_st16(pc, p);
                }
                // values of positions that no row of the item sees
                if (x0 < w.sp.lo || x0 + KT > w.sp.hi) {
                    if (!(ok = warp_wait_or_abort(&vfull[t % ST], (uint32_t)((t / ST) & 1), abort, a.status))) break;
                    uint8_t *v = smem + (size_t)(t % ST) * 2 * TILE + TILE;
                    for (int e = tid; e < KT * NCH * 8; e += 32 * PA_SOFTMAX) {
                        const int x = (e >> 3) % KT;
                        if (x0 + x < w.sp.lo || x0 + x >= w.sp.hi) *(uint4 *)(v + (size_t)e * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[t & 1]);
            }
            if (!ok) break;
            if (n > 0) {
                if (!(ok = warp_wait_or_abort(&pdone[(t - 1) & 1], (uint32_t)(((t - 1) >> 1) & 1), abort, a.status))) break;
                tc_fence_after();
            }
            if (!idle) {
                float theirs;
                if (!(ok = other(l, theirs))) break;
                l = half ? theirs + l : l + theirs;
            }
            const long long tok = w.s.q_lo + i;
            if (w.whole()) {
                const float inv = l > 0.0f ? 1.0f / l : 0.0f;
                uint16_t *op = (uint16_t *)a.out + tok * a.out_stride + (long long)h * HD + half * (HD / 2);
#pragma unroll 1
                for (int x = 0; x < (idle ? 0 : HD / 64); ++x) {
                    uint32_t v[32];
                    if (n > 0) {
                        tmem_ld32(lane_base + L::O + half * (HD / 2) + 32 * x, v);
                        tmem_wait_ld();
                    }
                    if (live)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            uint32_t y[4];
#pragma unroll
                            for (int d = 0; d < 4; ++d)
                                y[d] = l > 0.0f ? Half16<BF>::down(__uint_as_float(v[8 * e + 2 * d]) * inv,
                                                                   __uint_as_float(v[8 * e + 2 * d + 1]) * inv)
                                                : 0u;
                            *((uint4 *)(op + 32 * x) + e) = make_uint4(y[0], y[1], y[2], y[3]);
                        }
                }
                if (live && a.lse && half == 0)
                    a.lse[tok * a.n_q + h] = l > 0.0f ? 0.69314718055994530942f * (m + log2f(l)) : -INFINITY;
                tc_fence_before();
            } else {
                // this CTA's part of the item; the last of the item's CTAs adds them up
                const long long U = w.u - w.off;
                const int c0 = (int)div_count((U + 1) * sh.run.ctas + sh.run.total - 1, sh.run.total) - 1;
                const int c1 = (int)div_count((U + w.sp.units()) * sh.run.ctas + sh.run.total - 1, sh.run.total) - 1;
                const int me = blockIdx.x;
                float *rec = a.part + (size_t)(2 * me + (me == c0 ? 1 : 0)) * pa_record(HD);
#pragma unroll 1
                for (int x = 0; x < (idle ? 0 : HD / 64); ++x) {
                    uint32_t v[32];
                    tmem_ld32(lane_base + L::O + half * (HD / 2) + 32 * x, v);
                    tmem_wait_ld();
                    if (live)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            __stcg((uint4 *)rec + (size_t)(half * (HD / 8) + 8 * x + e) * PA_ROWS + row,
                                   make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]));
                }
                if (live && half == 0) __stcg((float2 *)(rec + (size_t)PA_ROWS * HD) + row, make_float2(m, l));
                tc_fence_before();
                __threadfence();
                if (!(ok = all_here())) break;
                if (tid == 0) {
                    const bool last = atomicAdd(a.count + c0, 1u) == (unsigned)(c1 - c0);
                    if (last) a.count[c0] = 0u;
                    __threadfence();
                    sh.last = last;
                }
                if (!(ok = all_here())) break;
                if (*(volatile int *)&sh.last) ok = pa_join<HD, BF>(a, w, c0, c1 - c0 + 1, rows, G, tq, sh.join, tid, all_here);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

namespace {

PFN_cuTensorMapEncodeTiled_v12000 pa_encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                       q == cudaDriverEntryPointSuccess
                   ? (PFN_cuTensorMapEncodeTiled_v12000)p
                   : nullptr;
    }();
    return fn;
}

// (value, slot, kv head, page) of a pool; a box is 64 values of `rows` slots.
bool pa_map(CUtensorMap *tm, const M27BPagedKV &kv, const void *pool, int rows) {
    auto enc = pa_encoder();
    if (!enc) return false;
    const cuuint64_t dim[4] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.page_size, (cuuint64_t)kv.n_kv, (cuuint64_t)kv.n_pages};
    const cuuint64_t stride[3] = {(cuuint64_t)kv.n_kv * kv.head_dim * 2, (cuuint64_t)kv.head_dim * 2,
                                  (cuuint64_t)kv.page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, one[4] = {1, 1, 1, 1};
    return enc(tm, kv.type == M27B_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
               const_cast<void *>(pool), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// CTAs of a launch: one per SM of the current device.
int pa_ctas() {
    static int sms[64] = {};
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 0;
    if (dev < 64 && sms[dev]) return sms[dev];
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    if (n > PA_MAX_CTAS) n = PA_MAX_CTAS;
    if (dev < 64) sms[dev] = n;
    return n;
}
constexpr int PA_SCRATCH_CTAS = 160;  // most CTAs the scratch has records for

template <int HD, bool BF>
cudaError_t pa_launch(const AttnArgs &a, const CUtensorMap &k, const CUtensorMap &v, int ctas, cudaStream_t st) {
    auto kern = k_paged_attn<HD, BF>;
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PaPlan<HD>::SMEM);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    return launch_pdl(kern, dim3(ctas), dim3(PA_THREADS), PaPlan<HD>::SMEM, st, a, k, v);
}

template <bool BF>
cudaError_t pa_launch_hd(const AttnArgs &a, const CUtensorMap &k, const CUtensorMap &v, int ctas, cudaStream_t st) {
    switch (a.kv.head_dim) {
    case 64: return pa_launch<64, BF>(a, k, v, ctas, st);
    case 128: return pa_launch<128, BF>(a, k, v, ctas, st);
    default: return pa_launch<256, BF>(a, k, v, ctas, st);
    }
}

}  // namespace
}  // namespace m27b

using namespace m27b;

extern "C" {

size_t m27b_paged_attn_scratch_bytes(int n_q, int n_kv, int head_dim) {
    if (n_kv < 1 || n_kv > 1024 || n_q < n_kv || n_q % n_kv || n_q / n_kv > 128) return 0;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    return PA_MAX_CTAS * sizeof(unsigned) + 2 * PA_SCRATCH_CTAS * pa_record(head_dim) * sizeof(float);
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
    if (kv->page_stride >= 1ll << 39) return paged_fail(err, err_cap, "%s: page_stride (%lld) too large", what, kv->page_stride);
    const int rows = kv->head_dim == 256 ? (kv->page_size < 64 ? kv->page_size : 64) : (kv->page_size < 128 ? kv->page_size : 128);
    CUtensorMap tk, tv;
    if (!pa_map(&tk, *kv, kv->k, rows) || !pa_map(&tv, *kv, kv->v, rows))
        return paged_fail(err, err_cap, "%s: the pools' tensor maps were refused", what);
    int ctas = pa_ctas();
    if (ctas < 1) return paged_fail(err, err_cap, "%s: no CUDA device", what);
    if (ctas > PA_SCRATCH_CTAS) ctas = PA_SCRATCH_CTAS;
    const AttnArgs a = {*kv, *batch, q, out, lse, q_stride, out_stride, n_q, window > 0 ? window : 0, scale,
                        (unsigned *)scratch, (float *)((char *)scratch + PA_MAX_CTAS * sizeof(unsigned)),
                        status_ptr_current()};
    return paged_ok(kv->type == M27B_TYPE_BF16 ? pa_launch_hd<true>(a, tk, tv, ctas, stream)
                                               : pa_launch_hd<false>(a, tk, tv, ctas, stream),
                    what, err, err_cap);
}

}  // extern "C"
