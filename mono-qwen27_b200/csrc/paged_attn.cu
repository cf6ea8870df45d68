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
// All items' units in a row are cut into one even run per worker, whatever the
// batch: a decode step of one long sequence is split over its positions, a
// batch of prompts over its rows, and no worker gets more than a unit above
// the mean.  Every worker finds its run itself from cu_q and lens.  An item
// that several workers share leaves one partial record (O, m, l of its rows)
// per worker in the scratch, and a second launch, whose blocks wait on the
// SMs for the first to end, adds the records in worker order.
//
// A worker is one CTA (k_paged_attn, one per SM), or for many rows a cluster of
// two CTAs (k_paged_attn_pair) that take 128 rows each and share the key tiles:
// each loads half of K's positions and half of V's columns, and the MMAs of the
// pair (cta_group::2, M = 256) read both halves.  A single CTA's 128 rows need
// 64 KB of keys and values per 1024 cycles of tensor work (head_dim 256, 64
// positions), which the shared memory cannot take in and hand to the MMAs at
// that rate; a pair needs half.
//
// What bounds it: decode (64 sequences of 300 to 8192 positions, 24 heads of
// 256 over 4, 680 MB of cache) the memory: 120 us, 5.7 TB/s; a chunk of 4096
// tokens over 8192 positions, same heads, the tensor pipe: 387 us with the pipe
// busy 83 % of it at full clocks, 430 to 460 us back to back under the power
// limit, 484 to 492 us a call from cold L2 (1.26 to 1.28 PFLOP/s); few rows and short contexts the latency of the launch, the first loads
// and the join: 13 us for one token over 769 positions.  The same chunk with 16
// heads of 128 over 8 (206 GFLOP, 224 us cold) and of 64 (255 us cold): the
// hand-offs between the roles; the tensor pipe is busy 46 and 19 % of the time,
// the exponentials' unit 49 and 41, the issue slots 36 and 38.
//
// A CTA's roles:
//   * warp 8 streams the key tiles into a ring of slots, in the order in which
//     the MMAs use them (K0 K1 V0 K2 V1 ...): TMA boxes of 64 values x the
//     positions of a page (or of the tile, if a page is longer), 128-byte
//     swizzle, each lane one box; a page outside the item's positions is a box
//     past the end of the pool, which reads zeros;
//   * warp 9 issues the MMAs: S = Q K^T with K (K-major) in shared memory, O += P
//     V with P in TMEM and V (N-major) in shared memory.  Q is in TMEM, in a
//     pair in shared memory.  In a pair the first CTA's warp issues;
//   * warps 0-7: the softmax of S, P into TMEM, and at the item's end O / l to
//     global memory.  In a single CTA warps w and w + 4 have the halves of the
//     same rows and tell each other their maximum (one tile's latency counts:
//     decode has few live rows); in a pair they take turns with whole tiles
//     and hand m on (throughput counts).  A warp none of whose rows is live
//     (decode: G rows of 128) only passes the barriers.
// TMEM (512 columns): O | Q | S | P, P (a pair: O | S (, S) | P, P).  S is free
// again once the warps have loaded it, so the next product runs while they
// compute; P has two buffers.  Steady state of the tensor pipe: P V of tile t,
// Q K of tile t + 2, P V of tile t + 1, ...
//
// m moves only when the running maximum has grown by more than 2^8 since it
// was set, so that O in TMEM is rescaled on few tiles.  For bf16 it is set to
// the maximum: weights stay below 2^8, far from the type's limits.  For f16 it is
// set 7 below: weights stay below 2^15 (f16 ends at 2^16), and the largest is at
// least 2^7, so that those which f16 holds with fewer than 11 bits (below 2^-14,
// with an absolute error of 2^-25) are below 2^-21 of it and their errors at
// most 2^-32 of it each.  Set to the maximum, a weight of 2^-25 of the largest is
// lost, and 40000 such positions beside a large one are 0.1 % of the sum.
//
// Rows of a V tile that no row of the sequence sees may hold anything: their
// weights are 0, but 0 * NaN is not, so the softmax warps overwrite them with
// zeros in shared memory before the product (the tiles at the ends only).
//
// Every wait is bounded (2 s; status 5 and the CTA's abort flag).
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
    struct PaItem *items;  // of each CTA: the item that begins in its run and ends in a later one
    float *part;           // two records per CTA
    int *status;
};

// An item whose records are to be joined (np = 0: none).
struct __align__(16) PaItem {
    int np, rows, tok, j;  // parts, rows, first token row, kv head
};

constexpr int PA_ROWS = 128;
constexpr int PA_SOFTMAX = 8;  // softmax warps: two for each 32 rows, each with half of a tile's positions
constexpr int PA_PRODUCER = PA_SOFTMAX, PA_ISSUER = PA_SOFTMAX + 1;
constexpr int PA_THREADS = (PA_SOFTMAX + 2) * 32;
template <bool BF> constexpr float PA_BELOW = BF ? 0.0f : 7.0f;     // m is set this far below the maximum (log2)
template <bool BF> constexpr float PA_SLACK = 8.0f + PA_BELOW<BF>;  // the maximum above m before m follows

template <int HD> struct PaPlan {
    static constexpr int KT = HD == 256 ? 64 : 128;  // positions per key tile
    static constexpr int SLOT = KT * HD * 2;         // bytes of a slot (K or V of a tile)
    static constexpr int SLOTS = 192 * 1024 / SLOT;
    static constexpr int O = 0, Q = HD, S = HD + HD / 2, P = S + KT;  // TMEM columns: O | Q | S | P, P
    static constexpr size_t SMEM = 1024 + (size_t)SLOTS * SLOT + 1024;
    static_assert(P + KT <= 512, "TMEM plan");
    static_assert(SMEM > MMA_SMEM_MIN && SMEM <= MMA_SMEM_LIMIT - 8192, "one CTA per SM");
};

// floats of a partial record: O[d / 4][row][4], then (m, l) of the rows
__host__ __device__ constexpr size_t pa_record(int hd) { return (size_t)PA_ROWS * (hd + 2); }

// ---- tensor core helpers ----

// D[tmem] (+)= A[tmem] B[smem], 16-bit operands, fp32 sums, one thread.
M27B_DI void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
// For a pair: D of both CTAs, A in TMEM or shared memory of each, B half in
// each.  The whole warp comes here and the lane with `lead` issues: operands
// that are the same in all lanes stay in uniform registers, which the
// instruction reads.
M27B_DI void pair_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
                 : "memory");
}
M27B_DI void pair_mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(lead)
                 : "memory");
}
M27B_DI uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
// The MMAs that the lead lane issued for the pair arrive on `bar` of both CTAs when they complete.
M27B_DI void pair_commit(uint32_t lead, uint32_t bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %2, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(bar),
        "h"((uint16_t)3), "r"(lead)
        : "memory");
}
M27B_DI void pair_tmem_alloc(uint32_t *slot) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
M27B_DI void pair_tmem_free(uint32_t tmem) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}
// All threads of the pair.
M27B_DI void pair_barrier() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The address, in the first or second CTA of the pair, of the barrier at this place.
M27B_DI uint32_t pair_bar(uint64_t *bar, int cta) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(bar)), "r"(cta));
    return r;
}
// Copies into this CTA that signal a barrier of either CTA of the pair.
M27B_DI void pair_load_4d(uint32_t dst, const CUtensorMap *tm, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, "
        "%4, %5}], [%6];" ::"r"(dst),
        "l"((unsigned long long)tm), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}
M27B_DI void pair_load_3d(uint32_t dst, const CUtensorMap *tm, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, "
        "%4}], [%5];" ::"r"(dst),
        "l"((unsigned long long)tm), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
// Arrive on the barrier at the same place in the first (or second) CTA of the pair.  What
// these arrivals announce is in TMEM or was written by copies, whose order the
// tcgen05 fences and the copies' own barriers give, so they carry no release
// at cluster scope (some 800 cycles each; zeroed V rows, ordinary stores, get a
// cluster fence of their own).
M27B_DI void pair_arrive(uint64_t *bar, int cta = 0) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(pair_bar(bar, cta)) : "memory");
}
// Matrix descriptor, 128-byte swizzle: 1024 bytes between groups of 8
// 128-byte rows; `lead` bytes between 64-value columns (N-major operands).
M27B_DI uint64_t umma_desc128(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// fp32 accumulator, f16 or bf16 operands, A K-major, B K-major or N-major.
template <bool BF, int M, int N, bool BMN>
constexpr uint32_t umma_idesc_f16() {
    return (1u << 4) | ((BF ? 1u : 0u) << 7) | ((BF ? 1u : 0u) << 10) | ((BMN ? 1u : 0u) << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
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
M27B_DI void tmem_ld16(uint32_t taddr, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
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
    const int cap = a.kv.n_cols * a.kv.page_size, end = a.bt.cu_q[b + 1];
    int len = s.row < 0 ? 0 : a.bt.lens[s.row];
    if (report && s.q_n > 0 && (s.row < 0 || len > cap)) paged_bad(a.status);
    len = max(0, min(len, cap));
    s.row = max(0, s.row);
    s.base = (int)max((long long)-(1 << 30), (long long)len - end + t.x);
    s.nrt = (s.q_n + tq - 1) / tq;
    return s;
}

// Positions [x, y) that some row of the sequence sees; the others may hold anything.
M27B_DI int2 pa_seen(const PaSeq &s, int window) {
    return make_int2(window > 0 ? max(0, s.base - window + 1) : 0, max(0, s.base + s.q_n));
}

// Positions [lo, hi) that row tile r sees, and its key tiles [kt0, kt1).
struct PaSpan {
    int lo, hi, kt0, kt1;
};
// Units of an item: its key tiles, and the time between two items (the pipeline
// drains, O leaves) in tiles.  Without it a worker with many short items runs
// behind: a decode batch of 64 sequences of 300 to 8192 positions ended after
// 103 us on the median CTA and 146 us on the last.  Swept on that batch and
// on a 4096-token chunk: 1, 2, 3, 4, 5, 6, 8 tiles 144, 133, 130, 122, 122, 123,
// 126 us; pairs 4, 6, 8, 10, 12 tiles 430, 430, 434, 435, 468 us.  Both with
// head_dim 256; 64 and 128 and items without tiles are charged the same, not swept.
constexpr int PA_EXTRA = 4, PAIR_EXTRA = 6;
template <int EX>
M27B_DI int pa_units(const PaSpan &s) { return s.kt1 - s.kt0 + EX; }
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
template <int KT, int EX>
M27B_DI long long pa_head_units(const PaSeq &s, int tq, int window) {
    const int lane = threadIdx.x & 31;
    long long u = 0;
    if (s.nrt <= 4)
        for (int r = 0; r < s.nrt; ++r) u += pa_units<EX>(pa_span<KT>(s, r, tq, window));
    for (unsigned big = __ballot_sync(0xffffffffu, s.nrt > 4); big; big &= big - 1) {
        const int src = __ffs(big) - 1;
        PaSeq o;
        o.q_n = __shfl_sync(0xffffffffu, s.q_n, src);
        o.base = __shfl_sync(0xffffffffu, s.base, src);
        o.nrt = __shfl_sync(0xffffffffu, s.nrt, src);
        long long v = 0;
        for (int r = lane; r < o.nrt; r += 32) v += pa_units<EX>(pa_span<KT>(o, r, tq, window));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (lane == src) u = v;
    }
    return u;
}

// A worker's run of units, and where it begins.
struct PaRun {
    long long total, begin, end;
    int workers;          // workers that have a run
    int b, j, r, off;     // first item, and units of it that belong to the workers before
    long long seq_off, head_units;  // the run's begin within sequence b; units of a kv head of it
    PaSeq seq;                      // sequence b
};

// x / y for counts that nearly always fit 32 bits (a 64-bit division is a
// routine of some hundred cycles, and the prologue has several in a row).
M27B_DI long long div_count(long long x, long long y) {
    return (x | y) >> 32 ? x / y : (long long)((unsigned)x / (unsigned)y);
}

// The item at hand, walked alike by every role.
template <int KT, int EX>
struct PaWalk {
    long long u, end;
    int tq, b, j, r, off;
    int take;  // units of this item in this run
    PaSeq s;
    PaSpan sp;

    M27B_DI void begin(const AttnArgs &a, const PaRun &run, int tq_) {
        tq = tq_, u = run.begin, end = run.end, b = run.b, j = run.j, r = run.r, off = run.off;
        s = run.seq;
        if (more()) span(a);
    }
    M27B_DI bool more() const { return u < end; }
    M27B_DI void span(const AttnArgs &a) {
        sp = pa_span<KT>(s, r, tq, a.window);
        take = (int)min((long long)(pa_units<EX>(sp) - off), end - u);
    }
    // key tiles of this item in this run
    M27B_DI int tiles() const { return max(0, off + take - EX) - max(0, off - EX); }
    M27B_DI int first() const { return sp.kt0 + max(0, off - EX); }
    M27B_DI int units() const { return pa_units<EX>(sp); }
    M27B_DI bool whole() const { return off == 0 && take == units(); }
    M27B_DI void next(const AttnArgs &a) {
        u += take;
        off = 0;
        if (!more()) return;
        if (++r == s.nrt) {
            r = 0;
            if (++j == a.kv.n_kv) {
                j = 0;
                do {
                    s = pa_seq(a, ++b, tq, false);
                } while (s.nrt == 0);  // units are left, so a sequence with tokens follows
            }
        }
        span(a);
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
    for (int w = 0; w < (int)blockDim.x / 32; ++w) {
        if (w < warp) before += red[w];
        all += red[w];
    }
    *total = all;
    return before + inc - v;
}

// All threads: fill `run` (shared memory) with the run of worker `me` of at most `most`.
template <int KT, int EX>
M27B_DI void pa_find_run(const AttnArgs &a, int tq, int me, int most, PaRun *run, long long *red) {
    const int n = a.bt.n_seq, nt = blockDim.x;
    long long total = 0, head = 0, u = 0, before = 0, sum;
    PaSeq s;
    for (int b0 = 0; b0 < n; b0 += nt) {
        const int b = b0 + threadIdx.x;
        s = {0, 0, 0, 0, 0};
        if (b < n) s = pa_seq(a, b, tq, blockIdx.x == 0);
        head = pa_head_units<KT, EX>(s, tq, a.window);
        u = head * a.kv.n_kv;
        before = pa_scan(u, red, &sum);
        total += sum;
    }
    const long long n_w = min((long long)most, total);
    const long long begin = me < n_w ? div_count(me * total, n_w) : 0,
                    end = me < n_w ? div_count((me + 1) * total, n_w) : 0;
    if (threadIdx.x == 0) {
        run->total = total, run->workers = (int)n_w, run->begin = begin, run->end = end;
        run->b = n;
    }
    __syncthreads();
    if (begin >= end) return;
    long long at = 0;
    for (int b0 = 0; b0 < n && at <= begin; b0 += nt) {
        const int b = b0 + threadIdx.x;
        if (n > nt) {
            s = {0, 0, 0, 0, 0};
            if (b < n) s = pa_seq(a, b, tq, false);
            head = pa_head_units<KT, EX>(s, tq, a.window);
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
            const int v = r0 + lane < s.nrt ? pa_units<EX>(pa_span<KT>(s, r0 + lane, tq, a.window)) : 0;
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
    uint32_t tmem;
    int abort;
};

// Page id of page p of the sequence for a copy: past the end of the pool (a box
// of zeros) where the item sees nothing of the page.
template <class Walk>
M27B_DI int pa_page(const AttnArgs &a, const Walk &w, const int *ids, int p, int shift) {
    if (p >= a.kv.n_cols || (p << shift) >= w.sp.hi || (p + 1) << shift <= w.sp.lo) return a.kv.n_pages;
    const int id = ids[p];
    if (id >= 0 && id < a.kv.n_pages) return id;
    paged_bad(a.status);
    return a.kv.n_pages;
}

// Bounded waits.  The timer (in 2^20 ns, one register) and the abort flag are
// looked at only after many tests (a test may itself wait a while in
// hardware): what stands between the roles' hand-offs is a test and a branch.
// No function call: the softmax warps hold their scores in registers here.
M27B_DI bool pa_give_up(uint32_t &t0, volatile int *abort, int *status) {
    if (*abort) return true;
    const uint32_t now = (uint32_t)(global_ns() >> 20) | 1u;
    if (t0 == 0) t0 = now;
    if (now - t0 <= (uint32_t)(M27B_WAIT_NS >> 20)) return false;
    *abort = 1;
    if (status) atomicCAS(status, 0, 5);
    return true;
}
M27B_DI bool pa_wait_at(uint32_t bar, uint32_t parity, volatile int *abort, int *status) {
    uint32_t t0 = 0;
    for (unsigned it = 1;; ++it) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((it & 63u) == 0 && pa_give_up(t0, abort, status)) return false;
    }
}
M27B_DI bool pa_wait(uint64_t *bar, uint32_t parity, volatile int *abort, int *status) {
    return pa_wait_at(smem_u32(bar), parity, abort, status);
}
M27B_DI bool pa_warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort, int *status) {
    return __all_sync(0xffffffffu, pa_wait(bar, parity, abort, status)) != 0;
}

// Lanes 4 g + i hold y[j] = element (i, j) of a 4 x 4 matrix of 16-byte
// elements; afterwards element (j, i).
M27B_DI void transpose4(uint4 (&y)[4]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int b = 1; b < 4; b <<= 1)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (!(j & b)) {
                // swap y[j | b] of lanes without bit b and y[j] of lanes with it
                const bool up = lane & b;
                uint4 give = up ? y[j] : y[j | b], got;
                got.x = __shfl_xor_sync(0xffffffffu, give.x, b), got.y = __shfl_xor_sync(0xffffffffu, give.y, b);
                got.z = __shfl_xor_sync(0xffffffffu, give.z, b), got.w = __shfl_xor_sync(0xffffffffu, give.w, b);
                if (up) y[j] = got;
                else y[j | b] = got;
            }
}

// The end of an item in this worker's run: this thread's part of its row's O
// (columns [part HD / PARTS, ..) of TMEM at `o`) to the output, or, if the worker
// has a part of the item only, O, m and l to its record.  `tok`: the first
// token row of the CTA's rows; `any`: there were tiles (else O is 0).  l is 0
// for a row that saw nothing, whose O is not read, and NaN where scores were.
template <int HD, bool BF, int PARTS, class Walk>
M27B_DI void pa_write(const AttnArgs &a, const Walk &w, const PaRun &run, int me, int cta, int tok, int G, int rows, int row,
                      int part, bool any, float m, float l, uint32_t o, PaItem &tail) {
    constexpr int COLS = HD / PARTS;
    const bool live = row < rows, idle = (row & ~31) >= rows;
    const int h = w.j * G + row % G;
    const long long at = tok + row / G;
    if (w.whole()) {
        if (idle) return;
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        const bool nothing = __any_sync(0xffffffffu, l == 0.0f);  // some row's O is not to be read
        // where quadruple row & 3 of 32 columns of rows (row & ~3) .. + 3 goes
        uint16_t *to[4];
        int i = (row & ~3) / G, g = (row & ~3) - i * G;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            to[r] = (row & ~3) + r < rows ? (uint16_t *)a.out + (tok + i) * a.out_stride + (long long)(w.j * G + g) * HD + part * COLS +
                                                8 * (row & 3)
                                          : nullptr;
            if (++g == G) g = 0, ++i;
        }
#pragma unroll 1
        for (int x = 0; x < COLS / 32; ++x) {
            uint32_t v[32];
            if (any) {
                tmem_ld32(o + part * COLS + 32 * x, v);
                tmem_wait_ld();
            }
            if (nothing && l == 0.0f)
#pragma unroll
                for (int e = 0; e < 32; ++e) v[e] = 0u;
            // four quadruples of 16 bits; then lane 4 g + j holds quadruple j of rows
            // 4 g .. 4 g + 3, so that a store has 64 bytes of a row together
            uint4 y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t z[4];
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    z[d] = Half16<BF>::down(__uint_as_float(v[8 * e + 2 * d]) * inv, __uint_as_float(v[8 * e + 2 * d + 1]) * inv);
                y[e] = make_uint4(z[0], z[1], z[2], z[3]);
            }
            transpose4(y);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (to[r]) *(uint4 *)(to[r] + 32 * x) = y[r];
        }
        if (live && a.lse && part == 0)
            a.lse[at * a.n_q + h] = l != 0.0f ? 0.69314718055994530942f * (m + log2f(l)) : -INFINITY;
    } else {
        // the item begins with worker c0 and ends with c1
        const long long U = w.u - w.off;
        const int c0 = (int)div_count((U + 1) * run.workers + run.total - 1, run.total) - 1;
        const int c1 = (int)div_count((U + w.units()) * run.workers + run.total - 1, run.total) - 1;
        if (me == c0) tail = {rows > 0 ? c1 - c0 + 1 : 0, rows, tok, w.j};
        if (idle) return;
        float *rec = a.part + (size_t)(2 * cta + (me == c0 ? 1 : 0)) * pa_record(HD);
#pragma unroll 1
        for (int x = 0; x < COLS / 32; ++x) {
            uint32_t v[32];
            tmem_ld32(o + part * COLS + 32 * x, v);
            tmem_wait_ld();
            if (live)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    __stcg((uint4 *)rec + (size_t)(part * (COLS / 4) + 8 * x + e) * PA_ROWS + row,
                           make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]));
        }
        if (live && part == 0) __stcg((float2 *)(rec + (size_t)PA_ROWS * HD) + row, make_float2(m, l));
    }
    tc_fence_before();
}

template <int HD, bool BF>
__global__ void __launch_bounds__(PA_THREADS, 1)
    k_paged_attn(const AttnArgs a, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv) {
    using L = PaPlan<HD>;
    constexpr int KT = L::KT, NS = L::SLOTS, SLOT = L::SLOT;
    extern __shared__ uint8_t pa_raw[];
    uint8_t *ring = (uint8_t *)(((uintptr_t)pa_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = (uint64_t *)(ring + (size_t)NS * SLOT);
    // full: a slot's copies have landed; empty: its MMAs are done
    uint64_t *full = bars, *empty = full + NS, *qfull = empty + NS, *sfull = qfull + 1, *sfree = sfull + 1,
             *pfull = sfree + 1, *pdone = pfull + 2, *drain = pdone + 2, *pair = drain + 1;
    __shared__ PaShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int me = blockIdx.x, G = a.n_q / a.kv.n_kv, tq = PA_ROWS / G;  // tokens of an item
    volatile int *abort = &sh.abort;

    if (warp == PA_PRODUCER) {
        for (int s = lane; s < 2 * NS; s += 32) mbar_init(&full[s], 1);
        if (lane < 4) mbar_init(&pair[lane], 2);
        if (lane < 2) {
            mbar_init(&pfull[lane], PA_SOFTMAX);
            mbar_init(&pdone[lane], 1);
        }
        if (lane == 0) {
            mbar_init(qfull, PA_SOFTMAX);
            mbar_init(sfull, 1);
            mbar_init(sfree, PA_SOFTMAX);
            mbar_init(drain, 1);
            sh.abort = 0;
        }
        fence_mbar_init();
    }
    if (warp == PA_ISSUER) {
        tmem_alloc(&sh.tmem, 512);
        tmem_relinquish();
    }
    pdl_wait();
    pdl_trigger();
    tc_fence_before();
    pa_find_run<KT, PA_EXTRA>(a, tq, me, gridDim.x, &sh.run, sh.red);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    PaWalk<KT, PA_EXTRA> w;
    w.begin(a, sh.run, tq);

    if (warp == PA_PRODUCER) {
        const int ps = a.kv.page_size, shift = 31 - __clz(ps);
        // lane = box: (64-value column, page of the tile)
        const int rows = min(ps, KT), np = KT / rows, pg = lane % np, ch = lane / np;
        const uint32_t base = smem_u32(ring);
        const uint32_t dst = ch * (KT * 128) + pg * rows * 128;
        int g = 0;
        bool ok = true;
        for (; ok && w.more(); w.next(a)) {
            const int n = w.tiles();
            if (n == 0) continue;
            const int *ids = a.kv.table + (long long)w.s.row * a.kv.n_cols;
            int have = -32, cur = 0;  // lane's page id of page have + lane of the sequence
            // page ids of the tile at x0 (and, in the same fetch, of the one before: its V comes after this K)
            auto page_of = [&](int p) { return __shfl_sync(0xffffffffu, cur, (p - have) & 31); };
            for (int i = 0; ok && i <= n; ++i) {
                if (i < n) {
                    const int x0 = (w.first() + i) * KT, plast = (x0 + KT - 1) >> shift;
                    if (plast >= have + 32) {
                        have = max(0, x0 - KT) >> shift;
                        cur = pa_page(a, w, ids, have + lane, shift);
                    }
                    const int s = g % NS, page = page_of((x0 >> shift) + pg);
                    if (g >= NS && !(ok = pa_warp_wait(&empty[s], (uint32_t)((g / NS - 1) & 1), abort, a.status))) break;
                    if (lane == 0) mbar_arrive_expect_tx(&full[s], SLOT);
                    __syncwarp();
                    if (ch < HD / 64) tma_load_4d(base + s * SLOT + dst, &tmk, ch * 64, x0 & (ps - 1), w.j, page, &full[s]);
                    ++g;
                }
                if (i > 0) {
                    const int x0 = (w.first() + i - 1) * KT, s = g % NS, page = page_of((x0 >> shift) + pg);
                    if (g >= NS && !(ok = pa_warp_wait(&empty[s], (uint32_t)((g / NS - 1) & 1), abort, a.status))) break;
                    if (lane == 0) mbar_arrive_expect_tx(&full[s], SLOT);
                    __syncwarp();
                    if (ch < HD / 64) tma_load_4d(base + s * SLOT + dst, &tmv, ch * 64, x0 & (ps - 1), w.j, page, &full[s]);
                    ++g;
                }
            }
        }
        // every copy lands before the CTA's shared memory is released (bounded)
        for (int i = max(0, g - NS); i < g; ++i) mbar_wait_bounded(&full[i % NS], (uint32_t)((i / NS) & 1), a.status, 5);
    } else if (warp == PA_ISSUER) {
        if (lane == 0) {
            constexpr uint32_t id_s = umma_idesc_f16<BF, 128, KT, false>(), id_o = umma_idesc_f16<BF, 128, HD, true>();
            const uint32_t base = smem_u32(ring);
            int t0 = 0, g = 0, item = 0;
            bool ok = true;
            auto landed = [&](int g) { return pa_wait(&full[g % NS], (uint32_t)((g / NS) & 1), abort, a.status); };
            for (; ok && w.more(); w.next(a)) {
                const int n = w.tiles();
                if (n == 0) continue;
                // S of tile t = Q K^T, once S has been read and the keys are there
                auto scores = [&](int t) {
                    if (t > 0 && !pa_wait(sfree, (uint32_t)((t - 1) & 1), abort, a.status)) return false;
                    if (!landed(g)) return false;
                    tc_fence_after();
                    const uint32_t k = base + (g % NS) * SLOT;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; ++kk)
                        umma_f16_ts(tmem + L::S, tmem + L::Q + kk * 8,
                                           umma_desc128(k + (kk / 4) * (KT * 128) + (kk % 4) * 32, 16), id_s, kk > 0);
                    umma_commit(sfull);
                    umma_commit(&empty[g % NS]);
                    ++g;
                    return true;
                };
                ok = pa_wait(qfull, (uint32_t)(item & 1), abort, a.status);
                tc_fence_after();
                ok = ok && scores(t0) && (n < 2 || scores(t0 + 1));
                for (int i = 0; ok && i < n; ++i) {
                    const int t = t0 + i;
                    if (!(ok = pa_wait(&pfull[t & 1], (uint32_t)((t >> 1) & 1), abort, a.status) && landed(g))) break;
                    tc_fence_after();
                    const uint32_t v = base + (g % NS) * SLOT;
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk)
                        umma_f16_ts(tmem + L::O, tmem + L::P + (t & 1) * (KT / 2) + kk * 8,
                                           umma_desc128(v + kk * 2048, KT * 128), id_o, i > 0 || kk > 0);
                    umma_commit(&empty[g % NS]);
                    umma_commit(&pdone[t & 1]);
                    ++g;
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
        int t = 0, g0 = 0, told = 0;
        bool ok = true;
        PaItem tail = {0, 0, 0, 0};
        // this row's value of the other half
        auto other = [&](float mine, float &theirs) {
            const int turn = told++ & 1;
            sh.half[turn][half][row] = mine;
            __syncwarp();
            if (lane == 0) mbar_arrive(&pair[quarter]);
            const bool here = pa_warp_wait(&pair[quarter], (uint32_t)turn, abort, a.status);
            theirs = *(volatile float *)&sh.half[turn][half ^ 1][row];
            return here;
        };
        // half of the row's Q of an item into TMEM
        auto load_q = [&](const PaWalk<KT, PA_EXTRA> &x) {
            const int i = x.r * tq + row / G;
            const bool live = row < tq * G && i < x.s.q_n;
            const uint16_t *qp = (const uint16_t *)a.q + (long long)(x.s.q_lo + i) * a.q_stride + (long long)(x.j * G + row % G) * HD +
                                 half * (HD / 2);
#pragma unroll
            for (int y = 0; y < HD / 64; ++y) {
                uint32_t v[16];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint4 z = live ? *((const uint4 *)(qp + 32 * y) + e) : make_uint4(0, 0, 0, 0);
                    v[4 * e] = z.x, v[4 * e + 1] = z.y, v[4 * e + 2] = z.z, v[4 * e + 3] = z.w;
                }
                tmem_st16(lane_base + L::Q + half * (HD / 4) + 16 * y, v);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(qfull);
        };
        if (w.more() && w.tiles() > 0) load_q(w);
        while (ok && w.more()) {
            const int2 seen = pa_seen(w.s, a.window);
            const int n = w.tiles(), i0 = w.r * tq, i = i0 + row / G, h = w.j * G + row % G;
            const int rows = min(tq, w.s.q_n - i0) * G;
            const bool live = row < rows, idle = 32 * quarter >= rows;  // idle: no row of this warp is live
            // a dead row's scores are garbage that no one reads
            const int hi = live ? w.s.base + i + 1 : 0x7fffffff;
            const int lo = live && a.window > 0 ? max(0, hi - a.window) : 0;
            float m = -INFINITY, l = 0.0f;  // m in units of c s
            for (int k = 0; k < n; ++k, ++t) {
                const int x0 = (w.first() + k) * KT;
                if (!(ok = pa_warp_wait(sfull, (uint32_t)(t & 1), abort, a.status))) break;
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
                        const uint32_t off = (uint32_t)(xh - lo), len = (uint32_t)max(0, hi - lo);
#pragma unroll
                        for (int x = 0; x < KH; ++x)
                            if (off + x >= len) s[x] = -INFINITY;
                    }
                    float tops[4] = {s[0], s[1], s[2], s[3]}, theirs;
#pragma unroll
                    for (int x = 4; x < KH; ++x) tops[x & 3] = fmaxf(tops[x & 3], s[x]);
                    const float mine = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    if (!(ok = other(mine, theirs))) break;
                    const float top = c * fmaxf(mine, theirs);
                    if (__any_sync(0xffffffffu, top > m + PA_SLACK<BF>)) {
                        const float to = top > m + PA_SLACK<BF> ? top - PA_BELOW<BF> : m;
                        const float f = m == -INFINITY ? 1.0f : ex2(m - to);
                        m = to;
                        l *= f;
                        if (k > 0) {
                            // this half's columns of O, once the products so far are done
                            if (!(ok = pa_warp_wait(&pdone[(t - 1) & 1], (uint32_t)(((t - 1) >> 1) & 1), abort, a.status)))
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
                    if (t >= 2 && !(ok = pa_warp_wait(&pdone[t & 1], (uint32_t)(((t - 2) >> 1) & 1), abort, a.status))) break;
                    const uint32_t pc = lane_base + L::P + (t & 1) * (KT / 2) + half * (KH / 2);
                    if constexpr (KH == 64) tmem_st32(pc, p);
                    else tmem_st16(pc, p);
                }
                // values of positions that no row of the sequence sees
                if (x0 < seen.x || x0 + KT > seen.y) {
                    const int g = g0 + (k == n - 1 ? 2 * n - 1 : 2 * k + 2);  // V's slot: K0 K1 V0 K2 V1 ...
                    if (!(ok = pa_warp_wait(&full[g % NS], (uint32_t)((g / NS) & 1), abort, a.status))) break;
                    uint8_t *v = ring + (size_t)(g % NS) * SLOT;
                    for (int e = tid; e < SLOT / 16; e += 32 * PA_SOFTMAX) {
                        const int x = (e >> 3) % KT;
                        if (x0 + x < seen.x || x0 + x >= seen.y) *(uint4 *)(v + (size_t)e * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&pfull[t & 1]);
            }
            if (!ok) break;
            g0 += 2 * n;
            // the next item's Q, while the last product here runs: the products
            // with this one are done, since their scores have been read
            PaWalk<KT, PA_EXTRA> next = w;
            next.next(a);
            if (next.more() && next.tiles() > 0) load_q(next);
            if (n > 0) {
                if (!(ok = pa_warp_wait(&pdone[(t - 1) & 1], (uint32_t)(((t - 1) >> 1) & 1), abort, a.status))) break;
                tc_fence_after();
            }
            if (!idle) {
                float theirs;
                if (!(ok = other(l, theirs))) break;
                l = half ? theirs + l : l + theirs;
            }
            pa_write<HD, BF, 2>(a, w, sh.run, me, blockIdx.x, w.s.q_lo + i0, G, rows, row, half, n > 0, m, l, lane_base + L::O, tail);
            w = next;
        }
        if (tid == 0) a.items[blockIdx.x] = tail;
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == PA_ISSUER) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- two CTAs a worker ----

template <int HD> struct PairPlan {
    static constexpr int KT = 128;                   // positions per key tile
    static constexpr int KR = KT / 2, VC = HD / 2;   // positions of K, columns of V in a CTA's slot
    static constexpr int SLOT = KR * HD * 2;
    static_assert(SLOT == KT * VC * 2, "slots");
    static constexpr int Q_BYTES = PA_ROWS * HD * 2;
    static constexpr int SLOTS = (192 * 1024 - Q_BYTES) / SLOT;
    static constexpr int NB = HD == 256 ? 1 : 2;     // buffers of S
    static constexpr int AHEAD = 2;                  // products Q K issued ahead of P V
    static constexpr int O = 0, S = HD, P = S + NB * KT;  // TMEM columns: O | S (, S) | P, P
    static constexpr size_t SMEM = 1024 + Q_BYTES + (size_t)SLOTS * SLOT + 1024;
    static_assert(P + KT <= 512, "TMEM plan");
    static_assert(SMEM > MMA_SMEM_MIN && SMEM <= MMA_SMEM_LIMIT - 8192, "one CTA per SM");
};
// Warps 0-7: softmax, a row per thread, warps 0-3 the even tiles and 4-7 the odd
// ones.  Registers: they hold a row of a tile; 2 x 128 threads of 216 and 128 of
// 72 are the 384 x 168 that the block is launched with.
constexpr int PAIR_SOFTMAX = 8;
constexpr int PAIR_PRODUCER = PAIR_SOFTMAX, PAIR_ISSUER = PAIR_SOFTMAX + 1;
constexpr int PAIR_THREADS = (PAIR_SOFTMAX + 4) * 32;
constexpr int PAIR_REGS_SOFTMAX = 216, PAIR_REGS_OTHER = 72;
static_assert(2 * PAIR_REGS_SOFTMAX + PAIR_REGS_OTHER <= 3 * 168, "register split");

template <int HD> struct PairShared {
    PaRun run;
    PaWalk<PairPlan<HD>::KT, PAIR_EXTRA> walk[PAIR_SOFTMAX][2];  // of each softmax warp: the item at hand and the next
    PaItem tail[PAIR_SOFTMAX];
    AttnArgs args;
    long long red[PAIR_THREADS / 32];
    uint64_t m[2][PA_ROWS];     // a row's m after a tile, by turns; above it the tile's number + 1
    float half[2][2][PA_ROWS];  // what the two warps of a row tell each other at an item's end
    uint32_t tmem;
    int abort;
};

// Two values at once (packed fp32 arithmetic).
M27B_DI uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
M27B_DI float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
M27B_DI uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
M27B_DI uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
M27B_DI float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The m that another warp stores with number `tag` (bounded, for a whole warp).
M27B_DI bool pair_follow(const uint64_t *p, uint32_t tag, float &m, volatile int *abort, int *status) {
    uint64_t v;
    const uint32_t at = smem_u32(p);
    uint32_t t0 = 0;
    bool here = true;
    for (unsigned it = 1;; ++it) {
        asm volatile("ld.volatile.shared.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
        if ((uint32_t)(v >> 32) == tag) break;
        if ((it & 255u) == 0 && pa_give_up(t0, abort, status)) {
            here = false;
            break;
        }
    }
    m = __uint_as_float((uint32_t)v);
    return __all_sync(0xffffffffu, here) != 0;
}

// pa_write for a pair's thread, out of line: inlined, its state costs the tile
// loop 100 spilled registers a tile.
template <int HD, bool BF>
__device__ __noinline__ void pair_write(const AttnArgs &a, const PaWalk<PairPlan<HD>::KT, PAIR_EXTRA> &w, const PaRun &run, int tok, int rows,
                                        bool any, float m, float l, uint32_t o, PaItem *tail) {
    const int warp = threadIdx.x >> 5, row = 32 * (warp & 3) + (threadIdx.x & 31);
    PaItem t = *tail;
    __syncwarp();
    pa_write<HD, BF, 2>(a, w, run, blockIdx.x >> 1, blockIdx.x, tok, a.n_q / a.kv.n_kv, rows, row, warp >> 2, any, m, l, o, t);
    if ((threadIdx.x & 31) == 0) *tail = t;
}

template <int HD, bool BF>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    k_paged_attn_pair(const AttnArgs a, const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                      const __grid_constant__ CUtensorMap tmq) {
    using L = PairPlan<HD>;
    constexpr int KT = L::KT, NS = L::SLOTS, SLOT = L::SLOT, NB = L::NB, AHEAD = L::AHEAD;
    extern __shared__ uint8_t pa_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)pa_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = smem + L::Q_BYTES;
    uint64_t *bars = (uint64_t *)(ring + (size_t)NS * SLOT);
    // full: a slot's copies have landed (in the first CTA, for those of both);
    // empty: its MMAs are done; sfull, pdone, odone, empty, qempty come to both
    // CTAs; sfree, pfull, oread are the first CTA's, for the warps of both; vlanded
    // tells the second CTA's softmax warps that a tile's V is there; odone has a
    // phase an item
    uint64_t *full = bars, *empty = full + NS, *qfull = empty + NS, *qempty = qfull + 1, *vlanded = qempty + 1, *sfull = vlanded + 2, *sfree = sfull + 2, *pfull = sfree + 2, *pdone = pfull + 2,
             *oread = pdone + 2, *odone = oread + 1, *drain = odone + 1, *pair = drain + 1;
    __shared__ PairShared<HD> sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = blockIdx.x & 1, me = blockIdx.x >> 1;
    const int G = a.n_q / a.kv.n_kv, tq = PA_ROWS / G, tqw = 2 * tq;  // tokens of a CTA's rows, of an item
    volatile int *abort = &sh.abort;

    if (warp == PAIR_PRODUCER) {
        for (int s = lane; s < 2 * NS; s += 32) mbar_init(&full[s], 1);
        if (lane < 4) mbar_init(&pair[lane], 2);
        if (lane < 2) {
            mbar_init(&sfull[lane], 1);
            mbar_init(&vlanded[lane], 1);
            mbar_init(&sfree[lane], PAIR_SOFTMAX);
            mbar_init(&pfull[lane], PAIR_SOFTMAX);
            mbar_init(&pdone[lane], 1);
        }
        if (lane == 0) {
            mbar_init(qfull, 1);
            mbar_init(qempty, 1);
            mbar_init(oread, 2 * PAIR_SOFTMAX);
            mbar_init(odone, 1);
            mbar_init(drain, 1);
            sh.abort = 0;
        }
        fence_mbar_init();
    }
    if (warp == PAIR_ISSUER) pair_tmem_alloc(&sh.tmem);
    if (tid == 0) sh.args = a;
    if (tid < 2 * PA_ROWS) sh.m[tid >> 7][tid & 127] = 0;
    pdl_wait();
    pdl_trigger();
    tc_fence_before();
    pa_find_run<KT, PAIR_EXTRA>(a, tqw, me, gridDim.x >> 1, &sh.run, sh.red);
    pair_barrier();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    auto fewer_registers = [] { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PAIR_REGS_OTHER)); };

    if (warp == PAIR_PRODUCER) {
        fewer_registers();
        PaWalk<KT, PAIR_EXTRA> w;
        w.begin(a, sh.run, tqw);
        const int ps = a.kv.page_size, shift = 31 - __clz(ps);
        // lane = box: (64-value column, page) of a K slot or a V slot
        const int krows = min(ps, L::KR), knp = L::KR / krows, vrows = min(ps, KT), vnp = KT / vrows;
        const int kpg = lane % knp, kch = lane / knp, vpg = lane % vnp, vch = lane / vnp;
        const uint32_t base = smem_u32(ring);
        const uint32_t kdst = kch * (L::KR * 128) + kpg * krows * 128, vdst = vch * (KT * 128) + vpg * vrows * 128;
        int g = 0, item = 0;
        bool ok = true;
        for (; ok && w.more(); w.next(a)) {
            const int n = w.tiles();
            if (n == 0) continue;
            const int *ids = a.kv.table + (long long)w.s.row * a.kv.n_cols;
            int have = -32, cur = 0;  // lane's page id of page have + lane of the sequence
            auto page_of = [&](int p) { return __shfl_sync(0xffffffffu, cur, (p - have) & 31); };
            for (int i = 0; ok && i < n + AHEAD; ++i) {
                if (i < n) {
                    const int x0 = (w.first() + i) * KT, plast = (x0 + KT - 1) >> shift;
                    if (plast >= have + 32) {
                        // from AHEAD tiles before on: that V comes after this K
                        have = max(0, x0 - AHEAD * KT) >> shift;
                        cur = pa_page(a, w, ids, have + lane, shift);
                    }
                    const int s = g % NS, xk = x0 + rank * L::KR, page = page_of((xk >> shift) + kpg);
                    if (g >= NS && !(ok = pa_warp_wait(&empty[s], (uint32_t)((g / NS - 1) & 1), abort, a.status))) break;
                    if (lane == 0 && rank == 0) mbar_arrive_expect_tx(&full[s], 2 * SLOT);
                    if (kch < HD / 64)
                        pair_load_4d(base + s * SLOT + kdst, &tmk, kch * 64, xk & (ps - 1), w.j, page, pair_bar(&full[s], 0));
                    ++g;
                }
                if (i == 0) {
                    // Q, once the last product with the item's before is done
                    if (item > 0 && !(ok = pa_warp_wait(qempty, (uint32_t)((item - 1) & 1), abort, a.status))) break;
                    if (lane == 0 && rank == 0) mbar_arrive_expect_tx(qfull, 2 * (HD / 64) * G * tq * 128);
                    if (lane < HD / 64)
                        pair_load_3d(smem_u32(smem) + lane * (PA_ROWS * 128), &tmq, lane * 64, w.j * G,
                                     w.s.q_lo + w.r * tqw + rank * tq, pair_bar(qfull, 0));
                    ++item;
                }
                if (i >= AHEAD) {
                    const int x0 = (w.first() + i - AHEAD) * KT, s = g % NS, page = page_of((x0 >> shift) + vpg);
                    if (g >= NS && !(ok = pa_warp_wait(&empty[s], (uint32_t)((g / NS - 1) & 1), abort, a.status))) break;
                    if (lane == 0 && rank == 0) mbar_arrive_expect_tx(&full[s], 2 * SLOT);
                    if (vch < L::VC / 64)
                        pair_load_4d(base + s * SLOT + vdst, &tmv, rank * L::VC + vch * 64, x0 & (ps - 1), w.j, page,
                                     pair_bar(&full[s], 0));
                    ++g;
                }
            }
        }
        // every copy lands before the pair's shared memory is released (bounded)
        if (rank == 0) {
            if (item > 0) mbar_wait_bounded(qfull, (uint32_t)((item - 1) & 1), a.status, 5);
            for (int i = max(0, g - NS); i < g; ++i) mbar_wait_bounded(&full[i % NS], (uint32_t)((i / NS) & 1), a.status, 5);
        }
    } else if (warp == PAIR_ISSUER) {
        fewer_registers();
        if (rank == 0) {
            // The warp stays together and one lane issues; its code is kept
            // small: what it does between two products is time the tensor
            // cores wait.
            constexpr uint32_t id_s = umma_idesc_f16<BF, 256, KT, false>(), id_o = umma_idesc_f16<BF, 256, HD, true>();
            const uint32_t lead = elect_one(), tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t kdesc = umma_desc128(smem_u32(ring), 16), vdesc = umma_desc128(smem_u32(ring), KT * 128),
                           qdesc = umma_desc128(smem_u32(smem), 16);
            const uint32_t full0 = smem_u32(full), empty0 = smem_u32(empty), sfull0 = smem_u32(sfull), sfree0 = smem_u32(sfree),
                           pfull0 = smem_u32(pfull), pdone0 = smem_u32(pdone);
            PaWalk<KT, PAIR_EXTRA> w;
            w.begin(a, sh.run, tqw);
            uint32_t t = 0, slot = 0, phase = 0, item = 0;  // t: tile of the next scores; phase: of the slot
            bool ok = true;
            auto used = [&] {
                pair_commit(lead, empty0 + 8 * slot);
                if (++slot == NS) slot = 0, phase ^= 1;
            };
            auto wait = [&](uint32_t bar, uint32_t parity) {
                return ok = __all_sync(0xffffffffu, pa_wait_at(bar, parity, abort, a.status)) != 0;
            };
            for (; ok && w.more(); w.next(a)) {
                const int n = __shfl_sync(0xffffffffu, w.tiles(), 0);
                if (n == 0) continue;
                if (!wait(smem_u32(qfull), item & 1)) break;
                // Q K runs ahead of P V, which waits for the softmax
                for (int i = 0; i < n + AHEAD; ++i) {
                    if (i < n) {
                        // S of tile t, once its buffer has been read and the keys are there
                        const uint32_t u = t - NB;
                        if (t >= NB && !wait(sfree0 + 8 * (u & 1), (u >> 1) & 1)) break;
                        if (!wait(full0 + 8 * slot, phase)) break;
                        tc_fence_after();
                        uint64_t kd = kdesc + (uint64_t)(slot * (SLOT / 16)), qd = qdesc;
                        const uint32_t d = tm + L::S + (NB == 2 ? (t & 1) * KT : 0);
#pragma unroll 1
                        for (int ch = 0; ch < HD / 64; ++ch, kd += L::KR * 128 / 16, qd += PA_ROWS * 128 / 16)
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) pair_mma_ss(lead, d, qd + 2 * kk, kd + 2 * kk, id_s, ch > 0 || kk > 0);
                        pair_commit(lead, sfull0 + 8 * (t & 1));
                        used();
                        if (i + 1 == n) pair_commit(lead, smem_u32(qempty));
                        ++t;
                    }
                    if (i < AHEAD) continue;
                    const uint32_t v = t - 1 - (i < n ? AHEAD : n + AHEAD - 1 - i);
                    if (!wait(pfull0 + 8 * (v & 1), (v >> 1) & 1)) break;
                    if (!wait(full0 + 8 * slot, phase)) break;
                    // O of the item before has been read
                    if (i == AHEAD && item > 0 && !wait(smem_u32(oread), (item - 1) & 1)) break;
                    tc_fence_after();
                    uint64_t vd = vdesc + (uint64_t)(slot * (SLOT / 16));
                    uint32_t pc = tm + L::P + (v & 1) * (KT / 2);
#pragma unroll 1
                    for (int half = 0; half < 2; ++half, vd += 4 * 128, pc += 32)
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            pair_mma_ts(lead, tm + L::O, pc + 8 * kk, vd + 128 * kk, id_o, i > AHEAD || half > 0 || kk > 0);
                    used();
                    pair_commit(lead, pdone0 + 8 * (v & 1));
                }
                if (ok) pair_commit(lead, smem_u32(odone));
                ++item;
            }
            // every MMA issued above (bounded, even after an abort)
            pair_commit(lead, smem_u32(drain));
        }
        // (the second CTA: the first one's last arrival here)
        mbar_wait_bounded(drain, 0u, a.status, 5);
        __syncwarp();
    } else if (warp >= PAIR_SOFTMAX) {
        fewer_registers();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PAIR_REGS_SOFTMAX));
        // row = TMEM lane; warps 0-3 take the even tiles, warps 4-7 the odd ones
        const int quarter = warp & 3, wg = warp >> 2, row = 32 * quarter + lane;
        const uint32_t lane_base = tmem + ((uint32_t)(32 * quarter) << 16);
        const float c = a.scale * 1.44269504088896340736f;  // log2 e
        int t0 = 0, u0 = 0, told = 0, zeroed = 0;  // u0: tiles of this quarter so far (of items where it has live rows)
        uint32_t ended = 0;                        // parity of odone's phase
        bool ok = true;
        if (lane == 0) sh.tail[warp] = PaItem{0, 0, 0, 0};
        // m after tile u of this quarter, from the warp that has the tile to the
        // other: one 64-bit word with its tile's number (two words of a vector access
        // have no order), so that no barrier is needed
        auto publish = [&](int u, float m) {
            const uint64_t v = (uint64_t)((uint32_t)u + 1) << 32 | __float_as_uint(m);
            asm volatile("st.volatile.shared.u64 [%0], %1;" ::"r"(smem_u32(&sh.m[u & 1][row])), "l"(v) : "memory");
        };
        auto follow = [&](int u, float &m) { return pair_follow(&sh.m[u & 1][row], (uint32_t)u + 1, m, abort, a.status); };
        // arrivals that both CTAs' warps make in the first
        auto arrive = [&](uint64_t *bar) {
            if (rank == 0) mbar_arrive(bar);
            else pair_arrive(bar);
        };
        // the walk's state is in shared memory, for registers' sake
        const int row_tok = row / G;
        int cur = 0;
        if (lane == 0) sh.walk[warp][0].begin(a, sh.run, tqw);
        __syncwarp();
        while (ok && sh.walk[warp][cur].more()) {
            const PaWalk<KT, PAIR_EXTRA> &w = sh.walk[warp][cur];
            const int n = w.tiles(), x_first = w.first() * KT;
            const int2 seen = pa_seen(w.s, a.window);
            const int i0 = w.r * tqw + rank * tq, rows = max(0, min(tq, w.s.q_n - i0)) * G;
            const bool live = row < rows, idle = 32 * quarter >= rows;  // idle: no row of this warp is live
            // a dead row's scores are garbage that no one reads
            const int hi = live ? w.s.base + i0 + row_tok + 1 : 0x7fffffff;
            const int lo = live && a.window > 0 ? max(0, hi - a.window) : 0;
            float m = -INFINITY, l = 0.0f;  // m in units of c s; l of this warp's tiles
            for (int k = (wg ^ t0) & 1; k < n; k += 2) {
                const int t = t0 + k, x0 = x_first + k * KT;
                if (!(ok = pa_warp_wait(&sfull[wg], (uint32_t)((t >> 1) & 1), abort, a.status))) break;
                if (idle) {
                    if (lane == 0) arrive(&sfree[wg]);
                    // as the others before they write P: the scores of t come before
                    // the product of t - 2 has its P, and an arrival for t must not
                    // be taken for one for t - 2
                    if (t >= 2 && !(ok = pa_warp_wait(&pdone[wg], (uint32_t)(((t - 2) >> 1) & 1), abort, a.status))) break;
                } else {
                    tc_fence_after();
                    float s[KT];
#pragma unroll
                    for (int x = 0; x < KT / 32; ++x) tmem_ld32(lane_base + L::S + (NB == 2 ? wg * KT : 0) + 32 * x, (uint32_t *)s + 32 * x);
                    tmem_wait_ld();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive(&sfree[wg]);
                    if (__any_sync(0xffffffffu, x0 < lo || x0 + KT > hi)) {
                        const uint32_t off = (uint32_t)(x0 - lo), len = (uint32_t)max(0, hi - lo);
#pragma unroll
                        for (int x = 0; x < KT; ++x)
                            if (off + x >= len) s[x] = -INFINITY;
                    }
                    float tops[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int x = 4; x < KT; x += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            tops[e] = x + 4 + e < KT ? max3(tops[e], s[x + e], s[x + 4 + e]) : fmaxf(tops[e], s[x + e]);
                    const float top = c * fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
                    // the other warps' m after the tile before, and ours
                    float before = -INFINITY;
                    if (k > 0 && !(ok = follow(u0 + k - 1, before))) break;
                    const float now = top > before + PA_SLACK<BF> ? top - PA_BELOW<BF> : before;
                    publish(u0 + k, now);
                    if (m != now) {
                        l *= m == -INFINITY ? 0.0f : ex2(m - now);
                        m = now;
                    }
                    if (k > 0 && __any_sync(0xffffffffu, now != before)) {
                        // O, once the products so far are done
                        if (!(ok = pa_warp_wait(&pdone[wg ^ 1], (uint32_t)(((t - 1) >> 1) & 1), abort, a.status))) break;
                        tc_fence_after();
                        const float f = before == -INFINITY ? 1.0f : ex2(before - now);
#pragma unroll 1
                        for (int x = 0; x < HD / 16; ++x) {
                            uint32_t v[16];
                            tmem_ld16(lane_base + L::O + 16 * x, v);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * f);
                            tmem_st16(lane_base + L::O + 16 * x, v);
                        }
                        tmem_wait_st();
                    }
                    const float mm = m == -INFINITY ? 0.0f : m;
                    const uint64_t c2 = pack2(c, c), m2 = pack2(-mm, -mm);
                    uint64_t sum[2] = {0, 0};
                    // P's buffer is free once the product of two tiles ago is done
                    if (t >= 2 && !(ok = pa_warp_wait(&pdone[wg], (uint32_t)(((t - 2) >> 1) & 1), abort, a.status))) break;
#pragma unroll
                    for (int x = 0; x < KT / 64; ++x) {
                        uint32_t p[32];
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float2 y = unpack2(fma2(pack2(s[64 * x + 2 * e], s[64 * x + 2 * e + 1]), c2, m2));
                            const float p0 = ex2(y.x), p1 = ex2(y.y);
                            sum[e & 1] = add2(sum[e & 1], pack2(p0, p1));
                            p[e] = Half16<BF>::down(p0, p1);
                        }
                        tmem_st32(lane_base + L::P + wg * (KT / 2) + 32 * x, p);
                    }
                    const float2 both = unpack2(add2(sum[0], sum[1]));
                    l += both.x + both.y;
                }
                // values of positions that no row of the sequence sees
                if (x0 < seen.x || x0 + KT > seen.y) {
                    const int g = 2 * t0 + min(n, k + 1 + AHEAD) + k;  // V's slot: after K of AHEAD tiles more
                    // the first CTA sees the copies of both land, and tells the
                    // second; not before tile t - 2 is done with in both, so
                    // that what it tells is not overtaken
                    if (t >= 2 && !(ok = pa_warp_wait(&pdone[wg], (uint32_t)(((t - 2) >> 1) & 1), abort, a.status))) break;
                    if (rank == 0) {
                        if (!(ok = pa_warp_wait(&full[g % NS], (uint32_t)((g / NS) & 1), abort, a.status))) break;
                        if (quarter == 0 && lane == 0) pair_arrive(&vlanded[wg], 1);
                    } else if (!(ok = pa_warp_wait(&vlanded[wg], (uint32_t)(zeroed++ & 1), abort, a.status))) break;
                    uint8_t *v = ring + (size_t)(g % NS) * SLOT;
                    for (int e = tid & 127; e < SLOT / 16; e += 128) {
                        const int x = (e >> 3) % KT;
                        if (x0 + x < seen.x || x0 + x >= seen.y) *(uint4 *)(v + (size_t)e * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async();
                    if (rank == 1) asm volatile("fence.acq_rel.cluster;" ::: "memory");
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive(&pfull[wg]);
            }
            if (!ok) break;
            if (lane == 0) {
                // the next item, while the last product runs
                sh.walk[warp][cur ^ 1] = w;
                sh.walk[warp][cur ^ 1].next(a);
            }
            if (n > 0) {
                // The item's products.  Not pdone of the last tile: the group that
                // does not own it may know pdone of four tiles ago only, and the
                // parity of a phase two early passes at once; an idle warp would
                // then arrive on oread while the item before is still being read.
                if (!(ok = pa_warp_wait(odone, ended, abort, a.status))) break;
                ended ^= 1u;
                tc_fence_after();
                if (!idle) {
                    const int last = t0 + n - 1;
                    // m of the last tile, and the other warp's sum under it
                    float end = m, theirs;
                    if ((last & 1) != wg && !(ok = follow(u0 + n - 1, end))) break;
                    l *= m == end ? 1.0f : m == -INFINITY ? 0.0f : ex2(m - end);
                    m = end;
                    const int turn = told++ & 1;
                    sh.half[turn][wg][row] = l;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&pair[quarter]);
                    if (!(ok = pa_warp_wait(&pair[quarter], (uint32_t)turn, abort, a.status))) break;
                    theirs = *(volatile float *)&sh.half[turn][wg ^ 1][row];
                    l = wg ? theirs + l : l + theirs;
                    u0 += n;
                }
            }
            pair_write<HD, BF>(sh.args, w, sh.run, w.s.q_lo + i0, rows, n > 0, m, l, lane_base + L::O, &sh.tail[warp]);
            if (n > 0) {
                __syncwarp();
                if (lane == 0) arrive(oread);
            }
            t0 += n;
            __syncwarp();
            cur ^= 1;
        }
        if (tid == 0) a.items[blockIdx.x] = sh.tail[0];
    }
    __syncwarp();
    tc_fence_before();
    pair_barrier();
    if (warp == PAIR_ISSUER) {
        __syncwarp();
        tc_fence_after();
        pair_tmem_free(tmem);
    }
}

constexpr int JOIN_THREADS = 128;

// Add up the records of item blockIdx.x (the tail of that CTA's run, if it has
// one) and write its rows.  A group of SP threads takes eight values of a row;
// thread p has parts p, p + SP, ..., four in flight, and the group adds its
// sums up, all in an order that the sizes fix.
template <int HD, bool BF, int SP>
M27B_DI void pa_join(const AttnArgs &a, const PaItem &it, int stride) {
    const int G = a.n_q / a.kv.n_kv, p = threadIdx.x % SP;
    const int first = blockIdx.x;
    auto record = [&](int x) { return a.part + (size_t)(2 * (first + stride * x) + (x == 0 ? 1 : 0)) * pa_record(HD); };
    const int n = it.rows * (HD / 8), per = JOIN_THREADS / SP;
    for (int e0 = blockIdx.y * per; e0 < n; e0 += gridDim.y * per) {
        const int e = min(n - 1, e0 + (int)threadIdx.x / SP), d8 = e / it.rows, row = e - d8 * it.rows;
        float m = -INFINITY, l = 0.0f, o[8] = {};
        for (int x0 = p; x0 < it.np; x0 += 4 * SP) {
            float2 ml[4];
            float4 y[4][2];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int x = x0 + q * SP;
                const bool in = x < it.np;
                const float *r = record(x);
                ml[q] = in ? __ldcg((const float2 *)(r + (size_t)PA_ROWS * HD) + row) : make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int v = 0; v < 2; ++v)
                    y[q][v] = in ? __ldcg((const float4 *)r + (size_t)(2 * d8 + v) * PA_ROWS + row) : make_float4(0, 0, 0, 0);
            }
            const float mn = fmaxf(m, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)));
            const float ref = mn == -INFINITY ? 0.0f : mn, f0 = ex2(m - ref);
            m = mn;
            l *= f0;
#pragma unroll
            for (int v = 0; v < 8; ++v) o[v] *= f0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (ml[q].y == 0.0f) continue;  // the part saw nothing (its O may be anything)
                const float f = ex2(ml[q].x - ref);
                l = fmaf(f, ml[q].y, l);
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    o[4 * v] = fmaf(f, y[q][v].x, o[4 * v]), o[4 * v + 1] = fmaf(f, y[q][v].y, o[4 * v + 1]);
                    o[4 * v + 2] = fmaf(f, y[q][v].z, o[4 * v + 2]), o[4 * v + 3] = fmaf(f, y[q][v].w, o[4 * v + 3]);
                }
            }
        }
        float mx = m;
#pragma unroll
        for (int d = 1; d < SP; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const float f = ex2(m - (mx == -INFINITY ? 0.0f : mx));
        l *= f;
#pragma unroll
        for (int v = 0; v < 8; ++v) o[v] *= f;
#pragma unroll
        for (int d = 1; d < SP; d <<= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, d);
#pragma unroll
            for (int v = 0; v < 8; ++v) o[v] += __shfl_xor_sync(0xffffffffu, o[v], d);
        }
        if (p != 0 || e0 + (int)threadIdx.x / SP >= n) continue;
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
        uint32_t y[4];
#pragma unroll
        for (int v = 0; v < 4; ++v) y[v] = Half16<BF>::down(o[2 * v] * inv, o[2 * v + 1] * inv);
        const long long tok = it.tok + row / G;
        const int h = it.j * G + row % G;
        *(uint4 *)((uint16_t *)a.out + tok * a.out_stride + (long long)h * HD + 8 * d8) = make_uint4(y[0], y[1], y[2], y[3]);
        if (d8 == 0 && a.lse)
            a.lse[tok * a.n_q + h] = l != 0.0f ? 0.69314718055994530942f * (mx + log2f(l)) : -INFINITY;
    }
}

// 80 registers of 128 threads fit on an SM beside a CTA of k_paged_attn, so that
// the first blocks wait there for its end (verify 29.5 -> 28.6 us, one token over
// 131071 positions 95.4 -> 93.8 us against blocks of 256).  Blocks that share
// the tasks of all items evenly took 1 to 5 us more: the scan of the items comes
// before the first read of a record.
template <int HD, bool BF>
__global__ void __launch_bounds__(JOIN_THREADS, 6) k_paged_join(const AttnArgs a, int stride) {
    pdl_wait();
    pdl_trigger();
    const PaItem it = a.items[blockIdx.x];
    if (it.np == 0) return;
    // the group size with the fewest round trips: those of a value (four parts
    // a thread each), times the values of a group
    const int tasks = it.rows * (HD / 8), threads = JOIN_THREADS * gridDim.y;
    auto trips = [&](int sp) { return (tasks * sp + threads - 1) / threads * (2 * ((it.np + 4 * sp - 1) / (4 * sp)) + 1); };
    const int t1 = trips(1), t2 = trips(2), t8 = trips(8);
    if (t1 <= t2 && t1 <= t8) pa_join<HD, BF, 1>(a, it, stride);
    else if (t2 <= t8) pa_join<HD, BF, 2>(a, it, stride);
    else pa_join<HD, BF, 8>(a, it, stride);
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
bool pa_pool_map(CUtensorMap *tm, const M27BPagedKV &kv, const void *pool, int rows) {
    auto enc = pa_encoder();
    if (!enc) return false;
    const cuuint64_t dim[4] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.page_size, (cuuint64_t)kv.n_kv, (cuuint64_t)kv.n_pages};
    const cuuint64_t stride[3] = {(cuuint64_t)kv.n_kv * kv.head_dim * 2, (cuuint64_t)kv.head_dim * 2,
                                  (cuuint64_t)kv.page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(kv.page_size < rows ? kv.page_size : rows), 1, 1}, one[4] = {1, 1, 1, 1};
    return enc(tm, kv.type == M27B_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
               const_cast<void *>(pool), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// (value, head, token) of q; a box is 64 values of the G heads of a kv head, tq tokens.
bool pa_q_map(CUtensorMap *tm, const AttnArgs &a, int G, int tq) {
    auto enc = pa_encoder();
    if (!enc) return false;
    const cuuint64_t dim[3] = {(cuuint64_t)a.kv.head_dim, (cuuint64_t)a.n_q, (cuuint64_t)a.bt.n_tok};
    const cuuint64_t stride[2] = {(cuuint64_t)a.kv.head_dim * 2, (cuuint64_t)a.q_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)tq}, one[3] = {1, 1, 1};
    return enc(tm, a.kv.type == M27B_TYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
               const_cast<void *>(a.q), dim, stride, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int PA_MAX_CTAS = 160;  // CTAs the scratch has records for

// CTAs of a launch: one per SM of the current device, an even number.
int pa_ctas() {
    static int sms[64] = {};
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 0;
    if (dev < 64 && sms[dev]) return sms[dev];
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    n = (n < PA_MAX_CTAS ? n : PA_MAX_CTAS) & ~1;
    if (dev < 64) sms[dev] = n;
    return n;
}

// Raise a kernel's shared-memory limit, once per device.
template <class K>
cudaError_t pa_ready(K kern, size_t smem, bool (&done)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess || (dev >= 0 && dev < 64 && done[dev])) return e;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
    return e;
}

// The join after it.  It asks for the same split of L1 as the kernel before
// (all shared memory), so that the SMs need not drain to change it.
template <int HD, bool BF>
cudaError_t pa_join_launch(const AttnArgs &a, int ctas, int stride, cudaStream_t st) {
    static bool ready[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        e = cudaFuncSetAttribute(k_paged_join<HD, BF>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    return launch_pdl(k_paged_join<HD, BF>, dim3(ctas, 16), dim3(JOIN_THREADS), 0, st, a, stride);
}

template <int HD, bool BF>
cudaError_t pa_launch(const AttnArgs &a, int G, bool pair, int ctas, cudaStream_t st, bool *maps) {
    CUtensorMap tk, tv, tq;
    cudaError_t e;
    if constexpr (HD >= 128) {
        if (pair) {
            using L = PairPlan<HD>;
            static bool ready[64] = {};
            *maps = pa_pool_map(&tk, a.kv, a.kv.k, L::KR) && pa_pool_map(&tv, a.kv, a.kv.v, L::KT) && pa_q_map(&tq, a, G, PA_ROWS / G);
            if (!*maps) return cudaSuccess;
            e = pa_ready(k_paged_attn_pair<HD, BF>, L::SMEM, ready);
            if (e == cudaSuccess) e = launch_pdl(k_paged_attn_pair<HD, BF>, dim3(ctas), dim3(PAIR_THREADS), L::SMEM, st, a, tk, tv, tq);
            return e != cudaSuccess ? e : pa_join_launch<HD, BF>(a, ctas, 2, st);
        }
    }
    using L = PaPlan<HD>;
    static bool ready[64] = {};
    *maps = pa_pool_map(&tk, a.kv, a.kv.k, L::KT) && pa_pool_map(&tv, a.kv, a.kv.v, L::KT);
    if (!*maps) return cudaSuccess;
    e = pa_ready(k_paged_attn<HD, BF>, L::SMEM, ready);
    if (e == cudaSuccess) e = launch_pdl(k_paged_attn<HD, BF>, dim3(ctas), dim3(PA_THREADS), L::SMEM, st, a, tk, tv);
    return e != cudaSuccess ? e : pa_join_launch<HD, BF>(a, ctas, 1, st);
}

template <bool BF>
cudaError_t pa_launch_hd(const AttnArgs &a, int G, bool pair, int ctas, cudaStream_t st, bool *maps) {
    switch (a.kv.head_dim) {
    case 64: return pa_launch<64, BF>(a, G, pair, ctas, st, maps);
    case 128: return pa_launch<128, BF>(a, G, pair, ctas, st, maps);
    default: return pa_launch<256, BF>(a, G, pair, ctas, st, maps);
    }
}

}  // namespace
}  // namespace m27b

using namespace m27b;

extern "C" {

size_t m27b_paged_attn_scratch_bytes(int n_q, int n_kv, int head_dim) {
    if (n_kv < 1 || n_kv > 1024 || n_q < n_kv || n_q % n_kv || n_q / n_kv > 128) return 0;
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return 0;
    return PA_MAX_CTAS * sizeof(PaItem) + 2 * PA_MAX_CTAS * pa_record(head_dim) * sizeof(float);
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
    const int ctas = pa_ctas(), G = n_q / kv->n_kv;
    if (ctas < 2) return paged_fail(err, err_cap, "%s: no CUDA device", what);
    // a window of all that a row of the table holds is none, so that the kernels'
    // differences of positions (2^30 at most on either side) stay in 32 bits
    if (window < 0 || window >= kv->n_cols * kv->page_size) window = 0;
    const AttnArgs a = {*kv, *batch, q, out, lse, q_stride, out_stride, n_q, window, scale,
                        (PaItem *)scratch, (float *)((char *)scratch + PA_MAX_CTAS * sizeof(PaItem)), status_ptr_current()};
    // Pairs of CTAs when a sequence has rows for one and a half, on average.  With
    // 128, 192, 256, 512 rows a sequence, microseconds by single CTAs and by pairs
    // from cold L2: 16 sequences of 2000 positions, head_dim 256: 62 72 78 140 and
    // 64 68 72 132; head_dim 128: 62 83 87 134 and 70 72 74 111; one sequence: 42 36
    // 38 36 and 36 38 40 38; a prompt of 4096 tokens over 8192 positions, 24 heads of
    // 256: 695 and 458, 16 heads of 128: 269 and 218.  (head_dim 64 has no pairs:
    // the tensor pipe is busy a fifth of the time there, so that what a pair saves
    // in shared memory is not what bounds it.)  The average is over the batch: 64
    // single tokens over 2000 positions take 120 us, a chunk of 512 or 2048 tokens
    // of another sequence 73 and 161, and both in one call 159 (single CTAs) and
    // 294 (pairs), head_dim 256.
    const bool pair = (long long)batch->n_tok * G >= 192ll * batch->n_seq;
    bool maps = false;
    const cudaError_t e = kv->type == M27B_TYPE_BF16 ? pa_launch_hd<true>(a, G, pair, ctas, stream, &maps)
                                                     : pa_launch_hd<false>(a, G, pair, ctas, stream, &maps);
    if (e == cudaSuccess && !maps) return paged_fail(err, err_cap, "%s: the tensor maps were refused", what);
    return paged_ok(e, what, err, err_cap);
}

}  // extern "C"
