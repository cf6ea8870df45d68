// paged_rope.cu — head RMSNorm, rotary positions and the append of new tokens
// to a paged cache (include/m27b_paged.h), in one pass over the projections.
//
//   x' = x * rsqrt(mean(x^2) + eps) * w                      (where w is given)
//   (u, v) -> (u c - v s, u s + v c) for each of the first n_rot / 2 pairs of
//   the head, (c, s) = the position's table entry; q to q_out, k to its slot
//   of the cache, v to its slot as it is; one rounding to 16 bits at the end.
//
// A warp has whole heads: lane l holds values [l V, l V + V), V = head_dim / 32,
// so the mean is one butterfly, and the second value of a half-layout pair
// lies n_rot / 2 values, a whole number of lanes, away.
// Bounded by the bytes: each projection value is read once and written once
// in 16 bits; the table (256 bytes a token at n_rot = 64) stays in L2.
#include "paged_common.cuh"
#include "qmv_blk.cuh"

namespace m27b {

struct RopeArgs {
    M27BPagedKV kv;
    M27BPagedBatch bt;
    M27BRope rope;
    M27BHeads h;
    void *q_out;
    long long q_out_stride;
    int *status;
};

M27B_DI void mbar_arrive_local(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Sequence of token t: the number of ends cu_q[1..n] at or before t (n: none).
// 32 probes a step.
M27B_DI int find_seq(const int *cu_q, int n, int t, int lane) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32, i = lo + lane * step + step - 1;
        const bool past = i < hi && cu_q[i + 1] <= t;
        lo += __popc(__ballot_sync(0xffffffffu, past)) * step;
        if (step == 1) break;
        hi = min(hi, lo + step - 1);
    }
    return min(lo, n);
}

template <bool F32, bool BF, int V>
M27B_DI void load_head(const void *base, long long off, float (&x)[V]) {
    if constexpr (F32) {
        const float *p = (const float *)base + off;
        if constexpr (V == 2) {
            const float2 t = __ldcs((const float2 *)p);
            x[0] = t.x, x[1] = t.y;
        } else {
#pragma unroll
            for (int c = 0; c < V / 4; ++c) {
                const float4 t = __ldcs((const float4 *)p + c);
                x[4 * c] = t.x, x[4 * c + 1] = t.y, x[4 * c + 2] = t.z, x[4 * c + 3] = t.w;
            }
        }
    } else {
        const uint16_t *p = (const uint16_t *)base + off;
        uint32_t w[V / 2];
        if constexpr (V == 2) w[0] = __ldcs((const unsigned *)p);
        else if constexpr (V == 4) {
            const uint2 t = __ldcs((const uint2 *)p);
            w[0] = t.x, w[1] = t.y;
        } else {
            const uint4 t = __ldcs((const uint4 *)p);
            w[0] = t.x, w[1] = t.y, w[2] = t.z, w[3] = t.w;
        }
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 f = Half16<BF>::up(w[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}

// Eight values from shared memory.
template <bool F32, bool BF>
M27B_DI void load8_smem(const uint8_t *p, float (&x)[8]) {
    if constexpr (F32) {
        const float4 u = *(const float4 *)p, v = *((const float4 *)p + 1);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else {
        const uint4 u = *(const uint4 *)p;
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = Half16<BF>::up(w[i]);
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    }
}

template <bool BF, int V>
M27B_DI void store_head(void *base, long long off, const float (&x)[V]) {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = Half16<BF>::down(x[2 * i], x[2 * i + 1]);
    uint16_t *p = (uint16_t *)base + off;
    if constexpr (V == 2) *(unsigned *)p = w[0];
    else if constexpr (V == 4) *(uint2 *)p = make_uint2(w[0], w[1]);
    else *(uint4 *)p = make_uint4(w[0], w[1], w[2], w[3]);
}

// A token's sequence, slot and rotary position; false (and a report) if it has none.
struct RopeToken {
    long long slot;  // values from the pools' start to the token's first kv head
    int rp;
};
M27B_DI bool rope_token(const RopeArgs &a, int t, int b, bool report, RopeToken &k) {
    if (b >= a.bt.n_seq || t < a.bt.cu_q[b]) return false;  // of no sequence
    const int row = seq_row(a.bt, b, a.kv.n_rows);
    const int p = row < 0 ? -1 : a.bt.lens[row] - a.bt.cu_q[b + 1] + t;
    k.rp = a.rope.positions ? a.rope.positions[t] : p;
    const int pc = p / a.kv.page_size;
    const int page = p >= 0 && pc < a.kv.n_cols ? a.kv.table[(long long)row * a.kv.n_cols + pc] : -1;
    if (page < 0 || page >= a.kv.n_pages || k.rp < 0 || k.rp >= a.rope.n_pos) {
        if (report) paged_bad(a.status);
        return false;
    }
    k.slot = page * a.kv.page_stride + (long long)(p - pc * a.kv.page_size) * a.kv.n_kv * a.kv.head_dim;
    return true;
}

// This lane's cos and sin, from the position's row of the table: pairs d0 / 2 ..
// (interleaved) or d0 mod (n_rot / 2) .. of lanes that turn.
template <int V>
M27B_DI void rope_factors(const RopeArgs &a, const float2 *tab, int d0, float2 (&cs)[V]) {
    const int half = a.rope.n_rot / 2;
    if (d0 >= a.rope.n_rot) return;
    const float4 *at = (const float4 *)(tab + (a.rope.interleaved ? d0 / 2 : d0 < half ? d0 : d0 - half));
    const int n = a.rope.interleaved ? V / 2 : V;
    if constexpr (V == 2) {
        cs[0] = *(const float2 *)at;
        if (n == 2) cs[1] = *((const float2 *)at + 1);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            if (2 * i < n) {
                const float4 y = at[i];
                cs[2 * i] = make_float2(y.x, y.y), cs[2 * i + 1] = make_float2(y.z, y.w);
            }
    }
}

// V consecutive fp32 of norm weights.
template <int V>
M27B_DI void norm_weights(const float *w, int d0, float (&v)[V]) {
    if constexpr (V == 2) {
        const float2 y = __ldg((const float2 *)(w + d0));
        v[0] = y.x, v[1] = y.y;
    } else {
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float4 y = __ldg((const float4 *)(w + d0) + i);
            v[4 * i] = y.x, v[4 * i + 1] = y.y, v[4 * i + 2] = y.z, v[4 * i + 3] = y.w;
        }
    }
}

// One head of a token: x (this lane's values) normalised and turned.
template <int V>
M27B_DI void norm_turn(const RopeArgs &a, bool norm, const float (&nw)[V], const float2 (&cs)[V], int d0, int lane, float (&x)[V]) {
    if (norm) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) ss = fmaf(x[i], x[i], ss);
        const float sc = 1.0f / sqrtf(warp_sum(ss) / (float)(32 * V) + a.h.eps);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = x[i] * sc * nw[i];
    }
    const bool turns = d0 < a.rope.n_rot;
    if (a.rope.interleaved) {
        if (turns)
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float u = x[2 * i], v = x[2 * i + 1];
                x[2 * i] = u * cs[i].x - v * cs[i].y;
                x[2 * i + 1] = u * cs[i].y + v * cs[i].x;
            }
    } else {
        const int half = a.rope.n_rot / 2, dl = half / V;  // lanes between the two values of a pair
        const bool first = d0 < half;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = __shfl_sync(0xffffffffu, x[i], first ? lane + dl : lane - dl);
        if (turns)
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = first ? x[i] * cs[i].x - o[i] * cs[i].y : o[i] * cs[i].y + x[i] * cs[i].x;
    }
}

// Few tokens: a warp takes one head of one token.  Its loads go out before the
// token's sequence, page and slot are looked up (four dependent reads).
template <bool F32, bool BF, int V>
__global__ void __launch_bounds__(256) k_rope_append(const RopeArgs a) {
    constexpr int HD = 32 * V;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, d0 = lane * V;
    const int rows = a.h.n_q + 2 * a.kv.n_kv;
    const long long w = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const long long t64 = w / rows;
    if (t64 >= a.bt.n_tok) return;
    const int t = (int)t64, r = (int)(w - t64 * rows), j = r - a.h.n_q;
    float x[V], nw[V];
    const float *norm = r < a.h.n_q ? a.h.q_norm : j < a.kv.n_kv ? a.h.k_norm : nullptr;
    if (r < a.h.n_q) load_head<F32, BF>(a.h.q, t * a.h.q_stride + (long long)r * HD + d0, x);
    else if (j < a.kv.n_kv) load_head<F32, BF>(a.h.k, t * a.h.k_stride + (long long)j * HD + d0, x);
    else load_head<F32, BF>(a.h.v, t * a.h.v_stride + (long long)(j - a.kv.n_kv) * HD + d0, x);
    if (norm) norm_weights<V>(norm, d0, nw);
    RopeToken k;
    if (!rope_token(a, t, find_seq(a.bt.cu_q, a.bt.n_seq, t, lane), lane == 0, k)) return;
    if (j >= a.kv.n_kv) {
        store_head<BF>(a.kv.v, k.slot + (long long)(j - a.kv.n_kv) * HD + d0, x);
        return;
    }
    float2 cs[V];
    rope_factors<V>(a, (const float2 *)a.rope.table + (long long)k.rp * (a.rope.n_rot / 2), d0, cs);
    norm_turn<V>(a, norm != nullptr, nw, cs, d0, lane, x);
    if (r < a.h.n_q) store_head<BF>(a.q_out, t * a.q_out_stride + (long long)r * HD + d0, x);
    else store_head<BF>(a.kv.k, k.slot + (long long)j * HD + d0, x);
}

// This lane's eight values of a head that LG lanes hold, normalised with
// weights w (if `norm`) and turned (if `turn`).  For the half layout cs has the
// sine's sign of the lane's place in the pair.  All lanes come here.
template <int LG>
M27B_DI void norm_turn8(const RopeArgs &a, bool norms, bool norm, bool turn, const float (&w)[8], const float2 (&cs)[8], int from, float (&x)[8]) {
    if (norms) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int o = LG / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float sc = rsqrtf(fmaf(ss, 1.0f / (8 * LG), a.h.eps));
        if (norm)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * sc * w[i];
    }
    if (a.rope.interleaved) {
        if (turn)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float u = x[2 * i], v = x[2 * i + 1];
                x[2 * i] = u * cs[i].x - v * cs[i].y, x[2 * i + 1] = u * cs[i].y + v * cs[i].x;
            }
    } else {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, x[i], from);
        if (turn)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], cs[i].x, o[i] * cs[i].y);
    }
}

// Many tokens: a unit is up to p.per heads of a token, at most 32 KB of
// projections.  A producer warp looks the units' tokens up, 32 at a time, and
// keeps p.stages units in flight in shared memory (bulk copies of the unit's
// q, k and v heads and of the position's row of the table); eight warps turn
// them, a lane eight values of a head.  The lookups' and the memory's latency,
// which hold the kernel above to half of the bandwidth, are then off the warps'
// path.  8192 tokens, from cold L2: 32 heads of 256 fp32 values 135 -> 74 us
// (403 MB, 5.4 TB/s), 32 heads of 128 bf16 values 102 -> 43 us (134 MB, 3.1
// TB/s).  The same heads in fp32 take no longer (49 us against 48 a call): with
// rows this short a unit's hand-offs bound it (1.6 us a unit and CTA), neither
// the issue slots, 55 % busy, nor the memory.  A warp with whole heads, as
// above, took 80 and 57 us; 12 and 16 warps 80 and 98 us, 47 and 68 us.
constexpr int ROPE_WARPS = 8, ROPE_MAX_STAGES = 8;
constexpr int ROPE_UNIT = 32 * 1024;
constexpr int ROPE_THREADS = (ROPE_WARPS + 1) * 32;
constexpr int ROPE_SMEM = 110 * 1024;  // of a CTA, two on an SM

// A unit's size and the stages that a CTA keeps of it.
struct RopeStream {
    int per, groups;         // heads of a unit, units of a token
    int stage, tab, stages;  // bytes of a stage and of its row of the table
};

template <bool F32, bool BF, int LG>
__global__ void __launch_bounds__(ROPE_THREADS, 2) k_rope_stream(const RopeArgs a, const RopeStream p, int wait_code) {
    constexpr int HD = 8 * LG, ES = F32 ? 4 : 2, HB = HD * ES, HW = 32 / LG;  // HW: heads of a warp at once
    extern __shared__ __align__(128) uint8_t rope_smem[];
    __shared__ uint64_t full[ROPE_MAX_STAGES], empty[ROPE_MAX_STAGES];
    __shared__ long long slots[ROPE_MAX_STAGES];  // the unit's slot; -1: token left out
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows = a.h.n_q + 2 * a.kv.n_kv;
    const long long units = (long long)a.bt.n_tok * p.groups, mine = blockIdx.x < units ? (units - 1 - blockIdx.x) / gridDim.x + 1 : 0;
    uint8_t *tabs = rope_smem + (size_t)p.stages * p.stage;
    if (tid == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], ROPE_WARPS);
        }
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    int s = 0;
    uint32_t turn = 0;  // parity of the ring's round
    // the unit at hand: group g of token t; gridDim.x units on
    int t = (int)(blockIdx.x / p.groups), g = (int)(blockIdx.x % p.groups);
    const int dt = (int)(gridDim.x / p.groups), dg = (int)(gridDim.x % p.groups);
    auto step = [&] {
        if (++s == p.stages) s = 0, turn ^= 1u;
        t += dt, g += dg;
        if (g >= p.groups) g -= p.groups, ++t;
    };
    if (warp == ROPE_WARPS) {
        bool ok = true;
        RopeToken k = {-1, 0};
        long long n = 0;
        for (; ok && n < mine; ++n) {
            if (n % 32 == 0) {
                // the next 32 units' tokens, one a lane
                const long long u = blockIdx.x + (n + lane) * (long long)gridDim.x;
                k.slot = -1;
                if (n + lane < mine) {
                    const int tl = (int)(u / p.groups);
                    int lo = 0, hi = a.bt.n_seq;
                    while (lo < hi) {
                        const int mid = (lo + hi) / 2;
                        if (a.bt.cu_q[mid + 1] <= tl) lo = mid + 1;
                        else hi = mid;
                    }
                    if (!rope_token(a, tl, lo, true, k)) k.slot = -1;
                }
                __syncwarp();
            }
            const long long slot = __shfl_sync(0xffffffffu, k.slot, (int)(n % 32));
            const int rp = __shfl_sync(0xffffffffu, k.rp, (int)(n % 32));
            if (lane == 0) {
                if (n >= p.stages && !mbar_wait_bounded(&empty[s], turn ^ 1u, a.status, wait_code)) ok = false;
                else {
                    const int r0 = g * p.per, r1 = min(rows, r0 + p.per);
                    slots[s] = slot;
                    if (slot < 0) mbar_arrive_local(&full[s]);
                    else {
                        const int nq = max(0, min(r1, a.h.n_q) - r0), kb = a.h.n_q + a.kv.n_kv;
                        const int k0 = max(r0, a.h.n_q), nk = max(0, min(r1, kb) - k0), v0 = max(r0, kb), nv = max(0, r1 - v0);
                        uint8_t *st = rope_smem + (size_t)s * p.stage;
                        const uint32_t tb = (uint32_t)a.rope.n_rot * 4;
                        mbar_arrive_expect_tx(&full[s], (uint32_t)(r1 - r0) * HB + tb);
                        bulk_copy_g2s(tabs + s * p.tab, a.rope.table + (long long)rp * a.rope.n_rot, tb, &full[s]);
                        if (nq) bulk_copy_g2s(st, (const uint8_t *)a.h.q + (t * a.h.q_stride + (long long)r0 * HD) * ES, nq * HB, &full[s]);
                        if (nk)
                            bulk_copy_g2s(st + (k0 - r0) * HB, (const uint8_t *)a.h.k + (t * a.h.k_stride + (long long)(k0 - a.h.n_q) * HD) * ES,
                                          nk * HB, &full[s]);
                        if (nv)
                            bulk_copy_g2s(st + (v0 - r0) * HB, (const uint8_t *)a.h.v + (t * a.h.v_stride + (long long)(v0 - kb) * HD) * ES,
                                          nv * HB, &full[s]);
                    }
                }
            }
            ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
            step();
        }
        // every copy lands before the shared memory is released (bounded)
        if (lane == 0)
            for (long long i = ok ? n : n - 1, e = i; i > 0 && e - i < p.stages; --i) {
                const long long round = (i - 1) / p.stages;
                mbar_wait_bounded(&full[(i - 1) - round * p.stages], (uint32_t)(round & 1), a.status, wait_code);
            }
        return;
    }
    const int d0 = 8 * (lane % LG), half = a.rope.n_rot / 2, kb = a.h.n_q + a.kv.n_kv;
    const bool turns = d0 < a.rope.n_rot, first = d0 < half, norms = a.h.q_norm || a.h.k_norm;
    const int from = first ? lane + half / 8 : lane - half / 8;  // the lane with the pairs' other values
    float qw[8] = {}, kw[8] = {};
    if (a.h.q_norm) norm_weights<8>(a.h.q_norm, d0, qw);
    if (a.h.k_norm) norm_weights<8>(a.h.k_norm, d0, kw);
    for (long long n = 0; n < mine; ++n) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[s], turn, a.status, wait_code))) return;
        const long long slot = slots[s];
        const int r0 = g * p.per, r1 = min(rows, r0 + p.per);
        if (slot >= 0) {
            uint16_t *qo = (uint16_t *)a.q_out + t * a.q_out_stride + d0;
            uint16_t *ko = (uint16_t *)a.kv.k + slot + d0, *vo = (uint16_t *)a.kv.v + slot + d0;
            const uint8_t *st = rope_smem + (size_t)s * p.stage;
            float2 cs[8];
            rope_factors<8>(a, (const float2 *)(tabs + s * p.tab), d0, cs);
            if (!a.rope.interleaved && first)
#pragma unroll
                for (int i = 0; i < 8; ++i) cs[i].y = -cs[i].y;
            // the warps take turns at the unit's rows, since the v heads are little
            // work (8192 tokens of 32 bf16 heads of 128: 45 -> 43 us)
            for (int rw = r0 + (warp + 3 * (int)n) % ROPE_WARPS * HW; rw < r1; rw += HW * ROPE_WARPS) {
                const int r = min(rw + lane / LG, r1 - 1);
                float x[8];
                load8_smem<F32, BF>(st + (r - r0) * HB + d0 * ES, x);
                const bool is_q = r < a.h.n_q, is_v = r >= kb;
                if (rw < kb) {
                    float w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = is_q ? qw[i] : kw[i];
                    norm_turn8<LG>(a, norms, is_q ? a.h.q_norm != nullptr : !is_v && a.h.k_norm, turns && !is_v, w, cs, from, x);
                }
                if (rw + lane / LG < r1) store_head<BF>(is_q ? qo : is_v ? vo : ko, (is_q ? r : is_v ? r - kb : r - a.h.n_q) * HD, x);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_local(&empty[s]);
        step();
    }
}

template <bool F32, bool BF, int V>
cudaError_t rope_launch_v(const RopeArgs &a, cudaStream_t st) {
    const int rows = a.h.n_q + 2 * a.kv.n_kv, hb = 32 * V * (F32 ? 4 : 2);
    RopeStream p;
    p.per = ROPE_UNIT / hb < rows ? ROPE_UNIT / hb : rows, p.groups = (rows + p.per - 1) / p.per;
    const long long units = (long long)a.bt.n_tok * p.groups, ctas = 2 * 148;
    // the stream once a CTA has two units (32 heads, microseconds by head and by
    // stream from cold L2: fp32 of 256, 148 tokens 10.2 and 12.3, 592 16.4 and
    // 16.4, 1184 26.6 and 20.5; bf16 of 128, 8.2 and 10.2, 14.3 and 12.3, 20.5 and 14.5)
    if (units >= ctas * 2) {
        p.stage = p.per * hb, p.tab = (a.rope.n_rot * 4 + 127) & ~127;
        p.stages = ROPE_SMEM / (p.stage + p.tab) < ROPE_MAX_STAGES ? ROPE_SMEM / (p.stage + p.tab) : ROPE_MAX_STAGES;
        static bool ready[64] = {};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        if (dev < 0 || dev >= 64 || !ready[dev]) {
            e = cudaFuncSetAttribute(k_rope_stream<F32, BF, 4 * V>, cudaFuncAttributeMaxDynamicSharedMemorySize, ROPE_SMEM);
            if (e != cudaSuccess) return e;
            if (dev >= 0 && dev < 64) ready[dev] = true;
        }
        return launch_pdl(k_rope_stream<F32, BF, 4 * V>, dim3((unsigned)ctas), dim3(ROPE_THREADS), (size_t)p.stages * (p.stage + p.tab), st, a, p, 5);
    }
    const dim3 grid((unsigned)(((long long)a.bt.n_tok * rows + 7) / 8)), block(256);
    return launch_pdl(k_rope_append<F32, BF, V>, grid, block, 0, st, a);
}

template <bool F32, bool BF>
cudaError_t rope_launch(const RopeArgs &a, cudaStream_t st) {
    switch (a.kv.head_dim) {
    case 64: return rope_launch_v<F32, BF, 2>(a, st);
    case 128: return rope_launch_v<F32, BF, 4>(a, st);
    default: return rope_launch_v<F32, BF, 8>(a, st);
    }
}

struct RopeTable {
    float2 *out;
    int n_pos, half;
    double theta;
    M27BRopeScaling s;
    double lo, hi, mul;
};

// One thread per (position, pair); the frequency and the angle in fp64, since
// an fp32 angle is off by up to 2^-24 of its size: 0.06 at a position of 10^6.
__global__ void __launch_bounds__(256) k_rope_table(const RopeTable a) {
    const long long n = (long long)a.n_pos * a.half;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const long long p = i / a.half;
        const int j = (int)(i - p * a.half);
        double f = pow(a.theta, -(double)j / a.half);
        if (a.s.kind == M27B_ROPE_LINEAR) f /= a.s.factor;
        if (a.s.kind == M27B_ROPE_YARN) {
            const double r = fmin(fmax((j - a.lo) / fmax(a.hi - a.lo, 0.001), 0.0), 1.0);
            f = f / a.s.factor * r + f * (1.0 - r);
        }
        double s, c;
        sincos((double)p * f, &s, &c);
        a.out[i] = make_float2((float)(c * a.mul), (float)(s * a.mul));
    }
}

bool paged_check_kv(const M27BPagedKV *kv, const char *what, char *err, size_t cap) {
    if (!kv) return paged_fail(err, cap, "%s: null cache", what);
    if (!kv->k || !kv->v || !kv->table) return paged_fail(err, cap, "%s: null pool or table", what);
    if (((uintptr_t)kv->k | (uintptr_t)kv->v) & 15u)
        return paged_fail(err, cap, "%s: pools must be 16-byte aligned", what);
    if (kv->type != M27B_TYPE_F16 && kv->type != M27B_TYPE_BF16)
        return paged_fail(err, cap, "%s: the cache's type must be f16 or bf16 (got %u)", what, kv->type);
    if (kv->page_size < 16 || kv->page_size > 256 || (kv->page_size & (kv->page_size - 1)))
        return paged_fail(err, cap, "%s: page_size must be 16, 32, 64, 128 or 256 (got %d)", what, kv->page_size);
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return paged_fail(err, cap, "%s: head_dim must be 64, 128 or 256 (got %d)", what, kv->head_dim);
    if (kv->n_kv < 1 || kv->n_kv > 1024) return paged_fail(err, cap, "%s: bad n_kv (%d)", what, kv->n_kv);
    if (kv->n_pages < 1 || kv->n_rows < 1 || kv->n_cols < 1)
        return paged_fail(err, cap, "%s: empty cache (%d pages, %d rows of %d)", what, kv->n_pages, kv->n_rows, kv->n_cols);
    if ((long long)kv->n_cols * kv->page_size > 0x3fffffffll)
        return paged_fail(err, cap, "%s: n_cols x page_size takes 31 bits or more", what);
    if (kv->page_stride < (long long)kv->page_size * kv->n_kv * kv->head_dim || kv->page_stride % 8)
        return paged_fail(err, cap, "%s: page_stride (%lld) must be a multiple of 8, at least a page", what, kv->page_stride);
    if (kv->page_stride > (1ll << 62) / 2 / kv->n_pages)
        return paged_fail(err, cap, "%s: page_stride (%lld) too large", what, kv->page_stride);
    return true;
}

bool paged_check_batch(const M27BPagedBatch *b, const M27BPagedKV *kv, const char *what, char *err, size_t cap) {
    if (!b || !b->cu_q || !b->lens) return paged_fail(err, cap, "%s: null batch, cu_q or lens", what);
    if (b->n_seq < 0 || b->n_tok < 0) return paged_fail(err, cap, "%s: bad n_seq (%d) or n_tok (%d)", what, b->n_seq, b->n_tok);
    if (!b->rows && b->n_seq > kv->n_rows)
        return paged_fail(err, cap, "%s: %d sequences and %d table rows", what, b->n_seq, kv->n_rows);
    return true;
}

}  // namespace m27b

using namespace m27b;

extern "C" {

bool m27b_rope_table(float *table, int n_pos, int n_rot, double theta, const M27BRopeScaling *scaling,
                     cudaStream_t stream, char *err, size_t err_cap) {
    const char *what = "m27b_rope_table";
    if (!table || ((uintptr_t)table & 7u)) return paged_fail(err, err_cap, "%s: table must be 8-byte aligned", what);
    if (n_pos < 1) return paged_fail(err, err_cap, "%s: n_pos must be positive (got %d)", what, n_pos);
    if (n_rot < 2 || n_rot % 2 || n_rot > 65536) return paged_fail(err, err_cap, "%s: n_rot must be even (got %d)", what, n_rot);
    if (!(theta > 0.0)) return paged_fail(err, err_cap, "%s: theta must be positive", what);
    RopeTable a = {};
    a.out = (float2 *)table, a.n_pos = n_pos, a.half = n_rot / 2, a.theta = theta, a.mul = 1.0;
    if (scaling) a.s = *scaling;
    if (a.s.kind < M27B_ROPE_NONE || a.s.kind > M27B_ROPE_YARN)
        return paged_fail(err, err_cap, "%s: unknown scaling %d", what, a.s.kind);
    if (a.s.kind != M27B_ROPE_NONE && !(a.s.factor >= 1.0f))
        return paged_fail(err, err_cap, "%s: the scaling factor must be at least 1", what);
    if (a.s.kind == M27B_ROPE_YARN) {
        if (a.s.original_ctx < 1 || !(a.s.beta_fast > 0.0f) || !(a.s.beta_slow > 0.0f) || theta == 1.0)
            return paged_fail(err, err_cap, "%s: yarn needs original_ctx, beta_fast and beta_slow", what);
        // pair that turns `beta` times over the original context
        auto pair = [&](double beta) {
            return n_rot * log(a.s.original_ctx / (2.0 * 3.14159265358979323846 * beta)) / (2.0 * log(theta));
        };
        a.lo = fmax(0.0, floor(pair(a.s.beta_fast)));
        a.hi = fmin((double)n_rot - 1.0, ceil(pair(a.s.beta_slow)));
        a.mul = a.s.attn_factor > 0.0f ? (double)a.s.attn_factor : 0.1 * log((double)a.s.factor) + 1.0;
    }
    const long long n = (long long)n_pos * a.half;
    const unsigned grid = (unsigned)((n + 255) / 256 < 16384 ? (n + 255) / 256 : 16384);
    k_rope_table<<<grid, 256, 0, stream>>>(a);
    return paged_ok(cudaGetLastError(), what, err, err_cap);
}

bool m27b_rope_append(const M27BPagedKV *kv, const M27BPagedBatch *batch, const M27BRope *rope, const M27BHeads *heads,
                      void *q_out, long long q_out_stride, cudaStream_t stream, char *err, size_t err_cap) {
    const char *what = "m27b_rope_append";
    if (!paged_check_kv(kv, what, err, err_cap) || !paged_check_batch(batch, kv, what, err, err_cap)) return false;
    if (!rope || !rope->table || ((uintptr_t)rope->table & 15u))
        return paged_fail(err, err_cap, "%s: the rope table must be 16-byte aligned", what);
    if (rope->n_pos < 1 || rope->n_rot < 16 || rope->n_rot % 16 || rope->n_rot > kv->head_dim)
        return paged_fail(err, err_cap, "%s: n_rot must be a multiple of 16, at most head_dim (got %d)", what, rope->n_rot);
    if (!batch->n_seq || !batch->n_tok) return paged_ok(cudaSuccess, what, err, err_cap);
    if (!heads || !heads->k || !heads->v) return paged_fail(err, err_cap, "%s: null k or v", what);
    if (heads->n_q < 0 || heads->n_q > 65536) return paged_fail(err, err_cap, "%s: bad n_q (%d)", what, heads->n_q);
    if (heads->n_q && (!heads->q || !q_out)) return paged_fail(err, err_cap, "%s: null q or q_out", what);
    const bool f32 = heads->src_type == M27B_TYPE_F32;
    if (!f32 && heads->src_type != kv->type)
        return paged_fail(err, err_cap, "%s: q, k, v must be f32 or of the cache's type (got %u)", what, heads->src_type);
    const int per16 = f32 ? 4 : 8;
    if (((uintptr_t)heads->q | (uintptr_t)heads->k | (uintptr_t)heads->v | (uintptr_t)q_out | (uintptr_t)heads->q_norm |
         (uintptr_t)heads->k_norm) & 15u)
        return paged_fail(err, err_cap, "%s: q, k, v, q_out and norm weights must be 16-byte aligned", what);
    if (heads->q_stride % per16 || heads->k_stride % per16 || heads->v_stride % per16 || q_out_stride % 8)
        return paged_fail(err, err_cap, "%s: strides must be multiples of 16 bytes", what);
    const long long hd = kv->head_dim;
    if (heads->k_stride < kv->n_kv * hd || heads->v_stride < kv->n_kv * hd ||
        (heads->n_q && (heads->q_stride < heads->n_q * hd || q_out_stride < heads->n_q * hd)))
        return paged_fail(err, err_cap, "%s: a token's stride is shorter than its heads", what);
    const void *q = heads->q;
    if (heads->n_q && q_out == q && (f32 || q_out_stride != heads->q_stride))
        return paged_fail(err, err_cap, "%s: q_out may be q only with its type and stride", what);
    if ((long long)batch->n_tok * (heads->n_q + 2 * kv->n_kv) > 0x7fffffffll * 8)
        return paged_fail(err, err_cap, "%s: too many heads", what);
    RopeArgs a = {*kv, *batch, *rope, *heads, q_out, q_out_stride, status_ptr_current()};
    const bool bf = kv->type == M27B_TYPE_BF16;
    cudaError_t e = f32 ? (bf ? rope_launch<true, true>(a, stream) : rope_launch<true, false>(a, stream))
                        : (bf ? rope_launch<false, true>(a, stream) : rope_launch<false, false>(a, stream));
    return paged_ok(e, what, err, err_cap);
}

}  // extern "C"
