// Attention over the 8-bit paged cache, up to 64 query rows a KV head (decode,
// verify), and the attention mass that eviction goes by.
//
// softmax(q K^T / sqrt(d)) V per row, row t of sequence b over entries
// 0 .. entry0[b] + t.  Memory-bound up to a block of 8 or 16 rows: 2 d bytes an
// entry and KV head, read (from HBM or L2) and widened once for each such block of
// query rows.  Keys are the rows of the tensor-core products (m16n8k16):
// S^T = K Q^T and O^T += V^T P^T, 8 query rows as columns, so that the few
// rows of a decode step waste little.  The cache's bytes are stored in operand
// order, so a lane's 16-byte shared-memory load is an operand after
// e4m3 -> f16, which is exact.
//
// Rounding: K and V enter exactly (block scales are powers of two: K's is
// multiplied into the fp32 scores, V's into the probabilities).  Queries are
// the sum of two f16 numbers (22 bits), so scores, and the mass, are what fp32
// arithmetic gives; probabilities are two f16 numbers for fp32 outputs, one
// for bf16 outputs; max, sum and O are fp32.
//
// One CTA per (key split, KV head, sequence x row block), two an SM.  A unit is
// 4 KB: the K and V of 16 tokens at d = 128, of 32 at d = 64; 8 units, one a
// warp, are a round, and the splits take the rounds in turns, so that a sequence
// far shorter than the capacity still reaches all its CTAs (4 x 8 heads, 8192
// entries of 32768: 39 us with a run of keys a split, 21 us in turns; a full one
// is the same).  A CTA's warps are on their own until the end: lane 0 fetches
// the warp's units with bulk copies into a ring, and each warp keeps (max, sum,
// O), merged in a fixed order.  Which split, warp and tile an entry goes to is
// fixed by its index alone and a row's arithmetic does not depend on the other
// rows of the call, so a verify row equals the decode step at that entry bit for
// bit.
// Measured (d 128, group 4, bf16): 262144 entries of 8 heads (537 MB) in 92 us,
// 5.8 TB/s, of which about 10 us are launch, first bytes and two merges; a warp
// needs about 1900 cycles a unit, so one CTA alone streams 27 GB/s, which bounds
// ragged batches.  6 warps with units of
// 8 KB (half the overhead a byte) were slower: 262144 entries 95 for 90 us.
//
// The running max is raised lazily: only when a score exceeds it by more than
// 8 (log2 units), which keeps the common tile free of shuffles and rescaling;
// probabilities stay below 2^8 and O / sum is exact either way.
#include <algorithm>

#include "attention_q8.cuh"

namespace dkv {

namespace {

constexpr int kQdKG = 8;               // key groups: the CTA's warps
constexpr int kQdUnit = 4096;          // bytes of a unit
constexpr int kQdDepth = 3;            // units of a warp's ring
constexpr int kQdThreads = 32 * kQdKG;
constexpr size_t kQdSmem = (size_t)kQdKG * kQdDepth * kQdUnit;
constexpr int kQdMinBytes = 1 << 17;   // codes a split streams where the library picks it, at least
constexpr float kQdLazy = 8.f;         // growth of the max that forces a rescale (log2 units)
constexpr int kQdBias = 6;             // probabilities enter as p * 2^6: f16 keeps 2^-30 of the max

DKV_DEV uint32_t pack_h2(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
DKV_DEV float2 unpack_h2(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
DKV_DEV void mma_f16_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
DKV_DEV uint32_t movm_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
// Page ids and scales of a warp's next tiles, one tile a lane; the K scale of a
// tile that must not be seen (bad page id, past the end) is negative, its V scale
// the smallest.
struct QdMeta {
    int pid;
    float ks, vs;
};

// NT: tiles of 8 query rows; PLO: probabilities as two f16 numbers (fp32
// outputs; one holds a weight to 2^-11, an eighth of a bf16 output's
// rounding).  PAIR (up to 4 rows): columns 4..7 of the score product hold the
// queries' lower parts, so one product gives both sums; the same numbers are
// multiplied and added as without, so a row's bits do not depend on it.
template <int D, int NT, bool PLO, bool PAIR>
__global__ void __launch_bounds__(kQdThreads, 16 / kQdKG) q8_decode_kernel(const __grid_constant__ Q8AttnArgs a) {
    constexpr int UT = kQdUnit / (2 * D);              // tokens a unit
    constexpr int TPU = UT / 16;                       // 16-token tiles a unit
    constexpr int UPB = 32 / TPU;                      // units whose tiles a warp's lanes describe at once
    constexpr int KS = D / 16, PS = D + 4, RB = 8 * NT;
    static_assert(!PAIR || NT == 1, "paired columns: one row tile");
    constexpr int QP = PAIR ? 1 : 2;                   // query operands a row tile
    static_assert(RB * PS * sizeof(float) <= kQdDepth * kQdUnit, "a warp's partial rows fit its ring");
    extern __shared__ __align__(128) uint8_t ring_all[];
    __shared__ __align__(8) uint64_t full_bar[kQdKG][kQdDepth];
    __shared__ uint2 qs[NT > 1 ? QP * NT * KS * 32 : 1];       // query operands (NT 1: in registers)
    __shared__ float ms[RB], ls[RB];
    __shared__ float gw[RB * kQdKG];
    __shared__ int failed;
    __shared__ int8_t own_eo[kQdKG][RB];
    const Q8View& v = a.v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* ring = ring_all + (size_t)warp * kQdDepth * kQdUnit;
    uint64_t* full = full_bar[warp];
    if (lane == 0) {
        for (int i = 0; i < kQdDepth; ++i) mbar_init(&full[i], 1);
        if (warp == 0) failed = 0;
        fence_async_shared();
    }
    __syncwarp();
    pdl_wait();            // queries and the new entries come from earlier kernels

    // one round of loads: the first page ids (any entry of the table row may be
    // read), the query rows, entry0 and n_rows
    const int s = blockIdx.x, h = blockIdx.y;
    const int b = blockIdx.z / a.n_rb, rb = blockIdx.z % a.n_rb;
    const int G = a.group, R_all = a.T * G;
    const int rbase = rb * RB, R = min(RB, R_all - rbase);
    const int32_t* tab = v.row(b);
    // first key of this warp's unit u: round u * n_splits + s of the sequence
    auto key_of = [&](int u) { return ((u * a.n_splits + s) * kQdKG + warp) * UT; };
    // page id of tile `lane` of the batch that starts at this warp's unit u0 (-1 beyond the table)
    auto load_pid = [&](int u0) {
        const long long key = (((long long)(u0 + lane / TPU) * a.n_splits + s) * kQdKG + warp) * UT + (lane % TPU) * 16;
        return key < v.capacity() ? q8_ld(tab + (key >> v.page_shift)) : -1;
    };
    const int first_pid = load_pid(0);
    const int qr = lane >> 2, qc = lane & 3;
    float2 xq[NT][KS][2];
    auto load_q = [&](int nt, int kk, int u) {
        const int r = nt * 8 + (PAIR ? qr & 3 : qr), gr = rbase + r;      // this lane's operand row
        return r < R ? q8_ld(reinterpret_cast<const float2*>(
                           a.q + (((size_t)b * a.T + gr / G) * v.n_kv * G + h * G + gr % G) * D + kk * 16 + u * 8 + 2 * qc))
                     : make_float2(0.f, 0.f);
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) xq[nt][kk][0] = load_q(nt, kk, 0), xq[nt][kk][1] = load_q(nt, kk, 1);
    const int n_tok = a.n_rows ? min(a.n_rows[b], a.T) : a.T;
    const int e0 = a.first(b);
    // the block's last token decides what is read
    const int t_last = min((rbase + R - 1) / G, n_tok - 1);
    const int n_keys = t_last >= rbase / G ? max(0, min(a.n_keys(b), e0 + t_last + 1)) : 0;
    if (s == 0 && h == 0 && rb == 0 && threadIdx.x == 0 && a.beyond(b)) atomicOr(a.err, kErrQ8Page);
    const int before = (n_keys + UT - 1) / UT - (s * kQdKG + warp), every = a.n_splits * kQdKG;
    const int mine = before > 0 ? (before + every - 1) / every : 0;      // this warp's units

    // -1 for tiles past the end and for bad ids (recorded; their keys are not seen)
    auto check_pid = [&](int u0, int pid) {
        const int u = u0 + lane / TPU;
        if (u >= mine || key_of(u) + (lane % TPU) * 16 >= n_keys) return -1;
        if (v.ok(pid)) return pid;
        atomicOr(a.err, kErrQ8Page);
        return -1;
    };
    auto load_scale = [&](int pid, float& ks, float& vs) {
        float2 sc = make_float2(-1.f, q8_pow2(kQ8ExpMin));
        if (pid >= 0) sc = q8_ld(reinterpret_cast<const float2*>(v.scale + v.scale_at(pid, h, 0)));
        ks = sc.x;
        vs = sc.y;
    };
    // unit u into ring slot `slot` (u % depth); pids: the page ids of its batch.
    // A tile is [K 16 d][V 16 d]; a 16-token page is one copy, of longer ones two
    const int rec = 2 * v.page * D;
    const uint8_t* base_h = v.codes + (size_t)h * rec;
    const size_t page_stride = (size_t)v.n_kv * rec;
    auto issue = [&](int u, int slot, int pids) {
        int pid[TPU], live = 0;
#pragma unroll
        for (int tt = 0; tt < TPU; ++tt) {
            pid[tt] = __shfl_sync(0xffffffffu, pids, (u % UPB) * TPU + tt);
            live += pid[tt] >= 0;
        }
        if (lane == 0) {
            uint8_t* to = ring + slot * kQdUnit;
            uint64_t* bar = &full[slot];
            mbar_expect_tx(bar, (uint32_t)(live * 32 * D));
#pragma unroll
            for (int tt = 0; tt < TPU; ++tt) {
                if (pid[tt] < 0) continue;
                const uint8_t* kp = base_h + (size_t)pid[tt] * page_stride;
                if (v.page == 16) {
                    bulk_g2s(to + tt * 32 * D, kp, 32 * D, bar);
                } else {
                    kp += ((key_of(u) + tt * 16) & (v.page - 1)) * D;
                    bulk_g2s(to + tt * 32 * D, kp, 16 * D, bar);
                    bulk_g2s(to + tt * 32 * D + 16 * D, kp + v.page * D, 16 * D, bar);
                }
            }
        }
        __syncwarp();
    };
    QdMeta cur{-1, -1.f, q8_pow2(kQ8ExpMin)}, nxt = cur;
    cur.pid = check_pid(0, first_pid);
    const int prologue = min(mine, kQdDepth);
    for (int u = 0; u < prologue; ++u) issue(u, u, cur.pid);     // (kQdDepth <= UPB)
    load_scale(cur.pid, cur.ks, cur.vs);

    // ---------------- queries: column qr of row tile nt, as hi (+ lo) f16
    // numbers of q * log2 e / sqrt(d) * 2^-x, x the row's exponent
    uint2 qreg[NT > 1 ? 1 : QP * KS];
    float cs[NT][2];                                   // 2^x of this thread's score columns
    int lim[NT][2];                                    // last visible entry of them
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float2(&x)[KS][2] = xq[nt];
        float am = 0.f;
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                x[kk][u].x *= a.scale;
                x[kk][u].y *= a.scale;
                am = fmaxf(am, fmaxf(fabsf(x[kk][u].x), fabsf(x[kk][u].y)));
            }
        am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
        am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
        // am = 1.m * 2^ex; an infinite row keeps its infinities
        const int ex = min(max((int)(__float_as_uint(am) >> 23) - 127, -126), 126);
        const float down = q8_pow2(-ex);
#pragma unroll
        for (int kk = 0; kk < KS; ++kk) {
            uint2 hi, lo;
            uint32_t* hp = &hi.x;
            uint32_t* lp = &lo.x;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float p = x[kk][u].x * down, q = x[kk][u].y * down;
                hp[u] = pack_h2(p, q);
                const float2 hf = unpack_h2(hp[u]);
                lp[u] = pack_h2(p - hf.x, q - hf.y);
            }
            if (NT > 1) {
                if (warp == kk % kQdKG) {              // (every warp holds the same rows)
                    qs[(kk * NT + nt) * 32 + lane] = hi;
                    qs[((KS + kk) * NT + nt) * 32 + lane] = lo;
                }
            } else if (PAIR) {
                qreg[kk] = qr < 4 ? hi : lo;
            } else {
                qreg[kk] = hi;
                qreg[(QP - 1) * KS + kk] = lo;
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            cs[nt][c] = __shfl_sync(0xffffffffu, q8_pow2(ex), (2 * qc + c) * 4);
            const int rc = nt * 8 + 2 * qc + c, t = (rbase + rc) / G;
            lim[nt][c] = rc < R && (!PAIR || qc < 2) && t < n_tok ? min(e0 + t, n_keys - 1) : -1;
        }
    }
    if (NT > 1) __syncthreads();
    auto query = [&](int piece, int kk, int nt) -> uint2 {
        if (NT > 1) return qs[((piece * KS + kk) * NT + nt) * 32 + lane];
        return qreg[piece * KS + kk];
    };

    // m: the running max (0 until a key was seen, for which thr is -infinity);
    // thr: the score that forces m up
    float m[NT][2], thr[NT][2], l[NT][2];
    float o[NT][KS][4];
    // O is in units of 2^(eo - kQdBias), eo the largest V exponent so far or one below
    // (probabilities, at most 2^8, then enter as p * 2^(bias + 1)); for a row that sees
    // no more when it grows (the growth may be more than fp32 spans) in those of own_eo
    int eo = q8_scale_exp(__shfl_sync(0xffffffffu, cur.vs, 0));
    if (lane < RB) own_eo[warp][lane] = (int8_t)-128;
    __syncwarp();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = l[nt][0] = l[nt][1] = 0.f;
        thr[nt][0] = thr[nt][1] = -INFINITY;
#pragma unroll
        for (int md = 0; md < KS; ++md) o[nt][md][0] = o[nt][md][1] = o[nt][md][2] = o[nt][md][3] = 0.f;
    }
    float* sc_base = a.scores ? a.scores + (((size_t)b * v.n_kv + h) * v.capacity()) * a.s_ld : nullptr;
    // entries up to here are seen by every row of the block that is there
    const int all_see = min(e0 + rbase / G, n_keys - 1);

    // ---- S^T of a unit, not yet scaled: keys qr (+8), columns 2qc, 2qc + 1 of
    // each row tile.  Two chains of products (the halves of each 32-dim block)
    // and the queries' lower parts apart, added in one order
    auto products = [&](const uint8_t* st, float (&sh)[TPU][NT][4]) {
#pragma unroll
        for (int tt = 0; tt < TPU; ++tt) {
            float x0[NT][4], x1[NT][4], y0[PAIR ? 1 : NT][4], y1[PAIR ? 1 : NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x0[nt][e] = x1[nt][e] = 0.f;
                    if (!PAIR) y0[nt][e] = y1[nt][e] = 0.f;
                }
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const uint4 w = *reinterpret_cast<const uint4*>(st + tt * 32 * D + j * 512);
                uint32_t a0[4], a1[4];
                q8_decode4(w.x, a0[0], a0[2]);
                q8_decode4(w.y, a0[1], a0[3]);
                q8_decode4(w.z, a1[0], a1[2]);
                q8_decode4(w.w, a1[1], a1[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint2 q0 = query(0, 2 * j, nt), q1 = query(0, 2 * j + 1, nt);
                    mma_f16_16816(x0[nt], a0, q0.x, q0.y);
                    mma_f16_16816(x1[nt], a1, q1.x, q1.y);
                    if (!PAIR) {
                        const uint2 p0 = query(1, 2 * j, nt), p1 = query(1, 2 * j + 1, nt);
                        mma_f16_16816(y0[nt], a0, p0.x, p0.y);
                        mma_f16_16816(y1[nt], a1, p1.x, p1.y);
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float hi = x0[nt][e] + x1[nt][e];
                    // paired: lane qc holds columns 2qc, + 1; qc + 2 their lower parts
                    const float lo = PAIR ? __shfl_xor_sync(0xffffffffu, hi, 2) : y0[PAIR ? 0 : nt][e] + y1[PAIR ? 0 : nt][e];
                    sh[tt][nt][e] = hi + lo;
                }
        }
    };
    auto arrived = [&](int u, int slot, uint32_t phase) {
        if (__all_sync(0xffffffffu, mbar_wait(&full[slot], phase, a.err))) return true;
        // a copy never came (error word 0x80): wait, bounded, for those still in flight
        if (lane == 0) {
            failed = 1;
            for (int w = u + 1; w < min(mine, u + kQdDepth); ++w)
                mbar_wait(&full[w % kQdDepth], (uint32_t)((w / kQdDepth) & 1), nullptr);
        }
        __syncwarp();
        return false;
    };

    // One row tile of d 128 (a unit of d 64 has two tiles to overlap): the next unit's scores are computed among this one's
    // probabilities and V products (a warp's own chain of latencies, not issue
    // slots, is what a unit takes)
    constexpr bool AHEAD = NT == 1 && D == 128;
    float sn[TPU][NT][4];
    int slot = 0;
    uint32_t phase = 0;
    bool go = mine > 0;
    if (AHEAD && go) {
        go = arrived(0, 0, 0u);
        products(ring + lane * 16, sn);
    }
    for (int u = 0; u < mine && go; ++u) {
        const int ub = u % UPB;
        if (ub == 0) {
            if (u > 0) cur = nxt;
            nxt.pid = check_pid(u + UPB, load_pid(u + UPB));
        } else if (ub == UPB / 2) {
            load_scale(nxt.pid, nxt.ks, nxt.vs);
        }
        const uint8_t* st = ring + slot * kQdUnit + lane * 16;
        const int slot1 = slot + 1 == kQdDepth ? 0 : slot + 1;
        const uint32_t phase1 = slot1 == 0 ? phase ^ 1u : phase;
        if (AHEAD ? u + 1 < mine && !arrived(u + 1, slot1, phase1) : !arrived(u, slot, phase)) break;
        const int key0 = key_of(u);
        float ks[TPU], vs[TPU];
        bool whole = key0 + UT - 1 <= all_see;         // every key of the unit is there for every row
#pragma unroll
        for (int tt = 0; tt < TPU; ++tt) {
            ks[tt] = __shfl_sync(0xffffffffu, cur.ks, ub * TPU + tt);
            vs[tt] = __shfl_sync(0xffffffffu, cur.vs, ub * TPU + tt);
            whole = whole && ks[tt] >= 0.f;
        }
        float sh[TPU][NT][4];
        bool grow = false;
        if (!AHEAD) products(st, sn);
#pragma unroll
        for (int tt = 0; tt < TPU; ++tt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) sh[tt][nt][e] = sn[tt][nt][e] * (cs[nt][e & 1] * ks[tt]);
        if (!whole) {
#pragma unroll
            for (int tt = 0; tt < TPU; ++tt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + tt * 16 + qr + (e >> 1) * 8;
                        if (key > lim[nt][e & 1] || ks[tt] < 0.f) sh[tt][nt][e] = -INFINITY;
                    }
        }
#pragma unroll
        for (int tt = 0; tt < TPU; ++tt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
                grow = grow || fmaxf(sh[tt][nt][0], sh[tt][nt][2]) > thr[nt][0] || fmaxf(sh[tt][nt][1], sh[tt][nt][3]) > thr[nt][1];
        if (sc_base) {
#pragma unroll
            for (int tt = 0; tt < TPU; ++tt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const int r = rbase + nt * 8 + 2 * qc, ka = key0 + tt * 16 + qr;
                    if (r < a.s_ld && (!PAIR || qc < 2)) {
                        if (ka < n_keys)
                            *reinterpret_cast<float2*>(sc_base + (size_t)ka * a.s_ld + r) =
                                make_float2(sh[tt][nt][0], sh[tt][nt][1]);
                        if (ka + 8 < n_keys)
                            *reinterpret_cast<float2*>(sc_base + (size_t)(ka + 8) * a.s_ld + r) =
                                make_float2(sh[tt][nt][2], sh[tt][nt][3]);
                    }
                }
        }
        if (__any_sync(0xffffffffu, grow)) {
            // raise the max of the columns that need it (alpha 1 for the others)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float al[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float t = -INFINITY;
#pragma unroll
                    for (int tt = 0; tt < TPU; ++tt) t = fmaxf(t, fmaxf(sh[tt][nt][c], sh[tt][nt][c + 2]));
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, off));
                    const bool up = t > thr[nt][c];
                    al[c] = !up ? 1.f : thr[nt][c] == -INFINITY ? 0.f : q8_ex2(m[nt][c] - t);
                    if (up) m[nt][c] = t, thr[nt][c] = t + kQdLazy;
                    l[nt][c] *= al[c];
                }
#pragma unroll
                for (int md = 0; md < KS; ++md) {
                    o[nt][md][0] *= al[0];
                    o[nt][md][1] *= al[1];
                    o[nt][md][2] *= al[0];
                    o[nt][md][3] *= al[1];
                }
            }
        }
        // (uniform) larger V values in a tile: O to their units, tile by
        // tile, so that a row's probabilities are rounded under the exponents of the
        // tiles it sees.  (A row that does not see this tile sees none behind it.)
        auto raise = [&](int tt, int ev) {
            const float dn = q8_pow2(max(eo - ev, -126));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const bool seen = whole || key0 + tt * 16 <= lim[nt][c];
                    int8_t& own = own_eo[warp][nt * 8 + 2 * qc + c];
                    if (!seen && qr == 0 && own < kQ8ExpMin) own = (int8_t)eo;
                    const float f = seen ? dn : 1.f;
#pragma unroll
                    for (int md = 0; md < KS; ++md) o[nt][md][c] *= f, o[nt][md][c + 2] *= f;
                }
            eo = ev;
        };
        auto weigh = [&](int tt, int ev) {
            const float vf = q8_pow2(max(ev - eo + kQdBias, -126));
            uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = q8_ex2(sh[tt][nt][e] - m[nt][e & 1]);
                l[nt][0] += p[0] + p[2];
                l[nt][1] += p[1] + p[3];
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const float x = p[2 * w] * vf, y = p[2 * w + 1] * vf;
                    const uint32_t hi = pack_h2(x, y);
                    ph[nt][w] = movm_trans(hi);
                    if (PLO) {
                        const float2 hf = unpack_h2(hi);
                        pl[nt][w] = movm_trans(pack_h2(x - hf.x, y - hf.y));
                    }
                }
            }
            const uint8_t* vb = st + tt * 32 * D + 16 * D;
            uint4 w[D / 32];
#pragma unroll
            for (int j = 0; j < D / 32; ++j) w[j] = *reinterpret_cast<const uint4*>(vb + j * 512);
            if (!whole) {
                // bytes of keys that are not there (past the end, bad page) as zeros:
                // their probability is 0, but 0 x NaN would not be
                const int ke = ks[tt] < 0.f ? 0 : n_keys - key0 - tt * 16;
                const uint32_t vm = (2 * qc < ke ? 0xffu : 0u) | (2 * qc + 1 < ke ? 0xff00u : 0u) |
                                    (2 * qc + 8 < ke ? 0xff0000u : 0u) | (2 * qc + 9 < ke ? 0xff000000u : 0u);
#pragma unroll
                for (int j = 0; j < D / 32; ++j) w[j].x &= vm, w[j].y &= vm, w[j].z &= vm, w[j].w &= vm;
            }
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                uint32_t a0[4], a1[4];
                q8_decode4(w[j].x, a0[0], a0[2]);
                q8_decode4(w[j].y, a0[1], a0[3]);
                q8_decode4(w[j].z, a1[0], a1[2]);
                q8_decode4(w[j].w, a1[1], a1[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma_f16_16816(o[nt][2 * j], a0, ph[nt][0], ph[nt][1]);
                    mma_f16_16816(o[nt][2 * j + 1], a1, ph[nt][0], ph[nt][1]);
                    if (PLO) {
                        mma_f16_16816(o[nt][2 * j], a0, pl[nt][0], pl[nt][1]);
                        mma_f16_16816(o[nt][2 * j + 1], a1, pl[nt][0], pl[nt][1]);
                    }
                }
            }
        };
        bool larger = false;
#pragma unroll
        for (int tt = 0; tt < TPU; ++tt) larger = larger || q8_scale_exp(vs[tt]) > eo + 1;
        if (TPU == 1 && larger) raise(0, q8_scale_exp(vs[0]));
        // (past the last unit: over stale bytes, unused)
        if (AHEAD) products(ring + slot1 * kQdUnit + lane * 16, sn);
        if (TPU > 1 && larger) {                       // (rare: below the tiles overlap)
#pragma unroll
            for (int tt = 0; tt < TPU; ++tt) {
                const int ev = q8_scale_exp(vs[tt]);
                if (ev > eo + 1) raise(tt, ev);
                weigh(tt, ev);
            }
        } else {
#pragma unroll
            for (int tt = 0; tt < TPU; ++tt) weigh(tt, q8_scale_exp(vs[tt]));
        }
        // the slot's bytes are in registers: refill it
        __syncwarp();
        const int un = u + kQdDepth;
        if (un < mine) issue(un, slot, ub + kQdDepth < UPB ? cur.pid : nxt.pid);
        slot = slot1;
        phase = phase1;
    }
    __syncwarp();

    // ---- this warp's (max, sum, O over the sum) of every row to its drained ring
    {
        float* mine_f = reinterpret_cast<float*>(ring);        // [RB][max, sum, -, -, O / sum]
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int own = own_eo[warp][nt * 8 + 2 * qc + c];
                const float un = q8_pow2((own < kQ8ExpMin ? eo : own) - kQdBias);
                float ll = l[nt][c];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) ll += __shfl_xor_sync(0xffffffffu, ll, off);
                // O goes on over the sum (1 and more where a key was seen): an average of
                // V, which fp32 holds whatever V is
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                // no key seen: -infinity (a row with NaN scores has a NaN sum, to be merged)
                const float mm = thr[nt][c] == -INFINITY && ll == ll ? -INFINITY : m[nt][c];
                float* to = mine_f + (nt * 8 + 2 * qc + c) * PS;
                if (qr == 0) {
                    to[0] = mm;
                    to[1] = ll;
                }
#pragma unroll
                for (int md = 0; md < KS; ++md) {
                    to[4 + 16 * md + qr] = o[nt][md][c] * inv * un;
                    to[4 + 16 * md + qr + 8] = o[nt][md][c + 2] * inv * un;
                }
            }
    }
    pdl_trigger();
    __syncthreads();
    const size_t bhr = ((size_t)b * v.n_kv + h) * a.n_rb + rb;
    const bool alone = a.n_splits == 1;
    float* mypart = alone ? nullptr : a.part + (bhr * a.n_splits + s) * (size_t)RB * PS;
    auto group_row = [&](int g, int r) { return reinterpret_cast<const float*>(ring_all + (size_t)g * kQdDepth * kQdUnit) + r * PS; };
    if (threadIdx.x < R) {
        const int r = threadIdx.x;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int g = 0; g < kQdKG; ++g) M = fmaxf(M, group_row(g, r)[0]);
#pragma unroll
        for (int g = 0; g < kQdKG; ++g) {
            const float mg = group_row(g, r)[0];
            const float w = mg == -INFINITY ? 0.f : group_row(g, r)[1] * q8_ex2(mg - M);
            L += w;
            gw[r * kQdKG + g] = w;
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
        for (int g = 0; g < kQdKG; ++g) gw[r * kQdKG + g] *= inv;
        if (failed) M = -INFINITY, L = 0.f;            // a failed split counts as empty
        ms[r] = M;
        ls[r] = L;
        if (!alone) *reinterpret_cast<float2*>(mypart + (size_t)r * PS) = make_float2(M, L);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * (D / 2); i += kQdThreads) {
        const int r = i / (D / 2), e = i % (D / 2) * 2;
        float x0 = 0.f, x1 = 0.f;
#pragma unroll
        for (int g = 0; g < kQdKG; ++g) {
            const float w = gw[r * kQdKG + g];
            if (w != 0.f) {
                const float2 y = *reinterpret_cast<const float2*>(group_row(g, r) + 4 + e);
                x0 += y.x * w;
                x1 += y.y * w;
            }
        }
        if (alone) {
            q8_store2<D>(a, b, h, rbase + r, n_tok, e, x0, x1);
        } else {
            *reinterpret_cast<float2*>(mypart + (size_t)r * PS + 4 + e) = make_float2(x0, x1);
        }
    }
    if (!alone) {
        q8_merge_splits<D, RB>(a, bhr, b, h, rbase, R, n_tok);
    } else if (a.stats) {
        for (int r = threadIdx.x; r < R; r += kQdThreads)
            a.stats[((size_t)b * v.n_kv + h) * R_all + rbase + r] =
                make_float2(ms[r], ls[r] == 0.f || (rbase + r) / G >= n_tok ? 0.f : 1.f / ls[r]);
    }
}

// mass[b][h][j] += sum over the call's rows of p_j: the scores of the pass
// above under the merged (max, sum), rows in order (no atomics).
// A thread takes kMassKeys keys, kMassThreads apart, W rows of each at a time (8:
// a sector a load pair; rows of 2 scores: 2), whose loads are in flight together.
// (Two rows at a time, each sector fetched four times: 42 rows over 3 x 6 x 36337
// entries 75 us; so, 38 us.)
constexpr int kMassThreads = 256, kMassKeys = 4;
template <int W>
__global__ void __launch_bounds__(kMassThreads) q8_mass_kernel(Q8AttnArgs a, float* mass) {
    __shared__ float2 st_s[kQ8MaxRows + 8];        // (max, 1 / sum) of a row
    __shared__ int last_s[kQ8MaxRows + 8];         // a row's scores exist up to its own entry
    pdl_wait();
    const int h = blockIdx.y, b = blockIdx.z, R = a.T * a.group;
    const int n = a.n_keys(b), e0 = a.first(b), key0 = blockIdx.x * kMassThreads * kMassKeys + threadIdx.x;
    if ((int)(blockIdx.x * kMassThreads * kMassKeys) >= n) return;
    const size_t bh = (size_t)b * a.v.n_kv + h, cap = a.v.capacity();
    float old[kMassKeys], sum[kMassKeys];
    const float* sc = a.scores + (bh * cap + key0) * a.s_ld;
    constexpr int V = W == 2 ? 2 : 4;              // scores a load
    float x[kMassKeys][W];
    auto load = [&](int r) {
#pragma unroll
        for (int k = 0; k < kMassKeys; ++k)
#pragma unroll
            for (int w = 0; w < W; w += V) {
                const float* at = sc + (size_t)k * kMassThreads * a.s_ld + r + w;
                if (key0 + k * kMassThreads >= n || r + w >= a.s_ld) continue;
                if (V == 2) {
                    const float2 y = __ldcg(reinterpret_cast<const float2*>(at));
                    x[k][w] = y.x, x[k][w + 1] = y.y;
                } else {
                    const float4 y = __ldcg(reinterpret_cast<const float4*>(at));
                    x[k][w] = y.x, x[k][w + 1] = y.y, x[k][w + V - 2] = y.z, x[k][w + V - 1] = y.w;
                }
            }
    };
#pragma unroll
    for (int k = 0; k < kMassKeys; ++k) {
        sum[k] = 0.f;
        old[k] = key0 + k * kMassThreads < n ? mass[bh * cap + key0 + k * kMassThreads] : 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) x[k][w] = 0.f;
    }
    load(0);
    for (int r = threadIdx.x; r < kQ8MaxRows + 8; r += kMassThreads) {
        st_s[r] = r < R ? a.stats[bh * R + r] : make_float2(0.f, 0.f);
        last_s[r] = e0 + r / a.group;
    }
    __syncthreads();
    for (int r = 0; r < R; r += W) {
        if (r > 0) load(r);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 st = st_s[r + w];
            const int last = last_s[r + w];
#pragma unroll
            for (int k = 0; k < kMassKeys; ++k)
                if (st.y != 0.f && key0 + k * kMassThreads <= last) sum[k] += q8_ex2(x[k][w] - st.x) * st.y;
        }
    }
    pdl_trigger();
#pragma unroll
    for (int k = 0; k < kMassKeys; ++k)
        if (key0 + k * kMassThreads < n) mass[bh * cap + key0 + k * kMassThreads] = old[k] + sum[k];
}

// Query rows a CTA: 16, or 8 where the rows come in an odd number of eights (at
// d = 64, where a block of 16 takes 1.5 times one of 8, up to three of them).
// 4 x 8 heads, 32768 entries, bf16 outputs, in eights and in sixteens: d 128 20 rows
// 127 and 150 us, 36 rows 207 and 219, 56 rows 287 and 287 (fp32 309 and 322); d 64
// 20 rows 80 and 81, 36 rows 127 and 117.
int row_block(int R, int d) {
    const int e = (R + 7) / 8;
    return e % 2 && (d == 128 || e <= 3) ? 8 : 16;
}

template <int D, int NT, bool PLO, bool PAIR>
cudaError_t launch_decode(const Q8AttnArgs& a, dim3 grid, cudaStream_t st) {
    const cudaError_t e = allow_smem_max_once<q8_decode_kernel<D, NT, PLO, PAIR>>();
    if (e != cudaSuccess) return e;
    return launch_pdl(q8_decode_kernel<D, NT, PLO, PAIR>, grid, dim3(kQdThreads), kQdSmem, st, a);
}
template <int D, bool PLO>
cudaError_t launch_decode_rows(const Q8AttnArgs& a, int R, dim3 grid, cudaStream_t st) {
    return R <= 4 ? launch_decode<D, 1, PLO, true>(a, grid, st)
                  : row_block(R, D) == 8 ? launch_decode<D, 1, PLO, false>(a, grid, st)
                                      : launch_decode<D, 2, PLO, false>(a, grid, st);
}

// Splits of the key axis.  Where the caller names no length: one wave of two
// CTAs an SM over (sequence, head, split), and at least 128 KB of codes a split
// when the capacity is full.  They depend on the batch, the heads and the
// capacity only, so a sequence's verify and decode calls share them.
int split_count(dkv_dims dims, int capacity, int split_keys) {
    if (split_keys > 0) return (int)(((long long)capacity + split_keys - 1) / split_keys);
    const int ctas = std::max(1, 2 * 148 / std::max(1, dims.batch * dims.n_kv));
    return (int)std::max(1ll, std::min<long long>(ctas, (long long)capacity * 2 * dims.d / kQdMinBytes));
}

size_t decode_work(dkv_dims dims, int R, int capacity, int split_keys, bool mass, Q8AttnArgs* a, Arena* ar) {
    const int rb = row_block(R, dims.d), n_rb = (R + rb - 1) / rb, ns = split_count(dims, capacity, split_keys);
    const size_t bh = (size_t)dims.batch * dims.n_kv;
    const size_t part = bh * n_rb * ns * rb * (dims.d + 4), s_ld = R <= 2 ? 2 : (size_t)(R + 3) / 4 * 4;
    if (a) {
        a->tickets = ar->take<unsigned>(kQ8Tickets);
        a->part = ar->take<float>(part);
        a->scores = mass ? ar->take<float>(bh * capacity * s_ld) : nullptr;
        a->stats = mass ? ar->take<float2>(bh * R) : nullptr;
        a->s_ld = (int)s_ld;
        a->n_rb = n_rb;
        a->n_splits = ns;
    }
    size_t b = kQ8Tickets * sizeof(unsigned) + align_up(part * sizeof(float), 256);
    if (mass) b += align_up(bh * capacity * s_ld * sizeof(float), 256) + align_up(bh * R * sizeof(float2), 256);
    return b + 1024;
}

}  // namespace

size_t attn_q8_work_upto(dkv_dims dims, int group, int max_T, int capacity, bool mass) {
    const int T1 = std::min(max_T, std::max(1, kQ8MaxRows / group));
    size_t w = dkv_q8_attn_work_bytes(dims, group, T1, capacity, 0, mass ? 1 : 0);
    // (rows of a prompt chunk count in blocks of 128 or 256: one T of each block count)
    for (long long R = kQ8MaxRows + 1; R <= (long long)max_T * group; R = (R + 127) / 128 * 128 + 1)
        w = std::max(w, attn_q8_prefill_work(dims, 1, (int)std::min(R, 1ll << 24), capacity));
    return w;
}
}  // namespace dkv

using namespace dkv;

extern "C" size_t dkv_q8_attn_work_bytes(dkv_dims dims, int group, int T, int capacity, int split_keys, int note_mass) {
    if (dims.batch < 1 || dims.n_kv < 1 || group < 1 || T < 1 || capacity < 1) return 0;
    const long long R = (long long)T * group;
    if (R > (1 << 24) || capacity > (1 << 30) || (split_keys > 0 && split_keys % 128)) return 0;
    if (R > kQ8MaxRows) return attn_q8_prefill_work(dims, group, T, capacity);
    return decode_work(dims, (int)R, capacity, split_keys, note_mass != 0, nullptr, nullptr);
}

extern "C" int dkv_q8_attn(const dkv_q8_cache* cache, dkv_dims dims, int layer, int group, int T, const float* q,
                           const int32_t* entry0, const int32_t* n_rows, void* out, int out_dtype, int split_keys,
                           float* mass, void* work, size_t work_bytes, void* stream) {
    Q8AttnArgs a{};
    DKV_TRY(q8_view("dkv_q8_attn", cache, dims, layer, &a.v));
    DKV_REQUIRE(q && entry0 && out, "dkv_q8_attn: arrays required");
    DKV_REQUIRE(group >= 1 && T >= 1 && (long long)T * group <= (1 << 24), "dkv_q8_attn: group %d, T %d", group, T);
    DKV_REQUIRE(out_dtype == DKV_F32 || out_dtype == DKV_BF16, "dkv_q8_attn: out dtype %d", out_dtype);
    DKV_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)work & 15) == 0,
                "dkv_q8_attn: q, out and work must be 16-byte aligned");
    const int R = T * group, cap = a.v.capacity();
    DKV_REQUIRE(split_keys <= 0 || split_keys % 128 == 0, "dkv_q8_attn: split_keys %d (a multiple of 128, or 0)",
                split_keys);
    DKV_UNSUPPORTED(!mass || R <= kQ8MaxRows, "dkv_q8_attn: the mass of %d query rows a head (at most %d)", R,
                    kQ8MaxRows);
    a.group = group;
    a.T = T;
    a.batch = dims.batch;
    a.q = q;
    a.entry0 = entry0;
    a.n_rows = n_rows;
    a.out = out;
    a.out_dtype = out_dtype;
    a.scale = 1.4426950408889634f / sqrtf((float)dims.d);
    a.err = device_error_word();
    DKV_REQUIRE(a.err, "dkv_q8_attn: device error word unavailable");
    cudaStream_t st = (cudaStream_t)stream;
    if (R > kQ8MaxRows) {
        // more rows (a prompt chunk): the tcgen05 kernel, which picks its own splits
        DKV_REQUIRE(work && work_bytes >= attn_q8_prefill_work(dims, group, T, cap),
                    "dkv_q8_attn: work buffer of %zu bytes is too small", work_bytes);
        return attn_q8_prefill(a, dims, work, work_bytes, st);
    }
    DKV_REQUIRE(work && work_bytes >= decode_work(dims, R, cap, split_keys, mass != nullptr, nullptr, nullptr),
                "dkv_q8_attn: work buffer of %zu bytes is too small", work_bytes);
    Arena ar(work, work_bytes);
    decode_work(dims, R, cap, split_keys, mass != nullptr, &a, &ar);
    DKV_REQUIRE(a.tickets && a.part && (!mass || (a.scores && a.stats)), "dkv_q8_attn: work buffer");
    const size_t n_tk = (size_t)dims.batch * dims.n_kv * a.n_rb;
    DKV_REQUIRE((a.n_splits == 1 || n_tk <= kQ8Tickets) && (size_t)dims.batch * a.n_rb <= 65535,
                "dkv_q8_attn: batch x heads x row blocks too large");
    const dim3 grid((unsigned)a.n_splits, (unsigned)dims.n_kv, (unsigned)(dims.batch * a.n_rb));
    ProfScope ps(DKV_PROF_ATTN_FULL, 0.0, st);
    cudaError_t e;
    const bool plo = out_dtype == DKV_F32;
    if (dims.d == 128)
        e = plo ? launch_decode_rows<128, true>(a, R, grid, st) : launch_decode_rows<128, false>(a, R, grid, st);
    else
        e = plo ? launch_decode_rows<64, true>(a, R, grid, st) : launch_decode_rows<64, false>(a, R, grid, st);
    DKV_CUDA(e);
    if (mass) {
        const dim3 mg((unsigned)((cap + kMassThreads * kMassKeys - 1) / (kMassThreads * kMassKeys)), (unsigned)dims.n_kv,
                      (unsigned)dims.batch);
        // (after more than one wave an early start takes SMs from the CTAs that are
        // still to come: 42 rows over 3 x 6 x 36337 entries 257 us, 242 us without)
        if ((size_t)grid.x * grid.y * grid.z <= 2 * 148)
            DKV_CUDA(a.s_ld == 2 ? launch_pdl(q8_mass_kernel<2>, mg, dim3(kMassThreads), 0, st, a, mass)
                                 : launch_pdl(q8_mass_kernel<8>, mg, dim3(kMassThreads), 0, st, a, mass));
        else if (a.s_ld == 2)
            q8_mass_kernel<2><<<mg, kMassThreads, 0, st>>>(a, mass);
        else
            q8_mass_kernel<8><<<mg, kMassThreads, 0, st>>>(a, mass);
        DKV_LAUNCHED();
    }
    return DKV_OK;
}
