// Attention over the 8-bit paged cache, up to 64 query rows a KV head (decode,
// verify), and the attention mass that eviction goes by.
//
// softmax(q K^T / sqrt(d)) V per row, row t of sequence b over entries
// 0 .. entry0[b] + t.  Memory-bound: 2 d bytes an entry and KV head, read once
// for all rows.  Keys are the rows of the tensor-core products (m16n8k16):
// S^T = K Q^T and O^T += V^T P^T, 8 query rows as columns, so that the few
// rows of a decode step waste little.  The cache's bytes are stored in operand
// order, so a lane's 16-byte shared-memory load is an operand after
// e4m3 -> f16, which is exact.
//
// Rounding: K and V enter exactly (block scales are powers of two: K's is
// multiplied into the fp32 scores, V's into the probabilities).  Queries are
// the sum of two f16 numbers (22 bits), probabilities too, so what is rounded
// is what fp32 arithmetic rounds; max, sum and outputs are fp32.
//
// One CTA per (key split, KV head, sequence x row block).  A producer warp
// streams 16 KB stages with bulk copies (one contiguous record of K and V per
// page and head) through a ring; 4 warps per row group take every fourth
// 16-token tile of a stage and keep (max, sum, O) of their own, merged in a
// fixed order.  Split boundaries are absolute key positions and a row's
// arithmetic does not depend on the other rows of the call, so a verify row
// equals the decode step at that entry bit for bit.
//
// The running max is raised lazily: only when a score exceeds it by more than
// 8 (log2 units), which keeps the common tile free of shuffles and rescaling;
// probabilities stay below 2^8 and O / sum is exact either way.
#include <algorithm>

#include "attention_q8.cuh"

namespace dkv {

namespace {

constexpr int kQdStage = 16384;        // bytes of a ring stage
constexpr int kQdKG = 4;               // key groups (warps a row group)
constexpr int kQdMaxSplit = 8192;      // keys a split may have (page ids and scales staged in shared memory)
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
DKV_DEV void mbar_arrive1(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}

// NT: tiles of 8 query rows a warp carries; RG: row groups of 4 warps.
template <int NT, int RG>
struct QdGeo {
    static constexpr int ROWS = 8 * NT * RG;           // query rows a CTA
    static constexpr int WARPS = kQdKG * RG;
    static constexpr int THREADS = 32 * (WARPS + 1);   // + the producer warp
    static constexpr int STAGES = RG > 1 ? 10 : 5;     // one CTA an SM, or two
    static constexpr int CTAS = RG > 1 ? 1 : 2;
    static constexpr size_t SMEM = (size_t)STAGES * kQdStage;
};

template <int D, int NT, int RG>
__global__ void __launch_bounds__(QdGeo<NT, RG>::THREADS, QdGeo<NT, RG>::CTAS) q8_decode_kernel(const __grid_constant__ Q8AttnArgs a) {
    using Geo = QdGeo<NT, RG>;
    constexpr int KEYS = kQdStage / (2 * D);           // keys a stage
    constexpr int TPW = KEYS / 16 / kQdKG;             // tiles a warp takes of a stage
    constexpr int KS = D / 16, PS = D + 2, RB = Geo::ROWS;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ __align__(8) uint64_t full_bar[Geo::STAGES], empty_bar[Geo::STAGES];
    __shared__ int32_t page_s[kQdMaxSplit / 16];
    __shared__ float2 scale_s[kQdMaxSplit / 16];
    __shared__ float ms[RB], ls[RB];
    __shared__ int failed;
    const Q8View& v = a.v;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < Geo::STAGES; ++i) {
            mbar_init(&full_bar[i], 1);
            mbar_init(&empty_bar[i], Geo::WARPS);
        }
        failed = 0;
        fence_async_shared();
    }
    pdl_trigger();
    pdl_wait();            // queries and the new entries come from earlier kernels

    const int s = blockIdx.x, h = blockIdx.y;
    const int b = blockIdx.z / a.n_rb, rb = blockIdx.z % a.n_rb;
    const int G = a.group, R_all = a.T * G;
    const int rbase = rb * RB, R = min(RB, R_all - rbase);
    const int n_tok = a.n_rows ? min(a.n_rows[b], a.T) : a.T;
    const int e0 = a.entry0[b];
    const int k0 = s * a.split;
    // the block's last token decides what is read
    const int t_last = min((rbase + R - 1) / G, n_tok - 1);
    const int n_keys = t_last >= rbase / G ? max(0, min(a.n_keys(b), e0 + t_last + 1)) : 0;
    const int kend = min(n_keys, k0 + a.split);
    const int psx = min(v.page, KEYS);                 // tokens of a page inside a stage
    const int n_pg = kend > k0 ? (kend - k0 + v.page - 1) >> v.page_shift : 0;
    if (s == 0 && h == 0 && rb == 0 && threadIdx.x == 0 && a.beyond(b)) atomicOr(a.err, kErrQ8Page);
    // page ids and scales of the split: a page with a bad id gets -1 and its keys are not seen
    for (int i = threadIdx.x; i < n_pg; i += Geo::THREADS) {
        const int pid = __ldg(v.row(b) + (k0 >> v.page_shift) + i);
        const bool ok = v.ok(pid);
        page_s[i] = ok ? pid : -1;
        scale_s[i] = ok ? *reinterpret_cast<const float2*>(v.scale + v.scale_at(pid, h, 0)) : make_float2(1.f, 1.f);
        if (!ok) atomicOr(a.err, kErrQ8Page);
    }
    __syncthreads();
    const int n_st = kend > k0 ? (kend - k0 + KEYS - 1) / KEYS : 0;

    float m[NT][2], l[NT][2];
    float o[NT][KS][4];
    int eo = kQ8ExpMin;                                // O is in units of 2^(eo - kQdBias)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int md = 0; md < KS; ++md) o[nt][md][0] = o[nt][md][1] = o[nt][md][2] = o[nt][md][3] = 0.f;
    }
    const int kg = warp % kQdKG, rg = warp / kQdKG;
    const int qr = lane >> 2, qc = lane & 3;

    if (warp == Geo::WARPS) {
        // ---------------- producer: lane j copies page j of a stage
        for (int it = 0; it < n_st; ++it) {
            const int slot = it % Geo::STAGES;
            if (it >= Geo::STAGES &&
                !__all_sync(0xffffffffu, mbar_wait(&empty_bar[slot], (uint32_t)((it / Geo::STAGES - 1) & 1), a.err))) {
                if (lane == 0) failed = 1;
                break;
            }
            const int t0 = k0 + it * KEYS;
            uint8_t* dst = ring + (size_t)slot * kQdStage;
            const int live = (min(kend - t0, KEYS) + psx - 1) / psx;     // page parts with a visible key
            const int pid = lane < live ? page_s[(t0 + lane * psx - k0) >> v.page_shift] : -1;
            const int parts = __popc(__ballot_sync(0xffffffffu, pid >= 0));
            if (lane == 0) mbar_expect_tx(&full_bar[slot], (uint32_t)(parts * psx * 2 * D));
            __syncwarp();
            if (pid >= 0) {
                const int in_page = (t0 + lane * psx) & (v.page - 1);
                const uint8_t* kp = v.side(pid, h, 0) + (size_t)in_page * D;
                uint8_t* to = dst + (size_t)lane * psx * 2 * D;
                if (psx == v.page) {
                    bulk_g2s(to, kp, (uint32_t)(psx * 2 * D), &full_bar[slot]);
                } else {
                    bulk_g2s(to, kp, (uint32_t)(psx * D), &full_bar[slot]);
                    bulk_g2s(to + psx * D, v.side(pid, h, 1) + (size_t)in_page * D, (uint32_t)(psx * D),
                             &full_bar[slot]);
                }
            }
            __syncwarp();
        }
    } else {
        // ---------------- queries: column qr of row tile nt, as hi + lo f16
        // numbers of q * log2 e / sqrt(d) * 2^-x, x the row's exponent
        uint32_t qh[NT][KS][2], ql[NT][KS][2];
        float cs[NT][2];                               // 2^x of this thread's score columns
        int lim[NT][2];                                // last visible entry of them
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = (rg * NT + nt) * 8 + qr;     // this lane's operand row
            const int gr = rbase + r;
            const float* qv = r < R ? a.q + (((size_t)b * a.T + gr / G) * v.n_kv * G + h * G + gr % G) * D : nullptr;
            float2 x[KS][2];
            float am = 0.f;
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    x[kk][u] = qv ? __ldg(reinterpret_cast<const float2*>(qv + kk * 16 + u * 8 + 2 * qc))
                                  : make_float2(0.f, 0.f);
                    x[kk][u].x *= a.scale;
                    x[kk][u].y *= a.scale;
                    am = fmaxf(am, fmaxf(fabsf(x[kk][u].x), fabsf(x[kk][u].y)));
                }
            am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
            am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
            // am = 1.m * 2^ex; an infinite row keeps its infinities
            const int ex = min(max((int)(__float_as_uint(am) >> 23) - 127, -100), 126);
            const float down = q8_pow2(-ex);
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float p = x[kk][u].x * down, q = x[kk][u].y * down;
                    qh[nt][kk][u] = pack_h2(p, q);
                    const float2 hi = unpack_h2(qh[nt][kk][u]);
                    ql[nt][kk][u] = pack_h2(p - hi.x, q - hi.y);
                }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                cs[nt][c] = __shfl_sync(0xffffffffu, q8_pow2(ex), (2 * qc + c) * 4);
                const int rc = (rg * NT + nt) * 8 + 2 * qc + c, t = (rbase + rc) / G;
                lim[nt][c] = rc < R && t < n_tok ? min(e0 + t, n_keys - 1) : -1;
            }
        }
        const int row0 = rbase + rg * NT * 8 + 2 * qc;     // row of score column (nt 0, c 0)
        float* sc_base = a.scores ? a.scores + (((size_t)b * v.n_kv + h) * v.capacity()) * a.s_ld : nullptr;

        for (int it = 0; it < n_st; ++it) {
            const int slot = it % Geo::STAGES, t0 = k0 + it * KEYS;
            const uint8_t* st = ring + (size_t)slot * kQdStage;
            if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[slot], (uint32_t)((it / Geo::STAGES) & 1), a.err))) {
                if (lane == 0) failed = 1;
                break;
            }
#pragma unroll
            for (int tw = 0; tw < TPW; ++tw) {
                const int tile = tw * kQdKG + kg, key0 = t0 + tile * 16;
                if (key0 >= kend) break;
                const int part = tile * 16 / psx, inside = tile * 16 % psx;
                const uint8_t* kb = st + (size_t)part * psx * 2 * D + (size_t)inside * D + lane * 16;
                const uint8_t* vb = kb + psx * D;
                const int pi = (key0 - k0) >> v.page_shift;
                const bool bad = page_s[pi] < 0;
                const float2 sc2 = scale_s[pi];
                // ---- S^T: keys qr (+8), columns 2qc, 2qc + 1 of each row tile
                float sh[NT][4], sl[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sh[nt][e] = sl[nt][e] = 0.f;
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const uint4 w = *reinterpret_cast<const uint4*>(kb + j * 512);
                    uint32_t a0[4], a1[4];
                    q8_decode4(w.x, a0[0], a0[2]);
                    q8_decode4(w.y, a0[1], a0[3]);
                    q8_decode4(w.z, a1[0], a1[2]);
                    q8_decode4(w.w, a1[1], a1[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_f16_16816(sh[nt], a0, qh[nt][2 * j][0], qh[nt][2 * j][1]);
                        mma_f16_16816(sl[nt], a0, ql[nt][2 * j][0], ql[nt][2 * j][1]);
                        mma_f16_16816(sh[nt], a1, qh[nt][2 * j + 1][0], qh[nt][2 * j + 1][1]);
                        mma_f16_16816(sl[nt], a1, ql[nt][2 * j + 1][0], ql[nt][2 * j + 1][1]);
                    }
                }
                const int ka = key0 + qr, kb2 = ka + 8;
                bool grow = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float f = cs[nt][c] * sc2.x;
                        const int last = bad ? -1 : lim[nt][c];
                        const float x = ka <= last ? (sh[nt][c] + sl[nt][c]) * f : -INFINITY;
                        const float y = kb2 <= last ? (sh[nt][c + 2] + sl[nt][c + 2]) * f : -INFINITY;
                        sh[nt][c] = x;
                        sh[nt][c + 2] = y;
                        grow = grow || fmaxf(x, y) > m[nt][c] + kQdLazy;
                    }
                if (sc_base) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const int r = row0 + nt * 8;
                        if (r < a.s_ld && r - rbase < RB) {
                            if (ka < kend)
                                *reinterpret_cast<float2*>(sc_base + (size_t)ka * a.s_ld + r) =
                                    make_float2(sh[nt][0], sh[nt][1]);
                            if (kb2 < kend)
                                *reinterpret_cast<float2*>(sc_base + (size_t)kb2 * a.s_ld + r) =
                                    make_float2(sh[nt][2], sh[nt][3]);
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
                            float t = fmaxf(sh[nt][c], sh[nt][c + 2]);
#pragma unroll
                            for (int off = 4; off < 32; off <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, off));
                            const bool up = t > m[nt][c] + kQdLazy;
                            al[c] = up ? q8_ex2(m[nt][c] - t) : 1.f;
                            if (up) m[nt][c] = t;
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
                const int ev = q8_scale_exp(sc2.y);
                if (ev > eo) {                         // (uniform) larger V values: O to their units
                    const float dn = q8_pow2(max(eo - ev, -126));
                    eo = ev;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int md = 0; md < KS; ++md)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[nt][md][e] *= dn;
                }
                const float vf = q8_pow2(max(ev - eo + kQdBias, -126));
                uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        p[e] = sh[nt][e] == -INFINITY ? 0.f : q8_ex2(sh[nt][e] - m[nt][e & 1]);
                        if (e >= 2) l[nt][e & 1] += p[e - 2] + p[e];
                        p[e] = p[e];
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float x = p[2 * u] * vf, y = p[2 * u + 1] * vf;
                        const uint32_t hi = pack_h2(x, y);
                        const float2 hf = unpack_h2(hi);
                        ph[nt][u] = movm_trans(hi);
                        pl[nt][u] = movm_trans(pack_h2(x - hf.x, y - hf.y));
                    }
                }
                // bytes of keys that are not there (past the end, bad page) as zeros:
                // their probability is 0, but 0 x NaN would not be
                uint32_t vm = 0xffffffffu;
                if (key0 + 16 > kend || bad) {
                    vm = 0u;
                    const int ke = bad ? 0 : kend - key0;
                    if (2 * qc < ke) vm |= 0xffu;
                    if (2 * qc + 1 < ke) vm |= 0xff00u;
                    if (2 * qc + 8 < ke) vm |= 0xff0000u;
                    if (2 * qc + 9 < ke) vm |= 0xff000000u;
                }
#pragma unroll
                for (int j = 0; j < D / 32; ++j) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vb + j * 512);
                    uint32_t a0[4], a1[4];
                    q8_decode4(w.x & vm, a0[0], a0[2]);
                    q8_decode4(w.y & vm, a0[1], a0[3]);
                    q8_decode4(w.z & vm, a1[0], a1[2]);
                    q8_decode4(w.w & vm, a1[1], a1[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_f16_16816(o[nt][2 * j], a0, ph[nt][0], ph[nt][1]);
                        mma_f16_16816(o[nt][2 * j + 1], a1, ph[nt][0], ph[nt][1]);
                        mma_f16_16816(o[nt][2 * j], a0, pl[nt][0], pl[nt][1]);
                        mma_f16_16816(o[nt][2 * j + 1], a1, pl[nt][0], pl[nt][1]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive1(&empty_bar[slot]);
        }
    }
    __syncthreads();
    if (failed) {
        // a wait ran out (error word 0x80): wait, bounded, for the copies still
        // in flight before the ring is reused; the split counts as empty
        if (threadIdx.x == 0)
            for (int it = max(0, n_st - Geo::STAGES); it < n_st; ++it)
                mbar_wait(&full_bar[it % Geo::STAGES], (uint32_t)((it / Geo::STAGES) & 1), nullptr);
        __syncthreads();
    }

    // ---- the key groups' (max, sum, O) of every row to the drained ring
    float* mrg = reinterpret_cast<float*>(ring);           // [KG][RB][D + 2]
    if (warp < Geo::WARPS) {
        const float un = q8_pow2(eo) * q8_pow2(-kQdBias);  // (eo - bias may pass the smallest exponent)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float ll = l[nt][c];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) ll += __shfl_xor_sync(0xffffffffu, ll, off);
                // a row with NaN scores has no max: give it one, so that its NaN sum is merged
                const float mm = ll != ll && m[nt][c] == -INFINITY ? 0.f : m[nt][c];
                float* to = mrg + ((size_t)kg * RB + (rg * NT + nt) * 8 + 2 * qc + c) * PS;
                if (qr == 0) {
                    to[0] = mm;
                    to[1] = ll;
                }
#pragma unroll
                for (int md = 0; md < KS; ++md) {
                    to[2 + 16 * md + qr] = o[nt][md][c] * un;
                    to[2 + 16 * md + qr + 8] = o[nt][md][c + 2] * un;
                }
            }
    }
    __syncthreads();
    const size_t bhr = ((size_t)b * v.n_kv + h) * a.n_rb + rb;
    const bool alone = a.n_splits == 1;
    float* mypart = alone ? nullptr : a.part + (bhr * a.n_splits + s) * (size_t)RB * PS;
    // group weights first (in place over the maxima), then the sums
    for (int r = threadIdx.x; r < R; r += Geo::THREADS) {
        float M = -INFINITY, L = 0.f, w[kQdKG];
#pragma unroll
        for (int g = 0; g < kQdKG; ++g) M = fmaxf(M, mrg[((size_t)g * RB + r) * PS]);
#pragma unroll
        for (int g = 0; g < kQdKG; ++g) {
            const float mg = mrg[((size_t)g * RB + r) * PS];
            w[g] = mg == -INFINITY ? 0.f : q8_ex2(mg - M);
            if (w[g] != 0.f) L += mrg[((size_t)g * RB + r) * PS + 1] * w[g];
            mrg[((size_t)g * RB + r) * PS] = w[g];
        }
        if (failed) M = -INFINITY, L = 0.f;
        ms[r] = M;
        ls[r] = L;
        if (!alone) {
            mypart[(size_t)r * PS] = M;
            mypart[(size_t)r * PS + 1] = L;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * (D / 2); i += Geo::THREADS) {
        const int r = i / (D / 2), e = i % (D / 2) * 2;
        float x0 = 0.f, x1 = 0.f;
#pragma unroll
        for (int g = 0; g < kQdKG; ++g) {
            const float* at = mrg + ((size_t)g * RB + r) * PS;
            const float w = at[0];
            if (w != 0.f) {
                const float2 y = *reinterpret_cast<const float2*>(at + 2 + e);
                x0 += y.x * w;
                x1 += y.y * w;
            }
        }
        if (alone) {
            const float L = ls[r];
            q8_store2<D>(a, b, h, rbase + r, n_tok, e, L == 0.f ? 0.f : x0 / L, L == 0.f ? 0.f : x1 / L);
        } else {
            *reinterpret_cast<float2*>(mypart + (size_t)r * PS + 2 + e) = make_float2(x0, x1);
        }
    }
    if (!alone && !q8_merge_splits<D, RB>(a, bhr, b, h, rbase, R, n_tok, mrg, Geo::SMEM, ms, ls)) return;
    if (a.stats)
        for (int r = threadIdx.x; r < R; r += Geo::THREADS)
            a.stats[((size_t)b * v.n_kv + h) * R_all + rbase + r] =
                make_float2(ms[r], ls[r] == 0.f ? 0.f : 1.f / ls[r]);
}

// mass[b][h][j] += sum over the call's rows of p_j: the scores of the pass
// above under the merged (max, sum), rows in order (no atomics).
constexpr int kMassThreads = 256;
__global__ void __launch_bounds__(kMassThreads) q8_mass_kernel(Q8AttnArgs a, float* mass) {
    __shared__ float2 st_s[kQ8MaxRows];
    pdl_trigger();
    pdl_wait();
    const int h = blockIdx.y, b = blockIdx.z, R = a.T * a.group;
    const int n = a.n_keys(b);
    if ((int)(blockIdx.x * kMassThreads) >= n) return;
    const size_t bh = (size_t)b * a.v.n_kv + h;
    for (int r = threadIdx.x; r < R; r += kMassThreads) st_s[r] = a.stats[bh * R + r];
    __syncthreads();
    const int key = blockIdx.x * kMassThreads + threadIdx.x;
    if (key >= n) return;
    const float* sc = a.scores + (bh * a.v.capacity() + key) * a.s_ld;
    // a row block's scores exist up to its last token's entry only
    float sum = 0.f;
    const int e0 = a.entry0[b];
    for (int r = 0; r < R; r += 2) {
        const float2 x = __ldcg(reinterpret_cast<const float2*>(sc + r));
        const float2 s0 = st_s[r], s1 = r + 1 < R ? st_s[r + 1] : make_float2(0.f, 0.f);
        if (s0.y != 0.f && key <= e0 + r / a.group) sum += q8_ex2(x.x - s0.x) * s0.y;
        if (s1.y != 0.f && key <= e0 + (r + 1) / a.group) sum += q8_ex2(x.y - s1.x) * s1.y;
    }
    mass[bh * a.v.capacity() + key] += sum;
}

template <int D, int NT, int RG>
cudaError_t launch_decode(const Q8AttnArgs& a, dim3 grid, cudaStream_t st) {
    using Geo = QdGeo<NT, RG>;
    static_assert(Geo::SMEM >= (size_t)kQdKG * Geo::ROWS * (D + 2) * sizeof(float), "the merge fits the ring");
    const cudaError_t e = allow_smem_max_once<q8_decode_kernel<D, NT, RG>>();
    if (e != cudaSuccess) return e;
    return launch_pdl(q8_decode_kernel<D, NT, RG>, grid, dim3(Geo::THREADS), Geo::SMEM, st, a);
}

// Query rows a CTA: 8, 16 or 32.
int row_block(int R) { return R <= 8 ? 8 : R <= 16 ? 16 : 32; }

// Keys per split (a multiple of 128) where the caller names none: one wave of
// two CTAs an SM over (sequence, head, split), from 256 keys up to the staged
// limit.  It depends on the batch, the heads and the capacity only, so a
// sequence's verify and decode calls share it.
int default_split(int batch, int n_kv, int capacity) {
    const int ctas = std::max(1, 2 * 148 / std::max(1, batch * n_kv));
    const int keys = (int)(((long long)capacity + ctas - 1) / ctas);
    return std::min(std::max((keys + 127) / 128 * 128, 256), kQdMaxSplit);
}

int pick_split(int batch, int n_kv, int capacity, int split_keys) {
    return split_keys > 0 ? split_keys : default_split(batch, n_kv, capacity);
}

size_t decode_work(dkv_dims dims, int R, int capacity, int split, bool mass, Q8AttnArgs* a, Arena* ar) {
    const int rb = row_block(R), n_rb = (R + rb - 1) / rb, ns = std::max(1, (capacity + split - 1) / split);
    const size_t bh = (size_t)dims.batch * dims.n_kv;
    const size_t part = bh * n_rb * ns * rb * (dims.d + 2), s_ld = (size_t)(R + 1) / 2 * 2;
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
}  // namespace dkv

using namespace dkv;

extern "C" size_t dkv_q8_attn_work_bytes(dkv_dims dims, int group, int T, int capacity, int split_keys, int note_mass) {
    if (dims.batch < 1 || dims.n_kv < 1 || group < 1 || T < 1 || capacity < 1) return 0;
    const long long R = (long long)T * group;
    if (R > (1 << 24)) return 0;
    if (R > kQ8MaxRows) return attn_q8_prefill_work(dims, group, T, capacity);
    return decode_work(dims, (int)R, capacity, pick_split(dims.batch, dims.n_kv, capacity, split_keys), note_mass != 0,
                       nullptr, nullptr);
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
    DKV_REQUIRE(split_keys <= kQdMaxSplit && (split_keys <= 0 || split_keys % 128 == 0),
                "dkv_q8_attn: split_keys %d (a multiple of 128 up to %d, or 0)", split_keys, kQdMaxSplit);
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
    a.split = pick_split(dims.batch, dims.n_kv, cap, split_keys);
    DKV_REQUIRE(work && work_bytes >= decode_work(dims, R, cap, a.split, mass != nullptr, nullptr, nullptr),
                "dkv_q8_attn: work buffer of %zu bytes is too small", work_bytes);
    Arena ar(work, work_bytes);
    decode_work(dims, R, cap, a.split, mass != nullptr, &a, &ar);
    DKV_REQUIRE(a.tickets && a.part && (!mass || (a.scores && a.stats)), "dkv_q8_attn: work buffer");
    const size_t n_tk = (size_t)dims.batch * dims.n_kv * a.n_rb;
    DKV_REQUIRE(n_tk <= kQ8Tickets && (size_t)dims.batch * a.n_rb <= 65535,
                "dkv_q8_attn: batch x heads x row blocks too large");
    const dim3 grid((unsigned)a.n_splits, (unsigned)dims.n_kv, (unsigned)(dims.batch * a.n_rb));
    ProfScope ps(DKV_PROF_ATTN_FULL, 0.0, st);
    cudaError_t e;
    const int rb = row_block(R);
    if (dims.d == 128)
        e = rb == 8 ? launch_decode<128, 1, 1>(a, grid, st)
                    : rb == 16 ? launch_decode<128, 2, 1>(a, grid, st) : launch_decode<128, 2, 2>(a, grid, st);
    else
        e = rb == 8 ? launch_decode<64, 1, 1>(a, grid, st)
                    : rb == 16 ? launch_decode<64, 2, 1>(a, grid, st) : launch_decode<64, 2, 2>(a, grid, st);
    DKV_CUDA(e);
    if (mass)
        DKV_CUDA(launch_pdl(q8_mass_kernel, dim3((unsigned)((cap + kMassThreads - 1) / kMassThreads), (unsigned)dims.n_kv, (unsigned)dims.batch),
                            dim3(kMassThreads), 0, st, a, mass));
    return DKV_OK;
}
